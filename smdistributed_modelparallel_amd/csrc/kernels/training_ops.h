// Bindings of the embedding, block-norm and gradient-norm operators (training_ops.cpp).
#pragma once
#include <torch/extension.h>

void register_training_ops(py::module_& m);
