"""grad_norm / clip_grad_norm_ on the CPU: values, refusals and the clip of parameter lists."""
import math

import pytest
import torch

from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm, grad_power


def _grads(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(3, 5, generator=g), torch.randn(7, generator=g).bfloat16(), torch.empty(0),
            torch.randn(2, 2, 2, generator=g).half()]


def _norm64(ts, inf):
    flat = torch.cat([t.double().flatten() for t in ts])
    return float(flat.abs().max() if inf else flat.norm())


@pytest.mark.parametrize("p", [2.0, math.inf])
def test_norm_and_clip(p):
    ts = _grads()
    want = _norm64(ts, p == math.inf) * 0.25
    assert float(grad_norm(ts, p, 0.25)) == pytest.approx(want, rel=1e-6)
    before = [t.clone() for t in ts]
    assert float(clip_grad_norm_(ts, want / 2, p, 0.25)) == pytest.approx(want, rel=1e-6)
    for t, b in zip(ts, before):
        exact = b.double() * 0.125  # (1e-6 / norm below the tolerance)
        assert torch.allclose(t.double(), exact, rtol=torch.finfo(t.dtype).eps / 2 + 5e-6, atol=1e-30)


def test_clip_matches_torch_on_parameters():
    from smdistributed_modelparallel_amd.optimizers import clip_grad_norm_ as clip_params

    for max_norm in (0.5, 1e6, math.inf):
        a = [torch.nn.Parameter(torch.zeros(4, 3)), torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(2))]
        for q in a[:2]:
            q.grad = torch.randn(q.shape, generator=torch.Generator().manual_seed(q.numel()))
        b = [torch.nn.Parameter(q.detach().clone()) for q in a]
        for q, r in zip(a[:2], b):
            r.grad = q.grad.clone()
        n, m = clip_params(a, max_norm), torch.nn.utils.clip_grad_norm_(b, max_norm)
        assert torch.allclose(n, m)
        for q, r in zip(a[:2], b):
            assert torch.allclose(q.grad, r.grad)
        assert a[2].grad is None
    assert float(clip_params([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0


def test_out_in_another_type_leaves_the_gradients():
    ts = _grads(1)
    before, out = [t.clone() for t in ts], [torch.full(t.shape, 9.0) for t in ts]
    norm = clip_grad_norm_(ts, 1e9, scale=0.5, out=out)
    assert float(norm) == pytest.approx(_norm64(ts, False) * 0.5, rel=1e-6)
    for t, b, o in zip(ts, before, out):
        assert torch.equal(t, b) and torch.equal(o, t.float() * 0.5)


def test_no_tensors_and_no_elements():
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    assert float(grad_power([])) == 0.0
    empty = [torch.empty(0), torch.empty(3, 0)]
    assert float(clip_grad_norm_(empty, 1.0)) == 0.0 and float(grad_norm(empty, math.inf)) == 0.0


_T = torch.zeros(4)
_BIG = torch.zeros(12)


@pytest.mark.parametrize("args,kwargs", [
    (([_T], -1.0), {}),
    (([_T], math.nan), {}),
    (([_T], 1.0), {"norm_type": 1.0}),
    (([_T], 1.0), {"norm_type": 0}),
    (([_T], 1.0), {"scale": 0.0}),
    (([_T], 1.0), {"scale": math.inf}),
    (([_T.double()], 1.0), {}),
    (([_T.long()], 1.0), {}),
    (([_T.to_sparse()], 1.0), {}),
    (([None], 1.0), {}),
    (([_T], 1.0), {"out": []}),
    (([_T], 1.0), {"out": [_T[:3]]}),
    (([_T], 1.0), {"out": [_T.double()]}),
    (([torch.zeros(1).expand(4)], 1.0), {}),
    (([_T, _T], 1.0), {}),
    (([_BIG[:8], _BIG[4:]], 1.0), {}),
    (([_BIG[:6], _BIG[6:]], 1.0), {"out": [_BIG[6:], _BIG[:6]]}),
])
def test_refusals(args, kwargs):
    with pytest.raises(SMPInvalidArgumentError):
        clip_grad_norm_(*args, **kwargs)
    assert not _BIG.any()


def test_clip_master_grads_by_largest_value_over_stages():
    from tests.dist_utils import run_workers

    assert all("OK clip" in o for o in run_workers("clip_inf", 2, timeout=120))


def test_clip_master_grads_of_a_model_in_64_bits():
    from tests.dist_utils import run_workers

    assert all("OK clip" in o for o in run_workers("clip_fp64", 2, timeout=120))
