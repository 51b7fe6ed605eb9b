"""Worker (pp=2, CPU): ``clip_master_grads`` and the step of a model in fp64."""
import math

import torch
import torch.nn as nn

import smdistributed_modelparallel_amd.torch as smp


class Net(nn.Module):
    def __init__(self):
        super().__init__()
        self.a = nn.Linear(6, 8)
        self.b = nn.Linear(8, 1)

    def forward(self, x):
        return self.b(torch.tanh(self.a(x))).pow(2).mean()


def main():
    torch.manual_seed(0)
    smp.init({"pipeline_parallel_degree": 2, "microbatches": 1, "auto_partition": False, "default_partition": 0})
    net, ref = Net().double(), Net().double()
    ref.load_state_dict(net.state_dict())
    smp.set_partition(net.b, 1)
    model = smp.DistributedModel(net)
    opt = smp.DistributedOptimizer(torch.optim.SGD(model.parameters(), lr=0.5))

    @smp.step
    def train(model, x):
        loss = model(x)
        model.backward(loss)
        return loss

    x = torch.randn(8, 6, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    for norm_type in (2, math.inf):
        opt.zero_grad()
        train(model, x)
        ref.zero_grad()
        ref(x).backward()
        norm = opt.clip_master_grads(1e-3, norm_type)
        want = torch.nn.utils.clip_grad_norm_(ref.parameters(), 1e-3, norm_type)
        assert abs(float(norm) - float(want)) <= 2.0 ** -23 * float(want), (norm_type, norm, want)
        opt._clip_coef = None
    opt.clip_master_grads(1e-3)
    opt.step()
    print(f"rank {smp.rank()} OK clip", flush=True)
    smp.barrier()


if __name__ == "__main__":
    main()
