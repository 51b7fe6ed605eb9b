"""Worker (pp=2, CPU): ``clip_master_grads`` with the largest-value norm over the pipeline's stages."""
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
    net, ref = Net(), Net()
    ref.load_state_dict(net.state_dict())
    smp.set_partition(net.b, 1)
    model = smp.DistributedModel(net)
    opt = smp.DistributedOptimizer(torch.optim.SGD(model.parameters(), lr=0.5))
    ref_opt = torch.optim.SGD(ref.parameters(), lr=0.5)

    @smp.step
    def train(model, x):
        loss = model(x)
        model.backward(loss)
        return loss

    for norm_type in (math.inf, 2):
        x = torch.randn(8, 6, generator=torch.Generator().manual_seed(1))
        opt.zero_grad()
        train(model, x)
        ref_opt.zero_grad()
        ref(x).backward()
        norm = opt.clip_master_grads(1e-3, norm_type)
        want = torch.nn.utils.clip_grad_norm_(ref.parameters(), 1e-3, norm_type)
        assert abs(float(norm) - float(want)) <= 1e-5 * float(want), (norm_type, norm, want)
        opt.step()
        ref_opt.step()
        full = dict(ref.named_parameters())
        for n, p in model.local_named_parameters():
            assert torch.allclose(p, full[n], rtol=1e-5, atol=1e-7), n
    # a NaN of one stage reaches all of them
    for bad in range(2):
        opt.zero_grad()
        train(model, x)
        if smp.pp_rank() == bad:
            next(p for _, p in model.local_named_parameters()).grad[0] = math.nan
        assert math.isnan(float(opt.clip_master_grads(1.0, math.inf))), bad
        opt._clip_coef = None
    try:
        opt.clip_master_grads(1.0, 1)
    except ValueError:
        print(f"rank {smp.rank()} OK clip", flush=True)
    smp.barrier()


if __name__ == "__main__":
    main()
