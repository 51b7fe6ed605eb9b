"""block_norm / rms_norm / FusedBlockNorm on the CPU: values, gradients by differences, refusals."""
import pytest
import torch

from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
from smdistributed_modelparallel_amd.ops.layernorm import add_layer_norm, block_norm, layer_norm, rms_norm
from tests import block_norm_ref as ref


def _inputs(rms, post, gate, seed=0, b=2, s=3, d=6):
    g = torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g)

    shape = {"none": None, "scalar": (), "channel": (d,), "sample": (b, 1, d), "places": (1, s, d), "rows": (b, s, 1),
             "full": (b, s, d)}[gate]
    return {"x": r(b, s, d), "residual": r(b, s, d), "weight": r(d), "bias": None if rms else r(d),
            "post_weight": r(d) if post else None, "post_bias": r(d) if post and not rms else None,
            "gate": None if shape is None else r(*shape)}


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "sample", "places", "rows", "full"])
def test_values_and_gradients(rms, post, gate):
    t = _inputs(rms, post, gate)
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    y, s = block_norm(leaf["x"], leaf["residual"], leaf["weight"], leaf["bias"], leaf["post_weight"],
                      leaf["post_bias"], leaf["gate"], residual_scale=0.5, rms=rms)
    g = torch.Generator().manual_seed(9)
    dy, ds = torch.randn(y.shape, generator=g), torch.randn(y.shape, generator=g)
    want = ref.exact(t, 0.5, 1e-5, rms, dy, ds)
    torch.testing.assert_close(y.double(), want["y"], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(s.double(), want["s"], rtol=1e-5, atol=1e-6)
    names = [k for k, v in leaf.items() if v is not None]
    for k, got in zip(names, torch.autograd.grad([y, s], [leaf[k] for k in names], [dy, ds])):
        torch.testing.assert_close(got.double(), want["d" + k], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("rms", [False, True])
def test_reference_gradients_are_the_differences(rms):
    """The oracle of these tests against central differences in 64 bits."""
    t = {k: None if v is None else v.double() for k, v in _inputs(rms, True, "sample", seed=4).items()}
    g = torch.Generator().manual_seed(5)
    dy, ds = (torch.randn(2, 3, 6, generator=g, dtype=torch.float64) for _ in range(2))
    want = ref.exact(t, 0.7, 1e-5, rms, dy, ds)
    for k, v in t.items():
        if v is None:
            continue
        for i in (0, v.numel() - 1):
            side = []
            for h in (1e-6, -1e-6):
                u = dict(t, **{k: v.clone()})
                u[k].view(-1)[i] += h
                out = ref.exact(u, 0.7, 1e-5, rms)
                side.append(float((out["y"] * dy).sum() + (out["s"] * ds).sum()))
            assert abs((side[0] - side[1]) / 2e-6 - float(want["d" + k].view(-1)[i])) < 1e-6


def test_plain_forms_are_the_existing_operators():
    t = _inputs(False, False, "none")
    y, s = block_norm(t["x"], t["residual"], t["weight"], t["bias"])
    ry, rs = add_layer_norm(t["x"], t["residual"], t["weight"], t["bias"])
    torch.testing.assert_close(y, ry)
    assert torch.equal(s, rs)
    u = t["x"] - t["x"].mean(-1, keepdim=True)
    torch.testing.assert_close(rms_norm(u, t["weight"]), layer_norm(u, t["weight"], None))


def test_module():
    from smdistributed_modelparallel_amd import nn as smp_nn

    m = smp_nn.FusedBlockNorm(6, gate=0.25, residual_scale=2.0)
    x, r = torch.randn(2, 3, 6), torch.randn(2, 3, 6)
    y, s = m(x, r)
    torch.testing.assert_close(s, r + 0.5 * layer_norm(x, None, None))
    torch.testing.assert_close(y, layer_norm(s, None, None))
    (y.sum() + s.sum()).backward()
    assert sorted(n for n, p in m.named_parameters() if p.grad is not None) == ["bias", "gate", "post_bias",
                                                                                "post_weight", "weight"]
    m = smp_nn.FusedBlockNorm(6, rms=True, post_norm=False)
    assert [n for n, _ in m.named_parameters()] == ["weight"]
    _, s = m(x, r, gate=torch.full((2, 1, 6), 3.0))
    torch.testing.assert_close(s, r + 3 * x)


def test_no_rows():
    w = torch.ones(4, requires_grad=True)
    y, s = block_norm(torch.empty(0, 3, 4), torch.empty(0, 3, 4), w)
    assert y.shape == s.shape == (0, 3, 4)


_X, _W = torch.zeros(2, 3, 8), torch.ones(8)


@pytest.mark.parametrize("args,kwargs", [
    ((_X, _X[:1], _W), {}),
    ((_X, _X.half(), _W), {}),
    ((_X.double(), _X.double(), _W.double()), {}),
    ((_X.long(), _X.long(), _W), {}),
    ((_X, _X, _W[:7]), {}),
    ((_X, _X, None), {}),
    ((_X, _X, _W.half()), {}),
    ((_X, _X, _W), {"bias": _W.half()}),
    ((_X, _X, _W), {"bias": _W[:4]}),
    ((_X, _X, _W), {"post_bias": _W}),
    ((_X, _X, _W), {"post_weight": _W.half()}),
    ((_X.half(), _X.half(), _W), {"post_weight": _W.half()}),
    ((_X, _X, _W), {"gate": _W[:7]}),
    ((_X, _X, _W), {"gate": _W.half()}),
    ((_X, _X, _W), {"gate": torch.ones(3, 1, 8)}),
    ((_X, _X, _W), {"gate": torch.ones(1, 2, 3, 8)}),
    ((_X, _X, _W), {"residual_scale": float("inf")}),
    ((_X, _X, _W), {"eps": -1e-5}),
    ((torch.zeros(1, 16385), torch.zeros(1, 16385), torch.ones(16385)), {}),
    ((torch.zeros(3, 0), torch.zeros(3, 0), torch.ones(0)), {}),
    ((torch.zeros(1).half().expand((1 << 30) + 1, 1), torch.zeros(1).half().expand((1 << 30) + 1, 1), torch.ones(1)), {}),
])
def test_refusals(args, kwargs):
    with pytest.raises(SMPInvalidArgumentError):
        block_norm(*args, **kwargs)


@pytest.mark.parametrize("args", [(_X, _W[:7]), (_X, _W.half()), (_X.long(), _W), (_X, _W, float("nan"))])
def test_rms_norm_refusals(args):
    with pytest.raises(SMPInvalidArgumentError):
        rms_norm(*args)
