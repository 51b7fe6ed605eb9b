"""The gradient-norm kernels against 64-bit arithmetic.

Squares are summed in 64 bits, so the norm is off by its rounding to fp32 alone (2^-24, taken
twice for the 64-bit sums); a clipped gradient by the fp32 rounding of the factor and of the
product (2^-24 each) and by its rounding into its type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def norm64(ts, p):
    if p == math.inf:
        return max([float(t.double().abs().max()) for t in ts if t.numel()], default=0.0)
    return math.sqrt(sum(float(t.double().pow(2).sum()) for t in ts))


def within(got, exact):
    dt = torch.finfo(got.dtype)
    bound = (dt.eps / 2 + 3 * U32) * exact.abs() + dt.tiny * dt.eps
    assert bool(((got.double() - exact).abs() <= bound).all())


def factor(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


def make(sizes, dtypes, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LISTS = {"one": [1], "odd": [1, 7, 8, 9, 255, 2049, 16384, 16385, 0, 100003], "many": list(range(1, 700, 2)),
         "large": [30_000_001, 5, 4_000_000]}


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in DTYPES] + [DTYPES], ids=["f32", "f16", "bf16", "mixed"])
def test_norm_and_clip(name, p, dtypes):
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm

    ts = make(LISTS[name], dtypes)
    want = norm64(ts, p)
    assert float(grad_norm(ts, p)) == pytest.approx(want, rel=3 * U32)
    before = [t.clone() for t in ts]
    assert float(clip_grad_norm_(ts, 2 * want, p)) == pytest.approx(want, rel=3 * U32)
    assert all(torch.equal(t, b) for t, b in zip(ts, before))  # within the norm: untouched
    f = factor(want / 4, want / 9)
    out = [torch.full_like(t, 7.0, dtype=DTYPES[i % 3]) for i, t in enumerate(ts)]
    clip_grad_norm_(ts, want / 9, p, scale=0.25, out=out)
    assert all(torch.equal(t, b) for t, b in zip(ts, before))
    for b, o in zip(before, out):
        within(o, b.double() * (0.25 * f))
    clip_grad_norm_(ts, want / 9, p, scale=0.25)
    for b, t in zip(before, ts):
        within(t, b.double() * (0.25 * f))


def test_squares_that_leave_fp32():
    """Sums of squares far above and below fp32's range."""
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm

    for std in (1e30, 1e-30):
        ts = make([1000, 50000], [torch.float32, torch.bfloat16], std=std)
        want = norm64(ts, 2.0)
        assert float(grad_norm(ts)) == pytest.approx(want, rel=3 * U32)
        before = [t.clone() for t in ts]
        clip_grad_norm_(ts, want / 2)
        for b, t in zip(before, ts):
            within(t, b.double() * factor(want, want / 2))


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(p, dtype):
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm

    ts = make([70_000, 33], [dtype])
    ts[0][65_537] = -math.inf
    assert float(grad_norm(ts, p)) == math.inf
    clip_grad_norm_(ts, 1.0, p)  # multiplied by zero
    assert ts[0][65_537].isnan() and ts[0][:65_537].eq(0).all() and ts[1].eq(0).all()
    ts = make([70_000, 33], [dtype])
    ts[0][3], ts[1][32] = math.inf, math.nan
    assert math.isnan(float(grad_norm(ts, p)))
    clip_grad_norm_(ts, 1.0, p)
    assert all(t.isnan().all() for t in ts)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Starts off 16 bytes, transposed, sliced and expanded tensors."""
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm

    base = make([40_001], [dtype])[0]
    wide = make([64 * 50], [dtype], seed=2)[0].view(64, 50)
    ts = [base[1:], wide[:, :20], wide[:, 25:].t(), make([60], [dtype], seed=3)[0].view(3, 4, 5).permute(2, 0, 1)]
    want = norm64(ts, 2.0)
    assert float(grad_norm(ts)) == pytest.approx(want, rel=3 * U32)
    assert float(grad_norm([ts[0], torch.ones(1, device="cuda", dtype=dtype).expand(9, 9)])) == pytest.approx(
        math.hypot(norm64(ts[:1], 2.0), 9.0), rel=3 * U32)
    before, kept = [t.clone() for t in ts], wide[:, 20:25].clone()
    first = base[0].clone()
    clip_grad_norm_(ts, want / 3)
    for b, t in zip(before, ts):
        within(t, b.double() * factor(want, want / 3))
    assert torch.equal(wide[:, 20:25], kept) and base[0] == first
    out = torch.empty(20, 64, device="cuda").t()
    clip_grad_norm_([wide[:, :20]], math.inf, out=[out])
    assert torch.equal(out, wide[:, :20].float())


def test_shared_memory_is_refused():
    from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

    x = torch.ones(100, device="cuda")
    for grads, out in (([x, x], None), ([x[:60], x[50:]], None), ([x[:50], x[50:]], [x[50:], x[:50]]),
                       ([x[:50].bfloat16()], [x[:50]])):
        if out is not None and grads[0].dtype == torch.bfloat16:
            clip_grad_norm_(grads, math.inf, out=out)
            continue
        with pytest.raises(SMPInvalidArgumentError):
            clip_grad_norm_(grads, 0.1, out=out)
    with pytest.raises(SMPInvalidArgumentError):
        clip_grad_norm_([x, torch.ones(3)], 1.0)
    assert x.eq(1).all()


def test_one_memory_as_two_types_is_refused():
    from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

    for device in ("cpu", "cuda"):
        x = torch.ones(100, device=device, dtype=torch.float16)
        with pytest.raises(SMPInvalidArgumentError):
            clip_grad_norm_([x], 100.0, out=[x.view(torch.bfloat16)])
        assert x.eq(1).all()


def test_parameters_of_a_model():
    from smdistributed_modelparallel_amd.optimizers import clip_grad_norm_

    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(50, 70), torch.nn.LayerNorm(70), torch.nn.Linear(70, 3)).cuda()
    m(torch.randn(9, 50, device="cuda")).pow(2).sum().backward()
    grads = [q.grad.clone() for q in m.parameters()]
    want = norm64(grads, 2.0)
    assert float(clip_grad_norm_(m.parameters(), want / 2)) == pytest.approx(want, rel=3 * U32)
    for q, g in zip(m.parameters(), grads):
        within(q.grad, g.double() * factor(want, want / 2))


def test_same_bits_and_graph_replays():
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

    ts = make([3_000_000] + list(range(1, 300)), DTYPES)
    out = [torch.empty_like(t, dtype=torch.float32) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_grad_norm_(ts, 3.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(ts, 3.0, out=out)
    for k in range(3):
        for t in ts:
            t.normal_(std=10.0 ** -k)
        graph.replay()
        torch.cuda.synchronize()
        got = [norm.clone()] + [o.clone() for o in out]
        eager = [clip_grad_norm_(ts, 3.0, out=out)] + out
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_inference_tensors():
    """They have no versions to count."""
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

    with torch.inference_mode():
        x = torch.ones(16, device="cuda")
        assert float(clip_grad_norm_([x], 2.0)) == 4.0
    assert float(clip_grad_norm_([x], 1.0)) == pytest.approx(2.0, rel=1e-6)
    assert float(x.sum()) == pytest.approx(4.0, rel=1e-6)
