"""The block-norm kernels against 64-bit arithmetic, held to the bounds of block_norm_ref.slack
and one rounding (half a step) into each output's type."""
import pytest
import torch

from tests import block_norm_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def within(name, got, exact, slack):
    dt = torch.finfo(got.dtype)
    bound = slack + dt.eps / 2 * (exact.abs() + slack) + dt.tiny * dt.eps
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), (
        f"{name}: {int((~(err <= bound)).sum())} of {err.numel()} values off, worst {float((err / bound).max())} bounds")


def inputs(shape, dtype, wdtype, rms, post, gate, seed=0, mean=0.3, gdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, s, d = shape

    def r(*n, dt=dtype, m=0.0, std=1.0):
        return (torch.randn(n, generator=g, device="cuda") * std + m).to(dt)

    gshape = {"none": None, "scalar": (), "channel": (d,), "sample": (b, 1, d), "places": (1, s, d),
              "rows": (b, s, 1), "full": (b, s, d)}[gate]
    return {"x": r(b, s, d, m=mean), "residual": r(b, s, d, m=-mean, std=2.0), "weight": r(d, dt=wdtype, m=1.0, std=0.2),
            "bias": None if rms else r(d, dt=wdtype), "post_weight": r(d, dt=wdtype, m=1.0, std=0.2) if post else None,
            "post_bias": r(d, dt=wdtype) if post and not rms else None,
            "gate": None if gshape is None else r(*gshape, dt=gdtype or dtype, m=0.5)}


def call(t, alpha, eps, rms):
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    return block_norm(t["x"], t["residual"], t["weight"], t["bias"], t["post_weight"], t["post_bias"], t["gate"], alpha,
                      eps, rms)


def check(shape, dtype, wdtype=None, rms=False, post=True, gate="none", alpha=0.5, eps=1e-5, use=("y", "s"), **kw):
    t = inputs(shape, dtype, wdtype or dtype, rms, post, gate, **kw)
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    y, s = call(leaf, alpha, eps, rms)
    assert y.shape == s.shape == torch.Size(shape) and y.dtype == s.dtype == dtype
    g = torch.Generator(device="cuda").manual_seed(11)
    dy, ds = ((torch.randn(shape, generator=g, device="cuda") * 0.5).to(dtype) if n in use else None for n in ("y", "s"))
    outs = [(o, d) for o, d in ((y, dy), (s, ds)) if d is not None]
    names = [k for k, v in leaf.items() if v is not None and (dy is not None or k not in ("weight", "bias"))]
    grads = torch.autograd.grad([o for o, _ in outs], [leaf[k] for k in names], [d for _, d in outs])
    want, slack = ref.exact(t, alpha, eps, rms, dy, ds), ref.slack(t, alpha, eps, rms, dy, ds)
    within("y", y, want["y"], slack["y"])
    within("s", s, want["s"], slack["s"])
    for k, got in zip(names, grads):
        within("d" + k, got, want["d" + k], slack["d" + k])
    return [y, s, *grads]


SHAPES = [(1, 1, 1), (1, 1, 64), (2, 3, 7), (3, 5, 8), (1, 700, 40), (5, 41, 512), (2, 129, 1600), (7, 33, 1601),
          (3, 50, 2056), (2, 20, 4096), (2, 9, 6144), (3, 5, 6145), (1, 7, 8192), (1, 5, 8193), (2, 3, 12288), (1, 3, 16384),
          (9, 100, 65), (4, 11, 128), (3, 70, 129), (3, 50, 250), (2, 40, 257), (2, 17, 5000)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", DTYPES)
def test_sizes(shape, dtype):
    check(shape, dtype, gate="channel")
    check(shape, dtype, torch.float32, rms=True, gate="sample")


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "sample", "places", "rows", "full"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                          (torch.bfloat16, torch.float32)])
def test_forms(dtype, wdtype, rms, post, gate):
    check((6, 37, 200), dtype, wdtype, rms, post, gate, alpha=-0.75)


@pytest.mark.parametrize("use", [("y",), ("s",)])
@pytest.mark.parametrize("post", [False, True])
def test_one_output_used(use, post):
    check((3, 40, 136), torch.bfloat16, post=post, gate="channel", use=use)


@pytest.mark.parametrize("shape,gate", [((3000, 3, 24), "sample"), ((30, 300, 24), "full"), ((600, 40, 72), "sample"),
                                        ((2, 9000, 48), "sample"), ((1, 20000, 96), "channel"), ((9000, 2, 16), "none"),
                                        ((5, 300, 6152), "sample"), ((700, 2, 6200), "sample"), ((3, 90, 8192), "full"),
                                        ((40, 40, 9001), "channel")])
def test_many_rows(shape, gate):
    """More gate rows than units, fewer, and one for all rows; fp32 gate beside 16-bit rows."""
    check(shape, torch.bfloat16, torch.float32, gate=gate, gdtype=torch.float32)


def test_only_some_gradients():
    t = inputs((4, 9, 80), torch.float32, torch.float32, False, True, "channel")
    want = ref.exact(t, 1.0, 1e-5, False, torch.ones(4, 9, 80, device="cuda"), None)
    slack = ref.slack(t, 1.0, 1e-5, False, torch.ones(4, 9, 80, device="cuda"), None)
    for k in ("x", "residual", "gate", "post_bias", "weight"):
        leaf = dict(t, **{k: t[k].clone().requires_grad_()})
        y, _ = call(leaf, 1.0, 1e-5, False)
        (got,) = torch.autograd.grad(y.sum(), leaf[k])  # an expanded gradient
        within("d" + k, got, want["d" + k], slack["d" + k])


def test_layouts():
    """Transposed and sliced rows, gates and gradients, off 16 bytes and not."""
    t = inputs((5, 12, 104), torch.bfloat16, torch.bfloat16, False, True, "sample")
    u = dict(t)
    u["x"] = t["x"].transpose(0, 1).contiguous().transpose(0, 1)
    u["residual"] = torch.cat([t["residual"], t["residual"]], -1)[..., :104]
    u["gate"] = torch.cat([t["gate"], t["gate"]], 1)[:, :1]
    u["weight"] = torch.stack([t["weight"], t["weight"]], -1)[:, 0]
    big = torch.empty(104 * 60 + 1, device="cuda", dtype=torch.bfloat16)
    v = dict(t, x=big[1:].view(5, 12, 104).copy_(t["x"]))
    base = call(t, 0.5, 1e-5, False)
    for other in (u, v):
        assert all(torch.equal(a, b) for a, b in zip(base, call(other, 0.5, 1e-5, False)))
    leaf = {k: None if x is None else x.detach().requires_grad_() for k, x in u.items()}
    y, s = call(leaf, 0.5, 1e-5, False)
    dy = torch.randn(12, 104, 5, device="cuda").bfloat16().permute(2, 0, 1)
    names = [k for k, x in leaf.items() if x is not None]
    want, slack = ref.exact(t, 0.5, 1e-5, False, dy), ref.slack(t, 0.5, 1e-5, False, dy)
    for k, got in zip(names, torch.autograd.grad(y, [leaf[k] for k in names], dy)):
        within("d" + k, got, want["d" + k], slack["d" + k])


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_zero_and_infinite_rows(dtype, rms):
    """Rows without deviation are finite; infinities and NaN stay in their rows."""
    t = inputs((1, 6, 48), dtype, dtype, rms, True, "none")
    for k in ("x", "residual"):
        t[k][0, 0] = 0.0
        t[k][0, 1] = 3.0
    t["x"][0, 2, 5] = float("inf")
    t["x"][0, 3, 47] = float("nan")
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    y, s = call(leaf, 1.0, 1e-5, rms)
    dx, = torch.autograd.grad(y, leaf["x"], torch.ones_like(y))
    # a zero row of x and residual: both norms multiply the gradient by 1e-5 ** -0.5 = 316, together
    # 1e5, which fp16 (65504 at most) cannot hold: infinite exactly where the definition is too large
    want = ref.exact({k: v if v is None else v[:, [0, 1, 4, 5]] for k, v in t.items() if v is None or v.dim() == 3}
                     | {k: v for k, v in t.items() if v is not None and v.dim() == 1}, 1.0, 1e-5, rms,
                     torch.ones_like(y[:, [0, 1, 4, 5]]))["dx"]
    over = want.abs() > torch.finfo(dtype).max * (1 + 2.0 ** -12)
    assert torch.equal(dx[:, [0, 1, 4, 5]].isinf(), over) and not dx[0, [2, 3]].isfinite().all(-1).any()
    for o in (y, s):
        assert o[0, [0, 1, 4, 5]].isfinite().all() and not o[0, [2, 3]].isfinite().all(-1).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 1601, 4096])
def test_rms_norm(dtype, d):
    from smdistributed_modelparallel_amd.ops.layernorm import rms_norm

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 50, d, generator=g, device="cuda").to(dtype).requires_grad_()
    w = torch.randn(d, generator=g, device="cuda").requires_grad_()
    dy = torch.randn(3, 50, d, generator=g, device="cuda").to(dtype)
    y = rms_norm(x, w, 1e-6)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    # the definition with nothing added: block_norm of a zero block
    t = {"x": torch.zeros_like(x), "residual": x, "weight": w}
    want, slack = ref.exact(t, 1.0, 1e-6, True, dy), ref.slack(t, 1.0, 1e-6, True, dy)
    within("y", y, want["y"], slack["y"])
    within("dx", dx, want["dresidual"], slack["dresidual"])
    within("dw", dw, want["dweight"], slack["dweight"])


def test_bound_gradients_and_a_shared_parameter():
    """Parameters bound to the flat gradient buffer are added to in place; one that serves as both
    weights gets the sum."""
    t = inputs((3, 70, 160), torch.bfloat16, torch.bfloat16, False, True, "channel")
    names = ("weight", "bias", "post_bias", "gate")
    p = {k: torch.nn.Parameter(t[k].clone()) for k in names}
    start = {}
    for k, q in p.items():
        q.grad = torch.randn_like(q)
        q._smp_fused_grad = True
        start[k] = q.grad.clone()
    x, r = t["x"].requires_grad_(), t["residual"].requires_grad_()
    u = {"x": x, "residual": r, "post_weight": p["weight"], **p}
    y, s = call(u, 0.5, 1e-5, False)
    dy, ds = torch.randn_like(y), torch.randn_like(s)
    torch.autograd.backward([y, s], [dy, ds])
    want, slack = ref.exact(u, 0.5, 1e-5, False, dy, ds), ref.slack(u, 0.5, 1e-5, False, dy, ds)
    eps = torch.finfo(torch.bfloat16).eps
    for k in names:
        exact, room = want["d" + k], slack["d" + k]
        if k == "weight":  # two contributions, the second rounded by itself and added to the bound gradient
            other = want["dpost_weight"]
            room = room + slack["dpost_weight"] + eps / 2 * (exact.abs() + other.abs() + start[k].double().abs() + room)
            exact = exact + other
        within(k, p[k].grad, exact + start[k].double(), room + ref.FEW * start[k].double().abs())


def test_second_derivatives_are_refused():
    t = inputs((2, 3, 16), torch.float32, torch.float32, False, True, "none")
    x = t["x"].requires_grad_()
    y, _ = call(t, 1.0, 1e-5, False)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()


def test_no_rows_on_the_gpu():
    w = torch.ones(8, device="cuda", requires_grad=True)
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y, s = call({"x": x, "residual": x, "weight": w, "bias": None, "post_weight": w, "post_bias": None, "gate": None},
                1.0, 1e-5, True)
    dx, dw = torch.autograd.grad((y + s).sum(), [x, w])
    assert y.shape == dx.shape == (0, 8) and torch.equal(dw, torch.zeros_like(w))


def test_same_bits_and_graph_replays():
    t = inputs((4, 300, 328), torch.bfloat16, torch.float32, False, True, "sample")
    leaf = {k: None if v is None else v.requires_grad_() for k, v in t.items()}
    dy, ds = (torch.randn(4, 300, 328, device="cuda").bfloat16() for _ in range(2))
    names = [k for k, v in leaf.items() if v is not None]

    def step():
        y, s = call(leaf, 0.5, 1e-5, False)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], [leaf[k] for k in names], [dy, ds])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        with torch.no_grad():
            leaf["x"].normal_()
            leaf["gate"].normal_()
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step()):
            assert torch.equal(a, e)


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are right, and the weight gradients see all rows."""
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    rows, d = 270_000, 8192
    x = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
    r = torch.zeros_like(x)
    t = inputs((1, 2, d), torch.bfloat16, torch.float32, False, True, "channel")
    x[-2:], r[-2:] = t["x"][0], t["residual"][0]
    names = ("weight", "bias", "post_weight", "post_bias", "gate")
    leaf = {k: t[k].clone().requires_grad_() for k in names}
    x.requires_grad_()
    y, s = block_norm(x, r, leaf["weight"], leaf["bias"], leaf["post_weight"], leaf["post_bias"], leaf["gate"], 0.5)
    dy = torch.zeros_like(y)
    dy[-2:] = torch.randn(2, d, device="cuda").bfloat16()
    grads = torch.autograd.grad(y, [x] + [leaf[k] for k in names], dy)
    want, slack = ref.exact(t, 0.5, 1e-5, False, dy[-2:].unsqueeze(0)), ref.slack(t, 0.5, 1e-5, False, dy[-2:].unsqueeze(0))
    within("y", y.detach()[-2:], want["y"][0], slack["y"][0])
    within("s", s.detach()[-2:], want["s"][0], slack["s"][0])
    within("dx", grads[0][-2:], want["dx"][0], slack["dx"][0])
    for k, g in zip(names, grads[1:]):  # rows without gradient add zeros
        within("d" + k, g, want["d" + k], slack["d" + k])


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_autocast_takes_the_residuals_type(device):
    from smdistributed_modelparallel_amd.nn import FusedBlockNorm

    torch.manual_seed(0)
    lin, norm = torch.nn.Linear(48, 48).to(device), FusedBlockNorm(48, gate=0.5).to(device)
    r = torch.randn(5, 48, device=device)
    with torch.autocast(device, dtype=torch.bfloat16):
        x = lin(r)
        y, s = norm(x, r)
    assert x.dtype == torch.bfloat16 and y.dtype == s.dtype == torch.float32
    y2, s2 = norm(x.float(), r)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    y.sum().backward()
    assert lin.weight.grad.isfinite().all()


def test_bound_gradients_stay_out_of_other_passes():
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    x = torch.randn(6, 40, device="cuda").requires_grad_()
    w = torch.randn(40, device="cuda").requires_grad_()
    (expect,) = torch.autograd.grad(block_norm(x, x, w)[0].sum(), w)
    w.grad, w._smp_fused_grad = torch.zeros_like(w), True
    slot = w.grad
    (dw,) = torch.autograd.grad(block_norm(x, x, w)[0].sum(), w)
    assert torch.equal(dw, expect) and slot.eq(0).all()
    block_norm(x, x, w)[0].sum().backward(inputs=[w])
    assert w.grad is slot and torch.equal(slot, expect)


def test_capture_beside_an_eager_graph_is_refused():
    """Autograd would take the gradient on the default stream, which a capture cannot include."""
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    x, r = (torch.randn(9, 32, device="cuda") for _ in range(2))
    w = torch.randn(32, device="cuda").requires_grad_()
    dy = torch.randn(9, 32, device="cuda")
    eager, _ = block_norm(x, r, w)
    (expect,) = torch.autograd.grad(eager, w, dy, retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = block_norm(x, r, w)
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(y, w, dy)
    assert torch.equal(torch.autograd.grad(eager, w, dy)[0], expect)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "scalar", "channel", "sample", "places", "rows", "full"])
@pytest.mark.parametrize("shape", [(0, 3, 8), (2, 0, 8), (0, 0, 8), (0, 3, 7000)])
def test_no_rows_with_a_gate(shape, gate, post):
    t = inputs(shape, torch.bfloat16, torch.float32, False, post, gate, gdtype=torch.float32)
    leaf = {k: None if v is None else v.clone().requires_grad_() for k, v in t.items()}
    with torch.no_grad():
        assert all(o.shape == shape for o in call(leaf, 0.5, 1e-5, False))
    y, s = call(leaf, 0.5, 1e-5, False)
    assert y.shape == s.shape == shape and y.dtype == s.dtype == torch.bfloat16
    names = [k for k, v in leaf.items() if v is not None]
    for k, g in zip(names, torch.autograd.grad([y, s], [leaf[k] for k in names], [torch.empty_like(y)] * 2)):
        assert g.shape == leaf[k].shape and g.dtype == leaf[k].dtype and not g.any(), k


def test_no_rows_of_a_module_with_a_gate():
    from smdistributed_modelparallel_amd.nn import FusedBlockNorm

    m = FusedBlockNorm(24, gate=0.5).cuda()
    for p in m.parameters():
        p.grad, p._smp_fused_grad = torch.ones_like(p), True
    x = torch.empty(0, 5, 24, device="cuda", requires_grad=True)
    y, s = m(x, x)
    (y.sum() + s.sum()).backward()
    assert x.grad.shape == x.shape and all(p.grad.eq(1).all() for p in m.parameters())


def test_one_row_of_a_flat_gate():
    """Rows without leading dimensions."""
    check((1, 1, 40), torch.float32, gate="channel")
    t = {k: None if v is None else v.view(40) for k, v in
         inputs((1, 1, 40), torch.float32, torch.float32, False, True, "full").items()}
    y, s = call(t, 0.5, 1e-5, False)
    want, slack = ref.exact(t, 0.5, 1e-5, False), ref.slack(t, 0.5, 1e-5, False)
    within("y", y, want["y"], slack["y"])
    within("s", s, want["s"], slack["s"])


def test_hooks_of_bound_parameters_get_their_gradients():
    t = inputs((3, 50, 72), torch.float32, torch.float32, False, True, "channel")
    names = ("weight", "bias", "post_weight", "post_bias", "gate")
    u = {k: torch.nn.Parameter(v) if k in names else v for k, v in t.items()}
    dy, ds = (torch.randn(3, 50, 72, device="cuda") for _ in range(2))
    expect = dict(zip(names, torch.autograd.grad(call(u, 0.5, 1e-5, False), [u[k] for k in names], [dy, ds])))
    seen = {}
    for k in names:
        u[k].grad, u[k]._smp_fused_grad = torch.zeros_like(u[k]), True
        u[k].register_hook(lambda g, k=k: seen.update({k: g.clone()}) or 3 * g)
    torch.autograd.backward(call(u, 0.5, 1e-5, False), [dy, ds])
    for k in names:
        assert torch.equal(seen[k], expect[k]) and torch.equal(u[k].grad, 3 * expect[k]), k


@pytest.mark.parametrize("device", ["cpu", "cuda"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_keeps_a_fp32_gate(device, dtype):
    """Beside 16-bit rows the gate and its gradient have the same bits with and without autocast."""
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    g = torch.Generator().manual_seed(4)
    x, r = (torch.randn(4, 3, 48, generator=g).to(device, dtype) for _ in range(2))
    w, dy, ds = torch.randn(48, generator=g).to(device), *(torch.randn(4, 3, 48, generator=g).to(device, dtype) for _ in range(2))
    for shape in ((48,), (4, 1, 48), (4, 3, 48)):
        gate = torch.randn(shape, generator=g).to(device).requires_grad_()
        plain = block_norm(x, r, w, gate=gate)
        plain += torch.autograd.grad(plain, gate, [dy, ds])
        with torch.autocast(device, dtype=torch.bfloat16):
            cast = block_norm(x, r, w, gate=gate)
        cast += torch.autograd.grad(cast, gate, [dy, ds])
        assert cast[2].dtype == torch.float32
        assert all(torch.equal(a, b) for a, b in zip(plain, cast))


@pytest.mark.parametrize("rows,d", [((1 << 29) + 11, 1), ((1 << 25) + 5, 66), (700_000, 6145)])
def test_more_rows_than_one_launch_takes(rows, d):
    """A row's results have the same bits whatever rows the call has beside it."""
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    g = torch.Generator(device="cuda").manual_seed(5)
    w, pw = (torch.rand(d, generator=g, device="cuda") + 0.5 for _ in range(2))
    x = torch.empty(rows, d, device="cuda", dtype=torch.float16).normal_(generator=g)
    threads = 8 if d == 1 else 16 if d == 66 else 832
    most = (1 << 28) // threads  # rows of a launch
    places = sorted({0, rows - 40, *(k * most - 20 for k in range(1, rows // most + 1))})
    assert len(places) > 2
    x.requires_grad_()
    y, s = block_norm(x, x, w, post_weight=pw, rms=True)
    (dx,) = torch.autograd.grad(y, x, y.detach())
    for at in places:
        part = x.detach()[at:at + 40].clone().requires_grad_()
        py, ps = block_norm(part, part, w, post_weight=pw, rms=True)
        assert torch.equal(y[at:at + 40], py) and torch.equal(s[at:at + 40], ps)
        assert torch.equal(dx[at:at + 40], torch.autograd.grad(py, part, py.detach())[0])
