"""The embedding kernels against plain 64-bit arithmetic.

Bounds: the forward adds two fp32 products' roundings (2^-24 of each term, twice) and one
rounding into the output type; a gradient that is the fp32 sum of k rows is off by at most
k * 2^-24 of the sum of their magnitudes, and rounded once.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, exact, slack):
    """|got - exact| <= slack + half a step of the result; subnormals of the type round absolutely."""
    dt = got.dtype
    bound = slack + half_step(dt) * (exact.abs() + slack) + torch.finfo(dt).tiny * torch.finfo(dt).eps
    err = (got.double() - exact).abs()
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} values off, worst {float((err - bound).max())}"


def table_grad(ids, dy, rows, scale, skip=None):
    """(gradient, slack) in 64 bits; ids outside the table and `skip` take none."""
    ids, dy = ids.reshape(-1), dy.double().reshape(-1, dy.shape[-1])
    keep = (ids >= 0) & (ids < rows)
    if skip is not None:
        keep &= ids != skip
    ids, dy = ids[keep], dy[keep]
    z = torch.zeros(rows, dy.shape[-1], dtype=torch.float64, device=dy.device)
    count = torch.bincount(ids, minlength=rows).double().unsqueeze(1)
    total, size = z.index_add(0, ids, dy) * scale, z.index_add(0, ids, dy.abs()) * abs(scale)
    return total, (count + 2) * U32 * size


def forward(ids, w, scale, start, pos, p):
    rows = w.shape[0]
    local = ids - (start or 0)
    out = w.double()[local.clamp(0, rows - 1)] * scale
    if start is not None:
        out = out * ((local >= 0) & (local < rows)).unsqueeze(-1)
    slack = out.abs()
    if p is not None:
        out, slack = out + p.double()[pos], slack + p.double()[pos].abs()
    return out, 2 * U32 * slack


def check(b, s, rows, dim, dtype, ids=None, scale=1.0, padding=None, start=None, positions="none", idt=torch.long,
          seed=0, strided=False):
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    g = torch.Generator(device="cuda").manual_seed(seed)
    vocab = rows if start is None else rows + 2 * start + 1
    if ids is None:
        ids = torch.randint(0, vocab, (b, s), generator=g, device="cuda")
    ids = ids.to(idt)
    w = torch.randn(rows, dim + 8 if strided else dim, generator=g, device="cuda").to(dtype)[:, :dim].requires_grad_()
    p = pos = None
    if positions != "none":
        p = torch.randn(s + 3, dim, generator=g, device="cuda").to(dtype).requires_grad_()
        pos = torch.arange(s, device="cuda").expand(b, s)
        if positions == "given":
            pos = pos + torch.randint(0, 4, (b, 1), generator=g, device="cuda")
    y = embedding(ids, w, padding_idx=padding, scale=scale, vocab_start=start,
                  position_ids=pos if positions == "given" else None, position_weight=p)
    assert y.shape == (b, s, dim) and y.dtype == dtype
    within(y, *forward(ids.long(), w.detach(), scale, start, pos, None if p is None else p.detach()))
    dy = torch.randn(b, s, dim, generator=g, device="cuda").to(dtype)
    grads = torch.autograd.grad(y, [w] if p is None else [w, p], dy)
    skip = None if padding is None else padding - (start or 0)
    within(grads[0], *table_grad(ids.long() - (start or 0), dy, rows, scale, skip))
    if p is not None:
        within(grads[1], *table_grad(pos, dy, s + 3, 1.0))
    return grads


DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,s,rows,dim", [(1, 1, 1, 1), (1, 1, 7, 64), (2, 3, 5, 1601), (3, 77, 300, 8), (5, 100, 50, 40),
                                          (4, 600, 1000, 264), (2, 1025, 70000, 24)])
def test_sizes(b, s, rows, dim, dtype):
    check(b, s, rows, dim, dtype)


@pytest.mark.parametrize("b,s,rows,dim", [(8, 5000, 60000, 16), (3, 16384, 1023, 9), (3, 16384, 1024, 8), (1, 700001, 3000, 8),
                                          (1, 600000, 1200000, 2), (2, 9000, 2, 3000), (64, 17, 40, 9000),
                                          (2, 300, 300000, 8), (1, 131072, 262144, 8), (1, 131073, 5000, 16)])
def test_long_lists(b, s, rows, dim):
    """Lists that many blocks sort, one to three passes, rows of several column slabs."""
    check(b, s, rows, dim, torch.bfloat16, positions="implicit")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("positions", ["none", "implicit", "given"])
@pytest.mark.parametrize("b,s,rows,dim", [(2, 256, 1, 8), (1, 512, 3, 512), (1, 513, 3, 16), (16, 1, 30000, 1027), (2, 65, 2500, 520),
                                          (3, 100, 1048576, 12), (3, 99, 1048577, 12), (1, 15, 1000, 16384), (7, 64, 5, 585),
                                          (7, 64, 5, 586), (1, 1, 2, 1)])
def test_short_lists(b, s, rows, dim, positions, dtype):
    """At the limits of the kernel for short lists and just beyond them; few rows of many tokens."""
    check(b, s, rows, dim, dtype, positions=positions, padding=rows - 1 if rows > 1 else None, scale=0.5)


@pytest.mark.parametrize("positions", ["none", "implicit", "given"])
@pytest.mark.parametrize("b,s,rows,dim,dtype", [(4, 5000, 900, 264, torch.bfloat16), (3, 6000, 60000, 264, torch.float32),
                                                (3, 6000, 2000, 521, torch.float16), (80, 300, 5000, 600, torch.float32),
                                                (2, 9000, 1100000, 257, torch.bfloat16)])
def test_long_lists_of_wide_rows(positions, b, s, rows, dim, dtype):
    """Position sums and zeros that run beside the sort of the tokens."""
    check(b, s, rows, dim, dtype, positions=positions, padding=5)


@pytest.mark.parametrize("positions", ["implicit", "given"])
@pytest.mark.parametrize("dtype,dim", [(torch.float32, 36), (torch.bfloat16, 1600), (torch.float16, 37)])
def test_positions_and_scale(positions, dtype, dim):
    check(3, 65, 40, dim, dtype, positions=positions, scale=dim ** 0.5, padding=3)


@pytest.mark.parametrize("start", [0, 13])
@pytest.mark.parametrize("dtype", DTYPES)
def test_vocabulary_shard(start, dtype):
    check(3, 50, 20, 72, dtype, start=start, padding=start + 2, scale=0.25, idt=torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,dim", [(40, 64), (5000, 200), (20000, 33)])
def test_one_token_everywhere(dtype, n, dim):
    """The longest segment: all positions hold the same token."""
    check(1, n, 9, dim, dtype, ids=torch.full((1, n), 4, device="cuda"))


def test_all_padding_and_all_foreign():
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(6, 16, device="cuda", requires_grad=True)
    ids = torch.full((2, 9), 5, device="cuda")
    (dw,) = torch.autograd.grad(embedding(ids, w, padding_idx=-1).sum(), w)  # an expanded gradient
    assert torch.equal(dw, torch.zeros_like(dw))
    y = embedding(ids, w, vocab_start=6)
    assert torch.equal(y, torch.zeros_like(y))
    (dw,) = torch.autograd.grad(y, w, torch.full_like(y, float("nan")))
    assert torch.equal(dw, torch.zeros_like(dw))


def test_ids_outside_the_table_are_nan_rows():
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(6, 16, device="cuda", requires_grad=True)
    p = torch.randn(4, 16, device="cuda")
    ids = torch.tensor([0, 6, -1, 2 ** 40, 5], device="cuda")
    y = embedding(ids, w)
    assert y.isnan().all(1).tolist() == [False, True, True, True, False]
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert dw[:, 0].tolist() == [1, 0, 0, 0, 0, 1]
    y = embedding(ids.clamp(0, 5), w, position_ids=torch.tensor([0, 4, -1, 3, 2], device="cuda"), position_weight=p)
    assert y.isnan().all(1).tolist() == [False, True, True, False, False]


def test_infinite_gradients_stay_in_their_row():
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(8, 8, device="cuda", requires_grad=True)
    ids = torch.tensor([1, 2, 2, 3], device="cuda")
    dy = torch.ones(4, 8, device="cuda")
    dy[1] = float("inf")
    dy[3] = float("nan")
    (dw,) = torch.autograd.grad(embedding(ids, w), w, dy)
    assert torch.isfinite(dw[[0, 1, 4, 5, 6, 7]]).all() and dw[2].isinf().all() and dw[3].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Strided ids, rows and gradients, and a table whose rows start off 16 bytes."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    check(4, 30, 25, 48, dtype, strided=True)
    check(4, 30, 25, 45, dtype, strided=True)
    ids = torch.randint(0, 25, (30, 8), device="cuda")[::2, ::2].t()
    w = torch.randn(25 * 48 + 1, device="cuda").to(dtype)[1:].view(25, 48).requires_grad_()
    y = embedding(ids, w)
    within(y, *forward(ids, w.detach(), 1.0, None, None, None))
    dy = torch.randn(48, 4, 15, device="cuda").to(dtype).permute(1, 2, 0)
    (dw,) = torch.autograd.grad(y, w, dy)
    within(dw, *table_grad(ids, dy, 25, 1.0))
    wt = torch.randn(48, 25, device="cuda").to(dtype).t().requires_grad_()  # columns dense instead of rows
    y = embedding(ids, wt)
    within(y, *forward(ids, wt.detach(), 1.0, None, None, None))
    (dw,) = torch.autograd.grad(y, wt, dy)
    within(dw, *table_grad(ids, dy, 25, 1.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [50, 3000, 40000])
def test_bound_gradient_accumulates_in_place(dtype, n):
    """A parameter bound to the flat gradient buffer: touched rows grow, the others keep their bits."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.nn.Parameter(torch.randn(700, 40, generator=g, device="cuda").to(dtype))
    p = torch.nn.Parameter(torch.randn(64, 40, generator=g, device="cuda").to(dtype))
    n = n // 50 * 50
    ids = torch.randint(0, 300, (n // 50, 50), generator=g, device="cuda")
    before = {}
    for t in (w, p):
        t.grad = torch.randn(t.shape, generator=g, device="cuda").to(dtype)
        t._smp_fused_grad = True
        before[t] = t.grad.clone()
    hooks = []
    w.register_post_accumulate_grad_hook(lambda t: hooks.append(t))
    dy = torch.randn(n // 50, 50, 40, generator=g, device="cuda").to(dtype)
    embedding(ids, w, position_weight=p, scale=2.0).backward(dy)
    assert len(hooks) == 1 and hooks[0] is w
    for t, at, scale in ((w, ids, 2.0), (p, torch.arange(50, device="cuda").expand(n // 50, 50), 1.0)):
        total, slack = table_grad(at, dy, t.shape[0], scale)
        seen = torch.bincount(at.reshape(-1), minlength=t.shape[0]) > 0
        within(t.grad[seen], (total + before[t].double())[seen], (slack + 2 * U32 * before[t].double().abs())[seen])
        assert torch.equal(t.grad[~seen], before[t][~seen])


def test_one_parameter_as_both_tables():
    """Bound and dense gradients of a table that serves for tokens and positions alike."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    g = torch.Generator(device="cuda").manual_seed(8)
    ids = torch.randint(0, 50, (6, 40), generator=g, device="cuda")
    pos = torch.arange(40, device="cuda").expand(6, 40)
    dy = torch.randn(6, 40, 520, generator=g, device="cuda")
    w = torch.nn.Parameter(torch.randn(50, 520, generator=g, device="cuda"))
    total, slack = (a + b for a, b in zip(table_grad(ids, dy, 50, 2.0), table_grad(pos, dy, 50, 1.0)))
    (dw,) = torch.autograd.grad(embedding(ids, w, scale=2.0, position_weight=w), w, dy)
    within(dw, total, 2 * slack)
    w.grad, w._smp_fused_grad = torch.zeros_like(w), True
    embedding(ids, w, scale=2.0, position_weight=w).backward(dy)
    within(w.grad, total, 2 * slack)


@pytest.mark.parametrize("frozen", [None, "token", "position"])
@pytest.mark.parametrize("given", [False, True])
def test_second_derivative(frozen, given):
    """The gradients are linear in dy: their derivative looks the rows of the second gradients up, but
    not that of the padding token.  A third pass goes the other way again."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, p, a, b = (torch.randn(n, 20, device="cuda") for n in (9, 6, 9, 6))
    ids = torch.tensor([[1, 8, 3, 3], [3, 0, 1, 7]], device="cuda")
    pos = torch.tensor([[5, 4, 0, 1], [2, 2, 3, 0]], device="cuda") if given else None
    dy = torch.randn(2, 4, 20, device="cuda", requires_grad=True)
    leaves = [t.requires_grad_() for t, name in ((w, "token"), (p, "position")) if name != frozen]
    second = [t.requires_grad_() for t, name in ((a, "token"), (b, "position")) if name != frozen]
    y = embedding(ids, w, padding_idx=3, scale=0.5, position_ids=pos, position_weight=p)
    grads = torch.autograd.grad(y, leaves, dy, create_graph=True)
    assert all(torch.equal(g, e) for g, e in zip(grads, torch.autograd.grad(y, leaves, dy)))
    (ddy,) = torch.autograd.grad(grads, dy, second, create_graph=True)
    expect = torch.zeros_like(dy)
    if frozen != "token":
        expect = expect + 0.5 * a[ids] * (ids != 3).unsqueeze(-1)
    if frozen != "position":
        expect = expect + b[pos if given else torch.arange(4, device="cuda")]
    assert float((ddy - expect).detach().abs().max()) <= 2.0 ** -23 * float(expect.detach().abs().max())
    for g, e in zip(torch.autograd.grad(ddy, second, dy.detach()), grads):
        assert torch.equal(g, e)


def test_bound_gradients_stay_out_of_other_passes():
    """torch.autograd.grad returns the gradient of a bound table, a pass that builds a graph keeps it
    in that graph, backward(inputs=...) adds it in place."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, v = (torch.randn(9, 24, device="cuda").requires_grad_() for _ in range(2))
    w.grad, w._smp_fused_grad = torch.ones_like(w), True
    slot = w.grad
    ids = torch.tensor([4, 4, 1], device="cuda")
    count = torch.zeros_like(w)
    count[4], count[1] = 2.0, 1.0
    (dw,) = torch.autograd.grad(embedding(ids, w).sum(), w)
    assert torch.equal(dw, count) and slot.eq(1).all()
    (embedding(ids, w) * embedding(ids, v)).sum().backward(inputs=[v])
    assert slot.eq(1).all() and v.grad is not None
    embedding(ids, w).sum().backward(inputs=[w])
    assert w.grad is slot and torch.equal(slot, 1 + count)
    dy = torch.ones(3, 24, device="cuda", requires_grad=True)
    embedding(ids, w).backward(dy, create_graph=True)
    assert slot.eq(1 + count).all() and torch.equal(w.grad, 1 + 2 * count)
    (ddy,) = torch.autograd.grad(w.grad.sum(), dy)
    assert ddy.eq(1).all()


def test_table_changed_before_the_backward():
    """The tables' values are not part of the gradient: an optimizer may have changed them."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(6, 16, device="cuda", requires_grad=True)
    y = embedding(torch.tensor([1, 1, 5], device="cuda"), w)
    with torch.no_grad():
        w.zero_()
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert dw[:, 0].tolist() == [0, 2, 0, 0, 0, 1]


def test_same_bits_on_every_run_and_stream():
    g1 = check(8, 1000, 500, 200, torch.float32, seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g2 = check(8, 1000, 500, 200, torch.float32, seed=5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(g1[0], g2[0])


def test_offsets_past_32_bits():
    """A table and an output of more than 2^31 elements."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    rows, dim = 600_000, 4096
    w = torch.zeros(rows, dim, device="cuda", dtype=torch.bfloat16)
    w[-1], w[300_000] = 2.0, 3.0
    ids = torch.zeros(550_000, device="cuda", dtype=torch.long)
    ids[-1], ids[-2] = rows - 1, 300_000
    w.requires_grad_()
    y = embedding(ids, w)
    assert y[-1].eq(2).all() and y[-2].eq(3).all() and y[-3].eq(0).all()
    dy = torch.zeros_like(y)
    dy[-1], dy[-2] = 1.0, 4.0
    (dw,) = torch.autograd.grad(y, w, dy)
    assert dw[-1].eq(1).all() and dw[300_000].eq(4).all() and float(dw.sum(dtype=torch.float64)) == 5 * dim


@pytest.mark.parametrize("b", [3, 50, 200])
def test_graph_replays(b):
    """Forward and backward captured: every replay on new ids gives what the eager call gives."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(900, 64, device="cuda").requires_grad_()
    p = torch.randn(130, 64, device="cuda").requires_grad_()
    ids = torch.randint(0, 900, (b, 128), device="cuda")
    dy = torch.randn(b, 128, 64, device="cuda")

    def step():
        y = embedding(ids, w, position_weight=p, scale=0.5, padding_idx=7)
        return [y.detach(), *torch.autograd.grad(y, [w, p], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        ids.copy_(torch.randint(0, 900 >> (4 * k), (b, 128), device="cuda"))
        dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, step()):
            assert torch.equal(a, e)


@pytest.mark.parametrize("positions", [False, True])
def test_no_tokens(positions):
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, p = (torch.randn(n, 20, device="cuda", requires_grad=True) for n in (7, 5))
    for shape in ((0,), (3, 0), (0, 4)):
        y = embedding(torch.empty(shape, dtype=torch.long, device="cuda"), w, position_weight=p if positions else None)
        assert y.shape == shape + (20,)
        leaves = [w, p] if positions else [w]
        for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
            assert torch.equal(g, torch.zeros_like(t))


def test_two_streams_at_once():
    """Calls of two streams share nothing: each gives what it gives alone."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    def work(k):
        g = torch.Generator(device="cuda").manual_seed(k)
        w = torch.randn(4000, 512, generator=g, device="cuda").requires_grad_()
        ids = torch.randint(0, 4000 >> k, (9000,), generator=g, device="cuda")
        dy = torch.randn(9000, 512, generator=g, device="cuda")
        return w, ids, dy

    def step(w, ids, dy):
        y = embedding(ids, w)
        return [y.detach()] + list(torch.autograd.grad(y, w, dy))

    data = [work(k) for k in range(2)]
    alone = [step(*d) for d in data]
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for _ in range(3):
        both = []
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                both.append(step(*d))
        torch.cuda.synchronize()
        for a, b in zip(alone, both):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_capture_beside_an_eager_graph_is_refused():
    """Autograd would take the gradient on the default stream, which a capture cannot include."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.randn(30, 16, device="cuda").requires_grad_()
    ids = torch.randint(0, 30, (40,), device="cuda")
    dy = torch.randn(40, 16, device="cuda")
    eager = embedding(ids, w)
    (expect,) = torch.autograd.grad(eager, w, dy, retain_graph=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = embedding(ids, w)
        with pytest.raises(RuntimeError, match="alive"):
            torch.autograd.grad(y, w, dy)
    assert torch.equal(torch.autograd.grad(eager, w, dy)[0], expect)
    del eager, y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dw,) = torch.autograd.grad(embedding(ids, w), w, dy)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, expect)


@pytest.mark.parametrize("rows", [262144, 262145, 300000, 1100000])
@pytest.mark.parametrize("shape", [(0,), (3, 0), (0, 4)])
def test_no_tokens_of_large_tables(rows, shape):
    """An empty batch of a table of any size: dense gradients are zeros, bound ones stay as they are."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    ids = torch.empty(shape, dtype=torch.long, device="cuda")
    for positions in (None, "implicit", "given"):
        w, p = (torch.randn(rows, 9, device="cuda", requires_grad=True) for _ in range(2))
        kw = {} if positions is None else {"position_weight": p}
        if positions == "given":
            kw["position_ids"] = ids
        leaves = [w] if positions is None else [w, p]
        y = embedding(ids, w, padding_idx=rows - 1, **kw)
        assert y.shape == shape + (9,)
        for g, t in zip(torch.autograd.grad(y, leaves, torch.empty_like(y), retain_graph=True), leaves):
            assert g.shape == t.shape and not g.any()
        for t in leaves:
            t.grad, t._smp_fused_grad = torch.ones_like(t), True
        embedding(ids, w, **kw).backward(torch.empty_like(y))
        assert all(t.grad.eq(1).all() for t in leaves)


@pytest.mark.parametrize("of", ["tensor", "accumulator"])
def test_hooks_of_a_bound_table_get_its_gradient(of):
    """A tensor hook may change the gradient before it is added (rows masked here); a hook of the
    accumulator sees it."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    g = torch.Generator(device="cuda").manual_seed(2)
    w, p = (torch.nn.Parameter(torch.randn(n, 24, generator=g, device="cuda")) for n in (9, 6))
    ids = torch.tensor([[4, 4, 1, 8], [0, 4, 2, 2]], device="cuda")
    dy = torch.randn(2, 4, 24, generator=g, device="cuda")
    expect = torch.autograd.grad(embedding(ids, w, scale=2.0, position_weight=p), [w, p], dy)
    for t in (w, p):
        t.grad, t._smp_fused_grad = torch.ones_like(t), True
    slots = [w.grad, p.grad]
    mask = (torch.arange(9, device="cuda") % 2 == 0).float().unsqueeze(1)
    seen = []
    if of == "tensor":
        handle = w.register_hook(lambda g: seen.append(g.clone()) or g * mask)
    else:
        accumulator = w.expand_as(w).grad_fn.next_functions[0][0]
        handle = accumulator.register_hook(lambda _, grads: seen.append(grads[0].clone()) and None)
    embedding(ids, w, scale=2.0, position_weight=p).backward(dy)
    assert w.grad is slots[0] and p.grad is slots[1]
    assert len(seen) == 1 and torch.equal(seen[0], expect[0])
    assert torch.equal(w.grad, 1 + expect[0] * (mask if of == "tensor" else 1))
    assert float((p.grad - 1 - expect[1]).abs().max()) <= 2 * U32 * float(1 + expect[1].abs().max())
    handle.remove()
    embedding(ids, w, scale=2.0, position_weight=p).backward(dy)
    assert len(seen) == 1 and w.grad is slots[0]


@pytest.mark.parametrize("n", [0, 900])
@pytest.mark.parametrize("rows,dim", [((1 << 25) + 37, 8), ((1 << 28) + 100, 1), ((1 << 25) + 4, 33), (40_000, 600_000)])
def test_gradients_of_very_large_tables(rows, dim, n):
    """More rows to clear than one launch has blocks for."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w = torch.ones(rows, dim, device="cuda", dtype=torch.float16).requires_grad_()
    ids = torch.randint(0, rows, (n,), device="cuda")
    ids[:2], ids[2:3] = rows - 1, 0
    y = embedding(ids, w)
    assert y.eq(1).all()
    (dw,) = torch.autograd.grad(y, w, y.detach())
    assert torch.equal(dw[:, 0], torch.bincount(ids, minlength=rows).half())
    filled = sum(int(part.count_nonzero()) for part in dw.split(max((1 << 28) // dim, 1)))
    assert torch.equal(dw[:, 0], dw[:, -1]) and filled == ids.unique().numel() * dim


def test_most_tokens():
    """The longest list: the radix sort of 2^27 tokens."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    n, rows = 1 << 27, 30000
    w = torch.randn(rows, 1, device="cuda").requires_grad_()
    ids = torch.randint(0, rows, (n,), device="cuda", dtype=torch.int32)
    y = embedding(ids, w)
    assert torch.equal(y[:, 0], w.detach()[:, 0][ids.long()])
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(dw[:, 0], torch.bincount(ids, minlength=rows).float())


def test_tables_of_one_column():
    """Their last stride may be anything; so may the first one of tables of one row."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    ids = torch.tensor([3, 0, 3, 9], device="cuda")
    base = torch.randn(10, 10, device="cuda")
    for w in (torch.randn(1, 10, device="cuda").t(), base[2:3].t(), base[:, 2:3], base[:1, :1].expand(10, 1)):
        for p in (None, torch.randn(1, 4, device="cuda").t()):
            w = w.detach().requires_grad_()
            y = embedding(ids, w, position_weight=p)
            assert torch.equal(y, w.detach()[ids] + (0.0 if p is None else p))
            (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
            assert dw[:, 0].tolist() == [1, 0, 0, 2, 0, 0, 0, 0, 0, 1]
    row = base[:, 4:5].t()
    y = embedding(torch.zeros(3, dtype=torch.long, device="cuda"), row)
    assert torch.equal(y, row.expand(3, 10))
