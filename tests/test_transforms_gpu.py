"""embedding and block_norm where a kernel's launch alone would lose something: dual numbers,
function transforms, compiled functions, traces, dispatch modes.

The embedding is linear in its tables, so its results are held to the formula: one rounding of fp32
(2^-24) for the product and one for the sum, taken twice.  block_norm's tangents are held to the
64-bit definition's within 2^-14 of the largest: a row's sums are off by 64 * 2^-24, and two norms
whose weights and deviations are of the size of one multiply that by 16 at most.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests import block_norm_ref as ref

pytestmark = pytest.mark.gpu
FEW = 4 * 2.0 ** -24


def near(got, want, bound=FEW):
    assert got.shape == want.shape
    assert float((got.double() - want.double()).abs().max()) <= bound * float(want.double().abs().max())


def tables():
    g = torch.Generator(device="cuda").manual_seed(0)
    w, p, tw, tp = (torch.randn(n, 24, generator=g, device="cuda") for n in (9, 6, 9, 6))
    ids = torch.tensor([[1, 8, 3, 3], [3, 0, 1, 7]], device="cuda")
    return w, p, tw, tp, ids


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("start", [None, 2])
def test_embedding_tangents(start, leaf, no_grad):
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, p, tw, tp, ids = tables()
    local = ids - (start or 0)
    held = ((local >= 0) & (local < 9)).unsqueeze(-1)
    want = 0.5 * tw[local.clamp(0, 8)] * held + tp[:4]
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        w, p = w.requires_grad_(leaf), p.requires_grad_(leaf)
        out = embedding(ids, fwd.make_dual(w, tw), scale=0.5, vocab_start=start, position_weight=fwd.make_dual(p, tp))
        y, t = fwd.unpack_dual(out)
        near(t, want)
        near(y, embedding(ids, w.detach(), scale=0.5, vocab_start=start, position_weight=p.detach()))
        # one table alone, the other frozen
        t = fwd.unpack_dual(embedding(ids, w.detach(), scale=0.5, vocab_start=start,
                                      position_weight=fwd.make_dual(p, tp))).tangent
        near(t, tp[:4].expand(2, 4, 24))


def test_module_tangents():
    from smdistributed_modelparallel_amd.nn import DistributedEmbedding

    m = DistributedEmbedding(9, 24, padding_idx=3).cuda()
    _, _, tw, _, ids = tables()
    _, t = torch.func.jvp(lambda w: torch.func.functional_call(m, {"weight": w}, (ids,)), (m.weight.detach(),), (tw,))
    near(t, tw[ids])


def test_embedding_gradients_of_dual_and_batched_rows():
    """The gradient is linear in dy: its tangent is the gradient of dy's tangent, a batch's one for each."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, p, _, _, ids = tables()
    w.requires_grad_(), p.requires_grad_()
    for kw in ({"position_weight": p}, {"position_weight": p, "position_ids": ids % 6}):
        y = embedding(ids, w, padding_idx=3, scale=0.5, **kw)
        dy, t, u = (torch.randn(2, 4, 24, device="cuda") for _ in range(3))
        want = [torch.autograd.grad(y, [w, p], d, retain_graph=True) for d in (dy, t, u)]
        with fwd.dual_level():
            for i, g in enumerate(torch.autograd.grad(y, [w, p], fwd.make_dual(dy, t), retain_graph=True)):
                g, tangent = fwd.unpack_dual(g)
                near(g, want[0][i])
                near(tangent, want[1][i])
        batch = torch.autograd.grad(y, [w, p], torch.stack([dy, t, u]), is_grads_batched=True, retain_graph=True)
        for i, g in enumerate(batch):
            near(g, torch.stack([v[i] for v in want]))


def test_embedding_in_function_transforms():
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    w, p, tw, _, ids = tables()
    dy = torch.randn(2, 4, 24, device="cuda")

    def f(w):
        return (embedding(ids, w, padding_idx=3, scale=0.5, position_weight=p) * dy).sum()

    leaf = w.clone().requires_grad_()
    near(torch.func.grad(f)(w), torch.autograd.grad(f(leaf), leaf)[0])
    near(torch.vmap(lambda i: embedding(i, w))(ids), w[ids])
    near(torch.vmap(lambda v: embedding(ids, v))(torch.stack([w, tw])), torch.stack([w[ids], tw[ids]]))
    outside = torch.tensor([0, 9, -1], device="cuda")
    y = torch.vmap(lambda i: embedding(i, w))(outside.expand(2, 3))
    assert y.isnan().all(-1).tolist() == [[False, True, True]] * 2


def test_traces_replay_the_call():
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm, rms_norm

    w, p, _, _, ids = tables()
    v = torch.randn(24, device="cuda")

    def f(ids):
        x = embedding(ids, w, position_weight=p)
        return (*block_norm(x, 2 * x, v, gate=v), rms_norm(x, v))

    traced = torch.jit.trace(f, ids, check_trace=False)
    for other in (ids, (ids + 1) % 9):
        for a, b in zip(traced(other), f(other)):
            near(a, b, 2.0 ** -14)


def test_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    with FakeTensorMode():
        w = torch.empty(9, 24, device="cuda", dtype=torch.bfloat16)
        y = embedding(torch.zeros(2, 4, dtype=torch.long, device="cuda"), w)
        assert y.shape == (2, 4, 24) and y.dtype == torch.bfloat16 and y.is_cuda
        y, s = block_norm(y, y, w[0])
        assert y.shape == s.shape == (2, 4, 24) and s.is_cuda
    y = embedding(torch.zeros(2, 4, dtype=torch.long, device="cuda").new_zeros(1), torch.ones(3, 8, device="cuda"))
    assert y.eq(1).all()


def block_inputs(d=40, post=True):
    g = torch.Generator(device="cuda").manual_seed(3)

    def r(*n):
        return torch.randn(*n, generator=g, device="cuda")

    t = {"x": r(3, 5, d), "residual": r(3, 5, d), "weight": r(d), "bias": r(d), "gate": r(3, 1, d)}
    return t if not post else t | {"post_weight": r(d), "post_bias": r(d)}


def block(t, alpha=0.5):
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    return block_norm(t["x"], t["residual"], t["weight"], t["bias"], t.get("post_weight"), t.get("post_bias"),
                      t["gate"], alpha)


def block64(t, alpha=0.5):
    h = ref.norm(t["x"], t["post_weight"], t["post_bias"], 1e-5, False) if "post_weight" in t else t["x"]
    s = t["residual"] + alpha * t["gate"] * h
    return ref.norm(s, t["weight"], t["bias"], 1e-5, False), s


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("no_grad", [False, True])
def test_block_norm_tangents(no_grad, post):
    t = block_inputs(post=post)
    tangents = {k: torch.randn_like(v) for k, v in t.items()}
    _, want = torch.func.jvp(lambda *a: block64(dict(zip(t, a))), tuple(v.double() for v in t.values()),
                             tuple(v.double() for v in tangents.values()))
    with fwd.dual_level(), torch.set_grad_enabled(not no_grad):
        out = block({k: fwd.make_dual(v, tangents[k]) for k, v in t.items()})
        for o, e, plain in zip(out, want, block(t)):
            near(fwd.unpack_dual(o).tangent, e, 2.0 ** -14)
            near(fwd.unpack_dual(o).primal, plain, 2.0 ** -14)


def test_rms_norm_tangent():
    from smdistributed_modelparallel_amd.ops.layernorm import rms_norm

    x, w, t = (torch.randn(n, device="cuda") for n in ((7, 40), (40,), (7, 40)))
    _, want = torch.func.jvp(lambda v: ref.norm(v, w.double(), None, 1e-5, True), (x.double(),), (t.double(),))
    with fwd.dual_level():
        near(fwd.unpack_dual(rms_norm(fwd.make_dual(x, t), w)).tangent, want, 2.0 ** -14)


def test_block_norm_in_function_transforms():
    t = block_inputs()
    leaf = {k: v.clone().requires_grad_() for k, v in t.items()}
    loss = sum(o.square().sum() for o in block(leaf))
    want = dict(zip(leaf, torch.autograd.grad(loss, list(leaf.values()))))
    got = torch.func.grad(lambda u: sum(o.square().sum() for o in block(u)))(t)
    for k in t:
        near(got[k], want[k], 2.0 ** -14)
    y, s = torch.vmap(lambda x, r: block({**t, "x": x, "residual": r, "gate": t["gate"][0]}))(t["x"], t["residual"])
    e = block({**t, "gate": t["gate"][:1].expand(3, 1, 40)})
    near(y, e[0], 2.0 ** -14)
    near(s, e[1], 2.0 ** -14)


def test_block_norm_refuses_gradients_that_are_no_plain_tensors():
    t = block_inputs()
    x = t["x"].requires_grad_()
    y, _ = block(t)
    dy = torch.ones_like(y)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="plain tensor"):
        torch.autograd.grad(y, x, fwd.make_dual(dy, dy), retain_graph=True)
    with pytest.raises(RuntimeError, match="plain tensor"):
        torch.autograd.grad(y, x, dy.expand(2, *dy.shape), is_grads_batched=True, retain_graph=True)
    assert torch.autograd.grad(y, x, dy)[0].isfinite().all()


def test_gradient_norm_refuses_tensors_that_are_not_their_memory():
    """Fake, dual, batched and lazily negated tensors: nothing is read or written."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_, grad_norm, grad_power

    x = torch.ones(40, device="cuda")
    with FakeTensorMode():
        fake = torch.empty(40, device="cuda")
    negated = torch._neg_view(x)
    with fwd.dual_level():
        for bad in (fake, negated, fwd.make_dual(x.clone(), x)):
            for call in (grad_norm, grad_power, lambda ts: clip_grad_norm_(ts, 1.0)):
                with pytest.raises(SMPInvalidArgumentError):
                    call([x, bad])
            with pytest.raises(SMPInvalidArgumentError):
                clip_grad_norm_([x], 1.0, out=[bad])
    with pytest.raises(SMPInvalidArgumentError):
        torch.vmap(lambda t: grad_norm([t]))(x.view(4, 10))
    assert x.eq(1).all()


def test_compiled_in_one_graph():
    """torch.compile sees torch's operations, in values and gradients."""
    from smdistributed_modelparallel_amd.nn import DistributedEmbedding
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm, rms_norm

    w, p, _, _, ids = tables()
    m, v = DistributedEmbedding(9, 24, padding_idx=3).cuda(), torch.randn(24, device="cuda")
    w.requires_grad_()

    def f(ids):
        x = embedding(ids, w, scale=0.5, position_weight=p) + m(ids)
        return (*block_norm(x, 2 * x, v, gate=v), rms_norm(x, v))

    got, want = torch.compile(f, backend="eager", fullgraph=True)(ids), f(ids)
    for a, b in zip(got, want):
        near(a, b, 2.0 ** -14)
    dy = [torch.randn_like(o) for o in want]
    for a, b in zip(torch.autograd.grad(got, [w, m.weight], dy), torch.autograd.grad(want, [w, m.weight], dy)):
        near(a, b, 2.0 ** -14)
