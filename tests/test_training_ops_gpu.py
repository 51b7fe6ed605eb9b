"""The embedding, block-norm and gradient-norm operators together, as a training step uses them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Net(torch.nn.Module):
    """Embedding -> blocks (linear + gelu) joined by FusedBlockNorm -> tied head."""

    def __init__(self, vocab, d, layers, rms):
        from smdistributed_modelparallel_amd import nn as smp_nn

        super().__init__()
        self.tok = torch.nn.Parameter(torch.randn(vocab, d) * 0.3)
        self.pos = torch.nn.Parameter(torch.randn(40, d) * 0.1)
        self.first = torch.nn.Parameter(torch.ones(d))
        self.blocks = torch.nn.ModuleList(torch.nn.Linear(d, d) for _ in range(layers))
        self.norms = torch.nn.ModuleList(
            smp_nn.FusedBlockNorm(d, rms=rms, gate=0.5, residual_scale=0.7) for _ in range(layers))

    def forward(self, ids):
        from smdistributed_modelparallel_amd.ops.embedding import embedding
        from smdistributed_modelparallel_amd.ops.layernorm import rms_norm

        s = embedding(ids, self.tok, padding_idx=0, scale=2.0, position_weight=self.pos)
        y = rms_norm(s, self.first)
        for block, norm in zip(self.blocks, self.norms):
            y, s = norm(torch.nn.functional.gelu(block(y)), s)
        return y @ self.tok.t()


def reference(net, ids, rms, target):
    """The same in 64 bits by elementary operations; (loss, gradients by name)."""
    p = {n: t.detach().double().requires_grad_() for n, t in net.named_parameters()}

    def norm(v, w, b):
        c = v if rms else v - v.mean(-1, keepdim=True)
        out = c * (c.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * w
        return out if b is None else out + b

    keep = (ids != 0).unsqueeze(-1)
    tok = torch.where(keep, p["tok"][ids], p["tok"].detach()[ids])  # padding takes no gradient here
    s = 2.0 * tok + p["pos"][: ids.shape[1]]
    y = s * (s.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * p["first"]
    for i in range(len(net.blocks)):
        x = torch.nn.functional.gelu(y @ p[f"blocks.{i}.weight"].t() + p[f"blocks.{i}.bias"])
        k = f"norms.{i}."
        s = s + 0.7 * p[k + "gate"] * norm(x, p[k + "post_weight"], p.get(k + "post_bias"))
        y = norm(s, p[k + "weight"], p.get(k + "bias"))
    loss = torch.nn.functional.cross_entropy((y @ p["tok"].t()).flatten(0, 1), target.flatten())
    return loss, dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


@pytest.mark.parametrize("rms", [False, True])
def test_step(rms):
    from smdistributed_modelparallel_amd.optimizers import FusedAdam, clip_grad_norm_

    torch.manual_seed(0)
    net = Net(300, 136, 3, rms).cuda()
    ids = torch.randint(0, 300, (6, 33), device="cuda")
    ids[2, 20:] = 0
    target = torch.randint(0, 300, (6, 33), device="cuda")
    opt = FusedAdam(net.parameters(), lr=1e-3)
    for _ in range(2):
        want_loss, want = reference(net, ids, rms, target)
        opt.zero_grad()
        loss = torch.nn.functional.cross_entropy(net(ids).flatten(0, 1), target.flatten())
        loss.backward()
        # fp32 forward and backward of a few layers: some hundred roundings of 2^-24, and the sums' own
        assert abs(float(loss) - float(want_loss)) < 1e-4
        for n, q in net.named_parameters():
            assert float((q.grad.double() - want[n]).norm()) <= 1e-4 * float(want[n].norm()), n
        total = torch.stack([g.norm() for g in want.values()]).norm()
        assert abs(float(clip_grad_norm_(net.parameters(), 0.5 * float(total))) - float(total)) <= 1e-4 * float(total)
        clipped = torch.stack([q.grad.double().norm() for q in net.parameters()]).norm()
        assert abs(float(clipped) / float(total) - 0.5) <= 1e-4
        opt.step()


def test_same_bits_on_every_run():
    from smdistributed_modelparallel_amd.ops.multi_tensor import grad_norm

    runs = []
    for _ in range(2):
        torch.manual_seed(1)
        net = Net(500, 200, 2, False).cuda().bfloat16()
        ids = torch.randint(0, 500, (16, 40), device="cuda")
        net(ids).float().pow(2).mean().backward()
        grads = [q.grad for n, q in net.named_parameters() if not n.startswith("blocks")]
        runs.append([grad_norm(grads)] + grads)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("positions", [True, False])
def test_lm_head_model_uses_the_fused_lookup(positions, monkeypatch):
    """The GPT model's embeddings through the operator: logits of the same bits as by the modules,
    gradients within the rounding of one sum order."""
    from smdistributed_modelparallel_amd.models import build_gpt
    from smdistributed_modelparallel_amd.nn import transformer
    from smdistributed_modelparallel_amd.ops._ext import track_calls

    ids = torch.randint(0, 512, (4, 50), device="cuda")
    out = []
    for fused in (True, False):
        monkeypatch.setattr(transformer, "_FUSE_EMBEDDING", [fused])
        torch.manual_seed(3)
        m = build_gpt("gpt2-tiny", dropout=0.0, use_positional_embedding=positions, num_layers=2).cuda().bfloat16()
        with track_calls() as calls:
            loss, logits = m((ids, None, None, None, ids))
        assert ("embedding" in calls) == fused
        loss.backward()
        out.append((logits.detach(), {n: p.grad for n, p in m.named_parameters()}))
    assert torch.equal(out[0][0], out[1][0])
    for n, g in out[0][1].items():
        h = out[1][1][n].float()
        assert float((g.float() - h).norm()) <= 2.0 ** -8 * float(h.norm()), n
    hooked = []
    monkeypatch.setattr(transformer, "_FUSE_EMBEDDING", [True])
    m.word_embedding.register_forward_hook(lambda *a: hooked.append(1))
    with track_calls() as calls:
        m((ids, None, None, None, ids))
    assert hooked and "embedding" not in calls


def test_replaced_forward_of_an_embedding_module_is_called():
    from smdistributed_modelparallel_amd.models import build_gpt

    m = build_gpt("gpt2-tiny", dropout=0.0, num_layers=1).cuda().bfloat16()
    plain, called = m.word_embedding.forward, []
    m.word_embedding.forward = lambda ids: called.append(1) or plain(ids)
    ids = torch.randint(0, 512, (2, 9), device="cuda")
    m((ids, None, None, None, ids))
    assert called


def test_distributed_embedding_module():
    from smdistributed_modelparallel_amd.nn import DistributedEmbedding
    from smdistributed_modelparallel_amd.ops._ext import track_calls

    m = DistributedEmbedding(40, 24, padding_idx=3).cuda()
    ids = torch.randint(0, 40, (5, 7), device="cuda")
    with track_calls() as calls:
        y = m(ids)
    assert calls == {"embedding": 1} and torch.equal(y, m.weight[ids])
    y.sum().backward()
    assert torch.equal(m.weight.grad[:, 0], torch.bincount(ids.flatten(), minlength=40).float() * (torch.arange(40, device="cuda") != 3))
    assert m.double()(ids).dtype == torch.float64


def _bound(*tensors):
    out = [torch.nn.Parameter(t.clone()) for t in tensors]
    for t in out:
        t.grad, t._smp_fused_grad = torch.zeros_like(t), True
    return out


def test_bound_gradients_of_two_streams():
    """One bound parameter used on two streams of one graph gets the sum of both uses, also where the
    caller reads it without waiting for either stream itself."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    torch.manual_seed(0)
    table, scale = torch.randn(6000, 520, device="cuda"), torch.randn(520, device="cuda")
    ids = [torch.randint(0, 6000, (40000,), device="cuda") for _ in range(2)]
    x = [torch.randn(40000, 520, device="cuda") for _ in range(2)]
    dy = [torch.randn(40000, 520, device="cuda") for _ in range(2)]
    alone = []
    for k in range(2):
        w, v = table.clone().requires_grad_(), scale.clone().requires_grad_()
        outs = [embedding(ids[k], w), block_norm(x[k], x[k], v)[0]]
        alone.append(torch.autograd.grad(outs, [w, v], [dy[k], dy[k]]))
        del outs
    main, streams = torch.cuda.current_stream(), [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        w, v = _bound(table, scale)
        outs = []
        for k, s in enumerate(streams):
            s.wait_stream(main)
            with torch.cuda.stream(s):
                outs += [embedding(ids[k], w), block_norm(x[k], x[k], v)[0]]
        for s in streams:
            main.wait_stream(s)
        slots = [w.grad, v.grad]
        torch.autograd.backward(outs, [dy[0], dy[0], dy[1], dy[1]])
        got = [w.grad.clone(), v.grad.clone()]  # (on the caller's stream)
        assert w.grad is slots[0] and v.grad is slots[1]
        for g, a, b in zip(got, *alone):  # one rounding of the sum, in one order or the other
            assert float((g.double() - (a.double() + b.double())).abs().max()) <= 2.0 ** -23 * float((a.abs() + b.abs()).max())
        del outs


def test_bound_gradients_with_an_accumulator_of_another_stream():
    """The leaf's accumulator was made on another stream than the pass runs on, and is alive."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    torch.manual_seed(1)
    ids, dy = torch.randint(0, 6000, (40000,), device="cuda"), torch.randn(40000, 520, device="cuda")
    (w,) = _bound(torch.randn(6000, 520, device="cuda"))
    (expect,) = torch.autograd.grad(embedding(ids, w), w, dy)
    keep = w.expand_as(w)  # (its graph holds the accumulator, made on the default stream)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    for k in range(3):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y = embedding(ids, w)
        main.wait_stream(side)
        y.backward(dy)
        assert torch.equal(w.grad, (k + 1) * expect) or k == 2  # (1 and 2 times are exact)
        del y
    assert float((w.grad - 3 * expect).abs().max()) <= 2.0 ** -23 * float(w.grad.abs().max())
    assert keep.requires_grad


@pytest.mark.parametrize("side", [False, True])
def test_bound_gradients_need_no_dense_one(side):
    from smdistributed_modelparallel_amd.ops.embedding import embedding

    (w,) = _bound(torch.randn(50000, 520, device="cuda"))
    w.register_post_accumulate_grad_hook(lambda t: None)
    ids = torch.randint(0, 50000, (600,), device="cuda")
    dy = torch.ones(600, 520, device="cuda")
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        embedding(ids, w).backward(dy)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < w.nbytes / 4
    assert torch.equal(w.grad[:, 0], torch.bincount(ids, minlength=50000).float())


@pytest.mark.parametrize("late", [False, True])
def test_caller_waits_for_bound_gradients(late):
    """The pass runs on another stream than the caller's, which is busy; the caller reads at once."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    torch.manual_seed(2)
    w, v = _bound(torch.randn(3000, 136, device="cuda"), torch.randn(136, device="cuda"))
    ids, x = torch.randint(0, 3000, (2000,), device="cuda"), torch.randn(2000, 136, device="cuda")
    dy = torch.randn(2000, 136, device="cuda")
    outs = [embedding(ids, w), block_norm(x, x, v)[0]]
    expect = torch.autograd.grad(outs, [w, v], [dy, dy])
    del outs
    keep = [t.expand_as(t) for t in (w, v)] if late else None
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    side.wait_stream(main)
    with torch.cuda.stream(side):
        outs = [embedding(ids, w), block_norm(x, x, v)[0]]
        torch.cuda._sleep(100_000_000)
    torch.autograd.backward(outs, [dy, dy])
    got = [w.grad.clone(), v.grad.clone()]
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    assert keep is None or len(keep) == 2


def test_writes_in_place_are_seen_by_graphs():
    """What autograd saved before a clip, or before a bound gradient grew, it refuses to use after it."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm
    from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

    x = torch.randn(8, 16, device="cuda", requires_grad=True)

    def clip(g):
        clip_grad_norm_([g], 0.1)

    def clip_into(g):
        clip_grad_norm_([torch.ones_like(g)], 0.1, out=[g])

    def lookup(g):
        w = torch.nn.Parameter(torch.randn(8, 16, device="cuda"))
        w.grad, w._smp_fused_grad = g, True
        embedding(torch.tensor([1, 2], device="cuda"), w).sum().backward()
        assert w.grad is g

    def norm(g):
        w = torch.nn.Parameter(torch.randn(16, device="cuda"))
        w.grad, w._smp_fused_grad = g[0], True
        block_norm(x.detach(), x.detach(), w)[0].sum().backward()

    for write in (clip, clip_into, lookup, norm):
        g = torch.randn(8, 16, device="cuda")
        loss = (x * g).sum()
        write(g)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()


def test_captured_bound_gradients():
    """A captured backward adds to bound gradients at every replay what the eager one adds."""
    from smdistributed_modelparallel_amd.ops.embedding import embedding
    from smdistributed_modelparallel_amd.ops.layernorm import block_norm

    torch.manual_seed(4)
    table, place, scale = (torch.randn(n, device="cuda") for n in ((700, 136), (60, 136), (136,)))
    ids, dy = torch.randint(0, 700, (20, 50), device="cuda"), torch.randn(20, 50, 136, device="cuda")

    def step(w, p, v):
        x = embedding(ids, w, position_weight=p, padding_idx=3)
        y, s = block_norm(x, x, v, gate=v)
        torch.autograd.backward([y, s], [dy, dy])

    captured, eager = _bound(table, place, scale), _bound(table, place, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*captured)
    torch.cuda.current_stream().wait_stream(side)
    for t in captured:
        t.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*captured)
    for k in range(3):
        ids.copy_(torch.randint(0, 700 >> (3 * k), (20, 50), device="cuda"))
        dy.normal_()
        graph.replay()
        step(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(captured, eager))
