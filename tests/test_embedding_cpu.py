"""ops.embedding on the CPU: values and gradients of the plain path, and what the operator refuses."""
import pytest
import torch

from smdistributed_modelparallel_amd.backend.exceptions import SMPInvalidArgumentError
from smdistributed_modelparallel_amd.ops.embedding import embedding


def test_plain_embedding_is_torchs():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(11, 6, generator=g, requires_grad=True)
    ids = torch.randint(0, 11, (3, 5), generator=g)
    y = embedding(ids, w, padding_idx=-2)
    ref = torch.nn.functional.embedding(ids, w, padding_idx=9)
    assert torch.equal(y, ref)
    dy = torch.randn(3, 5, 6, generator=g)
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(ref, w, dy)[0])
    with pytest.raises(IndexError):
        embedding(torch.tensor([11]), w)


def test_scale_positions_and_differences():
    """Against finite differences, in 64 bits for the arithmetic of the test itself."""
    g = torch.Generator().manual_seed(1)
    w, p = torch.randn(7, 4, generator=g), torch.randn(9, 4, generator=g)
    ids, pos = torch.randint(0, 7, (2, 3), generator=g), torch.tensor([[4, 0, 8]])
    wl, pl = w.clone().requires_grad_(), p.clone().requires_grad_()
    y = embedding(ids, wl, scale=0.5, position_ids=pos, position_weight=pl)
    assert torch.allclose(y, 0.5 * w[ids] + p[pos.expand(2, 3)])
    dy = torch.randn(2, 3, 4, generator=g)
    dw, dp = torch.autograd.grad(y, (wl, pl), dy)
    for table, grad, other in ((w, dw, p), (p, dp, w)):
        for r, c in ((int(ids[0, 0]), 1), (4, 2)):
            hi = table.clone()
            hi[r, c] += 1.0  # the map is linear: a step of one is exact
            a = embedding(ids, hi if table is w else w, scale=0.5, position_ids=pos,
                          position_weight=hi if table is p else p)
            diff = ((a.double() - y.detach().double()) * dy.double()).sum()
            assert abs(float(diff - grad[r, c].double())) < 1e-5


def test_shards_add_up_to_the_whole_table():
    g = torch.Generator().manual_seed(2)
    w, ids = torch.randn(10, 4, generator=g), torch.randint(0, 10, (4, 3), generator=g)
    parts = [embedding(ids, w[a:b].clone(), vocab_start=a) for a, b in ((0, 4), (4, 5), (5, 10))]
    assert torch.equal(sum(parts), w[ids])
    whole = w.clone().requires_grad_()
    dy = torch.randn(4, 3, 4, generator=g)
    (ref,) = torch.autograd.grad(embedding(ids, whole, padding_idx=6), whole, dy)
    for a, b in ((0, 4), (4, 5), (5, 10)):
        shard = w[a:b].clone().requires_grad_()
        (got,) = torch.autograd.grad(embedding(ids, shard, padding_idx=6, vocab_start=a), shard, dy)
        assert torch.allclose(got, ref[a:b])


def test_no_tokens():
    w = torch.randn(5, 3, requires_grad=True)
    y = embedding(torch.empty(2, 0, dtype=torch.long), w, scale=2.0)
    assert y.shape == (2, 0, 3)
    assert torch.equal(torch.autograd.grad(y, w, torch.empty(2, 0, 3))[0], torch.zeros(5, 3))


_W = torch.zeros(5, 4)
_I = torch.zeros(2, 3, dtype=torch.long)


@pytest.mark.parametrize("args,kwargs", [
    ((_I.float(), _W), {}),
    ((_I.to(torch.int16), _W), {}),
    ((_I, _W[0]), {}),
    ((_I, _W.long()), {}),
    ((_I, _W.double()), {}),
    ((_I, _W[:, :0]), {}),
    ((_I, _W[:0]), {}),
    ((_I, _W), {"padding_idx": 5}),
    ((_I, _W), {"padding_idx": -6}),
    ((_I, _W), {"padding_idx": -1, "vocab_start": 5}),
    ((_I, _W), {"vocab_start": -1}),
    ((_I, _W), {"scale": float("nan")}),
    ((_I, _W), {"scale": float("inf")}),
    ((_I, _W), {"position_ids": _I}),
    ((_I, _W), {"position_weight": _W[:2]}),
    ((_I, _W), {"position_weight": _W[:, :3]}),
    ((_I, _W), {"position_weight": _W.half()}),
    ((_I[0, 0], _W), {"position_weight": _W}),
    ((_I, _W), {"position_weight": _W, "position_ids": _I[:, :2]}),
    ((_I, _W), {"position_weight": _W, "position_ids": _I.float()}),
])
def test_refusals(args, kwargs):
    with pytest.raises(SMPInvalidArgumentError):
        embedding(*args, **kwargs)


@pytest.mark.parametrize("n,rows,dim", [(1, 2, (1 << 24) + 1), (1, (1 << 31) - 1, 1), ((1 << 27) + 1, 2, 1), (1 << 27, 2, 1024),
                                        (16384, 2, 8388608)])
def test_sizes_beyond_a_launch_are_refused(n, rows, dim):
    """Expanded tensors: one element of memory each."""
    with pytest.raises(SMPInvalidArgumentError):
        embedding(torch.zeros(1, dtype=torch.long).expand(n), torch.zeros(1, 1).expand(rows, dim))
