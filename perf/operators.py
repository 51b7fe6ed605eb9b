"""What the embedding, block-norm and gradient-clipping operators are measured on.

Every case is one call as a training script (or, forward only, an evaluation or generation
loop) makes it.  ``run`` computes it in plain torch operations, or -- with ``own`` set --
through this package's operators:

* ``embed``: token embedding ``position[t] + scale * weight[id]`` and its gradients;
* ``block``: the norms around a block, ``h = norm(x)``, ``s = residual + alpha * gate * h``,
  ``y = norm(s)``, and their gradients;
* ``clip``: the global norm of a list of gradients, and the clipped gradients.
"""
import math

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ------------------------------------------------------------------------------ cases
def _embed(name, b, s, vocab, dim, dtype, train, positions="none", scale=1.0, pad=0.0, shards=1):
    return {"name": name, "op": "embed", "b": b, "s": s, "vocab": vocab, "dim": dim, "dtype": dtype, "train": train,
            "positions": positions, "scale": scale, "pad": pad, "shards": shards}


def _block(name, b, s, dim, dtype, train, kind="layer", post=True, gate="channel", alpha=1.0, wdtype=None):
    return {"name": name, "op": "block", "b": b, "s": s, "dim": dim, "dtype": dtype, "wdtype": wdtype or dtype,
            "train": train, "kind": kind, "post": post, "gate": gate, "alpha": alpha}


def _clip(name, layers, hidden, vocab, dtype, out, p="2", scale=1.0, clipped=True, mixed=False):
    return {"name": name, "op": "clip", "layers": layers, "hidden": hidden, "vocab": vocab, "dtype": dtype,
            "out": out, "p": p, "scale": scale, "clipped": clipped, "mixed": mixed}


def listed():
    return [
        # generation: one new token for each of 8 sequences, position given; latency is all there is
        _embed("embed-decode", 8, 1, 50257, 1600, "bfloat16", False, positions="given"),
        # one short fp32 sequence of a fine-tuning step, padded batch
        _embed("embed-short", 3, 77, 30522, 512, "float32", True, positions="implicit", pad=0.3),
        # GPT-2 XL's micro-batch of 32 x 2048 tokens (this repository's benchmark)
        _embed("embed-gpt2-xl", 32, 2048, 50257, 1600, "bfloat16", True, positions="implicit"),
        # one vocabulary shard of a GPT-NeoX-sized embedding under tensor parallelism, scaled
        _embed("embed-shard", 4, 2048, 50432, 6144, "float16", True, scale=0.5, shards=4),
        # generation: 8 rows through the norms around one block
        _block("block-decode", 8, 1, 1600, "bfloat16", False),
        # GPT-2 XL's hidden states, LayerNorm on both sides, learned per-channel gate
        _block("block-gpt2-xl", 8, 2048, 1600, "bfloat16", True, alpha=0.5),
        # root-mean-square norms with fp32 weights and one gate vector for each sample
        _block("block-rms-sample", 16, 1024, 4096, "bfloat16", True, kind="rms", gate="sample", wdtype="float32"),
        # an odd width and row count, fp16, no norm after the block
        _block("block-odd", 7, 333, 1601, "float16", True, post=False, gate="none"),
        # a small model's gradients, fp32: many short tensors, latency
        _clip("clip-small", 4, 128, 512, "float32", "same"),
        # fp16 gradients unscaled and clipped into fp32 master gradients
        _clip("clip-master", 12, 1600, 50257, "float16", "float32", scale=1.0 / 1024.0, mixed=True),
        # all of GPT-2 XL's gradients in bf16
        _clip("clip-gpt2-xl", 48, 1600, 50257, "bfloat16", "same"),
        # the largest absolute value as the norm
        _clip("clip-inf", 24, 1000, 30522, "bfloat16", "same", p="inf"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["embed", "block", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "clip":
        hidden = _log_int(rng, 48, 1600)
        c = _clip("", rng.randint(1, 40), hidden, _log_int(rng, 100, 50257), dtype, rng.choice(["same", "float32"]),
                  p=rng.choice(["2", "2", "inf"]), scale=rng.choice([1.0, 1.0 / 512.0]), clipped=rng.random() < 0.8,
                  mixed=rng.random() < 0.5)
    else:
        dim = _log_int(rng, 32, 8192)
        if rng.random() < 0.7:
            dim = (dim + 7) // 8 * 8
        tokens = max(1, min(_log_int(rng, 1, 65536), 100_000_000 // dim))
        s = _log_int(rng, 1, min(tokens, 4096))
        b = max(1, tokens // s)
        train = rng.random() < 0.75
        if op == "embed":
            vocab = min(_log_int(rng, 8, 50257), 80_000_000 // dim)
            shards = rng.choice([1, 1, 2, 4]) if b * s >= 64 else 1  # (a shard holds some of the tokens)
            c = _embed("", b, s, vocab, dim, dtype, train, rng.choice(["none", "implicit", "given"]) if shards == 1 else "none",
                       scale=rng.choice([1.0, 1.0, dim ** 0.5]), pad=rng.choice([0.0, 0.4]) if shards == 1 else 0.0,
                       shards=shards)
        else:
            if train:  # forward and backward hold more tensors than an embedding's
                b = max(1, min(b, 60_000_000 // (dim * s)))
            c = _block("", b, s, dim, dtype, train, rng.choice(["layer", "rms"]), rng.random() < 0.6,
                       rng.choice(["none", "channel", "sample", "full"]), alpha=rng.choice([1.0, 0.25]),
                       wdtype=rng.choice([dtype, "float32"]))
    del c["name"]
    return c


def _shard(c):
    """(rows held, first id held): the middle shard of the vocabulary."""
    rows = max(1, c["vocab"] // c["shards"])
    return rows, rows * (c["shards"] // 2)


def _positions_rows(c):
    """Rows of the position table: a few more than the sequence uses."""
    return c["s"] + 1 + c["s"] // 4


def _shapes(c):
    """The parameter shapes of a decoder with `layers` layers, as its gradients come."""
    h, out = c["hidden"], []
    for _ in range(c["layers"]):
        out += [(h,), (h,), (3 * h, h), (3 * h,), (h, h), (h,), (h,), (h,), (4 * h, h), (4 * h,), (h, 4 * h), (h,)]
    return out + [(c["vocab"], h), (h,), (h,)]


def _token_frequencies(vocab):
    """Words of natural text: the r-th most frequent one with probability ~ 1 / (r + 2.7)."""
    p = 1.0 / (torch.arange(vocab, dtype=torch.float64) + 2.7)
    return p / p.sum()


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DT[c["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype).mul_(std).add_(mean)

    st = {"case": c}
    if c["op"] == "embed":
        rows, start = _shard(c)
        n = c["b"] * c["s"]
        cdf = _token_frequencies(c["vocab"]).cumsum(0).to(dev)
        rank = torch.searchsorted(cdf, torch.rand(n, generator=g, device=dev, dtype=torch.float64)).clamp_(max=c["vocab"] - 1)
        ids = torch.randperm(c["vocab"], generator=g, device=dev)[rank].view(c["b"], c["s"])
        st["padding_idx"] = None
        if c["pad"]:  # the tail of every sequence is padding, of another length in each
            st["padding_idx"] = c["vocab"] - 1
            keep = (torch.rand(c["b"], 1, generator=g, device=dev) * 2 * c["pad"]).neg_().add_(1).mul_(c["s"])
            ids = torch.where(torch.arange(c["s"], device=dev) < keep, ids, torch.full_like(ids, c["vocab"] - 1))
        st["ids"] = ids.contiguous()
        st["vocab_start"] = start if c["shards"] > 1 else None
        st["weight"] = randn(rows, c["dim"], std=0.02)
        st["position_weight"] = st["position_ids"] = None
        if c["positions"] != "none":
            st["position_weight"] = randn(_positions_rows(c), c["dim"], std=0.01)
        if c["positions"] == "given":  # every sequence begins at a place of its own
            first = torch.randint(0, _positions_rows(c) - c["s"] + 1, (c["b"], 1), generator=g, device=dev)
            st["position_ids"] = first + torch.arange(c["s"], device=dev)
        if c["train"]:
            st["dy"] = randn(c["b"], c["s"], c["dim"], std=0.1)
            st["weight"].requires_grad_()
            if st["position_weight"] is not None:
                st["position_weight"].requires_grad_()
    elif c["op"] == "block":
        b, s, d, wdt = c["b"], c["s"], c["dim"], _DT[c["wdtype"]]
        st["x"], st["residual"] = randn(b, s, d, std=0.7, mean=0.1), randn(b, s, d, std=1.5, mean=-0.2)
        st["weight"] = randn(d, std=0.1, mean=1.0, dtype=wdt)
        st["bias"] = randn(d, std=0.1, dtype=wdt) if c["kind"] == "layer" else None
        st["post_weight"] = randn(d, std=0.1, mean=1.0, dtype=wdt) if c["post"] else None
        st["post_bias"] = randn(d, std=0.1, dtype=wdt) if c["post"] and c["kind"] == "layer" else None
        shape = {"channel": (d,), "sample": (b, 1, d), "full": (b, s, d)}.get(c["gate"])
        st["gate"] = None if shape is None else randn(*shape, std=0.3, mean=0.5, dtype=wdt if c["gate"] == "channel" else dt)
        if c["train"]:
            st["dy"], st["ds"] = randn(b, s, d, std=0.3), randn(b, s, d, std=0.2)
            for k in ("x", "residual", "weight", "bias", "post_weight", "post_bias", "gate"):
                if st[k] is not None:
                    st[k].requires_grad_()
    else:
        loss_scale = 1.0 / c["scale"]
        dts = [torch.float32 if c["mixed"] and len(s) == 1 else dt for s in _shapes(c)]  # norms and biases in fp32
        st["grads"] = [randn(*s, std=1e-3 * loss_scale, dtype=t) for s, t in zip(_shapes(c), dts)]
        # the clipped gradients go to one flat buffer for each type, every tensor at a multiple of 64 elements
        odt = [t.dtype if c["out"] == "same" else _DT[c["out"]] for t in st["grads"]]
        size = dict.fromkeys(odt, 0)
        at = []
        for t, o in zip(st["grads"], odt):
            at.append(size[o])
            size[o] += (t.numel() + 63) // 64 * 64
        st["flat"] = {o: torch.zeros(n, dtype=o, device=dev) for o, n in size.items()}
        st["out"] = [st["flat"][o][k:k + t.numel()].view(t.shape) for t, o, k in zip(st["grads"], odt, at)]
        n = sum(t.numel() for t in st["grads"])
        usual = 1e-3 * math.sqrt(n) if c["p"] == "2" else 4e-3
        st["max_norm"] = usual * (0.3 if c["clipped"] else 3.0)
    return st


# ----------------------------------------------------------------------------- one pass
def run(state):
    return {"embed": _run_embed, "block": _run_block, "clip": _run_clip}[state["case"]["op"]](state)


def _run_embed(st):
    c = st["case"]
    if own:
        from smdistributed_modelparallel_amd.ops.embedding import embedding

        def call():
            return embedding(st["ids"], st["weight"], padding_idx=st["padding_idx"], scale=c["scale"],
                             vocab_start=st["vocab_start"], position_ids=st["position_ids"],
                             position_weight=st["position_weight"])

        if not c["train"]:
            with torch.no_grad():
                return [call()]
        out = call()
        leaves = [t for t in (st["weight"], st["position_weight"]) if t is not None]
        return [out.detach(), *torch.autograd.grad(out, leaves, st["dy"])]

    with torch.no_grad():
        w, pw, dt = st["weight"], st["position_weight"], st["weight"].dtype
        local, held = st["ids"], None
        if st["vocab_start"] is not None:  # the other shards' tokens
            local = local - st["vocab_start"]
            held = (local >= 0) & (local < w.shape[0])
            local = torch.where(held, local, 0)
        y = w[local].float() * c["scale"]
        if held is not None:
            y = y * held.unsqueeze(-1)
        pos = None
        if pw is not None:
            pos = st["position_ids"]
            if pos is None:
                pos = torch.arange(c["s"], device=w.device).expand(c["b"], -1)
            y = y + pw[pos].float()
        outs = [y.to(dt)]
        if c["train"]:
            dy = st["dy"].float().reshape(-1, c["dim"])
            if st["padding_idx"] is not None:
                held = st["ids"] != st["padding_idx"]
            dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
            dw.index_add_(0, local.reshape(-1), dy if held is None else dy * held.reshape(-1, 1))
            outs.append((dw * c["scale"]).to(dt))
            if pw is not None:
                dp = torch.zeros(pw.shape, dtype=torch.float32, device=w.device)
                outs.append(dp.index_add_(0, pos.reshape(-1), dy).to(dt))
        return outs


_EPS = 1e-5


def _norm32(x, w, b, rms):
    """(normalised x, 1 / deviation, output) of the last dimension, fp32."""
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
    n = x * r
    return n, r, n * w.float() + (b.float() if b is not None else 0.0)


def _norm32_backward(dy, n, r, w, rms):
    g = dy * w.float()
    dx = g - n * (g * n).mean(-1, keepdim=True)
    if not rms:
        dx = dx - g.mean(-1, keepdim=True)
    return dx * r


def _run_block(st):
    c = st["case"]
    if own:
        from smdistributed_modelparallel_amd.ops.layernorm import block_norm

        def call():
            return block_norm(st["x"], st["residual"], st["weight"], st["bias"], post_weight=st["post_weight"],
                              post_bias=st["post_bias"], gate=st["gate"], residual_scale=c["alpha"], eps=_EPS,
                              rms=c["kind"] == "rms")

        if not c["train"]:
            with torch.no_grad():
                return list(call())
        y, s = call()
        leaves = [st[k] for k in ("x", "residual", "weight", "bias", "post_weight", "post_bias", "gate")
                  if st[k] is not None]
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [st["dy"], st["ds"]])]

    with torch.no_grad():
        rms, dt, gate = c["kind"] == "rms", st["x"].dtype, st["gate"]
        x, h = st["x"].float(), st["x"].float()
        if st["post_weight"] is not None:
            n2, r2, h = _norm32(x, st["post_weight"], st["post_bias"], rms)
        m = c["alpha"] * gate.float() if gate is not None else c["alpha"]
        s = st["residual"].float() + m * h
        n1, r1, y = _norm32(s, st["weight"], st["bias"], rms)
        outs = [y.to(dt), s.to(dt)]
        if not c["train"]:
            return outs
        dy = st["dy"].float()
        ds = _norm32_backward(dy, n1, r1, st["weight"], rms) + st["ds"].float()
        dh = m * ds
        dx = _norm32_backward(dh, n2, r2, st["post_weight"], rms) if st["post_weight"] is not None else dh
        grads = [dx.to(dt), ds.to(dt), (dy * n1).sum((0, 1)).to(st["weight"].dtype)]
        if st["bias"] is not None:
            grads.append(dy.sum((0, 1)).to(st["bias"].dtype))
        if st["post_weight"] is not None:
            grads.append((dh * n2).sum((0, 1)).to(st["post_weight"].dtype))
        if st["post_bias"] is not None:
            grads.append(dh.sum((0, 1)).to(st["post_bias"].dtype))
        if gate is not None:
            dg = c["alpha"] * ds * h
            if c["gate"] != "full":
                dg = dg.sum((0, 1)) if c["gate"] == "channel" else dg.sum(1, keepdim=True)
            grads.append(dg.to(gate.dtype))
        return outs + grads


def _run_clip(st):
    c = st["case"]
    if own:
        from smdistributed_modelparallel_amd.ops.multi_tensor import clip_grad_norm_

        norm = clip_grad_norm_(st["grads"], st["max_norm"], norm_type=float(c["p"]), scale=c["scale"], out=st["out"])
        return [norm, *st["flat"].values()]
    if c["p"] == "2":
        parts = [t.float().square().sum(dtype=torch.float64) for t in st["grads"]]
        norm = torch.stack(parts).sum().sqrt() * c["scale"]
    else:
        norm = torch.stack([t.float().abs().max() for t in st["grads"]]).max().double() * c["scale"]
    f = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0).mul(c["scale"]).float()
    [o.copy_(t.float() * f) for t, o in zip(st["grads"], st["out"])]
    return [norm.float(), *st["flat"].values()]


# ------------------------------------------------------------------------------- floors
def work(case):
    """Every input once (of a table, the rows that are looked up), every output once."""
    c = case
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    e = size[c["dtype"]]
    if c["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(c))
        small = sum(math.prod(s) for s in _shapes(c) if len(s) == 1) if c["mixed"] else 0
        read = (n - small) * e + small * 4
        return {"bytes": read + (read if c["out"] == "same" else 4 * n), "flops": 3 * n}
    n, d = c["b"] * c["s"], c["dim"]
    if c["op"] == "embed":
        rows, _ = _shard(c)
        seen = float((1 - (1 - _token_frequencies(c["vocab"])) ** n).sum()) / c["shards"]
        pos = _positions_rows(c) if c["positions"] != "none" else 0
        b = 8 * n + e * d * (seen + min(pos, n) + n)
        if c["train"]:
            b += e * d * (n + rows + pos)
        return {"bytes": int(b), "flops": n * d * (4 if c["train"] else 2)}
    gate = {"none": 0, "channel": d, "sample": c["b"] * d, "full": n * d}[c["gate"]]
    vectors = 4 * d * size[c["wdtype"]]
    if not c["train"]:
        return {"bytes": 4 * n * d * e + gate * e + vectors, "flops": 14 * n * d}
    return {"bytes": 8 * n * d * e + 2 * gate * e + 2 * vectors, "flops": 45 * n * d}


# -------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    st, c = prepare(case, seed), case
    if c["op"] == "embed":
        # forward by selecting rows of the tables with the shard's ids put at its end for the
        # others', gradients by adding up the rows of each token's group
        w, start = st["weight"].detach().double(), st["vocab_start"] or 0
        rows, flat = w.shape[0], st["ids"].reshape(-1) - start
        flat = torch.where((flat < 0) | (flat >= rows), torch.full_like(flat, rows), flat)
        y = c["scale"] * torch.cat([w, w.new_zeros(1, w.shape[1])]).index_select(0, flat)
        place = None
        if st["position_weight"] is not None:
            place = st["position_ids"] if st["position_ids"] is not None else torch.arange(c["s"], device=w.device).repeat(c["b"], 1)
            place = place.reshape(-1)
            y += st["position_weight"].detach().double().index_select(0, place)
        outs = [y.view(c["b"], c["s"], -1)]
        if c["train"]:
            dy = st["dy"].double().view(-1, c["dim"])

            def groups(keys, n):
                order = torch.argsort(keys, stable=True)
                got, count = torch.unique_consecutive(keys[order], return_counts=True)
                sums = torch.segment_reduce(dy[order], "sum", lengths=count, axis=0)
                return dy.new_zeros(n + 1, c["dim"]).index_copy_(0, got, sums)[:n]

            keys = flat
            if st["padding_idx"] is not None:
                keys = torch.where(flat == st["padding_idx"] - start, torch.full_like(flat, rows), flat)
            outs.append(c["scale"] * groups(keys, rows))
            if place is not None:
                outs.append(groups(place, st["position_weight"].shape[0]))
        return outs
    if c["op"] == "block":
        names = [k for k in ("x", "residual", "weight", "bias", "post_weight", "post_bias", "gate") if st[k] is not None]
        v = {k: st[k].detach().double().requires_grad_(c["train"]) for k in names}

        def norm(t, w, b):
            center = t if c["kind"] == "rms" else t - t.mean(-1, keepdim=True)
            out = center / (center.pow(2).mean(-1, keepdim=True) + _EPS).sqrt() * v[w]
            return out + v[b] if b in v else out

        h = norm(v["x"], "post_weight", "post_bias") if c["post"] else v["x"]
        s = v["residual"] + c["alpha"] * (h * v["gate"] if "gate" in v else h)
        y = norm(s, "weight", "bias")
        outs = [y.detach(), s.detach()]
        if c["train"]:
            outs += torch.autograd.grad([y, s], [v[k] for k in names], [st["dy"].double(), st["ds"].double()])
        return outs
    most, total = 0.0, 0.0
    for t in st["grads"]:
        u = c["scale"] * t.double().flatten()
        most, total = max(most, float(u.abs().max())), total + float(u.dot(u))
    norm = math.sqrt(total) if c["p"] == "2" else most
    f = min(1.0, st["max_norm"] / (norm + 1e-6))
    flat = {}
    for t, o in zip(st["grads"], st["out"]):
        clipped = torch.nn.functional.pad(t.double().flatten() * (c["scale"] * f), (0, -t.numel() % 64))
        flat.setdefault(o.dtype, []).append(clipped)
    return [torch.tensor(norm, dtype=torch.float64), *[torch.cat(parts) for parts in flat.values()]]
