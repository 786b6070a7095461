"""Cases and plain forms of the transformer training operators.

Three operators that follow one another on a transformer's path: the token
embedding (lookup with a scale, gradient by sorted tokens), the RMS norm of
queries and keys for each head with the position rotation in the same pass,
and attention with a sliding window and first tokens that stay visible.

    listed()            the cases that are measured
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program has in hand before the call, on the GPU
    run(state)          one pass: the plain form, or the framework's call
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the definition in 64 bits
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16,
          "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
_EPS = 1e-6


# ---- cases ----------------------------------------------------------------

def listed():
    return [
        # a handful of token ids at evaluation: what counts is latency
        {"name": "embed_few", "op": "embed", "train": False, "batch": 1,
         "seq": 5, "vocab": 30522, "hidden": 768, "weight": "bf16",
         "out": "bf16", "scaled": False, "padding": False},
        # BERT-base's training step: f32 weights, bf16 activations
        {"name": "embed_step", "op": "embed", "train": True, "batch": 32,
         "seq": 128, "vocab": 30522, "hidden": 768, "weight": "fp32",
         "out": "bf16", "scaled": False, "padding": False},
        # long padded sequences, a scaled embedding, odd width and vocabulary
        {"name": "embed_padded_odd", "op": "embed", "train": True,
         "batch": 7, "seq": 2045, "vocab": 32003, "hidden": 517,
         "weight": "fp16", "out": "fp16", "scaled": True, "padding": True},
        # the largest: 64k tokens a step in bf16
        {"name": "embed_large", "op": "embed", "train": True, "batch": 16,
         "seq": 4096, "vocab": 50000, "hidden": 1024, "weight": "bf16",
         "out": "bf16", "scaled": True, "padding": False},
        # one new token of each of 8 sequences, each at its own far position
        {"name": "qk_one_token", "op": "qk", "train": False, "batch": 8,
         "seq": 1, "q_heads": 16, "k_heads": 4, "dim": 128, "type": "fp16",
         "weight": "fp32", "positions": "each", "table": 40960},
        # BERT-base's training step
        {"name": "qk_step", "op": "qk", "train": True, "batch": 32,
         "seq": 128, "q_heads": 12, "k_heads": 12, "dim": 64,
         "type": "bf16", "weight": "fp32", "positions": "row",
         "table": 512},
        # long sequences with shared key heads
        {"name": "qk_long", "op": "qk", "train": True, "batch": 2,
         "seq": 8192, "q_heads": 32, "k_heads": 8, "dim": 128,
         "type": "bf16", "weight": "bf16", "positions": "row",
         "table": 8192},
        # one new token of 16 sequences over all their earlier keys
        {"name": "attn_one_token", "op": "attn", "train": False,
         "batch": 16, "rows": 1, "keys": 16000, "q_heads": 32,
         "k_heads": 8, "dim": 128, "type": "bf16", "window": 0, "sinks": 0,
         "causal": True, "ragged": True},
        # BERT-base's training step with local attention in both directions
        # and a first token that all see
        {"name": "attn_step_local", "op": "attn", "train": True,
         "batch": 32, "rows": 128, "keys": 128, "q_heads": 12,
         "k_heads": 12, "dim": 64, "type": "bf16", "window": 32,
         "sinks": 1, "causal": False, "ragged": False},
        # evaluation of a padded batch of odd lengths
        {"name": "attn_padded", "op": "attn", "train": False, "batch": 6,
         "rows": 1999, "keys": 1999, "q_heads": 12, "k_heads": 12,
         "dim": 64, "type": "fp16", "window": 257, "sinks": 3,
         "causal": True, "ragged": True},
        # a training step without a window
        {"name": "attn_full", "op": "attn", "train": True, "batch": 4,
         "rows": 2048, "keys": 2048, "q_heads": 16, "k_heads": 16,
         "dim": 64, "type": "bf16", "window": 0, "sinks": 0,
         "causal": True, "ragged": False},
        # the largest: a long sequence, shared key heads, window and sinks
        {"name": "attn_long", "op": "attn", "train": True, "batch": 1,
         "rows": 8192, "keys": 8192, "q_heads": 32, "k_heads": 8,
         "dim": 128, "type": "bf16", "window": 1024, "sinks": 4,
         "causal": True, "ragged": False},
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low),
                                              math.log(high + 1)))))


def draw(rng):
    op = rng.choice(["embed", "qk", "attn", "attn"])
    if op == "embed":
        seq = _spread(rng, 1, 4096)
        weight = rng.choice(["fp32", "bf16", "fp16"])
        return {"op": op, "train": rng.random() < 0.7,
                "batch": _spread(rng, 1, max(1, min(64, 65536 // seq))),
                "seq": seq, "vocab": _spread(rng, 1000, 50000),
                "hidden": (_spread(rng, 64, 1024) if rng.random() < 0.3
                           else 8 * _spread(rng, 8, 128)),
                "weight": weight,
                "out": "bf16" if weight == "fp32" and rng.random() < 0.6
                else weight,
                "scaled": rng.random() < 0.5, "padding": rng.random() < 0.5}
    k_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = k_heads * rng.choice([1, 2, 3, 4])
    if op == "qk":
        seq = _spread(rng, 1, 8192)
        return {"op": op, "train": rng.random() < 0.7,
                "batch": _spread(rng, 1, max(1, min(64, 16384 // seq))),
                "seq": seq, "q_heads": q_heads, "k_heads": k_heads,
                "dim": rng.choice([32, 64, 80, 96, 128]),
                "type": rng.choice(["fp32", "bf16", "fp16"]),
                "weight": "fp32", "positions": rng.choice(["row", "each"]),
                "table": seq + _spread(rng, 1, 32768)}
    train = rng.random() < 0.6
    rows = _spread(rng, 1, 4096)
    keys = rows
    if not train and rng.random() < 0.6:
        rows = min(rows, _spread(rng, 1, 64))
        keys = rows + _spread(rng, 1, 16000)
    most = max(1, min(32, (1 << 30) // (q_heads * rows * keys)))
    return {"op": op, "train": train, "batch": _spread(rng, 1, most),
            "rows": rows, "keys": keys, "q_heads": q_heads,
            "k_heads": k_heads, "dim": rng.choice([32, 64, 64, 80, 128, 128]),
            "type": rng.choice(["bf16", "bf16", "fp16"]),
            "window": rng.choice([0, _spread(rng, 1, 2048),
                                  _spread(rng, 1, 2048)]),
            "sinks": rng.choice([0, 1, 4, _spread(rng, 1, 200)]),
            "causal": rng.random() < 0.7, "ragged": rng.random() < 0.5}


# ---- inputs ---------------------------------------------------------------

def _lengths(case):
    """Keys that each sequence has: all, or a ragged batch's."""
    n, top = case["batch"], case["keys"]
    if not case["ragged"]:
        return [top] * n
    low = case["rows"] if case["rows"] < top else 1
    return [max(low, top - (b * 7919 + n) % max(1, (2 * top) // 3))
            for b in range(n)]


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = dict(case)
    if case["op"] == "embed":
        b, s, v, h = (case[n] for n in ("batch", "seq", "vocab", "hidden"))
        # token frequencies of text fall about as one over their rank
        u = torch.rand((b, s), generator=gen, device="cuda",
                       dtype=torch.float64)
        ids = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        mix = torch.randperm(v, generator=gen, device="cuda")
        ids = mix[ids]
        state["padding_idx"] = None
        if case["padding"]:  # each sequence ends in a run of one id
            state["padding_idx"] = 1
            ends = torch.randint(1, s + 1, (b, 1), generator=gen,
                                 device="cuda")
            past = torch.arange(s, device="cuda") >= ends
            ids = torch.where(past, torch.ones_like(ids), ids)
        state["ids"] = ids
        state["weight"] = _normal(gen, (v, h), _TYPES[case["weight"]], 0.02)
        state["scale"] = math.sqrt(h) if case["scaled"] else 1.0
        if case["train"]:
            state["weight"].requires_grad_(True)
            state["dout"] = _normal(gen, (b, s, h), _TYPES[case["out"]])
        return state
    hq, hk, d = case["q_heads"], case["k_heads"], case["dim"]
    dtype = _TYPES[case["type"]]
    if case["op"] == "qk":
        b, s = case["batch"], case["seq"]
        qkv = _normal(gen, (b, s, hq + 2 * hk, d), dtype)  # one projection's
        state["q"], state["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
        for n in ("q_weight", "k_weight"):
            state[n] = (1.0 + 0.1 * torch.randn(
                d, generator=gen, device="cuda")).to(_TYPES[case["weight"]])
        state["positions"] = None
        if case["positions"] == "each":
            start = torch.randint(0, case["table"] - s + 1, (b, 1),
                                  generator=gen, device="cuda")
            state["positions"] = start + torch.arange(s, device="cuda")
        angles = torch.arange(case["table"], device="cuda",
                              dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, d, 2, device="cuda",
                                   dtype=torch.float64) / d)
        state["rope"] = torch.cat([angles.cos(), angles.sin()], 1).float()
        if case["train"]:
            for n in ("q", "k", "q_weight", "k_weight"):
                state[n] = state[n].detach().requires_grad_(True)
            state["dq"] = _normal(gen, (b, s, hq, d), dtype)
            state["dk"] = _normal(gen, (b, s, hk, d), dtype)
        return state
    b, s, t = case["batch"], case["rows"], case["keys"]
    state["q"] = _normal(gen, (b, s, hq, d), dtype)
    if s == t:  # keys and values of one projection
        state["k"] = _normal(gen, (b, t, hk, d), dtype)
        state["v"] = _normal(gen, (b, t, hq + 2 * hk, d), dtype)[
            :, :, hq + hk:]
    else:  # held for each head
        state["k"] = _normal(gen, (b, hk, t, d), dtype).transpose(1, 2)
        state["v"] = _normal(gen, (b, hk, t, d), dtype).transpose(1, 2)
    state["lengths"] = state["starts"] = None
    if case["ragged"]:
        state["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32,
                                        device="cuda")
        if s != t:  # the rows are the last ones of each sequence
            state["starts"] = state["lengths"] - s
    if case["train"]:
        for n in ("q", "k", "v"):
            state[n] = state[n].detach().requires_grad_(True)
        state["dout"] = _normal(gen, (b, s, hq, d), dtype)
    return state


# ---- one pass -------------------------------------------------------------

def run(state):
    if state["op"] == "embed":
        return _run_embed(state)
    if state["op"] == "qk":
        return _run_qk(state)
    return _run_attn(state)


def _run_embed(state):
    ids, weight, scale = state["ids"], state["weight"], state["scale"]
    out_type, pad = _TYPES[state["out"]], state["padding_idx"]
    if own:
        from kungfu_amd.ops.fused_embedding import embedding

        out = embedding(ids, weight, scale=scale, padding_idx=pad,
                        out_dtype=out_type)
        if not state["train"]:
            return out
        return (out,) + torch.autograd.grad(out, weight, state["dout"])
    with torch.no_grad():
        out = (weight[ids].float() * scale).to(out_type)
        if not state["train"]:
            return out
        grad = torch.zeros(weight.shape, device=weight.device)
        grad.index_add_(0, ids.reshape(-1),
                        state["dout"].reshape(-1, weight.shape[1]).float())
        grad *= scale
        if pad is not None:
            grad[pad] = 0.0
        return out, grad.to(weight.dtype)


def _plain_norm_rope(x, w, rope, positions):
    x, half = x.float(), x.shape[-1] // 2
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    at = rope[:x.shape[1]] if positions is None else rope[positions]
    cos, sin = at[..., None, :half], at[..., None, half:]
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _run_qk(state):
    q, k, qw, kw = (state[n] for n in ("q", "k", "q_weight", "k_weight"))
    rope, positions = state["rope"], state["positions"]
    if own:
        from kungfu_amd.ops.qk_norm_rope import qk_norm_rope

        oq, ok = qk_norm_rope(q, k, qw, kw, rope, positions=positions,
                              eps=_EPS)
    else:
        oq = _plain_norm_rope(q, qw, rope, positions).to(q.dtype)
        ok = _plain_norm_rope(k, kw, rope, positions).to(k.dtype)
    if not state["train"]:
        return oq, ok
    return (oq, ok) + torch.autograd.grad(
        (oq, ok), (q, k, qw, kw), (state["dq"], state["dk"]))


def _plain_attention(state):
    q, k, v = (state[n].float().transpose(1, 2).contiguous()
               for n in ("q", "k", "v"))
    (b, hq, s, d), (hk, t) = q.shape, k.shape[1:3]
    at = torch.arange(s, device=q.device)
    j = torch.arange(t, device=q.device)
    starts, lengths = state["starts"], state["lengths"]
    p = (at + (t - s)).expand(b, s) if starts is None else \
        starts.long()[:, None] + at
    n = torch.full((b,), t, device=q.device) if lengths is None else lengths
    p, n = p[:, :, None], n[:, None, None]
    seen = (j < n) & (p < n)
    if state["window"]:
        seen = seen & (((p - j).abs() < state["window"]) |
                       (j < state["sinks"]))
    if state["causal"]:
        seen = seen & (j <= p)
    seen = seen[:, None, None]  # over the heads
    q = q.view(b, hk, hq // hk, s, d)
    scores = torch.matmul(q, k.transpose(-1, -2)[:, :, None].contiguous())
    scores = (scores * (d ** -0.5)).masked_fill(~seen, -math.inf)
    top = scores.detach().amax(-1, keepdim=True).clamp_min(-1e30)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, v[:, :, None]) / \
        torch.where(total == 0, torch.ones_like(total), total)
    return out.reshape(b, hq, s, d).transpose(1, 2).contiguous()


def _run_attn(state):
    q, k, v = state["q"], state["k"], state["v"]
    if own:
        from kungfu_amd.ops.window_attention import window_attention

        out = window_attention(q, k, v, window=state["window"] or None,
                               sinks=state["sinks"], causal=state["causal"],
                               lengths=state["lengths"],
                               starts=state["starts"])
    else:
        out = _plain_attention(state).to(q.dtype)
    if not state["train"]:
        return out
    return (out,) + torch.autograd.grad(out, (q, k, v), state["dout"])


# ---- what a pass cannot do without ----------------------------------------

def _visible(case):
    """(query, key) pairs that the mask leaves, and keys that any row sees,
    summed over the batch."""
    pairs = keys = 0
    w, sinks = case["window"], case["sinks"]
    for n in _lengths(case):
        start = n - case["rows"] if case["rows"] != case["keys"] else 0
        p = np.arange(start, start + case["rows"])
        p = p[p < n]
        hi = np.full_like(p, n) if not w else np.minimum(p + w, n)
        if case["causal"]:
            hi = np.minimum(hi, p + 1)
        lo = np.zeros_like(p) if not w else np.maximum(p - w + 1, 0)
        total = hi - lo
        if w:
            first = min(sinks, n)
            total = total + np.minimum(first, lo)
            if not case["causal"]:
                total = total + np.maximum(first - hi, 0)
        pairs += int(total.sum())
        if len(p):
            keys += int(min(n, hi.max() - lo.min() +
                            (min(sinks, lo.min()) if w else 0)))
    return pairs, keys


def work(case):
    if case["op"] == "embed":
        n, h = case["batch"] * case["seq"], case["hidden"]
        ws, os = _SIZE[case["weight"]], _SIZE[case["out"]]
        size = n * 8 + min(n, case["vocab"]) * h * ws + n * h * os
        flops = n * h
        if case["train"]:
            size += n * h * os + case["vocab"] * h * ws
            flops += 2 * n * h
        return {"bytes": size, "flops": flops}
    if case["op"] == "qk":
        rows = case["batch"] * case["seq"]
        n = rows * (case["q_heads"] + case["k_heads"]) * case["dim"]
        size = _SIZE[case["type"]]
        table = case["seq"] if case["positions"] == "row" else rows
        return {"bytes": (5 if case["train"] else 2) * n * size +
                min(table, case["table"]) * case["dim"] * 4,
                "flops": (24 if case["train"] else 8) * n}
    pairs, keys = _visible(case)
    size, d = _SIZE[case["type"]], case["dim"]
    q = case["batch"] * case["rows"] * case["q_heads"] * d
    kv = 2 * keys * case["k_heads"] * d
    moved = 2 * q + kv
    if case["train"]:  # and dout, dq, dk, dv
        moved += 2 * q + 2 * case["batch"] * case["keys"] * \
            case["k_heads"] * d
    return {"bytes": moved * size,
            "flops": (14 if case["train"] else 4) * pairs * d *
            case["q_heads"]}


# ---- the definition in 64 bits --------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embed":
            return _exact_embed(state)
        if case["op"] == "qk":
            return _exact_qk(state)
        return _exact_attn(case, state)


def _exact_embed(state):
    ids, weight = state["ids"], state["weight"].detach()
    out = weight.double().index_select(0, ids.flatten()) * state["scale"]
    out = out.view(*ids.shape, -1)
    if not state["train"]:
        return out
    # sum of the rows of each token: differences of running sums over the
    # rows in the order of their tokens, which 64 bits carry
    flat = ids.flatten()
    order = torch.argsort(flat)
    rows = state["dout"].flatten(0, 1).double().index_select(0, order)
    sums = torch.cat([torch.zeros_like(rows[:1]), rows.cumsum(0)])
    ends = torch.bincount(flat, minlength=weight.shape[0]).cumsum(0)
    grad = sums[ends]
    grad[1:] -= sums[ends[:-1]]
    grad *= state["scale"]
    if state["padding_idx"] is not None:
        grad[state["padding_idx"]] = 0.0
    return out, grad


def _exact_qk(state):
    outs, grads, weights = [], [], []
    for n in ("q", "k"):
        x = state[n].detach().double()
        w = state[n + "_weight"].detach().double()
        b, s, _, d = x.shape
        pos = state["positions"]
        if pos is None:
            pos = torch.arange(s, device=x.device).expand(b, s)
        angle = pos.double()[..., None] * 10000.0 ** (
            -2.0 * torch.arange(d // 2, device=x.device).double() / d)
        turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
        r = (x.square().sum(-1, keepdim=True) / d + _EPS).rsqrt()
        z = torch.complex(*(x * r * w).chunk(2, -1)) * turn
        outs.append(torch.cat([z.real, z.imag], -1))
        if not state["train"]:
            continue
        g = torch.complex(*state["d" + n].double().chunk(2, -1)) * \
            turn.conj()
        g = torch.cat([g.real, g.imag], -1)
        weights.append((g * x * r).sum((0, 1, 2)))
        g = g * w
        grads.append(r * g - x * r ** 3 * (g * x).sum(-1, keepdim=True) / d)
    return tuple(outs + grads + weights)


def _exact_attn(case, state):
    q, k, v = (state[n].detach() for n in ("q", "k", "v"))
    (b, s, hq, d), (t, hk) = q.shape, k.shape[1:3]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    dq = torch.zeros_like(out)
    dk = torch.zeros(k.shape, dtype=torch.float64, device=q.device)
    dv = torch.zeros_like(dk)
    i = torch.arange(s, device=q.device)[:, None]
    j = torch.arange(t, device=q.device)[None, :]
    for bi, n in enumerate(_lengths(case)):
        pos = i + ((n - s) if s != t else 0)
        dist = pos - j
        hide = (j >= n) | (pos >= n)
        if case["window"]:
            hide |= (dist.abs() >= case["window"]) & (j >= case["sinks"])
        if case["causal"]:
            hide |= dist < 0
        empty = hide.all(1, keepdim=True)
        for h in range(hq):
            g = h * hk // hq
            qh, kh, vh = (x.double() for x in (q[bi, :, h], k[bi, :, g],
                                               v[bi, :, g]))
            a = (qh @ kh.T) / math.sqrt(d)
            a[hide] = -math.inf
            a = torch.softmax(a, 1)
            a = torch.where(empty, torch.zeros_like(a), a)
            o = out[bi, :, h] = a @ vh
            if case["train"]:
                do = state["dout"][bi, :, h].double()
                dv[bi, :, g] += a.T @ do
                da = a * (do @ vh.T - (do * o).sum(1, keepdim=True))
                da /= math.sqrt(d)
                dq[bi, :, h] = da @ kh
                dk[bi, :, g] += da.T @ qh
    if not case["train"]:
        return out
    return out, dq, dk, dv
