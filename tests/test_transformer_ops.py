"""Embedding, query/key norm with rotation and window attention.

Each is compared with its definition in 64 bits. The tolerances are bounds,
element by element, of what the documented roundings can do: a value
rounded to a type is off by at most half a step, finfo.eps / 2 of itself,
and an f32 sum of n terms by n * 2^-24 of the sum of their magnitudes.
CPU tensors take the eager path, CUDA tensors the kernels.
"""
import math

import pytest
import torch

from kungfu_amd.ops.fused_embedding import FusedEmbedding, embedding
from kungfu_amd.ops.qk_norm_rope import (QKNormRope, qk_norm_rope,
                                         rope_table)
from kungfu_amd.ops.window_attention import window_attention

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
F32 = 2.0 ** -24
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def inside(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    # subnormals of the type round by an absolute step
    over = (got - want).abs() - bound - 1e-7
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, "%s: %.3g over its bound" % (what, worst)


def randn(gen, shape, dtype, device):
    return torch.randn(shape, generator=gen).to(dtype).to(device)


# ---- embedding ------------------------------------------------------------

def embed_oracle(ids, weight, scale, pad, dout):
    """out, dW, and the sums of magnitudes and row counts behind dW."""
    w, g = weight.detach().double().cpu(), dout.double().cpu()
    flat, g = ids.cpu().reshape(-1).long(), g.reshape(-1, w.shape[1])
    out = (w[flat] * scale).reshape(*ids.shape, -1)
    dw, mag = torch.zeros_like(w), torch.zeros_like(w)
    n = torch.zeros(w.shape[0], 1, dtype=torch.float64)
    for i, t in enumerate(flat.tolist()):
        if t != pad:
            dw[t] += g[i] * scale
            mag[t] += g[i].abs() * scale
            n[t] += 1
    return out, dw, mag, n


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("weight_t,out_t", [
    (FP32, FP32), (FP32, BF16), (FP32, F16), (BF16, BF16), (F16, F16),
    (BF16, FP32)])
@pytest.mark.parametrize("shape,vocab,hidden,spread", [
    ((1,), 1, 1, 1), ((3, 5), 7, 8, 7), ((2, 129), 300, 517, 300),
    ((4, 300), 65537, 24, 3), ((2500,), 1000, 40, 1),
    ((9, 1100), 255, 520, 255)])
def test_embedding(device, weight_t, out_t, shape, vocab, hidden, spread):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, spread, shape, generator=gen).to(device)
    w = randn(gen, (vocab, hidden), weight_t, device).requires_grad_(True)
    pad = 2 if vocab > 2 else None
    scale = math.sqrt(hidden)
    out = embedding(ids, w, scale, pad, out_t)
    dout = randn(gen, out.shape, out_t, device)
    dw, = torch.autograd.grad(out, w, dout)
    assert out.dtype == out_t and dw.dtype == weight_t
    want, dwant, mag, n = embed_oracle(ids, w, scale, pad, dout)
    inside(out, want, (half_step(out_t) + 3 * F32) * want.abs(), "out")
    if device == "cpu" and weight_t != FP32:
        # eager autograd adds the rows of a token in the weight's type
        return
    inside(dw, dwant, half_step(weight_t) * dwant.abs() +
           (n + 4) * F32 * 2 * mag, "dw")


@gpu
def test_embedding_rows_and_strides():
    """A weight that is a slice of wider rows, ids that are a transposed
    int32 view, and rows that are not 16-byte aligned."""
    gen = torch.Generator().manual_seed(2)
    for width, off in ((64, 0), (64, 3), (37, 5)):
        store = randn(gen, (90, width + 16), BF16, "cuda")
        w = store[:, off:off + width]
        ids = torch.randint(0, 90, (11, 13), generator=gen,
                            dtype=torch.int32).cuda().t()
        got = embedding(ids, w)
        assert torch.equal(got, w[ids.long()])


@gpu
@pytest.mark.parametrize("n", [0, 1, 31, 4095, 4096, 4097, 70001])
def test_embedding_gradient_of_whole_numbers(n):
    """Small whole numbers add without rounding in f32: the gradient is
    then exact whatever the order, whole chunks of one token among them."""
    gen = torch.Generator().manual_seed(n)
    for vocab, hot in ((5, 0.0), (3000, 0.6), (200000, 0.3)):
        ids = torch.randint(0, vocab, (n,), generator=gen)
        ids[torch.rand(n, generator=gen) < hot] = vocab // 2
        w = torch.zeros(vocab, 16, device="cuda", requires_grad=True)
        d = torch.randint(-3, 4, (n, 16), generator=gen).float().cuda()
        dw, = torch.autograd.grad(embedding(ids.cuda(), w), w, d)
        want = torch.zeros(vocab, 16, dtype=torch.float64)
        want.index_add_(0, ids, d.double().cpu())
        assert torch.equal(dw.double().cpu(), want)


@gpu
def test_embedding_ids_outside_the_table():
    w = torch.randn(10, 16, device="cuda", requires_grad=True)
    ids = torch.tensor([0, -1, 9, 10, 1 << 40, 3], device="cuda")
    out = embedding(ids, w)
    bad = torch.isnan(out).all(1).cpu()
    assert bad.tolist() == [False, True, False, True, True, False]
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    want = torch.zeros(10, 16)
    want[[0, 3, 9]] = 1
    assert torch.equal(dw.cpu(), want)


def test_embedding_refusals():
    w = torch.randn(10, 8)
    ids = torch.tensor([1, 2])
    with pytest.raises(TypeError):
        embedding(ids.float(), w)
    with pytest.raises(ValueError):
        embedding(ids, w[0])
    with pytest.raises(ValueError):
        embedding(ids, w, padding_idx=10)
    with pytest.raises(IndexError):
        embedding(torch.tensor([10]), w)
    with pytest.raises(ValueError):
        FusedEmbedding(10, 8, max_norm=1.0)
    with pytest.raises(ValueError):
        embedding(ids, torch.empty(2, 8, device="meta"))


def test_fused_embedding_module():
    m = FusedEmbedding(20, 8, padding_idx=3, scale=2.0)
    ids = torch.tensor([[1, 3], [4, 1]])
    out = m(ids)
    assert torch.equal(out, m.weight[ids] * 2.0)
    out.sum().backward()
    assert torch.equal(m.weight.grad[3], torch.zeros(8))
    assert torch.equal(m.weight.grad[1], torch.full((8,), 4.0))


# ---- query/key norm and rotation ------------------------------------------

def qk_oracle(x, w, rope, at, eps, dy):
    """y, dx, dw and their magnitudes for one of q and k."""
    x, dy = x.detach().double().cpu(), dy.double().cpu()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else \
        w.detach().double().cpu()
    if rope is None:
        c, s = (torch.full((1, 1, 1, D // 2), v, dtype=torch.float64)
                for v in (1.0, 0.0))
    else:
        c, s = rope.double().cpu()[at][:, :, None].chunk(2, -1)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    lo, hi = (x * r * w).chunk(2, -1)
    y = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    ymag = torch.cat([(lo * c).abs() + (hi * s).abs(),
                      (hi * c).abs() + (lo * s).abs()], -1)
    a, b = dy.chunk(2, -1)
    g = torch.cat([a * c + b * s, b * c - a * s], -1)
    gmag = torch.cat([(a * c).abs() + (b * s).abs(),
                      (b * c).abs() + (a * s).abs()], -1)
    h, hmag = g * w, gmag * w.abs()
    dx = r * h - x * r ** 3 * (h * x).mean(-1, keepdim=True)
    dxmag = r * hmag + x.abs() * r ** 3 * (hmag * x.abs()).mean(
        -1, keepdim=True)
    dw = (g * x * r).sum((0, 1, 2))
    return y, ymag, dx, dxmag, dw, (gmag * x.abs() * r).sum((0, 1, 2))


def qk_check(q, k, qw, kw, rope, positions, start, eps=1e-6):
    gen = torch.Generator().manual_seed(7)
    given = [t for t in (q, k, qw, kw) if t is not None]
    for t in given:
        t.requires_grad_(True)
    outs = qk_norm_rope(q, k, qw, kw, rope, positions, start, eps)
    dys = [randn(gen, o.shape, q.dtype, q.device) for o in outs]
    grads = iter(torch.autograd.grad(outs, given, dys))
    dx = [next(grads), next(grads)]
    dw = [None if w is None else next(grads) for w in (qw, kw)]
    B, S, _, D = q.shape
    at = torch.arange(start, start + S).expand(B, S) if positions is None \
        else positions.cpu().long().expand(B, S)
    u, e = half_step(q.dtype), (2 * D + 64) * F32
    for i, (x, w) in enumerate(((q, qw), (k, kw))):
        y, ymag, gx, gmag, gw, wmag = qk_oracle(x, w, rope, at, eps, dys[i])
        inside(outs[i], y, u * y.abs() + e * ymag, "y")
        inside(dx[i], gx, u * gx.abs() + 2 * e * gmag, "dx")
        if w is not None:
            n = B * S * x.shape[2]
            inside(dw[i], gw, half_step(w.dtype) * gw.abs() +
                   (e + n * F32) * wmag, "dw")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,weight_t", [(FP32, FP32), (BF16, FP32),
                                            (BF16, BF16), (F16, FP32)])
@pytest.mark.parametrize("B,S,Hq,Hk,D", [
    (1, 1, 1, 1, 2), (2, 3, 4, 2, 16), (1, 5, 3, 1, 10), (2, 67, 12, 12, 64),
    (1, 33, 32, 8, 128), (3, 9, 6, 2, 80), (2, 5, 5, 5, 512),
    (1, 700, 2, 1, 96)])
def test_qk_norm_rope(device, dtype, weight_t, B, S, Hq, Hk, D):
    gen = torch.Generator().manual_seed(3)
    qkv = randn(gen, (B, S, Hq + 2 * Hk, D), dtype, device)
    q, k = qkv[:, :, :Hq].detach(), qkv[:, :, Hq:Hq + Hk].detach()
    qw = (1 + 0.2 * torch.randn(D, generator=gen)).to(weight_t).to(device)
    kw = (1 + 0.2 * torch.randn(D, generator=gen)).to(weight_t).to(device)
    if device == "cpu" and weight_t == BF16:
        kw = qw = None  # eager autograd adds a bf16 weight's rows in steps
    rope = rope_table(S + 1000, D, device=device)
    qk_check(q, k, qw, kw, rope, None, 11)
    at = torch.randint(0, S + 1000, (B, S), generator=gen).to(device)
    qk_check(q, k, qw, kw, rope, at, 0)
    qk_check(q, k, qw, kw, rope, at[0].int(), 0)
    qk_check(q, k, None, kw, None, None, 0)


@gpu
@pytest.mark.parametrize("off", [1, 4, 8])
def test_qk_norm_rope_strides(off):
    """Rows that start anywhere, heads and tokens in another order, and a
    broadcast key head."""
    gen = torch.Generator().manual_seed(4)
    store = randn(gen, (2, 6, 21, 64 + off + 7), BF16, "cuda")
    q = store.transpose(1, 2)[..., off:off + 64].detach()
    one = randn(gen, (2, 21, 1, 64), BF16, "cuda")
    k = one.expand(2, 21, 6, 64).detach()
    rope = rope_table(64, 64, device="cuda")
    qk_check(q, k, None, None, rope, None, 0)
    w = torch.randn(64 + off, device="cuda")[off:].detach()
    qk_check(q, k, w, w.clone(), rope, None, 2)


def test_rope_table_far_positions():
    """Angles of far positions keep their fraction: against 64 bits."""
    t = rope_table(200001, 64)[200000].double()
    inv = [10000.0 ** (-2 * i / 64) for i in range(32)]
    want = torch.tensor([math.cos(200000 * f) for f in inv] +
                        [math.sin(200000 * f) for f in inv],
                        dtype=torch.float64)
    # 200000 * inv is off by a few 2^-53 of 200000 at most, 1e-10
    assert float((t - want).abs().max()) < 2.0 ** -24 + 1e-9


@gpu
def test_qk_positions_outside_the_table():
    q = torch.randn(1, 4, 2, 32, device="cuda")
    rope = rope_table(8, 32, device="cuda")
    at = torch.tensor([7, 8, -1, 0], device="cuda")
    y, _ = qk_norm_rope(q, q, rope=rope, positions=at)
    bad = torch.isnan(y).all(-1).all(-1)[0].tolist()
    assert bad == [False, True, True, False]
    assert torch.isfinite(y[0, [0, 3]]).all()


def test_qk_refusals():
    q, rope = torch.randn(1, 4, 2, 32), rope_table(8, 32)
    bad = [
        (ValueError, (q[0], q), {}),
        (ValueError, (q, q[:, :3]), {}),
        (ValueError, (q[..., :31], q[..., :31]), {}),
        (ValueError, (q, q.bfloat16()), {}),
        (ValueError, (q, q, torch.ones(31)), {}),
        (TypeError, (q, q, torch.ones(32).double()), {}),
        (ValueError, (q, q, None, None, rope[:, :30]), {}),
        (ValueError, (q, q, None, None, rope[:0]),
         {"positions": torch.arange(4)}),
        (ValueError, (q, q, None, None, rope), {"start": 5}),
        (ValueError, (q, q, None, None, rope), {"start": -1}),
        (ValueError, (q, q), {"positions": torch.arange(4)}),
        (ValueError, (q, q, None, None, rope),
         {"positions": torch.arange(3)}),
        (TypeError, (q, q, None, None, rope),
         {"positions": torch.arange(4.0)}),
        (IndexError, (q, q, None, None, rope),
         {"positions": torch.arange(4) + 5}),
        (IndexError, (q, q, None, None, rope),
         {"positions": torch.arange(4) - 1}),
    ]
    for error, args, kwargs in bad:
        with pytest.raises(error):
            qk_norm_rope(*args, **kwargs)
    with pytest.raises(ValueError):
        rope_table(8, 31)


@gpu
def test_qk_refusals_gpu():
    q = torch.randn(1, 2, 2, 514, device="cuda")
    with pytest.raises(ValueError):
        qk_norm_rope(q, q)
    with pytest.raises(TypeError):
        qk_norm_rope(q[..., :64].double(), q[..., :64].double())


@pytest.mark.parametrize("device", DEVICES)
def test_qk_gradient_by_differences(device):
    """Directional derivative of sum(dy * y) in f32: a step of 2^-6 leaves
    a third-order error of about 2^-12 and rounding of about
    2^-24 * sum|dy y| / 2^-6, together below 1 in 500 of the norm."""
    gen = torch.Generator().manual_seed(5)
    q, k = (randn(gen, (2, 5, h, 32), FP32, device).requires_grad_(True)
            for h in (4, 2))
    w = (1 + 0.2 * torch.randn(32, generator=gen)).to(device)
    w.requires_grad_(True)
    rope = rope_table(5, 32, device=device)
    dy = [randn(gen, t.shape, FP32, device) for t in (q, k)]

    def loss(q, k, w):
        y = qk_norm_rope(q, k, w, w, rope)
        return sum((a * b).double().sum() for a, b in zip(y, dy))

    grads = torch.autograd.grad(loss(q, k, w), (q, k, w))
    dirs = [randn(gen, t.shape, FP32, device) for t in (q, k, w)]
    h = 2.0 ** -6
    with torch.no_grad():
        up = loss(*(t + h * d for t, d in zip((q, k, w), dirs)))
        down = loss(*(t - h * d for t, d in zip((q, k, w), dirs)))
    slope = float((up - down) / (2 * h))
    want = sum(float((g.double() * d).sum()) for g, d in zip(grads, dirs))
    size = sum(float((g.double() * d).square().sum())
               for g, d in zip(grads, dirs)) ** 0.5
    assert abs(slope - want) < size / 20 + 1e-2


# ---- window attention -----------------------------------------------------

def mask_of(S, T, start, n, window, sinks, causal):
    p = torch.arange(start, start + S)[:, None]
    j = torch.arange(T)[None, :]
    see = (j < n) & (p >= 0) & (p < n)
    if window is not None:
        see &= ((p - j).abs() < window) | (j < sinks)
    if causal:
        see &= j <= p
    return see


def attn_oracle(q, k, v, dout, window, sinks, causal, lengths, starts,
                scale):
    """Outputs and gradients with bounds of their errors. u is the half
    step of the inputs' type: probabilities and their gradients are rounded
    to it before the second products, and each output once."""
    u = half_step(q.dtype)
    q, k, v, dout = (t.detach().double().cpu() for t in (q, k, v, dout))
    (B, S, Hq, D), (T, Hk) = q.shape, k.shape[1:3]
    res = {n: torch.zeros(t.shape, dtype=torch.float64)
           for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    bound = {n: torch.zeros_like(t) for n, t in res.items()}
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        start = T - S if starts is None else int(starts[b])
        see = mask_of(S, T, start, n, window, sinks, causal)
        rows, cols = see.any(1), see.any(0)
        for h in range(Hq):
            g = h * Hk // Hq
            qh = torch.where(rows[:, None], q[b, :, h], 0.0)
            do = torch.where(rows[:, None], dout[b, :, h], 0.0)
            kh = torch.where(cols[:, None], k[b, :, g], 0.0)
            vh = torch.where(cols[:, None], v[b, :, g], 0.0)
            x = (qh @ kh.T * scale).masked_fill(~see, -math.inf)
            top = x.amax(1, keepdim=True).clamp_min(-1e300)
            p = torch.exp(x - top)
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            o = p @ vh
            # f32 scores of exact products, exponentials and sums
            e = 6 * (D + 8) * F32 * (1 + float(
                (qh.abs() @ kh.abs().T).max() * scale)) + 2 * T * F32
            omag = p @ vh.abs()
            oerr = (u + e) * omag + u * o.abs()
            dp = do @ vh.T
            delta = (do * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            derr = (do.abs() * oerr).sum(1, keepdim=True) + \
                (D + 8) * F32 * (do.abs() @ vh.abs().T)
            dserr = (u + e) * ds.abs() + p * derr * (1 + u)
            res["out"][b, :, h] = o
            bound["out"][b, :, h] = oerr
            dq = ds @ kh * scale
            res["dq"][b, :, h] = dq
            bound["dq"][b, :, h] = scale * (
                (dserr + 2 * T * F32 * ds.abs()) @ kh.abs()) + u * dq.abs()
            res["dk"][b, :, g] += ds.T @ qh * scale
            bound["dk"][b, :, g] += scale * (
                (dserr + 2 * S * Hq * F32 * ds.abs()).T @ qh.abs())
            res["dv"][b, :, g] += p.T @ do
            bound["dv"][b, :, g] += (u + e + 2 * S * Hq * F32) * (
                p.T @ do.abs())
    for n in ("dk", "dv"):
        bound[n] += u * (res[n].abs() + bound[n])
    return res, bound


def attn_check(q, k, v, window=None, sinks=0, causal=True, lengths=None,
               starts=None, scale=None, seed=6):
    gen = torch.Generator().manual_seed(seed)
    dout = randn(gen, q.shape, q.dtype, q.device)
    at = [q.detach().requires_grad_(True), k.detach().requires_grad_(True),
          v.detach().requires_grad_(True)]
    move = [None if t is None else torch.tensor(t).to(q.device)
            for t in (lengths, starts)]
    out = window_attention(*at, window=window, sinks=sinks, causal=causal,
                           lengths=move[0], starts=move[1], scale=scale)
    grads = torch.autograd.grad(out, at, dout)
    with torch.no_grad():
        again = window_attention(*at, window=window, sinks=sinks,
                                 causal=causal, lengths=move[0],
                                 starts=move[1], scale=scale)
    assert torch.equal(out, again)
    want, bound = attn_oracle(q, k, v, dout, window, sinks, causal, lengths,
                              starts, scale or q.shape[-1] ** -0.5)
    for n, got in zip(("out", "dq", "dk", "dv"), (out,) + grads):
        inside(got, want[n], bound[n], n)
    return out, grads


SHAPES = [
    # B, S, T, Hq, Hk, D, window, sinks, causal
    (1, 1, 1, 1, 1, 8, None, 0, True),
    (2, 7, 7, 2, 1, 32, 1, 0, True),
    (2, 130, 130, 3, 3, 64, None, 0, True),
    (1, 200, 200, 4, 2, 64, None, 0, False),
    (1, 333, 333, 3, 1, 64, 50, 3, True),
    (2, 257, 257, 2, 2, 64, 33, 1, False),
    (1, 700, 700, 2, 1, 128, 100, 130, True),
    (1, 515, 515, 2, 2, 128, 64, 70, False),
    (1, 190, 190, 6, 2, 80, 65, 0, True),
    (1, 129, 129, 2, 1, 96, None, 0, False),
    (1, 64, 64, 5, 1, 40, 5, 200, True),
    (1, 1200, 1200, 1, 1, 32, 3, 2, True),
    (3, 1, 900, 8, 2, 128, None, 0, True),
    (2, 1, 900, 4, 4, 64, 65, 4, True),
    (2, 5, 300, 6, 3, 64, None, 0, True),
    (1, 40, 1500, 4, 1, 64, 200, 1, True),
    (1, 3, 70, 2, 2, 64, 4, 2, False),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,S,T,Hq,Hk,D,window,sinks,causal", SHAPES)
def test_window_attention(device, dtype, B, S, T, Hq, Hk, D, window, sinks,
                          causal):
    gen = torch.Generator().manual_seed(8)
    q = randn(gen, (B, S, Hq, D), dtype, device)
    k = randn(gen, (B, T, Hk, D), dtype, device)
    v = randn(gen, (B, T, Hk, D), dtype, device)
    attn_check(q, k, v, window, sinks, causal)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("S,T,window,sinks,causal,starts", [
    (150, 150, None, 0, False, None),
    (150, 150, 20, 2, True, None),
    (260, 260, 40, 3, False, None),
    (3, 400, None, 0, True, [397, 97, -1, -3]),
    (1, 400, 64, 2, True, [399, 99, 0, -1]),
    (200, 100, None, 0, True, [-100, 0, 50, 1 << 29]),
    (140, 400, 30, 1, True, [0, 10, 200, -50])])
def test_padded_batches(device, S, T, window, sinks, causal, starts):
    """Sequences of all lengths down to none; what lies behind them and
    queries outside them hold NaN and infinities, and neither show."""
    gen = torch.Generator().manual_seed(9)
    lengths = [T, T // 4, 1, 0]
    q = randn(gen, (4, S, 4, 64), BF16, device)
    k = randn(gen, (4, T, 2, 64), BF16, device)
    v = randn(gen, (4, T, 2, 64), BF16, device)
    for b, n in enumerate(lengths):
        start = T - S if starts is None else starts[b]
        for i in range(S):
            if not 0 <= start + i < n:
                q[b, i] = math.inf
        k[b, n:] = math.nan
        v[b, n:] = -math.inf
    out, grads = attn_check(q, k, v, window, sinks, causal, lengths, starts)
    for b, n in enumerate(lengths):
        start = T - S if starts is None else starts[b]
        for i in range(S):
            if not 0 <= start + i < n:
                assert not out[b, i].any() and not grads[0][b, i].any()
        assert not grads[1][b, n:].any() and not grads[2][b, n:].any()


@gpu
@pytest.mark.parametrize("D", [64, 128])
def test_attention_strides(D):
    """Slices of one projection, keys held for each head, a broadcast key
    head, rows that do not start at 16 bytes, reversed head order."""
    gen = torch.Generator().manual_seed(10)
    qkv = randn(gen, (2, 77, 8, D), BF16, "cuda")
    q, k, v = qkv.split([4, 2, 2], 2)
    attn_check(q, k, v, 30, 2)
    held = randn(gen, (2, 2, 77, D), BF16, "cuda").transpose(1, 2)
    attn_check(q, held, held, 30, 2)
    one = randn(gen, (2, 77, 1, D), BF16, "cuda").expand(2, 77, 2, D)
    attn_check(q, one, v, None, 0, False)
    odd = randn(gen, (2, 77, 2, D + 5), BF16, "cuda")[..., 3:3 + D]
    attn_check(q, odd, odd, 9, 1)
    moved = randn(gen, (77, 2, 4, D), BF16, "cuda").transpose(0, 1)
    attn_check(moved, k, v, 9, 1)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_extreme_scores(device):
    """Scores of some hundreds, and scores all alike."""
    gen = torch.Generator().manual_seed(11)
    q = randn(gen, (1, 96, 2, 64), BF16, device)
    k = randn(gen, (1, 96, 2, 64), BF16, device)
    v = randn(gen, (1, 96, 2, 64), BF16, device)
    attn_check(q, k, v, 40, 1, scale=1e-6)
    got = window_attention(q * 30, k * 30, v, window=1)
    assert torch.equal(got, v)  # each sees itself alone
    got = window_attention(q * 30, k * 30, v)
    assert torch.isfinite(got).all()


@gpu
def test_attention_long_rows_are_split():
    """Few rows over many keys: the keys are shared out and joined."""
    gen = torch.Generator().manual_seed(12)
    q = randn(gen, (1, 2, 4, 64), F16, "cuda")
    k = randn(gen, (1, 20011, 1, 64), F16, "cuda")
    v = randn(gen, (1, 20011, 1, 64), F16, "cuda")
    attn_check(q, k, v, None, 0)
    attn_check(q, k, v, 15000, 7, lengths=[19990], starts=[19985])
    q = randn(gen, (1, 150, 1, 128), BF16, "cuda")
    k = randn(gen, (1, 6000, 1, 128), BF16, "cuda")
    attn_check(q, k, k.clone(), None, 0)


@gpu
def test_attention_gradient_by_differences():
    """Directional derivative of the 64-bit definition by differences,
    against the kernels' gradients: f16 roundings (2^-11) of some hundred
    thousand independent terms leave well under 1 in 100."""
    gen = torch.Generator().manual_seed(13)
    q, k, v = (randn(gen, (1, 90, h, 64), F16, "cuda") for h in (4, 2, 2))
    dout = randn(gen, q.shape, F16, "cuda")
    at = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*at, window=25, sinks=2)
    grads = torch.autograd.grad(out, at, dout)
    dirs = [randn(gen, t.shape, torch.float64, "cpu") for t in at]
    # along the gradient itself too, so that the slope is not near zero
    dirs = [d + g.double().cpu() for d, g in zip(dirs, grads)]
    base = [t.detach().double().cpu() for t in at]

    def loss(sign):
        a = [t + sign * 1e-4 * d for t, d in zip(base, dirs)]
        o = window_attention(*a, window=25, sinks=2)
        return float((o * dout.double().cpu()).sum())

    slope = (loss(1) - loss(-1)) / 2e-4
    want = sum(float((g.double().cpu() * d).sum())
               for g, d in zip(grads, dirs))
    assert abs(slope - want) < 0.01 * abs(want)


def test_eager_attention_gradcheck():
    gen = torch.Generator().manual_seed(14)
    q, k, v = (torch.randn(2, 6, h, 8, generator=gen, dtype=torch.float64,
                           requires_grad=True) for h in (2, 1, 1))
    lengths = torch.tensor([6, 3])
    assert torch.autograd.gradcheck(
        lambda q, k, v: window_attention(q, k, v, window=2, sinks=1,
                                         lengths=lengths), (q, k, v))


def test_attention_refusals():
    q, k = torch.randn(2, 4, 4, 16), torch.randn(2, 6, 2, 16)
    bad = [
        ((q[0], k, k), {}),
        ((q, k, k[:, :5]), {}),
        ((q, k[:1], k[:1]), {}),
        ((q[:, :, :3], k, k), {}),
        ((q, k[..., :8], k[..., :8]), {}),
        ((q, k.half(), k), {}),
        ((q, k, k), {"window": 0}),
        ((q, k, k), {"sinks": -1}),
        ((q, k, k), {"scale": 0.0}),
        ((q, k, k), {"scale": -1.0}),
        ((q, k, k), {"scale": math.nan}),
        ((q, k, k), {"lengths": torch.tensor([1])}),
        ((k, q[:, :, :2], q[:, :, :2]), {}),  # more queries than keys
    ]
    for args, kwargs in bad:
        with pytest.raises(ValueError):
            window_attention(*args, **kwargs)
    with pytest.raises(TypeError):
        window_attention(q, k, k, lengths=torch.tensor([1.0, 2.0]))


@gpu
def test_attention_refusals_gpu():
    q = torch.randn(1, 4, 2, 64, device="cuda")
    with pytest.raises(TypeError):
        window_attention(q, q, q)
    q = q.bfloat16()
    with pytest.raises(ValueError):
        window_attention(q[..., :60], q[..., :60], q[..., :60])
    wide = torch.randn(1, 4, 2, 136, device="cuda").bfloat16()
    with pytest.raises(ValueError):
        window_attention(wide, wide, wide)
    with pytest.raises(ValueError):
        window_attention(q, q, q, lengths=torch.tensor([4]))


@pytest.mark.parametrize("device", DEVICES)
def test_attention_of_nothing(device):
    q = torch.zeros(1, 2, 2, 16, device=device, dtype=BF16)
    none = torch.zeros(1, 0, 2, 16, device=device, dtype=BF16)
    starts = torch.zeros(1, dtype=torch.int32, device=device)
    assert window_attention(none, q, q).shape == (1, 0, 2, 16)
    q.requires_grad_(True)
    out = window_attention(q, none, none, starts=starts)
    assert out.shape == q.shape and not out.any()
    dq, = torch.autograd.grad(out.float().sum(), q)
    assert not dq.any()


@gpu
def test_no_second_derivative():
    """A second differentiation is refused, not zero."""
    w = torch.randn(9, 16, device="cuda", requires_grad=True)
    ids = torch.arange(5, device="cuda")
    q = torch.randn(1, 4, 2, 32, device="cuda", requires_grad=True)
    a = torch.randn(1, 4, 2, 32, device="cuda").bfloat16()
    a.requires_grad_(True)
    for x, y in ((w, embedding(ids, w)), (q, qk_norm_rope(q, q)[0]),
                 (a, window_attention(a, a, a))):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        assert torch.isfinite(g).all()
        with pytest.raises(RuntimeError, match="second derivative"):
            g.sum().backward()


@gpu
def test_unused_outputs_and_inputs():
    """Gradients where only one of two outputs is used, where only some
    inputs want one, and where the gradient is broadcast."""
    gen = torch.Generator().manual_seed(21)
    q = randn(gen, (2, 9, 4, 32), BF16, "cuda").requires_grad_(True)
    k = randn(gen, (2, 9, 2, 32), BF16, "cuda").requires_grad_(True)
    y, z = qk_norm_rope(q, k)
    dq, dk = torch.autograd.grad(y.sum(), (q, k))
    want, = torch.autograd.grad(qk_norm_rope(q, k.detach())[0].sum(), q)
    assert torch.equal(dq, want) and not dk.any()
    v = randn(gen, (2, 9, 2, 32), BF16, "cuda")
    every = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    all_of = torch.autograd.grad(window_attention(*every).sum(), every)
    for i in range(3):
        some = [t.detach().requires_grad_(j == i)
                for j, t in enumerate(every)]
        one, = torch.autograd.grad(window_attention(*some).sum(), some[i])
        assert torch.equal(one, all_of[i])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_empty_batches(device, shape):
    """No tokens: empty outputs, and zeros for what has a gradient."""
    w = torch.randn(9, 16, device=device, requires_grad=True)
    ids = torch.zeros(shape, dtype=torch.int64, device=device)
    x = embedding(ids, w)
    dw, = torch.autograd.grad(x.sum(), w)
    assert x.shape == shape + (16,) and not dw.any()
    q = torch.zeros(*shape, 2, 32, device=device, requires_grad=True)
    a = torch.ones(32, device=device, requires_grad=True)
    y, z = qk_norm_rope(q, q, a, a, rope_table(8, 32, device=device))
    dq, da = torch.autograd.grad(y.sum() + z.sum(), (q, a))
    assert y.shape == dq.shape == q.shape and not da.any()
    h = torch.zeros(*shape, 2, 32, device=device, dtype=BF16)
    h.requires_grad_(True)
    dh, = torch.autograd.grad(window_attention(h, h, h).float().sum(), h)
    assert dh.shape == h.shape


@gpu
def test_steps_free_what_they_kept():
    a = block_inputs("cuda", BF16)
    leaves = [t for t in a if t.requires_grad]

    def step():
        torch.autograd.grad(block(*a, 4).float().sum(), leaves)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated()

    step()
    held = [step() for _ in range(4)]
    assert len(set(held)) == 1


@gpu
def test_changed_inputs_are_noticed():
    """A backward whose kept inputs were changed in place raises."""
    q = torch.randn(1, 8, 2, 32, device="cuda").bfloat16()
    x = q.clone().requires_grad_(True)
    k = q.clone()
    out = window_attention(x, k, q)
    k.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        out.float().sum().backward()


@gpu
def test_lengths_and_positions_of_any_layout():
    """int64 and int32, strided, far out of range."""
    gen = torch.Generator().manual_seed(22)
    q = randn(gen, (4, 40, 2, 64), BF16, "cuda")
    want = window_attention(q, q, q, lengths=torch.tensor(
        [40, 0, 7, 0], dtype=torch.int32, device="cuda"))
    far = torch.tensor([[1 << 40, 9], [-(1 << 40), 9], [7, 9], [0, 9]],
                       device="cuda")
    assert torch.equal(want, window_attention(q, q, q, lengths=far[:, 0]))
    starts = torch.tensor([0, 0, 0, 1 << 40], device="cuda")
    got = window_attention(q, q, q, starts=starts)
    assert torch.equal(got[:3], window_attention(q[:3], q[:3], q[:3]))
    assert not got[3].any()
    rope = rope_table(90, 64, device="cuda")
    at = torch.randint(0, 90, (40, 4), generator=gen).cuda()
    y = qk_norm_rope(q, q, rope=rope, positions=at.t())[0]
    assert torch.equal(y, qk_norm_rope(q, q, rope=rope, positions=at.t()
                                       .contiguous().int())[0])


# ---- offsets past 32 bits ----

@gpu
def test_embedding_of_a_table_past_32_bits():
    """Rows whose first element is past 2^31."""
    V, H = (1 << 21) + 77, 1024
    w = torch.zeros(V, H, dtype=BF16, device="cuda")
    ids = torch.tensor([V - 1, 5, 1 << 21, V - 1], device="cuda")
    gen = torch.Generator().manual_seed(18)
    rows = randn(gen, (3, H), BF16, "cuda")
    for i, n in enumerate((V - 1, 5, 1 << 21)):
        w[n] = rows[i]
    w.requires_grad_(True)
    out = embedding(ids, w)
    assert torch.equal(out, rows[[0, 1, 2, 0]])
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    for n, k in ((V - 1, 2), (5, 1), (1 << 21, 1)):
        assert (dw[n] == k).all()
    assert float(dw.sum(dtype=torch.float32)) == 4 * H


@gpu
def test_norm_rope_of_rows_past_32_bits():
    S, Hq, D = 140011, 120, 128
    gen = torch.Generator().manual_seed(19)
    q = torch.zeros(1, S, Hq, D, dtype=BF16, device="cuda")
    k = torch.zeros(1, S, 1, D, dtype=BF16, device="cuda")
    at = [0, S // 2, S - 1]
    for n in at:
        q[:, n] = randn(gen, (1, Hq, D), BF16, "cuda")
    rope = rope_table(S, D, device="cuda")
    q.requires_grad_(True)
    y, _ = qk_norm_rope(q, k, rope=rope)
    dq, = torch.autograd.grad(y, q, torch.ones_like(y))
    for n in at:
        few = q.detach()[:, n:n + 1].clone().requires_grad_(True)
        z, _ = qk_norm_rope(few, few[:, :, :1].detach(), rope=rope, start=n)
        assert torch.equal(z, y[:, n:n + 1])
        dz, = torch.autograd.grad(z, few, torch.ones_like(z))
        assert torch.equal(dz, dq[:, n:n + 1])


@gpu
def test_attention_of_a_cache_past_32_bits():
    """A long cache of which the window and the first tokens are seen."""
    T, H, D = (1 << 21) + 1003, 8, 128
    gen = torch.Generator().manual_seed(20)
    k = torch.full((1, T, H, D), 0.5, dtype=BF16, device="cuda")
    v = torch.full((1, T, H, D), -2.0, dtype=BF16, device="cuda")
    seen = list(range(3)) + list(range(T - 80, T))
    for t in (k, v):
        t[:, seen] = randn(gen, (1, len(seen), H, D), BF16, "cuda")
    q = randn(gen, (1, 2, 16, D), BF16, "cuda")
    dout = randn(gen, q.shape, BF16, "cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = window_attention(*leaves, window=79, sinks=3)
    grads = torch.autograd.grad(out, leaves, dout)
    # the same rows and keys alone
    few = [q.detach().clone().requires_grad_(True)] + [
        t.detach()[:, seen].clone().requires_grad_(True) for t in (k, v)]
    want, bound = attn_oracle(*few, dout, 79, 3, True, None, None,
                              D ** -0.5)
    inside(out, want["out"], bound["out"], "out")
    inside(grads[0], want["dq"], bound["dq"], "dq")
    for i, n in ((1, "dk"), (2, "dv")):
        inside(grads[i][:, seen], want[n], bound[n], n)
        assert not grads[i][:, 3:T - 80].any()


# ---- together -------------------------------------------------------------

def block(ids, table, qw, kw, proj, rope, heads, lengths=None):
    """Embedding, one projection, norm and rotation, windowed attention."""
    x = embedding(ids, table, scale=2.0, out_dtype=proj.dtype)
    qkv = torch.matmul(x, proj).view(*ids.shape, heads * 2, -1)
    q, k, v = qkv.split([heads, heads // 2, heads // 2], 2)
    q, k = qk_norm_rope(q, k, qw, kw, rope)
    return window_attention(q, k, v, window=24, sinks=2, lengths=lengths)


def block_inputs(device, dtype, D=64, heads=4):
    gen = torch.Generator().manual_seed(15)
    ids = torch.randint(0, 50, (3, 70), generator=gen).to(device)
    table = randn(gen, (50, 32), FP32, device).requires_grad_(True)
    qw, kw = (torch.ones(D, device=device, requires_grad=True)
              for _ in range(2))
    proj = (randn(gen, (32, 2 * heads * D), FP32, "cpu") / 8).to(dtype)
    proj = proj.to(device).requires_grad_(True)
    rope = rope_table(70, D, device=device)
    return ids, table, qw, kw, proj, rope


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_block_against_eager(dtype):
    """The three operators in a row on the GPU, with their gradients,
    against the same call on the CPU in 64 bits: the outputs' relative
    errors in the 2-norm stay within some roundings of the activations
    (about six in a row forward, twice that backward, of half a step
    each, adding as independent ones at most linearly)."""
    a = block_inputs("cuda", dtype)
    lengths = torch.tensor([70, 33, 1], device="cuda")
    out = block(*a, 4, lengths=lengths)
    gen = torch.Generator().manual_seed(16)
    dout = randn(gen, out.shape, dtype, "cuda")
    leaves = [t for t in a if t.requires_grad]
    grads = torch.autograd.grad(out, leaves, dout)

    c = [t.detach().cpu() for t in a]
    c = [t.double().requires_grad_(True) if t.is_floating_point() and
         t is not c[5] else t for t in c]
    c[5] = a[5].cpu()
    ids, table, qw, kw, proj, rope = c
    x = table[ids] * 2.0
    qkv = torch.matmul(x, proj).view(3, 70, 8, 64)
    q, k, v = qkv.split([4, 2, 2], 2)

    def norm_rope(t, w):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        cs, sn = rope.double()[:, None].chunk(2, -1)
        lo, hi = t.chunk(2, -1)
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1)

    want = window_attention(norm_rope(q, qw), norm_rope(k, kw), v,
                            window=24, sinks=2, lengths=lengths.cpu())
    wants = torch.autograd.grad(want, [table, qw, kw, proj],
                                dout.double().cpu())
    u = half_step(dtype)
    rel = float((out.double().cpu() - want).norm() / want.norm())
    assert rel < 6 * u, rel
    for g, w in zip(grads, wants):
        rel = float((g.double().cpu() - w).norm() / w.norm())
        assert rel < 12 * u, rel


@gpu
def test_block_repeats_on_streams_and_in_graphs():
    """The same bits on another stream, and from a captured step that is
    replayed on new inputs between eager work."""
    a = block_inputs("cuda", BF16)
    ids, leaves = a[0], [t for t in a if t.requires_grad]

    def step():
        # detached: while an eager graph of the leaves lives, a captured
        # backward would wait for the stream that graph was made on
        out = block(*a, 4)
        return (out.detach(),) + torch.autograd.grad(out, leaves,
                                                     torch.ones_like(out))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for x, y in zip(first, other):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        ids.copy_((ids * 7 + turn) % 50)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(held, want):
            assert torch.equal(x, y)


@gpu
def test_two_graphs_keep_their_workspaces():
    """Two captured calls that each have a workspace, replayed in turn."""
    gen = torch.Generator().manual_seed(17)
    q = randn(gen, (1, 1, 4, 64), BF16, "cuda")
    ks = [randn(gen, (1, 9000, 1, 64), BF16, "cuda") for _ in range(2)]
    window_attention(q, ks[0], ks[0])
    graphs, held = [], []
    for k in ks:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(window_attention(q, k, k))
        graphs.append(g)
    for turn in range(3):
        q.copy_(randn(gen, q.shape, BF16, "cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for k, h in zip(ks, held):
            assert torch.equal(h, window_attention(q, k, k))


def test_norm_module_parameters():
    m = QKNormRope(16)
    q = torch.randn(1, 3, 2, 16)
    y, z = m(q, q, rope_table(3, 16))
    (y.sum() + z.sum()).backward()
    assert m.q_weight.grad.shape == (16,) and m.k_weight.grad is not None
