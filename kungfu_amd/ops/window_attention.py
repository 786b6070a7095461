"""Attention with a sliding window and first tokens that stay visible.

Wraps csrc/hip/window_attention.hip: one pass over the visible key tiles
with a running softmax forward (tiles that the mask hides are not read),
and a backward that writes every gradient once, in a fixed order, so that
results repeat bit by bit. Key heads may be fewer than query heads, batches
may be padded, and q, k and v may be slices of one projection's output.

On CPU tensors the same is computed by eager torch.
"""
import math

import torch

from kungfu_amd.ops import hip

_MOST = 1 << 30


def _check(q, k, v, window, sinks, lengths, starts, scale):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be (batch, length, heads, width)")
    if k.shape != v.shape:
        raise ValueError("k %s and v %s differ" %
                         (tuple(k.shape), tuple(v.shape)))
    B, S, Hq, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError("q %s and k %s differ in batch or width" %
                         (tuple(q.shape), tuple(k.shape)))
    if k.shape[2] == 0 or Hq % k.shape[2]:
        raise ValueError("%d query heads cannot share %d key heads" %
                         (Hq, k.shape[2]))
    if not (q.dtype == k.dtype == v.dtype) or \
            not (q.device == k.device == v.device):
        raise ValueError("q, k and v must be of one type and device")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1, not %d" % window)
    if sinks < 0:
        raise ValueError("sinks must be at least 0, not %d" % sinks)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite, not %r" % scale)
    for name, t in (("lengths", lengths), ("starts", starts)):
        if t is not None:
            hip.check_ints(name, t, [(B,)], q.device)
    if starts is None and S > k.shape[1]:
        raise ValueError("%d queries for %d keys need starts" %
                         (S, k.shape[1]))
    if q.is_cuda:
        if q.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("q, k and v must be bfloat16 or float16, not %s"
                            % q.dtype)
        if D % 8 or not 8 <= D <= 128:
            raise ValueError("the head width must be a multiple of 8 up to "
                             "128, not %d" % D)
        if max(S * (Hq // k.shape[2]), k.shape[1], B * k.shape[2]) >= _MOST:
            raise ValueError("window_attention is limited to 2^30 rows of a "
                             "key head and keys")


def _eager(q, k, v, window, sinks, causal, lengths, starts, scale):
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    (B, S, Hq, D), (T, Hk) = q.shape, k.shape[1:3]
    p = torch.arange(S, device=q.device) + (
        T - S if starts is None else starts.long()[:, None])
    p = p.expand(B, S)[:, :, None]
    j = torch.arange(T, device=q.device)
    n = torch.full((B,), T, device=q.device) if lengths is None else \
        lengths.long().clamp(0, T)
    n = n[:, None, None]
    seen = (j < n) & (p >= 0) & (p < n)
    if window is not None:
        seen = seen & (((p - j).abs() < window) | (j < sinks))
    if causal:
        seen = seen & (j <= p)
    seen = seen[:, None, None]
    # what lies behind a sequence is not read, whatever it holds
    q, k, v = (t.to(wide) for t in (q, k, v))
    q = torch.where(((p >= 0) & (p < n))[..., None], q, torch.zeros_like(q))
    if lengths is not None:
        held = (j < n[:, 0])[:, :, None, None]
        k = torch.where(held, k, torch.zeros_like(k))
        v = torch.where(held, v, torch.zeros_like(v))
    q = q.transpose(1, 2).reshape(B, Hk, Hq // Hk, S, D)
    k = k.transpose(1, 2)[:, :, None]
    v = v.transpose(1, 2)[:, :, None]
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    x = x.masked_fill(~seen, -math.inf)
    top = x.detach().amax(-1, keepdim=True) if T else x.sum(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top),
                                  top))
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x, v) / torch.where(total == 0,
                                           torch.ones_like(total), total)
    return out.reshape(B, Hq, S, D).transpose(1, 2)


def _int32(t):
    """Positions as the kernels read them; far ones stay far."""
    if t.dtype == torch.int64:
        t = t.clamp(-_MOST, _MOST).to(torch.int32)
    return t.contiguous()


def window_attention(q, k, v, window=None, sinks=0, causal=True,
                     lengths=None, starts=None, scale=None):
    """Attention of q (batch, queries, heads, width) over k and v (batch,
    keys, key heads, width); returns (batch, queries, heads, width).

    Query i of a sequence has position starts[b] + i (default: the queries
    are the last of the keys). It sees key j when |position - j| < window
    or j < sinks, and where causal only up to its own position; window None
    is no window. lengths (batch,): keys that each sequence has (default
    all); what lies behind them is not read, and a query whose position is
    outside its sequence sees nothing: its output and gradients are zeros.
    scale is width^-1/2 by default. Query head h reads key head
    h * key heads / heads. Keys and values inside a sequence have to be
    finite, also where a mask hides them from some queries.

    On the GPU: bf16 or f16 (f32 under autocast is cast as autocast says),
    a width that is a multiple of 8 up to 128. Probabilities are rounded to
    that type for the product with v, and so are their gradients for the
    products with q and k (in f16 those overflow past 65504); all sums are
    f32.
    """
    if q.is_cuda and torch.is_autocast_enabled("cuda"):
        to = torch.get_autocast_dtype("cuda")
        q, k, v = (t.to(to) if t.dtype == torch.float32 else t
                   for t in (q, k, v))
    window = None if window is None else int(window)
    sinks = int(sinks)
    scale = float(scale) if scale is not None else \
        1.0 / math.sqrt(max(1, q.shape[-1]))
    _check(q, k, v, window, sinks, lengths, starts, scale)
    if not q.is_cuda:
        # the products too are of wide operands, also under autocast
        with torch.autocast("cpu", enabled=False):
            return _eager(q, k, v, window, sinks, causal, lengths, starts,
                          scale).to(q.dtype)
    if 0 in q.shape or 0 in k.shape:
        # no row, or none that sees anything
        every = torch.ones((), dtype=torch.bool, device=q.device)
        q, k, v = (t.masked_fill(every, 0) for t in (q, k, v))
        return q + k.sum() + v.sum()
    if lengths is not None:
        lengths = _int32(lengths)
    if starts is not None:
        starts = _int32(starts)
    return hip.nodes().window_attention(
        q, k, v, lengths, starts, _MOST if window is None else
        min(window, _MOST), min(sinks, _MOST), bool(causal), scale,
        hip.stream_of(q))
