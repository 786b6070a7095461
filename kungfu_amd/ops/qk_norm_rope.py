"""RMS norm of queries and keys for each head with the position rotation.

Wraps csrc/hip/qk_norm_rope.hip: one pass over q and k forward, one over
their gradients backward, both in one launch; the norm is computed again in
the backward from the rows that it reads anyway, so nothing but q and k is
kept. q and k may be slices of one projection's output, no copy is made of
them.

On CPU tensors the same is computed by eager torch.
"""
import torch

from kungfu_amd.ops import hip

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def rope_table(length, dim, base=10000.0, device=None):
    """Angles of `length` positions for heads of `dim`: (length, dim) f32,
    the cosines of the dim/2 angles, then the sines. The angle of position
    p and pair i is p * base^(-2 i / dim), computed in 64 bits: p of some
    10^5 leaves 32 bits only two digits after the point."""
    if dim < 2 or dim % 2:
        raise ValueError("rotation needs an even head width, not %d" % dim)
    inv = torch.pow(float(base), -torch.arange(
        0, dim, 2, dtype=torch.float64, device=device) / dim)
    angles = torch.arange(length, dtype=torch.float64,
                          device=device)[:, None] * inv
    return torch.cat([angles.cos(), angles.sin()], 1).float()


def _check(q, k, weights, rope, positions, start):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be (batch, length, heads, width)")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q %s and k %s differ in more than heads" %
                         (tuple(q.shape), tuple(k.shape)))
    if q.dtype != k.dtype or q.device != k.device:
        raise ValueError("q and k must be of one type and device")
    B, S, _, D = q.shape
    if D < 2 or D % 2:
        raise ValueError("the head width must be even, not %d" % D)
    given = [w for w in weights if w is not None]
    for w in given:
        if tuple(w.shape) != (D,) or w.device != q.device:
            raise ValueError("a norm weight must be (%d,) on %s" %
                             (D, q.device))
        if w.dtype not in (torch.float32, q.dtype) or \
                w.dtype != given[0].dtype:
            raise TypeError("norm weights must both be float32 or %s" %
                            q.dtype)
    if rope is None:
        if positions is not None:
            raise ValueError("positions without a rope table")
    else:
        if rope.dim() != 2 or rope.shape[1] != D or not rope.shape[0] or \
                rope.dtype != torch.float32 or rope.device != q.device:
            raise ValueError("rope must be (positions, %d) float32 on %s" %
                             (D, q.device))
        if rope.requires_grad and torch.is_grad_enabled():
            raise ValueError("rope is a table of constants and gets no "
                             "gradient")
        if positions is not None:
            hip.check_ints("positions", positions, [(S,), (B, S)], q.device)
        elif start < 0 or start + S > rope.shape[0]:
            raise ValueError("positions %d..%d are outside a table of %d" %
                             (start, start + S - 1, rope.shape[0]))
    if q.is_cuda:
        if q.dtype not in _FLOATS:
            raise TypeError("q must be float32, bfloat16 or float16, not %s"
                            % q.dtype)
        if D > 512:
            raise ValueError("head width %d is over 512" % D)
        if B * S >= 1 << 30 or q.shape[2] + k.shape[2] > 1 << 16:
            raise ValueError("qk_norm_rope is limited to 2^30 tokens and "
                             "2^16 heads")


def _eager(x, w, rope, positions, start, eps):
    up = x.double() if x.dtype == torch.float64 else x.float()
    up = up * torch.rsqrt(up.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        up = up * w.to(up.dtype)
    if rope is not None:
        S = x.shape[1]
        if positions is None:
            at = rope[start:start + S]
        else:
            if positions.numel() and (
                    int(positions.min()) < 0 or
                    int(positions.max()) >= rope.shape[0]):
                raise IndexError("a position is outside a table of %d" %
                                 rope.shape[0])
            at = rope[positions.long()]
        cos, sin = at.to(up.dtype)[..., None, :].chunk(2, -1)
        lo, hi = up.chunk(2, -1)
        up = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return up.to(x.dtype)


def _dense_rows(t):
    return t if t.stride(-1) == 1 else t.contiguous()


def qk_norm_rope(q, k, q_weight=None, k_weight=None, rope=None,
                 positions=None, start=0, eps=1e-6):
    """Norms and rotates q (batch, length, heads, width) and k (batch,
    length, key heads, width); returns both, dense.

    Each head's row is divided by the root of its mean square plus eps and
    multiplied by the weight (width,), float32 or q's type, where there is
    one. Where there is a table (`rope_table`), the pairs (i, i + width/2)
    are then turned by the angles of the row's position: `positions`,
    (length,) or (batch, length) int32 or int64, else start, start + 1, ...
    The table has no gradient, and one that asks for it is refused.

    The width is even and at most 512. Without `positions` the range is
    checked here. A position in `positions` outside the table raises on the
    CPU; on the GPU, where reading it back would hold up the stream, the
    rows at it are NaN, get zeros as gradients and add to none.
    """
    start, eps = int(start), float(eps)
    _check(q, k, (q_weight, k_weight), rope, positions, start)
    if not q.is_cuda:
        return (_eager(q, q_weight, rope, positions, start, eps),
                _eager(k, k_weight, rope, positions, start, eps))
    q, k = _dense_rows(q), _dense_rows(k)
    if rope is not None:
        rope = rope.contiguous()
    if q_weight is not None:
        q_weight = q_weight.contiguous()
    if k_weight is not None:
        k_weight = k_weight.contiguous()
    return hip.nodes().qk_norm_rope(q, k, q_weight, k_weight, rope,
                                    positions, start, eps, hip.stream_of(q))


class QKNormRope(torch.nn.Module):
    """Norm weights of one layer's queries and keys, in f32."""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.eps = eps
        self.q_weight = torch.nn.Parameter(torch.ones(dim))
        self.k_weight = torch.nn.Parameter(torch.ones(dim))

    def forward(self, q, k, rope=None, positions=None, start=0):
        return qk_norm_rope(q, k, self.q_weight, self.k_weight, rope,
                            positions, start, self.eps)
