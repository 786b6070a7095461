"""Variants of the transformer operators' kernels that only unusual sizes
reach, and orders of dimensions, against the definitions in 64 bits."""
import pytest
import torch

from kungfu_amd.ops.fused_embedding import embedding
from kungfu_amd.ops.qk_norm_rope import qk_norm_rope, rope_table
from kungfu_amd.ops.window_attention import window_attention
from test_transformer_ops import (BF16, F16, F32, FP32, attn_check, mask_of,
                                  qk_oracle, randn)

gpu = pytest.mark.gpu


# ---- embedding ------------------------------------------------------------

@gpu
@pytest.mark.parametrize("n,vocab,hot", [
    (131072, 70001, 0.0),   # the most tiles that every block counts itself
    (131073, 70001, 0.0),   # one tile more: their counts are summed before
    (140001, 5, 0.0), (200003, 300, 0.5), (262144 + 9, 90000, 0.2)])
def test_gradient_of_many_ids(n, vocab, hot):
    """Small whole numbers add without rounding: exact in any order."""
    gen = torch.Generator().manual_seed(n)
    ids = torch.randint(0, vocab, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < hot] = vocab // 3
    w = torch.zeros(vocab, 8, device="cuda", requires_grad=True)
    d = torch.randint(-3, 4, (n, 8), generator=gen).float()
    dw, = torch.autograd.grad(embedding(ids.cuda(), w, 1.0, 1), w, d.cuda())
    want = torch.zeros(vocab, 8, dtype=torch.float64)
    want.index_add_(0, ids, d.double())
    want[1] = 0
    assert torch.equal(dw.double().cpu(), want)


@gpu
@pytest.mark.parametrize("width", [520, 1027])
def test_gradient_of_a_frequent_token_in_slices(width):
    """Chunks of chunks of one token's rows, where a row is several waves'."""
    n, vocab = 20011, 40
    gen = torch.Generator().manual_seed(width)
    ids = torch.randint(0, vocab, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < 0.7] = 11
    w = torch.zeros(vocab, width, device="cuda", requires_grad=True)
    d = torch.randint(-3, 4, (n, width), generator=gen).float()
    dw, = torch.autograd.grad(embedding(ids.cuda(), w), w, d.cuda())
    want = torch.zeros(vocab, width, dtype=torch.float64)
    want.index_add_(0, ids, d.double())
    assert torch.equal(dw.double().cpu(), want)


# ---- query/key norm and rotation ------------------------------------------

@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_norm_gradient_by_differences(device):
    """The gradient along a direction against central differences of the
    definition in 64 bits, whose own error is of the order of 1e-9. What
    the f32 gradient may be off by is summed over its elements."""
    gen = torch.Generator().manual_seed(41)
    D = 32
    q, k = (randn(gen, (2, 5, h, D), FP32, device) for h in (4, 2))
    w = (1 + 0.2 * torch.randn(D, generator=gen)).to(device)
    rope = rope_table(5, D, device=device)
    dys = [randn(gen, t.shape, FP32, device) for t in (q, k)]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, w, w)]
    grads = torch.autograd.grad(qk_norm_rope(*leaves, rope=rope), leaves,
                                dys)
    dirs = [torch.randn(t.shape, generator=gen, dtype=torch.float64)
            for t in leaves]
    base = [t.double().cpu() for t in (q, k, w, w)]
    cs, sn = rope.double().cpu()[:, None].chunk(2, -1)

    def loss(step):
        total = 0.0
        at = [b + step * d for b, d in zip(base, dirs)]
        for x, u, dy in ((at[0], at[2], dys[0]), (at[1], at[3], dys[1])):
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * u
            lo, hi = x.chunk(2, -1)
            y = torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1)
            total += float((y * dy.double().cpu()).sum())
        return total

    slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = sum(float((g.double().cpu() * d).sum())
              for g, d in zip(grads, dirs))
    e, bound = (2 * D + 64) * F32, 1e-6
    at = torch.arange(5).expand(2, 5)
    for i, x in enumerate((q, k)):
        _, _, gx, gmag, gw, wmag = qk_oracle(x, w, rope, at, 1e-6, dys[i])
        n = x.numel() // D
        bound += float(((F32 * gx.abs() + 2 * e * gmag) *
                        dirs[i].abs()).sum())
        bound += float(((F32 * gw.abs() + (e + n * F32) * wmag) *
                        dirs[2 + i].abs()).sum())
    assert abs(got - slope) < bound
    assert bound < 0.01 * abs(slope)


# ---- window attention -----------------------------------------------------

@gpu
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_narrow_windows_with_split_keys(dtype, D):
    """Blocks of 64 rows whose keys, most of them first tokens, are shared
    out and joined, forward and for dq."""
    gen = torch.Generator().manual_seed(42)
    q, k, v = (randn(gen, (1, 1500, h, D), dtype, "cuda") for h in (2, 1, 1))
    attn_check(q, k, v, 300, 1100, True)
    attn_check(q[:, :700], k[:, :1200], v[:, :1200], 90, 1100, False,
               lengths=[1190], starts=[480])


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_in_parts(causal, D):
    """Few blocks of keys, no window: the rows that see them are cut."""
    gen = torch.Generator().manual_seed(43)
    q, k, v = (randn(gen, (1, 1500, h, D), BF16, "cuda") for h in (4, 2, 2))
    attn_check(q, k, v, None, 0, causal)
    attn_check(q, k, v, None, 0, causal, lengths=[1111])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("S,D,window,sinks,causal", [
    (130, 64, 2, 0, False), (700, 128, 9, 4, True), (300, 32, 3, 20, False),
    (32, 96, None, 0, False), (5, 64, None, 0, True), (200, 80, 32, 0, True)])
def test_gradients_of_rows_that_see_few_keys(dtype, S, D, window, sinks,
                                             causal):
    """Values have a common offset, which gradients of the scores are free
    of. Each of those, w (dw - sum w dw), is off by its rounding to the type
    as an operand and by f32 errors of its parts, and not by roundings of
    the weights that the output was summed with."""
    gen = torch.Generator().manual_seed(45)
    q, k, v, dout = (randn(gen, (1, S, 2, D), FP32, "cpu") for _ in range(4))
    q, k, v, dout = (t.to(dtype).cuda() for t in (q, k, v + 16, dout))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(
        window_attention(*leaves, window=window, sinks=sinks, causal=causal),
        leaves[:2], dout)
    u, scale = torch.finfo(dtype).eps / 2, D ** -0.5
    see = mask_of(S, S, 0, S, window, sinks, causal)
    for h in range(2):
        a, b, c, g = (t.detach()[0, :, h].double().cpu()
                      for t in (q, k, v, dout))
        x = (a @ b.T * scale).masked_fill(~see, -float("inf"))
        p, dp = torch.softmax(x, 1), g @ c.T
        delta = (p * dp).sum(1, keepdim=True)
        ds = p * (dp - delta)
        # f32 scores, exponentials and sums: of D products, of S weights
        e = 6 * (D + 8) * F32 * (1 + float(
            (a.abs() @ b.abs().T).max() * scale)) + 2 * S * F32
        most = (g.abs() @ c.abs().T).masked_fill(~see, 0).amax(
            1, keepdim=True)
        derr = (u + e) * ds.abs() + (1 + u) * p * 2 * e * most
        for t, want, bound in (
                (got[0], ds @ b * scale, derr @ b.abs() * scale),
                (got[1], ds.T @ a * scale, derr.T @ a.abs() * scale)):
            t = t[0, :, h].double().cpu()
            over = (t - want).abs() - bound * (1 + u) - u * want.abs()
            assert float(over.max()) < 1e-7


@gpu
def test_orders_of_dimensions():
    """Queries held for each head, and batches next to each other."""
    gen = torch.Generator().manual_seed(44)
    q = randn(gen, (2, 6, 90, 64), BF16, "cuda").transpose(1, 2)
    k, v = (randn(gen, (90, 3, 2, 64), BF16, "cuda").permute(2, 0, 1, 3)
            for _ in range(2))
    assert q.stride(2) > q.stride(1) and k.stride(1) > k.stride(0)
    attn_check(q, k, v, 30, 2)
    attn_check(q, k, v, None, 0, False, lengths=[90, 41])
