"""Calls of the transformer operators that differ from the plain ones: rows
at positions outside the table, derivatives and traces that the operators
do not have, checkpoints, workspaces of unusual plans."""
import math

import pytest
import torch

from kungfu_amd.ops.qk_norm_rope import qk_norm_rope, rope_table

gpu = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def randn(gen, shape, dtype, device):
    return torch.randn(shape, generator=gen).to(dtype).to(device)


# ---- positions outside the table ------------------------------------------

@gpu
@pytest.mark.parametrize("D", [64, 80, 10])
@pytest.mark.parametrize("dtype,weight_t", [(FP32, FP32), (BF16, FP32),
                                            (F16, F16)])
def test_rows_outside_the_table_have_no_gradient(dtype, weight_t, D):
    """They get zeros and add nothing to the weights' gradients, whatever
    they and their gradients hold: the same bits as with any position
    inside the table and gradients of zero there."""
    gen = torch.Generator().manual_seed(31)
    B, S, P = 2, 37, 50
    q, k = (randn(gen, (B, S, h, D), dtype, "cuda") for h in (5, 2))
    w = [(1 + 0.2 * torch.randn(D, generator=gen)).to(weight_t).cuda()
         for _ in range(2)]
    dys = [randn(gen, t.shape, dtype, "cuda") for t in (q, k)]
    rope = rope_table(P, D, device="cuda")
    at = torch.randint(0, P, (B, S), generator=gen).cuda()
    bad = torch.zeros(B, S, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[0, 36] = bad[1, 0] = bad[1, 17] = True

    def grads(q, k, at, dys):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
        outs = qk_norm_rope(*leaves, rope=rope, positions=at)
        return outs, torch.autograd.grad(outs, leaves, dys)

    want_out, want = grads(q, k, at, [
        d.masked_fill(bad[..., None, None], 0) for d in dys])
    far = at.clone()
    far[bad] = torch.tensor([-1, P, 1 << 40, -(1 << 40)], device="cuda")
    q[bad], k[bad] = math.inf, math.nan
    dys[0][bad], dys[1][bad] = math.nan, -math.inf
    out, got = grads(q, k, far, dys)
    for a, b in zip(out, want_out):
        assert torch.isnan(a[bad]).all()
        assert torch.equal(a[~bad], b[~bad])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert not got[0][bad].any() and not got[1][bad].any()
