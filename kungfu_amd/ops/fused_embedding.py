"""Embedding lookup with a scale, and its gradient by sorted tokens.

Wraps csrc/hip/embedding.hip. The lookup reads each row once and writes it
scaled in the activations' type, with no cast pass after it. The gradient
sums the rows of each token in one fixed order (a stable radix sort of the
ids, no atomics), in f32 with one rounding at the end, so it repeats bit by
bit; torch's nn.Embedding rounds after each of several steps and needs a
cast of the gradient where the activations are of another type.

On CPU tensors the same is computed by eager torch.
"""
import torch

from kungfu_amd.ops import hip

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check(ids, weight, padding_idx, out_dtype):
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("ids must be int32 or int64, not %s" % ids.dtype)
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError("weight must be a (tokens, width) matrix, not %s" %
                         (tuple(weight.shape),))
    if ids.device != weight.device:
        raise ValueError("ids are on %s, weight is on %s" %
                         (ids.device, weight.device))
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError("padding_idx %d is outside %d tokens" %
                         (padding_idx, weight.shape[0]))
    if not weight.is_cuda:
        return
    if weight.dtype not in _FLOATS:
        raise TypeError("weight must be float32, bfloat16 or float16, not "
                        "%s" % weight.dtype)
    if out_dtype not in (torch.float32, weight.dtype) and \
            weight.dtype != torch.float32:
        raise TypeError("no lookup of %s rows as %s" %
                        (weight.dtype, out_dtype))
    if out_dtype not in _FLOATS:
        raise TypeError("no lookup as %s" % out_dtype)
    if ids.numel() >= 1 << 30 or weight.shape[0] >= 1 << 30 or \
            weight.shape[1] > 1 << 20:
        raise ValueError("embedding is limited to 2^30 ids, 2^30 tokens and "
                         "a width of 2^20")


def embedding(ids, weight, scale=1.0, padding_idx=None, out_dtype=None):
    """scale * weight[ids], as `out_dtype` (default: the weight's type).

    ids: int32 or int64, any shape. weight: (tokens, width), f32, bf16 or
    f16; `out_dtype` is f32 or the weight's type, or any of the three for
    f32 weights. The row `padding_idx` is looked up as any other and gets no
    gradient. The gradient is dense, of the weight's type.

    An id outside the table raises on the CPU. On the GPU, where reading it
    back would hold up the stream, its output row is NaN and it adds to no
    gradient.
    """
    out_dtype = weight.dtype if out_dtype is None else out_dtype
    scale = float(scale)
    _check(ids, weight, padding_idx, out_dtype)
    if not weight.is_cuda:
        rows = torch.nn.functional.embedding(ids, weight, padding_idx)
        if weight.dtype != torch.float64:
            rows = rows.float()
        return (rows * scale).to(out_dtype)
    if weight.stride(1) != 1 and weight.shape[1] > 1:
        weight = weight.contiguous()
    return hip.nodes().embedding(
        ids.contiguous(), weight, scale,
        -1 if padding_idx is None else padding_idx, out_dtype,
        hip.stream_of(weight))


class FusedEmbedding(torch.nn.Embedding):
    """nn.Embedding with a scale and an output type of its own."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None,
                 scale=1.0, out_dtype=None, **kwargs):
        for name in ("max_norm", "scale_grad_by_freq", "sparse"):
            if kwargs.get(name):
                raise ValueError("FusedEmbedding has no %s" % name)
        super().__init__(num_embeddings, embedding_dim, padding_idx,
                         **kwargs)
        self.scale = scale
        self.out_dtype = out_dtype

    def forward(self, ids, out_dtype=None):
        """`out_dtype`: of this call, where the module has none of its own."""
        return embedding(ids, self.weight, self.scale, self.padding_idx,
                         self.out_dtype or out_dtype)
