"""BERT-base encoder (masked-LM head) for the SMA + gradient-noise-scale
benchmark config.

Self-contained transformer encoder with BERT-base dimensions (L=12, H=768,
A=12, ~110M params); attention uses torch's fused SDPA, which lowers to the
ROCm flash-attention path on MI355X.

Options beside the plain encoder, each off by default: `fused_embed` (the
lookup in the activations' type, gradient by sorted tokens), `qk_norm` and
`rotary` (norm of queries and keys for each head, positions by rotation
instead of an embedding), `window`/`sinks`/`causal` (attention to near and
first tokens), and padded batches by `lengths`. On the GPU all but the first
need 16-bit activations: bf16 weights, or autocast.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from kungfu_amd.ops.fused_linear import KfLinear


def _make_ln(hidden, fused):
    if fused:
        from kungfu_amd.ops.fused_ln import FusedLayerNorm

        return FusedLayerNorm(hidden)
    return nn.LayerNorm(hidden)


def _make_embed(n, hidden, fused):
    if fused:
        from kungfu_amd.ops.fused_embedding import FusedEmbedding

        return FusedEmbedding(n, hidden)
    return nn.Embedding(n, hidden)


class BertLayer(nn.Module):
    def __init__(self, hidden, heads, ffn, fused_ln=False, qk_norm=False,
                 window=None, sinks=0, causal=False):
        super().__init__()
        self.heads = heads
        self.window = window
        self.sinks = sinks
        self.causal = causal
        self.qk = None
        if qk_norm:
            from kungfu_amd.ops.qk_norm_rope import QKNormRope

            self.qk = QKNormRope(hidden // heads)
        # KfLinear = nn.Linear + fused column-sum bias-grad kernel
        # (native autograd fallback outside the bf16-master conditions)
        self.qkv = KfLinear(hidden, 3 * hidden)
        self.proj = KfLinear(hidden, hidden)
        self.ln1 = _make_ln(hidden, fused_ln)
        self.fc1 = KfLinear(hidden, ffn)
        self.fc2 = KfLinear(ffn, hidden)
        self.ln2 = _make_ln(hidden, fused_ln)

    def attend(self, qkv, rope, lengths):
        if self.qk is None and rope is None and self.window is None and \
                not self.causal and lengths is None:
            q, k, v = (t.transpose(1, 2) for t in qkv.unbind(2))
            a = F.scaled_dot_product_attention(q, k, v)
            return a.transpose(1, 2)
        from kungfu_amd.ops.window_attention import window_attention

        q, k, v = qkv.unbind(2)
        if self.qk is not None:
            q, k = self.qk(q, k, rope)
        return window_attention(q, k, v, window=self.window,
                                sinks=self.sinks, causal=self.causal,
                                lengths=lengths)

    def forward(self, x, rope=None, lengths=None):
        b, s, h = x.shape
        qkv = self.qkv(x).view(b, s, 3, self.heads, h // self.heads)
        a = self.attend(qkv, rope, lengths).reshape(b, s, h)
        x = self.ln1(x + self.proj(a))
        x = self.ln2(x + self.fc2(F.gelu(self.fc1(x))))
        return x


class Bert(nn.Module):
    def __init__(self, vocab=30522, hidden=768, layers=12, heads=12,
                 ffn=3072, max_len=512, fused_ln=False, fused_embed=False,
                 qk_norm=False, rotary=False, window=None, sinks=0,
                 causal=False):
        super().__init__()
        if rotary and not qk_norm:
            raise ValueError("rotary positions need qk_norm")
        self.fused_ln = fused_ln
        self.fused_embed = fused_embed
        self.tok = _make_embed(vocab, hidden, fused_embed)
        self.pos = None
        if not rotary:
            self.pos = _make_embed(max_len, hidden, fused_embed)
        self.rotary = (max_len, hidden // heads) if rotary else None
        self._rope = None
        self.ln = _make_ln(hidden, fused_ln)
        self.blocks = nn.ModuleList(
            [BertLayer(hidden, heads, ffn, fused_ln=fused_ln,
                       qk_norm=qk_norm, window=window, sinks=sinks,
                       causal=causal)
             for _ in range(layers)])
        self.head = KfLinear(hidden, vocab)
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, std=0.02)
                nn.init.zeros_(m.bias)
            elif isinstance(m, nn.Embedding):
                nn.init.normal_(m.weight, std=0.02)

    def _embed(self, ids):
        low = self.fused_ln and ids.is_cuda
        if low and self.fused_embed and self.pos is None:
            # in the activations' type: no cast of the rows after it
            x = self.tok(ids, out_dtype=torch.bfloat16)
        else:  # rows that are added are rounded after that, once
            x = self.tok(ids)
        if self.pos is not None:
            if self.fused_embed and ids.shape[1] > self.pos.num_embeddings:
                # the lookup on the GPU would answer NaN
                raise IndexError("%d tokens for %d positions" %
                                 (ids.shape[1], self.pos.num_embeddings))
            pos = torch.arange(ids.shape[1], device=ids.device).unsqueeze(0)
            x = x + self.pos(pos)
        if low:
            x = x.to(torch.bfloat16)  # embeddings stay fp32 under autocast
        return self.ln(x)

    def _angles(self, device):
        # no buffer: the table stays f32 when the model's type is changed
        if self.rotary is None:
            return None
        if self._rope is None or self._rope.device != device:
            from kungfu_amd.ops.qk_norm_rope import rope_table

            # a tensor of inference mode could not be trained with
            with torch.inference_mode(False):
                if device.type == "cuda" and \
                        torch.cuda.is_current_stream_capturing():
                    # there after a replay only: not for other calls
                    return rope_table(*self.rotary, device=device)
                # the copy waits, so that any stream can use it
                self._rope = rope_table(*self.rotary).to(device)
        return self._rope

    def forward(self, ids, lengths=None):
        """Logits of every token. `lengths` (batch,) are the tokens that
        each sequence of a padded batch has: no token attends to what lies
        behind them."""
        x = self._embed(ids)
        rope = self._angles(ids.device)
        for blk in self.blocks:
            x = blk(x, rope, lengths)
        return self.head(x)


def bert_base(vocab=30522, max_len=512, fused_ln=False, **options):
    return Bert(vocab=vocab, max_len=max_len, fused_ln=fused_ln, **options)
