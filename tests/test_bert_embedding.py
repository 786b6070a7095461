"""BERT's embedding where `fused_embed` is set: it goes through its modules."""
import pytest
import torch

from kungfu_amd.models.bert import Bert
from kungfu_amd.ops.fused_embedding import FusedEmbedding

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def make(seed, **options):
    torch.manual_seed(seed)
    return Bert(vocab=97, hidden=128, layers=1, heads=2, ffn=160, max_len=64,
                fused_embed=True, **options)


def ids_of(b, s, device):
    gen = torch.Generator().manual_seed(1)
    return torch.randint(0, 97, (b, s), generator=gen).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("fused_ln", [False, True])
def test_hooks_and_settings_of_the_modules(device, rotary, fused_ln):
    m = make(1, qk_norm=rotary, rotary=rotary, fused_ln=fused_ln).to(device)
    x, ran = ids_of(2, 9, device), []
    tables = [t for t in (m.tok, m.pos) if t is not None]
    for t in tables:
        t.register_forward_hook(lambda t, args, out: ran.append(t))
    plain = m._embed(x)
    assert ran == tables
    # the scale of the module is its own: none leaves the positions alone
    m.tok.scale = 0.0
    bare = m._embed(x)
    assert not torch.equal(bare, plain)
    if not rotary:
        assert torch.equal(bare[0], bare[1])


@gpu
@pytest.mark.parametrize("rotary", [False, True])
def test_rows_are_rounded_once(rotary):
    """What the first norm reads is the sum of f32 rows, rounded to bf16:
    the same bits as without the option."""
    m = make(2, qk_norm=rotary, rotary=rotary, fused_ln=True).cuda()
    x, read = ids_of(2, 50, "cuda"), []
    m.ln.register_forward_pre_hook(lambda ln, args: read.append(args[0]))
    m._embed(x)
    want = m.tok.weight[x]
    if not rotary:
        want = want + m.pos.weight[:50]
    assert read[0].dtype == torch.bfloat16
    assert torch.equal(read[0], want.bfloat16())


@pytest.mark.parametrize("device", DEVICES)
def test_a_module_keeps_its_own_type(device):
    m = FusedEmbedding(9, 16, out_dtype=torch.float16).to(device)
    x = torch.tensor([1, 8], device=device)
    assert m(x, out_dtype=torch.bfloat16).dtype == torch.float16
    m.out_dtype = None
    assert m(x, out_dtype=torch.bfloat16).dtype == torch.bfloat16
    assert m(x).dtype == torch.float32
