"""BERT with the transformer operators: what each option means, and its
gradients."""
import pytest
import torch

from kungfu_amd.models.bert import Bert
from kungfu_amd.utils.precision import convert_bf16_master

gpu = pytest.mark.gpu
SMALL = dict(vocab=97, hidden=128, layers=2, heads=2, ffn=160, max_len=64)
EVERY = dict(fused_embed=True, qk_norm=True, rotary=True, window=6, sinks=2)


def make(seed=0, **options):
    torch.manual_seed(seed)
    return Bert(**SMALL, **options)


def ids_of(b, s, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, SMALL["vocab"], (b, s), generator=gen)


def test_defaults_are_the_plain_encoder():
    m = make()
    names = set(dict(m.named_parameters()))
    assert {"tok.weight", "pos.weight", "head.weight"} <= names
    assert not any(".qk." in n for n in names)
    x = ids_of(2, 9)
    # all tokens see each other: the window attention without a mask is the
    # same function, up to f32 roundings of sums of 128 terms
    full = m(x)
    same = m(x, lengths=torch.tensor([9, 9]))
    assert torch.allclose(full, same, atol=1e-5)


def test_fused_embedding_is_the_same_function():
    a, b = make(3), make(3, fused_embed=True)
    x = ids_of(2, 9)
    assert torch.equal(a(x), b(x))
    for m in (a, b):
        m(x).square().mean().backward()
    # both add the rows of a token in f32, in another order
    assert torch.allclose(a.tok.weight.grad, b.tok.weight.grad, atol=1e-6)
    assert torch.allclose(a.pos.weight.grad, b.pos.weight.grad, atol=1e-6)


@pytest.mark.parametrize("options", [{}, EVERY, dict(EVERY, causal=True)])
def test_padding_does_not_show(options):
    """Logits of a padded batch's tokens are those of the sequence alone."""
    m = make(4, **options)
    x = ids_of(3, 20)
    lengths = torch.tensor([20, 7, 1])
    out = m(x, lengths=lengths)
    for b, n in enumerate(lengths.tolist()):
        alone = m(x[b:b + 1, :n], lengths=torch.tensor([n]))
        assert torch.allclose(out[b, :n], alone[0], atol=1e-5)


def test_causal_and_window_limit_what_is_seen():
    m = make(5, causal=True)
    x = ids_of(1, 16)
    y = x.clone()
    y[0, 9:] = (y[0, 9:] + 1) % SMALL["vocab"]
    a, b = m(x), m(y)
    assert torch.equal(a[0, :9], b[0, :9]) and not torch.equal(a, b)
    # two layers of a window of 3 reach 4 tokens to each side, and token 0
    # is seen by all but sees only its own neighbours
    m = make(5, window=3, sinks=1)
    y = x.clone()
    y[0, 15] = (y[0, 15] + 1) % SMALL["vocab"]
    a, b = m(x), m(y)
    assert torch.equal(a[0, :11], b[0, :11])
    assert not torch.equal(a[0, 11:], b[0, 11:])


def test_rotary_has_no_position_embedding():
    m = make(6, qk_norm=True, rotary=True)
    assert m.pos is None
    assert "rope" not in "".join(m.state_dict())
    x = ids_of(1, 12)
    x[0, 5] = (x[0, 3] + 1) % SMALL["vocab"]
    out = m(x)
    # order matters
    y = x.clone()
    y[0, 3], y[0, 5] = x[0, 5], x[0, 3]
    assert not torch.allclose(out[0, 0], m(y)[0, 0])
    # the table keeps f32 when the model is cast
    m.double()(x)
    assert m._rope.dtype == torch.float32
    with pytest.raises(ValueError):
        Bert(**SMALL, rotary=True)
    with pytest.raises(ValueError):
        m(ids_of(1, SMALL["max_len"] + 1))


def test_every_parameter_gets_a_gradient():
    m = make(7, **EVERY)
    m(ids_of(2, 20), lengths=torch.tensor([20, 5])).square().mean() \
        .backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and p.grad.abs().sum() > 0, n


@gpu
@pytest.mark.parametrize("options", [
    EVERY, dict(EVERY, causal=True), dict(fused_embed=True, window=4)])
@pytest.mark.parametrize("mode", ["master", "autocast"])
def test_gradients_on_the_gpu(options, mode):
    """A bf16 step's gradients against the same model's in f32 on the CPU.
    Between a parameter and the logits lie about 20 roundings of the
    activations and as many of their gradients, of half a step (2^-8) each
    at most; adding linearly they stay under 40 * 2^-8 = 0.16 of the
    gradient's norm."""
    m = make(8, fused_ln=True, **options)
    x, lengths = ids_of(3, 40), torch.tensor([40, 17, 1])
    on = m.cuda()
    if mode == "master":
        convert_bf16_master(on)
    gen = torch.Generator().manual_seed(9)
    weight = torch.randn(3, 40, SMALL["vocab"], generator=gen)
    weight[1, 17:] = weight[2, 1:] = 0  # a loss of the tokens that are there
    with torch.autocast("cuda", dtype=torch.bfloat16,
                        enabled=mode == "autocast"):
        out = on(x.cuda(), lengths=lengths.cuda())
    loss = (out.float() * weight.cuda()).sum()
    names = [n for n, _ in on.named_parameters()]
    got = torch.autograd.grad(loss, list(on.parameters()))
    ref = make(8, fused_ln=True, **options)
    ref.load_state_dict({n: t.float().cpu()
                         for n, t in on.state_dict().items()})
    want = torch.autograd.grad(
        (ref(x, lengths=lengths) * weight).sum(), list(ref.parameters()))
    for n, g, w in zip(names, got, want):
        if n.endswith("qkv.bias"):
            # without rotation or norm a bias of the keys moves all scores
            # of a query alike: a third of it has no gradient but roundings
            continue
        rel = float((g.float().cpu() - w).norm() / w.norm())
        assert rel < 0.16, (n, rel)


@gpu
def test_step_in_a_graph():
    """A captured training step of the model, replayed between eager
    passes, follows the eager step. The norms and biases of the model add
    with atomics, so their last bits, and after them roundings to bf16, may
    differ from run to run: by 2^-8 of a value each, 0.02 for some of them
    one after another."""
    m = make(10, fused_ln=True, **EVERY).cuda()
    convert_bf16_master(m)
    x = ids_of(4, 48).cuda()
    params = list(m.parameters())

    def step():
        loss = m(x).float().square().mean()
        return torch.autograd.grad(loss, params)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    ours = [i for i, (n, _) in enumerate(m.named_parameters())
            if n == "tok.weight" or n.endswith(("q_weight", "k_weight"))]
    for turn in range(3):
        x.copy_((x * 5 + turn) % SMALL["vocab"])
        graph.replay()
        torch.cuda.synchronize()
        first = [held[i].clone() for i in ours]
        with torch.no_grad():
            m(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for i, f in zip(ours, first):
            assert torch.isfinite(f).all()
            rel = float((f.float() - want[i].float()).norm() /
                        want[i].float().norm())
            assert rel < 0.02, rel


def test_trains_after_inference_mode():
    """The first call may be one of inference mode: what the model keeps of
    it, the angles, serves training too."""
    m = make(12, **EVERY)
    x = ids_of(2, 9)
    with torch.inference_mode():
        seen = m(x)
    out = m(x)
    out.square().mean().backward()
    assert torch.equal(out, seen)
    assert all(p.grad is not None for p in m.parameters())


def test_too_long_a_batch_is_refused():
    """Also where the lookup itself would not raise, on the GPU."""
    for options in (dict(fused_embed=True), EVERY):
        m = make(13, **options)
        m(ids_of(1, 64))
        with pytest.raises((ValueError, IndexError), match="64"):
            m(ids_of(1, 65))


@gpu
def test_angles_of_a_captured_first_call_are_not_kept():
    """What a graph computes is there after a replay only: a call outside
    the graph makes its own."""
    m = make(14, **EVERY).cuda()
    device = m.tok.weight.device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m._angles(device)
    eager = m._angles(device).clone()
    assert m._angles(device) is m._angles(device)
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        # 64-bit cosines and sines of two libraries, rounded once to f32
        assert torch.allclose(held, eager, rtol=0, atol=2.0 ** -24)
        assert float(eager[0, 0]) == 1.0
