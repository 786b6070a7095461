"""Calls of the transformer operators at the edge of what they are for:
derivatives and traces that they do not have, checkpoints, rows at
positions outside the table, plans of unusual sizes."""
import ctypes
import math

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.checkpoint import checkpoint

from kungfu_amd.ops import hip
from kungfu_amd.ops.fused_embedding import embedding
from kungfu_amd.ops.qk_norm_rope import qk_norm_rope, rope_table
from kungfu_amd.ops.window_attention import window_attention
from test_transformer_ops import attn_check

gpu = pytest.mark.gpu
BF16, F16, FP32 = torch.bfloat16, torch.float16, torch.float32


def randn(gen, shape, dtype, device):
    return torch.randn(shape, generator=gen).to(dtype).to(device)


# ---- the operators as functions of one leaf -------------------------------
# On the GPU by their entry points. On the CPU those would take the eager
# path; there the nodes are called themselves, over stand-ins of the kernels
# that compute nothing: what is tested is what the nodes are to autograd.

@pytest.fixture
def stand_ins():
    """The table of the kernels, its launches (csrc/hip/kernel_api.h)
    replaced by functions that return success."""
    hip_so = pytest.importorskip("kungfu_amd._hip")
    pytest.importorskip("kungfu_amd._nodes")
    where = ctypes.pythonapi.PyCapsule_GetPointer
    where.restype = ctypes.c_void_p
    where.argtypes = [ctypes.py_object, ctypes.c_char_p]
    table = (ctypes.c_void_p * 9).from_address(
        where(hip_so.kernels, b"kungfu_amd.kernels"))
    kept = list(table)
    done = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: 0)
    for i in LAUNCHES:
        table[i] = ctypes.cast(done, ctypes.c_void_p).value
    yield table
    table[:] = kept


LAUNCHES = [2, 3, 5, 7, 8]  # embedding, its gradient, norm, attention, its


def on_cpu(name, x):
    """The node `name` as a function of x, in f32 or what it takes."""
    if name == "embedding":
        return hip.nodes().embedding(torch.tensor([1, 3, 3]), x, 2.0, -1,
                                     x.dtype, 0)
    if name == "qk_norm_rope":
        return hip.nodes().qk_norm_rope(x, x, None, None, None, None, 0,
                                        1e-6, 0)[0]
    return hip.nodes().window_attention(x, x, x, None, None, 4, 0, True, 1.0,
                                        0)


def on_gpu(name, x):
    if name == "embedding":
        return embedding(torch.tensor([1, 3, 3], device="cuda"), x, 2.0)
    if name == "qk_norm_rope":
        return qk_norm_rope(x, x)[0]
    return window_attention(x, x, x, window=4)


def leaf(name, device):
    gen = torch.Generator().manual_seed(32)
    shape = (5, 32) if name == "embedding" else (1, 6, 2, 32)
    dtype = BF16 if name == "window_attention" else FP32
    return randn(gen, shape, dtype, device).requires_grad_(True)


OPERATORS = ["embedding", "qk_norm_rope", "window_attention"]


# ---- the interpreter's lock -----------------------------------------------

@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", OPERATORS)
def test_launches_do_not_hold_the_interpreter(name, grad, stand_ins):
    """In place of the launches, the function that says whether its thread
    holds the lock: 1, which is an error code here, if it does."""
    holds = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p)
    for i in LAUNCHES:
        stand_ins[i] = holds.value
    x = leaf(name, "cpu")
    with torch.set_grad_enabled(grad):
        y = on_cpu(name, x)
    if grad:
        torch.autograd.grad(y, x, torch.ones_like(y))


# ---- second derivatives ---------------------------------------------------

def second_derivative(name, op, device):
    """A term that goes through the operator's gradient next to one that
    goes past it: no way of differentiating may drop the first."""
    x = leaf(name, device)
    beside = leaf(name, device)

    def loss():
        y = op(name, x)
        g, = torch.autograd.grad((y * beside.sum()).square().sum(), x,
                                 create_graph=True)
        return g.square().sum() + x.square().sum() + beside.square().sum()

    for t in (x, beside):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(loss(), t)
        with pytest.raises(RuntimeError, match="second derivative"):
            loss().backward(inputs=[t])
    with pytest.raises(RuntimeError, match="second derivative"):
        loss().backward()
    # a graph that is made and not used does no harm
    other = leaf(name, device)
    got, = torch.autograd.grad(loss() + other.square().sum(), other)
    assert torch.equal(got, 2 * other.detach())


@pytest.mark.parametrize("name", OPERATORS)
def test_second_derivative_of_a_node(name, stand_ins):
    second_derivative(name, on_cpu, "cpu")


@gpu
@pytest.mark.parametrize("name", OPERATORS)
def test_second_derivative(name):
    second_derivative(name, on_gpu, "cuda")


@gpu
def test_embedding_gradient_of_a_constant_has_no_derivative():
    """The gradient does not depend on the weight where the output's does
    not: what is beside it is differentiated as ever."""
    w = leaf("embedding", "cuda")
    g, = torch.autograd.grad(on_gpu("embedding", w).sum(), w,
                             create_graph=True)
    got, = torch.autograd.grad(g.sum() + w.square().sum(), w)
    assert torch.equal(got, 2 * w.detach())


# ---- forward-mode derivatives ---------------------------------------------

def forward_mode(name, op, device):
    """Refused, of the inputs and of the gradients that come in: an output
    without a tangent would be a derivative of zero."""
    x = leaf(name, device)
    y = op(name, x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(
            x.detach(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            op(name, dual)
        dy = torch.autograd.forward_ad.make_dual(
            torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)
    for transform in (lambda f: torch.func.jvp(f, (x.detach(),),
                                               (torch.ones_like(x),)),
                      lambda f: torch.func.vmap(f)(x.detach()[None])):
        with pytest.raises(RuntimeError):
            transform(lambda t: op(name, t))


@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode_of_a_node(name, stand_ins):
    forward_mode(name, on_cpu, "cpu")


@gpu
@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode(name):
    forward_mode(name, on_gpu, "cuda")


# ---- tracers --------------------------------------------------------------

def tracers(name, op, device):
    """Refused: a trace would hold the output's allocation, and not what
    fills it."""
    x = leaf(name, device)
    y = op(name, x)
    dy = torch.ones_like(y)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: op(name, t), (x.detach(),),
                        check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda t: op(name, t))(x.detach())
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda t: torch.autograd.grad(y, x, t)[0])(dy)
    # a program that is compiled runs it as it is
    torch._dynamo.reset()
    run = torch.compile(lambda t: op(name, t * 1.0) + 0.0, backend="eager")
    assert run(x.detach()).shape == y.shape
    return run(x.detach()), y


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", OPERATORS)
def test_tracers_of_a_node(name, stand_ins):
    tracers(name, on_cpu, "cpu")


@gpu
@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", OPERATORS)
def test_tracers(name):
    got, want = tracers(name, on_gpu, "cuda")
    assert torch.equal(got, want)


# ---- checkpoints ----------------------------------------------------------

def checkpointed(name, op, device):
    """A region that ends in the operator: its inputs are computed again
    while its backward asks for them."""
    x = leaf(name, device)

    def region(t):
        return op(name, (t * 2.0).square())

    for reentrant in (False, True):
        y = checkpoint(region, x, use_reentrant=reentrant)
        y.backward(torch.ones_like(y))
        dx, x.grad = x.grad, None
        yield dx, torch.autograd.grad(region(x), x, torch.ones_like(y))[0]


@pytest.mark.parametrize("name", OPERATORS)
def test_checkpoint_of_a_node(name, stand_ins):
    for got, want in checkpointed(name, on_cpu, "cpu"):
        assert got.shape == want.shape


@gpu
@pytest.mark.parametrize("name", OPERATORS)
def test_checkpoint(name):
    for got, want in checkpointed(name, on_gpu, "cuda"):
        assert torch.equal(got, want)


# ---- kept tensors in another layout ---------------------------------------

@gpu
@pytest.mark.parametrize("name", OPERATORS)
def test_hooks_may_change_the_layout_of_kept_tensors(name):
    """What a hook gives back has the kept tensor's values, type and size,
    and strides of its own; or was on the host in between."""
    def turned(t):  # the last dimension is the widest apart
        return t.movedim(-1, 0).contiguous().movedim(0, -1)

    x = leaf(name, "cuda")
    assert name == "embedding" or turned(x).stride(-1) != 1

    def step():
        y = on_gpu(name, x)
        return torch.autograd.grad(y, x, torch.ones_like(y))[0]

    def attend():
        k = x.detach()
        lengths = torch.tensor([[5, 9]], device="cuda")[:, 0]
        y = window_attention(x, k, k, window=4, lengths=lengths)
        return torch.autograd.grad(y, x, torch.ones_like(y))[0]

    for run in (step, attend) if name == "window_attention" else (step,):
        want = run()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned):
            got = run()
        assert torch.equal(got, want)
        with torch.autograd.graph.save_on_cpu():
            got = run()
        assert torch.equal(got, want)


# ---- what has no gradient -------------------------------------------------

@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_a_table_that_wants_a_gradient_is_refused(device):
    q = torch.randn(1, 4, 2, 32, device=device)
    rope = rope_table(4, 32, device=device).requires_grad_(True)
    for x in (q, q.clone().requires_grad_(True)):
        with pytest.raises(ValueError, match="gradient"):
            qk_norm_rope(x, x, rope=rope)
    with torch.no_grad():
        assert torch.equal(qk_norm_rope(q, q, rope=rope)[0],
                           qk_norm_rope(q, q, rope=rope.detach())[0])


# ---- how attention's backward is cut ---------------------------------------

def backward_workspace(B, S, T, Hk, G, D, window, sinks, causal):
    hip_so = pytest.importorskip("kungfu_amd._hip")
    size = ctypes.CDLL(hip_so.__file__).kf_attn_ws
    size.restype = ctypes.c_longlong
    return size((ctypes.c_longlong * 9)(
        B, S, T, Hk, G, D, window or 1 << 30, sinks, causal), 1)


def test_workspace_of_the_backward():
    """Beside a value for each row, bounded whatever the sizes: 1024 parts
    of first tokens' blocks and seven parts a place of the others, two f32
    sums of 128 x 128 each, for 512 places; and 1.5 times the places of 128
    rows for dq (at 64 columns, 768 places of half the size)."""
    most = (1024 + 7 * 512) * 2 * 128 * 128 * 4 + 768 * 128 * 128 * 4
    for B, Hk in ((1, 1), (1, 8), (2, 4), (4, 16), (32, 12), (7, 37)):
        for G in (1, 4, 32):
            for T in (1, 129, 1000, 4096, 8192, 50000, 131072, 1 << 20):
                for window in (None, 1, 64, 128, 600, 4096):
                    for sinks in (0, 1, 4, 200, 1024, 100000):
                        for D in (32, 64, 128):
                            for causal in (0, 1):
                                size = backward_workspace(
                                    B, T, T, Hk, G, D, window, sinks, causal)
                                assert 0 < size <= most + 256 + \
                                    4 * B * T * Hk * G, (
                                        B, Hk, G, T, window, sinks, D,
                                        causal)


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("B,T,Hq,Hk,D,window,sinks", [
    (4, 600, 16, 16, 64, 30, 590),   # first tokens' blocks whole
    (1, 1000, 24, 8, 64, 40, 900),   # in fewer parts than the rows ask for
    (1, 600, 16, 16, 64, 30, 590),   # in as many
    (2, 900, 8, 4, 128, 100, 700)])
def test_many_first_tokens(B, T, Hq, Hk, D, window, sinks, causal):
    gen = torch.Generator().manual_seed(33)
    q, k, v = (randn(gen, (B, T, h, D), BF16, "cuda") for h in (Hq, Hk, Hk))
    attn_check(q, k, v, window, sinks, causal)


# ---- autocast on the CPU --------------------------------------------------

@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_eager_attention_under_autocast(dtype):
    """Scores, softmax and sums stay in 32 bits: the same values and
    gradients as without autocast."""
    gen = torch.Generator().manual_seed(34)
    leaves = [randn(gen, (2, 40, h, 32), dtype, "cpu").requires_grad_(True)
              for h in (4, 2, 2)]

    def step(on):
        with torch.autocast("cpu", dtype=BF16, enabled=on):
            out = window_attention(*leaves, window=9, sinks=1)
        return (out,) + torch.autograd.grad(out, leaves,
                                            torch.ones_like(out))

    for a, b in zip(step(True), step(False)):
        assert a.dtype == dtype and torch.equal(a, b)


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
