"""Row operators on the CPU: calls that are allowed and rare, and what
``activations_8bit`` does with tensors that are no activations."""

import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from yet_another_mobilenet_series_amd import ops
from yet_another_mobilenet_series_amd.ops import backend
from yet_another_mobilenet_series_amd.ops import rows as R


# ---------------------------------------------------------------------------
# forward-mode derivatives
# ---------------------------------------------------------------------------

@pytest.mark.skipif(not backend.extension_available(),
                    reason="the extension is not built")
@pytest.mark.parametrize("grad_mode", [True, False])
def test_the_extension_refuses_tangents(grad_mode):
    """The refusal comes before anything is launched, so that it is seen
    without a GPU too."""
    ext = R.ext()
    x, w = torch.randn(4, 8), torch.randn(8)

    def join(h, x, w):
        return ext.join(h, x, None, None, None, None, w, None, False, True,
                        True, 0, 0, 1e-6, 1.0, False)

    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dx = forward_ad.make_dual(x, torch.ones_like(x))
        dw = forward_ad.make_dual(w, torch.ones_like(w))
        for call in (lambda: ext.bias_act(dx, None, 1, False),
                     lambda: ext.bias_act(x, dw, 1, True),
                     lambda: ext.linear8(dx, x, None),
                     lambda: ext.linear8(x, x, dw[:4]),
                     lambda: join(None, dx, None), lambda: join(x, x, dw),
                     lambda: join(dx, x, w)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_tangents_pass_through_the_reference():
    x, t = torch.randn(5, 8), torch.randn(5, 8)
    with forward_ad.dual_level():
        u = forward_ad.unpack_dual(ops.row_norm(forward_ad.make_dual(x, t)))
    a = 1e-3
    want = (ops.row_norm((x + a * t).double())
            - ops.row_norm((x - a * t).double())) / (2 * a)
    assert torch.allclose(u.tangent.double(), want, atol=1e-4)


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------

def test_the_context_leaves_what_the_codec_does_not_take(monkeypatch):
    """A tensor of too many chunks, or a layer of too many inputs, is handled
    as without the context instead of ending the forward pass."""
    one = torch.empty(1)
    assert R._fits(one.expand((1 << 29) - 1, 1))
    assert not R._fits(one.expand(1 << 29, 1))       # 4 chunks a row
    assert not R._fits(one.expand(1 << 24, 1024))    # 128
    assert R._fits(one.expand((1 << 24) - 1, 1024))
    assert not R._fits(one.expand(1, 1 << 30))
    monkeypatch.setattr(R, "_fits", lambda t: t.shape[-1] < 64)
    x = torch.randn(4, 64)
    w = torch.randn(64, 64, requires_grad=True)
    with ops.activations_8bit(min_numel=1):
        y = torch.tanh(x @ w)
    got, = torch.autograd.grad(y.sum(), w)
    want, = torch.autograd.grad(torch.tanh(x @ w).sum(), w)
    assert torch.equal(got, want)

    w16 = one.expand(16, 1024)
    assert R.linear_fits(one.expand((1 << 24) - 1, 1024), w16)
    assert not R.linear_fits(one.expand(1 << 24, 1024), w16)
    assert not R.linear_fits(one.expand(1 << 20, 64), one.expand(1 << 17, 64))
    assert not R.linear_fits(one.expand(2, (1 << 22) + 1),
                             one.expand(1, (1 << 22) + 1))
    monkeypatch.setattr(R, "MAX_LINEAR_CHANNELS", 32)
    x = x.requires_grad_()
    with ops.activations_8bit(min_numel=1):
        y = ops.linear(x, w)
    got, = torch.autograd.grad(y.square().sum(), w)
    want, = torch.autograd.grad(ops.linear(x, w).square().sum(), w)
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# weights inside activations_8bit
# ---------------------------------------------------------------------------

def _grads(run, *wanted, context):
    """The gradients of run()'s sum of squares' neighbour (a fixed gradient)
    and the shapes of what was packed."""
    packed = []
    pack = R.pack_activation

    def spy(t):
        packed.append(tuple(t.shape))
        return pack(t)

    R.pack_activation = spy
    try:
        if context:
            with ops.activations_8bit(min_numel=1):
                y = run()
        else:
            y = run()
    finally:
        R.pack_activation = pack
    dy = torch.linspace(-1, 1, y.numel()).view(y.shape).to(y.dtype)
    return torch.autograd.grad(y, wanted, dy), packed


def _weight(form):
    """A weight [24, 40] made by `form` from parameters (or none), as a
    function that a forward pass calls."""
    torch.manual_seed(6)
    p = torch.nn.Parameter(torch.randn(24, 40))
    g = torch.nn.Parameter(torch.rand(24, 1) + 0.5)
    q = torch.nn.Parameter(torch.randn(40, 24))
    a, b = (torch.nn.Parameter(torch.randn(*s)) for s in ((24, 5), (5, 40)))
    mask = (torch.rand(24, 40) > 0.5).float()
    frozen = torch.nn.Parameter(torch.randn(24, 40), requires_grad=False)
    conv = torch.nn.Parameter(torch.randn(24, 40, 1, 1))
    buffer = torch.randn(24, 40)
    normed = torch.nn.utils.parametrizations.weight_norm(
        torch.nn.Linear(40, 24, bias=False))
    return {
        "parameter": lambda: p,
        "frozen": lambda: frozen,
        "frozen, cast": lambda: frozen.double().float(),
        "frozen, its data": lambda: frozen.data * 1.0,
        "1x1 filter, viewed and cast":
            lambda: conv.view(24, 40).double().float(),
        "transposed copy": lambda: q.t().contiguous(),
        "weight norm": lambda: g * p / p.norm(dim=1, keepdim=True),
        "parametrised": lambda: normed.weight,
        "scaled": lambda: 0.5 * p,
        "concatenated": lambda: torch.cat([p[:7], frozen[7:]]),
        "masked": lambda: p * mask,
        "low rank": lambda: a @ b,
        "plain": lambda: buffer,
        "plain, wants a gradient":
            lambda w=buffer.clone().requires_grad_(): w,
    }[form]


WEIGHTS = ["parameter", "frozen", "frozen, cast", "frozen, its data",
           "1x1 filter, viewed and cast", "transposed copy", "weight norm",
           "parametrised", "scaled", "concatenated", "masked", "low rank",
           "plain", "plain, wants a gradient"]


@pytest.mark.parametrize("layer", ["linear", "conv", "matmul", "ops.linear",
                                   "ops.conv"])
@pytest.mark.parametrize("form", WEIGHTS)
def test_weights_are_saved_as_they_are(form, layer):
    """dx comes from the weight itself, however the weight is made."""
    weight = _weight(form)
    x = torch.randn(6, 40, requires_grad=True)

    def run():
        w, v = weight(), x * 1.0
        if layer == "linear":
            return torch.nn.functional.linear(v, w)
        if layer == "conv":
            return torch.nn.functional.conv2d(v[:, :, None, None],
                                              w[:, :, None, None])
        if layer == "matmul":
            return v @ w.t()
        if layer == "ops.linear":
            return ops.linear(v, w)
        return ops.conv_bn_act(v[:, :, None, None], w[:, :, None, None],
                               None, None, None, None)

    (want,), _ = _grads(run, x, context=False)
    (got,), packed = _grads(run, x, context=True)
    assert torch.equal(got, want)
    assert not any(s[:2] in ((24, 40), (40, 24)) for s in packed)


@pytest.mark.parametrize("form", ["weight norm", "scaled", "masked"])
def test_activations_beside_made_weights_are_packed(form):
    weight = _weight(form)
    x = torch.randn(6, 40)
    p = torch.nn.Parameter(torch.randn(24, 24))

    def run():
        return torch.tanh(x @ weight().t()) @ p

    _, packed = _grads(run, p, context=True)
    assert packed.count((6, 40)) == 1 and packed.count((6, 24)) >= 1


@pytest.mark.parametrize("frozen", [False, True])
def test_weights_under_autocast(frozen):
    m = torch.nn.Sequential(torch.nn.Linear(40, 24), torch.nn.Linear(24, 16))
    m.requires_grad_(not frozen)
    x = torch.randn(6, 40, requires_grad=True)

    def run():
        with torch.autocast("cpu", torch.bfloat16):
            return m(x * 1.0)

    (want,), _ = _grads(run, x, context=False)
    (got,), packed = _grads(run, x, context=True)
    assert torch.equal(got, want)
    assert frozen or set(packed) == {(6, 40), (6, 24)}


def test_functional_call_and_attention():
    m = torch.nn.MultiheadAttention(32, 4, batch_first=True)
    x = torch.randn(2, 5, 32, requires_grad=True)
    plain = {k: v.detach().clone() for k, v in m.named_parameters()}

    def run():
        v = x * 1.0
        return torch.func.functional_call(m, plain, (v, v, v))[0]

    _, packed = _grads(run, x, context=True)
    assert packed and not any(s in ((96, 32), (32, 96), (32, 32))
                              for s in packed)


def test_an_input_that_wants_a_gradient_leaves_the_rest_packed():
    """It is a leaf, and as such like a weight; what follows from it is
    not."""
    x = torch.randn(6, 40, requires_grad=True)
    w = torch.nn.Parameter(torch.randn(24, 40))
    _, packed = _grads(lambda: torch.tanh(torch.tanh(x) @ w.t()), x,
                       context=True)
    assert packed.count((6, 40)) >= 1 and packed.count((6, 24)) == 1


def test_nested_contexts_and_threads_know_the_same_weights():
    import threading
    weight = _weight("weight norm")
    x = torch.randn(6, 40, requires_grad=True)

    def run(inner=contextlib.nullcontext):
        w = weight()
        with inner():
            return torch.nn.functional.linear(x * 1.0, w) + (x * 1.0) @ w.t()

    (want,), _ = _grads(run, x, context=False)
    (got,), _ = _grads(
        lambda: run(lambda: ops.activations_8bit(min_numel=1)), x,
        context=True)
    assert torch.equal(got, want) and not R.saving_8bit()
    seen = []
    with ops.activations_8bit():
        t = threading.Thread(target=lambda: seen.append(R.saving_8bit()))
        t.start()
        t.join()
        assert R.saving_8bit()
    assert seen == [False]


def test_sparse_operands_stay_as_they_are():
    p = torch.nn.Parameter(torch.randn(40, 24))
    x = torch.randn(6, 40)
    adjacency = torch.eye(6).to_sparse()

    def run():
        return torch.tanh(torch.sparse.mm(adjacency, x @ p))

    (got,), packed = _grads(run, p, context=True)
    assert set(packed) == {(6, 40), (6, 24)}
    assert bool(got.isfinite().all())


# ---------------------------------------------------------------------------
# gradients that divide by what is saved
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("fn", [
    torch.log, torch.sqrt, torch.log1p, lambda v: v ** 0.5, lambda v: 1 / v,
    lambda v: v / v.flip(0), lambda v: torch.nn.functional.normalize(v, dim=0),
    lambda v: v.std(0), lambda v: torch.linalg.vector_norm(v, dim=1),
    lambda v: v.norm(dim=1), lambda v: torch.div(2.0, v)],
    ids="log sqrt log1p pow reciprocal div normalize std vector_norm norm "
        "torch.div".split())
def test_finite_gradients_stay_finite(fn):
    """Positive maps with values below a unit of their group."""
    torch.manual_seed(7)
    x = torch.rand(64, 64).pow(8) + 1e-12
    x.requires_grad_()

    def run():
        return fn(x * 1.0)

    (want,), _ = _grads(run, x, context=False)
    (got,), _ = _grads(run, x, context=True)
    assert bool(want.isfinite().all())
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# layouts
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("op", ["row_norm", "bias_act", "norm_residual",
                                "linear"])
def test_rows_are_the_last_axis_in_any_layout(op):
    """A 4D tensor whose memory happens to be that of a channels_last map:
    its rows are kept, not its second axis."""
    torch.manual_seed(8)
    x = torch.randn(40, 1, 6, 5).permute(1, 2, 3, 0) * torch.arange(1.0, 41)
    x = x.contiguous(memory_format=torch.channels_last)
    assert x.is_contiguous(memory_format=torch.channels_last)
    dy = torch.randn(x.shape)
    w = torch.randn(40, 40)

    def grad(v):
        v = v.detach().requires_grad_()
        s = torch.ones(40, requires_grad=True)
        y = {"row_norm": lambda: ops.row_norm(v, s, save8=True),
             "bias_act": lambda: ops.bias_act(v, s, "hswish", save8=True),
             "norm_residual": lambda: ops.norm_residual(
                 v, v, scale=s, gate=v, next_norm=True, save8=True)[1],
             "linear": lambda: ops.linear(v, w * s, None, save8=True)}[op]()
        return torch.autograd.grad(y, [v, s], dy)

    for a, b in zip(grad(x), grad(x.contiguous())):
        assert torch.equal(a, b)
