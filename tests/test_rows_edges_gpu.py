"""Row operators on the GPU where values, types and sizes are at their ends,
against their definitions in 64 bits or the same call on plain inputs."""

import pytest
import torch

from yet_another_mobilenet_series_amd import ops

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DEV = "cuda:0"
U32 = 2.0 ** -24


def _rand(seed, *shape, dtype=F32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _within(got, want, scale, what=""):
    """Half a step of the output's type, and `scale` for the arithmetic."""
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * want.abs() + scale + 2 * fi.smallest_normal
    off = (got.detach().double() - want).abs()
    assert bool((off <= tol).all()), (what, float((off / tol).max()))


# ---------------------------------------------------------------------------
# FC layer: weights of more bits than bf16
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("wtype", [F32, F16])
@pytest.mark.parametrize("m,k,n,bias", [
    (1, 1, 1, True), (3, 33, 17, True), (1, 1280, 1000, True),
    (256, 1280, 1000, True), (65, 96, 129, False), (1021, 965, 499, True),
    (20001, 24, 72, True), (333, 2048, 512, False), (3001, 1000, 5003, True)])
def test_linear_uses_what_weights_have_beyond_bf16(wtype, m, k, n, bias):
    """Weights go in as two bf16 parts, which leave at most 2^-7 2^-8 of a
    weight out; sums in fp32 add at most 256 2^-24 of their terms."""
    x = _rand(m + k, m, k, dtype=BF16).requires_grad_()
    w = (_rand(n, n, k) / k ** 0.5).to(wtype).requires_grad_()
    b = _rand(7, n).requires_grad_() if bias else None
    dy = _rand(11, m, n, dtype=BF16)
    y = ops.linear(x, w, b, save8=True)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    x64, w64, d64 = (t.detach().double() for t in (x, w, dy))
    b64 = b.detach().double() if bias else torch.zeros(n, device=DEV).double()
    err = 256 * U32 + 2.0 ** -15
    _within(y, x64 @ w64.t() + b64,
            err * (x64.abs() @ w64.abs().t() + b64.abs()), "y")
    _within(dx, d64 @ w64, err * (d64.abs() @ w64.abs()), "dx")
    assert dw.dtype is wtype


@pytest.mark.parametrize("m,k,n", [(5, 40, 24), (300, 320, 264)])
def test_linear_keeps_infinite_and_largest_weights_apart(m, k, n):
    """The largest fp32 stays finite, an infinity gives infinities and no
    NaN, a NaN (with any payload) NaN, each in its own column of y."""
    x = _rand(1, m, k, dtype=BF16).abs() + 0.5
    w = _rand(2, n, k) / k
    w[1, 3] = float("inf")
    w[2, 4] = -float("inf")
    w[3, 5] = torch.finfo(F32).max
    w[4, 6] = torch.tensor(0x7F800001, dtype=torch.int32).view(F32)
    y = ops.linear(x * 2.0 ** -10, w, None, save8=True).float()
    assert bool((y[:, 1] == float("inf")).all())
    assert bool((y[:, 2] == -float("inf")).all())
    assert bool(y[:, 4].isnan().all())
    rest = [j for j in range(n) if j not in (1, 2, 4)]
    want = (x.double() * 2.0 ** -10) @ w[rest].double().t()
    assert bool((y[:, rest].double() - want).abs().le(
        2.0 ** -7 * want.abs() + 1e-6).all())
