"""Row operators: activations kept in 8 bits, and norms over channels.

A row is the last axis of a tensor (for an NHWC map: ``x.permute(0, 2, 3,
1)``, a free view of a channels_last tensor).  Two families, made to be used
together:

- What a backward pass needs can be kept in 8 bits.  :func:`pack_activation`
  is the codec; :func:`bias_act`, :func:`row_norm`, :func:`norm_residual` and
  ``linear`` take ``save8=True`` and then keep their inputs so, and read the
  codes in their backward kernels; :func:`activations_8bit` switches that on
  for a whole forward pass and packs what every other operator saves.
- :func:`row_norm` and :func:`norm_residual` are the norms before and after a
  residual block, the latter fused with the block's gate, its scale, the
  residual sum and the next block's norm.

**What 8 bits hold.**  Groups of 32 neighbouring channels share a power of
two, the smallest one with ``max|x| <= 127`` units; values are whole units.
Every value is off by at most half a unit (a whole one in the top binade of
the dtype, where nothing may round up to infinity).  A group that holds a
non-finite value gives its infinities back and NaN for all the rest.

**What the gradients mean.**  With ``save8`` the output is computed from the
true inputs, and the gradient is the operator's at the values that the codes
stand for: bit for bit the gradient of the same call on the unpacked inputs.
It can be taken once: there is no gradient of the gradient.

Dispatch is that of the op layer: GPU tensors run the HIP kernels
(csrc/act8.hip, rownorm_*, linear8.hip; their autograd is C++ too,
autograd_rows.cpp), CPU tensors and
``engine_mode() == "reference"`` a composition of torch operations.
"""

from __future__ import annotations

import contextlib
import functools
import threading
from typing import Callable, Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch.overrides import TorchFunctionMode
from torch.utils.weak import WeakTensorKeyDictionary

from .backend import ext, use_hip

GROUP = 32
#: fp16 has no step below 2^-24; below 2^-126 an fp32 unit is not normal
_LEAST = {torch.float16: -24, torch.bfloat16: -126, torch.float32: -126}
#: the unit of the dtype's top binade, where codes stop at 63
_LAST = {torch.float16: 10, torch.bfloat16: 122, torch.float32: 122}
MAX_NORM_CHANNELS = 16384
#: inputs and outputs of an FC layer whose input is kept in 8 bits
MAX_LINEAR_CHANNELS = 1 << 22

_GATE_NONE, _GATE_FULL, _GATE_GROUP = 0, 1, 2
_GATE_SIGMOID = 5
_ACT_HSIGMOID = 4
F32 = torch.float32


# ---------------------------------------------------------------------------
# rows
# ---------------------------------------------------------------------------

def _rows(x: torch.Tensor) -> torch.Tensor:
    """[rows, C]: a view where there is one."""
    c = x.shape[-1]
    return x if x.dim() == 2 else x.reshape(x.numel() // c, c)


def _check_rows(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} needs a last axis of channels, got shape "
                         f"{tuple(x.shape)}")


def _check_gpu_dtype(x: torch.Tensor, name: str) -> None:
    if x.dtype not in _LEAST:
        raise TypeError(f"{name} must be bf16, fp16 or fp32, got {x.dtype}")


def _param(p: Optional[torch.Tensor], c: int, name: str,
           x: torch.Tensor) -> None:
    if p is None:
        return
    if p.dim() != 1 or p.shape[0] != c:
        raise ValueError(f"{name} must have shape ({c},), got "
                         f"{tuple(p.shape)}")
    if p.device != x.device:
        raise ValueError(f"{name} is on {p.device}, the rows on {x.device}")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in tensors)


# ---------------------------------------------------------------------------
# the 8-bit form
# ---------------------------------------------------------------------------

class PackedActivation:
    """A tensor kept in 8 bits: ``codes`` (int8, [rows, C]), ``exponents``
    (uint8, one per 32 channels of a row; the unit is 2^(e - 127), 255 marks
    a group with a non-finite value), and what it was: ``shape``, ``dtype``,
    and whether its rows are the channels of a channels_last map."""

    __slots__ = ("codes", "exponents", "shape", "dtype", "nhwc")

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor,
                 shape: torch.Size, dtype: torch.dtype,
                 nhwc: bool = False) -> None:
        self.codes = codes
        self.exponents = exponents
        self.shape = shape
        self.dtype = dtype
        self.nhwc = nhwc

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exponents.numel()

    def unpack(self) -> torch.Tensor:
        """The values that the codes stand for, in the original dtype."""
        shape = self.shape
        if self.nhwc:
            n, c, h, w = shape
            shape = (n, h, w, c)
        if use_hip(self.codes):
            y = ext().unpack(self.codes, self.exponents, self.dtype, shape)
        else:
            y = _ref_unpack(self.codes, self.exponents,
                            self.dtype).view(shape)
        return y.permute(0, 3, 1, 2) if self.nhwc else y

    def __repr__(self) -> str:
        return (f"PackedActivation(shape={tuple(self.shape)}, "
                f"dtype={self.dtype}, nbytes={self.nbytes})")


def _is_nhwc(x: torch.Tensor) -> bool:
    return (x.dim() == 4
            and x.is_contiguous(memory_format=torch.channels_last)
            and not (x.is_contiguous() and x.shape[3] >= x.shape[1]))


def _fits(x: torch.Tensor) -> bool:
    """Whether the codec takes x in one call (2^31 chunks of 8 channels, rows
    padded to groups; 2^30 channels)."""
    c = x.shape[1 if _is_nhwc(x) else -1]
    return c < 1 << 30 and x.numel() // c * -(-c // GROUP) * 4 < 1 << 31


def pack_activation(x: torch.Tensor) -> PackedActivation:
    """Keep ``x`` in 8 bits.  Rows are the last axis; of a 4D channels_last
    tensor they are the channels.  (A tensor with one channel or one pixel
    is both: its rows are the longer axis.)"""
    _check_rows(x, "x")
    _check_gpu_dtype(x, "x")
    nhwc = _is_nhwc(x)
    rows = x.permute(0, 2, 3, 1) if nhwc else x
    if use_hip(x):
        codes, exps = ext().pack(rows)
    else:
        codes, exps = _ref_pack(_rows(rows.detach()))
    return PackedActivation(codes, exps, x.shape, x.dtype, nhwc)


def _ref_pack(rows: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    m, c = rows.shape
    g = (c + GROUP - 1) // GROUP
    v = F.pad(rows.float(), (0, g * GROUP - c)).view(m, g, GROUP)
    finite = torch.isfinite(v)
    sound = finite.all(dim=2, keepdim=True)
    a = torch.where(sound, v, 0.0)
    # |x| max = f * 2^p with f in [1/2, 1): 127 is 127/128 of 2^7
    f, p = torch.frexp(a.abs().amax(dim=2, keepdim=True))
    least = _LEAST[rows.dtype]
    e = (p - 7 + (f > 127 / 128).to(p.dtype)).clamp(min=least)
    e = torch.where(f > 0, e, least)
    top = torch.where(e >= _LAST[rows.dtype], 63.0, 127.0)
    unit = ((e + 127) << 23).to(torch.int32).view(F32)
    q = torch.minimum(torch.maximum(torch.round(a / unit), -top), top)
    q = torch.where(sound, q, torch.where(torch.isinf(v), torch.sign(v), 0.0))
    e = torch.where(sound, e + 127, 255)
    codes = q.to(torch.int8).view(m, g * GROUP)[:, :c].contiguous()
    return codes, e.to(torch.uint8).view(m, g)


def _ref_unpack(codes: torch.Tensor, exps: torch.Tensor,
                dtype: torch.dtype) -> torch.Tensor:
    c = codes.shape[1]
    unit = (exps.to(torch.int32) << 23).view(F32)
    unit = unit.repeat_interleave(GROUP, dim=1)[:, :c]
    return (codes.float() * unit).to(dtype)


# ---------------------------------------------------------------------------
# keeping everything in 8 bits
# ---------------------------------------------------------------------------

_local = threading.local()


def saving_8bit() -> bool:
    """Whether the calling thread is inside :func:`activations_8bit`."""
    return getattr(_local, "depth", 0) > 0


def _resolve(save8: Optional[bool]) -> bool:
    return saving_8bit() if save8 is None else bool(save8)


# Which saved tensors are weights, and stay as they are.  A weight is told by
# what it is (a parameter) or by how it is used (the weight argument of a
# layer); a mode that sees torch's calls follows what is made of parameters,
# and the framework's own layers name their weights (with_weights).

class _Call:
    """The call that is running: its weights and its other tensors."""

    __slots__ = ("weights", "others", "all", "casts")

    def __init__(self, weights, others=(), all=False, casts=True) -> None:
        self.weights = weights
        self.others = others  # those that are kept as they are, too
        self.all = all        # everything is: it makes a weight, or divides
        self.casts = casts    # autocast may have copied them

    def keeps(self, t: torch.Tensor) -> bool:
        if self.all:
            return True
        where = t.untyped_storage().data_ptr()
        return any(
            w.layout is torch.strided
            and (w.untyped_storage().data_ptr() == where
                 or (self.casts and w.numel() == t.numel()
                     and w.dtype != t.dtype))
            for group in (self.weights, self.others) for w in group)


def with_weights(fn: Callable, weights, *args):
    """``fn(*args)``, a layer of the framework; inside
    :func:`activations_8bit` its ``weights`` are saved as they are."""
    if not saving_8bit():
        return fn(*args)
    outer = getattr(_local, "call", None)
    _local.call = _Call([w for w in weights if w is not None], casts=False)
    try:
        with torch._C.DisableTorchFunction():
            return fn(*args)
    finally:
        _local.call = outer


def _unwatched(fn: Callable) -> Callable:
    """An operator of this module: the mode of :func:`activations_8bit` has
    nothing to see in it, and would see every attribute that it checks (some
    25 of a join, 2 us each)."""
    @functools.wraps(fn)
    def call(*args, **kwargs):
        if not saving_8bit():
            return fn(*args, **kwargs)
        with torch._C.DisableTorchFunction():
            return fn(*args, **kwargs)
    return call


#: torch's layers, and where their weight is among the arguments
_WEIGHT_AT = {"linear": 1, "bilinear": 2, "prelu": 1,
              **{f"conv{t}{d}d": 1 for d in (1, 2, 3)
                 for t in ("", "_transpose")}}
#: products, of which a tensor without a graph is an operand like a weight
_PRODUCTS = {*_WEIGHT_AT, "matmul", "__matmul__", "__rmatmul__", "mm", "bmm",
             "addmm", "baddbmm", "addbmm", "einsum", "tensordot", "mv",
             "inner", "outer", "multi_head_attention_forward"}
#: what divides by the tensors it saves: small values of a group become zero,
#: and a finite gradient infinite
_DIVIDES = {"div", "div_", "divide", "true_divide", "__truediv__", "__idiv__",
            "__itruediv__", "__rdiv__", "__rtruediv__", "reciprocal", "log",
            "log2", "log10", "log1p", "xlogy", "logit", "sqrt", "pow",
            "__pow__", "__rpow__", "float_power", "norm", "vector_norm",
            "linalg_vector_norm", "normalize", "cosine_similarity", "std",
            "std_mean", "prod", "cumprod", "atan2", "acosh", "asinh",
            "lgamma", "digamma"}
#: what a plain tensor, no larger than it, does to a weight: masking it
_MASKS = {"mul", "__mul__", "__rmul__", "where", "masked_fill"}


class _WeightsMode(TorchFunctionMode):
    """Sees the calls inside :func:`activations_8bit` and tells the saved
    tensors that are weights from the others."""

    def __init__(self) -> None:
        super().__init__()
        self.made = WeakTensorKeyDictionary()  # of parameters alone

    def of_parameters(self, t: torch.Tensor) -> bool:
        base = t if t._base is None else t._base
        return (isinstance(base, torch.nn.Parameter)
                or isinstance(t, torch.nn.Parameter)
                or (len(self.made) > 0
                    and (t in self.made or base in self.made)))

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = kwargs or {}
        name = getattr(func, "__name__", "")
        if name == "__get__":
            out = func(*args, **kwargs)
            if isinstance(out, torch.Tensor) and self.of_parameters(args[0]):
                self.made[out] = True  # W.data
            return out
        tensors = []
        for a in (*args, *kwargs.values()):
            if isinstance(a, torch.Tensor):
                tensors.append(a)
            elif isinstance(a, (list, tuple)):
                tensors += [t for t in a if isinstance(t, torch.Tensor)]
        if not tensors:
            return func(*args, **kwargs)
        params = [self.of_parameters(t) for t in tensors]
        at, used = _WEIGHT_AT.get(name), None
        if at is not None:
            used = kwargs.get("weight", args[at] if at < len(args) else None)
        weights, rest = [], []
        for t, p in zip(tensors, params):
            (weights if p or t is used or _is_weight(t) else rest).append(t)
        # a tensor without a graph beside one that has it: a coefficient of
        # a product, or one that is broadcast
        most = max((t.numel() for t in rest if t.requires_grad), default=-1)
        plain = [t for t in rest if not t.requires_grad and most >= 0
                 and (name in _PRODUCTS or t.numel() < most)]
        alone = all(params) or (
            name in _MASKS and any(params)
            and not any(t.requires_grad for t in rest)
            and max(t.numel() for t in weights)
            >= max((t.numel() for t in rest), default=0))
        outer = getattr(_local, "call", None)
        _local.call = _Call(weights, plain, alone or name in _DIVIDES)
        try:
            out = func(*args, **kwargs)
        finally:
            _local.call = outer
        if alone:
            for t in out if isinstance(out, (list, tuple)) else (out,):
                if isinstance(t, torch.Tensor):
                    self.made[t] = True
        return out


def _is_weight(t: torch.Tensor) -> bool:
    """A parameter (frozen or not), another leaf that wants a gradient, what
    a single operator (a cast) made of a parameter that wants one, or a view
    of any of these."""
    base = t if t._base is None else t._base
    if isinstance(base, torch.nn.Parameter):
        return True
    if base.is_leaf or t.is_leaf:
        return base.is_leaf and base.requires_grad
    nodes = base.grad_fn.next_functions
    return len(nodes) == 1 and isinstance(
        getattr(nodes[0][0], "variable", None), torch.nn.Parameter)


@contextlib.contextmanager
def activations_8bit(min_numel: int = 1 << 16):
    """Keep the activations of the forward pass run inside in 8 bits.

    The row operators and ``linear`` run as with ``save8=True``; what any
    other operator saves for its backward pass is packed on saving and
    unpacked on use, if it is a dense bf16, fp16 or fp32 tensor of two or
    more axes and at least ``min_numel`` elements, not a weight and not too
    large for one call; that holds for an operator called with
    ``save8=False`` too.  Put the model's forward inside and the loss outside: what a loss
    saves are gradients, not activations.

    Weights are: parameters, frozen or not, and other leaves that want a
    gradient; views of these; what is made inside from parameters alone, by
    any number of operators, and from a parameter and a mask; the weight
    argument of a layer (this framework's, torch's linear, bilinear, prelu
    and convolutions), whatever tensor it is; and a tensor without a graph
    that is multiplied with one that has it (a buffer).
    Anything else, as a weight made before the context and handed to
    ``matmul``, or to an autograd function of your own, is an activation.

    Small values of a group become zero, and a gradient that divides by them
    infinite.  Torch's operators that do so (division, ``log``, ``sqrt``,
    powers, norms and the like) are therefore left alone; an autograd function
    of your own that does belongs outside.

    Each operator keeps codes of its own, 1 + 1/32 bytes a value.  A tensor
    that several operators save costs that for each of them, where it would
    otherwise be saved once (2 bytes a value in bf16).

    A region under ``torch.utils.checkpoint`` is computed again in the
    backward pass, outside: pass ``save8`` to the operators in it (a region
    that is not computed again as it was raises an error there)."""
    if min_numel < 0:
        raise ValueError(f"min_numel must not be negative, got {min_numel}")

    outer = getattr(_local, "mode", None)
    mode = _WeightsMode() if outer is None else outer

    def pack(t: torch.Tensor):
        with torch._C.DisableTorchFunction():
            if (t.dtype not in _LEAST or t.layout is not torch.strided
                    or t.dim() < 2 or t.numel() == 0
                    or t.numel() < min_numel or not _fits(t)
                    or _is_weight(t) or mode.of_parameters(t)):
                return t
            call = getattr(_local, "call", None)
            return (t if call is not None and call.keeps(t)
                    else pack_activation(t))

    def unpack(kept):
        return kept.unpack() if isinstance(kept, PackedActivation) else kept

    with (mode if outer is None else contextlib.nullcontext()), \
            torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        _local.depth = getattr(_local, "depth", 0) + 1
        _local.mode = mode
        try:
            yield
        finally:
            _local.depth -= 1
            _local.mode = outer


class _Keep8Fn(torch.autograd.Function):
    """Reference: ``fn(*tensors)``, with the gradient of fn at the unpacked
    values of the tensors named by ``kept``."""

    @staticmethod
    def forward(ctx, fn: Callable, kept: Tuple[bool, ...], *tensors):
        with torch.no_grad():
            out = fn(*tensors)
        saved, ctx.form = [], []
        for t, k in zip(tensors, kept):
            if t is not None and k:
                # by rows, whatever the layout: not as pack_activation, which
                # takes the channels of a channels_last map
                _check_gpu_dtype(t, "what is kept in 8 bits")
                saved += _ref_pack(_rows(t.detach()))
                ctx.form.append((t.shape, t.dtype))
            else:
                saved.append(t)
                ctx.form.append(None)
        ctx.save_for_backward(*saved)
        ctx.fn = fn
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *douts):
        saved, args = iter(ctx.saved_tensors), []
        for f in ctx.form:
            t = next(saved)
            if f is not None:
                t = PackedActivation(t, next(saved), *f).unpack()
            args.append(t)
        needs = ctx.needs_input_grad[2:]
        args = [t if t is None else t.detach().requires_grad_(n)
                for t, n in zip(args, needs)]
        with torch.enable_grad():
            outs = ctx.fn(*args)
        outs = outs if isinstance(outs, tuple) else (outs,)
        leaves = [t for t in args if t is not None and t.requires_grad]
        grads = iter(torch.autograd.grad(outs, leaves, douts,
                                         allow_unused=True))
        return (None, None) + tuple(
            next(grads) if t is not None and t.requires_grad else None
            for t in args)


def _reference(fn: Callable, kept: Tuple[bool, ...], save8: bool, *tensors):
    if save8 and _wants_grad(*tensors):
        return _Keep8Fn.apply(fn, kept, *tensors)
    return fn(*tensors)


def _up(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.dtype is torch.float64 else t.float()


# ---------------------------------------------------------------------------
# bias + activation
# ---------------------------------------------------------------------------

@_unwatched
def bias_act(z: torch.Tensor, bias: Optional[torch.Tensor] = None,
             act: Union[int, str] = 0, save8: Optional[bool] = None
             ) -> torch.Tensor:
    """``act(z + bias)`` over the last axis, in the dtype of ``z``.

    ``act`` is an activation's name or code; ``save8`` keeps ``z`` in 8 bits
    for the backward pass (default: as :func:`activations_8bit` says)."""
    from .functional import act_code, apply_act
    _check_rows(z, "z")
    code = act_code(act)
    if not 0 <= code <= 3:
        raise ValueError(f"bad act code {code}")
    _param(bias, z.shape[-1], "bias", z)
    save8 = _resolve(save8)
    if use_hip(z):
        _check_gpu_dtype(z, "z")
        return ext().bias_act(z, bias, code, save8)

    def fn(z, bias):
        v = _up(z)
        if bias is not None:
            v = v + _up(bias)
        return apply_act(v, code).to(z.dtype)

    return _reference(fn, (True, False), save8, z, bias)


# ---------------------------------------------------------------------------
# FC layer on an input kept in 8 bits
# ---------------------------------------------------------------------------

def linear_fits(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether :func:`linear8` takes a layer of this size: its channels, the
    codec's chunks, and 2^24 tiles of 64 x 64 for each of its products."""
    if weight.dim() != 2 or weight.numel() == 0:
        return True  # refused by name
    n, k = weight.shape
    m = x.numel() // k
    t = [-(-v // 64) for v in (m, n, k)]
    return (max(n, k) <= MAX_LINEAR_CHANNELS
            and m * -(-k // GROUP) * 4 < 1 << 31
            and max(t[0] * t[1], t[0] * t[2], t[1] * t[2]) < 1 << 24)


@_unwatched
def linear8(x: torch.Tensor, weight: torch.Tensor,
            bias: Optional[torch.Tensor], act: int,
            save8: bool = True) -> torch.Tensor:
    """``linear`` with ``save8``: ``act(x @ weight.T + bias)`` over the last
    axis of x; x, and z = x @ weight.T where there is an activation, are
    kept in 8 bits.  GPU: bf16 in and out (like ``linear``, rows of other
    dtypes are rounded to it); weights count with 15 bits and more."""
    _check_rows(x, "x")
    if (x.dim() > 2 and weight.dim() == 2 and x.shape[-1] != weight.shape[1]
            and x.shape[1:].numel() == weight.shape[1]):
        x = x.flatten(1)  # pooled maps, as `linear` takes them
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight must be [out, {x.shape[-1]}], got "
                         f"{tuple(weight.shape)}")
    if weight.shape[0] < 1:
        raise ValueError("weight has no outputs")
    if use_hip(x) and max(weight.shape) > MAX_LINEAR_CHANNELS:
        raise ValueError(f"an FC layer with save8 takes at most "
                         f"{MAX_LINEAR_CHANNELS} inputs and outputs, got "
                         f"{tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, x on {x.device}")
    _param(bias, weight.shape[0], "bias", x)
    if use_hip(x):
        z = with_weights(ext().linear8, (weight,), x, weight,
                         bias if act == 0 else None)
    else:
        z = with_weights(_reference, (weight,),
                         lambda x, w, b: F.linear(x, w, b),
                         (True, False, False), save8, x, weight,
                         bias if act == 0 else None)
    return z if act == 0 else bias_act(z, bias, act, save8)


# ---------------------------------------------------------------------------
# norms over channels
# ---------------------------------------------------------------------------

def _kind(kind: str, eps: float, *biases) -> bool:
    if kind not in ("rms", "layer"):
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if kind == "rms" and any(b is not None for b in biases):
        raise ValueError("an rms norm has no bias")
    return kind == "layer"


def _ref_norm(v, w, b, layer: bool, eps: float):
    if layer:
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        v = v * _up(w)
    return v if b is None else v + _up(b)


def _check_norm_rows(x: torch.Tensor, name: str) -> None:
    _check_rows(x, name)
    if use_hip(x):
        _check_gpu_dtype(x, name)
        if x.shape[-1] > MAX_NORM_CHANNELS:
            raise ValueError(f"norms take at most {MAX_NORM_CHANNELS} "
                             f"channels, got {x.shape[-1]}")


@_unwatched
def row_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
             bias: Optional[torch.Tensor] = None, *, kind: str = "rms",
             eps: float = 1e-6, save8: Optional[bool] = None
             ) -> torch.Tensor:
    """The norm before a block: every row of x over its last axis.

    ``kind="rms"``: ``weight * x / sqrt(mean(x^2) + eps)``;
    ``kind="layer"``: the same of ``x - mean(x)``, plus ``bias``.  Statistics
    are fp32, the result has the dtype of x.  ``save8`` keeps x in 8 bits
    for the backward pass (default: as :func:`activations_8bit` says)."""
    _check_norm_rows(x, "x")
    layer = _kind(kind, eps, bias)
    c = x.shape[-1]
    _param(weight, c, "weight", x)
    _param(bias, c, "bias", x)
    save8 = _resolve(save8)
    if use_hip(x):
        return ext().join(None, x, None, None, None, None, weight, bias,
                          layer, False, True, _GATE_NONE, 0, eps, 1.0,
                          save8)[0]

    def fn(x, w, b):
        return _ref_norm(_up(x), w, b, layer, eps).to(x.dtype)

    return _reference(fn, (True, False, False), save8, x, weight, bias)


def _gate_code(name: str) -> int:
    codes = {"identity": 0, "hsigmoid": _ACT_HSIGMOID,
             "sigmoid": _GATE_SIGMOID}
    try:
        return codes[name]
    except (KeyError, TypeError):
        raise ValueError(f"gate_act must be one of {sorted(codes)}, got "
                         f"{name!r}") from None


@_unwatched
def norm_residual(
    h: torch.Tensor, x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None, *,
    gate: Optional[torch.Tensor] = None, gate_act: str = "identity",
    scale: Union[None, float, torch.Tensor] = None,
    post_norm: bool = True, next_norm: bool = False,
    next_weight: Optional[torch.Tensor] = None,
    next_bias: Optional[torch.Tensor] = None,
    kind: str = "rms", eps: float = 1e-6, save8: Optional[bool] = None,
):
    """The join after a residual block, in one pass over its rows::

        y = x + scale * gate_act(gate) * N(h)      N: row_norm of h
        u = N'(y)                                  the next block's norm

    ``h`` is the block's output and ``x`` the residual stream.  ``gate``
    has the shape of x, or ``(x.shape[0], x.shape[-1])`` for one gate per
    image or sequence and channel; ``gate_act`` is "identity", "hsigmoid" or
    "sigmoid".  ``scale`` is a number or one value per channel.
    ``post_norm=False`` takes h as it is; ``next_norm=True`` returns
    ``(y, u)`` instead of ``y``, with u computed from y before it is
    rounded.  ``weight``/``bias`` and ``next_weight``/``next_bias`` are the
    two norms' parameters.  ``save8`` keeps h, x and the gate in 8 bits for
    the backward pass (default: as :func:`activations_8bit` says)."""
    _check_norm_rows(x, "x")
    _check_norm_rows(h, "h")
    layer = _kind(kind, eps, bias, next_bias)
    c = x.shape[-1]
    if h.shape != x.shape or h.dtype != x.dtype or h.device != x.device:
        raise ValueError(
            f"h and x must agree: {tuple(h.shape)} {h.dtype} {h.device}, "
            f"{tuple(x.shape)} {x.dtype} {x.device}")
    if not post_norm and (weight is not None or bias is not None):
        raise ValueError("weight and bias belong to the post norm")
    if not next_norm and (next_weight is not None or next_bias is not None):
        raise ValueError("next_weight and next_bias belong to the next norm")
    gact = _gate_code(gate_act)
    gmode = _GATE_NONE
    if gate is not None:
        if gate.dtype != x.dtype or gate.device != x.device:
            raise ValueError(f"gate must be {x.dtype} on {x.device}, got "
                             f"{gate.dtype} on {gate.device}")
        if gate.shape == x.shape:
            gmode = _GATE_FULL
        elif x.dim() >= 3 and tuple(gate.shape) == (x.shape[0], c):
            # one row each is a gate for every row
            gmode = (_GATE_FULL if x.numel() == gate.numel()
                     else _GATE_GROUP)
        else:
            raise ValueError(
                f"gate must have shape {tuple(x.shape)}"
                + (f" or {(x.shape[0], c)}" if x.dim() >= 3 else "")
                + f", got {tuple(gate.shape)}")
    elif gact != 0:
        raise ValueError("gate_act without a gate")
    alpha = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        alpha, scale = float(scale), None
    for p, name in ((weight, "weight"), (bias, "bias"), (scale, "scale"),
                    (next_weight, "next_weight"), (next_bias, "next_bias")):
        _param(p, c, name, x)
    save8 = _resolve(save8)
    tensors = (h, x, gate, weight, bias, scale, next_weight, next_bias)
    if use_hip(x):
        outs = ext().join(*tensors, layer, post_norm, next_norm, gmode, gact,
                          eps, alpha, save8)
        return tuple(outs) if next_norm else outs[0]

    def fn(h, x, gate, w, b, scale, w2, b2):
        t = _up(h)
        if post_norm:
            t = _ref_norm(t, w, b, layer, eps)
        if gate is not None:
            g = _up(gate)
            if gate.shape != x.shape:
                g = g.view((g.shape[0],) + (1,) * (x.dim() - 2) + (c,))
            t = t * (torch.sigmoid(g) if gact == _GATE_SIGMOID else
                     F.hardsigmoid(g) if gact == _ACT_HSIGMOID else g)
        t = t * alpha
        if scale is not None:
            t = t * _up(scale)
        y = _up(x) + t
        if not next_norm:
            return y.to(x.dtype)
        return (y.to(x.dtype),
                _ref_norm(y, w2, b2, layer, eps).to(x.dtype))

    return _reference(fn, (True, True, True) + (False,) * 5, save8, *tensors)
