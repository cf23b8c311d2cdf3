"""Low-bit operators of the model's own forward and backward step, between two outer steps.

The compression ops (``prime_amd.ops``) hold what a worker sends in 8-bit codes; these hold what it
computes with: activations as 8-bit codes with one scale per row, weights as 4-bit codes with one
scale per group of a row.

    rms_norm_quantize           RMS norm of rows as int8 or e4m3 codes with one scale per row
    add_rms_norm_quantize       the same after the residual's addition, which it returns too
    rms_norm_quantize_backward  gradients of the norm's input and weight, straight through the codes
    quantize_4bit               a weight matrix as 4-bit codes with a scale per 32, 64 or 128
    dequantize_4bit             the matrix such codes stand for
    matvec_4bit                 products of a few rows (floating point, or int8 codes with scales) with it

The norm stands in for src/zeroband/models/norms.py:128,176; the others have no counterpart there.

Registered as ``torch.library`` ops in the namespace ``prime_lowbit`` (``prime::`` is the closed set
of the compression path), for ROCm tensors only: a CPU tensor reaches no kernel and the dispatcher
raises.  The functions below take plain CUDA tensors of an eager call straight to the C ABI and everything
else (fake and CPU tensors, tensor subclasses, calls under ``torch.compile``, a tracer, a dispatch mode or a
``torch.func`` transform, forward-mode duals) to the dispatcher.  Every call runs on the current stream of its tensors'
device, allocates its outputs (and the backward pass its scratch) from torch's caching allocator,
and can be captured into a HIP graph.

Codes carry no gradient, so a call whose inputs require one, or carry a tangent, is refused while gradients
are being recorded; inside a ``torch.autograd.Function`` (or ``torch.no_grad()``) pair
``add_rms_norm_quantize`` with ``rms_norm_quantize_backward``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _raw_stream, _stream

GROUP_SIZES = (32, 64, 128)
CODE_DTYPES = (torch.int8, torch.float8_e4m3fn)
MAX_DIM = 1 << 30

# element types of the C ABI
_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_SCALES = (torch.float32, torch.bfloat16)

_LIB = torch.library.Library("prime_lowbit", "DEF")
_LIB.define("rms_norm_quantize(Tensor x, Tensor weight, float eps=1e-06, ScalarType dtype=int8) -> (Tensor, Tensor, Tensor)")
_LIB.define("add_rms_norm_quantize(Tensor x, Tensor residual, Tensor weight, float eps=1e-06, ScalarType dtype=int8) "
            "-> (Tensor, Tensor, Tensor, Tensor)")
_LIB.define("rms_norm_quantize_backward(Tensor grad, Tensor hidden, Tensor weight, Tensor inv_rms, Tensor? grad_hidden=None) -> (Tensor, Tensor)")
_LIB.define("quantize_4bit(Tensor weight, int group_size=128, ScalarType scale_dtype=bfloat16) -> (Tensor, Tensor)")
_LIB.define("dequantize_4bit(Tensor packed, Tensor scales, int? columns=None, ScalarType dtype=float) -> Tensor")
_LIB.define("matvec_4bit(Tensor x, Tensor packed, Tensor scales, Tensor? x_scales=None, ScalarType? dtype=None) -> Tensor")


# looked up once: a call's time on the host is what bounds the small ones
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_compiling = torch.compiler.is_compiling
_dispatch_modes = torch._C._len_torch_dispatch_stack
_transform = torch._C._functorch.peek_interpreter_stack
_tracing_state = torch._C._get_tracing_state
_stream_of = _raw_stream if _raw_stream is not None else lambda index: _stream(torch.device("cuda", index))


def _fail(name: str, what: str):
    raise RuntimeError(f"{name}: {what}")


def _no_gradient(name: str):
    _fail(name, "records no gradient; call it inside a torch.autograd.Function or under torch.no_grad()")


def _check_inputs(name: str, dev: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    """One device, and no gradient asked of an op that records none."""
    grads = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if t.device != dev:
            _fail(name, f"all tensors must live on one device, got {t.device} beside {dev}")
        if grads and t.requires_grad:
            _no_gradient(name)


def _wants_gradient(*tensors: Optional[torch.Tensor]) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return torch.is_grad_enabled()
    return False


def _rows(t: torch.Tensor, dim: int) -> Tuple[torch.Tensor, int]:
    """(``t``, or a copy where its strides ask for one, elements from row to row): rows of ``dim`` consecutive elements."""
    if t.is_contiguous():
        return t, dim
    v = t if t.dim() == 2 else t.reshape(-1, dim)
    if v.stride(1) != 1 and dim > 1:
        v = v.contiguous()
    return v, v.stride(0)


def _like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised dense tensor of ``t``'s shape (from a dense one in half the time)."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else torch.empty(t.shape, dtype=dtype, device=t.device)


def _check_norm(name: str, x: torch.Tensor, weight: torch.Tensor, like: Tuple[Tuple[str, Optional[torch.Tensor]], ...] = ()) -> int:
    if x.dtype not in _FLOATS:
        _fail(name, f"expected Float, BFloat16 or Half rows but found {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > MAX_DIM:
        _fail(name, f"rows of 1 to 2^30 elements are needed, got shape {tuple(x.shape)}")
    dim = x.shape[-1]
    if weight.dim() != 1 or weight.shape[0] != dim:
        _fail(name, f"weight needs shape ({dim},), got {tuple(weight.shape)}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        _fail(name, f"weight must be Float or of the rows' type {x.dtype}, got {weight.dtype}")
    for what, t in like:
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            _fail(name, f"{what} must have shape {tuple(x.shape)} and type {x.dtype}, got {tuple(t.shape)} and {t.dtype}")
    return dim


def _check_norm_call(name: str, x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float, dtype: torch.dtype) -> None:
    _check_norm(name, x, weight, (("residual", residual),))
    if dtype not in CODE_DTYPES:
        _fail(name, f"codes are torch.int8 or torch.float8_e4m3fn, got {dtype}")
    if not eps >= 0.0:
        _fail(name, f"eps must not be negative, got {eps}")
    _check_inputs(name, x.device, x, residual, weight)


def _check_backward_call(name: str, grad: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor, inv_rms: torch.Tensor,
                         grad_hidden: Optional[torch.Tensor]) -> None:
    _check_norm(name, hidden, weight, (("grad", grad), ("grad_hidden", grad_hidden)))
    if inv_rms.dtype != torch.float32 or inv_rms.shape != hidden.shape[:-1]:
        _fail(name, f"inv_rms must be Float of shape {tuple(hidden.shape[:-1])}, got {inv_rms.dtype} of {tuple(inv_rms.shape)}")
    _check_inputs(name, hidden.device, grad, hidden, weight, inv_rms, grad_hidden)


def _norm(name: str, x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float, dtype: torch.dtype):
    xt, wt, shape, dev = x.dtype, weight.dtype, x.shape, x.device
    # one expression for the calls that are right; the checks that say what is wrong run only for the others
    if not (xt in _FLOATS and len(shape) > 0 and weight.shape == shape[-1:] and 0 < shape[-1] <= MAX_DIM and (wt is xt or wt is torch.float32)
            and dtype in CODE_DTYPES and eps >= 0.0 and weight.device == dev
            and (residual is None or (residual.shape == shape and residual.dtype is xt and residual.device == dev))
            and not _wants_gradient(x, weight, residual)):
        _check_norm_call(name, x, residual, weight, eps, dtype)
    dim = shape[-1]
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _norm(name, x, residual, weight, eps, dtype)
    lib = _lib.load()
    lead = shape[:-1]
    x2, xs = _rows(x, dim)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    codes = _like(x, dtype)
    scales = x.new_empty(lead, dtype=torch.float32)
    inv_rms = x.new_empty(lead, dtype=torch.float32)
    hidden = None
    rp = hp = None
    rs = 0
    if residual is not None:
        r2, rs = _rows(residual, dim)
        hidden = _like(x, xt)
        rp, hp = r2.data_ptr(), hidden.data_ptr()
    rc = lib.prime_rms_norm_quantize(x2.data_ptr(), xs, rp, rs, weight.data_ptr(), x.numel() // dim, dim, _TYPE[xt], _TYPE[wt], _TYPE[dtype], eps,
                                     codes.data_ptr(), scales.data_ptr(), hp, inv_rms.data_ptr(), _stream_of(dev.index))
    if rc:
        _lib.check(rc, "prime_rms_norm_quantize")
    return codes, scales, hidden, inv_rms


def _rms_norm_quantize(x, weight, eps=1e-6, dtype=torch.int8):
    codes, scales, _, inv_rms = _norm("rms_norm_quantize", x, None, weight, eps, dtype)
    return codes, scales, inv_rms


def _add_rms_norm_quantize(x, residual, weight, eps=1e-6, dtype=torch.int8):
    return _norm("add_rms_norm_quantize", x, residual, weight, eps, dtype)


def _rms_norm_quantize_backward(grad, hidden, weight, inv_rms, grad_hidden=None):
    name = "rms_norm_quantize_backward"
    ht, wt, shape, dev = hidden.dtype, weight.dtype, hidden.shape, hidden.device
    if not (ht in _FLOATS and len(shape) > 0 and weight.shape == shape[-1:] and 0 < shape[-1] <= MAX_DIM and (wt is ht or wt is torch.float32)
            and grad.shape == shape and grad.dtype is ht and inv_rms.dtype is torch.float32 and inv_rms.shape == shape[:-1]
            and grad.device == dev and weight.device == dev and inv_rms.device == dev
            and (grad_hidden is None or (grad_hidden.shape == shape and grad_hidden.dtype is ht and grad_hidden.device == dev))
            and not _wants_gradient(grad, hidden, weight, inv_rms, grad_hidden)):
        _check_backward_call(name, grad, hidden, weight, inv_rms, grad_hidden)
    dim = shape[-1]
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _rms_norm_quantize_backward(grad, hidden, weight, inv_rms, grad_hidden)
    lib = _lib.load()
    g2, gs = _rows(grad, dim)
    h2, hs = _rows(hidden, dim)
    dp, ds = None, 0
    if grad_hidden is not None:
        d2, ds = _rows(grad_hidden, dim)
        dp = d2.data_ptr()
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if not inv_rms.is_contiguous():
        inv_rms = inv_rms.contiguous()
    rows = hidden.numel() // dim
    grad_x = _like(hidden, ht)
    grad_weight = torch.empty_like(weight)
    # the call's own scratch and no workspace of the stream: a captured call keeps it in its graph's memory
    nbytes = lib.prime_rms_norm_backward_scratch_bytes(rows, dim)
    scratch = hidden.new_empty((nbytes,), dtype=torch.uint8)
    rc = lib.prime_rms_norm_quantize_backward(g2.data_ptr(), gs, h2.data_ptr(), hs, weight.data_ptr(), inv_rms.data_ptr(), dp, ds, rows, dim,
                                              _TYPE[ht], _TYPE[wt], grad_x.data_ptr(), grad_weight.data_ptr(), scratch.data_ptr(), nbytes, _stream_of(dev.index))
    if rc:
        _lib.check(rc, "prime_rms_norm_quantize_backward")
    return grad_x, grad_weight


def _groups(name: str, k: int, group_size: int) -> int:
    if group_size not in GROUP_SIZES:
        _fail(name, f"group size must be one of {GROUP_SIZES}, got {group_size}")
    return -(-k // group_size)


def _check_quantize(name: str, weight: torch.Tensor, group_size: int, scale_dtype: torch.dtype) -> Tuple[int, int, int]:
    """(rows, columns, groups of a row) of a matrix to be packed."""
    if weight.dtype not in _FLOATS:
        _fail(name, f"expected a Float, BFloat16 or Half weight but found {weight.dtype}")
    if weight.dim() != 2 or weight.shape[1] < 1 or weight.shape[1] > MAX_DIM:
        _fail(name, f"a matrix with rows of 1 to 2^30 weights is needed, got shape {tuple(weight.shape)}")
    if scale_dtype not in _SCALES:
        _fail(name, f"scales are torch.bfloat16 or torch.float32, got {scale_dtype}")
    if _wants_gradient(weight):
        _no_gradient(name)
    n, k = weight.shape
    return n, k, _groups(name, k, group_size)


def _quantize_4bit(weight, group_size=128, scale_dtype=torch.bfloat16):
    n, k, groups = _check_quantize("quantize_4bit", weight, group_size, scale_dtype)
    dev = weight.device
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _quantize_4bit(weight, group_size, scale_dtype)
    lib = _lib.load()
    w, stride = _rows(weight, k)
    packed = weight.new_empty((n, groups * group_size // 2), dtype=torch.uint8)
    scales = weight.new_empty((n, groups), dtype=scale_dtype)
    rc = lib.prime_quantize_4bit(w.data_ptr(), stride, n, k, _TYPE[w.dtype], group_size, _TYPE[scale_dtype], packed.data_ptr(),
                                 scales.data_ptr(), _stream_of(dev.index))
    if rc:
        _lib.check(rc, "prime_quantize_4bit")
    return packed, scales


def _check_packed(name: str, packed: torch.Tensor, scales: torch.Tensor, columns: Optional[int]) -> Tuple[int, int, int]:
    """(rows, columns, group size) of a 4-bit matrix."""
    if packed.dtype is torch.uint8 and scales.dtype in _SCALES and packed.dim() == 2 and scales.dim() == 2:
        n, held = packed.shape
        rows, groups = scales.shape
        held *= 2
        if rows == n and groups > 0:
            group = held // groups
            k = held if columns is None else columns
            if group in GROUP_SIZES and group * groups == held <= MAX_DIM and held - group < k <= held:
                return n, k, group
    if packed.dtype != torch.uint8 or scales.dtype not in _SCALES:
        _fail(name, f"expected Byte codes and Float or BFloat16 scales but found {packed.dtype} and {scales.dtype}")
    if packed.dim() != 2 or scales.dim() != 2 or packed.shape[0] != scales.shape[0] or scales.shape[1] < 1:
        _fail(name, f"codes and scales must be matrices with the same rows, got shapes {tuple(packed.shape)} and {tuple(scales.shape)}")
    held, groups = 2 * packed.shape[1], scales.shape[1]
    group = held // groups
    if group not in GROUP_SIZES or group * groups != held or held > MAX_DIM:
        _fail(name, f"{held} codes and {groups} scales a row do not make groups of {GROUP_SIZES}")
    k = held if columns is None else int(columns)
    if not held - group < k <= held:
        _fail(name, f"rows of {groups} groups of {group} hold {held - group + 1} to {held} columns, not {k}")
    return packed.shape[0], k, group


def _dense_rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() or t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check_dequantize(name: str, packed: torch.Tensor, scales: torch.Tensor, columns: Optional[int], dtype: torch.dtype) -> Tuple[int, int, int]:
    sizes = _check_packed(name, packed, scales, columns)
    if dtype not in _FLOATS:
        _fail(name, f"weights are Float, BFloat16 or Half, got {dtype}")
    if scales.device != packed.device or _wants_gradient(scales):
        _check_inputs(name, packed.device, packed, scales)
    return sizes


def _dequantize_4bit(packed, scales, columns=None, dtype=torch.float32):
    n, k, group = _check_dequantize("dequantize_4bit", packed, scales, columns, dtype)
    dev = packed.device
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _dequantize_4bit(packed, scales, columns, dtype)
    lib = _lib.load()
    packed, scales = _dense_rows(packed), _dense_rows(scales)
    out = packed.new_empty((n, k), dtype=dtype)
    rc = lib.prime_dequantize_4bit(packed.data_ptr(), packed.stride(0), scales.data_ptr(), scales.stride(0), n, k, group, _TYPE[scales.dtype],
                                   out.data_ptr(), _TYPE[dtype], _stream_of(dev.index))
    if rc:
        _lib.check(rc, "prime_dequantize_4bit")
    return out


def _check_matvec(name: str, x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, x_scales: Optional[torch.Tensor],
                  dtype: Optional[torch.dtype]) -> Tuple[int, int, int, torch.dtype]:
    if x.dtype not in _FLOATS and x.dtype != torch.int8:
        _fail(name, f"expected Float, BFloat16, Half or Char rows but found {x.dtype}")
    if x.dim() < 1:
        _fail(name, "rows are needed, got a scalar")
    n, k, group = _check_packed(name, packed, scales, x.shape[-1])
    if (x.dtype == torch.int8) != (x_scales is not None):
        _fail(name, "int8 rows come with x_scales, and no others do")
    if x_scales is not None and (x_scales.dtype != torch.float32 or x_scales.shape != x.shape[:-1]):
        _fail(name, f"x_scales must be Float of shape {tuple(x.shape[:-1])}, got {x_scales.dtype} of {tuple(x_scales.shape)}")
    if dtype is None:
        dtype = torch.float32 if x.dtype == torch.int8 else x.dtype
    if dtype not in _FLOATS:
        _fail(name, f"products are Float, BFloat16 or Half, got {dtype}")
    dev = x.device
    if packed.device != dev or scales.device != dev or (x_scales is not None and x_scales.device != dev) or _wants_gradient(x, scales, x_scales):
        _check_inputs(name, dev, x, packed, scales, x_scales)
    return n, k, group, dtype


def _matvec_4bit(x, packed, scales, x_scales=None, dtype=None):
    n, k, group, dtype = _check_matvec("matvec_4bit", x, packed, scales, x_scales, dtype)
    dev = x.device
    if _current_device() != dev.index:
        with torch.cuda.device(dev):
            return _matvec_4bit(x, packed, scales, x_scales, dtype)
    lib = _lib.load()
    x2, stride = _rows(x, k)
    packed, scales = _dense_rows(packed), _dense_rows(scales)
    xp = None
    if x_scales is not None:
        x_scales = x_scales.contiguous()
        xp = x_scales.data_ptr()
    shape = x.shape
    out = x.new_empty((shape[0], n) if len(shape) == 2 else shape[:-1] + (n,), dtype=dtype)
    rc = lib.prime_matvec_4bit(x2.data_ptr(), stride, _TYPE[x.dtype], xp, packed.data_ptr(), packed.stride(0), scales.data_ptr(), scales.stride(0),
                               x.numel() // k, n, k, group, _TYPE[scales.dtype], out.data_ptr(), _TYPE[dtype], _stream_of(dev.index))
    if rc:
        _lib.check(rc, "prime_matvec_4bit")
    return out


_LIB.impl("rms_norm_quantize", _rms_norm_quantize, "CUDA")
_LIB.impl("add_rms_norm_quantize", _add_rms_norm_quantize, "CUDA")
_LIB.impl("rms_norm_quantize_backward", _rms_norm_quantize_backward, "CUDA")
_LIB.impl("quantize_4bit", _quantize_4bit, "CUDA")
_LIB.impl("dequantize_4bit", _dequantize_4bit, "CUDA")
_LIB.impl("matvec_4bit", _matvec_4bit, "CUDA")


# What the dispatcher asks first where gradients could be recorded: it refuses, in reverse and in forward mode, what the ops could only drop.
def _refusal_of_gradients(name: str):
    op = getattr(torch.ops.prime_lowbit, name).default

    def kernel(*args, **kwargs):
        reverse = torch.is_grad_enabled()
        forward = forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()
        if reverse or forward:
            for t in (*args, *kwargs.values()):
                if isinstance(t, torch.Tensor) and ((reverse and t.requires_grad) or (forward and forward_ad.unpack_dual(t).tangent is not None)):
                    _no_gradient(name)
        with torch._C._AutoDispatchBelowAutograd():
            return op(*args, **kwargs)

    return kernel


for _name in ("rms_norm_quantize", "add_rms_norm_quantize", "rms_norm_quantize_backward", "quantize_4bit", "dequantize_4bit", "matvec_4bit"):
    _LIB.impl(_name, _refusal_of_gradients(_name), "Autograd")


# shape-only implementations so the ops can be traced: the same checks, no kernel
@torch.library.register_fake("prime_lowbit::rms_norm_quantize")
def _(x, weight, eps=1e-6, dtype=torch.int8):
    _check_norm_call("rms_norm_quantize", x, None, weight, eps, dtype)
    lead = x.shape[:-1]
    return x.new_empty(x.shape, dtype=dtype), x.new_empty(lead, dtype=torch.float32), x.new_empty(lead, dtype=torch.float32)


@torch.library.register_fake("prime_lowbit::add_rms_norm_quantize")
def _(x, residual, weight, eps=1e-6, dtype=torch.int8):
    _check_norm_call("add_rms_norm_quantize", x, residual, weight, eps, dtype)
    lead = x.shape[:-1]
    return (x.new_empty(x.shape, dtype=dtype), x.new_empty(lead, dtype=torch.float32), x.new_empty(x.shape),
            x.new_empty(lead, dtype=torch.float32))


@torch.library.register_fake("prime_lowbit::rms_norm_quantize_backward")
def _(grad, hidden, weight, inv_rms, grad_hidden=None):
    _check_backward_call("rms_norm_quantize_backward", grad, hidden, weight, inv_rms, grad_hidden)
    return hidden.new_empty(hidden.shape), weight.new_empty(weight.shape)


@torch.library.register_fake("prime_lowbit::quantize_4bit")
def _(weight, group_size=128, scale_dtype=torch.bfloat16):
    n, _, groups = _check_quantize("quantize_4bit", weight, group_size, scale_dtype)
    return weight.new_empty((n, groups * group_size // 2), dtype=torch.uint8), weight.new_empty((n, groups), dtype=scale_dtype)


@torch.library.register_fake("prime_lowbit::dequantize_4bit")
def _(packed, scales, columns=None, dtype=torch.float32):
    n, k, _ = _check_dequantize("dequantize_4bit", packed, scales, columns, dtype)
    return packed.new_empty((n, k), dtype=dtype)


@torch.library.register_fake("prime_lowbit::matvec_4bit")
def _(x, packed, scales, x_scales=None, dtype=None):
    n, _, _, dtype = _check_matvec("matvec_4bit", x, packed, scales, x_scales, dtype)
    return x.new_empty(x.shape[:-1] + (n,), dtype=dtype)


def _eager() -> bool:
    """No compiler, tracer, dispatch mode, ``torch.func`` transform or forward-mode level that would have to see the op."""
    return not (_compiling() or _dispatch_modes() or _transform() is not None or forward_ad._current_level >= 0 or _tracing_state() is not None)


def _plain(first: torch.Tensor, *others: Optional[torch.Tensor]) -> bool:
    """An eager call on tensors whose memory holds their values."""
    if not (_eager() and first.is_cuda and type(first) in _PLAIN and not first.is_neg()):
        return False
    for t in others:
        if t is not None and (type(t) not in _PLAIN or t.is_neg()):
            return False
    return True


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, dtype: torch.dtype = torch.int8):
    """RMS norm of the rows of ``x`` ([..., dim], Float, BFloat16 or Half) times ``weight`` ([dim], Float or the rows' type)
    as 8-bit codes: (codes like ``x`` in ``dtype``, int8 or e4m3; scales and inv_rms, Float, one a row), with
    ``codes * scales`` standing for ``x * inv_rms * weight`` and inv_rms = 1 / sqrt(mean(x^2) + eps).

    The scale is the largest of a row over 127 (448), and a code the nearest number of its type, ties to
    even, exactly.  A row that holds a value that is not finite gets scale NaN and codes 0."""
    if _plain(x, weight):
        return _rms_norm_quantize(x, weight, eps, dtype)
    return torch.ops.prime_lowbit.rms_norm_quantize(x, weight, eps, dtype)


def add_rms_norm_quantize(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, dtype: torch.dtype = torch.int8):
    """``rms_norm_quantize`` of ``hidden = x + residual`` (one type and shape; the sum is rounded to that type before it is
    normalised): (codes, scales, hidden, inv_rms)."""
    if _plain(x, residual, weight):
        return _add_rms_norm_quantize(x, residual, weight, eps, dtype)
    return torch.ops.prime_lowbit.add_rms_norm_quantize(x, residual, weight, eps, dtype)


def rms_norm_quantize_backward(grad: torch.Tensor, hidden: torch.Tensor, weight: torch.Tensor, inv_rms: torch.Tensor,
                               grad_hidden: Optional[torch.Tensor] = None):
    """Gradients of the norm, straight through the rounding to codes: (grad_x, grad_weight) from ``grad``, that of
    ``codes * scales``, and ``grad_hidden``, that of the stored sum (optional).  ``hidden`` is what the forward pass returned
    (its ``x`` without a residual); grad_x is the gradient of ``x`` and of the residual alike."""
    if _plain(hidden, grad, weight, inv_rms, grad_hidden):
        return _rms_norm_quantize_backward(grad, hidden, weight, inv_rms, grad_hidden)
    return torch.ops.prime_lowbit.rms_norm_quantize_backward(grad, hidden, weight, inv_rms, grad_hidden)


def quantize_4bit(weight: torch.Tensor, group_size: int = 128, scale_dtype: torch.dtype = torch.bfloat16):
    """A matrix [n, k] (Float, BFloat16 or Half) as 4-bit codes with a scale per ``group_size`` (32, 64 or 128) consecutive
    weights of a row: (packed, Byte [n, ceil(k / group_size) * group_size / 2], the even element in the lower half,
    two's complement; scales, ``scale_dtype`` [n, ceil(k / group_size)]).  The scale is the group's largest magnitude over
    7; codes lie within -7 .. 7 and are the nearest integers, ties to even, exactly.  A group that holds a value
    that is not finite gets scale NaN and codes 0."""
    if _plain(weight):
        return _quantize_4bit(weight, group_size, scale_dtype)
    return torch.ops.prime_lowbit.quantize_4bit(weight, group_size, scale_dtype)


def dequantize_4bit(packed: torch.Tensor, scales: torch.Tensor, columns: Optional[int] = None, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The matrix [n, columns] that 4-bit codes stand for: ``code * scale`` in 32 bits, rounded to ``dtype``.  ``columns``: the
    row length before it was filled up to whole groups (default: all that the codes hold)."""
    if _plain(packed, scales):
        return _dequantize_4bit(packed, scales, columns, dtype)
    return torch.ops.prime_lowbit.dequantize_4bit(packed, scales, columns, dtype)


def matvec_4bit(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, x_scales: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ dequantize_4bit(packed, scales, k).T`` for ``x`` [..., k], without the matrix: [..., n].  ``x`` is Float, BFloat16 or
    Half, or int8 codes with ``x_scales`` (Float, one a row), as ``rms_norm_quantize`` gives them (sums within a group exact).
    ``dtype``: of the products, rounded once; default the rows' type, Float for int8 rows.

    Floating rows are summed in 32 bits, of exact products with the codes, in an order that depends on the number of rows (so the last
    bits of a row's products can too); of Float columns what lies below 2^-133 is dropped.  A row that holds a value that is not
    finite has no finite products (other rows are not touched), and magnitudes beyond 2^120 may overflow before their group's scale is
    applied.  At most 2^26 outputs; rows of ``packed`` and ``scales`` may be slices of a larger matrix,
    less than 4 GiB apart.  Meant for the rows of a decoding step; for hundreds of rows take ``dequantize_4bit`` and a library
    product."""
    if _plain(x, packed, scales, x_scales):
        return _matvec_4bit(x, packed, scales, x_scales, dtype)
    return torch.ops.prime_lowbit.matvec_4bit(x, packed, scales, x_scales, dtype)
