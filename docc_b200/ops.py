"""Array-level host API over the C ABI.

Each function accepts either numpy arrays (host memory: the call stages the data
through the device, docc's "WithTransfers" flavour) or torch CUDA tensors (device
pointers, asynchronous on the library's current stream). Mixed inputs are an error.
Outputs have the kind of the inputs. All calls are forward: outputs carry no gradient.

Stream ordering of device calls: the library's current stream is, by default, a private
non-blocking stream of the calling thread that is NOT ordered after torch's streams. Code that
mixes torch operations and these calls on the same tensors must either route the library to
torch's stream first (``set_stream(torch.cuda.current_stream().cuda_stream)``, which the front
ends in ``docc_b200.torch`` / ``docc_b200.python`` do on every call) or synchronise around the
calls (``torch.cuda.synchronize()`` before, ``sync()`` after).
"""
from __future__ import annotations

import ctypes
import math
import warnings

import numpy as np

from . import _lib
from ._lib import BlockParams, call

ROW_MAJOR, COL_MAJOR = 101, 102
NO_TRANS, TRANS = 111, 112
FLAG_HOST_PTRS, FLAG_FP32_EXACT = 1, 2
ACT_NONE, ACT_GELU_ERF, ACT_RELU, ACT_TANH, ACT_SIGMOID, ACT_EXP, ACT_ERF, ACT_SQRT, ACT_ABS = range(9)
EW_ADD, EW_SUB, EW_MUL, EW_DIV, EW_MAX, EW_MIN = range(6)
RED_SUM, RED_MAX, RED_MIN, RED_MEAN, RED_STD = range(5)

_i64 = ctypes.c_int64
_vp = ctypes.c_void_p


class DeviceArray:
    """A C-order array in device memory obtained from ``docc_b200_malloc`` (the runtime's pool).

    This is what a container of an offloaded SDFG is between its H2D and D2H transfer nodes: the
    front ends keep intermediates in DeviceArrays so that consecutive library nodes exchange no
    data with the host. Freed through ``docc_b200_free`` when the last reference goes away."""

    is_cuda = True

    def __init__(self, shape, dtype):
        self.shape = tuple(int(v) for v in shape)
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape, dtype=np.int64)) * self.dtype.itemsize if self.shape else self.dtype.itemsize
        ptr = _vp()
        call("docc_b200_malloc", ctypes.byref(ptr), max(self.nbytes, 1))
        self._ptr = ptr.value
        self._owner = None

    @property
    def ndim(self):
        return len(self.shape)

    def data_ptr(self):
        return self._ptr

    def is_contiguous(self):
        return True

    @classmethod
    def from_numpy(cls, a):
        a = np.ascontiguousarray(a)
        out = cls(a.shape, a.dtype)
        if a.nbytes:
            call("docc_b200_h2d", _vp(out._ptr), _vp(a.ctypes.data), a.nbytes)
        return out

    def to_numpy(self):
        out = np.empty(self.shape, dtype=self.dtype)
        if out.nbytes:
            call("docc_b200_d2h", _vp(out.ctypes.data), _vp(self._ptr), out.nbytes)
        return out

    def reshape(self, *shape):
        shape = shape[0] if len(shape) == 1 and isinstance(shape[0], (tuple, list)) else shape
        shape = list(shape)
        n = int(np.prod(self.shape, dtype=np.int64)) if self.shape else 1
        if -1 in shape:
            known = int(np.prod([v for v in shape if v != -1], dtype=np.int64)) if len(shape) > 1 else 1
            shape[shape.index(-1)] = n // max(known, 1)
        if int(np.prod(shape, dtype=np.int64)) != n:
            raise ValueError("reshape changes the number of elements")
        view = object.__new__(DeviceArray)
        view.shape, view.dtype, view.nbytes, view._ptr = tuple(shape), self.dtype, self.nbytes, self._ptr
        view._owner = self._owner or self  # keeps the allocation alive
        return view

    def __del__(self):
        if getattr(self, "_owner", None) is None and getattr(self, "_ptr", None):
            try:
                _lib.lib().docc_b200_free(_vp(self._ptr))
            except Exception:
                pass
            self._ptr = None


_torch_types = {}  # type -> whether torch defines it


def _is_torch(x) -> bool:
    kind = type(x)
    known = _torch_types.get(kind)
    if known is None:
        known = _torch_types[kind] = kind.__module__.startswith("torch")
    return known


_type_names = {}  # dtype of either library -> its name


def _type_name(dtype) -> str:
    name = _type_names.get(dtype)
    if name is None:
        name = _type_names[dtype] = str(dtype)[6:] if str(dtype).startswith("torch.") else np.dtype(dtype).name
    return name


_PRECISIONS = {"float64": ord("d"), "float32": ord("s"), "float16": ord("h"), "bfloat16": ord("b")}


def _prec(x) -> int:
    name = _type_name(x.dtype)
    try:
        return _PRECISIONS[name]
    except KeyError:
        raise TypeError(f"unsupported element type {name}") from None


def _ptr(x):
    if x is None:
        return _vp(0)
    if _is_torch(x) or isinstance(x, DeviceArray):
        return _vp(x.data_ptr())
    return _vp(x.ctypes.data)


def _arr(seq):
    seq = [int(v) for v in seq]
    return (_i64 * max(len(seq), 1))(*seq)


def _kind(*xs):
    """Returns (flags, empty_like factory) after checking all arrays live on the same side."""
    xs = [x for x in xs if x is not None]
    torch_side = [_is_torch(x) or isinstance(x, DeviceArray) for x in xs]
    if any(torch_side) and not all(torch_side):
        raise TypeError("mix of host arrays and device tensors")
    if all(torch_side):
        for x in xs:
            if not x.is_cuda:
                raise TypeError("torch tensors must live on a CUDA device (pass numpy arrays for host data)")
            if not x.is_contiguous():
                raise ValueError("tensors must be contiguous")
        return 0
    for x in xs:
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError("arrays must be C-contiguous")
    return FLAG_HOST_PTRS


def _empty(like, shape, dtype=None):
    if isinstance(like, DeviceArray):
        return DeviceArray(shape, dtype or like.dtype)
    if _is_torch(like):
        import torch

        return torch.empty(tuple(shape), dtype=dtype or like.dtype, device=like.device)
    return np.empty(tuple(shape), dtype=dtype or like.dtype)


def _scalar(prec, value):
    return ctypes.c_double(value) if prec == ord("d") else ctypes.c_float(value)


def init(device: int = 0) -> None:
    call("docc_b200_init", int(device))


def sync() -> None:
    call("docc_b200_sync")


def set_stream(stream_handle) -> None:
    """Route launches of the calling thread to ``stream_handle`` (a cudaStream_t value, e.g.
    ``torch.cuda.current_stream().cuda_stream``). ``None`` restores the library's own stream; the
    value 0 names the legacy default stream and is passed on as CUDA's ``cudaStreamLegacy`` handle."""
    if stream_handle is None:
        call("docc_b200_set_stream", _vp(0))
    else:
        call("docc_b200_set_stream", _vp(int(stream_handle) or 1))


def launch_count(reset: bool = False) -> int:
    return int(_lib.lib().docc_b200_launch_count(1 if reset else 0))


def gemm(A, B, C=None, alpha=1.0, beta=0.0, transa=False, transb=False, layout=ROW_MAJOR, flags=0):
    """C = alpha*op(A)*op(B) + beta*C (GEMMNode). 2-D arrays; for COL_MAJOR the arrays hold the
    matrices transposed, as a Fortran caller would see them."""
    flags |= _kind(A, B, C)
    prec = _prec(A)
    if layout == ROW_MAJOR:
        m, k = (A.shape[1], A.shape[0]) if transa else A.shape
        n = B.shape[0] if transb else B.shape[1]
        c_shape = (m, n)
    else:
        k, m = (A.shape[1], A.shape[0]) if transa else A.shape
        n = B.shape[1] if transb else B.shape[0]
        c_shape = (n, m)
    if C is None:
        C = _empty(A, c_shape)
        beta = 0.0
    al, be = _scalar(prec, alpha), _scalar(prec, beta)
    call("docc_b200_gemm", prec, layout, TRANS if transa else NO_TRANS, TRANS if transb else NO_TRANS, m, n, k,
         ctypes.cast(ctypes.pointer(al), _vp), _ptr(A), A.shape[-1], _ptr(B), B.shape[-1],
         ctypes.cast(ctypes.pointer(be), _vp), _ptr(C), C.shape[-1], flags)
    return C


def gemm_strided(precision, layout, transa, transb, m, n, k, alpha, A, lda, B, ldb, beta, C, ldc, flags=0):
    """GEMM on flat buffers with explicit leading dimensions, the form docc's generated code passes to BLAS
    (gemm_node.cpp:441-520): ``C`` is updated in place. ``precision`` is one of 'h', 's', 'd', 'b'."""
    flags |= _kind(A, B, C)
    prec = ord(precision)
    if prec != _prec(A) or prec != _prec(B) or prec != _prec(C):
        raise TypeError(f"gemm_strided: operands are not all of precision {precision!r}")
    al, be = _scalar(prec, float(alpha)), _scalar(prec, float(beta))
    call("docc_b200_gemm", prec, int(layout), TRANS if transa else NO_TRANS, TRANS if transb else NO_TRANS, int(m), int(n), int(k),
         ctypes.cast(ctypes.pointer(al), _vp), _ptr(A), int(lda), _ptr(B), int(ldb),
         ctypes.cast(ctypes.pointer(be), _vp), _ptr(C), int(ldc), flags)
    return C


def matmul(A, B, flags=0):
    """Batched row-major matmul with numpy broadcasting rules on the batch dims (MatMulNode)."""
    flags |= _kind(A, B)
    m, k = A.shape[-2:]
    n = B.shape[-1]
    batch_shape = tuple(np.broadcast_shapes(tuple(A.shape[:-2]), tuple(B.shape[:-2])))
    batch = int(np.prod(batch_shape)) if batch_shape else 1
    sa = 0 if A.ndim == 2 else m * k
    sb = 0 if B.ndim == 2 else k * n
    if A.ndim > 2 and tuple(A.shape[:-2]) != batch_shape or B.ndim > 2 and tuple(B.shape[:-2]) != batch_shape:
        raise ValueError("batch dims must match exactly or the operand must be 2-D")
    Y = _empty(A, batch_shape + (m, n))
    call("docc_b200_matmul", _prec(A), batch, m, n, k, _ptr(A), k, sa, _ptr(B), n, sb, _ptr(Y), n, m * n, flags)
    return Y


def linear(X, W, bias=None, act=ACT_NONE, residual=None, alpha=1.0, flags=0):
    """Y = act(alpha * X W^T + bias) + residual with the torch Linear weight layout [out, in]."""
    flags |= _kind(X, W, bias, residual)
    if bias is not None:
        # the ABI reads the bias as fp32 for 16-bit operands and in the operand type otherwise
        want = ord("s") if _prec(X) in (ord("h"), ord("b")) else _prec(X)
        if _prec(bias) != want:
            raise TypeError(f"linear: bias must be {'float32' if want == ord('s') else 'float64'} for {chr(_prec(X))!r} operands")
    k = X.shape[-1]
    m = int(np.prod(X.shape[:-1]))
    n = W.shape[0]
    # the ABI sees pointers and leading dimensions only: extents and types are checked here
    if W.ndim != 2 or W.shape[1] != k or _prec(W) != _prec(X):
        raise ValueError(f"linear: weight {tuple(W.shape)} does not match inputs of width {k} and type {chr(_prec(X))!r}")
    if bias is not None and int(np.prod(bias.shape)) != n:
        raise ValueError(f"linear: bias has {int(np.prod(bias.shape))} elements for {n} output features")
    if residual is not None and (tuple(residual.shape) != tuple(X.shape[:-1]) + (n,) or _prec(residual) != _prec(X)):
        raise ValueError("linear: the residual must have the shape and type of the output (broadcast it first)")
    Y = _empty(X, tuple(X.shape[:-1]) + (n,))
    call("docc_b200_gemm_epilogue", _prec(X), TRANS, m, n, k, float(alpha), _ptr(X), k, _ptr(W), k, _ptr(bias), int(act),
         _ptr(residual), n, _ptr(Y), n, flags)
    return Y


def softmax(X, axes=None, flags=0):
    flags |= _kind(X)
    if axes is None:
        axes = list(range(X.ndim))
    if np.isscalar(axes):
        axes = [axes]
    Y = _empty(X, X.shape)
    call("docc_b200_softmax", _prec(X), X.ndim, _arr(X.shape), len(axes), _arr(axes), _ptr(X), _ptr(Y), flags)
    return Y


def reduce(op, X, axes, flags=0):
    flags |= _kind(X)
    if np.isscalar(axes):
        axes = [axes]
    norm = sorted(a % X.ndim for a in axes)
    out_shape = tuple(s for d, s in enumerate(X.shape) if d not in norm)
    Y = _empty(X, out_shape)
    call("docc_b200_reduce", int(op), _prec(X), X.ndim, _arr(X.shape), len(axes), _arr(axes), _ptr(X), _ptr(Y), flags)
    return Y


def conv_out_shape(x_shape, k_shape, strides, pads, dilations, c_out):
    sr = len(k_shape)
    out = [x_shape[0], c_out]
    for i in range(sr):
        num = x_shape[2 + i] + pads[i] + pads[sr + i] - dilations[i] * (k_shape[i] - 1) - 1
        out.append(0 if num < 0 else num // strides[i] + 1)
    return tuple(out)


def conv(X, W, bias=None, strides=None, pads=None, dilations=None, group=1, out_dtype=None, flags=0):
    """N-D cross-correlation in NC(D..) layout (ConvNode). ``pads`` = [begin..., end...]."""
    flags |= _kind(X, W, bias)
    sr = X.ndim - 2
    strides = list(strides or [1] * sr)
    pads = list(pads or [0] * (2 * sr))
    dilations = list(dilations or [1] * sr)
    k_shape = tuple(W.shape[2:])
    c_out = W.shape[0]
    prec_in = _prec(X)
    if out_dtype is None:
        prec_out = ord("s") if prec_in in (ord("b"), ord("h")) else prec_in
    else:
        prec_out = _prec(np.empty(0, dtype=out_dtype)) if not _is_torch(X) else _prec(_empty(X, (0,), out_dtype))
    if _is_torch(X):
        import torch

        odt = {ord("s"): torch.float32, ord("d"): torch.float64, ord("b"): torch.bfloat16, ord("h"): torch.float16}[prec_out]
    else:
        odt = {ord("s"): np.float32, ord("d"): np.float64, ord("h"): np.float16}.get(prec_out, X.dtype)
    Y = _empty(X, conv_out_shape(tuple(X.shape), k_shape, strides, pads, dilations, c_out), odt)
    call("docc_b200_conv", prec_in, prec_out, sr, _arr(X.shape), _arr(k_shape), _arr(strides), _arr(pads), _arr(dilations),
         c_out, int(group), _ptr(X), _ptr(W), _ptr(bias), _ptr(Y), flags)
    return Y


def attention(Q, K, V, scale=None, causal=False, flags=0):
    """softmax(scale * Q K^T [+ causal mask]) V on contiguous [B,H,S,D] arrays."""
    flags |= _kind(Q, K, V)
    B, H, Sq, D = Q.shape
    Skv = K.shape[2]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    O = _empty(Q, Q.shape)
    null = ctypes.cast(None, ctypes.POINTER(_i64))
    call("docc_b200_attention", _prec(Q), B, H, Sq, Skv, D, float(scale), int(bool(causal)), _ptr(Q), null, _ptr(K), null,
         _ptr(V), null, _ptr(O), null, flags)
    return O


def layernorm(X, gamma=None, beta=None, eps=1e-5, flags=0):
    flags |= _kind(X, gamma, beta)
    cols = X.shape[-1]
    rows = int(np.prod(X.shape[:-1]))
    Y = _empty(X, X.shape)
    call("docc_b200_layernorm", _prec(X), rows, cols, _ptr(X), _ptr(gamma), _ptr(beta), float(eps), _ptr(Y), flags)
    return Y


# ---- the decoder step: RMS norm, rotary positions and the paged cache, attention over it, log-probabilities -----------------------
# These calls are short on the device, so that what the host does around them is most of a step: the helpers ask a tensor for as
# little as the checks need.
_Pairs, _Triples = _i64 * 2, _i64 * 3
_torch = None  # the module, once one of its tensors has been met (an import statement costs as much as several of the checks)


def _torch_module():
    global _torch
    if _torch is None:
        import torch

        _torch = torch
    return _torch


def _addr(x):
    """The address of an array of either side, or None."""
    if x is None:
        return None
    try:
        return x.data_ptr()
    except AttributeError:
        return x.ctypes.data


_NATIVE = ("docc_b200_rmsnorm", "docc_b200_rmsnorm_q8", "docc_b200_rope", "docc_b200_rope_append", "docc_b200_paged_attention",
           "docc_b200_token_logprobs")
_native = None  # the compiled form of these calls for torch tensors (docc_b200/host): None until the first of them, False if there is none


def _compiled(x):
    """The module that takes the ordinary call on torch tensors; it answers None to every other, which then runs here. False before the
    first torch tensor has been met, and where the module has not been built for this torch and interpreter."""
    global _native
    if _native is None:
        if not _is_torch(x):
            return False
        from importlib.machinery import ExtensionFileLoader
        from importlib.util import module_from_spec, spec_from_loader

        from .build import HOST_NAME, host_path

        path = host_path()
        if path is None:  # a tensor type of another package
            return False
        try:
            loader = ExtensionFileLoader(HOST_NAME, path)
            module = module_from_spec(spec_from_loader(loader.name, loader))
            loader.exec_module(module)
        except ImportError as e:
            warnings.warn(f"{path} cannot be loaded ({e}): these calls take their Python path, which is 4-13 us slower. "
                          "Run `python -m docc_b200.build`.", RuntimeWarning, stacklevel=3)
            _native = False
            return False
        module.bind(*(ctypes.cast(getattr(_lib.lib(), name), _vp).value for name in _NATIVE), _lib.check)
        _native = module
    return _native


def _side(*xs):
    """``_kind`` without its demand for contiguity, for entries that take strides: flags, after checking that all arrays live on the
    same side and, for torch tensors, on the device that the calling thread's launches go to."""
    host = device = False
    current = None
    for x in xs:
        if x is None:
            continue
        if _is_torch(x):
            at = x.get_device()
            if at != current:
                if at < 0:
                    raise TypeError("torch tensors must live on a CUDA device (pass numpy arrays for host data)")
                if current is None:
                    current = (_torch or _torch_module()).cuda.current_device()
                if at != current:
                    raise ValueError(f"tensor on cuda:{at} while the calling thread's device is cuda:{current}")
            device = True
        elif isinstance(x, DeviceArray):
            device = True
        else:
            if not x.flags["C_CONTIGUOUS"]:
                raise ValueError("arrays must be C-contiguous")
            host = True
    if host and device:
        raise TypeError("mix of host arrays and device tensors")
    return FLAG_HOST_PTRS if host else 0


def _new_like(x):
    """An uninitialised contiguous array of x's kind, shape and element type."""
    if _is_torch(x) and x.is_contiguous():
        return (_torch or _torch_module()).empty_like(x)
    return _new(x, x.shape)


def _new(x, shape, name=None):
    """An uninitialised contiguous array of x's kind, of element type ``name`` (None: x's own)."""
    if _is_torch(x):
        if name is None:
            return x.new_empty(shape)
        return x.new_empty(shape, dtype=_like(x, name))
    return _empty(x, shape, None if name is None else np.dtype(name))


def _heads_strides(x, name, written=False):
    """The strides array of a tensor whose last dimension is contiguous, or NULL if all of it is. One that is written may not be
    a broadcast view, whose elements share memory."""
    if not _is_torch(x) or x.is_contiguous():
        return None
    s, shape = x.stride(), x.shape
    if s[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    if written and 0 in s:
        for d, v in enumerate(s):
            if v == 0 and shape[d] > 1:
                raise ValueError(f"{name}: a broadcast view cannot be written")
    return _Pairs(s[0], s[1]) if len(s) == 3 else _Triples(s[0], s[1], s[2])


def _rows_of(x, name):
    """(rows, cols, row stride) of a tensor seen as rows over its last dimension; the leading dimensions must be one strided run."""
    shape = x.shape
    cols, rows = shape[-1], 1
    for s in shape[:-1]:
        rows *= s
    if not _is_torch(x) or x.is_contiguous():
        return rows, cols, cols
    s, run, step = x.stride(), None, None
    for d in range(x.ndim - 2, -1, -1):
        if shape[d] == 1:
            continue
        if run is None:
            run = step = s[d]
        if s[d] != step:
            raise ValueError(f"{name}: the leading dimensions are not one run of rows")
        step *= shape[d]
    if (s[-1] != 1 and cols > 1) or (run is not None and run < cols):
        raise ValueError(f"{name}: rows must be contiguous and must not overlap")
    return rows, cols, cols if run is None else run


def _want(x, dtype, name, shape=None):
    if _type_name(x.dtype) != dtype:
        raise TypeError(f"{name} must be {dtype}, not {_type_name(x.dtype)}")
    if shape is not None and x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(x.shape)}")
    if _is_torch(x) and not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


_torch_dtypes = {}


def _like(x, name):
    """The element type ``name`` in the library ``x`` comes from."""
    if _is_torch(x):
        got = _torch_dtypes.get(name)
        if got is None:
            got = _torch_dtypes[name] = getattr(_torch_module(), name)
        return got
    return np.dtype(name)


def _rms_inputs(X, gamma, residual, flags):
    flags |= _side(X, gamma, residual)
    if X.ndim == 0:
        raise ValueError("rmsnorm: a scalar has no rows")
    rows, cols, ldx = _rows_of(X, "rmsnorm")
    ldr = 0
    if gamma is not None:
        _want(gamma, "float32", "rmsnorm: gamma", (cols,))
    if residual is not None:
        if residual.shape != X.shape or residual.dtype != X.dtype:
            raise ValueError("rmsnorm: the residual must have the shape and type of the input")
        ldr = _rows_of(residual, "rmsnorm: residual")[2]
    return rows, cols, ldx, ldr, flags


def rmsnorm(X, gamma=None, residual=None, eps=1e-6, flags=0):
    """``Y = s / sqrt(mean(s^2) + eps) * gamma`` over the last dimension, ``s = X + residual``. Returns Y, or with a residual
    ``(Y, S)``: S is s in the input's type, the residual of what follows. ``gamma`` is float32."""
    native = _native or _compiled(X)
    if native and not flags:
        got = native.rmsnorm(X, gamma, residual, eps)
        if got is not None:
            return got
    rows, cols, ldx, ldr, flags = _rms_inputs(X, gamma, residual, flags)
    Y = _new_like(X)
    S = _new_like(X) if residual is not None else None
    call("docc_b200_rmsnorm", _prec(X), rows, cols, _addr(X), ldx, _addr(residual), ldr, _addr(gamma), eps, _addr(S), _addr(Y), flags)
    return Y if residual is None else (Y, S)


def rmsnorm_quant(X, gamma=None, residual=None, eps=1e-6, group=0, flags=0):
    """The norm of ``rmsnorm`` with an 8-bit output: ``(Q, scales)``, or ``(Q, scales, S)`` with a residual. Q holds e4m3 values
    (``torch.float8_e4m3fn``; their codes as uint8 for other arrays) and ``Q * scales`` stands for the norm, with one float32 scale
    per ``group`` of 128 columns or, with group 0, per row: scales have shape ``X.shape[:-1] + (groups,)``."""
    native = _native or _compiled(X)
    if native and not flags:
        got = native.rmsnorm_quant(X, gamma, residual, eps, group)
        if got is not None:
            return got
    rows, cols, ldx, ldr, flags = _rms_inputs(X, gamma, residual, flags)
    if group not in (0, 128):
        raise ValueError("rmsnorm_quant: group must be 0 (whole rows) or 128")
    Q = _new(X, X.shape, "float8_e4m3fn" if _is_torch(X) else "uint8")
    scales = _new(X, tuple(X.shape[:-1]) + (1 if group == 0 else -(-cols // group),), "float32")
    S = _new_like(X) if residual is not None else None
    call("docc_b200_rmsnorm_q8", _prec(X), rows, cols, _addr(X), ldx, _addr(residual), ldr, _addr(gamma), eps, group, _addr(S), _addr(Q),
         _addr(scales), flags)
    return (Q, scales) if residual is None else (Q, scales, S)


def rope_frequencies(rotary_dim, base=10000.0, scaling="none", factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0):
    """``(inv_freq, mscale)`` for ``rope``: radians per position of each pair as a float64 numpy array (``base ** (-2i / rotary_dim)``,
    to be moved to the device once), and the factor of cosine and sine. ``scaling`` stretches a context trained at
    ``original_length`` by ``factor``: ``"linear"`` divides every frequency; ``"ntk"`` raises the base so that the slowest pair is
    divided by ``factor`` and the fastest kept; ``"yarn"`` divides the pairs that turn less than ``beta_slow`` times within
    ``original_length``, keeps those that turn more than ``beta_fast`` times, blends between, and sets
    ``mscale = 0.1 ln(factor) + 1``."""
    rotary_dim = int(rotary_dim)
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rope_frequencies: rotary_dim must be even")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("rope_frequencies: base must be above 1 and factor at least 1")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    freq = float(base) ** (-2.0 * i / max(rotary_dim, 1))
    if scaling == "none":
        return freq, 1.0
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "ntk":
        if rotary_dim <= 2:
            raise ValueError("rope_frequencies: 'ntk' needs more than one pair")
        return (base * factor ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim), 1.0
    if scaling != "yarn":
        raise ValueError(f"rope_frequencies: unknown scaling {scaling!r}")
    if original_length is None or not beta_fast > beta_slow:
        raise ValueError("rope_frequencies: 'yarn' needs original_length, and beta_fast above beta_slow")
    pair_of = lambda turns: rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
    stretched = np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    return freq / factor * stretched + freq * (1.0 - stretched), 0.1 * math.log(factor) + 1.0


def _rope_inputs(x, positions, inv_freq, name):
    _want(positions, "int64", f"{name}: positions", (x.shape[0],))
    _want(inv_freq, "float64", f"{name}: inv_freq")
    if inv_freq.ndim != 1 or 2 * inv_freq.shape[0] > x.shape[2]:
        raise ValueError(f"{name}: inv_freq must hold one frequency per pair, at most D / 2")


def _out_like(x, out, name):
    if out is None:
        return _new_like(x)
    if out.shape != x.shape or out.dtype != x.dtype:
        raise ValueError(f"{name}: out must have the shape and type of the query")
    return out


def rope(X, positions, inv_freq, interleaved=False, mscale=1.0, inverse=False, out=None, flags=0):
    """Rotary positions on X [tokens, heads, D] (``docc_b200_rope``): ``positions`` int64 [tokens], ``inv_freq`` float64
    [rotary_dim / 2] on the side of X (``rope_frequencies``). ``inverse`` applies the transpose, which is the gradient. ``out`` may be
    X itself."""
    native = _native or _compiled(X)
    if native and not flags:
        got = native.rope(X, positions, inv_freq, interleaved, mscale, inverse, out)
        if got is not None:
            return got
    flags |= _side(X, positions, inv_freq, out)
    if X.ndim != 3:
        raise ValueError("rope: X must be [tokens, heads, D]")
    T, H, D = X.shape
    _rope_inputs(X, positions, inv_freq, "rope")
    out = _out_like(X, out, "rope")
    call("docc_b200_rope", _prec(X), T, H, D, 2 * inv_freq.shape[0], 1 if interleaved else 0, 1 if inverse else 0, _addr(X),
         _heads_strides(X, "rope: X"), _addr(positions), _addr(inv_freq), mscale, _addr(out), _heads_strides(out, "rope: out", True), flags)
    return out


def _cache(q, k_cache, v_cache, Hkv, D, name):
    """(pages, page_size, strides of K, strides of V) of a cache [pages, Hkv, page_size, D] (views of other layouts included)."""
    shape = k_cache.shape
    if v_cache.shape != shape:
        raise ValueError(f"{name}: the two caches differ in shape")
    if len(shape) != 4 or shape[1] != Hkv or shape[3] != D or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{name}: caches must be [pages, {Hkv}, page_size, {D}] of the type of the query")
    return shape[0], shape[2], _heads_strides(k_cache, f"{name}: k_cache", True), _heads_strides(v_cache, f"{name}: v_cache", True)


def rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved=False, mscale=1.0, out=None, flags=0):
    """Rotates q [tokens, Hq, D] and k [tokens, Hkv, D] and writes the rotated k and v into the paged cache
    [pages, Hkv, page_size, D] at ``slots`` (int64 [tokens]: page * page_size + place; negative: not written). Returns the rotated q
    (``out``, which may be q itself). Device tensors only; the slots of one call must differ."""
    native = _native or _compiled(q)
    if native and not flags:
        got = native.rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved, mscale, out)
        if got is not None:
            return got
    if _side(q, k, v, positions, inv_freq, k_cache, v_cache, slots, out):
        raise TypeError("rope_append: the cache lives on the device; host arrays are not taken")
    if q.ndim != 3 or k.ndim != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("rope_append: q must be [tokens, Hq, D], k and v [tokens, Hkv, D]")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("rope_append: q, k and v differ in type")
    _rope_inputs(q, positions, inv_freq, "rope_append")
    _want(slots, "int64", "rope_append: slots", (T,))
    pages, page_size, ks, vs = _cache(q, k_cache, v_cache, Hkv, D, "rope_append")
    out = _out_like(q, out, "rope_append")
    call("docc_b200_rope_append", _prec(q), T, Hq, Hkv, D, 2 * inv_freq.shape[0], 1 if interleaved else 0, _addr(q),
         _heads_strides(q, "rope_append: q"), _addr(k), _heads_strides(k, "rope_append: k"), _addr(v), _heads_strides(v, "rope_append: v"),
         _addr(positions), _addr(inv_freq), mscale, _addr(out), _heads_strides(out, "rope_append: out", True), _addr(k_cache), ks,
         _addr(v_cache), vs, pages, page_size, _addr(slots), flags)
    return out


_scratch_bytes = {}  # (device, query heads per key-value head, D) -> bytes: what the size of the scratch depends on


def paged_attention(q, k_cache, v_cache, page_table, lengths, scale=None, softcap=0.0, window=0, return_lse=False, out=None, flags=0):
    """Attention of one new token per sequence, q [B, Hq, D], over a paged cache [pages, Hkv, page_size, D]; the cache must already
    hold the new token (``rope_append``). ``page_table`` int32 [B, max_pages], ``lengths`` int32 [B]: token j of sequence b is at place
    ``j % page_size`` of page ``page_table[b, j // page_size]``. ``window`` > 0 keeps the last ``window`` tokens, ``softcap`` > 0 caps
    the scores (``docc_b200_paged_attention``). Returns the output [B, Hq, D], with ``return_lse`` also the float32 [B, Hq]
    logarithm of the softmax's denominator. Sequences of length 0 give zeros and -inf. Device tensors only.

    While torch captures a graph the scratch comes from torch's allocator, so that the graph owns what it replays with; otherwise it
    is the library's, ordered on the calling thread's stream."""
    native = _native or _compiled(q)
    if native and not flags:
        got = native.paged_attention(q, k_cache, v_cache, page_table, lengths, scale, softcap, window, return_lse, out)
        if got is not None:
            return got
    if _side(q, k_cache, v_cache, page_table, lengths, out):
        raise TypeError("paged_attention: the cache lives on the device; host arrays are not taken")
    if q.ndim != 3 or k_cache.ndim != 4:
        raise ValueError("paged_attention: q must be [B, Hq, D] and the caches [pages, Hkv, page_size, D]")
    B, Hq, D = q.shape
    Hkv, prec = k_cache.shape[1], _prec(q)
    pages, page_size, ks, vs = _cache(q, k_cache, v_cache, Hkv, D, "paged_attention")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"paged_attention: {Hq} query heads are not a multiple of {Hkv} key-value heads")
    _want(lengths, "int32", "paged_attention: lengths", (B,))
    if page_table.ndim != 2:
        raise ValueError("paged_attention: page_table must be [B, max_pages]")
    most = page_table.shape[1]
    _want(page_table, "int32", "paged_attention: page_table", (B, most))
    out = _out_like(q, out, "paged_attention")
    lse = _new(q, (B, Hq), "float32") if return_lse else None
    work, bytes_ = None, 0
    if _is_torch(q) and _torch_module().cuda.is_current_stream_capturing():
        key = (q.get_device(), Hq // Hkv, D)
        bytes_ = _scratch_bytes.get(key)
        if bytes_ is None:
            size = ctypes.c_size_t()
            call("docc_b200_paged_attention_workspace", prec, 1, Hq, Hkv, D, ctypes.byref(size))
            bytes_ = _scratch_bytes[key] = size.value
        work = _new(q, bytes_, "uint8")
    call("docc_b200_paged_attention", prec, B, Hq, Hkv, D, 1.0 / math.sqrt(max(D, 1)) if scale is None else scale, softcap, window,
         _addr(q), _heads_strides(q, "paged_attention: q"), _addr(k_cache), ks, _addr(v_cache), vs, pages, page_size, _addr(page_table),
         most, most, _addr(lengths), _addr(out), _heads_strides(out, "paged_attention: out", True), _addr(lse), _addr(work), bytes_, flags)
    return (out, lse) if return_lse else out


def token_logprobs(logits, ids, k=0, scale=1.0, flags=0):
    """``(logp, entropy, top_ids, top_logp)`` of logits [rows, vocab] under ``softmax(scale * logits)``: the log-probability of token
    ``ids[row]`` (int64; an id outside the vocabulary gives NaN), the distribution's entropy, and the ``k`` <= 32 most likely tokens
    with their log-probabilities (ties to the lowest index). float32, indices int64; [rows, k] for the last two."""
    native = _native or _compiled(logits)
    if native and not flags:
        got = native.token_logprobs(logits, ids, k, scale)
        if got is not None:
            return got
    flags |= _side(logits, ids)
    if logits.ndim != 2:
        raise ValueError("token_logprobs: logits must be [rows, vocab]")
    rows, vocab, ldx = _rows_of(logits, "token_logprobs")
    _want(ids, "int64", "token_logprobs: ids", (rows,))
    if _is_torch(logits):
        logp, entropy = _new(logits, (2, rows), "float32").unbind(0)
    else:
        logp, entropy = _new(logits, (rows,), "float32"), _new(logits, (rows,), "float32")
    width = k if 0 <= k <= 32 else 0  # nothing is allocated for a k that the call refuses
    top_ids, top_logp = _new(ids, (rows, width)), _new(logits, (rows, width), "float32")
    call("docc_b200_token_logprobs", _prec(logits), rows, vocab, _addr(logits), ldx, scale, _addr(ids), _addr(logp), _addr(entropy), k,
         _addr(top_ids), _addr(top_logp), flags)
    return logp, entropy, top_ids, top_logp


def bias_act(X, scale=1.0, bias=None, act=ACT_NONE, residual=None, flags=0):
    flags |= _kind(X, bias, residual)
    cols = X.shape[-1] if X.ndim else 1
    rows = int(np.prod(X.shape[:-1])) if X.ndim else 1
    Y = _empty(X, X.shape)
    call("docc_b200_bias_act", _prec(X), rows, cols, _ptr(X), float(scale), _ptr(bias), int(act), _ptr(residual), _ptr(Y), flags)
    return Y


def binary(op, A, B, flags=0):
    flags |= _kind(A, B)
    if tuple(A.shape) != tuple(B.shape):
        raise ValueError("binary: shapes differ (broadcast with numpy/torch first)")
    Y = _empty(A, A.shape)
    n = int(np.prod(A.shape)) if A.ndim else 1
    call("docc_b200_binary", int(op), _prec(A), n, _ptr(A), _ptr(B), _ptr(Y), flags)
    return Y


def cast(X, dtype, flags=0):
    flags |= _kind(X)
    Y = _empty(X, X.shape, dtype)
    n = int(np.prod(X.shape)) if X.ndim else 1
    call("docc_b200_cast", _prec(X), _prec(Y), n, _ptr(X), _ptr(Y), flags)
    return Y


BLOCK_FIELDS = ("ln1_g", "ln1_b", "w_qkv", "b_qkv", "w_o", "b_o", "ln2_g", "ln2_b", "w_1", "b_1", "w_2", "b_2")


def transformer_block(x, params, n_heads, eps=1e-5, flags=0):
    """Pre-LN encoder block; ``params`` maps the ``docc_b200_block_params`` field names to arrays."""
    tensors = [params.get(f) for f in BLOCK_FIELDS]
    flags |= _kind(x, *tensors)
    Bn, S, d = x.shape
    bp = BlockParams()
    bp.batch, bp.seq, bp.d_model, bp.n_heads, bp.d_ff, bp.eps = Bn, S, d, int(n_heads), params["w_1"].shape[0], float(eps)
    for f, t in zip(BLOCK_FIELDS, tensors):
        setattr(bp, f, _ptr(t).value or 0)
    y = _empty(x, x.shape)
    call("docc_b200_transformer_block", _prec(x), ctypes.byref(bp), _ptr(x), _ptr(y), flags)
    return y
