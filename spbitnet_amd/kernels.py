"""Python mirror of the reference's kernel host API for the sparse-ternary
path (include/spbitnet/sparse_ternary_kernels.h:16-48 and
include/spbitnet/inference_kernels.h:19-30 of the reference): same names,
same argument order and meaning, device tensors in place of raw pointers.

Each call checks on the host that every tensor is on the GPU, has the dtype
the kernel expects, is contiguous and is at least as large as the shape
arguments require, then launches through the C ABI on the given stream
(default: torch's current stream).  Failures raise SpbError; rows == 0 or
cols == 0 is a no-op, as in the reference.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib

_HALF_KIND = {torch.float16: "f16", torch.bfloat16: "bf16"}


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        # the current stream's pointer: 0.2 us, where torch.cuda.current_stream()
        # builds a Stream object in 2.8 us, a third of a small call
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()) or None
    if isinstance(stream, int):
        return stream or None
    return stream.cuda_stream or None


def _dev(t: torch.Tensor, name: str, dtype, min_numel: int) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.numel() < min_numel:
        raise ValueError(f"{name} holds {t.numel()} elements, needs at least {min_numel}")
    return t.data_ptr()


def _weights(meta, values, rows, cols, meta_row_stride, values_row_stride):
    if rows < 0 or cols < 0:
        raise ValueError(f"negative shape ({rows}, {cols})")
    if cols % 4:
        raise ValueError(f"cols={cols} is not a multiple of 4")
    if meta_row_stride < (cols // 4 + 7) // 8 or values_row_stride < (cols // 4 + 15) // 16:
        raise ValueError("row strides are smaller than the format requires")
    need_m = rows * meta_row_stride if rows and cols else 0
    need_v = rows * values_row_stride if rows and cols else 0
    pm = _dev(meta, "meta", (torch.int32, torch.uint32), need_m)
    pv = _dev(values, "values", (torch.int32, torch.uint32), need_v)
    return pm, pv


def sparse_ternary_unpack_gpu(meta, values, out, rows, cols, meta_row_stride,
                              values_row_stride, stream=None):
    """reference src/kernels/sparse_ternary.cu:240-254"""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    po = _dev(out, "out", torch.int8, rows * cols)
    _lib.check(_lib.load().spb_sparse_ternary_unpack(pm, pv, po, rows, cols, meta_row_stride,
                                                     values_row_stride, _stream_ptr(stream)),
               "sparse_ternary_unpack_gpu")


def sparse_ternary_gemv_gpu(meta, values, x, y, rows, cols, meta_row_stride,
                            values_row_stride, stream=None, resident=False):
    """reference src/kernels/sparse_ternary.cu:256-272 (int8 x -> int32 y).
    resident=True loads the weights on the default cache policy
    (spb_sparse_ternary_gemv_resident: matrices that stay in the Infinity
    Cache between calls) instead of the streaming one."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    empty = rows == 0 or cols == 0
    px = _dev(x, "x", torch.int8, 0 if empty else cols)
    py = _dev(y, "y", torch.int32, 0 if empty else rows)
    L = _lib.load()
    fn = L.spb_sparse_ternary_gemv_resident if resident else L.spb_sparse_ternary_gemv
    _lib.check(fn(pm, pv, px, py, rows, cols, meta_row_stride, values_row_stride,
                  _stream_ptr(stream)), "sparse_ternary_gemv_gpu")


def fused_sparse_bitlinear_gpu(meta, values, x, output, d_absmax, gamma, rows, cols,
                               meta_row_stride, values_row_stride, stream=None):
    """reference src/kernels/sparse_ternary.cu:274-291; x/output fp16 or bf16."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    if x.dtype not in _HALF_KIND:
        raise TypeError("x must be float16 or bfloat16")
    kind = _HALF_KIND[x.dtype]
    empty = rows == 0 or cols == 0
    px = _dev(x, "x", x.dtype, 0 if empty else cols)
    po = _dev(output, "output", x.dtype, 0 if empty else rows)
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    fn = getattr(_lib.load(), f"spb_fused_sparse_bitlinear_{kind}")
    _lib.check(fn(pm, pv, px, po, pa, float(gamma), rows, cols, meta_row_stride,
                  values_row_stride, _stream_ptr(stream)), "fused_sparse_bitlinear_gpu")


def absmax_reduce_gpu(input, d_absmax, size, stream=None):
    """reference src/kernels/inference_kernels.cu:549-553"""
    if input.dtype not in _HALF_KIND:
        raise TypeError("input must be float16 or bfloat16")
    pi = _dev(input, "input", input.dtype, size)
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    fn = getattr(_lib.load(), f"spb_absmax_reduce_{_HALF_KIND[input.dtype]}")
    _lib.check(fn(pi, pa, size, _stream_ptr(stream)), "absmax_reduce_gpu")


def absmax_quantize_gpu(input, output, d_absmax, size, stream=None):
    """reference src/kernels/inference_kernels.cu:543-547"""
    if input.dtype not in _HALF_KIND:
        raise TypeError("input must be float16 or bfloat16")
    pi = _dev(input, "input", input.dtype, size)
    po = _dev(output, "output", torch.int8, size)
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    fn = getattr(_lib.load(), f"spb_absmax_quantize_{_HALF_KIND[input.dtype]}")
    _lib.check(fn(pi, po, pa, size, _stream_ptr(stream)), "absmax_quantize_gpu")


def dequantize_gpu(input, output, d_absmax, gamma, size, stream=None):
    """reference src/kernels/inference_kernels.cu:555-561; output fp16 or bf16."""
    if output.dtype not in _HALF_KIND:
        raise TypeError("output must be float16 or bfloat16")
    pi = _dev(input, "input", torch.int32, size)
    po = _dev(output, "output", output.dtype, size)
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    fn = getattr(_lib.load(), f"spb_dequantize_{_HALF_KIND[output.dtype]}")
    _lib.check(fn(pi, po, pa, float(gamma), size, _stream_ptr(stream)), "dequantize_gpu")


# ---- batched GEMM (replaces the reference's cuSPARSELt path) ------------------

def sparse_ternary_gemm_gpu(meta, values, X, Y, rows, cols, n, meta_row_stride,
                            values_row_stride, stream=None, kernel="auto"):
    """Y[t][r] = sum_c W[r][c] X[t][c] (int32), X int8 [n][cols], Y int32 [n][rows].

    Replaces CuSparseLtGemm::execute (reference src/cusparselt_backend.cu:186-207);
    kernel="auto" uses the matrix-core kernel where the shape allows,
    kernel="addsub" the bit-plane GEMV kernel over tokens (the comparator)."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    if n < 0:
        raise ValueError("negative batch")
    empty = rows == 0 or cols == 0 or n == 0
    px = _dev(X, "X", torch.int8, 0 if empty else n * cols)
    py = _dev(Y, "Y", torch.int32, 0 if empty else n * rows)
    L = _lib.load()
    fn = L.spb_sparse_ternary_gemm if kernel == "auto" else L.spb_sparse_ternary_gemm_addsub
    _lib.check(fn(pm, pv, px, py, rows, cols, n, meta_row_stride, values_row_stride,
                  _stream_ptr(stream)), "sparse_ternary_gemm_gpu")


def gemm_kernel_id(meta, values, X, rows, cols, n, meta_row_stride, values_row_stride) -> int:
    """Kernel spb_sparse_ternary_gemm would run for these arguments: 2 the
    staged matrix-core kernel, 1 the direct matrix-core kernel, 0 the general
    kernel."""
    return _lib.load().spb_sparse_ternary_gemm_kernel_id(
        meta.data_ptr(), values.data_ptr(), X.data_ptr(), rows, cols, n, meta_row_stride,
        values_row_stride)


# ---- 2:4 structured-sparse int8 GEMM (the cuSPARSELt backend) ---------------

def sparse_i8_compressed_size(m: int, k: int) -> int:
    """Bytes of the compressed operand of an m x k int8 matrix (the size query
    of cusparseLtSpMMACompressedSize, reference src/cusparselt_backend.cu:140-146)."""
    L = _lib.load()
    n = L.spb_sparse_i8_compressed_size(m, k)
    if n < 0:
        _lib.check(1, "sparse_i8_compressed_size")
    return int(n)


def sparse_i8_prune_check(d_weights, m: int, k: int, stream=None) -> int:
    """Groups of the int8 [m][k] matrix with more than two non-zeros
    (0 = already 2:4), cusparseLtSpMMAPruneCheck as prepare uses it
    (reference src/cusparselt_backend.cu:123-136)."""
    pa = _dev(d_weights, "d_weights", torch.int8, m * k)
    res = torch.empty(1, dtype=torch.int32, device=d_weights.device)
    _lib.check(_lib.load().spb_sparse_i8_prune_check(pa, m, k, res.data_ptr(),
                                                       _stream_ptr(stream)),
               "sparse_i8_prune_check")
    return int(res.item())


class CuSparseLtGemm:
    """CuSparseLtGemm (reference include/spbitnet/cusparselt_backend.h:28-77,
    src/cusparselt_backend.cu:38-219): D[m,n] = A_pruned[m,k] * B[k,n] with
    int32 accumulation on the int8 sparse matrix cores.

    prepare(d_weights) prunes a device int8 [m][k] row-major matrix (any int8
    values, k a multiple of 4) to 2:4 along k -- the two largest |a| of each
    group of four, on equal magnitudes the higher index; groups with at most
    two non-zeros are kept whole -- and compresses it into a device buffer
    this object owns.  execute(d_B, d_D) takes B int8 [k x n] column-major
    (a [n][k] tensor) and writes D int32 [m x n] column-major (a [n][m]
    tensor).  Any n >= 1 (the reference needs n >= 16)."""

    def __init__(self, m: int, k: int, n: int, device="cuda"):
        if n < 1:
            raise ValueError("n must be >= 1")
        self._m, self._k, self._n = m, k, n
        size = sparse_i8_compressed_size(m, k)
        self._comp = torch.empty(max(size, 16), dtype=torch.uint8, device=device)
        self._prepared = False

    def m(self) -> int:
        return self._m

    def k(self) -> int:
        return self._k

    def n(self) -> int:
        return self._n

    def prepare(self, d_weights, stream=None) -> None:
        """Prune to 2:4 and compress (src/cusparselt_backend.cu:107-166)."""
        pa = _dev(d_weights, "d_weights", torch.int8, self._m * self._k)
        _lib.check(_lib.load().spb_sparse_i8_prune_compress(
            pa, None, self._comp.data_ptr(), self._m, self._k, _stream_ptr(stream)),
            "CuSparseLtGemm.prepare")
        self._prepared = True

    def execute(self, d_B, d_D, stream=None) -> None:
        """D = A_pruned * B (src/cusparselt_backend.cu:173-207)."""
        if not self._prepared:
            raise RuntimeError("CuSparseLtGemm.execute() called before prepare()")
        pb = _dev(d_B, "d_B", torch.int8, self._n * self._k)
        pd = _dev(d_D, "d_D", torch.int32, self._n * self._m)
        _lib.check(_lib.load().spb_sparse_i8_gemm(self._comp.data_ptr(), pb, pd, self._m,
                                                    self._k, self._n, _stream_ptr(stream)),
                   "CuSparseLtGemm.execute")

    def get_pruned_weights(self, d_out, stream=None) -> None:
        """The pruned dense int8 [m][k] matrix (src/cusparselt_backend.cu:209-217)."""
        if not self._prepared:
            raise RuntimeError("CuSparseLtGemm.get_pruned_weights(): not prepared")
        po = _dev(d_out, "d_out", torch.int8, self._m * self._k)
        _lib.check(_lib.load().spb_sparse_i8_decompress(self._comp.data_ptr(), po, self._m,
                                                          self._k, _stream_ptr(stream)),
                   "CuSparseLtGemm.get_pruned_weights")

    def kernel_id(self, d_B) -> int:
        """1 when execute runs the matrix-core kernel for d_B, 0 the general one."""
        return _lib.load().spb_sparse_i8_gemm_kernel_id(self._comp.data_ptr(), d_B.data_ptr(),
                                                        self._m, self._k, self._n)


# ---- bit-plane activation layout (no reference counterpart) -----------------

def planes_words(cols: int) -> int:
    """uint32 words of the plane layout of a `cols`-column activation."""
    return 8 * ((cols + 31) // 32)


def activation_planes_gpu(x, planes, cols, stream=None):
    """int8 x[cols] -> bit-plane layout (word [w*8+b] = plane b of columns 32w..32w+31)."""
    px = _dev(x, "x", torch.int8, cols)
    pp = _dev(planes, "planes", (torch.int32, torch.uint32), planes_words(cols))
    _lib.check(_lib.load().spb_activation_planes(px, pp, cols, _stream_ptr(stream)),
               "activation_planes_gpu")


def absmax_quantize_planes_gpu(input, planes, d_absmax, size, output=None, stream=None):
    """absmax + int8 quantisation emitting the plane layout (and the int8 vector if given)."""
    if input.dtype not in _HALF_KIND:
        raise TypeError("input must be float16 or bfloat16")
    pi = _dev(input, "input", input.dtype, size)
    pp = _dev(planes, "planes", (torch.int32, torch.uint32), planes_words(size))
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    po = _dev(output, "output", torch.int8, size) if output is not None else None
    fn = getattr(_lib.load(), f"spb_absmax_quantize_planes_{_HALF_KIND[input.dtype]}")
    _lib.check(fn(pi, pp, po, pa, size, _stream_ptr(stream)), "absmax_quantize_planes_gpu")


def sparse_ternary_gemv_planes_gpu(meta, values, planes, y, rows, cols, meta_row_stride,
                                   values_row_stride, stream=None):
    """sparse_ternary_gemv_gpu with plane-layout activations."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    empty = rows == 0 or cols == 0
    pp = _dev(planes, "planes", (torch.int32, torch.uint32), 0 if empty else planes_words(cols))
    py = _dev(y, "y", torch.int32, 0 if empty else rows)
    _lib.check(_lib.load().spb_sparse_ternary_gemv_planes(pm, pv, pp, py, rows, cols,
                                                          meta_row_stride, values_row_stride,
                                                          _stream_ptr(stream)),
               "sparse_ternary_gemv_planes_gpu")


def fused_sparse_bitlinear_planes_gpu(meta, values, planes, output, d_absmax, gamma, rows, cols,
                                      meta_row_stride, values_row_stride, stream=None):
    """GEMV on plane activations + the reference's dequant epilogue; output fp16 or bf16."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    if output.dtype not in _HALF_KIND:
        raise TypeError("output must be float16 or bfloat16")
    empty = rows == 0 or cols == 0
    pp = _dev(planes, "planes", (torch.int32, torch.uint32), 0 if empty else planes_words(cols))
    po = _dev(output, "output", output.dtype, 0 if empty else rows)
    pa = _dev(d_absmax, "d_absmax", torch.float32, 1)
    fn = getattr(_lib.load(), f"spb_fused_sparse_bitlinear_planes_{_HALF_KIND[output.dtype]}")
    _lib.check(fn(pm, pv, pp, po, pa, float(gamma), rows, cols, meta_row_stride,
                  values_row_stride, _stream_ptr(stream)), "fused_sparse_bitlinear_planes_gpu")


def gemv_kernel_id(meta, values, rows, cols, meta_row_stride, values_row_stride) -> int:
    """1 if the bit-plane GEMV kernel would run for these arguments, else 0."""
    return _lib.load().spb_sparse_ternary_gemv_kernel_id(
        meta.data_ptr(), values.data_ptr(), rows, cols, meta_row_stride, values_row_stride)


def bitlinear_workspace_size(cols: int) -> int:
    """Bytes of the workspace bitlinear_gpu needs for `cols` input columns."""
    return int(_lib.load().spb_bitlinear_workspace_size(int(cols)))


def bitlinear_gpu(meta, values, x, output, gamma, rows, cols, meta_row_stride,
                  values_row_stride, workspace, stream=None):
    """InferenceEngine::bitlinear (reference src/inference.cu:106-117) as one
    call: absmax, quantisation, sparse GEMV and dequantisation, with the
    absmax scratch (and the activation planes) in `workspace`, a uint8 GPU
    tensor of at least bitlinear_workspace_size(cols) bytes."""
    pm, pv = _weights(meta, values, rows, cols, meta_row_stride, values_row_stride)
    empty = rows == 0 or cols == 0
    kind = _HALF_KIND.get(x.dtype)
    if kind is None:
        raise TypeError(f"x has dtype {x.dtype}, expected float16 or bfloat16")
    px = _dev(x, "x", x.dtype, 0 if empty else cols)
    po = _dev(output, "output", x.dtype, 0 if empty else rows)
    need = 0 if empty else bitlinear_workspace_size(cols)
    pw = _dev(workspace, "workspace", torch.uint8, need)
    fn = getattr(_lib.load(), f"spb_bitlinear_{kind}")
    _lib.check(fn(pm, pv, px, po, float(gamma), rows, cols, meta_row_stride, values_row_stride,
                  pw, workspace.numel(), _stream_ptr(stream)), "bitlinear_gpu")


# ---- batches of tokens over a paged cache (no reference counterpart) ---------

_ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


# These calls are short (a decode step's rotation runs 2.6 us), so their checks
# are: one condition per tensor, and the reason is looked for when it fails.

_Tensor = torch.Tensor
_raw_stream = torch._C._cuda_getCurrentRawStream
_INT_MAX = 2 ** 31 - 1


# ctypes passes the low 32 bits of what is longer, so numbers are looked at before.

def _int32(x, name: str):
    if not -_INT_MAX <= x <= _INT_MAX:
        raise ValueError(f"{name} {x} does not fit in 32 bits")
    return x


def _too_long(shape, name: str):
    raise ValueError(f"{name} has shape {tuple(shape)}, which does not fit in 32 bits")


def _sizes(shape, name: str) -> None:
    if max(shape) > _INT_MAX:
        _too_long(shape, name)


def _device(t, name: str) -> int:
    """The index of the GPU that a call runs on: t's, which must be the current one."""
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name} must be a GPU tensor")
    if dev != torch._C._cuda_getDevice():
        raise ValueError(f"{name} is on {t.device}, the current device is "
                         f"cuda:{torch.cuda.current_device()}")
    return dev


def _kind(t, name: str) -> str:
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    kind = _HALF_KIND.get(t.dtype)
    if kind is None:
        raise TypeError(f"{name} has dtype {t.dtype}, expected float16 or bfloat16")
    return kind


def _refuse(t, name: str, dtype, shape, dev: int):
    """Raises what is wrong with a tensor; returns if its layout is."""
    if _device(t, name) != dev:
        raise ValueError(f"{name} is on {t.device}, others are on cuda:{dev}")
    if t.dtype != dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _heads(t, name: str, dtype, shape, dev: int) -> Tuple[int, int]:
    """Pointer and token stride of a [tokens][heads][head_dim] tensor whose
    tokens' heads are contiguous (a part of a stacked projection may be one)."""
    if (not isinstance(t, _Tensor) or t.get_device() != dev or t.dtype != dtype
            or t.shape != shape):
        _refuse(t, name, dtype, shape, dev)
    st, (n, heads, hd) = t.stride(), shape
    if st[2] != 1 or (heads > 1 and st[1] != hd):
        raise ValueError(f"{name}: a token's heads must be contiguous")
    return t.data_ptr(), st[0] if n > 1 else heads * hd


def _flat(t, name: str, dtype, shape, dev: int) -> int:
    """Pointer of a contiguous tensor."""
    if (not isinstance(t, _Tensor) or t.get_device() != dev or t.dtype != dtype
            or t.shape != shape):
        _refuse(t, name, dtype, shape, dev)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _on(stream, dev: int):
    return (_raw_stream(dev) or None) if stream is None else _stream_ptr(stream)


def rope_inv_freq(rotary_dim: int, theta: float = 10000.0, scaling: str = "none",
                  factor: float = 1.0, original_positions: int = 0, beta_fast: float = 32.0,
                  beta_slow: float = 1.0) -> Tuple[torch.Tensor, float]:
    """Radians per position of each pair (float64, on the host) and the factor of
    the rotated pairs, for scaling "none", "linear", "ntk" or "yarn"
    (spb_rope_inv_freq)."""
    if scaling not in _ROPE_SCALING:
        raise ValueError(f"scaling must be one of {sorted(_ROPE_SCALING)}, not {scaling!r}")
    rotary_dim = _int32(int(rotary_dim), "rotary_dim")
    original_positions = _int32(int(original_positions), "original_positions")
    out = torch.empty(max(rotary_dim // 2, 1), dtype=torch.float64)
    scale = ctypes.c_float()
    _lib.check(_lib.load().spb_rope_inv_freq(out.data_ptr(), ctypes.addressof(scale),
                                             rotary_dim, float(theta),
                                             _ROPE_SCALING[scaling], float(factor),
                                             original_positions, float(beta_fast),
                                             float(beta_slow)), "rope_inv_freq")
    return out, scale.value


class _Descriptor:
    """What a call passes on as a C struct of pointers and sizes, taken once.  Its
    attributes hold the tensors and say the sizes that the calls check others against;
    one set afterwards would free the memory behind a pointer or let a smaller tensor
    pass, so that is refused.  A program may add attributes of its own."""

    _fixed = ()  # names, once _ptr is set (last)

    def _keep(self, name):
        if name in self._fixed:
            raise AttributeError(f"{name} of a {type(self).__name__} cannot be changed: make "
                                 "another (the contents of its tensors may be)")

    def __setattr__(self, name, value):
        self._keep(name)
        object.__setattr__(self, name, value)
        if name == "_ptr":
            object.__setattr__(self, "_fixed", frozenset(self.__dict__) | {"_fixed"})

    def __delattr__(self, name):
        self._keep(name)
        object.__delattr__(self, name)


class Rope(_Descriptor):
    """A rotation (spb_rope): inv_freq, float64 radians per position of each pair
    (rotary_dim / 2 of them, moved to the GPU if they are not there), the factor
    of the rotated pairs and their layout: pairs (2i, 2i + 1) when interleaved,
    else (i, i + rotary_dim / 2)."""

    def __init__(self, inv_freq: torch.Tensor, scale: float = 1.0, interleaved: bool = True):
        if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or inv_freq.numel() < 1:
            raise ValueError("inv_freq must be a float64 vector")
        if not inv_freq.is_cuda:
            inv_freq = inv_freq.to(torch.device("cuda", torch.cuda.current_device()))
        self.inv_freq = inv_freq.contiguous()
        self._dev = _device(self.inv_freq, "inv_freq")
        self.rotary_dim = 2 * inv_freq.numel()
        self.scale, self.interleaved = float(scale), bool(interleaved)
        self._c = _lib.RopeC(self.inv_freq.data_ptr(), self.rotary_dim, int(self.interleaved),
                             self.scale)
        self._ptr = ctypes.addressof(self._c)

    @staticmethod
    def scaled(rotary_dim: int, theta: float = 10000.0, interleaved: bool = True,
               **scaling) -> "Rope":
        """The rotation of rope_inv_freq(rotary_dim, theta, **scaling)."""
        f, scale = rope_inv_freq(rotary_dim, theta, **scaling)
        return Rope(f, scale, interleaved)


def _no(x, kind, name: str):
    raise TypeError(f"{name} must be a {kind.__name__}, not {type(x).__name__}")


def _same_device(x, kind, name: str, dev: int) -> None:
    if not isinstance(x, kind):
        _no(x, kind, name)
    if x._dev != dev:
        raise ValueError(f"{name} is on cuda:{x._dev}, the tensors are on cuda:{dev}")


def rope_tokens_gpu(x, output, positions, rope: Rope, stream=None):
    """Rotates the heads of x [tokens][heads][head_dim] to positions (int32
    [tokens]; a negative one is padding, its output stays as it was) into output,
    which may be x (spb_rope_tokens_*)."""
    kind = _kind(x, "x")
    shape, dt = x.shape, x.dtype
    if len(shape) != 3:
        raise ValueError("x must be [tokens][heads][head_dim]")
    n, heads, hd = shape
    if n > _INT_MAX or heads > _INT_MAX or hd > _INT_MAX:
        _too_long(shape, "x")
    dev = _device(x, "x")
    px, sx = _heads(x, "x", dt, shape, dev)
    py, sy = _heads(output, "output", dt, shape, dev)
    pp = _flat(positions, "positions", torch.int32, (n,), dev)
    _same_device(rope, Rope, "rope", dev)
    L = _lib.load()
    fn = L.spb_rope_tokens_f16 if kind == "f16" else L.spb_rope_tokens_bf16
    _lib.check(fn(px, py, pp, rope._ptr, n, heads, hd, sx, sy, _on(stream, dev)),
               "rope_tokens_gpu")


def qk_norm_rope_gpu(q, k, q_output, k_output, q_weight, k_weight, positions,
                     rope: Optional[Rope], eps: float = 1e-5, stream=None):
    """RMSNorm of every head of q [tokens][heads][head_dim] and k
    [tokens][kv heads][head_dim] with the weights (float32 [head_dim]), then the
    rotation to positions, in one pass (spb_qk_norm_rope_*).  rope None: norms
    only.  The outputs may be q and k."""
    kind = _kind(q, "q")
    _kind(k, "k")
    qs, ks, dt, dev = q.shape, k.shape, q.dtype, _device(q, "q")
    if len(qs) != 3 or len(ks) != 3 or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError("q and k must be [tokens][heads][head_dim] with the same tokens and "
                         "head_dim")
    n, nh, hd = qs
    if n > _INT_MAX or nh > _INT_MAX or hd > _INT_MAX:
        _too_long(qs, "q")
    if ks[1] > _INT_MAX:
        _too_long(ks, "k")
    pq, sq = _heads(q, "q", dt, qs, dev)
    pk, sk = _heads(k, "k", dt, ks, dev)
    pqo, sqo = _heads(q_output, "q_output", dt, qs, dev)
    pko, sko = _heads(k_output, "k_output", dt, ks, dev)
    pqw = _flat(q_weight, "q_weight", torch.float32, (hd,), dev)
    pkw = _flat(k_weight, "k_weight", torch.float32, (hd,), dev)
    pp = pr = None
    if rope is not None:
        pp = _flat(positions, "positions", torch.int32, (n,), dev)
        _same_device(rope, Rope, "rope", dev)
        pr = rope._ptr
    L = _lib.load()
    fn = L.spb_qk_norm_rope_f16 if kind == "f16" else L.spb_qk_norm_rope_bf16
    _lib.check(fn(pq, pk, pqo, pko, pqw, pkw, pp, pr, n, nh, ks[1], hd, sq, sk, sqo, sko, eps,
                  _on(stream, dev)), "qk_norm_rope_gpu")


class PagedKVCache(_Descriptor):
    """A pool of pages (spb_paged_cache) in two tensors k and v
    [pages][kv heads][page_size][head_dim] (fp16 or bf16) of equal strides; the
    last dimension is contiguous, so pages laid out [page_size][kv heads][head_dim]
    come as a transposed view.  Keeps the tensors alive."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        self.kind = _kind(k, "k")
        self._dev = _device(k, "k")
        if _device(v, "v") != self._dev or v.dtype != k.dtype:
            raise TypeError(f"v is {v.dtype} on {v.device}, expected {k.dtype} on {k.device}")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [pages][kv heads][page_size][head_dim]")
        _sizes(k.shape, "each of k and v")
        if k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v must have the same strides and a contiguous last dimension")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        st = k.stride()
        self._c = _lib.PagedCacheC(k.data_ptr(), v.data_ptr(), st[0], st[1], st[2],
                                   self.num_pages, self.page_size, self.num_kv_heads,
                                   self.head_dim)
        self._ptr = ctypes.addressof(self._c)


class PagedBatch(_Descriptor):
    """A batch of new tokens (spb_paged_batch): int32 GPU tensors token_starts
    [sequences + 1], kv_lens [sequences] and page_table [sequences][width];
    num_tokens rows in the token tensors (those past token_starts' last entry are
    padding); max_new, the most new tokens of a sequence, if the program knows it.
    The tensors are read by the calls, so a program may refill them between
    calls (and between replays of a captured one); the object itself is fixed, as are
    a Rope and a PagedKVCache."""

    def __init__(self, token_starts, kv_lens, page_table, num_tokens: int, max_new: int = 0):
        if not isinstance(kv_lens, torch.Tensor) or kv_lens.dim() != 1:
            raise ValueError("kv_lens must be a vector")
        if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
            raise ValueError("page_table must be [sequences][width]")
        _sizes(kv_lens.shape, "kv_lens")
        _sizes(page_table.shape, "page_table")
        n, width = kv_lens.numel(), page_table.shape[1]
        num_tokens, max_new = _int32(int(num_tokens), "num_tokens"), _int32(int(max_new), "max_new")
        if num_tokens < 0 or max_new < 0:
            raise ValueError("negative number of tokens")
        self._dev = dev = _device(kv_lens, "kv_lens")
        self.token_starts, self.kv_lens, self.page_table = token_starts, kv_lens, page_table
        self.num_seqs, self.num_tokens, self.max_new = n, num_tokens, max_new
        self._c = _lib.PagedBatchC(_flat(token_starts, "token_starts", torch.int32, (n + 1,), dev),
                                   _flat(kv_lens, "kv_lens", torch.int32, (n,), dev),
                                   _flat(page_table, "page_table", torch.int32, (n, width), dev),
                                   n, width, self.num_tokens, self.max_new)
        self._ptr = ctypes.addressof(self._c)


def paged_append_gpu(cache: PagedKVCache, batch: PagedBatch, k, v, rope: Optional[Rope] = None,
                     q=None, q_output=None, q_weight=None, k_weight=None, eps: float = 1e-5,
                     stream=None):
    """Writes the batch's k and v [tokens][kv heads][head_dim] into their pages, the
    keys rotated to their positions on the way (rope None: as they are), and, if q
    [tokens][heads][head_dim] is given, rotates it into q_output (which may be q)
    in the same launch.  q_weight / k_weight (float32 [head_dim]): RMSNorm before
    the rotation (spb_paged_append_*)."""
    if not isinstance(cache, PagedKVCache):
        _no(cache, PagedKVCache, "cache")
    dev = _device(cache.k, "the cache")
    _same_device(batch, PagedBatch, "batch", dev)
    n, hd, dt = batch.num_tokens, cache.head_dim, cache.dtype
    pk = pv = pq = pqo = pqw = pkw = pr = None
    sk = sv = sq = sqo = nh = 0
    if k is not None or v is not None:
        shape = (n, cache.num_kv_heads, hd)
        pk, sk = _heads(k, "k", dt, shape, dev)
        pv, sv = _heads(v, "v", dt, shape, dev)
    if q is not None or q_output is not None:
        _kind(q, "q")
        nh = q.shape[1] if q.dim() == 3 else 0
        if nh > _INT_MAX:
            _too_long(q.shape, "q")
        shape = (n, nh, hd)
        pq, sq = _heads(q, "q", dt, shape, dev)
        pqo, sqo = _heads(q_output, "q_output", dt, shape, dev)
    if q_weight is not None:
        pqw = _flat(q_weight, "q_weight", torch.float32, (hd,), dev)
    if k_weight is not None:
        pkw = _flat(k_weight, "k_weight", torch.float32, (hd,), dev)
    if rope is not None:
        _same_device(rope, Rope, "rope", dev)
        pr = rope._ptr
    L = _lib.load()
    fn = L.spb_paged_append_f16 if cache.kind == "f16" else L.spb_paged_append_bf16
    _lib.check(fn(cache._ptr, batch._ptr, pk, pv, pq, pqo, sk, sv, sq, sqo, nh, pqw, pkw, eps, pr,
                  _on(stream, dev)), "paged_append_gpu")


def paged_attention_workspace_size(num_heads: int, num_kv_heads: int, head_dim: int) -> int:
    """Bytes of the workspace that paged_attention_gpu needs for these heads."""
    n = int(_lib.load().spb_paged_attention_workspace_size(
        _int32(num_heads, "num_heads"), _int32(num_kv_heads, "num_kv_heads"),
        _int32(head_dim, "head_dim")))
    if n == 0:
        _lib.check(1, "paged_attention_workspace_size")
    return n


def paged_attention_gpu(cache: PagedKVCache, batch: PagedBatch, q, output, workspace,
                        scale: Optional[float] = None, causal: bool = True, window: int = 0,
                        stream=None):
    """Attention of the batch's queries q [tokens][heads][head_dim] over their
    sequences' pages into output (which may be q): position p sees positions j <= p
    when causal, j > p - window when window > 0, and the whole cached length
    otherwise.  scale None: head_dim ** -0.5.  workspace: a contiguous uint8 GPU
    tensor of paged_attention_workspace_size bytes (spb_paged_attention_*)."""
    if not isinstance(cache, PagedKVCache):
        _no(cache, PagedKVCache, "cache")
    dev = _device(cache.k, "the cache")
    _same_device(batch, PagedBatch, "batch", dev)
    hd, dt = cache.head_dim, cache.dtype
    _kind(q, "q")
    nh = q.shape[1] if q.dim() == 3 else 0
    if nh > _INT_MAX:
        _too_long(q.shape, "q")
    shape = (batch.num_tokens, nh, hd)
    window = _int32(window, "window")
    pq, sq = _heads(q, "q", dt, shape, dev)
    po, so = _heads(output, "output", dt, shape, dev)
    size = workspace.numel() if isinstance(workspace, _Tensor) else 0
    pw = _flat(workspace, "workspace", torch.uint8, (size,), dev)
    L = _lib.load()
    fn = L.spb_paged_attention_f16 if cache.kind == "f16" else L.spb_paged_attention_bf16
    _lib.check(fn(cache._ptr, batch._ptr, pq, po, sq, so, nh,
                  hd ** -0.5 if scale is None else scale, 1 if causal else 0, window, pw, size,
                  _on(stream, dev)), "paged_attention_gpu")


# ---- what each request of a shared batch brings of its own (no reference counterpart)

_MAX_SECTIONS = 4
_LOGITS_KIND = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}


class Adapters(_Descriptor):
    """A pool of low-rank adapters of one projection (spb_adapters): a
    [adapters][sections * rank][cols] and b [adapters][rows][rank] (fp16 or bf16, last
    dimension contiguous, strides multiples of 8), scales float32 [adapters] and, where
    adapters have fewer ranks than the pool, ranks int32 [adapters].  sections: the rows
    of each part of a stacked projection, each with `rank` rows of a (None: one part).
    Keeps the tensors alive; their contents may be changed between calls."""

    def __init__(self, a, b, scales, ranks=None, sections=None):
        self.kind = _kind(a, "a")
        _kind(b, "b")
        if a.dim() != 3 or b.dim() != 3 or b.shape[0] != a.shape[0]:
            raise ValueError("a and b must be [adapters][sections * rank][cols] and "
                             "[adapters][rows][rank]")
        _sizes(a.shape, "a")
        _sizes(b.shape, "b")
        self._dev = dev = _device(a, "a")
        if _device(b, "b") != dev or b.dtype != a.dtype:
            raise TypeError(f"b is {b.dtype} on {b.device}, expected {a.dtype} on {a.device}")
        num, rows, rank = b.shape
        parts = (rows,) if sections is None else tuple(_int32(int(s), "a section")
                                                       for s in sections)
        if not 1 <= len(parts) <= _MAX_SECTIONS or min(parts) < 1 or sum(parts) != rows:
            raise ValueError(f"sections {parts} must be 1 to {_MAX_SECTIONS} numbers that sum up "
                             f"to the {rows} rows of b")
        if a.shape[1] != len(parts) * rank:
            raise ValueError(f"a has {a.shape[1]} rows, expected {len(parts)} sections of rank "
                             f"{rank}")
        for t, name in ((a, "a"), (b, "b")):
            if t.shape[2] > 1 and t.stride(2) != 1:
                raise ValueError(f"{name}: the last dimension must be contiguous")
        self.a, self.b, self.scales, self.ranks = a, b, scales, ranks
        self.dtype, self.num_adapters, self.rows, self.rank = a.dtype, num, rows, rank
        self.cols, self.sections = a.shape[2], parts
        ps = _flat(scales, "scales", torch.float32, (num,), dev)
        pr = None if ranks is None else _flat(ranks, "ranks", torch.int32, (num,), dev)
        self._c = _lib.AdaptersC(a.data_ptr(), b.data_ptr(), ps, pr, a.stride(0), a.stride(1),
                                 b.stride(0), b.stride(1), num, rank, self.cols, len(parts),
                                 (ctypes.c_int * _MAX_SECTIONS)(*parts))
        self._ptr = ctypes.addressof(self._c)


def _rows(t, name: str, dtype, shape, dev: int) -> Tuple[int, int]:
    """Pointer and row stride of a matrix with contiguous rows."""
    if (not isinstance(t, _Tensor) or t.get_device() != dev or t.dtype != dtype
            or t.shape != shape):
        _refuse(t, name, dtype, shape, dev)
    st = t.stride()
    if st[1] != 1 and shape[1] > 1:
        raise ValueError(f"{name}: rows must be contiguous")
    return t.data_ptr(), st[0] if shape[0] > 1 else shape[1]


def adapters_workspace_size(adapters: Adapters, num_tokens: int) -> int:
    """Bytes of the workspace that adapters_gpu needs for at most num_tokens tokens."""
    if not isinstance(adapters, Adapters):
        _no(adapters, Adapters, "adapters")
    n = int(_lib.load().spb_adapters_workspace_size(adapters._ptr,
                                                    _int32(num_tokens, "num_tokens")))
    if n == 0:
        _lib.check(1, "adapters_workspace_size")
    return n


def adapters_gpu(adapters: Adapters, ids, x, base, output, workspace, stream=None):
    """output[t] = base[t] + scale * B (A x[t]) with the adapter ids[t] (int32 [tokens];
    outside the pool: none, output[t] = base[t]).  x [tokens][cols]; base, what the
    shared projection gave for x, and output, which may be base, [tokens][rows].
    workspace: a contiguous uint8 GPU tensor of adapters_workspace_size bytes
    (spb_adapters_*)."""
    if not isinstance(adapters, Adapters):
        _no(adapters, Adapters, "adapters")
    dev, dt = _device(adapters.a, "adapters"), adapters.dtype
    if not isinstance(ids, _Tensor) or ids.dim() != 1:
        raise ValueError("ids must be a vector")
    n = ids.shape[0]
    if n > _INT_MAX:
        _too_long(ids.shape, "ids")
    pi = _flat(ids, "ids", torch.int32, (n,), dev)
    px, sx = _rows(x, "x", dt, (n, adapters.cols), dev)
    pb, sb = _rows(base, "base", dt, (n, adapters.rows), dev)
    po, so = _rows(output, "output", dt, (n, adapters.rows), dev)
    size = workspace.numel() if isinstance(workspace, _Tensor) else 0
    pw = _flat(workspace, "workspace", torch.uint8, (size,), dev)
    L = _lib.load()
    fn = L.spb_adapters_f16 if adapters.kind == "f16" else L.spb_adapters_bf16
    _lib.check(fn(adapters._ptr, pi, px, pb, po, n, sx, sb, so, pw, size, _on(stream, dev)),
               "adapters_gpu")


class Sampling(_Descriptor):
    """Settings of sample_gpu (spb_sampling), each a number for all rows or a GPU vector
    with one for each: temperature (float32; 0: greedy), top_k (int32; 0: all), top_p
    (float32; 1: all) and min_p (float32; 0: all).  Vectors are read by the calls, so a
    program may refill them between calls (and between replays of a captured one)."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        self._dev, self.rows = None, None
        ptrs, numbers = [], []
        for name, x, dtype, off in (("temperature", temperature, torch.float32, 1.0),
                                    ("top_k", top_k, torch.int32, 0),
                                    ("top_p", top_p, torch.float32, 1.0),
                                    ("min_p", min_p, torch.float32, 0.0)):
            if isinstance(x, _Tensor):
                if x.dim() != 1:
                    raise ValueError(f"{name} must be a number or a vector")
                _sizes((*x.shape, 0), name)
                dev = _device(x, name)
                if self._dev is not None and (dev, x.shape[0]) != (self._dev, self.rows):
                    raise ValueError(f"{name} has {x.shape[0]} rows on cuda:{dev}, others "
                                     f"{self.rows} on cuda:{self._dev}")
                self._dev, self.rows = dev, x.shape[0]
                ptrs.append(_flat(x, name, dtype, x.shape, dev))
                numbers.append(off)
            else:
                ptrs.append(None)
                numbers.append(_int32(int(x), name) if dtype is torch.int32 else float(x))
        self.temperature, self.top_k, self.top_p, self.min_p = temperature, top_k, top_p, min_p
        t, k, p, m = numbers
        if not t >= 0 or k < 0 or not 0 <= p <= 1 or not 0 <= m <= 1:
            raise ValueError(f"temperature {t} and top_k {k} must not be negative, top_p {p} and "
                             f"min_p {m} must be in [0, 1]")
        self._c = _lib.SamplingC(*ptrs, t, k, p, m)
        self._ptr = ctypes.addressof(self._c)


def _logits(t) -> str:
    if not isinstance(t, _Tensor):
        raise TypeError("logits must be a torch.Tensor")
    kind = _LOGITS_KIND.get(t.dtype)
    if kind is None:
        raise TypeError(f"logits have dtype {t.dtype}, expected float32, float16 or bfloat16")
    if t.dim() != 2:
        raise ValueError("logits must be [rows][vocab]")
    if max(t.shape) > _INT_MAX:
        _too_long(t.shape, "logits")
    return kind


def sample_workspace_size(rows: int, vocab: int) -> int:
    """Bytes of the workspace that sample_gpu needs for at most `rows` rows."""
    n = int(_lib.load().spb_sample_workspace_size(_int32(rows, "rows"), _int32(vocab, "vocab")))
    if n == 0:
        _lib.check(1, "sample_workspace_size")
    return n


def sample_gpu(logits, uniforms, tokens, sampling: Sampling, workspace, logprobs=None,
               stream=None):
    """The next token of each row of logits [rows][vocab] (float32, fp16 or bf16) under
    the settings, into tokens (int32 [rows]): in the order of falling logits, equal ones by
    index, the first of the kept tokens whose weight with those before it passes
    uniforms[row] (float32, in [0, 1)) times the kept weight; -1 where all logits are minus
    infinity.  logprobs (float32 [rows]): the logarithm of its share of the kept weight.
    workspace: a contiguous uint8 GPU tensor of sample_workspace_size bytes (spb_sample_*)."""
    kind = _logits(logits)
    dev, (n, vocab) = _device(logits, "logits"), logits.shape
    pl, sl = _rows(logits, "logits", logits.dtype, logits.shape, dev)
    pu = _flat(uniforms, "uniforms", torch.float32, (n,), dev)
    pt = _flat(tokens, "tokens", torch.int32, (n,), dev)
    pp = None if logprobs is None else _flat(logprobs, "logprobs", torch.float32, (n,), dev)
    if not isinstance(sampling, Sampling):
        _no(sampling, Sampling, "sampling")
    if sampling._dev is not None and (sampling._dev != dev or sampling.rows != n):
        raise ValueError(f"sampling has {sampling.rows} rows on cuda:{sampling._dev}, logits {n} "
                         f"on cuda:{dev}")
    size = workspace.numel() if isinstance(workspace, _Tensor) else 0
    pw = _flat(workspace, "workspace", torch.uint8, (size,), dev)
    fn = getattr(_lib.load(), "spb_sample_" + kind)
    _lib.check(fn(pl, sl, pu, pt, pp, n, vocab, sampling._ptr, pw, size, _on(stream, dev)),
               "sample_gpu")


def token_logprobs_workspace_size(rows: int, vocab: int, top: int = 0) -> int:
    """Bytes of the workspace that token_logprobs_gpu needs for at most `rows` rows."""
    n = int(_lib.load().spb_token_logprobs_workspace_size(
        _int32(rows, "rows"), _int32(vocab, "vocab"), _int32(top, "top")))
    if n == 0:
        _lib.check(1, "token_logprobs_workspace_size")
    return n


def token_logprobs_gpu(logits, tokens, logprobs, workspace, top_ids=None, top_logprobs=None,
                       stream=None):
    """Log-probabilities of tokens (int32 [rows]; outside the vocabulary: padding, the
    row's outputs stay as they were) under logits [rows][vocab] (float32, fp16 or bf16), into
    logprobs (float32 [rows]; both None: not asked for), and the likeliest tokens of each
    row, the best first and equal ones by index, into top_ids (int32 [rows][top]) and
    top_logprobs (float32 [rows][top]).  workspace: a contiguous uint8 GPU tensor of
    token_logprobs_workspace_size bytes (spb_token_logprobs_*)."""
    kind = _logits(logits)
    dev, (n, vocab) = _device(logits, "logits"), logits.shape
    pl, sl = _rows(logits, "logits", logits.dtype, logits.shape, dev)
    pt = pp = pi = pv = None
    top = 0
    if tokens is not None or logprobs is not None:
        pt = _flat(tokens, "tokens", torch.int32, (n,), dev)
        pp = _flat(logprobs, "logprobs", torch.float32, (n,), dev)
    if top_ids is not None or top_logprobs is not None:
        if not isinstance(top_ids, _Tensor) or top_ids.dim() != 2:
            raise ValueError("top_ids must be [rows][top]")
        top = top_ids.shape[1]
        if top > _INT_MAX:
            _too_long(top_ids.shape, "top_ids")
        pi = _flat(top_ids, "top_ids", torch.int32, (n, top), dev)
        pv = _flat(top_logprobs, "top_logprobs", torch.float32, (n, top), dev)
    size = workspace.numel() if isinstance(workspace, _Tensor) else 0
    pw = _flat(workspace, "workspace", torch.uint8, (size,), dev)
    fn = getattr(_lib.load(), "spb_token_logprobs_" + kind)
    _lib.check(fn(pl, sl, pt, pp, pi, pv, n, vocab, top, pw, size, _on(stream, dev)),
               "token_logprobs_gpu")
