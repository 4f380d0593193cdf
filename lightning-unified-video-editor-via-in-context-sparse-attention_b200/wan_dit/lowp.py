"""Low-precision operators of the DiT: linear layers on microscaled 4-bit
operands, and a key/value cache held in 8 bits with the attention that reads
it (include/icsa_lowp.h; the kernels are in libicsa.so, there is no CPU
fallback).

    w = fp4_quantize(weight, "nvfp4", fp4_global_scale(weight))   # once, [N, K]
    y = fp4_linear(x, w, bias, activation="gelu_tanh")            # x: bf16 / f32 [M, K]

    cache = kv8_quantize(k, v, lengths)                           # [B, L, H, D]
    o = kv8_attention(q, cache)                                   # q: bf16 [B, Lq, Hq, D]

Every function takes and returns torch tensors on one CUDA device (which need
not be the current one) and runs on that device's current stream.  They
compute values only: no gradient is recorded, and fp4_linear and kv8_attention
refuse an input that requires one where gradients are enabled.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch

from in_context_sparse_attention import _capi

LOWP_EXPORTED = ("icsa_fp4_data_bytes", "icsa_fp4_scale_bytes", "icsa_fp4_quantize", "icsa_fp4_dequantize",
                 "icsa_fp4_linear_workspace_size", "icsa_fp4_linear", "icsa_fp4_linear_rows_workspace_size",
                 "icsa_fp4_linear_rows", "icsa_fp4_linear_scaled_rows_workspace_size", "icsa_fp4_linear_scaled_rows",
                 "icsa_kv8_quantize", "icsa_kv8_dequantize",
                 "icsa_kv8_attention_workspace_size", "icsa_kv8_attention_strided_workspace_size", "icsa_kv8_attention")

FP4_FORMATS = {"nvfp4": 0, "mxfp4": 1}
FP4_BLOCK = {"nvfp4": 16, "mxfp4": 32}
ACTIVATIONS = {None: 0, "gelu_tanh": 1}
KV8_TOKENS = 64     # tokens that share a scale

_DT = {torch.bfloat16: _capi.ICSA_BF16, torch.float32: _capi.ICSA_F32}


class _Kv8Desc(ctypes.Structure):
    """Mirror of struct icsa_kv8_cache."""
    _fields_ = [("B", ctypes.c_int), ("H", ctypes.c_int), ("L", ctypes.c_int), ("D", ctypes.c_int),
                ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p), ("lengths", ctypes.c_void_p)]


_lib = None


def _load():
    global _lib
    if _lib is not None:
        return _lib
    lib = _capi.load()
    for name in LOWP_EXPORTED:
        if not hasattr(lib, name):
            raise ImportError(f"{_capi.LIB_PATH} does not export {name}; rebuild it with `python build.py`")
    vp, i, i64, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    st, desc = ctypes.POINTER(i64), ctypes.POINTER(_Kv8Desc)
    for name, res, args in (
            ("icsa_fp4_data_bytes", sz, [i, i]),
            ("icsa_fp4_scale_bytes", sz, [i, i, i]),
            ("icsa_fp4_quantize", i, [vp, i, i64, i, i, i, f, vp, vp, vp]),
            ("icsa_fp4_dequantize", i, [vp, vp, i, i, i, f, vp, i, i64, vp]),
            ("icsa_fp4_linear_workspace_size", sz, [i, i, i]),
            ("icsa_fp4_linear", i, [i, vp, vp, f, vp, vp, f, vp, i, vp, i64, i, i, i, vp, sz, vp]),
            ("icsa_fp4_linear_rows_workspace_size", sz, [i, i, i, i]),
            ("icsa_fp4_linear_rows", i, [i, vp, i, i64, vp, vp, f, vp, i, vp, i64, i, i, i, vp, sz, vp]),
            ("icsa_fp4_linear_scaled_rows_workspace_size", sz, [i, i, i, i]),
            ("icsa_fp4_linear_scaled_rows", i, [i, vp, i, i64, vp, vp, f, vp, i, vp, i64, i, i, i, vp, sz, vp]),
            ("icsa_kv8_quantize", i, [desc, vp, vp, i, st, st, vp]),
            ("icsa_kv8_dequantize", i, [desc, vp, vp, i, vp]),
            ("icsa_kv8_attention_workspace_size", sz, [desc, i, i]),
            ("icsa_kv8_attention_strided_workspace_size", sz, [desc, i, i]),
            ("icsa_kv8_attention", i, [desc, vp, st, vp, i, i, vp, sz, vp])):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, res
    _lib = lib
    return lib


def _device(where, *tensors):
    """Index of the one CUDA device of the tensors (None entries are skipped)."""
    index = None
    for t in tensors:
        if t is None:
            continue
        i = t.get_device() if isinstance(t, torch.Tensor) else -1     # -1 on the CPU
        if i != index:
            if i < 0 or not t.is_cuda:
                raise ValueError(f"{where}: expected CUDA tensors")
            if index is not None:
                raise ValueError(f"{where}: tensors on cuda:{index} and cuda:{i}")
            index = i
    return index


def _no_gradient(where, t):
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{where}: no gradient is recorded; detach the inputs or call it under torch.no_grad()")


def _on(index, fn, *args):
    """fn(library, raw handle of the device's current stream, *args) with the device current."""
    lib = _lib or _load()
    if index == torch._C._cuda_getDevice():
        return fn(lib, torch._C._cuda_getCurrentRawStream(index), *args)
    with torch.cuda.device(index):
        return fn(lib, torch._C._cuda_getCurrentRawStream(index), *args)


# outputs are allocated with their strides given, the cheapest call
_empty = torch.empty_strided


def _bytes(like, n):
    """n bytes of workspace on the device of `like` (None for 0) and their address."""
    if not n:
        return None, None
    ws = _empty((n,), (1,), dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr()


# ---------------------------------------------------------------------------
# 4-bit tensors
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class Fp4Tensor:
    """A [rows, K] tensor in 4-bit storage (layout: include/icsa_lowp.h).

    data:   uint8 [rows, K' / 2], K' = K rounded up to 32, even element in the low half
    scales: uint8 [ceil(rows / 128), scale tiles along K, 32, 4, 4], row r and
            scale c of a tile at [r % 32, r // 32, c]
    """
    data: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    fmt: str
    global_scale: float = 1.0

    def __post_init__(self):
        if self.fmt not in FP4_FORMATS:
            raise ValueError(f"4-bit format {self.fmt!r}: expected one of {sorted(FP4_FORMATS)}")
        object.__setattr__(self, "shape", tuple(int(n) for n in self.shape))
        if len(self.shape) != 2 or self.shape[0] < 0 or self.shape[1] < 1:
            raise ValueError(f"Fp4Tensor: shape {self.shape} is not [rows, K] with K >= 1")
        data, scales = fp4_storage(*self.shape, self.fmt)
        for name, t, want in (("data", self.data, data), ("scales", self.scales, scales)):
            if t.dtype != torch.uint8 or t.shape != want or not t.is_contiguous():
                raise ValueError(f"Fp4Tensor: {name} must be contiguous uint8 {list(want)} for shape {list(self.shape)}")
        if self.data.get_device() != self.scales.get_device():
            raise ValueError("Fp4Tensor: data and scales on different devices")
        _check_global_scale(self.fmt, self.global_scale)

    @property
    def device(self):
        return self.data.device


@functools.lru_cache(maxsize=1024)
def fp4_storage(rows: int, K: int, fmt: str):
    """Shapes of `data` and `scales` of a [rows, K] Fp4Tensor."""
    tiles = 256 // (4 * FP4_BLOCK[fmt])
    return (rows, -(-K // 32) * 16), (-(-rows // 128), -(-K // 256) * tiles, 32, 4, 4)


def _check_global_scale(fmt, g):
    if not (isinstance(g, (int, float)) and 2.0 ** -149 <= g < 2.0 ** 128):     # (false for a NaN)
        raise ValueError(f"the global scale must be a positive finite float32 number, got {g!r}")
    if fmt == "mxfp4" and g != 1:
        raise ValueError("mxfp4 has no global scale (must be 1)")


def fp4_global_scale(x: torch.Tensor) -> float:
    """A global scale for nvfp4: the smallest power of two with which the
    largest magnitude of x is in range (448 x 6 steps), so that multiplying by
    it is exact.  Reads x and synchronises: for weights, once."""
    top = float(x.detach().abs().max()) if x.numel() else 0.0
    if not math.isfinite(top):
        raise ValueError("fp4_global_scale: x holds a NaN or an infinity")
    m, e = math.frexp(top / (6 * 448))
    return 1.0 if top == 0 else math.ldexp(1.0, max(min(e - (m == 0.5), 100), -100))


def fp4_row_scales(x: torch.Tensor) -> torch.Tensor:
    """f32 [rows, 1]: the global scales that fp4_linear(row_scales=True) gives
    the rows of x.  2^e, e the smallest with which the row's largest magnitude
    is in range (448 x 6 steps), in [-90, 90]; 1 for a row of zeros and for one
    with a NaN or an infinity."""
    top = x.detach().float().abs().amax(dim=1, keepdim=True)
    m, e = torch.frexp(top / (6 * 448))       # (the quotient of floats rounds to a power of two only where it is one)
    e = (e - (m == 0.5).int()).clamp(-90, 90)
    return torch.where((top > 0) & torch.isfinite(top), torch.ldexp(torch.ones_like(top), e), 1.0)


def _rows2d(where, x):
    """x as rows of contiguous elements that do not overlap, and their distance."""
    shape = x.shape
    if len(shape) != 2 or x.dtype not in _DT:
        raise ValueError(f"{where}: expected a 2-D bf16 or f32 tensor, got {x.dtype} {tuple(shape)}")
    rows, K = shape
    if K < 1:
        raise ValueError(f"{where}: no columns")
    ld, step = x.stride()
    if (K > 1 and step != 1) or (rows > 1 and ld < K):
        x, ld = x.contiguous(), K
    return x, (ld if rows > 1 else K)


def fp4_quantize(x: torch.Tensor, fmt: str = "nvfp4", global_scale: float = 1.0) -> Fp4Tensor:
    """x: bf16 or f32 [rows, K], any strides.  nvfp4: blocks of 16 with e4m3
    scales e4m3(amax / (6 global_scale)); mxfp4: blocks of 32 with
    power-of-two scales 2^(floor(log2 amax) - 2)."""
    if fmt not in FP4_FORMATS:
        raise ValueError(f"4-bit format {fmt!r}: expected one of {sorted(FP4_FORMATS)}")
    _check_global_scale(fmt, global_scale)
    index = _device("fp4_quantize", x)
    x, ld = _rows2d("fp4_quantize", x)
    return _on(index, _quantize, x, ld, fmt, float(global_scale))


def _quantize(lib, stream, x, ld, fmt, g):
    rows, K = x.shape
    (_, row), scales = fp4_storage(rows, K, fmt)
    device = x.device
    data = _empty((rows, row), (row, 1), dtype=torch.uint8, device=device)
    scales = _empty(scales, (scales[1] * 512, 512, 16, 4, 1), dtype=torch.uint8, device=device)
    code = lib.icsa_fp4_quantize(x.data_ptr(), _DT[x.dtype], ld, rows, K, FP4_FORMATS[fmt], g, data.data_ptr(),
                                 scales.data_ptr(), stream)
    if code:
        _capi.check(code, "icsa_fp4_quantize")
    t = object.__new__(Fp4Tensor)       # its tensors are as the constructor wants them
    t.__dict__.update(data=data, scales=scales, shape=(rows, K), fmt=fmt, global_scale=g)
    return t


def fp4_dequantize(t: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[rows, K] values of a 4-bit tensor, code * (block scale * global scale)."""
    if dtype not in _DT:
        raise ValueError(f"fp4_dequantize: dtype {dtype}, expected bf16 or f32")
    return _on(_device("fp4_dequantize", t.data, t.scales), _dequantize, t, dtype)


def _dequantize(lib, stream, t, dtype):
    rows, K = t.shape
    out = _empty((rows, K), (K, 1), dtype=dtype, device=t.data.device)
    code = lib.icsa_fp4_dequantize(t.data.data_ptr(), t.scales.data_ptr(), rows, K, FP4_FORMATS[t.fmt],
                                   t.global_scale, out.data_ptr(), _DT[dtype], K, stream)
    if code:
        _capi.check(code, "icsa_fp4_dequantize")
    return out


def fp4_linear(x, w: Fp4Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
               row_scales: bool = False) -> torch.Tensor:
    """bf16 [M, N] = act(x @ w^T + bias) with both operands in 4 bits.

    x: an Fp4Tensor [M, K] of w's format, or bf16 / f32 [M, K], which is
    quantised to it first.  w: [N, K].  bias: bf16 [N].  activation: None or
    "gelu_tanh".  row_scales: x is quantised with a global scale for each of
    its rows, a power of two found on the device, in place of 1.  nvfp4 needs
    that for rows that are not of order one: with scale 1 a block of 16 below
    0.0059 becomes zero, below 0.09 it loses bits, and above 2688 it
    saturates.  (mxfp4 has the range by itself: no difference.)"""
    if activation not in ACTIVATIONS:
        raise ValueError(f"fp4_linear: activation {activation!r}, expected one of {list(ACTIVATIONS)}")
    if not isinstance(w, Fp4Tensor):
        raise ValueError("fp4_linear: w must be an Fp4Tensor (fp4_quantize)")
    N, K = w.shape
    if N < 1:
        raise ValueError("fp4_linear: w has no rows")
    if len(x.shape) != 2 or x.shape[1] != K:
        raise ValueError(f"fp4_linear: x {tuple(x.shape)} and w {w.shape} differ in K")
    if bias is not None:
        if bias.dtype != torch.bfloat16 or bias.shape != (N,):
            raise ValueError(f"fp4_linear: bias must be bf16 [{N}]")
        _no_gradient("fp4_linear", bias)
        bias = bias.contiguous()
    if isinstance(x, Fp4Tensor):
        if x.fmt != w.fmt:
            raise ValueError(f"fp4_linear: x is {x.fmt}, w is {w.fmt}")
        if row_scales:
            raise ValueError("fp4_linear: row_scales is for rows that are still to be quantised")
        return _on(_device("fp4_linear", x.data, x.scales, w.data, w.scales, bias), _linear, x, w, bias, activation)
    _no_gradient("fp4_linear", x)
    index = _device("fp4_linear", x, w.data, w.scales, bias)
    x, ld = _rows2d("fp4_linear", x)
    return _on(index, _linear_rows, x, ld, w, bias, activation, row_scales and w.fmt == "nvfp4")


@functools.lru_cache(maxsize=1024)
def _linear_workspace(index, fmt, M, N, K, scaled=False):
    """Workspace bytes of icsa_fp4_linear (fmt None) or icsa_fp4_linear[_scaled]_rows; the device is current."""
    if fmt is None:
        return _lib.icsa_fp4_linear_workspace_size(M, N, K)
    if scaled:
        return _lib.icsa_fp4_linear_scaled_rows_workspace_size(FP4_FORMATS[fmt], M, N, K)
    return _lib.icsa_fp4_linear_rows_workspace_size(FP4_FORMATS[fmt], M, N, K)


def _linear(lib, stream, a, w, bias, activation):
    (M, K), N = a.shape, w.shape[0]
    out = _empty((M, N), (N, 1), dtype=torch.bfloat16, device=a.data.device)
    size = _linear_workspace(a.data.get_device(), None, M, N, K)
    ws, ptr = _bytes(out, size)
    code = lib.icsa_fp4_linear(FP4_FORMATS[w.fmt], a.data.data_ptr(), a.scales.data_ptr(), a.global_scale,
                               w.data.data_ptr(), w.scales.data_ptr(), w.global_scale,
                               bias.data_ptr() if bias is not None else None, ACTIVATIONS[activation], out.data_ptr(),
                               N, M, N, K, ptr, size, stream)
    if code:
        _capi.check(code, "icsa_fp4_linear")
    return out


def _linear_rows(lib, stream, x, ld, w, bias, activation, scaled):
    (M, K), N = x.shape, w.shape[0]
    out = _empty((M, N), (N, 1), dtype=torch.bfloat16, device=x.device)
    size = _linear_workspace(x.get_device(), w.fmt, M, N, K, scaled)
    ws, ptr = _bytes(out, size)
    fn = lib.icsa_fp4_linear_scaled_rows if scaled else lib.icsa_fp4_linear_rows
    code = fn(FP4_FORMATS[w.fmt], x.data_ptr(), _DT[x.dtype], ld, w.data.data_ptr(), w.scales.data_ptr(),
              w.global_scale, bias.data_ptr() if bias is not None else None, ACTIVATIONS[activation], out.data_ptr(),
              N, M, N, K, ptr, size, stream)
    if code:
        _capi.check(code, fn.__name__)
    return out


# ---------------------------------------------------------------------------
# 8-bit key/value cache
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class Kv8Cache:
    """Keys and values of B sequences in e4m3 (layout: include/icsa_lowp.h).

    k: float8_e4m3fn [B, H, nb, 64, D], v: float8_e4m3fn [B, H, nb, D, 64]
    (nb blocks of 64 tokens); k_scale, v_scale: f32 [B, H, nb], powers of two;
    L: tokens the cache has room for; lengths: int32 [B] on the device, the
    valid tokens of each sequence, or None (all L)."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    L: int
    lengths: Optional[torch.Tensor] = None

    def __post_init__(self):
        if self.k.dim() != 5 or self.k.shape[3] != KV8_TOKENS or self.k.shape[4] not in (64, 128):
            raise ValueError(f"Kv8Cache: k {tuple(self.k.shape)} is not [B, H, nb, 64, D] with D 64 or 128")
        B, H, nb, T, D = self.k.shape
        if self.L < 1 or nb != -(-self.L // T):
            raise ValueError(f"Kv8Cache: {nb} blocks do not hold L={self.L} tokens")
        for name, t, shape, dt in (("k", self.k, (B, H, nb, T, D), torch.float8_e4m3fn),
                                   ("v", self.v, (B, H, nb, D, T), torch.float8_e4m3fn),
                                   ("k_scale", self.k_scale, (B, H, nb), torch.float32),
                                   ("v_scale", self.v_scale, (B, H, nb), torch.float32)):
            if t.shape != shape or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"Kv8Cache: {name} must be contiguous {dt} {list(shape)}")
        _check_lengths("Kv8Cache", self.lengths, B)
        index = self.k.get_device()
        if any(t.get_device() != index for t in (self.v, self.k_scale, self.v_scale)) or (
                self.lengths is not None and self.lengths.get_device() != index):
            raise ValueError("Kv8Cache: tensors on different devices")

    @property
    def device(self):
        return self.k.device

    def _desc(self):
        B, H, _, _, D = self.k.shape
        return _Kv8Desc(B, H, self.L, D, self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                        self.v_scale.data_ptr(), self.lengths.data_ptr() if self.lengths is not None else None)


def _check_lengths(where, lengths, B):
    if lengths is not None and (lengths.dtype != torch.int32 or lengths.shape != (B,) or not lengths.is_contiguous()):
        raise ValueError(f"{where}: lengths must be contiguous int32 [{B}]")


@functools.lru_cache(maxsize=1024)
def _int64x3(a, b, c):
    return (ctypes.c_int64 * 3)(a, b, c)


def _strides(shape, strides):
    """Batch, token and head strides; 0 for an axis of one."""
    (B, L, H, _), (sb, st, sh, _) = shape, strides
    return _int64x3(sb if B > 1 else 0, st if L > 1 else 0, sh if H > 1 else 0)


def kv8_quantize(k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor] = None) -> Kv8Cache:
    """k, v: bf16 or f32 [B, L, H, D] with contiguous features; lengths: int32
    [B] on the device or None.  One scale for each block of 64 tokens and
    head, the smallest power of two with which the block's largest magnitude
    is at most 448.  Tokens behind a length are not read."""
    index = _device("kv8_quantize", k, v, lengths)
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _DT:
        raise ValueError(f"kv8_quantize: k {tuple(k.shape)} and v {tuple(v.shape)} must be bf16 or f32 [B, L, H, D]")
    B, L, H, D = shape = k.shape
    if D != 64 and D != 128:
        raise ValueError(f"kv8_quantize: head dim {D} (supported: 64, 128)")
    if B < 1 or L < 1 or H < 1:
        raise ValueError(f"kv8_quantize: empty k, v {tuple(shape)}")
    if lengths is not None:
        _check_lengths("kv8_quantize", lengths, B)
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1:
        k = k.contiguous()
        ks = k.stride()
    if vs[3] != 1:
        v = v.contiguous()
        vs = v.stride()
    return _on(index, _quantize_kv, k, v, lengths, shape, ks, vs)


def _quantize_kv(lib, stream, k, v, lengths, shape, ks, vs):
    B, L, H, D = shape
    nb = -(-L // KV8_TOKENS)
    device, T, n = k.device, KV8_TOKENS, nb * KV8_TOKENS * D
    codes = _empty((B, H, nb, T, D), (H * n, n, T * D, D, 1), dtype=torch.float8_e4m3fn, device=device)
    values = _empty((B, H, nb, D, T), (H * n, n, T * D, T, 1), dtype=torch.float8_e4m3fn, device=device)
    k_scale = _empty((B, H, nb), (H * nb, nb, 1), dtype=torch.float32, device=device)
    v_scale = torch.empty_like(k_scale)
    desc = _Kv8Desc(B, H, L, D, codes.data_ptr(), values.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                    lengths.data_ptr() if lengths is not None else None)
    code = lib.icsa_kv8_quantize(ctypes.byref(desc), k.data_ptr(), v.data_ptr(), _DT[k.dtype], _strides(shape, ks),
                                 _strides(shape, vs), stream)
    if code:
        _capi.check(code, "icsa_kv8_quantize")
    c = object.__new__(Kv8Cache)        # its tensors are as the constructor wants them
    c.__dict__.update(k=codes, v=values, k_scale=k_scale, v_scale=v_scale, L=L, lengths=lengths)
    return c


def kv8_dequantize(cache: Kv8Cache, dtype: torch.dtype = torch.bfloat16):
    """(k, v) [B, L, H, D], code * scale (exact in bf16); zero behind a length."""
    if dtype not in _DT:
        raise ValueError(f"kv8_dequantize: dtype {dtype}, expected bf16 or f32")
    return _on(_device("kv8_dequantize", cache.k), _dequantize_kv, cache, dtype)


def _dequantize_kv(lib, stream, cache, dtype):
    (B, H, _, _, D), L, device = cache.k.shape, cache.L, cache.k.device
    k = _empty((B, L, H, D), (L * H * D, H * D, D, 1), dtype=dtype, device=device)
    v = torch.empty_like(k)
    code = lib.icsa_kv8_dequantize(ctypes.byref(cache._desc()), k.data_ptr(), v.data_ptr(), _DT[dtype], stream)
    if code:
        _capi.check(code, "icsa_kv8_dequantize")
    return k, v


def kv8_attention(q: torch.Tensor, cache: Kv8Cache) -> torch.Tensor:
    """softmax(q k^T / sqrt(D)) v over the valid tokens of the cache, bf16
    [B, Lq, Hq, D]; zero for a sequence of length 0.  q: bf16 [B, Lq, Hq, D],
    Hq a multiple of the cache's heads (query heads h of one group share
    cache head h // (Hq / H))."""
    _no_gradient("kv8_attention", q)
    index = _device("kv8_attention", q, cache.k)
    B, H, _, _, D = cache.k.shape
    shape = q.shape
    if len(shape) != 4 or q.dtype != torch.bfloat16 or shape[0] != B or shape[3] != D or shape[2] % H or not shape[2]:
        raise ValueError(f"kv8_attention: q must be bf16 [{B}, Lq, a multiple of {H}, {D}], got {q.dtype} {tuple(shape)}")
    return _on(index, _attention, index, q, shape, cache, H)


@functools.lru_cache(maxsize=1024)
def _attention_workspace(index, B, H, L, D, Lq, Hq, strided=False):
    """Workspace bytes of icsa_kv8_attention; strided: for a q that is not rows,
    None where that would take another kernel.  The device is current."""
    desc = ctypes.byref(_Kv8Desc(B, H, L, D))
    size = _lib.icsa_kv8_attention_workspace_size(desc, Lq, Hq)
    if strided and size != _lib.icsa_kv8_attention_strided_workspace_size(desc, Lq, Hq):
        return None
    return size


def _attention(lib, stream, index, q, shape, cache, H):
    B, Lq, Hq, D = shape
    out = _empty((B, Lq, Hq, D), (Lq * Hq * D, Hq * D, D, 1), dtype=torch.bfloat16, device=q.device)
    if Lq == 0:
        return out
    sb, st, sh, sd = q.stride()
    # an axis of one has any stride
    sh = sh if Hq > 1 else D
    st = st if Lq > 1 else Hq * D
    sb = sb if B > 1 else Lq * st
    size = None
    if sd == 1 and not (sb | st | sh) % 8 and q.data_ptr() % 16 == 0:
        # rows of a wider GEMM output are taken as they are, other strides wherever the kernel for these sizes does
        strided = sh != D or st < Hq * D or sb != Lq * st
        size = _attention_workspace(index, B, H, cache.L, D, Lq, Hq, strided)
    if size is None:
        q = q.clone(memory_format=torch.contiguous_format)
        sb, st, sh = Lq * Hq * D, Hq * D, D
        size = _attention_workspace(index, B, H, cache.L, D, Lq, Hq)
    ws, ptr = _bytes(out, size)
    code = lib.icsa_kv8_attention(ctypes.byref(cache._desc()), q.data_ptr(), _int64x3(sb, st, sh), out.data_ptr(),
                                  Lq, Hq, ptr, size, stream)
    if code:
        _capi.check(code, "icsa_kv8_attention")
    return out
