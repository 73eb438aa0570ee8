"""Python binding of the gfx950 C ABI (include/quixicore_hip.h) over ctypes.

Tensors are torch tensors on the GPU; their data pointers and the current
torch stream are handed to the C ABI unchanged.  There is no CPU fallback:
importing this module without the built library raises, and every call runs
a HIP kernel.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_DIR = os.path.dirname(HERE)
LIB_PATH = os.path.join(PKG_DIR, "lib", "libquixicore_hip.so")
SYNTH_PATH = os.path.join(HERE, "libqcsynth.so")

Q8_0, Q4_0 = 0, 1
BLOCK_BYTES = {Q8_0: 34, Q4_0: 18}
STATUS = {0: "kOk", 1: "kInvalidShape", 2: "kUnsupportedFormat", 3: "kInvalidArgument",
          4: "kOutOfMemory", 5: "kDeviceError"}

if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} is not built; run `make -C quixicore-cpu_amd` (or __graft_entry__.build())")

_P = ctypes.c_void_p
_LL = ctypes.c_longlong
_I = ctypes.c_int

lib = ctypes.CDLL(LIB_PATH)

_SIGS = {
    "qc_hip_version": ([], ctypes.c_char_p),
    "qc_hip_last_error": ([], ctypes.c_char_p),
    "qc_hip_qgemv_packed_size": ([_I, _LL, _LL, ctypes.POINTER(ctypes.c_size_t)], _I),
    "qc_hip_qgemv_pack": ([_I, _P, _LL, _LL, _P, _P, _P], _I),
    "qc_hip_qgemv_unpack": ([_I, _P, _LL, _LL, _P, _P], _I),
    "qc_hip_qgemv": ([_I, _P, _P, _P, _LL, _LL, _P], _I),
    "qc_hip_qgemm": ([_I, _P, _P, _P, _LL, _LL, _LL, _P], _I),
    "qc_hip_qgemm_noalloc": ([_I, _P, _P, _P, _LL, _LL, _LL, _P], _I),
    "qc_hip_qgemv_w8a8": ([_I, _P, _P, _P, _LL, _LL, _P, _P], _I),
    "qc_hip_qgemv_up_gate": ([_I, _P, _P, _P, _P, _P, _LL, _LL, _P], _I),
    "qc_hip_qgemv_up_gate_activation": ([_I, _P, _P, _P, _P, _LL, _LL, _I, _P], _I),
    "qc_hip_qgemv_qkv": ([_I, _P, _P, _P, _P, _P, _P, _P, _LL, _LL, _LL, _P], _I),
    "qc_hip_cint8_project": ([_I, _P, _I, _P, _I, _LL, _P, _P, _P, _I, _P, _P, _LL, _P], _I),
    "qc_hip_qgemv_qkv_rope_kv": ([_I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _LL, _LL, _LL, _LL,
                                  _LL, _LL, _I, _I, _P], _I),
    "qc_hip_qgemv_w8a8_packed_size": ([_I, _LL, _LL, _P], _I),
    "qc_hip_qgemv_w8a8_variant": ([_I], ctypes.c_char_p),
    "qc_hip_quantize_int8": ([_P, _P, _P, _LL, _LL, _LL, _P, _P], _I),
    "qc_hip_int8_gemm": ([_P, _P, _P, _P, _P, _P, _P, _LL, _LL, _LL, _I, _P, _P], _I),
    "qc_hip_qgemm_w8a8": ([_P, _P, _P, _P, _P, _LL, _LL, _LL, _P, _P], _I),
    "qc_hip_int8_gemm_i32": ([_P, _P, _P, _LL, _LL, _LL, _P], _I),
    "qc_hip_nonfinite_scan": ([_P, _LL, _P, _P], _I),
    "qc_hip_qgemv_variant": ([_I], ctypes.c_char_p),
    "qc_hip_int8_gemm_variant": ([], ctypes.c_char_p),
    "qc_hip_set_gemv_rows_per_wave": ([_I], _I),
    "qc_hip_set_int8_gemm_route": ([_I], _I),
    "qc_hip_set_qgemm_plan": ([_I, _I], _I),
    "qc_hip_rms_norm_add_quant_int8": ([_P, _P, _P, _P, _P, _P, _LL, _LL, ctypes.c_float, _LL,
                                        _P, _P], _I),
    "qc_hip_quantize_int8_asymmetric": ([_P, _P, _P, _P, _LL, _LL, _P, _P], _I),
    "qc_hip_dequantize_int8_asymmetric": ([_P, _P, _P, _P, _LL, _LL, _P], _I),
    "qc_hip_set_norm_sequential_sum": ([_I], _I),
    "qc_hip_set_qgemm_panel": ([_I], _I),
    "qc_hip_set_qgemm_rows": ([_I], _I),
    "qc_hip_set_qgemm_fold": ([_I], _I),
    "qc_hip_set_cint8_dot": ([_I], _I),
    "qc_hip_stream_read": ([_P, _LL, _P, _I, _P], _I),
    "qc_hip_cint8_dequantize": ([_P, _P, _P, _P], _I),
    "qc_hip_cint8_quantized_gemm": ([_P, _P, _P, _P, _P], _I),
    "qc_hip_storage_to_f32": ([_P, _I, _LL, _P, _P], _I),
    "qc_hip_rope_table": ([_P, _P, _LL, _LL, _LL, ctypes.c_double, _P, _P], _I),
    "qc_hip_rope": ([_P, _P, _I, _LL, _LL, _LL, _LL, _LL, _LL, _LL, _LL, _P, _P, _P, _LL, _I, _P,
                     _P], _I),
    "qc_hip_kv8_append": ([_P, _P, _P, _LL, _P, _LL, _I, _P, _P], _I),
    "qc_hip_kv8_gather": ([_P, _P, _P, _LL, _P, _LL, _I, _I, _P, _P], _I),
    "qc_hip_kv8_attention": ([_P, _P, _P, _LL, _P, _LL, _I, _LL, ctypes.c_float, _I, _LL, _P, _P],
                             _I),
    "qc_hip_kv8_rope_append": ([_P, _P, _P, _LL, _P, _LL, _LL, _P, _LL, _P, _LL, _I, _P, _P, _P, _LL,
                                _LL, _I, _P, _P], _I),
    "qc_hip_kv8_tree_attention": ([_P, _P, _P, _LL, _P, _LL, _I, _LL, ctypes.c_float, _P, _LL, _P,
                                   _LL, _P, _P], _I),
    "qc_hip_kv8_keep": ([_P, _P, _P, _LL, _P, _P, _P, _P], _I),
    "qc_hip_mxfp4_moe": ([_P, _P, _LL, _P, _LL, _P, _LL, _I, _LL, _LL, _I, ctypes.c_float, _I, _P, _P,
                          _P], _I),
    "qc_hip_quantize_mxfp4": ([_P, _I, _LL, _P, _P, _LL, _LL, _P, _P], _I),
    "qc_hip_dequantize_mxfp4": ([_P, _P, _P, _I, _LL, _LL, _P], _I),
    "qc_hip_set_kv8_attention_route": ([_I], _I),
    "qc_hip_set_mxfp4_gemm_route": ([_I], _I),
    "qc_hip_mxfp4_gemm": ([_P, _P, _P, _P, _P, _I, _LL, _LL, _LL, _P], _I),
}
for _name, (_args, _res) in _SIGS.items():
    _fn = getattr(lib, _name)
    _fn.argtypes = _args
    _fn.restype = _res

EXPORTED = tuple(_SIGS)


class QcError(RuntimeError):
    def __init__(self, status, what):
        detail = lib.qc_hip_last_error().decode()
        super().__init__(f"{what}: {STATUS.get(status, status)}" + (f" ({detail})" if detail else ""))
        self.status = status


# A pointer argument is declared c_void_p, so a plain int is passed as it is; a
# one-projection call spends several us here, as long as its kernel, when every
# pointer is wrapped and the current stream looked up as a Stream object.
def _ptr(t):
    return None if t is None else t.data_ptr()


_raw_stream = None   # current stream handle of the current device


def _stream(stream):
    if stream is not None:
        return stream
    global _raw_stream
    if _raw_stream is None:
        import torch
        torch.cuda.current_stream()   # initialises the device
        c = torch._C
        if hasattr(c, "_cuda_getCurrentRawStream") and hasattr(c, "_cuda_getDevice"):
            raw, device = c._cuda_getCurrentRawStream, c._cuda_getDevice
            _raw_stream = lambda: raw(device())
        else:
            _raw_stream = lambda: torch.cuda.current_stream().cuda_stream
    return _raw_stream()


def _check(status, what):
    if status != 0:
        raise QcError(status, what)


def packed_size(fmt, n, k):
    size = ctypes.c_size_t(0)
    st = lib.qc_hip_qgemv_packed_size(fmt, n, k, ctypes.byref(size))
    return st, size.value


# Raw entry points: return the status integer (tests exercise error paths).
def qgemv_raw(fmt, packed, x, y, n, k, stream=None):
    return lib.qc_hip_qgemv(fmt, _ptr(packed), _ptr(x), _ptr(y), n, k, _stream(stream))


def qgemv_w8a8_raw(fmt, packed, x, y, n, k, dev_status=None, stream=None):
    return lib.qc_hip_qgemv_w8a8(fmt, _ptr(packed), _ptr(x), _ptr(y), n, k, _ptr(dev_status),
                                 _stream(stream))


def qgemv_up_gate_raw(fmt, p_up, p_gate, x, up, gate, n, k, stream=None):
    return lib.qc_hip_qgemv_up_gate(fmt, _ptr(p_up), _ptr(p_gate), _ptr(x), _ptr(up), _ptr(gate),
                                    n, k, _stream(stream))


def qgemv_up_gate_activation_raw(fmt, p_up, p_gate, x, out, n, k, gelu_tanh=True, stream=None):
    return lib.qc_hip_qgemv_up_gate_activation(fmt, _ptr(p_up), _ptr(p_gate), _ptr(x), _ptr(out),
                                               n, k, int(bool(gelu_tanh)), _stream(stream))


def qgemv_qkv_raw(fmt, pq, pk, pv, x, q, k_out, v_out, query_dim, kv_dim, input_dim, stream=None):
    return lib.qc_hip_qgemv_qkv(fmt, _ptr(pq), _ptr(pk), _ptr(pv), _ptr(x), _ptr(q), _ptr(k_out),
                                _ptr(v_out), query_dim, kv_dim, input_dim, _stream(stream))


def qgemv_qkv_rope_kv_raw(fmt, pq, pk, pv, x, cosine, sine, q, key_cache, value_cache,
                         query_heads, kv_heads, head_dim, input_dim, slots, max_position,
                         position, slot, stream=None):
    return lib.qc_hip_qgemv_qkv_rope_kv(fmt, _ptr(pq), _ptr(pk), _ptr(pv), _ptr(x), _ptr(cosine),
                                        _ptr(sine), _ptr(q), _ptr(key_cache), _ptr(value_cache),
                                        query_heads, kv_heads, head_dim, input_dim, slots,
                                        max_position, position, slot, _stream(stream))


class CInt8Weights(ctypes.Structure):
    """qc_cint8_weights (include/quixicore_hip.h)."""
    _fields_ = [("codes", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("zero_points", ctypes.c_void_p), ("rows", ctypes.c_longlong),
                ("cols", ctypes.c_longlong), ("groups", ctypes.c_longlong)]


STORAGE = {"f32": 0, "f16": 1, "bf16": 2}


def cint8_weights(codes, scales, zero_points, rows, cols, groups):
    """A qc_cint8_weights over device tensors; the caller keeps the tensors
    alive while the struct is in use (it holds raw pointers)."""
    return CInt8Weights(None if codes is None else codes.data_ptr(),
                        None if scales is None else scales.data_ptr(),
                        None if zero_points is None else zero_points.data_ptr(), rows, cols, groups)


def cint8_project_raw(mode, weights, x, x_type, m, ys, y_types, bias=None, activation=0,
                      rope_cos=None, rope_sin=None, head_dim=0, stream=None):
    """qc_hip_cint8_project: weights is a list of CInt8Weights, ys a list of
    output tensors (or None), types as STORAGE ids."""
    arr = (CInt8Weights * max(len(weights), 1))(*weights)
    yp = (ctypes.c_void_p * max(len(ys), 1))(*[None if y is None else y.data_ptr() for y in ys])
    yt = (ctypes.c_int * max(len(y_types), 1))(*y_types)
    return lib.qc_hip_cint8_project(mode, arr, len(weights), _ptr(x), x_type, m, yp, yt,
                                    _ptr(bias), activation, _ptr(rope_cos), _ptr(rope_sin),
                                    head_dim, _stream(stream))


def cint8_dequantize_raw(weights, out, group_index=None, stream=None):
    """qc_hip_cint8_dequantize: weights a CInt8Weights, out f32 [rows][cols]."""
    return lib.qc_hip_cint8_dequantize(ctypes.byref(weights), _ptr(group_index), _ptr(out),
                                       _stream(stream))


def cint8_quantized_gemm_raw(weights, activation, y, a_int_zero_points=None, stream=None):
    """qc_hip_cint8_quantized_gemm: weights / activation CInt8Weights, y f32 [m][n]."""
    return lib.qc_hip_cint8_quantized_gemm(ctypes.byref(weights), ctypes.byref(activation),
                                           _ptr(a_int_zero_points), _ptr(y), _stream(stream))


def storage_to_f32_raw(x, x_type, count, out, stream=None):
    """qc_hip_storage_to_f32: x of STORAGE type x_type, out f32 [count]."""
    return lib.qc_hip_storage_to_f32(_ptr(x), x_type, count, _ptr(out), _stream(stream))


def qgemm_raw(fmt, packed, x, y, m, n, k, stream=None):
    return lib.qc_hip_qgemm(fmt, _ptr(packed), _ptr(x), _ptr(y), m, n, k, _stream(stream))


def qgemm_noalloc_raw(fmt, packed, x, y, m, n, k, stream=None):
    return lib.qc_hip_qgemm_noalloc(fmt, _ptr(packed), _ptr(x), _ptr(y), m, n, k,
                                    _stream(stream))


def pack_raw(fmt, w, packed, n, k, dev_status=None, stream=None):
    return lib.qc_hip_qgemv_pack(fmt, _ptr(w), n, k, _ptr(packed), _ptr(dev_status),
                                 _stream(stream))


def unpack_raw(fmt, packed, w, n, k, stream=None):
    return lib.qc_hip_qgemv_unpack(fmt, _ptr(packed), n, k, _ptr(w), _stream(stream))


def quantize_int8_raw(x, codes, scales, rows, dim, group_size=0, dev_status=None, stream=None):
    return lib.qc_hip_quantize_int8(_ptr(x), _ptr(codes), _ptr(scales), rows, dim, group_size,
                                    _ptr(dev_status), _stream(stream))


def rms_norm_add_quant_int8_raw(x, residual, weight, codes, residual_out, scales, rows, hidden,
                                eps=1e-5, group_size=0, dev_status=None, stream=None):
    return lib.qc_hip_rms_norm_add_quant_int8(_ptr(x), _ptr(residual), _ptr(weight), _ptr(codes),
                                              _ptr(residual_out), _ptr(scales), rows, hidden, eps,
                                              group_size, _ptr(dev_status), _stream(stream))


def quantize_int8_asymmetric_raw(x, codes, scales, zero_points, rows, dim, dev_status=None,
                                 stream=None):
    return lib.qc_hip_quantize_int8_asymmetric(_ptr(x), _ptr(codes), _ptr(scales),
                                               _ptr(zero_points), rows, dim, _ptr(dev_status),
                                               _stream(stream))


def dequantize_int8_asymmetric_raw(codes, scales, zero_points, out, rows, dim, stream=None):
    return lib.qc_hip_dequantize_int8_asymmetric(_ptr(codes), _ptr(scales), _ptr(zero_points),
                                                 _ptr(out), rows, dim, _stream(stream))


def int8_gemm_raw(w, x, ws, as_, row_sum, zp, y, m, n, k, asymmetric=False, dev_status=None,
                  stream=None):
    return lib.qc_hip_int8_gemm(_ptr(w), _ptr(x), _ptr(ws), _ptr(as_), _ptr(row_sum), _ptr(zp),
                                _ptr(y), m, n, k, int(asymmetric), _ptr(dev_status),
                                _stream(stream))


def int8_gemm_i32_raw(w, x, acc, m, n, k, stream=None):
    return lib.qc_hip_int8_gemm_i32(_ptr(w), _ptr(x), _ptr(acc), m, n, k, _stream(stream))


# Tensor-level helpers (torch GPU tensors in, new tensors out).
def pack(fmt, w):
    import torch
    n, k = w.shape
    st, size = packed_size(fmt, n, k)
    _check(st, "qgemv_packed_size")
    out = torch.empty(size, dtype=torch.uint8, device=w.device)
    _check(pack_raw(fmt, w, out, n, k), "qgemv_pack")
    return out


def unpack(fmt, packed, n, k):
    import torch
    out = torch.empty((n, k), dtype=torch.float32, device=packed.device)
    _check(unpack_raw(fmt, packed, out, n, k), "qgemv_unpack")
    return out


def qgemv(fmt, packed, x, n, k, y=None):
    import torch
    if y is None:
        y = torch.empty(n, dtype=torch.float32, device=x.device)
    _check(qgemv_raw(fmt, packed, x, y, n, k), "qgemv")
    return y


def qgemv_w8a8(fmt, packed, x, n, k, y=None):
    import torch
    if y is None:
        y = torch.empty(n, dtype=torch.float32, device=x.device)
    _check(qgemv_w8a8_raw(fmt, packed, x, y, n, k), "qgemv_w8a8")
    return y


def qgemm(fmt, packed, x, n, k, y=None):
    import torch
    m = x.shape[0]
    if y is None:
        y = torch.empty((m, n), dtype=torch.float32, device=x.device)
    _check(qgemm_raw(fmt, packed, x, y, m, n, k), "qgemm")
    return y


def quantize_int8(x, group_size=0, dev_status=None):
    import torch
    rows, dim = x.shape
    g = dim if group_size == 0 else group_size
    codes = torch.empty((rows, dim), dtype=torch.int8, device=x.device)
    scales = torch.empty((rows, dim // g), dtype=torch.float32, device=x.device)
    _check(quantize_int8_raw(x, codes, scales, rows, dim, group_size, dev_status),
           "quantize_int8")
    return codes, scales


def int8_gemm(w, x, ws, as_, row_sum=None, zp=None, asymmetric=False, dev_status=None, y=None):
    import torch
    m, k = x.shape
    n = w.shape[0]
    if y is None:
        y = torch.empty((m, n), dtype=torch.float32, device=x.device)
    _check(int8_gemm_raw(w, x, ws, as_, row_sum, zp, y, m, n, k, asymmetric, dev_status),
           "int8_gemm")
    return y


def int8_gemm_i32(w, x):
    import torch
    m, k = x.shape
    n = w.shape[0]
    acc = torch.empty((m, n), dtype=torch.int32, device=x.device)
    _check(int8_gemm_i32_raw(w, x, acc, m, n, k), "int8_gemm_i32")
    return acc


# Rotary positions, the 8-bit key/value cache and MXFP4 (include/quixicore_hip.h).
# These helpers check what the C ABI cannot see: types, shapes, contiguity, and
# that tensors lie on the current device, whose stream the call goes to.
ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "turns": 3, "yarn": 4}


class RopeScaling(ctypes.Structure):
    """qc_rope_scaling (include/quixicore_hip.h)."""
    _fields_ = [("kind", ctypes.c_int), ("factor", ctypes.c_double),
                ("original_positions", ctypes.c_double), ("low_turns", ctypes.c_double),
                ("high_turns", ctypes.c_double), ("magnitude", ctypes.c_double)]


# The checks run on every call beside kernels of a few us: no tensor is looked at twice,
# and get_device() stands for comparing device objects.
_storage_ids = None   # torch dtype -> STORAGE id
_device = None        # index of the current device
_types = None         # (int32, uint8, float32)


def _start():
    global _storage_ids, _device, _types
    import torch
    torch.cuda.current_stream()   # initialises the device
    _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    _storage_ids = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    _types = (torch.int32, torch.uint8, torch.float32)


def _storage(t):
    """STORAGE id of a tensor's type."""
    if _storage_ids is None:
        _start()
    st = _storage_ids.get(t.dtype)
    if st is None:
        raise TypeError(f"f32, f16 or bf16 tensors: got {t.dtype}")
    return st


def _here(*tensors):
    """The tensors lie on the current device."""
    if _device is None:
        _start()
    now = _device()
    for t in tensors:
        if t.get_device() != now:
            raise ValueError(f"a tensor on {t.device}: the current device is cuda:{now}")


def _flat(what, dtype, *tensors):
    """Contiguous tensors of one type on the current device."""
    now = _device()
    for t in tensors:
        if t.dtype is not dtype or not t.is_contiguous() or t.get_device() != now:
            raise ValueError(f"{what}: contiguous {dtype} tensors on cuda:{now}")


def _status(dev_status):
    if dev_status is None:
        return None
    if dev_status.dtype is not _types[0] or dev_status.get_device() != _device():
        _flat("dev_status", _types[0], dev_status)
    return dev_status.data_ptr()


def _rows(what, t, heads, head_dim):
    """Row stride of token rows [tokens][heads * head_dim] or [tokens][heads][head_dim]."""
    shape, stride = t.shape, t.stride()
    n = len(shape)
    if n == 3:
        ok = shape[1] == heads and shape[2] == head_dim and stride[2] == 1 and (
            heads == 1 or stride[1] == head_dim)
    else:
        ok = n == 2 and shape[1] == heads * head_dim and stride[1] == 1
    if not ok:
        raise ValueError(f"{what}: rows of {heads} x {head_dim} elements side by side, got "
                         f"{tuple(shape)} with strides {stride}")
    return stride[0] if shape[0] > 1 else heads * head_dim


def rope_table(positions, rotary_dim, base=10000.0, scaling="none", factor=1.0,
               original_positions=0.0, low_turns=1.0, high_turns=32.0, magnitude=1.0,
               first_position=0):
    """(cosine, sine), f32 [positions][rotary_dim / 2], on the current device; scaling one of
    ROPE_SCALING (see qc_rope_scaling)."""
    import torch
    cosine = torch.empty((positions, rotary_dim // 2), dtype=torch.float32, device="cuda")
    sine = torch.empty_like(cosine)
    sc = RopeScaling(ROPE_SCALING[scaling], factor, original_positions, low_turns, high_turns,
                     magnitude)
    _check(lib.qc_hip_rope_table(_ptr(cosine), _ptr(sine), first_position, positions, rotary_dim,
                                 base, ctypes.addressof(sc), _stream(None)), "rope_table")
    return cosine, sine


def rope(x, cosine, sine, positions, interleaved=False, out=None, dev_status=None):
    """x [tokens][heads][head_dim] (token-major, head-major or strided) with the first 2 *
    cosine.shape[1] elements of every head rotated; out may be x.  Tokens at position -1 are
    left as they were (zeros in a new tensor)."""
    st = _storage(x)
    if x.dim() != 3 or x.stride(2) != 1:
        raise ValueError("rope: x is [tokens][heads][head_dim], elements side by side")
    if out is None:
        import torch
        out = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
    tokens, heads, head_dim = shape = x.shape
    xt, xh, _ = x.stride()
    yt, yh, side = out.stride()
    if out is not x and (side != 1 or out.shape != shape or out.dtype is not x.dtype):
        raise ValueError("rope: out is of x's shape and type")
    _here(x, out)
    _flat("rope tables", _types[2], cosine, sine)
    _flat("rope positions", _types[0], positions)
    most, half = table = cosine.shape
    if sine.shape != table or positions.numel() != tokens:
        raise ValueError("rope: tables [max_position][rotary_dim / 2], a position for each token")
    _check(lib.qc_hip_rope(x.data_ptr(), out.data_ptr(), st, tokens, heads, head_dim, 2 * half, xt,
                           xh, yt, yh, cosine.data_ptr(), sine.data_ptr(), positions.data_ptr(),
                           most, 1 if interleaved else 0, _status(dev_status), _stream(None)), "rope")
    return out


class Kv8Cache(ctypes.Structure):
    """qc_kv8_cache over int8 codes [pages][kv_heads][page_tokens][head_dim] and f32 scales
    [pages][kv_heads]; keeps the tensors alive."""
    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_longlong), ("kv_heads", ctypes.c_longlong),
                ("page_tokens", ctypes.c_longlong), ("head_dim", ctypes.c_longlong)]

    def __init__(self, k_codes, v_codes, k_scales, v_scales):
        import torch
        _here(k_codes)
        _flat("cache codes", torch.int8, k_codes, v_codes)
        _flat("cache scales", torch.float32, k_scales, v_scales)
        if (k_codes.dim() != 4 or v_codes.shape != k_codes.shape
                or k_scales.shape != k_codes.shape[:2] or v_scales.shape != k_codes.shape[:2]):
            raise ValueError("codes [pages][kv_heads][page_tokens][head_dim], scales [pages][kv_heads]")
        self.tensors = (k_codes, v_codes, k_scales, v_scales)
        self.device = k_codes.get_device()
        super().__init__(*[t.data_ptr() for t in self.tensors], *k_codes.shape)


class Kv8Batch(ctypes.Structure):
    """qc_kv8_batch over int32 block_table [seqs][columns], seq_start [seqs + 1] and
    kv_len [seqs]; keeps the tensors alive."""
    _fields_ = [("block_table", ctypes.c_void_p), ("seq_start", ctypes.c_void_p),
                ("kv_len", ctypes.c_void_p), ("seqs", ctypes.c_longlong),
                ("columns", ctypes.c_longlong), ("tokens", ctypes.c_longlong),
                ("max_new", ctypes.c_longlong), ("max_kv", ctypes.c_longlong)]

    def __init__(self, block_table, seq_start, kv_len, tokens, max_new, max_kv):
        import torch
        _here(block_table)
        _flat("batch", torch.int32, block_table, seq_start, kv_len)
        seqs, columns = block_table.shape
        if seq_start.numel() != seqs + 1 or kv_len.numel() != seqs:
            raise ValueError("block_table [seqs][columns], seq_start [seqs + 1], kv_len [seqs]")
        self.tensors = (block_table, seq_start, kv_len)
        self.device = block_table.get_device()
        super().__init__(*[t.data_ptr() for t in self.tensors], seqs, columns, tokens, max_new,
                         max_kv)


def _kv8_here(cache, batch, *tensors):
    """Everything on the current device (types were checked when the handles were made)."""
    now = _device()
    if cache.device != now or batch.device != now:
        raise ValueError(f"a cache on cuda:{cache.device}, a batch on cuda:{batch.device}: the "
                         f"current device is cuda:{now}")
    for t in tensors:
        if t.get_device() != now:
            raise ValueError(f"a tensor on {t.device}: the current device is cuda:{now}")


def kv8_cache(pages, kv_heads, page_tokens, head_dim):
    """An empty cache (zeros) on the current device."""
    import torch
    shape = (pages, kv_heads, page_tokens, head_dim)
    codes = [torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, kv_heads), dtype=torch.float32, device="cuda") for _ in range(2)]
    return Kv8Cache(*codes, *scales)


def kv8_append(cache, batch, k, v, dev_status=None):
    """Writes the batch's new tokens' k and v ([tokens][kv_heads][head_dim] or flat rows)."""
    st = _storage(k)
    _kv8_here(cache, batch, k, v)
    tokens, heads, head_dim = batch.tokens, cache.kv_heads, cache.head_dim
    if v.dtype is not k.dtype or k.shape[0] != tokens or v.shape[0] != tokens:
        raise ValueError("kv8_append: k and v of one type, a row for each of the batch's tokens")
    _check(lib.qc_hip_kv8_append(ctypes.addressof(cache), ctypes.addressof(batch), k.data_ptr(),
                                 _rows("k", k, heads, head_dim), v.data_ptr(),
                                 _rows("v", v, heads, head_dim), st, _status(dev_status),
                                 _stream(None)), "kv8_append")


def kv8_gather(cache, batch, dtype=None, k=None, v=None, dev_status=None):
    """(k, v) [tokens][kv_heads][head_dim]: the values the cache holds for the batch's
    tokens.  Rows of no sequence are left as they were (zeros in new tensors)."""
    tokens, heads, head_dim = batch.tokens, cache.kv_heads, cache.head_dim
    rest = 0
    if k is None and v is None:
        import torch
        k, v = torch.empty((2, tokens, heads, head_dim), dtype=dtype or torch.float32,
                           device=cache.tensors[0].device).unbind()
        rest = 1
    elif k is None or v is None:
        import torch
        given = v if k is None else k
        new = torch.zeros((tokens, heads, head_dim), dtype=given.dtype, device=given.device)
        k, v = (new, v) if k is None else (k, new)
    st = _storage(k)
    _kv8_here(cache, batch, k, v)
    if v.dtype is not k.dtype or k.shape[0] != tokens or v.shape[0] != tokens:
        raise ValueError("kv8_gather: k and v of one type, a row for each of the batch's tokens")
    _check(lib.qc_hip_kv8_gather(ctypes.addressof(cache), ctypes.addressof(batch), k.data_ptr(),
                                 _rows("k", k, heads, head_dim), v.data_ptr(),
                                 _rows("v", v, heads, head_dim), st, rest, _status(dev_status),
                                 _stream(None)), "kv8_gather")
    return k, v


def kv8_attention(cache, batch, q, scale=None, causal=True, window=0, out=None, dev_status=None):
    """softmax(scale q k^T) v of the batch's tokens over the cache: q [tokens][heads][head_dim]
    (rows may be strided), scale 1 / sqrt(head_dim) by default.  Rows of no sequence are left as
    they were (zeros in a new tensor)."""
    st = _storage(q)
    head_dim, shape = cache.head_dim, q.shape
    if len(shape) != 3 or shape[0] != batch.tokens:
        raise ValueError("kv8_attention: q is [tokens][heads][head_dim], a row for each of the batch's tokens")
    heads = shape[1]
    if out is None:
        import torch
        out = torch.zeros(shape, dtype=q.dtype, device=q.device)
    elif out.shape != shape or out.dtype is not q.dtype:
        raise ValueError("kv8_attention: out is of q's shape and type")
    _kv8_here(cache, batch, q, out)
    if scale is None:
        scale = head_dim ** -0.5
    _check(lib.qc_hip_kv8_attention(ctypes.addressof(cache), ctypes.addressof(batch), q.data_ptr(),
                                    _rows("q", q, heads, head_dim), out.data_ptr(),
                                    _rows("out", out, heads, head_dim), st, heads, scale,
                                    1 if causal else 0, window, _status(dev_status), _stream(None)),
           "kv8_attention")
    return out


def kv8_rope_append(cache, batch, q, k, v, cosine, sine, positions=None, interleaved=False, out=None,
                    dev_status=None):
    """Writes the batch's new tokens' k and v ([tokens][kv_heads][head_dim] or flat rows) into the
    cache, k turned by the tokens' positions (None: their places in their sequences), and returns q
    ([tokens][heads][head_dim], rows may be strided; None: no queries) turned likewise; out may be q.
    Rows of no sequence are left as they were (zeros in a new tensor)."""
    st = _storage(k)
    _kv8_here(cache, batch, k, v)
    tokens, kv_heads, head_dim = batch.tokens, cache.kv_heads, cache.head_dim
    if v.dtype is not k.dtype or k.shape[0] != tokens or v.shape[0] != tokens:
        raise ValueError("kv8_rope_append: k and v of one type, a row for each of the batch's tokens")
    _flat("rope tables", _types[2], cosine, sine)
    most, half = table = cosine.shape
    if sine.shape != table:
        raise ValueError("kv8_rope_append: tables [max_position][rotary_dim / 2]")
    at = None
    if positions is not None:
        _flat("rope positions", _types[0], positions)
        if positions.numel() != tokens:
            raise ValueError("kv8_rope_append: a position for each of the batch's tokens")
        at = positions.data_ptr()
    heads = qp = qs = op = os_ = 0
    if q is not None:
        shape = q.shape
        if len(shape) != 3 or shape[0] != tokens or q.dtype is not k.dtype:
            raise ValueError("kv8_rope_append: q is [tokens][heads][head_dim] of k's type, a row for each "
                             "of the batch's tokens")
        heads = shape[1]
        if out is None:
            import torch
            out = torch.zeros(shape, dtype=q.dtype, device=q.device)
        elif out.shape != shape or out.dtype is not q.dtype:
            raise ValueError("kv8_rope_append: out is of q's shape and type")
        _here(q, out)
        qp, op = q.data_ptr(), out.data_ptr()
        qs, os_ = _rows("q", q, heads, head_dim), _rows("out", out, heads, head_dim)
    _check(lib.qc_hip_kv8_rope_append(ctypes.addressof(cache), ctypes.addressof(batch), qp, qs, op, os_,
                                      heads, k.data_ptr(), _rows("k", k, kv_heads, head_dim),
                                      v.data_ptr(), _rows("v", v, kv_heads, head_dim), st,
                                      cosine.data_ptr(), sine.data_ptr(), at, most, 2 * half,
                                      1 if interleaved else 0, _status(dev_status), _stream(None)),
           "kv8_rope_append")
    return out


def kv8_tree_attention(cache, batch, q, mask, scale=None, positions=None, window=0, out=None,
                       dev_status=None):
    """kv8_attention for trees of drafted tokens: each of a sequence's new tokens sees what was there
    before them, and of them those whose bits are set in its row of mask (int32 [tokens][words], bit b %
    32 of word b / 32; itself too only by its bit).  With a window, positions (int32 [tokens]) are the
    rows' own and the window cuts what was there before."""
    st = _storage(q)
    head_dim, shape = cache.head_dim, q.shape
    if len(shape) != 3 or shape[0] != batch.tokens:
        raise ValueError("kv8_tree_attention: q is [tokens][heads][head_dim], a row for each of the "
                         "batch's tokens")
    heads = shape[1]
    if out is None:
        import torch
        out = torch.zeros(shape, dtype=q.dtype, device=q.device)
    elif out.shape != shape or out.dtype is not q.dtype:
        raise ValueError("kv8_tree_attention: out is of q's shape and type")
    _kv8_here(cache, batch, q, out)
    _flat("kv8_tree_attention's mask", _types[0], mask)
    if mask.dim() != 2 or mask.shape[0] != batch.tokens:
        raise ValueError("kv8_tree_attention: mask is [tokens][words]")
    at = None
    if positions is not None:
        _flat("kv8_tree_attention's positions", _types[0], positions)
        if positions.numel() != batch.tokens:
            raise ValueError("kv8_tree_attention: a position for each of the batch's tokens")
        at = positions.data_ptr()
    if scale is None:
        scale = head_dim ** -0.5
    _check(lib.qc_hip_kv8_tree_attention(ctypes.addressof(cache), ctypes.addressof(batch),
                                         q.data_ptr(), _rows("q", q, heads, head_dim),
                                         out.data_ptr(), _rows("out", out, heads, head_dim), st,
                                         heads, scale, mask.data_ptr(), mask.shape[1], at, window,
                                         _status(dev_status), _stream(None)), "kv8_tree_attention")
    return out


def kv8_keep(cache, batch, kept, count, out=None, dev_status=None):
    """The accepted ones of each sequence's new tokens (kept int32 [seqs][columns], count[seqs] ascending
    indexes of them) close up behind what was there before; returns the new lengths (int32 [seqs]).
    Sequences in error are left as they were, their lengths in a new tensor too (their kv_len)."""
    if _device is None:
        _start()
    _kv8_here(cache, batch)
    _flat("kv8_keep", _types[0], kept, count)
    if kept.dim() != 2 or kept.shape[0] != batch.seqs or count.numel() != batch.seqs:
        raise ValueError("kv8_keep: kept [seqs][columns], count [seqs]")
    if out is None:
        out = batch.tensors[2].clone()
    else:
        _flat("kv8_keep's lengths", _types[0], out)
        if out.numel() != batch.seqs:
            raise ValueError("kv8_keep: a length for each sequence")
    _check(lib.qc_hip_kv8_keep(ctypes.addressof(cache), ctypes.addressof(batch), kept.data_ptr(),
                               kept.shape[1], count.data_ptr(), out.data_ptr(), _status(dev_status),
                               _stream(None)), "kv8_keep")
    return out


class Mxfp4Moe(ctypes.Structure):
    """qc_mxfp4_moe over router [experts][dim], bias f32 [experts] or None, and uint8 codes
    [experts][rows][k / 2] and scales [experts][rows][k / 32] of gate_up (gate rows, then up rows) and
    down; keeps the tensors alive."""
    _fields_ = [("router", ctypes.c_void_p), ("router_bias", ctypes.c_void_p),
                ("gate_up_codes", ctypes.c_void_p), ("gate_up_scales", ctypes.c_void_p),
                ("down_codes", ctypes.c_void_p), ("down_scales", ctypes.c_void_p),
                ("router_type", ctypes.c_int), ("experts", ctypes.c_longlong),
                ("dim", ctypes.c_longlong), ("inter", ctypes.c_longlong)]

    def __init__(self, router, gate_up_codes, gate_up_scales, down_codes, down_scales, bias=None):
        import torch
        st = _storage(router)
        _here(router)
        _flat("router", router.dtype, router)
        _flat("expert weights", torch.uint8, gate_up_codes, gate_up_scales, down_codes, down_scales)
        experts, dim = router.shape
        inter = 2 * down_codes.shape[-1]
        for name, t, shape in (("gate_up codes", gate_up_codes, (experts, 2 * inter, dim // 2)),
                               ("gate_up scales", gate_up_scales, (experts, 2 * inter, dim // 32)),
                               ("down codes", down_codes, (experts, dim, inter // 2)),
                               ("down scales", down_scales, (experts, dim, inter // 32))):
            if t.shape != shape:
                raise ValueError(f"{name}: {shape} expected, got {tuple(t.shape)}")
        if bias is not None:
            _flat("router bias", torch.float32, bias)
            if bias.numel() != experts:
                raise ValueError("router bias: one for each expert")
        self.tensors = (router, bias, gate_up_codes, gate_up_scales, down_codes, down_scales)
        self.device = router.get_device()
        super().__init__(*[None if t is None else t.data_ptr() for t in self.tensors], st, experts, dim,
                         inter)


def mxfp4_moe(layer, x, top_k, normalize=True, weight_scale=1.0, gelu_tanh=False, residual=None,
              out=None):
    """(y, ids, weights) of a mixture-of-experts feed-forward: y [tokens][dim] = residual + sum_s
    weights[s] down_e(act(gate_e x) * up_e x), e = ids[s], over each token's top_k experts; x, residual
    and out: rows may be strided, out may be residual or x."""
    import torch
    st = _storage(x)
    if layer.device != _device():
        raise ValueError(f"experts on cuda:{layer.device}: the current device is cuda:{_device()}")
    _here(x)
    shape = x.shape
    if len(shape) != 2 or shape[1] != layer.dim or x.stride(1) != 1:
        raise ValueError("mxfp4_moe: x is [tokens][dim], elements side by side")
    tokens = shape[0]
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    for t in (out, residual):
        if t is None:
            continue
        _here(t)
        if t.shape != shape or t.dtype is not x.dtype or t.stride(1) != 1:
            raise ValueError("mxfp4_moe: out and residual are of x's shape and type, elements side by side")
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=x.device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=x.device)
    res, res_stride = (None, 0) if residual is None else (residual.data_ptr(), residual.stride(0))
    _check(lib.qc_hip_mxfp4_moe(ctypes.addressof(layer), x.data_ptr(), x.stride(0), res, res_stride,
                                out.data_ptr(), out.stride(0), st, tokens, top_k, 1 if normalize else 0,
                                weight_scale, 1 if gelu_tanh else 0, ids.data_ptr(), weights.data_ptr(),
                                _stream(None)), "mxfp4_moe")
    return out, ids, weights


def quantize_mxfp4(x, dev_status=None):
    """(codes [rows][dim / 2], scales [rows][dim / 32]) uint8 of x [rows][dim] (rows may be
    strided).  Where dev_status becomes 3, the blocks in error hold anything."""
    import torch
    st = _storage(x)
    _here(x)
    stride = x.stride()
    if len(stride) != 2 or stride[1] != 1:
        raise ValueError("quantize_mxfp4: x is [rows][dim], elements side by side")
    rows, dim = x.shape
    codes = torch.empty((rows, dim // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((rows, dim // 32), dtype=torch.uint8, device=x.device)
    _check(lib.qc_hip_quantize_mxfp4(x.data_ptr(), st, stride[0], codes.data_ptr(),
                                     scales.data_ptr(), rows, dim, _status(dev_status),
                                     _stream(None)), "quantize_mxfp4")
    return codes, scales


def dequantize_mxfp4(codes, scales, dtype=None, out=None):
    """The values [rows][dim] that MXFP4 codes and scales stand for."""
    if _device is None:
        _start()
    _flat("mxfp4", _types[1], codes, scales)
    rows, half = codes.shape
    if out is None:
        import torch
        out = torch.empty((rows, 2 * half), dtype=dtype or torch.float32, device=codes.device)
    elif out.shape != (rows, 2 * half) or not out.is_contiguous():
        raise ValueError("dequantize_mxfp4: out is [rows][dim], contiguous")
    else:
        _here(out)
    if scales.shape != (rows, half // 16):
        raise ValueError("dequantize_mxfp4: codes [rows][dim / 2], scales [rows][dim / 32]")
    _check(lib.qc_hip_dequantize_mxfp4(codes.data_ptr(), scales.data_ptr(), out.data_ptr(),
                                       _storage(out), rows, 2 * half, _stream(None)),
           "dequantize_mxfp4")
    return out


def mxfp4_gemm(w_codes, w_scales, x_codes, x_scales, dtype=None, y=None):
    """y [m][n] = x . w^T of MXFP4 matrices w [n][k] and x [m][k]."""
    if _device is None:
        _start()
    _flat("mxfp4_gemm", _types[1], w_codes, w_scales, x_codes, x_scales)
    n, half = w_codes.shape
    m, other = x_codes.shape
    blocks = half // 16
    if other != half or w_scales.shape != (n, blocks) or x_scales.shape != (m, blocks):
        raise ValueError("mxfp4_gemm: codes [rows][k / 2], scales [rows][k / 32]")
    if y is None:
        import torch
        y = torch.empty((m, n), dtype=dtype or torch.float32, device=x_codes.device)
    elif y.shape != (m, n) or not y.is_contiguous():
        raise ValueError("mxfp4_gemm: y is [m][n], contiguous")
    else:
        _here(y)
    _check(lib.qc_hip_mxfp4_gemm(w_codes.data_ptr(), w_scales.data_ptr(), x_codes.data_ptr(),
                                 x_scales.data_ptr(), y.data_ptr(), _storage(y), m, n, 2 * half,
                                 _stream(None)), "mxfp4_gemm")
    return y


def set_kv8_attention_route(route=0):
    """0 = from the sizes, 1 / 2 = the cache read directly for 16 / 32 rows a workgroup,
    3 = laid out for MFMA tiles first."""
    _check(lib.qc_hip_set_kv8_attention_route(route), "set_kv8_attention_route")


def set_mxfp4_gemm_route(route=0):
    """0 = from the sizes, 1..7 = tiles of 32 x 32 to 256 x 256 rows of w and x."""
    _check(lib.qc_hip_set_mxfp4_gemm_route(route), "set_mxfp4_gemm_route")


def set_gemv_rows_per_wave(rows):
    _check(lib.qc_hip_set_gemv_rows_per_wave(rows), "set_gemv_rows_per_wave")


def set_qgemm_plan(waves=0, stages=0):
    """Small-batch GEMM work split: waves per workgroup (4/8) and K stages
    per workgroup (1/2/4/8/16); 0 = from the shape."""
    _check(lib.qc_hip_set_qgemm_plan(waves, stages), "set_qgemm_plan")


def set_qgemm_panel(mode=0):
    """qgemm route for M >= 2: 0 = 2-D GEMM for M >= 33 (q4_0: 17), -1 = never,
    1 / 2 = always with one / two K ranges."""
    _check(lib.qc_hip_set_qgemm_panel(mode), "set_qgemm_panel")


def set_qgemm_rows(mode=0):
    """qgemm route for 2 <= M <= 8: 0 = by shape (exact-digit rows kernel for
    M = 2, and M <= 4 with N <= 8192, at K <= 4096), -1 = never (MFMA
    small-batch kernels), 1 = always."""
    _check(lib.qc_hip_set_qgemm_rows(mode), "set_qgemm_rows")


def set_cint8_dot(mode=0):
    """Canonical int8 projections: 0 = the row-plane route (int8 MFMA) for two
    or more activation rows (three, or five for groups of 32, with group
    scales), from some tens of rows the f16 MFMA route where it is the faster,
    else the exact digit-dot kernels where they apply; 1 = never either MFMA
    route; -1 = always the f32 kernel."""
    _check(lib.qc_hip_set_cint8_dot(mode), "set_cint8_dot")


def set_qgemm_fold(mode=0):
    """Digit-layout small-batch GEMM: 0 = builds its own digits where it can
    (no prep launch), -1 = always runs the prep launch (same bits)."""
    _check(lib.qc_hip_set_qgemm_fold(mode), "set_qgemm_fold")


def set_norm_sequential_sum(on):
    """Replay the element-order sum of squares for every row of
    rms_norm_add_quant_int8 (results are identical either way)."""
    _check(lib.qc_hip_set_norm_sequential_sum(int(bool(on))), "set_norm_sequential_sum")


def rms_norm_add_quant_int8(x, residual, weight, eps=1e-5, group_size=0, dev_status=None):
    """Returns (codes, residual_out, scales)."""
    import torch
    rows, hidden = x.shape
    g = hidden if group_size == 0 else group_size
    codes = torch.empty((rows, hidden), dtype=torch.int8, device=x.device)
    resid = torch.empty((rows, hidden), dtype=torch.float32, device=x.device)
    scales = torch.empty((rows, hidden // g), dtype=torch.float32, device=x.device)
    _check(rms_norm_add_quant_int8_raw(x, residual, weight, codes, resid, scales, rows, hidden,
                                       eps, group_size, dev_status), "rms_norm_add_quant_int8")
    return codes, resid, scales


def quantize_int8_asymmetric(x, dev_status=None):
    """Returns (codes, scales, zero_points)."""
    import torch
    rows, dim = x.shape
    codes = torch.empty((rows, dim), dtype=torch.int8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    zps = torch.empty(rows, dtype=torch.int32, device=x.device)
    _check(quantize_int8_asymmetric_raw(x, codes, scales, zps, rows, dim, dev_status),
           "quantize_int8_asymmetric")
    return codes, scales, zps


def set_int8_gemm_route(route):
    """0 = from the shape, 1 = full-line ring, 2 = 64-byte-step DMA,
    3 = register-staged, 4 = one thread per output."""
    _check(lib.qc_hip_set_int8_gemm_route(route), "set_int8_gemm_route")


def qgemv_variant(fmt):
    return lib.qc_hip_qgemv_variant(fmt).decode()


def qgemv_w8a8_variant(fmt):
    return lib.qc_hip_qgemv_w8a8_variant(fmt).decode()


def int8_gemm_variant():
    return lib.qc_hip_int8_gemm_variant().decode()


def version():
    return lib.qc_hip_version().decode()
