"""Loader of the MI355X decode-kernel library and the torch-facing op module.

Drop-in for the reference's ``runtime/ext.py`` (:9-20): ``load()`` returns an object with the six ops of the pybind
module ``decode_kernels`` (kernels/bindings.cpp:90-99) — same names, argument order, in-place/out-param conventions
and error behaviour (``RuntimeError`` for every TORCH_CHECK of kernels/bindings.cpp:18-88). Instead of a JIT nvcc
build it loads ``libdk_amd.so``, a hipcc-built C-ABI library (include/dk_amd.h), through ctypes; every op launches on
torch's current HIP stream, so the ops are capturable with ``torch.cuda.graph`` (a hipGraph on ROCm).

There is no CPU path: without the built library ``load()`` raises.
"""
import ctypes
import pathlib

import torch

PKG_DIR = pathlib.Path(__file__).resolve().parents[1]
LIB_PATH = PKG_DIR / "libdk_amd.so"
HEADER = PKG_DIR.parent / "include" / "dk_amd.h"

# Every exported entry point, with its ctypes signature (kept in the order of include/dk_amd.h).
_P, _I, _F, _Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
_L = ctypes.c_longlong
SIGNATURES = {
    "dk_last_error": ([], ctypes.c_char_p),
    "dk_runtime_version": ([], _I),
    "dk_gemv_w4a16": ([_I, _I, _I, _I, _P, _P, _P, _P, _I, _I, _I, _P], _I),
    "dk_gemv_w4a16_rmsnorm": ([_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _F, _P, _P, _I, _I, _I, _P], _I),
    "dk_gemv_w4a16_gate_up": ([_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _F, _P, _P, _I, _I, _I, _P], _I),
    "dk_gemv_w4a16_qkv_rope": ([_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _F, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I,
                                _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "dk_gemv_w4a16_attn": ([_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _I, _I, _I,
                            _P], _I),
    "dk_gemv_f16": ([_I, _I, _I, _P, _P, _P, _I, _I, _P], _I),
    "dk_gemv_f16_rmsnorm": ([_I, _I, _I, _P, _P, _P, _P, _F, _P, _P, _I, _I, _P], _I),
    "dk_gemm_w4a16": ([_P, _P, _P, _P, _I, _I, _I, _I, _I, _P], _I),
    "dk_gemm_w4a16_workspace_bytes": ([_I, _I, _I, _I, _I], _Z),
    "dk_gemm_w4a16_ws_splits": ([_I, _I, _I, _I, _I, _Z], _I),
    "dk_gemm_w4a16_kernel": ([_I, _I, _I, _I, _I, _I], ctypes.c_char_p),
    "dk_gemm_w4a16_ws": ([_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _Z, _P], _I),
    "dk_rope_append_rows": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "dk_rmsnorm_rows_parts": ([_P, _P, _I, ctypes.c_longlong, _P, _P, _P, _I, _I, _F, _P], _I),
    "dk_rmsnorm_rows": ([_P, _P, _I, _P, _P, _P, _P, _I, _I, _F, _P], _I),
    "dk_attention_prefill": ([_P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "dk_bw_read": ([_P, _Z, _P, _I, _I, _I, _I, _P], _I),
    "dk_paged_attention": ([_I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P], _I),
    "dk_paged_attention_split": ([_I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P], _I),
    "dk_paged_attention_noalloc": ([_I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "dk_paged_attention_noalloc_bytes": ([_I, _I, _I], _Z),
    "dk_attention_decode": ([_P, _P, _P, _I, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P],
                            _I),
    "dk_add_rmsnorm": ([_P, _P, _P, _P, _I, _F, _P], _I),
    "dk_swiglu": ([_P, _P, _I, _P], _I),
    "dk_rope_append": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "dk_argmax_advance": ([_P, _I, _P, _P, _P], _I),
    "dk_argmax_advance_split": ([_P, _I, _P, _P, _P, _P], _I),
    "dk_qk_norm_rope_append_rows": ([_P, _P, _P, _F, _P, _P, _P, _P, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _I, _I,
                                     _I, _P], _I),
    "dk_attention_tree_workspace_bytes": ([_I, _I, _I, _I, _I], _Z),
    "dk_attention_tree": ([_P, _L, _P, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z, _P], _I),
    "dk_token_logprobs_workspace_bytes": ([_I, _I, _I, _I], _Z),
    "dk_token_logprobs": ([_P, _I, _L, _P, _P, _P, _P, _P, _I, _I, _I, _P, _Z, _P], _I),
    "dk_tree_accept": ([_P, _P, _P, _L, _I, _P, _P, _I, _P, _I, _I, _I, _I, _I, _P, _P, _P, _P], _I),
    "dk_kv8_append_rows": ([_P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _P, _L, _I, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "dk_kv8_read": ([_P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P], _I),
    "dk_attention_window_workspace_bytes": ([_I, _I, _I, _I, _I, _I, _I, _I], _Z),
    "dk_attention_kv8_decode": ([_P, _P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z,
                                 _P], _I),
    "dk_attention_window": ([_P, _L, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z, _P],
                            _I),
    "dk_quantize_w4": ([_P, _P, _P, _I, _I, _I, _I, _P], _I),
}

_EXT = None


def open_library(path=LIB_PATH):
    """dlopen the library and bind every entry point (no GPU needed). torch is imported first so the library resolves
    libamdhip64 to the HIP runtime torch already loaded (one runtime per process)."""
    if not pathlib.Path(path).exists():
        raise RuntimeError(f"{path} is not built: run `make -C llm-decode-kernels_amd/csrc` "
                           "(or __graft_entry__.build()); there is no CPU fallback")
    lib = ctypes.CDLL(str(path))
    for name, (argtypes, restype) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    return lib


def _check_cuda(t, name):
    if not (t.is_cuda and t.is_contiguous()):
        raise RuntimeError(f"{name} must be a contiguous CUDA tensor")


def _check_dtype(t, dtype, name):
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


def _stream(t):
    """The handle of torch's current stream on t's device. As the raw handle (0.08 us): building the Stream object of
    torch.cuda.current_stream took 2.1 us of an op's 8.5 us of host time, more than half of the smallest GEMV's 2.6 us
    of GPU time again."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _check_all(what, device, *tensors):
    """(tensor or None, name, dtype) triples: contiguous CUDA tensors of their type, all on `device` (an index, -1 for none).
    Returns their addresses. One pass with three questions per tensor: asked one by one, with an address each later, they were
    2.5 us of an op's 9 us of host time."""
    ptrs = []
    for t, name, dtype in tensors:
        if t is None:
            ptrs.append(None)
            continue
        if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or device < 0:
            _check_cuda(t, name)
            if t.dtype != dtype:
                raise RuntimeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
            raise RuntimeError(f"{what}: {name} is on another device than the other tensors")
        ptrs.append(t.data_ptr())
    return ptrs


def _addresses(what, device, spec, *tensors):
    """_check_all with the names and types as one constant, ((name, dtype), ...): 0.5 us of host time less per call."""
    ptrs = []
    for t, (name, dtype) in zip(tensors, spec):
        if t is None:
            ptrs.append(None)
        elif t.dtype is dtype and t.get_device() == device and t.is_contiguous() and device >= 0:
            ptrs.append(t.data_ptr())
        else:
            _check_all(what, device, (t, name, dtype))
    return ptrs


def _workspace(what, device, t):
    """(address, bytes) of a workspace on `device`, of nothing for None."""
    if t is None:
        return None, 0
    if t.get_device() != device or not t.is_contiguous():
        _check_cuda(t, "workspace")
        raise RuntimeError(f"{what}: workspace is on another device than the other tensors")
    return t.data_ptr(), t.nbytes


def _ints(*sizes):
    """Sizes as C ints; ctypes would pass a larger one on without its high bits."""
    out = []
    for n in sizes:
        n = int(n)
        if not -0x80000000 <= n <= 0x7FFFFFFF:
            raise RuntimeError(f"a size of {n} does not fit 32 bits")
        out.append(n)
    return out


LOGITS_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
CACHE_DTYPES = {torch.float16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
KV8_BLOCK = 16  # tokens that share a scale


def _kv8_specs(*spec):
    """The spec of _addresses with the codes' type in the place of None, for either type."""
    return {d: tuple((n, d if t is None else t) for n, t in spec) for d in (torch.int8, torch.float8_e4m3fn)}


_CACHE_SPEC = (("bt", torch.int32), ("kc", None), ("vc", None), ("ks", torch.float32), ("vs", torch.float32))
_APPEND_SPEC = _kv8_specs(("qkv", torch.float16), ("cos_t", torch.float32), ("sin_t", torch.float32), ("pos", torch.int32),
                          *_CACHE_SPEC)
_READ_SPEC = _kv8_specs(*_CACHE_SPEC, ("k_out", torch.float16), ("v_out", torch.float16))
_KV8_SPEC = _kv8_specs(("pos", torch.int32), *_CACHE_SPEC, ("out", torch.float16))
_DECODE_SPEC = _kv8_specs(("qkv", torch.float16), ("cos_t", torch.float32), ("sin_t", torch.float32), ("pos", torch.int32),
                          *_CACHE_SPEC, ("out", torch.float16))
_WINDOW_SPEC = (("pos", torch.int32), ("bt", torch.int32), ("kc", torch.float16), ("vc", torch.float16), ("ks", torch.float32),
                ("vs", torch.float32), ("out", torch.float16))


class DecodeKernels:
    """The op module. Every method validates like the reference binding, then calls one C entry point."""

    def __init__(self, lib):
        self.lib = lib

    def _call(self, fn, *args):
        rc = fn(*args)
        if rc != 0:
            raise RuntimeError(self.lib.dk_last_error().decode() or f"decode kernel error {rc}")

    # kernels/bindings.cpp:27-38
    def gemv_w4a16(self, stage, R, warps, pf, packed, sz, x, y, group):
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (y, "y")):
            _check_cuda(t, n)
        N, K = packed.size(0), packed.size(1) * 8
        if K % 32 != 0 or K % group != 0:
            raise RuntimeError("K must be a multiple of 32 and of the group size")
        if group < 32:
            raise RuntimeError("group must be >= 32 (one uint4 never straddles a group)")
        if not (x.numel() == K and y.numel() == N and sz.size(0) == N and sz.size(1) == K // group):
            raise RuntimeError("gemv_w4a16: shape mismatch between packed, sz, x and y")
        _check_dtype(packed, torch.int32, "packed")
        for t, n in ((x, "x"), (y, "y"), (sz, "sz")):
            _check_dtype(t, torch.float16, n)
        self._call(self.lib.dk_gemv_w4a16, int(stage), int(R), int(warps), int(pf), packed.data_ptr(), sz.data_ptr(),
                   x.data_ptr(), y.data_ptr(), N, K, int(group), _stream(x))

    def _gemv_shape(self, packed, sz, y, K, group):
        N = packed.size(0)
        if packed.size(1) * 8 != K or y.numel() != N or sz.size(0) != N or sz.size(1) != K // group:
            raise RuntimeError("gemv: shape mismatch between packed, sz, x and y")
        _check_dtype(packed, torch.int32, "packed")
        _check_dtype(sz, torch.float16, "sz")
        _check_dtype(y, torch.float16, "y")
        return N

    # add_rmsnorm (kernels/bindings.cpp:64-72) fused into the gemv_w4a16 that follows it
    def gemv_w4a16_rmsnorm(self, stage, R, warps, pf, packed, sz, x, row, delta, norm_w, eps, x_out, y, group):
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (norm_w, "norm_w"), (y, "y")):
            _check_cuda(t, n)
        K = norm_w.numel()
        N = self._gemv_shape(packed, sz, y, K, group)
        if row is None and x.numel() != K:
            raise RuntimeError("gemv_w4a16_rmsnorm: x must hold K values (or be a [*, K] table with row)")
        if row is not None and (x.dim() != 2 or x.size(1) != K or row.dtype != torch.int64 or delta is not None):
            raise RuntimeError("gemv_w4a16_rmsnorm: row needs an int64 index into a [*, K] x and no delta")
        for t, n in ((x, "x"), (norm_w, "norm_w")):
            _check_dtype(t, torch.float16, n)
        ptr = lambda t: None if t is None else t.data_ptr()
        for t, n in ((delta, "delta"), (x_out, "x_out"), (row, "row")):
            if t is not None:
                _check_cuda(t, n)
        for t, n in ((delta, "delta"), (x_out, "x_out")):
            if t is not None and (t.numel() != K or t.dtype != torch.float16):
                raise RuntimeError(f"gemv_w4a16_rmsnorm: {n} must be fp16 [K]")
        self._call(self.lib.dk_gemv_w4a16_rmsnorm, int(stage), int(R), int(warps), int(pf), packed.data_ptr(),
                   sz.data_ptr(), x.data_ptr(), ptr(row), ptr(delta), norm_w.data_ptr(), float(eps), ptr(x_out),
                   y.data_ptr(), N, K, int(group), _stream(x))

    # gemv_w4a16 of the interleaved gate|up rows followed by swiglu (kernels/bindings.cpp:27-38, 74-79), one launch;
    # the input is x itself (norm_w None) or the residual + RMSNorm of gemv_w4a16_rmsnorm
    def gemv_w4a16_gate_up(self, stage, R, warps, pf, packed, sz, x, row, delta, norm_w, eps, x_out, act, group):
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (act, "act")):
            _check_cuda(t, n)
        K = packed.size(1) * 8
        N = packed.size(0)
        if N % 2 != 0 or act.numel() * 2 != N or sz.size(0) != N or sz.size(1) != K // group:
            raise RuntimeError("gemv_w4a16_gate_up: packed/sz need 2I interleaved rows and act I entries")
        _check_dtype(packed, torch.int32, "packed")
        _check_dtype(sz, torch.float16, "sz")
        _check_dtype(act, torch.float16, "act")
        _check_dtype(x, torch.float16, "x")
        if norm_w is None:
            if row is not None or delta is not None or x_out is not None or x.numel() != K:
                raise RuntimeError("gemv_w4a16_gate_up: without norm_w, x must hold K values and row/delta/x_out be None")
        else:
            _check_cuda(norm_w, "norm_w")
            _check_dtype(norm_w, torch.float16, "norm_w")
            if norm_w.numel() != K:
                raise RuntimeError("gemv_w4a16_gate_up: norm_w must hold K values")
            if row is None and x.numel() != K:
                raise RuntimeError("gemv_w4a16_gate_up: x must hold K values (or be a [*, K] table with row)")
            if row is not None and (x.dim() != 2 or x.size(1) != K or row.dtype != torch.int64 or delta is not None):
                raise RuntimeError("gemv_w4a16_gate_up: row needs an int64 index into a [*, K] x and no delta")
            for t, n in ((delta, "delta"), (x_out, "x_out"), (row, "row")):
                if t is not None:
                    _check_cuda(t, n)
            for t, n in ((delta, "delta"), (x_out, "x_out")):
                if t is not None and (t.numel() != K or t.dtype != torch.float16):
                    raise RuntimeError(f"gemv_w4a16_gate_up: {n} must be fp16 [K]")
        ptr = lambda t: None if t is None else t.data_ptr()
        self._call(self.lib.dk_gemv_w4a16_gate_up, int(stage), int(R), int(warps), int(pf), packed.data_ptr(),
                   sz.data_ptr(), x.data_ptr(), ptr(row), ptr(delta), ptr(norm_w), float(eps), ptr(x_out),
                   act.data_ptr(), N, K, int(group), _stream(x))

    # gemv_w4a16 of the qkv rows stored as per-head rotation pairs followed by rope_append (kernels/bindings.cpp
    # gemv_w4a16 then rope_append), one launch; the input is x itself (norm_w None) or the residual + RMSNorm input
    def gemv_w4a16_qkv_rope(self, stage, R, warps, pf, packed, sz, x, row, delta, norm_w, eps, x_out, qkv, cos_t,
                            sin_t, pos, bt, kc, vc, n_q, n_kv, group):
        """Shapes and dtypes are checked first, then that every tensor is a contiguous CUDA tensor, so no bad
        argument reaches the kernel."""
        what = "gemv_w4a16_qkv_rope"
        if kc.dim() != 4 or vc.shape != kc.shape or kc.size(1) != n_kv:
            raise RuntimeError(f"{what}: cache must be [pages, n_kv, P, head_dim] (kc and vc alike)")
        D = kc.size(3)
        K = packed.size(1) * 8
        N = (n_q + 2 * n_kv) * D
        if packed.dim() != 2 or packed.size(0) != N or qkv.numel() != N:
            raise RuntimeError(f"{what}: packed must hold (n_q + 2 n_kv) * head_dim rows and qkv as many values")
        if K % 32 != 0 or group < 32 or K % group != 0:
            raise RuntimeError(f"{what}: K must be a multiple of 32 and of the group size (>= 32)")
        self._gemv_shape(packed, sz, qkv, K, group)
        if cos_t.dim() != 2 or cos_t.size(1) * 2 != D or sin_t.shape != cos_t.shape:
            raise RuntimeError(f"{what}: cos_t and sin_t must both be [max_pos, head_dim / 2]")
        for t, n in ((x, "x"), (kc, "kc"), (vc, "vc")):
            _check_dtype(t, torch.float16, n)
        for t, n in ((cos_t, "cos_t"), (sin_t, "sin_t")):
            _check_dtype(t, torch.float32, n)
        for t, n in ((pos, "pos"), (bt, "bt")):
            _check_dtype(t, torch.int32, n)
        if pos.numel() < 1:
            raise RuntimeError(f"{what}: pos must hold the position (int32 [1])")
        if norm_w is None:
            if row is not None or delta is not None or x_out is not None or x.numel() != K:
                raise RuntimeError(f"{what}: without norm_w, x must hold K values and row/delta/x_out be None")
        else:
            if norm_w.numel() != K or norm_w.dtype != torch.float16:
                raise RuntimeError(f"{what}: norm_w must be fp16 [K]")
            if row is None and x.numel() != K:
                raise RuntimeError(f"{what}: x must hold K values (or be a [*, K] table with row)")
            if row is not None and (x.dim() != 2 or x.size(1) != K or row.dtype != torch.int64 or row.numel() != 1
                                    or delta is not None):
                raise RuntimeError(f"{what}: row needs one int64 index into a [*, K] x and no delta")
            for t, n in ((delta, "delta"), (x_out, "x_out")):
                if t is not None and (t.numel() != K or t.dtype != torch.float16):
                    raise RuntimeError(f"{what}: {n} must be fp16 [K]")
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (qkv, "qkv"), (cos_t, "cos_t"), (sin_t, "sin_t"),
                     (pos, "pos"), (bt, "bt"), (kc, "kc"), (vc, "vc"), (row, "row"), (delta, "delta"),
                     (norm_w, "norm_w"), (x_out, "x_out")):
            if t is not None:
                _check_cuda(t, n)
        ptr = lambda t: None if t is None else t.data_ptr()
        self._call(self.lib.dk_gemv_w4a16_qkv_rope, int(stage), int(R), int(warps), int(pf), packed.data_ptr(),
                   sz.data_ptr(), x.data_ptr(), ptr(row), ptr(delta), ptr(norm_w), float(eps), ptr(x_out),
                   qkv.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), pos.data_ptr(), bt.data_ptr(), kc.data_ptr(),
                   vc.data_ptr(), int(n_q), int(n_kv), D, kc.size(2), cos_t.size(0), kc.size(0), bt.numel(), K,
                   int(group), _stream(x))

    def _f16_shape(self, w, x, y, what):
        for t, n in ((w, "w"), (x, "x"), (y, "y")):
            _check_cuda(t, n)
            _check_dtype(t, torch.float16, n)
        if w.dim() != 2 or x.numel() != w.size(1) or y.numel() != w.size(0):
            raise RuntimeError(f"{what}: w must be [N, K], x [K] and y [N]")
        return w.size(0), w.size(1)

    # the fp16 LM head's torch.mm(x, W^T) (runtime/model.py:187) as a HIP GEMV
    def gemv_f16(self, R, warps, pf, w, x, y):
        N, Kd = self._f16_shape(w, x, y, "gemv_f16")
        self._call(self.lib.dk_gemv_f16, int(R), int(warps), int(pf), w.data_ptr(), x.data_ptr(), y.data_ptr(), N, Kd,
                   _stream(x))

    # add_rmsnorm (kernels/bindings.cpp:64-72) fused into the fp16 GEMV that follows it
    def gemv_f16_rmsnorm(self, R, warps, pf, w, x, delta, norm_w, eps, x_out, y):
        N, Kd = self._f16_shape(w, x, y, "gemv_f16_rmsnorm")
        _check_cuda(norm_w, "norm_w")
        for t, n in ((delta, "delta"), (norm_w, "norm_w"), (x_out, "x_out")):
            if t is not None:
                _check_cuda(t, n)
                if t.numel() != Kd or t.dtype != torch.float16:
                    raise RuntimeError(f"gemv_f16_rmsnorm: {n} must be fp16 [K]")
        ptr = lambda t: None if t is None else t.data_ptr()
        self._call(self.lib.dk_gemv_f16_rmsnorm, int(R), int(warps), int(pf), w.data_ptr(), x.data_ptr(), ptr(delta),
                   norm_w.data_ptr(), float(eps), ptr(x_out), y.data_ptr(), N, Kd, _stream(x))

    # prefill projections: Y = X . dequant(W)^T (epilogue 1: SwiGLU of interleaved gate/up pairs)
    def gemm_workspace_bytes(self, M, N, K, group, epilogue=0):
        """Bytes of split-K workspace dk_gemm_w4a16_ws uses for this shape (0: it does not split)."""
        return int(self.lib.dk_gemm_w4a16_workspace_bytes(int(M), int(N), int(K), int(group), int(epilogue)))

    def gemm_kernel(self, M, N, K, group, epilogue=0, splits=1):
        """Name of the kernel and tile that a GEMM of this shape runs over that many k ranges."""
        return self.lib.dk_gemm_w4a16_kernel(int(M), int(N), int(K), int(group), int(epilogue), int(splits)).decode()

    def gemm_w4a16(self, packed, sz, x, y, group, epilogue=0, workspace=None):
        """y = x . dequant(W)^T (epilogue 1: SwiGLU of interleaved gate/up rows); `workspace` (a CUDA tensor of
        gemm_workspace_bytes bytes) lets the shapes that do not fill the CUs split K."""
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (y, "y")):
            _check_cuda(t, n)
        N, K = packed.size(0), packed.size(1) * 8
        if x.dim() != 2 or x.size(1) != K:
            raise RuntimeError("gemm_w4a16: x must be [M, K]")
        M = x.size(0)
        if sz.size(0) != N or sz.size(1) != K // group or y.shape != (M, N // (1 + int(epilogue))):
            raise RuntimeError("gemm_w4a16: sz must be [N, K/G, 2] and y [M, N] (epilogue 1: [M, N/2])")
        _check_dtype(packed, torch.int32, "packed")
        for t, n in ((sz, "sz"), (x, "x"), (y, "y")):
            _check_dtype(t, torch.float16, n)
        if workspace is None:
            self._call(self.lib.dk_gemm_w4a16, packed.data_ptr(), sz.data_ptr(), x.data_ptr(), y.data_ptr(), M, N, K,
                       int(group), int(epilogue), _stream(x))
            return
        _check_cuda(workspace, "workspace")
        self._call(self.lib.dk_gemm_w4a16_ws, packed.data_ptr(), sz.data_ptr(), x.data_ptr(), y.data_ptr(), M, N, K,
                   int(group), int(epilogue), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                   _stream(x))

    def gemm_w4a16_parts(self, packed, sz, x, group, workspace):
        """The split-K GEMM's fp32 partials alone (no reduce launch), left in `workspace`; returns them as a [S, M, N]
        float32 view of it. Only for shapes that split (gemm_workspace_bytes(M, N, K, group) > 0)."""
        for t, n in ((packed, "packed"), (sz, "sz"), (x, "x"), (workspace, "workspace")):
            _check_cuda(t, n)
        N, K = packed.size(0), packed.size(1) * 8
        if x.dim() != 2 or x.size(1) != K:
            raise RuntimeError("gemm_w4a16_parts: x must be [M, K]")
        M = x.size(0)
        if sz.size(0) != N or sz.size(1) != K // group:
            raise RuntimeError("gemm_w4a16_parts: sz must be [N, K/G, 2]")
        _check_dtype(packed, torch.int32, "packed")
        for t, n in ((sz, "sz"), (x, "x")):
            _check_dtype(t, torch.float16, n)
        need = self.gemm_workspace_bytes(M, N, K, group)
        self._call(self.lib.dk_gemm_w4a16_ws, packed.data_ptr(), sz.data_ptr(), x.data_ptr(), None, M, N, K,
                   int(group), 2, workspace.data_ptr(), workspace.numel() * workspace.element_size(), _stream(x))
        S = need // (M * N * 4)
        return workspace.view(torch.uint8)[:need].view(torch.float32).view(S, M, N)

    # prefill: residual + RMSNorm of M rows whose delta is split-K partials [S, M, H] (a view; rows contiguous)
    def rmsnorm_rows_parts(self, x_in, parts, w, x_out, out, eps):
        for t, n in ((x_in, "x_in"), (w, "w"), (x_out, "x_out"), (out, "out")):
            _check_cuda(t, n)
            _check_dtype(t, torch.float16, n)
        if not parts.is_cuda or parts.dtype != torch.float32 or parts.dim() != 3:
            raise RuntimeError("rmsnorm_rows_parts: parts must be a CUDA float32 [S, M, H] view")
        S, M, H = parts.shape
        if parts.stride(2) != 1 or parts.stride(1) != H or out.shape != (M, H) or x_in.shape != (M, H):
            raise RuntimeError("rmsnorm_rows_parts: parts [S, M, H] with contiguous rows; x_in, out [M, H]")
        self._call(self.lib.dk_rmsnorm_rows_parts, x_in.data_ptr(), parts.data_ptr(), S, parts.stride(0),
                   w.data_ptr(), x_out.data_ptr(), out.data_ptr(), M, H, float(eps), _stream(x_in))

    # prefill: rope_append over M token rows (row m at position *pos + m)
    def rope_append_rows(self, qkv, cos_t, sin_t, pos, bt, kc, vc, n_q, n_kv):
        for t, n in ((qkv, "qkv"), (cos_t, "cos_t"), (sin_t, "sin_t"), (pos, "pos"), (bt, "bt"), (kc, "kc"),
                     (vc, "vc")):
            _check_cuda(t, n)
        D = kc.size(3)
        if qkv.dim() != 2 or qkv.size(1) != (n_q + 2 * n_kv) * D:
            raise RuntimeError("rope_append_rows: qkv must be [M, (n_q + 2 n_kv) * D]")
        self._call(self.lib.dk_rope_append_rows, qkv.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), pos.data_ptr(),
                   bt.data_ptr(), kc.data_ptr(), vc.data_ptr(), qkv.size(0), int(n_q), int(n_kv), D, kc.size(2),
                   cos_t.size(0), kc.size(0), bt.numel(), _stream(qkv))

    # prefill: residual + RMSNorm of M rows (rows: optional int64 gather index into x_in)
    def rmsnorm_rows(self, x_in, rows, delta, w, x_out, out, eps):
        for t, n in ((x_in, "x_in"), (w, "w"), (x_out, "x_out"), (out, "out")):
            _check_cuda(t, n)
            _check_dtype(t, torch.float16, n)
        M, H = out.shape
        if x_out.shape != (M, H) or w.numel() != H or x_in.size(-1) != H or (delta is not None and delta.shape != (M, H)):
            raise RuntimeError("rmsnorm_rows: x_out, out, delta [M, H], w [H], x_in [*, H]")
        if rows is not None and (rows.dtype != torch.int64 or rows.numel() != M):
            raise RuntimeError("rmsnorm_rows: rows must be int64 [M]")
        if rows is None and x_in.shape != (M, H):
            raise RuntimeError("rmsnorm_rows: without rows x_in must be [M, H]")
        ptr = lambda t: None if t is None else t.data_ptr()
        self._call(self.lib.dk_rmsnorm_rows, x_in.data_ptr(), ptr(rows), x_in.numel() // H, ptr(delta), w.data_ptr(),
                   x_out.data_ptr(), out.data_ptr(), M, H, float(eps), _stream(out))

    # prefill: causal attention of M rows over the paged cache
    def attention_prefill(self, qkv, pos, bt, kc, vc, n_q, n_kv, max_ctx, out):
        for t, n in ((qkv, "qkv"), (pos, "pos"), (bt, "bt"), (kc, "kc"), (vc, "vc"), (out, "out")):
            _check_cuda(t, n)
        D = kc.size(3)
        M = qkv.size(0)
        if qkv.dim() != 2 or qkv.size(1) != (n_q + 2 * n_kv) * D or out.shape != (M, n_q * D):
            raise RuntimeError("attention_prefill: qkv [M, (n_q + 2 n_kv) * D] and out [M, n_q * D]")
        self._call(self.lib.dk_attention_prefill, qkv.data_ptr(), pos.data_ptr(), bt.data_ptr(), bt.numel(),
                   kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.size(2), int(n_q), int(n_kv), D, M, int(max_ctx),
                   out.data_ptr(), _stream(qkv))

    # kernels/bindings.cpp:40-43
    def bw_read(self, buf, sink, blocks, threads, unroll):
        """Read probe over buf with the caller's grid (blocks x threads, `unroll` 16-byte loads in flight per lane).
        A sink of at least blocks * threads / 64 32-bit words receives per-wave sums of the words read (slot
        b * threads / 64 + w), which add up to the 32-bit word sum of the buffer; a smaller sink is not written."""
        _check_cuda(buf, "buf")
        _check_cuda(sink, "sink")
        words = sink.numel() * sink.element_size() // 4
        if words < 1:
            raise RuntimeError("bw_read: sink must hold at least one 32-bit word")
        self._call(self.lib.dk_bw_read, buf.data_ptr(), buf.numel() * buf.element_size(), sink.data_ptr(), words,
                   int(blocks), int(threads), int(unroll), _stream(buf))

    # the checks of kernels/bindings.cpp:45-62 (head_dim generalised from 64 to {64, 128}) -> C arguments
    def _attention_args(self, q, kc, vc, bt, pos, part_size, o_part, m_part, l_part, out, version):
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (bt, "bt"), (pos, "pos"), (out, "out"),
                     (o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part")):
            _check_cuda(t, n)
        if kc.dim() != 4 or kc.size(3) not in (64, 128) or vc.shape != kc.shape:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        if bt.dtype != torch.int32 or pos.dtype != torch.int32:
            raise RuntimeError("bt and pos must be int32")
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (out, "out")):
            _check_dtype(t, torch.float16, n)
        for t, n in ((o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part")):
            _check_dtype(t, torch.float32, n)
        D = kc.size(3)
        n_q, n_kv, P = q.numel() // D, kc.size(1), kc.size(2)
        if n_q * D != q.numel() or n_q % n_kv != 0 or (n_q // n_kv) not in (1, 2, 4, 8):
            raise RuntimeError("heads-per-group must be 1/2/4/8")
        if part_size <= 0:
            raise RuntimeError("part_size must be > 0")
        if version not in (1, 2, 3, 4, 5):
            raise RuntimeError("attention version must be 1..5")
        max_splits = o_part.size(1)
        if not (o_part.size(0) == n_q and o_part.size(2) == D and m_part.size(0) == n_q and l_part.size(0) == n_q
                and m_part.size(1) == max_splits and l_part.size(1) == max_splits and out.numel() == n_q * D):
            raise RuntimeError("paged_attention: split buffers must be o [n_q, S, D], m/l [n_q, S], out [n_q, D]")
        return (int(version), q.data_ptr(), kc.data_ptr(), vc.data_ptr(), bt.data_ptr(), pos.data_ptr(), n_q, n_kv, D,
                P, kc.size(0), bt.numel(), int(part_size), max_splits, o_part.data_ptr(), m_part.data_ptr(),
                l_part.data_ptr(), out.data_ptr(), _stream(q))

    # kernels/bindings.cpp:45-62 (head_dim generalised from 64 to {64, 128})
    def paged_attention(self, q, kc, vc, bt, pos, part_size, o_part, m_part, l_part, out, version=2):
        self._call(self.lib.dk_paged_attention,
                   *self._attention_args(q, kc, vc, bt, pos, part_size, o_part, m_part, l_part, out, version))

    # paged_attention's split kernel alone (no combine): with one live split it writes out, otherwise the partials
    # are left for gemv_w4a16_attn, the o projection that merges them in its prologue
    def paged_attention_split(self, q, kc, vc, bt, pos, part_size, o_part, m_part, l_part, out, version=5):
        self._call(self.lib.dk_paged_attention_split,
                   *self._attention_args(q, kc, vc, bt, pos, part_size, o_part, m_part, l_part, out, version))

    # the combine of paged_attention (kernels/paged_attention.cu:368-427) fused as the x prologue of gemv_w4a16 (the
    # o projection, runtime/model.py:220-222): y = W . combine(o_part, m_part, l_part), or W . attn with one live split
    def gemv_w4a16_attn(self, stage, R, warps, pf, packed, sz, o_part, m_part, l_part, attn, pos, bt, page, part_size,
                        max_pos, y, group):
        for t, n in ((packed, "packed"), (sz, "sz"), (o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part"),
                     (attn, "attn"), (pos, "pos"), (bt, "bt"), (y, "y")):
            _check_cuda(t, n)
        for t, n in ((o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part")):
            _check_dtype(t, torch.float32, n)
        _check_dtype(attn, torch.float16, "attn")
        if pos.dtype != torch.int32 or bt.dtype != torch.int32:
            raise RuntimeError("pos and bt must be int32")
        if o_part.dim() != 3:
            raise RuntimeError("gemv_w4a16_attn: o_part must be [n_q, S, D]")
        n_q, S, D = o_part.shape
        if m_part.shape != (n_q, S) or l_part.shape != (n_q, S) or attn.numel() != n_q * D:
            raise RuntimeError("gemv_w4a16_attn: split buffers must be o [n_q, S, D], m/l [n_q, S], attn [n_q * D]")
        K = n_q * D
        N = self._gemv_shape(packed, sz, y, K, group)
        self._call(self.lib.dk_gemv_w4a16_attn, int(stage), int(R), int(warps), int(pf), packed.data_ptr(),
                   sz.data_ptr(), o_part.data_ptr(), m_part.data_ptr(), l_part.data_ptr(), attn.data_ptr(),
                   pos.data_ptr(), bt.numel(), int(page), int(part_size), S, int(max_pos), n_q, D, y.data_ptr(), N, K,
                   int(group), _stream(y))

    # paged_attention with its split partials in the library's per-device scratch array (no caller buffers, no
    # allocation); calls that overlap on one GPU race
    def paged_attention_noalloc(self, q, kc, vc, bt, pos, part_size, max_splits, out, version=5):
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (bt, "bt"), (pos, "pos"), (out, "out")):
            _check_cuda(t, n)
        if kc.dim() != 4 or kc.size(3) not in (64, 128) or vc.shape != kc.shape:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        if bt.dtype != torch.int32 or pos.dtype != torch.int32:
            raise RuntimeError("bt and pos must be int32")
        for t, n in ((q, "q"), (kc, "kc"), (vc, "vc"), (out, "out")):
            _check_dtype(t, torch.float16, n)
        D = kc.size(3)
        n_q, n_kv, P = q.numel() // D, kc.size(1), kc.size(2)
        if n_q * D != q.numel() or out.numel() != n_q * D:
            raise RuntimeError("paged_attention_noalloc: q and out must hold n_q * head_dim values")
        with torch.cuda.device(q.device):      # the scratch address is resolved on the current device
            self._call(self.lib.dk_paged_attention_noalloc, int(version), q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                       bt.data_ptr(), pos.data_ptr(), n_q, n_kv, D, P, kc.size(0), bt.numel(), int(part_size),
                       int(max_splits), out.data_ptr(), _stream(q))

    def paged_attention_noalloc_bytes(self, n_q, head_dim, max_splits):
        return int(self.lib.dk_paged_attention_noalloc_bytes(int(n_q), int(head_dim), int(max_splits)))

    # rope_append (kernels/bindings.cpp:81-88) + paged_attention (kernels/bindings.cpp:45-62) fused into one launch
    def attention_decode(self, qkv, cos_t, sin_t, pos, bt, kc, vc, n_q, n_kv, part_size, o_part, m_part, l_part,
                         out, impl=0):
        """impl: 0 or 1 = block kernel, 3 = lean MFMA kernel (pages >= 16 tokens, part_size a multiple of 16 up to
        512, 256 at head_dim 128); 2 (an MFMA kernel since removed) is rejected. The split kernel is followed by the
        combine kernel."""
        for t, n in ((qkv, "qkv"), (cos_t, "cos_t"), (sin_t, "sin_t"), (pos, "pos"), (bt, "bt"), (kc, "kc"),
                     (vc, "vc"), (o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part"), (out, "out")):
            _check_cuda(t, n)
        if kc.dim() != 4 or kc.size(3) not in (64, 128) or vc.shape != kc.shape or kc.size(1) != n_kv:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        D = kc.size(3)
        if qkv.numel() != (n_q + 2 * n_kv) * D or cos_t.dim() != 2 or cos_t.size(1) != D // 2 \
                or sin_t.shape != cos_t.shape:
            raise RuntimeError("attention_decode: qkv must hold (n_q + 2 n_kv) * D values and cos/sin [max_pos, D/2]")
        for t, n in ((qkv, "qkv"), (kc, "kc"), (vc, "vc"), (out, "out")):
            _check_dtype(t, torch.float16, n)
        for t, n in ((cos_t, "cos_t"), (sin_t, "sin_t"), (o_part, "o_part"), (m_part, "m_part"), (l_part, "l_part")):
            _check_dtype(t, torch.float32, n)
        for t, n in ((pos, "pos"), (bt, "bt")):
            _check_dtype(t, torch.int32, n)
        if n_q % n_kv != 0 or (n_q // n_kv) not in (1, 2, 4, 8):
            raise RuntimeError("heads-per-group must be 1/2/4/8")
        max_splits = o_part.size(1)
        if not (o_part.size(0) == n_q and o_part.size(2) == D and m_part.shape == (n_q, max_splits)
                and l_part.shape == (n_q, max_splits) and out.numel() == n_q * D):
            raise RuntimeError("attention_decode: buffers must be o [n_q, S, D], m/l [n_q, S], out [n_q, D]")
        self._call(self.lib.dk_attention_decode, qkv.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), cos_t.size(0),
                   pos.data_ptr(), bt.data_ptr(), bt.numel(), kc.data_ptr(), vc.data_ptr(), kc.size(0), kc.size(2),
                   int(n_q), int(n_kv), D, int(part_size), max_splits, int(impl), o_part.data_ptr(),
                   m_part.data_ptr(), l_part.data_ptr(), out.data_ptr(), _stream(qkv))

    # kernels/bindings.cpp:64-72
    def add_rmsnorm(self, x, delta, w, out, eps):
        _check_cuda(x, "x")
        _check_cuda(w, "w")
        _check_cuda(out, "out")
        if x.numel() % 8 != 0:
            raise RuntimeError("add_rmsnorm: numel must be a multiple of 8")
        if w.numel() != x.numel() or out.numel() != x.numel():
            raise RuntimeError("add_rmsnorm: x, w and out must have the same size")
        for t, n in ((x, "x"), (w, "w"), (out, "out")):
            _check_dtype(t, torch.float16, n)
        d = None
        if delta is not None:
            _check_cuda(delta, "delta")
            _check_dtype(delta, torch.float16, "delta")
            if delta.numel() != x.numel():
                raise RuntimeError("add_rmsnorm: delta must have the size of x")
            d = delta.data_ptr()
        self._call(self.lib.dk_add_rmsnorm, x.data_ptr(), d, w.data_ptr(), out.data_ptr(), x.numel(), float(eps),
                   _stream(x))

    # kernels/bindings.cpp:74-79
    def swiglu(self, gu, out):
        _check_cuda(gu, "gu")
        _check_cuda(out, "out")
        if not (out.numel() % 8 == 0 and gu.numel() == 2 * out.numel()):
            raise RuntimeError("swiglu: out.numel() % 8 == 0 and gu.numel() == 2 * out.numel() required")
        _check_dtype(gu, torch.float16, "gu")
        _check_dtype(out, torch.float16, "out")
        self._call(self.lib.dk_swiglu, gu.data_ptr(), out.data_ptr(), out.numel(), _stream(gu))

    # kernels/bindings.cpp:81-88 (head_dim generalised from 64 to {64, 128})
    def rope_append(self, qkv, cos_t, sin_t, pos, bt, kc, vc, n_q, n_kv):
        for t, n in ((qkv, "qkv"), (cos_t, "cos_t"), (sin_t, "sin_t"), (kc, "kc"), (vc, "vc"), (pos, "pos"),
                     (bt, "bt")):
            _check_cuda(t, n)
        if kc.dim() != 4 or kc.size(3) not in (64, 128) or vc.shape != kc.shape or kc.size(1) != n_kv:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        D = kc.size(3)
        if qkv.numel() != (n_q + 2 * n_kv) * D or cos_t.dim() != 2 or cos_t.size(1) != D // 2 \
                or sin_t.shape != cos_t.shape:
            raise RuntimeError("rope_append: qkv must hold (n_q + 2 n_kv) * D values and cos/sin [max_pos, D/2]")
        _check_dtype(qkv, torch.float16, "qkv")
        _check_dtype(cos_t, torch.float32, "cos_t")
        _check_dtype(sin_t, torch.float32, "sin_t")
        if bt.dtype != torch.int32 or pos.dtype != torch.int32:
            raise RuntimeError("bt and pos must be int32")
        self._call(self.lib.dk_rope_append, qkv.data_ptr(), cos_t.data_ptr(), sin_t.data_ptr(), pos.data_ptr(),
                   bt.data_ptr(), kc.data_ptr(), vc.data_ptr(), int(n_q), int(n_kv), D, kc.size(2), cos_t.size(0),
                   kc.size(0), bt.numel(), _stream(qkv))

    # runtime/model.py:232-233 (torch.argmax into tok, then pos += 1) as one launch
    def argmax_advance(self, logits, tok, pos=None):
        _check_cuda(logits, "logits")
        _check_cuda(tok, "tok")
        _check_dtype(logits, torch.float16, "logits")
        _check_dtype(tok, torch.int64, "tok")
        p = None
        if pos is not None:
            _check_cuda(pos, "pos")
            _check_dtype(pos, torch.int32, "pos")
            p = pos.data_ptr()
        self._call(self.lib.dk_argmax_advance, logits.data_ptr(), logits.numel(), tok.data_ptr(), p, _stream(logits))

    def argmax_advance_split(self, logits, tok, pos, work):
        """argmax_advance over ceil(V / 4096) workgroups that meet through `work` (int64 [2], zero before the first
        call, left zero by every call; one work buffer per stream of calls)."""
        _check_cuda(logits, "logits")
        _check_cuda(tok, "tok")
        _check_cuda(work, "work")
        _check_dtype(logits, torch.float16, "logits")
        _check_dtype(tok, torch.int64, "tok")
        _check_dtype(work, torch.int64, "work")
        if work.numel() != 2:
            raise RuntimeError("argmax_advance_split: work must be int64 [2]")
        p = None
        if pos is not None:
            _check_cuda(pos, "pos")
            _check_dtype(pos, torch.int32, "pos")
            p = pos.data_ptr()
        self._call(self.lib.dk_argmax_advance_split, logits.data_ptr(), logits.numel(), tok.data_ptr(), p,
                   work.data_ptr(), _stream(logits))

    def _call_on(self, device, fn, *args):
        """_call with the stream of `device` as the last argument and that device current (the default stream's handle
        names the current device's)."""
        stream = torch._C._cuda_getCurrentRawStream(device)
        if device == torch._C._cuda_getDevice():
            rc = fn(*args, stream)
            if rc != 0:
                raise RuntimeError(self.lib.dk_last_error().decode() or f"decode kernel error {rc}")
            return
        with torch.cuda.device(device):
            self._call(fn, *args, stream)

    # rows of a prompt or of a drafted tree: per-head RMSNorm of q and k (models with q_norm / k_norm), RoPE, KV append
    def qk_norm_rope_append_rows(self, qkv, q_w, k_w, eps, cos_t, sin_t, pos, depth, bt, kc, vc, n_q, n_kv, q_out=None):
        """Row m of qkv [M, (n_q + 2 n_kv) * D] is cache token *pos + m and rotates at *pos + depth[m] (depth None: as a
        prompt, *pos + m). q_w, k_w [D] (None: no norm) weight the RMSNorm of each q and k head. The rotated q goes to
        q_out [M, n_q * D] (rows may be strided; None: in place in qkv), rotated k and v to the cache."""
        what, dev = "qk_norm_rope_append_rows", qkv.get_device()
        p_qkv, p_qw, p_kw, p_cos, p_sin, p_pos, p_depth, p_bt, p_kc, p_vc = _check_all(
            what, dev, (qkv, "qkv", torch.float16), (q_w, "q_w", torch.float16), (k_w, "k_w", torch.float16),
            (cos_t, "cos_t", torch.float32), (sin_t, "sin_t", torch.float32), (pos, "pos", torch.int32),
            (depth, "depth", torch.int32), (bt, "bt", torch.int32), (kc, "kc", torch.float16), (vc, "vc", torch.float16))
        cache, table, rows = kc.shape, cos_t.shape, qkv.shape
        if len(cache) != 4 or cache[3] not in (64, 128) or vc.shape != cache or cache[1] != n_kv:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        D = cache[3]
        row = (n_q + 2 * n_kv) * D
        if len(rows) != 2 or rows[1] != row or len(table) != 2 or table[1] * 2 != D or sin_t.shape != table \
                or pos.numel() < 1:
            raise RuntimeError(f"{what}: qkv must be [M, (n_q + 2 n_kv) * D], cos and sin [max_pos, D/2], pos [1]")
        M = rows[0]
        if depth is not None and depth.numel() != M:
            raise RuntimeError(f"{what}: depth must be int32 [M]")
        if (q_w is None) != (k_w is None) or (q_w is not None and (q_w.numel() != D or k_w.numel() != D)):
            raise RuntimeError(f"{what}: q_w and k_w must both be [D] or both None")
        if q_out is None:
            p_out, q_stride = p_qkv, row
        else:
            if q_out.dtype is not torch.float16 or q_out.get_device() != dev or q_out.shape != (M, n_q * D) \
                    or q_out.stride(1) != 1:
                raise RuntimeError(f"{what}: q_out must be a CUDA fp16 [M, n_q * D] with contiguous rows")
            p_out = q_out.data_ptr()
            q_stride = q_out.stride(0) if M > 1 else row if p_out == p_qkv else n_q * D
        self._call_on(dev, self.lib.dk_qk_norm_rope_append_rows, p_qkv, p_qw, p_kw, float(eps), p_cos, p_sin, p_pos, p_depth,
                      p_bt, p_kc, p_vc, p_out, q_stride, M, int(n_q), int(n_kv), D, cache[2], table[0], cache[0], bt.numel())

    # attention of the nodes of a drafted token tree (speculative decoding) over the paged cache
    def attention_tree_workspace_bytes(self, M, n_q, n_kv, head_dim, max_ctx):
        """Bytes of split workspace that attention_tree can use for these sizes (0: it does not split)."""
        return int(self.lib.dk_attention_tree_workspace_bytes(*_ints(M, n_q, n_kv, head_dim, max_ctx)))

    def attention_tree(self, q, mask, pos, bt, kc, vc, max_ctx, out, workspace=None):
        """q [M, n_q, D] or [M, n_q * D] (rows may be strided, e.g. the q part of qkv rows), rotated; node i attends the
        tokens [0, *pos) and the nodes j (tokens *pos + j, in the cache already) whose bit j % 64 of mask[i, j // 64] is
        set (mask int64 [M, ceil(M / 64)]; None: a chain, j <= i). max_ctx: *pos + M or more. out [M, n_q * D]."""
        what, dev = "attention_tree", q.get_device()
        p_mask, p_pos, p_bt, p_kc, p_vc, p_out = _check_all(
            what, dev, (mask, "mask", torch.int64), (pos, "pos", torch.int32), (bt, "bt", torch.int32),
            (kc, "kc", torch.float16), (vc, "vc", torch.float16), (out, "out", torch.float16))
        cache, rows = kc.shape, q.shape
        if len(cache) != 4 or cache[3] not in (64, 128) or vc.shape != cache:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
        D, strides = cache[3], q.stride()
        if q.dtype is not torch.float16 or len(rows) not in (2, 3) or strides[-1] != 1 \
                or (len(rows) == 3 and (rows[2] != D or (rows[1] > 1 and strides[1] != D))):
            raise RuntimeError(f"{what}: q must be a CUDA fp16 [M, n_q, D] or [M, n_q * D] with contiguous rows")
        M = rows[0]
        width = rows[1] if len(rows) == 2 else rows[1] * D
        if width % D != 0 or out.shape != (M, width) or pos.numel() < 1:
            raise RuntimeError(f"{what}: q rows must hold n_q * D values, out be [M, n_q * D] and pos [1]")
        if mask is not None and mask.shape != (M, (M + 63) // 64):
            raise RuntimeError(f"{what}: mask must be int64 [M, ceil(M / 64)]")
        max_ctx = int(max_ctx)
        if not -0x80000000 <= max_ctx <= 0x7FFFFFFF:
            _ints(max_ctx)
        p_ws, ws_bytes = _workspace(what, dev, workspace)
        self._call_on(dev, self.lib.dk_attention_tree, q.data_ptr(), strides[0] if M > 1 else width, p_mask, p_pos, p_bt,
                      bt.numel(), p_kc, p_vc, cache[0], cache[2], width // D, cache[1], D, M, max_ctx, p_out, p_ws,
                      ws_bytes)

    # log probabilities of given tokens with entropy and top alternatives (the picks of a verified tree, prompt scoring)
    def token_logprobs_workspace_bytes(self, M, V, k, dtype=torch.float16):
        """Bytes of split workspace that token_logprobs can use for these sizes (0: it does not split)."""
        if dtype not in LOGITS_DTYPES:
            raise RuntimeError(f"token_logprobs: logits must be fp16, bf16 or fp32, got {dtype}")
        return int(self.lib.dk_token_logprobs_workspace_bytes(*_ints(M, V, k), LOGITS_DTYPES[dtype]))

    def token_logprobs(self, logits, tokens, logprobs, entropy=None, top_ids=None, top_logprobs=None, workspace=None):
        """logits [M, V] (fp16, bf16 or fp32; rows may be strided): logprobs[m] of the ids tokens[m], entropy[m] and the k
        largest logits' ids and log probabilities (top_ids int64, top_logprobs [M, k], k <= 32; descending, the lowest
        index first among equals). Outputs fp32; any of them may be None (tokens and logprobs together)."""
        what, dev = "token_logprobs", logits.get_device()
        p_tokens, p_logprobs, p_entropy, p_ids, p_top = _check_all(
            what, dev, (tokens, "tokens", torch.int64), (logprobs, "logprobs", torch.float32),
            (entropy, "entropy", torch.float32), (top_ids, "top_ids", torch.int64),
            (top_logprobs, "top_logprobs", torch.float32))
        dtype, rows = LOGITS_DTYPES.get(logits.dtype), logits.shape
        if dev < 0 or dtype is None or len(rows) != 2 or (logits.stride(1) != 1 and rows[1] > 1):
            raise RuntimeError(f"{what}: logits must be a CUDA fp16, bf16 or fp32 [M, V] with contiguous rows")
        M, V = rows
        if M > 0x7FFFFFFF or V > 0x7FFFFFFF:
            _ints(M, V)
        for t, name in ((tokens, "tokens"), (logprobs, "logprobs"), (entropy, "entropy")):
            if t is not None and t.numel() != M:
                raise RuntimeError(f"{what}: {name} must hold M values")
        k = 0 if top_ids is None else top_ids.size(-1)
        if (top_ids is None) != (top_logprobs is None) \
                or (top_ids is not None and (k == 0 or not top_ids.shape == top_logprobs.shape == (M, k))):
            raise RuntimeError(f"{what}: top_ids and top_logprobs must both be [M, k] or both None")
        p_ws, ws_bytes = _workspace(what, dev, workspace)
        self._call_on(dev, self.lib.dk_token_logprobs, logits.data_ptr(), dtype, logits.stride(0) if M > 1 else V, p_tokens,
                      p_logprobs, p_entropy, p_ids, p_top, M, V, k, p_ws, ws_bytes)

    # the greedy walk down a verified tree, and its cache rows made contiguous
    def tree_accept(self, tokens, parents, picks, pos, bt, kv, path, count, tok):
        """tokens int64 [M], parents int32 [M] (node 0 the root, parents[c] < c), picks int64 [M] (the model's pick after
        each node; may be strided, e.g. top_ids[:, 0]) -> path int32 [M] (the accepted nodes, then -1), count int32 [1],
        tok int64 [1] (the next pending token); kv [..., pages, n_kv, P, D] (any leading sizes, e.g. layers and K / V; None:
        no move): the rows of tokens *pos + path[t] move to *pos + t in every cache. pos stays: the caller adds count."""
        what, dev = "tree_accept", tokens.get_device()
        p_tokens, p_parents, p_pos, p_bt, p_kv, p_path, p_count, p_tok = _check_all(
            what, dev, (tokens, "tokens", torch.int64), (parents, "parents", torch.int32), (pos, "pos", torch.int32),
            (bt, "bt", torch.int32), (kv, "kv", torch.float16), (path, "path", torch.int32), (count, "count", torch.int32),
            (tok, "tok", torch.int64))
        M = tokens.numel()
        if picks.dtype is not torch.int64 or picks.get_device() != dev or picks.shape != (M,):
            raise RuntimeError(f"{what}: picks must be a CUDA int64 [M]")
        if parents.numel() != M or path.numel() != M or count.numel() != 1 or tok.numel() != 1:
            raise RuntimeError(f"{what}: parents and path must hold M values, count and tok one")
        if kv is None:
            n_caches, cache = 0, (0, 0, 0, 0)
        else:
            cache = kv.shape[-4:]
            if len(cache) < 4 or cache[3] not in (64, 128):
                raise RuntimeError("cache must be [pages, n_kv, P, 64|128]")
            n_caches = kv.numel() // max(1, cache[0] * cache[1] * cache[2] * cache[3])
        self._call_on(dev, self.lib.dk_tree_accept, p_tokens, p_parents, picks.data_ptr(), picks.stride(0) if M > 1 else 1, M,
                      p_pos, p_bt, 0 if bt is None else bt.numel(), p_kv, n_caches, cache[0], cache[1], cache[2], cache[3],
                      p_path, p_count, p_tok)

    def _kv8_cache(self, what, kc, vc, ks, vs):
        """Shape and type of an 8-bit cache: (its type's number, [pages, n_kv, P, D])."""
        cache, dtype = kc.shape, CACHE_DTYPES.get(kc.dtype, 0)
        if dtype == 0:
            raise RuntimeError(f"{what}: kc and vc must be int8 or float8_e4m3fn, got {kc.dtype}")
        if len(cache) != 4 or cache[3] not in (64, 128) or vc.shape != cache or cache[2] % KV8_BLOCK:
            raise RuntimeError("cache must be [pages, n_kv, P, 64|128], of an 8-bit cache P a multiple of 16")
        scales = (cache[0], cache[1], cache[2] // KV8_BLOCK)
        if ks.shape != scales or vs.shape != scales:
            raise RuntimeError(f"{what}: ks and vs must be [pages, n_kv, P / {KV8_BLOCK}]")
        return dtype, cache

    # rows of a prompt, or one token, rotated and appended to a cache of 8-bit codes
    def kv8_append_rows(self, qkv, cos_t, sin_t, pos, bt, kc, vc, ks, vs, n_q, n_kv, q_out=None):
        """rope_append_rows into an 8-bit cache: row m of qkv [M, (n_q + 2 n_kv) * D] is token *pos + m. kc, vc int8 or
        float8_e4m3fn [pages, n_kv, P, D], ks, vs fp32 [pages, n_kv, P / 16]: a value is code * scale, one scale for 16
        tokens, a power of two. The rotated q goes to q_out [M, n_q * D] (rows may be strided; None: in place in qkv). cos_t
        and sin_t None: no rotation. Rows behind the new ones in a block count as absent."""
        what, dev = "kv8_append_rows", qkv.get_device()
        dtype, cache = self._kv8_cache(what, kc, vc, ks, vs)
        p_qkv, p_cos, p_sin, p_pos, p_bt, p_kc, p_vc, p_ks, p_vs = _addresses(
            what, dev, _APPEND_SPEC[kc.dtype], qkv, cos_t, sin_t, pos, bt, kc, vc, ks, vs)
        rows, D = qkv.shape, cache[3]
        row = (n_q + 2 * n_kv) * D
        if len(rows) != 2 or rows[1] != row or cache[1] != n_kv or pos.numel() < 1:
            raise RuntimeError(f"{what}: qkv must be [M, (n_q + 2 n_kv) * D], pos [1]")
        if (cos_t is None) != (sin_t is None) \
                or (cos_t is not None and (cos_t.dim() != 2 or cos_t.size(1) * 2 != D or sin_t.shape != cos_t.shape)):
            raise RuntimeError(f"{what}: cos_t and sin_t must both be [max_pos, D/2] or both None")
        M = rows[0]
        if q_out is None:
            p_out, q_stride = p_qkv, row
        else:
            if q_out.dtype is not torch.float16 or q_out.get_device() != dev or q_out.shape != (M, n_q * D) \
                    or q_out.stride(1) != 1:
                raise RuntimeError(f"{what}: q_out must be a CUDA fp16 [M, n_q * D] with contiguous rows")
            p_out = q_out.data_ptr()
            q_stride = q_out.stride(0) if M > 1 else row if p_out == p_qkv else n_q * D
        self._call_on(dev, self.lib.dk_kv8_append_rows, p_qkv, p_cos, p_sin, p_pos, p_bt, p_kc, p_vc, p_ks, p_vs, dtype, p_out,
                      q_stride, M, int(n_q), int(n_kv), D, cache[2], 0 if cos_t is None else cos_t.size(0), cache[0],
                      bt.numel())

    # tokens of an 8-bit cache as fp16 rows
    def kv8_read(self, bt, kc, vc, ks, vs, start, k_out, v_out):
        """Tokens [start, start + n) of the 8-bit cache as fp16 rows k_out, v_out [n, n_kv, D] (or [n, n_kv * D]); tokens
        without a mapped page read as zeros."""
        what, dev = "kv8_read", k_out.get_device()
        dtype, cache = self._kv8_cache(what, kc, vc, ks, vs)
        p_bt, p_kc, p_vc, p_ks, p_vs, p_k, p_v = _addresses(what, dev, _READ_SPEC[kc.dtype], bt, kc, vc, ks, vs, k_out, v_out)
        n = k_out.size(0) if k_out.dim() else 0
        if n < 1 or k_out.numel() != n * cache[1] * cache[3] or v_out.shape != k_out.shape:
            raise RuntimeError(f"{what}: k_out and v_out must be [n, n_kv, D], n >= 1")
        self._call_on(dev, self.lib.dk_kv8_read, p_bt, bt.numel(), p_kc, p_vc, p_ks, p_vs, dtype, cache[0], cache[2], cache[1],
                      cache[3], *_ints(start, n), p_k, p_v)

    # attention of rows under a sliding window with sinks, over fp16 or 8-bit caches
    def attention_window_workspace_bytes(self, M, n_q, n_kv, head_dim, max_ctx, window=0, sinks=0, dtype=torch.float16):
        """Bytes of split workspace that attention_window (dtype of the cache fp16) or attention_kv8 (int8, float8_e4m3fn)
        can use for these sizes (0: it does not split)."""
        if dtype not in CACHE_DTYPES:
            raise RuntimeError(f"attention_window: the cache must be fp16, int8 or float8_e4m3fn, got {dtype}")
        return int(self.lib.dk_attention_window_workspace_bytes(*_ints(M, n_q, n_kv, head_dim, max_ctx, window, sinks),
                                                                CACHE_DTYPES[dtype]))

    def _attention_window(self, what, spec, q, pos, bt, kc, vc, ks, vs, dtype, cache, max_ctx, out, window, sinks, workspace):
        dev = q.get_device()
        p_pos, p_bt, p_kc, p_vc, p_ks, p_vs, p_out = _addresses(what, dev, spec, pos, bt, kc, vc, ks, vs, out)
        rows, strides, D = q.shape, q.stride(), cache[3]
        if q.dtype is not torch.float16 or len(rows) not in (2, 3) or strides[-1] != 1 \
                or (len(rows) == 3 and (rows[2] != D or (rows[1] > 1 and strides[1] != D))):
            raise RuntimeError(f"{what}: q must be a CUDA fp16 [M, n_q, D] or [M, n_q * D] with contiguous rows")
        M = rows[0]
        width = rows[1] if len(rows) == 2 else rows[1] * D
        if width % D != 0 or out.shape != (M, width) or pos.numel() < 1:
            raise RuntimeError(f"{what}: q rows must hold n_q * D values, out be [M, n_q * D] and pos [1]")
        max_ctx, window, sinks = int(max_ctx), int(window), int(sinks)
        if not 0 <= max_ctx | window | sinks <= 0x7FFFFFFF:
            _ints(max_ctx, window, sinks)
        p_ws, ws_bytes = _workspace(what, dev, workspace)
        self._call_on(dev, self.lib.dk_attention_window, q.data_ptr(), strides[0] if M > 1 else width, p_pos, p_bt, bt.numel(),
                      p_kc, p_vc, p_ks, p_vs, dtype, cache[0], cache[2], width // D, cache[1], D, M, max_ctx, window, sinks,
                      p_out, p_ws, ws_bytes)

    def attention_window(self, q, pos, bt, kc, vc, max_ctx, out, window=0, sinks=0, workspace=None):
        """q [M, n_q, D] or [M, n_q * D] (rows may be strided), rotated; row m is at position p = *pos + m and attends the
        tokens t <= p of the cache that are in its window (t > p - window; 0: no window) or sinks (t < sinks). max_ctx:
        *pos + M or more. out [M, n_q * D]."""
        cache = kc.shape
        if kc.dtype is not torch.float16 or len(cache) != 4 or cache[3] not in (64, 128) or vc.shape != cache:
            raise RuntimeError("cache must be fp16 [pages, n_kv, P, 64|128]")
        self._attention_window("attention_window", _WINDOW_SPEC, q, pos, bt, kc, vc, None, None, 0, cache, max_ctx, out, window,
                               sinks, workspace)

    def attention_kv8(self, q, pos, bt, kc, vc, ks, vs, max_ctx, out, window=0, sinks=0, workspace=None):
        """attention_window over an 8-bit cache (kv8_append_rows), by default without a window."""
        dtype, cache = self._kv8_cache("attention_kv8", kc, vc, ks, vs)
        self._attention_window("attention_kv8", _KV8_SPEC[kc.dtype], q, pos, bt, kc, vc, ks, vs, dtype, cache, max_ctx, out,
                               window, sinks, workspace)

    def attention_kv8_decode(self, qkv, cos_t, sin_t, pos, bt, kc, vc, ks, vs, n_q, n_kv, max_ctx, out, window=0, sinks=0,
                             workspace=None):
        """kv8_append_rows of one token, the fused qkv vector [(n_q + 2 n_kv) * D] (which stays as it is), and attention_kv8
        of its rotated q, in the launches of the attention. out [n_q * D]; workspace as for attention_kv8 with M = 1."""
        what, dev = "attention_kv8_decode", qkv.get_device()
        dtype, cache = self._kv8_cache(what, kc, vc, ks, vs)
        p_qkv, p_cos, p_sin, p_pos, p_bt, p_kc, p_vc, p_ks, p_vs, p_out = _addresses(
            what, dev, _DECODE_SPEC[kc.dtype], qkv, cos_t, sin_t, pos, bt, kc, vc, ks, vs, out)
        D = cache[3]
        if cos_t is None or sin_t is None or cos_t.dim() != 2 or cos_t.size(1) * 2 != D or sin_t.shape != cos_t.shape:
            raise RuntimeError(f"{what}: cos_t and sin_t must be [max_pos, D/2]")
        if qkv.numel() != (n_q + 2 * n_kv) * D or cache[1] != n_kv or out.numel() != n_q * D or pos.numel() < 1:
            raise RuntimeError(f"{what}: qkv must hold (n_q + 2 n_kv) * D values, out n_q * D and pos one")
        p_ws, ws_bytes = _workspace(what, dev, workspace)
        self._call_on(dev, self.lib.dk_attention_kv8_decode, p_qkv, p_cos, p_sin, cos_t.size(0), p_pos, p_bt, bt.numel(), p_kc,
                      p_vc, p_ks, p_vs, dtype, cache[0], cache[2], *_ints(n_q, n_kv), D, *_ints(max_ctx, window, sinks), p_out,
                      p_ws, ws_bytes)

    # runtime/quant.py:42-48,100-124 on the GPU
    def quantize_w4(self, w, packed, sz, group, clip=False):
        for t, n in ((w, "w"), (packed, "packed"), (sz, "sz")):
            _check_cuda(t, n)
        N, K = w.shape
        if not (packed.shape == (N, K // 8) and sz.shape == (N, K // group, 2)):
            raise RuntimeError("quantize_w4: packed must be [N, K/8] int32 and sz [N, K/G, 2] fp16")
        _check_dtype(w, torch.float16, "w")
        _check_dtype(packed, torch.int32, "packed")
        _check_dtype(sz, torch.float16, "sz")
        self._call(self.lib.dk_quantize_w4, w.data_ptr(), packed.data_ptr(), sz.data_ptr(), N, K, int(group),
                   int(bool(clip)), _stream(w))


def load(verbose=False):
    """Load (once) and return the op module. Raises RuntimeError if the library is missing or not loadable."""
    global _EXT
    if _EXT is None:
        lib = open_library()
        _EXT = DecodeKernels(lib)
        if verbose:
            print(f"loaded {LIB_PATH} (HIP runtime {lib.dk_runtime_version()})")
    return _EXT
