"""ctypes binding of libsid_hip.so: torch tensors in, raw device pointers out.

Each method checks its tensors the way the reference's TORCH_CHECKs do
(sid/csrc/flash_decode.cu:325-345, 386-395) and raises RuntimeError on a violation or on
a non-zero status from the library (message from `sid_last_error()`). Launches go on
torch's current stream of the tensors' device, so they order with surrounding torch work
and are captured by `torch.cuda.graph` like any torch op.
"""

from __future__ import annotations

import ctypes
from pathlib import Path

import torch

_i32, _i64, _f32, _vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

# name -> argtypes (every entry point returns int status)
_SIGNATURES = {
    "sid_reshape_and_cache": [_vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i64, _vp],
    "sid_flash_decode_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i64, _i32,
                             _i32, _f32, _vp, _vp, _i32, _i32, _vp, _vp],
    "sid_extend_attention_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i64, _i32, _i32, _i32,
                                 _i64, _i32, _i32, _f32, _vp, _i64, _vp, _vp],
    "sid_rmsnorm": [_vp, _vp, _vp, _i64, _i32, _f32, _vp],
    "sid_fused_add_rmsnorm": [_vp, _vp, _vp, _i64, _i32, _f32, _vp],
    "sid_rope_apply": [_vp, _vp, _vp, _vp, _i64, _i32, _i32, _i32, _i64, _vp],
    "sid_linear": [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _i32, _vp],
    "sid_linear_partials": [_vp, _i64, _vp, _vp, _i64, _i64, _i64, _vp],
    "sid_fused_add_rmsnorm_partials": [_vp, _i32, _vp, _vp, _vp, _i64, _i32, _f32, _vp],
    "sid_silu_mul_partials": [_vp, _i32, _vp, _i64, _i64, _vp],
    "sid_qkv_post": [_vp, _vp, _i32, _i64, _i32, _i32, _i32, _vp, _vp, _f32, _vp, _vp, _i64, _vp,
                     _vp, _vp, _vp, _i64, _vp],
    "sid_silu_mul": [_vp, _vp, _i64, _i64, _vp],
    "sid_linear_silu_mul": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "sid_gather_rows": [_vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "sid_argmax_rows": [_vp, _i64, _vp, _i64, _i64, _vp],
    "sid_build_paged_decode_indices": [_vp, _i64, _i64, _i32, _vp, _vp, _vp, _vp, _i32, _vp],
    "sid_flash_decode_segments_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i64,
                                      _i32, _i32, _i32, _i32, _i32, _vp, _f32, _vp, _vp, _i32,
                                      _i32, _vp, _vp],
    "sid_flash_decode_workers_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i64,
                                     _i32, _i32, _i32, _i32, _i32, _vp, _f32, _vp, _vp, _i32,
                                     _i32, _vp, _i32, _vp],
    "sid_flash_decode_segments_fwd_noalloc": [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32,
                                              _i32, _i64, _i32, _i32, _i32, _i32, _i32, _vp,
                                              _f32, _vp, _vp],
    "sid_sample_rows": [_vp, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _vp, _i64, _vp, _vp],
    "sid_linear_sample": [_vp, _i64, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _vp, _i64, _vp, _vp,
                          _i32, _vp],
    "sid_linear_argmax": [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _vp],
    "sid_linear_residual": [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i64, _vp],
    "sid_rmsnorm_linear_silu_mul": [_vp, _i32, _vp, _f32, _vp, _vp, _i64, _i64, _i64, _vp],
    "sid_rmsnorm_qkv_post": [_vp, _i32, _vp, _f32, _vp, _i64, _i64, _i32, _i32, _i32, _vp, _vp,
                             _vp, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _vp],
    "sid_rmsnorm_f32": [_vp, _vp, _vp, _i64, _i32, _f32, _vp],
    "sid_pack_decode_weight": [_vp, _vp, _i64, _i64, _i32, _vp],
    "sid_reshape_and_cache_fp8": [_vp, _i64, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _i32, _i32,
                                  _i64, _vp],
    "sid_gather_cache_fp8": [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i64, _vp],
    "sid_qkv_post_fp8": [_vp, _vp, _i32, _i64, _i32, _i32, _i32, _vp, _vp, _f32, _vp, _vp, _i64,
                         _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "sid_rmsnorm_qkv_post_fp8": [_vp, _i32, _vp, _f32, _vp, _i64, _i64, _i32, _i32, _i32, _vp,
                                 _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _vp, _i64, _vp],
    "sid_flash_decode_fp8_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i64,
                                 _i32, _i32, _i32, _i32, _i32, _vp, _f32, _vp, _vp, _i32, _i32,
                                 _vp, _i32, _vp],
    "sid_extend_attention_fp8_fwd": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i32, _i64, _i32, _i32,
                                     _i32, _i64, _i32, _i32, _f32, _vp, _i64, _vp, _vp],
}
EXPORTED = ("sid_last_error", "sid_abi_version", "sid_abi_revision",
            "sid_extend_attention_workspace_bytes",
            "sid_linear_argmax_workspace_bytes", "sid_sample_workspace_bytes",
            "sid_qwen3_extend_workspace_bytes", "sid_qwen3_extend_forward",
            "sid_qwen3_extend_forward_fp8", "sid_extend_attention_fp8_workspace_bytes",
            "sid_flash_decode_noalloc_scratch_bytes", "sid_linear_sample_workspace_bytes",
            "sid_extend_attention_query_rows", "sid_linear_tile", *_SIGNATURES)
ABI_VERSION = 22
ABI_REVISION = 1  # entry points added under that version (1: the 8-bit KV pool)


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _gpu(t: torch.Tensor, name: str, dtype: torch.dtype | None = None) -> None:
    # The messages are built only when they are raised: formatting them (a dtype's repr above
    # all) took half of an eager decode-attention call's host time (cache write + attention
    # of one request, two calls with 13 tensors: 31 us for 12 us of kernels).
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError(f"{name} must be a GPU tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")


_E4M3, _E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


# The usual case of an 8-bit pool's call, in one expression each: an eager call of a few rows is bound
# by the host, and these instead of a check for each tensor take one request's decode attention from
# 16.9 to 16.0 us and 64 rows' qkv_post from 13.6 to 12.8. False: the checks one by one say what
# is wrong.

def _usual_decode(q, kv_indptr, kv_indices, part_o, part_lse, o) -> bool:
    try:
        return (-1 < q.get_device() == kv_indptr.get_device() == kv_indices.get_device()
                == part_o.get_device() == part_lse.get_device() == o.get_device()
                and q.dtype is _BF16 and o.dtype is _BF16 and kv_indptr.dtype is _I32
                and kv_indices.dtype is _I32 and part_o.dtype is _F32 and part_lse.dtype is _F32
                and q.is_contiguous() and kv_indptr.is_contiguous() and kv_indices.is_contiguous()
                and part_o.is_contiguous() and part_lse.is_contiguous() and o.is_contiguous())
    except AttributeError:
        return False


def _usual_qkv(q_out, q_norm, k_norm, positions, cos_sin, slots) -> bool:
    try:
        return (-1 < q_out.get_device() == q_norm.get_device() == k_norm.get_device()
                == positions.get_device() == cos_sin.get_device() == slots.get_device()
                and q_out.dtype is _BF16 and q_norm.dtype is _BF16 and k_norm.dtype is _BF16
                and positions.dtype is _I64 and slots.dtype is _I64 and cos_sin.dtype is _F32
                and q_out.is_contiguous() and q_norm.is_contiguous() and k_norm.is_contiguous()
                and positions.is_contiguous() and slots.is_contiguous()
                and cos_sin.is_contiguous())
    except AttributeError:
        return False


def _same_device(device: int, *tensors) -> None:
    """Every tensor (None: absent) is on GPU `device` (an index)."""
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise RuntimeError(f"operands on {t.device} and GPU {device}: all must be on one device")


def _pool8(k_cache, v_cache, kv_scales, head_dim: int, device: int) -> tuple:
    """Checks an 8-bit KV pool (codes and their scales) on GPU `device`; its shape [S, HKV, D].
    One expression in the usual case (a decode step's eager call is bound by the host: these
    checks took 1.3 us of a one-row store's 8.4, now 0.6); the reason is looked for if it fails."""
    try:
        ks = k_cache.shape
        if (k_cache.dtype is _E4M3 and v_cache.dtype is _E4M3 and kv_scales.dtype is _E8M0
                and k_cache.get_device() == v_cache.get_device() == kv_scales.get_device() == device
                and k_cache.is_contiguous() and v_cache.is_contiguous()
                and kv_scales.is_contiguous() and len(ks) == 3 and ks[2] == head_dim
                and v_cache.shape == ks and kv_scales.shape == (ks[0], ks[1], 2)):
            return ks
    except AttributeError:
        pass
    _gpu(k_cache, "k_cache", _E4M3)
    _gpu(v_cache, "v_cache", _E4M3)
    _gpu(kv_scales, "kv_scales", _E8M0)
    if k_cache.dim() != 3 or ks[2] != head_dim or v_cache.shape != ks:
        raise RuntimeError(f"k_cache and v_cache must both be [S, HKV, {head_dim}]")
    if tuple(kv_scales.shape) != (ks[0], ks[1], 2):
        raise RuntimeError(f"kv_scales must be [S, HKV, 2] = [{ks[0]}, {ks[1]}, 2], got "
                           f"{list(kv_scales.shape)}")
    _same_device(device, k_cache, v_cache, kv_scales)
    raise AssertionError("unreachable")


def _ptr(t) -> int:
    """Device address of an optional tensor (0 for None)."""
    return 0 if t is None else t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    """torch's current stream of the tensor's device (the raw handle: no Stream object)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


class NativeLib:
    """The loaded library; method names and argument orders follow the reference ops."""

    def __init__(self, path: Path):
        self.path = Path(path)
        self.lib = ctypes.CDLL(str(self.path))
        self.lib.sid_last_error.restype = ctypes.c_char_p
        self.lib.sid_last_error.argtypes = []
        self.lib.sid_abi_version.restype = ctypes.c_int
        self.lib.sid_abi_version.argtypes = []
        ver = self.lib.sid_abi_version()
        _check(ver == ABI_VERSION, f"libsid_hip.so ABI {ver} != expected {ABI_VERSION}; rebuild")
        rev = self.lib.sid_abi_revision() if hasattr(self.lib, "sid_abi_revision") else 0
        _check(rev >= ABI_REVISION,
               f"libsid_hip.so ABI {ver} revision {rev} < expected {ABI_REVISION}; rebuild")
        self.lib.sid_extend_attention_workspace_bytes.restype = ctypes.c_int64
        self.lib.sid_extend_attention_workspace_bytes.argtypes = [_i32, _i64, _i32, _i32, _i32, _i32]
        self.lib.sid_extend_attention_fp8_workspace_bytes.restype = ctypes.c_int64
        self.lib.sid_extend_attention_fp8_workspace_bytes.argtypes = [_i32, _i64, _i32, _i32, _i32,
                                                                      _i32]
        self.lib.sid_extend_attention_query_rows.restype = ctypes.c_int
        self.lib.sid_extend_attention_query_rows.argtypes = [_i32, _i64, _i32, _i32]
        self.lib.sid_linear_tile.restype = ctypes.c_int
        self.lib.sid_linear_tile.argtypes = [_i64, _i64]
        self.lib.sid_linear_argmax_workspace_bytes.restype = ctypes.c_int64
        self.lib.sid_linear_argmax_workspace_bytes.argtypes = [_i64]
        self.lib.sid_sample_workspace_bytes.restype = ctypes.c_int64
        self.lib.sid_sample_workspace_bytes.argtypes = [_i64, _i64]
        self.lib.sid_linear_sample_workspace_bytes.restype = ctypes.c_int64
        self.lib.sid_linear_sample_workspace_bytes.argtypes = [_i64]
        self.lib.sid_flash_decode_noalloc_scratch_bytes.restype = ctypes.c_int64
        self.lib.sid_flash_decode_noalloc_scratch_bytes.argtypes = []
        for name, argtypes in _SIGNATURES.items():
            fn = getattr(self.lib, name)
            fn.argtypes = argtypes
            fn.restype = ctypes.c_int

    def _call(self, name: str, *args) -> None:
        rc = getattr(self.lib, name)(*args)
        if rc != 0:
            raise RuntimeError(f"{name}: {self.lib.sid_last_error().decode(errors='replace')}")

    def _launch(self, device: int, name: str, *args) -> None:
        """_call on GPU `device`'s current stream, with that device made current if it is not
        (the null stream belongs to the current device)."""
        if device != torch._C._cuda_getDevice():
            with torch.cuda.device(device):
                self._call(name, *args, torch._C._cuda_getCurrentRawStream(device))
            return
        if getattr(self.lib, name)(*args, torch._C._cuda_getCurrentRawStream(device)) != 0:
            raise RuntimeError(f"{name}: {self.lib.sid_last_error().decode(errors='replace')}")

    # ---- reference module `sid_flash_decode` (sid/csrc/flash_decode.cu:408-413) ----------

    def flash_decode_fwd(self, q, k_cache, v_cache, kv_indptr, kv_indices, num_splits,
                         max_splits: int, fixed_split_size: int, sm_scale: float,
                         part_o, part_lse, o, segment_size: int = 0,
                         grid_slots: int | None = None, variant: int = 0,
                         wg_order=None, workers: int = 0, kv_scales=None) -> None:
        """segment_size / grid_slots / variant / wg_order: see sid_flash_decode_segments_fwd
        (defaults: one segment per split, grid of max_splits slots = the reference's
        partition, the default workgroup shape, the grid's own order); workers > 0: stage 1
        by that many workgroups over the items of wg_order (sid_flash_decode_workers_fwd; entries
        flagged ORDER_EMPTY hold no tokens); kv_scales: the caches are an 8-bit pool
        (sid_flash_decode_fp8_fwd)."""
        usual = kv_scales is not None and _usual_decode(q, kv_indptr, kv_indices, part_o, part_lse, o)
        if not usual:
            _gpu(q, "q", torch.bfloat16)
        _check(q.dim() == 3, "q must be [B, HQ, D]")
        b, hq, d = qs = q.shape  # (each .shape builds a new object: taken once)
        if kv_scales is not None:
            ks = _pool8(k_cache, v_cache, kv_scales, d, q.get_device())
            if usual:
                _same_device(q.get_device(), num_splits, wg_order)
            else:
                _same_device(q.get_device(), kv_indptr, kv_indices, num_splits, part_o, part_lse,
                             o, wg_order)
        else:
            _gpu(k_cache, "k_cache", torch.bfloat16)
            _gpu(v_cache, "v_cache", torch.bfloat16)
            ks, vs = k_cache.shape, v_cache.shape
            for name, sh in (("k_cache", ks), ("v_cache", vs)):
                if not (len(sh) == 3 and sh[2] == d):
                    raise RuntimeError(f"{name} must be [slots, HKV, {d}]")
            _check(ks == vs, "k_cache and v_cache shapes differ")
        num_slots, hkv, _ = ks
        if not usual:
            _gpu(kv_indptr, "kv_indptr", torch.int32)
            _gpu(kv_indices, "kv_indices", torch.int32)
            _gpu(part_o, "part_o", torch.float32)
            _gpu(part_lse, "part_lse", torch.float32)
            _gpu(o, "o", torch.bfloat16)
        _check(kv_indptr.numel() == b + 1, "kv_indptr must have B+1 entries")
        if num_splits is not None:  # None: derived on the device from the lengths
            _gpu(num_splits, "num_splits", torch.int32)
            _check(num_splits.numel() == b, "num_splits must have B entries")
        po, pl = part_o.shape, part_lse.shape
        _check(len(po) == 4 and po[1] == hq and po[3] == d,
               "part_o workspace too small / wrong shape")
        _check(len(pl) == 3 and pl[1] == hq and pl[2] == po[2] and pl[0] >= po[0],
               "part_lse workspace shape mismatch")
        _check(o.shape == qs, "o must have q's shape")
        slots = int(max_splits) if grid_slots is None else int(grid_slots)
        order = self._order_ptr(wg_order, b * slots)
        _check(workers == 0 or wg_order is not None, "a worker launch needs wg_order")
        plan = (kv_indptr.data_ptr(), kv_indices.data_ptr(), _ptr(num_splits), b, hq, hkv, d,
                num_slots, int(max_splits), int(fixed_split_size), int(segment_size), slots,
                int(variant), order, float(sm_scale), part_o.data_ptr(), part_lse.data_ptr(),
                po[0], po[2], o.data_ptr(), int(workers))
        if kv_scales is not None:
            self._launch(q.get_device(), "sid_flash_decode_fp8_fwd", q.data_ptr(), k_cache.data_ptr(),
                         v_cache.data_ptr(), kv_scales.data_ptr(), *plan)
            return
        self._call("sid_flash_decode_workers_fwd", q.data_ptr(), k_cache.data_ptr(),
                   v_cache.data_ptr(), *plan, _stream(q))

    def flash_decode_fwd_noalloc(self, q, k_cache, v_cache, kv_indptr, kv_indices, num_splits,
                                 max_splits: int, fixed_split_size: int, sm_scale: float, o,
                                 segment_size: int = 0, grid_slots: int | None = None,
                                 variant: int = 0, wg_order=None) -> None:
        """flash_decode_fwd with the split partials in the library's static per-GPU scratch
        (no workspace argument, nothing allocated). Calls that overlap on one GPU race."""
        _gpu(q, "q", torch.bfloat16)
        _check(q.dim() == 3, "q must be [B, HQ, D]")
        b, hq, d = q.shape
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
            _gpu(t, name, torch.bfloat16)
            if not (t.dim() == 3 and t.shape[2] == d):
                raise RuntimeError(f"{name} must be [slots, HKV, {d}]")
        _check(k_cache.shape == v_cache.shape, "k_cache and v_cache shapes differ")
        _gpu(kv_indptr, "kv_indptr", torch.int32)
        _check(kv_indptr.numel() == b + 1, "kv_indptr must have B+1 entries")
        _gpu(kv_indices, "kv_indices", torch.int32)
        if num_splits is not None:  # None: derived on the device from the lengths
            _gpu(num_splits, "num_splits", torch.int32)
            _check(num_splits.numel() == b, "num_splits must have B entries")
        _gpu(o, "o", torch.bfloat16)
        _check(o.shape == q.shape, "o must have q's shape")
        slots = int(max_splits) if grid_slots is None else int(grid_slots)
        order = self._order_ptr(wg_order, b * slots)
        self._call("sid_flash_decode_segments_fwd_noalloc", q.data_ptr(), k_cache.data_ptr(),
                   v_cache.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(),
                   _ptr(num_splits), b, hq, k_cache.shape[1], d, k_cache.shape[0],
                   int(max_splits), int(fixed_split_size), int(segment_size), slots,
                   int(variant), order, float(sm_scale), o.data_ptr(), _stream(q))

    @staticmethod
    def _order_ptr(wg_order, n: int) -> int:
        if wg_order is None:
            return 0
        _gpu(wg_order, "wg_order", torch.int32)
        _check(wg_order.numel() >= n, "wg_order must have B * grid_slots entries")
        return wg_order.data_ptr()

    def reshape_and_cache(self, k, v, k_cache, v_cache, slot_mapping) -> None:
        _gpu(k, "k", torch.bfloat16)
        _gpu(v, "v", torch.bfloat16)
        ks, cs = k.shape, k_cache.shape
        _check(v.shape == ks, "v must have k's shape")
        _gpu(k_cache, "k_cache", torch.bfloat16)
        _gpu(v_cache, "v_cache", torch.bfloat16)
        _check(cs == v_cache.shape and len(cs) == 3, "bad cache shapes")
        _check(len(ks) == 3 and ks[1:] == cs[1:], "k must be [T, HKV, D] matching the cache")
        _gpu(slot_mapping, "slot_mapping", torch.int64)
        _check(slot_mapping.numel() == ks[0], "slot_mapping must have T entries")
        if ks[0] == 0:
            return
        self._call("sid_reshape_and_cache", k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
                   v_cache.data_ptr(), slot_mapping.data_ptr(), ks[0], cs[1], cs[2],
                   cs[0], _stream(k))

    # ---- 8-bit pool ----------------------------------------------------------------------

    def reshape_and_cache_fp8(self, k, v, k_cache, v_cache, kv_scales, slot_mapping) -> None:
        for name, x in (("k", k), ("v", v)):
            if not (isinstance(x, torch.Tensor) and x.is_cuda and x.dtype is torch.bfloat16):
                raise RuntimeError(f"{name} must be a bf16 GPU tensor")
        xs, device = k.shape, k.get_device()
        if len(xs) != 3 or v.shape != xs:
            raise RuntimeError("k must be [T, HKV, D], and v must have k's shape")
        t, hkv, d = xs
        cs = _pool8(k_cache, v_cache, kv_scales, d, device)
        if hkv != cs[1]:
            raise RuntimeError("k must be [T, HKV, D] matching the cache")
        _gpu(slot_mapping, "slot_mapping", torch.int64)
        if slot_mapping.numel() != t:
            raise RuntimeError("slot_mapping must have T entries")
        if v.get_device() != device or slot_mapping.get_device() != device:
            _same_device(device, v, slot_mapping)
        if t == 0:
            return
        sk, sv = k.stride(), v.stride()
        for name, s in (("k", sk), ("v", sv)):  # heads and dims dense, any token stride
            if s[2] != 1 or (s[1] != d and hkv > 1):
                raise RuntimeError(f"{name}'s heads and dims must be contiguous")
        one = t == 1
        self._launch(device, "sid_reshape_and_cache_fp8", k.data_ptr(), hkv * d if one else sk[0],
                     v.data_ptr(), hkv * d if one else sv[0], k_cache.data_ptr(),
                     v_cache.data_ptr(), kv_scales.data_ptr(), slot_mapping.data_ptr(), t, hkv, d,
                     cs[0])

    def gather_cache_fp8(self, k_cache, v_cache, kv_scales, slots, k, v) -> None:
        _gpu(slots, "slots", torch.int64)
        _gpu(k, "k", torch.bfloat16)
        _gpu(v, "v", torch.bfloat16)
        xs, device = k.shape, slots.get_device()
        if len(xs) != 3 or v.shape != xs:
            raise RuntimeError("k and v must both be [N, HKV, D]")
        cs = _pool8(k_cache, v_cache, kv_scales, xs[2], device)
        if xs[0] != slots.numel() or xs[1] != cs[1]:
            raise RuntimeError("k must be [N, HKV, D] matching the slots and the cache")
        _same_device(device, k, v)
        if xs[0] == 0:
            return
        self._launch(device, "sid_gather_cache_fp8", k_cache.data_ptr(), v_cache.data_ptr(),
                     kv_scales.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), *xs,
                     cs[0])

    # ---- the rest of the decode path ----------------------------------------------------

    def extend_attention_workspace_bytes(self, batch, total_q, hq, hkv, max_extend_len,
                                         max_kv_len, fp8: bool = False) -> int:
        fn = (self.lib.sid_extend_attention_fp8_workspace_bytes if fp8
              else self.lib.sid_extend_attention_workspace_bytes)
        return int(fn(batch, total_q, hq, hkv, max_extend_len, max_kv_len))

    def extend_attention_fwd(self, q, k_buffer, v_buffer, qo_indptr, kv_indptr, kv_indices,
                             max_extend_len: int, sm_scale: float, o, max_kv_len: int,
                             workspace=None, kv_scales=None) -> None:
        """kv_scales: the buffers are an 8-bit pool (sid_extend_attention_fp8_fwd)."""
        _gpu(q, "q_extend", torch.bfloat16)
        _check(q.dim() == 3, "q_extend must be [Text, HQ, D]")
        if kv_scales is not None:
            _pool8(k_buffer, v_buffer, kv_scales, q.shape[2], q.get_device())
            _same_device(q.get_device(), qo_indptr, kv_indptr, kv_indices, o, workspace)
        else:
            _gpu(k_buffer, "k_buffer", torch.bfloat16)
            _gpu(v_buffer, "v_buffer", torch.bfloat16)
            _check(k_buffer.shape == v_buffer.shape and k_buffer.dim() == 3
                   and k_buffer.shape[2] == q.shape[2], "bad KV buffer shapes")
        _gpu(qo_indptr, "qo_indptr", torch.int32)
        _gpu(kv_indptr, "kv_indptr", torch.int32)
        _gpu(kv_indices, "kv_indices", torch.int32)
        _check(qo_indptr.numel() == kv_indptr.numel(), "qo_indptr/kv_indptr length mismatch")
        _gpu(o, "o", torch.bfloat16)
        _check(o.shape == q.shape, "o must have q's shape")
        ws_ptr, ws_bytes = None, 0
        if workspace is not None:
            _gpu(workspace, "workspace", torch.uint8)
            ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel()
        rest = (qo_indptr.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(),
                qo_indptr.numel() - 1, q.shape[0], q.shape[1], k_buffer.shape[1], q.shape[2],
                k_buffer.shape[0], int(max_extend_len), int(max_kv_len), float(sm_scale), ws_ptr,
                ws_bytes, o.data_ptr())
        if kv_scales is not None:
            self._launch(q.get_device(), "sid_extend_attention_fp8_fwd", q.data_ptr(), k_buffer.data_ptr(),
                         v_buffer.data_ptr(), kv_scales.data_ptr(), *rest)
            return
        self._call("sid_extend_attention_fwd", q.data_ptr(), k_buffer.data_ptr(),
                   v_buffer.data_ptr(), *rest, _stream(q))

    def rmsnorm(self, x, w, out, eps: float) -> None:
        _gpu(x, "x", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        hidden = x.shape[-1]
        _check(w.numel() == hidden and out.shape == x.shape, "rmsnorm shape mismatch")
        self._call("sid_rmsnorm", x.data_ptr(), w.data_ptr(), out.data_ptr(),
                   x.numel() // max(hidden, 1), hidden, float(eps), _stream(x))

    def fused_add_rmsnorm(self, x, residual, w, eps: float) -> None:
        _gpu(x, "x", torch.bfloat16)
        _gpu(residual, "residual", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        hidden = x.shape[-1]
        _check(residual.shape == x.shape and w.numel() == hidden, "fused_add_rmsnorm shape mismatch")
        self._call("sid_fused_add_rmsnorm", x.data_ptr(), residual.data_ptr(), w.data_ptr(),
                   x.numel() // max(hidden, 1), hidden, float(eps), _stream(x))

    def rope_apply(self, q, k, positions, cos_sin) -> None:
        _gpu(q, "q", torch.bfloat16)
        _gpu(k, "k", torch.bfloat16)
        _gpu(positions, "positions", torch.int64)
        _gpu(cos_sin, "cos_sin", torch.float32)
        t, hq, d = q.shape
        _check(k.dim() == 3 and k.shape[0] == t and k.shape[2] == d, "k must be [T, HKV, D]")
        _check(positions.numel() == t, "positions must have T entries")
        _check(cos_sin.dim() == 2 and cos_sin.shape[1] == d, "cos_sin must be [max_pos, D]")
        self._call("sid_rope_apply", q.data_ptr(), k.data_ptr(), positions.data_ptr(),
                   cos_sin.data_ptr(), t, hq, k.shape[1], d, cos_sin.shape[0], _stream(q))

    def linear(self, x, w, bias, y, out_fp32: bool) -> None:
        m, k, n = self._linear_check(x, w)
        if bias is not None:
            _gpu(bias, "bias", torch.bfloat16)
            _check(bias.numel() == n, "bias must have N entries")
        _gpu(y, "out", torch.float32 if out_fp32 else torch.bfloat16)
        _check(tuple(y.shape) == (m, n), "out must be [M, N]")
        self._call("sid_linear", x.data_ptr(), x.stride(0) if m > 1 else k, w.data_ptr(),
                   bias.data_ptr() if bias is not None else None, y.data_ptr(), m, n, k,
                   1 if out_fp32 else 0, _stream(x))

    def linear_partials(self, x, w, partials) -> None:
        m, k, n = self._linear_check(x, w)
        _gpu(partials, "partials", torch.float32)
        _check(tuple(partials.shape) == (k // 256, m, n), "partials must be [K/256, M, N]")
        self._call("sid_linear_partials", x.data_ptr(), x.stride(0) if m > 1 else k,
                   w.data_ptr(), partials.data_ptr(), m, n, k, _stream(x))

    def linear_argmax_workspace_bytes(self, m: int) -> int:
        return int(self.lib.sid_linear_argmax_workspace_bytes(m))

    def linear_argmax(self, x, w, bias, logits, workspace, out) -> None:
        m, k, n = self._linear_check(x, w)
        if bias is not None:
            _gpu(bias, "bias", torch.bfloat16)
            _check(bias.numel() == n, "bias must have N entries")
        if logits is not None:
            _gpu(logits, "logits", torch.float32)
            _check(tuple(logits.shape) == (m, n), "logits must be [M, N]")
        _gpu(workspace, "workspace")
        _gpu(out, "out", torch.int64)
        _check(out.numel() == m, "out must have M entries")
        self._call("sid_linear_argmax", x.data_ptr(), x.stride(0) if m > 1 else k, w.data_ptr(),
                   bias.data_ptr() if bias is not None else None,
                   logits.data_ptr() if logits is not None else None, m, n, k,
                   workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                   out.data_ptr(), _stream(x))

    def linear_sample_workspace_bytes(self, m: int) -> int:
        return int(self.lib.sid_linear_sample_workspace_bytes(m))

    def linear_sample(self, x, w, temperatures, seeds, positions, workspace, out,
                      recompute_all: bool = False, tiles=None, logits=None) -> None:
        """tiles: None = grouping by row count; True = 128-column tiles; False = streaming
        waves."""
        m, k, n = self._linear_check(x, w)
        if logits is not None:
            _gpu(logits, "logits", torch.float32)
            _check(tuple(logits.shape) == (m, n), "logits must be [M, N]")
        for name, t, dt in (("temperatures", temperatures, torch.float32),
                            ("seeds", seeds, torch.int64), ("positions", positions, torch.int64),
                            ("out", out, torch.int64)):
            _gpu(t, name, dt)
            _check(t.numel() == m, f"{name} must have M entries")
        _gpu(workspace, "workspace")
        self._call("sid_linear_sample", x.data_ptr(), x.stride(0) if m > 1 else k, w.data_ptr(),
                   m, n, k, temperatures.data_ptr(), seeds.data_ptr(), positions.data_ptr(),
                   workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                   out.data_ptr(), logits.data_ptr() if logits is not None else None,
                   int(recompute_all) | {None: 0, True: 2, False: 4}[tiles], _stream(x))

    @staticmethod
    def _linear_check(x, w):
        _check(x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1,
               "x must be a 2-D bf16 GPU tensor with unit column stride")
        _gpu(w, "weight", torch.bfloat16)
        m, k = x.shape
        _check(w.dim() == 2 and w.shape[1] == k, f"weight must be [N, {k}]")
        return m, k, w.shape[0]

    def fused_add_rmsnorm_partials(self, partials, residual, w, out, eps: float) -> None:
        _gpu(partials, "partials", torch.float32)
        _gpu(residual, "residual", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        nch, rows, hidden = partials.shape
        _check(tuple(residual.shape) == (rows, hidden) and out.shape == residual.shape
               and w.numel() == hidden, "fused_add_rmsnorm_partials shape mismatch")
        self._call("sid_fused_add_rmsnorm_partials", partials.data_ptr(), nch, residual.data_ptr(),
                   w.data_ptr(), out.data_ptr(), rows, hidden, float(eps), _stream(out))

    def silu_mul_partials(self, partials, out) -> None:
        _gpu(partials, "partials", torch.float32)
        _gpu(out, "out", torch.bfloat16)
        nch, t, two_i = partials.shape
        _check(two_i % 2 == 0 and tuple(out.shape) == (t, two_i // 2), "silu_mul_partials shape")
        self._call("sid_silu_mul_partials", partials.data_ptr(), nch, out.data_ptr(), t,
                   two_i // 2, _stream(out))

    def qkv_post(self, qkv, partials, q_norm, k_norm, eps: float, positions, cos_sin, slots,
                 q_out, k_cache, v_cache, kv_scales=None) -> None:
        """kv_scales: the caches are an 8-bit pool (sid_qkv_post_fp8)."""
        _check((qkv is None) != (partials is None), "give exactly one of qkv and partials")
        if qkv is not None:
            _gpu(qkv, "qkv", torch.bfloat16)
            t, width, nch = qkv.shape[0], qkv.shape[1], 0
        else:
            _gpu(partials, "partials", torch.float32)
            nch, t, width = partials.shape
        usual = kv_scales is not None and _usual_qkv(q_out, q_norm, k_norm, positions, cos_sin, slots)
        if not usual:
            _gpu(q_out, "q_out", torch.bfloat16)
        _check(q_out.dim() == 3 and q_out.shape[0] == t, "q_out must be [T, HQ, D]")
        hq, d = q_out.shape[1], q_out.shape[2]
        self._cache_operands(k_cache, v_cache, kv_scales, d, q_out)
        hkv = k_cache.shape[1]
        _check(width == (hq + 2 * hkv) * d, "projection width != (HQ + 2*HKV) * D")
        if not usual:
            _gpu(q_norm, "q_norm", torch.bfloat16)
            _gpu(k_norm, "k_norm", torch.bfloat16)
            _gpu(positions, "positions", torch.int64)
            _gpu(slots, "slots", torch.int64)
            _gpu(cos_sin, "cos_sin", torch.float32)
        _check(positions.numel() == t and slots.numel() == t, "positions/slots must have T entries")
        args = (_ptr(qkv), _ptr(partials), nch, t, hq, hkv, d, q_norm.data_ptr(),
                k_norm.data_ptr(), float(eps), positions.data_ptr(), cos_sin.data_ptr(),
                cos_sin.shape[0], slots.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(),
                v_cache.data_ptr())
        if kv_scales is not None:
            if usual:
                _same_device(q_out.get_device(), qkv, partials)
            else:
                _same_device(q_out.get_device(), qkv, partials, q_norm, k_norm, positions, cos_sin,
                             slots)
            self._launch(q_out.get_device(), "sid_qkv_post_fp8", *args, kv_scales.data_ptr(), k_cache.shape[0])
            return
        self._call("sid_qkv_post", *args, k_cache.shape[0], _stream(q_out))

    @staticmethod
    def _cache_operands(k_cache, v_cache, kv_scales, d: int, q) -> None:
        if kv_scales is not None:
            _pool8(k_cache, v_cache, kv_scales, d, q.get_device())
            return
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            _gpu(c, name, torch.bfloat16)
            _check(c.dim() == 3 and c.shape[2] == d, f"{name} must be [S, HKV, D]")

    def linear_residual(self, x, w, residual, r32) -> None:
        """residual, r32 <- r = residual + bf16(x @ w^T) (fp32 r; residual = bf16(r))."""
        m, k, n = self._linear_check(x, w)
        _gpu(residual, "residual", torch.bfloat16)
        _gpu(r32, "r32", torch.float32)
        _check(tuple(residual.shape) == (m, n) and tuple(r32.shape) == (m, n),
               "residual / r32 must be [M, N]")
        self._call("sid_linear_residual", x.data_ptr(), x.stride(0), w.data_ptr(),
                   residual.data_ptr(), r32.data_ptr(), m, n, k, _stream(r32))

    @staticmethod
    def _norm_src(src):
        _check(src.is_cuda and src.dim() == 2 and src.is_contiguous()
               and src.dtype in (torch.float32, torch.bfloat16),
               "norm source must be a contiguous fp32 or bf16 [M, hidden] GPU tensor")
        return int(src.dtype == torch.float32)

    def rmsnorm_linear_silu_mul(self, src, norm_w, eps: float, w, out) -> None:
        """out <- silu_mul(bf16(rmsnorm(src) * norm_w) @ w^T), w = [gate rows | up rows]."""
        f32 = self._norm_src(src)
        _gpu(norm_w, "norm weight", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        m, hidden = src.shape
        _check(w.dim() == 2 and w.shape[1] == hidden and w.shape[0] % 2 == 0
               and norm_w.numel() == hidden, "rmsnorm_linear_silu_mul shapes")
        inter = w.shape[0] // 2
        _check(tuple(out.shape) == (m, inter), "out must be [M, I]")
        self._call("sid_rmsnorm_linear_silu_mul", src.data_ptr(), f32, norm_w.data_ptr(),
                   float(eps), w.data_ptr(), out.data_ptr(), m, hidden, inter, _stream(out))

    def rmsnorm_qkv_post(self, src, norm_w, eps: float, w, q_norm, k_norm, positions, cos_sin,
                         slots, q_out, k_cache, v_cache, kv_scales=None) -> None:
        """qkv_post over bf16(rmsnorm(src) * norm_w) @ w^T (one launch); kv_scales: the caches
        are an 8-bit pool (sid_rmsnorm_qkv_post_fp8)."""
        f32 = self._norm_src(src)
        m, hidden = src.shape
        _gpu(norm_w, "norm weight", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        _gpu(q_out, "q_out", torch.bfloat16)
        _check(q_out.dim() == 3 and q_out.shape[0] == m, "q_out must be [M, HQ, D]")
        hq, d = q_out.shape[1], q_out.shape[2]
        self._cache_operands(k_cache, v_cache, kv_scales, d, q_out)
        hkv = k_cache.shape[1]
        _check(w.dim() == 2 and w.shape[0] == (hq + 2 * hkv) * d and w.shape[1] == hidden
               and norm_w.numel() == hidden, "qkv weight must be [(HQ + 2*HKV) * D, hidden]")
        _gpu(q_norm, "q_norm", torch.bfloat16)
        _gpu(k_norm, "k_norm", torch.bfloat16)
        _gpu(positions, "positions", torch.int64)
        _gpu(slots, "slots", torch.int64)
        _gpu(cos_sin, "cos_sin", torch.float32)
        _check(positions.numel() == m and slots.numel() == m, "positions/slots must have M entries")
        args = (src.data_ptr(), f32, norm_w.data_ptr(), float(eps), w.data_ptr(), m, hidden, hq,
                hkv, d, q_norm.data_ptr(), k_norm.data_ptr(), positions.data_ptr(),
                cos_sin.data_ptr(), cos_sin.shape[0], slots.data_ptr(), q_out.data_ptr(),
                k_cache.data_ptr(), v_cache.data_ptr())
        if kv_scales is not None:
            _same_device(q_out.get_device(), src, norm_w, w, q_norm, k_norm, positions, cos_sin, slots)
            self._launch(q_out.get_device(), "sid_rmsnorm_qkv_post_fp8", *args, kv_scales.data_ptr(),
                         k_cache.shape[0])
            return
        self._call("sid_rmsnorm_qkv_post", *args, k_cache.shape[0], _stream(q_out))

    def pack_decode_weight(self, w, packed, gate_up: bool) -> None:
        """packed <- w [N, K] in the fragment-packed order of the decode-chain kernels."""
        _gpu(w, "weight", torch.bfloat16)
        _gpu(packed, "packed", torch.bfloat16)
        _check(w.dim() == 2 and packed.shape == w.shape, "packed must have the weight's shape")
        self._call("sid_pack_decode_weight", w.data_ptr(), packed.data_ptr(), w.shape[0],
                   w.shape[1], int(gate_up), _stream(packed))

    def rmsnorm_f32(self, x, w, out, eps: float) -> None:
        """out <- bf16(rmsnorm(x) * w) for fp32 rows x (rmsnorm's bits)."""
        _gpu(x, "x", torch.float32)
        _gpu(w, "weight", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        _check(x.dim() == 2 and out.shape == x.shape and w.numel() == x.shape[1], "rmsnorm_f32 shapes")
        self._call("sid_rmsnorm_f32", x.data_ptr(), w.data_ptr(), out.data_ptr(), x.shape[0],
                   x.shape[1], float(eps), _stream(out))

    def linear_silu_mul(self, x, w, out) -> None:
        _gpu(x, "x", torch.bfloat16)
        _gpu(w, "weight", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        _check(x.dim() == 2 and w.dim() == 2 and w.shape[1] == x.shape[1], "x / weight shapes")
        _check(w.shape[0] % 2 == 0 and tuple(out.shape) == (x.shape[0], w.shape[0] // 2),
               "linear_silu_mul: out must be [M, N/2]")
        self._call("sid_linear_silu_mul", x.data_ptr(), w.data_ptr(), out.data_ptr(), x.shape[0],
                   x.shape[1], w.shape[0] // 2, _stream(out))

    def silu_mul(self, gate_up, out) -> None:
        _gpu(gate_up, "gate_up", torch.bfloat16)
        _gpu(out, "out", torch.bfloat16)
        t, two_i = gate_up.shape
        _check(two_i % 2 == 0 and tuple(out.shape) == (t, two_i // 2), "silu_mul shape mismatch")
        self._call("sid_silu_mul", gate_up.data_ptr(), out.data_ptr(), t, two_i // 2, _stream(out))

    def gather_rows(self, table, idx, out) -> None:
        _gpu(table, "table", torch.bfloat16)
        _gpu(idx, "indices", torch.int64)
        _gpu(out, "out", torch.bfloat16)
        _check(out.shape[0] == idx.numel() and out.shape[1:] == table.shape[1:],
               "gather_rows shape mismatch")
        row = table[0].numel() if table.shape[0] > 0 else out[0].numel()
        self._call("sid_gather_rows", table.data_ptr(), idx.data_ptr(), out.data_ptr(),
                   idx.numel(), row, table.shape[0], _stream(out))

    def argmax_rows(self, logits, out) -> None:
        _check(logits.is_cuda and logits.dtype == torch.float32 and logits.dim() == 2
               and logits.stride(1) == 1, "logits must be 2-D fp32 on the GPU, unit column stride")
        _gpu(out, "out", torch.int64)
        _check(out.numel() == logits.shape[0], "out must have one entry per row")
        self._call("sid_argmax_rows", logits.data_ptr(), logits.stride(0), out.data_ptr(),
                   logits.shape[0], logits.shape[1], _stream(out))

    def sample_rows(self, logits, temperatures, top_ks, top_ps, seeds, positions, out) -> None:
        _check(logits.is_cuda and logits.dtype == torch.float32 and logits.dim() == 2
               and logits.stride(1) == 1, "logits must be 2-D fp32 on the GPU, unit column stride")
        r, v = logits.shape
        for name, t, dt in (("temperatures", temperatures, torch.float32),
                            ("top_ks", top_ks, torch.int64), ("top_ps", top_ps, torch.float32),
                            ("seeds", seeds, torch.int64), ("positions", positions, torch.int64),
                            ("out", out, torch.int64)):
            _gpu(t, name, dt)
            if t.numel() != r:
                raise RuntimeError(f"{name} must have one entry per row")
        if r == 0:
            return
        ws = torch.empty(int(self.lib.sid_sample_workspace_bytes(r, v)), dtype=torch.uint8,
                         device=logits.device)
        self._call("sid_sample_rows", logits.data_ptr(), logits.stride(0), temperatures.data_ptr(),
                   top_ks.data_ptr(), top_ps.data_ptr(), seeds.data_ptr(), positions.data_ptr(),
                   r, v, ws.data_ptr(), ws.numel(), out.data_ptr(), _stream(logits))

    def build_paged_decode_indices(self, block_tables, page_size: int, rows, new_slots,
                                   kv_indptr, kv_indices) -> None:
        _gpu(block_tables, "block_tables", torch.int32)
        _check(block_tables.dim() == 2, "block_tables must be [rows, max_pages]")
        _gpu(rows, "rows", torch.int64)
        _gpu(new_slots, "new_slots", torch.int64)
        _check(new_slots.numel() == rows.numel(), "new_slots must have B entries")
        _gpu(kv_indptr, "kv_indptr", torch.int32)
        _gpu(kv_indices, "kv_indices", torch.int32)
        _check(kv_indptr.numel() == rows.numel() + 1, "kv_indptr must have B+1 entries")
        self._call("sid_build_paged_decode_indices", block_tables.data_ptr(),
                   block_tables.shape[1], block_tables.shape[0], int(page_size), rows.data_ptr(),
                   new_slots.data_ptr(), kv_indptr.data_ptr(), kv_indices.data_ptr(),
                   rows.numel(), _stream(rows))
