"""Python binding of libmi355x.so (the gfx950 prefill backend).

Two layers, both plain ctypes over the C ABI in include/:
  * the kernel entry points of mi355x_kernels.h (device pointers, sizes, a HIP stream), with
    torch-tensor helpers: torch only allocates device memory and names the stream;
  * the backend's host layer of mi355x_backend.h (claim rules, graph compute, counters), which
    mirrors ggml-rocket.h.

There is no fallback: if the shared library is missing, `lib()` raises.
"""
from __future__ import annotations

import ctypes
import numbers
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libmi355x.so")

F32, F16, Q8_0, Q4_K, Q6_K, I32, I64, BF16, MXFP4 = 0, 1, 8, 12, 14, 26, 27, 30, 39
Q4_0, Q4_1, Q5_0, Q2_K, Q5_K = 2, 3, 6, 10, 13
F16_T = 0x101   # the library's tiled fp16 layout (16 x 32 tiles of 1 KB); not a ggml type
Q4_K_X = 0x10C  # Q4_K blocks regrouped by 32 rows, for expert stacks (MUL_MAT_ID); not a ggml type
Q8_0_X = 0x108  # Q8_0 blocks regrouped by 32 rows (quant plane, then scale plane); expert stacks only
MXFP4_X = 0x127  # MXFP4 blocks regrouped by 32 rows, as Q8_0_X; expert stacks only
Q6_K_X = 0x10E  # Q6_K blocks regrouped by 32 rows (four planes); expert stacks only
OK, E_ARG, E_DEVICE, E_UNSUPPORTED, E_NOMEM, E_IDS = 0, -1, -2, -3, -4, -5   # mi355x_status
BLOCK = {F16: 1, F32: 1, BF16: 1, Q8_0: 32, Q4_0: 32, Q4_K: 256, Q5_K: 256, Q6_K: 256, MXFP4: 32}
TYPE_SIZE = {F16: 2, F32: 4, BF16: 2, Q8_0: 34, Q4_0: 18, Q4_K: 144, Q5_K: 176, Q6_K: 210, MXFP4: 17}

_lib = None


class MI355XError(RuntimeError):
    pass


class GemmOut(ctypes.Structure):
    _fields_ = [("w_dev", ctypes.c_void_p), ("rows_total", ctypes.c_int64),
                ("row0", ctypes.c_int64), ("N", ctypes.c_int64),
                ("c_dev", ctypes.c_void_p), ("ldc", ctypes.c_int64)]


class DeviceInfo(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 64), ("compute_units", ctypes.c_int),
                ("lds_bytes_per_block", ctypes.c_int), ("clock_khz", ctypes.c_int),
                ("hbm_total", ctypes.c_size_t), ("hbm_free", ctypes.c_size_t)]


class FaArgs(ctypes.Structure):
    _fields_ = [("q_dev", ctypes.c_void_p), ("q_nb1", ctypes.c_int64), ("q_nb2", ctypes.c_int64),
                ("k_dev", ctypes.c_void_p), ("k_nb1", ctypes.c_int64), ("k_nb2", ctypes.c_int64),
                ("v_dev", ctypes.c_void_p), ("v_nb1", ctypes.c_int64), ("v_nb2", ctypes.c_int64),
                ("mask_dev", ctypes.c_void_p), ("mask_nb1", ctypes.c_int64),
                ("dst_dev", ctypes.c_void_p), ("dst_nb1", ctypes.c_int64), ("dst_nb2", ctypes.c_int64),
                ("D", ctypes.c_int), ("DV", ctypes.c_int), ("T", ctypes.c_int), ("H", ctypes.c_int),
                ("KV", ctypes.c_int), ("HK", ctypes.c_int),
                ("scale", ctypes.c_float), ("max_bias", ctypes.c_float), ("softcap", ctypes.c_float)]


class MoeArgs(ctypes.Structure):
    _fields_ = [("wtype", ctypes.c_int),
                ("as_dev", ctypes.c_void_p), ("n_expert", ctypes.c_int64), ("N", ctypes.c_int64),
                ("K", ctypes.c_int64),
                ("b_dev", ctypes.c_void_p), ("ne11", ctypes.c_int64), ("b_nb1", ctypes.c_int64),
                ("b_nb2", ctypes.c_int64),
                ("ids_dev", ctypes.c_void_p), ("n_used", ctypes.c_int64), ("ids_nb0", ctypes.c_int64),
                ("ids_nb1", ctypes.c_int64),
                ("n_tokens", ctypes.c_int64),
                ("dst_dev", ctypes.c_void_p), ("dst_nb1", ctypes.c_int64), ("dst_nb2", ctypes.c_int64)]


class KvRows(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int), ("q_dev", ctypes.c_void_p), ("d_dev", ctypes.c_void_p),
                ("n_rows", ctypes.c_int64), ("nb1", ctypes.c_int64), ("nb2", ctypes.c_int64),
                ("H", ctypes.c_int64), ("D", ctypes.c_int64),
                ("x_type", ctypes.c_int), ("x_dev", ctypes.c_void_p),
                ("x_nb1", ctypes.c_int64), ("x_nb2", ctypes.c_int64)]


class KvView(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int), ("q_dev", ctypes.c_void_p), ("d_dev", ctypes.c_void_p),
                ("nb1", ctypes.c_int64), ("nb2", ctypes.c_int64), ("nb3", ctypes.c_int64)]


class FaQArgs(ctypes.Structure):
    _fields_ = [("q_dev", ctypes.c_void_p), ("q_nb1", ctypes.c_int64), ("q_nb2", ctypes.c_int64), ("q_nb3", ctypes.c_int64),
                ("k", KvView), ("v", KvView),
                ("mask_dev", ctypes.c_void_p), ("mask_nb1", ctypes.c_int64), ("mask_nb3", ctypes.c_int64),
                ("dst_dev", ctypes.c_void_p), ("dst_nb1", ctypes.c_int64), ("dst_nb2", ctypes.c_int64), ("dst_nb3", ctypes.c_int64),
                ("q_type", ctypes.c_int), ("dst_type", ctypes.c_int),
                ("D", ctypes.c_int), ("DV", ctypes.c_int), ("T", ctypes.c_int), ("H", ctypes.c_int),
                ("KV", ctypes.c_int), ("HK", ctypes.c_int), ("S", ctypes.c_int),
                ("scale", ctypes.c_float), ("max_bias", ctypes.c_float), ("softcap", ctypes.c_float)]


class KvStepArgs(ctypes.Structure):
    _fields_ = [("table_dev", ctypes.c_void_p), ("table_nb", ctypes.c_int64), ("n_past_dev", ctypes.c_void_p),
                ("n_new_dev", ctypes.c_void_p), ("parent_dev", ctypes.c_void_p), ("parent_nb", ctypes.c_int64),
                ("n_table", ctypes.c_int64), ("S", ctypes.c_int), ("T", ctypes.c_int), ("page", ctypes.c_int)]


class KvAppendArgs(ctypes.Structure):
    _fields_ = [("step", KvStepArgs), ("k", KvRows), ("v", KvRows), ("k_nb3", ctypes.c_int64), ("v_nb3", ctypes.c_int64),
                ("q_dev", ctypes.c_void_p), ("q_nb1", ctypes.c_int64), ("q_nb2", ctypes.c_int64), ("q_nb3", ctypes.c_int64),
                ("qr_dev", ctypes.c_void_p), ("qr_nb1", ctypes.c_int64), ("qr_nb2", ctypes.c_int64), ("qr_nb3", ctypes.c_int64),
                ("q_type", ctypes.c_int), ("qr_type", ctypes.c_int), ("H", ctypes.c_int64), ("freq_dev", ctypes.c_void_p),
                ("pos_dev", ctypes.c_void_p), ("pos_nb", ctypes.c_int64), ("n_rot", ctypes.c_int), ("neox", ctypes.c_int),
                ("mscale", ctypes.c_float)]


class FaPArgs(ctypes.Structure):
    _fields_ = [("step", KvStepArgs), ("q_dev", ctypes.c_void_p), ("q_nb1", ctypes.c_int64), ("q_nb2", ctypes.c_int64),
                ("q_nb3", ctypes.c_int64), ("k", KvView), ("v", KvView), ("n_rows", ctypes.c_int64), ("dst_dev", ctypes.c_void_p),
                ("dst_nb1", ctypes.c_int64), ("dst_nb2", ctypes.c_int64), ("dst_nb3", ctypes.c_int64), ("q_type", ctypes.c_int),
                ("dst_type", ctypes.c_int), ("D", ctypes.c_int), ("DV", ctypes.c_int), ("H", ctypes.c_int), ("HK", ctypes.c_int),
                ("scale", ctypes.c_float), ("softcap", ctypes.c_float), ("max_kv", ctypes.c_int64), ("from_pages", ctypes.c_int)]


def lib():
    """Load the built backend library. Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise MI355XError(f"{LIB_PATH} is missing: build it first (python -c "
                          f"'import __graft_entry__ as g; g.build()')")
    L = ctypes.CDLL(LIB_PATH)
    i64, i32, vp, sz = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t
    f32 = ctypes.c_float
    L.mi355x_status_str.restype = ctypes.c_char_p
    L.mi355x_status_str.argtypes = [i32]
    L.mi355x_get_device_info.argtypes = [ctypes.POINTER(DeviceInfo)]
    L.mi355x_weight_bytes.restype = i64
    L.mi355x_weight_bytes.argtypes = [i32, i64, i64]
    L.mi355x_weight_pack.argtypes = [i32, vp, i64, i64, vp, vp]
    L.mi355x_weight_dequant_f16.argtypes = [i32, vp, i64, i64, vp, vp]
    L.mi355x_weight_f16_tiled.argtypes = [i32, vp, i64, i64, vp, vp]
    L.mi355x_pack_act.argtypes = [vp, i64, i64, i64, vp, vp, vp]
    L.mi355x_pack_act_tiled.argtypes = [vp, i64, i64, i64, vp, vp, vp]
    L.mi355x_gemm.argtypes = [i32, vp, vp, i64, i64, ctypes.POINTER(GemmOut), i32, vp]
    L.mi355x_gemm_workspace.restype = sz
    L.mi355x_gemm_workspace.argtypes = [i32, i64, i64, ctypes.POINTER(GemmOut), i32]
    L.mi355x_gemm_ws.argtypes = [i32, vp, vp, i64, i64, ctypes.POINTER(GemmOut), i32, vp, sz, i32, vp]
    L.mi355x_gemm_accumulates.argtypes = [i32, i64, i64, ctypes.POINTER(GemmOut), i32, sz]
    L.mi355x_pack_act_clear.argtypes = [i32, vp, i64, i64, i64, vp, vp, vp, i64, i64, vp]
    L.mi355x_mul_mat_workspace.restype = sz
    L.mi355x_mul_mat_workspace.argtypes = [i64, i64]
    L.mi355x_mul_mat_workspace_for.restype = sz
    L.mi355x_mul_mat_workspace_for.argtypes = [i32, i64, i64, i64]
    L.mi355x_mul_mat_decode_first.restype = i32
    L.mi355x_mul_mat_decode_first.argtypes = [i32, i64, i64, i64]
    L.mi355x_mul_mat.argtypes = [i32, vp, i64, i64, vp, i64, i64, vp, i64, vp, sz, vp]
    _bind_optional(L)
    _lib = L
    return L


def _bind_optional(L):
    """Entry points of later kernel families; bound when the library exports them."""
    i64, i32, vp, sz, f32 = ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_float
    if hasattr(L, "mi355x_flash_attn"):
        pa = ctypes.POINTER(FaArgs)
        L.mi355x_flash_attn_auto_split.restype = i32
        L.mi355x_flash_attn_auto_split.argtypes = [pa]
        L.mi355x_flash_attn_workspace.restype = sz
        L.mi355x_flash_attn_workspace.argtypes = [pa, i32]
        L.mi355x_flash_attn.argtypes = [pa, i32, vp, sz, vp]
        L.mi355x_flash_attn_ex.argtypes = [pa, i32, i32, vp, sz, vp]
    if hasattr(L, "mi355x_set_rows"):
        pq = ctypes.POINTER(FaQArgs)
        L.mi355x_set_rows.argtypes = [vp, i32, vp, i32, i64, vp, vp]
        L.mi355x_get_rows.argtypes = [vp, i32, vp, i32, i64, vp, vp]
        L.mi355x_flash_attn_q_workspace.restype = sz
        L.mi355x_flash_attn_q_workspace.argtypes = [pq, i32]
        L.mi355x_flash_attn_q.argtypes = [pq, i32, vp, sz, vp]
    if hasattr(L, "mi355x_kv_append"):
        pp, ps = ctypes.POINTER(FaPArgs), ctypes.POINTER(KvStepArgs)
        L.mi355x_kv_append.argtypes = [vp, vp, vp]
        L.mi355x_flash_attn_paged_workspace.restype = sz
        L.mi355x_flash_attn_paged_workspace.argtypes = [pp, i32]
        L.mi355x_flash_attn_paged.argtypes = [pp, i32, vp, sz, vp, vp]
        L.mi355x_kv_keep.argtypes = [ps, vp, i32, vp, i64, vp, i32, vp, vp]
    if hasattr(L, "mi355x_mul_mat_noalloc"):
        L.mi355x_mul_mat_noalloc.argtypes = [i32, vp, i64, i64, vp, i64, i64, vp, i64, vp]
    if hasattr(L, "mi355x_mul_mat_id"):
        pm = ctypes.POINTER(MoeArgs)
        L.mi355x_mul_mat_id_workspace.restype = sz
        L.mi355x_mul_mat_id_workspace.argtypes = [pm]
        L.mi355x_mul_mat_id.argtypes = [pm, vp, sz, vp, vp]


def check(status: int, what: str = "call"):
    if status != 0:
        msg = lib().mi355x_status_str(status).decode()
        raise MI355XError(f"{what}: status {status} ({msg})")


def status_str(status: int) -> str:
    return lib().mi355x_status_str(status).decode()


def device_info() -> dict:
    d = DeviceInfo()
    check(lib().mi355x_get_device_info(ctypes.byref(d)), "get_device_info")
    return {"name": d.name.decode(), "compute_units": d.compute_units,
            "lds_bytes_per_block": d.lds_bytes_per_block, "clock_khz": d.clock_khz,
            "hbm_total": d.hbm_total, "hbm_free": d.hbm_free}


# ---- torch helpers ------------------------------------------------------------------------

def _torch():
    import torch
    return torch


def stream_handle(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def weight_bytes(wtype: int, rows: int, K: int) -> int:
    return int(lib().mi355x_weight_bytes(wtype, rows, K))


def upload_weight(wtype: int, payload, rows: int, K: int, device="cuda"):
    """A ggml payload (numpy uint8 / uint16 / torch) -> its HBM layout, as a uint8 device tensor.
    Q4_K_X, Q8_0_X, Q6_K_X and MXFP4_X take the ggml blocks of their base type (rows % 32 == 0)
    and regroup them."""
    torch = _torch()
    import numpy as np
    if isinstance(payload, np.ndarray):
        raw = torch.from_numpy(np.ascontiguousarray(payload).view(np.uint8).reshape(-1)).to(device)
    else:
        raw = payload.contiguous().view(torch.uint8).reshape(-1).to(device)
    nbytes = weight_bytes(wtype, rows, K)
    if nbytes < 0 or raw.numel() != nbytes:
        raise MI355XError(f"payload of {raw.numel()} bytes is not {rows} rows of K={K} of type {wtype}")
    if wtype in (F16, Q4_K, Q5_K):
        return raw
    out = torch.empty(nbytes, dtype=torch.uint8, device=device)
    check(lib().mi355x_weight_pack(wtype, _ptr(raw), rows, K, _ptr(out), stream_handle()), "weight_pack")
    return out


def dequant_f16(wtype: int, w_dev, rows: int, K: int):
    torch = _torch()
    out = torch.empty((rows, K), dtype=torch.float16, device=w_dev.device)
    check(lib().mi355x_weight_dequant_f16(wtype, _ptr(w_dev), rows, K, _ptr(out), stream_handle()),
          "weight_dequant_f16")
    return out


def tile_f16(wtype: int, w_dev, rows: int, K: int):
    """A weight in HBM layout -> the tiled fp16 layout (F16_T), as a uint8 device tensor."""
    torch = _torch()
    out = torch.empty(weight_bytes(F16_T, rows, K), dtype=torch.uint8, device=w_dev.device)
    check(lib().mi355x_weight_f16_tiled(wtype, _ptr(w_dev), rows, K, _ptr(out), stream_handle()),
          "weight_f16_tiled")
    return out


def pack_act(x, tiled: bool = False):
    """F32 [M, K] -> (fp16 activations, row scales [M]). tiled: the F16_T layout over M rows,
    returned as [ceil(M/16)*16, K] (the padding rows are never read)."""
    torch = _torch()
    M, K = x.shape
    rows = (M + 15) // 16 * 16 if tiled else M
    a16 = torch.empty((rows, K), dtype=torch.float16, device=x.device)
    sc = torch.empty((M,), dtype=torch.float32, device=x.device)
    fn = lib().mi355x_pack_act_tiled if tiled else lib().mi355x_pack_act
    check(fn(_ptr(x), x.stride(0), M, K, _ptr(a16), _ptr(sc), stream_handle()), "pack_act")
    return a16, sc


def gemm(wtype: int, a16, scales, K: int, outs, split_workspace: bool = True):
    """outs: list of (w_dev, rows_total, row0, N, c_tensor). M = len(scales). With
    split_workspace, mi355x_gemm_ws with the workspace its fastest K split asks for; without,
    mi355x_gemm (K split at most two ways)."""
    arr = (GemmOut * len(outs))()
    for i, (w, rows_total, row0, N, c) in enumerate(outs):
        arr[i] = GemmOut(w.data_ptr(), rows_total, row0, N, c.data_ptr(), c.stride(0))
    M = scales.shape[0]
    if not split_workspace:
        check(lib().mi355x_gemm(wtype, _ptr(a16), _ptr(scales), M, K, arr, len(outs), stream_handle()), "gemm")
        return
    need = int(lib().mi355x_gemm_workspace(wtype, M, K, arr, len(outs)))
    ws = _torch().empty(max(need, 1), dtype=_torch().uint8, device=a16.device)
    check(lib().mi355x_gemm_ws(wtype, _ptr(a16), _ptr(scales), M, K, arr, len(outs), _ptr(ws), need, 0,
                               stream_handle()), "gemm_ws")


def mul_mat(wtype: int, w_dev, N: int, K: int, x, out=None, workspace=None):
    """dst[M, N] = x[M, K] . W[N, K]^T with W already in HBM layout."""
    torch = _torch()
    M = x.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=x.device)
    need = int(lib().mi355x_mul_mat_workspace_for(wtype, N, K, M))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    check(lib().mi355x_mul_mat(wtype, _ptr(w_dev), N, K, _ptr(x), x.stride(0), M, _ptr(out), out.stride(0),
                               _ptr(workspace), workspace.numel(), stream_handle()), "mul_mat")
    return out


def mul_mat_noalloc(wtype: int, w_dev, N: int, K: int, x, out):
    """mul_mat through mi355x_mul_mat_noalloc: the workspace is the library's static device
    scratch; `out` [M, >= N] is the caller's. Returns the status (no exception), so callers can
    check the size limit."""
    return lib().mi355x_mul_mat_noalloc(wtype, _ptr(w_dev), N, K, _ptr(x), x.stride(0), x.shape[0], _ptr(out),
                                        out.stride(0), stream_handle())


def _fa_args(q, k, v, mask, out, scale, softcap=0.0, max_bias=0.0):
    H, T, D = q.shape
    HK, KV, DV = v.shape
    return FaArgs(q.data_ptr(), q.stride(1), q.stride(0),
                  k.data_ptr(), k.stride(1), k.stride(0),
                  v.data_ptr(), v.stride(1), v.stride(0),
                  mask.data_ptr() if mask is not None else None, mask.stride(0) if mask is not None else 0,
                  out.data_ptr(), out.stride(1), out.stride(0),
                  D, DV, T, H, KV, HK, scale, max_bias, softcap)


def flash_attn_workspace(q, k, v, mask, out, scale: float = 1.0, softcap: float = 0.0, nsplit: int = 0) -> int:
    """Workspace bytes mi355x_flash_attn needs for these operands (0 for an unsupported op)."""
    return int(lib().mi355x_flash_attn_workspace(ctypes.byref(_fa_args(q, k, v, mask, out, scale, softcap)), nsplit))


FA_CLASSES_READY = 1


def flash_attn(q, k, v, mask, scale: float, softcap: float = 0.0, nsplit: int = 0, out=None,
               workspace=None, max_bias: float = 0.0, classes_ready: bool = False):
    """q [H, T, D] f32 (any strides with unit last-dim stride), k/v [HK, KV, D] fp16, mask
    [T', KV'] fp16 or None. Returns dst [T, H, D] f32. classes_ready: `workspace` holds the mask
    classes of an earlier call with the same mask, shapes and split (mi355x_flash_attn_ex)."""
    torch = _torch()
    H, T, D = q.shape
    HK, KV, DV = v.shape
    if out is None:
        out = torch.empty((T, H, DV), dtype=torch.float32, device=q.device)
    a = _fa_args(q, k, v, mask, out, scale, softcap, max_bias)
    need = int(lib().mi355x_flash_attn_workspace(ctypes.byref(a), nsplit))
    if need and (workspace is None or workspace.numel() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    wp = workspace.data_ptr() if need else None
    if classes_ready and workspace is None:
        raise MI355XError("flash_attn: classes_ready needs the workspace of the call that classified the mask")
    flags = FA_CLASSES_READY if classes_ready else 0
    check(lib().mi355x_flash_attn_ex(ctypes.byref(a), nsplit, flags, wp, need, stream_handle()), "flash_attn")
    return out


# ---- the quantized KV cache -----------------------------------------------------------------
# Decoding calls these once a layer and token, so they avoid what costs microseconds: a cache keeps its
# part of the C structs, and structs are filled in one call.

class KvCache:
    """A K or V cache on the device, of any leading dims: `q` holds the codes (Q8_0: int8 [..., D];
    Q4_0: uint8 [..., D / 2]; F16: the fp16 values, without `d`), `d` the blocks' fp16 scales
    [..., D / 32]. Both planes have the same element strides; permute and indexing of the leading dims
    give views."""

    __slots__ = ("type", "q", "d", "D", "shape", "nb", "dev", "_tail", "_rows", "_view")

    def __init__(self, ttype: int, q, d=None):
        torch = _torch()
        self.type, self.q, self.d = ttype, q, d
        want = {Q8_0: torch.int8, Q4_0: torch.uint8, F16: torch.float16}.get(ttype)
        if want is None or q.dtype != want or q.dim() < 2 or q.stride(-1) != 1:
            raise MI355XError(f"KvCache: type {ttype} does not hold codes of {q.dtype} {tuple(q.shape)}")
        per = 2 if ttype == Q4_0 else 1
        self.D = q.shape[-1] * per
        self.shape = tuple(q.shape[:-1]) + (self.D,)
        self.nb = tuple(s * per for s in q.stride()[:-1])
        self.dev = q.get_device()
        if ttype == F16:
            if d is not None:
                raise MI355XError("KvCache: an F16 cache has no scales")
        elif (d is None or d.dtype != torch.float16 or d.device != q.device or self.D % 32
              or tuple(d.shape) != self.shape[:-1] + (self.D // 32,) or (d.stride(-1) != 1 and d.shape[-1] > 1)
              or any(n > 1 and a != 32 * b for n, a, b in zip(q.shape[:-1], self.nb, d.stride()))):
            raise MI355XError("KvCache: the scales are not fp16 of the codes' shape and strides / 32")
        n, nb, qp, dp = len(self.shape), self.nb, q.data_ptr(), None if d is None else d.data_ptr()
        # the cache's part of mi355x_kv_rows ([rows, D] or [rows, H, D]) and of mi355x_fa_q_args ([(S,) HK, KV, D])
        self._tail = self.shape[1:]
        self._rows = {2: (ttype, qp, dp or 0, self.shape[0], nb[0], 0, 1, self.D),
                      3: (ttype, qp, dp or 0, self.shape[0], nb[0], nb[-1], self.shape[1], self.D)}.get(n)
        self._view = KvView(ttype, qp, dp, nb[-1], nb[-2], nb[0] if n == 4 else 0) if n in (3, 4) and d is not None else None

    def permute(self, *dims):
        """A view with the leading dims in another order; the last dim stays last."""
        lead = len(self.shape) - 1
        if len(dims) == lead:
            dims = dims + (lead,)
        if dims[-1] not in (lead, -1):
            raise MI355XError("KvCache.permute: the last dim stays last")
        return KvCache(self.type, self.q.permute(*dims), None if self.d is None else self.d.permute(*dims))

    def __getitem__(self, at):
        """A view by integers and slices of leading dims. Lists and tensors, which would copy, are refused."""
        ats = at if isinstance(at, tuple) else (at,)
        if len(ats) >= len(self.shape) or not all(isinstance(i, slice) or (isinstance(i, numbers.Integral) and not isinstance(i, bool)) for i in ats):
            raise MI355XError("KvCache: integers and slices of leading dims only")
        return KvCache(self.type, self.q[at], None if self.d is None else self.d[at])


def kv_cache(ttype: int, *shape, device="cuda") -> KvCache:
    """A cache of zeros of the logical shape [..., D]."""
    torch = _torch()
    lead, D = tuple(shape[:-1]), shape[-1]
    if ttype == F16:
        return KvCache(F16, torch.zeros(*lead, D, dtype=torch.float16, device=device))
    if ttype not in (Q8_0, Q4_0) or D % 32:
        raise MI355XError(f"kv_cache: type {ttype} does not hold rows of {D}")
    q = (torch.zeros(*lead, D, dtype=torch.int8, device=device) if ttype == Q8_0
         else torch.full((*lead, D // 2), 0x88, dtype=torch.uint8, device=device))
    return KvCache(ttype, q, torch.zeros(*lead, D // 32, dtype=torch.float16, device=device))


_plain = {}


def _plain_types():
    if not _plain:
        torch = _torch()
        _plain.update({torch.float32: F32, torch.float16: F16, torch.int32: I32, torch.int64: I64})
    return _plain


def _launch_stream(dev: int, what: str):
    """The current stream's handle, for tensors of the current device."""
    C = _torch()._C
    if dev < 0 or dev != C._cuda_getDevice():
        raise MI355XError(f"{what}: the tensors are not on the current GPU")
    return C._cuda_getCurrentRawStream(dev)


_KV_ROWS = struct.Struct("@iPPqqqqqiPqq")     # mi355x_kv_rows, field by field


def _kv_rows(caches, plain, n, what):
    """mi355x_kv_rows of caches [rows, H, D] or [rows, D] and their plain rows [n, H, D] or [n, D]."""
    types, out = _plain_types(), b""
    if not 1 <= len(caches) <= 4:
        raise MI355XError(f"{what}: one to four caches")
    for c, x in zip(caches, plain):
        stride, t, rows = x.stride(), types.get(x.dtype), c._rows
        if rows is None or x.shape != (n, *c._tail) or stride[-1] != 1 or (t != F32 and t != F16) or x.get_device() != c.dev:
            raise MI355XError(f"{what}: rows {x.dtype} {tuple(x.shape)} do not fit {n} rows of a cache {c.shape}")
        out += _KV_ROWS.pack(*rows, t, x.data_ptr(), stride[0], stride[1] if len(stride) == 3 else 0)
    return out


def _kv_index(idx, n, dev, what):
    """(address, ggml type, count) of the row indices."""
    if idx is None:
        return None, I32, n
    t = _plain_types().get(idx.dtype)
    if t not in (I32, I64) or idx.dim() != 1 or not idx.is_contiguous() or idx.get_device() != dev:
        raise MI355XError(f"{what}: indices are int32 or int64, contiguous, on the cache's device")
    return idx.data_ptr(), t, idx.shape[0]


def _kv_err(err, dev, what):
    if err is None:
        return None
    if _plain_types().get(err.dtype) != I32 or err.get_device() != dev or err.numel() < 1:
        raise MI355XError(f"{what}: err is an int32 on the cache's device")
    return err.data_ptr()


def set_rows(pairs, idx=None, err=None):
    """pairs: (cache, x) for up to four caches [rows, H, D] (or [rows, D]) and plain rows x [n, H, D]
    (F32 or F16): x[i] is quantized into cache row idx[i] (int32 or int64 [n]; None: i), one launch
    for every 16384 rows. err: a device int32 that an index out of range sets to 1. The caches must not overlap."""
    if not pairs:
        raise MI355XError("set_rows: one to four caches")
    caches, plain = zip(*pairs)
    dev = caches[0].dev
    ip, it, n = _kv_index(idx, plain[0].shape[0], dev, "set_rows")
    if any(c.dev != dev for c in caches):
        raise MI355XError("set_rows: caches on one device")
    arr = _kv_rows(caches, plain, n, "set_rows")
    check(lib().mi355x_set_rows(arr, len(caches), ip, it, n, _kv_err(err, dev, "set_rows"), _launch_stream(dev, "set_rows")), "set_rows")


def get_rows(caches, idx=None, dtype=None, out=None, err=None):
    """Rows idx[i] (None: all, in order) of each of up to four caches as plain values: a list of
    [n, H, D] (or [n, D]) tensors of `dtype` (F32 by default), or `out`. One launch for every 2^24 blocks of 32."""
    if not caches:
        raise MI355XError("get_rows: one to four caches")
    dev = caches[0].dev
    ip, it, n = _kv_index(idx, caches[0].shape[0], dev, "get_rows")
    if any(c.dev != dev for c in caches):
        raise MI355XError("get_rows: caches on one device")
    if out is None:
        dtype = dtype or _torch().float32
        out = [c.q.new_empty((n, *c._tail), dtype=dtype) for c in caches]
    elif len(out) != len(caches):
        raise MI355XError("get_rows: one output for every cache")
    arr = _kv_rows(caches, out, n, "get_rows")
    check(lib().mi355x_get_rows(arr, len(caches), ip, it, n, _kv_err(err, dev, "get_rows"), _launch_stream(dev, "get_rows")), "get_rows")
    return out


def _fa_q_args(q, k, v, mask, out, scale, softcap=0.0, max_bias=0.0):
    types, qs, os, kv = _plain_types(), q.shape, out.shape, v.shape
    nd, dev = len(qs), q.get_device()
    if nd not in (3, 4) or len(k.shape) != nd or len(kv) != nd or len(os) != nd:
        raise MI355XError("flash_attn_q: q, k, v and out are all [H, T, D]-shaped or all [S, H, T, D]-shaped")
    H, T, D = qs[-3], qs[-2], qs[-1]
    HK, KV, DV = kv[-3:]
    S = qs[0] if nd == 4 else 1
    if k.shape != kv[:-1] + (D,) or (nd == 4 and (kv[0] != S or os[0] != S)) or os[-3] != T or os[-2] != H or os[-1] != DV:
        raise MI355XError(f"flash_attn_q: q {tuple(qs)}, k {k.shape}, v {kv} and out {tuple(os)} do not fit")
    if k._view is None or v._view is None:
        raise MI355XError("flash_attn_q: an F16 cache is flash_attn's")
    qn, on, qt, ot = q.stride(), out.stride(), types.get(q.dtype), types.get(out.dtype)
    if qn[-1] != 1 or on[-1] != 1 or qt not in (F32, F16) or ot not in (F32, F16):
        raise MI355XError("flash_attn_q: q and out are F32 or F16 with contiguous rows")
    if k.dev != dev or v.dev != dev or out.get_device() != dev or (mask is not None and mask.get_device() != dev):
        raise MI355XError("flash_attn_q: all tensors on one device")
    mp, m1, m3 = None, 0, 0
    if mask is not None:
        ms, mn = mask.shape, mask.stride()
        if (types.get(mask.dtype) != F16 or mn[-1] != 1 or len(ms) not in (2, 3) or ms[-2] < T or ms[-1] < KV
                or (len(ms) == 3 and ms[0] not in (1, S))):
            raise MI355XError("flash_attn_q: the mask is fp16 [T', KV'], [1, T', KV'] or [S, T', KV'], T' >= T, KV' >= KV")
        mp, m1, m3 = mask.data_ptr(), mn[-2], mn[0] if len(ms) == 3 and ms[0] > 1 else 0
    return FaQArgs(q.data_ptr(), qn[-2], qn[-3], qn[0] if nd == 4 else 0, k._view, v._view, mp, m1, m3,
                   out.data_ptr(), on[-2], on[-3], on[0] if nd == 4 else 0, qt, ot, D, DV, T, H, KV, HK, S, scale, max_bias, softcap)


def flash_attn_q_workspace(q, k, v, mask, out, nsplit: int = 0) -> int:
    """Workspace bytes mi355x_flash_attn_q needs for these operands (0 for an unsupported op)."""
    return int(lib().mi355x_flash_attn_q_workspace(_fa_q_args(q, k, v, mask, out, 1.0), nsplit))


def flash_attn_q(q, k: KvCache, v: KvCache, mask, scale: float, softcap: float = 0.0, nsplit: int = 0, out=None, workspace=None,
                 max_bias: float = 0.0):
    """FLASH_ATTN_EXT over a quantized cache: q [H, T, D] or [S, H, T, D] (F32 or F16), k and v KvCache
    views [(S,) HK, KV, D] of Q8_0 or Q4_0, mask fp16 [T', KV'], [S, T', KV'] (S or 1) or None. Returns dst
    [(S,) T, H, DV], F32 unless `out` is F16."""
    torch = _torch()
    if out is None:
        H, T = q.shape[-3:-1]
        out = torch.empty(tuple(q.shape[:-3]) + (T, H, v.shape[-1]), dtype=torch.float32, device=q.device)
    a = _fa_q_args(q, k, v, mask, out, scale, softcap, max_bias)
    if workspace is None:
        need = int(lib().mi355x_flash_attn_q_workspace(a, nsplit))
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != k.dev:
        raise MI355XError("flash_attn_q: the workspace is on another device")
    check(lib().mi355x_flash_attn_q(a, nsplit, workspace.data_ptr(), workspace.nbytes, _launch_stream(k.dev, "flash_attn_q")),
          "flash_attn_q")
    return out


# ---- a KV cache in pages --------------------------------------------------------------------

def _set_once(self, name, value):
    """Of objects that hold their tensors' addresses: another tensor in a field would leave the old address in use."""
    if hasattr(self, name):
        raise MI355XError(f"{type(self).__name__}.{name} is fixed: make a new one, or change the tensor's values")
    object.__setattr__(self, name, value)


class KvStep:
    """A step of S sequences over caches in pages (mi355x_kv_step): page p of a cache [rows, HK, D] is its rows
    p * page .. p * page + page - 1; sequence s holds n_past[s] rows, found through the pages table[s] names, and
    adds up to T tokens, n_new[s] of them real (None: all), a chain or, with parents [S, T] (the number of the token
    before, -1: the rows held; T <= 64), a tree. All int32 on one device, read when a call runs, not when the step is
    made: a program keeps the step and changes the tensors' values."""

    __slots__ = ("table", "n_past", "n_new", "parents", "S", "T", "page", "dev", "args", "_raw")

    def __init__(self, table, n_past, T: int, page: int, n_new=None, parents=None):
        self.table, self.n_past, self.n_new, self.parents = table, n_past, n_new, parents
        self.S, self.T, self.page, self.dev = table.shape[0], int(T), int(page), table.get_device()
        i32 = _torch().int32
        for t, shape in ((table, (self.S, None)), (n_past, (self.S,)), (n_new, (self.S,)), (parents, (self.S, self.T))):
            if t is None:
                continue
            if (t.dtype != i32 or t.get_device() != self.dev or t.dim() != len(shape) or (t.shape[-1] > 1 and t.stride(-1) != 1)
                    or any(n is not None and n != m for n, m in zip(shape, t.shape))):
                raise MI355XError(f"KvStep: {t.dtype} {tuple(t.shape)} where an int32 of {shape} on the table's device is wanted")
        if self.page <= 0 or self.page % 32 or self.T < 0:
            raise MI355XError("KvStep: pages of whole 32-row tiles")
        if parents is not None and self.T > 64:
            raise MI355XError("KvStep: trees of at most 64 tokens")
        self.args = KvStepArgs(table.data_ptr(), table.stride(0), n_past.data_ptr(), None if n_new is None else n_new.data_ptr(),
                               None if parents is None else parents.data_ptr(), 0 if parents is None else parents.stride(0),
                               table.shape[1], self.S, self.T, self.page)
        self._raw = bytes(self.args)

    __setattr__ = _set_once


class Rope:
    """The position rotation of kv_append: pair i of a head's first 2 * len(freq) dims, (2 i, 2 i + 1) or with neox
    (i, i + len(freq)), turns by position * freq[i] (F32 on the device, radians a position); cosine and sine are
    multiplied by mscale. positions [S, T] int32, or None: n_past[s] plus a token's depth."""

    __slots__ = ("freq", "neox", "mscale", "positions", "dev", "_args")

    def __init__(self, freq, neox: bool = False, mscale: float = 1.0, positions=None):
        torch = _torch()
        if freq.dtype != torch.float32 or freq.dim() != 1 or not freq.is_contiguous() or freq.shape[0] % 4:
            raise MI355XError("Rope: freq is a contiguous F32 tensor of a multiple of 4 values")
        if positions is not None and (positions.dtype != torch.int32 or positions.dim() != 2 or positions.get_device() != freq.get_device()
                                      or (positions.shape[-1] > 1 and positions.stride(-1) != 1)):
            raise MI355XError("Rope: positions are int32 [S, T] on freq's device")
        self.freq, self.neox, self.mscale, self.positions, self.dev = freq, bool(neox), float(mscale), positions, freq.get_device()
        # its part of mi355x_kv_append_args
        self._args = (freq.data_ptr(), 0 if positions is None else positions.data_ptr(), 0 if positions is None else positions.stride(0),
                      2 * freq.shape[0], self.neox, self.mscale)

    __setattr__ = _set_once


def rope_freqs(n_rot: int, base: float = 10000.0, factors=None, device="cuda"):
    """base^(-2 i / n_rot), divided by factors[i] where given, formed in 64 bits: Rope's freq."""
    torch = _torch()
    f = base ** (-torch.arange(0, n_rot, 2, dtype=torch.float64) / n_rot)
    if factors is not None:
        f = f / torch.as_tensor(factors, dtype=torch.float64).cpu()
    return f.float().to(device)


# mi355x_kv_append_args behind the step and the two caches' rows: sequence strides, queries, rotation
_KV_APPEND = struct.Struct("@qqPqqqPqqqiiqPPqiif4x")
_NO_QUERIES = (0, 0, 0, 0, 0, 0, 0, 0, F32, F32, 0)
_NO_ROPE = (0, 0, 0, 0, 0, 1.0)


def _step_rows(c, x, step, what):
    """mi355x_kv_rows of cache [rows, H, D] and the step's plain rows x [S, T, H, D], with their sequence stride."""
    t, n, rows = _plain_types().get(x.dtype), x.stride(), c._rows
    if len(c.shape) != 3 or x.shape != (step.S, step.T, *c._tail) or n[3] != 1 or (t != F32 and t != F16) or x.get_device() != c.dev:
        raise MI355XError(f"{what}: rows {x.dtype} {tuple(x.shape)} do not fit {step.S} x {step.T} rows of a cache {c.shape}")
    return _KV_ROWS.pack(*rows, t, x.data_ptr(), n[1], n[2]), n[0]


def kv_append(step: KvStep, k_cache: KvCache, v_cache: KvCache, k, v, rope: Rope = None, q=None, q_out=None, err=None):
    """The step's new keys k [S, T, HK, D], rotated, and values v [S, T, HK, DV] (F32 or F16) into the rows of their
    tokens in the caches [rows, HK, D] and [rows, HK, DV], and the queries q [S, T, H, D], rotated, into q_out (a new tensor
    like q by default), which is returned. One launch. Rows of padding are left as they were. err: a device int32 that
    numbers out of range set to 1 (mi355x_kv_step)."""
    dev = step.dev
    if k_cache.dev != dev or v_cache.dev != dev:
        raise MI355XError("kv_append: the caches are on another device than the step")
    kr, k3 = _step_rows(k_cache, k, step, "kv_append")
    vr, v3 = _step_rows(v_cache, v, step, "kv_append")
    queries = _NO_QUERIES
    if q is None and q_out is not None:
        raise MI355XError("kv_append: q_out without q")
    if q is not None:
        if q_out is None:
            q_out = _torch().empty_like(q)
        types, shape, qn, on = _plain_types(), q.shape, q.stride(), q_out.stride()
        qt, ot = types.get(q.dtype), types.get(q_out.dtype)
        if (len(shape) != 4 or q_out.shape != shape or shape[0] != step.S or shape[1] != step.T or shape[3] != k_cache.D or qn[3] != 1 or on[3] != 1
                or (qt != F32 and qt != F16) or (ot != F32 and ot != F16) or q.get_device() != dev or q_out.get_device() != dev):
            raise MI355XError(f"kv_append: queries {q.dtype} {tuple(shape)} -> {q_out.dtype} {tuple(q_out.shape)} of a step of "
                              f"{step.S} x {step.T} tokens and heads of {k_cache.D}")
        queries = (q.data_ptr(), qn[1], qn[2], qn[0], q_out.data_ptr(), on[1], on[2], on[0], qt, ot, shape[2])
    turn = _NO_ROPE
    if rope is not None:
        if rope.dev != dev or (rope.positions is not None and rope.positions.shape != (step.S, step.T)):
            raise MI355XError("kv_append: the rotation is not this step's")
        turn = rope._args
    check(lib().mi355x_kv_append(step._raw + kr + vr + _KV_APPEND.pack(k3, v3, *queries, *turn), _kv_err(err, dev, "kv_append"),
                                 _launch_stream(dev, "kv_append")), "kv_append")
    return q_out


def kv_keep(step: KvStep, caches, path, n_keep=None, err=None):
    """The rows of the step's tokens path[s, i] (int32 [S, A], A <= 64, increasing) copied to those of tokens i, for i <
    n_keep[s] (int32 [S]; None: A each), in each of up to four caches [rows, H, D]: a path of accepted drafts becomes
    the next rows of its sequence. One launch."""
    dev, i32 = step.dev, _torch().int32
    if not 1 <= len(caches) <= 4 or any(c.dev != dev or c._rows is None for c in caches):
        raise MI355XError("kv_keep: one to four caches [rows, H, D] on the step's device")
    if path.dtype != i32 or path.dim() != 2 or path.shape[0] != step.S or path.get_device() != dev or (path.shape[1] > 1 and path.stride(1) != 1):
        raise MI355XError("kv_keep: path is int32 [S, A] on the step's device")
    if n_keep is not None and (n_keep.dtype != i32 or n_keep.shape != (step.S,) or n_keep.get_device() != dev or (step.S > 1 and n_keep.stride(0) != 1)):
        raise MI355XError("kv_keep: n_keep is int32 [S] on the step's device")
    rows = b"".join([_KV_ROWS.pack(*c._rows, F32, 0, 0, 0) for c in caches])
    check(lib().mi355x_kv_keep(step.args, rows, len(caches), path.data_ptr(), path.stride(0), None if n_keep is None else n_keep.data_ptr(),
                               path.shape[1], _kv_err(err, dev, "kv_keep"), _launch_stream(dev, "kv_keep")), "kv_keep")


def _fa_p_args(q, k, v, step, out, scale, softcap, max_kv, from_pages):
    types, qs, os = _plain_types(), q.shape, out.shape
    dev = step.dev
    if len(qs) != 4 or len(k.shape) != 3 or len(v.shape) != 3 or qs[0] != step.S or qs[2] != step.T or k.shape[-1] != qs[3] or k.shape[:2] != v.shape[:2]:
        raise MI355XError(f"flash_attn_paged: q {tuple(qs)}, k {k.shape} and v {v.shape} do not fit a step of {step.S} x {step.T} tokens")
    if os != (step.S, step.T, qs[1], v.shape[-1]):
        raise MI355XError(f"flash_attn_paged: out {tuple(os)}")
    qn, on, qt, ot = q.stride(), out.stride(), types.get(q.dtype), types.get(out.dtype)
    if qn[-1] != 1 or on[-1] != 1 or qt not in (F32, F16) or ot not in (F32, F16):
        raise MI355XError("flash_attn_paged: q and out are F32 or F16 with contiguous rows")
    if k.dev != dev or v.dev != dev or q.get_device() != dev or out.get_device() != dev:
        raise MI355XError("flash_attn_paged: all tensors on one device")
    kt, kq, kd, rows, k1, k2, HK, D = k._rows
    vt, vq, vd, _, v1, v2, _, DV = v._rows
    return FaPArgs(step.args, q.data_ptr(), qn[2], qn[1], qn[0], KvView(kt, kq, kd, k1, k2, 0), KvView(vt, vq, vd, v1, v2, 0), rows,
                   out.data_ptr(), on[2], on[1], on[0], qt, ot, D, DV, qs[1], HK, scale, softcap, max_kv, bool(from_pages))


def flash_attn_paged_workspace(q, k: KvCache, v: KvCache, step: KvStep, out, nsplit: int = 0, max_kv: int = 0, from_pages: bool = False) -> int:
    """Workspace bytes mi355x_flash_attn_paged needs for these operands (0 for an unsupported op)."""
    return int(lib().mi355x_flash_attn_paged_workspace(_fa_p_args(q, k, v, step, out, 1.0, 0.0, max_kv, from_pages), nsplit))


def flash_attn_paged(q, k: KvCache, v: KvCache, step: KvStep, scale: float, softcap: float = 0.0, nsplit: int = 0, out=None,
                     workspace=None, max_kv: int = 0, err=None, from_pages: bool = False):
    """Attention of a step's tokens, q [S, H, T, D] (F32 or F16), over caches in pages k [rows, HK, D] and v [rows, HK, DV]: each
    token sees the rows its sequence held, itself and the tokens above it. Returns dst [S, T, H, DV], F32 unless `out` is
    F16; padding is zeros. max_kv: a bound that no n_past + n_new passes (0: what the tables can hold), for which launch and
    workspace are planned; rows behind it are not read. from_pages: a quantized cache is read as it is stored, never decoded to fp16 first, which many
    rows of a chain may be: less rounding, longer calls."""
    torch = _torch()
    if out is None:
        out = torch.empty(q.shape[0], q.shape[2], q.shape[1], v.shape[-1], dtype=torch.float32, device=q.device)
    a = _fa_p_args(q, k, v, step, out, scale, softcap, max_kv, from_pages)
    if workspace is None:
        need = int(lib().mi355x_flash_attn_paged_workspace(a, nsplit))
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    elif workspace.get_device() != step.dev:
        raise MI355XError("flash_attn_paged: the workspace is on another device")
    check(lib().mi355x_flash_attn_paged(a, nsplit, workspace.data_ptr(), workspace.nbytes, _kv_err(err, step.dev, "flash_attn_paged"),
                                        _launch_stream(step.dev, "flash_attn_paged")), "flash_attn_paged")
    return out


def mul_mat_id(wtype: int, as_dev, n_expert: int, N: int, K: int, b, ids, out=None, workspace=None,
               err=None):
    """as_dev: expert panel in HBM layout (n_expert*N rows); b [T, ne11, K] f32; ids [T, n_used]
    int32. Returns dst [T, n_used, N] f32."""
    torch = _torch()
    T, ne11, _ = b.shape
    n_used = ids.shape[1]
    if out is None:
        out = torch.empty((T, n_used, N), dtype=torch.float32, device=b.device)
    a = MoeArgs(wtype, as_dev.data_ptr(), n_expert, N, K, b.data_ptr(), ne11, b.stride(1), b.stride(0),
                ids.data_ptr(), n_used, ids.stride(1), ids.stride(0), T,
                out.data_ptr(), out.stride(1), out.stride(0))
    need = int(lib().mi355x_mul_mat_id_workspace(ctypes.byref(a)))
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=b.device)
    check(lib().mi355x_mul_mat_id(ctypes.byref(a), _ptr(workspace), workspace.numel(),
                                  _ptr(err) if err is not None else None, stream_handle()), "mul_mat_id")
    return out


# ==== the backend host layer (include/mi355x_backend.h) =========================================
# A numpy-backed stand-in for the few ggml graph constructors the reference's tests use
# (ggml_new_tensor_*, ggml_mul_mat, ggml_mul_mat_id, ggml_flash_attn_ext, permute / view), with
# ggml's ne / nb conventions, so the host-layer tests read like the reference's.

OP_NONE, OP_MUL_MAT, OP_MUL_MAT_ID, OP_FLASH_ATTN_EXT, OP_RESHAPE, OP_VIEW, OP_PERMUTE, \
    OP_TRANSPOSE, OP_ADD, OP_SCALE, OP_OTHER = range(11)
BUF_NONE, BUF_HOST, BUF_REPACK, BUF_OTHER = range(4)
STATUS_SUCCESS, STATUS_FAILED = 0, -1
# ggml's published (block values, block bytes) of the types the descriptors here may carry
_TYPE_SIZE_ALL = {0: (1, 4), 1: (1, 2), 2: (32, 18), 3: (32, 20), 6: (32, 22), 7: (32, 24), 8: (32, 34),
                  10: (256, 84), 11: (256, 110), 12: (256, 144), 13: (256, 176), 14: (256, 210), 26: (1, 4),
                  30: (1, 2), 39: (32, 17)}


class Tensor(ctypes.Structure):
    pass


Tensor._fields_ = [("type", ctypes.c_int32), ("op", ctypes.c_int32),
                   ("ne", ctypes.c_int64 * 4), ("nb", ctypes.c_size_t * 4),
                   ("op_params", ctypes.c_int32 * 16), ("src", ctypes.POINTER(Tensor) * 10),
                   ("data", ctypes.c_void_p), ("name", ctypes.c_char * 64),
                   ("buffer_kind", ctypes.c_int32), ("buffer_id", ctypes.c_void_p),
                   ("buffer_size", ctypes.c_size_t)]


# ggml_to_float_t: (const void * src, float * dst, int64_t n)
TO_FLOAT_FN = ctypes.CFUNCTYPE(None, ctypes.c_void_p, ctypes.POINTER(ctypes.c_float), ctypes.c_int64)
_decoders = {}


def set_to_float(ttype, block, type_size, fn):
    """Registers a row decoder for a quantized type the kernels do not decode (the plugin passes
    ggml's to_float). `fn(src_addr, dst_float_ptr, n)`; kept alive for the process. Returns the
    status (0 or -1)."""
    cb = TO_FLOAT_FN(fn)
    st = host().mi355x_backend_set_to_float(ttype, block, type_size, cb)
    if st == 0:
        _decoders[ttype] = cb
    return st


def _bind_host(L):
    if getattr(L, "_host_bound", False):
        return L
    vp, i32, lng, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_size_t
    pt = ctypes.POINTER(Tensor)
    L.mi355x_backend_name.restype = ctypes.c_char_p
    L.mi355x_backend_description.restype = ctypes.c_char_p
    L.mi355x_backend_get_memory.argtypes = [ctypes.POINTER(sz), ctypes.POINTER(sz)]
    L.mi355x_backend_get_host_memory.argtypes = [ctypes.POINTER(sz), ctypes.POINTER(sz)]
    L.mi355x_backend_supports_op.restype = ctypes.c_bool
    L.mi355x_backend_supports_op.argtypes = [pt]
    L.mi355x_backend_offload_op.restype = ctypes.c_bool
    L.mi355x_backend_offload_op.argtypes = [pt]
    L.mi355x_backend_supports_buft.restype = ctypes.c_bool
    L.mi355x_backend_supports_buft.argtypes = [i32]
    L.mi355x_backend_init.restype = vp
    L.mi355x_backend_free.argtypes = [vp]
    L.mi355x_backend_is.restype = ctypes.c_bool
    L.mi355x_backend_is.argtypes = [vp]
    L.mi355x_backend_set_n_threads.argtypes = [vp, i32]
    L.mi355x_backend_get_n_threads.argtypes = [vp]
    L.mi355x_backend_set_quant_resident.argtypes = [vp, i32]
    L.mi355x_backend_graph_compute.argtypes = [vp, ctypes.POINTER(pt), i32]
    L.mi355x_backend_route_ops.restype = lng
    L.mi355x_backend_route_ops.argtypes = [vp, ctypes.c_char_p]
    L.mi355x_backend_cpu_fallbacks.restype = lng
    L.mi355x_backend_cpu_fallbacks.argtypes = [vp]
    L.mi355x_backend_moe_stats.argtypes = [vp, ctypes.POINTER(lng), ctypes.POINTER(lng)]
    L.mi355x_backend_route_stats.argtypes = [vp, ctypes.c_char_p, ctypes.POINTER(lng), ctypes.POINTER(lng),
                                                  ctypes.POINTER(lng)]
    L.mi355x_backend_inject_faults.argtypes = [vp, ctypes.c_char_p, i32]
    L.mi355x_backend_host_stats.argtypes = [vp, ctypes.POINTER(HostStats)]
    L.mi355x_backend_weight_key.argtypes = [pt, ctypes.c_char_p, i32]
    L.mi355x_backend_register_weight_source.argtypes = [pt, vp, sz]
    L.mi355x_backend_parse_mb.restype = ctypes.c_bool
    L.mi355x_backend_parse_mb.argtypes = [ctypes.c_char_p, ctypes.POINTER(sz)]
    L.mi355x_backend_set_to_float.restype = i32
    L.mi355x_backend_set_to_float.argtypes = [i32, ctypes.c_int64, ctypes.c_int64, TO_FLOAT_FN]
    L._host_bound = True
    return L


class HostStats(ctypes.Structure):
    """mi355x_host_stats: where graph_compute's time goes on the host."""
    _fields_ = [("calls", ctypes.c_long), ("fa_mirror_hits", ctypes.c_long), ("copyback_redone", ctypes.c_long),
                ("bytes_up", ctypes.c_double), ("bytes_down", ctypes.c_double), ("wall_s", ctypes.c_double),
                ("up_copy_s", ctypes.c_double), ("up_wait_s", ctypes.c_double), ("down_copy_s", ctypes.c_double),
                ("down_wait_s", ctypes.c_double), ("copy_api_s", ctypes.c_double), ("weight_s", ctypes.c_double),
                ("pieces_up", ctypes.c_long), ("pieces_down", ctypes.c_long)]


def host():
    return _bind_host(lib())


class Graph:
    """Owns the descriptors and numpy buffers of one graph (a ggml_context stand-in). With
    alloc=False (a no_alloc context) tensors have no data, as in a supports_op probe."""

    def __init__(self, alloc=True):
        self.alloc = alloc
        self.tensors = []
        self.keep = []

    def _new(self, ttype, ne, name=None, op=OP_NONE, srcs=(), data=None):
        import numpy as np
        t = Tensor()
        t.type = ttype
        t.op = op
        ne = list(ne) + [1] * (4 - len(ne))
        blk, bsz = _TYPE_SIZE_ALL[ttype]
        for i in range(4):
            t.ne[i] = ne[i]
        t.nb[0] = bsz
        t.nb[1] = bsz * (ne[0] // blk)
        t.nb[2] = t.nb[1] * ne[1]
        t.nb[3] = t.nb[2] * ne[2]
        for i, s in enumerate(srcs):
            if s is not None:
                t.src[i] = ctypes.pointer(s)
        if name:
            t.name = name.encode()[:63]
        nbytes = t.nb[3] * ne[3]
        if self.alloc and op in (OP_NONE, OP_MUL_MAT, OP_MUL_MAT_ID, OP_FLASH_ATTN_EXT, OP_OTHER, OP_ADD, OP_SCALE):
            buf = np.zeros(max(nbytes, 1), dtype=np.uint8) if data is None else data
            self.keep.append(buf)
            t.data = buf.ctypes.data
            t.buffer_kind = BUF_HOST
            t.buffer_size = buf.nbytes
            t.buffer_id = buf.ctypes.data
        self.tensors.append(t)
        return t

    def new_tensor(self, ttype, ne, name=None):
        return self._new(ttype, ne, name)

    def set(self, t, arr):
        import numpy as np
        a = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
        n = min(a.nbytes, t.buffer_size)
        ctypes.memmove(t.data, a.ctypes.data, n)

    def get(self, t, dtype, shape):
        import numpy as np
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        out = np.empty(shape, dtype=dtype)
        ctypes.memmove(out.ctypes.data, t.data, n)
        return out

    def mul_mat(self, a, b):
        return self._new(F32, [a.ne[1], b.ne[1], b.ne[2], b.ne[3]], op=OP_MUL_MAT, srcs=(a, b))

    def mul_mat_id(self, a, b, ids):
        return self._new(F32, [a.ne[1], ids.ne[0], b.ne[2], 1], op=OP_MUL_MAT_ID, srcs=(a, b, ids))

    def flash_attn_ext(self, q, k, v, mask, scale, max_bias=0.0, softcap=0.0, acc_prec=0):
        t = self._new(F32, [v.ne[0], q.ne[2], q.ne[1], q.ne[3]], op=OP_FLASH_ATTN_EXT, srcs=(q, k, v, mask))
        fp = (ctypes.c_float * 3)(scale, max_bias, softcap)
        ctypes.memmove(ctypes.addressof(t.op_params), fp, 12)
        if acc_prec:
            t.op_params[3] = acc_prec
        return t

    def op(self, ttype, ne, op, srcs=()):
        """A node of any other op (e.g. an ADD or a SCALE) for placement probes."""
        return self._new(ttype, ne, op=op, srcs=srcs)

    def permute_view(self, src, ne, nb, offset=0):
        """A strided view of `src` (ggml_view_* / ggml_permute): same bytes, new ne / nb."""
        t = Tensor()
        t.type = src.type
        t.op = OP_VIEW
        for i in range(4):
            t.ne[i] = ne[i]
            t.nb[i] = nb[i]
        t.src[0] = ctypes.pointer(src)
        if src.data:
            t.data = src.data + offset
            t.buffer_kind = src.buffer_kind
            t.buffer_size = src.buffer_size
            t.buffer_id = src.buffer_id
        self.tensors.append(t)
        return t


class Backend:
    """One backend instance (mi355x_backend_init .. free)."""

    def __init__(self):
        self.L = host()
        self.h = self.L.mi355x_backend_init()
        if not self.h:
            raise MI355XError("init failed")

    def free(self):
        if self.h:
            self.L.mi355x_backend_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def compute(self, nodes):
        arr = (ctypes.POINTER(Tensor) * len(nodes))(*[ctypes.pointer(n) for n in nodes])
        return self.L.mi355x_backend_graph_compute(self.h, arr, len(nodes))

    def route_ops(self, route=None):
        return self.L.mi355x_backend_route_ops(self.h, route.encode() if route else None)

    def cpu_fallbacks(self):
        return self.L.mi355x_backend_cpu_fallbacks(self.h)

    def moe_stats(self):
        a, b = ctypes.c_long(), ctypes.c_long()
        self.L.mi355x_backend_moe_stats(self.h, ctypes.byref(a), ctypes.byref(b))
        return a.value, b.value

    def route_stats(self, group):
        a, b, c = ctypes.c_long(), ctypes.c_long(), ctypes.c_long()
        self.L.mi355x_backend_route_stats(self.h, group.encode(), ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
        return a.value, b.value, c.value

    def set_quant_resident(self, mode):
        self.L.mi355x_backend_set_quant_resident(self.h, mode)

    def inject_faults(self, group, n):
        self.L.mi355x_backend_inject_faults(self.h, group.encode(), n)

    def host_stats(self):
        st = HostStats()
        self.L.mi355x_backend_host_stats(self.h, ctypes.byref(st))
        return {name: getattr(st, name) for name, _ in HostStats._fields_}


_registered = {}


def register_weight_source(t, src):
    """The original bytes of a weight whose tensor sits in CPU_REPACK (numpy array, or None to
    unregister); the array is kept alive while registered."""
    import numpy as np
    key = ctypes.addressof(t)
    if src is None:
        host().mi355x_backend_register_weight_source(ctypes.byref(t), None, 0)
        _registered.pop(key, None)
        return
    a = np.ascontiguousarray(src).view(np.uint8).reshape(-1)
    _registered[key] = a
    host().mi355x_backend_register_weight_source(ctypes.byref(t), ctypes.c_void_p(a.ctypes.data), a.nbytes)


def supports_op(t):
    return bool(host().mi355x_backend_supports_op(ctypes.byref(t)))


def offload_op(t):
    return bool(host().mi355x_backend_offload_op(ctypes.byref(t)))


def weight_key(t):
    buf = ctypes.create_string_buffer(256)
    host().mi355x_backend_weight_key(ctypes.byref(t), buf, 256)
    return buf.value.decode()


def parse_mb(text):
    v = ctypes.c_size_t(12345)
    ok = host().mi355x_backend_parse_mb(text.encode(), ctypes.byref(v))
    return ok, v.value
