// SPDX-License-Identifier: MIT
// The C ABI of the kernel library (include/mi355x_kernels.h): argument checks, HIP error
// mapping and launches. Nothing here allocates device memory.

#include "../../include/mi355x_kernels.h"

#include <hip/hip_runtime.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <cmath>

#include "mx_fa_dims.h"
#include "mx_kernels_impl.h"
#include "mx_weights.h"

namespace {

inline hipStream_t S(void * s) { return (hipStream_t)s; }

inline int hip_status(hipError_t e) {
    if (e == hipSuccess) return MI355X_OK;
    fprintf(stderr, "[mi355x] HIP error: %s\n", hipGetErrorString(e));
    return MI355X_E_DEVICE;
}

inline bool known_wtype(int wt) {
    return wt == mx::T_F16 || wt == mx::T_Q8_0 || wt == mx::T_Q4_0 || wt == mx::T_Q4_K || wt == mx::T_Q5_K ||
           wt == mx::T_Q6_K || wt == mx::T_MXFP4;
}

// the layouts regrouped by 32 rows, built from ggml blocks for expert stacks
inline bool x32_wtype(int wt) { return wt == mx::T_Q4_KX || wt == mx::T_Q8_0X || wt == mx::T_Q6_KX || wt == mx::T_MXFP4X; }

// the expert-stack layouts: every weight type, and the regrouped ones
inline bool known_moe_wtype(int wt) { return known_wtype(wt) || x32_wtype(wt); }

inline int64_t blck(int wt) {
    if (wt == mx::T_Q4_K || wt == mx::T_Q4_KX || wt == mx::T_Q5_K || wt == mx::T_Q6_K || wt == mx::T_Q6_KX) return 256;
    return (wt == mx::T_Q8_0 || wt == mx::T_Q8_0X || wt == mx::T_Q4_0 || wt == mx::T_MXFP4 || wt == mx::T_MXFP4X) ? 32 : 1;
}

inline bool aligned(const void * p, size_t a) { return ((uintptr_t)p % a) == 0; }

}  // namespace

extern "C" {

MI355X_API const char * mi355x_status_str(int st) {
    switch (st) {
        case MI355X_OK: return "ok";
        case MI355X_E_ARG: return "invalid argument";
        case MI355X_E_DEVICE: return "device error";
        case MI355X_E_UNSUPPORTED: return "unsupported";
        case MI355X_E_NOMEM: return "workspace too small";
        case MI355X_E_IDS: return "expert id out of range";
        default: return "unknown status";
    }
}

MI355X_API int mi355x_get_device_info(mi355x_device_info * out) {
    if (!out) return MI355X_E_ARG;
    memset(out, 0, sizeof(*out));
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_status(e);
    hipDeviceProp_t p;
    e = hipGetDeviceProperties(&p, dev);
    if (e != hipSuccess) return hip_status(e);
    snprintf(out->name, sizeof(out->name), "%s", p.gcnArchName);
    out->compute_units = p.multiProcessorCount;
    out->lds_bytes_per_block = (int)p.sharedMemPerBlock;
    out->clock_khz = p.clockRate;
    size_t fr = 0, tot = 0;
    if (hipMemGetInfo(&fr, &tot) == hipSuccess) {
        out->hbm_free = fr;
        out->hbm_total = tot;
    }
    return MI355X_OK;
}

MI355X_API int64_t mi355x_weight_bytes(int wtype, int64_t rows, int64_t K) {
    if (wtype == mx::T_F16T) return (rows < 0 || K <= 0 || K % 32) ? -1 : mx::packed_weight_bytes(wtype, rows, K);
    if (x32_wtype(wtype)) return (rows < 0 || K <= 0 || K % blck(wtype)) ? -1 : mx::packed_weight_bytes(wtype, rows, K);
    if (!known_wtype(wtype) || rows < 0 || K <= 0 || K % blck(wtype)) return -1;
    return mx::packed_weight_bytes(wtype, rows, K);
}

MI355X_API int mi355x_weight_pack(int wtype, const void * src_dev, int64_t rows, int64_t K,
                                  void * dst_dev, void * stream) {
    if (x32_wtype(wtype)) {   // from ggml blocks; a regrouping, so never in place
        if (rows < 0 || rows % 32 || K <= 0 || K % blck(wtype)) return MI355X_E_ARG;
        if (rows == 0) return MI355X_OK;
        if (!src_dev || !dst_dev || src_dev == dst_dev || !aligned(dst_dev, 16)) return MI355X_E_ARG;
        if (wtype == mx::T_Q4_KX) {
            if (!aligned(src_dev, 16)) return MI355X_E_ARG;
            return hip_status(mx::launch_pack_q4kx(src_dev, rows, K, dst_dev, S(stream)));
        }
        return hip_status(mx::launch_pack_x32(wtype, src_dev, rows, K, dst_dev, S(stream)));
    }
    if (!known_wtype(wtype) || rows < 0 || K <= 0 || K % blck(wtype) || K % 32) return MI355X_E_ARG;
    if (rows == 0) return MI355X_OK;
    if (!src_dev || !dst_dev) return MI355X_E_ARG;
    if ((wtype == mx::T_Q8_0 || wtype == mx::T_Q4_0 || wtype == mx::T_Q6_K || wtype == mx::T_MXFP4) && src_dev == dst_dev)
        return MI355X_E_ARG;
    return hip_status(mx::launch_pack_weight(wtype, src_dev, rows, K, dst_dev, S(stream)));
}

MI355X_API int mi355x_weight_dequant_f16(int wtype, const void * w_dev, int64_t rows, int64_t K,
                                         uint16_t * out_dev, void * stream) {
    if (!known_wtype(wtype) || rows < 0 || K <= 0 || K % blck(wtype) || K % 64) return MI355X_E_ARG;
    if (rows == 0) return MI355X_OK;
    if (!w_dev || !out_dev || !aligned(w_dev, 16) || !aligned(out_dev, 16)) return MI355X_E_ARG;
    return hip_status(mx::launch_dequant_f16(wtype, w_dev, rows, K, out_dev, S(stream)));
}

MI355X_API int mi355x_weight_f16_tiled(int wtype, const void * w_dev, int64_t rows, int64_t K,
                                       uint16_t * out_dev, void * stream) {
    if (!known_wtype(wtype) || rows < 0 || K <= 0 || K % blck(wtype) || K % 64) return MI355X_E_ARG;
    if (rows == 0) return MI355X_OK;
    if (!w_dev || !out_dev || !aligned(w_dev, 16) || !aligned(out_dev, 16) || w_dev == (const void *)out_dev)
        return MI355X_E_ARG;
    return hip_status(mx::launch_f16_tiled(wtype, w_dev, rows, K, out_dev, S(stream)));
}

MI355X_API int mi355x_convert_f16(int type, const void * src_dev, int64_t n, uint16_t * dst_dev, void * stream) {
    if ((type != mx::T_F32 && type != mx::T_BF16) || n < 0) return MI355X_E_ARG;
    if (n == 0) return MI355X_OK;
    if (!src_dev || !dst_dev || !aligned(src_dev, type == mx::T_F32 ? 4 : 2) || !aligned(dst_dev, 2)) return MI355X_E_ARG;
    return hip_status(mx::launch_convert_f16(type, src_dev, n, dst_dev, S(stream)));
}

// zc (optional): an output [M][ldzc] whose first zn columns the pack kernel also clears
static int pack_impl(bool tiled, const float * x_dev, int64_t ldx, int64_t M, int64_t K, uint16_t * a16_dev,
                     float * scales_dev, void * stream, float * zc, int64_t ldzc, int64_t zn) {
    if (M < 0 || K <= 0 || K % (tiled ? 32 : 4) || ldx < K || ldx % 4 || M > INT32_MAX - 15 || K > INT32_MAX)
        return MI355X_E_ARG;
    if (M == 0) return MI355X_OK;
    if (!x_dev || !a16_dev || !scales_dev || !aligned(x_dev, 16) || !aligned(a16_dev, 8)) return MI355X_E_ARG;
    if (zc && (ldzc < zn || zn > INT32_MAX)) return MI355X_E_ARG;
    return tiled ? hip_status(mx::launch_pack_act_tiled(x_dev, ldx, (int)M, (int)K, a16_dev, scales_dev, S(stream),
                                                        zc, ldzc, (int)zn))
                 : hip_status(mx::launch_pack_act(x_dev, ldx, (int)M, (int)K, a16_dev, K, scales_dev, S(stream), zc,
                                                  ldzc, (int)zn));
}

MI355X_API int mi355x_pack_act(const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                               uint16_t * a16_dev, float * scales_dev, void * stream) {
    return pack_impl(false, x_dev, ldx, M, K, a16_dev, scales_dev, stream, nullptr, 0, 0);
}

MI355X_API int mi355x_pack_act_tiled(const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                                     uint16_t * a16_dev, float * scales_dev, void * stream) {
    return pack_impl(true, x_dev, ldx, M, K, a16_dev, scales_dev, stream, nullptr, 0, 0);
}

MI355X_API int mi355x_pack_act_clear(int tiled, const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                                     uint16_t * a16_dev, float * scales_dev, float * clear_dev, int64_t ld_clear,
                                     int64_t n_clear, void * stream) {
    if (!clear_dev || n_clear <= 0 || !aligned(clear_dev, 4)) return MI355X_E_ARG;
    return pack_impl(tiled != 0, x_dev, ldx, M, K, a16_dev, scales_dev, stream, clear_dev, ld_clear, n_clear);
}

// The launch arguments of a GEMM, checked; `with_ptrs` also checks the operand pointers.
static int gemm_lower(int wtype, const uint16_t * a16_dev, const float * scales_dev, int64_t M, int64_t K,
                      const mi355x_gemm_out * outs, int n_out, bool with_ptrs, mx::GemmArgs & a) {
    const bool tiled = wtype == mx::T_F16T;
    if ((!known_wtype(wtype) && !tiled) || M < 0 || K <= 0 || K % 32 || K % blck(wtype) || M > INT32_MAX ||
        K > INT32_MAX)
        return MI355X_E_ARG;
    if (n_out < 1 || n_out > mx::GEMM_MAX_GROUPS || !outs) return MI355X_E_ARG;
    if (with_ptrs && M > 0 && (!a16_dev || !scales_dev || !aligned(a16_dev, 16))) return MI355X_E_ARG;
    memset(&a, 0, sizeof(a));
    a.A = a16_dev;
    a.scales = scales_dev;
    a.lda = K;
    a.M = (int)M;
    a.K = (int)K;
    a.m_tiles = (int)((M + 127) / 128);
    a.ng = n_out;
    int nt = 0;
    for (int i = 0; i < n_out; i++) {
        const mi355x_gemm_out & o = outs[i];
        if (o.N <= 0 || o.N % 16 || o.N > INT32_MAX || o.ldc < o.N || o.row0 < 0 || o.rows_total < o.row0 + o.N)
            return MI355X_E_ARG;
        if (with_ptrs && (!o.w_dev || !o.c_dev || !aligned(o.w_dev, 16))) return MI355X_E_ARG;
        a.g[i].W = o.w_dev;
        a.g[i].rows_total = o.rows_total;
        a.g[i].row0 = o.row0;
        a.g[i].N = (int)o.N;
        a.g[i].C = o.c_dev;
        a.g[i].ldc = o.ldc;
        a.g[i].ntile_begin = nt;
        nt += (int)((o.N + 127) / 128);
    }
    return MI355X_OK;
}

// c_zeroed: the outputs were cleared by the activation pack (mi355x_mul_mat); part / part_bytes:
// workspace for the partial sums of a K split past two ways
static int gemm_impl(int wtype, const uint16_t * a16_dev, const float * scales_dev, int64_t M, int64_t K,
                     const mi355x_gemm_out * outs, int n_out, void * stream, bool c_zeroed, void * part,
                     size_t part_bytes) {
    mx::GemmArgs a;
    const int st = gemm_lower(wtype, a16_dev, scales_dev, M, K, outs, n_out, true, a);
    if (st != MI355X_OK || M == 0) return st;
    if (part && !aligned(part, 16)) return MI355X_E_ARG;
    return hip_status(mx::launch_gemm(wtype, a, 0, S(stream), c_zeroed, (float *)part, part ? part_bytes : 0));
}

MI355X_API int mi355x_gemm(int wtype, const uint16_t * a16_dev, const float * scales_dev,
                           int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                           void * stream) {
    return gemm_impl(wtype, a16_dev, scales_dev, M, K, outs, n_out, stream, false, nullptr, 0);
}

MI355X_API size_t mi355x_gemm_workspace(int wtype, int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out) {
    mx::GemmArgs a;
    if (M <= 0 || gemm_lower(wtype, nullptr, nullptr, M, K, outs, n_out, false, a) != MI355X_OK) return 0;
    return mx::gemm_split_bytes(wtype, a);
}

MI355X_API int mi355x_gemm_accumulates(int wtype, int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                                       size_t workspace_bytes) {
    mx::GemmArgs a;
    const int st = gemm_lower(wtype, nullptr, nullptr, M, K, outs, n_out, false, a);
    if (st != MI355X_OK) return st;
    return M > 0 && mx::gemm_accumulates(wtype, a, workspace_bytes) ? 1 : 0;
}

MI355X_API int mi355x_gemm_ws(int wtype, const uint16_t * a16_dev, const float * scales_dev,
                              int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                              void * workspace_dev, size_t workspace_bytes, int flags, void * stream) {
    return gemm_impl(wtype, a16_dev, scales_dev, M, K, outs, n_out, stream, (flags & MI355X_GEMM_OUT_ZEROED) != 0,
                     workspace_dev, workspace_bytes);
}

// M rows rounded up to 16: the tiled layout's padding (the row-major pack uses M rows of it).
static size_t mul_mat_a16_bytes(int64_t M, int64_t K) {
    return ((size_t)((M + 15) / 16 * 16) * (size_t)K * 2 + 255) & ~(size_t)255;
}

MI355X_API size_t mi355x_mul_mat_workspace(int64_t M, int64_t K) {
    if (M <= 0 || K <= 0) return 0;
    return mul_mat_a16_bytes(M, K) + (size_t)M * 4;
}

// The K-split partials of mi355x_mul_mat start at this offset of its workspace.
static size_t mul_mat_part_offset(int64_t M, int64_t K) {
    return (mi355x_mul_mat_workspace(M, K) + 255) & ~(size_t)255;
}

static int device_cus() {
    static int cus = 0;   // read once: this may run while a stream is being captured
    if (cus == 0) {
        int dev = 0;
        hipDeviceProp_t p;
        cus = (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&p, dev) == hipSuccess &&
               p.multiProcessorCount > 0) ? p.multiProcessorCount : 256;
    }
    return cus;
}

// The share of the chip that an all-DMA launch of bm x 256 tiles keeps busy over its rounds.
static double tile_fill(int64_t M, int64_t N, int bm) {
    const int64_t t = ((M + bm - 1) / bm) * ((N + 255) / 256), cus = device_cus();
    return (double)t / (double)((t + cus - 1) / cus * cus);
}

// Where a weight decoded once per call into tiled fp16 (one pass over the weight, at HBM rate) and
// multiplied by the one-wave fp16 GEMM is faster than decoded inside the GEMM. Measured per call on
// MI355X with cold weights over N, K in {1024, 2048, 3072, 4096, 6144, 8192, 14336, 28672} and M 65-2048
// (in-GEMM time over decode-first time); never at M <= 128, where the skinny kernels win 1.1-2.5x.
//   Q6_K, Q5_K, MXFP4, Q4_0 (register-staged decode kernel): 1.1-2.3x from M 384 on; below that up to
//     2^25 weights, 0.95-1.5x, on larger panels 0.82-1.05x (MXFP4, its slowest in-GEMM decode, 1.15-1.4x
//     up to 2^26).
//   Q4_K and Q8_0 (all-DMA decode kernels):
//     up to 2^25 weights 0.95-1.7x from M 129 on, except that past 2^23 weights a K of 2 N or more is split
//     inside the all-DMA kernel, which is as fast (0.85-1.03x) up to M 767, and loses 1.1-1.6x beyond;
//     larger panels: from M 768 (Q8_0) or 1024 (Q4_K) on 1.0-1.5x. Below that the all-DMA kernel wins
//     where its tiles fill the chip (14336 x 4096 at M 512, 224 tiles: 0.93x) and loses 1.1-1.4x where
//     the last round is mostly empty (at M 600, 280 tiles); Q8_0 past 2^26 weights, whose decode pass
//     moves twice the bytes, only from M 768.
//     Q8_0 up to 2^25 weights stays inside too where that launch makes one full round: up to 256 rows its
//     K split, from K 4096 and 2^24 weights on (4096 x 4096 M 160 0.96x, 8192 x 4096 0.91x, 6144 x 5120 0.89x; not
//     5632 x 4096, whose six splits are 264 blocks: 1.36x; 8192 x 2560 1.10x), and up to 767 its tiles where they
//     take 0.85 of the chip (16384 x 1024 M 512 0.91x, 12800 x 2560 M 600 0.96x; 11008 x 2816 M 640, 0.84, 1.12x).
// Panels under 2^22 weights keep lines drawn with the older fp16 GEMM: such calls are a few
// microseconds of launches either way. Same fp16 weights and activations in both forms.
static bool mul_mat_decode_first(int wtype, int64_t M, int64_t N, int64_t K) {
    if (K % 64 || M <= 128) return false;
    const int64_t w = N * K;
    const bool panel = w >= ((int64_t)1 << 22), w25 = w <= ((int64_t)1 << 25), w26 = w <= ((int64_t)1 << 26);
    const bool split = K >= 2 * N && w > ((int64_t)1 << 23);
    switch (wtype) {
        case mx::T_Q6_K:
        case mx::T_Q5_K: return M >= 512 || (panel && (M >= 384 || w25));
        case mx::T_MXFP4: return M >= 512 || (panel && (M >= 384 || w26));
        case mx::T_Q4_0: return (panel && (M >= 384 || w25)) || (M >= 512 && (N >= K || M >= 1024));
        case mx::T_Q4_K:
            if (!panel) return M >= 512 && N >= K;
            if (split) return M >= 768;
            if (w25 || M >= 1024) return true;
            return M >= 384 && std::max(tile_fill(M, N, 128), tile_fill(M, N, 256)) < 0.8;
        case mx::T_Q8_0:
            if (!panel) return M >= 1024 || (M >= 512 && K % 256 && N >= K);
            if (split) return M >= 768;
            if (w25 && M < 768 && K % 256 == 0 && ((M <= 256 && K >= 4096 && w >= ((int64_t)1 << 24)) || tile_fill(M, N, 128) >= 0.85)) {
                mx::GemmArgs a;
                memset(&a, 0, sizeof(a));
                a.M = (int)M;
                a.K = (int)K;
                a.ng = 1;
                a.g[0].N = (int)N;
                if (mx::gemm_one_round(wtype, a)) return false;
            }
            if (w25 || M >= 768) return true;
            return M >= 384 && w26 && tile_fill(M, N, 128) < 0.8;
        default: return false;
    }
}

MI355X_API int mi355x_mul_mat_decode_first(int wtype, int64_t M, int64_t N, int64_t K) {
    return known_wtype(wtype) && N > 0 && K > 0 && mul_mat_decode_first(wtype, M, N, K) ? 1 : 0;
}

// The tiled fp16 weight of the decode-first form sits right after the pack; the K-split
// partials after it.
static size_t mul_mat_w16_bytes(int64_t N, int64_t K) {
    return ((size_t)mi355x_weight_bytes(mx::T_F16T, N, K) + 255) & ~(size_t)255;
}

MI355X_API size_t mi355x_mul_mat_workspace_for(int wtype, int64_t N, int64_t K, int64_t M) {
    const size_t need = mi355x_mul_mat_workspace(M, K);
    if (need == 0) return 0;
    const mi355x_gemm_out o = {nullptr, N, 0, N, nullptr, N};
    if (known_wtype(wtype) && N > 0 && mul_mat_decode_first(wtype, M, N, K))
        return mul_mat_part_offset(M, K) + mul_mat_w16_bytes(N, K) + mi355x_gemm_workspace(mx::T_F16T, M, K, &o, 1);
    const size_t part = mi355x_gemm_workspace(wtype, M, K, &o, 1);
    return part ? mul_mat_part_offset(M, K) + part : need;
}

MI355X_API int mi355x_mul_mat(int wtype, const void * w_dev, int64_t N, int64_t K,
                              const float * x_dev, int64_t ldx, int64_t M,
                              float * dst_dev, int64_t ldd,
                              void * workspace_dev, size_t workspace_bytes, void * stream) {
    if (M == 0) return MI355X_OK;
    const size_t need = mi355x_mul_mat_workspace(M, K);
    if (need == 0) return MI355X_E_ARG;
    if (!workspace_dev || workspace_bytes < need) return MI355X_E_NOMEM;
    uint16_t * a16 = (uint16_t *)workspace_dev;
    float * scales = (float *)((char *)workspace_dev + mul_mat_a16_bytes(M, K));
    // the room past the pack holds the decode-first form's fp16 weight, if it runs, then K-split
    // partials
    size_t poff = mul_mat_part_offset(M, K);
    uint16_t * w16 = nullptr;
    if (known_wtype(wtype) && N > 0 && N <= INT32_MAX && mul_mat_decode_first(wtype, M, N, K) &&
        workspace_bytes >= poff + mul_mat_w16_bytes(N, K)) {
        w16 = (uint16_t *)((char *)workspace_dev + poff);
        poff += mul_mat_w16_bytes(N, K);
    }
    void * part = workspace_bytes > poff ? (char *)workspace_dev + poff : nullptr;
    const size_t part_bytes = part ? workspace_bytes - poff : 0;
    if (w16) {   // checks the weight's type, K and alignment like any other call of it
        const int st = mi355x_weight_f16_tiled(wtype, w_dev, N, K, w16, stream);
        if (st != MI355X_OK) return st;
        wtype = mx::T_F16T;
        w_dev = w16;
    }
    // a GEMM that adds a two-way K split into dst has it cleared by the pack, in the same launch
    bool zero = false;
    if ((known_wtype(wtype) || wtype == mx::T_F16T) && K > 0 && K <= INT32_MAX && M <= INT32_MAX && N > 0 &&
        N <= INT32_MAX && dst_dev && ldd >= N) {
        mx::GemmArgs probe;
        memset(&probe, 0, sizeof(probe));
        probe.M = (int)M;
        probe.K = (int)K;
        probe.ng = 1;
        probe.g[0].N = (int)N;
        zero = mx::gemm_accumulates(wtype, probe, part_bytes);
    }
    int st = pack_impl(wtype == mx::T_F16T, x_dev, ldx, M, K, a16, scales, stream, zero ? dst_dev : nullptr, ldd, N);
    if (st != MI355X_OK) return st;
    mi355x_gemm_out o = {w_dev, N, 0, N, dst_dev, ldd};
    return gemm_impl(wtype, a16, scales, M, K, &o, 1, stream, zero, part, part_bytes);
}

// ---- FLASH_ATTN_EXT ---------------------------------------------------------------------------

// Head dims past the fused kernel's builds (dk or dv > 256): two GEMMs around a softmax pass
// (mx_fa_wide.hip).
static bool fa_is_wide(const mi355x_fa_args * a) {
    return !mx::fa_dims_supported(a->D, a->DV) && mx::fa_wide_dims(a->D, a->DV);
}
static constexpr int64_t FA_WIDE_MAX_KV = 1 << 20;

// The absorbed MLA (dk 576, dv 512) whose V is the first 512 dims of K, the same pointer and strides:
// the fused kernel (mx_fa_mla.hip), which reads one cache for both products and addresses a KV head's
// keys by 32-bit byte offsets. It wins from one token on (16 heads, n_kv 4096, two GEMMs against fused:
// T 1 60 / 41 us, T 512 247 / 116; T 16 n_kv 1024 43 / 34), so everything else about the call is free.
// Other head dims past 256, V elsewhere and n_kv past its class table take the two-GEMM path.
static bool fa_mla_sizes(const mi355x_fa_args * a) {
    return a->D == 576 && a->DV == 512 && a->KV >= 1 && a->KV <= mx::FA_MLA_MAX_KV &&
           (int64_t)a->H * a->T < ((int64_t)1 << 30);
}
static bool fa_is_mla(const mi355x_fa_args * a) {
    return fa_mla_sizes(a) && a->v_dev == a->k_dev && a->v_nb1 == a->k_nb1 && (a->HK == 1 || a->v_nb2 == a->k_nb2) &&
           a->k_nb1 >= a->D && ((int64_t)a->KV + 64) * a->k_nb1 * 2 < 0x7FFFFFFF;
}

static int fa_check(const mi355x_fa_args * a) {
    if (!a || !a->q_dev || !a->k_dev || !a->v_dev || !a->dst_dev) return MI355X_E_ARG;
    const bool wide = fa_is_wide(a);
    // dk, dv <= 256, multiples of 8 (fused kernel); else dk % 32 == 0, dv % 8 == 0 up to 1024
    if (!wide && !mx::fa_dims_supported(a->D, a->DV)) return MI355X_E_UNSUPPORTED;
    if (a->max_bias != 0.0f) return MI355X_E_UNSUPPORTED;
    if (a->T < 0 || a->H <= 0 || a->HK <= 0 || a->KV < 0 || a->H % a->HK) return MI355X_E_ARG;
    if (a->q_nb1 % 4 || a->q_nb2 % 4 || !aligned(a->q_dev, 16)) return MI355X_E_ARG;
    if (a->k_nb1 % 8 || a->k_nb2 % 8 || a->v_nb1 % 8 || a->v_nb2 % 8) return MI355X_E_ARG;
    if (!aligned(a->k_dev, 16) || !aligned(a->v_dev, 16)) return MI355X_E_ARG;
    if (a->dst_nb1 % 4 || a->dst_nb2 % 4 || !aligned(a->dst_dev, 16)) return MI355X_E_ARG;
    if (a->mask_dev && (a->mask_nb1 % 4 || a->mask_nb1 < a->KV || !aligned(a->mask_dev, 8))) return MI355X_E_ARG;
    if (wide ? (int64_t)a->KV > FA_WIDE_MAX_KV : (size_t)a->KV > mx::fa_max_kv(a->D, a->DV)) return MI355X_E_UNSUPPORTED;
    return MI355X_OK;
}

// Workspace of the wide path: fp16 queries and their row scales, one KV head's keys and
// transposed values, and one chunk of query rows' scores, fp16 P, 1 / row sums and output rows.
struct FaWideLayout {
    size_t q16, qsc, kc, vt, s, p16, psc, o, total;
    int kvp, rows_chunk;
};
static size_t up256_fa(size_t n) { return (n + 255) & ~(size_t)255; }
static FaWideLayout fa_wide_layout(const mi355x_fa_args * a) {
    FaWideLayout L;
    L.kvp = (int)((a->KV + 63) / 64 * 64);
    if (L.kvp == 0) L.kvp = 64;
    L.rows_chunk = mx::fa_wide_rows_chunk(a->T, a->H, a->HK, L.kvp);
    const size_t rows = (size_t)a->H * a->T, rc = (size_t)L.rows_chunk, kvp = (size_t)L.kvp;
    size_t o = 0;
    L.q16 = o;  o += up256_fa(rows * a->D * 2);
    L.qsc = o;  o += up256_fa(rows * 4);
    L.kc = o;   o += up256_fa(kvp * a->D * 2);
    L.vt = o;   o += up256_fa((size_t)a->DV * kvp * 2);
    L.s = o;    o += up256_fa(rc * kvp * 4);
    L.p16 = o;  o += up256_fa(rc * kvp * 2);
    L.psc = o;  o += up256_fa(rc * 4);
    L.o = o;    o += up256_fa(rc * a->DV * 4);
    L.total = o;
    return L;
}

static mx::FaArgs fa_lower(const mi355x_fa_args * a, int nsplit) {
    mx::FaArgs f;
    memset(&f, 0, sizeof(f));
    f.q = a->q_dev; f.k = a->k_dev; f.v = a->v_dev; f.mask = a->mask_dev; f.dst = a->dst_dev;
    f.q_nb1 = a->q_nb1; f.q_nb2 = a->q_nb2; f.k_nb1 = a->k_nb1; f.k_nb2 = a->k_nb2;
    f.v_nb1 = a->v_nb1; f.v_nb2 = a->v_nb2; f.mask_nb1 = a->mask_nb1;
    f.dst_nb1 = a->dst_nb1; f.dst_nb2 = a->dst_nb2;
    f.dk = a->D; f.dv = a->DV;
    mx::fa_pad_dims(a->D, a->DV, f.D, f.DV);   // the kernel's dims (checked by fa_check)
    f.T = a->T; f.H = a->H; f.HK = a->HK; f.KV = a->KV; f.nsplit = nsplit;
    f.tasks = 4;
    f.kvp = (int)((a->KV + 63) / 64 * 64);
    f.cls_stride = (f.kvp / 64 + 15) / 16 * 16;
    f.scale = a->scale; f.softcap = a->softcap;
    return f;
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace: mask classes [T/32][cls_stride] | 256 bytes, the first 16 zeroed by the prep kernel |
// partial O [nsplit][T][H][DV] f32 and (max, sum) [nsplit][T][H][2] f32 when nsplit > 1 (DV as
// the kernel is built).
struct FaLayout {
    size_t cls, zero, po, pml, total;
};
static FaLayout fa_layout(const mx::FaArgs & f) {
    FaLayout L;
    const size_t nqt = (size_t)(f.T + 31) / 32;
    const size_t rows = (size_t)f.T * f.H * f.nsplit;
    L.cls = 0;
    L.zero = L.cls + align256(nqt * (size_t)f.cls_stride);
    L.po = L.zero + 256;
    L.pml = L.po + (f.nsplit > 1 ? align256(rows * f.DV * 4) : 0);
    L.total = L.pml + (f.nsplit > 1 ? align256(rows * 8) : 0);
    return L;
}

// The launch of an op: wave tasks per block and KV split (nsplit_req > 0: that split). One block
// per CU (their LDS rings take 128 KB). A step is two 64-key tiles for every task of a block:
// measured at head dims 128 / 128 on MI355X, 2.4 us with four tasks a block and 1.55 us with
// two (half the MFMA work, but the same barrier, DMA and latency chain per step), scaled here by
// the MFMA work of other head dims. A split writes its unnormalised partials and reads them back
// in the combine launch (about 3 us plus the partial bytes at 6 TB/s: 8.6 us at 512 queries x 32
// heads split two ways), and keeps at least 12 key tiles. MI355X_FA_TASKS (2 or 4) pins the
// task count, for tests.
struct FaPlan {
    int tasks, nsplit;
};
static FaPlan fa_plan(const mi355x_fa_args * a, int nsplit_req) {
    mx::FaArgs f = fa_lower(a, 1);
    const int ntiles = (int)((a->KV + 63) / 64);
    const int cus = device_cus();
    int pin = 0;
    if (const char * e = getenv("MI355X_FA_TASKS"))
        if (*e) pin = atoi(e);
    const int max_by_len = ntiles / 12 > 0 ? ntiles / 12 : 1;
    FaPlan best{4, nsplit_req > 0 ? nsplit_req : 1};
    double best_us = 0.0;
    bool have = false;
    for (int tasks = 2; tasks <= 4; tasks += 2) {
        if (!mx::fa_tasks_ok(f.DV, tasks) || (pin && pin != tasks)) continue;
        f.tasks = tasks;
        const int nb = mx::fa_blocks_per_split(f);
        const double step_us = (tasks == 2 ? 1.55 : 2.4) * (f.D + f.DV) / 256.0;
        const int lo = nsplit_req > 0 ? nsplit_req : 1, hi = nsplit_req > 0 ? nsplit_req : std::min(max_by_len, 16);
        for (int ns = lo; ns <= hi; ns++) {
            const double rounds = (double)((int64_t)nb * ns + cus - 1) / cus;
            const int steps = ((ntiles + ns - 1) / ns + 1) / 2;
            const double part_mb = (double)ns * a->T * a->H * f.DV * 8.0 / 1e6;
            const double us = (int64_t)rounds * steps * step_us + (ns > 1 ? 3.0 + part_mb / 6.0 : 0.0);
            if (!have || us < best_us - 1e-9) {
                best = {tasks, ns};
                best_us = us;
                have = true;
            }
        }
    }
    return best;
}

// The fused MLA's launch arguments. KV split: a block takes about 2.9 us a key tile after some 12 us
// of prologue (measured at 16 heads, 512 queries, n_kv 4096); a split writes its partial rows and
// reads them back in the combine launch, which walks the splits in turn, at least 0.85 us each (16 heads, T 1-32: two
// tiles a split instead of four gain 6 us at 4 splits, nothing at 16 and lose 6 at 32; whole call T 8 n_kv 512
// with soft-cap and holes 36.0 -> 29.7).
static mx::FaArgs fa_mla_lower(const mi355x_fa_args * a) {
    mx::FaArgs f = fa_lower(a, 1);
    f.D = 576;
    f.DV = 512;
    const int ntiles = f.kvp / 64, cus = device_cus();
    const int64_t nb = mx::fa_mla_blocks(f);
    const double part_mb = (double)a->T * a->H * 512 * 8.0 / 1e6;
    double best = 0.0;
    for (int ns = 1; ns <= std::min(ntiles, 64); ns++) {
        const int64_t rounds = (nb * ns + cus - 1) / cus;
        const double us = (double)rounds * (12.0 + ((ntiles + ns - 1) / ns) * 2.9) + (ns > 1 ? 3.0 + ns * std::max(0.85, part_mb / 6.0) : 0.0);
        if (ns == 1 || us < best - 1e-9) {
            best = us;
            f.nsplit = ns;
        }
    }
    return f;
}

MI355X_API int mi355x_flash_attn_auto_split(const mi355x_fa_args * a) {
    if (fa_check(a) != MI355X_OK) return 1;
    if (fa_is_mla(a)) return fa_mla_lower(a).nsplit;
    return fa_is_wide(a) ? 1 : fa_plan(a, 0).nsplit;
}

MI355X_API size_t mi355x_flash_attn_workspace(const mi355x_fa_args * a, int nsplit) {
    if (fa_check(a) != MI355X_OK) return 0;
    if (fa_is_wide(a)) {   // by the sizes alone: where V lies decides between the two forms
        const size_t wide = fa_wide_layout(a).total;
        return fa_mla_sizes(a) ? std::max(wide, fa_layout(fa_mla_lower(a)).total) : wide;
    }
    if (nsplit <= 0) nsplit = fa_plan(a, 0).nsplit;
    if (nsplit > 64) return 0;
    return fa_layout(fa_lower(a, nsplit)).total;
}

MI355X_API int mi355x_flash_attn(const mi355x_fa_args * a, int nsplit,
                                 void * workspace_dev, size_t workspace_bytes, void * stream) {
    return mi355x_flash_attn_ex(a, nsplit, 0, workspace_dev, workspace_bytes, stream);
}

// The fused kernel of head dims up to 256 on the workspace ws; q_f16, dst_f16: q and dst hold fp16.
static mx::FaArgs fa_fused_args(const mi355x_fa_args * a, int nsplit, bool q_f16, bool dst_f16, char * ws, size_t * need) {
    const FaPlan plan = fa_plan(a, nsplit);
    mx::FaArgs f = fa_lower(a, plan.nsplit);
    f.tasks = plan.tasks;
    f.q_f16 = q_f16;
    f.dst_f16 = dst_f16;
    const FaLayout L = fa_layout(f);
    *need = L.total;
    f.cls = (uint8_t *)(ws + L.cls);
    f.kzero = (uint16_t *)(ws + L.zero);
    if (plan.nsplit > 1) {
        f.part_o = (float *)(ws + L.po);
        f.part_ml = (float *)(ws + L.pml);
    }
    return f;
}

MI355X_API int mi355x_flash_attn_ex(const mi355x_fa_args * a, int nsplit, int flags,
                                    void * workspace_dev, size_t workspace_bytes, void * stream) {
    if (flags & ~MI355X_FA_CLASSES_READY) return MI355X_E_ARG;
    const int st = fa_check(a);
    if (st != MI355X_OK) return st;
    if (a->T == 0) return MI355X_OK;
    if (fa_is_mla(a)) {
        mx::FaArgs f = fa_mla_lower(a);
        const FaLayout L = fa_layout(f);
        if (workspace_dev && workspace_bytes >= L.total && aligned(workspace_dev, 256)) {
            char * ws = (char *)workspace_dev;
            f.cls = (uint8_t *)(ws + L.cls);
            f.kzero = (uint16_t *)(ws + L.zero);
            f.part_o = (float *)(ws + L.po);
            f.part_ml = (float *)(ws + L.pml);
            return hip_status(mx::launch_fa_mla(f, true, S(stream)));
        }
    }
    if (fa_is_wide(a)) {
        const FaWideLayout L = fa_wide_layout(a);
        if (!workspace_dev || workspace_bytes < L.total || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
        char * ws = (char *)workspace_dev;
        mx::FaWideArgs w;
        memset(&w, 0, sizeof(w));
        w.q = a->q_dev; w.k = a->k_dev; w.v = a->v_dev; w.mask = a->mask_dev; w.dst = a->dst_dev;
        w.q_nb1 = a->q_nb1; w.q_nb2 = a->q_nb2; w.k_nb1 = a->k_nb1; w.k_nb2 = a->k_nb2;
        w.v_nb1 = a->v_nb1; w.v_nb2 = a->v_nb2; w.mask_nb1 = a->mask_nb1;
        w.dst_nb1 = a->dst_nb1; w.dst_nb2 = a->dst_nb2;
        w.dk = a->D; w.dv = a->DV; w.T = a->T; w.H = a->H; w.HK = a->HK; w.KV = a->KV;
        w.kvp = L.kvp; w.rows_chunk = L.rows_chunk;
        w.scale = a->scale; w.softcap = a->softcap;
        w.q16 = (uint16_t *)(ws + L.q16); w.qsc = (float *)(ws + L.qsc);
        w.kc = (uint16_t *)(ws + L.kc); w.vt = (uint16_t *)(ws + L.vt);
        w.s = (float *)(ws + L.s); w.p16 = (uint16_t *)(ws + L.p16);
        w.psc = (float *)(ws + L.psc); w.o = (float *)(ws + L.o);
        return hip_status(mx::launch_fa_wide(w, S(stream)));
    }
    if (nsplit > 64) return MI355X_E_ARG;
    size_t need;
    const mx::FaArgs f = fa_fused_args(a, nsplit, false, false, (char *)workspace_dev, &need);
    if (!workspace_dev || workspace_bytes < need || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
    return hip_status(mx::launch_fa(f, !(flags & MI355X_FA_CLASSES_READY), S(stream)));
}

// ---- the quantized KV cache ---------------------------------------------------------------------

static bool kv_type(int t) { return t == mx::T_Q8_0 || t == mx::T_Q4_0; }

// store: the caches are written, else the plain rows
static int kv_rows_lower(const mi355x_kv_rows * r, int n_out, const void * idx_dev, int idx_type, int64_t n, int32_t * err_dev,
                         bool store, mx::KvRowsArgs & a) {
    if (!r || n_out < 1 || n_out > mx::KV_MAX_OUT || n < 0 || n > (1 << 30)) return MI355X_E_ARG;
    if (idx_type != 26 && idx_type != 27) return MI355X_E_ARG;
    if (!aligned(idx_dev, idx_type == 27 ? 8 : 4) || !aligned(err_dev, 4)) return MI355X_E_ARG;
    memset(&a, 0, sizeof a);
    // 32-bit positions (fq_div) and threads of a launch: all outputs' blocks up to 2^30, a row's up to 2^24
    int64_t blocks = 0;
    for (int k = 0; k < n_out; k++) {
        const mi355x_kv_rows & s = r[k];
        if ((!kv_type(s.type) && s.type != mx::T_F16) || (s.x_type != mx::T_F32 && s.x_type != mx::T_F16)) return MI355X_E_ARG;
        if (s.H <= 0 || s.D <= 0 || s.D % 32 || s.H > INT32_MAX / s.D || s.n_rows < 0) return MI355X_E_ARG;
        if (s.nb1 < 0 || s.nb2 < 0 || s.nb1 % 32 || s.nb2 % 32 || s.x_nb1 < 0 || s.x_nb2 < 0 || s.x_nb1 % 8 || s.x_nb2 % 8)
            return MI355X_E_ARG;
        if (n > 0 && (!s.q_dev || !s.x_dev || !aligned(s.q_dev, 16) || !aligned(s.x_dev, 16))) return MI355X_E_ARG;
        if (n > 0 && s.type != mx::T_F16 && (!s.d_dev || !aligned(s.d_dev, 8))) return MI355X_E_ARG;
        if (!idx_dev && n > s.n_rows) return MI355X_E_ARG;
        for (int j = 0; j < k && n > 0; j++)   // one destination twice: written in no order
            if (store ? r[j].q_dev == s.q_dev : r[j].x_dev == s.x_dev) return MI355X_E_ARG;
        const int64_t bpr = s.H * (s.D / 32);
        if (bpr > (1 << 24) || (blocks += n * bpr) > (1 << 30)) return MI355X_E_ARG;
        mx::KvRowsOut & o = a.o[k];
        o.q = (uint8_t *)s.q_dev; o.d = s.d_dev; o.x = s.x_dev;
        o.nb1 = s.nb1; o.nb2 = s.nb2; o.x_nb1 = s.x_nb1; o.x_nb2 = s.x_nb2; o.n_rows = s.n_rows;
        o.type = s.type; o.H = (int)s.H; o.bph = (int)(s.D / 32); o.x_f16 = s.x_type == mx::T_F16;
    }
    a.n_out = n_out; a.n = (int)n; a.idx = idx_dev; a.idx64 = idx_type == 27; a.err = err_dev;
    return MI355X_OK;
}

MI355X_API int mi355x_set_rows(const mi355x_kv_rows * r, int n_out, const void * idx_dev, int idx_type, int64_t n,
                               int32_t * err_dev, void * stream) {
    mx::KvRowsArgs a;
    const int st = kv_rows_lower(r, n_out, idx_dev, idx_type, n, err_dev, true, a);
    return st != MI355X_OK || n == 0 ? st : hip_status(mx::launch_set_rows(a, S(stream)));
}

MI355X_API int mi355x_get_rows(const mi355x_kv_rows * r, int n_out, const void * idx_dev, int idx_type, int64_t n,
                               int32_t * err_dev, void * stream) {
    mx::KvRowsArgs a;
    const int st = kv_rows_lower(r, n_out, idx_dev, idx_type, n, err_dev, false, a);
    return st != MI355X_OK || n == 0 ? st : hip_status(mx::launch_get_rows(a, S(stream)));
}

static int fa_q_check_view(const mi355x_kv_view & w, bool empty) {
    if (!kv_type(w.type)) return MI355X_E_UNSUPPORTED;
    if ((!empty && (!w.q_dev || !w.d_dev)) || !aligned(w.q_dev, 16) || !aligned(w.d_dev, 8)) return MI355X_E_ARG;
    if (w.nb1 < 0 || w.nb2 < 0 || w.nb3 < 0 || w.nb1 % 32 || w.nb2 % 32 || w.nb3 % 32) return MI355X_E_ARG;
    return MI355X_OK;
}

static int fa_q_check(const mi355x_fa_q_args * a, int nsplit) {
    if (!a) return MI355X_E_ARG;
    const bool empty = a->T == 0 || a->S == 0;   // no query: nothing is read or written
    if (!empty && (!a->q_dev || !a->dst_dev)) return MI355X_E_ARG;
    if (a->D <= 0 || a->DV <= 0 || a->D % 32 || a->DV % 32 || !mx::fa_dims_supported(a->D, a->DV)) return MI355X_E_UNSUPPORTED;
    if (a->max_bias != 0.0f) return MI355X_E_UNSUPPORTED;
    for (const mi355x_kv_view * w : {&a->k, &a->v}) {
        const int st = fa_q_check_view(*w, empty || a->KV == 0);
        if (st != MI355X_OK) return st;
    }
    if (a->T < 0 || a->S < 0 || a->H <= 0 || a->HK <= 0 || a->KV < 0 || a->H % a->HK) return MI355X_E_ARG;
    if ((int64_t)a->KV * a->HK * ((a->D + a->DV) / 32) >= 1 << 29) return MI355X_E_UNSUPPORTED;
    // threads of a launch: row tiles of 16 rows of a sequence and KV head, up to 1024 threads and 64 splits; where keys
    // are split, 256 threads a tile and 16 (built) dims merge them, and 2^32 threads are too many
    const int64_t tiles = (int64_t)a->S * a->HK * (((int64_t)a->T * (a->H / a->HK) + 15) / 16);
    if (tiles > (1 << 21) / (nsplit > 1 ? nsplit : 1)) return MI355X_E_UNSUPPORTED;
    int D, DV;
    mx::fa_pad_dims(a->D, a->DV, D, DV);
    if (nsplit > 1 && tiles * DV >= 1 << 28) return MI355X_E_UNSUPPORTED;
    if ((int64_t)a->S * a->T * a->H > (1 << 30) || (size_t)a->KV > mx::fa_max_kv(a->D, a->DV)) return MI355X_E_UNSUPPORTED;
    for (int t : {a->q_type, a->dst_type})
        if (t != mx::T_F32 && t != mx::T_F16) return MI355X_E_ARG;
    const int64_t qa = a->q_type == mx::T_F16 ? 8 : 4;
    if (a->q_nb1 % qa || a->q_nb2 % qa || a->q_nb3 % qa || !aligned(a->q_dev, 16)) return MI355X_E_ARG;
    if (a->dst_nb1 % 4 || a->dst_nb2 % 4 || a->dst_nb3 % 4 || !aligned(a->dst_dev, a->dst_type == mx::T_F16 ? 8 : 16)) return MI355X_E_ARG;
    if (a->mask_dev && (a->mask_nb1 % 4 || a->mask_nb3 % 4 || a->mask_nb1 < a->KV || a->mask_nb3 < 0 || !aligned(a->mask_dev, 8)))
        return MI355X_E_ARG;
    return MI355X_OK;
}

// The view of sequence s.
static mx::KvView fa_q_view(const mi355x_kv_view & w, int64_t s) {
    mx::KvView v;
    v.q = (const uint8_t *)w.q_dev + s * w.nb3 / (w.type == mx::T_Q4_0 ? 2 : 1);
    v.d = w.d_dev + s * w.nb3 / 32;
    v.nb1 = w.nb1; v.nb2 = w.nb2; v.nb3 = w.nb3; v.type = w.type;
    return v;
}

// One sequence of the op over fp16 K and V at k16, v16, [HK][KV][D] each.
static mi355x_fa_args fa_q_lower(const mi355x_fa_q_args * a, int s, const uint16_t * k16, const uint16_t * v16) {
    mi355x_fa_args f;
    memset(&f, 0, sizeof f);
    const int64_t qe = a->q_type == mx::T_F16 ? 2 : 4, de = a->dst_type == mx::T_F16 ? 2 : 4;
    f.q_dev = (const float *)((const char *)a->q_dev + s * a->q_nb3 * qe); f.q_nb1 = a->q_nb1; f.q_nb2 = a->q_nb2;
    f.k_dev = k16; f.k_nb1 = a->D; f.k_nb2 = (int64_t)a->KV * a->D;
    f.v_dev = v16; f.v_nb1 = a->DV; f.v_nb2 = (int64_t)a->KV * a->DV;
    f.mask_dev = a->mask_dev ? a->mask_dev + s * a->mask_nb3 : nullptr; f.mask_nb1 = a->mask_nb1;
    f.dst_dev = (float *)((char *)a->dst_dev + s * a->dst_nb3 * de); f.dst_nb1 = a->dst_nb1; f.dst_nb2 = a->dst_nb2;
    f.D = a->D; f.DV = a->DV; f.T = a->T; f.H = a->H; f.KV = a->KV; f.HK = a->HK;
    f.scale = a->scale; f.softcap = a->softcap;
    return f;
}

// Rows a wave and KV splits of the kernels of mx_fa_q.h (nsplit > 0: that split).
static void fa_q_plan(mx::FaQArgs & f, int nsplit) {
    // Keys are split while compute units are idle, four tiles a block at least, and not at all up to 16 tiles,
    // which a block's waves take at once or twice: the second launch costs more (us whole, in splits of eight
    // tiles and of four, Q8_0: 300 keys 11.2, 11.3, 13.1; 1000 15.6, 13.2, 13.0; 4000 35, 15.1, 14.9; 1000 at
    // head dim 256 33, 19.2, 16.2). Never past one block a compute unit (32 sequences of 4096 keys, 256 blocks:
    // 69 whole, 79 in two splits; of different lengths 50 and 60).
    const int64_t cus = device_cus(), ntiles = (f.KV + 31) / 32;
    auto units = [&](int nq) { return (int64_t)f.S * f.HK * ((f.R + 16 * nq - 1) / (16 * nq)); };
    auto splits = [&](int nq) {
        return nsplit > 0 ? nsplit : ntiles <= 16 ? 1 : std::max<int64_t>(1, std::min<int64_t>({64, cus / std::max<int64_t>(1, units(nq)), ntiles / 4}));
    };
    // Two row tiles a wave (head dim 64) share the work of turning codes into operands: a key tile takes 1.75 times
    // as long as with one, and a block's start and end, which take as long as 60 key tiles, 85. They are taken
    // where a compute unit is done sooner (4-bit, 8 KV heads, us with one and two: 256 rows of 16384
    // keys 47 / 45, 512 73 / 70; 512 of 4096 26 / 29; 400 of 1531 16 / 20, 800 28 / 22). At head dim 128 their
    // registers leave one wave a SIMD, which was never less time (128 rows of 32768 keys 66 / 86).
    auto cost = [&](int nq) {
        const int64_t n = splits(nq), tiles = (ntiles + n - 1) / n;
        return (units(nq) * n + cus - 1) / cus * (nq == 2 ? 7 * tiles + 340 : 4 * tiles + 240);
    };
    f.nq = 1;
    if (mx::fa_q_max_nq(f.D) == 2 && f.R > 16) {
        const char * e = getenv("MI355X_FA_Q_ROWS");
        f.nq = e && *e ? (atoi(e) == 32 ? 2 : 1) : cost(2) < cost(1) ? 2 : 1;
    }
    f.nrt = (f.R + 16 * f.nq - 1) / (16 * f.nq);
    f.nsplit = (int)splits(f.nq);
    f.div_nrt = mx::fq_div_by(f.nrt); f.div_hk = mx::fq_div_by(f.HK); f.div_split = mx::fq_div_by(f.nsplit);
    f.div_g = mx::fq_div_by(f.G);
}

// The direct form: the kernel of mx_fa_q.h on the cache as it is stored.
static mx::FaQArgs fa_q_direct(const mi355x_fa_q_args * a, int nsplit) {
    mx::FaQArgs f;
    memset(&f, 0, sizeof f);
    f.q = a->q_dev; f.k = fa_q_view(a->k, 0); f.v = fa_q_view(a->v, 0); f.mask = a->mask_dev; f.dst = a->dst_dev;
    f.q_nb1 = a->q_nb1; f.q_nb2 = a->q_nb2; f.q_nb3 = a->q_nb3; f.mask_nb1 = a->mask_nb1; f.mask_nb3 = a->mask_nb3;
    f.dst_nb1 = a->dst_nb1; f.dst_nb2 = a->dst_nb2; f.dst_nb3 = a->dst_nb3;
    mx::fa_pad_dims(a->D, a->DV, f.D, f.DV);
    f.dk = a->D; f.dv = a->DV;
    f.T = a->T; f.HK = a->HK; f.KV = a->KV; f.S = a->S; f.G = a->H / a->HK; f.R = a->T * f.G;
    f.scale = a->scale; f.softcap = a->softcap;
    f.q_f16 = a->q_type == mx::T_F16; f.dst_f16 = a->dst_type == mx::T_F16;
    fa_q_plan(f, nsplit);
    return f;
}

// The direct form or decoding first. Direct attention turns codes into operands once for every 16 or 32
// rows, and with many rows that, not the memory, is its time; decoding turns them once and feeds the F16
// kernel, one sequence after another, in two or three launches and 14 us at least each. Direct up to R (D + DV) = 2^16
// (us direct / decoded, 8 KV heads, 4-bit, head dim 128: 128 rows of 8192 keys 28 / 43, 256 42 / 45, 384 61 / 52;
// 256 of 32768 115 / 126, 384 207 / 143; head dim 256, 16384 keys: 128 rows 95 / 148, 192 171 / 147), and up
// to 64 key tiles of 16 rows a compute unit and sequence, which are done before those launches are (512 rows of
// 1000 keys 17 / 25, 768 29 / 25; head dim 64, 1531 keys: 400 rows 16 / 23, 800 22 / 24; head dim 256, 1000
// keys, 512 rows 36 / 71; 32 sequences x 256 rows x 1024 187 / 641).
// Fewer keys than a tile's 32, whose loads the direct form does not bound a lane at a time, are always decoded first: 14 us
// for one sequence (300 keys 10 us), but 477 us for 32 sequences of 31 keys, one after another, where 32 keys take 9.
static bool fa_q_is_direct(const mi355x_fa_q_args * a) {
    if (a->KV < mx::FA_Q_MIN_KV || a->k.nb1 >= mx::FA_Q_MAX_NB1 || a->v.nb1 >= mx::FA_Q_MAX_NB1) return false;
    int D, DV;
    mx::fa_pad_dims(a->D, a->DV, D, DV);
    if (2 * a->D < D || 2 * a->DV < DV) return false;   // its loads of scales
    if (const char * e = getenv("MI355X_FA_Q_DIRECT"))
        if (*e) return atoi(e) != 0;
    const int64_t R = (int64_t)(a->H / a->HK) * a->T;
    return R * (D + DV) <= 65536 || a->HK * ((R + 15) / 16) * ((a->KV + 31) / 32) <= 64 * (int64_t)device_cus();
}
struct FaQDirectLayout {
    size_t po, pml, total;
};
static FaQDirectLayout fa_q_direct_layout(const mx::FaQArgs & f) {
    FaQDirectLayout L;
    const size_t parts = f.nsplit > 1 ? (size_t)f.S * f.HK * f.nrt * f.nsplit : 0;
    L.po = 0;
    L.pml = parts * f.nq * (f.DV / 16) * 1024;
    L.total = L.pml + align256(parts * f.nq * 16 * 8) + 256;
    return L;
}

// Workspace of the decode-first form: one sequence's K and V as fp16, then the fused kernel's own.
struct FaQLayout {
    size_t k, v, fa, total;
};
static FaQLayout fa_q_layout(const mi355x_fa_q_args * a, int nsplit) {
    FaQLayout L;
    const size_t rows = (size_t)a->HK * a->KV;
    L.k = 0;
    L.v = L.k + align256(rows * a->D * 2);
    L.fa = L.v + align256(rows * a->DV * 2);
    const mi355x_fa_args f = fa_q_lower(a, 0, nullptr, nullptr);
    if (nsplit <= 0) nsplit = fa_plan(&f, 0).nsplit;
    L.total = L.fa + align256(fa_layout(fa_lower(&f, nsplit)).total);
    return L;
}

MI355X_API size_t mi355x_flash_attn_q_workspace(const mi355x_fa_q_args * a, int nsplit) {
    if (nsplit > 64 || fa_q_check(a, nsplit) != MI355X_OK) return 0;
    if (a->T == 0 || a->S == 0) return 256;   // nothing to plan for; 0 would say that the op is not taken
    return fa_q_is_direct(a) ? fa_q_direct_layout(fa_q_direct(a, nsplit)).total : fa_q_layout(a, nsplit).total;
}

MI355X_API int mi355x_flash_attn_q(const mi355x_fa_q_args * a, int nsplit, void * workspace_dev, size_t workspace_bytes,
                                   void * stream) {
    if (nsplit > 64) return MI355X_E_ARG;
    const int st = fa_q_check(a, nsplit);
    if (st != MI355X_OK) return st;
    if (a->T == 0 || a->S == 0) return MI355X_OK;
    if (fa_q_is_direct(a)) {
        mx::FaQArgs f = fa_q_direct(a, nsplit);
        const FaQDirectLayout L = fa_q_direct_layout(f);
        if (!workspace_dev || workspace_bytes < L.total || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
        f.part_o = (float *)((char *)workspace_dev + L.po);
        f.part_ml = (float *)((char *)workspace_dev + L.pml);
        return hip_status(mx::launch_fa_q(f, S(stream)));
    }
    const FaQLayout L = fa_q_layout(a, nsplit);
    if (!workspace_dev || workspace_bytes < L.total || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
    char * ws = (char *)workspace_dev;
    for (int s = 0; s < a->S; s++) {
        const mi355x_fa_args one = fa_q_lower(a, s, (const uint16_t *)(ws + L.k), (const uint16_t *)(ws + L.v));
        size_t need;
        const mx::FaArgs f = fa_fused_args(&one, nsplit, a->q_type == mx::T_F16, a->dst_type == mx::T_F16, ws + L.fa, &need);
        if (need > workspace_bytes - L.fa) return MI355X_E_NOMEM;
        if (a->KV > 0) {
            mx::KvDecodeArgs d;
            d.k = fa_q_view(a->k, s);
            d.v = fa_q_view(a->v, s);
            d.k16 = (uint16_t *)(ws + L.k);
            d.v16 = (uint16_t *)(ws + L.v);
            d.HK = a->HK; d.KV = a->KV; d.D = a->D; d.DV = a->DV;
            const int e = hip_status(mx::launch_kv_decode(d, f, S(stream)));
            if (e != MI355X_OK) return e;
        }
        const int e = hip_status(mx::launch_fa(f, a->KV == 0, S(stream)));
        if (e != MI355X_OK) return e;
    }
    return MI355X_OK;
}

// ---- a KV cache in pages ------------------------------------------------------------------------

static int kv_step_lower(const mi355x_kv_step & s, int64_t n_rows, int32_t * err_dev, mx::KvStepArgs & a) {
    if (s.S < 0 || s.T < 0 || s.page <= 0 || s.page % 32 || s.n_table < 0 || s.table_nb < 0 || s.parent_nb < 0) return MI355X_E_ARG;
    if (!aligned(s.table_dev, 4) || !aligned(s.n_past_dev, 4) || !aligned(s.n_new_dev, 4) || !aligned(s.parent_dev, 4) || !aligned(err_dev, 4))
        return MI355X_E_ARG;
    if (s.n_table > (1 << 29) / s.page || (int64_t)s.S * s.T > 1 << 22 || n_rows < 0 || n_rows / s.page > INT32_MAX) return MI355X_E_ARG;
    if (s.parent_dev && s.T > mx::KV_TREE_MAX) return MI355X_E_ARG;
    if (s.S > 0 && s.T > 0 && (!s.table_dev || !s.n_past_dev || s.n_table < 1 || n_rows < s.page)) return MI355X_E_ARG;
    a.table = s.table_dev; a.n_past = s.n_past_dev; a.n_new = s.n_new_dev; a.parent = s.parent_dev; a.err = err_dev;
    a.table_nb = s.table_nb; a.parent_nb = s.parent_nb; a.n_table = (int)s.n_table; a.S = s.S; a.T = s.T; a.page = s.page;
    a.n_pages = (int)(n_rows / s.page);
    a.cap = (int)(s.n_table * s.page);
    a.div_page = mx::fq_div_by(s.page);
    return MI355X_OK;
}

MI355X_API int mi355x_kv_append(const mi355x_kv_append_args * p, int32_t * err_dev, void * stream) {
    if (!p) return MI355X_E_ARG;
    mx::KvAppendArgs a;
    memset(&a, 0, sizeof a);
    // the rows' own checks, as for a store of one row: a cache's rows and the sources' strides do not follow from a count here
    mi355x_kv_rows r[2] = {p->k, p->v};
    mx::KvRowsArgs rows;
    const int64_t n = (int64_t)p->step.S * p->step.T;
    if (r[0].n_rows < 0 || r[1].n_rows < 0) return MI355X_E_ARG;
    int st = kv_step_lower(p->step, std::min(r[0].n_rows, r[1].n_rows), err_dev, a.st);
    if (st != MI355X_OK) return st;
    st = kv_rows_lower(r, 2, nullptr, 26, n > 0, err_dev, true, rows);
    if (st != MI355X_OK) return st;
    const bool queries = p->q_dev || p->qr_dev;
    if (p->k_nb3 < 0 || p->v_nb3 < 0 || p->k_nb3 % 8 || p->v_nb3 % 8 || p->pos_nb < 0 || !aligned(p->pos_dev, 4) || !aligned(p->freq_dev, 4))
        return MI355X_E_ARG;
    if (p->n_rot < 0 || p->n_rot % 8 || p->n_rot > r[0].D || p->n_rot > 256 || (p->n_rot > 0 && n > 0 && !p->freq_dev)) return MI355X_E_ARG;
    if (r[0].H != r[1].H || (queries && (p->H <= 0 || p->H > INT32_MAX / r[0].D))) return MI355X_E_ARG;
    if (queries) {
        for (int t : {p->q_type, p->qr_type})
            if (t != mx::T_F32 && t != mx::T_F16) return MI355X_E_ARG;
        for (int64_t nb : {p->q_nb1, p->q_nb2, p->q_nb3, p->qr_nb1, p->qr_nb2, p->qr_nb3})
            if (nb < 0 || nb % 8) return MI355X_E_ARG;
        if (n > 0 && (!p->q_dev || !p->qr_dev)) return MI355X_E_ARG;
        if (!aligned(p->q_dev, 16) || !aligned(p->qr_dev, 16)) return MI355X_E_ARG;
        // in place: a value that another lane still pairs with its own must not be overwritten
        if (n > 0 && p->q_dev == p->qr_dev && (p->q_type != p->qr_type || p->q_nb1 != p->qr_nb1 || p->q_nb2 != p->qr_nb2 || p->q_nb3 != p->qr_nb3 ||
                                              (p->neox && p->n_rot)))
            return MI355X_E_ARG;
    }
    for (int k = 0; k < 2; k++) {
        mx::KvAppendRows & o = a.r[k];
        o.x = {r[k].x_dev, r[k].x_nb1, r[k].x_nb2, k ? p->v_nb3 : p->k_nb3, r[k].x_type == mx::T_F16};
        o.H = (int)r[k].H; o.bph = (int)(r[k].D / 32); o.rotate = k == 0;
        a.o[k] = rows.o[k];
    }
    a.r[2].x = {(void *)p->q_dev, p->q_nb1, p->q_nb2, p->q_nb3, p->q_type == mx::T_F16};
    a.r[2].H = (int)p->H; a.r[2].bph = a.r[0].bph; a.r[2].rotate = true;
    a.qr = {p->qr_dev, p->qr_nb1, p->qr_nb2, p->qr_nb3, p->qr_type == mx::T_F16};
    a.n_rows = queries ? 3 : 2;
    for (int k = 0; k < a.n_rows; k++)
        if ((int64_t)a.r[k].H * a.r[k].bph > 1 << 16) return MI355X_E_ARG;
    a.freq = p->freq_dev; a.pos = p->pos_dev; a.pos_nb = p->pos_nb; a.half = p->n_rot / 2; a.neox = p->neox != 0; a.mscale = p->mscale;
    return n == 0 ? MI355X_OK : hip_status(mx::launch_kv_append(a, S(stream)));
}

MI355X_API int mi355x_kv_keep(const mi355x_kv_step * step, const mi355x_kv_rows * r, int n_out, const int32_t * path_dev,
                              int64_t path_nb, const int32_t * n_keep_dev, int A, int32_t * err_dev, void * stream) {
    if (!step || !r || n_out < 1 || n_out > mx::KV_MAX_OUT || A < 0 || A > mx::KV_TREE_MAX || path_nb < 0) return MI355X_E_ARG;
    if (!aligned(path_dev, 4) || !aligned(n_keep_dev, 4)) return MI355X_E_ARG;
    const bool some = step->S > 0 && step->T > 0 && A > 0;
    if (some && !path_dev) return MI355X_E_ARG;
    mx::KvKeepArgs a;
    memset(&a, 0, sizeof a);
    int64_t n_rows = INT64_MAX;
    mi355x_kv_rows rows[mx::KV_MAX_OUT];
    for (int k = 0; k < n_out; k++) {   // x is not read: anything that the check of a store takes
        rows[k] = r[k];
        rows[k].x_type = mx::T_F32;
        rows[k].x_dev = rows[k].q_dev;
        rows[k].x_nb1 = rows[k].x_nb2 = 0;
        n_rows = std::min(n_rows, r[k].n_rows);
    }
    int st = kv_step_lower(*step, n_rows, err_dev, a.st);
    if (st != MI355X_OK) return st;
    mx::KvRowsArgs low;
    st = kv_rows_lower(rows, n_out, nullptr, 26, some, err_dev, true, low);
    if (st != MI355X_OK) return st;
    for (int k = 0; k < n_out; k++) {
        if (low.o[k].H * (int64_t)low.o[k].bph > 1 << 16) return MI355X_E_ARG;
        a.o[k] = low.o[k];
    }
    a.n_out = n_out; a.A = A; a.path = path_dev; a.n_keep = n_keep_dev; a.path_nb = path_nb;
    return some ? hip_status(mx::launch_kv_keep(a, S(stream))) : MI355X_OK;
}

// Rows a wave and KV splits over an fp16 cache (mx_fa_pf16.hip): the pair whose estimated time is least. Estimate: a CU holds
// `slots` blocks; a round of blocks takes a start and end and, for each of a wave's tiles, what a tile's chain takes or, if more, what
// the blocks beside each other on a CU take of its units; HBM sets a floor; a split adds the merge. The numbers (us) are fitted to
// some 900 times of 34 shapes a head dim, to 10 to 17 % each; the pair taken is 2 % from the best measured one in the mean (two
// tiles a wave where that filled the chip, and splits up to it: 14 %). Examples, 8 KV heads, best with one row tile / two:
// 512 rows of 16000 keys, head dim 64 56 / 42, 128 107 / 74; 64 rows, head dim 128 30 / 26; 256 rows of 1000 and of 4 sequences, head dim
// 64 12.6 / 15.2, 128 20.6 / 18.5. Not split past one round of blocks: 10 sequences of 3000 keys, 256 rows each, 82 whole and 90 in three.
// The fits are of 8 KV heads: over 18 shapes for each of 1, 4, 16 and 32 it is 5, 3, 2 and 2 % from the best in the mean, at worst 1 head with 32
// query heads of 64 (8 sequences of 4000 keys 15.0 us for 10.4).
struct FpCost {
    int slots[2];                     // one row tile a wave, two
    double ends, chain[2], unit[2];   // a block's start and end; a tile's chain; a CU's units, a tile of each block's waves
    double merge, merge_cu;           // the second launch, and more for each row tile a CU hands it
};
static FpCost fp_cost(int D) {
    return D <= 64    ? FpCost{{4, 3}, 4.2, {0.63, 0.82}, {0.35, 0.53}, 4.4, 0.4}
           : D <= 128 ? FpCost{{2, 2}, 3.9, {1.05, 1.2}, {0.7, 1.2}, 5.4, 1.0}
           : D <= 192 ? FpCost{{1, 1}, 4.1, {1.3, 1.8}, {1.3, 1.8}, 5.3, 1.0}
                      : FpCost{{1, 1}, 6.8, {1.9, 1.9}, {1.9, 1.9}, 5.2, 0.1};
}
static void fa_p_plan_f16(mx::FaPArgs & f, int nsplit) {
    const int64_t cus = device_cus(), ntiles = (f.KV + 31) / 32;
    const FpCost c = fp_cost(f.D);
    const double hbm = (double)f.S * ntiles * 64 * f.HK * (f.D + f.DV) / 4.6e6 + 4.0;
    int first = 1, last = f.D <= 192 && f.R > 16 ? 2 : 1;
    if (const char * e = getenv("MI355X_FA_Q_ROWS"))
        if (*e) first = last = atoi(e) == 32 && f.D <= 192 ? 2 : 1;
    double best = 0.0;
    f.nsplit = 0;
    for (int nq = first; nq <= last; nq++) {
        const int64_t units = (int64_t)f.S * f.HK * ((f.R + 16 * nq - 1) / (16 * nq)), room = c.slots[nq - 1] * cus;
        const int64_t most = nsplit > 0 ? nsplit : std::max<int64_t>(1, std::min<int64_t>({64, room / units, ntiles / 4}));
        for (int64_t ns = nsplit > 0 ? nsplit : 1; ns <= most; ns++) {
            const int64_t blocks = units * ns, chain = ((ntiles + ns - 1) / ns + 3) / 4, rest = blocks % room;
            auto round = [&](int64_t beside) { return c.ends + chain * std::max(c.chain[nq - 1], beside * c.unit[nq - 1]); };
            double t = blocks / room * round(c.slots[nq - 1]) + (rest ? round((rest + cus - 1) / cus) : 0.0);
            t = std::sqrt(std::sqrt(t * t * t * t + hbm * hbm * hbm * hbm));
            if (ns > 1) t += c.merge + c.merge_cu * nq * blocks / cus;
            if (!f.nsplit || t < best) {
                best = t;
                f.nq = nq;
                f.nsplit = (int)ns;
            }
        }
    }
    f.nrt = (f.R + 16 * f.nq - 1) / (16 * f.nq);
    f.div_nrt = mx::fq_div_by(f.nrt); f.div_hk = mx::fq_div_by(f.HK); f.div_split = mx::fq_div_by(f.nsplit); f.div_g = mx::fq_div_by(f.G);
}

static int fa_p_check(const mi355x_fa_p_args * a, int nsplit, mx::FaPArgs & f) {
    memset(&f, 0, sizeof f);
    if (!a) return MI355X_E_ARG;
    const int st = kv_step_lower(a->step, a->n_rows, nullptr, f.st);
    if (st != MI355X_OK) return st;
    const int Sn = a->step.S, T = a->step.T;
    const bool empty = T == 0 || Sn == 0;   // no query: nothing is read or written
    if (!empty && (!a->q_dev || !a->dst_dev)) return MI355X_E_ARG;
    if (a->D <= 0 || a->DV <= 0 || a->D % 32 || a->DV % 32 || !mx::fa_pad_dims(a->D, a->DV, f.D, f.DV)) return MI355X_E_UNSUPPORTED;
    if (2 * a->D < f.D || 2 * a->DV < f.DV) return MI355X_E_UNSUPPORTED;   // the loads of scales
    const bool f16 = a->k.type == mx::T_F16;
    for (const mi355x_kv_view * w : {&a->k, &a->v}) {
        if (f16 ? w->type != mx::T_F16 : !kv_type(w->type)) return MI355X_E_UNSUPPORTED;
        if (w->nb1 < 0 || w->nb2 < 0 || w->nb1 % 32 || w->nb2 % 32 || w->nb1 >= mx::FA_Q_MAX_NB1) return MI355X_E_ARG;
        if ((!empty && !w->q_dev) || !aligned(w->q_dev, 16)) return MI355X_E_ARG;
        if (!f16 && ((!empty && !w->d_dev) || !aligned(w->d_dev, 8))) return MI355X_E_ARG;
    }
    if (a->H <= 0 || a->HK <= 0 || a->H % a->HK || a->max_kv < 0 || nsplit > 64) return MI355X_E_ARG;
    const int64_t tiles = (int64_t)Sn * a->HK * (((int64_t)T * (a->H / a->HK) + 15) / 16);
    if (tiles > (1 << 21) / (nsplit > 1 ? nsplit : 1) || (nsplit > 1 && tiles * f.DV >= 1 << 28)) return MI355X_E_UNSUPPORTED;
    if ((int64_t)Sn * T * a->H > 1 << 30) return MI355X_E_UNSUPPORTED;
    for (int t : {a->q_type, a->dst_type})
        if (t != mx::T_F32 && t != mx::T_F16) return MI355X_E_ARG;
    const int64_t qa = a->q_type == mx::T_F16 ? 8 : 4;
    if (a->q_nb1 % qa || a->q_nb2 % qa || a->q_nb3 % qa || !aligned(a->q_dev, 16)) return MI355X_E_ARG;
    if (a->dst_nb1 % 4 || a->dst_nb2 % 4 || a->dst_nb3 % 4 || !aligned(a->dst_dev, a->dst_type == mx::T_F16 ? 8 : 16)) return MI355X_E_ARG;
    if (empty) return MI355X_OK;
    f.q = a->q_dev; f.dst = a->dst_dev;
    f.k = fa_q_view(a->k, 0); f.v = fa_q_view(a->v, 0);
    f.k.nb3 = f.v.nb3 = 0;
    f.q_nb1 = a->q_nb1; f.q_nb2 = a->q_nb2; f.q_nb3 = a->q_nb3;
    f.dst_nb1 = a->dst_nb1; f.dst_nb2 = a->dst_nb2; f.dst_nb3 = a->dst_nb3;
    f.dk = a->D; f.dv = a->DV;
    if (a->max_kv) f.st.cap = (int)std::min<int64_t>(a->max_kv, f.st.cap);
    f.KV = f.st.cap;
    f.T = T; f.S = Sn; f.HK = a->HK; f.G = a->H / a->HK; f.R = T * f.G;
    f.scale = a->scale; f.softcap = a->softcap;
    f.q_f16 = a->q_type == mx::T_F16; f.dst_f16 = a->dst_type == mx::T_F16;
    if (f16) fa_p_plan_f16(f, nsplit);
    else fa_q_plan(f, nsplit);
    f.div_tpp = mx::fq_div_by(a->step.page / 32);
    return MI355X_OK;
}

// Many rows of a chain over a quantized cache: decoded first, a sequence at a time, as mi355x_flash_attn_q, where that is estimated
// to take a tenth less (the direct form rounds less). Direct: a block's start, end and merge, and its waves' tiles, one after
// another; decoded: launches, the cache's values, the rows' products. The numbers (us) are measured ones of 8 KV heads, 8-bit, F32
// Q; direct / decoded: head dim 64, 384 rows of 16000 keys 76 / 54, of 4000 26 / 28; 128, 128 rows of 16000 50 / 69, 256 78 / 80, 288
// 138 / 83, 512 of 4000 43 / 40, of 1000 18 / 26; 192, 192 rows of 16000 144 / 93; 256, 128 115 / 146, 192 208 / 145, 160 of 4000 51 / 74.
// A tree has 64 tokens at most and is read as stored; an fp16 cache needs no decoding.
struct FpForms {
    int waves;                          // a block's
    double tile, launches, key, row;    // a tile of each; decoded: a sequence, a key of it, and with each row
};
static FpForms fp_forms(int D, int nq) {
    return D <= 64    ? nq == 2 ? FpForms{8, 1.9, 20.0, 1.9e-3, 0.6e-6} : FpForms{12, 1.55, 20.0, 1.9e-3, 0.6e-6}
           : D <= 128 ? FpForms{8, 2.06, 20.0, 2.4e-3, 5.2e-6}
           : D <= 192 ? FpForms{4, 2.2, 20.0, 3.3e-3, 6.6e-6}
                      : FpForms{4, 3.2, 50.0, 5.1e-3, 5.0e-6};
}
static bool fa_p_decodes(const mi355x_fa_p_args * a, const mx::FaPArgs & f) {
    if (a->from_pages || f.k.type == mx::T_F16 || f.st.parent || (size_t)f.KV > mx::fa_max_kv(f.dk, f.dv)) return false;
    if ((int64_t)f.KV * f.HK * ((f.dk + f.dv) / 32) >= 1 << 29) return false;
    if (const char * e = getenv("MI355X_FA_Q_DIRECT"))
        if (*e) return atoi(e) == 0;
    const FpForms c = fp_forms(f.D, f.nq);
    const int64_t cus = device_cus(), blocks = (int64_t)f.S * f.HK * f.nrt * f.nsplit, tiles = (f.KV + 31) / 32;
    const int64_t chain = ((tiles + f.nsplit - 1) / f.nsplit + c.waves - 1) / c.waves;
    const double direct = 12.0 + (double)((blocks + cus - 1) / cus) * chain * c.tile;
    const double decoded = f.S * (c.launches + f.HK / 8.0 * f.KV * (c.key + c.row * f.R));
    return 1.1 * decoded < direct;
}

// The decoded form of `count` tokens of sequence s, from `first` on: the op on fp16 K and V [HK][kvp][D] and the mask [count][kvp] that the
// decoding launch writes.
static mi355x_fa_args fa_p_lower(const mi355x_fa_p_args * a, const mx::FaPArgs & f, int s, int first, int count, char * k16, char * v16, char * mask) {
    mi355x_fa_args o;
    memset(&o, 0, sizeof o);
    const int64_t kvp = (f.KV + 63) / 64 * 64;
    o.q_dev = (const float *)((const char *)a->q_dev + (s * a->q_nb3 + first * a->q_nb1) * (f.q_f16 ? 2 : 4)); o.q_nb1 = a->q_nb1; o.q_nb2 = a->q_nb2;
    o.k_dev = (const uint16_t *)k16; o.k_nb1 = a->D; o.k_nb2 = kvp * a->D;
    o.v_dev = (const uint16_t *)v16; o.v_nb1 = a->DV; o.v_nb2 = kvp * a->DV;
    o.mask_dev = (const uint16_t *)mask; o.mask_nb1 = kvp;
    o.dst_dev = (float *)((char *)a->dst_dev + (s * a->dst_nb3 + first * a->dst_nb2) * (f.dst_f16 ? 2 : 4)); o.dst_nb1 = a->dst_nb1; o.dst_nb2 = a->dst_nb2;
    o.D = a->D; o.DV = a->DV; o.T = count; o.H = a->H; o.KV = (int)kvp; o.HK = a->HK;
    o.scale = a->scale; o.softcap = a->softcap;
    return o;
}
// Only the tiles along the chain's diagonal have a mask that is written and read, but it has a place for every tile. So that
// long chains over long caches do not take gigabytes for it, tokens go through in pieces whose mask is 2^26 values at most (128 MiB: 512 tokens
// of 131072 keys), or 32 tokens'; K and V are decoded once. The splits are those of a whole piece. (32 / 8 heads of 128, 4096 tokens of
// 131072 keys: 656 MiB and 9.9 ms, in one piece 1536 MiB and 9.75 ms; 16384 of 32768 keys 256 MiB for 1152, 7.2 ms either way.)
struct FaPLayout {
    size_t k, v, mask, fa, total;
    int piece, nsplit;
};
static FaPLayout fa_p_layout(const mi355x_fa_p_args * a, const mx::FaPArgs & f, int nsplit) {
    FaPLayout L;
    const size_t kvp = (size_t)(f.KV + 63) / 64 * 64;
    L.piece = (int)std::min<int64_t>(a->step.T, std::max<int64_t>(32, (1 << 26) / (int64_t)kvp / 32 * 32));
    L.k = 0;
    L.v = L.k + align256((size_t)a->HK * kvp * a->D * 2);
    L.mask = L.v + align256((size_t)a->HK * kvp * a->DV * 2);
    L.fa = L.mask + align256((size_t)L.piece * kvp * 2);
    const mi355x_fa_args one = fa_p_lower(a, f, 0, 0, L.piece, nullptr, nullptr, nullptr);
    L.nsplit = nsplit > 0 ? nsplit : fa_plan(&one, 0).nsplit;
    L.total = L.fa + align256(fa_layout(fa_lower(&one, L.nsplit)).total);
    return L;
}

MI355X_API size_t mi355x_flash_attn_paged_workspace(const mi355x_fa_p_args * a, int nsplit) {
    mx::FaPArgs f;
    if (fa_p_check(a, nsplit, f) != MI355X_OK) return 0;
    if (a->step.T == 0 || a->step.S == 0) return 256;
    return fa_p_decodes(a, f) ? fa_p_layout(a, f, nsplit).total : fa_q_direct_layout(f).total;
}

MI355X_API int mi355x_flash_attn_paged(const mi355x_fa_p_args * a, int nsplit, void * workspace_dev, size_t workspace_bytes,
                                       int32_t * err_dev, void * stream) {
    mx::FaPArgs f;
    const int st = fa_p_check(a, nsplit, f);
    if (st != MI355X_OK) return st;
    if (!aligned(err_dev, 4)) return MI355X_E_ARG;
    if (a->step.T == 0 || a->step.S == 0) return MI355X_OK;
    f.st.err = err_dev;
    if (fa_p_decodes(a, f)) {
        const FaPLayout L = fa_p_layout(a, f, nsplit);
        if (!workspace_dev || workspace_bytes < L.total || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
        char * ws = (char *)workspace_dev;
        for (int s = 0; s < a->step.S; s++)
            for (int first = 0; first < a->step.T; first += L.piece) {
                const mi355x_fa_args one = fa_p_lower(a, f, s, first, std::min(L.piece, a->step.T - first), ws + L.k, ws + L.v, ws + L.mask);
                size_t need;
                const mx::FaArgs g = fa_fused_args(&one, L.nsplit, f.q_f16, f.dst_f16, ws + L.fa, &need);
                if (need > workspace_bytes - L.fa) return MI355X_E_NOMEM;
                mx::KvDecodeArgs d;
                memset(&d, 0, sizeof d);
                d.k = f.k; d.v = f.v;
                d.k16 = (uint16_t *)(ws + L.k); d.v16 = (uint16_t *)(ws + L.v);
                d.HK = a->HK; d.KV = one.KV; d.D = a->D; d.DV = a->DV;
                int e = hip_status(mx::launch_kv_decode_paged(d, g, f.st, s, first, (uint16_t *)(ws + L.mask), S(stream)));
                if (e == MI355X_OK) e = hip_status(mx::launch_fa(g, false, S(stream)));
                if (e != MI355X_OK) return e;
            }
        return MI355X_OK;
    }
    const FaQDirectLayout L = fa_q_direct_layout(f);
    if (!workspace_dev || workspace_bytes < L.total || !aligned(workspace_dev, 256)) return MI355X_E_NOMEM;
    f.part_o = (float *)((char *)workspace_dev + L.po);
    f.part_ml = (float *)((char *)workspace_dev + L.pml);
    return hip_status(mx::launch_fa_p(f, S(stream)));
}

// ---- MUL_MAT_ID -------------------------------------------------------------------------------

namespace {

struct MoeLayout {
    size_t a16, scales, off, rows, tiles, n_tiles, err, zero, total;
};

inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

bool moe_layout(const mi355x_moe_args * a, MoeLayout & L) {
    if (!a || a->n_tokens < 0 || a->n_used <= 0 || a->ne11 <= 0 || a->n_expert <= 0 || a->K <= 0 || a->N <= 0)
        return false;
    const size_t rows_b = (size_t)a->n_tokens * a->ne11;
    const size_t R = (size_t)a->n_tokens * a->n_used;
    const size_t tiles = (size_t)mx::moe_max_tiles((int)a->n_tokens, (int)a->n_used, (int)a->n_expert);
    size_t o = 0;
    L.a16 = o;     o += up256(rows_b * a->K * 2);
    L.scales = o;  o += up256(rows_b * 4);
    L.off = o;     o += up256(((size_t)a->n_expert + 1) * 4);
    L.rows = o;    o += up256((R > 0 ? R : 1) * 4);
    L.tiles = o;   o += up256(tiles * 8);
    L.n_tiles = o; o += 256;
    L.err = o;     o += 256;
    L.zero = o;    o += 256;
    L.total = o;
    return true;
}

}  // namespace

MI355X_API size_t mi355x_mul_mat_id_workspace(const mi355x_moe_args * a) {
    MoeLayout L;
    return moe_layout(a, L) ? L.total : 0;
}

MI355X_API int mi355x_mul_mat_id(const mi355x_moe_args * a, void * workspace_dev, size_t workspace_bytes,
                                 int32_t * err_dev, void * stream) {
    MoeLayout L;
    if (!moe_layout(a, L)) return MI355X_E_ARG;
    if (!known_moe_wtype(a->wtype) || a->K % 32 || a->K % blck(a->wtype) || a->N % 16) return MI355X_E_ARG;
    // experts are whole 32-row groups, each plane's share of one expert under 2^31 bytes
    if (x32_wtype(a->wtype) && (a->N % 32 || a->N * a->K > ((int64_t)1 << 31))) return MI355X_E_ARG;
    if (!a->as_dev || !a->b_dev || !a->ids_dev || !a->dst_dev || !aligned(a->as_dev, 16) || !aligned(a->b_dev, 16))
        return MI355X_E_ARG;
    if (a->b_nb1 < a->K || a->b_nb1 % 4 || a->b_nb2 != a->ne11 * a->b_nb1) return MI355X_E_ARG;
    if (a->n_expert * a->N > INT32_MAX || a->n_tokens * a->n_used > INT32_MAX || a->n_expert > 8192 ||
        a->n_tokens * a->ne11 > INT32_MAX || a->K > INT32_MAX)
        return MI355X_E_ARG;
    if (a->n_tokens == 0) return MI355X_OK;
    if (!workspace_dev || workspace_bytes < L.total) return MI355X_E_NOMEM;
    char * ws = (char *)workspace_dev;
    mx::MoeArgs m;
    memset(&m, 0, sizeof(m));
    m.w = a->as_dev; m.E = (int)a->n_expert; m.N = (int)a->N; m.K = (int)a->K;
    m.b = a->b_dev; m.b_nb1 = a->b_nb1; m.ne11 = (int)a->ne11; m.T = (int)a->n_tokens; m.U = (int)a->n_used;
    m.ids = a->ids_dev; m.ids_nb0 = a->ids_nb0; m.ids_nb1 = a->ids_nb1;
    m.dst = a->dst_dev; m.dst_nb1 = a->dst_nb1; m.dst_nb2 = a->dst_nb2;
    m.a16 = (uint16_t *)(ws + L.a16);
    m.scales = (float *)(ws + L.scales);
    m.off = (int32_t *)(ws + L.off);
    m.rows = (int32_t *)(ws + L.rows);
    m.tiles = (int32_t *)(ws + L.tiles);
    m.n_tiles = (int32_t *)(ws + L.n_tiles);
    m.err = err_dev ? err_dev : (int32_t *)(ws + L.err);
    m.zero = (uint16_t *)(ws + L.zero);
    return hip_status(mx::launch_moe(a->wtype, m, S(stream)));
}

}  // extern "C"
