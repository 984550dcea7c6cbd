/* SPDX-License-Identifier: MIT
 *
 * mi355x_kernels.h -- the C ABI of the gfx950 prefill kernels (libmi355x.so).
 *
 * This is the device library of the backend: what librocketnpu is to the reference (its call
 * sites in ggml-rocket.cpp are cited per entry). Plain pointers, sizes and an opaque stream;
 * no ggml or torch types cross it. Every pointer named *_dev is device memory (HBM) that the
 * caller owns; the library allocates nothing inside these calls unless a comment says so.
 * `stream` is a hipStream_t (NULL = the legacy default stream). Every call is asynchronous on
 * that stream and returns a status (MI355X_OK = 0, or a negative code below).
 *
 * Layouts follow ggml's contiguous tensors:
 *   MUL_MAT      W [N][K] (src0 ne=[K,N]), X [M][K] F32 (src1 ne=[K,M]), dst [M][N] F32.
 *   FLASH_ATTN   q [H][T][D] F32, k [HK][KV][D] fp16, v [HK][KV][DV] fp16,
 *                mask [T'][KV'] fp16 (T' >= T, KV' >= KV), dst [T][H][DV] F32.
 *   MUL_MAT_ID   as [E][N][K], b [T][ne11][K] F32, ids [T][n_used] I32, dst [T][n_used][N] F32.
 *
 * Weight types are ggml type ids: F16 = 1, Q4_0 = 2, Q8_0 = 8, Q4_K = 12, Q5_K = 13, Q6_K = 14,
 * MXFP4 = 39. A weight reaches a GEMM in its HBM layout: F16, Q4_K and Q5_K are the ggml payload
 * unchanged; Q4_0, Q8_0, Q6_K and MXFP4 are re-laid out once by mi355x_weight_pack (same bytes,
 * split into 16-byte-aligned planes).
 */
#ifndef MI355X_KERNELS_H
#define MI355X_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI355X_API __attribute__((visibility("default")))

enum mi355x_status {
    MI355X_OK = 0,
    MI355X_E_ARG = -1,          /* a shape, stride, alignment or type the entry does not take */
    MI355X_E_DEVICE = -2,       /* a HIP error: launch, copy or allocation failure */
    MI355X_E_UNSUPPORTED = -3,  /* a structural decline (like ROCKET_E_UNSUPPORTED) */
    MI355X_E_NOMEM = -4,        /* workspace too small */
    MI355X_E_IDS = -5,          /* MUL_MAT_ID: an expert id outside [0, n_expert) */
};

enum mi355x_wtype { MI355X_F16 = 1, MI355X_Q4_0 = 2, MI355X_Q8_0 = 8, MI355X_Q4_K = 12, MI355X_Q5_K = 13,
                    MI355X_Q6_K = 14, MI355X_MXFP4 = 39,
                    /* not a ggml type: fp16 [rows][K] in 16 x 32 tiles of 1 KB, row-major inside,
                     * tile (r/16, k/32) at element ((r/16)*(K/32) + k/32)*512; rows padded to a
                     * multiple of 16 (padding never read). The resident fp16 form the GEMM streams
                     * fastest: each 64-lane load instruction reads one whole tile. */
                    MI355X_F16_T = 0x101,
                    /* not a ggml type: Q4_K blocks of [rows][K] (rows % 32 == 0) regrouped by 32
                     * rows, for expert stacks (mi355x_mul_mat_id only): for each group of 32 rows
                     * and 256-value block, the 32 rows' 16-byte headers (d, dmin, scales), then
                     * for each 64-value quarter the 32 rows' 32 bytes of nibbles. Same bytes as
                     * Q4_K; a wave's loads of a quarter are one contiguous KiB. Built from ggml
                     * Q4_K blocks by mi355x_weight_pack. */
                    MI355X_Q4_K_X = 0x10C,
                    /* not ggml types: Q8_0 / MXFP4 blocks of [rows][K] (rows % 32 == 0) regrouped
                     * by 32 rows, for expert stacks (mi355x_mul_mat_id only). Two planes, each in
                     * (32-row group, 32-value block, row) order: the quants (Q8_0: 32 int8 a
                     * block, MXFP4: 16 bytes of FP4 codes), then the block scales (Q8_0: fp16 d,
                     * MXFP4: the E8M0 byte). Same bytes as the ggml blocks; a wave's quant load
                     * of a block is 1 KiB (Q8_0) or 512 B (MXFP4) of consecutive bytes. Built from
                     * ggml blocks by mi355x_weight_pack. */
                    MI355X_Q8_0_X = 0x108, MI355X_MXFP4_X = 0x127,
                    /* not a ggml type: Q6_K blocks of [rows][K] (rows % 32 == 0) regrouped by 32
                     * rows, for expert stacks (mi355x_mul_mat_id only): the four planes ql, qh,
                     * scales, d, each in (32-row group, 256-value block) order, ql and qh as
                     * [16-byte chunk][row], scales as [row][16 bytes], d as [row]. Same bytes as
                     * the ggml blocks. Built from ggml Q6_K blocks by mi355x_weight_pack. */
                    MI355X_Q6_K_X = 0x10E };

typedef struct mi355x_device_info {
    char name[64];              /* e.g. "gfx950" */
    int  compute_units;
    int  lds_bytes_per_block;
    int  clock_khz;
    size_t hbm_total;
    size_t hbm_free;
} mi355x_device_info;

/* The current device's properties. Replaces rocket_hw_current() (ggml-rocket.cpp:4402, 7262)
 * and rocket_driver_name() (7273), which describe the NPU part and its driver. */
MI355X_API int mi355x_get_device_info(mi355x_device_info * out);

/* Human-readable text for a status code. */
MI355X_API const char * mi355x_status_str(int status);

/* ---- weights ------------------------------------------------------------------------------ */

/* Bytes of `rows` rows of K values of `wtype` in HBM layout (equal to the ggml payload size),
 * or -1 if K is not a whole number of the type's blocks. */
MI355X_API int64_t mi355x_weight_bytes(int wtype, int64_t rows, int64_t K);

/* ggml payload (device) -> HBM layout (device). For F16, Q4_K and Q5_K this is a copy (or
 * nothing, when src_dev == dst_dev); the split layouts need dst_dev != src_dev. Replaces the resident pack rocket_weights_pack (ggml-rocket.cpp:
 * 4362) and its segment form rocket_weights_pack_seg (5121). */
MI355X_API int mi355x_weight_pack(int wtype, const void * src_dev, int64_t rows, int64_t K,
                                  void * dst_dev, void * stream);

/* A weight in HBM layout -> fp16 [rows][K]: each value decoded exactly as ggml's dequantizer
 * does, then rounded once to fp16. The on-device form of rocket_weight_to_fp16 (ggml-rocket.cpp:
 * 3843-3931), used for the resident-fp16 ("prepacked-q") cache. */
MI355X_API int mi355x_weight_dequant_f16(int wtype, const void * w_dev, int64_t rows, int64_t K,
                                         uint16_t * out_dev, void * stream);

/* A weight in HBM layout (any weight type above) -> MI355X_F16_T, decoded exactly as
 * mi355x_weight_dequant_f16 decodes it (the same fp16 values, tiled). K % 64 == 0; out_dev holds
 * mi355x_weight_bytes(MI355X_F16_T, rows, K) bytes and does not alias w_dev. The tiled resident
 * form of rocket_weight_to_fp16 + the resident pack (ggml-rocket.cpp:3843-3931, 4362). */
MI355X_API int mi355x_weight_f16_tiled(int wtype, const void * w_dev, int64_t rows, int64_t K,
                                       uint16_t * out_dev, void * stream);

/* F32 (type 0) or BF16 (type 30) values -> fp16, round to nearest even: the resident form of an
 * F32 / BF16 weight (the F32 and BF16 branches of rocket_weight_to_fp16, ggml-rocket.cpp:
 * 3855-3890). n values; src 4- or 2-byte aligned, dst 2-byte aligned. */
MI355X_API int mi355x_convert_f16(int type, const void * src_dev, int64_t n, uint16_t * dst_dev, void * stream);

/* ---- MUL_MAT ----------------------------------------------------------------------------- */

/* F32 activations [M][ldx] -> fp16 [M][K] divided by each row's max |x| (1 for a zero row),
 * and the row scales [M]. The device form of rocket_pack_activations (ggml-rocket.cpp:
 * 1451-1502). K % 4 == 0, ldx % 4 == 0, x 16-byte aligned. */
MI355X_API int mi355x_pack_act(const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                               uint16_t * a16_dev, float * scales_dev, void * stream);

/* mi355x_pack_act (tiled != 0: mi355x_pack_act_tiled) that also clears columns [0, n_clear) of
 * the M rows of an F32 matrix clear_dev (row stride ld_clear elements): the output of a GEMM that
 * adds a two-way K split into it (mi355x_gemm_accumulates), cleared in the same launch instead
 * of by a fill of the GEMM's own (pass MI355X_GEMM_OUT_ZEROED to mi355x_gemm_ws). No counterpart
 * in the reference, whose NPU GEMM writes its output. */
MI355X_API int mi355x_pack_act_clear(int tiled, const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                                     uint16_t * a16_dev, float * scales_dev, float * clear_dev, int64_t ld_clear,
                                     int64_t n_clear, void * stream);

/* mi355x_pack_act with the fp16 output in the MI355X_F16_T layout (ceil(M/16)*16 rows; the
 * padding rows are never read), for a GEMM on MI355X_F16_T weights. K % 32 == 0. Same values and
 * scales as mi355x_pack_act (rocket_pack_activations, ggml-rocket.cpp:1451-1502). */
MI355X_API int mi355x_pack_act_tiled(const float * x_dev, int64_t ldx, int64_t M, int64_t K,
                                     uint16_t * a16_dev, float * scales_dev, void * stream);

/* One output of a (fused) GEMM launch. */
typedef struct mi355x_gemm_out {
    const void * w_dev;     /* weight panel in HBM layout */
    int64_t rows_total;     /* rows of the whole panel (the split layouts index planes by it) */
    int64_t row0;           /* first row of this weight in the panel */
    int64_t N;              /* rows of this weight = output columns; N % 16 == 0 */
    float * c_dev;          /* output [M][ldc] F32 */
    int64_t ldc;
} mi355x_gemm_out;

/* c[m][n] = scales[m] * sum_k a16[m][k] * w[row0 + n][k], for each of `n_out` (1..4) weights of
 * one type that share the activation, in ONE launch over their concatenated N. fp16 MFMA, fp32
 * accumulation, F32 output. K % 32 == 0 (and a whole number of the type's blocks). For
 * MI355X_F16_T weights a16 is tiled too (mi355x_pack_act_tiled).
 * Replaces rocket_matmul_fp16_prepacked (ggml-rocket.cpp:4449, 5144),
 * rocket_matmul_fp16_stream (4834), rocket_matmul_fp16_mt (4844) and the fused
 * rocket_matmul_fp16_stream_fused (5004).
 * Results are reproducible: equal inputs give equal bits on every call. A launch may split K
 * over blocks; this entry has no workspace, so it splits at most two ways, adding both parts
 * into the zeroed output (two addends on zero sum the same in either order). Wider splits, the
 * fast form for M <= 128 and for deep K, need mi355x_gemm_ws. */
MI355X_API int mi355x_gemm(int wtype, const uint16_t * a16_dev, const float * scales_dev,
                           int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                           void * stream);

/* Bytes of device workspace with which mi355x_gemm_ws runs this launch's fastest K split: one
 * F32 slab [M][sum of the outputs' N] per split when it splits more than two ways, else 0 (0 also
 * for invalid arguments; the pointers in `outs` are not read). */
MI355X_API size_t mi355x_gemm_workspace(int wtype, int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out);

/* mi355x_gemm with a workspace (16-byte aligned) for the partial sums of a K split past two ways.
 * Each split writes its slab; a second launch sums the slabs in split order into the outputs,
 * so the result does not depend on the order in which blocks finish (reproducible, as the CPU
 * backend's MUL_MAT is). With fewer bytes than mi355x_gemm_workspace asks, the split narrows to
 * what fits (down to two ways). The same bytes give the same bits on every call; a different
 * workspace size may pick a different split and round differently. */
MI355X_API int mi355x_gemm_ws(int wtype, const uint16_t * a16_dev, const float * scales_dev,
                              int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                              void * workspace_dev, size_t workspace_bytes, int flags, void * stream);

/* flags of mi355x_gemm_ws: the outputs are already zero (cleared by mi355x_pack_act_clear), so a
 * launch that adds a two-way split into them launches no fill of its own. */
#define MI355X_GEMM_OUT_ZEROED 1

/* 1 if mi355x_gemm_ws with `workspace_bytes` of workspace adds a two-way K split into zeroed
 * outputs for this launch (the outputs must then be zero: cleared by the caller, with
 * MI355X_GEMM_OUT_ZEROED, or by the launch itself), 0 if it writes them, or a negative status
 * for arguments mi355x_gemm_ws would refuse (the pointers in `outs` are not read). */
MI355X_API int mi355x_gemm_accumulates(int wtype, int64_t M, int64_t K, const mi355x_gemm_out * outs, int n_out,
                                       size_t workspace_bytes);

/* 1 if a MUL_MAT of M rows with this weight layout and N x K weight runs faster in the
 * decode-first form (the weight decoded once into tiled fp16, mi355x_weight_f16_tiled, then
 * multiplied as MI355X_F16_T) than decoded inside the GEMM, else 0 (lines measured on MI355X,
 * K % 64 == 0): never for M <= 128; above that for weights of 2^22 to 2^25 values, from M 384 (Q4_0,
 * Q5_K, Q6_K, MXFP4), 768 (Q8_0) or 1024 (Q4_K) for larger ones, with exceptions for Q4_K and
 * Q8_0 where the all-DMA kernel fills the chip or splits a deep K; smaller weights from M 512 or 1024.
 * No counterpart in the reference, whose per-call fp16 route always decodes first. */
MI355X_API int mi355x_mul_mat_decode_first(int wtype, int64_t M, int64_t N, int64_t K);

/* Workspace bytes mi355x_mul_mat needs for M rows of K: the activation pack. */
MI355X_API size_t mi355x_mul_mat_workspace(int64_t M, int64_t K);

/* Workspace bytes with which mi355x_mul_mat runs its fastest form for this shape: the pack,
 * then (from the next 256-byte boundary) the decode-first form's tiled fp16 weight where that
 * form runs (mi355x_mul_mat_decode_first), then the split
 * partials mi355x_gemm_workspace names. */
MI355X_API size_t mi355x_mul_mat_workspace_for(int wtype, int64_t N, int64_t K, int64_t M);

/* dst[M][ldd] = x[M][ldx] . w[N][K]^T: mi355x_pack_act (mi355x_pack_act_tiled for MI355X_F16_T)
 * then mi355x_gemm_ws, the activation pack at the start of `workspace_dev` and the K-split
 * partials in the bytes past it (mi355x_mul_mat_workspace_for sizes both; with only
 * mi355x_mul_mat_workspace bytes the split is at most two ways). Reproducible as mi355x_gemm_ws.
 * Decode-first form: where mi355x_mul_mat_decode_first says so, the weight is decoded once per
 * call into tiled fp16 in the workspace
 * (mi355x_weight_f16_tiled) and multiplied as MI355X_F16_T, when the workspace holds that
 * weight; the same fp16 weights and activations as the in-GEMM decode, faster at those shapes.
 * The whole MUL_MAT of ggml-rocket.cpp:4548-4871 on device. */
MI355X_API int mi355x_mul_mat(int wtype, const void * w_dev, int64_t N, int64_t K,
                              const float * x_dev, int64_t ldx, int64_t M,
                              float * dst_dev, int64_t ldd,
                              void * workspace_dev, size_t workspace_bytes, void * stream);

/* Bytes of the static device scratch of mi355x_mul_mat_noalloc (64 MiB per GPU). */
#define MI355X_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* mi355x_mul_mat without a workspace argument: no counterpart in the reference. For callers
 * that cannot allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). The workspace lives in a file-scope device array of
 * MI355X_NOALLOC_SCRATCH_BYTES per GPU, held until the process ends; the call allocates nothing
 * and frees nothing. Limit: mi355x_mul_mat_workspace(M, K) <= MI355X_NOALLOC_SCRATCH_BYTES
 * (e.g. M 2048 at K 14336), else MI355X_E_NOMEM with a message. Every call on one GPU shares
 * that GPU's array: calls that overlap on one GPU (two streams, two threads) race and must be
 * serialized by the caller. The first call on a device resolves the array's address there
 * (make it outside a stream capture); later calls may be captured. It computes exactly what
 * mi355x_mul_mat computes given MI355X_NOALLOC_SCRATCH_BYTES of workspace: the scratch holds
 * the activation pack, then, where the decode-first form runs (mi355x_mul_mat_decode_first) and
 * the pack plus the tiled fp16 weight fit, that weight, and the K-split partials in what is left.
 * So the form depends on the fit: a quantized weight whose fp16 image does not fit beside the
 * pack (e.g. Q6_K 8192 x 4096 at M 512: 4 MiB + 64 MiB) is decoded inside the GEMM here while
 * mi355x_mul_mat with mi355x_mul_mat_workspace_for bytes decodes it first; both forms meet the
 * same MUL_MAT bars, but their bits can differ in the last place. */
MI355X_API int mi355x_mul_mat_noalloc(int wtype, const void * w_dev, int64_t N, int64_t K,
                                      const float * x_dev, int64_t ldx, int64_t M,
                                      float * dst_dev, int64_t ldd, void * stream);

/* ---- FLASH_ATTN_EXT ---------------------------------------------------------------------- */

/* One attention op. Strides are in ELEMENTS, so strided ggml views (a KV-cache slice, a
 * permuted Q) are read in place. */
typedef struct mi355x_fa_args {
    const float * q_dev;      int64_t q_nb1, q_nb2;      /* token, head strides */
    const uint16_t * k_dev;   int64_t k_nb1, k_nb2;      /* key, kv-head strides (fp16) */
    const uint16_t * v_dev;   int64_t v_nb1, v_nb2;      /* key, kv-head strides (fp16) */
    const uint16_t * mask_dev; int64_t mask_nb1;         /* token stride; NULL = unmasked */
    float * dst_dev;          int64_t dst_nb1, dst_nb2;  /* head, token strides */
    int D, DV, T, H, KV, HK;
    float scale, max_bias, softcap;
} mi355x_fa_args;

/* The KV-split count mi355x_flash_attn uses when called with nsplit = 0 (for head dims past 256: 1, or the
 * fused MLA's own, whatever nsplit is). The launch is planned per
 * call: the block layout (two or four 32-query tasks per block) and the split that together
 * minimise an estimate from measured per-step costs; MI355X_FA_TASKS=2|4 in the environment pins
 * the layout (for tests). The result does not depend on the layout beyond fp32 summation order. */
MI355X_API int mi355x_flash_attn_auto_split(const mi355x_fa_args * a);

/* Workspace bytes for `nsplit` KV splits (0 = auto): the per-tile mask classes, 16 zero bytes
 * (the source of zero-padded head dims) and, for nsplit > 1, the partial outputs and their
 * (max, sum); for head dims past 256, the fp16 queries, one KV head's keys and transposed
 * values, and a chunk of query rows' scores and fp16 P (at most 64 MiB of F32 scores); for the
 * absorbed MLA's 576 / 512 the larger of that and the fused form's classes and partials (as above, with
 * a split of its own), so it does not depend on where V lies. Always
 * non-zero for a valid op; the workspace must be 256-byte aligned. */
MI355X_API size_t mi355x_flash_attn_workspace(const mi355x_fa_args * a, int nsplit);

/* dst = softmax(cap(scale * q.k) + mask) . v for every (token, head); head h reads KV head
 * h / (H / HK). On `stream`: a prep pass over the mask, the attention, and for a KV split a
 * launch that merges the splits.
 * Concurrent calls must not share a workspace. D and DV up to 256, multiples of 8, run fused (the
 * kernels are built for (64, 64), (128, 128), the MLA (192, 128) and (256, 256); other dims run
 * zero-padded on the smallest that holds them); past 256 (the absorbed MLA's 576 / 512: D % 32
 * == 0, DV % 8 == 0, both up to 1024) as two GEMMs around a softmax pass over a bounded chunk
 * of query rows at a time, with no KV split, or, for 576 / 512 with V the first 512 dims of K (v_dev ==
 * k_dev, the same strides), fused, choosing its own KV split; H % HK == 0; max_bias
 * must be 0 (no ALiBi); the mask
 * covers [T][KV] with mask_nb1 % 4 == 0; q rows and dst rows 16-byte aligned; k/v rows 16-byte
 * aligned. Rows whose every key is masked are written as zeros. Replaces
 * rocket_flash_attn_fp16_ctx / _mt (ggml-rocket.cpp:5589-5606) and, because no fp16 score
 * surface exists here, the range fallback rocket_fa_ref_f32 (5617-5626) as well. */
MI355X_API int mi355x_flash_attn(const mi355x_fa_args * a, int nsplit,
                                 void * workspace_dev, size_t workspace_bytes, void * stream);

/* mi355x_flash_attn with flags. MI355X_FA_CLASSES_READY: skip the prep pass, because this
 * workspace already holds its results for this mask -- written by an earlier call on the same
 * stream with the same mask bytes, T, KV, head dims and split (nsplit as resolved), and not
 * overwritten since. A graph's layers share one KQ mask per micro-batch, so the first attention
 * of the micro-batch classifies the mask tiles and the others reuse them. The flag is ignored for
 * head dims past 256. No counterpart in the reference (its NPU path has no prep pass). */
#define MI355X_FA_CLASSES_READY 1
MI355X_API int mi355x_flash_attn_ex(const mi355x_fa_args * a, int nsplit, int flags,
                                    void * workspace_dev, size_t workspace_bytes, void * stream);

/* ---- the quantized KV cache: SET_ROWS, GET_ROWS, FLASH_ATTN_EXT over it ---------------------- */

/* A cache of type MI355X_Q8_0 or MI355X_Q4_0 is two planes that share one set of element strides
 * (every stride a multiple of 32, the block length): the codes (element e at byte e for Q8_0, byte
 * e / 2 for Q4_0) and the blocks' fp16 scales (the scale of element e at index e / 32). Inside a
 * block of 32 the bytes are ggml's: Q8_0 an int8 a value, Q4_0 16 bytes with value j in the low and
 * value j + 16 in the high nibble of byte j; Q8_0 stands for d * code, Q4_0 for d * (code - 8). So a
 * cache that mi355x_weight_pack made from ggml blocks is one too, its scales right behind its codes.
 * An MI355X_F16 cache is the plain fp16 tensor, without scales. */

/* The rows of one cache and plain values beside them. Strides in ELEMENTS. */
typedef struct mi355x_kv_rows {
    int type;                 /* MI355X_Q8_0, MI355X_Q4_0 or MI355X_F16 */
    void * q_dev;             /* codes (F16: values) of the cache, 16-byte aligned */
    uint16_t * d_dev;         /* block scales, 8-byte aligned (F16: not read) */
    int64_t n_rows;           /* rows of the cache: an index lies in [0, n_rows) */
    int64_t nb1, nb2;         /* row and head strides of the cache */
    int64_t H, D;             /* heads a row, values a head (D % 32 == 0) */
    int x_type;               /* the plain values: 0 F32 or 1 F16 */
    void * x_dev;             /* [n][H][D], 16-byte aligned */
    int64_t x_nb1, x_nb2;     /* their row and head strides (multiples of 8) */
} mi355x_kv_rows;

/* ggml's SET_ROWS into a cache: row i of the plain values of each of `n_out` (1..4) caches is
 * quantized and written to cache row idx[i], for every i < n, all caches in the same launches (a layer's K and V
 * share their indices), one for every 16384 rows. idx_dev: int32 (idx_type 26) or int64 (27) [n] on the device, or NULL for idx[i] = i.
 * Where an index repeats, the row with the largest i stays, whole. An index outside [0, n_rows)
 * writes nothing and sets *err_dev (a device int32, may be NULL) to 1. Rows that no index names keep
 * their bytes.
 * Bits are those of ggml's reference quantizers: Q8_0 d = max|x| / 127, Q4_0 d = (the value of largest
 * magnitude, the first of equals) / -8, code = x * (1 / d) rounded half away from zero (Q4_0: plus 8.5,
 * truncated, at most 15), each step rounded to f32, d stored as fp16 (infinite past 65504, as
 * ggml's). A block that holds a NaN or an infinity, for which ggml defines nothing, is stored with
 * a NaN scale and reads back as NaN. F16: round to nearest even.
 * Caches of one call must not overlap (two at one address are refused; mi355x_get_rows: nor their x).
 * n and n * H * D / 32, summed over the caches, are at most 2^30, H * D / 32 at most 2^24.
 * No counterpart in the reference, whose host writes its caches on the CPU. */
MI355X_API int mi355x_set_rows(const mi355x_kv_rows * r, int n_out, const void * idx_dev, int idx_type, int64_t n,
                               int32_t * err_dev, void * stream);

/* ggml's GET_ROWS from a cache: cache row idx[i] as plain values in row i of x, for each of `n_out`
 * caches, in one launch for every 2^24 blocks. F32 values are exact; F16 ones are rounded once (mi355x_weight_dequant_f16's
 * values). Indices as in mi355x_set_rows; one outside [0, n_rows) leaves its row of x unwritten and
 * sets *err_dev. */
MI355X_API int mi355x_get_rows(const mi355x_kv_rows * r, int n_out, const void * idx_dev, int idx_type, int64_t n,
                               int32_t * err_dev, void * stream);

/* A quantized K or V: strides in ELEMENTS, multiples of 32. */
typedef struct mi355x_kv_view {
    int type;                          /* MI355X_Q8_0 or MI355X_Q4_0 */
    const void * q_dev;                /* codes, 16-byte aligned */
    const uint16_t * d_dev;            /* block scales, 8-byte aligned */
    int64_t nb1, nb2, nb3;             /* key, KV head and sequence strides */
} mi355x_kv_view;

/* One attention op over a quantized cache, for S sequences (ggml's ne[3]). Strides in ELEMENTS. */
typedef struct mi355x_fa_q_args {
    const void * q_dev;       int64_t q_nb1, q_nb2, q_nb3;     /* token, head, sequence strides */
    mi355x_kv_view k, v;
    const uint16_t * mask_dev; int64_t mask_nb1, mask_nb3;     /* fp16; token, sequence strides (nb3 0: one mask for all); NULL = unmasked */
    void * dst_dev;           int64_t dst_nb1, dst_nb2, dst_nb3;  /* head, token, sequence strides */
    int q_type, dst_type;                                      /* 0 F32 or 1 F16 */
    int D, DV, T, H, KV, HK, S;
    float scale, max_bias, softcap;
} mi355x_fa_q_args;

/* Workspace bytes of mi355x_flash_attn_q with `nsplit` KV splits (0 = its own choice); 0 for an op it
 * does not take (an op without query rows or sequences is taken and needs next to none). 256-byte aligned. */
MI355X_API size_t mi355x_flash_attn_q_workspace(const mi355x_fa_q_args * a, int nsplit);

/* mi355x_flash_attn with K and V in a quantized cache, each Q8_0 or Q4_0: dst = softmax(cap(scale *
 * q.k) + mask) . v. The products' operands are fp16, rounded once, sums F32: Q and P in both forms below, K's and
 * V's values where the cache is decoded first, P times the scale of V's block where it is read as stored (that product
 * is also off by up to 2^-32 of the largest scale of its 32 dims). An F32 dst holds values of that accuracy, some 4e-4 of an
 * output's norm. So that the values stay inside fp16, a scale counts as at most 515.5 (Q8_0: 65468 / 127) or 8188 (Q4_0:
 * 65504 / 8). D and DV are multiples of 32
 * up to 256; H % HK == 0; max_bias 0; KV * HK * (D + DV) / 32 < 2^29, and
 * S * HK row tiles of 16 (T * H / HK rows), times nsplit, at most 2^21 (with nsplit > 1, tiles times DV also below 2^28, DV
 * counted as 64, 128 or 256). A key that the mask hides from a
 * query (-inf) adds nothing to it, whatever the cache holds there, NaN included; a key with a scale
 * that is not finite makes the rows of the queries that see it NaN; rows whose every key is hidden are
 * written as zeros. q rows 16-byte, dst rows 16-byte (F16: 8), mask rows 8-byte aligned.
 * Few rows are taken by a kernel that reads the cache as it is stored, in any number of sequences; many by
 * decoding it to fp16 in the workspace, a sequence at a time, for the kernel of mi355x_flash_attn. The
 * choice follows measured costs; MI355X_FA_Q_DIRECT=1|0 pins it and MI355X_FA_Q_ROWS=16|32 the rows a
 * wave of the first takes at head dims up to 64, for measurements and tests.
 * Concurrent calls must not share a workspace. Equal inputs give equal bits. */
MI355X_API int mi355x_flash_attn_q(const mi355x_fa_q_args * a, int nsplit, void * workspace_dev, size_t workspace_bytes,
                                   void * stream);

/* ---- a KV cache in pages: append, attention of chains and trees of new tokens, keep ----------- */

/* A step of S sequences over caches in pages. The cache is rows [n_rows][HK][D], page p its rows p * page
 * up to p * page + page - 1 (rows behind the last whole page belong to none). Sequence s has logical rows j: row
 * table[s][j / page] * page + j % page of the cache. It holds n_past[s] of them; this step's tokens t < n_new[s] are its
 * logical rows n_past[s] + t, the others up to T are padding. parent[s][t], if given, makes the tokens a tree:
 * the number of the token that t follows, before its own, or -1 for one that follows the n_past rows;
 * without it each follows the one before. All of it is read on the device, when the call runs: a captured call
 * follows the lengths and tables of its replay. A token whose way up its parents meets any other number counts
 * as padding. n_past outside [0, n_table * page] counts as a sequence without new tokens, n_new outside [0, T] as
 * the nearest of the two; logical rows behind the table and rows of pages that the cache does not have are neither
 * read nor written. Each of these sets *err_dev of the call (a device int32, may be NULL) to 1; table entries that no
 * row needs are not looked at. */
typedef struct mi355x_kv_step {
    const int32_t * table_dev;  int64_t table_nb;    /* [S][n_table], sequence stride in elements */
    const int32_t * n_past_dev;                      /* [S] */
    const int32_t * n_new_dev;                       /* [S], or NULL: T */
    const int32_t * parent_dev; int64_t parent_nb;   /* [S][T], T <= 64, or NULL */
    int64_t n_table;                                 /* entries a sequence, n_table * page <= 2^29 */
    int S, T, page;                                  /* page: a multiple of 32; S * T <= 2^22 */
} mi355x_kv_step;

/* Position rotation and storing of a step's tokens: the keys x of `k`, rotated, and the values x of `v` go to the
 * rows of their tokens, as mi355x_set_rows stores them (types, bits and plain types as there; x_nb1 and x_nb2 are the
 * token and head strides, k_nb3 and v_nb3 the sequence strides; n_rows the caches' rows); the queries q [S][T][H][D of k],
 * rotated, to qr. q_dev NULL: no queries. q and qr are each F32 (0) or F16 (1); qr may be q where types and strides agree
 * and n_rot is 0 or the pairs are neighbours (neox 0).
 * Pair i < n_rot / 2 of a head's dims, (2 i, 2 i + 1) or with neox (i, i + n_rot / 2), turns by theta = p * freq_dev[i], p the
 * position pos_dev[s][t], or, without it, n_past[s] plus the number of tokens above t: c = cos(theta) * mscale and s
 * likewise are formed in 64 bits and rounded to f32, then a' = a c - b s and b' = a s + b c with every product and sum
 * rounded to f32; |theta| below 2^40. n_rot: a multiple of 8 up to D and 256, or 0. Dims from n_rot on stay as they are.
 * One launch, or one for every 2^16 tokens of a sequence, or for every so many sequences as may write 2048 pages.
 * Where tables share a page and two tokens' rows are one, the last token's (by sequence, then number) stays, whole.
 * Rows and queries of padding are left as they were. A token without a row in the cache is not stored; its query is
 * rotated. K and V are different caches. H * D / 32 of each at most 2^16. */
typedef struct mi355x_kv_append_args {
    mi355x_kv_step step;
    mi355x_kv_rows k, v;
    int64_t k_nb3, v_nb3;
    const void * q_dev;   int64_t q_nb1, q_nb2, q_nb3;      /* token, head, sequence strides, multiples of 8 */
    void * qr_dev;        int64_t qr_nb1, qr_nb2, qr_nb3;
    int q_type, qr_type;
    int64_t H;
    const float * freq_dev;
    const int32_t * pos_dev; int64_t pos_nb;                /* [S][T], sequence stride; or NULL */
    int n_rot, neox;
    float mscale;
} mi355x_kv_append_args;
MI355X_API int mi355x_kv_append(const mi355x_kv_append_args * a, int32_t * err_dev, void * stream);

/* Attention of a step's tokens over a cache in pages, K and V [n_rows][HK][D] each Q8_0 or Q4_0 (any mix), or both
 * F16 (values at q_dev, d_dev not read): dst[s][t] = softmax over the keys that t sees of cap(scale * q.k), times v.
 * Token t of sequence s sees its n_past[s] rows, itself and the tokens above it. Padding, and a token none of whose keys
 * lies in the cache, are written as zeros. A key that a token does not see adds nothing to it, whatever the cache holds there, NaN
 * included; one that it sees makes it NaN where a block's scale is not finite, and where an F16 V is not, that dim at least not
 * finite. Limits of the values as in mi355x_flash_attn_q; roundings, read from the pages, of the matrix unit's operands to
 * fp16: P times the scale of V's block (an fp16 cache: P) once, Q only where it is F32 and then by 2^-22 of itself and 2^-27 of its
 * row's largest value (F16: by 2^-35 of that one, where it is 128 or more and the cache quantized); an output
 * is 1.7e-4 of its norm from the 64-bit value then, and an fp16 one's own rounding 2.1e-4. Decoded first: as there.
 * max_kv: a number that no n_past + n_new passes (0: n_table * page). The launch and its workspace are planned for it;
 * it takes the place of n_table * page in what the step says of numbers out of range.
 * H % HK == 0; D and DV multiples of 32 up to 256, each at least half of what the kernels are built for (64 / 64, 128 / 128,
 * 192 / 128, 256 / 256, the smallest that holds both); S * HK row tiles of 16 (T * H / HK rows) as there. Few rows, trees and
 * fp16 caches are taken from the pages as they are; many rows of a chain over a quantized cache by decoding it to fp16 in
 * the workspace first, a sequence at a time: which of them follows from the sizes and max_kv, unless from_pages says that
 * the cache is read as it is (512 tokens of 8192 keys, 32 heads of 128 on 8: 289 us and 2.7e-4 for 107 and 4.7e-4).
 * MI355X_FA_Q_DIRECT=1|0 and MI355X_FA_Q_ROWS=16|32 pin the choices as there, for calls without from_pages. */
typedef struct mi355x_fa_p_args {
    mi355x_kv_step step;
    const void * q_dev;   int64_t q_nb1, q_nb2, q_nb3;         /* token, head, sequence strides */
    mi355x_kv_view k, v;                                       /* nb1 the row, nb2 the head stride; nb3 is not read */
    int64_t n_rows;                                            /* rows of K and of V */
    void * dst_dev;       int64_t dst_nb1, dst_nb2, dst_nb3;   /* head, token, sequence strides */
    int q_type, dst_type;                                      /* 0 F32 or 1 F16 */
    int D, DV, H, HK;
    float scale, softcap;
    int64_t max_kv;
    int from_pages;                                            /* not 0: never decoded first */
} mi355x_fa_p_args;
/* Workspace bytes of mi355x_flash_attn_paged with `nsplit` KV splits (0 = its own choice); 0 for an op that it does not
 * take. It follows the sizes and max_kv, not what lies on the device: partial results where keys are split, and decoded first one
 * sequence's K and V, max_kv keys as fp16, and 128 MiB at most (or 64 bytes a key). 256-byte aligned. */
MI355X_API size_t mi355x_flash_attn_paged_workspace(const mi355x_fa_p_args * a, int nsplit);
/* Concurrent calls must not share a workspace. Equal inputs give equal bits. */
MI355X_API int mi355x_flash_attn_paged(const mi355x_fa_p_args * a, int nsplit, void * workspace_dev, size_t workspace_bytes,
                                       int32_t * err_dev, void * stream);

/* Accepted tokens kept: for i = 0 .. n_keep[s] - 1 in this order, the row of token path[s][i] is copied to the row of token
 * i, bit by bit, in each of `n_out` (1..4) caches (the step's n_past then grows by n_keep). The rows' x is not read.
 * A path is increasing, its numbers below n_new[s]; n_keep NULL: A each. A sequence whose path or numbers are not so, or
 * whose rows are not all in the cache, is left as it is and sets *err_dev. A <= 64. Pages that a step moves
 * rows in belong to one sequence, once. */
MI355X_API int mi355x_kv_keep(const mi355x_kv_step * step, const mi355x_kv_rows * r, int n_out, const int32_t * path_dev,
                              int64_t path_nb, const int32_t * n_keep_dev, int A, int32_t * err_dev, void * stream);

/* ---- MUL_MAT_ID --------------------------------------------------------------------------- */

/* One expert-GEMM op. Strides in ELEMENTS. */
typedef struct mi355x_moe_args {
    int wtype;
    const void * as_dev;      int64_t n_expert, N, K;     /* experts [E][N][K], HBM layout over E*N rows */
    const float * b_dev;      int64_t ne11, b_nb1, b_nb2; /* activations [T][ne11][K]; rows contiguous */
    const int32_t * ids_dev;  int64_t n_used, ids_nb0, ids_nb1;  /* ids[t][s] */
    int64_t n_tokens;
    float * dst_dev;          int64_t dst_nb1, dst_nb2;   /* dst[t][s][:] */
} mi355x_moe_args;

/* Workspace bytes of mi355x_mul_mat_id for this op. */
MI355X_API size_t mi355x_mul_mat_id_workspace(const mi355x_moe_args * a);

/* dst[t][s][:] = as[ids[t][s]] . b[t][s % ne11][:] for every token t and slot s, in one device
 * pipeline with no host synchronisation: the distinct activation rows are packed once, the rows
 * are bucketed by expert on the device, and one grouped launch runs every (expert tile, N block)
 * with the expert's weight dequantized in LDS. An id outside [0, n_expert) leaves its row
 * unwritten and sets *err_dev (a device int32, may be NULL) to 1; the host-buffer path checks ids
 * before calling. K % 32 == 0 and a whole number of blocks, N % 16 == 0; for the layouts
 * regrouped by 32 rows (MI355X_*_X) N % 32 == 0 and N * K <= 2^31 (one expert's weights).
 * Replaces the per-expert loop of ggml-rocket.cpp:6783-6941 and its device calls
 * rocket_matmul_int8_prepacked_gw (6833) / rocket_matmul_fp16_mt (6922). */
MI355X_API int mi355x_mul_mat_id(const mi355x_moe_args * a, void * workspace_dev, size_t workspace_bytes,
                                 int32_t * err_dev, void * stream);

#ifdef __cplusplus
}
#endif

#endif /* MI355X_KERNELS_H */
