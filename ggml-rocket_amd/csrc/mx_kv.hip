// SPDX-License-Identifier: MIT
// SET_ROWS and GET_ROWS of a KV cache held as Q8_0, Q4_0 or F16 (the planes of mi355x_kv_rows).
//
// Per block of 32 values x_j (f32 arithmetic, every step rounded on its own, as ggml's reference
// quantizers):
//   Q8_0  d = max|x| / 127,            code_j = round_half_away(x_j * (1 / d)),        x_j ~ d * code_j
//   Q4_0  d = x_p / -8, p = argmax|x|, code_j = min(15, trunc(x_j * (1 / d) + 8.5)),   x_j ~ d * (code_j - 8)
// with d stored as fp16. Reading back multiplies the stored d by the code: exact in f32 (11 + 8 bits).
//
// Both are streams: bound by HBM for many rows and by a launch's latency for few. A block of 32 is
// the work of four lanes, a quad: lane l takes values 4l..4l+3 and 16+4l..16+4l+3, so it holds the
// two halves of its four Q4_0 bytes, reads pieces of 16 bytes (F32) or 8 (F16), and finds the block's maximum with
// two DPP exchanges inside the quad. Reading back, lane l takes values 8l..8l+7, one 16-byte store of fp16
// (its Q4_0 nibbles are the low or the high ones of eight bytes that two lanes read).

#include "mx_common.h"
#include "mx_fa_prep.h"
#include "mx_kernels_impl.h"
#include "mx_kv_rows.h"

namespace mx {

constexpr int KV_THREADS = 256;
constexpr int KV_BLOCKS = KV_THREADS / 4;   // 32-value blocks in flight in a workgroup
constexpr int KV_ROWS_MAX = 8;              // rows a workgroup of set_rows
constexpr int KV_ROWS_LAUNCH = 16384;       // and a launch of it
constexpr int KV_BLOCKS_LAUNCH = 1 << 24;   // blocks a launch of get_rows

__device__ __forceinline__ int64_t kv_index(const KvRowsArgs & a, int i) {
    if (!a.idx) return i;
    return a.idx64 ? ((const int64_t *)a.idx)[i] : (int64_t)((const int32_t *)a.idx)[i];
}

// The output whose workgroups hold `wg`.
__device__ __forceinline__ int kv_out_of(const KvRowsArgs & a, int wg) {
    int k = 0;
    while (k + 1 < a.n_out && wg >= a.o[k + 1].wg_begin) k++;
    return k;
}

// A workgroup takes rows_wg consecutive rows of output blockIdx.y. An index that a later row names again is
// dropped, so that the last of them stays whole whichever workgroup is first: every workgroup scans the
// indices behind its rows (8 n bytes at most out of L2, four of them in flight a thread) while its first
// block is on its way, against 4096 bits in LDS that its own indices set; only a hit is compared in full.
// (4091 rows of 2 x 1024: 15.8 us with every index compared with every row of the workgroup.)
__global__ void __launch_bounds__(KV_THREADS) set_rows_kernel(KvRowsArgs a) {
    __shared__ int64_t at_row[KV_ROWS_MAX];
    __shared__ int dead[KV_ROWS_MAX];
    __shared__ uint32_t named[128];
    const KvRowsOut & o = a.o[blockIdx.y];
    const int t = threadIdx.x, l = t % 4;
    const int r0 = (int)blockIdx.x * a.rows_wg, rows = min(a.rows_wg, a.n - r0);
    const int bpr = o.div_bpr.d, items = rows * bpr;
    auto load = [&](int it, float (&v)[8]) {
        const int r = fq_div(it, o.div_bpr), hb = it - r * bpr, h = fq_div(hb, o.div_bph), b = hb - h * o.bph;
        kv_load_plain(o, (int64_t)(r0 + r) * o.x_nb1 + (int64_t)h * o.x_nb2 + 32 * b, l, v);
    };
    float v[8];
    if (t / 4 < items) load(t / 4, v);
    if (t < 128) named[t] = 0;
    __syncthreads();
    if (t < rows) {
        const int64_t i = kv_index(a, r0 + t);
        const bool ok = i >= 0 && i < o.n_rows;
        at_row[t] = ok ? i : -1;
        dead[t] = !ok;
        if (!ok && a.err) *a.err = 1;
        if (ok) atomicOr(&named[(i & 4095) / 32], 1u << (i % 32));
    }
    __syncthreads();
    if (a.idx && a.n > r0 + 1) {
        for (int j0 = r0 + 1 + t; j0 < a.n; j0 += 4 * KV_THREADS) {
            int64_t i[4];
#pragma unroll
            for (int u = 0; u < 4; u++) i[u] = j0 + u * KV_THREADS < a.n ? kv_index(a, j0 + u * KV_THREADS) : -1;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i[u] >= 0 && (named[(i[u] & 4095) / 32] >> (i[u] % 32)) & 1u)
                    for (int r = 0; r < rows; r++)
                        if (i[u] == at_row[r] && j0 + u * KV_THREADS > r0 + r) dead[r] = 1;
        }
        __syncthreads();
    }
    for (int it = t / 4; it < items; it += KV_BLOCKS) {
        float w[8];
        if (it + KV_BLOCKS < items) load(it + KV_BLOCKS, w);
        const int r = fq_div(it, o.div_bpr), hb = it - r * bpr, h = fq_div(hb, o.div_bph), b = hb - h * o.bph;
        if (!dead[r]) kv_quantize(o, at_row[r] * o.nb1 + (int64_t)h * o.nb2 + 32 * b, l, v);   // the same for the quad
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = w[e];
    }
}

// A quad reads ILP blocks, KV_BLOCKS apart, all of them requested before the first is stored.
template <int ILP>
__global__ void __launch_bounds__(KV_THREADS) get_rows_kernel(KvRowsArgs a) {
    const KvRowsOut & o = a.o[kv_out_of(a, blockIdx.x)];
    const int t = threadIdx.x, l = t % 4;
    const int i0 = ((int)blockIdx.x - o.wg_begin) * (KV_BLOCKS * ILP) + t / 4, all = a.n * o.div_bpr.d;
    u32x4 x[ILP];
    uint16_t d[ILP];
    int64_t to[ILP];
    bool ok[ILP];
#pragma unroll
    for (int u = 0; u < ILP; u++) {
        const int it = i0 + u * KV_BLOCKS, rl = fq_div(min(it, all - 1), o.div_bpr), hb = min(it, all - 1) - rl * o.div_bpr.d;
        const int h = fq_div(hb, o.div_bph), b = hb - h * o.bph, r = a.first + rl;
        const int64_t i = kv_index(a, r);
        const bool in = i >= 0 && i < o.n_rows;
        if (!in && a.err) *a.err = 1;
        ok[u] = in && it < all;
        to[u] = (int64_t)r * o.x_nb1 + (int64_t)h * o.x_nb2 + 32 * b;
        const int64_t at = (in ? i : 0) * o.nb1 + (int64_t)h * o.nb2 + 32 * b;
        x[u] = u32x4{0, 0, 0, 0};
        d[u] = 0;
        if (ok[u]) {
            x[u] = kv_codes(o.type, o.q, at, l);
            if (o.type != T_F16) d[u] = o.d[at / 32];
        }
    }
#pragma unroll
    for (int u = 0; u < ILP; u++) {
        float v[8];
        kv_values(o.type, x[u], h2f_bits(d[u]), l, v);
        if (!ok[u]) continue;
        if (o.x_f16) {
            *(u32x4 *)((uint16_t *)o.x + to[u] + 8 * l) = kv_pack8(v);
        } else {
            float4v * p = (float4v *)((float *)o.x + to[u] + 8 * l);
            p[0] = float4v{v[0], v[1], v[2], v[3]};
            p[1] = float4v{v[4], v[5], v[6], v[7]};
        }
    }
}

// K and V of one sequence as fp16, for the fused attention: each value rounded once, by at most 2^-11 of itself (2^-25
// below 2^-14), since its products take fp16 operands and no F32 ones at their rate. A scale is held to the largest with which
// every value stays inside fp16. The attention hides a key by its score, but multiplies P = 0 by the
// key's V all the same, so V has to be finite: a V block whose scale is not stands for zeros here and
// makes the first value of that key's K a NaN instead, which reaches exactly the queries that see the key.
// The mask classes that the attention needs as well come from the same launch (a launch of their own 4.6 us).
// 2048 keys of 8 heads x 128 + 128 in Q8_0 5.5 us (13 MB), 8192 in Q4_0 16 us (43 MB, 2.7 TB/s; two and four
// blocks a quad 16 and 18 us, and stores past the caches 14 us but 3 us more in the attention).
__global__ void __launch_bounds__(KV_THREADS) kv_decode_kernel(KvDecodeArgs a, FaArgs f) {
    if ((int)blockIdx.x < a.n_prep) return fa_prep_block(f, blockIdx.x);
    const int t = threadIdx.x, l = t % 4;
    const int kb = a.D / 32, vb = a.DV / 32;
    // a key and head's blocks follow each other, K then V
    const int it = ((int)blockIdx.x - a.n_prep) * KV_BLOCKS + t / 4, kh = fq_div(it, a.div_blocks), b = it - kh * (kb + vb);
    const int j = fq_div(kh, a.div_hk), h = kh - j * a.HK;
    if (kh >= a.KV * a.HK) return;
    const bool is_v = b >= kb;
    const KvView & w = is_v ? a.v : a.k;
    const int blk = is_v ? b - kb : b;
    const int64_t at = j * w.nb1 + h * w.nb2 + 32 * blk;
    const u32x4 x = kv_codes(w.type, w.q, at, l);
    const uint16_t d = w.d[at / 32];
    const bool bad = (d & 0x7C00u) == 0x7C00u;
    bool poison = bad && !is_v;
    if (!is_v)   // a K block's quad looks at the V blocks blk, blk + kb, ...
        for (int i = blk; i < vb; i += kb) poison |= (a.v.d[(j * a.v.nb1 + h * a.v.nb2) / 32 + i] & 0x7C00u) == 0x7C00u;
    const float lim = kv_scale_limit(w.type), df = bad ? 0.0f : fmaxf(fminf(h2f_bits(d), lim), -lim);
    float v[8];
    kv_values(w.type, x, df, l, v);
    if (poison) v[0] = NAN;
    *(u32x4 *)((is_v ? a.v16 + (h * (int64_t)a.KV + j) * a.DV : a.k16 + (h * (int64_t)a.KV + j) * a.D) + 32 * blk + 8 * l) = kv_pack8(v);
}

hipError_t launch_kv_decode(const KvDecodeArgs & args, const FaArgs & f, hipStream_t st) {
    KvDecodeArgs a = args;
    a.div_blocks = fq_div_by((a.D + a.DV) / 32);
    a.div_hk = fq_div_by(a.HK);
    a.n_prep = fa_prep_blocks(f);
    const int64_t items = (int64_t)a.KV * a.HK * ((a.D + a.DV) / 32);
    hipLaunchKernelGGL(kv_decode_kernel, dim3((unsigned)(a.n_prep + (items + KV_BLOCKS - 1) / KV_BLOCKS)), dim3(KV_THREADS), 0, st, a, f);
    return hipGetLastError();
}

static void kv_divs(KvRowsArgs & a) {
    for (int k = 0; k < a.n_out; k++) {
        a.o[k].div_bpr = fq_div_by(a.o[k].H * a.o[k].bph);
        a.o[k].div_bph = fq_div_by(a.o[k].bph);
    }
}

// A launch takes KV_ROWS_LAUNCH rows at most, the next ones a next launch: the scans of later indices grow with the
// square of a launch's rows (8192 rows of 2 x 1024 without indices 18 us, with 24; 16384 29 and 50), and a
// repeated index in a later launch comes later by itself.
hipError_t launch_set_rows(KvRowsArgs a, hipStream_t st) {
    kv_divs(a);
    const int all = a.n;
    for (int r0 = 0; r0 < all; r0 += KV_ROWS_LAUNCH) {
        a.n = min(KV_ROWS_LAUNCH, all - r0);
        // one row a workgroup until the chip is full a few times over, then more: fewer index scans
        a.rows_wg = min(KV_ROWS_MAX, max(1, a.n / 512));
        hipLaunchKernelGGL(set_rows_kernel, dim3((a.n + a.rows_wg - 1) / a.rows_wg, a.n_out), dim3(KV_THREADS), 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (a.idx) a.idx = (const uint8_t *)a.idx + (int64_t)KV_ROWS_LAUNCH * (a.idx64 ? 8 : 4);
        for (int k = 0; k < a.n_out; k++) {
            KvRowsOut & o = a.o[k];
            o.x = (uint8_t *)o.x + KV_ROWS_LAUNCH * o.x_nb1 * (o.x_f16 ? 2 : 4);
            if (a.idx) continue;   // else row i is cache row i
            const int64_t e0 = KV_ROWS_LAUNCH * o.nb1;
            o.q += o.type == T_F16 ? 2 * e0 : o.type == T_Q4_0 ? e0 / 2 : e0;
            if (o.d) o.d += e0 / 32;
            o.n_rows -= KV_ROWS_LAUNCH;
        }
    }
    return hipSuccess;
}

template <int ILP>
static hipError_t get_rows_launch(KvRowsArgs a, hipStream_t st) {
    int wgs = 0;
    for (int k = 0; k < a.n_out; k++) {
        a.o[k].wg_begin = wgs;
        wgs += (int)(((int64_t)a.n * a.o[k].div_bpr.d + KV_BLOCKS * ILP - 1) / (KV_BLOCKS * ILP));
    }
    hipLaunchKernelGGL(get_rows_kernel<ILP>, dim3(wgs), dim3(KV_THREADS), 0, st, a);
    return hipGetLastError();
}

// Four blocks a quad where every output is F16 and there are 2^19 blocks at least, else one: more of them at once.
// (us with one and four, two caches of 8 x 128 in Q8_0: 512 rows as F16 3.2 / 5.2, as F32 3.8 / 5.6; 4096 8.1 / 8.8 and
// 11.9 / 13.1; 8192 12.2 / 11.7 and 18.9 / 19.3; 16384 27.8 / 26.6 and 41.4 / 42.5; 32768 47.4 / 46.1 and 73 / 82.)
// A launch takes KV_BLOCKS_LAUNCH blocks at most (or one row), so that its threads stay far from 2^32.
hipError_t launch_get_rows(KvRowsArgs a, hipStream_t st) {
    kv_divs(a);
    int bpr = 0;
    bool f16 = true;
    for (int k = 0; k < a.n_out; k++) {
        bpr += a.o[k].div_bpr.d;
        f16 = f16 && a.o[k].x_f16;
    }
    const int all = a.n, most = max(1, KV_BLOCKS_LAUNCH / bpr);
    for (a.first = 0; a.first < all; a.first += a.n) {
        a.n = min(most, all - a.first);
        const hipError_t e = f16 && (int64_t)a.n * bpr >= 1 << 19 ? get_rows_launch<4>(a, st) : get_rows_launch<1>(a, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace mx
