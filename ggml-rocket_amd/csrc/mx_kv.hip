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
// two halves of its four Q4_0 bytes, reads 16-byte pieces, and finds the block's maximum with two
// DPP exchanges inside the quad.

#include "mx_common.h"
#include "mx_kernels_impl.h"

namespace mx {

constexpr int KV_THREADS = 256;
constexpr int KV_BLOCKS = KV_THREADS / 4;   // 32-value blocks in flight in a workgroup
constexpr int KV_ROWS_MAX = 8;              // rows a workgroup of set_rows

template <int CTRL>
__device__ __forceinline__ uint32_t quad_dpp(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}
constexpr int QUAD_XOR1 = 0xB1, QUAD_XOR2 = 0x4E;   // quad_perm [1,0,3,2] and [2,3,0,1]

// Of two values the one of larger magnitude; the first where they are equal.
__device__ __forceinline__ float farther(float first, float second) {
    return fabsf(second) > fabsf(first) ? second : first;
}
// The same over a quad, each lane's value before those of the lanes above it.
__device__ __forceinline__ float quad_farther(float x, int l) {
    float y = __uint_as_float(quad_dpp<QUAD_XOR1>(__float_as_uint(x)));
    x = (l & 1) ? farther(y, x) : farther(x, y);
    y = __uint_as_float(quad_dpp<QUAD_XOR2>(__float_as_uint(x)));
    return (l & 2) ? farther(y, x) : farther(x, y);
}

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

// A lane's eight values of a plain block: 4l.. and 16+4l.. of the 32 at element offset `at`.
__device__ __forceinline__ void kv_load_plain(const KvRowsOut & o, int64_t at, int l, float (&v)[8]) {
    if (o.x_f16) {
        const uint16_t * p = (const uint16_t *)o.x + at + 4 * l;
        const half4 lo = *(const half4 *)p, hi = *(const half4 *)(p + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = (float)lo[e];
            v[4 + e] = (float)hi[e];
        }
    } else {
        const float * p = (const float *)o.x + at + 4 * l;
        const float4v lo = *(const float4v *)p, hi = *(const float4v *)(p + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = lo[e];
            v[4 + e] = hi[e];
        }
    }
}
__device__ __forceinline__ void kv_store_plain(const KvRowsOut & o, int64_t at, int l, const float (&v)[8]) {
    if (o.x_f16) {
        uint16_t * p = (uint16_t *)o.x + at + 4 * l;
        *(u32x2 *)p = u32x2{pack2h(v[0], v[1]), pack2h(v[2], v[3])};
        *(u32x2 *)(p + 16) = u32x2{pack2h(v[4], v[5]), pack2h(v[6], v[7])};
    } else {
        float * p = (float *)o.x + at + 4 * l;
        *(float4v *)p = float4v{v[0], v[1], v[2], v[3]};
        *(float4v *)(p + 16) = float4v{v[4], v[5], v[6], v[7]};
    }
}

// One block quantized by its quad and written at element offset `at` of the cache.
__device__ __forceinline__ void kv_quantize(const KvRowsOut & o, int64_t at, int l, const float (&v)[8]) {
    if (o.type == T_F16) {
        uint16_t * p = (uint16_t *)o.q + at + 4 * l;
        *(u32x2 *)p = u32x2{pack2h(v[0], v[1]), pack2h(v[2], v[3])};
        *(u32x2 *)(p + 16) = u32x2{pack2h(v[4], v[5]), pack2h(v[6], v[7])};
        return;
    }
    // the largest magnitude as an integer: its order is that of the floats, infinities and NaN last
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    top = max(top, quad_dpp<QUAD_XOR1>(top));
    top = max(top, quad_dpp<QUAD_XOR2>(top));
    const bool finite = top < 0x7F800000u;
    float d;
    if (o.type == T_Q8_0) {
        d = __uint_as_float(top) / 127.0f;
    } else {
        const float lo = quad_farther(farther(farther(v[0], v[1]), farther(v[2], v[3])), l);
        const float hi = quad_farther(farther(farther(v[4], v[5]), farther(v[6], v[7])), l);
        d = farther(lo, hi) / -8.0f;
    }
    float r = d != 0.0f ? 1.0f / d : 0.0f;
    // a scale too small for its reciprocal is far below fp16's smallest: the block stands for zeros
    if (!finite || !(fabsf(r) < INFINITY)) r = 0.0f;
    uint32_t c[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float y = finite ? mul_rn(v[e], r) : 0.0f;
        c[e] = o.type == T_Q8_0 ? (uint32_t)(int)__builtin_roundf(y) & 0xFFu
                                : (uint32_t)min(15, (int)sub_rn(y, -8.5f));
    }
    if (o.type == T_Q8_0) {
        uint8_t * p = o.q + at + 4 * l;
        *(uint32_t *)p = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
        *(uint32_t *)(p + 16) = c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24);
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) w |= (c[e] | (c[4 + e] << 4)) << (8 * e);
        *(uint32_t *)(o.q + at / 2 + 4 * l) = w;
    }
    if (l == 0) o.d[at / 32] = finite ? f2h_bits(d) : (uint16_t)0x7E00;
}

// A workgroup takes rows_wg consecutive rows of one output. An index that a later row names again
// is dropped, so that the last of them stays whole whichever workgroup is first: every workgroup
// scans the indices behind its rows (n * 8 bytes out of L2, while its first values are on their way).
__global__ void __launch_bounds__(KV_THREADS) set_rows_kernel(KvRowsArgs a) {
    __shared__ int64_t at_row[KV_ROWS_MAX];
    __shared__ int dead[KV_ROWS_MAX];
    const KvRowsOut & o = a.o[kv_out_of(a, blockIdx.x)];
    const int t = threadIdx.x, l = t % 4;
    const int r0 = ((int)blockIdx.x - o.wg_begin) * a.rows_wg, rows = min(a.rows_wg, a.n - r0);
    const int bpr = o.H * o.bph, items = rows * bpr;
    if (t < rows) {
        const int64_t i = kv_index(a, r0 + t);
        const bool ok = i >= 0 && i < o.n_rows;
        at_row[t] = ok ? i : -1;
        dead[t] = !ok;
        if (!ok && a.err) *a.err = 1;
    }
    __syncthreads();
    if (a.idx) {
        for (int j = r0 + 1 + t; j < a.n; j += KV_THREADS) {
            const int64_t i = kv_index(a, j);
            for (int r = 0; r < rows; r++)
                if (j > r0 + r && i == at_row[r]) dead[r] = 1;
        }
        __syncthreads();
    }
    for (int it = t / 4; it < items; it += KV_BLOCKS) {
        const int r = it / bpr, hb = it % bpr, h = hb / o.bph, b = hb % o.bph;
        if (dead[r]) continue;   // the same for the whole quad
        float v[8];
        kv_load_plain(o, (int64_t)(r0 + r) * o.x_nb1 + (int64_t)h * o.x_nb2 + 32 * b, l, v);
        kv_quantize(o, at_row[r] * o.nb1 + (int64_t)h * o.nb2 + 32 * b, l, v);
    }
}

// A quad's share of a quantized block at element offset `at`: the codes times d, exact in f32.
__device__ __forceinline__ void kv_values(int type, const uint8_t * q, float d, int64_t at, int l, float (&v)[8]) {
    if (type == T_Q8_0) {
        const uint32_t lo = *(const uint32_t *)(q + at + 4 * l), hi = *(const uint32_t *)(q + at + 16 + 4 * l);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = mul_rn(d, (float)(int8_t)(lo >> (8 * e)));
            v[4 + e] = mul_rn(d, (float)(int8_t)(hi >> (8 * e)));
        }
    } else {
        const uint32_t w = *(const uint32_t *)(q + at / 2 + 4 * l);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = mul_rn(d, (float)((int)((w >> (8 * e)) & 15u) - 8));
            v[4 + e] = mul_rn(d, (float)((int)((w >> (8 * e + 4)) & 15u) - 8));
        }
    }
}

__global__ void __launch_bounds__(KV_THREADS) get_rows_kernel(KvRowsArgs a) {
    const KvRowsOut & o = a.o[kv_out_of(a, blockIdx.x)];
    const int t = threadIdx.x, l = t % 4;
    const int bpr = o.H * o.bph;
    const int64_t it = (int64_t)((int)blockIdx.x - o.wg_begin) * KV_BLOCKS + t / 4;
    if (it >= (int64_t)a.n * bpr) return;
    const int r = (int)(it / bpr), hb = (int)(it % bpr), h = hb / o.bph, b = hb % o.bph;
    const int64_t i = kv_index(a, r);
    if (i < 0 || i >= o.n_rows) {
        if (a.err) *a.err = 1;
        return;
    }
    const int64_t at = i * o.nb1 + (int64_t)h * o.nb2 + 32 * b;
    float v[8];
    if (o.type == T_F16) {
        const uint16_t * p = (const uint16_t *)o.q + at + 4 * l;
        const half4 lo = *(const half4 *)p, hi = *(const half4 *)(p + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = (float)lo[e];
            v[4 + e] = (float)hi[e];
        }
    } else {
        kv_values(o.type, o.q, h2f_bits(o.d[at / 32]), at, l, v);
    }
    kv_store_plain(o, (int64_t)r * o.x_nb1 + (int64_t)h * o.x_nb2 + 32 * b, l, v);
}

// K and V of one sequence as fp16, for the fused attention. A scale is held to the largest with which
// every value stays inside fp16. The attention hides a key by its score, but multiplies P = 0 by the key's V all the same, so
// V has to be finite: a V block whose scale is not stands for zeros here and makes the first value of
// that key's K a NaN instead, which reaches exactly the queries that see the key.
__global__ void __launch_bounds__(KV_THREADS) kv_decode_kernel(KvDecodeArgs a) {
    const int t = threadIdx.x, l = t % 4;
    const int kb = a.D / 32, vb = a.DV / 32;
    const int64_t it = (int64_t)blockIdx.x * KV_BLOCKS + t / 4;
    const int64_t key_head = it / (kb + vb);
    const int b = (int)(it % (kb + vb));
    if (key_head >= (int64_t)a.KV * a.HK) return;
    const int64_t j = key_head / a.HK, h = key_head % a.HK;
    const bool is_v = b >= kb;
    const KvView & w = is_v ? a.v : a.k;
    const int blk = is_v ? b - kb : b;
    const int64_t at = j * w.nb1 + h * w.nb2 + 32 * blk;
    float d = h2f_bits(w.d[at / 32]);
    const bool bad = !(fabsf(d) < INFINITY);
    if (bad && is_v) d = 0.0f;
    const float lim = kv_scale_limit(w.type);
    d = fmaxf(fminf(d, lim), -lim);
    float v[8];
    kv_values(w.type, w.q, d, at, l, v);
    if (bad && !is_v) v[0] = NAN;
    if (b == 0 && l == 0) {
        const uint16_t * vd = a.v.d + (j * a.v.nb1 + h * a.v.nb2) / 32;
        for (int i = 0; i < vb; i++)
            if (!(fabsf(h2f_bits(vd[i])) < INFINITY)) v[0] = NAN;
    }
    uint16_t * p = (is_v ? a.v16 + (h * a.KV + j) * a.DV : a.k16 + (h * a.KV + j) * a.D) + 32 * blk + 4 * l;
    *(u32x2 *)p = u32x2{pack2h(v[0], v[1]), pack2h(v[2], v[3])};
    *(u32x2 *)(p + 16) = u32x2{pack2h(v[4], v[5]), pack2h(v[6], v[7])};
}

hipError_t launch_kv_decode(const KvDecodeArgs & a, hipStream_t st) {
    const int64_t items = (int64_t)a.KV * a.HK * ((a.D + a.DV) / 32);
    hipLaunchKernelGGL(kv_decode_kernel, dim3((unsigned)((items + KV_BLOCKS - 1) / KV_BLOCKS)), dim3(KV_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_set_rows(KvRowsArgs a, hipStream_t st) {
    // one row a workgroup until the chip is full several times over, then more: fewer index scans
    a.rows_wg = min(KV_ROWS_MAX, max(1, (int)((int64_t)a.n * a.n_out / 2048)));
    int wgs = 0;
    for (int k = 0; k < a.n_out; k++) {
        a.o[k].wg_begin = wgs;
        wgs += (a.n + a.rows_wg - 1) / a.rows_wg;
    }
    hipLaunchKernelGGL(set_rows_kernel, dim3(wgs), dim3(KV_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_get_rows(KvRowsArgs a, hipStream_t st) {
    int wgs = 0;
    for (int k = 0; k < a.n_out; k++) {
        a.o[k].wg_begin = wgs;
        wgs += (int)(((int64_t)a.n * a.o[k].H * a.o[k].bph + KV_BLOCKS - 1) / KV_BLOCKS);
    }
    hipLaunchKernelGGL(get_rows_kernel, dim3(wgs), dim3(KV_THREADS), 0, st, a);
    return hipGetLastError();
}

}  // namespace mx
