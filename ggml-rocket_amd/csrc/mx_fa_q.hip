// SPDX-License-Identifier: MIT
// FLASH_ATTN_EXT over a quantized cache: the launch that merges KV splits, and the dispatch by type.
#include "mx_fa_q.h"

namespace mx {

// Merges the splits of one O^T tile of one unit of rows: O = sum_s exp(m_s - M) O_s / sum_s exp(m_s - M) l_s.
// Every partial of the tile is requested at once, split i by wave i % 4, and the splits' weights are
// formed while they come: one memory round trip. Rows whose maxima are all -inf have sums of zero (or
// NaN, kept).
constexpr int FQ_MAX_SPLIT = 64;
__global__ void __launch_bounds__(256) fa_q_combine_kernel(FaQArgs a, int DV, int NQ) {
    __shared__ float sm[16][17], sl[16][17], sw[FQ_MAX_SPLIT][16];
    __shared__ float4v so[4][WAVE];
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE, r = lane % 16, g = lane / 16;
    const int TT = DV / 16, all = TT * NQ;
    const int at = blockIdx.x % all, n = at / TT, q = at % TT;
    const int unit = blockIdx.x / all;
    const int sh = fq_div(unit, a.div_nrt), s = fq_div(sh, a.div_hk), rt = unit - sh * a.nrt, hk = sh - s * a.HK;
    const float * po = a.part_o + (((int64_t)unit * a.nsplit * all + at) * WAVE + lane) * 4;
    float4v p[FQ_MAX_SPLIT / 4];
#pragma unroll
    for (int k = 0; k < FQ_MAX_SPLIT / 4; k++) {
        p[k] = float4v{0, 0, 0, 0};
        if (4 * k + wave < a.nsplit) p[k] = *(const float4v *)(po + (int64_t)(4 * k + wave) * all * WAVE * 4);
    }
    // thread (row t % 16, splits t / 16 + 16 k)
    const int row16 = t % 16, s0 = t / 16;
    const float * ml = a.part_ml + ((int64_t)unit * a.nsplit * NQ * 16 + n * 16 + row16) * 2;
    float m[FQ_MAX_SPLIT / 16], l[FQ_MAX_SPLIT / 16], M = -INFINITY;
#pragma unroll
    for (int k = 0; k < FQ_MAX_SPLIT / 16; k++) {
        m[k] = -INFINITY;
        l[k] = 0.0f;
        if (s0 + 16 * k < a.nsplit) {
            m[k] = ml[(int64_t)(s0 + 16 * k) * NQ * 32];
            l[k] = ml[(int64_t)(s0 + 16 * k) * NQ * 32 + 1];
        }
        M = fmaxf(M, m[k]);
    }
    sm[s0][row16] = M;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) M = fmaxf(M, sm[i][row16]);
    float L = 0.0f;
#pragma unroll
    for (int k = 0; k < FQ_MAX_SPLIT / 16; k++) {
        const float w = m[k] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m[k] - M) * FQ_LOG2E);
        L += w * l[k];
        if (s0 + 16 * k < FQ_MAX_SPLIT) sw[s0 + 16 * k][row16] = w;
    }
    sl[s0][row16] = L;
    __syncthreads();
    float4v v = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < FQ_MAX_SPLIT / 4; k++) {
        const float w = sw[4 * k + wave][r];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += w * p[k][e];
    }
    so[wave][lane] = v;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; w++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += so[w][lane][e];
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) L += sl[i][r];
    const int row = (rt * NQ + n) * 16 + r;
    if (row >= a.R) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const int tk = fq_div(row, a.div_g);
    const int64_t dst = (int64_t)s * a.dst_nb3 + (int64_t)tk * a.dst_nb2 + (int64_t)(hk * a.G + row - tk * a.G) * a.dst_nb1;
    fq_store4(a, dst, 16 * q + 4 * g, v, inv);
}

hipError_t launch_fa_q_combine(const FaQArgs & a, int DV, int NQ, hipStream_t st) {
    const int64_t units = (int64_t)a.S * a.HK * a.nrt;
    hipLaunchKernelGGL(fa_q_combine_kernel, dim3((unsigned)(units * (DV / 16) * NQ)), dim3(256), 0, st, a, DV, NQ);
    return hipGetLastError();
}

hipError_t launch_fa_q(const FaQArgs & a, hipStream_t st) {
    if (a.k.type == T_Q8_0) return a.v.type == T_Q8_0 ? launch_fa_q_Q8_0_Q8_0(a, st) : launch_fa_q_Q8_0_Q4_0(a, st);
    return a.v.type == T_Q8_0 ? launch_fa_q_Q4_0_Q8_0(a, st) : launch_fa_q_Q4_0_Q4_0(a, st);
}

hipError_t launch_fa_p(const FaPArgs & a, hipStream_t st) {
    if (a.k.type == T_F16) return launch_fa_p_F16(a, st);
    if (a.k.type == T_Q8_0) return a.v.type == T_Q8_0 ? launch_fa_p_Q8_0_Q8_0(a, st) : launch_fa_p_Q8_0_Q4_0(a, st);
    return a.v.type == T_Q8_0 ? launch_fa_p_Q4_0_Q8_0(a, st) : launch_fa_p_Q4_0_Q4_0(a, st);
}

}  // namespace mx
