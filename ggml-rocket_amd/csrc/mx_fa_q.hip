// SPDX-License-Identifier: MIT
// FLASH_ATTN_EXT over a quantized cache: the launch that merges KV splits, and the dispatch by type.
#include "mx_fa_q.h"

namespace mx {

// Merges the splits of one O^T tile of one unit of rows: O = sum_s exp(m_s - M) O_s / sum_s exp(m_s - M) l_s.
// Four waves take the splits in turn. Rows whose maxima are all -inf have sums of zero (or NaN, kept).
__global__ void __launch_bounds__(256) fa_q_combine_kernel(FaQArgs a, int vt, int DV, int NQ) {
    __shared__ float4v so[4][WAVE];
    __shared__ float sl[4][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, r = lane % 16, g = lane / 16;
    const int TT = DV / 16, all = TT * NQ;
    const int at = blockIdx.x % all, n = at / TT, q = at % TT;
    const int64_t unit = blockIdx.x / all;
    const int rt = (int)(unit % a.nrt), hk = (int)(unit / a.nrt % a.HK), s = (int)(unit / a.nrt / a.HK);
    const float * ml = a.part_ml + (unit * a.nsplit * NQ * 16 + n * 16 + r) * 2;
    const float * po = a.part_o + ((unit * a.nsplit * all + at) * WAVE + lane) * 4;
    const int64_t ml_st = NQ * 32, po_st = (int64_t)all * WAVE * 4;
    float M = -INFINITY;
    for (int i = 0; i < a.nsplit; i++) M = fmaxf(M, ml[i * ml_st]);
    float4v v = {0, 0, 0, 0};
    float L = 0.0f;
    for (int i = wave; i < a.nsplit; i += 4) {
        const float m = ml[i * ml_st], w = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - M) * FQ_LOG2E);
        const float4v p = *(const float4v *)(po + i * po_st);
        L += w * ml[i * ml_st + 1];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += w * p[e];
    }
    so[wave][lane] = v;
    sl[wave][lane] = L;
    __syncthreads();
    if (wave) return;
    for (int w = 1; w < 4; w++) {
        L += sl[w][lane];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += so[w][lane][e];
    }
    const int row = (rt * NQ + n) * 16 + r;
    if (row >= a.R) return;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const int64_t dst = (int64_t)s * a.dst_nb3 + (int64_t)(row / a.G) * a.dst_nb2 + (int64_t)(hk * a.G + row % a.G) * a.dst_nb1;
    const int vu = vt == T_Q8_0 || DV >= 128 ? 4 : 2;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int d = fq_dim(vt, vu, q, g, e);
        if (d < a.dv) {
            if (a.dst_f16) ((uint16_t *)a.dst)[dst + d] = f2h_bits(v[e] * inv);
            else ((float *)a.dst)[dst + d] = v[e] * inv;
        }
    }
}

hipError_t launch_fa_q_combine(const FaQArgs & a, int vt, int DV, int NQ, hipStream_t st) {
    const int64_t units = (int64_t)a.S * a.HK * a.nrt;
    hipLaunchKernelGGL(fa_q_combine_kernel, dim3((unsigned)(units * (DV / 16) * NQ)), dim3(256), 0, st, a, vt, DV, NQ);
    return hipGetLastError();
}

hipError_t launch_fa_q(const FaQArgs & a, hipStream_t st) {
    if (a.k.type == T_Q8_0) return a.v.type == T_Q8_0 ? launch_fa_q_Q8_0_Q8_0(a, st) : launch_fa_q_Q8_0_Q4_0(a, st);
    return a.v.type == T_Q8_0 ? launch_fa_q_Q4_0_Q8_0(a, st) : launch_fa_q_Q4_0_Q4_0(a, st);
}

}  // namespace mx
