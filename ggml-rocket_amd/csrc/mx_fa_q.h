// SPDX-License-Identifier: MIT
// FLASH_ATTN_EXT of few query rows over a quantized cache (Q8_0 / Q4_0 K and V), for gfx950: single
// tokens, drafts and short prompts. The cache is read once, as it is stored.
//
//   O[t,h,:] = softmax_j( cap(scale * q[h,t].k[hk,j]) + mask[t,j] ) . v[hk,j,:],  hk = h / G, G = H / HK
//
// The T * G query rows of one KV head share its keys, so they are the columns of the products: a wave
// takes 16 NQ rows and 32 keys at a time, in 16x16x32 MFMAs,
//   S^T = K . Q^T   (A: 16 keys x 32 dims, B: 32 dims x 16 rows)
//   O^T += V^T . P^T (A: 16 dims x 32 keys, B: 32 keys x 16 rows)
// with scores, softmax statistics and O in F32 and everything of a row in the four lanes of its
// column. A wave is on its own until its keys are done: no LDS tiles and no barriers, each 32-key
// tile's codes come straight into registers. The order of dims in a contraction and
// of keys in a tile is free, and chosen so that no lane needs another's data:
//   K   a lane holds one key and whole 16-byte pieces of its row; Q is laid out to match.
//   P   the S^T accumulators of two 16-key products are the P^T operand: slot e of lane group g is key
//       16 (e / 4) + 4 g + e % 4.
//   V   the lane of group g loads the same few bytes of those eight keys; v_perm_b32 picks one byte of
//       two keys into a pair of halves, which transposes V on the way to fp16.
// Codes become fp16 by integer operations: a byte under the exponent of 1024 is 1024 + byte, less the
// offset (exact), times the block's scale: the values of the cache rounded once. V's scales go through
// a few bytes of LDS a wave, which turns a key's row of scales into eight keys' scales of one block.
// The running maximum moves only when a score passes it by more than 8 in the exponent of 2 (P stays
// below 256, well inside fp16), so most tiles exchange nothing between lanes.
//
// A tile's K is loaded again, for the next tile, as soon as its scores are done, its V after O: the loads
// of one half of a tile are always in flight under the other half's work, and the registers hold one
// tile, so that several waves share a SIMD.
// The waves of a block take alternate tiles of the block's key range and merge through LDS at the end;
// the key range is split over blocks where there are too few of them, and a second launch merges those.
// Tiles that the mask hides from every row of a wave are not read: their mask is looked at before their
// loads are issued, and hidden tiles' loads are sent to the tile before (the number of loads in flight
// stays the same, which keeps the waits exact).

#pragma once

#include <type_traits>

#include "mx_common.h"
#include "mx_kernels_impl.h"
#include "mx_weights.h"

namespace mx {

constexpr int FQ_KEYS = 32;      // keys a tile
constexpr float FQ_LAZY = 8.0f / 1.4426950408889634f;
constexpr float FQ_LOG2E = 1.4426950408889634f;

// KT, VT: T_Q8_0 or T_Q4_0; DK, DV: the built head dims; NQ: 16-row query tiles a wave.
template <int KT, int VT, int DK, int DV, int NQ>
struct FqCfg {
    static constexpr int KRB = KT == T_Q8_0 ? DK : DK / 2, VRB = VT == T_Q8_0 ? DV : DV / 2;   // bytes a row
    static constexpr int CB = (KRB / 16) % 4 == 0 ? 16 : 8;   // a lane's piece of a key: the four lanes of
    static constexpr int KI = KRB / CB / 4;                   // a key take pieces g, g + 4, ...; KI each
    static constexpr int KS = DK / 32;                        // Q.K products
    static constexpr int SPP = KS / KI;                       // of them, per piece
    static constexpr int VU = VT == T_Q8_0 || DV >= 128 ? 4 : 2;   // a lane's bytes of a V row: u, u + 16, ...
    static constexpr int VJ = VRB / (16 * VU);
    static constexpr int VH = VT == T_Q4_0 ? 2 : 1;           // nibbles a byte
    static constexpr int TT = DV / 16;                        // O^T tiles, index (j * VU + byte) * VH + nibble
    static_assert(KRB % (4 * CB) == 0 && VJ * VU * VH == TT && SPP * KI == KS, "layout");
    static constexpr int VB = DV / 32, VS = DV / 64;          // V scales a key, and a lane (32 keys, two lanes each)
    // registers: a tile of codes, O, Q, scores and masks, the rest
    static constexpr int REGS = 2 * KI * (CB / 4) + 8 * VJ + (TT + KS) * 4 * NQ + 22 * NQ + 50;
    static constexpr int NW = REGS > 240 ? 4 : 8;             // waves a block
    static constexpr int CT = TT * NQ < 8 ? TT * NQ : 8;      // O^T tiles merged at a time
    static constexpr int SCALE_LDS = VB * FQ_KEYS * 2;        // a wave's V scales
    static constexpr int MERGE_LDS = NW * 16 * NQ * 8 + NW * CT * 1024;
    static constexpr int LDS = MERGE_LDS > NW * SCALE_LDS ? MERGE_LDS : NW * SCALE_LDS;
};

typedef uint32_t u32_alias __attribute__((may_alias));

// The element a lane's value i of O^T tile t is: its dim.
__device__ __forceinline__ int fq_dim(int vt, int vu, int t, int g, int i) {
    if (vt == T_Q8_0) return 64 * (t / 4) + 16 * g + 4 * i + t % 4;
    const int hi = t % 2, n = (t / 2) % vu, j = t / 2 / vu;
    return vu == 4 ? 32 * (g + 4 * j) + 4 * i + n + 16 * hi : 32 * (g / 2) + 8 * (g % 2) + 2 * i + n + 16 * hi;
}

// Maximum and sum over the four lanes of a column (l, l ^ 16, l ^ 32, l ^ 48), the same in each of them:
// v_permlane16_swap and v_permlane32_swap of a register with itself give every lane its pair's two
// values, without LDS.
__device__ __forceinline__ float fq_col_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float fq_col_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// n / d of a FqDiv made for d: the product is the quotient or one more.
__device__ __forceinline__ int fq_div(int n, const FqDiv & d) {
    const uint32_t q = __umulhi((uint32_t)n, d.mul);
    return d.d == 1 ? n : (int)(q * (uint32_t)d.d > (uint32_t)n ? q - 1 : q);
}

// A block's scale as the products take it: held to the largest with which every value stays inside
// fp16 (kv_scale_limit); infinite or NaN ones as `bad`.
template <int TYPE>
__device__ __forceinline__ uint16_t fq_scale(uint16_t bits, uint16_t bad) {
    constexpr uint16_t lim = TYPE == T_Q8_0 ? 0x6007 : 0x6FFF;
    const uint16_t mag = bits & 0x7FFFu;
    const uint16_t held = (uint16_t)(min(mag, lim) | (bits & 0x8000u));
    return mag >= 0x7C00u ? bad : held;
}

// Eight values of a key from its codes: a dword pair (Q8_0) or a dword (Q4_0: four low nibbles, four
// high ones), times d.
template <int KT>
__device__ __forceinline__ half8 fq_key(uint32_t x0, uint32_t x1, half2v d) {
    half2v p[4];
    if constexpr (KT == T_Q8_0) {
        const uint32_t a = x0 ^ 0x80808080u, b = x1 ^ 0x80808080u;
        const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        p[0] = (magic_pair(a, PERM_B01) + off) * d;
        p[1] = (magic_pair(a, PERM_B23) + off) * d;
        p[2] = (magic_pair(b, PERM_B01) + off) * d;
        p[3] = (magic_pair(b, PERM_B23) + off) * d;
    } else {
        const uint32_t a = x0 & 0x0F0F0F0Fu, b = (x0 >> 4) & 0x0F0F0F0Fu;
        const half2v off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        p[0] = (magic_pair(a, PERM_B01) + off) * d;
        p[1] = (magic_pair(a, PERM_B23) + off) * d;
        p[2] = (magic_pair(b, PERM_B01) + off) * d;
        p[3] = (magic_pair(b, PERM_B23) + off) * d;
    }
    half8 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r[2 * i] = p[i][0];
        r[2 * i + 1] = p[i][1];
    }
    return r;
}

template <int KT, int VT, int DK, int DV, int NQ>
__global__ void __launch_bounds__((FqCfg<KT, VT, DK, DV, NQ>::NW * WAVE))
fa_q_kernel(FaQArgs a) {
    using C = FqCfg<KT, VT, DK, DV, NQ>;
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int NW = C::NW;
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, g = lane / 16;

    // block -> (sequence, split, KV head, query rows): an XCD's run of blocks shares keys, and the KV
    // heads of a token lie side by side in a token-major cache
    int b = xcd_tile(blockIdx.x, gridDim.x), b1 = fq_div(b, a.div_nrt);
    const int rt = b - b1 * a.nrt;
    b = b1;
    b1 = fq_div(b, a.div_hk);
    const int hk = b - b1 * a.HK, s = fq_div(b1, a.div_split), split = b1 - s * a.nsplit;
    const int ntiles = (a.KV + FQ_KEYS - 1) / FQ_KEYS, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int tile0 = split * per, tile1 = min(ntiles, tile0 + per);

    // Tile t starts at key kb(t) = min(32 t, KV - 32), KV >= 32: a last partial tile is moved back and
    // its keys before 32 t, which the tile before has, do not count. So every load stays inside the
    // cache without a bound per lane: a scalar base and the lane's fixed 32-bit offset.
    const int kb_last = a.KV - FQ_KEYS;
    constexpr int KSH = KT == T_Q4_0, VSH = VT == T_Q4_0;   // elements to bytes
    const uint8_t * const kq = a.k.q + (((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) >> KSH);
    const uint8_t * const vq = a.v.q + (((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) >> VSH);
    const uint16_t * const kd = a.k.d + ((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) / 32;
    const uint16_t * const vd = a.v.d + ((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) / 32;
    const uint32_t knb = (uint32_t)a.k.nb1, vnb = (uint32_t)a.v.nb1;
    uint32_t ko[C::KI], kdo[C::KI];  // pieces of key r and their scales (a piece past dk: piece 0, Q is zero there)
#pragma unroll
    for (int i = 0; i < C::KI; i++) {
        int c = g + 4 * i;
        const int elems = KT == T_Q8_0 ? C::CB : 2 * C::CB;
        if (c * elems >= a.dk) c = 0;
        ko[i] = ((r * knb) >> KSH) + (uint32_t)(c * C::CB);
        kdo[i] = r * knb / 32 * 2 + (uint32_t)(c * elems / 32 * 2);
    }
    uint32_t vo[C::VJ];              // the lane's bytes of key 4 g's row of V
    int vblk[C::VJ];
#pragma unroll
    for (int j = 0; j < C::VJ; j++) {
        const int u = (r + 16 * j) * C::VU;                      // byte in the row
        vblk[j] = VT == T_Q8_0 ? u / 32 : u / 16;
        vo[j] = ((4 * g * vnb) >> VSH) + (32 * vblk[j] < a.dv ? (uint32_t)u : 0u);   // past dv: not stored
    }
    uint32_t vdo[C::VS];             // the V scales this lane fetches: key lane % 32
#pragma unroll
    for (int i = 0; i < C::VS; i++) {
        int blk = (lane / 32) * C::VS + i;
        if (32 * blk >= a.dv) blk = 0;
        vdo[i] = (uint32_t)(lane % 32) * vnb / 32 * 2 + 2 * blk;
    }

    uint32_t xk[2][C::KI][C::CB / 4], xv[8][C::VJ];   // the tile's codes
    uint16_t xkd[2][C::KI], xvd[C::VS];               // and scales
    auto load_k = [&](int t) {   // and V's scales, which are looked at with K's
        const int64_t kb = min(FQ_KEYS * t, kb_last);
        const uint8_t * vdt = (const uint8_t *)vd + kb * a.v.nb1 / 32 * 2;
#pragma unroll
        for (int i = 0; i < C::VS; i++) xvd[i] = *(const uint16_t *)(vdt + vdo[i]);
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int64_t at = (kb + 16 * hf) * a.k.nb1;
            const uint8_t * q = kq + (at >> KSH);
            const uint8_t * d = (const uint8_t *)kd + at / 32 * 2;
#pragma unroll
            for (int i = 0; i < C::KI; i++) {
                xkd[hf][i] = *(const uint16_t *)(d + kdo[i]);
                if constexpr (C::CB == 16) {
                    const u32x4 w = *(const u32x4 *)(q + ko[i]);
#pragma unroll
                    for (int e = 0; e < 4; e++) xk[hf][i][e] = w[e];
                } else {
                    const u32x2 w = *(const u32x2 *)(q + ko[i]);
#pragma unroll
                    for (int e = 0; e < 2; e++) xk[hf][i][e] = w[e];
                }
            }
        }
    };
    auto load_v = [&](int t) {
        const int64_t kb = min(FQ_KEYS * t, kb_last);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint8_t * q = vq + (((kb + 16 * (e / 4) + e % 4) * a.v.nb1) >> VSH);
#pragma unroll
            for (int j = 0; j < C::VJ; j++) {
                if constexpr (C::VU == 4) xv[e][j] = *(const uint32_t *)(q + vo[j]);
                else xv[e][j] = *(const uint16_t *)(q + vo[j]);
            }
        }
    };

    // this lane's rows: token and head
    int tok[NQ], head[NQ];
    bool ok[NQ];
    const uint16_t * mrow[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int row = (rt * NQ + n) * 16 + r;
        ok[n] = row < a.R;
        tok[n] = ok[n] ? fq_div(row, a.div_g) : 0;
        head[n] = hk * a.G + (ok[n] ? row - tok[n] * a.G : 0);
        mrow[n] = a.mask ? a.mask + (int64_t)s * a.mask_nb3 + (int64_t)tok[n] * a.mask_nb1 + 4 * g : (const uint16_t *)kq;
    }
    // without a mask the same loads read the first key's codes, and nothing looks at them: a load that
    // is sometimes issued would make every wait behind it a wait for all loads
    const int mstep = a.mask ? 1 : 0;
    typedef u32x2 Mask[NQ][2];   // this lane's four keys of either half tile
    auto load_mask = [&](Mask & x, int t) {
        const int kb = min(FQ_KEYS * t, kb_last);
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
                __builtin_memcpy(&x[n][hf], mrow[n] + (kb + 16 * hf) * mstep, 8);   // any alignment of 2 bytes
    };
    // whether some row of the wave sees some key of a tile
    auto seen = [&](const Mask & x) {
        if (!a.mask) return true;
        bool v = false;
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) v |= ok[n] && (x[n][hf][0] != 0xFC00FC00u || x[n][hf][1] != 0xFC00FC00u);
        return __builtin_amdgcn_readfirstlane((int)__any(v)) != 0;   // scalar
    };

    // the first tile is on its way while Q is converted
    int t = tile0 + wave;
    Mask mk0, mk1;
    if (t < tile1) {
        load_mask(mk0, t);
        load_mask(mk1, min(t + NW, ntiles - 1));
        load_k(t);
        load_v(t);
    }

    // Q in the B layout of the Q.K products, scaled, fp16; a row past fp16's range is divided by a
    // factor that multiplies its scores
    half8 qf[NQ][C::KS];
    float qfac[NQ];
    bool q_scaled = false;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int64_t at = (int64_t)s * a.q_nb3 + (int64_t)head[n] * a.q_nb2 + (int64_t)tok[n] * a.q_nb1;
        // a lane's dims of a product: runs of four at q_dim(st, 0) and q_dim(st, 1); past dk zeros
        auto q_dim = [&](int st, int hlf) {
            const int i = st / C::SPP, w = st % C::SPP, c = g + 4 * i;
            if constexpr (KT == T_Q8_0) return 16 * c + 8 * w + 4 * hlf;
            return (C::CB == 16 ? 32 * c : 32 * (c / 2) + 8 * (c % 2)) + 4 * w + 16 * hlf;
        };
        float v[C::KS][8], amax = 0.0f;
        if (a.q_f16) {
            half4 x[C::KS][2];
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int hlf = 0; hlf < 2; hlf++)
                    x[st][hlf] = *(const half4 *)((const uint16_t *)a.q + at + min(q_dim(st, hlf), a.dk - 4));
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int e = 0; e < 8; e++) v[st][e] = (float)x[st][e / 4][e % 4];
        } else {
            float4v x[C::KS][2];
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int hlf = 0; hlf < 2; hlf++) x[st][hlf] = *(const float4v *)((const float *)a.q + at + min(q_dim(st, hlf), a.dk - 4));
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int e = 0; e < 8; e++) v[st][e] = x[st][e / 4][e % 4];
        }
#pragma unroll
        for (int st = 0; st < C::KS; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[st][e] = ok[n] && q_dim(st, e / 4) < a.dk ? v[st][e] * a.scale : 0.0f;
                amax = fmaxf(amax, fabsf(v[st][e]));
            }
        amax = fq_col_max(amax);
        qfac[n] = amax > 65504.0f ? amax / 32768.0f : 1.0f;
        const float inv = 1.0f / qfac[n];
#pragma unroll
        for (int st = 0; st < C::KS; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) qf[n][st][e] = (_Float16)(qfac[n] == 1.0f ? v[st][e] : v[st][e] * inv);
        q_scaled |= qfac[n] != 1.0f;
        __builtin_amdgcn_sched_barrier(0);   // one tile's F32 rows at a time
    }
    q_scaled = __any(q_scaled);

    float4v o[NQ][C::TT];
    float m_run[NQ], l_run[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m_run[n] = -INFINITY;
        l_run[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < C::TT; t++) o[n][t] = float4v{0, 0, 0, 0};
    }
    const float cap2 = a.softcap != 0.0f ? 2.0f * FQ_LOG2E / a.softcap : 0.0f;
    uint8_t * const ws = smem + wave * C::SCALE_LDS;   // this wave's V scales [block][key]

    bool vis = t < tile1 && seen(mk0);
    while (t < tile1) {
        const bool next = t + NW < tile1;
        const int kb = min(FQ_KEYS * t, kb_last);
        // the lane offsets stay 32-bit registers beside scalar bases (widened outside the loop they would
        // be pairs, and every address a 64-bit addition)
#pragma unroll
        for (int i = 0; i < C::KI; i++) asm("" : "+v"(ko[i]), "+v"(kdo[i]));
#pragma unroll
        for (int i = 0; i < C::VJ; i++) asm("" : "+v"(vo[i]));
#pragma unroll
        for (int i = 0; i < C::VS; i++) asm("" : "+v"(vdo[i]));
        float4v sc[NQ][2];
        if (vis) {
            // V's scales into LDS, those that are not finite as zeros; their keys get a NaN K scale
            // instead, so that it is their scores that become NaN
            bool bad = false;
#pragma unroll
            for (int i = 0; i < C::VS; i++) {
                bad |= (xvd[i] & 0x7C00u) == 0x7C00u;
                *(uint16_t *)(ws + (((lane / 32) * C::VS + i) * FQ_KEYS + lane % 32) * 2) = fq_scale<VT>(xvd[i], 0);
            }
            const uint64_t bad_lanes = __ballot(bad);
            if (bad_lanes) {
                const uint32_t bad_keys = (uint32_t)bad_lanes | (uint32_t)(bad_lanes >> 32);
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
                    if ((bad_keys >> (16 * hf + r)) & 1u) xkd[hf][0] = 0x7E00;
            }
            asm volatile("" ::: "memory");   // one wave's LDS operations complete in order
            // ---- S^T = K . Q^T ----
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
#pragma unroll
                for (int n = 0; n < NQ; n++) sc[n][hf] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < C::KI; i++) {
                    const half2v d = h2_of(fq_scale<KT>(xkd[hf][i], 0x7E00) * 0x10001u);
#pragma unroll
                    for (int w = 0; w < C::SPP; w++) {
                        const half8 kf = KT == T_Q8_0 ? fq_key<KT>(xk[hf][i][(2 * w) % (C::CB / 4)], xk[hf][i][(2 * w + 1) % (C::CB / 4)], d)
                                                      : fq_key<KT>(xk[hf][i][w % (C::CB / 4)], 0, d);
#pragma unroll
                        for (int n = 0; n < NQ; n++)
                            sc[n][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[n][i * C::SPP + w], sc[n][hf], 0, 0, 0);
                    }
                }
            }
        }
        const bool vis1 = next && seen(mk1);
        const int tn = __builtin_amdgcn_readfirstlane(vis1 ? t + NW : t);
        load_k(tn);   // the next tile's, or this one's again
        half8 pf[NQ];
        if (vis) {
            // ---- scale back, cap, mask, softmax ----
            const bool part = kb < FQ_KEYS * t;
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                if (q_scaled) {
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[n][hf][e] *= qfac[n];
                }
                if (a.softcap != 0.0f) {
                    // cap * tanh(s / cap) = cap - 2 cap / (1 + exp(2 s / cap)): off by some 1e-7 of cap
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sc[n][hf][e] = fmaf(-2.0f * a.softcap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[n][hf][e] * cap2)), a.softcap);
                }
                if (a.mask) {
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float mv = h2f_bits((uint16_t)(mk0[n][hf][e / 2] >> (16 * (e % 2))));
                            sc[n][hf][e] = mv == -INFINITY ? -INFINITY : sc[n][hf][e] + mv;   // a hidden score may be NaN
                        }
                }
                if (part) {
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (kb + 16 * hf + 4 * g + e < FQ_KEYS * t) sc[n][hf][e] = -INFINITY;
                }
                float mt = -INFINITY;
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) mt = fmaxf(mt, sc[n][hf][e]);
                if (__any(mt > m_run[n] + FQ_LAZY)) {
                    mt = fq_col_max(mt);
                    const float m_new = fmaxf(m_run[n], mt);
                    const float alpha = m_run[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m_run[n] - m_new) * FQ_LOG2E);
                    m_run[n] = m_new;
                    l_run[n] *= alpha;
#pragma unroll
                    for (int q = 0; q < C::TT; q++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n][q][e] *= alpha;
                }
                const float mb = m_run[n] == -INFINITY ? 0.0f : m_run[n] * FQ_LOG2E;
                const half2v one2 = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const half2v p = h2_of(pack2h(__builtin_amdgcn_exp2f(fmaf(sc[n][hf][e], FQ_LOG2E, -mb)),
                                                      __builtin_amdgcn_exp2f(fmaf(sc[n][hf][e + 1], FQ_LOG2E, -mb))));
                        pf[n][4 * hf + e] = p[0];
                        pf[n][4 * hf + e + 1] = p[1];
                        l_run[n] = __builtin_amdgcn_fdot2(p, one2, l_run[n], false);   // the sum of what is multiplied
                    }
            }
        }
        // the mask moves up a tile here, where the one in flight has long come: a copy of a register that a
        // load behind the codes' still writes would wait for all of them
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                mk0[n][hf] = mk1[n][hf];
                asm volatile("" : "+v"(mk0[n][hf]));
            }
        load_mask(mk1, min(t + 2 * NW, ntiles - 1));
        if (vis) {
            // ---- O^T += V^T . P^T ----
#pragma unroll
            for (int j = 0; j < C::VJ; j++) {
                half2v d[4];
                {
                    const uint8_t * p = ws + vblk[j] * FQ_KEYS * 2 + 8 * g;
                    d[0] = h2_of(*(const u32_alias *)p);
                    d[1] = h2_of(*(const u32_alias *)(p + 4));
                    d[2] = h2_of(*(const u32_alias *)(p + 32));
                    d[3] = h2_of(*(const u32_alias *)(p + 36));
                }
#pragma unroll
                for (int n = 0; n < C::VU; n++) {
                    uint32_t y[4];   // byte n of keys (2 e, 2 e + 1), zero-extended
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        y[e] = __builtin_amdgcn_perm(xv[2 * e + 1][j], xv[2 * e][j], 0x0C000C00u | ((uint32_t)(4 + n) << 16) | (uint32_t)n);
#pragma unroll
                    for (int h = 0; h < C::VH; h++) {
                        half8 vf;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            half2v p;
                            if constexpr (VT == T_Q8_0) p = h2_of(y[e] ^ 0x64806480u) + half2v{(_Float16)-1152.0f, (_Float16)-1152.0f};
                            else p = h2_of(((h ? y[e] >> 4 : y[e]) & 0x000F000Fu) | 0x64006400u) + half2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
                            p = p * d[e];
                            vf[2 * e] = p[0];
                            vf[2 * e + 1] = p[1];
                        }
                        const int q = (j * C::VU + n) * C::VH + h;
#pragma unroll
                        for (int nq = 0; nq < NQ; nq++) o[nq][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[nq], o[nq][q], 0, 0, 0);
                    }
                }
            }
            asm volatile("" ::: "memory");   // the next tile's scales are written after these reads
        }
        load_v(tn);
        t += NW;
        vis = vis1;
    }

    // ---- merge the block's waves ----
    float * const sml = (float *)smem;                     // [NW][16 NQ][2]: (max, sum)
    float4v * const so = (float4v *)(smem + NW * 16 * NQ * 8);   // [NW][CT][64]
    __syncthreads();                                       // the scale areas are done with
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        l_run[n] = fq_col_sum(l_run[n]);
        if (g == 0) {
            sml[((wave * NQ + n) * 16 + r) * 2] = m_run[n];
            sml[((wave * NQ + n) * 16 + r) * 2 + 1] = l_run[n];
        }
    }
    __syncthreads();
    float M[NQ], L[NQ], wgt[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        M[n] = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) M[n] = fmaxf(M[n], sml[((w * NQ + n) * 16 + r) * 2]);
        L[n] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float mw = sml[((w * NQ + n) * 16 + r) * 2];
            L[n] += sml[((w * NQ + n) * 16 + r) * 2 + 1] * (mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((mw - M[n]) * FQ_LOG2E));
        }
        wgt[n] = m_run[n] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m_run[n] - M[n]) * FQ_LOG2E);
    }
    const int64_t unit = ((int64_t)(s * a.HK + hk) * a.nrt + rt) * a.nsplit + split;
    if (a.nsplit > 1 && wave == 0 && g == 0) {
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            float * ml = a.part_ml + (unit * NQ * 16 + n * 16 + r) * 2;
            ml[0] = M[n];
            ml[1] = L[n];
        }
    }
    constexpr int ALL = C::TT * NQ;
#pragma unroll
    for (int c0 = 0; c0 < ALL; c0 += C::CT) {
        if (c0) __syncthreads();
#pragma unroll
        for (int i = 0; i < C::CT; i++) {
            const int n = (c0 + i) / C::TT, q = (c0 + i) % C::TT;
            float4v v = o[n][q];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] *= wgt[n];
            so[(wave * C::CT + i) * WAVE + lane] = v;
        }
        __syncthreads();
        for (int i = wave; i < C::CT; i += NW) {
            float4v v = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const float4v p = so[(w * C::CT + i) * WAVE + lane];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += p[e];
            }
            const int at = c0 + i, n = at / C::TT, q = at % C::TT;
            if (a.nsplit > 1) {
                *(float4v *)(a.part_o + ((unit * ALL + at) * WAVE + lane) * 4) = v;
                continue;
            }
            const int row = (rt * NQ + n) * 16 + r;
            if (row >= a.R) continue;
            float Ln = L[0];
#pragma unroll
            for (int k = 1; k < NQ; k++)
                if (n == k) Ln = L[k];
            const float inv = Ln > 0.0f ? 1.0f / Ln : 0.0f;
            const int tk = fq_div(row, a.div_g);
            const int64_t dst = (int64_t)s * a.dst_nb3 + (int64_t)tk * a.dst_nb2 + (int64_t)(hk * a.G + row - tk * a.G) * a.dst_nb1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = fq_dim(VT, C::VU, q, g, e);
                if (d < a.dv) {
                    if (a.dst_f16) ((uint16_t *)a.dst)[dst + d] = f2h_bits(v[e] * inv);
                    else ((float *)a.dst)[dst + d] = v[e] * inv;
                }
            }
        }
    }
}

template <int KT, int VT, int DK, int DV, int NQ>
static hipError_t fq_launch(const FaQArgs & a, hipStream_t st) {
    using C = FqCfg<KT, VT, DK, DV, NQ>;
    static_assert(C::LDS <= 160 * 1024, "LDS");
    static bool done = false;
    if (!done) {
        const hipError_t e = hipFuncSetAttribute((const void *)fa_q_kernel<KT, VT, DK, DV, NQ>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
        if (e != hipSuccess) return e;
        done = true;
    }
    const int64_t units = (int64_t)a.S * a.HK * a.nrt;
    hipLaunchKernelGGL((fa_q_kernel<KT, VT, DK, DV, NQ>), dim3((unsigned)(units * a.nsplit)), dim3(C::NW * WAVE), C::LDS, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    return launch_fa_q_combine(a, VT, DV, NQ, st);
}

template <int KT, int VT, int DK, int DV>
static hipError_t fq_rows(const FaQArgs & a, hipStream_t st) {
    if (a.nq == 1) return fq_launch<KT, VT, DK, DV, 1>(a, st);
    if (a.nq == 2) return fq_launch<KT, VT, DK, DV, 2>(a, st);
    if constexpr (DV <= 128)
        if (a.nq == 4) return fq_launch<KT, VT, DK, DV, 4>(a, st);
    return hipErrorInvalidValue;
}

template <int KT, int VT>
static hipError_t fq_dims(const FaQArgs & a, hipStream_t st) {
    if (a.D == 64 && a.DV == 64) return fq_rows<KT, VT, 64, 64>(a, st);
    if (a.D == 128 && a.DV == 128) return fq_rows<KT, VT, 128, 128>(a, st);
    if (a.D == 192 && a.DV == 128) return fq_rows<KT, VT, 192, 128>(a, st);
    if (a.D == 256 && a.DV == 256) return fq_rows<KT, VT, 256, 256>(a, st);
    return hipErrorInvalidValue;
}

#define FQ_TYPES(K, V) \
    hipError_t launch_fa_q_##K##_##V(const FaQArgs & a, hipStream_t st) { return fq_dims<T_##K, T_##V>(a, st); }

}  // namespace mx
