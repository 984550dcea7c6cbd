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
// tile's codes come straight into registers, a tile ahead. The order of dims in a contraction and
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
// The waves of a block take alternate tiles of the block's key range and merge through LDS at the end;
// the key range is split over blocks where there are too few of them, and a second launch merges those.
// Tiles that the mask hides from every row of a wave are not read: their mask is looked at a tile
// before their loads are issued, and hidden tiles' loads are sent to the tile before (the number of
// loads in flight stays the same, which keeps the waits exact).

#pragma once

#include <type_traits>

#include "mx_common.h"
#include "mx_kernels_impl.h"
#include "mx_weights.h"

namespace mx {

constexpr int FQ_KEYS = 32;      // keys a tile
constexpr float FQ_LAZY = 8.0f / 1.4426950408889634f;
constexpr float FQ_LOG2E = 1.4426950408889634f;
constexpr float FQ_BIG = 512.0f; // scales below it keep every value (127 * d) inside fp16

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
    // registers: two tiles in flight, O, Q, masks, the rest
    static constexpr int REGS = 2 * (2 * KI * (CB / 4) + 8 * VJ) + (TT + KS) * 4 * NQ + 12 * NQ + 60;
    static constexpr int NW = REGS > 240 ? 4 : 8;             // waves a block, one or two a SIMD
    static constexpr int CT = TT * NQ < 8 ? TT * NQ : 8;      // O^T tiles merged at a time
    static constexpr int SCALE_LDS = VB * FQ_KEYS * 2 + FQ_KEYS * 4;   // a wave's V scales and poison
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

__device__ __forceinline__ float fq_xor16(float x) { return __shfl_xor(x, 16, WAVE); }
__device__ __forceinline__ float fq_xor32(float x) { return __shfl_xor(x, 32, WAVE); }

// Eight values of a key from its codes: a dword pair (Q8_0) or a dword (Q4_0: four low nibbles, four
// high ones), times d.
template <int KT, bool BIG>
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
    if constexpr (BIG) {
        const half2v top = {(_Float16)65504.0f, (_Float16)65504.0f};
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = __builtin_elementwise_max(__builtin_elementwise_min(p[i], top), -top);
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
    int b = xcd_tile(blockIdx.x, gridDim.x);
    const int rt = b % a.nrt;
    b /= a.nrt;
    const int hk = b % a.HK;
    b /= a.HK;
    const int split = b % a.nsplit, s = b / a.nsplit;
    const int ntiles = (a.KV + FQ_KEYS - 1) / FQ_KEYS, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int tile0 = split * per, tile1 = min(ntiles, tile0 + per);

    // this lane's rows: token and head
    int tok[NQ], head[NQ];
    bool ok[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int row = (rt * NQ + n) * 16 + r;
        ok[n] = row < a.R;
        tok[n] = ok[n] ? row / a.G : 0;
        head[n] = hk * a.G + (ok[n] ? row % a.G : 0);
    }

    // Q in the B layout of the Q.K products, scaled, fp16; a row past fp16's range is divided by a
    // factor that multiplies its scores
    half8 qf[NQ][C::KS];
    float qfac[NQ];
    bool q_scaled = false;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int64_t at = (int64_t)s * a.q_nb3 + (int64_t)head[n] * a.q_nb2 + (int64_t)tok[n] * a.q_nb1;
        float v[C::KS][8], amax = 0.0f;
#pragma unroll
        for (int st = 0; st < C::KS; st++) {
            // dims of the step's eight values: two runs of four
            const int i = st / C::SPP, w = st % C::SPP, c = g + 4 * i;
            int d0, d1;
            if constexpr (KT == T_Q8_0) {
                d0 = 16 * c + 8 * w;
                d1 = d0 + 4;
            } else {
                d0 = C::CB == 16 ? 32 * c + 4 * w : 32 * (c / 2) + 8 * (c % 2) + 4 * w;
                d1 = d0 + 16;
            }
#pragma unroll
            for (int hlf = 0; hlf < 2; hlf++) {
                const int d = hlf ? d1 : d0;
                float4v x = {0, 0, 0, 0};
                if (ok[n] && d < a.dk) {
                    if (a.q_f16) {
                        const half4 h = *(const half4 *)((const uint16_t *)a.q + at + d);
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = (float)h[e];
                    } else {
                        x = *(const float4v *)((const float *)a.q + at + d);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v[st][4 * hlf + e] = x[e] * a.scale;
                    amax = fmaxf(amax, fabsf(v[st][4 * hlf + e]));
                }
            }
        }
        amax = fmaxf(amax, fq_xor16(amax));
        amax = fmaxf(amax, fq_xor32(amax));
        qfac[n] = amax > 65504.0f ? amax / 32768.0f : 1.0f;
        const float inv = 1.0f / qfac[n];
#pragma unroll
        for (int st = 0; st < C::KS; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) qf[n][st][e] = (_Float16)(qfac[n] == 1.0f ? v[st][e] : v[st][e] * inv);
        q_scaled |= qfac[n] != 1.0f;
    }
    q_scaled = __any(q_scaled);

    // Tile t starts at key kb(t) = min(32 t, KV - 32): a last partial tile is moved back and its keys
    // before 32 t, which the tile before has, do not count. So every load stays inside the cache without
    // a bound per lane (a cache shorter than a tile: lane keys are held at its last).
    const int kb_last = max(a.KV - FQ_KEYS, 0);
    constexpr int KSH = KT == T_Q4_0, VSH = VT == T_Q4_0;   // elements to bytes
    const int klast = a.KV - 1;
    const uint8_t * const kq = a.k.q + (((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) >> KSH);
    const uint8_t * const vq = a.v.q + (((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) >> VSH);
    const uint16_t * const kd = a.k.d + ((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) / 32;
    const uint16_t * const vd = a.v.d + ((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) / 32;
    uint32_t ko[2], kdo[2];          // this lane's key in either half tile: byte offsets of row and scales
    uint32_t kco[C::KI], kcd[C::KI]; // pieces, and their scales' bytes (a piece past dk: piece 0, Q is zero there)
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
        const uint32_t key = (uint32_t)min(16 * hf + r, klast);
        ko[hf] = (key * (uint32_t)a.k.nb1) >> KSH;
        kdo[hf] = key * (uint32_t)a.k.nb1 / 32 * 2;
    }
#pragma unroll
    for (int i = 0; i < C::KI; i++) {
        int c = g + 4 * i;
        const int elems = KT == T_Q8_0 ? C::CB : 2 * C::CB;
        if (c * elems >= a.dk) c = 0;
        kco[i] = (uint32_t)(c * C::CB);
        kcd[i] = (uint32_t)(c * elems / 32 * 2);
    }
    uint32_t vo[8], vco[C::VJ];      // V rows of the lane's eight keys, and its bytes of them
#pragma unroll
    for (int e = 0; e < 8; e++) vo[e] = ((uint32_t)min(16 * (e / 4) + 4 * g + e % 4, klast) * (uint32_t)a.v.nb1) >> VSH;
    int vblk[C::VJ];
#pragma unroll
    for (int j = 0; j < C::VJ; j++) {
        const int u = (r + 16 * j) * C::VU;                      // byte in the row
        vblk[j] = VT == T_Q8_0 ? u / 32 : u / 16;
        vco[j] = 32 * vblk[j] < a.dv ? (uint32_t)u : 0u;         // past dv: not stored
    }
    uint32_t vdo[C::VS];             // the scales this lane fetches: key lane % 32
#pragma unroll
    for (int i = 0; i < C::VS; i++) {
        int blk = (lane / 32) * C::VS + i;
        if (32 * blk >= a.dv) blk = 0;
        vdo[i] = (uint32_t)min(lane % 32, klast) * (uint32_t)a.v.nb1 / 32 * 2 + 2 * blk;
    }
    const uint16_t * mrow[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++)
        mrow[n] = a.mask ? a.mask + (int64_t)s * a.mask_nb3 + (int64_t)tok[n] * a.mask_nb1 + 4 * g : nullptr;

    struct Tile {
        uint32_t k[2][C::KI][C::CB / 4];
        uint16_t kd[2][C::KI];
        uint32_t v[8][C::VJ];
        uint16_t vd[C::VS];
    };
    struct Mask {
        u32x2 m[NQ][2];   // this lane's four keys of either half tile
    };
    auto kb_of = [&](int t) { return min(FQ_KEYS * t, kb_last); };
    auto load = [&](Tile & x, int t) {
        const int64_t kb = kb_of(t);
        const uint8_t * kq_t = kq + ((kb * a.k.nb1) >> KSH);
        const uint8_t * vq_t = vq + ((kb * a.v.nb1) >> VSH);
        const uint8_t * kd_t = (const uint8_t *)(kd + kb * a.k.nb1 / 32);
        const uint8_t * vd_t = (const uint8_t *)(vd + kb * a.v.nb1 / 32);
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
            for (int i = 0; i < C::KI; i++) {
                if constexpr (C::CB == 16) {
                    const u32x4 w = *(const u32x4 *)(kq_t + (ko[hf] + kco[i]));
#pragma unroll
                    for (int e = 0; e < 4; e++) x.k[hf][i][e] = w[e];
                } else {
                    const u32x2 w = *(const u32x2 *)(kq_t + (ko[hf] + kco[i]));
#pragma unroll
                    for (int e = 0; e < 2; e++) x.k[hf][i][e] = w[e];
                }
                x.kd[hf][i] = *(const uint16_t *)(kd_t + (kdo[hf] + kcd[i]));
            }
#pragma unroll
        for (int i = 0; i < C::VS; i++) x.vd[i] = *(const uint16_t *)(vd_t + vdo[i]);
#pragma unroll
        for (int e = 0; e < 8; e++)
#pragma unroll
            for (int j = 0; j < C::VJ; j++) {
                if constexpr (C::VU == 4) x.v[e][j] = *(const uint32_t *)(vq_t + (vo[e] + vco[j]));
                else x.v[e][j] = *(const uint16_t *)(vq_t + (vo[e] + vco[j]));
            }
    };
    auto load_mask = [&](Mask & x, int t) {
        const int kb = kb_of(t);
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                x.m[n][hf] = u32x2{0, 0};
                if (!a.mask) continue;
                if (a.KV >= FQ_KEYS) {
                    __builtin_memcpy(&x.m[n][hf], mrow[n] + kb + 16 * hf, 8);   // any alignment of 2 bytes
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = mrow[n][min(16 * hf + e, klast - 4 * g)];
                    x.m[n][hf] = u32x2{w[0] | (w[1] << 16), w[2] | (w[3] << 16)};
                }
            }
    };
    // whether some row of the wave sees some key of a tile
    auto seen = [&](const Mask & x) {
        if (!a.mask) return true;
        bool v = false;
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t w = x.m[n][hf][e];
                    v |= ok[n] && ((w & 0xFFFFu) != 0xFC00u || (w >> 16) != 0xFC00u);
                }
        return (bool)__any(v);
    };

    float4v o[NQ][C::TT];
    float m_run[NQ], l_run[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m_run[n] = -INFINITY;
        l_run[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < C::TT; t++) o[n][t] = float4v{0, 0, 0, 0};
    }
    const float inv_cap = a.softcap != 0.0f ? 1.0f / a.softcap : 0.0f;
    // this wave's V scales [block][key], and in the rare case 32 poison values
    uint8_t * const ws = smem + wave * C::SCALE_LDS;
    float * const poison = (float *)(ws + C::VB * FQ_KEYS * 2);

    auto compute = [&](auto big_c, const Tile & x, const Mask & mk, int t) {
        constexpr bool BIG = decltype(big_c)::value;
        const int kb = kb_of(t);
        // V's scales into LDS; those that are not finite as zeros, their keys poisoned
#pragma unroll
        for (int i = 0; i < C::VS; i++) {
            uint16_t d = x.vd[i];
            if constexpr (BIG) d = (d & 0x7C00u) == 0x7C00u ? (uint16_t)0 : d;
            *(uint16_t *)(ws + (((lane / 32) * C::VS + i) * FQ_KEYS + lane % 32) * 2) = d;
        }
        if constexpr (BIG) {
            if (lane < 32) poison[lane] = 0.0f;
            asm volatile("" ::: "memory");
            bool bad = false;
#pragma unroll
            for (int i = 0; i < C::VS; i++) bad |= (x.vd[i] & 0x7C00u) == 0x7C00u;
            if (bad) poison[lane % 32] = NAN;
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int i = 0; i < C::KI; i++)
                    if ((x.kd[hf][i] & 0x7C00u) == 0x7C00u) poison[16 * hf + r] = NAN;
        }
        asm volatile("" ::: "memory");   // one wave's LDS operations complete in order
        // ---- scores ----
        float4v sc[NQ][2];
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
#pragma unroll
            for (int n = 0; n < NQ; n++) sc[n][hf] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < C::KI; i++) {
                uint32_t dbits = x.kd[hf][i];
                if constexpr (BIG) dbits = (dbits & 0x7C00u) == 0x7C00u ? 0u : dbits;
                const half2v d = h2_of(dbits * 0x10001u);
#pragma unroll
                for (int w = 0; w < C::SPP; w++) {
                    const half8 kf = KT == T_Q8_0 ? fq_key<KT, BIG>(x.k[hf][i][(2 * w) % (C::CB / 4)], x.k[hf][i][(2 * w + 1) % (C::CB / 4)], d)
                                                  : fq_key<KT, BIG>(x.k[hf][i][w % (C::CB / 4)], 0, d);
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        sc[n][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[n][i * C::SPP + w], sc[n][hf], 0, 0, 0);
                }
            }
        }
        // ---- scale back, cap, mask, softmax ----
        half8 pf[NQ];
        const bool part = kb < FQ_KEYS * t || kb + FQ_KEYS > a.KV;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            if (q_scaled) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[n][hf][e] *= qfac[n];
            }
            if (a.softcap != 0.0f) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[n][hf][e] = a.softcap * tanhf(sc[n][hf][e] * inv_cap);
            }
            if constexpr (BIG) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[n][hf][e] += poison[16 * hf + 4 * g + e];
            }
            if (a.mask) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float mv = h2f_bits((uint16_t)(mk.m[n][hf][e / 2] >> (16 * (e % 2))));
                        sc[n][hf][e] = mv == -INFINITY ? -INFINITY : sc[n][hf][e] + mv;   // a hidden score may be NaN
                    }
            }
            if (part) {
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = kb + 16 * hf + 4 * g + e;
                        if (j < FQ_KEYS * t || j >= a.KV) sc[n][hf][e] = -INFINITY;
                    }
            }
            float mt = -INFINITY;
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int e = 0; e < 4; e++) mt = fmaxf(mt, sc[n][hf][e]);
            if (__any(mt > m_run[n] + FQ_LAZY)) {
                mt = fmaxf(mt, fq_xor16(mt));
                mt = fmaxf(mt, fq_xor32(mt));
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
        // ---- O^T += V^T . P^T ----
#pragma unroll
        for (int j = 0; j < C::VJ; j++) {
            half2v d[4];
            {
                const uint8_t * p = ws + vblk[j] * FQ_KEYS * 2 + 8 * g;
                uint32_t w[4];
                w[0] = *(const u32_alias *)p;
                w[1] = *(const u32_alias *)(p + 4);
                w[2] = *(const u32_alias *)(p + 32);
                w[3] = *(const u32_alias *)(p + 36);
#pragma unroll
                for (int e = 0; e < 4; e++) d[e] = h2_of(w[e]);
            }
#pragma unroll
            for (int n = 0; n < C::VU; n++) {
                uint32_t y[4];   // byte n of keys (2 e, 2 e + 1), zero-extended
#pragma unroll
                for (int e = 0; e < 4; e++)
                    y[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][j], x.v[2 * e][j], 0x0C000C00u | ((uint32_t)(4 + n) << 16) | (uint32_t)n);
#pragma unroll
                for (int h = 0; h < C::VH; h++) {
                    half8 vf;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        half2v p;
                        if constexpr (VT == T_Q8_0) p = h2_of(y[e] ^ 0x64806480u) + half2v{(_Float16)-1152.0f, (_Float16)-1152.0f};
                        else p = h2_of(((h ? y[e] >> 4 : y[e]) & 0x000F000Fu) | 0x64006400u) + half2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
                        p = p * d[e];
                        if constexpr (BIG) {
                            const half2v top = {(_Float16)65504.0f, (_Float16)65504.0f};
                            p = __builtin_elementwise_max(__builtin_elementwise_min(p, top), -top);
                        }
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
    };
    // a scale of FQ_BIG or more, infinite or NaN
    auto any_big = [&](const Tile & x) {
        bool v = false;
#pragma unroll
        for (int i = 0; i < C::VS; i++) v |= (x.vd[i] & 0x7FFFu) >= 0x6000u;
#pragma unroll
        for (int hf = 0; hf < 2; hf++)
#pragma unroll
            for (int i = 0; i < C::KI; i++) v |= (x.kd[hf][i] & 0x7FFFu) >= 0x6000u;
        return (bool)__any(v);
    };

    int t = tile0 + wave;
    if (t < tile1) {
        Tile x[2];
        Mask mk[3];
        load_mask(mk[0], t);
        load_mask(mk[1], min(t + NW, ntiles - 1));
        bool vis = seen(mk[0]);
        load(x[0], t);
        for (;; ) {
#pragma unroll
            for (int ph = 0; ph < 2; ph++) {
                const bool vis1 = t + NW < tile1 && seen(mk[1]);
                load_mask(mk[2], min(t + 2 * NW, ntiles - 1));
                load(x[1 - ph], vis1 ? t + NW : t);
                if (vis) {
                    if (any_big(x[ph])) compute(std::true_type{}, x[ph], mk[0], t);
                    else compute(std::false_type{}, x[ph], mk[0], t);
                }
                t += NW;
                vis = vis1;
                mk[0] = mk[1];
                mk[1] = mk[2];
                if (t >= tile1) break;
            }
            if (t >= tile1) break;
        }
    }

    // ---- merge the block's waves ----
    float * const sml = (float *)smem;                     // [NW][16 NQ][2]: (max, sum)
    float4v * const so = (float4v *)(smem + NW * 16 * NQ * 8);   // [NW][CT][64]
    __syncthreads();                                       // the scale areas are done with
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        l_run[n] += fq_xor16(l_run[n]);
        l_run[n] += fq_xor32(l_run[n]);
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
        for (int w = 0; w < NW; w++) M[n] = fmaxf(M[n], sml[((w * NQ + n) * 16 + r) * 2]);
        L[n] = 0.0f;
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
            const int64_t dst = (int64_t)s * a.dst_nb3 + (int64_t)(row / a.G) * a.dst_nb2 + (int64_t)(hk * a.G + row % a.G) * a.dst_nb1;
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
