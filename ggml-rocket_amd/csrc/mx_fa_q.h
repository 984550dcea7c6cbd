// SPDX-License-Identifier: MIT
// FLASH_ATTN_EXT of few query rows over a quantized cache (Q8_0 / Q4_0 K and V), for gfx950: single
// tokens, drafts and short prompts. The cache is read once, as it is stored.
//
//   O[t,h,:] = softmax_j( cap(scale * q[h,t].k[hk,j]) + mask[t,j] ) . v[hk,j,:],  hk = h / G, G = H / HK
//
// The T * G query rows of one KV head share its keys, so they are the columns of the products: a wave
// takes 16 NQ rows and 32 keys at a time, in 16x16x32 MFMAs,
//   S^T = K . Q^T    (A: 16 keys x one block of 32 dims, B: 32 dims x 16 rows)
//   O^T += V^T . (P d)^T (A: 16 dims x 32 keys, B: 32 keys x 16 rows; d: V's scales of these dims' block)
// with scores, softmax statistics and O in F32 and everything of a row in the four lanes of its
// column. A wave is on its own until its keys are done: its tiles' codes come by LDS DMA into two buffers
// of its own, so there are no barriers in the loop. (Loaded straight into the operands' lanes, where
// neighbouring lanes are different keys, every load took the address unit a cycle a lane and the kernel
// waited for it: 978 cycles of it a tile at head dim 128; by DMA neighbouring lanes are neighbouring bytes.)
// The order of dims in a contraction and of keys in a tile is free, and chosen so that no lane needs
// another's data:
//   K   the lanes of group g hold bytes 8 g (Q8_0) or 4 g (Q4_0) on of every block of one key.
//   P   the S^T accumulators of two 16-key products are the P^T operand: slot e of lane group g is key
//       8 g + e, which product e / 4 has as its row 4 g + e % 4.
//   V   ds_read_b64_tr_b8 hands a lane of group g one byte of each of those eight keys, and v_perm_b32 puts
//       two of them into a pair of halves. The 16 dims of a product are 16 bytes of a row, of one block.
//
// What bounds it is the work of turning codes into operands, so that is kept to a few integer
// instructions a pair: an unsigned code u = code + 128 (Q8_0) or u = code (Q4_0, value u - 8) in the low
// bits of a half is the subnormal u 2^-24, which the matrix unit multiplies exactly. A high nibble left
// in place counts 16 times; its Q is divided by 16 beforehand, its O afterwards.
// (Exactly, but a sum's products are lined up by their operands' exponent fields, and a subnormal has that of 2^-14 however
// small it is: a block of four-bit codes is off by up to 40 times 2^-24 of sum |q u|, 5 in the mean, one of eight-bit codes by 2 and
// 0.3, one of normal halves by 1 and 0.2.)
//   K   one product is one block, so its scale multiplies the F32 result (S += d S_b), and the offset
//       is the product's start value, -128 (or -8) sum_dims q, a product of q with a constant: K is exact.
//   V   its scale multiplies P, once for a block's 32 dims, and the codes are exact. P d is held times 2^k, k such
//       that the largest d of that block of dims that the wave has seen is just below 2^7 (P goes to 2^8, see below;
//       k moves rarely, and O with it). The offset leaves at the end, as a multiple of the sum of the same P d.
// Roundings: Q, P and P d, once each, to fp16, the matrix unit's operands (F32 ones would take two products for each).
// Each is off by at most 2^-11 of itself; a P below 2^-14 by 2^-25, a P d by 2^-32 of the largest d of its dims. (With V's
// scales multiplied into V's halves, under one power of two for all dims, values 2^13 below the largest were lost, and the
// others rounded relative to their unsigned codes: 6e-4 of an output's norm from 64 bits; now 3.7e-4.)
//
// Scales go through a few bytes of LDS a wave, which turns a key's row of them into one block's of
// several keys. The running maximum moves only when a score passes it by more than 8 in the exponent of 2
// (P stays below 256, well inside fp16), so most tiles exchange nothing between lanes.
//
// Each part of a tile is requested two tiles ahead. The waves of a block take alternate tiles of the block's
// key range and merge through LDS at the end; the key range is split over blocks where there are too
// few of them, and a second launch merges those. Tiles that the mask hides from every row of a wave are left
// out: a lane looks at one tile's mask, for 64 of the wave's tiles at a time (only where at most 8 tokens
// share a wave; else every tile is read).
//
// Measured (this kernel; its merge is 4 us more where keys are split), 32 heads on 8 of head dim 128: one token
// on 1000 Q8_0 keys 9.4 us, on 32768 Q4_0 keys 16.7 us (38 MB, 2.3 TB/s); 32 sequences of 4096 Q8_0 keys 67 us
// (286 MB, 4.3 TB/s, the rate of a plain read), of 1 to 4096 keys 54 us (143 MB: the longest's 16 tiles a
// wave at some 2.5 us each). A block's start until its first data is 3 to 5 us, its end 2.5 us. A tile is the latency
// of its wave's own chain, not a unit at its limit (32768 Q4_0 keys: VALU instructions 0.23 of a wave's time, waits
// 0.24, matrix units 0.04 busy).
//
// A cache in pages (mi355x_flash_attn_paged; FaPArgs, `PG` below) is read by the same loop. A tile is 32 rows of one page, so its
// place is one table entry, which comes through the scalar cache a tile ahead: the counts that the waits go by stay
// as they are. The lengths are read on the device and a unit's keys are split evenly over its blocks, however many there
// are. Instead of a mask a row has a number of keys that it sees and, of the new tokens, a bit each (fp_sees: the ancestors of
// its node of the tree, from the parents by doubling, in each wave), looked at in the last tiles alone.
// Roundings there: P d, from F32, once; Q is exact where it is fp16 (a row of 128 and more loses 2^-35 of its largest value at most), its scale in K's F32
// scales, and two halves, hi + lo, off by 2^-22 of a value and 2^-27 of its row's largest, where it is F32 (one more product a block). An output is 1.7e-4 of its norm from 64 bits, 2.7e-4 as fp16, for 2.9e-4
// and 3.6e-4 with Q rounded and P rounded before d; an F32 Q takes 0 to 4 % longer than an fp16 one, 6 % with many rows.
// Measured (this kernel, its merge 4 us more): one token on 1000 Q8_0 keys 11.7 us, 32 sequences of 1 to 4096 keys 56 us (143 MB, 2.6
// TB/s; the longest ones' chain), a tree of 5 on 131072 Q4_0 keys 77 us (151 MB, 2.0 TB/s), of 16 on 16000 keys of head dim 256 42
// us. With many keys a wave's tile is 346 vector instructions and 24 products (the tree of 5); with two waves a SIMD vector
// instructions take 0.60 of its time, instructions of any kind 0.90, waits 0.16 of a wave's. What was taken out of it: the offsets'
// products are formed once before the loop, P d rounds in one instruction each and a nibble's mask needs no byte moved
// first (68 of 414 vector instructions and 8 of 32 products; the tree of 5 took 80.8 us with them). What did not help: two tiles
// side by side through each step (253 registers) took as long, blocks of four waves two a CU 53 us for 40 (32 sequences out of the
// last-level cache), twelve waves of 168 registers a quarter longer (28 spilled), the offsets as products instead of sums of P d
// 7 % longer, and parts made alike over all sequences by their lengths 59 us for 53.

#pragma once

#include <limits.h>

#include <type_traits>

#include "mx_common.h"
#include "mx_kernels_impl.h"
#include "mx_pages.h"
#include "mx_weights.h"

namespace mx {

constexpr int FQ_KEYS = 32;      // keys a tile
constexpr int FQ_LDS_MAX = 160 * 1024;
constexpr int FQ_BASE_REGS = 96;  // with 64 there are more waves and spills: 32768 Q4_0 keys 30.5 us a call, not 19.8
constexpr int FQ_SCAN_TOKENS = 8;
constexpr float FQ_LAZY = 8.0f / 1.4426950408889634f;
constexpr float FQ_LOG2E = 1.4426950408889634f;

// KT, VT: T_Q8_0 or T_Q4_0; DK, DV: the built head dims; NQ: 16-row query tiles a wave.
// PG: over a cache in pages.
template <int KT, int VT, int DK, int DV, int NQ, bool PG>
struct FqCfg {
    static constexpr int KRB = KT == T_Q8_0 ? DK : DK / 2, VRB = VT == T_Q8_0 ? DV : DV / 2;   // bytes a row
    static constexpr int KS = DK / 32;                        // blocks a K row: Q.K products
    static constexpr int KW = KT == T_Q8_0 ? 2 : 1;           // dwords of a block a lane holds
    // 16-byte chunks of a row in LDS (K: a power of two, 12 and 6 padded) and DMA instructions a tile
    static constexpr int KCH = KRB / 16 <= 2 ? 2 : KRB / 16 <= 4 ? 4 : KRB / 16 <= 8 ? 8 : 16, VCH = VRB / 16;
    static constexpr int KD = KCH / 2, VD = VCH / 2;
    static constexpr int STAGE = FQ_KEYS * 16 * (KCH + VCH);
    // Chunk c of row r lies at c ^ swz(r): the 16 rows that a read of one chunk takes then lie in 16
    // different chunk slots of LDS's 256-byte window. K rows lie in the order 16 h + 4 g + e (key 8 g + 4 h + e),
    // V rows in that of the keys.
    __device__ static __forceinline__ int kswz(int row) { return (row * KCH / 16) & (KCH - 1); }
    __device__ static __forceinline__ int vswz(int row) { return (row * VCH / 16) & (VCH - 1); }
    static constexpr int VH = VT == T_Q4_0 ? 2 : 1;           // nibbles a byte
    static constexpr int VN = 4 / VH;                         // chunks of two of V's blocks, read at a time
    // pages: a nibble's mask takes the other bytes away, so two of four bytes stay where they are
    static constexpr bool BY_TWOS = PG && VT == T_Q4_0;
    static constexpr int TT = DV / 16;                        // O^T tiles of 16 dims: chunk * VH + nibble
    static_assert(KRB == 16 * KS * KW && VCH * VH == TT, "layout");
    static constexpr int VB = DV / 32, VS = DV / 64, KSC = DK / 64;   // scales a key, and a lane (32 keys, two lanes each)
    static constexpr int KSL = KSC == 3 ? 4 : KSC, VSL = VS;  // and of a lane's load
    static constexpr int QN = NQ * KS * 64;                   // Q as B operands (pages: twice, halves hi and lo), then its rows' factors
    static constexpr int Q_LDS = (PG ? 2 : 1) * QN * 16 + NQ * 64;
    static constexpr int SCALE_LDS = KS * FQ_KEYS * 4 + VB * FQ_KEYS * 2;   // a wave's scales: K's F32, V's F16
    static constexpr int WAVE_LDS = SCALE_LDS + 2 * STAGE;
    // registers: O, scores and masks, a block of K and the offsets' product, the rest; the waves a SIMD they
    // leave room for, and as many in a block, one block a CU, as the buffers leave room for (5 tokens on 16384 Q4_0
    // keys of head dim 256: one wave a SIMD 28.4 us, two, which spill, 36.8)
    static constexpr int REGS = (TT * 4 + VB) * NQ + 30 * NQ + KD + VD + 6 * KS + KSC + VS + FQ_BASE_REGS;
    static constexpr int WPE = REGS <= 128 ? 4 : REGS <= 168 ? 3 : REGS <= 256 ? 2 : 1;
    static constexpr int FIT = (FQ_LDS_MAX - Q_LDS) / WAVE_LDS / 4 * 4;
    static constexpr int NW = FIT < 4 * WPE ? FIT : 4 * WPE;
    static_assert(NW >= 4, "LDS");
    // with two waves a SIMD or fewer and one query tile there is room to keep the offsets' products
    static constexpr bool KEEP_OFF = NQ == 1 && NW <= 8;
    static constexpr bool KEEP_Q = PG && NQ == 1 && NW == 4;  // and with one wave a SIMD Q itself
    static constexpr int CT = TT * NQ < 8 ? TT * NQ : 8;      // O^T tiles merged at a time
    static constexpr int LOOP_LDS = Q_LDS + NW * WAVE_LDS;
    static constexpr int MERGE_LDS = NW * 16 * NQ * 8 + NW * CT * 1024;
    static constexpr int LDS = MERGE_LDS > LOOP_LDS ? MERGE_LDS : LOOP_LDS;
};

typedef void __attribute__((address_space(3))) * fq_lptr_t;
// 16 bytes a lane into LDS, lane after lane, from byte `off` (below 2^31) of a wave-uniform address. As
// buffer loads: while a global load to LDS is pending, the compiler makes every wait for a register load
// one for all loads.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t fq_rsrc(const void * p) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, 0x7FFFFFFF, 0x00020000);
}
__device__ __forceinline__ void fq_dma16(__amdgpu_buffer_rsrc_t p, uint32_t off, void * l) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(p, (fq_lptr_t)l, 16, off, 0, 0, 0);
}
// No memory access moves across it; waits until at most N vector loads are outstanding.
template <int N>
__device__ __forceinline__ void fq_wait_vm() {
    static_assert(N >= 0 && N <= 63, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Eight bytes a lane out of LDS, transposed, from N addresses (bytes of LDS, OFF further): of the 8 x 16 bytes whose row
// i / 2 the lanes i of a group of 16 point at (the odd ones at its second half), lane i receives column i, row 0 lowest.
// As one statement with its wait: before a builtin of them the compiler would wait for every LDS DMA under way.
typedef int fq_v2i __attribute__((ext_vector_type(2)));
template <int N, int OFF>
__device__ __forceinline__ void fq_read_tr(const uint32_t (&a)[N], fq_v2i (&w)[N]) {
    static_assert(N == 2 || N == 4, "chunks");
    if constexpr (N == 2)
        asm volatile("ds_read_b64_tr_b8 %0, %2 offset:%4\n"
                     "ds_read_b64_tr_b8 %1, %3 offset:%4\n"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(w[0]), "=&v"(w[1])
                     : "v"(a[0]), "v"(a[1]), "n"(OFF)
                     : "memory");
    else
        asm volatile("ds_read_b64_tr_b8 %0, %4 offset:%8\n"
                     "ds_read_b64_tr_b8 %1, %5 offset:%8\n"
                     "ds_read_b64_tr_b8 %2, %6 offset:%8\n"
                     "ds_read_b64_tr_b8 %3, %7 offset:%8\n"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
                     : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(OFF)
                     : "memory");
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

// The maximum over the wave's lanes of the same parity: three rotations of the rows of 16, then across them.
__device__ __forceinline__ float fq_parity_max(float x) {
#define FQ_DPP_MAX(CTRL) x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true)))
    FQ_DPP_MAX(0x128);   // row_ror:8
    FQ_DPP_MAX(0x124);   // row_ror:4
    FQ_DPP_MAX(0x122);   // row_ror:2
#undef FQ_DPP_MAX
    return fq_col_max(x);
}
// Lane l's value, the same in every lane.
__device__ __forceinline__ float fq_lane(float x, int l) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
}

// A block's scale: held to the largest with which every value stays inside fp16 (kv_scale_limit), as
// where the cache is decoded first; infinite or NaN ones as `bad`.
template <int TYPE>
__device__ __forceinline__ float fq_scale(uint16_t bits, float bad) {
    const float d = fmaxf(fminf(h2f_bits(bits), kv_scale_limit(TYPE)), -kv_scale_limit(TYPE));
    return (bits & 0x7C00u) == 0x7C00u ? bad : d;
}

// N fp16 scales, of any alignment.
template <int N>
__device__ __forceinline__ uint64_t fq_load_scales(const uint8_t * p) {
    if constexpr (N == 1) return *(const uint16_t *)p;
    uint32_t lo, hi = 0;
    __builtin_memcpy(&lo, p, 4);
    if constexpr (N == 4) __builtin_memcpy(&hi, p + 4, 4);
    return (uint64_t)hi << 32 | lo;
}

// A lane's eight unsigned codes of a K block, each the low bits of a half. Q8_0: dims 8 g + 0..7. Q4_0:
// dims 4 g + {0, 2, 1, 3} and, 16 times as large, 16 + 4 g + {0, 2, 1, 3}.
template <int KT>
__device__ __forceinline__ half8 fq_key(const uint32_t * x) {
    u32x4 w;
    if constexpr (KT == T_Q8_0) {
        const uint32_t a = x[0] ^ 0x80808080u, b = x[1] ^ 0x80808080u;
        w = u32x4{__builtin_amdgcn_perm(0u, a, 0x0C010C00u), __builtin_amdgcn_perm(0u, a, 0x0C030C02u),
                  __builtin_amdgcn_perm(0u, b, 0x0C010C00u), __builtin_amdgcn_perm(0u, b, 0x0C030C02u)};
    } else {
        const uint32_t y = x[0] >> 8;
        w = u32x4{x[0] & 0x000F000Fu, y & 0x000F000Fu, x[0] & 0x00F000F0u, y & 0x00F000F0u};
    }
    return __builtin_bit_cast(half8, w);
}

// A lane's four dims from d on of an output row at dst, times inv.
__device__ __forceinline__ void fq_store4(const FaQArgs & a, int64_t dst, int d, const float4v & v, float inv) {
    if (d >= a.dv) return;
    if (a.dst_f16) *(u32x2 *)((uint16_t *)a.dst + dst + d) = u32x2{pack2h(v[0] * inv, v[1] * inv), pack2h(v[2] * inv, v[3] * inv)};
    else *(float4v *)((float *)a.dst + dst + d) = v * inv;
}

// Pages: row n of this lane (one of rt's 16 NQ) sees keys below lim[n] and, of the new tokens', those whose bits are set in
// anc[n]. Returns the number of first keys that every row sees; `up`: the parent of tree node `lane`.
template <int NQ>
__device__ __forceinline__ int fp_sees(const FaPArgs & a, int lane, int rt, int up, int n_past, int n_new, int tok_a, const bool (&ok)[NQ], int (&lim)[NQ],
                                       uint64_t (&anc)[NQ]) {
    const int room = a.st.cap - n_past;   // of new tokens
    const bool tree = a.st.parent != nullptr;
    const uint64_t node = tree ? tree_ancestors(up, lane) : 0;
    if (tree && lane < n_new && !node && a.st.err) *a.st.err = 1;
    const int all = n_past + (tree ? 0 : min(tok_a + 1, room));
    bool none = false;
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int tok = ok[n] ? fq_div((rt * NQ + n) * 16 + lane % 16, a.div_g) : 0;
        lim[n] = tok < n_new ? n_past : 0;
        anc[n] = 0;
        if (tree) {
            const uint32_t lo = (uint32_t)__shfl((int)(uint32_t)node, tok, WAVE), hi = (uint32_t)__shfl((int)(uint32_t)(node >> 32), tok, WAVE);
            anc[n] = tok < n_new ? (uint64_t)hi << 32 | lo : 0;
            if (!anc[n]) lim[n] = 0;
            if (room < KV_TREE_MAX) anc[n] &= ((uint64_t)1 << room) - 1;
        } else if (tok < n_new) {
            lim[n] = n_past + min(tok + 1, room);
        }
        none |= ok[n] && lim[n] < all;
    }
    return __any(none) ? 0 : all;
}
// Of keys j .. j + 7 those that a row sees, as bits.
__device__ __forceinline__ uint32_t fp_visible(int j, int n_past, int lim, uint64_t anc) {
    const int c = lim - j, u = j - n_past;
    uint32_t vis = c >= 8 ? 0xFFu : c > 0 ? (1u << c) - 1 : 0u;
    if (u > -8 && u < KV_TREE_MAX) vis |= (uint32_t)(u >= 0 ? anc >> u : anc << -u) & 0xFFu;
    return vis;
}

// A: FaQArgs, or FaPArgs for a cache in pages.
template <int KT, int VT, int DK, int DV, int NQ, class A>
__global__ void __launch_bounds__((FqCfg<KT, VT, DK, DV, NQ, std::is_same<A, FaPArgs>::value>::NW * WAVE))
__attribute__((amdgpu_waves_per_eu(FqCfg<KT, VT, DK, DV, NQ, std::is_same<A, FaPArgs>::value>::NW / 4, FqCfg<KT, VT, DK, DV, NQ, std::is_same<A, FaPArgs>::value>::NW / 4)))
fa_q_kernel(A a) {
    constexpr bool PG = std::is_same<A, FaPArgs>::value;
    using C = FqCfg<KT, VT, DK, DV, NQ, PG>;
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int NW = C::NW;
    // The arguments lie in host memory, a round trip of half a microsecond and more a cache line; used
    // here, one of each line, they all come at once instead of where each is first needed.
    asm volatile("" ::"s"(a.q), "s"(a.k.nb3), "s"(a.v.nb2), "s"(a.dst), "s"(a.mask_nb3), "s"(a.T), "s"(a.div_split.mul), "s"(a.softcap));
    if constexpr (PG) asm volatile("" ::"s"(a.st.table), "s"(a.st.parent_nb), "s"(a.div_tpp.mul));
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, g = lane / 16;

    // block -> (sequence, split, KV head, query rows): an XCD's run of blocks shares keys, and the KV
    // heads of a token lie side by side in a token-major cache
    int b = xcd_tile(blockIdx.x, gridDim.x), b1 = fq_div(b, a.div_nrt);
    const int rt = b - b1 * a.nrt;
    b = b1;
    b1 = fq_div(b, a.div_hk);
    const int hk = b - b1 * a.HK, s = fq_div(b1, a.div_split), split = b1 - s * a.nsplit;
    // pages: the first keys of the sequence, up to the last that a row of this block sees
    int n_past = 0, n_new = 0, keys = a.KV, up = -1;
    if constexpr (PG) {
        const StepOf sq = step_of(a.st, s);
        n_past = sq.past;
        n_new = sq.fresh;
        if (sq.bad && threadIdx.x == 0 && a.st.err) *a.st.err = 1;
        const int tok0 = fq_div(rt * 16 * NQ, a.div_g), tok1 = fq_div(min(a.R, (rt + 1) * 16 * NQ) - 1, a.div_g);
        const int seen = a.st.parent ? n_new : min(n_new, tok1 + 1);
        keys = tok0 < n_new ? min(n_past + seen, a.st.cap) : 0;
        if (a.st.parent && lane < a.T) up = a.st.parent[(int64_t)s * a.st.parent_nb + lane];
    }
    const int ntiles = (keys + FQ_KEYS - 1) / FQ_KEYS, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int tile0 = split * per, tile1 = min(ntiles, tile0 + per);

    // Tile t starts at key kb(t) = min(32 t, KV - 32), KV >= 32: a last partial tile is moved back and
    // its keys before 32 t, which the tile before has, do not count. So every load stays inside the
    // cache without a bound per lane: a scalar base and the lane's fixed 32-bit offset.
    // (In pages a tile is 32 rows of one page, all of them rows of the cache; the keys behind the last count for no row.)
    const int kb_last = PG ? INT_MAX : a.KV - FQ_KEYS;
    // Pages: the row where tile t begins, -1 for a tile of a page that the cache does not have
    auto page_of = [&](int t) -> int64_t {
        if constexpr (PG) {
            const int p = fq_div(t, a.div_tpp);
            const int64_t row = page_row(a.st, uniform_i32(a.st.table, (int64_t)s * a.st.table_nb + p));
            return row < 0 ? -1 : row + FQ_KEYS * (t - p * a.div_tpp.d);
        }
        return 0;
    };
    // the row that tile t is read from
    auto first_row = [&](int t, int64_t row) -> int64_t {
        if constexpr (PG) return row < 0 ? 0 : row;
        return min(FQ_KEYS * t, kb_last);
    };
    constexpr int KSH = KT == T_Q4_0, VSH = VT == T_Q4_0;   // elements to bytes
    const uint8_t * const kq = a.k.q + (((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) >> KSH);
    const uint8_t * const vq = a.v.q + (((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) >> VSH);
    const uint16_t * const kd = a.k.d + ((int64_t)s * a.k.nb3 + (int64_t)hk * a.k.nb2) / 32;
    const uint16_t * const vd = a.v.d + ((int64_t)s * a.v.nb3 + (int64_t)hk * a.v.nb2) / 32;
    const uint32_t knb = (uint32_t)a.k.nb1, vnb = (uint32_t)a.v.nb1;
    // chunks and scales past dk or dv: the first ones (Q is zero there, O is not stored)
    uint32_t kdma[C::KD], vdma[C::VD];   // this lane's chunk of each DMA instruction: byte offset from the tile
#pragma unroll
    for (int q = 0; q < C::KD; q++) {
        const int slot = q * WAVE + lane, row = slot / C::KCH, c = (slot % C::KCH) ^ C::kswz(row);
        const uint32_t key = row % 16 / 4 * 8 + row / 16 * 4 + row % 4;
        kdma[q] = ((key * knb) >> KSH) + (c * 16 < (a.dk >> KSH) ? 16 * c : 0);
    }
#pragma unroll
    for (int q = 0; q < C::VD; q++) {
        const int slot = q * WAVE + lane, c = (slot % C::VCH) ^ C::vswz(slot / C::VCH);
        const uint32_t key = slot / C::VCH;
        vdma[q] = ((key * vnb) >> VSH) + (c * 16 < (a.dv >> VSH) ? 16 * c : 0);
    }
    // The scales this lane fetches: key lane / 2, half of its blocks, in one load that stays inside the row
    // (dk and dv are at least half of the built dims): shifted down to the first of them, zeros behind the last.
    const int kn32 = a.dk / 32, vn32 = a.dv / 32, half = lane % 2;
    const int kfirst = min(half * C::KSC, kn32 - C::KSL), vfirst = min(half * C::VS, vn32 - C::VSL);
    const uint32_t kdo = (uint32_t)(lane / 2) * (knb / 32 * 2) + 2 * kfirst, vdo = (uint32_t)(lane / 2) * (vnb / 32 * 2) + 2 * vfirst;
    const int ksh = min(16 * (half * C::KSC - kfirst), 63), vsh = min(16 * (half * C::VS - vfirst), 63);
    // where this lane reads: bytes 4 KW g on of a K block (block i at kra ^ kra_i), and half a chunk of V row 8 g + r / 2
    // (chunk c at vra ^ 16 c)
    uint32_t kra = r * C::KCH * 16;
    kra += KT == T_Q8_0 ? ((C::kswz(r) ^ (g / 2)) << 4) + 8 * (g % 2) : (C::kswz(r) << 4) + 4 * g;
    const uint32_t vra = (8 * g + r / 2) * C::VRB + (C::vswz(8 * g + r / 2) << 4) + 8 * (r % 2);

    uint8_t * const wl = smem + C::Q_LDS + wave * C::WAVE_LDS;   // this wave's scales and buffers
    const uint32_t vlds = (uint32_t)(uintptr_t)(fq_lptr_t)wl;    // its LDS address
    float * const wk = (float *)wl;                              // K scales [block][key]
    uint16_t * const wv = (uint16_t *)(wk + C::KS * FQ_KEYS);    // V scales [block][key]
    auto dma_k = [&](int t, int64_t row, int buf) {
        const __amdgpu_buffer_rsrc_t kt = fq_rsrc(kq + ((first_row(t, row) * a.k.nb1) >> KSH));
        uint8_t * st = wl + C::SCALE_LDS + buf * C::STAGE;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int q = 0; q < C::KD; q++) fq_dma16(kt, kdma[q], st + q * 1024);
        asm volatile("" ::: "memory");
    };
    auto dma_v = [&](int t, int64_t row, int buf) {
        const __amdgpu_buffer_rsrc_t vt = fq_rsrc(vq + ((first_row(t, row) * a.v.nb1) >> VSH));
        uint8_t * st = wl + C::SCALE_LDS + buf * C::STAGE + FQ_KEYS * 16 * C::KCH;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int q = 0; q < C::VD; q++) fq_dma16(vt, vdma[q], st + q * 1024);
        asm volatile("" ::: "memory");
    };

    // this lane's rows
    bool ok[NQ];
    const uint16_t * mrow[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int row = (rt * NQ + n) * 16 + r;
        ok[n] = row < a.R;
        const int tok = ok[n] ? fq_div(row, a.div_g) : 0;
        mrow[n] = a.mask ? a.mask + (int64_t)s * a.mask_nb3 + (int64_t)tok * a.mask_nb1 + 8 * g : (const uint16_t *)kq;
    }
    // without a mask the same loads read the first key's codes, and nothing looks at them: a load that
    // is sometimes issued would make every wait behind it a wait for all loads
    const int mstep = a.mask ? 1 : 0;
    struct Side {              // what of a tile comes into registers
        uint64_t kd, vd;
        u32x4 m[NQ];           // the mask of this lane's eight keys
    };
    auto load_side = [&](Side & x, int t, int64_t row) {
        const int64_t kb = first_row(t, row);
        x.kd = fq_load_scales<C::KSL>((const uint8_t *)kd + kb * a.k.nb1 / 32 * 2 + kdo);
        x.vd = fq_load_scales<C::VSL>((const uint8_t *)vd + kb * a.v.nb1 / 32 * 2 + vdo);
        if constexpr (!PG) {
#pragma unroll
            for (int n = 0; n < NQ; n++) __builtin_memcpy(&x.m[n], mrow[n] + kb * mstep, 16);   // any alignment of 2 bytes
        }
    };
    // The wave's tiles are tile0 + wave + NW k. next() gives the next k that some row sees (-1: none): bits
    // of 64 of them, one lane a tile.
    const int nk = tile1 - tile0 > wave ? (tile1 - tile0 - wave + NW - 1) / NW : 0;
    const int tok_a = fq_div(rt * 16 * NQ, a.div_g), tok_b = fq_div(min(a.R, (rt + 1) * 16 * NQ) - 1, a.div_g);
    const bool scan = !PG && a.mask && tok_b - tok_a < FQ_SCAN_TOKENS;
    uint64_t todo = 0;
    int k0 = -64;              // the 64 that todo is for
    auto next = [&]() {
        while (todo == 0) {
            k0 += 64;
            if (k0 >= nk) return -1;
            const int k = k0 + lane;
            bool v = k < nk;
            if (v && scan) {
                const int kb = min(FQ_KEYS * (tile0 + wave + NW * k), kb_last);
                v = false;
                for (int tk = tok_a; tk <= tok_b; tk++) {
                    const uint16_t * p = a.mask + (int64_t)s * a.mask_nb3 + (int64_t)tk * a.mask_nb1 + kb;
                    u32x4 w[4];
                    __builtin_memcpy(w, p, 64);
#pragma unroll
                    for (int i = 0; i < 16; i++) v |= w[i / 4][i % 4] != 0xFC00FC00u;
                }
            }
            todo = __ballot(v);
        }
        const int k = k0 + __builtin_ctzll(todo);
        todo &= todo - 1;
        return __builtin_amdgcn_readfirstlane(k);
    };

    // Q in the B layout of the Q.K products, scaled, fp16, in LDS: wave n makes the operands of query tile n.
    // Its loads go out before the first tile's, which comes while Q is converted.
    half8 * const lq = (half8 *)smem;                                       // [NQ][KS][64]
    float * const lqf = (float *)(smem + C::Q_LDS - NQ * 64);               // [NQ][16]: 0 where no row needs a factor
    // a lane's dims of block st: runs of four at q_dim(st, 0) and q_dim(st, 1); past dk zeros
    auto q_dim = [&](int st, int hlf) { return 32 * st + (KT == T_Q8_0 ? 8 * g + 4 * hlf : 4 * g + 16 * hlf); };
    u32x4 qraw[C::KS][2];   // four values each: F32, or F16 in the first two words
    const int qrow = (rt * NQ + wave) * 16 + r;
    const bool qok = qrow < a.R;
    if (wave < NQ) {
        const int qtok = qok ? fq_div(qrow, a.div_g) : 0, qhead = hk * a.G + (qok ? qrow - qtok * a.G : 0);
        const int64_t at = (int64_t)s * a.q_nb3 + (int64_t)qhead * a.q_nb2 + (int64_t)qtok * a.q_nb1;
        if (a.q_f16) {
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int hlf = 0; hlf < 2; hlf++) {
                    const u32x2 w = *(const u32x2 *)((const uint16_t *)a.q + at + min(q_dim(st, hlf), a.dk - 4));
                    qraw[st][hlf] = u32x4{w[0], w[1], 0, 0};
                }
        } else {
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int hlf = 0; hlf < 2; hlf++) qraw[st][hlf] = *(const u32x4 *)((const float *)a.q + at + min(q_dim(st, hlf), a.dk - 4));
        }
    }

    // The first two tiles are requested before their masks are looked at; tiles that turn out hidden are
    // replaced once they have landed. Waves without tiles read some tile all the same: loads that are
    // sometimes issued would make every wait behind them a wait for all loads.
    const int tile_end = PG ? max(ntiles, 1) - 1 : ntiles - 1;
    int t = min(tile0 + wave, tile_end), tn = min(tile0 + wave + NW, tile_end);
    // Pages: the rows of both, and of the tile that is requested next (a wave's tiles follow each other: no mask hides
    // any): its table entry is on its way while this one's products are formed.
    int64_t row_t = page_of(t), row_n = page_of(tn), row_p = page_of(min(tn + NW, tile_end));
    Side x0, x1;
    auto request = [&]() {   // a tile's K, its scales and masks, its V, then the next tile's
        dma_k(t, row_t, 0);
        load_side(x0, t, row_t);
        dma_v(t, row_t, 0);
        dma_k(tn, row_n, 1);
        load_side(x1, tn, row_n);
        dma_v(tn, row_n, 1);
    };
    request();

    if (wave < NQ) {
        float v[C::KS][8], amax = 0.0f;
#pragma unroll
        for (int st = 0; st < C::KS; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t half = qraw[st][e / 4][e % 4 / 2] >> (16 * (e % 2));
                const float x = a.q_f16 ? h2f_bits((uint16_t)half) : __uint_as_float(qraw[st][e / 4][e % 4]);
                v[st][e] = qok && q_dim(st, e / 4) < a.dk ? (PG ? x : x * a.scale) : 0.0f;   // pages: K's scales carry it
                amax = fmaxf(amax, fabsf(v[st][e]));
            }
        amax = fq_col_max(amax);
        // a row outside [2^-6, 2^15] is divided by a factor that multiplies its scores (its largest value
        // goes to 2^4, so that the smaller ones, and 1/16 of them, keep their bits); the factor has a finite
        // reciprocal: values below 2^-116 then come out smaller than 2^4, and their scores are zero all the same
        // Pages: every row times 2^8, which K's scales take back; one outside [2^-2, 2^7) times the power of two (at most 2^127) that
        // brings its largest value to [2^14, 2^15). So the bits of an fp16 row stay, also of 1/16 of it, and an F32 row's low halves
        // keep theirs.
        float qfac, inv;
        if constexpr (PG) {
            const bool in = amax < 128.0f && (amax >= 0.25f || amax == 0.0f);
            const uint32_t e = in ? 127 : max((int)(__float_as_uint(amax) >> 23) - 6, 8);
            qfac = __uint_as_float(e << 23);
            inv = __uint_as_float((262u - e) << 23);
        } else {
            qfac = (amax > 32768.0f || (amax < 0.015625f && amax > 0.0f)) ? fmaxf(amax / 16.0f, 0x1p-120f) : 1.0f;
            inv = 1.0f / qfac;
        }
#pragma unroll
        for (int st = 0; st < C::KS; st++) {
            half8 qf, lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                // slot e of fq_key is value e (Q8_0), or 0, 2, 1, 3 of either half
                const float x = v[st][KT == T_Q8_0 ? e : (e & 4) | (e & 1) << 1 | (e & 2) >> 1] * inv;
                const float y = KT == T_Q4_0 && e >= 4 ? x * 0.0625f : x;
                qf[e] = (_Float16)y;
                lo[e] = (_Float16)(y - (float)qf[e]);
            }
            lq[(wave * C::KS + st) * WAVE + lane] = qf;
            if constexpr (PG) lq[C::QN + (wave * C::KS + st) * WAVE + lane] = lo;
        }
        if (g == 0) lqf[wave * 16 + r] = __any(qfac != 1.0f) ? qfac : 0.0f;
    }
    const int ka = next();
    int kn = ka >= 0 ? next() : -1;
    if (!PG && (ka > 0 || kn > 1)) {
        fq_wait_vm<0>();
        t = tile0 + wave + NW * ka;
        tn = kn >= 0 ? tile0 + wave + NW * kn : t;
        request();
    }
    int lim[NQ], full_to = INT_MAX;
    uint64_t anc[NQ];
    if constexpr (PG) full_to = fp_sees<NQ>(a, lane, rt, up, n_past, n_new, tok_a, ok, lim, anc);
    // a barrier for LDS alone: the first tiles' loads stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // the offsets' products: -128 2^-24 (Q8_0), -8 2^-24 and, for high nibbles, -128 2^-24 (Q4_0) in every
    // element, as bits of halves
    constexpr uint32_t kOffLo = KT == T_Q8_0 ? 0x80808080u : 0x80088008u, kOffHi = 0x80808080u;
    u32x4 koff = {kOffLo, kOffLo, kOffHi, kOffHi};
    float4v o[NQ][C::TT];      // O^T without the offsets
    float oc[NQ][C::VB];       // sum P d 2^k of each block, this lane's keys
    float m_run[NQ], l_run[NQ];
    bool scaled[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        scaled[n] = __any(lqf[n * 16 + r] != 0.0f);
        m_run[n] = -INFINITY;
        l_run[n] = 0.0f;
#pragma unroll
        for (int t = 0; t < C::TT; t++) o[n][t] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < C::VB; b++) oc[n][b] = 0.0f;
    }
    float vscale[C::VS];        // 2^k of this lane's blocks, half VS + i
    uint32_t vtop[C::VS];       // the largest scale each is for, as fp16 bits: 2^(7 - k)
#pragma unroll
    for (int i = 0; i < C::VS; i++) {
        vscale[i] = 1.0f;
        vtop[i] = 0;
    }
    const half2v one2 = {(_Float16)1.0f, (_Float16)1.0f};
    half8 kq_hi[C::KEEP_Q ? C::KS : 1], kq_lo[C::KEEP_Q ? C::KS : 1];
    if constexpr (C::KEEP_Q)
#pragma unroll
        for (int i = 0; i < C::KS; i++) {
            kq_hi[i] = lq[i * WAVE + lane];
            kq_lo[i] = lq[C::QN + i * WAVE + lane];
        }
    const bool q_two = PG && !a.q_f16;   // an fp16 Q is its hi
    float4v kept_off[PG && C::KEEP_OFF ? C::KS : 1];   // the offsets' products (the compiler leaves them in the loop's two forms)
    if constexpr (PG && C::KEEP_OFF)
#pragma unroll
        for (int i = 0; i < C::KS; i++) {
            const half8 hi = C::KEEP_Q ? kq_hi[i] : lq[i * WAVE + lane], lo = C::KEEP_Q ? kq_lo[i] : lq[C::QN + i * WAVE + lane];
            kept_off[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, koff), hi, float4v{0, 0, 0, 0}, 0, 0, 0);
            if (q_two) kept_off[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, koff), lo, kept_off[i], 0, 0, 0);
        }
    const float kscale = PG ? 65536.0f * a.scale : 16777216.0f;   // pages: Q holds 2^8
    const float cap2 = a.softcap != 0.0f ? 2.0f * FQ_LOG2E / a.softcap : 0.0f;

    // Tile t in buffer BUF, with its scales and masks in x. Everything of a tile is requested two tiles ahead, each
    // part as soon as the one that it takes the place of has been used, and waited for apart, so nearly two
    // tiles' time is there for it. (Requested and waited for as one, a wave waited 0.9 us of a tile's
    // 2.6 for it: 32 sequences of up to 4096 keys, Q8_0, head dim 128.) Returns false after the last tile.
    auto tile = [&](Side & x, auto buffer) __attribute__((always_inline)) {
        constexpr int BUF = decltype(buffer)::value;
        constexpr int SL = PG ? 2 : 2 + NQ;              // loads of load_side
        // K's codes and x have landed; behind them V, and the next tile's three
        fq_wait_vm<C::VD + C::KD + SL + C::VD>();
        const int kb = min(FQ_KEYS * t, kb_last);
        const uint8_t * const st = wl + C::SCALE_LDS + BUF * C::STAGE;
        if constexpr (!C::KEEP_OFF) asm("" : "+v"(koff));   // else the offsets' products would move out of the loop
        float4v sc[NQ][2];
        {
            // ---- S^T = K . Q^T, each block's product times its scale (and 2^24) ----
#pragma unroll
            for (int i = 0; i < C::KSC; i++)
                wk[(half * C::KSC + i) * FQ_KEYS + lane / 2] = fq_scale<KT>((uint16_t)((x.kd >> ksh) >> (16 * i)), NAN) * kscale;
            asm volatile("" ::: "memory");   // one wave's LDS operations complete in order
#pragma unroll
            for (int n = 0; n < NQ; n++) sc[n][0] = sc[n][1] = float4v{0, 0, 0, 0};
            auto products = [&](auto two) __attribute__((always_inline)) {   // two: Q in halves hi and lo
#pragma unroll
            for (int i = 0; i < C::KS; i++) {
                float4v off[NQ];
                half8 qf[NQ];
#pragma unroll
                for (int n = 0; n < NQ; n++) qf[n] = C::KEEP_Q ? kq_hi[i] : lq[(n * C::KS + i) * WAVE + lane];
#pragma unroll
                for (int n = 0; n < NQ; n++)
                    off[n] = PG && C::KEEP_OFF ? kept_off[i] : __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, koff), qf[n], float4v{0, 0, 0, 0}, 0, 0, 0);
                half8 ql[NQ];
                if constexpr (decltype(two)::value)
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        ql[n] = C::KEEP_Q ? kq_lo[i] : lq[C::QN + (n * C::KS + i) * WAVE + lane];
                        if constexpr (!PG || !C::KEEP_OFF)
                            off[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, koff), ql[n], off[n], 0, 0, 0);
                    }
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float4v d = *(const float4v *)(wk + i * FQ_KEYS + 8 * g + 4 * hf);
                    uint32_t kx[2];
                    if constexpr (C::KW == 2) {
                        const u32x2 w = *(const u32x2 *)(st + (kra ^ (uint32_t)(32 * i)) + hf * 256 * C::KCH);
                        kx[0] = w[0];
                        kx[1] = w[1];
                    } else {
                        kx[0] = *(const uint32_t *)(st + (kra ^ (uint32_t)(16 * i)) + hf * 256 * C::KCH);
                    }
                    const half8 kf = fq_key<KT>(kx);
#pragma unroll
                    for (int n = 0; n < NQ; n++) {
                        float4v p = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[n], off[n], 0, 0, 0);
                        if constexpr (decltype(two)::value) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[n], p, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[n][hf][e] = fmaf(p[e], d[e], sc[n][hf][e]);
                    }
                }
                if (!C::KEEP_OFF) __builtin_amdgcn_sched_barrier(0);   // not every block's operands at once
            }
            };
            if constexpr (PG) {
                if (q_two) products(std::true_type{});
                else products(std::false_type{});
            } else {
                products(std::false_type{});
            }
        }
        // K's codes have been read: the ones of the tile after the next come in their place (the last ones
        // again, where there is none: the number of loads in flight stays what the waits count)
        const int k2 = kn >= 0 ? next() : -1;
        const int t2 = k2 >= 0 ? tile0 + wave + NW * k2 : tn;
        const int64_t row2 = k2 >= 0 ? row_p : row_n;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        dma_k(t2, row2, BUF);
        if constexpr (PG) row_p = page_of(min(t2 + NW, tile_end));
        u32x4 pf[NQ];       // P, fp16
        float px[NQ][8];    // pages: P
        {
            // ---- scale back, cap, mask, softmax ----
            const bool part = kb < FQ_KEYS * t;
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                if (scaled[n]) {
                    const float qfac = lqf[n * 16 + r];
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[n][hf][e] *= qfac;
                }
                if (a.softcap != 0.0f) {
                    // cap * tanh(s / cap) = cap - 2 cap / (1 + exp(2 s / cap)): off by some 1e-7 of cap
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sc[n][hf][e] = fmaf(-2.0f * a.softcap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[n][hf][e] * cap2)), a.softcap);
                }
                if constexpr (PG) {
                    if (FQ_KEYS * (t + 1) > full_to || row_t < 0) {
                        if (row_t < 0 && a.st.err) *a.st.err = 1;
                        const uint32_t vis = row_t < 0 ? 0 : fp_visible(FQ_KEYS * t + 8 * g, n_past, lim[n], anc[n]);
#pragma unroll
                        for (int hf = 0; hf < 2; hf++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (!((vis >> (4 * hf + e)) & 1u)) sc[n][hf][e] = -INFINITY;   // a hidden score may be NaN
                    }
                } else if (a.mask && __any((x.m[n][0] | x.m[n][1] | x.m[n][2] | x.m[n][3]) != 0)) {
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float mv = h2f_bits((uint16_t)(x.m[n][2 * hf + e / 2] >> (16 * (e % 2))));
                            sc[n][hf][e] = mv == -INFINITY ? -INFINITY : sc[n][hf][e] + mv;   // a hidden score may be NaN
                        }
                }
                if (!PG && part) {
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (kb + 8 * g + 4 * hf + e < FQ_KEYS * t) sc[n][hf][e] = -INFINITY;
                }
            }
            // ---- V's scales (key lane / 2): the power of two a block's are held under; into LDS times it ----
            float dv[C::VS];
            bool bad = false, larger = false;
#pragma unroll
            for (int i = 0; i < C::VS; i++) {
                const uint16_t bits = (uint16_t)((x.vd >> vsh) >> (16 * i));
                bad |= (bits & 0x7C00u) == 0x7C00u;
                dv[i] = fq_scale<VT>(bits, 0.0f);
                larger |= (bits & 0x7FFFu) > vtop[i];
            }
            if (__any(larger)) {
                // a larger scale than any before, or one that is not finite (which stands for zero and makes
                // the row sums of the rows that see its key NaN); keys that no row sees count as zeros
                bool hidden = false;
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int e = 0; e < 8; e++) hidden |= ok[n] && sc[n][e / 4][e % 4] == -INFINITY;
                if (__any(hidden)) {
                    uint32_t seen_keys = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        bool any = false;
#pragma unroll
                        for (int n = 0; n < NQ; n++) any |= ok[n] && sc[n][e / 4][e % 4] != -INFINITY;
                        const uint64_t rows = __ballot(any);
#pragma unroll
                        for (int gg = 0; gg < 4; gg++)
                            seen_keys |= (uint32_t)(((rows >> (16 * gg)) & 0xFFFFu) != 0) << (8 * gg + e);
                    }
                    const bool mine = (seen_keys >> (lane / 2)) & 1u;
                    bad &= mine;
#pragma unroll
                    for (int i = 0; i < C::VS; i++) dv[i] = mine ? dv[i] : 0.0f;
                }
                const uint64_t bad_lanes = __ballot(bad);
                if (bad_lanes) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if ((bad_lanes >> (2 * (8 * g + e))) & 3u) {
#pragma unroll
                            for (int n = 0; n < NQ; n++)
                                if (sc[n][e / 4][e % 4] != -INFINITY) l_run[n] = NAN;
                        }
                }
#pragma unroll
                for (int i = 0; i < C::VS; i++) {
                    const float dmax = fq_parity_max(fabsf(dv[i]));
                    // a power of two at least as large, by its exponent
                    const uint32_t pow2 = (__float_as_uint(dmax) + 0x7FFFFFu) & 0x7F800000u;
                    const float next_scale = __uint_as_float((261u << 23) - pow2);   // 2^7 / pow2
                    float f = 1.0f;
                    if (dmax > 0.0f && (vtop[i] == 0 || next_scale < vscale[i])) {
                        f = next_scale * __builtin_amdgcn_rcpf(vscale[i]);   // powers of two: exact
                        vscale[i] = next_scale;
                        vtop[i] = f2h_bits(__uint_as_float(pow2));
                    }
#pragma unroll
                    for (int hb = 0; hb < 2; hb++) {
                        const int b = hb * C::VS + i;
                        const float fb = fq_lane(f, hb);
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            oc[n][b] *= fb;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                o[n][2 * b][e] *= fb;
                                o[n][2 * b + 1][e] *= fb;
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < C::VS; i++) wv[(half * C::VS + i) * FQ_KEYS + lane / 2] = f2h_bits(dv[i] * vscale[i]);
            asm volatile("" ::: "memory");
#pragma unroll
            for (int n = 0; n < NQ; n++) {
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
#pragma unroll
                    for (int b = 0; b < C::VB; b++) oc[n][b] *= alpha;
                }
                const float mb = m_run[n] == -INFINITY ? 0.0f : m_run[n] * FQ_LOG2E;
                if constexpr (PG) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        px[n][e] = __builtin_amdgcn_exp2f(fmaf(sc[n][e / 4][e % 4], FQ_LOG2E, -mb));
                        l_run[n] += px[n][e];
                    }
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float s0 = sc[n][e / 2][2 * (e % 2)], s1 = sc[n][e / 2][2 * (e % 2) + 1];
                    pf[n][e] = pack2h(__builtin_amdgcn_exp2f(fmaf(s0, FQ_LOG2E, -mb)), __builtin_amdgcn_exp2f(fmaf(s1, FQ_LOG2E, -mb)));
                    l_run[n] = __builtin_amdgcn_fdot2(h2_of(pf[n][e]), one2, l_run[n], false);   // the sum of what is multiplied
                }
            }
        }
        asm volatile("" ::: "memory");
        load_side(x, t2, row2);
        fq_wait_vm<C::KD + SL + C::VD + C::KD + SL>();   // this tile's V has landed
        {
            // ---- O^T += V^T . (P d 2^k)^T, two blocks of 32 dims at a time ----
#pragma unroll
            for (int c0 = 0; c0 < C::VCH; c0 += C::VN) {
                const uint16_t * const wd = wv + c0 * C::VH / 2 * FQ_KEYS + 8 * g;
                const u32x4 d[2] = {*(const u32x4 *)wd, *(const u32x4 *)(wd + FQ_KEYS)};
                uint32_t va[C::VN];
                fq_v2i w[C::VN];
#pragma unroll
                for (int c = 0; c < C::VN; c++) va[c] = vlds + (vra ^ (uint32_t)(16 * (c0 + c)));
                fq_read_tr<C::VN, C::SCALE_LDS + BUF * C::STAGE + FQ_KEYS * 16 * C::KCH>(va, w);
                u32x4 pd[NQ];
#pragma unroll
                for (int c = 0; c < C::VN; c++) {
                    const int b = (c0 + c) * C::VH / 2;
                    if ((c0 + c) * C::VH % 2 == 0) {   // a block's first chunk
#pragma unroll
                        for (int n = 0; n < NQ; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                if constexpr (PG) {   // rounded once (with the addition one instruction each, without it 2 1/2)
                                    const int k0 = C::BY_TWOS ? 4 * (e / 2) + e % 2 : 2 * e, k1 = k0 + (C::BY_TWOS ? 2 : 1);
                                    pd[n][e] = u_of(half2v{(_Float16)fmaf(px[n][k0], (float)h2_of(d[b % 2][k0 / 2])[k0 % 2], 0.0f),
                                                           (_Float16)fmaf(px[n][k1], (float)h2_of(d[b % 2][k1 / 2])[k1 % 2], 0.0f)});
                                } else {
                                    pd[n][e] = u_of(h2_of(pf[n][e]) * h2_of(d[b % 2][e]));
                                }
                                oc[n][b] = __builtin_amdgcn_fdot2(h2_of(pd[n][e]), one2, oc[n][b], false);
                            }
                    }
                    const uint32_t flip = VT == T_Q8_0 ? 0x80808080u : 0u, xl = (uint32_t)w[c][0] ^ flip, xh = (uint32_t)w[c][1] ^ flip;
                    // bytes of keys (2 e, 2 e + 1), zero-extended, or those of keys (0, 2), (1, 3), (4, 6), (5, 7) in the low ones
                    const u32x4 y = C::BY_TWOS ? u32x4{xl, xl >> 8, xh, xh >> 8}
                                               : u32x4{__builtin_amdgcn_perm(0u, xl, 0x0C010C00u), __builtin_amdgcn_perm(0u, xl, 0x0C030C02u),
                                                       __builtin_amdgcn_perm(0u, xh, 0x0C010C00u), __builtin_amdgcn_perm(0u, xh, 0x0C030C02u)};
#pragma unroll
                    for (int h = 0; h < C::VH; h++) {
                        const u32x4 u = VT == T_Q8_0 ? y : h ? y & 0x00F000F0u : y & 0x000F000Fu;
                        const int q = (c0 + c) * C::VH + h;
#pragma unroll
                        for (int n = 0; n < NQ; n++)
                            o[n][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, u), __builtin_bit_cast(half8, pd[n]), o[n][q], 0, 0, 0);
                    }
                    if (!C::KEEP_OFF) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        dma_v(t2, row2, BUF);
        if (kn < 0) return false;
        t = tn;
        tn = t2;
        row_t = row_n;
        row_n = row2;
        kn = k2;
        return true;
    };
    if (ka >= 0)
        while (tile(x0, std::integral_constant<int, 0>{}) && tile(x1, std::integral_constant<int, 1>{})) {}
    fq_wait_vm<0>();   // no DMA may still write what the merge reuses

    // ---- merge the block's waves ----
    float * const sml = (float *)smem;                     // [NW][16 NQ][2]: (max, sum)
    float4v * const so = (float4v *)(smem + NW * 16 * NQ * 8);   // [NW][CT][64]
    __syncthreads();                                       // the scale areas are done with
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        l_run[n] = fq_col_sum(l_run[n]);
#pragma unroll
        for (int b = 0; b < C::VB; b++) oc[n][b] = fq_col_sum(oc[n][b]);
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
            // values: the offset off (in units of 2^-24 d), then 2^24, 2^-k and a high nibble's 1/16
            constexpr float kOff = VT == T_Q8_0 ? 128.0f : 8.0f;
            const bool high = VT == T_Q4_0 && q % 2;
            float4v v = o[n][q];
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] = fmaf(oc[n][q / 2], -kOff, v[e] * (high ? 1048576.0f : 16777216.0f)) *
                       (wgt[n] * __builtin_amdgcn_rcpf(fq_lane(vscale[q / 2 % C::VS], q / 2 / C::VS)));
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
            const float inv = Ln == 0.0f ? 0.0f : 1.0f / Ln;   // no key seen: zeros; a NaN stays
            const int tk = fq_div(row, a.div_g);
            const int64_t dst = (int64_t)s * a.dst_nb3 + (int64_t)tk * a.dst_nb2 + (int64_t)(hk * a.G + row - tk * a.G) * a.dst_nb1;
            fq_store4(a, dst, 16 * q + 4 * g, v, inv);
        }
    }
}

template <int KT, int VT, int DK, int DV, int NQ, class A>
static hipError_t fq_launch(const A & a, hipStream_t st) {
    using C = FqCfg<KT, VT, DK, DV, NQ, std::is_same<A, FaPArgs>::value>;
    static_assert(C::LDS <= 160 * 1024, "LDS");
    static LdsAllowed done;
    const hipError_t l = allow_lds((const void *)fa_q_kernel<KT, VT, DK, DV, NQ, A>, C::LDS, done);
    if (l != hipSuccess) return l;
    const int64_t units = (int64_t)a.S * a.HK * a.nrt;
    hipLaunchKernelGGL((fa_q_kernel<KT, VT, DK, DV, NQ, A>), dim3((unsigned)(units * a.nsplit)), dim3(C::NW * WAVE), C::LDS, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    return launch_fa_q_combine(a, DV, NQ, st);
}

template <int KT, int VT, int DK, int DV, class A>
static hipError_t fq_rows(const A & a, hipStream_t st) {
    if (a.nq == 1) return fq_launch<KT, VT, DK, DV, 1>(a, st);
    if constexpr (DK == 64)
        if (a.nq == 2) return fq_launch<KT, VT, DK, DV, 2>(a, st);
    return hipErrorInvalidValue;
}

template <int KT, int VT, class A>
static hipError_t fq_dims(const A & a, hipStream_t st) {
    if (a.D == 64 && a.DV == 64) return fq_rows<KT, VT, 64, 64>(a, st);
    if (a.D == 128 && a.DV == 128) return fq_rows<KT, VT, 128, 128>(a, st);
    if (a.D == 192 && a.DV == 128) return fq_rows<KT, VT, 192, 128>(a, st);
    if (a.D == 256 && a.DV == 256) return fq_rows<KT, VT, 256, 256>(a, st);
    return hipErrorInvalidValue;
}

#define FQ_TYPES(K, V) \
    hipError_t launch_fa_q_##K##_##V(const FaQArgs & a, hipStream_t st) { return fq_dims<T_##K, T_##V>(a, st); }
#define FP_TYPES(K, V) \
    hipError_t launch_fa_p_##K##_##V(const FaPArgs & a, hipStream_t st) { return fq_dims<T_##K, T_##V>(a, st); }

}  // namespace mx
