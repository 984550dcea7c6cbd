// SPDX-License-Identifier: MIT
// Attention of few query rows over an fp16 cache in pages, for gfx950: single tokens, trees of drafts, short prompts.
//
//   O[t,h,:] = softmax over the keys that t sees of cap(scale * q[h,t].k[hk,j]), times v[hk,j,:],  hk = h / G, G = H / HK
//
// The plan of mx_fa_q.h without its codes: a wave takes 16 NQ query rows of a KV head and 32 keys at a time, S^T = K . Q^T and
// O^T += V^T . P^T in 16x16x32 MFMAs, so that everything of a row is in the four lanes of its column; K and V come by LDS
// DMA into buffers of the wave's own and no barrier is in the loop. K's operand is one 16-byte read of LDS (a key's eight
// dims), V's two transposing reads (ds_read_b64_tr_b16: the lanes i of a group of 16 point at 4 dims of key i / 4, and lane
// i receives dim i of the four keys).
// Roundings: P, once, to fp16. Q is exact: an fp16 one as it is, an F32 one as the sum of two halves, hi + lo, off by 2^-22 of a value and
// 2^-39 of its row's largest (a second product in the loop, 8 more MFMAs a tile at head dim 128); its scale multiplies the F32 scores. K and V are exact, scores,
// statistics, sums and O F32. An output is 1.7e-4 of its norm from 64 bits, as fp16 2.7e-4.
//
// Bound by HBM with few rows: one token on 32768 keys of 8 x (128 + 128) 31 us (134 MB, 4.3 TB/s) and 4 for the merge, 32
// sequences of 1 to 4096 keys 67 us (275 MB, 4.1 TB/s). With many rows by a wave's work on a tile and the blocks' starts and
// ends, some 8 us: 10 sequences x 256 rows of up to 3065 keys at head dim 64 48 us, 2048 rows of 8192 keys 116 us. Small blocks
// of four waves with one tile each, several a CU, overlap those: for the same single token 31 us with eight waves or two
// tiles a wave, 28 with these (out of the last-level cache), at head dim 64 22 and 18.6; 2048 rows 163 and, two row tiles a wave, 102;
// 4 x 2048 rows of 2000 keys at head dim 64 with three blocks a CU 74, with two of two tiles a wave 90, blocks of six waves 131, of twelve 113.
//
// A key that a row does not see has P = 0, and 0 times a V that is no number would still be none. So in the tiles that
// hold such a key (the last ones of a sequence; all tiles of a block with padding) those of its values that are not finite
// count as zeros, and the rows that do see the key get a sum of NaN instead.

#include "mx_fa_q.h"

namespace mx {

// NW: waves a block, with a tile each in LDS; WPE: waves a SIMD, whose registers they share.
template <int DK, int DV, int NQ, int NW>
struct FpCfg {
    static constexpr int KS = DK / 32, TT = DV / 16;
    // 16-byte chunks of a row (K: a power of two), DMA instructions a tile
    static constexpr int KCH = DK <= 64 ? 8 : DK <= 128 ? 16 : 32, VCH = DV / 8, KD = KCH / 2, VD = VCH / 2;
    static constexpr int K_BYTES = FQ_KEYS * 16 * KCH, STAGE = K_BYTES + FQ_KEYS * 16 * VCH, VRB = 16 * VCH;
    // Chunk c of K row r lies at c ^ kswz(r), so that the 16 rows of a read lie in 16 different chunks of LDS's 256-byte
    // window; chunk c of V row r at c ^ 2 vswz(r): the eight 32-byte pieces that 32 lanes read (keys 8 g + 0..3 or 4..7, g two
    // neighbours) in eight different places of it.
    __device__ static __forceinline__ int kswz(int r) { return KCH >= 16 ? r & 15 : (r / 2) & 7; }
    __device__ static __forceinline__ int vswz(int r) { return VCH >= 16 ? (r & 3) | (r >> 1 & 4) : (r >> 1 & 1) | (r >> 2 & 2); }
    static constexpr int CT = TT * NQ < 8 ? TT * NQ : 8;      // O^T tiles merged at a time
    static constexpr int Q_LO = NW * STAGE;                   // the halves lo of Q: [NQ][KS][64], behind the tiles
    static constexpr int LOOP_LDS = Q_LO + NQ * KS * 1024;
    static constexpr int MERGE_LDS = NW * 16 * NQ * 8 + NW * CT * 1024;
    static constexpr int LDS = MERGE_LDS > LOOP_LDS ? MERGE_LDS : LOOP_LDS;
    static_assert(LDS <= FQ_LDS_MAX, "LDS");
};

// V^T operands of four tiles of 16 dims from addresses a[i] (keys 8 g ..) and ROWS4 behind them (keys 8 g + 4 ..):
// one statement with its wait, as fq_read_tr.
template <int ROWS4>
__device__ __forceinline__ void fp_read_tr(const uint32_t (&a)[4], fq_v2i (&w)[8]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n"
                 "ds_read_b64_tr_b16 %1, %8 offset:%13\n"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n"
                 "ds_read_b64_tr_b16 %3, %9 offset:%13\n"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n"
                 "ds_read_b64_tr_b16 %5, %10 offset:%13\n"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n"
                 "ds_read_b64_tr_b16 %7, %11 offset:%13\n"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(w[4]), "=&v"(w[5]), "=&v"(w[6]), "=&v"(w[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(0), "n"(ROWS4)
                 : "memory");
}

// Bits of the halves of x that are not finite: 0x8000 of each.
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) { return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

template <int DK, int DV, int NQ, int NW, int WPE, bool QF32>
__global__ void __launch_bounds__((NW * WAVE)) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) fa_pf16_kernel(FaPArgs a) {
    using C = FpCfg<DK, DV, NQ, NW>;
    extern __shared__ __align__(16) uint8_t smem[];
    asm volatile("" ::"s"(a.q), "s"(a.k.nb3), "s"(a.v.nb2), "s"(a.dst), "s"(a.dst_nb3), "s"(a.T), "s"(a.div_split.mul), "s"(a.softcap), "s"(a.st.table),
                 "s"(a.st.parent_nb), "s"(a.div_tpp.mul));   // all lines of the arguments at once
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int r = lane % 16, g = lane / 16;

    // block -> (sequence, split, KV head, query rows), as fa_q_kernel
    int b = xcd_tile(blockIdx.x, gridDim.x), b1 = fq_div(b, a.div_nrt);
    const int rt = b - b1 * a.nrt;
    b = b1;
    b1 = fq_div(b, a.div_hk);
    const int hk = b - b1 * a.HK, s = fq_div(b1, a.div_split), split = b1 - s * a.nsplit;
    const StepOf sq = step_of(a.st, s);
    const int n_past = sq.past, n_new = sq.fresh;
    if (sq.bad && threadIdx.x == 0 && a.st.err) *a.st.err = 1;
    const int tok_a = fq_div(rt * 16 * NQ, a.div_g), tok_b = fq_div(min(a.R, (rt + 1) * 16 * NQ) - 1, a.div_g);
    const int seen = a.st.parent ? n_new : min(n_new, tok_b + 1);
    const int keys = tok_a < n_new ? min(n_past + seen, a.st.cap) : 0;
    const int up = a.st.parent && lane < a.T ? a.st.parent[(int64_t)s * a.st.parent_nb + lane] : -1;
    const int ntiles = (keys + FQ_KEYS - 1) / FQ_KEYS, per = (ntiles + a.nsplit - 1) / a.nsplit;
    const int tile0 = split * per, tile1 = min(ntiles, tile0 + per), tile_end = max(ntiles, 1) - 1;

    // Q in the B layout of the Q.K products: lane (row r, dims 8 g + 0..7 of a block of 32); past dk zeros. QF32: F32, two halves
    bool ok[NQ];
    int tok[NQ];
    int64_t qat[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int row = (rt * NQ + n) * 16 + r;
        ok[n] = row < a.R;
        tok[n] = ok[n] ? fq_div(row, a.div_g) : 0;
        const int head = hk * a.G + (ok[n] ? row - tok[n] * a.G : 0);
        qat[n] = (int64_t)s * a.q_nb3 + (int64_t)head * a.q_nb2 + (int64_t)tok[n] * a.q_nb1 + 8 * g;
    }
    u32x4 qraw[NQ][C::KS][2];   // eight values each: F32, or F16 in the first
    if constexpr (!QF32) {
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int st = 0; st < C::KS; st++) {
                qraw[n][st][0] = *(const u32x4 *)((const uint16_t *)a.q + qat[n] + (32 * st < a.dk ? 32 * st : 0));
                qraw[n][st][1] = u32x4{0, 0, 0, 0};
            }
    } else {
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int st = 0; st < C::KS; st++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    qraw[n][st][h] = *(const u32x4 *)((const float *)a.q + qat[n] + (32 * st < a.dk ? 32 * st : 0) + 4 * h);
    }

    const uint16_t * const kq = (const uint16_t *)a.k.q + (int64_t)hk * a.k.nb2;
    const uint16_t * const vq = (const uint16_t *)a.v.q + (int64_t)hk * a.v.nb2;
    // this lane's chunk of each DMA instruction: byte offset from the tile's first row; chunks past dk or dv the first ones
    uint32_t kdma[C::KD], vdma[C::VD];
#pragma unroll
    for (int q = 0; q < C::KD; q++) {
        const int slot = q * WAVE + lane, row = slot / C::KCH, c = (slot % C::KCH) ^ C::kswz(row);
        const uint32_t key = row % 16 / 4 * 8 + row / 16 * 4 + row % 4;   // K rows lie in the order 16 h + 4 g + e (key 8 g + 4 h + e)
        kdma[q] = key * 2 * (uint32_t)a.k.nb1 + (c * 8 < a.dk ? 16 * c : 0);
    }
#pragma unroll
    for (int q = 0; q < C::VD; q++) {
        const int slot = q * WAVE + lane, key = slot / C::VCH, c = (slot % C::VCH) ^ (2 * C::vswz(key));
        vdma[q] = key * 2 * (uint32_t)a.v.nb1 + (c * 8 < a.dv ? 16 * c : 0);
    }
    uint8_t * const wl = smem + wave * C::STAGE;
    // where this lane reads: chunk 4 i + g of K row r (i: kra ^ 64 i), 4 dims of V row 8 g + r / 4 (tile of 16 dims i: vra ^ 32 i)
    const uint32_t kra = r * C::KCH * 16 + ((g ^ C::kswz(r)) << 4);
    const int vrow = 8 * g + r / 4;
    const uint32_t vra = (uint32_t)(uintptr_t)(fq_lptr_t)wl + C::K_BYTES + vrow * C::VRB + (((r % 4 / 2) ^ (2 * C::vswz(vrow))) << 4) + 8 * (r % 2);

    auto page_of = [&](int t) -> int64_t {   // the row where tile t begins, -1 for a tile of a page that the cache does not have
        const int p = fq_div(t, a.div_tpp);
        const int64_t row = page_row(a.st, uniform_i32(a.st.table, (int64_t)s * a.st.table_nb + p));
        return row < 0 ? -1 : row + FQ_KEYS * (t - p * a.div_tpp.d);
    };
    auto dma_k = [&](int64_t row) {
        const __amdgpu_buffer_rsrc_t kt = fq_rsrc(kq + max(row, (int64_t)0) * a.k.nb1);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int q = 0; q < C::KD; q++) fq_dma16(kt, kdma[q], wl + q * 1024);
        asm volatile("" ::: "memory");
    };
    auto dma_v = [&](int64_t row) {
        const __amdgpu_buffer_rsrc_t vt = fq_rsrc(vq + max(row, (int64_t)0) * a.v.nb1);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int q = 0; q < C::VD; q++) fq_dma16(vt, vdma[q], wl + C::K_BYTES + q * 1024);
        asm volatile("" ::: "memory");
    };
    // The wave's tiles are tile0 + wave + NW k, k < nk. Waves without a tile read one all
    // the same, and behind the last the last again: the loads in flight stay what the waits count.
    const int nk = tile1 - tile0 > wave ? (tile1 - tile0 - wave + NW - 1) / NW : 0;
    int t = min(tile0 + wave, tile_end);
    int64_t row_t = page_of(t), row_n = page_of(min(t + NW, tile_end));
    dma_k(row_t);
    dma_v(row_t);

    // Q in halves; an F32 row times the power of two that brings its largest value to [2^14, 2^15) (at most 2^111), so that its low halves
    // keep their bits; the scale takes it back
    half8 qf[NQ][C::KS];
    half8 * const ql = (half8 *)(smem + C::Q_LO);
    float sfac[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        float amax = 0.0f;
        auto value = [&](int st, int e) {
            const float x = !QF32 ? h2f_bits((uint16_t)(qraw[n][st][0][e / 2] >> (16 * (e % 2)))) : __uint_as_float(qraw[n][st][e / 4][e % 4]);
            return ok[n] && 32 * st < a.dk ? x : 0.0f;
        };
#pragma unroll
        for (int st = 0; st < C::KS; st++)
#pragma unroll
            for (int e = 0; e < 8; e++) amax = fmaxf(amax, fabsf(value(st, e)));
        amax = fq_col_max(amax);
        const uint32_t e2 = QF32 ? max((int)(__float_as_uint(amax) >> 23) - 14, 16) : 127;
        const float qfac = __uint_as_float(e2 << 23), inv = __uint_as_float((254u - e2) << 23);
        sfac[n] = a.scale * qfac;
#pragma unroll
        for (int st = 0; st < C::KS; st++) {
            half8 lo;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = value(st, e) * inv;
                qf[n][st][e] = (_Float16)x;
                lo[e] = (_Float16)(x - (float)qf[n][st][e]);
            }
            if (QF32 && wave == 0) ql[(n * C::KS + st) * WAVE + lane] = lo;
        }
    }
    // a barrier for LDS alone: the first tiles' loads stay in flight
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int lim[NQ];
    uint64_t anc[NQ];
    const int full_to = fp_sees<NQ>(a, lane, rt, up, n_past, n_new, tok_a, ok, lim, anc);

    float4v o[NQ][C::TT];
    float m_run[NQ], l_run[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m_run[n] = -INFINITY;
        l_run[n] = 0.0f;
#pragma unroll
        for (int q = 0; q < C::TT; q++) o[n][q] = float4v{0, 0, 0, 0};
    }
    const half2v one2 = {(_Float16)1.0f, (_Float16)1.0f};
    const float cap2 = a.softcap != 0.0f ? 2.0f * FQ_LOG2E / a.softcap : 0.0f;

    for (int k = 0; k < nk; k++) {
        fq_wait_vm<C::VD>();   // K has landed
        float4v sc[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++) sc[n][0] = sc[n][1] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < C::KS; i++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++) {
                const half8 kf = *(const half8 *)(wl + (kra ^ (uint32_t)(64 * i)) + hf * 256 * C::KCH);
#pragma unroll
                for (int n = 0; n < NQ; n++) sc[n][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[n][i], sc[n][hf], 0, 0, 0);
                if constexpr (QF32)
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        sc[n][hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[(n * C::KS + i) * WAVE + lane], sc[n][hf], 0, 0, 0);
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        dma_k(row_n);
        const bool masked = FQ_KEYS * (t + 1) > full_to || row_t < 0;
        uint32_t vis[NQ];   // masked: which of this lane's eight keys row n sees
        u32x4 pf[NQ];       // P, fp16
        if (masked && row_t < 0 && a.st.err) *a.st.err = 1;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[n][hf][e] *= sfac[n];
            if (a.softcap != 0.0f) {
                // cap * tanh(s / cap) = cap - 2 cap / (1 + exp(2 s / cap)): off by some 1e-7 of cap
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        sc[n][hf][e] = fmaf(-2.0f * a.softcap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(sc[n][hf][e] * cap2)), a.softcap);
            }
            vis[n] = 0xFFu;
            if (masked) {
                vis[n] = row_t < 0 ? 0 : fp_visible(FQ_KEYS * t + 8 * g, n_past, lim[n], anc[n]);
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (!((vis[n] >> (4 * hf + e)) & 1u)) sc[n][hf][e] = -INFINITY;   // a hidden score may be NaN
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
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float s0 = sc[n][e / 2][2 * (e % 2)], s1 = sc[n][e / 2][2 * (e % 2) + 1];
                pf[n][e] = pack2h(__builtin_amdgcn_exp2f(fmaf(s0, FQ_LOG2E, -mb)), __builtin_amdgcn_exp2f(fmaf(s1, FQ_LOG2E, -mb)));
                l_run[n] = __builtin_amdgcn_fdot2(h2_of(pf[n][e]), one2, l_run[n], false);   // the sum of what is multiplied
            }
        }
        fq_wait_vm<C::KD>();   // V has landed
        // ---- O^T += V^T . P^T; shut: all bits of the halves of keys hidden from some row ----
        auto pv = [&](auto some, const u32x4 & shut, uint32_t & bad) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < C::TT; q += 4) {
                uint32_t va[4];
                fq_v2i w[8];
#pragma unroll
                for (int i = 0; i < 4; i++) va[i] = vra ^ (uint32_t)(32 * (q + i));
                fp_read_tr<4 * C::VRB>(va, w);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    u32x4 x = {(uint32_t)w[2 * i][0], (uint32_t)w[2 * i][1], (uint32_t)w[2 * i + 1][0], (uint32_t)w[2 * i + 1][1]};
                    if constexpr (decltype(some)::value) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t nf = not_finite2(x[e]) & shut[e];
                            x[e] &= ~((nf >> 15) * 0xFFFFu);
                            bad |= ((nf >> 15 & 1u) | (nf >> 30 & 2u)) << (2 * e);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NQ; n++)
                        o[n][q + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, pf[n]), o[n][q + i], 0, 0, 0);
                }
            }
        };
        uint32_t bad = 0;   // of this lane's keys: shut ones with a value that is not finite
        if (!masked) {
            pv(std::false_type{}, u32x4{0, 0, 0, 0}, bad);
        } else {
            uint32_t hidden = 0;
            u32x4 shut = {0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NQ; n++) hidden |= ok[n] ? ~vis[n] & 0xFFu : 0u;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint64_t rows = __ballot((hidden >> e) & 1u);
                if ((rows >> (16 * g)) & 0xFFFFu) shut[e / 2] |= 0xFFFFu << (16 * (e % 2));
            }
            pv(std::true_type{}, shut, bad);
            if (__any(bad != 0)) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const uint64_t dims = __ballot((bad >> e) & 1u);
                    if ((dims >> (16 * g)) & 0xFFFFu)
#pragma unroll
                        for (int n = 0; n < NQ; n++)
                            if ((vis[n] >> e) & 1u) l_run[n] = NAN;
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        dma_v(row_n);
        t += NW;
        row_t = row_n;
        row_n = page_of(min(t + NW, tile_end));
    }
    fq_wait_vm<0>();   // no DMA may still write what the merge reuses

    // ---- merge the block's waves, as fa_q_kernel ----
    float * const sml = (float *)smem;                           // [NW][16 NQ][2]: (max, sum)
    float4v * const so = (float4v *)(smem + NW * 16 * NQ * 8);   // [NW][CT][64]
    __syncthreads();
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
            so[(wave * C::CT + i) * WAVE + lane] = o[n][q] * wgt[n];
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

template <int DK, int DV, int NQ, int NW, int WPE, bool QF32>
static hipError_t fp_launch_q(const FaPArgs & a, hipStream_t st) {
    using C = FpCfg<DK, DV, NQ, NW>;
    static LdsAllowed done;
    const hipError_t l = allow_lds((const void *)fa_pf16_kernel<DK, DV, NQ, NW, WPE, QF32>, C::LDS, done);
    if (l != hipSuccess) return l;
    const int64_t units = (int64_t)a.S * a.HK * a.nrt;
    hipLaunchKernelGGL((fa_pf16_kernel<DK, DV, NQ, NW, WPE, QF32>), dim3((unsigned)(units * a.nsplit)), dim3(NW * WAVE), C::LDS, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    return launch_fa_q_combine(a, DV, NQ, st);
}

template <int DK, int DV, int NQ, int NW, int WPE>
static hipError_t fp_launch(const FaPArgs & a, hipStream_t st) {
    return a.q_f16 ? fp_launch_q<DK, DV, NQ, NW, WPE, false>(a, st) : fp_launch_q<DK, DV, NQ, NW, WPE, true>(a, st);
}

hipError_t launch_fa_p_F16(const FaPArgs & a, hipStream_t st) {
    if (a.D == 64 && a.DV == 64) return a.nq == 2 ? fp_launch<64, 64, 2, 4, 3>(a, st) : fp_launch<64, 64, 1, 4, 4>(a, st);
    if (a.D == 128 && a.DV == 128) return a.nq == 2 ? fp_launch<128, 128, 2, 4, 2>(a, st) : fp_launch<128, 128, 1, 4, 2>(a, st);
    if (a.D == 192 && a.DV == 128) return a.nq == 2 ? fp_launch<192, 128, 2, 4, 1>(a, st) : fp_launch<192, 128, 1, 4, 1>(a, st);
    if (a.nq == 1 && a.D == 256 && a.DV == 256) return fp_launch<256, 256, 1, 4, 1>(a, st);
    return hipErrorInvalidValue;
}

}  // namespace mx
