// SPDX-License-Identifier: MIT
// A KV cache in pages: new tokens' keys and values stored at their sequences' ends, with the position rotation
// of keys and queries, and accepted drafts moved to where the sequence goes on.
//
// Token t of sequence s has logical row j = n_past[s] + t, cache row table[s][j / page] * page + j % page and position
// p = n_past[s] + depth(t) (or a given one). Its keys and queries are rotated in pairs (a, b) of dims, pair i by
//   theta = p freq[i] in 64 bits,  c = f32(m cos theta),  s = f32(m sin theta)
//   a' = f32(f32(a c) - f32(b s)),  b' = f32(f32(a s) + f32(b c))
// every step rounded on its own, so the codes made of them are the definition's bits: an angle in 32 bits is off by
// 2^-24 of itself, 0.004 rad at position 65536, half a step of 8 bits and more.
//
// Append reads every value once and writes rows and queries: HBM bounds many tokens, latency a few. The sines are taken once
// a token and pair, not once a head, by the workgroup whose heads share them. Blocks of 32 are the work of a quad, as in
// mx_kv.hip.

#include <algorithm>

#include "mx_common.h"
#include "mx_fa_prep.h"
#include "mx_kernels_impl.h"
#include "mx_kv_rows.h"
#include "mx_pages.h"

namespace mx {

constexpr int AP_THREADS = 256;
constexpr int AP_BLOCKS = AP_THREADS / 4;   // quads
constexpr int AP_TOK = 16;                  // tokens a workgroup
constexpr int AP_HALF = 128;                // pairs at most (head dim 256)

// A lane's eight values, two runs of four: the first at `at`, the second `apart` values on (wide: 4, one 16-byte piece of F16).
__device__ __forceinline__ void ap_load8(const KvPlainRows & x, int64_t at, bool wide, u32x4 (&raw)[2]) {
    if (!x.f16) {
        const float * p = (const float *)x.x + at;
        raw[0] = *(const u32x4 *)p;
        raw[1] = *(const u32x4 *)(p + (wide ? 4 : 16));
    } else if (wide) {
        raw[0] = *(const u32x4 *)((const uint16_t *)x.x + at);
    } else {
        const uint16_t * p = (const uint16_t *)x.x + at;
        const u32x2 lo = *(const u32x2 *)p, hi = *(const u32x2 *)(p + 16);
        raw[0] = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
}
__device__ __forceinline__ float ap_value(bool f16, const u32x4 (&raw)[2], int e) {
    return f16 ? h2f_bits((uint16_t)(raw[0][e / 2] >> (16 * (e % 2)))) : __uint_as_float(raw[e / 4][e % 4]);
}

// Sine and cosine of x, |x| < 2^40, off by some 2^-53: x less a multiple k of pi / 2, whose three parts take 159 bits of it, then
// the Taylor series up to x^17 and x^18 (|r| <= pi / 4: the next terms are below 1e-19). The library's sincos also
// takes arguments of any size, with 60 registers, which left room for half as many workgroups.
__device__ __forceinline__ void ap_sincos(double x, double & sn, double & cn) {
    const double k = rint(x * 0.6366197723675814);
    const double r = fma(-k, -1.4973849048591698e-33, fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, x))), z = r * r;
    double s = 1.0 / 355687428096000.0, c = -1.0 / 6402373705728000.0;   // 17!, 18!
    s = fma(s, z, -1.0 / 1307674368000.0);
    c = fma(c, z, 1.0 / 20922789888000.0);
    s = fma(s, z, 1.0 / 6227020800.0);
    c = fma(c, z, -1.0 / 87178291200.0);
    s = fma(s, z, -1.0 / 39916800.0);
    c = fma(c, z, 1.0 / 479001600.0);
    s = fma(s, z, 1.0 / 362880.0);
    c = fma(c, z, -1.0 / 3628800.0);
    s = fma(s, z, -1.0 / 5040.0);
    c = fma(c, z, 1.0 / 40320.0);
    s = fma(s, z, 1.0 / 120.0);
    c = fma(c, z, -1.0 / 720.0);
    s = fma(s, z, -1.0 / 6.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    s = fma(s, z * r, r);
    c = fma(c, z, 1.0);
    const int q = (int)(int64_t)k & 3;   // sin(r + q pi / 2)
    const double a = q & 1 ? c : s, b = q & 1 ? s : c;
    sn = q & 2 ? -a : a;
    cn = (q + 1) & 2 ? -b : b;
}

// A workgroup takes tok_wg tokens of a sequence, one after the other, or one of `parts` of a token's blocks, of K, of V or of
// Q. A quad stays at its place of the row, block b of head h, and goes from token to token, the next block on its way
// meanwhile. Where nothing is quantized lane l takes values 8 l .. 8 l + 7 of a block, else 4 l .. and 16 + 4 l ..
// (kv_quantize). 4091 tokens of 32 + 8 + 8 heads x 128, all F16 (101 MB) 29.6 us, from F32 into Q8_0 (185 MB) 44 us, 4.2 TB/s; a
// single token 5.3 us, its chain of loads (lengths, table) and the barriers. A wave waits 0.7 of its time, for that chain
// most of all: with at most eight tokens a workgroup 30.1 and 47 us, with four blocks a thread requested at once 33.
// A row that a later token (of this sequence or the next ones) has too, because tables share a page where they are
// written, is left to the last of them, so that it is whole: every workgroup of K and V looks at the pages that the
// step writes behind its own.
template <bool NEOX>
__global__ void __launch_bounds__(AP_THREADS) kv_append_kernel(KvAppendArgs a) {
    __shared__ float cs[AP_TOK][AP_HALF][2];
    __shared__ int64_t at_row[AP_TOK];   // element offset of the token's row
    __shared__ int pos[AP_TOK], entry[AP_TOK], off[AP_TOK], dead[AP_TOK];   // dead: 1 its row is not written, 2 nor its query
    const int t = threadIdx.x, l = t % 4;
    int what = 0;
    while (what + 1 < a.n_rows && (int)blockIdx.x >= a.r[what + 1].wg_begin) what++;
    const KvAppendRows & r = a.r[what];
    const int wg = (int)blockIdx.x - r.wg_begin, grp = fq_div(wg, r.div_parts), part = wg - grp * r.parts;
    const int s = fq_div(grp, r.div_groups), t0 = (grp - s * r.groups) * r.tok_wg;
    const int end = min(r.items, (part + 1) * r.per);
    const int rotated = r.rotate ? 2 * a.half : 0;
    const bool wide = r.wide, x_f16 = r.x.f16;
    const int run0 = wide ? 8 * l : 4 * l, apart = wide ? 4 : 16;   // this lane's two runs of four values of a block
    // quad -> (token of the first few, place in the row); places go on by `across`, tokens by `down`
    const int across = min(r.per, AP_BLOCKS), down = r.down, quad = t / 4;
    const int tok0 = fq_div(quad, r.div_across), hb0 = part * r.per + quad - tok0 * across;
    struct At {
        int hb, tok, j;   // j: this lane's first dim of its head
        int64_t x, o;     // element offset of its value in the source of token t0, and in a row of the destination
    };
    const KvPlainRows & xr = r.x;
    const int64_t o_nb2 = what == 2 ? a.qr.nb2 : a.o[what].nb2;
    auto place = [&](int hb, int tok) {
        const int h = fq_div(hb, r.div_bph), j = 32 * (hb - h * r.bph) + run0;
        return At{hb, tok, j, (int64_t)s * xr.nb3 + (int64_t)t0 * xr.nb1 + (int64_t)h * xr.nb2 + j, (int64_t)h * o_nb2 + j};
    };
    u32x4 v[2], w[2];   // a block's values and those they are paired with
    auto load = [&](const At & p) {
        const int64_t at = p.x + p.tok * xr.nb1;
        ap_load8(xr, at, wide, v);
        if constexpr (NEOX) {
            if (wide) {   // half is a multiple of 8
                if (p.j < rotated) ap_load8(xr, at + (p.j < a.half ? a.half : -a.half), true, w);
            } else {
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const int j = p.j + 16 * g;
                    if (j >= rotated) continue;
                    const int64_t from = at + 16 * g + (j < a.half ? a.half : -a.half);
                    if (x_f16) {
                        const u32x2 y = *(const u32x2 *)((const uint16_t *)xr.x + from);
                        w[0][2 * g] = y[0];
                        w[0][2 * g + 1] = y[1];
                    } else {
                        w[g] = *(const u32x4 *)((const float *)xr.x + from);
                    }
                }
            }
        }
    };
    At p = place(hb0, tok0);
    // quads left over have nothing to do; padding's sources are there to be read
    if (tok0 < down && hb0 < end && tok0 < min(r.tok_wg, a.count - t0)) load(p);

    const StepOf sq = step_of(a.st, s);
    const int toks = min(r.tok_wg, min(sq.fresh - a.first, a.count) - t0);
    if (sq.bad && t == 0 && t0 == 0 && a.st.err) *a.st.err = 1;
    if (toks <= 0) return;
    // page k of those that this launch writes for sequence s2, rows [p0, p0 + n2) of it: the page's first row and its entry, or -1 for none
    struct Later {
        int s2, first, p0, n2, e;
    };
    auto later = [&](int i) {
        Later x = {0, 0, 0, 0, -1};
        if (what == 2 || i >= a.st.S * a.span) return x;
        x.s2 = fq_div(i, a.div_span);
        const int past = a.st.n_past[x.s2];
        x.n2 = min((a.st.n_new ? min(a.st.n_new[x.s2], a.st.T) : a.st.T) - a.first, a.count);
        if (past < 0 || past > a.st.cap || x.n2 <= 0) return x;
        x.p0 = past + a.first;
        const int pi = fq_div(x.p0, a.st.div_page) + i - x.s2 * a.span;
        x.first = pi * a.st.page;
        if (pi < a.st.n_table && x.first - x.p0 < x.n2) x.e = a.st.table[(int64_t)x.s2 * a.st.table_nb + pi];
        return x;
    };
    // whether token i of sequence s2 is one of a chain, or has a way up the tree's parents
    auto stored = [&](int s2, int i) {
        while (a.st.parent && i >= 0) {
            const int up = a.st.parent[(int64_t)s2 * a.st.parent_nb + i];
            i = up < i ? up : -2;
        }
        return i >= -1;
    };
    Later next = later(s * a.span + t);
    // ---- rows and positions of the tokens ----
    if (t < WAVE) {
        int depth = a.first + t0 + t;
        if (a.st.parent) {   // at most 64 tokens: first is 0
            const uint64_t anc = tree_ancestors(t < a.st.T ? a.st.parent[(int64_t)s * a.st.parent_nb + t] : -1, t);
            depth = __shfl(__popcll(anc) - 1, t0 + t, WAVE);
        }
        if (t < toks) {
            const int j = sq.past + a.first + t0 + t, pi = fq_div(j, a.st.div_page);
            const int e = pi < a.st.n_table ? a.st.table[(int64_t)s * a.st.table_nb + pi] : -1;
            const int64_t row = page_row(a.st, e);
            entry[t] = e;
            off[t] = j - pi * a.st.page;
            at_row[t] = what < 2 ? (row + off[t]) * a.o[what].nb1 : (int64_t)s * a.qr.nb3 + (int64_t)(t0 + t) * a.qr.nb1;
            pos[t] = a.pos ? a.pos[(int64_t)s * a.pos_nb + t0 + t] : sq.past + depth;
            dead[t] = depth < 0 ? 2 : row < 0 ? 1 : 0;
            if (dead[t] && a.st.err) *a.st.err = 1;
        }
    }
    __syncthreads();
    // ---- the sines, and the later owners of the rows ----
    for (int i = t; i < toks * (rotated / 2); i += AP_THREADS) {
        const int tok = fq_div(i, a.div_half), p = i - tok * a.half;
        double sn, c;
        ap_sincos((double)pos[tok] * (double)a.freq[p], sn, c);
        cs[tok][p][0] = (float)(c * (double)a.mscale);
        cs[tok][p][1] = (float)(sn * (double)a.mscale);
    }
    for (int i = s * a.span + t; what < 2 && i < a.st.S * a.span; i += AP_THREADS) {
        const Later x = next;
        next = later(i + AP_THREADS);
        for (int u = 0; u < toks; u++) {
            const int j = x.first + off[u];   // the row of s2 that token u's is
            if (x.e >= 0 && x.e == entry[u] && j >= x.p0 && j - x.p0 < x.n2 && (x.s2 > s || j > sq.past + a.first + t0 + u) && stored(x.s2, j - x.p0)) dead[u] |= 1;
        }
    }
    __syncthreads();
    // ---- blocks ----
    if (tok0 >= down || tok0 >= toks) return;
    while (p.hb < end) {
        const At c = p;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = ap_value(x_f16, v, e);
        float z[8];
        if constexpr (NEOX) {
#pragma unroll
            for (int e = 0; e < 8; e++) z[e] = ap_value(x_f16, w, e);
        }
        p.tok += down;
        if (p.tok >= toks) p = place(p.hb + across, tok0);
        if (p.hb < end) load(p);
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const int j = c.j + g * apart;
            if (j >= rotated) continue;
            if constexpr (NEOX) {
                const bool second = j >= a.half;
                const float * k = cs[c.tok][second ? j - a.half : j];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = mul_rn(y[4 * g + e], k[2 * e]), q = mul_rn(z[4 * g + e], k[2 * e + 1]);
                    y[4 * g + e] = sub_rn(x, second ? -q : q);
                }
            } else {
                const float * k = cs[c.tok][j / 2];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float x0 = y[4 * g + e], x1 = y[4 * g + e + 1];
                    y[4 * g + e] = sub_rn(mul_rn(x0, k[e]), mul_rn(x1, k[e + 1]));
                    y[4 * g + e + 1] = sub_rn(mul_rn(x0, k[e + 1]), -mul_rn(x1, k[e]));
                }
            }
        }
        const int64_t at = at_row[c.tok] + c.o;
        if (what == 2) {
            if (dead[c.tok] >= 2) continue;
            if (a.qr.f16) {
                uint16_t * to = (uint16_t *)a.qr.x + at;
                const u32x4 q = kv_pack8(y);
                if (wide) {
                    *(u32x4 *)to = q;
                } else {
                    *(u32x2 *)to = u32x2{q[0], q[1]};
                    *(u32x2 *)(to + 16) = u32x2{q[2], q[3]};
                }
            } else {
                float * to = (float *)a.qr.x + at;
                *(float4v *)to = float4v{y[0], y[1], y[2], y[3]};
                *(float4v *)(to + apart) = float4v{y[4], y[5], y[6], y[7]};
            }
        } else if (!dead[c.tok]) {   // the same for the quad
            const KvRowsOut & o = a.o[what];
            if (wide) *(u32x4 *)((uint16_t *)o.q + at) = kv_pack8(y);
            else kv_quantize(o, at - run0, l, y);
        }
    }
}

// A block a quad while that makes fewer than 2048 workgroups, then more: up to AP_TOK whole tokens a workgroup.
static hipError_t append_launch(KvAppendArgs a, hipStream_t st) {
    int64_t all = 0, wgs = 0;
    for (int k = 0; k < a.n_rows; k++) all += (int64_t)a.st.S * a.count * a.r[k].H * a.r[k].bph;
    const int64_t most = std::max<int64_t>(AP_BLOCKS, all / 2048);
    for (int k = 0; k < a.n_rows; k++) {
        KvAppendRows & r = a.r[k];
        r.items = r.H * r.bph;
        r.tok_wg = (int)std::min<int64_t>({std::max<int64_t>(1, most / r.items), AP_TOK, a.count});
        r.parts = most >= r.items ? 1 : (int)((r.items + most - 1) / most);
        r.per = (r.items + r.parts - 1) / r.parts;
        r.groups = (a.count + r.tok_wg - 1) / r.tok_wg;
        r.down = std::max(1, AP_BLOCKS / r.per);
        r.wide = (k == 2 || a.o[k].type == T_F16) && (!r.rotate || !a.neox || a.half % 8 == 0);
        r.wg_begin = (int)wgs;
        wgs += (int64_t)a.st.S * r.groups * r.parts;
        r.div_bph = fq_div_by(r.bph); r.div_parts = fq_div_by(r.parts); r.div_groups = fq_div_by(r.groups);
        r.div_across = fq_div_by(std::min(r.per, AP_BLOCKS));
    }
    a.div_half = fq_div_by(std::max(1, a.half));
    a.div_span = fq_div_by(a.span);
    if (a.neox) hipLaunchKernelGGL(kv_append_kernel<true>, dim3((unsigned)wgs), dim3(AP_THREADS), 0, st, a);
    else hipLaunchKernelGGL(kv_append_kernel<false>, dim3((unsigned)wgs), dim3(AP_THREADS), 0, st, a);
    return hipGetLastError();
}

static void advance(KvPlainRows & x, int64_t s, int64_t t) { x.x = (uint8_t *)x.x + (s * x.nb3 + t * x.nb1) * (x.f16 ? 2 : 4); }

// A launch takes AP_TOKENS tokens of a sequence at most, or sequences that write AP_PAGES pages at most, the next ones a next
// launch, where a row that is named again comes later by itself: what its workgroups look through for later owners grows
// with the square of a launch.
constexpr int AP_TOKENS = 1 << 16, AP_PAGES = 2048;
hipError_t launch_kv_append(KvAppendArgs a, hipStream_t st) {
    const int S = a.st.S, T = a.st.T, count = std::min(T, AP_TOKENS);
    a.span = (count + a.st.page - 2) / a.st.page + 1;   // pages that a sequence's rows may touch
    const int many = count < T ? 1 : std::max(1, AP_PAGES / a.span);
    for (int s = 0; s < S; s += many)
        for (int t = 0; t < T; t += count) {
            KvAppendArgs b = a;
            b.st.S = std::min(many, S - s);
            b.first = t;
            b.count = std::min(count, T - t);
            b.st.table += s * a.st.table_nb;
            b.st.n_past += s;
            if (a.st.n_new) b.st.n_new += s;
            if (a.st.parent) b.st.parent += s * a.st.parent_nb;
            if (a.pos) b.pos += s * a.pos_nb + t;
            for (int k = 0; k < a.n_rows; k++) advance(b.r[k].x, s, t);
            if (a.n_rows > 2) advance(b.qr, s, t);
            const hipError_t e = append_launch(b, st);
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

// A thread moves one block of 32 values and its scale, row after row. Source path[i] lies at or behind
// destination i and behind every earlier source, so in that order no row is read after it was written: what is read for
// i' > i lies behind i. KEEP_ILP rows are read before the first of them is written.
constexpr int KEEP_ILP = 4;
__global__ void __launch_bounds__(AP_THREADS) kv_keep_kernel(KvKeepArgs a) {
    __shared__ int64_t from[KV_TREE_MAX], to[KV_TREE_MAX];
    __shared__ int no;
    const int t = threadIdx.x, s = blockIdx.x / a.wgs, wg = blockIdx.x % a.wgs;
    const KvRowsOut & o = a.o[blockIdx.y];
    const StepOf sq = step_of(a.st, s);
    const int n = a.n_keep ? uniform_i32(a.n_keep, s) : a.A;
    if (t == 0) no = sq.bad || n < 0 || n > a.A;
    __syncthreads();
    if (t < KV_TREE_MAX && t < min(n, a.A)) {
        const int32_t * path = a.path + (int64_t)s * a.path_nb;
        const int p = path[t], before = t ? path[t - 1] : -1;
        bool ok = p >= t && p > before && p < sq.fresh;
        if (ok) {
            const int js = sq.past + p, jd = sq.past + t, ps = fq_div(js, a.st.div_page), pd = fq_div(jd, a.st.div_page);
            const int32_t * table = a.st.table + (int64_t)s * a.st.table_nb;
            const int64_t rs = ps < a.st.n_table ? page_row(a.st, table[ps]) : -1, rd = pd < a.st.n_table ? page_row(a.st, table[pd]) : -1;
            ok = rs >= 0 && rd >= 0;
            from[t] = rs + js - ps * a.st.page;
            to[t] = rd + jd - pd * a.st.page;
        }
        if (!ok) no = 1;
    }
    __syncthreads();
    if (no) {
        if (t == 0 && a.st.err) *a.st.err = 1;
        return;
    }
    const int hb = wg * AP_THREADS + t;
    if (hb >= o.div_bpr.d) return;
    const int h = fq_div(hb, o.div_bph), b = hb - h * o.bph;
    const int64_t at = (int64_t)h * o.nb2 + 32 * b;
    const int shift = o.type == T_F16 ? -1 : o.type == T_Q4_0;   // elements to bytes
    const int pieces = o.type == T_F16 ? 4 : o.type == T_Q8_0 ? 2 : 1;
    auto bytes = [&](int64_t e) { return shift < 0 ? 2 * e : e >> shift; };
    for (int i0 = 0; i0 < n; i0 += KEEP_ILP) {
        u32x4 x[KEEP_ILP][4];
        uint16_t d[KEEP_ILP];
#pragma unroll
        for (int u = 0; u < KEEP_ILP; u++) {
            if (i0 + u >= n) continue;
            const int64_t e = from[i0 + u] * o.nb1 + at;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c < pieces) x[u][c] = *(const u32x4 *)(o.q + bytes(e) + 16 * c);
            if (o.type != T_F16) d[u] = o.d[e / 32];
        }
#pragma unroll
        for (int u = 0; u < KEEP_ILP; u++) {
            if (i0 + u >= n || from[i0 + u] == to[i0 + u]) continue;
            const int64_t e = to[i0 + u] * o.nb1 + at;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c < pieces) *(u32x4 *)(o.q + bytes(e) + 16 * c) = x[u][c];
            if (o.type != T_F16) o.d[e / 32] = d[u];
        }
    }
}

hipError_t launch_kv_keep(KvKeepArgs a, hipStream_t st) {
    int bpr = 0;
    for (int k = 0; k < a.n_out; k++) {
        a.o[k].div_bpr = fq_div_by(a.o[k].H * a.o[k].bph);
        a.o[k].div_bph = fq_div_by(a.o[k].bph);
        bpr = std::max(bpr, a.o[k].div_bpr.d);
    }
    a.wgs = (bpr + AP_THREADS - 1) / AP_THREADS;
    const int S = a.st.S, many = std::max(1, (1 << 23) / a.wgs);   // threads of a launch below 2^32
    for (int s = 0; s < S; s += many) {
        KvKeepArgs b = a;
        b.st.S = std::min(many, S - s);
        b.st.table += s * a.st.table_nb;
        b.st.n_past += s;
        if (a.st.n_new) b.st.n_new += s;
        b.path += s * a.path_nb;
        if (a.n_keep) b.n_keep += s;
        hipLaunchKernelGGL(kv_keep_kernel, dim3((unsigned)(b.st.S * a.wgs), a.n_out), dim3(AP_THREADS), 0, st, b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// A sequence's rows out of their pages as fp16 for the fused attention (kv_decode_kernel has the values and what becomes of
// scales that are not finite), and its mask classes: token tq of f, the step's first + tq, sees the keys below n_past + first + tq + 1, padding none. Only
// tiles of which a token sees some keys and not all need a mask; it is written for those alone. Keys of the
// last tile of 64 behind the sequence's last and those of pages that the cache does not have are zeros.
__global__ void __launch_bounds__(AP_THREADS) kv_decode_paged_kernel(KvDecodeArgs a, FaArgs f, KvStepArgs st, int s, int first, uint16_t * mask) {
    const int t = threadIdx.x, l = t % 4;
    const StepOf sq = step_of(st, s);
    const int keys = sq.fresh ? min(sq.past + sq.fresh, st.cap) : 0;
    auto row_of = [&](int j) -> int64_t {
        const int p = fq_div(j, st.div_page);
        const int64_t r = p < st.n_table ? page_row(st, st.table[(int64_t)s * st.table_nb + p]) : -1;
        return r < 0 ? -1 : r + j - p * st.page;
    };
    if ((int)blockIdx.x < a.n_prep) {
        // a wave per (32 tokens, 64 keys): lane l has 32 of the keys for token l / 2
        if (blockIdx.x == 0 && t < 8) f.kzero[t] = 0;
        if (blockIdx.x == 0 && t == 0 && sq.bad && st.err) *st.err = 1;
        const int lane = t % WAVE, ct = (int)blockIdx.x * 4 + t / WAVE, nqt = (f.T + FA_QW - 1) / FA_QW;
        if (ct >= nqt * f.cls_stride) return;
        const int qt = ct / f.cls_stride, kt = ct - qt * f.cls_stride;
        const int tq = qt * FA_QW + lane / 2, jb = kt * FA_BKV + 32 * (lane % 2);
        int n = first + tq < sq.fresh && tq < f.T ? min(max(min(sq.past + first + tq + 1, keys) - jb, 0), 32) : 0;
        if (n > 0 && row_of(jb) < 0) {
            if (st.err) *st.err = 1;
            n = 0;
        }
        const bool any = __any(n > 0), all = __all(tq >= f.T || n == 32);
        if (lane == 0) f.cls[ct] = !any ? FA_TILE_SKIP : all ? FA_TILE_FULL : FA_TILE_MIXED;
        if (!any || all || tq >= f.T) return;
        u32x4 * m = (u32x4 *)(mask + (int64_t)tq * f.mask_nb1 + jb);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (8 * i + 2 * e < n ? 0u : 0xFC00u) | (8 * i + 2 * e + 1 < n ? 0u : 0xFC000000u);
            m[i] = w;
        }
        return;
    }
    const int kb = a.D / 32, vb = a.DV / 32;
    const int it = ((int)blockIdx.x - a.n_prep) * AP_BLOCKS + t / 4, kh = fq_div(it, a.div_blocks), b = it - kh * (kb + vb);
    const int j = fq_div(kh, a.div_hk), h = kh - j * a.HK;
    if (j >= min(a.KV, (keys + FA_BKV - 1) / FA_BKV * FA_BKV)) return;
    const bool is_v = b >= kb;
    const int blk = is_v ? b - kb : b;
    const int64_t row = j < keys ? row_of(j) : -1;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row >= 0) {
        const int64_t at = row * (is_v ? a.v.nb1 : a.k.nb1) + h * (is_v ? a.v.nb2 : a.k.nb2) + 32 * blk;
        const int type = is_v ? a.v.type : a.k.type;
        const u32x4 x = kv_codes(type, is_v ? a.v.q : a.k.q, at, l);
        const uint16_t d = (is_v ? a.v.d : a.k.d)[at / 32];
        const bool bad = (d & 0x7C00u) == 0x7C00u;
        bool poison = bad && !is_v;
        if (!is_v)   // a K block's quad looks at the V blocks blk, blk + kb, ...
            for (int i = blk; i < vb; i += kb) poison |= (a.v.d[(row * a.v.nb1 + h * a.v.nb2) / 32 + i] & 0x7C00u) == 0x7C00u;
        const float lim = kv_scale_limit(type);
        kv_values(type, x, bad ? 0.0f : fmaxf(fminf(h2f_bits(d), lim), -lim), l, v);
        if (poison) v[0] = NAN;
    }
    *(u32x4 *)((is_v ? a.v16 + (h * (int64_t)a.KV + j) * a.DV : a.k16 + (h * (int64_t)a.KV + j) * a.D) + 32 * blk + 8 * l) = kv_pack8(v);
}

hipError_t launch_kv_decode_paged(const KvDecodeArgs & args, const FaArgs & f, const KvStepArgs & st, int s, int first, uint16_t * mask, hipStream_t stream) {
    KvDecodeArgs a = args;
    a.div_blocks = fq_div_by((a.D + a.DV) / 32);
    a.div_hk = fq_div_by(a.HK);
    a.n_prep = fa_prep_blocks(f);
    const int64_t items = first ? 0 : (int64_t)a.KV * a.HK * ((a.D + a.DV) / 32);
    hipLaunchKernelGGL(kv_decode_paged_kernel, dim3((unsigned)(a.n_prep + (items + AP_BLOCKS - 1) / AP_BLOCKS)), dim3(AP_THREADS), 0, stream, a, f, st, s, first, mask);
    return hipGetLastError();
}

}  // namespace mx
