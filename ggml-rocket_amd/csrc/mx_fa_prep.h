// SPDX-License-Identifier: MIT
// The mask classes of the fused attention: one byte per 32-query x 64-key tile (every key masked, no key
// masked and no bias, or mixed), written before it by a launch of its own or by one that also does
// other work.
#pragma once

#include "mx_common.h"
#include "mx_kernels_impl.h"

namespace mx {

constexpr int FA_BKV = 64;      // keys per tile
constexpr int FA_QW = 32;       // query rows per wave task

enum : uint8_t { FA_TILE_SKIP = 0, FA_TILE_FULL = 1, FA_TILE_MIXED = 2 };

// Block b, of 256 threads, of fa_prep_blocks.
__device__ __forceinline__ void fa_prep_block(const FaArgs & a, int b) {
    const int t = threadIdx.x;
    const int nkt = a.kvp / FA_BKV;
    if (b == 0 && t < 8) a.kzero[t] = 0;   // the K and V source of the padded columns
    const int nqt = (a.T + FA_QW - 1) / FA_QW;
    const int nct = nqt * a.cls_stride;   // rows padded to cls_stride entries (padding: skip)
    const int cb = b;
    if (cb * 4 < nct) {
        // one wave per (query tile, key tile): lane l scans row l/2, keys 32*(l%2) .. +31
        const int wave = t / WAVE, lane = t % WAVE;
        const int ct = cb * 4 + wave;
        if (ct >= nct) return;
        const int qt = ct / a.cls_stride, kt = ct % a.cls_stride;
        bool vis = false, nz = false;
        if (kt >= nkt) {
            vis = false;                              // padding entry
        } else if (a.mask) {
            const int tq = qt * FA_QW + lane / 2;
            const int jb = kt * FA_BKV + 32 * (lane % 2);
            if (tq < a.T) {
                const uint16_t * mr = a.mask + (int64_t)tq * a.mask_nb1 + jb;
                if (jb + 32 <= a.KV) {
                    // 8 independent 8-byte loads (rows are 8-byte aligned)
                    u32x2 w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = *(const u32x2 *)(mr + 4 * i);
#pragma unroll
                    for (int i = 0; i < 8; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float m = h2f_bits((uint16_t)((w[i][e / 2] >> (16 * (e % 2))) & 0xFFFFu));
                            vis |= (m != -INFINITY);
                            nz |= (m != 0.0f);
                        }
                } else {
                    for (int j = 0; j < 32; j++) {
                        if (jb + j < a.KV) {
                            const float m = h2f_bits(mr[j]);
                            vis |= (m != -INFINITY);
                            nz |= (m != 0.0f);
                        }
                    }
                }
            }
        } else {
            vis = true;
        }
        const bool any_vis = __any(vis), any_nz = __any(nz);
        if (lane == 0) a.cls[ct] = !any_vis ? FA_TILE_SKIP : (any_nz ? FA_TILE_MIXED : FA_TILE_FULL);
        return;
    }
}

}  // namespace mx
