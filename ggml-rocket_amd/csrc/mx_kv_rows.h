// SPDX-License-Identifier: MIT
// One block of 32 values of a KV cache, the work of a quad of lanes: its plain values, their quantization
// and what the codes stand for (the formulas are at the head of mx_kv.hip).
#pragma once

#include "mx_common.h"
#include "mx_kernels_impl.h"

namespace mx {

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

// Lane l's codes of a block at element offset `at`: Q8_0 eight bytes, Q4_0 the eight that hold its
// nibbles, F16 eight values.
__device__ __forceinline__ u32x4 kv_codes(int type, const uint8_t * q, int64_t at, int l) {
    if (type == T_F16) return *(const u32x4 *)((const uint16_t *)q + at + 8 * l);
    const u32x2 x = *(const u32x2 *)(type == T_Q8_0 ? q + at + 8 * l : q + at / 2 + 8 * (l % 2));
    return u32x4{x[0], x[1], 0, 0};
}
// Their values: the codes times d, exact in f32.
__device__ __forceinline__ void kv_values(int type, const u32x4 & x, float d, int l, float (&v)[8]) {
    if (type == T_F16) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = h2f_bits((uint16_t)(x[e / 2] >> (16 * (e % 2))));
    } else if (type == T_Q8_0) {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = mul_rn(d, (float)(int8_t)(x[e / 4] >> (8 * (e % 4))));
    } else {
        const u32x2 n = {x[0] >> (4 * (l / 2)), x[1] >> (4 * (l / 2))};
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = mul_rn(d, (float)((int)((n[e / 4] >> (8 * (e % 4))) & 15u) - 8));
    }
}
__device__ __forceinline__ u32x4 kv_pack8(const float (&v)[8]) {
    return u32x4{pack2h(v[0], v[1]), pack2h(v[2], v[3]), pack2h(v[4], v[5]), pack2h(v[6], v[7])};
}

}  // namespace mx
