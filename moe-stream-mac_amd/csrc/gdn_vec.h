// Vector loads and stores of the streaming kernels (V elements at a time, converted to and from fp32) and sums over
// groups of lanes.
#pragma once

#include "gdn_common.h"

namespace gdn {
namespace ops {

// Sum over aligned groups of L lanes (every lane of the wave active); all lanes of a group get the same bits.
template <int L>
__device__ __forceinline__ float group_sum(float x) {
    static_assert(L == 1 || L == 2 || L == 4 || L == 8 || L == 16 || L == 32 || L == 64, "L is a power of two");
    if constexpr (L >= 2) x += dpp_mov<DPP_QUAD_1032>(x);
    if constexpr (L >= 4) x += dpp_mov<DPP_QUAD_2301>(x);
    if constexpr (L >= 8) x += dpp_mov<DPP_ROW_HALF_MIRROR>(x);
    if constexpr (L >= 16) x += dpp_mov<DPP_ROW_MIRROR>(x);
    if constexpr (L >= 32) x += lane_xor16(x);
    if constexpr (L >= 64) x += lane_xor32(x);
    return x;
}

__device__ __forceinline__ float half_bits_to_f32(uint32_t h) {
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

// V consecutive elements starting at element i (i % V == 0, buffer base 16-byte aligned).
template <int V>
__device__ __forceinline__ void loadv(const void *p, size_t i, int dt, float (&o)[V]) {
    if constexpr (V == 1) {
        o[0] = load_as_f32(p, i, dt);
    } else if constexpr (V == 4) {
        if (dt == DT_F32) {
            const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
            o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
        } else {
            const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
            const uint32_t w[2] = {u.x, u.y};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (dt == DT_BF16) {
                    o[2 * j] = __uint_as_float(w[j] << 16);
                    o[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                } else {
                    o[2 * j] = half_bits_to_f32(w[j]);
                    o[2 * j + 1] = half_bits_to_f32(w[j] >> 16);
                }
            }
        }
    } else {
        static_assert(V == 8, "V is 1, 4 or 8");
        if (dt == DT_F32) {
            const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
            const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + 4);
            o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
            o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (dt == DT_BF16) {
                    o[2 * j] = __uint_as_float(w[j] << 16);
                    o[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                } else {
                    o[2 * j] = half_bits_to_f32(w[j]);
                    o[2 * j + 1] = half_bits_to_f32(w[j] >> 16);
                }
            }
        }
    }
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int dt) {
    if (dt == DT_BF16) return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
    return (uint32_t)__half_as_ushort(__float2half(a)) | ((uint32_t)__half_as_ushort(__float2half(b)) << 16);
}

// The same by gfx950's v_cvt_pk_bf16_f32: one instruction for the two.
__device__ __forceinline__ uint32_t pack2_cvt(float a, float b, int dt) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    if (dt == DT_BF16) return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
    return pack2(a, b, dt);
}

template <int V>
__device__ __forceinline__ void storev(void *p, size_t i, int dt, const float (&o)[V]) {
    if constexpr (V == 1) {
        store_from_f32(p, i, o[0], dt);
    } else if constexpr (V == 4) {
        if (dt == DT_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(o[0], o[1], o[2], o[3]);
        } else {
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i) =
                make_uint2(pack2(o[0], o[1], dt), pack2(o[2], o[3], dt));
        }
    } else {
        static_assert(V == 8, "V is 1, 4 or 8");
        if (dt == DT_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = make_float4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<float4 *>(static_cast<float *>(p) + i + 4) = make_float4(o[4], o[5], o[6], o[7]);
        } else {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) =
                make_uint4(pack2(o[0], o[1], dt), pack2(o[2], o[3], dt), pack2(o[4], o[5], dt),
                           pack2(o[6], o[7], dt));
        }
    }
}

// The same from any element on: the card takes vector accesses at every address, and 16 bytes across a border cost less than
// element by element.
template <int V, int DT>
__device__ __forceinline__ void loadv_any(const void *p, int64_t i, float (&o)[V]) {
    static_assert(V == 4 || V == 8, "V is 4 or 8");
    typedef uint32_t w4 __attribute__((ext_vector_type(4)));
    typedef uint32_t w2 __attribute__((ext_vector_type(2)));
    typedef w4 any4 __attribute__((aligned(2)));
    typedef w2 any2 __attribute__((aligned(2)));
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            const w4 u = *reinterpret_cast<const any4 *>(static_cast<const float *>(p) + i + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * h + j] = __uint_as_float(u[j]);
        }
    } else {
        uint32_t w[V / 2];
        if constexpr (V == 8) {
            const w4 u = *reinterpret_cast<const any4 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = u[j];
        } else {
            const w2 u = *reinterpret_cast<const any2 *>(static_cast<const uint16_t *>(p) + i);
            w[0] = u[0];
            w[1] = u[1];
        }
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            o[2 * j] = DT == DT_BF16 ? __uint_as_float(w[j] << 16) : half_bits_to_f32(w[j]);
            o[2 * j + 1] = DT == DT_BF16 ? __uint_as_float(w[j] & 0xffff0000u) : half_bits_to_f32(w[j] >> 16);
        }
    }
}

template <int V, int DT>
__device__ __forceinline__ void storev_any(void *p, int64_t i, const float (&o)[V]) {
    static_assert(V == 4 || V == 8, "V is 4 or 8");
    typedef uint32_t w4 __attribute__((ext_vector_type(4)));
    typedef uint32_t w2 __attribute__((ext_vector_type(2)));
    typedef w4 any4 __attribute__((aligned(2)));
    typedef w2 any2 __attribute__((aligned(2)));
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int h = 0; h < V / 4; ++h)
            *reinterpret_cast<any4 *>(static_cast<float *>(p) + i + 4 * h) =
                w4{__float_as_uint(o[4 * h]), __float_as_uint(o[4 * h + 1]), __float_as_uint(o[4 * h + 2]),
                   __float_as_uint(o[4 * h + 3])};
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) w[j] = pack2_cvt(o[2 * j], o[2 * j + 1], DT);
        if constexpr (V == 8)
            *reinterpret_cast<any4 *>(static_cast<uint16_t *>(p) + i) = w4{w[0], w[1], w[2], w[3]};
        else
            *reinterpret_cast<any2 *>(static_cast<uint16_t *>(p) + i) = w2{w[0], w[1]};
    }
}

// The first n of V elements (n may be V or more, or less than one); the rest are zeros, or not stored.
template <int V, int DT>
__device__ __forceinline__ void load_first(const void *p, int64_t i, int64_t n, float (&o)[V]) {
    if (n >= V) {
        loadv_any<V, DT>(p, i, o);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = j < n ? load_as_f32(p, i + j, DT) : 0.f;
    }
}
template <int V, int DT>
__device__ __forceinline__ void store_first(void *p, int64_t i, int64_t n, const float (&o)[V]) {
    if (n >= V) {
        storev_any<V, DT>(p, i, o);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) store_from_f32(p, i + j, o[j], DT);
    }
}

}  // namespace ops
}  // namespace gdn
