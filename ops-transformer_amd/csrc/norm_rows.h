// What the norms of rows share: pieces of eight elements of any type, and the int8 rows with a scale each.
#pragma once

#include <cmath>

#include "moe_front.h"

namespace moe_front {

template <typename Codec>
struct Packet {  // eight elements as they lie in memory
    uint4 q[sizeof(typename Codec::Storage) / 2];
};

template <typename Codec>
__device__ __forceinline__ void Unpack(const Packet<Codec>& p, float (&v)[8]) {
    const typename Codec::Storage* const raw = reinterpret_cast<const typename Codec::Storage*>(&p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Codec::Load(raw[i]);
}

template <typename Codec>
__device__ __forceinline__ Packet<Codec> Pack(const float (&v)[8]) {
    Packet<Codec> p;
    if constexpr (std::is_same_v<Codec, Bf16>) {
        typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
        typedef float F32x2 __attribute__((ext_vector_type(2)));
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(F32x2{v[2 * i], v[2 * i + 1]}, Bf16x2));
        p.q[0] = uint4{w[0], w[1], w[2], w[3]};
    } else {
        typename Codec::Storage raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = Codec::Store(v[i]);
        __builtin_memcpy(&p, raw, sizeof(p));
    }
    return p;
}

// `count` (1 to 8) elements from `at` on, zeros behind them, and back.
template <bool kGrid, typename Codec>
__device__ __forceinline__ Packet<Codec> LoadPacket(const void* base, int64_t at, int count) {
    const typename Codec::Storage* const from = static_cast<const typename Codec::Storage*>(base) + at;
    Packet<Codec> p;
    if constexpr (kGrid) {
        p = *reinterpret_cast<const Packet<Codec>*>(from);
    } else if (count == 8) {
        __builtin_memcpy(&p, from, sizeof(p));
    } else {
        typename Codec::Storage raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = i < count ? from[i] : typename Codec::Storage{};
        __builtin_memcpy(&p, raw, sizeof(p));
    }
    return p;
}
template <bool kGrid, typename Storage, typename P>
__device__ __forceinline__ void StorePacket(void* base, int64_t at, int count, const P& p) {
    static_assert(sizeof(P) == 8 * sizeof(Storage));
    Storage* const to = static_cast<Storage*>(base) + at;
    if constexpr (kGrid) {
        *reinterpret_cast<P*>(to) = p;
    } else if (count == 8) {
        __builtin_memcpy(to, &p, sizeof(p));
    } else {
        Storage raw[8];
        __builtin_memcpy(raw, &p, sizeof(p));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i < count) to[i] = raw[i];
        }
    }
}

// What a row's reduction settles.
struct RowScales {
    float r;      // of the norm
    float scale;  // of the int8 row
    float up;     // w is taken times `up`, so that the quotient below stays a normal number in both parts for rows of tiny and of huge values
    float inv;    // 127 / (max|w| up), and what is left of it behind its rounding; 0 where the row's int8 values are zeros
    float rest;
};

// sumSquares and maxBits (the bits of max|w|, whose order as unsigned numbers is that of the values, NaN last) are the row's.
__device__ __forceinline__ RowScales ScalesOf(float sumSquares, uint32_t maxBits, int64_t cols, float eps) {
    RowScales s;
    const float mean = sumSquares / static_cast<float>(cols) + eps;
    s.r = mean == 0.f ? 0.f : 1.f / sqrtf(mean);
    const float m = __uint_as_float(maxBits);
    s.scale = m * s.r / 127.f;
    s.up = m < 0x1p-100f ? 0x1p100f : m > 0x1p100f ? 0x1p-100f : 1.f;
    s.inv = s.scale > 0.f && s.scale < INFINITY ? 127.f / (m * s.up) : 0.f;
    s.rest = fmaf(-s.inv, m * s.up, 127.f) * s.inv * (1.f / 127.f);
    return s;
}

// 127 w / max to the nearest whole number, half to even.  The factor has twice fp32's bits: a value in the middle between two whole numbers, as one in
// 25 000 of 16-bit rows is, is seen to be there (rounded to fp32 the factor took one in six of those to the odd number).  No |w| passes the maximum, so
// nothing passes 127.
__device__ __forceinline__ int32_t Quantised(float w, const RowScales& s) {
    const float v = w * s.up;
    return s.inv == 0.f ? 0 : static_cast<int32_t>(rintf(fmaf(v, s.inv, v * s.rest)));
}

}  // namespace moe_front
