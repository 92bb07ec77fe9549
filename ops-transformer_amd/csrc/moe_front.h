// What the operators in front of the expert FFN share: element types, reductions over a wave, checks of shapes and memory.
#pragma once

#include <hip/hip_fp16.h>

#include <cstdint>
#include <type_traits>

#include "opapi_common.h"

namespace moe_front {

constexpr int kWave = 64;

// Element types as the kernels read and write them; Store rounds to nearest even.
struct F32 {
    using Storage = float;
    static constexpr aclDataType kType = ACL_FLOAT;
    __device__ static float Load(Storage v) { return v; }
    __device__ static Storage Store(float f) { return f; }
};
struct F16 {
    using Storage = uint16_t;
    static constexpr aclDataType kType = ACL_FLOAT16;
    __device__ static float Load(Storage v) { return __half2float(__ushort_as_half(v)); }
    __device__ static Storage Store(float f) { return __half_as_ushort(__float2half_rn(f)); }
};
struct Bf16 {
    using Storage = uint16_t;
    static constexpr aclDataType kType = ACL_BF16;
    __device__ static float Load(Storage v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
    __device__ static Storage Store(float f) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f)); }
};

template <typename T>
__device__ __forceinline__ T WaveSum(T v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ uint32_t WaveMax(uint32_t v) {
    for (int d = 32; d > 0; d >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d)));
    return v;
}

inline bool IsFloating(const aclTensor* t) { return t->dtype == ACL_FLOAT || t->dtype == ACL_FLOAT16 || t->dtype == ACL_BF16; }

// t has the extents of x, its last one replaced by `last` (negative: left out).
inline bool SameButLast(const aclTensor* t, const aclTensor* x, int64_t last) {
    const size_t lead = x->dims.size() - 1;
    if (t->dims.size() != lead + (last < 0 ? 0 : 1)) return false;
    for (size_t i = 0; i < lead; ++i) {
        if (t->dims[i] != x->dims[i]) return false;
    }
    return last < 0 || t->dims.back() == last;
}

// Rows of a tensor of rank 2 or 3 whose extents are at most 2^31 - 1 each; -1 where there are more than kMaxRows.
constexpr int64_t kMaxRows = 1 << 26;
inline int64_t RowsOf(const aclTensor* x) {
    const int64_t rows = x->dims.size() == 2 ? x->dims[0] : x->dims[0] * x->dims[1];
    return rows <= kMaxRows ? rows : -1;
}

// A grid has fewer than 2^32 threads in its first direction: workgroups are numbered over two.
inline dim3 GridOf(int64_t groups) {
    constexpr int64_t kLine = 1 << 20;
    return groups <= kLine ? dim3(static_cast<unsigned>(groups)) : dim3(static_cast<unsigned>(kLine), static_cast<unsigned>((groups + kLine - 1) / kLine));
}
__device__ __forceinline__ int64_t GroupIndex() { return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x; }

// Without elements any strides do.
inline bool InOrder(const aclTensor* t) { return opapi::IsEmpty(t) || opapi::IsContiguous(t); }

// Whether two contiguous tensors have memory in common.
inline bool Overlap(const aclTensor* a, const aclTensor* b) {
    if (opapi::IsEmpty(a) || opapi::IsEmpty(b)) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(opapi::DataPtr(a)), pb = reinterpret_cast<uintptr_t>(opapi::DataPtr(b));
    const uint64_t na = static_cast<uint64_t>(opapi::Numel(a)) * opapi::ElemSize(a->dtype);
    const uint64_t nb = static_cast<uint64_t>(opapi::Numel(b)) * opapi::ElemSize(b->dtype);
    return pa < pb + nb && pb < pa + na;
}

}  // namespace moe_front
