// What the operators on rows of router logits with sequences share: rows of scores in registers, sums over the lanes of a row, which rows make up a sequence.
#pragma once

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <new>

#include "moe_front.h"

namespace moe_front {

constexpr int64_t kMaxRouterExperts = 2048;
constexpr int64_t kMaxRouterPicks = 64;

// Rows of a batch cut into `count` sequences by count + 1 offsets, or one sequence of all rows (offsets null).  Offsets are the caller's data: they are
// held to the rows there are, so that a bad one gives unspecified values and no access outside the tensors.
struct Sequences {
    const void* offsets;
    int32_t isInt64;
    int32_t count;
    int64_t rows;

    __device__ __forceinline__ int64_t Start(int64_t i) const {
        if (offsets == nullptr) return i == 0 ? 0 : rows;
        const int64_t at = isInt64 ? static_cast<const int64_t*>(offsets)[i] : static_cast<const int32_t*>(offsets)[i];
        return at < 0 ? 0 : at > rows ? rows : at;
    }
    // The last sequence that starts at or in front of `row`: -1 in front of the first, `count` behind the last.
    __device__ __forceinline__ int32_t Of(int64_t row) const {
        int64_t lo = -1, hi = static_cast<int64_t>(count) + 1;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (Start(mid) <= row) lo = mid;
            else hi = mid;
        }
        return static_cast<int32_t>(lo);
    }
};

// The value of the lane that is a fixed step away, over a row of sixteen lanes without a trip through LDS.
template <int kCtl>
__device__ __forceinline__ float DppLane(float v) {
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(__float_as_uint(v)), kCtl, 0xF, 0xF, true)));
}

// f over the values of kLanes neighbouring lanes (a power of two), the same bits in each of them.  Where the lanes of four, and of eight, agree already,
// reversing a half row or a row pairs the right ones.
template <int kLanes, typename F>
__device__ __forceinline__ float OverLanes(float v, F f) {
    if constexpr (kLanes >= 2) v = f(v, DppLane<0xB1>(v));   // quad_perm 1 0 3 2
    if constexpr (kLanes >= 4) v = f(v, DppLane<0x4E>(v));   // quad_perm 2 3 0 1
    if constexpr (kLanes >= 8) v = f(v, DppLane<0x141>(v));  // row_half_mirror
    if constexpr (kLanes >= 16) v = f(v, DppLane<0x140>(v)); // row_mirror
    if constexpr (kLanes >= 32) {
        const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(both[0]), __uint_as_float(both[1]));
    }
    if constexpr (kLanes >= 64) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(both[0]), __uint_as_float(both[1]));
    }
    return v;
}
template <int kLanes>
__device__ __forceinline__ float SumOver(float v) {
    return OverLanes<kLanes>(v, [](float a, float b) { return a + b; });
}
// A NaN among the values is passed over.
template <int kLanes>
__device__ __forceinline__ float MaxOver(float v) {
    return OverLanes<kLanes>(v, [](float a, float b) { return fmaxf(a, b); });
}

// e^x for x <= 0 to about three units of 2^-24: the product with log2(e) in two parts, so that its rounding does not grow with x.  Below 2^-126: zero.
__device__ __forceinline__ float ExpOfNegative(float x) {
    constexpr float kLog2e = 1.44269502162933349609f, kLog2eRest = 1.925963033500e-8f, kLn2 = 0.693147182464599609375f;
    const float hi = x * kLog2e;
    const float lo = fmaf(x, kLog2e, -hi) + x * kLog2eRest;
    const float e = __builtin_amdgcn_exp2f(hi);
    return x < -87.33f ? 0.f : fmaf(e, lo * kLn2, e);  // (of -inf: lo is none)
}

// sigmoid(x) and 1 - sigmoid(x), each to its own precision.
struct Sigmoid {
    float p, rest;
};
__device__ __forceinline__ Sigmoid SigmoidOf(float x) {
    const float t = ExpOfNegative(-fabsf(x));
    const float far = 1.f / (1.f + t), near = t * far;
    return x < 0.f ? Sigmoid{near, far} : Sigmoid{far, near};
}

// A row of experts lies over kLanes lanes in pieces of four: piece p of lane l holds experts 4 (p kLanes + l) to + 3.
template <int kLanes, int kPieces>
struct RowOf {
    static constexpr int kEach = 4 * kPieces;
    static constexpr int kWidth = kLanes * kEach;  // most experts
    __device__ static __forceinline__ int At(int p, int l) { return 4 * (p * kLanes + l); }

    // Behind the last expert: `fill`.  A piece that is whole is one load, wherever it begins.
    template <typename Codec>
    __device__ static __forceinline__ void Load(const typename Codec::Storage* row, int experts, int l, float fill, float (&v)[kEach]) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = At(p, l);
            typename Codec::Storage raw[4];
            if (at + 4 <= experts) {
                __builtin_memcpy(raw, row + at, sizeof(raw));
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * p + i] = Codec::Load(raw[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * p + i] = at + i < experts ? Codec::Load(row[at + i]) : fill;
            }
        }
    }
    template <typename Codec>
    __device__ static __forceinline__ void Store(typename Codec::Storage* row, int experts, int l, const float (&v)[kEach]) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = At(p, l);
            if (at + 4 <= experts) {
                typename Codec::Storage raw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i] = Codec::Store(v[4 * p + i]);
                __builtin_memcpy(row + at, raw, sizeof(raw));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (at + i < experts) row[at + i] = Codec::Store(v[4 * p + i]);
                }
            }
        }
    }
};

// Softmax of a row of logits: x -> p, and what makes a logit's p of it.  A row without a logit above -inf has zeros; NaN and +inf give NaN throughout.
struct Softmax {
    float top, inverse;
    __device__ __forceinline__ float Of(float x) const { return ExpOfNegative(x - top) * inverse; }
};
template <int kLanes, int kEach>
__device__ __forceinline__ Softmax SoftmaxOf(float (&v)[kEach]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < kEach; ++i) top = fmaxf(top, v[i]);
    top = MaxOver<kLanes>(top);
    if (top == -INFINITY) top = 0.f;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        v[i] = ExpOfNegative(v[i] - top);
        sum += v[i];
    }
    sum = SumOver<kLanes>(sum);
    const Softmax s{top, sum == 0.f ? 0.f : 1.f / sum};
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] *= s.inverse;
    return s;
}

// Shares of the row's sum of sigmoid scores, from the scores p.  Where every score is nearly lost in fp32 they are in the proportions of e^x, taken from
// the largest logit; a row without a logit above -inf has zeros.
template <int kLanes, int kEach>
__device__ __forceinline__ void SharesOf(const float (&x)[kEach], const float (&p)[kEach], float (&share)[kEach]) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += p[i];
    sum = SumOver<kLanes>(sum);
#pragma unroll
    for (int i = 0; i < kEach; ++i) share[i] = p[i];
    if (sum < 0x1p-60f) {  // (the lanes of a row agree)
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
        top = MaxOver<kLanes>(top);
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            share[i] = top == -INFINITY ? 0.f : ExpOfNegative(x[i] - top);
            sum += share[i];
        }
        sum = SumOver<kLanes>(sum);
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) share[i] *= inverse;
}

// f(lanes, pieces) of the layout for rows of so many experts, as integral constants: the fewest lanes whose pieces of four hold them, then the fewest pieces.
template <typename F>
void ForRowLayout(int64_t experts, F f) {
    auto with = [&](auto lanes, auto pieces) { f(lanes, pieces); };
    using std::integral_constant;
    if (experts <= 8) with(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    else if (experts <= 16) with(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (experts <= 32) with(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (experts <= 64) with(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (experts <= 128) with(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (experts <= 256) with(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (experts <= 512) with(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (experts <= 1024) with(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else with(integral_constant<int, 64>{}, integral_constant<int, 8>{});
}

// ------------------------------------------------------------------------------------------------ checks of the first phases
constexpr int64_t kMaxSequences = 1 << 20;

inline bool HasExtents(const aclTensor* t, std::initializer_list<int64_t> dims) {
    return t->dims.size() == dims.size() && std::equal(dims.begin(), dims.end(), t->dims.begin());
}

// Logits, expert ids and sequences: what both operators ask of them.
inline aclnnStatus CheckRouterRows(const aclTensor* x, const aclTensor* expertIdx, const aclTensor* seqOffsets, int64_t scoreType, int64_t* rows,
                                   int64_t* experts, int64_t* k, int64_t* sequences) {
    using namespace opapi;
    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    *experts = x->dims.back();
    OPAPI_CHECK(*experts >= 1 && *experts <= kMaxRouterExperts, kInvalid, "x has %lld experts; this operator takes 1 to %lld experts", (long long)*experts,
                (long long)kMaxRouterExperts);
    *rows = RowsOf(x);
    OPAPI_CHECK(*rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
    *k = expertIdx->dims.empty() ? 0 : expertIdx->dims.back();
    OPAPI_CHECK(expertIdx->dtype == ACL_INT32 && SameButLast(expertIdx, x, *k), kInvalid, "expertIdx %s must be INT32 of x's extents %s with the last replaced",
                ShapeStr(expertIdx).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(*k >= 1 && *k <= kMaxRouterPicks, kInvalid, "expertIdx has %lld ids a row; this operator takes 1 to %lld", (long long)*k,
                (long long)kMaxRouterPicks);
    OPAPI_CHECK(scoreType == 0 || scoreType == 1, kInvalid, "scoreType (=%lld) must be 0 or 1", (long long)scoreType);
    *sequences = 1;
    if (seqOffsets != nullptr) {
        OPAPI_CHECK(seqOffsets->dtype == ACL_INT32 || seqOffsets->dtype == ACL_INT64, kInvalid, "seqOffsets must be INT32 or INT64");
        OPAPI_CHECK(seqOffsets->dims.size() == 1 && seqOffsets->dims[0] >= 2 && seqOffsets->dims[0] <= kMaxSequences + 1, kInvalid,
                    "seqOffsets %s must be [S + 1] of 1 to %lld sequences", ShapeStr(seqOffsets).c_str(), (long long)kMaxSequences);
        *sequences = seqOffsets->dims[0] - 1;
    }
    return ACLNN_SUCCESS;
}

// Outputs are contiguous and apart from each other and from the inputs, and everything that has elements has memory.
inline aclnnStatus CheckMemory(std::initializer_list<const aclTensor*> ins, std::initializer_list<const aclTensor*> outs) {
    using namespace opapi;
    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (*o == nullptr) continue;
        OPAPI_CHECK(InOrder(*o), kInvalid, "the outputs must be contiguous");
        OPAPI_CHECK(IsEmpty(*o) || (*o)->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an output carries no device memory");
        for (auto p = outs.begin(); p != o; ++p) OPAPI_CHECK(!Overlap(*o, *p), kInvalid, "two outputs share memory");
    }
    for (const aclTensor* in : ins) {
        if (in == nullptr) continue;
        OPAPI_CHECK(IsEmpty(in) || in->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an input carries no device memory");
        if (!IsContiguous(in)) continue;  // read from a copy that is made first
        for (const aclTensor* out : outs) OPAPI_CHECK(!Overlap(out, in), kInvalid, "an output shares memory with an input");
    }
    return ACLNN_SUCCESS;
}

}  // namespace moe_front
