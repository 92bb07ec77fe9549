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
    // The last sequence that starts at or in front of `row`, the same in all lanes of a whole wave: -1 in front of the first, `count` behind the last.  The
    // lanes look at 64 places at a time, so that the round trips are one for up to 63 sequences and four for the most.  Whatever the offsets are, the
    // sequence starts at or in front of the row, and the next one, at `end`, behind it (behind the last: all rows).  `beyond`: where the next one
    // ends, if it was seen on the way; else -1.
    __device__ __forceinline__ int32_t Of(int64_t row, int64_t& end, int64_t& beyond) const {
        int32_t lo = -1, hi = count + 1;
        end = rows;
        beyond = -1;
        while (hi - lo > 1) {
            const int32_t step = (hi - lo - 2) / kWave + 1;
            const int32_t at = lo + (static_cast<int32_t>(threadIdx.x % kWave) + 1) * step;
            const int32_t start = at < hi ? static_cast<int32_t>(Start(at)) : 0;
            const uint64_t behind = __ballot(at >= hi || start > row);
            const int32_t steps = behind == 0 ? kWave : __builtin_ctzll(behind);  // that do not lead behind the row
            if (behind != 0 && lo + (steps + 1) * step < hi) {
                if (step == 1 && steps + 1 < kWave && lo + steps + 2 < hi) beyond = __shfl(start, steps + 1);
                hi = lo + (steps + 1) * step;
                end = __shfl(start, steps);
            }
            lo += steps * step;
        }
        return lo;
    }
};

// The sequence of a row in the lane's own place, from that of a row in front of it: the next one, if it is not further.
__device__ __forceinline__ int32_t SequenceBehind(const Sequences& s, int32_t sequence, int64_t row, int64_t& end) {
    end = s.rows;
    if (sequence + 1 >= s.count) return sequence + 1;
    end = s.Start(sequence + 2);
    if (end > row) return sequence + 1;
    int32_t lo = sequence + 1, hi = s.count + 1;
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) / 2;
        if (s.Start(mid) <= row) lo = mid;
        else hi = mid;
    }
    end = hi <= s.count ? s.Start(hi) : s.rows;
    return lo;
}

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

// 1 / v of numbers that neither it nor they are near the ends of fp32's range, to about a unit of 2^-24 (a division takes three times as long).
__device__ __forceinline__ float Reciprocal(float v) {
    const float r = __builtin_amdgcn_rcpf(v);
    return fmaf(fmaf(-v, r, 1.f), r, r);
}

constexpr float kLog2e = 1.44269502162933349609f;

// e^(x - top) for x <= top: the product with log2(e) with what its rounding leaves, so that only the difference's own rounding is |x - top| units of 2^-24,
// and the rest four.  0 of -inf, and below 2^-126.
struct ExpFrom {
    float top;
    __device__ __forceinline__ explicit ExpFrom(float t) : top(t) {}
    __device__ __forceinline__ float operator()(float x) const {
        constexpr float kLn2 = 0.693147182464599609375f, kLog2eRest = 1.925963033500e-8f;
        const float d = x - top, hi = d * kLog2e;
        const float lo = fmaf(d, kLog2e, -hi) + d * kLog2eRest;
        const float e = __builtin_amdgcn_exp2f(hi);
        return d < -88.f ? 0.f : fmaf(e, lo * kLn2, e);  // (of -inf: lo is none)
    }
};

// sigmoid(x) and 1 - sigmoid(x), each to its own precision: |x| + 4 units of 2^-24.  (Of e^-x past fp32's range the reciprocal is 0, and below a half the
// difference from 1 is the more exact: no value needs a case of its own.)
// What the product's rounding leaves is not carried, as ExpFrom carries it: with it balance and gradient of 16384 x 256 logits take 3 % longer, and the gradient's
// error, 1.2e-7 in the 2-norm, is the same, since logits are small numbers; at -20 a score has 1.4e-6.
struct Sigmoid {
    float p, rest;
};
__device__ __forceinline__ Sigmoid SigmoidOf(float x) {
    const float t = __builtin_amdgcn_exp2f(x * -kLog2e);
    const float p = __builtin_amdgcn_rcpf(1.f + t);
    return Sigmoid{p, p > 0.5f ? t * p : 1.f - p};
}

// -inf in an element type.
template <typename Codec>
__device__ __forceinline__ typename Codec::Storage Nothing() {
    if constexpr (std::is_same_v<Codec, F32>) return -INFINITY;
    else return std::is_same_v<Codec, F16> ? 0xfc00 : 0xff80;
}

// A row of experts lies over kLanes lanes in pieces of four: piece p of lane l holds experts 4 (p kLanes + l) to + 3.
template <int kLanes, int kPieces>
struct RowOf {
    static constexpr int kEach = 4 * kPieces;
    static constexpr int kWidth = kLanes * kEach;  // most experts
    __device__ static __forceinline__ int At(int p, int l) { return 4 * (p * kLanes + l); }

    // A lane's pieces as they come from memory: one load each without a branch and without a use, so that several rows' are on their way together.  A piece
    // that would end behind the row is the row's last four elements.
    template <typename T>
    struct Raw {
        T e[kEach];
    };
    // (`rows`, the same for the wave, and where the lane's row begins behind it: an address in scalar registers with 32 bits of the lane's own.)
    template <typename T>
    __device__ static __forceinline__ Raw<T> Ask(const T* rows, uint32_t begin, int experts, int l) {
        Raw<T> raw;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            if (kLanes == 2 && experts < 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) raw.e[4 * p + i] = rows[begin + static_cast<uint32_t>(min(i, experts - 1))];
            } else {
                __builtin_memcpy(raw.e + 4 * p, rows + (begin + static_cast<uint32_t>(min(At(p, l), experts - 4))), 4 * sizeof(T));
            }
        }
        return raw;
    }
    // Their elements in their places; behind the last expert: `fill`.
    template <typename T>
    __device__ static __forceinline__ void Place(const Raw<T>& raw, int experts, int l, T fill, T (&v)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = raw.e[i];
        if (experts == kWidth) return;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = At(p, l), behind = kLanes == 2 && experts < 4 ? 0 : at - min(at, experts - 4);
            T* const e = v + 4 * p;
            const bool one = (behind & 1) != 0, two = (behind & 2) != 0;  // three in two steps
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = one ? (i < 3 ? e[i + 1] : fill) : e[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = two ? (i < 2 ? e[i + 2] : fill) : e[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = at + i < experts ? e[i] : fill;
        }
    }
    template <typename Codec>
    __device__ static __forceinline__ void Logits(const Raw<typename Codec::Storage>& raw, int experts, int l, float (&v)[kEach]) {
        typename Codec::Storage placed[kEach];
        Place(raw, experts, l, Nothing<Codec>(), placed);
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = Codec::Load(placed[i]);
    }
    template <typename Codec>
    __device__ static __forceinline__ void Store(typename Codec::Storage* rows, uint32_t begin, int experts, int l, const float (&v)[kEach]) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            const int at = At(p, l);
            typename Codec::Storage* const row = rows + (begin + static_cast<uint32_t>(at));
            if (at + 4 <= experts) {
                typename Codec::Storage raw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[i] = Codec::Store(v[4 * p + i]);
                __builtin_memcpy(row, raw, sizeof(raw));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (at + i < experts) row[i] = Codec::Store(v[4 * p + i]);
                }
            }
        }
    }
};

// The largest of a row's logits, as the point that exponentials are taken from: 0 for a row without a logit above -inf.  A NaN is passed over.
template <int kLanes, int kEach>
__device__ __forceinline__ float TopOf(const float (&v)[kEach]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < kEach; ++i) top = fmaxf(top, v[i]);
    top = MaxOver<kLanes>(top);
    return top == -INFINITY ? 0.f : top;
}

// Softmax of a row of logits in their place.  A row without a logit above -inf has zeros; NaN and +inf give NaN throughout.
template <int kLanes, int kEach>
__device__ __forceinline__ void SoftmaxOf(float (&v)[kEach]) {
    const ExpFrom e(TopOf<kLanes>(v));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        v[i] = e(v[i]);
        sum += v[i];
    }
    sum = SumOver<kLanes>(sum);
    const float inverse = sum == 0.f ? 0.f : Reciprocal(sum);
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] *= inverse;
}

// Shares of the row's sum of sigmoid scores.  Where that sum is below kLostSum the scores are nearly or wholly lost in fp32: they are in the proportions of
// e^x then, which is the softmax (a row without a logit above -inf has zeros).
constexpr float kLostSum = 0x1p-60f;
// e^-v of a v above this is zero in 64 bits, too.
constexpr float kLostIn64 = 745.f;
template <int kLanes, int kEach>
__device__ __forceinline__ void LostSharesOf(const float (&x)[kEach], float (&share)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) share[i] = x[i];
    SoftmaxOf<kLanes>(share);
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
