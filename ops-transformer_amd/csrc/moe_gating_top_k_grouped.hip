// aclnnMoeGatingTopKGrouped for gfx950: softmax or sigmoid scores, a bias that moves the choice only, groups, top-k.
//
// Two experts change places when their t = p + bias do, and near the top of 256 sigmoid scores a pair within fp32's rounding of an exponential
// comes up in one row of some thousands.  t is therefore computed and compared in 64 bits, as order-preserving 64-bit keys (the bits of a
// double mapped so that unsigned comparison equals that of the numbers, NaN on top): the choice is that of the formula, whatever the
// exponential's last bit.  Key 0 marks an expert that is taken or lies in a group that was left out; it is below every real value, -inf
// (an expert of logit -inf) among them.
#include "moe_front.h"

#include <cmath>

#include "aclnnop/aclnn_moe_gating_top_k_grouped.h"

namespace {

using namespace moe_front;

constexpr int64_t kMaxExperts = 2048;
constexpr int64_t kMaxPicks = 64;

struct GatingArgs {
    const void* x;
    const float* bias;        // optional
    const uint8_t* finished;  // optional, one byte per row
    void* y;
    int32_t* expertIdx;
    float* scores;            // optional
    int64_t rows;
    int32_t experts;
    int32_t k;
    int32_t groups;
    int32_t kGroup;
    int32_t topTwo;           // a group's value is the sum of its two largest t
    int32_t sigmoid;
    int32_t renorm;
    float factor;
    double eps;
};

__device__ __forceinline__ uint64_t KeyOf(double d) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(d));
    if (d != d) return ~0ull;
    return (u >> 63) != 0 ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double ValueOf(uint64_t key) {
    if (key == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
    return __longlong_as_double(static_cast<long long>((key >> 63) != 0 ? key & 0x7fffffffffffffffull : ~key));
}

__device__ __forceinline__ double WaveSum64(double v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// The largest key of the wave and the lowest index that holds it; every lane brings the largest of its own and that one's lowest index.
__device__ __forceinline__ void WaveArgMax(uint64_t& key, int32_t& idx) {
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t otherKey = __shfl_xor(static_cast<unsigned long long>(key), d);
        const int32_t otherIdx = __shfl_xor(idx, d);
        if (otherKey > key || (otherKey == key && otherIdx < idx)) {
            key = otherKey;
            idx = otherIdx;
        }
    }
}

// p of one logit.  shift and sum are the row's largest logit and sum of exponentials under softmax.
__device__ __forceinline__ double ScoreOf(float x, bool sigmoid, double shift, double sum) {
    if (x == -INFINITY) return 0.0;
    return sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - shift) / sum;
}

// One wave per row, the keys in LDS.
template <typename Codec, typename Out>
__global__ __launch_bounds__(kWave) void GatingAnyKernel(GatingArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char ldsRaw[];
    uint64_t* const keys = reinterpret_cast<uint64_t*>(ldsRaw);     // [experts]
    uint64_t* const groupKeys = keys + a.experts;                   // [groups]
    const int lane = threadIdx.x;
    const int64_t row = GroupIndex();
    if (row >= a.rows) return;
    const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x) + row * a.experts;

    double shift = 0.0, sum = 1.0;
    if (a.sigmoid == 0) {
        float top = -INFINITY;
        bool nan = false;
        for (int c = lane; c < a.experts; c += kWave) {
            const float v = Codec::Load(x[c]);
            top = fmaxf(top, v);
            nan |= v != v;
        }
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        shift = __any(nan) ? NAN : top;
        sum = 0.0;
        for (int c = lane; c < a.experts; c += kWave) sum += ScoreOf(Codec::Load(x[c]), false, shift, 1.0);
        sum = WaveSum64(sum);
    }
    for (int c = lane; c < a.experts; c += kWave) {
        const float v = Codec::Load(x[c]);
        const double p = ScoreOf(v, a.sigmoid != 0, shift, sum);
        if (a.scores != nullptr) a.scores[row * a.experts + c] = static_cast<float>(p);
        keys[c] = KeyOf(v == -INFINITY ? -INFINITY : a.bias == nullptr ? p : p + static_cast<double>(a.bias[c]));
    }
    __syncthreads();

    if (a.kGroup < a.groups) {
        const int size = a.experts / a.groups;
        for (int g = lane; g < a.groups; g += kWave) {
            uint64_t first = 0, second = 0;
            for (int c = g * size; c < (g + 1) * size; ++c) {
                const uint64_t key = keys[c];
                if (key > first) {
                    second = first;
                    first = key;
                } else if (key > second) {
                    second = key;
                }
            }
            const double one = ValueOf(first), two = ValueOf(second);
            groupKeys[g] = a.topTwo != 0 && two != -INFINITY ? KeyOf(one + two) : first;
        }
        __syncthreads();
        for (int j = 0; j < a.kGroup; ++j) {
            uint64_t best = 0;
            int32_t at = INT32_MAX;
            for (int g = lane; g < a.groups; g += kWave) {
                if (groupKeys[g] > best) {
                    best = groupKeys[g];
                    at = g;
                }
            }
            WaveArgMax(best, at);
            __syncthreads();
            if (lane == 0) groupKeys[at] = 0;  // stays
            __syncthreads();
        }
        for (int c = lane; c < a.experts; c += kWave) {
            if (groupKeys[c / size] != 0) keys[c] = 0;
        }
        __syncthreads();
    }

    int32_t pick = 0;  // of lane j: the j-th
    for (int j = 0; j < a.k; ++j) {
        uint64_t best = 0;
        int32_t at = INT32_MAX;
        for (int c = lane; c < a.experts; c += kWave) {
            if (keys[c] > best) {
                best = keys[c];
                at = c;
            }
        }
        WaveArgMax(best, at);
        if (lane == j) pick = at;
        __syncthreads();
        if (lane == 0) keys[at] = 0;
        __syncthreads();
    }

    double y = lane < a.k ? ScoreOf(Codec::Load(x[pick]), a.sigmoid != 0, shift, sum) : 0.0;
    if (a.renorm != 0) {
        const double total = WaveSum64(y) + a.eps;
        y = total == 0.0 ? 0.0 : y / total;
    }
    if (lane < a.k) {
        const bool done = a.finished != nullptr && a.finished[row] != 0;
        static_cast<typename Out::Storage*>(a.y)[row * a.k + lane] = Out::Store(static_cast<float>(y * a.factor));
        a.expertIdx[row * a.k + lane] = done ? a.experts : pick;
    }
}

class GatingExecutor : public aclOpExecutor {
   public:
    GatingArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType outType = ACL_FLOAT;

    template <typename Codec, typename Out>
    void Launch(hipStream_t stream) const {
        const size_t lds = (static_cast<size_t>(args.experts) + args.groups) * 8;
        hipLaunchKernelGGL((GatingAnyKernel<Codec, Out>), GridOf(args.rows), dim3(kWave), lds, stream, args);
    }

    template <typename Codec>
    void LaunchFor(hipStream_t stream) const {
        if (outType == Codec::kType) Launch<Codec, Codec>(stream);
        else Launch<Codec, F32>(stream);
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("gating_topk_grouped", stream);
        if (dtype == ACL_FLOAT) Launch<F32, F32>(stream);
        else if (dtype == ACL_FLOAT16) LaunchFor<F16>(stream);
        else LaunchFor<Bf16>(stream);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) {
            opapi::SetError("aclnnMoeGatingTopKGrouped: launch failed: %s", hipGetErrorString(err));
            return ACLNN_ERR_RUNTIME_ERROR;
        }
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeGatingTopKGroupedGetWorkspaceSize(
    const aclTensor* x, const aclTensor* biasOptional, const aclTensor* finishedOptional, int64_t k, int64_t kGroup,
    int64_t groupCount, int64_t groupSelectMode, int64_t scoreType, int64_t renorm, double routedScalingFactor, double eps,
    const aclTensor* yOut, const aclTensor* expertIdxOut, const aclTensor* scoresOutOptional, uint64_t* workspaceSize,
    aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(yOut, "yOut");
    OPAPI_CHECK_NOTNULL(expertIdxOut, "expertIdxOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, biasOptional, finishedOptional, yOut, expertIdxOut, scoresOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    const int64_t experts = x->dims.back();
    OPAPI_CHECK(experts > 0 && experts <= kMaxExperts, kInvalid, "the last extent of x (=%lld) must be 1 to %lld experts", (long long)experts,
                (long long)kMaxExperts);
    const int64_t rows = RowsOf(x);
    OPAPI_CHECK(rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
    OPAPI_CHECK(groupCount >= 1 && groupCount <= experts && experts % groupCount == 0, kInvalid,
                "groupCount (=%lld) must divide the %lld experts", (long long)groupCount, (long long)experts);
    OPAPI_CHECK(kGroup >= 1 && kGroup <= groupCount, kInvalid, "kGroup (=%lld) must be 1 to groupCount (=%lld)", (long long)kGroup,
                (long long)groupCount);
    OPAPI_CHECK(groupSelectMode == 0 || groupSelectMode == 1, kInvalid, "groupSelectMode (=%lld) must be 0 or 1", (long long)groupSelectMode);
    OPAPI_CHECK(groupSelectMode == 0 || kGroup == groupCount || experts / groupCount >= 2, kInvalid,
                "groupSelectMode 1 adds two experts of a group, which has one");
    OPAPI_CHECK(scoreType == 0 || scoreType == 1, kInvalid, "scoreType (=%lld) must be 0 or 1", (long long)scoreType);
    OPAPI_CHECK(renorm == 0 || renorm == 1, kInvalid, "renorm (=%lld) must be 0 or 1", (long long)renorm);
    OPAPI_CHECK(k >= 1 && k <= kMaxPicks && k <= experts / groupCount * kGroup, kInvalid,
                "k (=%lld) must be 1 to %lld and at most the %lld experts of the groups that stay", (long long)k, (long long)kMaxPicks,
                (long long)(experts / groupCount * kGroup));
    OPAPI_CHECK(std::isfinite(routedScalingFactor), kInvalid, "routedScalingFactor must be a number");
    OPAPI_CHECK(eps >= 0 && std::isfinite(eps), kInvalid, "eps must be a number of at least 0");
    OPAPI_CHECK(biasOptional == nullptr || (biasOptional->dtype == ACL_FLOAT && biasOptional->dims.size() == 1 && biasOptional->dims[0] == experts),
                kInvalid, "bias must be FLOAT [%lld]", (long long)experts);
    OPAPI_CHECK(finishedOptional == nullptr || (finishedOptional->dtype == ACL_BOOL && SameButLast(finishedOptional, x, -1)), kInvalid,
                "finished must be BOOL of x's extents without the last");
    OPAPI_CHECK((yOut->dtype == x->dtype || yOut->dtype == ACL_FLOAT) && SameButLast(yOut, x, k), kInvalid,
                "yOut %s must be of x's type or FLOAT, x's extents %s with the last replaced by k", ShapeStr(yOut).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(expertIdxOut->dtype == ACL_INT32 && SameButLast(expertIdxOut, x, k), kInvalid,
                "expertIdxOut %s must be INT32, x's extents %s with the last replaced by k", ShapeStr(expertIdxOut).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(scoresOutOptional == nullptr || (scoresOutOptional->dtype == ACL_FLOAT && SameButLast(scoresOutOptional, x, experts)), kInvalid,
                "scoresOut %s must be FLOAT of x's extents %s", ShapeStr(scoresOutOptional).c_str(), ShapeStr(x).c_str());
    const aclTensor* const ins[] = {x, biasOptional, finishedOptional};
    const aclTensor* const outs[] = {yOut, expertIdxOut, scoresOutOptional};
    for (int o = 0; o < 3; ++o) {
        if (outs[o] == nullptr) continue;
        OPAPI_CHECK(InOrder(outs[o]), kInvalid, "the outputs must be contiguous");
        OPAPI_CHECK(rows == 0 || outs[o]->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an output carries no device memory");
        for (int p = 0; p < o; ++p) OPAPI_CHECK(!Overlap(outs[o], outs[p]), kInvalid, "two outputs share memory");
    }
    for (const aclTensor* in : ins) {
        if (in == nullptr) continue;
        OPAPI_CHECK(rows == 0 || in->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an input carries no device memory");
        for (const aclTensor* out : outs) {
            OPAPI_CHECK(!IsContiguous(in) || !Overlap(out, in), kInvalid, "an output shares memory with an input");
        }
    }

    auto* ex = new (std::nothrow) GatingExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    ex->dtype = x->dtype;
    ex->outType = yOut->dtype;
    OPAPI_BIND(ex, x, &ex->args.x);
    OPAPI_BIND(ex, biasOptional, &ex->args.bias);
    OPAPI_BIND(ex, finishedOptional, &ex->args.finished);
    ex->args.y = DataPtr(yOut);
    ex->args.expertIdx = reinterpret_cast<int32_t*>(DataPtr(expertIdxOut));
    ex->args.scores = reinterpret_cast<float*>(DataPtr(scoresOutOptional));
    ex->args.rows = rows;
    ex->args.experts = static_cast<int32_t>(experts);
    ex->args.k = static_cast<int32_t>(k);
    ex->args.groups = static_cast<int32_t>(groupCount);
    ex->args.kGroup = static_cast<int32_t>(kGroup);
    ex->args.topTwo = static_cast<int32_t>(groupSelectMode);
    ex->args.sigmoid = static_cast<int32_t>(scoreType);
    ex->args.renorm = static_cast<int32_t>(renorm);
    ex->args.factor = static_cast<float>(routedScalingFactor);
    ex->args.eps = eps;
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeGatingTopKGrouped(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                 aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
