// aclnnMoeGatingTopKGroupedGrad for gfx950: the gradients of picked weights and of the balance loss with respect to the logits.
//
// Both are a row's scores times something less a mean, and the scores are made anew from the logits: one read and one write of a row.  With q_j = p_j / t
// of the picked ones and A = sum dy_j p_j, the renormalised weights have dp_j = F (dy_j - A / t) / t, and their mean under the softmax is
// F A / t (1 - sum p / t) = F (A / t) (eps / t): formed so, it is not the difference of two sums that cancel.  The picks' dp goes through LDS from the lane
// that has the pick to the one that has the expert.
#include "router_rows.h"

#include "aclnnop/aclnn_moe_gating_top_k_grouped_grad.h"

namespace {

using namespace moe_front;

struct GradArgs {
    const void* x;
    const int32_t* expertIdx;
    const void* yGrad;         // optional
    const float* lossGrad;     // optional, with counts and seqRows
    const int32_t* counts;
    const int32_t* seqRows;
    Sequences sequences;
    void* xGrad;
    int32_t experts;
    int32_t k;
    int32_t yGradIsFloat;
    int32_t renorm;
    float factor;
    float eps;
    int32_t waveRows;          // rows of a wave, one behind the other
};

constexpr int kGradThreads = 256;
constexpr int kGradWaves = kGradThreads / kWave;

template <typename Codec, typename Out, int kLanes, int kPieces, bool kSigmoid>
__global__ __launch_bounds__(kGradThreads) void GatingGradKernel(GradArgs a) {
    using Row = RowOf<kLanes, kPieces>;
    constexpr int kEach = Row::kEach;
    constexpr int kRowsAtOnce = kWave / kLanes;
    __shared__ float4 picked[kGradWaves][kRowsAtOnce][Row::kWidth / 4];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, l = lane % kLanes, side = lane / kLanes;
    float* const mine = reinterpret_cast<float*>(picked[wave][side]);
    const bool weights = a.yGrad != nullptr, balance = a.lossGrad != nullptr;
    if (weights) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) picked[wave][side][Row::At(p, l) / 4] = float4{0.f, 0.f, 0.f, 0.f};
    }
    // The rows of a wave follow each other, `side` by side: their sequence changes seldom, and with it the counts in registers.
    const int64_t first = (GroupIndex() * kGradWaves + wave) * a.waveRows, last = min(first + a.waveRows, a.sequences.rows);
    int32_t sequence = -2;  // of this row, its end, and what its loss gives each share
    int64_t sequenceEnd = -1;
    float shareGrad[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) shareGrad[i] = 0.f;
    for (int64_t row = first + side; row < last; row += kRowsAtOnce) {
        const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x) + row * a.experts;
        const int32_t* const idx = a.expertIdx + row * a.k;
        auto isExpert = [&](int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts); };
        float v[kEach];
        Row::template Load<Codec>(x, a.experts, l, -INFINITY, v);
        const bool live = isExpert(idx[0]);
        if (balance && row >= sequenceEnd) {
            sequence = a.sequences.Of(row);
            const bool inside = sequence >= 0 && sequence < a.sequences.count;
            sequenceEnd = inside ? a.sequences.Start(sequence + 1) : sequence < 0 ? a.sequences.Start(0) : a.sequences.rows;
            const float n = inside ? static_cast<float>(a.seqRows[sequence]) : 0.f;
            const float each = n > 0.f ? a.lossGrad[sequence] * (static_cast<float>(a.experts) / static_cast<float>(a.k)) / n / n : 0.f;
#pragma unroll
            for (int p = 0; p < kPieces; ++p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = Row::At(p, l) + i;
                    shareGrad[4 * p + i] = n > 0.f && e < a.experts ? each * static_cast<float>(a.counts[static_cast<int64_t>(sequence) * a.experts + e]) : 0.f;
                }
            }
        }
        // scores: p, and 1 - p of sigmoid ones
        float p[kEach], rest[kEach];
        Softmax softmax{};
        if constexpr (kSigmoid) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const Sigmoid s = SigmoidOf(v[i]);
                p[i] = s.p;
                rest[i] = s.rest;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) p[i] = v[i];
            softmax = SoftmaxOf<kLanes>(p);
        }
        float grad[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) grad[i] = 0.f;
        if (weights) {
            auto yGradOf = [&](int j) {
                const int64_t at = row * a.k + j;
                return a.yGradIsFloat ? static_cast<const float*>(a.yGrad)[at] : Codec::Load(static_cast<const typename Codec::Storage*>(a.yGrad)[at]);
            };
            auto scoreOf = [&](int32_t id) {
                const float logit = Codec::Load(x[id]);
                if constexpr (kSigmoid) return SigmoidOf(logit).p;
                else return softmax.Of(logit);
            };
            float sum = 0.f, weighted = 0.f;
            int32_t id0 = -1;  // the lane's first pick, kept
            float y0 = 0.f;
            for (int j = l; j < a.k; j += kLanes) {
                const int32_t id = idx[j];
                const float y = yGradOf(j);
                if (j == l) {
                    id0 = id;
                    y0 = y;
                }
                if (!isExpert(id)) continue;
                const float score = scoreOf(id);
                sum += score;
                weighted += y * score;
            }
            sum = SumOver<kLanes>(sum);
            weighted = SumOver<kLanes>(weighted);
            float mean = 0.f, scale = a.factor, all = a.factor * weighted;
            if (a.renorm) {
                const float total = sum + a.eps;
                scale = total == 0.f ? 0.f : a.factor / total;
                mean = total == 0.f ? 0.f : weighted / total;
                all = total == 0.f ? 0.f : a.factor * mean * (a.eps / total);
                if (sum == 0.f) scale = mean = all = 0.f;
            }
            for (int j = l; j < a.k; j += kLanes) {
                const int32_t id = j == l ? id0 : idx[j];
                const float y = j == l ? y0 : yGradOf(j);
                if (isExpert(id)) atomicAdd(mine + id, scale * (y - mean));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < kPieces; ++q) {
                float4* const at = &picked[wave][side][Row::At(q, l) / 4];
                const float4 dp = *at;
                *at = float4{0.f, 0.f, 0.f, 0.f};  // for the next row
                const float d[4] = {dp.x, dp.y, dp.z, dp.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (kSigmoid) grad[4 * q + i] = d[i] * p[4 * q + i] * rest[4 * q + i];
                    else grad[4 * q + i] = p[4 * q + i] * (d[i] - all);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (balance) {
            float share[kEach];
            if constexpr (kSigmoid) {
                SharesOf<kLanes>(v, p, share);
            } else {
#pragma unroll
                for (int i = 0; i < kEach; ++i) share[i] = p[i];
            }
            float mean = 0.f;
#pragma unroll
            for (int i = 0; i < kEach; ++i) mean = fmaf(shareGrad[i], share[i], mean);
            mean = SumOver<kLanes>(mean);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                float g = share[i] * (shareGrad[i] - mean);
                if constexpr (kSigmoid) g *= rest[i];
                grad[i] += sequence >= 0 && sequence < a.sequences.count ? g : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i) grad[i] = live ? grad[i] : 0.f;
        Row::template Store<Out>(static_cast<typename Out::Storage*>(a.xGrad) + row * a.experts, a.experts, l, grad);
    }
}

class GatingGradExecutor : public aclOpExecutor {
   public:
    GradArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType outType = ACL_FLOAT;
    bool sigmoid = false;

    template <typename Codec, typename Out>
    void Launch(hipStream_t stream) {
        ForRowLayout(args.experts, [&](auto lanes, auto pieces) {
            constexpr int kLanes = decltype(lanes)::value, kPieces = decltype(pieces)::value;
            constexpr int64_t kRowsAtOnce = kWave / kLanes;
            const int64_t waves = 8 * 1024;  // two rounds of the chip's 256 x 4 SIMDs, four waves each
            int64_t each = (args.sequences.rows + waves - 1) / waves;
            each = (each + kRowsAtOnce - 1) / kRowsAtOnce * kRowsAtOnce;
            if (each > 64 * kRowsAtOnce) each = 64 * kRowsAtOnce;
            args.waveRows = static_cast<int32_t>(each);
            const int64_t groups = (args.sequences.rows + each * kGradWaves - 1) / (each * kGradWaves);
            if (sigmoid) hipLaunchKernelGGL((GatingGradKernel<Codec, Out, kLanes, kPieces, true>), GridOf(groups), dim3(kGradThreads), 0, stream, args);
            else hipLaunchKernelGGL((GatingGradKernel<Codec, Out, kLanes, kPieces, false>), GridOf(groups), dim3(kGradThreads), 0, stream, args);
        });
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.sequences.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("gating_grad", stream);
        if (dtype == ACL_FLOAT) Launch<F32, F32>(stream);
        else if (dtype == ACL_FLOAT16) outType == ACL_FLOAT ? Launch<F16, F32>(stream) : Launch<F16, F16>(stream);
        else outType == ACL_FLOAT ? Launch<Bf16, F32>(stream) : Launch<Bf16, Bf16>(stream);
        const hipError_t err = hipGetLastError();
        OPAPI_CHECK(err == hipSuccess, ACLNN_ERR_RUNTIME_ERROR, "aclnnMoeGatingTopKGroupedGrad: launch failed: %s", hipGetErrorString(err));
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeGatingTopKGroupedGradGetWorkspaceSize(
    const aclTensor* x, const aclTensor* expertIdx, const aclTensor* yGradOptional, const aclTensor* lossGradOptional, const aclTensor* countsOptional,
    const aclTensor* rowsOptional, const aclTensor* seqOffsetsOptional, int64_t scoreType, int64_t renorm, double routedScalingFactor, double eps,
    const aclTensor* xGradOut, uint64_t* workspaceSize, aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(expertIdx, "expertIdx");
    OPAPI_CHECK_NOTNULL(xGradOut, "xGradOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, expertIdx, yGradOptional, lossGradOptional, countsOptional, rowsOptional, seqOffsetsOptional, xGradOut);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    int64_t rows = 0, experts = 0, k = 0, sequences = 0;
    const aclnnStatus router = CheckRouterRows(x, expertIdx, seqOffsetsOptional, scoreType, &rows, &experts, &k, &sequences);
    if (router != ACLNN_SUCCESS) return router;
    OPAPI_CHECK(renorm == 0 || renorm == 1, kInvalid, "renorm (=%lld) must be 0 or 1", (long long)renorm);
    OPAPI_CHECK(std::isfinite(static_cast<float>(routedScalingFactor)), kInvalid, "routedScalingFactor must be a finite number");
    OPAPI_CHECK(eps >= 0 && eps <= 1e30, kInvalid, "eps must be a number of at least 0");
    const bool balance = lossGradOptional != nullptr;
    OPAPI_CHECK(balance == (countsOptional != nullptr) && balance == (rowsOptional != nullptr), ACLNN_ERR_PARAM_NULLPTR,
                "lossGrad, counts and rows belong together");
    OPAPI_CHECK(balance || yGradOptional != nullptr, ACLNN_ERR_PARAM_NULLPTR, "neither yGrad nor lossGrad is given");
    OPAPI_CHECK(balance || seqOffsetsOptional == nullptr, kInvalid, "seqOffsets belongs to lossGrad, which is not given");
    OPAPI_CHECK(yGradOptional == nullptr || ((yGradOptional->dtype == x->dtype || yGradOptional->dtype == ACL_FLOAT) && SameButLast(yGradOptional, x, k)),
                kInvalid, "yGrad %s must be of x's type or FLOAT and of expertIdx's extents %s", ShapeStr(yGradOptional).c_str(), ShapeStr(expertIdx).c_str());
    if (balance) {
        OPAPI_CHECK(lossGradOptional->dtype == ACL_FLOAT && HasExtents(lossGradOptional, {sequences}), kInvalid, "lossGrad %s must be FLOAT [%lld]",
                    ShapeStr(lossGradOptional).c_str(), (long long)sequences);
        OPAPI_CHECK(countsOptional->dtype == ACL_INT32 && HasExtents(countsOptional, {sequences, experts}), kInvalid, "counts %s must be INT32 [%lld,%lld]",
                    ShapeStr(countsOptional).c_str(), (long long)sequences, (long long)experts);
        OPAPI_CHECK(rowsOptional->dtype == ACL_INT32 && HasExtents(rowsOptional, {sequences}), kInvalid, "rows %s must be INT32 [%lld]",
                    ShapeStr(rowsOptional).c_str(), (long long)sequences);
    }
    OPAPI_CHECK((xGradOut->dtype == x->dtype || xGradOut->dtype == ACL_FLOAT) && SameButLast(xGradOut, x, experts), kInvalid,
                "xGradOut %s must be of x's type or FLOAT and of x's extents %s", ShapeStr(xGradOut).c_str(), ShapeStr(x).c_str());
    const aclnnStatus memory =
        CheckMemory({x, expertIdx, yGradOptional, lossGradOptional, countsOptional, rowsOptional, seqOffsetsOptional}, {xGradOut});
    if (memory != ACLNN_SUCCESS) return memory;

    auto* ex = new (std::nothrow) GatingGradExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    GradArgs& a = ex->args;
    ex->dtype = x->dtype;
    ex->outType = xGradOut->dtype;
    ex->sigmoid = scoreType == 1;
    OPAPI_BIND(ex, x, &a.x);
    OPAPI_BIND(ex, expertIdx, &a.expertIdx);
    OPAPI_BIND(ex, yGradOptional, &a.yGrad);
    OPAPI_BIND(ex, lossGradOptional, &a.lossGrad);
    OPAPI_BIND(ex, countsOptional, &a.counts);
    OPAPI_BIND(ex, rowsOptional, &a.seqRows);
    OPAPI_BIND(ex, seqOffsetsOptional, &a.sequences.offsets);
    a.sequences.isInt64 = seqOffsetsOptional != nullptr && seqOffsetsOptional->dtype == ACL_INT64;
    a.sequences.count = static_cast<int32_t>(sequences);
    a.sequences.rows = rows;
    a.xGrad = DataPtr(xGradOut);
    a.experts = static_cast<int32_t>(experts);
    a.k = static_cast<int32_t>(k);
    a.yGradIsFloat = yGradOptional != nullptr && yGradOptional->dtype == ACL_FLOAT;
    a.renorm = static_cast<int32_t>(renorm);
    a.factor = static_cast<float>(routedScalingFactor);
    a.eps = static_cast<float>(eps);
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeGatingTopKGroupedGrad(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
