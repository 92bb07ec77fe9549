// aclnnMoeGatingTopKGroupedGrad for gfx950: the gradients of picked weights and of the balance loss with respect to the logits.
//
// Both are a row's scores times something less a mean, and the scores are made anew from the logits: one read and one write of a row.  With t = sum p + eps of
// the picked ones, q_j = p_j / t and M = sum dy_j q_j, the renormalised weights have p_j dp_j = F q_j (dy_j - M), and the mean of dp under the softmax is
// F M (1 - sum p / t) = F M eps / t: formed so, it is not the difference of two sums that cancel.  The picks' p dp goes through LDS from the lane that has
// the pick to the one that has the expert.
//
// What bounds it: few rows, a launch and two round trips (256 x 8: 4.4 us, most of it the host's); many, no one thing (16384 x 256 fp32: 10.4 us, where the
// bytes, 34.6 MB, take 6.7 at a copy's rate): a score is six instructions, its gradient ten, and four sums cross the lanes, together 62 % of the SIMDs'
// issue; and the waves wait 52 % of their cycles, for those sums and for the offsets and then the sequence's tables in front of their four rows.
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
    float expertsPerPick;      // experts / k, and the other way round
    float picksPerExpert;
    int32_t waveRows;          // rows of a wave, one behind the other
};

constexpr int kGradThreads = 256;
constexpr int kGradWaves = kGradThreads / kWave;

// What is asked for of a row before the one in front of it is done.
template <typename Raw>
struct RowInputs {
    Raw x;
    int32_t first;  // its first id
    int32_t id;     // the lane's pick, the first of its own where a row has more picks than lanes, and its gradient
    float y;
};

// A row has the fewest lanes that hold it, four experts each, as the balance's kernel has it, and a wave's rows follow each other, the next asked for before the
// present one is done.  Scores are held unnormalised, so that their sum, that of the picked ones and both means are reduced side by side.
template <typename Codec, typename Out, int kLanes, int kPieces, bool kSigmoid>
__global__ __launch_bounds__(kGradThreads) void GatingGradKernel(GradArgs a) {
    using Row = RowOf<kLanes, kPieces>;
    constexpr int kEach = Row::kEach;
    constexpr int kRowsAtOnce = kWave / kLanes;
    __shared__ float4 scores[kGradWaves][kRowsAtOnce][Row::kWidth / 4];
    __shared__ float4 picked[kGradWaves][kRowsAtOnce][Row::kWidth / 4];  // zero between rows
    using X = typename Codec::Storage;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, l = lane % kLanes, side = lane / kLanes;
    const float* const scoreOf = reinterpret_cast<const float*>(scores[wave][side]);
    float* const pickedOf = reinterpret_cast<float*>(picked[wave][side]);
    const bool weights = a.yGrad != nullptr, balance = a.lossGrad != nullptr;
    auto isExpert = [&](int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts); };
    // The rows of a wave follow each other, `side` by side: their sequence changes seldom, and with it the counts in registers.
    const int64_t first = (GroupIndex() * kGradWaves + wave) * a.waveRows;
    if (first >= a.sequences.rows) return;
    const int32_t rows = static_cast<int32_t>(min(static_cast<int64_t>(a.waveRows), a.sequences.rows - first));
    // What the wave's rows begin at, and the lane's own row behind those of the ones beside it.
    const X* const xRows = static_cast<const X*>(a.x) + first * a.experts;
    typename Out::Storage* const outRows = static_cast<typename Out::Storage*>(a.xGrad) + first * a.experts;
    const int32_t* const idxRows = a.expertIdx + first * a.k;
    const float* const yRowsFloat = static_cast<const float*>(a.yGrad) + first * a.k;
    const X* const yRows = static_cast<const X*>(a.yGrad) + first * a.k;
    auto yGradOf = [&](uint32_t at) { return a.yGradIsFloat ? yRowsFloat[at] : Codec::Load(yRows[at]); };
    using Inputs = RowInputs<typename Row::template Raw<X>>;
    Inputs in;
    auto load = [&](int32_t row) {
        const uint32_t pick = static_cast<uint32_t>(row) * static_cast<uint32_t>(a.k);
        in.x = Row::Ask(xRows, static_cast<uint32_t>(row) * static_cast<uint32_t>(a.experts), a.experts, l);
        in.first = idxRows[pick];
        in.id = -1;
        in.y = 0.f;
        if (weights && l < a.k) {
            in.id = idxRows[pick + l];
            in.y = yGradOf(pick + l);
        }
    };
    if (side < rows) load(side);
    if (weights) {
#pragma unroll
        for (int p = 0; p < kPieces; ++p) picked[wave][side][Row::At(p, l) / 4] = float4{0.f, 0.f, 0.f, 0.f};
    }
    int32_t sequence = -2;     // of the row, and where it ends, from the wave's first row on
    int32_t sequenceEnd = -1;
    bool inside = false;       // whether it is one
    float shareGrad[kEach];    // what its loss gives each share
#pragma unroll
    for (int i = 0; i < kEach; ++i) shareGrad[i] = 0.f;
    // The loads of a sequence go out together, those of rows in none being of another one's.
    auto enter = [&](int32_t s, int64_t end) {
        sequenceEnd = static_cast<int32_t>(min(end - first, static_cast<int64_t>(1) << 30));
        sequence = s;
        inside = s >= 0 && s < a.sequences.count;
        const int32_t at = s < 0 ? 0 : min(s, a.sequences.count - 1);
        const int32_t live = a.seqRows[at];
        const float lossGrad = a.lossGrad[at];
        const auto raw = Row::Ask(a.counts, static_cast<uint32_t>(at) * static_cast<uint32_t>(a.experts), a.experts, l);
        int32_t counts[kEach];
        Row::Place(raw, a.experts, l, 0, counts);
        const float n = static_cast<float>(live);
        const float each = live > 0 ? lossGrad * a.expertsPerPick / n / n : 0.f;
        // Of the counts, their distances from the even one: what all have alike gives shares, whose sum is 1, nothing, and where a batch is spread as the loss wants it
        // the counts' own products and their mean would cancel.
        const uint32_t even = static_cast<uint32_t>(static_cast<int32_t>(fminf(rintf(n * a.picksPerExpert), 0x1p30f)));
#pragma unroll
        for (int i = 0; i < kEach; ++i) shareGrad[i] = live > 0 ? each * static_cast<float>(static_cast<int32_t>(static_cast<uint32_t>(counts[i]) - even)) : 0.f;
    };
    if (balance) {
        int64_t end, beyond;
        const int32_t s = a.sequences.Of(first, end, beyond);
        enter(s, end);
    }
    for (int32_t base = 0; base < rows; base += kRowsAtOnce) {
        const int32_t row = base + side;
        if (row >= rows) break;  // (the lanes of a row agree)
        if (balance && row >= sequenceEnd && sequence < a.sequences.count) {
            int64_t end;
            const int32_t s = SequenceBehind(a.sequences, sequence, first + row, end);
            enter(s, end);
        }
        const Inputs now = in;
        if (row + kRowsAtOnce < rows) load(row + kRowsAtOnce);
        const uint32_t pick = static_cast<uint32_t>(row) * static_cast<uint32_t>(a.k);
        float x[kEach];
        Row::template Logits<Codec>(now.x, a.experts, l, x);
        // p: sigmoid's score, with rest = 1 - p, or softmax's before its division by the sum
        float p[kEach], rest[kSigmoid ? kEach : 1];
        if constexpr (kSigmoid) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const Sigmoid s = SigmoidOf(x[i]);
                p[i] = s.p;
                rest[i] = s.rest;
            }
        } else {
            const ExpFrom e(TopOf<kLanes>(x));
#pragma unroll
            for (int i = 0; i < kEach; ++i) p[i] = e(x[i]);
        }
        float sum = 0.f, shared = 0.f, score = 0.f, pickedSum = 0.f, weighted = 0.f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            sum += p[i];
            shared = fmaf(shareGrad[i], p[i], shared);
        }
        // The lane's part of the picks' sums, of scores that go through LDS.
        auto pickSums = [&](const float (&s)[kEach]) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < kPieces; ++q) scores[wave][side][Row::At(q, l) / 4] = float4{s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            score = pickedSum = weighted = 0.f;
            if (isExpert(now.id)) {
                score = scoreOf[now.id];
                pickedSum = score;
                weighted = now.y * score;
            }
            for (int j = l + kLanes; j < a.k; j += kLanes) {
                const int32_t id = idxRows[pick + j];
                if (!isExpert(id)) continue;
                pickedSum += scoreOf[id];
                weighted = fmaf(yGradOf(pick + j), scoreOf[id], weighted);
            }
        };
        if (weights) pickSums(p);
        sum = SumOver<kLanes>(sum);
        shared = SumOver<kLanes>(shared);
        if (weights) {
            pickedSum = SumOver<kLanes>(pickedSum);
            weighted = SumOver<kLanes>(weighted);
        }
        float eps = kSigmoid ? a.eps : a.eps * sum;  // beside the picks' scores as they are held
        if (__builtin_expect(weights && a.renorm && pickedSum < kLostSum, 0)) {
            // Rare (the lanes of a row agree): scores, or their products with yGrad, are nearly or wholly lost in fp32.  They are taken from the largest pick
            // then instead of from the row's top, or from 1.  (16384 x 256: 1 % of its time for the branch, 3 % of the weights' alone.)
            const X* const logits = xRows + static_cast<uint32_t>(row) * static_cast<uint32_t>(a.experts);
            float top = isExpert(now.id) ? Codec::Load(logits[now.id]) : -INFINITY;
            for (int j = l + kLanes; j < a.k; j += kLanes) {
                const int32_t id = idxRows[pick + j];
                if (isExpert(id)) top = fmaxf(top, Codec::Load(logits[id]));
            }
            top = MaxOver<kLanes>(top);
            const float up = (kSigmoid ? 0.f : TopOf<kLanes>(x)) - top;  // e^up times as large
            if (up > kLostIn64) {
                pickedSum = 0.f;
            } else {
                const ExpFrom e(top);
                float s[kEach];
#pragma unroll
                for (int i = 0; i < kEach; ++i) s[i] = kSigmoid ? e(x[i]) * rest[i] : e(x[i]);
                pickSums(s);
                pickedSum = SumOver<kLanes>(pickedSum);
                weighted = SumOver<kLanes>(weighted);
                const float half = ExpFrom(-0.5f * up)(0.f);
                eps = a.eps * half * half * (kSigmoid ? 1.f : sum);
                if (a.eps == 0.f) eps = 0.f;
                else if (up > 176.f || !(eps < 1e37f)) eps = pickedSum = 0.f;  // beside eps they are below fp32's range
            }
        }
        const float inverse = sum == 0.f ? 0.f : Reciprocal(sum);
        if constexpr (!kSigmoid) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) p[i] *= inverse;
        }
        float grad[kEach];
        if (weights) {
            // The picked scores are divided once, softmax's by the row's sum or by the picked ones': first by the one and then by the other, small ones
            // would be lost between.
            float mean = 0.f, part = kSigmoid ? 1.f : inverse, all = a.factor * (weighted * part);
            if (a.renorm) {
                part = pickedSum == 0.f ? 0.f : Reciprocal(eps + pickedSum);
                mean = weighted * part;
                all = a.factor * mean * (eps * part);
            }
            if (isExpert(now.id)) atomicAdd(pickedOf + now.id, a.factor * (score * part) * (now.y - mean));
            for (int j = l + kLanes; j < a.k; j += kLanes) {
                const int32_t id = idxRows[pick + j];
                if (isExpert(id)) atomicAdd(pickedOf + id, a.factor * (scoreOf[id] * part) * (yGradOf(pick + j) - mean));
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
                    if constexpr (kSigmoid) grad[4 * q + i] = d[i] * rest[4 * q + i];
                    else grad[4 * q + i] = fmaf(p[4 * q + i], -all, d[i]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) grad[i] = 0.f;
        }
        if (balance && inside) {
            float share[kEach], mean = shared * inverse;
#pragma unroll
            for (int i = 0; i < kEach; ++i) share[i] = kSigmoid ? p[i] * inverse : p[i];
            if (kSigmoid && sum < kLostSum) {  // (the lanes of a row agree)
                LostSharesOf<kLanes>(x, share);
                mean = 0.f;
#pragma unroll
                for (int i = 0; i < kEach; ++i) mean = fmaf(shareGrad[i], share[i], mean);
                mean = SumOver<kLanes>(mean);
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const float d = shareGrad[i] - mean;
                if constexpr (kSigmoid) grad[i] = fmaf(share[i] * rest[i], d, grad[i]);
                else grad[i] = fmaf(share[i], d, grad[i]);
            }
        }
        const bool live = isExpert(now.first);
#pragma unroll
        for (int i = 0; i < kEach; ++i) grad[i] = live ? grad[i] : 0.f;
        Row::template Store<Out>(outRows, static_cast<uint32_t>(row) * static_cast<uint32_t>(a.experts), a.experts, l, grad);
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
            // Four waves for each of the 256 x 4 SIMDs: 16384 x 256 10.4 us, half as many 12.9, twice 10.9, four times 12.3.
            const int64_t waves = 4 * 1024;
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
    a.expertsPerPick = static_cast<float>(experts) / static_cast<float>(k);
    a.picksPerExpert = static_cast<float>(k) / static_cast<float>(experts);
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
