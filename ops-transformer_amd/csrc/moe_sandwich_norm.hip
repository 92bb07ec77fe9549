// aclnnMoeSandwichNorm for gfx950: s = a residual + b gate * (rms_norm(x) * postGamma), n = rms_norm(s) * preGamma, int8 rows of n * smooth.
//
// Two reductions over a row, the second on what the first one settles: the row stays in registers from its load to its last output, so it crosses the
// memory once, and the memory bounds it: 8192 x 7168 bf16 with a gate per channel (470 MB) 87.5 us a call, 5.37 TB/s, part of them from the memory-side cache
// (89.2 the traced kernel); 4096 x 12000 77.3 (393 MB, 5.1 TB/s); 64 x 4096 a launch, 5.0.  Rows of 16 bits off the four-byte grid take 1.3 times as long
// (4096 x 7167 59.7, where their bytes take 45): their loads and stores of eight elements straddle words.  int8 rows take longer than their bytes, too (8192 x 7168
// in place of 16-bit ones 113 us).  Sums, factors, u, v and n are fp32; what is rounded is s (to the stream's type, and that rounded value is what is normalised),
// n where it leaves, and y, which is made as aclnnMoeAddRmsNormQuant makes it (norm_rows.h).
#include "sandwich_norm.h"

#include "aclnnop/aclnn_moe_sandwich_norm.h"

namespace {

using namespace moe_front;

struct SandwichArgs {
    const void* x;
    const void* residual;
    const void* post;      // optional
    const void* gate;      // optional
    const void* pre;       // optional
    const float* smooth;   // optional
    void* sum;             // may be x's or residual's memory
    void* norm;            // optional
    int8_t* y;             // optional, with scale
    float* scale;
    float* postRstd;       // optional
    float* preRstd;        // optional
    int64_t rows;
    int64_t cols;
    int32_t gateKind;
    int32_t sigmoid;
    int32_t gateIsFloat;
    float residualScale;
    float branchScale;
    float eps;
};

__device__ __forceinline__ float FactorOf(float sumSquares, int64_t cols, float eps) {
    const float mean = sumSquares / static_cast<float>(cols) + eps;
    return mean == 0.f ? 0.f : 1.f / sqrtf(mean);
}

template <typename Codec>
__device__ __forceinline__ float RowGate(const SandwichArgs& a, int64_t row) {
    if (a.gateKind != kGateRow) return 1.f;
    const float raw = a.gateIsFloat ? static_cast<const float*>(a.gate)[row] : Codec::Load(static_cast<const typename Codec::Storage*>(a.gate)[row]);
    return Gated(raw, a.sigmoid);
}

// Rows in pieces of eight elements, up to kPackets of them a lane; a workgroup takes every gridDim.x-th row and asks for the next one before the
// present one is begun (where the registers hold both, else before it is reduced the second time).  Gammas and a gate per channel stay in registers.
// Up to 4096 values a lane has one piece, up to 12288 two on up to 768 lanes, up to 16384 four on 512: four of 9000 columns' take 71.5 us at 4096 rows
// where two take 60.9, and more than 768 lanes have no registers for two.

template <typename Codec, int kPackets, bool kGate>
struct NormRows {
    Packet<Codec> x[kPackets], residual[kPackets], gate[kGate ? kPackets : 1];
    float rowGate = 1.f;
};

template <typename Codec, typename Gamma, int kPackets, int kThreads, int kGate, bool kTail>
__global__ __launch_bounds__(kThreads) void SandwichPacketsKernel(SandwichArgs a) {
    using Storage = typename Codec::Storage;
    constexpr int kMaxWaves = kThreads / kWave;
    constexpr bool kHeld = kGate == kHeldPackets, kRead = kGate == kReadPackets;
    constexpr bool kEarly = kPackets == 1 || (kPackets == 2 && sizeof(Storage) == 2);
    __shared__ float postSums[2][kMaxWaves][1];
    __shared__ float2 partial[2][kMaxWaves];
    const int threads = blockDim.x, waves = threads / kWave, tid = threadIdx.x;
    const int cols = static_cast<int>(a.cols);
    const bool post = a.post != nullptr, pre = a.pre != nullptr;
    const Pieces<kPackets, kTail> at(cols, threads, tid);
    Packet<Gamma> postGamma[kPackets], preGamma[kPackets], gateHeld[kHeld ? kPackets : 1];
#pragma unroll
    for (int p = 0; p < kPackets; ++p) {
        if (post) postGamma[p] = at.template Load<Gamma>(a.post, 0, p);
        if (pre) preGamma[p] = at.template Load<Gamma>(a.pre, 0, p);
        if constexpr (kHeld) gateHeld[p] = at.template Load<Gamma>(a.gate, 0, p);
    }
    using Rows = NormRows<Codec, kPackets, kRead>;
    auto load = [&](Rows& to, int64_t row) {
        const int64_t begin = row * cols;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            to.x[p] = at.template Load<Codec>(a.x, begin, p);
            to.residual[p] = at.template Load<Codec>(a.residual, begin, p);
            if constexpr (kRead) to.gate[p] = at.template Load<Codec>(a.gate, begin, p);
        }
        if constexpr (kGate == kNoPackets) to.rowGate = RowGate<Codec>(a, row);
    };
    int64_t row = blockIdx.x;
    // One row; `following` takes the next one where it is asked for early, else `in` does.
    auto step = [&](Rows& in, Rows& following, int parity) __attribute__((always_inline)) {
        const int64_t begin = row * cols, next = row + gridDim.x;
        if constexpr (kEarly) load(following, min(next, a.rows - 1));
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            HoldPacked<Gamma>(postGamma[p]);
            HoldPacked<Gamma>(preGamma[p]);
            if constexpr (kHeld) HoldPacked<Gamma>(gateHeld[p]);
        }
        float postRstd = 0.f;
        if (post) {
            float squares[1] = {0.f};
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                float v[8], part = 0.f;
                Unpack<Codec>(in.x[p], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float own = at.Own(v[i], p, i);
                    part = fmaf(own, own, part);
                }
                squares[0] += at.Counted(part, p);
            }
            SumsOverGroup<1, kMaxWaves>(squares, waves, parity, postSums);
            postRstd = FactorOf(squares[0], a.cols, a.eps);
            if (a.postRstd != nullptr && tid == 0) a.postRstd[row] = postRstd;
        }
        Packet<Codec> s[kPackets];
        float sumSquares = 0.f;
        uint32_t maxBits = 0;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            float v[8], w[8], g[8];
            Unpack<Codec>(in.x[p], v);
            Unpack<Codec>(in.residual[p], w);
            if (post) {
                Unpack<Gamma>(postGamma[p], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] * postRstd * g[i];
            }
            if constexpr (kHeld) {
                Unpack<Gamma>(gateHeld[p], g);
                OpenGates(g, a.sigmoid);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= g[i];
            } else if constexpr (kRead) {
                Unpack<Codec>(in.gate[p], g);
                OpenGates(g, a.sigmoid);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= g[i];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= in.rowGate;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(a.residualScale, w[i], a.branchScale * v[i]);
            s[p] = Pack<Codec>(v);
            at.template StoreOwn<Storage>(a.sum, begin, p, s[p]);  // it may lie where another lane has yet to read what is not its own
            if (!pre) continue;
            Unpack<Codec>(s[p], v);
            Unpack<Gamma>(preGamma[p], g);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float own = at.Own(v[i], p, i);  // twice: of another lane's element there may be an infinite value here, made of its sum in place
                part = fmaf(own, own, part);
            }
            sumSquares += at.Counted(part, p);
            if (a.y != nullptr) {
                float smooth[8];
                if (a.smooth != nullptr) {
                    Unpack<F32>(at.template Load<F32>(a.smooth, 0, p), smooth);
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] *= smooth[i];
                }
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(fabsf(at.Own(v[i] * g[i], p, i))));
                if (kTail || at.skip[p] == 0) maxBits = max(maxBits, most);
            }
        }
        if constexpr (!kEarly) {
            __builtin_amdgcn_sched_barrier(0);  // not in front of the last uses
            load(in, min(next, a.rows - 1));
        }
        if (pre) {
            sumSquares = SumOver<kWave>(sumSquares);
            if (a.y != nullptr) maxBits = WaveMax(maxBits);
            if (waves > 1) {
                if (tid % kWave == 0) partial[parity][tid / kWave] = float2{sumSquares, __uint_as_float(maxBits)};
                __syncthreads();  // two buffers in turn: one barrier a reduction
                sumSquares = partial[parity][0].x;
                maxBits = __float_as_uint(partial[parity][0].y);
                for (int w = 1; w < waves; ++w) {
                    sumSquares += partial[parity][w].x;
                    maxBits = max(maxBits, __float_as_uint(partial[parity][w].y));
                }
            }
            const RowScales scales = ScalesOf(sumSquares, maxBits, a.cols, a.eps);
            if (tid == 0) {
                if (a.preRstd != nullptr) a.preRstd[row] = scales.r;
                if (a.scale != nullptr) a.scale[row] = scales.scale;
            }
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                float v[8], g[8];
                Unpack<Codec>(s[p], v);
                Unpack<Gamma>(preGamma[p], g);
                if (a.norm != nullptr) {
                    float n[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) n[i] = v[i] * scales.r * g[i];
                    at.template StoreOwn<Storage>(a.norm, begin, p, Pack<Codec>(n));
                }
                if (a.y != nullptr) {
                    float smooth[8];
                    if (a.smooth != nullptr) {
                        Unpack<F32>(at.template Load<F32>(a.smooth, 0, p), smooth);
#pragma unroll
                        for (int i = 0; i < 8; ++i) g[i] *= smooth[i];
                    }
                    uint32_t q[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[i / 4] |= (static_cast<uint32_t>(Quantised(v[i] * g[i], scales)) & 0xffu) << (i % 4 * 8);
                    at.template StoreOwn<int8_t>(a.y, begin, p, uint2{q[0], q[1]});
                }
            }
        }
        row = next;
    };
    Rows first;
    load(first, row);
    if constexpr (kEarly) {
        // The two rows take turns where they lie: moved, a row's loads would have to have ended, and the stores behind them.
        Rows second;
        while (true) {
            step(first, second, 0);
            if (row >= a.rows) break;
            step(second, first, 1);
            if (row >= a.rows) break;
        }
    } else {
        for (int parity = 0; row < a.rows; parity ^= 1) step(first, first, parity);
    }
}

// Rows of any length: a workgroup per row, one element at a time, the row read again behind each reduction (from the sum once that is written, by the
// same lane: it may lie in x's or the residual's memory), squares added up in 64 bits.
template <typename Codec, typename Gamma>
__global__ __launch_bounds__(kAnyThreads) void SandwichAnyKernel(SandwichArgs a) {
    using S = typename Codec::Storage;
    __shared__ double sums[kAnyThreads / kWave];
    __shared__ uint32_t maxima[kAnyThreads / kWave];
    const int64_t row = GroupIndex();
    if (row >= a.rows) return;
    const int64_t at = row * a.cols;
    const S* const x = static_cast<const S*>(a.x) + at;
    const S* const residual = static_cast<const S*>(a.residual) + at;
    S* const sum = static_cast<S*>(a.sum) + at;
    auto weight = [&](const void* w, int64_t c) { return Gamma::Load(static_cast<const typename Gamma::Storage*>(w)[c]); };
    float rstd = 0.f;
    if (a.post != nullptr) {
        double squares = 0.0;
        for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
            const double v = Codec::Load(x[c]);
            squares = fma(v, v, squares);
        }
        rstd = FactorOf(static_cast<float>(SumOfGroup(squares, sums)), a.cols, a.eps);
        if (a.postRstd != nullptr && threadIdx.x == 0) a.postRstd[row] = rstd;
    }
    const float rowGate = RowGate<Codec>(a, row);
    double squares = 0.0;
    uint32_t maxBits = 0;
    auto scaled = [&](float s, int64_t c) { return s * weight(a.pre, c) * (a.smooth == nullptr ? 1.f : a.smooth[c]); };
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        float v = Codec::Load(x[c]);
        if (a.post != nullptr) v = v * rstd * weight(a.post, c);
        if (a.gateKind == kGateChannel) v *= Gated(weight(a.gate, c), a.sigmoid);
        else if (a.gateKind == kGateEach) v *= Gated(Codec::Load(static_cast<const S*>(a.gate)[at + c]), a.sigmoid);
        else v *= rowGate;
        const S raw = Codec::Store(fmaf(a.residualScale, Codec::Load(residual[c]), a.branchScale * v));
        sum[c] = raw;
        if (a.pre == nullptr) continue;
        const float s = Codec::Load(raw);
        squares = fma(static_cast<double>(s), static_cast<double>(s), squares);
        if (a.y != nullptr) maxBits = max(maxBits, __float_as_uint(fabsf(scaled(s, c))));
    }
    if (a.pre == nullptr) return;
    squares = SumOfGroup(squares, sums);
    maxBits = WaveMax(maxBits);
    if (threadIdx.x % kWave == 0) maxima[threadIdx.x / kWave] = maxBits;
    __syncthreads();
    for (int w = 0; w < kAnyThreads / kWave; ++w) maxBits = max(maxBits, maxima[w]);
    const RowScales scales = ScalesOf(static_cast<float>(squares), maxBits, a.cols, a.eps);
    if (threadIdx.x == 0) {
        if (a.preRstd != nullptr) a.preRstd[row] = scales.r;
        if (a.scale != nullptr) a.scale[row] = scales.scale;
    }
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        const float s = Codec::Load(sum[c]);
        if (a.norm != nullptr) static_cast<S*>(a.norm)[at + c] = Codec::Store(s * scales.r * weight(a.pre, c));
        if (a.y != nullptr) a.y[at + c] = static_cast<int8_t>(Quantised(scaled(s, c), scales));
    }
}

class SandwichExecutor : public aclOpExecutor {
   public:
    SandwichArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType weightType = ACL_FLOAT;

    template <typename Codec, typename Gamma, int kPackets, int kThreads, int kGate>
    void LaunchPackets(hipStream_t stream) const {
        const int64_t lanes = ((args.cols + 7) / 8 + kPackets - 1) / kPackets;
        const int threads = static_cast<int>((lanes + kWave - 1) / kWave * kWave);
        const bool tail = args.cols % 8 != 0;
        // Workgroups a CU.  One piece: 16 waves, and three workgroups of five or six (8192 x 2880 38.5 us, with two of six 42.9, with four 39.3; with a gate a row
        // 42.7, 53.4 and 42.4; 8192 x 4096 38.4 with two, with one 42.6, with four 41; 8192 x 1024 13.2 with eight, with ten 14.3).  Two: 12 waves (8192 x 7168
        // 87.9 with one workgroup, with two 93.1; 8192 x 4608 59.9 with two, with three 67.7), and two workgroups where the tail's instructions want company
        // (4096 x 7167 63.0, with one 82).
        const int64_t each = kPackets == 1                     ? (threads > 4 * kWave ? 18 : 16) * kWave / threads
                             : tail && kThreads == kFewThreads ? 2
                                                               : std::max(1, 12 * kWave / threads);
        const int64_t groups = std::min<int64_t>(args.rows, kCus * each);
        const dim3 grid(static_cast<unsigned>(groups));
        if (tail) hipLaunchKernelGGL((SandwichPacketsKernel<Codec, Gamma, kPackets, kThreads, kGate, true>), grid, dim3(threads), 0, stream, args);
        else hipLaunchKernelGGL((SandwichPacketsKernel<Codec, Gamma, kPackets, kThreads, kGate, false>), grid, dim3(threads), 0, stream, args);
    }

    template <typename Codec, typename Gamma, int kPackets, int kThreads>
    void ForGate(hipStream_t stream) const {
        const int packets = GatePackets(args.gateKind);
        if (packets == kHeldPackets) LaunchPackets<Codec, Gamma, kPackets, kThreads, kHeldPackets>(stream);
        else if (packets == kReadPackets) LaunchPackets<Codec, Gamma, kPackets, kThreads, kReadPackets>(stream);
        else LaunchPackets<Codec, Gamma, kPackets, kThreads, kNoPackets>(stream);
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("sandwich_norm", stream);
        ForTypes(dtype, weightType, [&](auto codec, auto gamma) {
            using Codec = decltype(codec);
            using Gamma = decltype(gamma);
            const int64_t lanes = (args.cols + 7) / 8;
            if (args.cols < 8 || args.cols > kPacketCols) {
                hipLaunchKernelGGL((SandwichAnyKernel<Codec, Gamma>), GridOf(args.rows), dim3(kAnyThreads), 0, stream, args);
            } else if (lanes <= kFewThreads) {
                ForGate<Codec, Gamma, 1, kFewThreads>(stream);
            } else if (lanes <= 2 * kFewThreads) {
                ForGate<Codec, Gamma, 2, kFewThreads>(stream);
            } else if (lanes <= 2 * kManyThreads) {
                ForGate<Codec, Gamma, 2, kManyThreads>(stream);
            } else {
                ForGate<Codec, Gamma, kMaxPackets, kFewThreads>(stream);
            }
        });
        const hipError_t err = hipGetLastError();
        OPAPI_CHECK(err == hipSuccess, ACLNN_ERR_RUNTIME_ERROR, "aclnnMoeSandwichNorm: launch failed: %s", hipGetErrorString(err));
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeSandwichNormGetWorkspaceSize(
    const aclTensor* x, const aclTensor* residual, const aclTensor* postGammaOptional, const aclTensor* gateOptional, const aclTensor* preGammaOptional,
    const aclTensor* smoothScaleOptional, int64_t gateType, double residualScale, double branchScale, double epsilon, const aclTensor* sumOut,
    const aclTensor* normOutOptional, const aclTensor* yOutOptional, const aclTensor* scaleOutOptional, const aclTensor* postRstdOutOptional,
    const aclTensor* preRstdOutOptional, uint64_t* workspaceSize, aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(residual, "residual");
    OPAPI_CHECK_NOTNULL(sumOut, "sumOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, residual, postGammaOptional, gateOptional, preGammaOptional, smoothScaleOptional, sumOut, normOutOptional, yOutOptional,
                        scaleOutOptional, postRstdOutOptional, preRstdOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    SandwichShape shape;
    const aclnnStatus checked = CheckSandwich(x, postGammaOptional, gateOptional, preGammaOptional, gateType, residualScale, branchScale, &shape);
    if (checked != ACLNN_SUCCESS) return checked;
    OPAPI_CHECK(epsilon >= 0 && epsilon <= 1e30, kInvalid, "epsilon must be a number of at least 0");
    OPAPI_CHECK(Like(residual, x), kInvalid, "residual %s must have x's type and extents %s", ShapeStr(residual).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(Like(sumOut, x), kInvalid, "sumOut %s must have x's type and extents %s", ShapeStr(sumOut).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(Like(normOutOptional, x), kInvalid, "normOut %s must have x's type and extents %s", ShapeStr(normOutOptional).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK((yOutOptional == nullptr) == (scaleOutOptional == nullptr), ACLNN_ERR_PARAM_NULLPTR, "yOut and scaleOut belong together");
    OPAPI_CHECK(yOutOptional == nullptr || (yOutOptional->dtype == ACL_INT8 && SameButLast(yOutOptional, x, shape.cols)), kInvalid,
                "yOut %s must be INT8 of x's extents %s", ShapeStr(yOutOptional).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(PerRow(scaleOutOptional, x), kInvalid, "scaleOut %s must be FLOAT of x's extents %s without the last", ShapeStr(scaleOutOptional).c_str(),
                ShapeStr(x).c_str());
    OPAPI_CHECK(PerRow(postRstdOutOptional, x), kInvalid, "postRstdOut %s must be FLOAT of x's extents %s without the last",
                ShapeStr(postRstdOutOptional).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(PerRow(preRstdOutOptional, x), kInvalid, "preRstdOut %s must be FLOAT of x's extents %s without the last",
                ShapeStr(preRstdOutOptional).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(smoothScaleOptional == nullptr || (smoothScaleOptional->dtype == ACL_FLOAT && HasExtents(smoothScaleOptional, {shape.cols})), kInvalid,
                "smoothScale must be FLOAT [%lld]", (long long)shape.cols);
    OPAPI_CHECK(yOutOptional != nullptr || smoothScaleOptional == nullptr, kInvalid, "smoothScale goes into yOut, which is not given");
    OPAPI_CHECK(preGammaOptional != nullptr || (normOutOptional == nullptr && yOutOptional == nullptr && preRstdOutOptional == nullptr), kInvalid,
                "normOut, yOut and preRstdOut are of the norm with preGamma, which is not given");
    OPAPI_CHECK(preGammaOptional == nullptr || normOutOptional != nullptr || yOutOptional != nullptr || preRstdOutOptional != nullptr, ACLNN_ERR_PARAM_NULLPTR,
                "preGamma is given, but none of its norm's outputs");
    OPAPI_CHECK(postGammaOptional != nullptr || postRstdOutOptional == nullptr, kInvalid, "postRstdOut is of the norm with postGamma, which is not given");
    const aclTensor* const apart[] = {normOutOptional, yOutOptional, scaleOutOptional, postRstdOutOptional, preRstdOutOptional};
    const aclnnStatus memory =
        CheckMemory({x, residual, postGammaOptional, gateOptional, preGammaOptional, smoothScaleOptional}, {apart[0], apart[1], apart[2], apart[3], apart[4]});
    if (memory != ACLNN_SUCCESS) return memory;
    OPAPI_CHECK(InOrder(sumOut), kInvalid, "the outputs must be contiguous");
    OPAPI_CHECK(IsEmpty(sumOut) || sumOut->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an output carries no device memory");
    for (const aclTensor* out : apart) OPAPI_CHECK(!Overlap(out, sumOut), kInvalid, "two outputs share memory");
    for (const aclTensor* in : {x, residual, postGammaOptional, gateOptional, preGammaOptional, smoothScaleOptional}) {
        if (in == nullptr || !IsContiguous(in)) continue;
        const bool inPlace = (in == x || in == residual) && DataPtr(in) == DataPtr(sumOut);
        OPAPI_CHECK(inPlace || !Overlap(sumOut, in), kInvalid, "an output shares memory with an input");
    }

    auto* ex = new (std::nothrow) SandwichExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    SandwichArgs& a = ex->args;
    ex->dtype = x->dtype;
    ex->weightType = shape.weightType;
    OPAPI_BIND(ex, x, &a.x);
    OPAPI_BIND(ex, residual, &a.residual);
    OPAPI_BIND(ex, postGammaOptional, &a.post);
    OPAPI_BIND(ex, gateOptional, &a.gate);
    OPAPI_BIND(ex, preGammaOptional, &a.pre);
    OPAPI_BIND(ex, smoothScaleOptional, &a.smooth);
    a.sum = DataPtr(sumOut);
    a.norm = DataPtr(normOutOptional);
    a.y = reinterpret_cast<int8_t*>(DataPtr(yOutOptional));
    a.scale = reinterpret_cast<float*>(DataPtr(scaleOutOptional));
    a.postRstd = reinterpret_cast<float*>(DataPtr(postRstdOutOptional));
    a.preRstd = reinterpret_cast<float*>(DataPtr(preRstdOutOptional));
    a.rows = shape.rows;
    a.cols = shape.cols;
    a.gateKind = shape.gateKind;
    a.gateIsFloat = shape.gateIsFloat;
    a.sigmoid = static_cast<int32_t>(gateType);
    a.residualScale = static_cast<float>(residualScale);
    a.branchScale = static_cast<float>(branchScale);
    a.eps = static_cast<float>(epsilon);
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeSandwichNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
