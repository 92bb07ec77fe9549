// aclnnMoeSandwichNormGrad for gfx950: from the gradients of the sum and of its norm to those of the block's output, the residual, both gammas and the gate.
//
// With x^ = x postRstd and s^ = s preRstd a row needs one sum behind the other, sum(dn preGamma s^) for dS and sum(du postGamma x^) for xGrad: it stays in
// registers from its loads to its stores.  A workgroup takes every gridDim.x-th row and adds up what its lanes' columns owe the gammas and a gate per
// channel in registers; a second kernel adds up the workgroups.
#include "sandwich_norm.h"

#include "aclnnop/aclnn_moe_sandwich_norm_grad.h"

namespace {

using namespace moe_front;

// Column sums, by their place in the workspace.
enum { kPostSums, kPreSums, kGateSums, kColumnSums };

struct SandwichGradArgs {
    const void* x;           // read where there is a post norm or a gate
    const void* s;           // with norm, pre and preRstd
    const void* sumGrad;     // optional
    const void* normGrad;
    const void* post;        // optional, with postRstd
    const void* gate;        // optional
    const void* pre;
    const float* postRstd;
    const float* preRstd;
    void* xGrad;             // optional
    void* residualGrad;      // optional
    void* gateGrad;          // optional
    float* columnGrads[kColumnSums];  // outputs, optional
    float* columnSums[kColumnSums];   // workspace: [groups, cols] each
    float* rowMeans;         // workspace of rows in two passes: [rows, 2]
    int64_t rows;
    int64_t cols;
    int64_t groups;          // that columns are summed over
    int32_t gateKind;
    int32_t sigmoid;
    int32_t gateIsFloat;
    float residualScale;
    float branchScale;
};

// d g / d gate, of g = Gated(gate).
__device__ __forceinline__ float GateSlope(float gate, int sigmoid) {
    if (!sigmoid) return 1.f;
    const Sigmoid s = SigmoidOf(gate);
    return s.p * s.rest;
}
template <typename Codec>
__device__ __forceinline__ float RawRowGate(const SandwichGradArgs& a, int64_t row) {
    return a.gateIsFloat ? static_cast<const float*>(a.gate)[row] : Codec::Load(static_cast<const typename Codec::Storage*>(a.gate)[row]);
}

constexpr int kMaxPacketThreads = 512;

template <typename Codec, typename Gamma, int kPackets, int kGate>
__global__ __launch_bounds__(kMaxPacketThreads) void SandwichGradKernel(SandwichGradArgs a) {
    using P = Packet<Codec>;
    using Storage = typename Codec::Storage;
    constexpr int kMaxWaves = kMaxPacketThreads / kWave;
    constexpr bool kHeld = kGate == kHeldPackets, kRead = kGate == kReadPackets;
    __shared__ float preSums[2][kMaxWaves][1];
    __shared__ float postSums[2][kMaxWaves][2];
    const int threads = blockDim.x, waves = threads / kWave, tid = threadIdx.x;
    const int cols = static_cast<int>(a.cols);
    const float each = 1.f / static_cast<float>(a.cols);
    const bool post = a.post != nullptr, pre = a.pre != nullptr, gated = a.gateKind != kGateNone, rowGated = a.gateKind == kGateRow;
    const bool needsX = post || gated, sums = a.sumGrad != nullptr;
    P x[kPackets], s[kPackets], sumGrad[kPackets], normGrad[kPackets], gateRow[kRead ? kPackets : 1];
    Packet<Gamma> postGamma[kPackets], preGamma[kPackets];
    float gateHeld[kHeld ? kPackets : 1][8];
    float postSum[kPackets][8], preSum[kPackets][8], gateSum[kHeld ? kPackets : 1][8];
    float postRstd = 1.f, preRstd = 0.f, rawGate = 0.f;
    bool here[kPackets];
    auto at = [&](int p) { return (p * threads + tid) * 8; };
    auto count = [&](int p) { return min(cols - at(p), 8); };
#pragma unroll
    for (int p = 0; p < kPackets; ++p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            postSum[p][i] = preSum[p][i] = 0.f;
            if constexpr (kHeld) gateSum[p][i] = 0.f;
        }
        here[p] = at(p) < cols;
        if (!here[p]) continue;
        if (post) postGamma[p] = LoadPacket<false, Gamma>(a.post, at(p), count(p));
        if (pre) preGamma[p] = LoadPacket<false, Gamma>(a.pre, at(p), count(p));
        if constexpr (kHeld) {
            Unpack<Gamma>(LoadPacket<false, Gamma>(a.gate, at(p), count(p)), gateHeld[p]);
#pragma unroll
            for (int i = 0; i < 8; ++i) gateHeld[p][i] = Gated(gateHeld[p][i], a.sigmoid);
        }
    }
    auto load = [&](int64_t row) {
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            const int64_t from = row * cols + at(p);
            if (pre) {
                s[p] = LoadPacket<false, Codec>(a.s, from, count(p));
                normGrad[p] = LoadPacket<false, Codec>(a.normGrad, from, count(p));
            }
            if (sums) sumGrad[p] = LoadPacket<false, Codec>(a.sumGrad, from, count(p));
            if (needsX) x[p] = LoadPacket<false, Codec>(a.x, from, count(p));
            if constexpr (kRead) gateRow[p] = LoadPacket<false, Codec>(a.gate, from, count(p));
        }
        if (post) postRstd = a.postRstd[row];
        if (pre) preRstd = a.preRstd[row];
        if (kGate == kNoPackets && rowGated) rawGate = RawRowGate<Codec>(a, row);
    };
    int64_t row = blockIdx.x;
    if (row < a.rows) load(row);
    for (int parity = 0; row < a.rows; parity ^= 1) {
        // dS
        float d[kPackets][8];
        float preMean[1] = {0.f};
        if (pre) {
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                if (!here[p]) continue;
                float v[8], g[8];
                Unpack<Codec>(s[p], v);
                Unpack<Codec>(normGrad[p], d[p]);
                Unpack<Gamma>(preGamma[p], g);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float normed = v[i] * preRstd;
                    preSum[p][i] = fmaf(d[p][i], normed, preSum[p][i]);
                    d[p][i] *= g[i];
                    preMean[0] = fmaf(d[p][i], normed, preMean[0]);
                }
            }
            SumsOverGroup<1, kMaxWaves>(preMean, waves, parity, preSums);
            preMean[0] *= each;
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                if (!here[p]) continue;
                float v[8];
                Unpack<Codec>(s[p], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[p][i] = preRstd * (d[p][i] - v[i] * preRstd * preMean[0]);
            }
        }
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            if (sums) {
                float v[8];
                Unpack<Codec>(sumGrad[p], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[p][i] = pre ? d[p][i] + v[i] : v[i];
            }
            if (a.residualGrad != nullptr) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = a.residualScale * d[p][i];
                StorePacket<false, Storage>(a.residualGrad, row * cols + at(p), count(p), Pack<Codec>(v));
            }
        }
        // through the gate and the post norm's weights
        const float rowGate = rowGated ? Gated(rawGate, a.sigmoid) : 1.f;
        float rowSums[2] = {0.f, 0.f};  // du postGamma x^, dv u
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            float xs[8], g[8];
            if (needsX) Unpack<Codec>(x[p], xs);
            if (post) Unpack<Gamma>(postGamma[p], g);
            float gateEach[8], gateGrad[8];
            if constexpr (kRead) Unpack<Codec>(gateRow[p], gateEach);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = a.branchScale * d[p][i];
                const float normed = needsX ? xs[i] * postRstd : 0.f;
                const float u = post ? normed * g[i] : normed;
                if constexpr (kHeld) {
                    gateSum[p][i] = fmaf(v, u, gateSum[p][i]);
                    v *= gateHeld[p][i];
                } else if constexpr (kRead) {
                    float open = gateEach[i], slope = 1.f;
                    if (a.sigmoid) {
                        const Sigmoid sg = SigmoidOf(gateEach[i]);
                        open = sg.p;
                        slope = sg.p * sg.rest;
                    }
                    gateGrad[i] = v * u * slope;
                    v *= open;
                } else {
                    rowSums[1] = fmaf(v, u, rowSums[1]);
                    v *= rowGate;
                }
                if (post) {
                    postSum[p][i] = fmaf(v, normed, postSum[p][i]);
                    v *= g[i];
                    rowSums[0] = fmaf(v, normed, rowSums[0]);
                }
                d[p][i] = v;
            }
            if constexpr (kRead) {
                if (a.gateGrad != nullptr) StorePacket<false, Storage>(a.gateGrad, row * cols + at(p), count(p), Pack<Codec>(gateGrad));
            }
        }
        // The row's own values are needed once more: x is unpacked before the next row's loads take its place.
        const float rstd = postRstd, raw = rawGate;
        float xs[kPackets][8];
        if (post) {
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                if (here[p]) Unpack<Codec>(x[p], xs[p]);
            }
        }
        const int64_t next = row + gridDim.x;
        if (next < a.rows) load(next);
        if (post || rowGated) SumsOverGroup<2, kMaxWaves>(rowSums, waves, parity, postSums);
        if (rowGated && a.gateGrad != nullptr && tid == 0) static_cast<float*>(a.gateGrad)[row] = rowSums[1] * GateSlope(raw, a.sigmoid);
        if (a.xGrad != nullptr) {
            const float mean = rowSums[0] * each;
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                if (!here[p]) continue;
                if (post) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[p][i] = rstd * (d[p][i] - xs[p][i] * rstd * mean);
                }
                StorePacket<false, Storage>(a.xGrad, row * cols + at(p), count(p), Pack<Codec>(d[p]));
            }
        }
        row = next;
    }
    const int64_t mine = static_cast<int64_t>(blockIdx.x) * cols;
    auto leave = [&](int which, const float (&sum)[8], int p) {
        if (a.columnGrads[which] == nullptr) return;
        float* const to = a.columnSums[which] + mine + at(p);
        for (int i = 0; i < 8; ++i) {
            if (i < count(p)) to[i] = sum[i];
        }
    };
#pragma unroll
    for (int p = 0; p < kPackets; ++p) {
        if (!here[p]) continue;
        leave(kPostSums, postSum[p], p);
        leave(kPreSums, preSum[p], p);
        if constexpr (kHeld) leave(kGateSums, gateSum[p], p);
    }
}

// Longer rows, read behind each sum again: a workgroup a row, which leaves the row's two means for the columns' sums.
constexpr int kAnyThreads = 256;

__device__ __forceinline__ double SumOfGroup(double v, double (&lds)[kAnyThreads / kWave]) {
    v = WaveSum(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kAnyThreads / kWave; ++w) v += lds[w];
    return v;
}

// What the two kernels of long rows make of an element.
template <typename Codec, typename Gamma>
struct Element {
    const SandwichGradArgs& a;
    int64_t row;
    float preRstd, postRstd, rawGate;

    __device__ Element(const SandwichGradArgs& args, int64_t r) : a(args), row(r), preRstd(0.f), postRstd(1.f), rawGate(0.f) {
        if (a.pre != nullptr) preRstd = a.preRstd[row];
        if (a.post != nullptr) postRstd = a.postRstd[row];
        if (a.gateKind == kGateRow) rawGate = RawRowGate<Codec>(a, row);
    }
    __device__ float Value(const void* t, int64_t c) const { return Codec::Load(static_cast<const typename Codec::Storage*>(t)[row * a.cols + c]); }
    __device__ float Weight(const void* t, int64_t c) const { return Gamma::Load(static_cast<const typename Gamma::Storage*>(t)[c]); }
    __device__ float NormedSum(int64_t c) const { return Value(a.s, c) * preRstd; }
    __device__ float NormedX(int64_t c) const { return a.post != nullptr || a.gateKind != kGateNone ? Value(a.x, c) * postRstd : 0.f; }
    __device__ float SumGrad(int64_t c, float preMean) const {
        float d = 0.f;
        if (a.pre != nullptr) d = preRstd * (Value(a.normGrad, c) * Weight(a.pre, c) - NormedSum(c) * preMean);
        return a.sumGrad != nullptr ? d + Value(a.sumGrad, c) : d;
    }
    __device__ float RawGate(int64_t c) const {
        return a.gateKind == kGateChannel ? Weight(a.gate, c) : a.gateKind == kGateEach ? Value(a.gate, c) : rawGate;
    }
    __device__ float Open(int64_t c) const { return a.gateKind == kGateNone ? 1.f : Gated(RawGate(c), a.sigmoid); }
    __device__ float Unit(int64_t c, float normedX) const { return a.post != nullptr ? normedX * Weight(a.post, c) : normedX; }
};

template <typename Codec, typename Gamma>
__global__ __launch_bounds__(kAnyThreads) void SandwichGradRowsKernel(SandwichGradArgs a) {
    using S = typename Codec::Storage;
    __shared__ double lds[kAnyThreads / kWave];
    const int64_t row = GroupIndex();
    if (row >= a.rows) return;
    const Element<Codec, Gamma> el(a, row);
    const int64_t at = row * a.cols;
    double sum = 0.0;
    if (a.pre != nullptr) {
        for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) sum += static_cast<double>(el.Value(a.normGrad, c) * el.Weight(a.pre, c)) * el.NormedSum(c);
        sum = SumOfGroup(sum, lds);
    }
    const float preMean = static_cast<float>(sum / static_cast<double>(a.cols));
    double postSum = 0.0, gateSum = 0.0;
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        const float d = el.SumGrad(c, preMean);
        if (a.residualGrad != nullptr) static_cast<S*>(a.residualGrad)[at + c] = Codec::Store(a.residualScale * d);
        const float v = a.branchScale * d, normed = el.NormedX(c), u = el.Unit(c, normed);
        if (a.gateKind == kGateEach && a.gateGrad != nullptr) static_cast<S*>(a.gateGrad)[at + c] = Codec::Store(v * u * GateSlope(el.RawGate(c), a.sigmoid));
        gateSum += static_cast<double>(v) * u;
        if (a.post != nullptr) postSum += static_cast<double>(v * el.Open(c) * el.Weight(a.post, c)) * normed;
    }
    if (a.gateKind == kGateRow) {
        gateSum = SumOfGroup(gateSum, lds);
        if (a.gateGrad != nullptr && threadIdx.x == 0) static_cast<float*>(a.gateGrad)[row] = static_cast<float>(gateSum) * GateSlope(el.rawGate, a.sigmoid);
    }
    if (a.post != nullptr) postSum = SumOfGroup(postSum, lds);
    if (threadIdx.x == 0) a.rowMeans[row] = preMean;
    if (a.xGrad == nullptr) return;
    const float postMean = static_cast<float>(postSum / static_cast<double>(a.cols));
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        float v = a.branchScale * el.SumGrad(c, preMean) * el.Open(c);
        if (a.post != nullptr) v = el.postRstd * (v * el.Weight(a.post, c) - el.NormedX(c) * postMean);
        static_cast<S*>(a.xGrad)[at + c] = Codec::Store(v);
    }
}

// A workgroup takes kAnyThreads columns of the rows of one group.
constexpr int kColumnRows = 512;

template <typename Codec, typename Gamma>
__global__ __launch_bounds__(kAnyThreads) void SandwichGradColumnsKernel(SandwichGradArgs a) {
    const int64_t blocks = (a.cols + kAnyThreads - 1) / kAnyThreads;
    const int64_t group = GroupIndex() / blocks;
    const int64_t c = GroupIndex() % blocks * kAnyThreads + threadIdx.x;
    if (group >= a.groups || c >= a.cols) return;
    float sums[kColumnSums] = {0.f, 0.f, 0.f};
    for (int64_t row = group; row < a.rows; row += a.groups) {
        const Element<Codec, Gamma> el(a, row);
        if (a.pre != nullptr) sums[kPreSums] = fmaf(el.Value(a.normGrad, c), el.NormedSum(c), sums[kPreSums]);
        if (a.post == nullptr && a.gateKind != kGateChannel) continue;
        const float v = a.branchScale * el.SumGrad(c, a.rowMeans[row]), normed = el.NormedX(c);
        sums[kGateSums] = fmaf(v, el.Unit(c, normed), sums[kGateSums]);
        sums[kPostSums] = fmaf(v * el.Open(c), normed, sums[kPostSums]);
    }
    for (int i = 0; i < kColumnSums; ++i) {
        if (a.columnGrads[i] != nullptr) a.columnSums[i][group * a.cols + c] = sums[i];
    }
}

// One of the column sums (blockIdx.y), kWave columns a workgroup: the groups' sums in their order, in runs side by side.
constexpr int kFinishThreads = 1024;

template <typename Gamma>
__global__ __launch_bounds__(kFinishThreads) void SandwichGradFinishKernel(SandwichGradArgs a) {
    constexpr int kRuns = kFinishThreads / kWave;
    __shared__ double sums[kRuns][kWave];
    const int which = blockIdx.y;
    if (a.columnGrads[which] == nullptr) return;
    const int run = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kWave + lane;
    double sum = 0.0;
    if (c < a.cols) {
#pragma unroll 4
        for (int64_t g = run; g < a.groups; g += kRuns) sum += a.columnSums[which][g * a.cols + c];
    }
    sums[run][lane] = sum;
    __syncthreads();
    if (run != 0 || c >= a.cols) return;
    sum = 0.0;
    for (int r = 0; r < kRuns; ++r) sum += sums[r][lane];
    if (which == kGateSums) sum *= GateSlope(Gamma::Load(static_cast<const typename Gamma::Storage*>(a.gate)[c]), a.sigmoid);
    a.columnGrads[which][c] = static_cast<float>(sum);
}

// Rows of up to 8192 values stay in registers, with what their columns owe.
constexpr int kMaxPackets = 2;
constexpr int64_t kPacketCols = 8ll * kMaxPacketThreads * kMaxPackets;

class SandwichGradExecutor : public aclOpExecutor {
   public:
    SandwichGradArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType weightType = ACL_FLOAT;
    uint64_t offMeans = 0, offSums = 0;
    int threads = 0;

    bool Columns() const { return args.columnGrads[kPostSums] != nullptr || args.columnGrads[kPreSums] != nullptr || args.columnGrads[kGateSums] != nullptr; }

    // Returns the workspace's size.
    uint64_t Plan() {
        uint64_t bytes = 0;
        if (args.cols > kPacketCols) {
            args.groups = (args.rows + kColumnRows - 1) / kColumnRows;
            // enough workgroups side by side for the columns' sums of short batches
            const int64_t blocks = (args.cols + kAnyThreads - 1) / kAnyThreads;
            const int64_t wanted = std::min<int64_t>((2048 + blocks - 1) / blocks, (args.rows + 7) / 8);
            if (args.groups < wanted) args.groups = wanted;
            bytes = opapi::AlignUp(4 * static_cast<uint64_t>(args.rows), 16);
        } else {
            const int64_t lanes = (args.cols + 7) / 8;
            const int64_t packets = lanes <= kMaxPacketThreads ? 1 : kMaxPackets;
            threads = static_cast<int>(((lanes + packets - 1) / packets + kWave - 1) / kWave * kWave);
            args.groups = 256 * std::max(1, kMaxPacketThreads / threads);
            if (args.groups < (args.rows + kColumnRows - 1) / kColumnRows) args.groups = (args.rows + kColumnRows - 1) / kColumnRows;
            if (args.groups > args.rows) args.groups = args.rows;
        }
        offSums = bytes;
        for (float* grads : args.columnGrads) {
            if (grads != nullptr) bytes += opapi::AlignUp(4 * static_cast<uint64_t>(args.groups) * static_cast<uint64_t>(args.cols), 16);
        }
        return bytes;
    }

    template <typename Codec, typename Gamma, int kPackets>
    void ForGate(hipStream_t stream) const {
        const int packets = GatePackets(args.gateKind);
        const dim3 grid(static_cast<unsigned>(args.groups));
        if (packets == kHeldPackets) hipLaunchKernelGGL((SandwichGradKernel<Codec, Gamma, kPackets, kHeldPackets>), grid, dim3(threads), 0, stream, args);
        else if (packets == kReadPackets) hipLaunchKernelGGL((SandwichGradKernel<Codec, Gamma, kPackets, kReadPackets>), grid, dim3(threads), 0, stream, args);
        else hipLaunchKernelGGL((SandwichGradKernel<Codec, Gamma, kPackets, kNoPackets>), grid, dim3(threads), 0, stream, args);
    }

    aclnnStatus Run(void* workspace, hipStream_t stream) override {
        OPAPI_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, ACLNN_ERR_PARAM_INVALID, "aclnnMoeSandwichNormGrad: the workspace must be 16-byte aligned");
        char* at = static_cast<char*>(workspace);
        args.rowMeans = reinterpret_cast<float*>(at);
        at += offSums;
        for (int i = 0; i < kColumnSums; ++i) {
            if (args.columnGrads[i] == nullptr) continue;
            args.columnSums[i] = reinterpret_cast<float*>(at);
            at += opapi::AlignUp(4 * static_cast<uint64_t>(args.groups) * static_cast<uint64_t>(args.cols), 16);
        }
        ForTypes(dtype, weightType, [&](auto codec, auto gamma) {
            using Codec = decltype(codec);
            using Gamma = decltype(gamma);
            if (args.rows > 0) {
                opapi::KernelTimer timer("sandwich_norm_grad", stream);
                if (args.cols > kPacketCols) {
                    hipLaunchKernelGGL((SandwichGradRowsKernel<Codec, Gamma>), GridOf(args.rows), dim3(kAnyThreads), 0, stream, args);
                    const int64_t blocks = (args.cols + kAnyThreads - 1) / kAnyThreads;
                    if (Columns()) hipLaunchKernelGGL((SandwichGradColumnsKernel<Codec, Gamma>), GridOf(blocks * args.groups), dim3(kAnyThreads), 0, stream, args);
                } else if (args.cols <= 8 * kMaxPacketThreads) {
                    ForGate<Codec, Gamma, 1>(stream);
                } else {
                    ForGate<Codec, Gamma, kMaxPackets>(stream);
                }
            }
            if (Columns()) {
                opapi::KernelTimer timer("sandwich_norm_grad_columns", stream);
                const dim3 grid(static_cast<unsigned>((args.cols + kWave - 1) / kWave), kColumnSums);
                hipLaunchKernelGGL((SandwichGradFinishKernel<Gamma>), grid, dim3(kFinishThreads), 0, stream, args);
            }
        });
        const hipError_t err = hipGetLastError();
        OPAPI_CHECK(err == hipSuccess, ACLNN_ERR_RUNTIME_ERROR, "aclnnMoeSandwichNormGrad: launch failed: %s", hipGetErrorString(err));
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeSandwichNormGradGetWorkspaceSize(
    const aclTensor* x, const aclTensor* sumOptional, const aclTensor* sumGradOptional, const aclTensor* normGradOptional,
    const aclTensor* postGammaOptional, const aclTensor* gateOptional, const aclTensor* preGammaOptional, const aclTensor* postRstdOptional,
    const aclTensor* preRstdOptional, int64_t gateType, double residualScale, double branchScale, const aclTensor* xGradOutOptional,
    const aclTensor* residualGradOutOptional, const aclTensor* postGammaGradOutOptional, const aclTensor* gateGradOutOptional,
    const aclTensor* preGammaGradOutOptional, uint64_t* workspaceSize, aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, sumOptional, sumGradOptional, normGradOptional, postGammaOptional, gateOptional, preGammaOptional, postRstdOptional, preRstdOptional,
                        xGradOutOptional, residualGradOutOptional, postGammaGradOutOptional, gateGradOutOptional, preGammaGradOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    SandwichShape shape;
    const aclnnStatus checked = CheckSandwich(x, postGammaOptional, gateOptional, preGammaOptional, gateType, residualScale, branchScale, &shape);
    if (checked != ACLNN_SUCCESS) return checked;
    OPAPI_CHECK(shape.cols <= (1 << 24), kInvalid, "the rows have %lld values; this operator takes up to 16777216", (long long)shape.cols);
    const bool pre = preGammaOptional != nullptr;
    OPAPI_CHECK((normGradOptional != nullptr) == pre && (preRstdOptional != nullptr) == pre && (sumOptional != nullptr || !pre), ACLNN_ERR_PARAM_NULLPTR,
                "normGrad, preGamma and preRstd belong together, and sum with them");
    OPAPI_CHECK((postGammaOptional == nullptr) == (postRstdOptional == nullptr), ACLNN_ERR_PARAM_NULLPTR, "postGamma and postRstd belong together");
    OPAPI_CHECK(pre || sumGradOptional != nullptr, ACLNN_ERR_PARAM_NULLPTR, "neither sumGrad nor normGrad is given");
    struct Named {
        const aclTensor* t;
        const char* name;
    };
    for (const Named& n : {Named{sumOptional, "sum"}, Named{sumGradOptional, "sumGrad"}, Named{normGradOptional, "normGrad"}, Named{xGradOutOptional, "xGradOut"},
                           Named{residualGradOutOptional, "residualGradOut"}}) {
        OPAPI_CHECK(Like(n.t, x), kInvalid, "%s %s must have x's type and extents %s", n.name, ShapeStr(n.t).c_str(), ShapeStr(x).c_str());
    }
    for (const Named& n : {Named{postRstdOptional, "postRstd"}, Named{preRstdOptional, "preRstd"}}) {
        OPAPI_CHECK(PerRow(n.t, x), kInvalid, "%s %s must be FLOAT of x's extents %s without the last", n.name, ShapeStr(n.t).c_str(), ShapeStr(x).c_str());
    }
    OPAPI_CHECK(postGammaGradOutOptional == nullptr || postGammaOptional != nullptr, kInvalid, "postGammaGradOut is given without postGamma");
    OPAPI_CHECK(preGammaGradOutOptional == nullptr || pre, kInvalid, "preGammaGradOut is given without preGamma");
    OPAPI_CHECK(gateGradOutOptional == nullptr || gateOptional != nullptr, kInvalid, "gateGradOut is given without a gate");
    for (const Named& n : {Named{postGammaGradOutOptional, "postGammaGradOut"}, Named{preGammaGradOutOptional, "preGammaGradOut"}}) {
        OPAPI_CHECK(n.t == nullptr || (n.t->dtype == ACL_FLOAT && HasExtents(n.t, {shape.cols})), kInvalid, "%s %s must be FLOAT [%lld]", n.name,
                    ShapeStr(n.t).c_str(), (long long)shape.cols);
    }
    if (gateGradOutOptional != nullptr) {
        OPAPI_CHECK(gateGradOutOptional->dtype == (shape.gateKind == kGateEach ? x->dtype : ACL_FLOAT) && gateGradOutOptional->dims == gateOptional->dims, kInvalid,
                    "gateGradOut %s must have the gate's extents %s, in FLOAT where the gate is shared and in x's type where it is not",
                    ShapeStr(gateGradOutOptional).c_str(), ShapeStr(gateOptional).c_str());
    }
    OPAPI_CHECK(xGradOutOptional != nullptr || residualGradOutOptional != nullptr || postGammaGradOutOptional != nullptr || gateGradOutOptional != nullptr ||
                    preGammaGradOutOptional != nullptr,
                ACLNN_ERR_PARAM_NULLPTR, "no output is given");
    const aclnnStatus memory =
        CheckMemory({x, sumOptional, sumGradOptional, normGradOptional, postGammaOptional, gateOptional, preGammaOptional, postRstdOptional, preRstdOptional},
                    {xGradOutOptional, residualGradOutOptional, postGammaGradOutOptional, gateGradOutOptional, preGammaGradOutOptional});
    if (memory != ACLNN_SUCCESS) return memory;

    auto* ex = new (std::nothrow) SandwichGradExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    SandwichGradArgs& a = ex->args;
    ex->dtype = x->dtype;
    ex->weightType = shape.weightType;
    OPAPI_BIND(ex, x, &a.x);
    if (pre) OPAPI_BIND(ex, sumOptional, &a.s);  // not read without
    OPAPI_BIND(ex, sumGradOptional, &a.sumGrad);
    OPAPI_BIND(ex, normGradOptional, &a.normGrad);
    OPAPI_BIND(ex, postGammaOptional, &a.post);
    OPAPI_BIND(ex, gateOptional, &a.gate);
    OPAPI_BIND(ex, preGammaOptional, &a.pre);
    OPAPI_BIND(ex, postRstdOptional, &a.postRstd);
    OPAPI_BIND(ex, preRstdOptional, &a.preRstd);
    a.xGrad = DataPtr(xGradOutOptional);
    a.residualGrad = DataPtr(residualGradOutOptional);
    a.columnGrads[kPostSums] = reinterpret_cast<float*>(DataPtr(postGammaGradOutOptional));
    a.columnGrads[kPreSums] = reinterpret_cast<float*>(DataPtr(preGammaGradOutOptional));
    if (shape.gateKind == kGateChannel) a.columnGrads[kGateSums] = reinterpret_cast<float*>(DataPtr(gateGradOutOptional));
    else a.gateGrad = DataPtr(gateGradOutOptional);
    a.rows = shape.rows;
    a.cols = shape.cols;
    a.gateKind = shape.gateKind;
    a.gateIsFloat = shape.gateIsFloat;
    a.sigmoid = static_cast<int32_t>(gateType);
    a.residualScale = static_cast<float>(residualScale);
    a.branchScale = static_cast<float>(branchScale);
    ex->SealWorkspace(ex->Plan());
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeSandwichNormGrad(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
