// aclnnMoeSandwichNormGrad for gfx950: from the gradients of the sum and of its norm to those of the block's output, the residual, both gammas and the gate.
//
// With x^ = x postRstd and s^ = s preRstd a row needs one sum behind the other, sum(dn preGamma s^) for dS and sum(du postGamma x^) for xGrad: it stays in
// registers from its loads to its stores, and the memory bounds it: 8192 x 7168 bf16 with both norms (705 MB) 137 us, 5.15 TB/s; 4096 x 12000 138 (590 MB);
// rows of 16 bits off the four-byte grid 1.45 times their bytes' time (4096 x 7167 100 us).  Few rows: two launches (64 x 4096 9.7 us).
//
// A workgroup takes every gridDim.x-th row, or several short ones at once, and adds up what its lanes' columns owe the gammas and a gate per channel in
// registers; a second kernel adds up the workgroups.
#include "sandwich_norm.h"

#include "aclnnop/aclnn_moe_sandwich_norm_grad.h"

namespace {

using namespace moe_front;

// Column sums, by their place in the workspace: of dn s^, and of the branch.  Where a gate per channel opens by g, postGammaGrad = g S and gateGrad = slope
// postGamma S of the one S = sum of dv x^; else S = sum of du x^ is postGammaGrad itself.
enum { kPreSums, kBranchSums, kColumnSums };

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
    float* preGammaGrad;     // optional
    float* postGammaGrad;    // optional
    float* channelGrad;      // optional: gateGrad of a gate per channel
    float* columnSums[kColumnSums];  // workspace: [groups, cols] each, null where not wanted
    float* rowMeans;         // workspace of longer rows: [rows]
    int64_t rows;
    int64_t cols;
    int64_t groups;          // that columns are summed over
    int32_t rowThreads;      // of a workgroup, which takes as many rows at once as it has times these
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

// What is read of a row.
template <typename Codec, int kPackets, bool kGate>
struct GradRows {
    Packet<Codec> x[kPackets], s[kPackets], sumGrad[kPackets], normGrad[kPackets], gate[kGate ? kPackets : 1];
    float postRstd = 1.f, preRstd = 0.f, rawGate = 0.f;
};

// kSumsInLds: the column sums of a workgroup, where its registers have no room for them beside the row (each lane adds to its own 16 bytes, no conflicts:
// with them in registers 4096 x 12000 rows went to scratch memory and took 912 us).
template <typename Codec, typename Gamma, int kPackets, int kThreads>
constexpr bool kSumsInLds = kPackets == 4 || kThreads == kManyThreads || (kPackets == 2 && sizeof(typename Codec::Storage) + sizeof(typename Gamma::Storage) == 8);

template <typename Codec, typename Gamma, int kPackets, int kThreads, int kGate, bool kPre, bool kTail>
__global__ __launch_bounds__(kThreads) void SandwichGradKernel(SandwichGradArgs a) {
    using Storage = typename Codec::Storage;
    constexpr int kMaxWaves = kThreads / kWave;
    constexpr bool kHeld = kGate == kHeldPackets, kRead = kGate == kReadPackets;
    constexpr bool kLds = kSumsInLds<Codec, Gamma, kPackets, kThreads>;
    // Where the registers hold a second row, the next one is asked for before the present one is begun, else when its loads have found their last use.
    constexpr bool kEarly = kPackets == 1 || (kPackets == 2 && sizeof(Storage) == 2);
    // Weights stay in registers, packed, or are read again for every row, from the caches.
    constexpr bool kHoldWeights = kPackets < 4 && kThreads == kFewThreads;
    __shared__ float preSums[2][kMaxWaves][1];
    __shared__ float postSums[2][kMaxWaves][2];
    extern __shared__ float4 ldsSums[];  // kLds: [kColumnSums][kPackets][2][threads], each lane its own
    // One piece a lane: rows of few waves lie side by side in a workgroup.
    const int threads = kPackets == 1 ? a.rowThreads : blockDim.x, waves = threads / kWave;
    const int side = kPackets == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / threads) : 0, sides = kPackets == 1 ? blockDim.x / threads : 1;
    const int tid = threadIdx.x - side * threads;
    const int cols = static_cast<int>(a.cols);
    const float each = 1.f / static_cast<float>(a.cols);
    const bool post = a.post != nullptr, gated = a.gateKind != kGateNone, rowGated = a.gateKind == kGateRow;
    const bool sums = a.sumGrad != nullptr, branchSums = post || kHeld;
    const Pieces<kPackets, kTail> at(cols, threads, tid);
    constexpr int kHeldPackets = kHoldWeights ? kPackets : 1;
    Packet<Gamma> postHeld[kHeldPackets], preHeld[kPre ? kHeldPackets : 1], gateHeld[kHeld ? kHeldPackets : 1];
    auto weights = [&](const Packet<Gamma>* held, const void* w, int p) {
        if constexpr (kHoldWeights) return held[p];
        else return at.template Load<Gamma>(w, 0, p);
    };
    float sumHeld[kLds ? 1 : kColumnSums][kLds ? 1 : kPackets][8];
    auto addToColumns = [&](int which, int p, const float (&v)[8], bool counts) {
        if constexpr (kLds) {
            float4* const to = ldsSums + ((which * kPackets + p) * 2) * threads + tid;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 t = to[h * threads];
                t.x += v[4 * h];
                t.y += v[4 * h + 1];
                t.z += v[4 * h + 2];
                t.w += v[4 * h + 3];
                to[h * threads] = t;
            }
        } else if (counts) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sumHeld[which][p][i] += v[i];
        }
    };
#pragma unroll
    for (int p = 0; p < kPackets; ++p) {
#pragma unroll
        for (int c = 0; c < kColumnSums; ++c) {
            if constexpr (kLds) {
                ldsSums[((c * kPackets + p) * 2) * threads + tid] = ldsSums[((c * kPackets + p) * 2 + 1) * threads + tid] = float4{0.f, 0.f, 0.f, 0.f};
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) sumHeld[c][p][i] = 0.f;
            }
        }
        if constexpr (kHoldWeights) {
            if (post) postHeld[p] = at.template Load<Gamma>(a.post, 0, p);
            if constexpr (kPre) preHeld[p] = at.template Load<Gamma>(a.pre, 0, p);
            if constexpr (kHeld) gateHeld[p] = at.template Load<Gamma>(a.gate, 0, p);
        }
    }
    // Every row's loads, and as many: of tensors that are absent or not needed another one's are loaded in their place, which are at hand then.
    const void* const readX = post || gated ? a.x : kPre ? a.s : a.sumGrad;
    const void* const readSumGrad = sums ? a.sumGrad : a.normGrad;
    const float* const readRstd = post ? a.postRstd : kPre ? a.preRstd : nullptr;
    auto load = [&](GradRows<Codec, kPackets, kRead>& to, int64_t row) {
        const int64_t begin = row * cols;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if constexpr (kPre) {
                to.s[p] = at.template Load<Codec>(a.s, begin, p);
                to.normGrad[p] = at.template Load<Codec>(a.normGrad, begin, p);
            }
            to.sumGrad[p] = at.template Load<Codec>(readSumGrad, begin, p);
            to.x[p] = at.template Load<Codec>(readX, begin, p);
            if constexpr (kRead) to.gate[p] = at.template Load<Codec>(a.gate, begin, p);
        }
        if (readRstd != nullptr) to.postRstd = readRstd[row];
        if constexpr (kPre) to.preRstd = a.preRstd[row];
        if (kGate == kNoPackets && rowGated) to.rawGate = RawRowGate<Codec>(a, row);
    };
    const int64_t stride = static_cast<int64_t>(gridDim.x) * sides;
    int64_t base = static_cast<int64_t>(blockIdx.x) * sides;  // the first of the rows side by side: it goes on for all or for none
    // One row; `following` takes the next one where it is asked for early, else `in` does.
    auto step = [&](GradRows<Codec, kPackets, kRead>& in, GradRows<Codec, kPackets, kRead>& following, int parity) __attribute__((always_inline)) {
        // Behind the last row: that one once more, which counts in no column.
        const int64_t row = min(base + side, a.rows - 1), begin = row * cols, next = min(base + side + stride, a.rows - 1);
        const bool counts = kPackets > 1 || base + side < a.rows;
        if constexpr (kEarly) load(following, next);
        if constexpr (kHoldWeights) {
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                HoldPacked<Gamma>(postHeld[p]);
                if constexpr (kPre) HoldPacked<Gamma>(preHeld[p]);
                if constexpr (kHeld) HoldPacked<Gamma>(gateHeld[p]);
            }
        }
        const float postRstd = post ? in.postRstd : 1.f, raw = in.rawGate;
        // dS
        float d[kPackets][8];
        if constexpr (kPre) {
            const float preRstd = in.preRstd;
            float preMean[1] = {0.f};
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                float v[8], g[8], terms[8], part = 0.f;
                Unpack<Codec>(in.s[p], v);
                Unpack<Codec>(in.normGrad[p], d[p]);
                Unpack<Gamma>(weights(preHeld, a.pre, p), g);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    terms[i] = d[p][i] * (v[i] * preRstd);
                    part = fmaf(at.Own(terms[i], p, i), g[i], part);
                    d[p][i] *= g[i];
                }
                addToColumns(kPreSums, p, terms, counts);
                preMean[0] += at.Counted(part, p);
            }
            SumsOverGroup<1, kMaxWaves>(preMean, waves, parity, preSums, side * waves);
            preMean[0] *= each;
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                float v[8];
                Unpack<Codec>(in.s[p], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[p][i] = preRstd * (d[p][i] - v[i] * preRstd * preMean[0]);
            }
        }
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!kPre || sums) {
                float v[8];
                Unpack<Codec>(in.sumGrad[p], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[p][i] = kPre ? d[p][i] + v[i] : v[i];
            }
            if (a.residualGrad != nullptr) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = a.residualScale * d[p][i];
                at.template Store<Storage>(a.residualGrad, begin, p, Pack<Codec>(v));
            }
        }
        // through the gate and the post norm's weights
        const float rowGate = rowGated ? Gated(raw, a.sigmoid) : 1.f;
        float rowSums[2] = {0.f, 0.f};  // du postGamma x^, dv u
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            float xs[8], g[8], gate[8], gateGrad[8], terms[8], parts[2] = {0.f, 0.f};
            Unpack<Codec>(in.x[p], xs);
            if (post) {
                Unpack<Gamma>(weights(postHeld, a.post, p), g);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = 1.f;
            }
            float slope[8];
            if constexpr (kRead) {
                Unpack<Codec>(in.gate[p], gate);
                OpenGates(gate, slope, a.sigmoid);
            } else if constexpr (kHeld) {
                Unpack<Gamma>(weights(gateHeld, a.gate, p), gate);
                OpenGates(gate, a.sigmoid);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = a.branchScale * d[p][i];
                const float normed = xs[i] * postRstd;
                if constexpr (kHeld) {
                    terms[i] = v * normed;
                    v *= gate[i];
                } else if constexpr (kRead) {
                    gateGrad[i] = v * (normed * g[i]) * slope[i];
                    v *= gate[i];
                    terms[i] = v * normed;
                } else {
                    parts[1] = fmaf(at.Own(v * normed, p, i), g[i], parts[1]);
                    v *= rowGate;
                    terms[i] = v * normed;
                }
                v *= g[i];
                parts[0] = fmaf(at.Own(v, p, i), normed, parts[0]);
                d[p][i] = v;
            }
            if (branchSums) addToColumns(kBranchSums, p, terms, counts);
            rowSums[0] += at.Counted(parts[0], p);
            rowSums[1] += at.Counted(parts[1], p);
            if constexpr (kRead) {
                if (a.gateGrad != nullptr) at.template Store<Storage>(a.gateGrad, begin, p, Pack<Codec>(gateGrad));
            }
        }
        Packet<Codec> x[kPackets];  // needed once more
#pragma unroll
        for (int p = 0; p < kPackets; ++p) x[p] = in.x[p];
        if constexpr (!kEarly) {
            __builtin_amdgcn_sched_barrier(0);  // not in front of the last uses
            load(in, next);
        }
        if (post || rowGated) SumsOverGroup<2, kMaxWaves>(rowSums, waves, parity, postSums, side * waves);
        if (rowGated && a.gateGrad != nullptr && tid == 0) static_cast<float*>(a.gateGrad)[row] = rowSums[1] * GateSlope(raw, a.sigmoid);
        if (a.xGrad != nullptr) {
            const float mean = rowSums[0] * each;
#pragma unroll
            for (int p = 0; p < kPackets; ++p) {
                if (post) {
                    float xs[8];
                    Unpack<Codec>(x[p], xs);
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[p][i] = postRstd * (d[p][i] - xs[i] * postRstd * mean);
                }
                at.template Store<Storage>(a.xGrad, begin, p, Pack<Codec>(d[p]));
            }
        }
        base += stride;
    };
    GradRows<Codec, kPackets, kRead> first;
    load(first, min(base + side, a.rows - 1));
    if constexpr (kPackets == 1) {
        // The two rows take turns where they lie: moved, a row's loads would have to have ended, and the stores behind them.
        GradRows<Codec, kPackets, kRead> second;
        while (true) {
            step(first, second, 0);
            if (base >= a.rows) break;
            step(second, first, 1);
            if (base >= a.rows) break;
        }
    } else if constexpr (kEarly) {
        GradRows<Codec, kPackets, kRead> second;
        for (int parity = 0; base < a.rows; parity ^= 1) {
            step(first, second, parity);
            first = second;
        }
    } else {
        for (int parity = 0; base < a.rows; parity ^= 1) step(first, first, parity);
    }
    if (kPackets == 1 && sides > 1) {  // the sums of the rows side by side, to the first of them
        static_assert(kPackets > 1 || kLds || kColumnSums * kPackets * 8 == 16, "four pieces of four");
        float4* const to = ldsSums + threadIdx.x;
        if constexpr (!kLds) {
#pragma unroll
            for (int q = 0; q < 4; ++q) to[q * blockDim.x] = *reinterpret_cast<const float4*>(&sumHeld[q / 2][0][q % 2 * 4]);
            __syncthreads();
            if (side > 0) return;
            for (int s = 1; s < sides; ++s) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 more = to[q * blockDim.x + s * threads];
                    float* const sum = &sumHeld[q / 2][0][q % 2 * 4];
                    sum[0] += more.x;
                    sum[1] += more.y;
                    sum[2] += more.z;
                    sum[3] += more.w;
                }
            }
        }
    }
    const int64_t mine = static_cast<int64_t>(blockIdx.x) * cols;
#pragma unroll
    for (int c = 0; c < kColumnSums; ++c) {
        if (a.columnSums[c] == nullptr) continue;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            Packet<F32> piece;
            if constexpr (kLds) {
#pragma unroll
                for (int h = 0; h < 2; ++h) piece.q[h] = __builtin_bit_cast(uint4, ldsSums[((c * kPackets + p) * 2 + h) * threads + tid]);
            } else {
                __builtin_memcpy(&piece, sumHeld[c][p], sizeof(piece));
            }
            at.template Store<float>(a.columnSums[c], mine, p, piece);
        }
    }
}

// Longer rows, read behind each sum again: a workgroup a row, which leaves the pre norm's mean of the row for the columns' sums.
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
    float sums[kColumnSums] = {0.f, 0.f};
    for (int64_t row = group; row < a.rows; row += a.groups) {
        const Element<Codec, Gamma> el(a, row);
        if (a.pre != nullptr) sums[kPreSums] = fmaf(el.Value(a.normGrad, c), el.NormedSum(c), sums[kPreSums]);
        if (a.columnSums[kBranchSums] == nullptr) continue;
        const float v = a.branchScale * el.SumGrad(c, a.rowMeans[row]);
        sums[kBranchSums] = fmaf(a.gateKind == kGateChannel ? v : v * el.Open(c), el.NormedX(c), sums[kBranchSums]);
    }
    for (int i = 0; i < kColumnSums; ++i) {
        if (a.columnSums[i] != nullptr) a.columnSums[i][group * a.cols + c] = sums[i];
    }
}

// One of the column sums (blockIdx.y), kWave columns a workgroup: the groups' sums in their order, in runs side by side.
constexpr int kFinishThreads = 1024;

template <typename Gamma>
__global__ __launch_bounds__(kFinishThreads) void SandwichGradFinishKernel(SandwichGradArgs a) {
    constexpr int kRuns = kFinishThreads / kWave;
    __shared__ double sums[kRuns][kWave];
    const int which = blockIdx.y;
    const float* const columnSums = a.columnSums[which];  // (of no rows: none, and the sums are zeros)
    if (which == kPreSums ? a.preGammaGrad == nullptr : a.postGammaGrad == nullptr && a.channelGrad == nullptr) return;
    const int run = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kWave + lane;
    double sum = 0.0;
    if (c < a.cols) {
#pragma unroll 8
        for (int64_t g = run; g < a.groups; g += kRuns) sum += columnSums[g * a.cols + c];
    }
    sums[run][lane] = sum;
    __syncthreads();
    if (run != 0 || c >= a.cols) return;
    sum = 0.0;
    for (int r = 0; r < kRuns; ++r) sum += sums[r][lane];
    if (which == kPreSums) {
        a.preGammaGrad[c] = static_cast<float>(sum);
        return;
    }
    auto weight = [&](const void* w) { return Gamma::Load(static_cast<const typename Gamma::Storage*>(w)[c]); };
    if (a.gateKind != kGateChannel) {
        a.postGammaGrad[c] = static_cast<float>(sum);
        return;
    }
    const float gate = weight(a.gate);
    if (a.postGammaGrad != nullptr) a.postGammaGrad[c] = static_cast<float>(sum * Gated(gate, a.sigmoid));
    if (a.channelGrad != nullptr) a.channelGrad[c] = static_cast<float>(sum * GateSlope(gate, a.sigmoid) * (a.post != nullptr ? weight(a.post) : 1.f));
}

// Rows of eight to 16384 values are one workgroup's at a time: one piece a lane up to 4096 values, two on up to 512 lanes, two on up to 768, whose 168 registers
// hold them with the sums in LDS (4096 x 12000 bf16 138 us, 2048 x 12000 fp32 139; four pieces on 384 lanes 157 and 238; two on 1024, with 128 registers, 202
// and 211), and four above 12288 values (3000 x 16384 156 us; an element at a time 755).

class SandwichGradExecutor : public aclOpExecutor {
   public:
    SandwichGradArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType weightType = ACL_FLOAT;
    uint64_t offMeans = 0, offSums = 0;
    int threads = 0, sides = 1;  // of a row; rows side by side in a workgroup

    // Which column sums are wanted.
    bool Wants(int which) const { return which == kPreSums ? args.preGammaGrad != nullptr : args.postGammaGrad != nullptr || args.channelGrad != nullptr; }
    bool Columns() const { return Wants(kPreSums) || Wants(kBranchSums); }
    bool InPackets() const { return args.cols >= 8 && args.cols <= kPacketCols; }

    // Returns the workspace's size.
    uint64_t Plan() {
        uint64_t bytes = 0;
        if (!InPackets()) {
            args.groups = (args.rows + kColumnRows - 1) / kColumnRows;
            // enough workgroups side by side for the columns' sums of short batches
            const int64_t blocks = (args.cols + kAnyThreads - 1) / kAnyThreads;
            const int64_t wanted = std::min<int64_t>((2048 + blocks - 1) / blocks, (args.rows + 7) / 8);
            if (args.groups < wanted) args.groups = wanted;
            bytes = opapi::AlignUp(4 * static_cast<uint64_t>(args.rows), 16);
        } else {
            const int64_t lanes = (args.cols + 7) / 8;
            const int64_t packets = lanes <= kFewThreads ? 1 : lanes <= 2 * kManyThreads ? 2 : kMaxPackets;
            threads = static_cast<int>(((lanes + packets - 1) / packets + kWave - 1) / kWave * kWave);
            const int64_t waves = threads / kWave;
            // Rows of one or two waves lie side by side in a workgroup of eight, whose column sums are joined before they leave it (8192 x 512 15.5 us, a
            // workgroup each 20.5; 16384 x 1024 45.4 and 47.8); of four they would wait for each other (16384 x 2048 83.8 and 81.9).
            sides = packets == 1 && waves <= 2 ? kFewThreads / kWave / waves : 1;
            args.rowThreads = threads;
            args.groups = kCus * std::max<int64_t>(1, kFewThreads / kWave / (waves * sides));
            // Above, a CU's workgroups have eight waves together; twelve or more (twice the workgroups) cost more in column sums than they hide: 8192 x 7168
            // 152 us instead of 137, 4096 x 4608 65 instead of 60.  Workgroups of five to eight waves with one piece a lane and many rows
            // have registers for two a CU: 8192 x 4096 55.8 us, with one 63.6; 2880 columns with a gate each 151 and 196.
            if (packets == 1 && waves > 4 && args.rows >= 8 * 2 * kCus) args.groups = 2 * kCus;
            const int64_t rows = (args.rows + sides - 1) / sides;  // one behind the other
            if (args.groups < (args.rows + kColumnRows - 1) / kColumnRows) args.groups = (args.rows + kColumnRows - 1) / kColumnRows;
            if (args.groups > rows) args.groups = rows;
        }
        offSums = bytes;
        for (int i = 0; i < kColumnSums; ++i) {
            if (Wants(i)) bytes += opapi::AlignUp(4 * static_cast<uint64_t>(args.groups) * static_cast<uint64_t>(args.cols), 16);
        }
        return bytes;
    }

    template <typename Codec, typename Gamma, int kPackets, int kThreads, int kGate, bool kPre, bool kTail>
    hipError_t LaunchKernel(hipStream_t stream) const {
        const auto kernel = SandwichGradKernel<Codec, Gamma, kPackets, kThreads, kGate, kPre, kTail>;
        int lds = 0;
        if constexpr (kSumsInLds<Codec, Gamma, kPackets, kThreads>) {
            static std::atomic<uint64_t> done{0};
            constexpr int kMost = kColumnSums * kPackets * 2 * kThreads * static_cast<int>(sizeof(float4));
            lds = kMost / kThreads * threads;
            const hipError_t e = opapi::EnsureDynamicLds(reinterpret_cast<const void*>(kernel), kMost, done);
            if (e != hipSuccess) return e;
        }
        if (sides > 1) lds = sides * threads * kColumnSums * 8 * static_cast<int>(sizeof(float));
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(args.groups)), dim3(static_cast<unsigned>(sides * threads)), static_cast<unsigned>(lds), stream,
                           args);
        return hipSuccess;
    }

    template <typename Codec, typename Gamma, int kPackets, int kThreads, int kGate>
    hipError_t LaunchPackets(hipStream_t stream) const {
        const bool tail = args.cols % 8 != 0;
        if (args.pre != nullptr && tail) return LaunchKernel<Codec, Gamma, kPackets, kThreads, kGate, true, true>(stream);
        if (args.pre != nullptr) return LaunchKernel<Codec, Gamma, kPackets, kThreads, kGate, true, false>(stream);
        if (tail) return LaunchKernel<Codec, Gamma, kPackets, kThreads, kGate, false, true>(stream);
        return LaunchKernel<Codec, Gamma, kPackets, kThreads, kGate, false, false>(stream);
    }

    template <typename Codec, typename Gamma, int kPackets, int kThreads>
    hipError_t ForGate(hipStream_t stream) const {
        const int packets = GatePackets(args.gateKind);
        if (packets == kHeldPackets) return LaunchPackets<Codec, Gamma, kPackets, kThreads, kHeldPackets>(stream);
        if (packets == kReadPackets) return LaunchPackets<Codec, Gamma, kPackets, kThreads, kReadPackets>(stream);
        return LaunchPackets<Codec, Gamma, kPackets, kThreads, kNoPackets>(stream);
    }

    aclnnStatus Run(void* workspace, hipStream_t stream) override {
        OPAPI_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, ACLNN_ERR_PARAM_INVALID, "aclnnMoeSandwichNormGrad: the workspace must be 16-byte aligned");
        char* at = static_cast<char*>(workspace);
        args.rowMeans = reinterpret_cast<float*>(at);
        at += offSums;
        for (int i = 0; i < kColumnSums; ++i) {
            if (!Wants(i)) continue;
            args.columnSums[i] = reinterpret_cast<float*>(at);
            at += opapi::AlignUp(4 * static_cast<uint64_t>(args.groups) * static_cast<uint64_t>(args.cols), 16);
        }
        hipError_t err = hipSuccess;
        ForTypes(dtype, weightType, [&](auto codec, auto gamma) {
            using Codec = decltype(codec);
            using Gamma = decltype(gamma);
            if (args.rows > 0) {
                opapi::KernelTimer timer("sandwich_norm_grad", stream);
                const int64_t lanes = (args.cols + 7) / 8;
                if (!InPackets()) {
                    hipLaunchKernelGGL((SandwichGradRowsKernel<Codec, Gamma>), GridOf(args.rows), dim3(kAnyThreads), 0, stream, args);
                    const int64_t blocks = (args.cols + kAnyThreads - 1) / kAnyThreads;
                    if (Columns()) hipLaunchKernelGGL((SandwichGradColumnsKernel<Codec, Gamma>), GridOf(blocks * args.groups), dim3(kAnyThreads), 0, stream, args);
                } else if (lanes <= kFewThreads) {
                    err = ForGate<Codec, Gamma, 1, kFewThreads>(stream);
                } else if (lanes <= 2 * kFewThreads) {
                    err = ForGate<Codec, Gamma, 2, kFewThreads>(stream);
                } else if (lanes <= 2 * kManyThreads) {
                    err = ForGate<Codec, Gamma, 2, kManyThreads>(stream);
                } else {
                    err = ForGate<Codec, Gamma, kMaxPackets, kFewThreads>(stream);
                }
            }
            if (Columns()) {
                opapi::KernelTimer timer("sandwich_norm_grad_columns", stream);
                const dim3 grid(static_cast<unsigned>((args.cols + kWave - 1) / kWave), kColumnSums);
                hipLaunchKernelGGL((SandwichGradFinishKernel<Gamma>), grid, dim3(kFinishThreads), 0, stream, args);
            }
        });
        if (err == hipSuccess) err = hipGetLastError();
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
    a.postGammaGrad = reinterpret_cast<float*>(DataPtr(postGammaGradOutOptional));
    a.preGammaGrad = reinterpret_cast<float*>(DataPtr(preGammaGradOutOptional));
    if (shape.gateKind == kGateChannel) a.channelGrad = reinterpret_cast<float*>(DataPtr(gateGradOutOptional));
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
