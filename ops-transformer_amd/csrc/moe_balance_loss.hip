// aclnnMoeBalanceLoss for gfx950: picks and mean probabilities per expert and sequence, and the sum of their products.
//
// The batch is cut into chunks of rows, a workgroup each, and a chunk is cut where a sequence ends.  Walking along the rows, every step goes to the next
// chunk or to the next sequence: the piece that chunk c has of sequence s is number c + s, and of s there are pieces from its first chunk to its
// last.  So the pieces' sums lie in a table of chunks + sequences entries without a count or an offset made beforehand, and a second kernel adds up those
// of each sequence in their order.  One chunk and one sequence: the first kernel finishes by itself.
//
// What bounds it: round trips and launches, not bytes.  16384 x 256 fp32 rows (17 MB, 3.3 us at a copy's 5.2 TB/s) take 12.6 us, 7.3 of them this kernel's
// (a pass of 32 rows per workgroup is a load, a row's sum across the lanes, a reciprocal) and 5 the second one's, which waits for sums that other XCDs
// wrote.  Its work in the first kernel's last workgroup would need counters that somebody has set to zero before, a launch again.
#include "router_rows.h"

#include "aclnnop/aclnn_moe_balance_loss.h"

namespace {

using namespace moe_front;

struct BalanceArgs {
    const void* x;
    const int32_t* expertIdx;
    Sequences sequences;
    int32_t experts;
    int32_t k;
    int32_t sigmoid;
    int32_t chunkRows;
    int32_t chunks;
    int32_t alone;  // one workgroup makes everything
    // outputs
    float* loss;
    int32_t* counts;
    int32_t* rowsOut;
    float* prob;  // optional
    // workspace, by piece
    float* pieceSums;       // [pieces, experts]
    int32_t* pieceCounts;   // [pieces, experts]
    int32_t* pieceRows;     // [pieces]
    double* lossParts;      // [sequences, parts]
    uint32_t* tickets;      // [sequences]
};

constexpr int kChunkThreads = 512;
constexpr int kChunkWaves = kChunkThreads / kWave;
// A lane's rows in flight: their loads and reductions overlap (4096 x 256 in four sequences 11.1 us, with one row 12.6; rows of more than 512 experts have no
// registers for two: 2048 x 2048 17.6 us, with two 19.9).
constexpr int UnrollOf(int pieces) { return pieces <= 2 ? 2 : 1; }
// Chunks: as many as there are CUs (16384 x 256 12.6 us; with 128 14.9, with 512 15.6), of at least two passes, whose loads overlap, or kMinChunkRows where a
// pass holds many narrow rows (16384 x 8 in eight sequences 10.1 us; of two passes, 1024 rows, 13.5), and of at most so many that a lane's fp32 sums stay short.
constexpr int64_t kMostChunks = 256, kMinChunkRows = 128, kMaxChunkRows = 4096;
// One sequence of up to so many passes is one workgroup's: it spares the second launch (96 x 256, six passes: 7.0 us, in two launches 8.1; eight passes of
// 128 rows 8.5 and 8.1, of 4096 rows of eight experts 14.7 and 9.5).
constexpr int64_t kAlonePasses = 6;
// A workgroup of the second kernel takes few experts in many runs of pieces, or, where a sequence has few pieces, many in few: 16384 x 256 in one sequence
// (256 pieces) 12.6 us with few and 16.6 with many, in 64 sequences (five pieces) 19.0 and 14.9.  Fewer than 64 leave more parts of the loss to join (32: 13.5).
constexpr int kFinishThreads = 1024;
constexpr int kFinishFew = 64, kFinishMany = 256;
constexpr int64_t kFewPieces = 64;

template <typename Codec, int kLanes, int kPieces, bool kSigmoid, bool kCut>
__global__ __launch_bounds__(kChunkThreads) void BalanceChunkKernel(BalanceArgs a) {
    using Row = RowOf<kLanes, kPieces>;
    constexpr int kEach = Row::kEach;
    constexpr int kRowsAtOnce = kWave / kLanes;
    constexpr int kUnroll = UnrollOf(kPieces);
    constexpr int kStride = kChunkWaves * kRowsAtOnce;
    // kCut: sequences may end inside a chunk.  The rows of two go in one pass, where LDS has room for both tables (packed batch of 3011 x 160 in 7
    // sequences 12.3 -> 11.0 us; without offsets the second sums cost 0.7 us for nothing).
    constexpr int kAtOnce = kCut && kPieces <= 2 ? 2 : 1;
    __shared__ alignas(16) float sums[kAtOnce][kChunkWaves][Row::kWidth];
    __shared__ int32_t picked[kAtOnce][Row::kWidth];
    __shared__ int32_t live[kAtOnce];
    __shared__ double finishing[kChunkWaves];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, l = lane % kLanes, side = lane / kLanes;
    const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x);
    auto isExpert = [&](int32_t id) { return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.experts); };

    auto totalOf = [&](int q, int e) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kChunkWaves; ++w) total += sums[q][w][e];
        return total;
    };
    const Sequences& seqs = a.sequences;
    int64_t first = static_cast<int64_t>(blockIdx.x) * a.chunkRows, last = min(first + a.chunkRows, seqs.rows);
    if (a.alone) {
        first = seqs.Start(0);
        last = max(first, seqs.Start(1));
    }
    // Rows that a lane has in flight: those of the next pass are asked for before the present one's scores are worked out, those of the first one, and
    // each lane's first id, before the workgroup looks for their sequence.
    typename Row::template Raw<typename Codec::Storage> raw[kUnroll];
    int32_t rowIds[kUnroll], id = -1, rowId = -1;
    // rows from `at` on, the same for the wave, its lanes `side` by side
    auto load = [&](int64_t at, int64_t end) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t row = min(at + u * kStride, end - 1);
            const uint32_t beside = kRowsAtOnce == 1 ? 0 : min(static_cast<uint32_t>(side), static_cast<uint32_t>(end - 1 - row));
            rowIds[u] = (a.expertIdx + row * a.k)[beside * static_cast<uint32_t>(a.k)];
            raw[u] = Row::Ask(x + row * a.experts, beside * static_cast<uint32_t>(a.experts), a.experts, l);
        }
    };
    auto loadFirst = [&](int64_t begin, int64_t end) {
        if (begin + wave * kRowsAtOnce < end) load(begin + wave * kRowsAtOnce, end);
        if (tid < (end - begin) * a.k) {
            id = a.expertIdx[begin * a.k + tid];
            rowId = a.expertIdx[(begin + tid / a.k) * a.k];
        }
    };
    loadFirst(first, last);
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
        for (int e = tid; e < a.experts; e += kChunkThreads) picked[q][e] = 0;
        if (tid == 0) live[q] = 0;
    }
    if (blockIdx.x == 0 && !a.alone) {  // for the second kernel
        for (int s = tid; s < seqs.count; s += kChunkThreads) a.tickets[s] = 0;
    }
    __syncthreads();
    for (int64_t at = first;;) {
        int32_t s = 0;
        int64_t border = last, end = last;  // of sequence s, and of the rows of this pass: those behind the border are of sequence s + 1
        if (!a.alone) {
            if (at >= last) return;
            if constexpr (kCut) {
                // whatever the offsets are, s starts at or in front of `at` and ends behind it
                int64_t beyond;
                s = seqs.Of(at, border, beyond);
                if (s >= seqs.count) return;
                border = min(last, border);
                end = border;
                if (s < 0) {
                    at = border;
                    if (at < last) loadFirst(at, last);
                    continue;
                }
                if (kAtOnce == 2 && border < last && s + 1 < seqs.count) end = max(border, min(last, beyond >= 0 ? beyond : seqs.Start(s + 2)));
            }
        }
        const bool both = end > border;
        float sum[kAtOnce][kEach];
        int32_t counted[kAtOnce];
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
            counted[q] = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum[q][i] = 0.f;
        }
#pragma unroll 1
        for (int64_t row = at + wave * kRowsAtOnce; row < end; row += kUnroll * kStride) {
            // Scores, for softmax before their division by the sum.  Row by row without a branch: the rows' reductions overlap.
            float p[kUnroll][kEach], total[kUnroll];
            bool counts[kUnroll], lost = false;
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                counts[u] = row + u * kStride + side < end && isExpert(rowIds[u]);
                Row::template Logits<Codec>(raw[u], a.experts, l, p[u]);
            }
            if (row + kUnroll * kStride < end) load(row + kUnroll * kStride, end);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if constexpr (kSigmoid) {
#pragma unroll
                    for (int i = 0; i < kEach; ++i) p[u][i] = SigmoidOf(p[u][i]).p;
                } else {
                    const ExpFrom e(TopOf<kLanes>(p[u]));
#pragma unroll
                    for (int i = 0; i < kEach; ++i) p[u][i] = e(p[u][i]);
                }
                total[u] = 0.f;
#pragma unroll
                for (int i = 0; i < kEach; ++i) total[u] += p[u][i];
                total[u] = SumOver<kLanes>(total[u]);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const bool behind = kAtOnce == 2 && row + u * kStride + side >= border;
#pragma unroll
                for (int q = 0; q < kAtOnce; ++q) counted[q] += counts[u] && l == 0 && behind == (q == 1) ? 1 : 0;
                if (kSigmoid && counts[u] && total[u] < kLostSum) {
                    lost = true;
                    counts[u] = false;
                }
                const float inverse = total[u] == 0.f ? 0.f : Reciprocal(total[u]);
#pragma unroll
                for (int q = 0; q < kAtOnce; ++q) {
                    const bool here = counts[u] && behind == (q == 1);
#pragma unroll
                    for (int i = 0; i < kEach; ++i) sum[q][i] = here ? fmaf(p[u][i], inverse, sum[q][i]) : sum[q][i];
                }
            }
            if (kSigmoid && lost) {  // rare, and made again (the lanes of a row agree)
#pragma unroll 1
                for (int64_t again = row + side; again < min(row + kUnroll * kStride, end); again += kStride) {
                    float v[kEach], share[kEach], scores = 0.f;
                    Row::template Logits<Codec>(Row::Ask(x + again * a.experts, 0, a.experts, l), a.experts, l, v);
#pragma unroll
                    for (int i = 0; i < kEach; ++i) scores += SigmoidOf(v[i]).p;
                    if (!(SumOver<kLanes>(scores) < kLostSum) || !isExpert(a.expertIdx[again * a.k])) continue;
                    LostSharesOf<kLanes>(v, share);
#pragma unroll
                    for (int q = 0; q < kAtOnce; ++q) {
#pragma unroll
                        for (int i = 0; i < kEach; ++i) sum[q][i] += (kAtOnce == 2 && again >= border) == (q == 1) ? share[i] : 0.f;
                    }
                }
            }
        }
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
            counted[q] = WaveSum(counted[q]);
            if (lane == 0 && counted[q] != 0) atomicAdd(&live[q], counted[q]);
        }
        const int32_t ids = static_cast<int32_t>(end - at) * a.k, idsBefore = static_cast<int32_t>(border - at) * a.k;
        if (tid < ids && isExpert(rowId) && isExpert(id)) atomicAdd(&picked[kAtOnce == 2 && tid >= idsBefore ? 1 : 0][id], 1);
#pragma unroll 1
        for (int32_t i = tid + kChunkThreads; i < ids; i += kChunkThreads) {
            const int32_t* const idx = a.expertIdx + at * a.k;
            const int32_t more = idx[i];
            if (isExpert(idx[i / a.k * a.k]) && isExpert(more)) atomicAdd(&picked[kAtOnce == 2 && i >= idsBefore ? 1 : 0][more], 1);
        }
        if (end < last) loadFirst(end, last);  // what comes behind, on its way meanwhile
        // the rows side by side in a wave; the waves are added up when they are read
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q) {
            if (q == 1 && !both) break;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
#pragma unroll
                for (int d = kLanes; d < kWave; d <<= 1) sum[q][i] += __shfl_xor(sum[q][i], d);
            }
            if (lane < kLanes) {
#pragma unroll
                for (int p = 0; p < kPieces; ++p) {
                    *reinterpret_cast<float4*>(&sums[q][wave][Row::At(p, l)]) = float4{sum[q][4 * p], sum[q][4 * p + 1], sum[q][4 * p + 2], sum[q][4 * p + 3]};
                }
            }
        }
        __syncthreads();
        if (a.alone) break;
        for (int q = 0; q < (both ? 2 : 1); ++q) {
            const int64_t piece = static_cast<int64_t>(blockIdx.x) + s + q;
#pragma unroll 1
            for (int e = tid; e < a.experts; e += kChunkThreads) {
                a.pieceSums[piece * a.experts + e] = totalOf(q, e);
                a.pieceCounts[piece * a.experts + e] = picked[q][e];
                picked[q][e] = 0;  // for the next sequences
            }
            if (tid == 0) {
                a.pieceRows[piece] = live[q];
                live[q] = 0;
            }
        }
        at = end;
        if (at >= last) return;
        __syncthreads();
    }
    const double n = live[0] > 0 ? live[0] : 1;
    double loss = 0.0;
#pragma unroll 1
    for (int e = tid; e < a.experts; e += kChunkThreads) {
        const double mean = totalOf(0, e) / n;
        a.counts[e] = picked[0][e];
        if (a.prob != nullptr) a.prob[e] = static_cast<float>(mean);
        loss += mean * picked[0][e];
    }
    loss = WaveSum(loss);
    if (lane == 0) finishing[wave] = loss;
    __syncthreads();
    if (tid != 0) return;
    loss = 0.0;
    for (int w = 0; w < kChunkWaves; ++w) loss += finishing[w];
    a.loss[0] = static_cast<float>(loss * a.experts / (a.k * n));
    a.rowsOut[0] = live[0];
}

// A sequence and kExperts of its experts: the pieces' sums in their order, in runs side by side.  Where one workgroup does not hold all experts, the one
// of a sequence that ends last adds up the loss, part by part in their order.
template <int kExperts>
__global__ __launch_bounds__(kFinishThreads) void BalanceFinishKernel(BalanceArgs a) {
    constexpr int kRuns = kFinishThreads / kExperts, kWaves = kExperts / kWave;
    __shared__ double sums[kRuns][kExperts];
    __shared__ int32_t picks[kRuns][kExperts];
    __shared__ int32_t rowsOf[kFinishThreads / kWave];
    __shared__ double losses[kWaves];
    // (32 bits hold every sequence's parts, and every row: divisions of 64 would be a good part of this kernel)
    const uint32_t group = static_cast<uint32_t>(GroupIndex()), parts = static_cast<uint32_t>(a.experts + kExperts - 1) / kExperts;
    const uint32_t whose = parts == 1 ? group : group / parts;
    if (whose >= static_cast<uint32_t>(a.sequences.count)) return;
    const int64_t s = whose;
    const int part = static_cast<int>(group - whose * parts);
    const int tid = threadIdx.x, run = tid / kExperts, lane = tid % kExperts;
    const int e = part * kExperts + lane;
    const int64_t begin = a.sequences.Start(s), end = a.sequences.Start(s + 1);
    int64_t from = 0, to = 0;
    if (begin < end) {
        const uint32_t chunkRows = static_cast<uint32_t>(a.chunkRows);
        from = static_cast<uint32_t>(begin) / chunkRows + s;
        to = static_cast<uint32_t>(end - 1) / chunkRows + 1 + s;
    }
    int32_t live = 0;
    for (int64_t p = from + tid; p < to; p += kFinishThreads) live += a.pieceRows[p];
    double sum = 0.0;
    int32_t count = 0;
    if (e < a.experts) {
#pragma unroll 8
        for (int64_t p = from + run; p < to; p += kRuns) {
            sum += a.pieceSums[p * a.experts + e];
            count += a.pieceCounts[p * a.experts + e];
        }
    }
    for (int d = 32; d > 0; d >>= 1) live += __shfl_xor(live, d);
    if (tid % kWave == 0) rowsOf[tid / kWave] = live;
    sums[run][lane] = sum;
    picks[run][lane] = count;
    __syncthreads();
    live = 0;
    for (int w = 0; w < kFinishThreads / kWave; ++w) live += rowsOf[w];
    const double n = live > 0 ? live : 1;
    double loss = 0.0;
    if (run == 0) {
        sum = 0.0;
        count = 0;
        for (int r = 0; r < kRuns; ++r) {
            sum += sums[r][lane];
            count += picks[r][lane];
        }
        const double mean = sum / n;
        if (e < a.experts) {
            a.counts[s * a.experts + e] = count;
            if (a.prob != nullptr) a.prob[s * a.experts + e] = static_cast<float>(mean);
        }
        loss = WaveSum(mean * count);
        if (tid % kWave == 0) losses[tid / kWave] = loss;
    }
    if constexpr (kWaves > 1) __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < kWaves; ++w) loss += losses[w];
    if (parts > 1) {
        double* const all = a.lossParts + s * parts;
        __hip_atomic_store(all + part, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__hip_atomic_fetch_add(a.tickets + s, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) != parts - 1) return;
        loss = 0.0;
        for (uint32_t i = 0; i < parts; ++i) loss += __hip_atomic_load(all + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    a.loss[s] = static_cast<float>(loss * a.experts / (a.k * n));
    a.rowsOut[s] = live;
}

class BalanceExecutor : public aclOpExecutor {
   public:
    BalanceArgs args{};
    aclDataType dtype = ACL_FLOAT;
    int64_t finishExperts = 0;  // of a workgroup of the second kernel
    uint64_t offRows = 0, offCounts = 0, offLoss = 0, offTickets = 0, offSums = 0;

    template <typename Codec>
    void Launch(hipStream_t stream) const {
        ForRowLayout(args.experts, [&](auto lanes, auto pieces) {
            constexpr int kLanes = decltype(lanes)::value, kPieces = decltype(pieces)::value;
            const dim3 grid(static_cast<unsigned>(args.chunks));
            const bool cut = args.sequences.offsets != nullptr && !args.alone;
            auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kChunkThreads), 0, stream, args); };
            if (args.sigmoid) cut ? launch(BalanceChunkKernel<Codec, kLanes, kPieces, true, true>) : launch(BalanceChunkKernel<Codec, kLanes, kPieces, true, false>);
            else cut ? launch(BalanceChunkKernel<Codec, kLanes, kPieces, false, true>) : launch(BalanceChunkKernel<Codec, kLanes, kPieces, false, false>);
        });
    }

    aclnnStatus Run(void* workspace, hipStream_t stream) override {
        if (!args.alone) {
            OPAPI_CHECK(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, ACLNN_ERR_PARAM_INVALID, "aclnnMoeBalanceLoss: the workspace must be 16-byte aligned");
            char* const at = static_cast<char*>(workspace);
            args.lossParts = reinterpret_cast<double*>(at + offLoss);
            args.tickets = reinterpret_cast<uint32_t*>(at + offTickets);
            args.pieceRows = reinterpret_cast<int32_t*>(at + offRows);
            args.pieceCounts = reinterpret_cast<int32_t*>(at + offCounts);
            args.pieceSums = reinterpret_cast<float*>(at + offSums);
        }
        {
            opapi::KernelTimer timer("balance_chunks", stream);
            if (dtype == ACL_FLOAT) Launch<F32>(stream);
            else if (dtype == ACL_FLOAT16) Launch<F16>(stream);
            else Launch<Bf16>(stream);
        }
        if (!args.alone) {
            opapi::KernelTimer timer("balance_finish", stream);
            const int64_t parts = (args.experts + finishExperts - 1) / finishExperts;
            const dim3 grid = GridOf(parts * args.sequences.count);
            if (finishExperts == kFinishFew) hipLaunchKernelGGL(BalanceFinishKernel<kFinishFew>, grid, dim3(kFinishThreads), 0, stream, args);
            else hipLaunchKernelGGL(BalanceFinishKernel<kFinishMany>, grid, dim3(kFinishThreads), 0, stream, args);
        }
        const hipError_t err = hipGetLastError();
        OPAPI_CHECK(err == hipSuccess, ACLNN_ERR_RUNTIME_ERROR, "aclnnMoeBalanceLoss: launch failed: %s", hipGetErrorString(err));
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeBalanceLossGetWorkspaceSize(const aclTensor* x, const aclTensor* expertIdx, const aclTensor* seqOffsetsOptional,
                                                           int64_t scoreType, const aclTensor* lossOut, const aclTensor* countsOut,
                                                           const aclTensor* rowsOut, const aclTensor* probOutOptional, uint64_t* workspaceSize,
                                                           aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(expertIdx, "expertIdx");
    OPAPI_CHECK_NOTNULL(lossOut, "lossOut");
    OPAPI_CHECK_NOTNULL(countsOut, "countsOut");
    OPAPI_CHECK_NOTNULL(rowsOut, "rowsOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, expertIdx, seqOffsetsOptional, lossOut, countsOut, rowsOut, probOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    int64_t rows = 0, experts = 0, k = 0, sequences = 0;
    const aclnnStatus router = CheckRouterRows(x, expertIdx, seqOffsetsOptional, scoreType, &rows, &experts, &k, &sequences);
    if (router != ACLNN_SUCCESS) return router;
    OPAPI_CHECK(rows * k <= 2147483647ll, kInvalid, "x has %lld rows of %lld picks; counts in INT32 hold up to 2147483647 ids", (long long)rows, (long long)k);
    OPAPI_CHECK(lossOut->dtype == ACL_FLOAT && HasExtents(lossOut, {sequences}), kInvalid, "lossOut %s must be FLOAT [%lld]", ShapeStr(lossOut).c_str(),
                (long long)sequences);
    OPAPI_CHECK(rowsOut->dtype == ACL_INT32 && HasExtents(rowsOut, {sequences}), kInvalid, "rowsOut %s must be INT32 [%lld]", ShapeStr(rowsOut).c_str(),
                (long long)sequences);
    OPAPI_CHECK(countsOut->dtype == ACL_INT32 && HasExtents(countsOut, {sequences, experts}), kInvalid, "countsOut %s must be INT32 [%lld,%lld]",
                ShapeStr(countsOut).c_str(), (long long)sequences, (long long)experts);
    OPAPI_CHECK(probOutOptional == nullptr || (probOutOptional->dtype == ACL_FLOAT && HasExtents(probOutOptional, {sequences, experts})), kInvalid,
                "probOut %s must be FLOAT [%lld,%lld]", ShapeStr(probOutOptional).c_str(), (long long)sequences, (long long)experts);
    const aclnnStatus memory = CheckMemory({x, expertIdx, seqOffsetsOptional}, {lossOut, countsOut, rowsOut, probOutOptional});
    if (memory != ACLNN_SUCCESS) return memory;

    auto* ex = new (std::nothrow) BalanceExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    BalanceArgs& a = ex->args;
    ex->dtype = x->dtype;
    OPAPI_BIND(ex, x, &a.x);
    OPAPI_BIND(ex, expertIdx, &a.expertIdx);
    OPAPI_BIND(ex, seqOffsetsOptional, &a.sequences.offsets);
    a.sequences.isInt64 = seqOffsetsOptional != nullptr && seqOffsetsOptional->dtype == ACL_INT64;
    a.sequences.count = static_cast<int32_t>(sequences);
    a.sequences.rows = rows;
    a.experts = static_cast<int32_t>(experts);
    a.k = static_cast<int32_t>(k);
    a.sigmoid = scoreType == 1;
    a.loss = reinterpret_cast<float*>(DataPtr(lossOut));
    a.counts = reinterpret_cast<int32_t*>(DataPtr(countsOut));
    a.rowsOut = reinterpret_cast<int32_t*>(DataPtr(rowsOut));
    a.prob = reinterpret_cast<float*>(DataPtr(probOutOptional));
    int passRows = 1;
    ForRowLayout(experts, [&](auto lanes, auto pieces) { passRows = kChunkWaves * (kWave / decltype(lanes)::value) * UnrollOf(decltype(pieces)::value); });
    a.alone = sequences == 1 && rows <= kAlonePasses * passRows;
    int64_t chunkRows = (rows + kMostChunks - 1) / kMostChunks;
    chunkRows = std::max(chunkRows, std::min<int64_t>(2 * passRows, kMinChunkRows));
    if (chunkRows > kMaxChunkRows) chunkRows = kMaxChunkRows;
    a.chunkRows = static_cast<int32_t>(chunkRows);
    a.chunks = a.alone ? 1 : static_cast<int32_t>((rows + chunkRows - 1) / chunkRows);
    if (a.chunks < 1) a.chunks = 1;  // of no rows: the outputs are zeros all the same
    uint64_t bytes = 0;
    if (!a.alone) {
        const uint64_t pieces = static_cast<uint64_t>(a.chunks) + static_cast<uint64_t>(sequences);
        ex->finishExperts = a.chunks / sequences <= kFewPieces && experts > kFinishFew ? kFinishMany : kFinishFew;
        const uint64_t parts = static_cast<uint64_t>((experts + ex->finishExperts - 1) / ex->finishExperts);
        auto take = [&](uint64_t size) {
            const uint64_t at = bytes;
            bytes = AlignUp(bytes + size, 16);
            return at;
        };
        ex->offLoss = take(8 * parts * static_cast<uint64_t>(sequences));
        ex->offTickets = take(4 * static_cast<uint64_t>(sequences));
        ex->offRows = take(4 * pieces);
        ex->offCounts = take(4 * pieces * static_cast<uint64_t>(experts));
        ex->offSums = take(4 * pieces * static_cast<uint64_t>(experts));
    }
    ex->SealWorkspace(bytes);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeBalanceLoss(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
