// aclnnMoeAddRmsNormQuant for gfx950: s = x + residual, n = rms_norm(s) * gamma, int8 rows of n * smooth with a scale each.
//
// With r = 1 / sqrt(mean(s^2) + eps) the scale's maximum is max|s r gamma smooth| = r max|s gamma smooth|, and r cancels in
// v / scale: y = round(127 w / max|w|) with w = s gamma smooth.  So one reduction over the row yields the sum of squares and the
// maximum together, and the row is done after a single exchange between its waves.  Sums, r, n and w are fp32; what is rounded is s
// (to the stream's type, and that rounded value is what is normalised: norm and sum agree whether or not the sum is asked for), n where
// it leaves, and y.
#include "norm_rows.h"

#include <cmath>

#include "aclnnop/aclnn_moe_add_rms_norm_quant.h"

namespace {

using namespace moe_front;

struct NormArgs {
    const void* x;
    const void* residual;  // optional
    const void* gamma;
    const float* smooth;   // optional
    int8_t* y;             // optional, with scale
    float* scale;
    void* norm;            // optional
    void* sum;             // optional; may be x's or residual's memory
    int64_t rows;
    int64_t cols;
    float eps;
};

template <int kWaves>
__device__ __forceinline__ void ReduceRow(double& sumSquares, uint32_t& maxBits) {
    sumSquares = WaveSum(sumSquares);
    maxBits = WaveMax(maxBits);
    if constexpr (kWaves > 1) {
        __shared__ double sums[kWaves];
        __shared__ uint32_t maxima[kWaves];
        if (threadIdx.x % kWave == 0) {
            sums[threadIdx.x / kWave] = sumSquares;
            maxima[threadIdx.x / kWave] = maxBits;
        }
        __syncthreads();
        sumSquares = sums[0];
        maxBits = maxima[0];
        for (int w = 1; w < kWaves; ++w) {
            sumSquares += sums[w];
            maxBits = max(maxBits, maxima[w]);
        }
    }
}

// Rows of any length: a workgroup per row, one element at a time, the row read again for the outputs (from the sum where that
// was written, by the same lane: it may lie in x's memory).  A lane adds up a 256th of the row, one square behind the other: in 64 bits, since
// in 32 the error grows with the row (2^22 equal values: 1800 units of 2^-24 in the sum, which is 1 / 18000 of the norm).  An element at a time twice
// is what bounds it: 4096 x 16392 bf16 271 us, where 16384 columns take 125 in packets; a single row has one CU to itself (65536 columns 143).
constexpr int kAnyThreads = 256;

template <typename Codec, typename Gamma>
__global__ __launch_bounds__(kAnyThreads) void NormQuantAnyKernel(NormArgs a) {
    using S = typename Codec::Storage;
    const int64_t row = GroupIndex();
    if (row >= a.rows) return;
    const int64_t at = row * a.cols;
    const S* const x = static_cast<const S*>(a.x) + at;
    const S* const residual = a.residual == nullptr ? nullptr : static_cast<const S*>(a.residual) + at;
    S* const sum = a.sum == nullptr ? nullptr : static_cast<S*>(a.sum) + at;
    const typename Gamma::Storage* const gamma = static_cast<const typename Gamma::Storage*>(a.gamma);
    double sumSquares = 0.0;
    uint32_t maxBits = 0;
    auto rounded = [&](int64_t c) { return residual == nullptr ? x[c] : Codec::Store(Codec::Load(x[c]) + Codec::Load(residual[c])); };
    auto weight = [&](int64_t c) { return a.smooth == nullptr ? 1.f : a.smooth[c]; };
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        const S raw = rounded(c);
        if (sum != nullptr) sum[c] = raw;
        const float s = Codec::Load(raw);
        sumSquares = fma(static_cast<double>(s), static_cast<double>(s), sumSquares);
        maxBits = max(maxBits, __float_as_uint(fabsf(s * Gamma::Load(gamma[c]) * weight(c))));
    }
    ReduceRow<kAnyThreads / kWave>(sumSquares, maxBits);
    const RowScales scales = ScalesOf(static_cast<float>(sumSquares), maxBits, a.cols, a.eps);
    if (a.scale != nullptr && threadIdx.x == 0) a.scale[row] = scales.scale;
    for (int64_t c = threadIdx.x; c < a.cols; c += kAnyThreads) {
        const float s = Codec::Load(sum != nullptr ? sum[c] : rounded(c));
        const float g = Gamma::Load(gamma[c]);
        if (a.norm != nullptr) static_cast<S*>(a.norm)[at + c] = Codec::Store(s * scales.r * g);
        if (a.y != nullptr) a.y[at + c] = static_cast<int8_t>(Quantised(s * g * weight(c), scales));
    }
}

// Rows in pieces of eight elements, up to kPackets of them per lane, read once and kept in registers from the reduction to the
// outputs.  A workgroup takes every gridDim.x-th row: gamma and smooth stay with it, and the next row is asked for before the present one is
// reduced.  What bounds it is HBM: 8192 x 7168 bf16 with a residual, all outputs, 94 us alone, 96 to 99 in a row of calls: 5.3 to 5.6 TB/s, with what the
// memory-side cache still holds (a copy of 1 GiB moves 5.2; the kernel that reads rows twice, an element at a time: 350 us); one row of 4096 3.4 us, a launch and one round trip.  As few packets a lane as
// 512 threads allow: on two and four the same row takes 0.3 and 1.6 us longer, 4096 x 4096 fp32 (54 us) 1 and 5.  Workgroups: 4096 at most, for the
// widest rows 100 us against 103 to 104 for 512 to 2048; narrow rows 2048 (16384 x 1024: 31.5 us, with 4096 33.3, with 1024 37.8).
// Off the 16-byte grid (kGrid false) pieces are read and written where they lie, which the vector memory instructions do at any address, and a row's last
// one by its elements: 8192 x 7167 bf16 172 us (246 twice and an element at a time), 64 x 7167 6.5 (19).  Pieces on the grid whose first and last are another
// row's in part: 148 to 157, but rows of 3001 42 instead of 33.
constexpr int kMaxPacketThreads = 512;
constexpr int kMaxPackets = 4;

template <typename Codec, typename Gamma, int kPackets, bool kSmooth, bool kGrid>
__global__ __launch_bounds__(kMaxPacketThreads) void NormQuantPacketsKernel(NormArgs a) {
    using P = Packet<Codec>;
    using Storage = typename Codec::Storage;
    __shared__ float2 partial[2][kMaxPacketThreads / kWave];
    const int threads = blockDim.x, waves = threads / kWave, tid = threadIdx.x;
    const int cols = static_cast<int>(a.cols);
    P x[kPackets], r[kPackets];
    Packet<Gamma> gamma[kPackets];
    Packet<F32> smooth[kSmooth ? kPackets : 1];
    bool here[kPackets];
    auto at = [&](int p) { return (p * threads + tid) * 8; };
    auto count = [&](int p) { return min(cols - at(p), 8); };
#pragma unroll
    for (int p = 0; p < kPackets; ++p) {
        here[p] = at(p) < cols;
        if (here[p]) {
            gamma[p] = LoadPacket<kGrid, Gamma>(a.gamma, at(p), count(p));
            if constexpr (kSmooth) smooth[p] = LoadPacket<kGrid, F32>(a.smooth, at(p), count(p));
        }
    }
    auto load = [&](int64_t row) {
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            x[p] = LoadPacket<kGrid, Codec>(a.x, row * cols + at(p), count(p));
            if (a.residual != nullptr) r[p] = LoadPacket<kGrid, Codec>(a.residual, row * cols + at(p), count(p));
        }
    };
    int64_t row = blockIdx.x;
    load(row);
    for (int parity = 0; row < a.rows; parity ^= 1) {
        P s[kPackets];
        float sumSquares = 0.f;
        uint32_t maxBits = 0;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            float v[8];
            s[p] = x[p];
            Unpack<Codec>(x[p], v);
            if (a.residual != nullptr) {
                float w[8];
                Unpack<Codec>(r[p], w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += w[i];
                s[p] = Pack<Codec>(v);
                Unpack<Codec>(s[p], v);
            }
            if (a.sum != nullptr) StorePacket<kGrid, Storage>(a.sum, row * cols + at(p), count(p), s[p]);
            float g[8];
            Unpack<Gamma>(gamma[p], g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sumSquares = fmaf(v[i], v[i], sumSquares);
                float w = v[i] * g[i];
                if constexpr (kSmooth) w *= reinterpret_cast<const float*>(&smooth[p])[i];
                maxBits = max(maxBits, __float_as_uint(fabsf(w)));
            }
        }
        const int64_t next = row + gridDim.x;
        if (next < a.rows) load(next);
        sumSquares = WaveSum(sumSquares);
        maxBits = WaveMax(maxBits);
        if (waves > 1) {
            if (tid % kWave == 0) partial[parity][tid / kWave] = float2{sumSquares, __uint_as_float(maxBits)};
            __syncthreads();  // two buffers in turn: one barrier a row
            sumSquares = partial[parity][0].x;
            maxBits = __float_as_uint(partial[parity][0].y);
            for (int w = 1; w < waves; ++w) {
                sumSquares += partial[parity][w].x;
                maxBits = max(maxBits, __float_as_uint(partial[parity][w].y));
            }
        }
        const RowScales scales = ScalesOf(sumSquares, maxBits, a.cols, a.eps);
        if (a.scale != nullptr && tid == 0) a.scale[row] = scales.scale;
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            if (!here[p]) continue;
            float v[8], g[8];
            Unpack<Codec>(s[p], v);
            Unpack<Gamma>(gamma[p], g);
            if (a.norm != nullptr) {
                float n[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) n[i] = v[i] * scales.r * g[i];
                StorePacket<kGrid, Storage>(a.norm, row * cols + at(p), count(p), Pack<Codec>(n));
            }
            if (a.y != nullptr) {
                uint32_t q[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float w = v[i] * g[i];
                    if constexpr (kSmooth) w *= reinterpret_cast<const float*>(&smooth[p])[i];
                    q[i / 4] |= (static_cast<uint32_t>(Quantised(w, scales)) & 0xffu) << (i % 4 * 8);
                }
                StorePacket<kGrid, int8_t>(a.y, row * cols + at(p), count(p), uint2{q[0], q[1]});
            }
        }
        row = next;
    }
}

class NormQuantExecutor : public aclOpExecutor {
   public:
    NormArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType gammaType = ACL_FLOAT;

    // Every tensor starts on the boundaries that packets are read and written at, row after row.
    bool OnGrid() const {
        auto on = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
        return args.cols % 8 == 0 && on(args.x, 16) && on(args.residual, 16) &&
               on(args.gamma, 16) && on(args.smooth, 16) && on(args.norm, 16) && on(args.sum, 16) && on(args.y, 8);
    }

    template <typename Codec, typename Gamma, int kPackets, bool kGrid>
    void LaunchPackets(hipStream_t stream) const {
        const int64_t lanes = ((args.cols + 7) / 8 + kPackets - 1) / kPackets;
        const int threads = static_cast<int>((lanes + kWave - 1) / kWave * kWave);
        int64_t groups = args.rows;
        const int64_t most = threads >= 256 ? 4096 : 2048;
        if (groups > most) groups = most;
        if (args.smooth != nullptr) {
            hipLaunchKernelGGL((NormQuantPacketsKernel<Codec, Gamma, kPackets, true, kGrid>), dim3(static_cast<unsigned>(groups)), dim3(threads), 0, stream, args);
        } else {
            hipLaunchKernelGGL((NormQuantPacketsKernel<Codec, Gamma, kPackets, false, kGrid>), dim3(static_cast<unsigned>(groups)), dim3(threads), 0, stream, args);
        }
    }

    template <typename Codec, typename Gamma>
    void Launch(hipStream_t stream) const {
        if (args.cols > 8 * kMaxPacketThreads * kMaxPackets) {
            hipLaunchKernelGGL((NormQuantAnyKernel<Codec, Gamma>), GridOf(args.rows), dim3(kAnyThreads), 0, stream, args);
        } else if (OnGrid()) {
            ChoosePackets<Codec, Gamma, true>(stream);
        } else {
            ChoosePackets<Codec, Gamma, false>(stream);
        }
    }

    template <typename Codec, typename Gamma, bool kGrid>
    void ChoosePackets(hipStream_t stream) const {
        const int64_t lanes = (args.cols + 7) / 8;
        if (lanes <= kMaxPacketThreads) LaunchPackets<Codec, Gamma, 1, kGrid>(stream);
        else if (lanes <= 2 * kMaxPacketThreads) LaunchPackets<Codec, Gamma, 2, kGrid>(stream);
        else LaunchPackets<Codec, Gamma, 4, kGrid>(stream);
    }

    template <typename Codec>
    void LaunchFor(hipStream_t stream) const {
        if (gammaType == Codec::kType) Launch<Codec, Codec>(stream);
        else Launch<Codec, F32>(stream);
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("add_rms_norm_quant", stream);
        if (dtype == ACL_FLOAT) Launch<F32, F32>(stream);
        else if (dtype == ACL_FLOAT16) LaunchFor<F16>(stream);
        else LaunchFor<Bf16>(stream);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) {
            opapi::SetError("aclnnMoeAddRmsNormQuant: launch failed: %s", hipGetErrorString(err));
            return ACLNN_ERR_RUNTIME_ERROR;
        }
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeAddRmsNormQuantGetWorkspaceSize(
    const aclTensor* x, const aclTensor* residualOptional, const aclTensor* gamma, const aclTensor* smoothScaleOptional,
    double epsilon, const aclTensor* yOutOptional, const aclTensor* scaleOutOptional, const aclTensor* normOutOptional,
    const aclTensor* sumOutOptional, uint64_t* workspaceSize, aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(gamma, "gamma");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, residualOptional, gamma, smoothScaleOptional, yOutOptional, scaleOutOptional, normOutOptional, sumOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    const int64_t cols = x->dims.back();
    OPAPI_CHECK(cols > 0, kInvalid, "the last extent of x is zero");
    const int64_t rows = RowsOf(x);
    OPAPI_CHECK(rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
    OPAPI_CHECK((gamma->dtype == x->dtype || gamma->dtype == ACL_FLOAT) && gamma->dims.size() == 1 && gamma->dims[0] == cols, kInvalid,
                "gamma must be [%lld] of x's type or FLOAT", (long long)cols);
    OPAPI_CHECK(smoothScaleOptional == nullptr || (smoothScaleOptional->dtype == ACL_FLOAT && smoothScaleOptional->dims.size() == 1 &&
                                                   smoothScaleOptional->dims[0] == cols),
                kInvalid, "smoothScale must be FLOAT [%lld]", (long long)cols);
    OPAPI_CHECK(epsilon >= 0 && epsilon <= 1e30, kInvalid, "epsilon must be a number of at least 0");
    OPAPI_CHECK((yOutOptional == nullptr) == (scaleOutOptional == nullptr), ACLNN_ERR_PARAM_NULLPTR, "yOut and scaleOut belong together");
    OPAPI_CHECK(yOutOptional != nullptr || normOutOptional != nullptr, ACLNN_ERR_PARAM_NULLPTR, "neither yOut nor normOut is given");
    OPAPI_CHECK(yOutOptional != nullptr || smoothScaleOptional == nullptr, kInvalid, "smoothScale goes into yOut, which is not given");
    if (residualOptional != nullptr) {
        OPAPI_CHECK(residualOptional->dtype == x->dtype && SameButLast(residualOptional, x, cols), kInvalid,
                    "residual %s must have x's type and extents %s", ShapeStr(residualOptional).c_str(), ShapeStr(x).c_str());
    }
    for (const aclTensor* t : {normOutOptional, sumOutOptional}) {
        OPAPI_CHECK(t == nullptr || (t->dtype == x->dtype && SameButLast(t, x, cols)), kInvalid,
                    "%s %s must have x's type and extents %s", t == normOutOptional ? "normOut" : "sumOut", ShapeStr(t).c_str(),
                    ShapeStr(x).c_str());
    }
    if (yOutOptional != nullptr) {
        OPAPI_CHECK(yOutOptional->dtype == ACL_INT8 && SameButLast(yOutOptional, x, cols), kInvalid, "yOut %s must be INT8 of x's extents %s",
                    ShapeStr(yOutOptional).c_str(), ShapeStr(x).c_str());
        OPAPI_CHECK(scaleOutOptional->dtype == ACL_FLOAT && SameButLast(scaleOutOptional, x, -1), kInvalid,
                    "scaleOut %s must be FLOAT of x's extents %s without the last", ShapeStr(scaleOutOptional).c_str(), ShapeStr(x).c_str());
    }
    const aclTensor* const ins[] = {x, residualOptional, gamma, smoothScaleOptional};
    const aclTensor* const outs[] = {sumOutOptional, normOutOptional, yOutOptional, scaleOutOptional};
    for (int o = 0; o < 4; ++o) {
        if (outs[o] == nullptr) continue;
        OPAPI_CHECK(InOrder(outs[o]), kInvalid, "the outputs must be contiguous");
        OPAPI_CHECK(rows == 0 || outs[o]->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an output carries no device memory");
        for (int p = 0; p < o; ++p) OPAPI_CHECK(!Overlap(outs[o], outs[p]), kInvalid, "two outputs share memory");
    }
    for (int i = 0; i < 4; ++i) {
        if (ins[i] == nullptr) continue;
        OPAPI_CHECK(rows == 0 || ins[i]->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an input carries no device memory");
        if (!IsContiguous(ins[i])) continue;  // read from a copy that is made first
        for (int o = 0; o < 4; ++o) {
            const bool inPlace = o == 0 && i < 2 && outs[o] != nullptr && DataPtr(outs[o]) == DataPtr(ins[i]);
            OPAPI_CHECK(inPlace || !Overlap(outs[o], ins[i]), kInvalid, "an output shares memory with an input");
        }
    }

    auto* ex = new (std::nothrow) NormQuantExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    ex->dtype = x->dtype;
    ex->gammaType = gamma->dtype;
    OPAPI_BIND(ex, x, &ex->args.x);
    OPAPI_BIND(ex, residualOptional, &ex->args.residual);
    OPAPI_BIND(ex, gamma, &ex->args.gamma);
    OPAPI_BIND(ex, smoothScaleOptional, &ex->args.smooth);
    ex->args.y = reinterpret_cast<int8_t*>(DataPtr(yOutOptional));
    ex->args.scale = reinterpret_cast<float*>(DataPtr(scaleOutOptional));
    ex->args.norm = DataPtr(normOutOptional);
    ex->args.sum = DataPtr(sumOutOptional);
    ex->args.rows = rows;
    ex->args.cols = cols;
    ex->args.eps = static_cast<float>(epsilon);
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeAddRmsNormQuant(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                               aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
