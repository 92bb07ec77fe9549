// aclnnMoeRouterLogits for gfx950: fp32 logits = x @ weight^T, x of 16 or 32 bits, weight of x's type or fp32.
#include "moe_front.h"

#include "aclnnop/aclnn_moe_router_logits.h"

namespace {

using namespace moe_front;

constexpr int64_t kMaxExperts = 4096;

struct LogitsArgs {
    const void* x;
    const void* weight;
    float* logits;
    int64_t rows;
    int64_t cols;
    int32_t experts;
};

// A workgroup per 16 rows and 16 experts, one product per thread, the columns 32 at a time through LDS.
constexpr int kTile = 16;
constexpr int kStep = 32;

template <typename Codec, typename Weight>
__global__ __launch_bounds__(kTile * kTile) void RouterLogitsAnyKernel(LogitsArgs a) {
    __shared__ float xs[kTile][kStep + 1];
    __shared__ float ws[kTile][kStep + 1];
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile;
    const int expert0 = blockIdx.y * kTile;
    const int r = threadIdx.x / kTile, e = threadIdx.x % kTile;
    float acc = 0.f;
    for (int64_t c0 = 0; c0 < a.cols; c0 += kStep) {
        for (int i = threadIdx.x; i < kTile * kStep; i += kTile * kTile) {
            const int line = i / kStep;
            const int64_t c = c0 + i % kStep;
            xs[line][i % kStep] = row0 + line < a.rows && c < a.cols
                                      ? Codec::Load(static_cast<const typename Codec::Storage*>(a.x)[(row0 + line) * a.cols + c]) : 0.f;
            ws[line][i % kStep] = expert0 + line < a.experts && c < a.cols
                                      ? Weight::Load(static_cast<const typename Weight::Storage*>(a.weight)[(expert0 + line) * a.cols + c]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kStep; ++i) acc = fmaf(xs[r][i], ws[e][i], acc);
        __syncthreads();
    }
    if (row0 + r < a.rows && expert0 + e < a.experts) a.logits[(row0 + r) * a.experts + expert0 + e] = acc;
}

class LogitsExecutor : public aclOpExecutor {
   public:
    LogitsArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType weightType = ACL_FLOAT;

    template <typename Codec, typename Weight>
    void Launch(hipStream_t stream) const {
        const dim3 grid(static_cast<unsigned>((args.rows + kTile - 1) / kTile), static_cast<unsigned>((args.experts + kTile - 1) / kTile));
        hipLaunchKernelGGL((RouterLogitsAnyKernel<Codec, Weight>), grid, dim3(kTile * kTile), 0, stream, args);
    }

    template <typename Codec>
    void LaunchFor(hipStream_t stream) const {
        if (weightType == Codec::kType) Launch<Codec, Codec>(stream);
        else Launch<Codec, F32>(stream);
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("router_logits", stream);
        if (dtype == ACL_FLOAT) Launch<F32, F32>(stream);
        else if (dtype == ACL_FLOAT16) LaunchFor<F16>(stream);
        else LaunchFor<Bf16>(stream);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) {
            opapi::SetError("aclnnMoeRouterLogits: launch failed: %s", hipGetErrorString(err));
            return ACLNN_ERR_RUNTIME_ERROR;
        }
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeRouterLogitsGetWorkspaceSize(const aclTensor* x, const aclTensor* weight, const aclTensor* logitsOut,
                                                            uint64_t* workspaceSize, aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(weight, "weight");
    OPAPI_CHECK_NOTNULL(logitsOut, "logitsOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, weight, logitsOut);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    const int64_t cols = x->dims.back();
    OPAPI_CHECK(cols > 0, kInvalid, "the last extent of x is zero");
    const int64_t rows = RowsOf(x);
    OPAPI_CHECK(rows >= 0, kInvalid, "x has more than 2147483647 rows");
    OPAPI_CHECK(weight->dtype == x->dtype || weight->dtype == ACL_FLOAT, kInvalid, "weight must be of x's type or FLOAT");
    OPAPI_CHECK(weight->dims.size() == 2 && weight->dims[1] == cols, kInvalid, "weight %s must be [experts, %lld]", ShapeStr(weight).c_str(),
                (long long)cols);
    const int64_t experts = weight->dims[0];
    OPAPI_CHECK(experts > 0 && experts <= kMaxExperts, kInvalid, "weight has %lld experts, this build takes 1 to %lld", (long long)experts,
                (long long)kMaxExperts);
    OPAPI_CHECK(logitsOut->dtype == ACL_FLOAT && SameButLast(logitsOut, x, experts), kInvalid,
                "logitsOut %s must be FLOAT, x's extents %s with the last replaced by %lld", ShapeStr(logitsOut).c_str(), ShapeStr(x).c_str(),
                (long long)experts);
    OPAPI_CHECK(InOrder(logitsOut), kInvalid, "the outputs must be contiguous");
    for (const aclTensor* t : {x, weight, logitsOut}) {
        OPAPI_CHECK(rows == 0 || t->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "a tensor carries no device memory");
        OPAPI_CHECK(t == logitsOut || !IsContiguous(t) || !Overlap(t, logitsOut), kInvalid, "an output shares memory with an input");
    }

    auto* ex = new (std::nothrow) LogitsExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    ex->dtype = x->dtype;
    ex->weightType = weight->dtype;
    OPAPI_BIND(ex, x, &ex->args.x);
    OPAPI_BIND(ex, weight, &ex->args.weight);
    ex->args.logits = reinterpret_cast<float*>(DataPtr(logitsOut));
    ex->args.rows = rows;
    ex->args.cols = cols;
    ex->args.experts = static_cast<int32_t>(experts);
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeRouterLogits(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
