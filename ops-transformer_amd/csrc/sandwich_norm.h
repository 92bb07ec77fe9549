// What aclnnMoeSandwichNorm and its gradient share: the gate's forms, sums over a workgroup's waves, and the checks of their first phases.
#pragma once

#include <algorithm>
#include <initializer_list>
#include <new>

#include "norm_rows.h"
#include "router_rows.h"

namespace moe_front {

// How a gate is shared.  kGateRow is a factor of the row, kGateChannel lies in registers beside the gammas, kGateEach is read with the rows.
enum GateKind { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateEach = 3 };

// The kernels are made for gates in registers, gates read with the rows, and neither.
constexpr int kNoPackets = 0, kHeldPackets = 1, kReadPackets = 2;
inline int GatePackets(int kind) { return kind == kGateChannel ? kHeldPackets : kind == kGateEach ? kReadPackets : kNoPackets; }

__device__ __forceinline__ float Gated(float gate, int sigmoid) { return sigmoid ? SigmoidOf(gate).p : gate; }
// Eight gates opened (and their slopes), the choice made once: made element by element both sides are worked out.
__device__ __forceinline__ void OpenGates(float (&gate)[8], int sigmoid) {
    if (!sigmoid) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) gate[i] = SigmoidOf(gate[i]).p;
}
__device__ __forceinline__ void OpenGates(float (&gate)[8], float (&slope)[8], int sigmoid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) slope[i] = 1.f;
    if (!sigmoid) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const Sigmoid s = SigmoidOf(gate[i]);
        gate[i] = s.p;
        slope[i] = s.p * s.rest;
    }
}

// kCount sums over a workgroup, or `waves` of it from `first` on, the same bits in every lane.  `parity` alternates between calls that follow each other: one
// barrier a call.
template <int kCount, int kMaxWaves>
__device__ __forceinline__ void SumsOverGroup(float (&v)[kCount], int waves, int parity, float (&lds)[2][kMaxWaves][kCount], int first = 0) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = SumOver<kWave>(v[i]);
    if (waves == 1) return;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) lds[parity][threadIdx.x / kWave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = lds[parity][first][i];
    for (int w = 1; w < waves; ++w) {
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] += lds[parity][first + w][i];
    }
}

// The piece itself, through a statement the optimiser cannot see through: what a loop makes of it is not made in front of the loop and held (weights of 16
// bits, unpacked, take twice their registers, and a gate's sigmoid as many again).
template <typename Codec>
__device__ __forceinline__ void HoldPacked(Packet<Codec>& piece) {
    if constexpr (sizeof(typename Codec::Storage) == 4) return;
#pragma unroll
    for (uint4& q : piece.q) asm volatile("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w));
}

// Rows of eight to kPacketCols values lie on a workgroup's lanes in pieces of eight: one a lane on up to kFewThreads lanes, two on these or up to kManyThreads, four
// on kFewThreads.  Others are read an element at a time by kAnyThreads lanes.
constexpr int kFewThreads = 512, kManyThreads = 768, kAnyThreads = 256;
constexpr int kMaxPackets = 4;
constexpr int64_t kPacketCols = 8ll * kFewThreads * kMaxPackets;
constexpr int64_t kCus = 256;

// The sum over a workgroup of kAnyThreads, the same bits in every lane.
__device__ __forceinline__ double SumOfGroup(double v, double (&lds)[kAnyThreads / kWave]) {
    v = WaveSum(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kAnyThreads / kWave; ++w) v += lds[w];
    return v;
}

// Where a lane's pieces of eight elements lie in a row of `cols`, at least eight.  Every lane has each of its pieces: one that would end behind the row is the
// row's last eight elements, the first `skip` of which are other lanes' (all eight of a piece that would begin behind it; kTail: cols is no multiple of eight,
// else there are no others).  So loads are without a branch, the compiler knows how many there are, and a wait for one row's need not be one for the
// next row's: with branches 8192 x 7168 rows waited for all of them (105 us instead of 93 with two workgroups a CU).
template <int kPackets, bool kTail>
struct Pieces {
    uint32_t from[kPackets];
    int skip[kPackets];

    __device__ __forceinline__ Pieces(int cols, int threads, int tid) {
#pragma unroll
        for (int p = 0; p < kPackets; ++p) {
            const int at = (p * threads + tid) * 8;
            from[p] = static_cast<uint32_t>(min(at, cols - 8));
            skip[p] = min(at - static_cast<int>(from[p]), 8);
        }
    }
    // Sums are of the lane's own elements: Own() of each term, Counted() of the piece's.
    __device__ __forceinline__ float Own(float v, int p, int i) const { return kTail && i < skip[p] ? 0.f : v; }
    __device__ __forceinline__ float Counted(float part, int p) const { return kTail || skip[p] == 0 ? part : 0.f; }
    // `row`: where the row begins, the same for the wave.
    template <typename Codec>
    __device__ __forceinline__ Packet<Codec> Load(const void* base, int64_t row, int p) const {
        Packet<Codec> piece;
        __builtin_memcpy(&piece, static_cast<const typename Codec::Storage*>(base) + row + from[p], sizeof(piece));
        return piece;
    }
    // All eight: what two lanes have of an element has to be the same bits.
    template <typename Storage, typename P>
    __device__ __forceinline__ void Store(void* base, int64_t row, int p, const P& piece) const {
        __builtin_memcpy(static_cast<Storage*>(base) + row + from[p], &piece, sizeof(piece));
    }
    // The lane's own.
    template <typename Storage, typename P>
    __device__ __forceinline__ void StoreOwn(void* base, int64_t row, int p, const P& piece) const {
        Storage* const to = static_cast<Storage*>(base) + row + from[p];
        if (skip[p] == 0) {
            __builtin_memcpy(to, &piece, sizeof(piece));
        } else if (kTail) {
            Storage raw[8];
            __builtin_memcpy(raw, &piece, sizeof(piece));
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                if (i >= skip[p]) to[i] = raw[i];
            }
        }
    }
};

// The weights that go with the channels, gammas and a gate per channel, share a type: x's, or FLOAT.
struct SandwichShape {
    int64_t rows = 0, cols = 0;
    int gateKind = kGateNone;
    bool gateIsFloat = false;  // of a value per row
    aclDataType weightType = ACL_FLOAT;
};

inline aclnnStatus CheckSandwich(const aclTensor* x, const aclTensor* postGamma, const aclTensor* gate, const aclTensor* preGamma, int64_t gateType,
                                 double residualScale, double branchScale, SandwichShape* shape) {
    using namespace opapi;
    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    const int64_t cols = x->dims.back();
    OPAPI_CHECK(cols > 0, kInvalid, "the last extent of x is zero");
    shape->cols = cols;
    shape->rows = RowsOf(x);
    OPAPI_CHECK(shape->rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
    shape->weightType = x->dtype;
    const aclTensor* const first = postGamma != nullptr ? postGamma : preGamma;
    for (const aclTensor* gamma : {postGamma, preGamma}) {
        OPAPI_CHECK(gamma == nullptr || ((gamma->dtype == x->dtype || gamma->dtype == ACL_FLOAT) && HasExtents(gamma, {cols})), kInvalid,
                    "%s %s must be [%lld] of x's type or FLOAT", gamma == postGamma ? "postGamma" : "preGamma", ShapeStr(gamma).c_str(), (long long)cols);
        OPAPI_CHECK(gamma == nullptr || gamma->dtype == first->dtype, kInvalid, "postGamma and preGamma must have one type");
    }
    if (first != nullptr) shape->weightType = first->dtype;
    OPAPI_CHECK(gateType == 0 || gateType == 1, kInvalid, "gateType (=%lld) must be 0 or 1", (long long)gateType);
    OPAPI_CHECK(std::isfinite(static_cast<float>(residualScale)) && std::isfinite(static_cast<float>(branchScale)), kInvalid,
                "residualScale and branchScale must be finite numbers");
    if (gate == nullptr) return ACLNN_SUCCESS;
    const bool floating = gate->dtype == x->dtype || gate->dtype == ACL_FLOAT;
    if (HasExtents(gate, {cols})) {
        OPAPI_CHECK(floating && (first == nullptr || gate->dtype == first->dtype), kInvalid,
                    "a gate [%lld] must be of x's type or FLOAT, and of the gammas' type", (long long)cols);
        shape->gateKind = kGateChannel;
        shape->weightType = gate->dtype;
    } else if (SameButLast(gate, x, 1)) {
        OPAPI_CHECK(floating, kInvalid, "a gate of a value per row must be of x's type or FLOAT");
        shape->gateKind = kGateRow;
        shape->gateIsFloat = gate->dtype == ACL_FLOAT;
    } else {
        OPAPI_CHECK(SameButLast(gate, x, cols) && gate->dtype == x->dtype, kInvalid,
                    "gate %s must be [%lld], x's extents %s with the last one 1, or these and x's type", ShapeStr(gate).c_str(), (long long)cols,
                    ShapeStr(x).c_str());
        shape->gateKind = kGateEach;
    }
    return ACLNN_SUCCESS;
}

// A tensor of x's type and extents (absent ones pass).
inline bool Like(const aclTensor* t, const aclTensor* x) { return t == nullptr || (t->dtype == x->dtype && SameButLast(t, x, x->dims.back())); }
// A FLOAT of x's rows.
inline bool PerRow(const aclTensor* t, const aclTensor* x) { return t == nullptr || (t->dtype == ACL_FLOAT && SameButLast(t, x, -1)); }

// f(element type, weights' type) as tags.
template <typename F>
void ForTypes(aclDataType type, aclDataType weightType, F f) {
    if (type == ACL_FLOAT) f(F32{}, F32{});
    else if (type == ACL_FLOAT16) weightType == type ? f(F16{}, F16{}) : f(F16{}, F32{});
    else weightType == type ? f(Bf16{}, Bf16{}) : f(Bf16{}, F32{});
}

}  // namespace moe_front
