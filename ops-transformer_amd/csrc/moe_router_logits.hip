// aclnnMoeRouterLogits for gfx950: fp32 logits = x @ weight^T, x of 16 or 32 bits, weight of x's type or fp32.
//
// The matrix instructions take 16-bit operands, and an operand of more bits is a sum of bf16 parts of eight significant bits each: fp32 = three parts
// and fp16 (next to fp32 weights) = two, both without a remainder.  Where both sides have several, each part is the nearest to what those before it
// leave: a part a_i (i from 0) is at most 2^-8i of |x|, a product a_i b_j at most 2^-8(i+j) of |x w|, so those with i + j <= 2 are summed; of the rest
// two are at most 2^-24 of |x w|, fp32's rounding of a product, and one 2^-32.  (Parts that are cut off are up to twice as large each and have one
// sign: 2^-21 of |x w| in all, which in sums of few products showed.)  bf16 rows on fp32 weights leave nothing out, and their weights are cut off:
// 600 x 7168 x 256 21.0 us, 22.6 with the nearest.  They take three instructions in place of one, fp16 rows five, fp32 rows six: with every bit
// of both sides, at several times the rate of the fp32 matrix instructions.  Sums are fp32, in an order that only sizes decide.
#include "moe_front.h"

#include <cmath>

#include "aclnnop/aclnn_moe_router_logits.h"
#include "opapi_profile.h"

namespace {

using namespace moe_front;

constexpr int64_t kMaxExperts = 4096;
constexpr double kMaxThreads = 4294967040.0;  // of a launch: fewer than 2^32, in whole workgroups

struct LogitsArgs {
    const void* x;
    const void* weight;
    float* logits;    // [splits, rows, experts] where the columns are split, the operator's output otherwise
    int64_t rows;
    int64_t cols;
    int64_t splitCols;  // columns of a split
    int32_t experts;
};

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));
typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef float F32x16 __attribute__((ext_vector_type(16)));

// Eight neighbouring values of one row as they lie in memory.
template <typename Codec>
struct Raw {
    uint4 q[sizeof(typename Codec::Storage) / 2];
};

// They need no alignment but their own, the vector memory instructions take any: 8192 x 7167 x 256 with fp32 weights 102 us, bf16 64 (312 and 368 an element at a
// time), 64 x 7167 x 256 13.0 and 14.7 (38 and 37), where 7168 columns take 93, 54, 8.2 and 5.5.
template <typename Codec>
__device__ __forceinline__ Raw<Codec> LoadWhole(const typename Codec::Storage* at) {
    Raw<Codec> r;
    __builtin_memcpy(&r, at, sizeof(r));
    return r;
}

// Values from column c on of a row, of rows on 16 bytes that are whole numbers of them; those behind `end`, which is on them too, are zeros.
template <typename Codec>
__device__ __forceinline__ Raw<Codec> LoadRaw(const typename Codec::Storage* row, int64_t c, int64_t end) {
    constexpr int kPieces = sizeof(typename Codec::Storage) / 2, kPer = 8 / kPieces;
    Raw<Codec> r;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        r.q[i] = c + i * kPer < end ? *reinterpret_cast<const uint4*>(row + c + i * kPer) : uint4{0, 0, 0, 0};
    }
    return r;
}
// The same of any row: what lies behind `end` is read with the rest and dropped, but for the tensor's last values (up to `limit`), which are read one by one.
template <typename Codec>
__device__ __forceinline__ Raw<Codec> LoadEnd(const typename Codec::Storage* row, int64_t c, int64_t end, const typename Codec::Storage* limit) {
    using Storage = typename Codec::Storage;
    Storage v[8] = {};
    if (c < end) {
        if (limit - (row + c) >= 8) {
            __builtin_memcpy(v, row + c, sizeof(v));
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < end ? v[i] : Storage{};
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = c + i < end ? row[c + i] : Storage{};
        }
    }
    Raw<Codec> r;
    __builtin_memcpy(&r, v, sizeof(r));
    return r;
}

// The same in two steps, for loads that are under way while others are used: the pieces, those from `end` on replaced by the row's last ones, and zeros in
// their place once they are there.
template <typename Codec>
__device__ __forceinline__ Raw<Codec> LoadClamped(const typename Codec::Storage* row, int64_t c, int64_t end) {
    constexpr int kPieces = sizeof(typename Codec::Storage) / 2, kPer = 8 / kPieces;
    Raw<Codec> r;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) r.q[i] = *reinterpret_cast<const uint4*>(row + min(c + i * kPer, end - kPer));
    return r;
}
template <typename Codec, bool kAligned>
__device__ __forceinline__ void ClearBehind(Raw<Codec>& r, int64_t c, int64_t end) {
    constexpr int kPieces = sizeof(typename Codec::Storage) / 2, kPer = 8 / kPieces;
    if constexpr (kAligned) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (c + i * kPer >= end) r.q[i] = uint4{0, 0, 0, 0};
        }
    }
}

// Operands of the matrix instructions: one of the type itself, or kParts of bf16.
template <typename Codec, int kParts>
struct Parts {
    uint4 p[kParts];
};

// The upper halves of two values, cut off; and the nearest bf16 to each.
__device__ __forceinline__ uint32_t CutTwo(float even, float odd) {
    return __builtin_amdgcn_perm(__float_as_uint(odd), __float_as_uint(even), 0x07060302u);
}
__device__ __forceinline__ uint32_t NearestTwo(float even, float odd) {
    typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
    typedef float F32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(F32x2{even, odd}, Bf16x2));
}

template <typename Codec, int kParts, bool kNearest>
__device__ __forceinline__ Parts<Codec, kParts> PartsOf(const Raw<Codec>& r) {
    Parts<Codec, kParts> out;
    if constexpr (kParts == 1) {
        static_assert(sizeof(typename Codec::Storage) == 2);
        out.p[0] = r.q[0];
    } else {
        uint32_t words[kParts][4];
#pragma unroll
        for (int pair = 0; pair < 4; ++pair) {
            float v[2];
            if constexpr (std::is_same_v<Codec, F32>) {
                const uint4 q = r.q[pair / 2];
                v[0] = __uint_as_float(pair % 2 == 0 ? q.x : q.z);
                v[1] = __uint_as_float(pair % 2 == 0 ? q.y : q.w);
            } else {
                const uint4 q = r.q[0];
                const uint32_t two = pair == 0 ? q.x : pair == 1 ? q.y : pair == 2 ? q.z : q.w;
                v[0] = Codec::Load(static_cast<uint16_t>(two));
                v[1] = Codec::Load(static_cast<uint16_t>(two >> 16));
            }
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                if constexpr (kNearest) {
                    words[part][pair] = NearestTwo(v[0], v[1]);
                    v[0] -= __uint_as_float(words[part][pair] << 16);
                    v[1] -= __uint_as_float(words[part][pair] & 0xffff0000u);
                } else {
                    words[part][pair] = CutTwo(v[0], v[1]);
                    v[0] -= __uint_as_float(__float_as_uint(v[0]) & 0xffff0000u);
                    v[1] -= __uint_as_float(__float_as_uint(v[1]) & 0xffff0000u);
                }
            }
        }
#pragma unroll
        for (int part = 0; part < kParts; ++part) out.p[part] = uint4{words[part][0], words[part][1], words[part][2], words[part][3]};
    }
    return out;
}

// Element types of the two sides and the number of parts of each.
template <typename X, typename W>
struct Sides {
    using XType = X;
    using WType = W;
    static constexpr bool kSame16 = std::is_same_v<X, W> && sizeof(typename X::Storage) == 2;
    static constexpr int kX = kSame16 || std::is_same_v<X, Bf16> ? 1 : std::is_same_v<X, F16> ? 2 : 3;
    static constexpr int kW = kSame16 ? 1 : 3;
    static constexpr bool kNearest = kX > 1;  // parts that leave the least to the products that are left out
    static constexpr bool kHalf = kSame16 && std::is_same_v<X, F16>;  // fp16 instructions; bf16 otherwise
};

template <bool kHalf>
__device__ __forceinline__ F32x4 Multiply(const uint4& a, const uint4& b, F32x4 c) {  // 16 x 16 x 32
    if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16x8, a), __builtin_bit_cast(F16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}
template <bool kHalf>
__device__ __forceinline__ F32x16 Multiply(const uint4& a, const uint4& b, F32x16 c) {  // 32 x 32 x 16
    if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(F16x8, a), __builtin_bit_cast(F16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}

// Few rows: operands go from memory to registers, the waves of a workgroup share its columns, 32 at a time in turn, and add up through LDS.  A workgroup makes
// kM x kN tiles of 16 rows and 16 experts.  With kSub > 1 (kM = kN = 1) the sixteen lines of either operand are 16 / kSub rows or experts times kSub
// neighbouring runs of 32 columns: the products of a run with itself, one in kSub, are what is added up, and a workgroup streams fewer experts' weights.
// What bounds it: one round trip to memory and the launch for a row (1 x 4096 x 128, bf16 2.9 us), the time a CU takes to bring in its share for a decode step
// (64 x 7168 x 256, fp32 weights 8.2, fp16 and fp32 rows on them 10.0 and 11.4: 256 workgroups of 350 KB, of which the L2 serves all but 14.4 MB; that is the
// shape's doing, whose workgroups take all columns), memory for prompts of few experts (16384 x 4096 x 8 22 us alone, 26 in a row of calls: a copy's rate).
template <typename S, int kM, int kN, int kSub, int kWaves, bool kAligned>
__global__ __launch_bounds__(kWave * kWaves) void RouterLogitsSlimKernel(LogitsArgs a) {
    using X = typename S::XType;
    using W = typename S::WType;
    constexpr int kLines = 16 / kSub;
    __shared__ F32x4 sums[kWaves * kM * kN][kWave];
    constexpr int kDepth = kM * kN > 1 ? 2 : 4;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int line = lane % 16 / kSub, sub = lane % 16 % kSub;
    // Workgroups go round robin over the eight XCDs: neighbours take different experts, whose weights then come to one L2 each.
    const int tilesN = (a.experts + kLines * kN - 1) / (kLines * kN);
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / tilesN) * (kLines * kM);
    const int expert0 = static_cast<int>(blockIdx.x % tilesN) * (kLines * kN);
    const int64_t end = a.cols;
    const typename X::Storage* x[kM];
    const typename W::Storage* w[kN];
#pragma unroll
    for (int m = 0; m < kM; ++m) x[m] = static_cast<const typename X::Storage*>(a.x) + min(row0 + m * kLines + line, a.rows - 1) * a.cols;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
        w[n] = static_cast<const typename W::Storage*>(a.weight) + static_cast<int64_t>(min(expert0 + n * kLines + line, a.experts - 1)) * a.cols;
    }
    const typename X::Storage* const xLimit = static_cast<const typename X::Storage*>(a.x) + a.rows * a.cols;
    const typename W::Storage* const wLimit = static_cast<const typename W::Storage*>(a.weight) + a.experts * a.cols;
    F32x4 acc[kM][kN] = {};
    const int at = (lane / 16 * kSub + sub) * 8;
    // kCount runs of 32 kSub columns from `base` on, a round of all waves apart; kWhole: all of them end within the row.
    constexpr int kRound = kWaves * kSub * 32;
    auto pass = [&](int64_t base, auto countOf, auto wholeOf) {
        constexpr int kCount = decltype(countOf)::value;
        Raw<X> xr[kCount][kM];
        Raw<W> wr[kCount][kN];
#pragma unroll
        for (int d = 0; d < kCount; ++d) {
            const int64_t c = base + d * kRound + at;
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                if constexpr (kAligned) wr[d][n] = LoadRaw<W>(w[n], c, end);
                else if constexpr (decltype(wholeOf)::value) wr[d][n] = LoadWhole<W>(w[n] + c);
                else wr[d][n] = LoadEnd<W>(w[n], c, end, wLimit);
            }
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                if constexpr (kAligned) xr[d][m] = LoadRaw<X>(x[m], c, end);
                else if constexpr (decltype(wholeOf)::value) xr[d][m] = LoadWhole<X>(x[m] + c);
                else xr[d][m] = LoadEnd<X>(x[m], c, end, xLimit);
            }
        }
#pragma unroll
        for (int d = 0; d < kCount; ++d) {
            Parts<X, S::kX> xp[kM];
#pragma unroll
            for (int m = 0; m < kM; ++m) xp[m] = PartsOf<X, S::kX, S::kNearest>(xr[d][m]);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
                const Parts<W, S::kW> wp = PartsOf<W, S::kW, S::kNearest>(wr[d][n]);
#pragma unroll
                for (int m = 0; m < kM; ++m) {
#pragma unroll
                    for (int i = S::kX - 1; i >= 0; --i) {
#pragma unroll
                        for (int j = S::kW - 1; j >= 0; --j) {
                            if (i + j <= 2) acc[m][n] = Multiply<S::kHalf>(xp[m].p[i], wp.p[j], acc[m][n]);
                        }
                    }
                }
            }
        }
    };
    using One = std::integral_constant<int, 1>;
    using Depth = std::integral_constant<int, kDepth>;
    int64_t base = wave * (kSub * 32);
    if constexpr (kAligned) {
        for (; base < end; base += kDepth * kRound) pass(base, Depth{}, std::false_type{});
    } else {
        for (; base + (kDepth - 1) * kRound + kSub * 32 <= end; base += kDepth * kRound) pass(base, Depth{}, std::true_type{});
        for (; base + kSub * 32 <= end; base += kRound) pass(base, One{}, std::true_type{});
        if (base < end) pass(base, One{}, std::false_type{});
    }
    // of a tile, lane l holds the columns l % 16 of the lines l / 16 * 4 + 0 .. 3
#pragma unroll
    for (int m = 0; m < kM; ++m) {
#pragma unroll
        for (int n = 0; n < kN; ++n) sums[wave * kM * kN + m * kN + n][lane] = acc[m][n];
    }
    __syncthreads();
    const float* const all = reinterpret_cast<const float*>(sums);
    for (int i = threadIdx.x; i < kLines * kM * kLines * kN; i += kWave * kWaves) {
        const int r = i / (kLines * kN), e = i % (kLines * kN);
        const int64_t row = row0 + r;
        const int expert = expert0 + e;
        const int tile = r / kLines * kN + e / kLines;
        float sum = 0.f;
        for (int v = 0; v < kWaves; ++v) {
#pragma unroll
            for (int t = 0; t < kSub; ++t) {
                const int i16 = r % kLines * kSub + t, j16 = e % kLines * kSub + t;
                sum += all[((v * kM * kN + tile) * kWave + i16 / 4 * 16 + j16) * 4 + i16 % 4];
            }
        }
        if (row < a.rows && expert < a.experts) a.logits[row * a.experts + expert] = sum;
    }
}

// Many rows: eight waves, kWavesM x kWavesN of them with kMt tiles of 32 x 32 products each, one below the other.  Rows and weights come through LDS, two buffers
// deep.  Rows are cut into parts on the way in, since every wave of a line reads them; weights of fp32 stay whole and are cut by the one wave (kWavesM of
// them) that has those experts: four bytes of theirs are moved in place of six.  Lines in LDS are 16 bytes longer than their columns, so that eight
// lanes of a fragment read meet eight different sets of banks.
// What bounds it: 8192 x 7168 x 256, fp32 weights 85 us and 7 for adding the splits up; 64 are the three parts' products at the rate of a large matrix product
// (1409 TFLOP/s).  The matrix instructions are under way for 59 % of the time that CUs work, cutting weights into parts takes another 45 % of the vector
// unit's, at 1.7 GHz.  fp16 and fp32 rows on fp32 weights 136 and 169 us, 107 and 128 of them five and six parts' products.  With bf16 weights
// 48 in 128 x 256 tiles and four splits, for which the costs below take 128 x 128 in two (53 to 56); 25 are the bytes.  Products a fragment ahead and 64 columns
// a step took 600 x 7168 x 256 from 22.7 to 20.0 us, 16384 x 2880 x 60 from 38.7 to 28.4.
constexpr int kTileThreads = 512;

template <typename S, int kWavesM, int kWavesN, int kMt>
struct TileShape {
    static constexpr int kBm = kWavesM * kMt * 32, kBn = kWavesN * 32;
    static constexpr int kWSize = sizeof(typename S::WType::Storage);
    static constexpr int kBk = S::kX == 1 && (S::kW == 1 || kBn < 256) ? 64 : 32;
    static constexpr int kXPitch = kBk * 2 + 16, kWPitch = kBk * kWSize + 16;
    static constexpr int kXBytes = S::kX * kBm * kXPitch;
    static constexpr int kStage = kXBytes + kBn * kWPitch;
    static constexpr int kBytes = 2 * kStage;
};

template <typename S, int kWavesM, int kWavesN, int kMt, bool kAligned>
__global__ __attribute__((amdgpu_flat_work_group_size(kTileThreads, kTileThreads), amdgpu_waves_per_eu(2))) void
RouterLogitsTileKernel(LogitsArgs a, int tilesN, int groups) {
    static_assert(kWavesM * kWavesN == kTileThreads / kWave);
    using X = typename S::XType;
    using W = typename S::WType;
    using Shape = TileShape<S, kWavesM, kWavesN, kMt>;
    constexpr int kBm = Shape::kBm, kBn = Shape::kBn, kBk = Shape::kBk, kChunks = kBk / 8;
    constexpr int kLineStep = kTileThreads / kChunks;
    constexpr int kXLoads = (kBm + kLineStep - 1) / kLineStep, kWLoads = (kBn + kLineStep - 1) / kLineStep;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    // Workgroups go round robin over the eight XCDs; those of one XCD take neighbouring rows of the same columns, whose weights their L2 holds.
    const int linear = blockIdx.x, perXcd = groups / 8;
    const int id = linear < perXcd * 8 ? linear % 8 * perXcd + linear / 8 : linear;
    const int tileN = id % tilesN, rest = id / tilesN;
    const int tilesM = static_cast<int>((a.rows + kBm - 1) / kBm);
    const int64_t row0 = static_cast<int64_t>(rest % tilesM) * kBm;
    const int split = rest / tilesM;
    const int expert0 = tileN * kBn;
    const int64_t begin = split * a.splitCols, end = min(a.cols, begin + a.splitCols);
    const int steps = static_cast<int>((end - begin + kBk - 1) / kBk);

    const int chunk = tid % kChunks, lineOf = tid / kChunks;
    const typename X::Storage* x[kXLoads];
    const typename W::Storage* w[kWLoads];
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
        x[i] = static_cast<const typename X::Storage*>(a.x) + min(row0 + lineOf + i * kLineStep, a.rows - 1) * a.cols;
    }
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) {
        w[i] = static_cast<const typename W::Storage*>(a.weight) + static_cast<int64_t>(min(expert0 + lineOf + i * kLineStep, a.experts - 1)) * a.cols;
    }
    Raw<X> xr[kXLoads];
    Raw<W> wr[kWLoads];
    // Rows and weights are asked for half a step apart, each a whole step ahead of the store into LDS: there is always half a stage under way.
    auto columnOf = [&](int step) { return begin + static_cast<int64_t>(step) * kBk + chunk * 8; };
    auto isTail = [&](int step) { return begin + static_cast<int64_t>(step + 1) * kBk > end; };
    auto load = [&](auto codec, const auto* row, const auto* limit, int step) {
        using Codec = decltype(codec);
        if constexpr (kAligned) return LoadClamped<Codec>(row, columnOf(step), end);
        else return isTail(step) ? LoadEnd<Codec>(row, columnOf(step), end, limit) : LoadWhole<Codec>(row + columnOf(step));
    };
    const typename X::Storage* const xLimit = static_cast<const typename X::Storage*>(a.x) + a.rows * a.cols;
    const typename W::Storage* const wLimit = static_cast<const typename W::Storage*>(a.weight) + a.experts * a.cols;
    auto loadX = [&](int step) {
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) {
            if (kBm % kLineStep == 0 || lineOf + i * kLineStep < kBm) xr[i] = load(X{}, x[i], xLimit, step);
        }
    };
    auto loadW = [&](int step) {
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) {
            if (kBn % kLineStep == 0 || lineOf + i * kLineStep < kBn) wr[i] = load(W{}, w[i], wLimit, step);
        }
    };
    auto storeW = [&](int step) {
        unsigned char* const stage = lds + step % 2 * Shape::kStage;
        if (isTail(step)) {
#pragma unroll
            for (int i = 0; i < kWLoads; ++i) ClearBehind<W, kAligned>(wr[i], columnOf(step), end);
        }
#pragma unroll
        for (int i = 0; i < kWLoads; ++i) {
            if (kBn % kLineStep != 0 && lineOf + i * kLineStep >= kBn) continue;
            uint4* const to = reinterpret_cast<uint4*>(stage + Shape::kXBytes + (lineOf + i * kLineStep) * Shape::kWPitch + chunk * (8 * Shape::kWSize));
#pragma unroll
            for (int q = 0; q < Shape::kWSize / 2; ++q) to[q] = wr[i].q[q];
        }
    };
    auto storeX = [&](int step) {
        unsigned char* const stage = lds + step % 2 * Shape::kStage;
        if (isTail(step)) {
#pragma unroll
            for (int i = 0; i < kXLoads; ++i) ClearBehind<X, kAligned>(xr[i], columnOf(step), end);
        }
#pragma unroll
        for (int i = 0; i < kXLoads; ++i) {
            if (kBm % kLineStep != 0 && lineOf + i * kLineStep >= kBm) continue;
            const Parts<X, S::kX> parts = PartsOf<X, S::kX, S::kNearest>(xr[i]);
#pragma unroll
            for (int p = 0; p < S::kX; ++p) {
                *reinterpret_cast<uint4*>(stage + (p * kBm + lineOf + i * kLineStep) * Shape::kXPitch + chunk * 16) = parts.p[p];
            }
        }
    };

    F32x16 acc[kMt] = {};
    const int waveN = wave % kWavesN, waveM = wave / kWavesN;
    const int xAt = (waveM * (kMt * 32) + lane % 32) * Shape::kXPitch + lane / 32 * 16;
    const int wAt = Shape::kXBytes + (waveN * 32 + lane % 32) * Shape::kWPitch + lane / 32 * (8 * Shape::kWSize);
    // Fragments are read one product of 16 columns ahead, or every product waits for its own; the scheduling barriers keep the compiler to that.
    struct Fragments {
        uint4 x[S::kX][kMt];
        Raw<W> w;
    };
    auto read = [&](const unsigned char* stage, int k, Fragments& f) {
#pragma unroll
        for (int q = 0; q < Shape::kWSize / 2; ++q) f.w.q[q] = reinterpret_cast<const uint4*>(stage + wAt + k * (16 * Shape::kWSize))[q];
#pragma unroll
        for (int p = 0; p < S::kX; ++p) {
#pragma unroll
            for (int m = 0; m < kMt; ++m) f.x[p][m] = *reinterpret_cast<const uint4*>(stage + xAt + (p * kBm + m * 32) * Shape::kXPitch + k * 32);
        }
    };
    auto multiply = [&](const Fragments& f) {
        const Parts<W, S::kW> wf = PartsOf<W, S::kW, S::kNearest>(f.w);
#pragma unroll
        for (int i = S::kX - 1; i >= 0; --i) {
#pragma unroll
            for (int j = S::kW - 1; j >= 0; --j) {
                if (i + j > 2) continue;
#pragma unroll
                for (int m = 0; m < kMt; ++m) acc[m] = Multiply<S::kHalf>(f.x[i][m], wf.p[j], acc[m]);
            }
        }
    };
    loadX(0);
    loadW(0);
    storeX(0);
    loadX(1);
    storeW(0);
    loadW(1);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const unsigned char* const stage = lds + step % 2 * Shape::kStage;
        constexpr int kProducts = kBk / 16;
        Fragments f[2];
        read(stage, 0, f[0]);
#pragma unroll
        for (int k = 0; k < kProducts; ++k) {
            if (k + 1 < kProducts) read(stage, k + 1, f[(k + 1) % 2]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(f[k % 2]);
            __builtin_amdgcn_sched_barrier(0);
            if (k == 0) {
                storeX(step + 1);
                loadX(step + 2);
            }
            if (k == kProducts / 2) {
                storeW(step + 1);
                loadW(step + 2);
            }
        }
        __syncthreads();
    }
    // of a tile, lane l holds column l % 32 of the lines 8 (i / 4) + 4 (l / 32) + i % 4, i = 0 .. 15
    float* const out = a.logits + static_cast<int64_t>(split) * a.rows * a.experts;
    const int expert = expert0 + waveN * 32 + lane % 32;
#pragma unroll
    for (int m = 0; m < kMt; ++m) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int64_t row = row0 + (waveM * kMt + m) * 32 + 8 * (i / 4) + 4 * (lane / 32) + i % 4;
            if (row < a.rows && expert < a.experts) out[row * a.experts + expert] = acc[m][i];
        }
    }
}

// Adds the splits up, in their order.
constexpr int kAddThreads = 256;

template <int kVec>
__global__ __launch_bounds__(kAddThreads) void AddSplitsKernel(const float* partial, float* logits, int64_t count, int splits) {
    typedef float Vec __attribute__((ext_vector_type(kVec)));
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kAddThreads + threadIdx.x;
    if (i * kVec >= count) return;
    Vec sum = reinterpret_cast<const Vec*>(partial)[i];
#pragma unroll 4
    for (int s = 1; s < splits; ++s) sum += reinterpret_cast<const Vec*>(partial + s * count)[i];
    reinterpret_cast<Vec*>(logits)[i] = sum;
}

// What there is to choose from, in the order of LaunchPlan, and what a call is taken to cost: fitted to 320 000 measurements of 50 900 calls over the operator's
// range (1 to 16384 rows, 4 to 512 experts, 512 to 8192 columns, all types).  In nine of ten the fit is 0.77 to 1.18 of what was measured; the choice by it costs
// 1.8 % more than the best shape in the mean, 7 % in one call of ten, 50 % at worst (columns off the 16-byte grid 1.4 % in the mean, odd ones of 16 bits 2.8).
// A shape each kind of call needs: without the slim kernels decode takes longer (64 x 7168 x 256, fp32 weights: 12.3 against 8.3 us, one row 10.8 against
// 3.5), without the tiles a prompt does (8192 x 7168 x 256, fp32 weights: 332 against 94 us).
struct Slim {
    int m, n, sub, waves;
};
struct Tile {
    int rows, experts;
};
constexpr int kSlims = 6, kTiles = 5;
constexpr Slim kSlim[kSlims] = {{1, 1, 16, 4}, {1, 1, 4, 8}, {2, 1, 4, 8}, {1, 1, 2, 8}, {2, 1, 2, 8}, {2, 2, 2, 8}};
constexpr Tile kTile[kTiles] = {{128, 64}, {128, 128}, {128, 256}, {256, 64}, {256, 128}};
// us: of a launch; of 100 KB that come to a CU, eight waves that start and the cutting into parts, for each workgroup that a CU gets in turn; of a megabyte of
// operands
constexpr double kSlimUs[] = {3.10, 1.00, 0.235, 1.136, 0.091};
// us: of a launch; a step of one part and of several; 100 KB, and the products at 2.5 PFLOP/s over all CUs; adding splits up, and a megabyte of them; a workgroup
constexpr double kTileUs[] = {4.01, 0.0135, 0.301, 0.930, 1.058, 2.48, 0.376, 1.84};

class LogitsExecutor : public aclOpExecutor {
   public:
    LogitsArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType weightType = ACL_FLOAT;
    // The plan, made from sizes and types alone: the workspace that is asked for does not hang on addresses.  Tensors whose extents are on the 16-byte grid and
    // whose addresses are not run the shape chosen for the grid, by its kernel for rows off it.
    int kernel = 0;  // of kSlim, then of kTile
    int splits = 1;

    void Plan() {
        const double T = static_cast<double>(args.rows), K = static_cast<double>(args.cols), E = args.experts;
        const double xSize = static_cast<double>(opapi::ElemSize(dtype)), wSize = static_cast<double>(opapi::ElemSize(weightType));
        const bool same16 = dtype == weightType && dtype != ACL_FLOAT;
        const int xParts = same16 || dtype == ACL_BF16 ? 1 : dtype == ACL_FLOAT16 ? 2 : 3;
        // bytes off the 16-byte grid take longer to come, most of all where rows start between two words and each is read by many
        const int64_t rowBytes[] = {args.cols * opapi::ElemSize(dtype), args.cols * opapi::ElemSize(weightType)};
        const double slimBytes = rowBytes[0] % 4 != 0 ? 3 : rowBytes[0] % 16 != 0 || rowBytes[1] % 16 != 0 ? 1.5 : 1, tileBytes = slimBytes > 1 ? 1.5 : 1;
        const double products = same16 ? 1 : xParts == 1 ? 3 : xParts == 2 ? 5 : 6;
        auto over = [](double n, double d) { return std::ceil(n / d); };
        double best = 0;
        const double operands = (T * K * xSize + E * K * wSize) * 1e-6, streamed = kSlimUs[0] + 0.19 * operands;  // at a copy's 5.2 TB/s
        auto offer = [&](double us, int which, int split) {
            if (us < streamed) us = streamed;
            if (best != 0 && us >= best) return;
            best = us;
            kernel = which;
            splits = split;
        };
        for (int i = 0; i < kSlims; ++i) {
            const Slim& v = kSlim[i];
            const double rows = 16 / v.sub * v.m, experts = 16 / v.sub * v.n;
            if (over(T, rows) * over(E, experts) * v.waves * kWave > kMaxThreads) continue;
            const double rounds = over(over(T, rows) * over(E, experts), 256), steps = over(K, 32 * v.sub * v.waves) * v.waves / 4;
            const double cuts = ((same16 ? 0 : 3) * v.n + (xParts > 1 ? 3 : 0) * v.m) * steps * 32 / 2400;
            offer(kSlimUs[0] + kSlimUs[4] * operands + rounds * (kSlimUs[1] * slimBytes * K * (rows * xSize + experts * wSize) * 1e-5 + kSlimUs[2] * v.waves / 8 + kSlimUs[3] * cuts), i, 1);
        }
        for (int i = 0; i < kTiles; ++i) {
            const Tile& v = kTile[i];
            if (v.rows > 128 && xParts > 1) continue;
            const double tiles = over(T, v.rows) * over(E, v.experts), bk = same16 || (xParts == 1 && v.experts < 256) ? 64 : 32;
            if (tiles * kTileThreads > kMaxThreads) continue;
            const double perCu = 2 * (xParts * v.rows * (2 * bk + 16) + v.experts * (wSize * bk + 16)) > 80 * 1024 ? 1 : 2;
            for (const int target : {128, 256, 512}) {
                int split = static_cast<int>(target / tiles);
                if (split < 1) split = 1;
                if (split > 1 && K / split < 128) continue;
                const double cols = over(K / split, 64) * 64, used = over(K, cols), rounds = over(tiles * used, 256);
                const double turns = over(rounds, perCu), bytes = cols * (v.rows * xSize + v.experts * wSize);
                const double flops = v.rows * v.experts * cols * products * 2;
                double us = kTileUs[0] + turns * (kTileUs[same16 ? 1 : 2] * cols / bk + kTileUs[7]) + rounds * (kTileUs[3] * tileBytes * bytes * 1e-5 + kTileUs[4] * flops * 256 / 2.5e9);
                if (used > 1) us += kTileUs[5] + kTileUs[6] * used * T * E * 4e-6;
                offer(us, kSlims + i, static_cast<int>(used));
            }
        }
        args.splitCols = static_cast<int64_t>(over(K / splits, 64)) * 64;
    }

    uint64_t OwnBytes() const { return splits > 1 ? static_cast<uint64_t>(splits) * args.rows * args.experts * sizeof(float) : 0; }

    template <typename S, int kM, int kN, int kSub, int kWaves, bool kAligned>
    hipError_t LaunchSlim(const LogitsArgs& a, hipStream_t stream) const {
        constexpr int kLines = 16 / kSub;
        const int64_t groups = (a.rows + kLines * kM - 1) / (kLines * kM) * ((a.experts + kLines * kN - 1) / (kLines * kN));
        hipLaunchKernelGGL((RouterLogitsSlimKernel<S, kM, kN, kSub, kWaves, kAligned>), dim3(static_cast<unsigned>(groups)), dim3(kWave * kWaves), 0, stream, a);
        return hipGetLastError();
    }

    template <typename S, int kWavesM, int kWavesN, int kMt, bool kAligned>
    hipError_t LaunchTile(const LogitsArgs& a, hipStream_t stream) const {
        using Shape = TileShape<S, kWavesM, kWavesN, kMt>;
        auto kernel = RouterLogitsTileKernel<S, kWavesM, kWavesN, kMt, kAligned>;
        static_assert(Shape::kBytes <= 160 * 1024);
        static std::atomic<uint64_t> optedIn{0};
        const hipError_t attr = opapi::EnsureDynamicLds(reinterpret_cast<const void*>(kernel), Shape::kBytes, optedIn);
        if (attr != hipSuccess) return attr;
        const int tilesN = static_cast<int>((a.experts + Shape::kBn - 1) / Shape::kBn);
        const int64_t groups = (a.rows + Shape::kBm - 1) / Shape::kBm * tilesN * splits;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(kTileThreads), Shape::kBytes, stream, a, tilesN, static_cast<int>(groups));
        return hipGetLastError();
    }

    template <typename S, bool kAligned>
    hipError_t LaunchPlan(const LogitsArgs& a, hipStream_t stream) const {
        switch (kernel) {
            case 0: return LaunchSlim<S, 1, 1, 16, 4, kAligned>(a, stream);
            case 1: return LaunchSlim<S, 1, 1, 4, 8, kAligned>(a, stream);
            case 2: return LaunchSlim<S, 2, 1, 4, 8, kAligned>(a, stream);
            case 3: return LaunchSlim<S, 1, 1, 2, 8, kAligned>(a, stream);
            case 4: return LaunchSlim<S, 2, 1, 2, 8, kAligned>(a, stream);
            case 5: return LaunchSlim<S, 2, 2, 2, 8, kAligned>(a, stream);
            case 6: return LaunchTile<S, 4, 2, 1, kAligned>(a, stream);
            case 7: return LaunchTile<S, 2, 4, 2, kAligned>(a, stream);
            case 8: return LaunchTile<S, 1, 8, 4, kAligned>(a, stream);
            default: break;
        }
        if constexpr (S::kX == 1) return kernel == 9 ? LaunchTile<S, 4, 2, 2, kAligned>(a, stream) : LaunchTile<S, 2, 4, 4, kAligned>(a, stream);
        return hipErrorInvalidValue;  // not planned for rows of several parts
    }

    template <typename X, typename W>
    hipError_t Launch(const LogitsArgs& a, hipStream_t stream) const {
        auto onGrid = [&](const void* p, size_t size) {
            return reinterpret_cast<uintptr_t>(p) % 16 == 0 && static_cast<uint64_t>(a.cols) * size % 16 == 0;
        };
        const bool aligned = onGrid(a.x, sizeof(typename X::Storage)) && onGrid(a.weight, sizeof(typename W::Storage));
        opapi::KernelTimer timer("router_logits", stream);
        return aligned ? LaunchPlan<Sides<X, W>, true>(a, stream) : LaunchPlan<Sides<X, W>, false>(a, stream);
    }

    aclnnStatus Run(void* workspace, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        OPAPI_CHECK(OwnBytes() == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, ACLNN_ERR_PARAM_INVALID,
                    "aclnnMoeRouterLogits: the workspace must be 16-byte aligned");
        hipError_t err;
        LogitsArgs a = args;
        float* const partial = static_cast<float*>(workspace);
        if (splits > 1) a.logits = partial;
        if (dtype == ACL_FLOAT) err = Launch<F32, F32>(a, stream);
        else if (dtype == ACL_FLOAT16) err = weightType == ACL_FLOAT ? Launch<F16, F32>(a, stream) : Launch<F16, F16>(a, stream);
        else err = weightType == ACL_FLOAT ? Launch<Bf16, F32>(a, stream) : Launch<Bf16, Bf16>(a, stream);
        if (err == hipSuccess && splits > 1) {
            opapi::KernelTimer timer("router_logits_add", stream);
            const int64_t count = args.rows * args.experts;
            const int vec = count % 4 == 0 && reinterpret_cast<uintptr_t>(args.logits) % 16 == 0 ? 4 : 1;
            const unsigned blocks = static_cast<unsigned>((count / vec + kAddThreads - 1) / kAddThreads);
            if (vec == 4) hipLaunchKernelGGL(AddSplitsKernel<4>, dim3(blocks), dim3(kAddThreads), 0, stream, partial, args.logits, count, splits);
            else hipLaunchKernelGGL(AddSplitsKernel<1>, dim3(blocks), dim3(kAddThreads), 0, stream, partial, args.logits, count, splits);
            err = hipGetLastError();
        }
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
    OPAPI_CHECK(rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
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
    if (rows > 0) ex->Plan();
    ex->SealWorkspace(ex->OwnBytes());
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

extern "C" int opapiRouterLogitsPlan(int xType, int weightType, int64_t rows, int64_t cols, int64_t experts, int* shape, int* splits) {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK(shape != nullptr && splits != nullptr, ACLNN_ERR_PARAM_NULLPTR, "shape or splits is null");
    const auto floating = [](int type) { return type == ACL_FLOAT || type == ACL_FLOAT16 || type == ACL_BF16; };
    OPAPI_CHECK(floating(xType) && (weightType == xType || weightType == ACL_FLOAT), ACLNN_ERR_PARAM_INVALID,
                "x must be FLOAT, FLOAT16 or BF16, weight of x's type or FLOAT");
    OPAPI_CHECK(rows > 0 && rows <= kMaxRows && cols > 0 && cols <= 2147483647ll && experts > 0 && experts <= kMaxExperts, ACLNN_ERR_PARAM_INVALID,
                "rows, cols or experts are out of range");
    LogitsExecutor ex;
    ex.dtype = static_cast<aclDataType>(xType);
    ex.weightType = static_cast<aclDataType>(weightType);
    ex.args.rows = rows;
    ex.args.cols = cols;
    ex.args.experts = static_cast<int32_t>(experts);
    ex.Plan();
    *shape = ex.kernel;
    *splits = ex.splits;
    return ACLNN_SUCCESS;
}
