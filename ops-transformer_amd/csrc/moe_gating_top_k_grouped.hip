// aclnnMoeGatingTopKGrouped for gfx950: softmax or sigmoid scores, a bias that moves the choice only, groups, top-k.
//
// Two experts change places when their t = p + bias do, and near the top of 256 sigmoid scores a pair within fp32's rounding of an exponential
// comes up in one row of some thousands.  The choice is defined in 64 bits, and every row is chosen as if it were made there: the
// fast kernel works on fp32 scores whose error it can bound, and where two values that decide something are closer than that, the wave makes
// that row again in 64 bits.  Without a bias t is a monotone function of the logit: logits are compared in its place, exactly.
// Keys are order-preserving: the bits of a number mapped so that unsigned comparison equals that of the numbers, NaN on top.  Key 0 marks an
// expert that is taken or lies in a group that was left out; it is below every real value, -inf (an expert of logit -inf) among them.
#include "moe_front.h"

#include <cmath>

#include "aclnnop/aclnn_moe_gating_top_k_grouped.h"

namespace {

using namespace moe_front;

constexpr int64_t kMaxExperts = 2048;
constexpr int64_t kMaxPicks = 64;

struct GatingArgs {
    const void* x;
    const float* bias;        // optional
    const uint8_t* finished;  // optional, one byte per row
    void* y;
    int32_t* expertIdx;
    float* scores;            // optional
    int64_t rows;
    int32_t experts;
    int32_t k;
    int32_t groups;
    int32_t kGroup;
    int32_t topTwo;           // a group's value is the sum of its two largest t
    int32_t sigmoid;
    int32_t renorm;
    int32_t packets;          // lanes have all of their experts or none (1), or all of them have (2), and rows start on the lanes' boundaries
    int32_t biasPackets;      // so does the bias
    uint32_t groupMagic;      // (c * groupMagic) >> 21 = c / (experts / groups) for c < 512
    double factor;
    double eps;
};

__device__ __forceinline__ uint64_t KeyOf(double d) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(d));
    if (d != d) return ~0ull;
    return (u >> 63) != 0 ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double ValueOf(uint64_t key) {
    if (key == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
    return __longlong_as_double(static_cast<long long>((key >> 63) != 0 ? key & 0x7fffffffffffffffull : ~key));
}

// -0 as 0, whose key is another's.
__device__ __forceinline__ float Unsigned0(float f) { return f + 0.f; }

__device__ __forceinline__ double WaveSum64(double v) {
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// The largest key of the wave and the lowest index that holds it; every lane brings the largest of its own and that one's lowest index.
__device__ __forceinline__ void WaveArgMax(uint64_t& key, int32_t& idx) {
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t otherKey = __shfl_xor(static_cast<unsigned long long>(key), d);
        const int32_t otherIdx = __shfl_xor(idx, d);
        if (otherKey > key || (otherKey == key && otherIdx < idx)) {
            key = otherKey;
            idx = otherIdx;
        }
    }
}

// p of one logit.  shift and sum are the row's largest logit and sum of exponentials under softmax.
__device__ __forceinline__ double ScoreOf(float x, bool sigmoid, double shift, double sum) {
    if (x == -INFINITY) return 0.0;
    return sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : exp(static_cast<double>(x) - shift) / sum;
}

// What one lane of the wave has written to LDS, the others read: the wave's accesses are carried out in order, the compiler must keep them so.
__device__ __forceinline__ void WaveSync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A row by one wave in 64 bits.  keys: [experts + groups] in LDS, the wave's own.
template <typename Codec, typename Out>
__device__ void ExactRow(const GatingArgs& a, int64_t row, int lane, uint64_t* keys, bool writeScores) {
    uint64_t* const groupKeys = keys + a.experts;
    const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x) + row * a.experts;
    const bool sigmoid = a.sigmoid != 0;

    double shift = 0.0, sum = 1.0;
    if (!sigmoid) {
        float top = -INFINITY;
        bool nan = false;
        for (int c = lane; c < a.experts; c += kWave) {
            const float v = Codec::Load(x[c]);
            top = fmaxf(top, v);
            nan |= v != v;
        }
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        shift = __any(nan) ? NAN : top;
        sum = 0.0;
        for (int c = lane; c < a.experts; c += kWave) sum += ScoreOf(Codec::Load(x[c]), false, shift, 1.0);
        sum = WaveSum64(sum);
    }
    for (int c = lane; c < a.experts; c += kWave) {
        const float v = Codec::Load(x[c]);
        const double p = a.bias != nullptr || writeScores ? ScoreOf(v, sigmoid, shift, sum) : 0.0;
        if (writeScores) a.scores[row * a.experts + c] = static_cast<float>(p);
        keys[c] = KeyOf(v == -INFINITY ? -INFINITY : a.bias == nullptr ? static_cast<double>(Unsigned0(v)) : p + static_cast<double>(a.bias[c]));
    }
    WaveSync();

    if (a.kGroup < a.groups) {
        const int size = a.experts / a.groups;
        for (int g = lane; g < a.groups; g += kWave) {
            uint64_t first = 0, second = 0;
            for (int c = g * size; c < (g + 1) * size; ++c) {
                const uint64_t key = keys[c];
                if (key > first) {
                    second = first;
                    first = key;
                } else if (key > second) {
                    second = key;
                }
            }
            double one = ValueOf(first), two = ValueOf(second);
            if (a.topTwo != 0 && two != -INFINITY) {
                if (a.bias == nullptr) {
                    one = ScoreOf(static_cast<float>(one), sigmoid, shift, sum);
                    two = ScoreOf(static_cast<float>(two), sigmoid, shift, sum);
                }
                first = KeyOf(one + two);
            } else if (a.topTwo != 0 && a.bias == nullptr && one != -INFINITY) {
                first = KeyOf(ScoreOf(static_cast<float>(one), sigmoid, shift, sum));
            }
            groupKeys[g] = first;
        }
        WaveSync();
        for (int j = 0; j < a.kGroup; ++j) {
            uint64_t best = 0;
            int32_t at = INT32_MAX;
            for (int g = lane; g < a.groups; g += kWave) {
                if (groupKeys[g] > best) {
                    best = groupKeys[g];
                    at = g;
                }
            }
            WaveArgMax(best, at);
            WaveSync();
            if (lane == 0) groupKeys[at] = 0;  // stays
            WaveSync();
        }
        for (int c = lane; c < a.experts; c += kWave) {
            if (groupKeys[c / size] != 0) keys[c] = 0;
        }
        WaveSync();
    }

    int32_t pick = 0;  // of lane j: the j-th
    for (int j = 0; j < a.k; ++j) {
        uint64_t best = 0;
        int32_t at = INT32_MAX;
        for (int c = lane; c < a.experts; c += kWave) {
            if (keys[c] > best) {
                best = keys[c];
                at = c;
            }
        }
        WaveArgMax(best, at);
        if (lane == j) pick = at;
        WaveSync();
        if (lane == 0) keys[at] = 0;
        WaveSync();
    }

    double y = lane < a.k ? ScoreOf(Codec::Load(x[pick]), sigmoid, shift, sum) : 0.0;
    if (a.renorm != 0) {
        const double total = WaveSum64(y) + a.eps;
        y = total == 0.0 ? 0.0 : y / total;
    }
    if (lane < a.k) {
        const bool done = a.finished != nullptr && a.finished[row] != 0;
        static_cast<typename Out::Storage*>(a.y)[row * a.k + lane] = Out::Store(static_cast<float>(y * a.factor));
        a.expertIdx[row * a.k + lane] = done ? a.experts : pick;
    }
}

// Any row: one wave each.
template <typename Codec, typename Out>
__global__ __launch_bounds__(kWave) void GatingAnyKernel(GatingArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char ldsRaw[];
    const int64_t row = GroupIndex();
    if (row < a.rows) ExactRow<Codec, Out>(a, row, threadIdx.x, reinterpret_cast<uint64_t*>(ldsRaw), a.scores != nullptr);
}

// Reductions over the kLanes (16 or 64) neighbouring lanes that share a row; every one of them has the result.
template <int kLanes, typename T, typename Op>
__device__ __forceinline__ T RowReduce(T v, Op op) {
    auto ror = [](T t, auto ctl) __attribute__((always_inline)) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, t), decltype(ctl)::value, 0xF, 0xF, true));
    };
    v = op(v, ror(v, std::integral_constant<int, 0x128>{}));  // row_ror:8
    v = op(v, ror(v, std::integral_constant<int, 0x124>{}));
    v = op(v, ror(v, std::integral_constant<int, 0x122>{}));
    v = op(v, ror(v, std::integral_constant<int, 0x121>{}));
    if constexpr (kLanes == 64) {
        auto lane = [&](int l) { return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
        v = op(op(lane(0), lane(16)), op(lane(32), lane(48)));
    }
    return v;
}
template <int kLanes>
__device__ __forceinline__ uint32_t RowMax(uint32_t v) { return RowReduce<kLanes>(v, [](uint32_t p, uint32_t q) { return max(p, q); }); }
template <int kLanes>
__device__ __forceinline__ uint32_t RowMin(uint32_t v) { return RowReduce<kLanes>(v, [](uint32_t p, uint32_t q) { return min(p, q); }); }
template <int kLanes>
__device__ __forceinline__ double RowSum(double v) {
    auto ror = [](double d, auto ctl) __attribute__((always_inline)) {
        const long long u = __double_as_longlong(d);
        const int lo = __builtin_amdgcn_mov_dpp(static_cast<int>(u), decltype(ctl)::value, 0xF, 0xF, true);
        const int hi = __builtin_amdgcn_mov_dpp(static_cast<int>(u >> 32), decltype(ctl)::value, 0xF, 0xF, true);
        return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo)));
    };
    v += ror(v, std::integral_constant<int, 0x128>{});
    v += ror(v, std::integral_constant<int, 0x124>{});
    v += ror(v, std::integral_constant<int, 0x122>{});
    v += ror(v, std::integral_constant<int, 0x121>{});
    if constexpr (kLanes == 64) {
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
    }
    return v;
}

// The lowest lane of the wave that holds the largest key; uniform.  The upper halves settle it nearly always.
__device__ __forceinline__ int WaveHolder(uint64_t key) {
    const uint32_t hi = static_cast<uint32_t>(key >> 32), lo = static_cast<uint32_t>(key);
    const bool top = hi == RowMax<64>(hi);
    uint64_t holders = __ballot(top);
    if ((holders & (holders - 1)) != 0) {
        const uint32_t low = RowMax<64>(top ? lo : 0u);
        holders = __ballot(top && lo == low);
    }
    return __ffsll(static_cast<unsigned long long>(holders)) - 1;
}

__device__ __forceinline__ uint32_t Key32(float f) {
    const uint32_t u = __float_as_uint(f);
    return f != f ? 0xffc00000u : (u & 0x80000000u) != 0 ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float Value32(uint32_t key) { return __uint_as_float((key & 0x80000000u) != 0 ? (key & 0x7fffffffu) : ~key); }

// Key32 of a number that is no NaN.
__device__ __forceinline__ uint32_t NumberKey(float f) {
    const int32_t u = __builtin_bit_cast(int32_t, f);
    return static_cast<uint32_t>(u) ^ (static_cast<uint32_t>(u >> 31) | 0x80000000u);
}

// exp(d) for d <= 0 to an fp32 unit in the last place (0 below e^-110): the product with log2(e) to twice fp32's bits, its tail put back behind the
// instruction.
__device__ __forceinline__ float ExpNotAbove1(float d) {
    d = d < -110.f ? -110.f : d;
    const float h = d * 0x1.715476p+0f;
    const float tail = fmaf(d, 0x1.715476p+0f, -h) + d * 0x1.4ae0cp-26f;
    const float e = __builtin_amdgcn_exp2f(h);
    return fmaf(e, tail * 0x1.62e43p-1f, e);
}

// The kPer values of a lane; absent ones are -inf.
template <typename Codec, int kPer>
__device__ __forceinline__ void LoadLane(const GatingArgs& a, const typename Codec::Storage* x, int l, float (&v)[kPer]) {
    if (a.packets != 0) {
        constexpr int kPiece = kPer * sizeof(typename Codec::Storage) >= 16 ? 16 / sizeof(typename Codec::Storage) : kPer;
        struct alignas(kPiece * sizeof(typename Codec::Storage)) Piece {
            typename Codec::Storage e[kPiece];
        };
        auto read = [&] {
#pragma unroll
            for (int i = 0; i < kPer; i += kPiece) {
                const Piece piece = *reinterpret_cast<const Piece*>(x + l * kPer + i);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) v[i + j] = Codec::Load(piece.e[j]);
            }
        };
        if (a.packets == 2) {
            read();
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[i] = -INFINITY;
            if (l * kPer < a.experts) read();
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = l * kPer + i < a.experts ? Codec::Load(x[l * kPer + i]) : -INFINITY;
    }
}

// y and the index of a row's picks, the j-th of them, whose logit is x, in its lane j.
template <typename Out, int kLanes>
__device__ __forceinline__ void WritePicks(const GatingArgs& a, int64_t row, int l, int32_t pick, float x, double shift, double sum) {
    double y = l < a.k ? ScoreOf(x, a.sigmoid != 0, shift, sum) : 0.0;
    if (a.renorm != 0) {
        const double total = RowSum<kLanes>(y) + a.eps;
        y = total == 0.0 ? 0.0 : y / total;
    }
    if (l < a.k) {
        const bool done = a.finished != nullptr && a.finished[row] != 0;
        static_cast<typename Out::Storage*>(a.y)[row * a.k + l] = Out::Store(static_cast<float>(y * a.factor));
        a.expertIdx[row * a.k + l] = done ? a.experts : pick;
    }
}

// A row of up to 64 * kPer experts, at most 64 groups, by one wave in 64 bits: lane l holds experts l * kPer + i, the keys in registers.  lds: 12 bytes an
// expert, the wave's own, for groups whose experts are not those of whole lanes and for the logits of the picks.  What bounds it is latency: a pick is a
// maximum over four rotations inside a row of sixteen lanes, four lane reads and a ballot (256 experts, 8 picks: 4.7 us, with sigmoid, bias and groups
// 5.8; with the keys in LDS and the arg-max over twelve shuffles 10.9 and 15.8), a value's exponential in 64 bits a chain of fifty instructions
// (301 x 160, softmax, with and without the scores 6.0 and 5.9 us; with a branch for each value 7.3).
template <typename Codec, typename Out, int kPer>
__device__ __forceinline__ void WaveRow(const GatingArgs& a, int64_t row, int lane, uint64_t* lds, bool writeScores) {
    const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x) + row * a.experts;
    const bool sigmoid = a.sigmoid != 0, biased = a.bias != nullptr, grouped = a.kGroup < a.groups;
    float v[kPer];
    LoadLane<Codec, kPer>(a, x, lane, v);
    float* const values = reinterpret_cast<float*>(lds + a.experts);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (lane * kPer + i < a.experts) values[lane * kPer + i] = v[i];
    }
    // p as ScoreOf has it, without branches for each: exponentials in 64 bits are long chains, which run side by side
    double shift = 0.0, sum = 1.0, p[kPer] = {};
    if (sigmoid) {
        if (biased || writeScores) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) p[i] = 1.0 / (1.0 + exp(-static_cast<double>(v[i])));  // 0 of -inf
        }
    } else {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) most = max(most, Key32(v[i]));
        shift = Value32(RowMax<64>(most));
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            p[i] = exp(static_cast<double>(v[i]) - shift);
            p[i] = v[i] == -INFINITY ? 0.0 : p[i];
            sum += p[i];
        }
        sum = RowSum<64>(sum);
        if (biased || writeScores) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) p[i] = v[i] == -INFINITY ? 0.0 : p[i] / sum;
        }
    }
    uint64_t keys[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = lane * kPer + i;
        if (writeScores && c < a.experts) a.scores[row * a.experts + c] = static_cast<float>(p[i]);
        double t = Unsigned0(v[i]);
        if (biased) t = v[i] == -INFINITY ? t : p[i] + static_cast<double>(a.bias[c < a.experts ? c : 0]);
        keys[i] = c < a.experts ? KeyOf(t) : 0;
    }
    if (grouped) {
        // the lanes are shared out among the groups, a power of two each
        const int size = a.experts / a.groups;
        const int share = kWave >> (32 - __builtin_clz(a.groups * 2 - 1) - 1);
        const int group = lane / share;
        uint64_t one = 0, two = 0;
        auto take = [&](uint64_t key) {
            two = key > one ? one : key > two ? key : two;
            one = key > one ? key : one;
        };
        if (share * kPer == size) {  // a group's experts are those of its lanes
#pragma unroll
            for (int i = 0; i < kPer; ++i) take(keys[i]);
        } else {
            WaveSync();
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (lane * kPer + i < a.experts) lds[lane * kPer + i] = keys[i];
            }
            WaveSync();
            if (group < a.groups) {
                for (int c = lane % share; c < size; c += share) take(lds[group * size + c]);
            }
        }
        for (int d = 1; d < share; d <<= 1) {
            const uint64_t otherOne = __shfl_xor(static_cast<unsigned long long>(one), d), otherTwo = __shfl_xor(static_cast<unsigned long long>(two), d);
            const uint64_t less = one > otherOne ? otherOne : one, second = two > otherTwo ? two : otherTwo;
            two = less > second ? less : second;
            one = one > otherOne ? one : otherOne;
        }
        if (a.topTwo != 0 && one != 0) {
            double first = ValueOf(one), second = two == 0 ? -INFINITY : ValueOf(two);
            if (!biased) {
                if (first != -INFINITY) first = ScoreOf(static_cast<float>(first), sigmoid, shift, sum);
                if (second != -INFINITY) second = ScoreOf(static_cast<float>(second), sigmoid, shift, sum);
            }
            one = KeyOf(second == -INFINITY ? first : first + second);
        }
        if (lane % share != 0) one = 0;
        uint64_t kept = 0;
        for (int j = 0; j < a.kGroup; ++j) {
            const int holder = WaveHolder(one);
            kept |= 1ull << (holder / share);
            if (lane == holder) one = 0;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const uint32_t c = lane * kPer + i;
            if ((kept >> ((c * a.groupMagic >> 21) & 63) & 1) == 0) keys[i] = 0;
        }
    }
    int32_t pick = 0;
    for (int j = 0; j < a.k; ++j) {
        uint64_t best = keys[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < kPer; ++i) {
            if (keys[i] > best) {  // equal keys: the lower expert stays
                best = keys[i];
                at = i;
            }
        }
        const int holder = WaveHolder(best);
        const int taken = __builtin_amdgcn_readlane(at, holder);
        if (lane == j) pick = holder * kPer + taken;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (lane == holder && i == taken) keys[i] = 0;
        }
    }
    WaveSync();
    WritePicks<Out, 64>(a, row, lane, pick, values[pick], shift, sum);
}

constexpr int kRowWaves = 4;  // of a workgroup

// LDS of a wave: a row's keys in 64 bits and its logits; or an fp32 value per expert of its four rows, then their picks.
constexpr uint32_t WaveBytes(int experts) { return static_cast<uint32_t>(experts < 16 ? 16 : experts) * 16; }

template <typename Codec, typename Out, int kPer>
__global__ __launch_bounds__(kWave * kRowWaves) void GatingWaveKernel(GatingArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char ldsRaw[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t row = GroupIndex() * kRowWaves + wave;
    if (row < a.rows) WaveRow<Codec, Out, kPer>(a, row, lane, reinterpret_cast<uint64_t*>(ldsRaw + wave * WaveBytes(a.experts)), a.scores != nullptr);
}

// Rows of up to 16 * kPer experts, at most 16 picks and groups: four rows a wave, sixteen lanes each, fp32 keys in registers.  Lane l of a row holds experts
// l * kPer + i, so that among equal values the lower lane has the lower index; within a lane the number i goes into the lowest bits of the key, which
// makes a lane's keys different.  `bound` is the last key that a lane gave away: of the differences key - bound modulo 2^32 the largest is that of the next
// smaller key.
// Errors, u = 2^-24: p is within 8 u top of itself (an exponential and its argument, the sum in 64 bits, a reciprocal), t = p + bias rounds once.
// Values that decide something and lie closer: the row is made again by the whole wave, in 64 bits.
// What bounds it is the number of instructions: 16384 x 256, sigmoid, bias, 4 of 8 groups, 8 picks 15.6 us (16.8 MB of logits are 3.3), of which a row that
// is made twice is 3: 980 vector instructions a wave, near half of them in the nine rounds of picking, and a wave waits for 39 % of its time;
// softmax without bias or groups, bf16 8.4.  Rows without an infinity or a NaN are spared what those need: 16.0 and 9.0 without.  Rows that end
// between two lanes are read in packets too: 384 experts, bf16, sigmoid, bias 18.6 us, an element at a time 36.  A bias of -inf or the lowest value, on
// one expert or on many, leaves the others' places no bits: every row is made again then, 40 to 45 us in place of 15.6 (by 64 lanes alone 27).
template <typename Codec, typename Out, int kPer>
__global__ __launch_bounds__(kWave * kRowWaves) void GatingQuadKernel(GatingArgs a) {
    constexpr int kLanes = 16, kBits = kPer == 1 ? 0 : kPer == 2 ? 1 : kPer == 4 ? 2 : kPer == 8 ? 3 : kPer == 16 ? 4 : 5;
    constexpr int kPlaceBits = 27;
    constexpr uint32_t kLow = (1u << kBits) - 1;
    constexpr float kU = 0x1p-24f;
    extern __shared__ __attribute__((aligned(16))) unsigned char ldsRaw[];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int l = lane % kLanes, first = lane - l;  // place in the row, the row's first lane
    const int64_t rowsFrom = (GroupIndex() * kRowWaves + wave) * 4;
    if (rowsFrom >= a.rows) return;
    const int64_t row = min(rowsFrom + lane / kLanes, a.rows - 1);
    const bool mine = rowsFrom + lane / kLanes < a.rows;
    unsigned char* const own = ldsRaw + wave * WaveBytes(a.experts);
    float* const values = reinterpret_cast<float*>(own) + lane / kLanes * a.experts;  // of the row, while groups are chosen

    const typename Codec::Storage* const x = static_cast<const typename Codec::Storage*>(a.x) + row * a.experts;
    const bool sigmoid = a.sigmoid != 0, biased = a.bias != nullptr, grouped = a.kGroup < a.groups;
    float v[kPer], b[kPer];
    LoadLane<Codec, kPer>(a, x, l, v);
    if (biased) {
        if (a.biasPackets != 0) {
            constexpr int kPiece = kPer < 4 ? kPer : 4;
            struct alignas(kPiece * 4) Piece {
                float e[kPiece];
            };
            const float* const own = a.bias + min(l * kPer, a.experts - kPer);
#pragma unroll
            for (int i = 0; i < kPer; i += kPiece) {
                const Piece piece = *reinterpret_cast<const Piece*>(own + i);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) b[i + j] = piece.e[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) b[i] = a.bias[min(l * kPer + i, a.experts - 1)];
        }
    }
    float all = v[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) all += v[i];
    const bool plain = __all(fabsf(all) < INFINITY || l * kPer >= a.experts);  // no NaN and no infinity in any of the wave's rows
    bool close = false;  // uniform over the row: it is made again, for values too close to be told apart here, or a NaN
    if (!plain) {
        bool nan = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) nan |= v[i] != v[i];
        close = RowMax<kLanes>(nan ? 1u : 0u) != 0;
    }

    float shift = 0.f, top = 1.f;  // top: no p of the row is larger
    double sum = 1.0;
    if (!sigmoid) {
        float most = v[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) most = fmaxf(most, v[i]);
        shift = RowReduce<kLanes>(most, [](float p, float q) { return fmaxf(p, q); });
        if (shift == -INFINITY) shift = 0.f;  // nothing but -inf
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += static_cast<double>(ExpNotAbove1(v[i] - shift));
        sum = RowSum<kLanes>(sum);
        top = 1.f / static_cast<float>(sum);
    }
    float t[kPer];  // what is compared
    if (biased || (grouped && a.topTwo != 0)) {
        if (sigmoid) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) t[i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v[i] * -0x1.715476p+0f));
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) t[i] = __builtin_amdgcn_exp2f((v[i] - shift) * 0x1.715476p+0f) * top;
        }
    }
    if (a.scores != nullptr && mine) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (l * kPer + i < a.experts) a.scores[row * a.experts + l * kPer + i] = static_cast<float>(ScoreOf(v[i], sigmoid, shift, sum));
        }
    }
    float low = 0.f, high = top;  // low <= t <= high
    bool spread = true;           // they have a distance that places can be taken of
    if (biased) {
        float least = b[0], most = b[0];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            least = fminf(least, b[i]);
            most = fmaxf(most, b[i]);
            t[i] += b[i];
        }
        low = RowReduce<kLanes>(least, [](float p, float q) { return fminf(p, q); });
        high = top + RowReduce<kLanes>(most, [](float p, float q) { return fmaxf(p, q); });
        // not where a bias is an infinity, nor where all are equal and so large that no p shows beside them (16 experts of 2^24)
        spread = high - low > 0.f && high - low < INFINITY;
        close |= !spread;
    }
    const float largest = fmaxf(fabsf(low), fabsf(high));
    if (biased || (grouped && a.topTwo != 0)) {
        if (!plain) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) t[i] = v[i] == -INFINITY ? -INFINITY : t[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) t[i] = Unsigned0(v[i]);
    }

    uint32_t kept = ~0u;  // groups, a bit each
    int group = 0;
    bool whole = false;   // a group's experts are those of its lanes
    if (grouped) {
        const int size = a.experts / a.groups;
        const int logShare = 4 - (32 - __builtin_clz(a.groups * 2 - 1) - 1), share = 1 << logShare;  // lanes of a group, a power of two
        group = l >> logShare;
        whole = share * kPer == size;
        uint32_t one = 0, two = 0;
        auto take = [&](float value) {
            const uint32_t key = NumberKey(value);
            two = max(two, min(one, key));
            one = max(one, key);
        };
        if (whole) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) take(t[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (l * kPer + i < a.experts) values[l * kPer + i] = t[i];
            }
            WaveSync();
            if (group < a.groups) {
                for (int c = l & (share - 1); c < size; c += share) take(values[group * size + c]);
            }
            WaveSync();
        }
        for (int d = 1; d < share; d <<= 1) {
            const uint32_t otherOne = __shfl_xor(one, d), otherTwo = __shfl_xor(two, d);
            two = max(min(one, otherOne), max(two, otherTwo));
            one = max(one, otherOne);
        }
        uint32_t value = 0;
        if ((l & (share - 1)) == 0 && group < a.groups) {
            value = a.topTwo != 0 && two != 0 && Value32(two) != -INFINITY ? NumberKey(Value32(one) + Value32(two)) : one;
        }
        kept = 0;
        uint32_t last = 0;
        for (int j = 0; j < a.kGroup; ++j) {
            last = RowMax<kLanes>(value);
            const uint32_t at = RowMin<kLanes>(value == last ? l : kLanes - 1);
            kept |= 1u << (at >> logShare);
            if (l == static_cast<int>(at)) value = 0;
        }
        const uint32_t next = RowMax<kLanes>(value);
        if (biased || a.topTwo != 0) close |= !(Value32(last) - Value32(next) > kU * (32.f * top + 16.f * largest));
        if (!biased && a.topTwo != 0) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) t[i] = Unsigned0(v[i]);
        }
    }

    // Without a bias a key is the logit's, cut: exact for 16 bits, and fp32 ones that agree in what is left are too close.  With one it is t's place
    // between low and high in 2^27ths, from 32 on, and 1 for -inf.
    uint32_t keys[kPer];
    uint32_t tooClose;  // a difference of two keys
    if (biased) {
        const float scale = spread ? 0x0.ffffp27f / (high - low) : 0.f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) t[i] = fmaf(t[i] - low, scale, 32.f);
        if (!plain || !spread) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) t[i] = __builtin_amdgcn_fmed3f(t[i], 1.f, 0x0.fffffp27f);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) keys[i] = static_cast<uint32_t>(t[i]) << (32 - kPlaceBits) | (kLow - i);
        // the difference to low, the product and the whole number round once each: 8, 8 and 1 units at most
        const float units = (16.f * top + 2.f * largest) * kU * scale * 1.01f + 36.f;
        tooClose = units < 0x1p26f ? static_cast<uint32_t>(units) << (32 - kPlaceBits) : ~0u;
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) keys[i] = (NumberKey(t[i]) & ~kLow) | (kLow - i);
        tooClose = 0;
    }
    const bool exact = !biased && (sizeof(typename Codec::Storage) == 2 || kBits == 0);
    // what is not looked at: experts that are not there, or in a group that was left out (no branches for each: a third of the kernel's time)
    if (grouped || a.experts != kLanes * kPer) {
        auto mask = [&](uint32_t c) {
            const uint32_t stays = grouped ? kept >> ((c * a.groupMagic >> 21) & 31) & 1 : 1u;
            return 0u - (c < static_cast<uint32_t>(a.experts) ? stays : 0u);
        };
        if ((grouped ? a.experts / a.groups : a.experts) % kPer == 0) {
            const uint32_t stays = mask(l * kPer);
#pragma unroll
            for (int i = 0; i < kPer; ++i) keys[i] &= stays;
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) keys[i] &= mask(l * kPer + i);
        }
    }
    const uint32_t upper = biased ? ~31u : ~kLow, lowest = biased ? 2u << (32 - kPlaceBits) : 0x00800000u;  // below: -inf, or none left
    int32_t* const picks = reinterpret_cast<int32_t*>(own) + lane / kLanes * kLanes;
    uint32_t before = ~0u, bound = 0;
    for (int j = 0; j <= a.k; ++j) {
        uint32_t best = 0u - bound;  // none left
#pragma unroll
        for (int i = 0; i < kPer; ++i) best = max(best, keys[i] - bound);
        best += bound;
        const uint32_t most = RowMax<kLanes>(best & upper);
        close |= !exact && j > 0 && most >= lowest && before - most <= tooClose;
        before = most;
        if (j == a.k) break;
        const uint64_t holders = __ballot((best & upper) == most) >> first;  // from the row's first lane on
        if (l == __builtin_ctz(static_cast<uint32_t>(holders))) {
            picks[j] = l * kPer + static_cast<int32_t>(kLow - (best & kLow));
            bound = best;
        }
    }
    WaveSync();
    const int32_t pick = l < a.k ? picks[l] : 0;
    WaveSync();
    if (!close && mine) WritePicks<Out, kLanes>(a, row, l, pick, Codec::Load(x[pick]), shift, sum);
    for (uint64_t again = __ballot(close && mine && l == 0); again != 0; again &= again - 1) {
        const int64_t which = rowsFrom + (__ffsll(static_cast<unsigned long long>(again)) - 1) / kLanes;
        GatingArgs whole = a;
        whole.packets = 0;
        WaveRow<Codec, Out, (kPer + 3) / 4>(whole, which, lane, reinterpret_cast<uint64_t*>(own), false);
    }
}

class GatingExecutor : public aclOpExecutor {
   public:
    GatingArgs args{};
    aclDataType dtype = ACL_FLOAT;
    aclDataType outType = ACL_FLOAT;

    // The arguments of a kernel whose rows are lanes of kPer experts.
    template <typename Codec>
    GatingArgs ForLanes(int lanes, int per) const {
        GatingArgs g = args;
        const size_t bytes = per * sizeof(typename Codec::Storage), piece = bytes < 16 ? bytes : 16;
        g.packets = g.experts % per == 0 && reinterpret_cast<uintptr_t>(g.x) % piece == 0 ? (g.experts == lanes * per ? 2 : 1) : 0;
        g.biasPackets = g.experts % per == 0 && reinterpret_cast<uintptr_t>(g.bias) % 16 == 0 ? 1 : 0;
        return g;
    }

    template <typename Codec, typename Out, int kPer>
    void LaunchWaves(hipStream_t stream) const {
        hipLaunchKernelGGL((GatingWaveKernel<Codec, Out, kPer>), GridOf((args.rows + kRowWaves - 1) / kRowWaves), dim3(kWave * kRowWaves),
                           kRowWaves * WaveBytes(args.experts), stream, ForLanes<Codec>(kWave, kPer));
    }

    template <typename Codec, typename Out, int kPer>
    void LaunchQuads(hipStream_t stream) const {
        hipLaunchKernelGGL((GatingQuadKernel<Codec, Out, kPer>), GridOf((args.rows + 4 * kRowWaves - 1) / (4 * kRowWaves)), dim3(kWave * kRowWaves),
                           kRowWaves * WaveBytes(args.experts), stream, ForLanes<Codec>(16, kPer));
    }

    template <typename Codec, typename Out>
    void Launch(hipStream_t stream) const {
        const int E = args.experts;
        // Sixteen lanes a row make more rows at a time and take longer for one, most of all with a bias, where one row in a thousand is
        // made twice.  us by sixteen and by 64 lanes: 256 experts, sigmoid, bias, 4 of 8 groups 9.6 and 6.6 at 1024 rows, 9.7 and 9.9 at 4096, 15.0 and
        // 27.0 at 16384; softmax without a bias 4.9 and 5.3, 5.0 and 7.9, 8.3 and 20.6.
        const bool many = args.rows > (args.bias != nullptr ? 4000 : 1024);
        if (many && E <= 512 && args.k <= 16 && args.groups <= 16) {
            if (E <= 16) LaunchQuads<Codec, Out, 1>(stream);
            else if (E <= 32) LaunchQuads<Codec, Out, 2>(stream);
            else if (E <= 64) LaunchQuads<Codec, Out, 4>(stream);
            else if (E <= 128) LaunchQuads<Codec, Out, 8>(stream);
            else if (E <= 256) LaunchQuads<Codec, Out, 16>(stream);
            else LaunchQuads<Codec, Out, 32>(stream);
        } else if (E <= 512 && args.groups <= kWave) {
            if (E <= 64) LaunchWaves<Codec, Out, 1>(stream);
            else if (E <= 128) LaunchWaves<Codec, Out, 2>(stream);
            else if (E <= 256) LaunchWaves<Codec, Out, 4>(stream);
            else LaunchWaves<Codec, Out, 8>(stream);
        } else {
            const size_t lds = (static_cast<size_t>(E) + args.groups) * 8;
            hipLaunchKernelGGL((GatingAnyKernel<Codec, Out>), GridOf(args.rows), dim3(kWave), lds, stream, args);
        }
    }

    template <typename Codec>
    void LaunchFor(hipStream_t stream) const {
        if (outType == Codec::kType) Launch<Codec, Codec>(stream);
        else Launch<Codec, F32>(stream);
    }

    aclnnStatus Run(void*, hipStream_t stream) override {
        if (args.rows == 0) return ACLNN_SUCCESS;
        opapi::KernelTimer timer("gating_topk_grouped", stream);
        if (dtype == ACL_FLOAT) Launch<F32, F32>(stream);
        else if (dtype == ACL_FLOAT16) LaunchFor<F16>(stream);
        else LaunchFor<Bf16>(stream);
        const hipError_t err = hipGetLastError();
        if (err != hipSuccess) {
            opapi::SetError("aclnnMoeGatingTopKGrouped: launch failed: %s", hipGetErrorString(err));
            return ACLNN_ERR_RUNTIME_ERROR;
        }
        return ACLNN_SUCCESS;
    }
};

}  // namespace

extern "C" aclnnStatus aclnnMoeGatingTopKGroupedGetWorkspaceSize(
    const aclTensor* x, const aclTensor* biasOptional, const aclTensor* finishedOptional, int64_t k, int64_t kGroup,
    int64_t groupCount, int64_t groupSelectMode, int64_t scoreType, int64_t renorm, double routedScalingFactor, double eps,
    const aclTensor* yOut, const aclTensor* expertIdxOut, const aclTensor* scoresOutOptional, uint64_t* workspaceSize,
    aclOpExecutor** executor) try {
    using namespace opapi;
    ClearError();
    OPAPI_CHECK_NOTNULL(x, "x");
    OPAPI_CHECK_NOTNULL(yOut, "yOut");
    OPAPI_CHECK_NOTNULL(expertIdxOut, "expertIdxOut");
    OPAPI_CHECK_NOTNULL(workspaceSize, "workspaceSize");
    OPAPI_CHECK_NOTNULL(executor, "executor");
    OPAPI_CHECK_EXTENTS(x, biasOptional, finishedOptional, yOut, expertIdxOut, scoresOutOptional);

    constexpr aclnnStatus kInvalid = ACLNN_ERR_PARAM_INVALID;
    OPAPI_CHECK(IsFloating(x), kInvalid, "x must be FLOAT, FLOAT16 or BF16");
    OPAPI_CHECK(x->dims.size() == 2 || x->dims.size() == 3, kInvalid, "x must have rank 2 or 3, not %zu", x->dims.size());
    for (int64_t d : x->dims) OPAPI_CHECK(d <= 2147483647ll, kInvalid, "an extent of x is larger than 2147483647");
    const int64_t experts = x->dims.back();
    OPAPI_CHECK(experts > 0 && experts <= kMaxExperts, kInvalid, "the last extent of x (=%lld) must be 1 to %lld experts", (long long)experts,
                (long long)kMaxExperts);
    const int64_t rows = RowsOf(x);
    OPAPI_CHECK(rows >= 0, kInvalid, "x has more than %lld rows", (long long)kMaxRows);
    OPAPI_CHECK(groupCount >= 1 && groupCount <= experts && experts % groupCount == 0, kInvalid,
                "groupCount (=%lld) must divide the %lld experts", (long long)groupCount, (long long)experts);
    OPAPI_CHECK(kGroup >= 1 && kGroup <= groupCount, kInvalid, "kGroup (=%lld) must be 1 to groupCount (=%lld)", (long long)kGroup,
                (long long)groupCount);
    OPAPI_CHECK(groupSelectMode == 0 || groupSelectMode == 1, kInvalid, "groupSelectMode (=%lld) must be 0 or 1", (long long)groupSelectMode);
    OPAPI_CHECK(groupSelectMode == 0 || kGroup == groupCount || experts / groupCount >= 2, kInvalid,
                "groupSelectMode 1 adds two experts of a group, which has one");
    OPAPI_CHECK(scoreType == 0 || scoreType == 1, kInvalid, "scoreType (=%lld) must be 0 or 1", (long long)scoreType);
    OPAPI_CHECK(renorm == 0 || renorm == 1, kInvalid, "renorm (=%lld) must be 0 or 1", (long long)renorm);
    OPAPI_CHECK(k >= 1 && k <= kMaxPicks && k <= experts / groupCount * kGroup, kInvalid,
                "k (=%lld) must be 1 to %lld and at most the %lld experts of the groups that stay", (long long)k, (long long)kMaxPicks,
                (long long)(experts / groupCount * kGroup));
    OPAPI_CHECK(std::isfinite(routedScalingFactor), kInvalid, "routedScalingFactor must be a number");
    OPAPI_CHECK(eps >= 0 && std::isfinite(eps), kInvalid, "eps must be a number of at least 0");
    OPAPI_CHECK(biasOptional == nullptr || (biasOptional->dtype == ACL_FLOAT && biasOptional->dims.size() == 1 && biasOptional->dims[0] == experts),
                kInvalid, "bias must be FLOAT [%lld]", (long long)experts);
    OPAPI_CHECK(finishedOptional == nullptr || (finishedOptional->dtype == ACL_BOOL && SameButLast(finishedOptional, x, -1)), kInvalid,
                "finished must be BOOL of x's extents without the last");
    OPAPI_CHECK((yOut->dtype == x->dtype || yOut->dtype == ACL_FLOAT) && SameButLast(yOut, x, k), kInvalid,
                "yOut %s must be of x's type or FLOAT, x's extents %s with the last replaced by k", ShapeStr(yOut).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(expertIdxOut->dtype == ACL_INT32 && SameButLast(expertIdxOut, x, k), kInvalid,
                "expertIdxOut %s must be INT32, x's extents %s with the last replaced by k", ShapeStr(expertIdxOut).c_str(), ShapeStr(x).c_str());
    OPAPI_CHECK(scoresOutOptional == nullptr || (scoresOutOptional->dtype == ACL_FLOAT && SameButLast(scoresOutOptional, x, experts)), kInvalid,
                "scoresOut %s must be FLOAT of x's extents %s", ShapeStr(scoresOutOptional).c_str(), ShapeStr(x).c_str());
    const aclTensor* const ins[] = {x, biasOptional, finishedOptional};
    const aclTensor* const outs[] = {yOut, expertIdxOut, scoresOutOptional};
    for (int o = 0; o < 3; ++o) {
        if (outs[o] == nullptr) continue;
        OPAPI_CHECK(InOrder(outs[o]), kInvalid, "the outputs must be contiguous");
        OPAPI_CHECK(rows == 0 || outs[o]->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an output carries no device memory");
        for (int p = 0; p < o; ++p) OPAPI_CHECK(!Overlap(outs[o], outs[p]), kInvalid, "two outputs share memory");
    }
    for (const aclTensor* in : ins) {
        if (in == nullptr) continue;
        OPAPI_CHECK(rows == 0 || in->data != nullptr, ACLNN_ERR_PARAM_NULLPTR, "an input carries no device memory");
        for (const aclTensor* out : outs) {
            OPAPI_CHECK(!IsContiguous(in) || !Overlap(out, in), kInvalid, "an output shares memory with an input");
        }
    }

    auto* ex = new (std::nothrow) GatingExecutor();
    OPAPI_CHECK(ex != nullptr, ACLNN_ERR_INNER_CREATE_EXECUTOR, "out of host memory");
    ex->dtype = x->dtype;
    ex->outType = yOut->dtype;
    OPAPI_BIND(ex, x, &ex->args.x);
    OPAPI_BIND(ex, biasOptional, &ex->args.bias);
    OPAPI_BIND(ex, finishedOptional, &ex->args.finished);
    ex->args.y = DataPtr(yOut);
    ex->args.expertIdx = reinterpret_cast<int32_t*>(DataPtr(expertIdxOut));
    ex->args.scores = reinterpret_cast<float*>(DataPtr(scoresOutOptional));
    ex->args.rows = rows;
    ex->args.experts = static_cast<int32_t>(experts);
    ex->args.k = static_cast<int32_t>(k);
    ex->args.groups = static_cast<int32_t>(groupCount);
    ex->args.kGroup = static_cast<int32_t>(kGroup);
    ex->args.topTwo = static_cast<int32_t>(groupSelectMode);
    ex->args.sigmoid = static_cast<int32_t>(scoreType);
    ex->args.renorm = static_cast<int32_t>(renorm);
    ex->args.factor = routedScalingFactor;
    ex->args.eps = eps;
    const int64_t size = experts / groupCount;
    ex->args.groupMagic = static_cast<uint32_t>(((1ll << 21) + size - 1) / size);
    ex->SealWorkspace(0);
    *workspaceSize = ex->workspaceBytes;
    *executor = ex;
    return ACLNN_SUCCESS;
} catch (...) {  // no exception may cross the C boundary
    opapi::SetError("out of host memory");
    return ACLNN_ERR_INNER;
}

extern "C" aclnnStatus aclnnMoeGatingTopKGrouped(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                 aclrtStream stream) {
    return opapi::RunAndRelease(workspace, workspaceSize, executor, stream);
}
