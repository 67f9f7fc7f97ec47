// Token sampling: one token for each row of logits x[0..V), by a given random
// number u in [0, 1).  With w_i = exp((x_i - max x) / T):
//
//   A = tokens with w_i >= min_p                    (min-p)
//   K = the first top_k of A by (x descending, index ascending)
//   P = the smallest prefix of K in that order with mass >= top_p * mass(K)
//   token = the first i, in index order, with  sum_{j <= i, j in P} w_j > u * mass(P)
//
// T = 0 takes the largest logit (lowest index).  The log probability is the
// model's own: x_token - max x - log sum_i exp(x_i - max x), over all tokens,
// in 64 bits up to its one rounding (exponentials, counted_partition).
//
// Exactness.  The nucleus and the draw compare sums of up to 2^19 weights with
// the border between two tokens, where fp32 sums would choose another token
// than the definition once in a few thousand draws.  Weights are therefore
// 64-bit fixed point, w * 2^s with s = min(51, 62 - ceil(log2 V)): each is
// computed in double precision (relative error below 2e-13) and rounded once;
// sums of integers are exact and do not depend on their order, so the same
// inputs give the same token whatever the launch shape.  What the rounding costs:
// a sum is off by half a unit a token at most, by 2^-27 of the largest weight in all
// for 2^18 tokens (some 2^-36 where the roundings are of either sign), which is how
// often a random number can find another token than the definition's.  Tokens
// lighter than 2^-(s+1) weigh nothing, so random numbers between 0 and 2^-24, which
// fp32 generators do not give, pass them over; for 0 itself tokens are counted down
// to double precision's smallest weight.  The exponential is
// table driven (Tang, 1989): 2^-n/256 from a table of 256 values times a Taylor
// polynomial of degree 3 in the remainder (at most ln 2 / 512, so 2e-13 off).
// Double-precision steps are what bounds it: tables of 64 and 16 values meet
// fewer bank conflicts, but need degrees 4 and 5, and take 45.7 and 46.7 us
// where this one takes 44.6 (64 uncut fp32 rows of 248320).
//
// Layout of the work.  A cluster of 1 to 16 CTAs takes one row, a CTA one
// contiguous share.  The row is read from HBM once: a small share then stays
// in shared memory, later passes over a large one find it in L2.  While the
// logits come in, a CTA counts them by their leading 16 bits (a bf16's own
// value); the merged counts say where a cut lies.  From there:
//   - where at most kList tokens can be kept, they are pushed to the first CTA,
//     which ranks them and draws;
//   - a bf16 row is known but for its order: masses are counts times weights,
//     a cut is a value and a number of equal logits, and only the slab that
//     holds the drawn token is weighed (of a large share first the quarter,
//     by counts that are kept apart for each);
//   - for fp16 and fp32 the counts bound the masses, and the tokens of the bins
//     that can hold the border are weighed one by one;
//   - uncut fp16 and fp32 rows are weighed slab by slab, and drawn from;
//   - rows that the counts do not hold (many tiny values, a largest logit
//     outside +-128) search a cut by bins of value.
//
// What bounds it.  Not HBM (64 uncut fp32 rows of 248320 take 44.9 us, 1.42
// TB/s): the small cases wait for some ten steps between the CTAs of a row (17.6
// us for one row; the merge of the counts 4.2 of them, an exchange 0.8 to 2.3),
// the large ones for the shared-memory counts, a weight's double-precision
// arithmetic and instruction issue: 2.6 instructions a clock over the whole kernel
// for 256 bf16 rows, and 10.3 clocks for a warp's 32 weights where two CTAs share
// an SM (13.6 for one alone).  256 bf16 rows with a nucleus of many thousand
// tokens take 110 us (1.16 TB/s) against 729 with a weight for every logit.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <cfloat>
#include <climits>

#include "../../include/ornith_moe_b200.h"
#include "abi_check.h"
#include "nvtx_range.h"

namespace ornith {
void count_launches(int n);

namespace sample {
namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxCluster = 16, kMaxVocab = 1 << 19, kSms = 148;
// Bins of a search, candidates that it ranks; tokens of a list: 19 us against 24 with 256 for 7 rows of 4099.
constexpr int kBins = 1024, kCap = 256, kList = 2 * kThreads;
// Vectors of a thread in flight: 111 us for 256 rows of 248320 with four, 113 with two.
constexpr int kAhead = 4;
// Parts of a bf16 CTA's logits that do not stay on chip, counted apart in 16 bits (kPartVecs * 8 < 2^16), so that the
// drawn token is sought in one of them: 111 us against 206 for 256 rows of 248320, 44 against 56 for 64.
constexpr int kParts = 4, kPartVecs = 255 * 32, kMaxVecs = kParts * kPartVecs;
// 16-byte vectors that one CTA or two of an SM keep on chip.  Where both fit, 19.4 us against 20.3 from L2 for 7 rows
// of 4099; 8192 for two, which leaves one CTA on an SM: 67 us against 44 for 64 rows.
constexpr int kAloneVecs = 1 << 13, kSharedVecs = 3 << 10;
constexpr int kStep = 8, kSlabs = kMaxVecs / 32 / kStep + kWarps;  // rows of 32 vectors in a slab; slabs of a CTA
constexpr float kMaxTemperature = 1e30f;
constexpr uint32_t kFlagNonfinite = 1, kFlagParameter = 2, kFlagNothingLeft = 4, kFlagBounds = 128;

struct Args {
    const void* logits;
    int64_t stride;  // values between rows
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t* tokens;
    float* logprobs;
    uint32_t* flags;
    int vocab, vecs;  // vecs: 16-byte vectors of a row for one CTA
    int resident;     // they stay in shared memory
    int part_vecs;    // bf16: vectors (a multiple of 32) of a part that is counted apart, or 0
};

template <int TY>
struct Elem;  // values of one 16-byte vector, as fp32 (exact)
template <>
struct Elem<0> {
    static constexpr int E = 8, kBytes = 2;
    static __device__ __forceinline__ float one(const void* p) { return __bfloat162float(*static_cast<const __nv_bfloat16*>(p)); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[E]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    // the largest value of a vector (of those that are not NaN)
    static __device__ __forceinline__ float largest(const uint4& v) {
        uint32_t a, b;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
        asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
        asm("max.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
        return fmaxf(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
    }
    static constexpr uint32_t kNone = 0xff80ff80u;  // a vector's word of two -inf
    static constexpr float kLowest = -3.3895313892515355e38f;
};
template <>
struct Elem<1> {
    static constexpr int E = 8, kBytes = 2;
    static __device__ __forceinline__ float one(const void* p) { return __half2float(*static_cast<const __half*>(p)); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[E]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __half2float(__ushort_as_half(uint16_t(w[i] & 0xffffu)));
            x[2 * i + 1] = __half2float(__ushort_as_half(uint16_t(w[i] >> 16)));
        }
    }
    static __device__ __forceinline__ float largest(const uint4& v) {
        uint32_t a, b;
        asm("max.f16x2 %0, %1, %2;" : "=r"(a) : "r"(v.x), "r"(v.y));
        asm("max.f16x2 %0, %1, %2;" : "=r"(b) : "r"(v.z), "r"(v.w));
        asm("max.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
        return fmaxf(__half2float(__ushort_as_half(uint16_t(a & 0xffffu))),
                     __half2float(__ushort_as_half(uint16_t(a >> 16))));
    }
    static constexpr uint32_t kNone = 0xfc00fc00u;
    static constexpr float kLowest = -65504.f;
};
template <>
struct Elem<2> {
    static constexpr int E = 4, kBytes = 4;
    static __device__ __forceinline__ float one(const void* p) { return *static_cast<const float*>(p); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[E]) {
        x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float largest(const uint4& v) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                     fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static constexpr uint32_t kNone = 0xff800000u;
    static constexpr float kLowest = -FLT_MAX;
};

struct Pair {
    u64 a, b;
};

// The search of a cut among the values of a range (cut_row).
struct Search {
    u64 mass[kBins], tmass[kBins];       // this CTA's histogram, the row's
    uint32_t cnt[kBins], tcnt[kBins];
    u64 gw[kCap];
    float lv[kCap], gv[kCap];            // candidates of this CTA, of the row
    int li[kCap], gi[kCap];
    uint32_t ln;
};

// Counts of the logits' leading 16 bits: 4352 codes of magnitude 2^-10 to 128,
// and all below 2^-10 as one.
constexpr int kOctaves = 17, kCodes = kOctaves * 128;
constexpr uint32_t kFirstCode = (134 - kOctaves) << 7;         // of 2^-10
// Bins by value, largest first: the tiny between, the negative from a multiple of 4 on (three bins stay empty).
constexpr int kTinyBin = kCodes, kNegative = kCodes + 4, kValueBins = kNegative + kCodes;
constexpr int kPerThread = (kValueBins + kThreads - 1) / kThreads, kTinyCap = 256;
// The tokens that can be kept, where they are few: pushed to the first CTA.
struct List {
    u64 weight[kList];                             // by rank
    float v[kList];
    int i[kList];
};
struct Values {
    union {
        alignas(16) uint32_t own[2 * kCodes + 4];  // by code: positive, negative, tiny
        List list;                                 // once the counts are merged
    };
    alignas(16) uint32_t all[kPerThread * kThreads];  // the row's, by value
    float tiny[kTinyCap];                          // this CTA's tiny logits (bf16 rows)
    uint8_t tiny_part[kTinyCap];                   // and where they lie
    u64 tiny_mass[kMaxCluster];                    // pushed
    u64 tiny_sum[kMaxCluster];                     // pushed: of exp(x), times 2^50
};

// A bin's largest and smallest value; the same for bf16 but in the tiny one.
__device__ __forceinline__ int code_of(int bin) {
    return bin < kTinyBin ? kCodes - 1 - bin : bin < kNegative ? 2 * kCodes : bin - kNegative + kCodes;
}
__device__ __forceinline__ uint32_t magnitude_of(int bin) {
    return (uint32_t(bin < kTinyBin ? kCodes - 1 - bin : bin - kNegative) + kFirstCode) << 16;
}
__device__ __forceinline__ float near_edge(int bin) {  // the edge next to zero
    if (bin >= kTinyBin && bin < kNegative) return 0.f;
    return __uint_as_float(magnitude_of(bin) | (bin < kTinyBin ? 0u : 0x80000000u));
}
__device__ __forceinline__ float far_edge(int bin) {
    return __uint_as_float(__float_as_uint(near_edge(bin)) | 0xffffu);
}
__device__ __forceinline__ float bin_top(int bin) {
    if (bin >= kTinyBin && bin < kNegative) return __uint_as_float((kFirstCode << 16) - 1);
    return bin < kTinyBin ? far_edge(bin) : near_edge(bin);
}
__device__ __forceinline__ float bin_bottom(int bin) {
    if (bin >= kTinyBin && bin < kNegative) return -__uint_as_float((kFirstCode << 16) - 1);
    return bin < kTinyBin ? near_edge(bin) : far_edge(bin);
}

struct alignas(16) Shared {
    union {
        Search search;
        Values values;
    };
    float ordered_v[kList];              // the list by bin
    int ordered_i[kList];
    uint32_t listed;
    double pow256[256];                  // 2^(s - j/256)
    Pair slot[2][kMaxCluster];           // pushed by every CTA of the cluster in turn
    u64 slab[kSlabs];                    // kept mass of each slab, in index order
    Pair red[kWarps];
    Pair part[kMaxCluster];              // fp16, fp32: every CTA's largest logit, sum of exponentials against it
    u64 bound[2];
    uint32_t part_here[kParts], part_kept[kParts];  // the border's value in the parts of the token's CTA
    int found, found_bin;
};

// The dynamic shared memory of a CTA: this, then the vectors that stay on chip.
extern __shared__ uint4 dynamic[];
__device__ __forceinline__ Shared& shared() { return *reinterpret_cast<Shared*>(dynamic); }
__device__ __forceinline__ uint4* vectors() { return dynamic + sizeof(Shared) / 16; }
// In their place where they do not: for fp16 and fp32, what the pass over a nucleus's masses leaves for the steps after
// it - the tokens of the bins that can hold the border, and the mass of each slab above them.  64 flat rows of 248320,
// top-p 0.9: 102 us in fp16 and 107 in fp32, against 158 and 182 with three passes more over the logits.
constexpr int kRegion = 5120;
struct Region {
    u64 slab[kSlabs];
    float v[kRegion];
    int slot[kRegion];
    uint32_t n;  // above kRegion: not all are here
};
__device__ __forceinline__ Region& region() { return *reinterpret_cast<Region*>(vectors()); }
// For bf16, counts of part 2i + j in half j of parts()[i * 2 * kCodes + code].
__device__ __forceinline__ uint32_t* parts() { return reinterpret_cast<uint32_t*>(vectors()); }
__device__ __forceinline__ uint32_t part_count(int code, int part) {
    return (parts()[(part >> 1) * 2 * kCodes + code] >> (16 * (part & 1))) & 0xffffu;
}

__device__ __forceinline__ float as_float(u64 v) { return __uint_as_float(uint32_t(v)); }
__device__ __forceinline__ u64 as_bits(float v) { return __float_as_uint(v); }

// The values of a 16-byte vector of which only a part lies in the row.
template <int TY>
__device__ __noinline__ uint4 edge_vector(const char* begin, int i0, int vocab) {
    constexpr int E = Elem<TY>::E, kBytes = Elem<TY>::kBytes;
    uint32_t w[4] = {Elem<TY>::kNone, Elem<TY>::kNone, Elem<TY>::kNone, Elem<TY>::kNone};
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (i0 + e >= 0 && i0 + e < vocab) {
            if (kBytes == 2) {
                const uint32_t h = reinterpret_cast<const uint16_t*>(begin)[i0 + e];
                w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | h << 16 : (w[e / 2] & 0xffff0000u) | h;
            } else {
                w[e & 3] = reinterpret_cast<const uint32_t*>(begin)[i0 + e];
            }
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 2^s exp(-d / T) for d >= 0, with step = 256 log2(e) / T; no more than 600 T.
__device__ __forceinline__ double scaled_exp(double d, double step) {
    constexpr double a = 0.69314718055994530942 / 256, kRound = 0x1.8p52;
    const double shifted = __fma_rn(d, step, kRound);  // n = rint(256 d log2(e) / T) in its low bits
    const int n = __double2loint(shifted);
    const double f = __fma_rn(d, step, -__dsub_rn(shifted, kRound));
    double p = __fma_rn(f, -a * a * a / 6, a * a / 2);
    p = __fma_rn(p, f, -a);
    p = __fma_rn(p, f, 1.0);
    const double v = __dmul_rn(shared().pow256[n & 255], p);
    return __hiloint2double(__double2hiint(v) + (n & ~255) * -4096, __double2loint(v));  // times 2^-(n / 256)
}
constexpr double kStep1 = 256 * 1.4426950408889634074;  // at T = 1
// 2^-s
__device__ __forceinline__ double unit() { return __hiloint2double((2046 << 20) - __double2hiint(shared().pow256[0]), 0); }

// What every thread of a row's cluster knows.
template <int TY>
struct Row {
    using El = Elem<TY>;
    static constexpr int E = El::E;
    bool resident;        // this CTA's vectors are in shared memory
    int head, tail;       // vectors of which only a part lies in the row, or -1
    const uint4* source;  // where they lie in the tensor
    const char* begin;    // the row's first logit
    int vocab, nvec, first;  // first: index of slot 0 (below 0 where the row starts inside a vector)
    int rank, size, parity;
    float top;            // the largest logit
    double step;          // 256 log2(e) / T
    bool count_mode;      // u = 0: any token of positive weight counts as one
    float weigh_from;     // no logit below this has a weight
    float edge, tie_v;    // kept: x >= edge, or x == tie_v and index <= tie_i
    int tie_i;

    __device__ __forceinline__ uint4 vec(int v) const {
        if (resident) return vectors()[v];
        return v != head && v != tail ? __ldcg(source + v) : edge_vector<TY>(begin, first + v * E, vocab);
    }
    __device__ __forceinline__ bool kept(float x, int slot) const {
        return x >= edge || (x == tie_v && first + slot <= tie_i);
    }
    // From here on only vectors [from, from + count).
    __device__ void narrow(int from, int count) {
        source += from, first += from * E, nvec = count;
        head = from == 0 ? head : -1, tail = tail >= from && tail < from + count ? tail - from : -1;
    }
    __device__ void keep_from(float v) { edge = fmaxf(v, -FLT_MAX), tie_v = 0.f, tie_i = -1; }
    __device__ void cut_at(float v, int index) { edge = nextafterf(v, INFINITY), tie_v = v, tie_i = index; }

    template <class F>
    __device__ __forceinline__ void each(F f) const {
        each_vector([&](int v, const uint4& q) {
            float x[E];
            El::unpack(q, x);
#pragma unroll
            for (int e = 0; e < E; ++e) f(x[e], v * E + e);
        });
    }
    template <class F>
    __device__ __forceinline__ void each_vector(F f) const {
#pragma unroll 1
        for (int b = threadIdx.x; b < nvec; b += kAhead * kThreads) {
            uint4 q[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (b + j * kThreads < nvec) q[j] = vec(b + j * kThreads);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int v = b + j * kThreads;
                if (v >= nvec) break;
                f(v, q[j]);
            }
        }
    }

    // By mass, or (count) by number of tokens that have a weight in double precision: down to half its smallest
    // number, 2^-1075.
    __device__ void weigh(bool count, int frac, float T) {
        count_mode = count;
        const double reach = 0.69314718055994530942 * (count ? 1075 : frac + 1);
        weigh_from = fmaxf(-FLT_MAX, __double2float_ru(double(top) - reach * double(T)));
    }

    // 2^52 + the fixed-point weight, as the bits of a double; 2^52 where not `in`.
    __device__ __forceinline__ u64 raw_weight(float x, bool in) const {
        const double v = scaled_exp(__dsub_rn(double(top), double(x)), step);
        const int high = in ? __double2hiint(v) : 0;
        return u64(__double_as_longlong(__dadd_rn(__hiloint2double(high, __double2loint(v)), 0x1p52)));
    }
    static constexpr u64 kRawZero = 0x4330000000000000ull;
    __device__ __forceinline__ u64 weight(float x) const {
        if (count_mode) return x >= weigh_from;
        return raw_weight(x, x >= weigh_from) - kRawZero;
    }
    // Weights and their sum, without branches between them: a chain of double-precision steps is long, and its
    // latency is hidden only by others beside it.
    template <int N>
    __device__ __forceinline__ void weights(const float (&x)[N], u64 (&w)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = raw_weight(x[i], x[i] >= weigh_from) - kRawZero;
        if (count_mode) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = x[i] >= weigh_from;
        }
    }
    // Adds the kept mass of vector v, whose values are in q, to `sum`, and that at low or high and above to two parts.
    // TIES: equal logits lie on both sides of the cut.  No value below `from` is kept.
    template <bool TIES, bool PARTS>
    __device__ __forceinline__ void add_kept(int v, const uint4& q, float from, u64& sum, float low, float high, Pair& parts) const {
        if (El::largest(q) < from) return;
        float x[E];
        El::unpack(q, x);
        bool in[E];
#pragma unroll
        for (int e = 0; e < E; ++e) in[e] = TIES ? kept(x[e], v * E + e) && x[e] >= weigh_from : x[e] >= from;
        if (count_mode) {
#pragma unroll
            for (int e = 0; e < E; ++e) sum += in[e];
            return;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const u64 raw = raw_weight(x[e], in[e]);
            sum += raw;
            if (PARTS) {
                parts.a += x[e] >= low ? raw - kRawZero : 0;
                parts.b += x[e] >= high ? raw - kRawZero : 0;
            }
        }
        sum -= E * kRawZero;
    }
    // The vectors of a warp: `steps` rows of 32, so that a slab, kStep of them, is a range of the row.  f(v, vector)
    // for each, done(slab) by the whole warp after each slab.
    __device__ __forceinline__ int steps() const { return (nvec + 32 * kWarps - 1) / (32 * kWarps); }
    template <class F, class D>
    __device__ __forceinline__ void each_slab(F f, D done) const {
        static_assert(kStep % kAhead == 0, "whole batches");
        const int n = steps(), warp_from = (int(threadIdx.x) >> 5) * n * 32, from = warp_from + int(threadIdx.x & 31);
#pragma unroll 1
        for (int s = 0; s < n; s += kStep) {
#pragma unroll 1
            for (int b = s; b < min(s + kStep, n); b += kAhead) {
                const int v = from + 32 * b, last = warp_from + 32 * (b + kAhead) - 1;
                uint4 q[kAhead];
                // a batch that lies in the row as a whole, the same for the warp
                if (b + kAhead <= n && last < nvec && last != tail && warp_from + 32 * b != head) {
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) q[j] = resident ? vectors()[v + 32 * j] : __ldcg(source + v + 32 * j);
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) f(v + 32 * j, q[j]);
                } else {
#pragma unroll 1
                    for (int j = 0; j < kAhead; ++j)
                        if (b + j < n && v + 32 * j < nvec) f(v + 32 * j, vec(v + 32 * j));
                }
            }
            done(s / kStep);
        }
    }

    // Everyone's pair, in rank order, after all have pushed theirs.  The two
    // buffers alternate: a CTA writes a buffer again only after a later
    // exchange, which its readers join when they have read it.
    __device__ const Pair* exchange(const Pair& mine) {
        Pair* box = shared().slot[parity];
        auto cluster = cg::this_cluster();
        if (int(threadIdx.x) < size) *cluster.map_shared_rank(box + rank, threadIdx.x) = mine;
        cluster.sync();
        parity ^= 1;
        return box;
    }
};

template <class Op>
__device__ __forceinline__ Pair block_reduce(Pair v, Op op) {
    Shared& sh = shared();
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Pair o{__shfl_xor_sync(0xffffffffu, v.a, d), __shfl_xor_sync(0xffffffffu, v.b, d)};
        v = op(v, o);
    }
    __syncthreads();  // red may still be read from the call before
    if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.red[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int d = kWarps / 2; d > 0; d >>= 1) {
        const Pair o{__shfl_xor_sync(0xffffffffu, v.a, d), __shfl_xor_sync(0xffffffffu, v.b, d)};
        v = op(v, o);
    }
    return v;
}

__device__ __forceinline__ u64 warp_exclusive(u64 v) {
    u64 inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const u64 o = __shfl_up_sync(0xffffffffu, inc, d);
        if ((threadIdx.x & 31) >= d) inc += o;
    }
    return inc - v;
}

// Exclusive prefix of one value per thread over the block.
__device__ __forceinline__ u64 block_exclusive(u64 v) {
    Shared& sh = shared();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u64 prior = warp_exclusive(v);
    __syncthreads();
    if (lane == 31) sh.red[warp].a = prior + v;
    __syncthreads();
    u64 before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
        if (w < warp) before += sh.red[w].a;
    return before + prior;
}

// Exclusive prefix of a float per thread over the block, and the sum of all.
__device__ __forceinline__ void block_exclusive_float(float v, float& before, float& total) {
    Shared& sh = shared();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float inc = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const float o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 31) sh.red[warp].a = u64(__float_as_uint(inc));
    __syncthreads();
    before = __shfl_up_sync(0xffffffffu, inc, 1);
    if (lane == 0) before = 0.f;
    total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w == warp) before += total;
        total += __uint_as_float(uint32_t(sh.red[w].a));
    }
}

// Tokens in the bins before `bin`, from counts that lie kPerThread to a thread.
__device__ u64 count_above(int first, u64 before, const uint32_t (&cnt)[kPerThread], int bin) {
    Shared& sh = shared();
    __syncthreads();
    if (first <= bin && bin < first + kPerThread) {
        u64 c = before;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i)
            if (first + i < bin) c += cnt[i];
        sh.bound[0] = c;
    }
    __syncthreads();
    return sh.bound[0];
}

// (n + d - 1) / d for n < 2^63 and 1 <= d: a quotient in double precision, put right.
__device__ __forceinline__ u64 ceil_div(u64 n, u64 d) {
    u64 q = u64(__ddiv_rn(double(n), double(d)));
    while (q > 0 && (q - 1) * d >= n) --q;
    while (q * d < n) ++q;
    return q;
}

__device__ __forceinline__ int slabs_of_warp(int steps) { return (steps + kStep - 1) / kStep; }

// Sums of slabs, in index order -> the slab that running sum `target` falls
// into and the sum before it.  For one warp.
__device__ __forceinline__ int find_slab(int slabs, u64 target, u64& sum) {
    const Shared& sh = shared();
    const int lane = threadIdx.x & 31, per_lane = (slabs + 31) / 32;
    int slab = min(lane * per_lane, slabs);
    const int end = min(slab + per_lane, slabs);
    u64 part = 0;
    for (int i = slab; i < end; ++i) part += sh.slab[i];
    sum += warp_exclusive(part);
    const bool here = sum <= target && target < sum + part;
    if (here)
        while (sum + sh.slab[slab] <= target) sum += sh.slab[slab++];
    const int from = max(0, __ffs(__ballot_sync(0xffffffffu, here)) - 1);
    slab = __shfl_sync(0xffffffffu, slab, from), sum = __shfl_sync(0xffffffffu, sum, from);
    return slab;
}

// The value whose weight (weigh(x, slot)) running sum `target` falls into,
// `ahead` before this CTA's slabs; found(x, slot) by one thread.  Every warp
// finds the slab, a warp adds up each of its steps, and the first warp goes
// through the step.
template <int TY, class W, class F>
__device__ __forceinline__ void find_value(const Row<TY>& r, u64 ahead, u64 target, W weigh, F found) {
    constexpr int E = Elem<TY>::E;
    static_assert(kStep <= kWarps, "a warp for each step");
    Shared& sh = shared();
    const int n = r.steps(), each = slabs_of_warp(n), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int slab = find_slab(kWarps * each, target, ahead), first = slab / each * n, from = first + slab % each * kStep;
    const auto step_mass = [&](int step, u64 (&w)[E], float (&x)[E]) {
        const int v = step * 32 + lane;
        u64 vec = 0;
        if (v < r.nvec) Elem<TY>::unpack(r.vec(v), x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            w[e] = v < r.nvec ? weigh(x[e], v * E + e) : 0;
            vec += w[e];
        }
        return vec;
    };
    u64 w[E] = {};
    float x[E];
    if (warp < kStep) {
        u64 sum = from + warp < first + n ? step_mass(from + warp, w, x) : 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) sh.red[warp].a = sum;
    }
    __syncthreads();
    int step = 0;
    while (step < kStep - 1 && ahead + sh.red[step].a <= target) ahead += sh.red[step++].a;
    if (warp == step) {  // it has the values at hand
        u64 vec = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) vec += w[e];
        u64 at = ahead + warp_exclusive(vec);
        if (at <= target && target < at + vec) {
            bool done = false;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                at += w[e];
                if (!done && at > target) found(x[e], ((from + step) * 32 + lane) * E + e), done = true;
            }
        }
    }
}

// The index of this CTA's `nth` kept token (from 1) whose logit is `value`; -1
// where it has fewer.
template <int TY>
__device__ int nth_equal(const Row<TY>& r, float value, u64 nth) {
    constexpr int E = Elem<TY>::E;
    Shared& sh = shared();
    const int n = r.steps(), each = slabs_of_warp(n), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();  // slab may still be read
    if (threadIdx.x == 0) sh.found_bin = -1;
    uint32_t ties = 0;
    r.each_slab(
        [&](int v, const uint4& q) {
            if (Elem<TY>::largest(q) < value) return;
            float x[E];
            Elem<TY>::unpack(q, x);
#pragma unroll
            for (int e = 0; e < E; ++e) ties += x[e] == value && r.kept(value, v * E + e);
        },
        [&](int slab) {
            ties = __reduce_add_sync(0xffffffffu, ties);
            if (lane == 0) sh.slab[warp * each + slab] = ties;
            ties = 0;
        });
    __syncthreads();
    if (nth > 0 && n > 0)
        find_value(r, 0, nth - 1, [&](float x, int slot) { return u64(x == value && r.kept(value, slot)); },
                   [&](float, int slot) { sh.found_bin = r.first + slot; });
    __syncthreads();
    return sh.found_bin;
}

// Cuts the kept set inside [lo, hi], which holds at most `n` of it: `base`
// tokens (mass, where MASS) lie above, and the smallest prefix by (value,
// index) with `target` stays.  Where there is no such prefix nothing is cut.
// Every CTA of the cluster takes the same decisions from the same merged sums.
// `g`: holds all of this CTA's tokens in [lo, hi], or null.  Returns whether
// there was a prefix.
template <int TY, bool MASS>
__device__ bool cut_row(Row<TY>& r, float lo, float hi, u64 base, u64 target, u64 n, const Region* g = nullptr) {
    Shared& sh = shared();
    Search& f = sh.search;
    auto cluster = cg::this_cluster();
    const int per = kBins / r.size;  // bins that one CTA merges
    float scale = 0.f, lift = 1.f;   // of the last histogram
    int border = -1;                 // its bin, where there was one
    auto bin = [&](float x) { return max(0, min(kBins - 1, __float2int_rz(__fmul_rn(__fmul_rn(__fsub_rn(hi, x), lift), scale)))); };
    // Few logits lie in the range once it is narrow: one branch for the others.
    auto inside = [&](float x, int slot) {
        return (x >= lo & x <= hi) && r.kept(x, slot) && (border < 0 || bin(x) == border);
    };
    const auto each = [&](auto f) {
        if (TY != 0 && MASS && g)
            for (int i = threadIdx.x; i < int(g->n); i += kThreads) f(g->v[i], g->slot[i]);
        else
            r.each(f);
    };
    while (n > u64(kCap)) {
        border = -1;
        // A range below 2^-118 has no scale in fp32: it would go to the two ends of the histogram, and a round would
        // take one value off it.
        lift = __fsub_rn(hi, lo) < 0x1p-64f ? 0x1p80f : 1.f;
        scale = __fdiv_rn(float(kBins), __fmul_rn(__fsub_rn(hi, lo), lift));
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            f.cnt[b] = f.tcnt[b] = 0;
            if (MASS) f.mass[b] = f.tmass[b] = 0;
        }
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
        each([&](float x, int slot) {
            if (inside(x, slot)) {
                const int b = bin(x);
                atomicAdd(&f.cnt[b], 1u);
                if (MASS) atomicAdd(&f.mass[b], r.weight(x));
            }
        });
        cluster.sync();
        // this CTA's range of bins, by teams of threads that share the CTAs to read
        const int teams = max(1, kThreads / per), team = int(threadIdx.x) / per;
        if (team < teams)
            for (int i = int(threadIdx.x) % per; i < per; i += kThreads) {
                const int b = r.rank * per + i;
                uint32_t c = 0;
                u64 w = 0;
                for (int q = team; q < r.size; q += teams) {
                    c += *cluster.map_shared_rank(&f.cnt[b], q);
                    if (MASS) w += *cluster.map_shared_rank(&f.mass[b], q);
                }
                if (c) atomicAdd(&f.tcnt[b], c);
                if (MASS && w) atomicAdd(&f.tmass[b], w);
            }
        __syncthreads();
        for (int i = threadIdx.x; i < per * (r.size - 1); i += kThreads) {
            const int to = (r.rank + 1 + i / per) & (r.size - 1), b = r.rank * per + i % per;
            *cluster.map_shared_rank(&f.tcnt[b], to) = f.tcnt[b];
            if (MASS) *cluster.map_shared_rank(&f.tmass[b], to) = f.tmass[b];
        }
        cluster.sync();
        // two bins a thread, from the largest values down
        const int b0 = 2 * threadIdx.x;
        const u64 v0 = MASS ? f.tmass[b0] : f.tcnt[b0], v1 = MASS ? f.tmass[b0 + 1] : f.tcnt[b0 + 1];
        const u64 at = base + block_exclusive(v0 + v1);
        if (at < target && target <= at + v0) sh.found_bin = b0, sh.bound[1] = at, sh.found = 1;
        if (at + v0 < target && target <= at + v0 + v1) sh.found_bin = b0 + 1, sh.bound[1] = at + v0, sh.found = 1;
        __syncthreads();
        if (!sh.found) return false;
        border = sh.found_bin, base = sh.bound[1];
        n = f.tcnt[border];
        __syncthreads();  // found is written again
        if (n <= u64(kCap)) break;
        // the values left: all alike, or split
        float mn = INFINITY, mx = -INFINITY;
        each([&](float x, int slot) {
            if (inside(x, slot)) mn = fminf(mn, x), mx = fmaxf(mx, x);
        });
        auto range = [](Pair p, Pair q) {
            return Pair{as_bits(fminf(as_float(p.a), as_float(q.a))), as_bits(fmaxf(as_float(p.b), as_float(q.b)))};
        };
        Pair own = block_reduce(Pair{as_bits(mn), as_bits(mx)}, range);
        const Pair* all = r.exchange(own);
        for (int q = 0; q < r.size; ++q) own = range(own, all[q]);
        lo = as_float(own.a), hi = as_float(own.b), border = -1;
        if (!(lo < hi)) {
            if (lo > hi) return false;  // none
            // equal logits: the lowest indices are kept
            u64 need = target - base;
            if (MASS) {
                const u64 w = r.weight(hi);
                if (w == 0) return false;
                need = ceil_div(need, w);
            }
            u64 ties = 0;
            each([&](float x, int slot) { ties += inside(x, slot); });
            auto add = [](Pair p, Pair q) { return Pair{p.a + q.a, 0}; };
            all = r.exchange(block_reduce(Pair{ties, 0}, add));
            u64 ahead = 0;
            for (int q = 0; q < r.rank; ++q) ahead += all[q].a;
            const int mine = nth_equal(r, hi, ahead < need ? need - ahead : 0);
            all = r.exchange(Pair{u64(uint32_t(mine)), 0});
            int index = -1;
            for (int q = 0; q < r.size; ++q) index = max(index, int(uint32_t(all[q].a)));
            if (index >= 0) r.cut_at(hi, index);
            return index >= 0;
        }
    }
    // rank the tokens left exactly; the exchange before tells every CTA that nobody reads the lists any more
    r.exchange(Pair{0, 0});
    if (threadIdx.x == 0) f.ln = 0, sh.found = 0;
    __syncthreads();
    each([&](float x, int slot) {
        if (inside(x, slot)) {
            const uint32_t at_list = atomicAdd(&f.ln, 1u);
            if (at_list < uint32_t(kCap)) f.lv[at_list] = x, f.li[at_list] = r.first + slot;
        }
    });
    cluster.sync();
    // every CTA's count, then each thread one candidate of the row
    if (int(threadIdx.x) < r.size) sh.slab[threadIdx.x] = *cluster.map_shared_rank(&f.ln, threadIdx.x);
    __syncthreads();
    int from = 0, owner = -1, at_owner = 0;
    for (int q = 0; q < r.size; ++q) {
        const int m = min(int(sh.slab[q]), kCap - from);
        if (int(threadIdx.x) >= from && int(threadIdx.x) < from + m) owner = q, at_owner = threadIdx.x - from;
        from += m;
    }
    if (owner >= 0) {
        f.gv[threadIdx.x] = *cluster.map_shared_rank(&f.lv[at_owner], owner);
        f.gi[threadIdx.x] = *cluster.map_shared_rank(&f.li[at_owner], owner);
    }
    __syncthreads();
    int place = 0;
    float x = 0.f;
    int index = 0;
    const bool mine = int(threadIdx.x) < from;
    if (mine) {
        x = f.gv[threadIdx.x], index = f.gi[threadIdx.x];
        for (int j = 0; j < from; ++j) place += f.gv[j] > x || (f.gv[j] == x && f.gi[j] < index);
        f.gw[place] = MASS ? r.weight(x) : 1;
    }
    __syncthreads();
    const u64 w = mine ? f.gw[threadIdx.x] : 0;
    const u64 sum = base + block_exclusive(w);
    if (sum < target && target <= sum + w) sh.found_bin = threadIdx.x, sh.found = 1;  // its place
    __syncthreads();
    const bool found = sh.found;
    if (mine && found && place == sh.found_bin) sh.bound[0] = as_bits(x), sh.bound[1] = u64(uint32_t(index));
    __syncthreads();
    if (found) r.cut_at(as_float(sh.bound[0]), int(uint32_t(sh.bound[1])));
    __syncthreads();
    return found;
}

// The kept mass of each slab of this CTA into sh.slab, and their sum.
template <int TY, bool TIES>
__device__ u64 slab_masses(const Row<TY>& r) {
    const int n = r.steps(), each = slabs_of_warp(n), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float from = fmaxf(TIES ? r.tie_v : r.edge, r.weigh_from);
    u64 mine = 0, sum = 0;
    Pair none{0, 0};
    __syncthreads();  // slab may still be read
    r.each_slab([&](int v, const uint4& q) { r.template add_kept<TIES, false>(v, q, from, sum, 0.f, 0.f, none); },
                [&](int slab) {
                    if (__any_sync(0xffffffffu, sum != 0)) {
#pragma unroll
                        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    }
                    if (lane == 0) shared().slab[warp * each + slab] = sum;
                    mine += sum, sum = 0;
                });
    return lane == 0 ? mine : 0;
}
template <int TY>
__device__ u64 slab_masses(const Row<TY>& r) {
    return r.tie_i < 0 ? slab_masses<TY, false>(r) : slab_masses<TY, true>(r);
}

// The kept mass in this thread's vectors, and that at low or high and above (by mass, not by number).
template <int TY, bool PARTS>
__device__ u64 kept_mass(const Row<TY>& r, float low, float high, Pair& parts) {
    u64 sum = 0;
    parts = Pair{0, 0};
    const bool ties = r.tie_i >= 0;
    const float from = fmaxf(ties ? r.tie_v : r.edge, r.weigh_from);
    if (ties)
        r.each_slab([&](int v, const uint4& q) { r.template add_kept<true, PARTS>(v, q, from, sum, low, high, parts); }, [](int) {});
    else
        r.each_slab([&](int v, const uint4& q) { r.template add_kept<false, PARTS>(v, q, from, sum, low, high, parts); }, [](int) {});
    return sum;
}

// The same, with the tokens from low to below high and the slabs' masses at
// high and above kept in region().  The caller has set n to 0.
template <int TY, bool TIES>
__device__ u64 mass_and_region(const Row<TY>& r, float low, float high, Pair& parts) {
    constexpr int E = Elem<TY>::E;
    Region& g = region();
    const int each = slabs_of_warp(r.steps()), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float from = fmaxf(TIES ? r.tie_v : r.edge, r.weigh_from);
    u64 sum = 0, above = 0;
    parts = Pair{0, 0};
    r.each_slab(
        [&](int v, const uint4& q) {
            r.template add_kept<TIES, true>(v, q, from, sum, low, high, parts);
            if (Elem<TY>::largest(q) < low) return;
            float x[E];
            Elem<TY>::unpack(q, x);
            uint32_t in = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) in |= uint32_t(x[e] >= low & x[e] < high) << e;
            if (in == 0) return;
            uint32_t at = atomicAdd(&g.n, uint32_t(__popc(in)));
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in >> e & 1) {
                    if (at < uint32_t(kRegion)) g.v[at] = x[e], g.slot[at] = v * E + e;
                    ++at;
                }
        },
        [&](int slab) {
            u64 here = parts.b;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) here += __shfl_xor_sync(0xffffffffu, here, d);
            if (lane == 0) g.slab[warp * each + slab] = here, above += here;
            parts.b = 0;
        });
    parts.b = above;
    return sum;
}

// slab_masses from a region whose border has been found.
template <int TY>
__device__ u64 slab_masses(const Row<TY>& r, const Region& g) {
    constexpr int E = Elem<TY>::E;
    Shared& sh = shared();
    const int n = r.steps(), each = slabs_of_warp(n);
    __syncthreads();  // slab may still be read
    for (int i = threadIdx.x; i < kWarps * each; i += kThreads) sh.slab[i] = g.slab[i];
    __syncthreads();
    for (int i = threadIdx.x; i < int(g.n); i += kThreads)
        if (r.kept(g.v[i], g.slot[i])) {
            const int row = g.slot[i] / (32 * E), warp = row / n;
            atomicAdd(&sh.slab[warp * each + (row - warp * n) / kStep], r.weight(g.v[i]));
        }
    __syncthreads();
    u64 mine = 0;
    for (int i = threadIdx.x; i < kWarps * each; i += kThreads) mine += sh.slab[i];
    return mine;
}

// The log probability of a token x: `sum` is that of exp(logit - top) over all
// tokens, 1 at least and 2^19 at most.  In 64 bits up to here, rounded once: the
// logarithm is an fp32 one put right by a Newton step, whose remainder is below
// 1e-12 (a chain of a third of a double-precision logarithm's steps, in which
// every row waits for one thread).
__device__ __forceinline__ float log_probability(float x, float top, double sum) {
    const float guess = logf(float(sum));
    const double rest = __fma_rn(__dmul_rn(sum, unit()), scaled_exp(double(guess), kStep1), -1.0);
    return float((double(x) - double(top)) - double(guess) - rest);
}

// For the CTA that holds the token.
template <int TY>
__device__ void write_token(const Row<TY>& r, const Args& a, int row, u64 ahead, u64 target, double z) {
    find_value(r, ahead, target, [&](float x, int slot) { return r.kept(x, slot) ? r.weight(x) : 0; },
               [&](float x, int slot) {
                   a.tokens[row] = r.first + slot;
                   if (a.logprobs) a.logprobs[row] = log_probability(x, r.top, z);
               });
}

__device__ __forceinline__ double as_double(u64 v) { return __longlong_as_double(static_cast<long long>(v)); }
__device__ __forceinline__ u64 as_bits(double v) { return u64(__double_as_longlong(v)); }
__device__ __forceinline__ Pair add_doubles(Pair p, Pair q) { return Pair{as_bits(as_double(p.a) + as_double(q.a)), 0}; }

// The sum of exp(x - top) over this CTA's logits.  Those up to kReach below `top`
// are taken in 64 bits: for fp16 and fp32 they are few, and a row's sum can rest
// on one of them.  The others go through fp32 one vector at a time, each off by
// at most (|x - top| + 4) steps of 2^-24 of itself and 7 of its vector's sum;
// they have e^-2 at most each, so what is left of these steps averages out.
// Vectors are joined in 64 bits.  64 flat fp32 rows of 248320 at T = 0.7: 60.7 us
// in all, 64.9 where the fp32 ones start at 3, 78 with all in 64 bits, and 59.4
// with all in fp32.
template <int TY>
__device__ double exponentials(const Row<TY>& r, float top) {
    constexpr int E = Elem<TY>::E;
    double sum = 0.0, close = 0.0;
    constexpr float kReach = TY == 0 ? 600.f : 2.f;
    const float near = __fsub_rn(top, kReach);
    r.each_vector([&](int, const uint4& q) {
        float x[E], part = 0.f;
        Elem<TY>::unpack(q, x);
#pragma unroll
        for (int e = 0; e < E; ++e) part += x[e] >= near ? 0.f : expf(__fsub_rn(x[e], top));
        sum += double(part);
        if (Elem<TY>::largest(q) >= near) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (x[e] >= near) close += scaled_exp(double(top) - double(x[e]), kStep1);
        }
    });
    return as_double(block_reduce(Pair{as_bits(__fma_rn(close, unit(), sum)), 0}, add_doubles).a);
}
__device__ __forceinline__ Pair add_pairs(Pair p, Pair q) { return Pair{p.a + q.a, p.b + q.b}; }

// floor(u * mass): the token is the first whose running mass is above it.
__device__ __forceinline__ u64 drawn(u64 mass, float u) { return __umul64hi(mass, __double2ull_rz(double(u) * 0x1p64)); }
// ceil(p * mass), 1 at least, for p < 1.
__device__ __forceinline__ u64 nucleus(u64 mass, float p) {
    const u64 share = __double2ull_rz(double(p) * 0x1p64);
    return max(u64(1), __umul64hi(mass, share) + (mass * share != 0));
}

// The sum of a row's exponentials from what every CTA has of it.  For a warp:
// every lane gets it.
template <int TY>
__device__ double joined_partition(const Row<TY>& r) {
    double z = 0.0;
    const int lane = threadIdx.x & 31;
    if (lane < r.size) {
        const Pair part = shared().part[lane];
        const float local = as_float(part.a);
        if (local >= r.top - 600.f) z = as_double(part.b) * (scaled_exp(double(r.top) - double(local), kStep1) * unit());
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
    return z;
}

// The same from a bf16 row's counts, for a block.  The tiny bin's values are not
// alike (by up to two per mille in their exponentials): theirs are summed apart.
__device__ double counted_partition(const Row<0>& r) {
    const Values& h = shared().values;
    double sum = 0.0;
#pragma unroll 3
    for (int i = 0; i < kPerThread; ++i) {
        const int bin = int(threadIdx.x) * kPerThread + i;
        const uint32_t c = h.all[bin];
        if (c && bin != kTinyBin) sum = __fma_rn(double(c), scaled_exp(double(r.top) - double(near_edge(bin)), kStep1), sum);
    }
    sum *= unit();
    if (threadIdx.x == 0 && h.all[kTinyBin]) {
        u64 tiny = 0;
        for (int q = 0; q < r.size; ++q) tiny += h.tiny_sum[q];
        sum += double(tiny) * 0x1p-50 * exp(-double(r.top));
    }
    return as_double(block_reduce(Pair{as_bits(sum), 0}, add_doubles).a);
}

// Pushes the tokens at `bottom` or above to the cluster's first CTA.  The caller
// synchronises the cluster next, and has made sure that the row has no more than
// kList of them, by counts that no cut has clipped: every token of the border's
// value is pushed, also those that top-k leaves out.  (A longer list would have
// lost tokens: draw_from_list refuses it.)
template <int TY>
__device__ void push_list(const Row<TY>& r, float bottom) {
    auto cluster = cg::this_cluster();
    List& l = *cluster.map_shared_rank(&shared().values.list, 0);
    uint32_t* const listed = cluster.map_shared_rank(&shared().listed, 0);
    r.each_vector([&](int v, const uint4& q) {
        if (Elem<TY>::largest(q) < bottom) return;
        float x[Elem<TY>::E];
        Elem<TY>::unpack(q, x);
#pragma unroll
        for (int e = 0; e < Elem<TY>::E; ++e)
            if (x[e] >= bottom) {
                const uint32_t at = atomicAdd(listed, 1u);
                if (at < uint32_t(kList)) l.v[at] = x[e], l.i[at] = r.first + v * Elem<TY>::E + e;
            }
    });
}

// Ranks the list by (value, index) into itself, with the weights of the first
// `limit`.  Few tokens are compared with each other; more are first put in
// order of their bins, whose counts say where each bin starts.
template <int TY>
__device__ __forceinline__ void rank_list(const Row<TY>& r, int n, u64 limit) {
    Shared& sh = shared();
    List& l = sh.values.list;
    const int tid = threadIdx.x;
    const auto before = [](float x, int i, float y, int j) { return x > y || (x == y && i < j); };
    const auto put = [&](int rank, float x, int index) {
        l.weight[rank] = u64(rank) < limit ? r.weight(x) : 0, l.v[rank] = x, l.i[rank] = index;
    };
    if (n <= kThreads / 2) {
        const int e = tid >> 1, half = tid & 1;  // two threads a token
        int rank = 0, index = 0;
        float x = 0.f;
        if (e < n) {
            x = l.v[e], index = l.i[e];
            for (int j = half; j < n; j += 2) rank += before(l.v[j], l.i[j], x, index);
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        __syncthreads();
        if (e < n && half == 0) put(rank, x, index);
        __syncthreads();
        return;
    }
    uint32_t* const start = sh.values.all;
    const auto bin_of = [](float x) {
        const uint32_t bits = __float_as_uint(x), code = ((bits >> 16) & 0x7fffu) - kFirstCode;
        return int(code < uint32_t(kCodes) ? (bits >> 31 ? kNegative + code : kCodes - 1 - code) : uint32_t(kTinyBin));
    };
    uint32_t count = 0;
    for (int i = 0; i < kPerThread; ++i) count += start[tid * kPerThread + i];
    uint32_t at = uint32_t(block_exclusive(count));
    for (int i = 0; i < kPerThread; ++i) {
        const uint32_t c = start[tid * kPerThread + i];
        start[tid * kPerThread + i] = at, at += c;
    }
    __syncthreads();
    for (int e = tid; e < n; e += kThreads) {
        const float x = l.v[e];
        const uint32_t place = min(atomicAdd(&start[bin_of(x)], 1u), uint32_t(kList - 1));
        sh.ordered_v[place] = x, sh.ordered_i[place] = l.i[e];
    }
    __syncthreads();
    // start is now each listed bin's end; all the bins before one are listed whole
    for (int e = tid; e < n; e += kThreads) {
        const float x = sh.ordered_v[e];
        const int index = sh.ordered_i[e], bin = bin_of(x), to = min(int(start[bin]), n);
        int rank = bin ? min(int(start[bin - 1]), n) : 0;
        const int from = rank;
        for (int j = from; j < to; ++j) rank += before(sh.ordered_v[j], sh.ordered_i[j], x, index);
        put(rank, x, index);
    }
    __syncthreads();
}

// The first CTA ranks its list, applies top-k (`limit`) and top-p and draws.
// `whole`: the mass that top-p refers to; 0: that of the first `limit`.
template <int TY>
__device__ void draw_from_list(const Row<TY>& r, const Args& a, int row, u64 limit, float p, float u, u64 whole) {
    Shared& sh = shared();
    List& l = sh.values.list;
    const int tid = threadIdx.x, n = int(sh.listed);
    if (n > kList) {
        if (tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, kFlagBounds);
        }
        return;
    }
    double z = 1.0;
    if (a.logprobs) {
        if constexpr (TY == 0)
            z = counted_partition(r);
        else
            z = joined_partition(r);
    }
    rank_list(r, n, limit);
    // two ranks a thread
    if (tid == 0) sh.found_bin = int(min(u64(n), limit)) - 1;
    const u64 w0 = 2 * tid < n ? l.weight[2 * tid] : 0, w1 = 2 * tid + 1 < n ? l.weight[2 * tid + 1] : 0;
    const u64 before = block_exclusive(w0 + w1);
    if (p < 1.f) {
        if (tid == kThreads - 1) sh.bound[0] = before + w0 + w1;
        __syncthreads();
        const u64 target = nucleus(whole ? whole : sh.bound[0], p);
        if (before < target && target <= before + w0) sh.found_bin = 2 * tid;
        if (before + w0 < target && target <= before + w0 + w1) sh.found_bin = 2 * tid + 1;
    }
    __syncthreads();
    const int keep = sh.found_bin + 1;
    const u64 mass = block_reduce(Pair{(2 * tid < keep ? w0 : 0) + (2 * tid + 1 < keep ? w1 : 0), 0}, add_pairs).a;
    const u64 target = drawn(mass, u);
    const auto answer = [&](int rank) {
        a.tokens[row] = l.i[rank];
        if (a.logprobs) a.logprobs[row] = log_probability(l.v[rank], r.top, z);
    };
    if (keep <= kThreads / 2) {
        // mass up to each kept token in index order, by two threads
        const int e = tid >> 1, half = tid & 1;
        u64 w = 0, upto = 0;
        if (e < keep) {
            const int index = l.i[e];
            w = l.weight[e];
            for (int j = half; j < keep; j += 2)
                if (l.i[j] <= index) upto += l.weight[j];
        }
        upto += __shfl_xor_sync(0xffffffffu, upto, 1);
        if (half == 0 && upto > target && upto - w <= target) answer(e);
        return;
    }
    // by ranges of indices first: the mass of each, the one that holds the token, then its few tokens
    u64* const range = reinterpret_cast<u64*>(sh.values.all);
    const int shift = max(0, 32 - __clz(a.vocab - 1) - 9);  // at most kThreads = 2^9 ranges
    range[tid] = 0;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    for (int e = tid; e < keep; e += kThreads) atomicAdd(&range[l.i[e] >> shift], l.weight[e]);
    __syncthreads();
    const u64 in_range = range[tid], ahead = block_exclusive(in_range);
    if (ahead <= target && target < ahead + in_range) sh.found_bin = tid, sh.bound[1] = ahead;
    __syncthreads();
    const int of = sh.found_bin;
    for (int e = tid; e < keep; e += kThreads)
        if (l.i[e] >> shift == of) sh.ordered_i[atomicAdd(&sh.listed, 1u)] = e;
    __syncthreads();
    const int few = int(sh.listed);
    for (int e = tid; e < few; e += kThreads) {
        const int rank = sh.ordered_i[e], index = l.i[rank];
        u64 upto = sh.bound[1];
        for (int j = 0; j < few; ++j)
            if (l.i[sh.ordered_i[j]] <= index) upto += l.weight[sh.ordered_i[j]];
        if (upto > target && upto - l.weight[rank] <= target) answer(rank);
    }
}

// Kept masses of the CTAs -> the one that holds the token finds it.  from_mass:
// that mass is the sum of exponentials for the log probability too (off by half a
// unit of 2^-s a token at most, so by 2^-27 in all for 2^18 tokens).
template <int TY>
__device__ void draw_from_row(Row<TY>& r, const Args& a, int row, float u, bool from_mass, const Region* g = nullptr) {
    const Pair own = block_reduce(Pair{g ? slab_masses(r, *g) : slab_masses(r), 0}, add_pairs);
    const Pair* all = r.exchange(own);
    u64 whole = 0, ahead = 0;
    for (int q = 0; q < r.size; ++q) {
        if (q < r.rank) ahead += all[q].a;
        whole += all[q].a;
    }
    const u64 target = drawn(whole, u);
    if (ahead <= target && target < ahead + own.a)
        write_token(r, a, row, ahead, target,
                    !a.logprobs ? 1.0 : from_mass ? double(whole) * unit() : joined_partition(r));
}

// The row's counts, by value, in every CTA; and for bf16 the mass of the tiny,
// with `logprobs` the sum of their exponentials too (integers: in any order).
// Each CTA adds up a range of codes, four at a time, in its own copy of the
// result, and pushes that to the others.
template <int TY>
__device__ u64 merge_counts(const Row<TY>& r, uint32_t tiny_count, bool logprobs) {
    Values& h = shared().values;
    auto cluster = cg::this_cluster();
    const int tid = threadIdx.x, quads = 2 * kCodes / 4 / r.size, first = r.rank * quads;
    const auto place = [](int quad) {  // the bins of codes 4 * quad + {0..3}: backwards for the positive ones
        return 4 * quad < kCodes ? kCodes - 4 - 4 * quad : kNegative + 4 * quad - kCodes;
    };
    const int teams = max(1, kThreads / quads), team = tid / quads;  // of threads that share the CTAs to read
    if (r.size > 1 && team < teams)
        for (int i = first + tid % quads; i < first + quads; i += kThreads) {
            uint4 sum = make_uint4(0, 0, 0, 0);
            for (int q = team; q < r.size; q += 4 * teams) {  // four loads from other CTAs at a time
                uint4 part[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    part[j] = q + j * teams < r.size
                                  ? *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&h.own[4 * i], q + j * teams))
                                  : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sum.x += part[j].x, sum.y += part[j].y, sum.z += part[j].z, sum.w += part[j].w;
            }
            uint32_t* bins = &h.all[place(i)];
            const bool back = 4 * i < kCodes;
            if (sum.x) atomicAdd(bins + (back ? 3 : 0), sum.x);
            if (sum.y) atomicAdd(bins + (back ? 2 : 1), sum.y);
            if (sum.z) atomicAdd(bins + (back ? 1 : 2), sum.z);
            if (sum.w) atomicAdd(bins + (back ? 0 : 3), sum.w);
        }
    if (r.size == 1)
        for (int i = tid; i < 2 * kCodes; i += kThreads)
            h.all[i < kCodes ? kCodes - 1 - i : i - kCodes + kNegative] = h.own[i];
    if (tid == 0) h.all[kTinyBin] = tiny_count;
    u64 own_tiny = 0;
    if (TY == 0) {
        const int tiny = int(h.own[2 * kCodes]);
        if ((tid & ~31) < tiny) {  // whole warps
            u64 w = tid < tiny ? r.weight(h.tiny[tid]) : 0;
            u64 e = tid < tiny && logprobs ? __double2ull_rn(exp(double(h.tiny[tid])) * 0x1p50) : 0;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d), e += __shfl_xor_sync(0xffffffffu, e, d);
            if ((tid & 31) == 0) atomicAdd(&shared().bound[0], w), atomicAdd(&shared().bound[1], e);
        }
    }
    __syncthreads();
    if (TY == 0) {
        own_tiny = shared().bound[0];
        if (tid < r.size) {
            *cluster.map_shared_rank(&h.tiny_mass[r.rank], tid) = own_tiny;
            *cluster.map_shared_rank(&h.tiny_sum[r.rank], tid) = shared().bound[1];
        }
    }
    for (int i = tid; i < quads * (r.size - 1); i += kThreads) {
        const int to = (r.rank + 1 + i / quads) & (r.size - 1), at = place(first + i % quads);
        *reinterpret_cast<uint4*>(cluster.map_shared_rank(&h.all[at], to)) = *reinterpret_cast<const uint4*>(&h.all[at]);
    }
    cluster.sync();
    return own_tiny;
}

// A row whose counts are whole: every logit has a bin, or no weight.  Returns
// false, in every CTA alike, where a cut of a bf16 row falls among its tiny
// logits; such a row goes the general way.
template <int TY>
__device__ bool counted_row(Row<TY>& r, const Args& a, int row, int k, float p, float u, float floor_v, bool greedy,
                            uint32_t tiny_count) {
    Shared& sh = shared();
    Values& h = sh.values;
    auto cluster = cg::this_cluster();
    const int tid = threadIdx.x;
    const u64 own_tiny = merge_counts(r, tiny_count, a.logprobs);
    const u64 limit = greedy ? 1 : k > 0 && k < a.vocab ? u64(k) : ~u64(0);
    if (greedy) p = 1.f;

    if (a.vocab <= kList && (limit != ~u64(0) || p < 1.f)) {
        push_list(r, fmaxf(bin_bottom(kValueBins - 1), floor_v));
        cluster.sync();
        if (r.rank == 0) draw_from_list(r, a, row, limit, p, u, 0);
        return true;
    }

    // this thread's bins, largest values first; the border of top-k
    const int first = tid * kPerThread;
    uint32_t cnt[kPerThread];
    u64 count = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        cnt[i] = (TY == 0 ? near_edge(first + i) : bin_top(first + i)) >= floor_v ? h.all[first + i] : 0;
        count += cnt[i];
    }
    if (tid == 0) sh.found = 0;
    u64 seen = block_exclusive(count);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        if (seen < limit && limit <= seen + cnt[i])
            sh.found = 1, sh.found_bin = first + i, sh.bound[0] = seen, sh.bound[1] = seen + cnt[i];
        const uint32_t had = cnt[i];
        cnt[i] = seen >= limit ? 0 : uint32_t(min(u64(had), limit - seen));
        seen += had;
    }
    __syncthreads();
    const bool by_count = sh.found;
    int border = by_count ? sh.found_bin : INT_MAX;
    const u64 before = sh.bound[0], listed = sh.bound[1];
    if (by_count && listed <= u64(kList)) {
        push_list(r, fmaxf(TY == 0 && border != kTinyBin ? near_edge(border) : bin_bottom(border), floor_v));
        cluster.sync();
        if (r.rank == 0) {
            draw_from_list(r, a, row, limit, p, u, 0);
        }
        return true;
    }

    if constexpr (TY == 0) {
        u64 ties = by_count ? limit - before : 0;  // kept of the border's value
        if (by_count && border == kTinyBin && limit < listed) return false;
        u64 tiny_mass = 0;
        for (int q = 0; q < r.size; ++q) tiny_mass += h.tiny_mass[q];
        u64 weight[kPerThread], mass = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; i += 3) {
            static_assert(kPerThread % 3 == 0, "three weights at a time");
            u64 three[3] = {0, 0, 0};
            if (__any_sync(0xffffffffu, cnt[i] | cnt[i + 1] | cnt[i + 2])) {
                const float v[3] = {near_edge(first + i), near_edge(first + i + 1), near_edge(first + i + 2)};
                r.weights(v, three);
            }
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                weight[i + j] = cnt[i + j] ? three[j] : 0;
                mass += first + i + j == kTinyBin ? (cnt[i + j] ? tiny_mass : 0) : cnt[i + j] * weight[i + j];
            }
        }
        if (p < 1.f) {
            const u64 ahead = block_exclusive(mass);
            if (tid == kThreads - 1) sh.bound[0] = ahead + mass;
            __syncthreads();
            const u64 whole = sh.bound[0], target = nucleus(whole, p);
            if (ahead < target && target <= ahead + mass) {
                u64 at = ahead, w = 0, kept = 0;
                int bin = 0;
                u64 c = seen - count;  // tokens above this thread's bins
#pragma unroll
                for (int i = 0; i < kPerThread; ++i) {
                    const u64 m = first + i == kTinyBin ? (cnt[i] ? tiny_mass : 0) : cnt[i] * weight[i];
                    c += cnt[i];
                    if (at < target && target <= at + m) bin = first + i, w = weight[i], sh.bound[1] = at, kept = c;
                    at += m;
                }
                sh.found_bin = bin, sh.found = int(min(kept, u64(INT_MAX)));
                if (bin != kTinyBin) sh.bound[1] = ceil_div(target - sh.bound[1], w);
            }
            __syncthreads();
            const int nucleus_border = min(max(sh.found_bin, 0), kValueBins - 1);
            // of top-k's border only a part is in cnt, and more than kList tokens lie at it or above
            const bool tied = by_count && nucleus_border == border;
            border = nucleus_border, ties = sh.bound[1];
            if (border == kTinyBin) return false;
            if (sh.found <= kList && !tied) {
                push_list(r, near_edge(border));
                cluster.sync();
                if (r.rank == 0) draw_from_list(r, a, row, limit, p, u, whole);
                return true;
            }
        }
        u64 here = 0, mine = 0;  // of the border's value in this CTA, and of the kept
        if (border != INT_MAX) {
            // counts of the border's value in the CTAs before this one
            if (tid < r.size) sh.slab[tid] = *cluster.map_shared_rank(&h.own[code_of(border)], tid);
            __syncthreads();
            u64 prior = 0;
            for (int q = 0; q < r.rank; ++q) prior += sh.slab[q];
            here = sh.slab[r.rank];
            mine = prior >= ties ? 0 : min(here, ties - prior);
        }
        mass = 0;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const int bin = first + i;
            if (bin != kTinyBin && weight[i] && bin <= border)
                mass += (bin == border ? mine : h.own[code_of(bin)]) * weight[i];
        }
        if (tid == 0 && border >= kTinyBin && floor_v <= 0.f) mass += own_tiny;
        const Pair own = block_reduce(Pair{mass, 0}, add_pairs);
        const Pair* all = r.exchange(own);
        u64 whole = 0, ahead = 0;
        for (int q = 0; q < r.size; ++q) {
            if (q < r.rank) ahead += all[q].a;
            whole += all[q].a;
        }
        const u64 target = drawn(whole, u);
        if (ahead > target || target >= ahead + own.a) return true;
        // the CTA that holds the token
        const double z = a.logprobs ? counted_partition(r) : 1.0;
        u64 target_at = ahead;
        if (a.part_vecs) {
            // the part that holds it, by the parts' counts
            u64 of[kParts] = {0, 0, 0, 0};
#pragma unroll 1
            for (int i = 0; i < kPerThread; ++i) {
                const int bin = first + i;
                if (bin == border) {
                    u64 left = mine;
                    for (int q = 0; q < kParts; ++q) {
                        const uint32_t c = bin == kTinyBin ? 0 : part_count(code_of(bin), q);
                        const u64 keep = min(left, u64(c));
                        sh.part_here[q] = c, sh.part_kept[q] = uint32_t(keep), left -= keep;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int bin = first + i;
                if (bin != kTinyBin && weight[i] && bin <= border) {
#pragma unroll
                    for (int q = 0; q < kParts; ++q)
                        of[q] += (bin == border ? sh.part_kept[q] : part_count(code_of(bin), q)) * weight[i];
                }
            }
            if (border >= kTinyBin && floor_v <= 0.f && tid < int(h.own[2 * kCodes])) {
                const u64 w = r.weight(h.tiny[tid]);
#pragma unroll
                for (int q = 0; q < kParts; ++q) of[q] += h.tiny_part[tid] == q ? w : 0;
            }
            const Pair front = block_reduce(Pair{of[0], of[1]}, add_pairs), back = block_reduce(Pair{of[2], of[3]}, add_pairs);
            const u64 sums[kParts] = {front.a, front.b, back.a, back.b};
            int part = 0;
#pragma unroll
            for (int q = 0; q < kParts - 1; ++q)
                if (part == q && target_at + sums[q] <= target) target_at += sums[q], part = q + 1;
            const int from = part * a.part_vecs;
            r.narrow(from, min(a.part_vecs, r.nvec - from));
            if (border != INT_MAX) here = sh.part_here[part], mine = sh.part_kept[part];
        }
        if (border == kTinyBin) {
            r.keep_from(bin_bottom(kTinyBin));  // all of the tiny
        } else if (border != INT_MAX) {
            const float v = near_edge(border);
            if (mine == here)
                r.keep_from(v);
            else if (mine == 0)
                r.keep_from(nextafterf(v, INFINITY));
            else
                r.cut_at(v, nth_equal(r, v, mine));
        }
        slab_masses(r);
        __syncthreads();
        write_token(r, a, row, target_at, target, z);
        return true;
    } else {
        // the search below uses the histogram's memory: the counts are in registers, and its own exchanges wait for all
        if (p < 1.f) {
            // The bins' masses by their middle values are some per mille off, so the border almost always lies in
            // the bins from 1.5% of the mass before its estimate to 1.5% after; the exact masses below tell.
            const float per_t = fminf(float(r.step * (1.0 / (256.0 * 1.4426950408889634074))), 1e37f);
            float estimate = 0.f, masses[kPerThread];
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const float middle = fminf(0.5f * bin_bottom(first + i) + 0.5f * bin_top(first + i), r.top);
                masses[i] = cnt[i] ? float(cnt[i]) * expf((middle - r.top) * per_t) : 0.f;
                estimate += masses[i];
            }
            float at, total;
            block_exclusive_float(estimate, at, total);
            const float can = (p - 0.015f) * total, must = (p + 0.015f) * total;
            if (tid == 0) sh.found_bin = 0, sh.found = kValueBins - 1;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                if (at < can && can <= at + masses[i]) atomicMax(&sh.found_bin, first + i);
                if (at < must && must <= at + masses[i]) atomicMin(&sh.found, first + i);
                at += masses[i];
            }
            __syncthreads();
            const int open = sh.found_bin, close = sh.found;
            // tokens above the first bin and up to the last
            const u64 counts_open = count_above(first, seen - count, cnt, open);
            const u64 counts_close = count_above(first, seen - count, cnt, close + 1);
            if (by_count) cut_row<TY, false>(r, fmaxf(bin_bottom(border), floor_v), bin_top(border), before, limit, listed - before);
            const float bottom = fmaxf(bin_bottom(close), floor_v);
            const bool few = counts_close <= u64(kList) && !by_count;
            if (few) push_list(r, bottom);
            // the exact masses: of all, of the bins up to the last, above the first
            const float edge = bin_top(open);
            const bool keep = !r.resident && !few;
            Pair parts;
            u64 own;
            if (keep) {
                if (tid == 0) region().n = 0;
                __syncthreads();
                const float above = nextafterf(edge, INFINITY);
                own = r.tie_i < 0 ? mass_and_region<TY, false>(r, bottom, above, parts) : mass_and_region<TY, true>(r, bottom, above, parts);
            } else {
                own = kept_mass<TY, true>(r, bottom, nextafterf(edge, INFINITY), parts);
            }
            const Pair* all = r.exchange(block_reduce(Pair{own, parts.a}, add_pairs));
            Pair mass{0, 0};
            for (int q = 0; q < r.size; ++q) mass = add_pairs(mass, all[q]);
            const u64 target = nucleus(mass.a, p);
            const bool low_enough = mass.b >= target;
            if (few && low_enough) {
                if (r.rank == 0) draw_from_list(r, a, row, limit, p, u, mass.a);
                return true;
            }
            all = r.exchange(block_reduce(Pair{parts.b, 0}, add_pairs));
            u64 base = 0;
            for (int q = 0; q < r.size; ++q) base += all[q].a;
            const bool high_enough = base < target;
            const bool proved = low_enough && high_enough;
            const Region* g = keep && proved && region().n <= uint32_t(kRegion) ? &region() : nullptr;
            const bool cut = cut_row<TY, true>(r, low_enough ? bottom : r.weigh_from, high_enough ? edge : r.top, high_enough ? base : 0,
                                               target, proved ? counts_close - counts_open : a.vocab, g);
            draw_from_row(r, a, row, u, false, cut ? g : nullptr);
            return true;
        } else if (by_count) {
            cut_row<TY, false>(r, fmaxf(bin_bottom(border), floor_v), bin_top(border), before, limit, listed - before);
        }
        draw_from_row(r, a, row, u, false);
        return true;
    }
}

// *shared += v where offset < 4 kCodes, without a branch: eight of them in a
// row would each part and join the warp again.
__device__ __forceinline__ void add_coded(uint32_t offset, uint32_t shared_address, uint32_t v) {
    asm volatile("{ .reg .pred p; setp.lt.u32 p, %0, %3; @p red.shared.add.u32 [%1], %2; }" ::"r"(offset), "r"(shared_address),
                 "r"(v), "n"(4 * kCodes)
                 : "memory");
}
__device__ __forceinline__ void add_shared(uint32_t shared_address, uint32_t v) {
    asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(shared_address), "r"(v) : "memory");
}

// The values of a counted vector above -128 that have no code.  1: NaN or
// +inf; 2: 128 or more, 8: too many tiny ones.  (4: -128 or less but not -inf.)
template <int TY>
__device__ __noinline__ uint32_t note_others(const uint4 q, int part) {
    constexpr int E = Elem<TY>::E;
    Values& h = shared().values;
    float x[E];
    Elem<TY>::unpack(q, x);
    uint32_t notes = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float size_of = fabsf(x[e]);
        if (!(x[e] < INFINITY)) {
            notes |= 1;
        } else if (x[e] >= 128.f) {
            notes |= 2;
        } else if (size_of < 0x1p-10f) {
            const uint32_t at = atomicAdd(&h.own[2 * kCodes], 1u);
            if (TY == 0) {
                if (at < uint32_t(kTinyCap)) h.tiny[at] = x[e], h.tiny_part[at] = uint8_t(part);
                else notes |= 8;
            }
        }
    }
    return notes;
}

// The notes of a vector that has values without a code.
template <int TY>
__device__ __forceinline__ uint32_t classify(const uint4& q, const float* x, int part) {
    bool others = false, masked = false;
#pragma unroll
    for (int e = 0; e < Elem<TY>::E; ++e) {
        others = others | !(fabsf(x[e]) >= 0x1p-10f & x[e] < 128.f);
        masked = masked | (x[e] <= -128.f & x[e] > -INFINITY);
    }
    return (others ? note_others<TY>(q, part) : 0) | uint32_t(masked) << 2;
}

// 4 kCodes where a half of the word is negative, else 0: the half's sign in all bits (byte 1's or byte 3's, by the
// replicating mode of prmt), multiplied, as the multiplier has less to do here than the integer unit.
template <int SELECTOR>
__device__ __forceinline__ uint32_t negative_offset(uint32_t word) {
    uint32_t sign;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(sign) : "r"(word), "n"(SELECTOR));
    return sign * uint32_t(-4 * kCodes);
}

// Counts eight bf16 values by their bits.  Whether all have a code is asked of
// pairs (magnitude - kFirstCode < kCodes); a warp of which all have adds eight
// times five instructions a value, any other one tests each value.
__device__ __forceinline__ uint32_t count_pairs(const uint4& q, int part, const uint32_t* counts, uint32_t one) {
    constexpr uint32_t kPair = 0x10001u, kMagnitude = 0x7fff * kPair, kShift = (0x10000u - kFirstCode) * kPair;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const uint32_t at = uint32_t(__cvta_generic_to_shared(counts));
    const auto above = [](uint32_t pair) { return max(pair & 0xffffu, pair >> 16) >= uint32_t(kCodes); };
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) most = __viaddmax_u16x2(w[i] & kMagnitude, kShift, most);
    if (!__any_sync(__activemask(), above(most))) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t low = 4 * (w[i] & 0x7fffu) + (at - 4 * kFirstCode);
            const uint32_t high = ((w[i] & 0x7fff0000u) >> 14) + (at - 4 * kFirstCode);
            add_shared(low + negative_offset<0x9999>(w[i]), one);
            add_shared(high + negative_offset<0xbbbb>(w[i]), one);
        }
        return 0;
    }
    // the same with -inf as 2 - 2^-7, and every value tested
    most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t infinite = __heq2_mask(reinterpret_cast<const __nv_bfloat162&>(w[i]), __float2bfloat162_rn(-INFINITY));
        most = __viaddmax_u16x2((w[i] & kMagnitude & ~infinite) | (infinite & 0x3fff * kPair), kShift, most);
        const uint32_t low = 4 * (w[i] & 0x7fffu) - 4 * kFirstCode, high = ((w[i] & 0x7fff0000u) >> 14) - 4 * kFirstCode;
        add_coded(low, low + at + negative_offset<0x9999>(w[i]), one);
        add_coded(high, high + at + negative_offset<0xbbbb>(w[i]), one);
    }
    if (!above(most)) return 0;
    float x[8];
    Elem<0>::unpack(q, x);
    return classify<0>(q, x, part);
}

// One cluster per row.  The barrier of a cluster is the hardware's: all its
// CTAs are resident together and take every barrier, as all decisions that
// lead to one are taken from exchanged values.
template <int TY>
__global__ __launch_bounds__(kThreads, 2) void sample_kernel(const Args a) {
    using El = Elem<TY>;
    constexpr int E = El::E, kBatch = 4;
    Shared& sh = shared();
    auto cluster = cg::this_cluster();
    cluster.barrier_arrive();  // waited for before the first access to another CTA's shared memory
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int row = blockIdx.x / size, tid = threadIdx.x;

    // this CTA's share of the row: whole 16-byte vectors of memory, values outside the row as -inf
    const char* begin = static_cast<const char*>(a.logits) + int64_t(row) * a.stride * El::kBytes;
    const int lead = int(reinterpret_cast<uintptr_t>(begin) % 16) / El::kBytes;
    const int total_vecs = (lead + a.vocab + E - 1) / E;
    const int v0 = min(rank * a.vecs, total_vecs), nvec = min(a.vecs, total_vecs - v0);
    const uint4* base = reinterpret_cast<const uint4*>(begin - lead * El::kBytes) + v0;
    const int i_first = v0 * E - lead;  // index of the first value
    const bool resident = a.resident;   // the logits stay in shared memory; else later passes find them in L2
    const int head = i_first < 0 ? 0 : -1, tail = v0 + nvec == total_vecs && (lead + a.vocab) % E ? nvec - 1 : -1;
    uint4 q[kBatch];
    auto fetch = [&](int b) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = b + j * kThreads + tid;
            if (v < nvec)
                q[j] = v != head && v != tail ? __ldcg(base + v) : edge_vector<TY>(begin, i_first + v * E, a.vocab);
        }
    };
    fetch(0);

    const float T = a.temperature ? a.temperature[row] : 1.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.uniform[row];
    const bool valid = T >= 0.f && T <= kMaxTemperature && p >= 0.f && min_p >= 0.f && min_p <= 1.f && u >= 0.f && u < 1.f;
    if (!valid) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, kFlagParameter);
        }
        cluster.barrier_wait();
        return;
    }
    const bool greedy = T == 0.f || k == 1, cuts = greedy || (k > 0 && k < a.vocab) || p < 1.f;
    const bool counting = TY == 0 || cuts;
    const double step = greedy ? 0.0 : 256.0 * 1.4426950408889634074 / double(T);
    const double depth = min_p > 0.f && !greedy ? double(T) * log(double(min_p)) : 0.0;  // of min-p's border
    Values& h = sh.values;
    if (counting) {
        for (int i = tid; i < int(sizeof(h.own) / 16); i += kThreads) reinterpret_cast<uint4*>(h.own)[i] = make_uint4(0, 0, 0, 0);
        for (int i = tid; i < int(sizeof(h.all) / 16); i += kThreads) reinterpret_cast<uint4*>(h.all)[i] = make_uint4(0, 0, 0, 0);
    }
    const int frac = min(51, 62 - (32 - __clz((a.vocab - 1) | 1)));  // s
    if (TY == 0 && a.part_vecs)
        for (int i = tid; i < kCodes; i += kThreads) vectors()[i] = make_uint4(0, 0, 0, 0);  // kParts / 2 * 2 * kCodes words
    if (tid < 256) sh.pow256[tid] = exp2(frac - tid * (1.0 / 256));
    if (tid == 0) sh.listed = 0, sh.bound[0] = sh.bound[1] = 0;
    __syncthreads();
    float top = -INFINITY;
    bool strange = false;
    uint32_t notes = 0;  // of note_others
    for (int b = 0; b < nvec; b += kBatch * kThreads) {
        uint4 now[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) now[j] = q[j];
        if (b + kBatch * kThreads < nvec) fetch(b + kBatch * kThreads);  // in flight meanwhile
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = b + j * kThreads + tid;
            if (v >= nvec) break;
            if (resident) vectors()[v] = now[j];
            if (TY == 0) {
                const int part = a.part_vecs ? (v >= a.part_vecs) + (v >= 2 * a.part_vecs) + (v >= 3 * a.part_vecs) : 0;
                notes |= count_pairs(now[j], part, a.part_vecs ? parts() + (part >> 1) * 2 * kCodes : h.own, 1u << (16 * (part & 1)));
            } else {
                float x[E];
                El::unpack(now[j], x);
                if (counting) {
                    const uint32_t counts_at = uint32_t(__cvta_generic_to_shared(h.own));
                    bool plain = true;  // every value has a code, or is -inf
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t bits = __float_as_uint(x[e]), code = ((bits >> 16) & 0x7fffu) - kFirstCode;
                        add_coded(4 * code, counts_at + 4 * (code + (bits >> 31) * kCodes), 1u);
                        plain = plain & (code < uint32_t(kCodes) | x[e] == -INFINITY);
                    }
                    if (!plain) notes |= classify<TY>(now[j], x, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) strange = strange | !(x[e] < INFINITY);
                }
            }
            top = fmaxf(top, El::largest(now[j]));
        }
    }

    Row<TY> r{resident, head, tail, base, begin, a.vocab, nvec, i_first, rank, size, 0};
    auto join = [](Pair x, Pair y) { return Pair{as_bits(fmaxf(as_float(x.a), as_float(y.a))), x.b | y.b}; };
    const Pair mine = block_reduce(Pair{as_bits(top), notes | uint32_t(strange)}, join);
    if (TY == 0 && a.part_vecs)
        for (int i = tid; i < 2 * kCodes; i += kThreads) {
            uint32_t c = 0;
#pragma unroll
            for (int part = 0; part < kParts; ++part) c += part_count(i, part);
            h.own[i] = c;
        }
    // Uncut at T = 1, the weights are those exponentials (fp16, fp32; the counts of bf16 give them anyhow).
    const bool from_mass = TY != 0 && a.logprobs && T == 1.f && !cuts && min_p == 0.f && u != 0.f;
    // sum of exponentials for the log probability, against this CTA's largest logit; a bf16 row takes it from its counts
    double sum = 0.0;
    if (TY != 0 && a.logprobs && !from_mass) sum = exponentials(r, as_float(mine.a));
    cluster.barrier_wait();
    const uint32_t own_tiny = counting ? h.own[2 * kCodes] : 0;
    const Pair* all = r.exchange(Pair{mine.a | (mine.b | own_tiny << 8) << 32, as_bits(sum)});
    uint32_t tiny_count = 0;
    top = -INFINITY, notes = 0;
    for (int i = 0; i < size; ++i) {
        const uint32_t high = uint32_t(all[i].a >> 32);
        top = fmaxf(top, as_float(all[i].a)), notes |= high & 255u, tiny_count += high >> 8;
    }
    if (TY != 0 && tid < size) sh.part[tid] = all[tid];  // read after a later barrier
    if ((notes & 1) || top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, notes & 1 ? kFlagNonfinite : kFlagNothingLeft);
        }
        return;
    }
    r.top = top;
    r.step = step;
    r.weigh(u == 0.f && !greedy, frac, T);
    // w >= min_p as a comparison of logits, which is exact
    float floor_v = -INFINITY;
    if (min_p > 0.f && !greedy) floor_v = __double2float_ru(double(top) + depth);
    r.keep_from(floor_v);
    if (counting) {
        // The counts must hold every logit that has a weight: below -128 none has from 37 T on.  A bf16 row also
        // needs its largest logit and min-p's border outside the tiny bin, where values are not told apart.
        const float heat = greedy ? 1.f : fmaxf(T, 1.f);
        bool whole = !(notes & 10) && top > -128.f && !r.count_mode && (!(notes & 4) || top + 128.f >= 37.f * heat);
        if (TY == 0) whole = whole && fabsf(top) > bin_top(kTinyBin) && !(fabsf(floor_v) <= bin_top(kTinyBin));
        if (whole && counted_row(r, a, row, k, p, u, floor_v, greedy, tiny_count)) return;
        cluster.sync();  // the counts' memory is used again
    }

    // The general way: rows without a cut, and those that the counts do not tell enough about.
    if (TY == 0 && a.logprobs) {
        const double own = exponentials(r, top);
        if (tid < size) *cluster.map_shared_rank(&sh.part[rank], tid) = Pair{as_bits(top), as_bits(own)};
        cluster.sync();
    }
    const bool by_count = greedy || (k > 0 && k < a.vocab), by_mass = p < 1.f && !greedy;
    if (by_count || by_mass) {
        // The values that a cut searches: from the smallest logit but -inf and the type's lowest value, which usually
        // masks.  Below 746 T under the top every weight is zero in double precision, so the order there never
        // matters; in fixed point that holds from 37 T (2^-53) on.
        float low = INFINITY;
        r.each([&](float x, int) {
            if (x > El::kLowest) low = fminf(low, x);
        });
        auto least = [](Pair x, Pair y) { return Pair{as_bits(fminf(as_float(x.a), as_float(y.a))), 0}; };
        all = r.exchange(block_reduce(Pair{as_bits(low), 0}, least));
        for (int i = 0; i < size; ++i) low = fminf(low, as_float(all[i].a));
        if (double(top) - 746.0 * double(T) <= double(El::kLowest)) low = El::kLowest;
        const auto from = [&](double units) {
            return fminf(top, fmaxf(fmaxf(low, __double2float_rd(double(top) - units * double(T))), floor_v));
        };
        if (by_count) cut_row<TY, false>(r, from(746.0), top, 0, greedy ? 1 : u64(k), a.vocab);
        if (by_mass) {
            const bool counted = r.count_mode;
            r.weigh(false, frac, T);  // the nucleus goes by mass for u = 0 too
            Pair none;
            all = r.exchange(block_reduce(Pair{kept_mass<TY, false>(r, 0.f, 0.f, none), 0}, add_pairs));
            u64 mass = 0;
            for (int i = 0; i < size; ++i) mass += all[i].a;
            cut_row<TY, true>(r, from(37.0), top, 0, nucleus(mass, p), a.vocab);
            r.weigh(counted, frac, T);
        }
    }
    draw_from_row(r, a, row, u, from_mass);
}

std::atomic<bool> g_attr[3][64];

}  // namespace sample
}  // namespace ornith

using namespace ornith;

extern "C" cudaError_t ornith_moe_b200_sample_launch(const void* logits, int64_t stride, int type,
                                                     const void* temperature, const void* top_k, const void* top_p,
                                                     const void* min_p, const void* uniform, void* tokens,
                                                     void* logprobs, void* flags, int M, int vocab,
                                                     cudaStream_t stream) {
    using namespace sample;
    if (M < 0 || vocab < 1 || vocab > kMaxVocab || type < 0 || type > 2) return cudaErrorInvalidValue;
    if (M == 0) return cudaSuccess;
    if (M == 1) stride = vocab;
    // the rows' extent in bytes fits 64 bits, so that the checks below see all of it
    if (stride < vocab || stride > (int64_t(1) << 40) || M > (int64_t(1) << 60) / stride) return cudaErrorInvalidValue;
    const int bytes = type == 2 ? 4 : 2, per_vec = 16 / bytes;
    const size_t rows4 = size_t(M) * 4, row_bytes = (size_t(M - 1) * size_t(stride) + size_t(vocab)) * bytes;
    for (const void* param : {temperature, top_k, top_p, min_p}) {  // each may be null
        const void* const ptr[5] = {param, logits, uniform, tokens, flags};
        const size_t size[5] = {rows4, row_bytes, rows4, rows4, 4};
        const uintptr_t align[5] = {4, uintptr_t(bytes), 4, 4, 4};
        if (!buffers_ok(ptr, size, align, 3, 0)) return cudaErrorInvalidValue;
        if (!logprobs) continue;
        const void* const with[6] = {param, logits, uniform, tokens, flags, logprobs};
        const size_t with_size[6] = {rows4, row_bytes, rows4, rows4, 4, rows4};
        const uintptr_t with_align[6] = {4, uintptr_t(bytes), 4, 4, 4, 4};
        if (!buffers_ok(with, with_size, with_align, 3, 0)) return cudaErrorInvalidValue;
    }
    // A row may start inside a 16-byte vector and then takes one more.
    const int total_vecs = (vocab + per_vec - 1 + per_vec - 1) / per_vec;
    // CTAs a row: the largest power of two that runs at once (two on each SM), as the steps between two passes over
    // the logits take much the same time for a large share as for a small one: 44 us for 64 mixed rows against 56 with
    // half as many and 61 with twice, 111 against 127 with twice for 256.  No share above kMaxVecs; none below 4 KB
    // (1 and 16 KB measure the same).
    int size = 1;
    while (size < kMaxCluster && ((total_vecs + size - 1) / size > kMaxVecs ||
                                  (int64_t(M) * size * 2 <= 2 * kSms && total_vecs / size > 512)))
        size *= 2;
    if (int64_t(M) * size > INT_MAX) return cudaErrorInvalidValue;
    NvtxRange range("ornith.sample");
    Args a{};
    a.logits = logits, a.stride = stride;
    a.temperature = static_cast<const float*>(temperature);
    a.top_k = static_cast<const int32_t*>(top_k);
    a.top_p = static_cast<const float*>(top_p), a.min_p = static_cast<const float*>(min_p);
    a.uniform = static_cast<const float*>(uniform);
    a.tokens = static_cast<int32_t*>(tokens), a.logprobs = static_cast<float*>(logprobs);
    a.flags = static_cast<uint32_t*>(flags);
    a.vocab = vocab, a.vecs = (total_vecs + size - 1) / size;
    a.resident = a.vecs <= (int64_t(M) * size <= kSms ? kAloneVecs : kSharedVecs);
    void (*const kernels[3])(Args) = {sample_kernel<0>, sample_kernel<1>, sample_kernel<2>};
    auto kernel = kernels[type];
    int device = 0;
    cudaError_t st = cudaGetDevice(&device);
    if (st != cudaSuccess) return st;
    if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
    std::atomic<bool>& done = g_attr[type][device];
    if (!done.load(std::memory_order_acquire)) {
        st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Shared)) + kAloneVecs * 16);
        if (st == cudaSuccess) st = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (st != cudaSuccess) return st;
        done.store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(M) * unsigned(size));
    cfg.blockDim = dim3(kThreads);
    a.part_vecs = type == 0 && !a.resident && a.vecs >= kParts * kThreads ? (a.vecs + 32 * kParts - 1) / (32 * kParts) * 32 : 0;
    cfg.dynamicSmemBytes = sizeof(Shared) + (a.resident ? size_t(a.vecs) * 16 : type ? sizeof(Region) : a.part_vecs ? size_t(kCodes) * 16 : 0);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    count_launches(1);
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
