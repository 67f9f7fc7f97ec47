// Token sampling: one token for each row of logits x[0..V), by a given random
// number u in [0, 1).  With w_i = exp((x_i - max x) / T):
//
//   A = tokens with w_i >= min_p                    (min-p)
//   K = the first top_k of A by (x descending, index ascending)
//   P = the smallest prefix of K in that order with mass >= top_p * mass(K)
//   token = the first i, in index order, with  sum_{j <= i, j in P} w_j > u * mass(P)
//
// T = 0 takes the largest logit (lowest index).  The log probability is the
// model's own: x_token - max x - log sum_i exp(x_i - max x), over all tokens.
//
// Exactness.  The nucleus and the draw compare sums of up to 2^19 weights with
// the border between two tokens, where fp32 sums would choose another token
// than the definition once in a few thousand draws.  Weights are therefore
// 64-bit fixed point, w * 2^s with s = min(51, 62 - ceil(log2 V)): each is
// computed in double precision (relative error below 1e-13) and rounded once;
// sums of integers are exact and do not depend on their order, so the same
// inputs give the same token whatever the launch shape.  The exponential is
// table driven (Tang, 1989): 2^-n/64 from a table of 64 values times a Taylor
// polynomial of degree 4 in the remainder.
//
// Layout of the work.  A cluster of 1 to 16 CTAs takes one row: every CTA
// keeps its share of the logits in shared memory, so the row is read from HBM
// once, however many steps the selection takes.  A cut (top-k or top-p) is
// found by histograms over the value range, merged through distributed shared
// memory; the bin that holds the border is ranked exactly when it has few
// tokens, split again when it has many, and resolved by index when all its
// logits are equal.
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
constexpr int kBins = 1024, kCap = 256;
constexpr int kMaxVecs = (kMaxVocab / 4 + 1 + kMaxCluster - 1) / kMaxCluster;       // 16-byte vectors of a CTA
constexpr int kSlabs = (kMaxVecs + kThreads - 1) / kThreads * kWarps;               // (turn, warp) pairs of a CTA
constexpr float kMaxTemperature = 1e30f;
constexpr uint32_t kFlagNonfinite = 1, kFlagParameter = 2, kFlagNothingLeft = 4;

struct Args {
    const void* logits;
    int64_t stride;  // values between rows
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t* top_k;
    int32_t* tokens;
    float* logprobs;
    uint32_t* flags;
    int vocab, vecs;  // vecs: 16-byte vectors of the row that one CTA keeps
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
    static constexpr uint32_t kNone = 0xff800000u;
    static constexpr float kLowest = -FLT_MAX;
};

struct Pair {
    u64 a, b;
};

// The search of a cut by value ranges.
struct Search {
    u64 mass[kBins], tmass[kBins];       // this CTA's histogram, the row's
    uint32_t cnt[kBins], tcnt[kBins];
    u64 gw[kCap];
    float lv[kCap], gv[kCap];            // candidates of this CTA, of the row
    int li[kCap], gi[kCap];
    uint32_t ln;
};

// The value histogram of a bf16 row (see value_row).
constexpr int kCodes = 19 * 128;                              // magnitudes from 2^-12 up to 128
constexpr int kTinyBin = kCodes, kValueBins = 2 * kCodes + 1;  // by value, largest first; zero and below 2^-12 between
constexpr int kPerThread = (kValueBins + kThreads - 1) / kThreads, kTinyCap = 64;
struct Values {
    uint32_t own[kValueBins];                      // by code: positive, negative, tiny
    uint32_t all[kPerThread * kThreads];           // the row's, by value
    float tiny[kTinyCap];                          // this CTA's tiny logits
    u64 tiny_mass[kMaxCluster];                    // pushed
    uint32_t tiny_n;
};

struct Shared {
    union {
        Search search;
        Values values;
    };
    double pow64[64];                    // 2^(-j/64)
    Pair slot[2][kMaxCluster];           // pushed by every CTA of the cluster in turn
    u64 slab[kSlabs];                    // kept mass of each (turn, warp) in index order
    Pair red[kWarps];
    u64 bound[2];
    int found, found_bin;
};

__device__ __forceinline__ float as_float(u64 v) { return __uint_as_float(uint32_t(v)); }
__device__ __forceinline__ u64 as_bits(float v) { return __float_as_uint(v); }

// What every thread of a row's cluster knows.
template <int TY>
struct Row {
    using El = Elem<TY>;
    Shared& sh;
    const uint4* data;  // this CTA's vectors
    int nvec, first;    // first: index of slot 0 (below 0 where the row starts inside a vector)
    int rank, size, parity;
    float top;          // the largest logit
    double step;        // 64 log2(e) / T
    int frac;           // s of the fixed point
    bool count_mode;    // u = 0: any token of positive weight counts as one
    float cut_v;        // kept: x > cut_v, or x == cut_v and index <= cut_i
    int cut_i;

    __device__ __forceinline__ bool kept(float x, int slot) const {
        return x > cut_v || (x == cut_v && first + slot <= cut_i);
    }

    template <class F>
    __device__ __forceinline__ void each(F f) const {
        for (int v = threadIdx.x; v < nvec; v += kThreads) {
            float x[El::E];
            El::unpack(data[v], x);
#pragma unroll
            for (int e = 0; e < El::E; ++e) f(x[e], v * El::E + e);
        }
    }

    __device__ __forceinline__ u64 weight(float x) const {
        const double y = __dmul_rn(__dsub_rn(double(top), double(x)), step);
        if (count_mode) return y < 64.0 * 1074.0 ? 1 : 0;
        if (!(y < 64.0 * (frac + 1))) return 0;  // below half a unit (and -inf)
        const double shifted = __dadd_rn(y, 0x1.8p52);
        const int n = __double2loint(shifted);
        const double f = __dsub_rn(y, __dsub_rn(shifted, 0x1.8p52));
        constexpr double a = 0.69314718055994530942 / 64;
        double p = __fma_rn(f, a * a * a * a / 24, -a * a * a / 6);
        p = __fma_rn(p, f, a * a / 2);
        p = __fma_rn(p, f, -a);
        p = __fma_rn(p, f, 1.0);
        const double v = __dmul_rn(sh.pow64[n & 63], p);
        const double scaled = __hiloint2double(__double2hiint(v) + ((frac - (n >> 6)) << 20), __double2loint(v));
        return u64(__double_as_longlong(__dadd_rn(scaled, 0x1p52))) & 0xfffffffffffffull;
    }

    // Everyone's pair, in rank order, after all have pushed theirs.  The two
    // buffers alternate: a CTA writes a buffer again only after a later
    // exchange, which its readers join when they have read it.
    __device__ const Pair* exchange(const Pair& mine) {
        Pair* box = sh.slot[parity];
        auto cluster = cg::this_cluster();
        if (int(threadIdx.x) < size) *cluster.map_shared_rank(box + rank, threadIdx.x) = mine;
        cluster.sync();
        parity ^= 1;
        return box;
    }
};

template <class Op>
__device__ __forceinline__ Pair block_reduce(Shared& sh, Pair v, Op op) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const Pair o{__shfl_xor_sync(0xffffffffu, v.a, d), __shfl_xor_sync(0xffffffffu, v.b, d)};
        v = op(v, o);
    }
    __syncthreads();  // red may still be read from the call before
    if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh.red[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v = op(v, sh.red[w]);
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
__device__ __forceinline__ u64 block_exclusive(Shared& sh, u64 v) {
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

// The smallest prefix of the kept tokens, by (value, index), that has `k`
// tokens (MASS false) or `share` / 2^64 of their mass, becomes the kept set.
// Every CTA of the cluster takes the same decisions from the same merged sums.
template <int TY, bool MASS>
__device__ void cut_row(Row<TY>& r, float low, u64 k, u64 share) {
    Shared& sh = r.sh;
    auto cluster = cg::this_cluster();
    const int per = kBins / r.size;  // bins that one CTA merges
    float hi = r.top, lo = low;
    u64 base = 0, target = k;
    for (bool first_level = true;; first_level = false) {
        const float scale = __fdiv_rn(float(kBins), __fsub_rn(hi, lo));
        auto bin = [&](float x) { return max(0, min(kBins - 1, __float2int_rz(__fmul_rn(__fsub_rn(hi, x), scale)))); };
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            sh.search.cnt[b] = 0;
            if (MASS) sh.search.mass[b] = 0;
        }
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
        r.each([&](float x, int slot) {
            if (x >= lo && x <= hi && r.kept(x, slot)) {
                const int b = bin(x);
                atomicAdd(&sh.search.cnt[b], 1u);
                if (MASS) atomicAdd(&sh.search.mass[b], r.weight(x));
            }
        });
        cluster.sync();  // also: nobody reads the list of a search before this one any more
        if (threadIdx.x == 0) sh.search.ln = 0;
        for (int i = threadIdx.x; i < per; i += kThreads) {
            const int b = r.rank * per + i;
            uint32_t c = 0;
            u64 w = 0;
            for (int q = 0; q < r.size; ++q) {
                c += *cluster.map_shared_rank(&sh.search.cnt[b], q);
                if (MASS) w += *cluster.map_shared_rank(&sh.search.mass[b], q);
            }
            for (int q = 0; q < r.size; ++q) {
                *cluster.map_shared_rank(&sh.search.tcnt[b], q) = c;
                if (MASS) *cluster.map_shared_rank(&sh.search.tmass[b], q) = w;
            }
        }
        cluster.sync();
        // two bins a thread, from the largest values down
        const int b0 = 2 * threadIdx.x;
        const u64 v0 = MASS ? sh.search.tmass[b0] : sh.search.tcnt[b0], v1 = MASS ? sh.search.tmass[b0 + 1] : sh.search.tcnt[b0 + 1];
        const u64 before = block_exclusive(sh, v0 + v1);
        if (first_level) {
            if (threadIdx.x == kThreads - 1) sh.bound[0] = before + v0 + v1;
            __syncthreads();
            const u64 total = sh.bound[0];
            if (MASS)
                target = max(u64(1), __umul64hi(total, share) + (total * share != 0));
            else if (total <= target)
                return;
        }
        const u64 at = base + before;
        if (at < target && target <= at + v0) sh.found_bin = b0, sh.bound[1] = at, sh.found = 1;
        if (at + v0 < target && target <= at + v0 + v1) sh.found_bin = b0 + 1, sh.bound[1] = at + v0, sh.found = 1;
        __syncthreads();
        if (!sh.found) return;  // no mass at all: nothing to cut
        const int border = sh.found_bin;
        const uint32_t n = sh.search.tcnt[border];
        base = sh.bound[1];
        if (n <= uint32_t(kCap)) {
            // rank the border's tokens exactly
            r.each([&](float x, int slot) {
                if (x >= lo && x <= hi && r.kept(x, slot) && bin(x) == border) {
                    const uint32_t at_list = atomicAdd(&sh.search.ln, 1u);
                    if (at_list < uint32_t(kCap)) sh.search.lv[at_list] = x, sh.search.li[at_list] = r.first + slot;
                }
            });
            cluster.sync();
            // every CTA's count, then each thread one candidate of the row
            if (int(threadIdx.x) < r.size)
                sh.slab[threadIdx.x] = *cluster.map_shared_rank(&sh.search.ln, threadIdx.x);
            __syncthreads();
            int from = 0, owner = -1, at_owner = 0;
            for (int q = 0; q < r.size; ++q) {
                const int m = min(int(sh.slab[q]), kCap - from);
                if (int(threadIdx.x) >= from && int(threadIdx.x) < from + m) owner = q, at_owner = threadIdx.x - from;
                from += m;
            }
            if (owner >= 0) {
                sh.search.gv[threadIdx.x] = *cluster.map_shared_rank(&sh.search.lv[at_owner], owner);
                sh.search.gi[threadIdx.x] = *cluster.map_shared_rank(&sh.search.li[at_owner], owner);
            }
            __syncthreads();
            int place = 0;
            float x = 0.f;
            int index = 0;
            const bool mine = int(threadIdx.x) < from;
            if (mine) {
                x = sh.search.gv[threadIdx.x], index = sh.search.gi[threadIdx.x];
                for (int j = 0; j < from; ++j) place += sh.search.gv[j] > x || (sh.search.gv[j] == x && sh.search.gi[j] < index);
                sh.search.gw[place] = MASS ? r.weight(x) : 1;
            }
            __syncthreads();
            const u64 w = int(threadIdx.x) < from ? sh.search.gw[threadIdx.x] : 0;
            const u64 sum = base + block_exclusive(sh, w);
            if (sum < target && target <= sum + w) sh.found_bin = threadIdx.x;  // its place
            __syncthreads();
            const int last = sh.found_bin;
            if (mine && place == last) sh.bound[0] = as_bits(x), sh.bound[1] = u64(uint32_t(index));
            __syncthreads();
            r.cut_v = as_float(sh.bound[0]), r.cut_i = int(uint32_t(sh.bound[1]));
            __syncthreads();
            return;
        }
        // the border's smallest and largest value
        float mn = INFINITY, mx = -INFINITY;
        r.each([&](float x, int slot) {
            if (x >= lo && x <= hi && r.kept(x, slot) && bin(x) == border) mn = fminf(mn, x), mx = fmaxf(mx, x);
        });
        auto range = [](Pair p, Pair q) {
            return Pair{as_bits(fminf(as_float(p.a), as_float(q.a))), as_bits(fmaxf(as_float(p.b), as_float(q.b)))};
        };
        Pair own = block_reduce(sh, Pair{as_bits(mn), as_bits(mx)}, range);
        const Pair* all = r.exchange(own);
        for (int q = 0; q < r.size; ++q) own = range(own, all[q]);
        lo = as_float(own.a), hi = as_float(own.b);
        if (lo < hi) continue;
        // equal logits: the lowest indices are kept
        u64 need = target - base;
        if (MASS) {
            const u64 w = r.weight(hi);
            need = (need + w - 1) / w;
        }
        const int per_thread = (r.nvec * Row<TY>::El::E + kThreads - 1) / kThreads;
        const int s0 = min(int(threadIdx.x) * per_thread, r.nvec * Row<TY>::El::E);
        const int s1 = min(s0 + per_thread, r.nvec * Row<TY>::El::E);
        const auto value = [&](int slot) {
            return Row<TY>::El::one(reinterpret_cast<const char*>(r.data) + size_t(slot) * Row<TY>::El::kBytes);
        };
        u64 ties = 0;
        for (int s = s0; s < s1; ++s) ties += value(s) == hi && r.kept(hi, s);
        const u64 prior = block_exclusive(sh, ties);
        if (threadIdx.x == kThreads - 1) sh.bound[0] = prior + ties;
        __syncthreads();
        all = r.exchange(Pair{sh.bound[0], 0});
        u64 ahead = 0;
        for (int q = 0; q < r.rank; ++q) ahead += all[q].a;
        if (threadIdx.x == 0) sh.found_bin = -1;
        __syncthreads();
        u64 rankth = ahead + prior;
        if (rankth < need && need <= rankth + ties)
            for (int s = s0; s < s1; ++s)
                if (value(s) == hi && r.kept(hi, s) && ++rankth == need) sh.found_bin = r.first + s;
        __syncthreads();
        all = r.exchange(Pair{u64(uint32_t(sh.found_bin)), 0});
        int index = -1;
        for (int q = 0; q < r.size; ++q) index = max(index, int(uint32_t(all[q].a)));
        r.cut_v = hi, r.cut_i = index;
        return;
    }
}

// The kept mass of each (turn, warp) of this CTA into sh.slab, and its sum.
// Vectors v = turn * kThreads + thread of a warp are consecutive in the row,
// so slabs in order are in index order.
template <int TY>
__device__ __forceinline__ u64 vector_mass(const Row<TY>& r, int v, u64 (&w)[Elem<TY>::E]) {
    constexpr int E = Elem<TY>::E;
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = 0;
    if (v < r.nvec) {
        float x[E];
        Elem<TY>::unpack(r.data[v], x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (r.kept(x[e], v * E + e)) w[e] = r.weight(x[e]);
            sum += w[e];
        }
    }
    return sum;
}

template <int TY>
__device__ u64 slab_masses(const Row<TY>& r, int turns) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 mine = 0;
    for (int turn = 0; turn < turns; ++turn) {
        u64 w[Elem<TY>::E];
        u64 sum = vector_mass(r, turn * kThreads + int(threadIdx.x), w);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) r.sh.slab[turn * kWarps + warp] = sum;
        mine += sum;
    }
    return lane == 0 ? mine : 0;
}

// The log probability of a token x: sums of exp(logit - top) over the largest
// logits (`tops` of them) and the others.
struct Partition {
    double tops, others;
    __device__ float of(float x, float top) const {
        return float((double(x) - double(top)) - (log(tops) + log1p(others / tops)));
    }
};

// One warp of the CTA that holds the token: its slab, its lane, its value.
template <int TY>
__device__ void write_token(const Row<TY>& r, const Args& a, int row, u64 ahead, u64 target, int turns,
                            const Partition& z) {
    constexpr int E = Elem<TY>::E;
    const Shared& sh = r.sh;
    const int lane = threadIdx.x & 31;
    const int slabs = turns * kWarps, per_lane = (slabs + 31) / 32;
    int slab = lane * per_lane;
    u64 part = 0;
    for (int i = slab; i < min(slab + per_lane, slabs); ++i) part += sh.slab[i];
    u64 sum = ahead + warp_exclusive(part);
    const bool here = sum <= target && target < sum + part;
    if (here)
        while (sum + sh.slab[slab] <= target) sum += sh.slab[slab++];
    const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    slab = __shfl_sync(0xffffffffu, slab, from), sum = __shfl_sync(0xffffffffu, sum, from);
    u64 w[E];
    const int v = (slab / kWarps) * kThreads + (slab % kWarps) * 32 + lane;
    const u64 vec = vector_mass(r, v, w);
    u64 at = sum + warp_exclusive(vec);
    if (at <= target && target < at + vec) {
        float x[E];
        Elem<TY>::unpack(r.data[v], x);
        bool done = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += w[e];
            if (!done && at > target) {
                a.tokens[row] = r.first + v * E + e;
                if (a.logprobs) a.logprobs[row] = z.of(x[e], r.top);
                done = true;
            }
        }
    }
}

__device__ __forceinline__ Pair add_doubles(Pair p, Pair q) {
    return Pair{u64(__double_as_longlong(__longlong_as_double(p.a) + __longlong_as_double(q.a))),
                u64(__double_as_longlong(__longlong_as_double(p.b) + __longlong_as_double(q.b)))};
}

// The index of this CTA's `nth` token (from 1) whose logit is `value`.
template <int TY>
__device__ int nth_equal(const Row<TY>& r, float value, u64 nth) {
    const int slots = r.nvec * Elem<TY>::E, per_thread = (slots + kThreads - 1) / kThreads;
    const int s0 = min(int(threadIdx.x) * per_thread, slots), s1 = min(s0 + per_thread, slots);
    const auto at = [&](int slot) {
        return Elem<TY>::one(reinterpret_cast<const char*>(r.data) + size_t(slot) * Elem<TY>::kBytes);
    };
    u64 ties = 0;
    for (int s = s0; s < s1; ++s) ties += at(s) == value;
    u64 rankth = block_exclusive(r.sh, ties);
    if (rankth < nth && nth <= rankth + ties)
        for (int s = s0; s < s1; ++s)
            if (at(s) == value && ++rankth == nth) r.sh.found_bin = r.first + s;
    __syncthreads();
    return r.sh.found_bin;
}

// A bf16 row by its values.  A row of 10^5 logits has a few thousand distinct
// values, so counts of each value, an exact histogram over the 4864 codes of
// magnitude 2^-12 to 128, hold everything but the order: masses are counts
// times weights, a cut is a value and a number of equal logits, and only the
// CTA that holds the token goes over its logits again.  One shared-memory
// count a logit replaces a double-precision exponential a logit.  The few
// logits below 2^-12 are kept in a list and weighted one by one.
//
// Returns false, in every CTA alike, where a cut falls among those: the row
// then goes the general way.
__device__ bool value_row(Row<0>& r, const Args& a, int row, float T, int k, float p, float u, float floor_v,
                          bool greedy) {
    Shared& sh = r.sh;
    Values& h = sh.values;
    auto cluster = cg::this_cluster();
    const int tid = threadIdx.x, size = r.size;
    const auto code_of = [](int bin) { return bin < kTinyBin ? kCodes - 1 - bin : bin == kTinyBin ? 2 * kCodes : bin - 1; };
    const auto value_of = [](int bin) {
        const int magnitude = bin < kTinyBin ? kCodes - 1 - bin : bin - 1 - kCodes;
        const float v = __uint_as_float(uint32_t(magnitude + (115 << 7)) << 16);
        return bin < kTinyBin ? v : bin == kTinyBin ? 0.f : -v;
    };
    const int per = (kValueBins + size - 1) / size;
    for (int i = tid; i < per; i += kThreads) {
        const int bin = r.rank * per + i;
        if (bin >= kValueBins) break;
        const int code = code_of(bin);
        uint32_t c = 0;
        for (int q = 0; q < size; ++q) c += *cluster.map_shared_rank(&h.own[code], q);
        for (int q = 0; q < size; ++q) *cluster.map_shared_rank(&h.all[bin], q) = c;
    }
    auto add = [](Pair x, Pair y) { return Pair{x.a + y.a, x.b + y.b}; };
    const u64 own_tiny =
        block_reduce(sh, Pair{tid < int(h.own[2 * kCodes]) ? r.weight(h.tiny[tid]) : 0, 0}, add).a;
    if (tid < size) *cluster.map_shared_rank(&h.tiny_mass[r.rank], tid) = own_tiny;
    cluster.sync();

    // this thread's values, largest first
    const int first = tid * kPerThread;
    uint32_t cnt[kPerThread];
    u64 weight[kPerThread], count = 0, tiny_mass = 0;
    for (int q = 0; q < size; ++q) tiny_mass += h.tiny_mass[q];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const float v = value_of(first + i);
        cnt[i] = v >= floor_v ? h.all[first + i] : 0;
        weight[i] = cnt[i] ? (greedy ? 1 : r.weight(v)) : 0;
        count += cnt[i];
    }
    if (tid == 0) sh.found = 0;
    const bool by_count = greedy || (k > 0 && k < a.vocab);
    const u64 limit = greedy ? 1 : u64(k);
    u64 mass = 0;
    const u64 before = by_count ? block_exclusive(sh, count) : 0;
    u64 seen = before;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
        const int bin = first + i;
        const uint32_t had = cnt[i];
        if (by_count) {
            cnt[i] = seen >= limit ? 0 : uint32_t(min(u64(had), limit - seen));
            if (seen < limit && limit <= seen + had) {
                sh.found = 1, sh.found_bin = bin, sh.bound[1] = limit - seen;
                if (bin == kTinyBin && cnt[i] < had) sh.found = 2;
            }
            seen += had;
        }
        mass += bin == kTinyBin ? (cnt[i] ? tiny_mass : 0) : cnt[i] * weight[i];
    }
    if (p < 1.f && !greedy) {
        const u64 ahead = block_exclusive(sh, mass);
        if (tid == kThreads - 1) sh.bound[0] = ahead + mass;
        __syncthreads();
        const u64 total = sh.bound[0];
        const bool stuck = sh.found == 2;
        __syncthreads();  // found and bound are written again below
        if (stuck) return false;
        const u64 share = __double2ull_rz(double(p) * 0x1p64);
        const u64 target = max(u64(1), __umul64hi(total, share) + (total * share != 0));
        if (ahead < target && target <= ahead + mass) {
            u64 at = ahead;
#pragma unroll
            for (int i = 0; i < kPerThread; ++i) {
                const int bin = first + i;
                const u64 m = bin == kTinyBin ? (cnt[i] ? tiny_mass : 0) : cnt[i] * weight[i];
                if (at < target && target <= at + m) {
                    sh.found = 1, sh.found_bin = bin;
                    if (bin == kTinyBin)
                        sh.found = 2;
                    else
                        sh.bound[1] = (target - at + weight[i] - 1) / weight[i];
                }
                at += m;
            }
        }
    }
    __syncthreads();
    if (sh.found == 2) return false;
    const int border = sh.found ? sh.found_bin : INT_MAX;
    const u64 ties = sh.bound[1];  // kept of the border's value
    u64 here = 0, mine = 0;        // of that value in this CTA, and of the kept
    if (sh.found) {
        // counts of the border's value in the CTAs before this one
        if (tid < size) sh.slab[tid] = *cluster.map_shared_rank(&h.own[code_of(border)], tid);
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
        if (bin == border)
            mass += mine * (bin == kTinyBin ? 0 : weight[i]);
        else if (bin < border && bin < kValueBins && bin != kTinyBin && weight[i])
            mass += h.own[code_of(bin)] * weight[i];
    }
    if (tid == 0 && border >= kTinyBin && floor_v <= 0.f) mass += own_tiny;
    const Pair own = block_reduce(sh, Pair{mass, 0}, add);
    const Pair* box = r.exchange(own);
    u64 whole = 0, ahead = 0;
    for (int q = 0; q < size; ++q) {
        if (q < r.rank) ahead += box[q].a;
        whole += box[q].a;
    }
    const u64 target = __umul64hi(whole, __double2ull_rz(double(u) * 0x1p64));  // floor(u * mass): token has sum > it
    if (ahead > target || target >= ahead + own.a) return true;

    // The CTA that holds the token.
    r.cut_v = floor_v, r.cut_i = INT_MAX;
    if (floor_v == -INFINITY) r.cut_i = -1;
    if (border != INT_MAX) {
        r.cut_v = value_of(border);
        if (border == kTinyBin)
            r.cut_v = -0x1p-12f, r.cut_i = -1;  // all of the tiny
        else if (mine == here)
            r.cut_i = INT_MAX;
        else
            r.cut_i = mine ? nth_equal(r, r.cut_v, mine) : -1;
    }
    Partition z{1.0, 0.0};
    if (a.logprobs) {
        float others = 0.f, tops = 0.f;
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) {
            const float v = value_of(first + i), c = float(h.all[first + i]);
            if (v == r.top)
                tops += c;
            else if (c > 0.f)
                others = __fmaf_rn(c, expf(__fsub_rn(v, r.top)), others);
        }
        const Pair sums = block_reduce(
            sh, Pair{u64(__double_as_longlong(tops)), u64(__double_as_longlong(others))}, add_doubles);
        z.tops = __longlong_as_double(sums.a), z.others = __longlong_as_double(sums.b);
    }
    const int turns = (a.vecs + kThreads - 1) / kThreads;
    if (greedy) {
        // the border is the largest logit and the token its first
        const int index = nth_equal(r, r.top, 1);
        if (tid == 0) {
            a.tokens[row] = index;
            if (a.logprobs) a.logprobs[row] = z.of(r.top, r.top);
        }
        return true;
    }
    slab_masses(r, turns);
    __syncthreads();
    if (tid < 32) write_token(r, a, row, ahead, target, turns, z);
    return true;
}

// The values of a 16-byte vector of which only a part lies in the row.
template <int TY>
__device__ __forceinline__ uint4 edge_vector(const char* begin, int i0, int vocab) {
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

// One cluster per row.  The barrier of a cluster is the hardware's: all its
// CTAs are resident together and take every barrier, as all decisions that
// lead to one are taken from exchanged values.
template <int TY>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Args a) {
    using El = Elem<TY>;
    constexpr int E = El::E, kBatch = 4;
    extern __shared__ uint4 data[];
    __shared__ Shared sh;
    auto cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int row = blockIdx.x / size, tid = threadIdx.x;

    const float T = a.temperature ? a.temperature[row] : 1.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.uniform[row];
    if (!(T >= 0.f && T <= kMaxTemperature) || !(p >= 0.f) || !(min_p >= 0.f && min_p <= 1.f) ||
        !(u >= 0.f && u < 1.f)) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, kFlagParameter);
        }
        return;
    }
    cluster.barrier_arrive();  // waited for before the first access to another CTA's shared memory
    const bool greedy = T == 0.f || k == 1;

    // this CTA's share of the row: whole 16-byte vectors of memory, values outside the row as -inf
    const char* begin = static_cast<const char*>(a.logits) + int64_t(row) * a.stride * El::kBytes;
    const int lead = int(reinterpret_cast<uintptr_t>(begin) % 16) / El::kBytes;
    const int total_vecs = (lead + a.vocab + E - 1) / E;
    const int v0 = min(rank * a.vecs, total_vecs), nvec = min(a.vecs, total_vecs - v0);
    const uint4* base = reinterpret_cast<const uint4*>(begin - lead * El::kBytes) + v0;
    const int i_first = v0 * E - lead;  // index of the first value
    float top = -INFINITY;
    uint32_t notes = 0;  // 1: NaN or +inf; bf16: 2: 128 or more, 4: -128 or less but not -inf, 8: too many tiny
    for (int b = 0; b == 0 || b < nvec; b += kBatch * kThreads) {
        uint4 q[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = b + j * kThreads + tid, i0 = i_first + v * E;
            if (v < nvec)
                q[j] = i0 >= 0 && i0 + E <= a.vocab ? __ldcs(base + v) : edge_vector<TY>(begin, i0, a.vocab);
        }
        if (b == 0) {
            if (tid < 64) sh.pow64[tid] = exp2(-tid * (1.0 / 64));
            if (TY == 0) {
                for (int i = tid; i < kValueBins; i += kThreads) sh.values.own[i] = 0;
                for (int i = kValueBins + tid; i < kPerThread * kThreads; i += kThreads) sh.values.all[i] = 0;
                if (tid == 0) sh.values.tiny_n = 0;
                __syncthreads();
            }
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int v = b + j * kThreads + tid;
            if (v >= nvec) break;
            data[v] = q[j];
            float x[E];
            El::unpack(q[j], x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                top = fmaxf(top, x[e]);
                if (TY == 0) {
                    const uint32_t bits = __float_as_uint(x[e]) >> 16, magnitude = bits & 0x7fffu;
                    const uint32_t code = magnitude - (115u << 7);
                    if (code < uint32_t(kCodes)) {
                        atomicAdd(&sh.values.own[code + (bits >> 15) * kCodes], 1u);
                    } else if (magnitude < (115u << 7)) {
                        const uint32_t at = atomicAdd(&sh.values.tiny_n, 1u);
                        if (at < uint32_t(kTinyCap)) sh.values.tiny[at] = x[e];
                        else notes |= 8;
                    } else if (!(x[e] < INFINITY)) {
                        notes |= 1;
                    } else if (x[e] != -INFINITY) {
                        notes |= x[e] > 0.f ? 2 : 4;
                    }
                } else if (!(x[e] < INFINITY)) {
                    notes |= 1;
                }
            }
        }
    }

    Row<TY> r{sh, data, nvec, i_first, rank, size, 0};
    auto join = [](Pair x, Pair y) { return Pair{as_bits(fmaxf(as_float(x.a), as_float(y.a))), x.b | y.b}; };
    Pair own = block_reduce(sh, Pair{as_bits(top), notes}, join);
    if (TY == 0 && tid == 0) sh.values.own[2 * kCodes] = min(sh.values.tiny_n, uint32_t(kTinyCap));
    cluster.barrier_wait();
    const Pair* all = r.exchange(own);
    for (int q = 0; q < size; ++q) own = join(own, all[q]);
    top = as_float(own.a), notes = uint32_t(own.b);
    if ((notes & 1) || top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, notes & 1 ? kFlagNonfinite : kFlagNothingLeft);
        }
        return;
    }
    r.top = top;
    r.step = greedy ? 0.0 : 64.0 * 1.4426950408889634074 / double(T);
    r.frac = min(51, 62 - (32 - __clz((a.vocab - 1) | 1)));
    r.count_mode = false;
    // w >= min_p as a comparison of logits, which is exact
    float floor_v = -INFINITY;
    if (min_p > 0.f && !greedy) floor_v = __double2float_ru(double(top) + double(T) * log(double(min_p)));
    if (TY == 0) {
        // Every logit but the tiny ones has a code of its own, or no weight: below -128 that takes 37 T.
        const float heat = greedy ? 1.f : fmaxf(T, 1.f);
        if (!(notes & 10) && top > -128.f && fabsf(top) >= 0x1p-12f && u != 0.f &&
            (!(notes & 4) || top + 128.f >= 37.f * heat) && !(fabsf(floor_v) < 0x1p-12f)) {
            if constexpr (TY == 0)
                if (value_row(r, a, row, T, k, p, u, floor_v, greedy)) return;
        }
        cluster.sync();  // the histogram's memory is used again
    }

    // the smallest logit but -inf and the type's lowest value, which usually masks
    float low = INFINITY;
    r.each([&](float x, int) {
        if (x > El::kLowest) low = fminf(low, x);
    });
    // log sum exp over all tokens: the largest logits counted, the others summed
    Partition z{1.0, 0.0};
    float others = 0.f, equal = 0.f;
    if (a.logprobs)
        r.each([&](float x, int) {
            if (x == top)
                equal += 1.f;
            else
                others += expf(__fsub_rn(x, top));
        });
    auto least = [](Pair x, Pair y) { return Pair{as_bits(fminf(as_float(x.a), as_float(y.a))), 0}; };
    own = block_reduce(sh, Pair{as_bits(low), 0}, least);
    low = as_float(own.a);
    if (a.logprobs) {
        own = block_reduce(sh, Pair{u64(__double_as_longlong(equal)), u64(__double_as_longlong(others))}, add_doubles);
        all = r.exchange(own);
        own = all[0];
        for (int q = 1; q < size; ++q) own = add_doubles(own, all[q]);
        z.tops = __longlong_as_double(own.a), z.others = __longlong_as_double(own.b);
    }

    if (greedy) {
        int index = INT_MAX;
        r.each([&](float x, int slot) {
            if (x == top) index = min(index, r.first + slot);
        });
        auto first = [](Pair x, Pair y) { return Pair{min(x.a, y.a), 0}; };
        own = block_reduce(sh, Pair{u64(index), 0}, first);
        all = r.exchange(own);
        for (int q = 0; q < size; ++q) own = first(own, all[q]);
        if (rank == 0 && tid == 0) {
            a.tokens[row] = int(own.a);
            if (a.logprobs) a.logprobs[row] = z.of(top, top);
        }
        return;
    }

    r.cut_v = floor_v, r.cut_i = min_p > 0.f ? INT_MAX : -1;
    if ((k > 0 && k < a.vocab) || p < 1.f) {
        all = r.exchange(Pair{as_bits(low), 0});
        for (int q = 0; q < size; ++q) low = fminf(low, as_float(all[q].a));
        // The values a cut searches.  Below 746 T under the top every weight is
        // zero in double precision, so the order there never matters; in fixed
        // point that holds from 37 T (2^-53) on.
        if (double(top) - 746.0 * double(T) <= double(El::kLowest)) low = El::kLowest;
    }
    if (k > 0 && k < a.vocab) {
        const float floor_k = fmaxf(low, __double2float_rd(double(top) - 746.0 * double(T)));
        cut_row<TY, false>(r, fminf(top, fmaxf(floor_k, r.cut_v)), u64(k), 0);
    }
    if (p < 1.f) {
        const float floor_p = fmaxf(low, __double2float_rd(double(top) - 37.0 * double(T)));
        cut_row<TY, true>(r, fminf(top, fmaxf(floor_p, r.cut_v)), 0, __double2ull_rz(double(p) * 0x1p64));
    }

    r.count_mode = u == 0.f;
    const int turns = (a.vecs + kThreads - 1) / kThreads;
    auto add = [](Pair x, Pair y) { return Pair{x.a + y.a, 0}; };
    own = block_reduce(sh, Pair{slab_masses(r, turns), 0}, add);
    all = r.exchange(own);
    u64 whole = 0, ahead = 0;
    for (int q = 0; q < size; ++q) {
        if (q < rank) ahead += all[q].a;
        whole += all[q].a;
    }
    const u64 target = __umul64hi(whole, __double2ull_rz(double(u) * 0x1p64));  // floor(u * mass): token has sum > it
    if (ahead <= target && target < ahead + own.a && tid < 32) write_token(r, a, row, ahead, target, turns, z);
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
    if (stride < vocab || stride > (int64_t(1) << 40)) return cudaErrorInvalidValue;
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
    // CTAs a row: so many that a share is at most 64 KB (three or more CTAs fit
    // an SM), and with few rows as many as give every SM a share of 8 KB or more.
    int size = 1;
    while (size < kMaxCluster && ((total_vecs + size - 1) / size * 16 > 64 * 1024 ||
                                  (int64_t(M) * size < kSms && total_vecs / size * 16 > 16 * 1024)))
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
    void (*const kernels[3])(Args) = {sample_kernel<0>, sample_kernel<1>, sample_kernel<2>};
    auto kernel = kernels[type];
    int device = 0;
    cudaError_t st = cudaGetDevice(&device);
    if (st != cudaSuccess) return st;
    if (device < 0 || device >= 64) return cudaErrorInvalidDevice;
    std::atomic<bool>& done = g_attr[type][device];
    if (!done.load(std::memory_order_acquire)) {
        st = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMaxVecs + 1) * 16);
        if (st == cudaSuccess) st = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (st != cudaSuccess) return st;
        done.store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(M) * unsigned(size));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = size_t(a.vecs) * 16;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    count_launches(1);
    return cudaLaunchKernelEx(&cfg, kernel, a);
}
