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

struct Shared {
    u64 mass[kBins], tmass[kBins];       // this CTA's histogram, the row's
    uint32_t cnt[kBins], tcnt[kBins];
    double pow64[64];                    // 2^(-j/64)
    Pair slot[2][kMaxCluster];           // pushed by every CTA of the cluster in turn
    u64 slab[kSlabs];                    // kept mass of each (turn, warp) in index order
    u64 gw[kCap];
    float lv[kCap], gv[kCap];            // candidates of this CTA, of the row
    int li[kCap], gi[kCap];
    Pair red[kWarps];
    u64 bound[2];
    uint32_t ln;
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
            sh.cnt[b] = 0;
            if (MASS) sh.mass[b] = 0;
        }
        if (threadIdx.x == 0) sh.found = 0;
        __syncthreads();
        r.each([&](float x, int slot) {
            if (x >= lo && x <= hi && r.kept(x, slot)) {
                const int b = bin(x);
                atomicAdd(&sh.cnt[b], 1u);
                if (MASS) atomicAdd(&sh.mass[b], r.weight(x));
            }
        });
        cluster.sync();  // also: nobody reads the list of a search before this one any more
        if (threadIdx.x == 0) sh.ln = 0;
        for (int i = threadIdx.x; i < per; i += kThreads) {
            const int b = r.rank * per + i;
            uint32_t c = 0;
            u64 w = 0;
            for (int q = 0; q < r.size; ++q) {
                c += *cluster.map_shared_rank(&sh.cnt[b], q);
                if (MASS) w += *cluster.map_shared_rank(&sh.mass[b], q);
            }
            for (int q = 0; q < r.size; ++q) {
                *cluster.map_shared_rank(&sh.tcnt[b], q) = c;
                if (MASS) *cluster.map_shared_rank(&sh.tmass[b], q) = w;
            }
        }
        cluster.sync();
        // two bins a thread, from the largest values down
        const int b0 = 2 * threadIdx.x;
        const u64 v0 = MASS ? sh.tmass[b0] : sh.tcnt[b0], v1 = MASS ? sh.tmass[b0 + 1] : sh.tcnt[b0 + 1];
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
        const uint32_t n = sh.tcnt[border];
        base = sh.bound[1];
        if (n <= uint32_t(kCap)) {
            // rank the border's tokens exactly
            r.each([&](float x, int slot) {
                if (x >= lo && x <= hi && r.kept(x, slot) && bin(x) == border) {
                    const uint32_t at_list = atomicAdd(&sh.ln, 1u);
                    if (at_list < uint32_t(kCap)) sh.lv[at_list] = x, sh.li[at_list] = r.first + slot;
                }
            });
            cluster.sync();
            int from = 0;
            for (int q = 0; q < r.size; ++q) {
                const int m = min(int(*cluster.map_shared_rank(&sh.ln, q)), kCap - from);
                for (int i = threadIdx.x; i < m; i += kThreads) {
                    sh.gv[from + i] = *cluster.map_shared_rank(&sh.lv[i], q);
                    sh.gi[from + i] = *cluster.map_shared_rank(&sh.li[i], q);
                }
                from += m;
            }
            __syncthreads();
            int place = 0;
            float x = 0.f;
            int index = 0;
            const bool mine = int(threadIdx.x) < from;
            if (mine) {
                x = sh.gv[threadIdx.x], index = sh.gi[threadIdx.x];
                for (int j = 0; j < from; ++j) place += sh.gv[j] > x || (sh.gv[j] == x && sh.gi[j] < index);
                sh.gw[place] = MASS ? r.weight(x) : 1;
            }
            __syncthreads();
            const u64 w = int(threadIdx.x) < from ? sh.gw[threadIdx.x] : 0;
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

// One cluster per row.  The barrier of a cluster is the hardware's: all its
// CTAs are resident together and take every barrier, as all decisions that
// lead to one are taken from exchanged values.
template <int TY>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Args a) {
    using El = Elem<TY>;
    constexpr int E = El::E;
    extern __shared__ uint4 data[];
    __shared__ Shared sh;
    auto cluster = cg::this_cluster();
    const int size = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int row = blockIdx.x / size, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

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
    const bool greedy = T == 0.f || k == 1;

    // this CTA's share of the row: whole 16-byte vectors of memory, values outside the row as -inf
    const char* begin = static_cast<const char*>(a.logits) + int64_t(row) * a.stride * El::kBytes;
    const int lead = int(reinterpret_cast<uintptr_t>(begin) % 16) / El::kBytes;
    const int total_vecs = (lead + a.vocab + E - 1) / E;
    const int v0 = min(rank * a.vecs, total_vecs), nvec = min(a.vecs, total_vecs - v0);
    const char* base = begin - lead * El::kBytes;
    float top = -INFINITY, low = INFINITY;
    bool bad = false;
    for (int v = tid; v < nvec; v += kThreads) {
        const int i0 = (v0 + v) * E - lead;  // index of the vector's first value
        uint4 q;
        if (i0 >= 0 && i0 + E <= a.vocab) {
            q = __ldcs(reinterpret_cast<const uint4*>(base) + v0 + v);
        } else {
            q = make_uint4(El::kNone, El::kNone, El::kNone, El::kNone);
            data[v] = q;
            for (int e = 0; e < E; ++e)
                if (i0 + e >= 0 && i0 + e < a.vocab) {
                    if (El::kBytes == 2)
                        reinterpret_cast<uint16_t*>(data + v)[e] =
                            reinterpret_cast<const uint16_t*>(begin)[i0 + e];
                    else
                        reinterpret_cast<uint32_t*>(data + v)[e] =
                            reinterpret_cast<const uint32_t*>(begin)[i0 + e];
                }
            q = data[v];
        }
        data[v] = q;
        float x[E];
        El::unpack(q, x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            bad |= !(x[e] < INFINITY);
            top = fmaxf(top, x[e]);
            if (x[e] > El::kLowest) low = fminf(low, x[e]);
        }
    }
    if (tid < 64) sh.pow64[tid] = exp2(-tid * (1.0 / 64));

    Row<TY> r{sh, data, nvec, v0 * E - lead, rank, size, 0};
    auto span = [](Pair p, Pair q) {
        return Pair{as_bits(fmaxf(as_float(p.a), as_float(q.a))) | ((p.a | q.a) & (1ull << 32)),
                    as_bits(fminf(as_float(p.b), as_float(q.b)))};
    };
    Pair own = block_reduce(sh, Pair{as_bits(top) | (u64(bad) << 32), as_bits(low)}, span);
    cluster.sync();  // every CTA of the cluster runs: its shared memory may be written
    const Pair* all = r.exchange(own);
    for (int q = 0; q < size; ++q) own = span(own, all[q]);
    top = as_float(own.a), low = as_float(own.b), bad = own.a >> 32;
    if (bad || top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            a.tokens[row] = -1;
            if (a.logprobs) a.logprobs[row] = NAN;
            atomicOr(a.flags, bad ? kFlagNonfinite : kFlagNothingLeft);
        }
        return;
    }
    r.top = top;

    // log sum exp over all tokens: the largest logits counted, the others summed
    double others = 0.0, tops = 0.0;
    if (a.logprobs) {
        float sum = 0.f, equal = 0.f;
        r.each([&](float x, int) {
            if (x == top)
                equal += 1.f;
            else
                sum += expf(__fsub_rn(x, top));
        });
        auto add = [](Pair p, Pair q) {
            return Pair{u64(__double_as_longlong(__longlong_as_double(p.a) + __longlong_as_double(q.a))),
                        u64(__double_as_longlong(__longlong_as_double(p.b) + __longlong_as_double(q.b)))};
        };
        own = block_reduce(sh, Pair{u64(__double_as_longlong(sum)), u64(__double_as_longlong(equal))}, add);
        all = r.exchange(own);
        for (int q = 0; q < size; ++q)
            others += __longlong_as_double(all[q].a), tops += __longlong_as_double(all[q].b);
    }
    auto answer = [&](int index, float x) {
        a.tokens[row] = index;
        if (a.logprobs) a.logprobs[row] = float((double(x) - double(top)) - (log(tops) + log1p(others / tops)));
    };

    if (greedy) {
        int index = INT_MAX;
        r.each([&](float x, int slot) {
            if (x == top) index = min(index, r.first + slot);
        });
        auto least = [](Pair p, Pair q) { return Pair{min(p.a, q.a), 0}; };
        own = block_reduce(sh, Pair{u64(index), 0}, least);
        all = r.exchange(own);
        for (int q = 0; q < size; ++q) own = least(own, all[q]);
        if (rank == 0 && tid == 0) answer(int(own.a), top);
        return;
    }

    r.step = 64.0 * 1.4426950408889634074 / double(T);
    r.frac = min(51, 62 - (32 - __clz(a.vocab - 1 | 1)));
    r.count_mode = false;
    r.cut_v = -INFINITY, r.cut_i = -1;
    if (min_p > 0.f) {
        // w >= min_p as a comparison of logits, which is exact
        r.cut_v = __double2float_ru(double(top) + double(T) * log(double(min_p)));
        r.cut_i = INT_MAX;
    }
    // The values a cut searches.  Below 746 T under the top every weight is zero
    // in double precision, so the order there never matters; in fixed point
    // that holds from 37 T (2^-53) on.  Above `low` lies every logit but -inf
    // and the type's lowest value, which usually masks.
    if (double(top) - 746.0 * double(T) <= double(El::kLowest)) low = El::kLowest;
    if (k > 0 && k < a.vocab) {
        const float floor_v = fmaxf(low, __double2float_rd(double(top) - 746.0 * double(T)));
        cut_row<TY, false>(r, fminf(top, fmaxf(floor_v, r.cut_v)), u64(k), 0);
    }
    if (p < 1.f) {
        const float floor_v = fmaxf(low, __double2float_rd(double(top) - 37.0 * double(T)));
        cut_row<TY, true>(r, fminf(top, fmaxf(floor_v, r.cut_v)), 0, __double2ull_rz(double(p) * 0x1p64));
    }

    // The draw.  Vectors v = turn * kThreads + thread of a warp are consecutive
    // in the row, so (turn, warp) sums in order are sums in index order.
    r.count_mode = u == 0.f;
    const int turns = (a.vecs + kThreads - 1) / kThreads;
    auto vector_mass = [&](int v, u64 (&w)[E]) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = 0;
        if (v < nvec) {
            float x[E];
            El::unpack(data[v], x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (r.kept(x[e], v * E + e)) w[e] = r.weight(x[e]);
                sum += w[e];
            }
        }
        return sum;
    };
    u64 mine = 0;
    for (int turn = 0; turn < turns; ++turn) {
        u64 w[E];
        u64 sum = vector_mass(turn * kThreads + tid, w);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) sh.slab[turn * kWarps + warp] = sum;
        mine += sum;
    }
    auto add = [](Pair p, Pair q) { return Pair{p.a + q.a, 0}; };
    own = block_reduce(sh, Pair{lane == 0 ? mine : 0, 0}, add);
    all = r.exchange(own);
    u64 whole = 0, ahead = 0;
    for (int q = 0; q < size; ++q) {
        if (q < rank) ahead += all[q].a;
        whole += all[q].a;
    }
    const u64 target = __umul64hi(whole, __double2ull_rz(double(u) * 0x1p64));  // floor(u * mass): token has sum > it
    if (ahead > target || target >= ahead + own.a || warp != 0) return;
    // this CTA's first warp: the slab, then the lane, then the value
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
    const u64 vec = vector_mass(v, w);
    u64 at = sum + warp_exclusive(vec);
    if (at <= target && target < at + vec) {
        float x[E];
        El::unpack(data[v], x);
        bool done = false;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += w[e];
            if (!done && at > target) {
                answer(r.first + v * E + e, x[e]);
                done = true;
            }
        }
    }
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
