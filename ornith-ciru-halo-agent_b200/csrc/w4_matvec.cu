// Matrix-vector products of 1 to 16 rows with 4-bit weights and group scales:
//
//   out[m][n] = sum_g s[n][g] * sum_{k in group g} x[m][k] * (c[n][k] - z[n][g])
//
// codes c and zero points z in 0..15 (z = 8 without zero points), bf16 or fp16
// activations as they are, groups of 32, 64, 128 or 256 values of K.  It stands
// beside the G256 projections for checkpoints in the ordinary 4-bit form (no
// Hadamard rotation, no quantised activations).
//
// Arithmetic.  c - z is an integer of at most 4 bits and a sign, exact in bf16
// and fp16, so every product x * (c - z) is exact in fp32.  A group's products
// (32 to 256, 2 to 16 chained steps) are summed in the tensor core's fp32
// accumulator; each group's sum is scaled and added to the row's fp32 sum with one
// FMA; the only rounding below fp32 is the store in the output's type.
//
// Layout.  A tile is 16 rows of N times 64 values of K = 512 bytes, lane
// l = 4r + t holding 16 of them as four words, one per mma.m16n8k16 step, in
// that instruction's A-fragment order: word w of lane (r, t) covers rows r and
// r + 8 and k = 64c + 32(w / 2) + 8t + 4(w % 2) + {0..3}.  Bits 4j of the two
// half words hold the two values of fragment register j, so (word >> 4j) &
// 0x000f000f is the register up to an exponent.  The order of k inside a step
// is free as long as both operands agree; this one keeps every step inside 32
// consecutive values (the smallest group) and makes a lane's activations for
// two steps 16 consecutive bytes of x.
//
// What bounds it: the stream of the codes, N*K/2 bytes.  One warp reads a tile
// with one 16-byte load per lane, two or four tiles ahead in registers.  248320
// x 2048 with groups of 128 for one bf16 row: 55.8 us, 263 MB at 4.72 TB/s (0.72
// of a copy's measured 6.55); groups of 64 with zero points, 8 rows: 69.0 us,
// 4.09 TB/s (0.62).  There the warps issue 2.3 and 2.5 instructions a clock, most
// of them to take a nibble out and centre it (the integer units are busy for 57 %
// of the time), so loads come no faster; a ring of asynchronous copies in a
// persistent kernel took 71 and 90 us.  12288 x 2048 takes 5.0 us for one row and
// 8.6 for 16 with groups of 32, 2048 x 512 2.1: the launch, and one latency of
// memory for the codes and one for the join.
//
// For more than 16 rows a caller has to come again and the codes are streamed
// again: it is a kernel for decode steps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/ornith_moe_b200.h"
#include "abi_check.h"
#include "nvtx_range.h"

namespace ornith {
void count_launches(int n);

namespace w4 {

constexpr int kMaxM = 16, kMaxK = 16384, kMaxN = 1 << 22, kSms = 148;
constexpr uint32_t kFlagProjection = 4, kFlagStored = 8;  // the dense library's bits

bool shape_ok(int N, int K, int group) {
    return N > 0 && N <= kMaxN && K > 0 && K <= kMaxK && (group == 32 || group == 64 || group == 128 || group == 256) &&
           K % group == 0;
}
inline int row_tiles(int N) { return (N + 15) / 16; }
inline int k_chunks(int K) { return (K + 63) / 64; }

// ---------------------------------------------------------------------------
// layout, once per weight
// ---------------------------------------------------------------------------

// One thread per word of a tile; codes U32[N][K/8], value 8j + d of a row in
// bits 4d of word j.  Rows past N and values past K are code 0: the first are
// not stored, the second never enter a product (see the half-chunk test).
__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const uint32_t* codes, uint32_t* tiles, int N, int K,
                                                            size_t words) {
    const size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= words) return;
    const int chunks = (K + 63) / 64;
    const int w = int(i & 3), lane = int((i >> 2) & 31), r = lane >> 2, t = lane & 3;
    const size_t tile = i >> 7;
    const int c = int(tile % chunks), row = int(tile / chunks) * 16 + r;
    const int k = 64 * c + 32 * (w >> 1) + 8 * t + 4 * (w & 1);
    uint32_t four[2] = {0u, 0u};  // nibbles k..k+3 of rows r and r + 8
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (row + 8 * h < N && k < K)
            four[h] = (codes[size_t(row + 8 * h) * (K / 8) + k / 8] >> (4 * (k & 7))) & 0xffffu;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e)  // e: low or high half of the register
#pragma unroll
        for (int p = 0; p < 2; ++p)  // p: first or second pair of k
#pragma unroll
            for (int h = 0; h < 2; ++h)
                word |= ((four[h] >> (4 * (2 * p + e))) & 15u) << (16 * e + 4 * (2 * p + h));
    tiles[i] = word;
}

// Scales 16-bit [N][K/G] -> [row tile][group][r] pairs (row r, row r + 8);
// zero points u8 likewise, a pair in two bytes.
__global__ __launch_bounds__(256) void w4_pack_meta_kernel(const uint16_t* scales, const uint8_t* zeros,
                                                           uint32_t* tile_scales, uint16_t* tile_zeros, int N,
                                                           int groups, size_t pairs) {
    const size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= pairs) return;
    const int r = int(i & 7);
    const size_t tg = i >> 3;
    const int g = int(tg % groups), row = int(tg / groups) * 16 + r;
    uint32_t s = 0, z = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (row + 8 * h < N) {
            const size_t at = size_t(row + 8 * h) * groups + g;
            s |= uint32_t(scales[at]) << (16 * h);
            if (zeros) z |= (zeros[at] & 15u) << (8 * h);
        }
    tile_scales[i] = s;
    if (zeros) tile_zeros[i] = uint16_t(z);
}

// ---------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------

struct Args {
    const void* x;
    int64_t x_stride;  // values between rows of x
    const uint4* tiles;
    const uint32_t* scales;
    const uint16_t* zeros;  // pairs of bytes
    void* out;
    uint32_t* flags;
    // per_warp: chunks of one warp, a multiple of a group's; split: warps that share a row tile
    int M, N, K, chunks, groups, per_warp, split, out_f32;
};

// A fragment register as the codes' exponent trick leaves it, 128 + c (bf16) or
// 1024 + c (fp16) in each half, and the exact step down to c - z: one FMA with
// one and -(128 + z) or -(1024 + z).
template <bool F16>
struct Num {
    static constexpr uint32_t kMagic = F16 ? 0x64006400u : 0x43004300u;
    static constexpr uint32_t kOne = F16 ? 0x3c003c00u : 0x3f803f80u;
    static constexpr uint32_t kBias = F16 ? 0xe4u : 0xc3u;  // high byte of -(1024 + z), -(128 + z)
    // -(1024 + z) or -(128 + z) in both halves, z the low (half 0) or high byte of a pair
    static __device__ __forceinline__ uint32_t bias(uint32_t pair, int half) {
        return __byte_perm(pair, kBias, half ? 0x4141 : 0x4040);
    }
    // (v & mask) | magic in one instruction
    static __device__ __forceinline__ uint32_t nibbles(uint32_t v) {
        uint32_t d;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(v), "r"(0x000f000fu), "r"(kMagic));
        return d;
    }
    static __device__ __forceinline__ uint32_t centred(uint32_t v, uint32_t bias) {
        uint32_t d;
        if (F16)
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(kOne), "r"(bias));
        else
            asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(kOne), "r"(bias));
        return d;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                               bool opens) {
        const float c[4] = {opens ? 0.f : d[0], opens ? 0.f : d[1], opens ? 0.f : d[2], opens ? 0.f : d[3]};
        if (F16)
            asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                "{%10,%11,%12,%13};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
                  "f"(c[3]));
        else
            asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                "{%10,%11,%12,%13};"
                : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
                  "f"(c[3]));
    }
};

template <bool F16>
__device__ __forceinline__ float scale_value(uint32_t bits16) {
    return F16 ? __half2float(__ushort_as_half(uint16_t(bits16))) : __uint_as_float(bits16 << 16);
}

// Streamed once: do not keep the codes in L1.
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// `split` warps of a CTA (a power of two) share TILES row tiles, each with a
// range of their chunks, and join their sums through shared memory.  MT: tiles
// of 8 activation rows; S16: fp16 scales.  Rows past M repeat the last one:
// columns of the product are independent and theirs are not stored.
//
// CTAs of four warps and at least 20 warps on an SM where a warp takes two row
// tiles: 68 us for 8 rows of the head, against 78 with eight warps to a CTA
// and 94 with registers cut for 28 warps.
template <int TILES>
constexpr int kWarps = TILES == 2 ? 4 : 8;
template <bool F16, bool S16, int MT, bool ZP, int GROUP, int TILES>
__global__ __launch_bounds__(kWarps<TILES> * 32, TILES == 2 ? 5 : 3) void w4_matvec_kernel(const Args a) {
    constexpr int kThreads = kWarps<TILES> * 32;
    constexpr int kRuns = GROUP == 32 ? 2 : 1;             // groups in a chunk
    constexpr int kSpan = GROUP < 64 ? 1 : GROUP / 64;     // chunks of a group
    // Chunks in flight.  Registers, and with them warps, count for more than depth where a warp
    // holds two tiles of rows or of N: 2 against 4 took 76 us against 85 for 8 rows of the head.
    constexpr int kAhead = (MT * TILES > 1 || GROUP == 32) && kSpan <= 2 ? 2 : 4;
    constexpr int kMeta = kAhead / kSpan;                  // scales in flight, per run
    __shared__ float joined[kWarps<TILES>][TILES][16][8 * MT + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int part = warp & (a.split - 1);
    const int per_cta = kWarps<TILES> / a.split;  // warps of different row tiles
    const int row_tile = (blockIdx.x * per_cta + warp / a.split) * TILES, row_tiles = (a.N + 15) / 16;
    const int first = part * a.per_warp;
    int left = row_tile < row_tiles ? min(a.per_warp, a.chunks - first) : 0;
    float acc[TILES][MT][4];
#pragma unroll
    for (int q = 0; q < TILES; ++q)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[q][i][j] = 0.f;

    if (left > 0) {
        const uint4* tile[TILES];
        const uint32_t* scale[TILES];
        const uint16_t* zero[TILES];
#pragma unroll
        for (int q = 0; q < TILES; ++q) {
            const int of = min(row_tile + q, row_tiles - 1);  // an odd last tile is computed twice, stored once
            tile[q] = a.tiles + (size_t(of) * a.chunks + first) * 32 + lane;
            const size_t meta = (size_t(of) * a.groups + first / kSpan * kRuns) * 8 + r;
            scale[q] = a.scales + meta;
            zero[q] = ZP ? a.zeros + meta : nullptr;
        }
        const uint16_t* x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
            x[i] = static_cast<const uint16_t*>(a.x) + min(8 * i + r, a.M - 1) * a.x_stride + 64 * first + 8 * t;
        // a K of 32 more than a multiple of 64 ends in half a chunk, without the second group
        int halves = GROUP == 32 ? a.K / 32 - 2 * first : 0;
        uint4 code[TILES][kAhead];
        uint32_t sc[TILES][kMeta][kRuns], zp[TILES][kMeta][kRuns];
        // chunk d of the next kAhead, `at` chunks further on; the first chunk of a group brings its scale
        auto fetch = [&](int d, int at) {
#pragma unroll
            for (int q = 0; q < TILES; ++q) code[q][d] = load_stream(tile[q] + (at + d) * 32);
            if (d % kSpan == 0) {
#pragma unroll
                for (int h = 0; h < kRuns; ++h)
                    if (h == 0 || halves > 2 * (at + d) + h) {
                        const int g = (at + d) / kSpan * kRuns + h;
#pragma unroll
                        for (int q = 0; q < TILES; ++q) {
                            sc[q][d / kSpan][h] = __ldg(scale[q] + g * 8);
                            if (ZP) zp[q][d / kSpan][h] = __ldg(zero[q] + g * 8);
                        }
                    }
            }
        };
#pragma unroll
        for (int d = 0; d < kAhead; ++d)
            if (d < left) fetch(d, 0);
        float run[TILES][MT][4];
        while (left > 0) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                if (d >= left) break;
                uint4 b[2][MT];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        if (h == 0 || GROUP != 32 || halves > 2 * d + h)
                            b[h][i] = __ldg(reinterpret_cast<const uint4*>(x[i] + 64 * d + 32 * h));
                uint4 word[TILES];
                uint32_t s2[TILES][kRuns], bias[TILES][kRuns][2];
#pragma unroll
                for (int q = 0; q < TILES; ++q) {
                    word[q] = code[q][d];
#pragma unroll
                    for (int h = 0; h < kRuns; ++h) {
                        s2[q][h] = sc[q][d / kSpan][h];
                        const uint32_t z = ZP ? zp[q][d / kSpan][h] : 0x808u;
                        bias[q][h][0] = Num<F16>::bias(z, 0), bias[q][h][1] = Num<F16>::bias(z, 1);
                    }
                }
                // the group's scale is still needed by its later chunks: fetch after its last
                if (d % kSpan == kSpan - 1) {
#pragma unroll
                    for (int e = d - kSpan + 1; e <= d; ++e)
                        if (left > kAhead + e) fetch(e, kAhead);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (GROUP == 32 && h == 1 && halves <= 2 * d + 1) break;  // the same for the whole warp
                    const int g = kRuns == 2 ? h : 0;
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int q = 0; q < TILES; ++q) {
                            const uint32_t w = h ? (p ? word[q].w : word[q].z) : (p ? word[q].y : word[q].x);
                            uint32_t frag[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                frag[j] = Num<F16>::centred(Num<F16>::nibbles(w >> (4 * j)), bias[q][g][j & 1]);
                            const bool opens = p == 0 && (kRuns == 2 || (h == 0 && d % kSpan == 0));
#pragma unroll
                            for (int i = 0; i < MT; ++i)
                                Num<F16>::mma(run[q][i], frag, p ? b[h][i].z : b[h][i].x, p ? b[h][i].w : b[h][i].y,
                                              opens);
                        }
                    if (kRuns == 2 || (h == 1 && d % kSpan == kSpan - 1)) {
#pragma unroll
                        for (int q = 0; q < TILES; ++q) {
                            const float lo = scale_value<S16>(s2[q][g] & 0xffffu);
                            const float hi = scale_value<S16>(s2[q][g] >> 16);
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                acc[q][i][0] = __fmaf_rn(lo, run[q][i][0], acc[q][i][0]);
                                acc[q][i][1] = __fmaf_rn(lo, run[q][i][1], acc[q][i][1]);
                                acc[q][i][2] = __fmaf_rn(hi, run[q][i][2], acc[q][i][2]);
                                acc[q][i][3] = __fmaf_rn(hi, run[q][i][3], acc[q][i][3]);
                            }
                        }
                    }
                }
            }
            left -= kAhead, halves -= 2 * kAhead;
#pragma unroll
            for (int q = 0; q < TILES; ++q) {
                tile[q] += kAhead * 32, scale[q] += kMeta * kRuns * 8;
                if (ZP) zero[q] += kMeta * kRuns * 8;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) x[i] += kAhead * 64;
        }
    }
#pragma unroll
    for (int q = 0; q < TILES; ++q)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                joined[warp][q][r + 8 * (j >> 1)][8 * i + 2 * t + (j & 1)] = acc[q][i][j];
    __syncthreads();
    uint32_t fault = 0;
    const int rows = 16 * TILES * per_cta;  // rows of N of this CTA
    for (int i = threadIdx.x; i < rows * a.M; i += kThreads) {
        const int m = i / rows, row = i % rows, n = blockIdx.x * rows + row;
        if (n >= a.N) continue;
        float v = 0.f;
        for (int p = 0; p < a.split; ++p)
            v = __fadd_rn(v, joined[row / (16 * TILES) * a.split + p][row / 16 % TILES][row & 15][m]);
        if (!isfinite(v)) fault |= kFlagProjection;
        const size_t at = size_t(m) * a.N + n;
        if (a.out_f32) {
            static_cast<float*>(a.out)[at] = v;
        } else if (F16) {
            const __half h = __float2half_rn(v);
            if (!isfinite(__half2float(h))) fault |= kFlagStored;
            static_cast<__half*>(a.out)[at] = h;
        } else {
            const __nv_bfloat16 h = __float2bfloat16_rn(v);
            if (!isfinite(__bfloat162float(h))) fault |= kFlagStored;
            static_cast<__nv_bfloat16*>(a.out)[at] = h;
        }
    }
    if (fault) atomicOr(a.flags, fault);
}

template <bool F16, bool S16, int MT, bool ZP, int TILES>
void launch(const Args& a, int group, int blocks, cudaStream_t stream) {
    auto* kernel = group == 32    ? w4_matvec_kernel<F16, S16, MT, ZP, 32, TILES>
                   : group == 64  ? w4_matvec_kernel<F16, S16, MT, ZP, 64, TILES>
                   : group == 128 ? w4_matvec_kernel<F16, S16, MT, ZP, 128, TILES>
                                  : w4_matvec_kernel<F16, S16, MT, ZP, 256, TILES>;
    kernel<<<blocks, kWarps<TILES> * 32, 0, stream>>>(a);
}

}  // namespace w4
}  // namespace ornith

using namespace ornith;

extern "C" cudaError_t ornith_moe_b200_w4_pack(const void* codes, const void* scales, const void* zeros, void* tiles,
                                               void* tile_scales, void* tile_zeros, int N, int K, int group,
                                               cudaStream_t stream) {
    using namespace w4;
    if (!shape_ok(N, K, group) || (zeros == nullptr) != (tile_zeros == nullptr)) return cudaErrorInvalidValue;
    const int groups = K / group;
    const size_t words = size_t(row_tiles(N)) * k_chunks(K) * 128, pairs = size_t(row_tiles(N)) * groups * 8;
    const void* const ptr[5] = {codes, scales, tiles, tile_scales, nullptr};
    const size_t size[5] = {size_t(N) * K / 2, size_t(N) * groups * 2, words * 4, pairs * 4, 0};
    const uintptr_t align[5] = {4, 2, 16, 4, 1};
    if (!buffers_ok(ptr, size, align, 2, 4)) return cudaErrorInvalidValue;
    if (zeros) {
        const void* const zptr[6] = {codes, scales, zeros, tiles, tile_scales, tile_zeros};
        const size_t zsize[6] = {size[0], size[1], size_t(N) * groups, size[2], size[3], pairs * 2};
        const uintptr_t zalign[6] = {4, 2, 1, 16, 4, 2};
        if (!buffers_ok(zptr, zsize, zalign, 3)) return cudaErrorInvalidValue;
    }
    count_launches(2);
    w4_pack_codes_kernel<<<unsigned((words + 255) / 256), 256, 0, stream>>>(static_cast<const uint32_t*>(codes),
                                                                            static_cast<uint32_t*>(tiles), N, K, words);
    cudaError_t st = cudaGetLastError();
    if (st != cudaSuccess) return st;
    w4_pack_meta_kernel<<<unsigned((pairs + 255) / 256), 256, 0, stream>>>(
        static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), static_cast<uint32_t*>(tile_scales),
        static_cast<uint16_t*>(tile_zeros), N, groups, pairs);
    return cudaGetLastError();
}

extern "C" cudaError_t ornith_moe_b200_w4_launch(const void* x, int64_t x_stride, int x_type, const void* tiles,
                                                 const void* tile_scales, int scale_type, const void* tile_zeros,
                                                 void* out, int out_type, void* flags, int M, int N, int K, int group,
                                                 cudaStream_t stream) {
    using namespace w4;
    if (!shape_ok(N, K, group) || M < 0 || M > kMaxM || x_type < 0 || x_type > 1 || scale_type < 0 || scale_type > 1 ||
        (out_type != x_type && out_type != 2))
        return cudaErrorInvalidValue;
    if (M == 0) return cudaSuccess;
    // every row of x starts on 16 bytes and rows do not overlap; the stride of a single row is not used
    if (x_stride < K || x_stride % 8 || x_stride > (int64_t(1) << 40)) {
        if (M != 1) return cudaErrorInvalidValue;
        x_stride = 0;
    }
    const int groups = K / group;
    const size_t pairs = size_t(row_tiles(N)) * groups * 8;
    const void* const ptr[6] = {x, tiles, tile_scales, tile_zeros, out, flags};
    const size_t size[6] = {(size_t(M - 1) * size_t(x_stride) + size_t(K)) * 2, size_t(row_tiles(N)) * k_chunks(K) * 512,
                            pairs * 4, pairs * 2, size_t(M) * N * (out_type == 2 ? 4 : 2), 4};
    const uintptr_t align[6] = {16, 16, 4, 2, uintptr_t(out_type == 2 ? 4 : 2), 4};
    if (!buffers_ok(ptr, size, align, 4, 3)) return cudaErrorInvalidValue;  // zero points may be null
    NvtxRange range("ornith.w4");
    Args a{};
    a.x = x, a.x_stride = x_stride;
    a.tiles = static_cast<const uint4*>(tiles);
    a.scales = static_cast<const uint32_t*>(tile_scales);
    a.zeros = static_cast<const uint16_t*>(tile_zeros);
    a.out = out, a.flags = static_cast<uint32_t*>(flags);
    a.M = M, a.N = N, a.K = K, a.chunks = k_chunks(K), a.groups = groups;
    a.out_f32 = out_type == 2;
    const int span = group < 64 ? 1 : group / 64, units = (a.chunks + span - 1) / span;
    // Row tiles of a warp: two share its activations where that leaves 16 warps on each SM.  248320 x 2048: 55.3 us
    // for one row and 67.4 for 8 (57.3 and 84.6 with one tile); below the limit, 65536 x 2048 takes 18.2 us with one
    // tile and 19.8 with two, 32768 x 2048 for 8 rows 11.2 and 12.2.
    const int tiles_each = row_tiles(N) >= 2 * kSms * 16 ? 2 : 1, sets = (row_tiles(N) + tiles_each - 1) / tiles_each;
    const int warps = tiles_each == 2 ? kWarps<2> : kWarps<1>;
    // Warps that share row tiles: as few as keep 16 warps on each SM.  12288 x 2048 takes 5.0 us for one row and 7.0
    // for 16; 6.4 and 9.0 with 8 warps, 5.6 and 8.1 with 32.
    a.split = 1;
    while (a.split < warps && a.split < units && sets * a.split < kSms * 16) a.split *= 2;
    a.per_warp = (units + a.split - 1) / a.split * span;
    const int per_cta = warps / a.split, blocks = (sets + per_cta - 1) / per_cta;
    count_launches(1);
    using Launch = void (*)(const Args&, int, int, cudaStream_t);
#define ORNITH_W4(F16, S16, MT)                                              \
    {{launch<F16, S16, MT, false, 1>, launch<F16, S16, MT, false, 2>}, \
     {launch<F16, S16, MT, true, 1>, launch<F16, S16, MT, true, 2>}}
    static constexpr Launch table[2][2][2][2][2] = {
        {{ORNITH_W4(false, false, 1), ORNITH_W4(false, false, 2)}, {ORNITH_W4(false, true, 1), ORNITH_W4(false, true, 2)}},
        {{ORNITH_W4(true, false, 1), ORNITH_W4(true, false, 2)}, {ORNITH_W4(true, true, 1), ORNITH_W4(true, true, 2)}}};
#undef ORNITH_W4
    table[x_type][scale_type][M > 8][tile_zeros != nullptr][tiles_each - 1](a, group, blocks, stream);
    return cudaGetLastError();
}
