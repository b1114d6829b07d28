// Dense products of few rows (up to 128) on tcgen05: D[m][n] = sum_k A[m][k] B[n][k], stored as out[n][m] (m contiguous), for
//   * 4-bit microscaled operands (kind::mxf4, 2^x scales of 32 elements taken from tensor memory) and 16-bit ones (kind::f16),
//   * weights A whose rows run along K, or (16 bit) along m, so that dx needs no transposed copy,
//   * one A, or two with an accumulator each (gate and up) that the epilogue joins: act(g) * u.
// m is the feature that is contiguous in the output: lane l of TMEM row quarter q holds m = 32 q + l, so that the stores of a column
// are whole 64- or 128-byte lines without a trip through shared memory, a block of 32 features is one warp's column (the epilogue
// can quantise), and few tokens make narrow tiles (n from 16) under full-height ones of weights, whose bytes are what such a product costs.
//
// One CTA: warp 0 moves tiles by TMA through a ring of stages of 128 bytes of K a row, warp 1 issues the MMAs, eight warps read the
// accumulators (two a row quarter).  Few results: a cluster splits K and its CTAs' partial sums are added through distributed shared
// memory in ascending rank order (no workspace, no atomics: the same bits on every run).
//
// What bounds it: the weights' bytes, and for the smallest the launch.  4-bit 65536 x 8192 (285 MB) 16 tokens 47.4 us (6.0 TB/s), 65536 x 4096 8 tokens 26.3
// (5.4); gated bf16, 4 tokens, 4096 -> 10240 (168 MB) 28.8 (5.8; lower tiles that would share the weights evenly over the SMs change nothing); 4-bit
// 4096 x 4096, one token, 4.2 to 4.7 for the 1.4 that its bytes take: about half until the first operands are there, the rest products and the join.
//
// Up to 128 rows, as beyond that the other kernel's tiles are faster.  us a call here / there at 64, 96, 128 tokens: 4-bit 4096 x 4096 5.5 / 9.0, 6.9 / 9.3,
// 7.3 / 9.6; 8192 -> 16384 17.5 / 17.6, 17.5 / 18.0, 18.6 / 18.3; gated bf16 4096 -> 10240 with pre 34.5 / 41.1, 42.6 / 42.3, 46.0 / 43.9; dx of
// 2048 -> 5632, dg and du included, 14.9 / 22.7, 16.3 / 22.8, 18.4 / 22.7.  Accumulators for 16, 32, 64 or 128 rows, the fewest that hold them: up to 64, two blocks share an SM.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "dense_plan.h"
#include "dnb_common.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.cuh"

namespace dnb {
namespace dt {
using namespace tcp;

constexpr int TM = 128;             // rows of A in a tile
constexpr int NTHREADS = 320;
constexpr int EPI_WARPS = 8;
constexpr int kWaitStage = 27, kWaitAcc = 28, kWaitDrain = 29;  // status codes of the waits
// Chunks of K of the longest sum.  A tile's results are waited for while its sum runs, 0.3 to 0.7 us a chunk, and a wait gives up after half a second.
constexpr int kMostChunks = 1 << 19;

enum Act { ACT_NONE = -1, ACT_SILU = 0, ACT_GELU = 1 };

struct Params {
    CUtensorMap a[2], b[2];         // b[1]: of the second pass
    const uint8_t* sa[2];           // scale tiles of A (4 bit)
    const uint8_t* sb;              // and of B
    int M, N, K;
    int passes;                     // 2: the sum goes on over a[1], b[1]
    int splits, chunks, share[9];   // parts of K, in chunks, and where each begins
    int bn;                         // rows of B that are loaded and multiplied: N rounded up to 16
    int idesc_type;                 // 16 bit: 0 fp16, 1 bf16
    int out_type, act;
    void* out;
    uint8_t* out_scales;            // MXFP4 results
    float* pre;                     // gate and up before the activation [2][N][M], or null
    size_t ldo;                     // elements between rows of out
    int* status;
};

// Blocks that share an SM never ask for more tensor memory together than it has (one would wait for the other, and clusters for one another): those
// of half of it or less take over a third of an SM's 228 KB of shared memory, the others too much to stand beside one of those.
constexpr size_t kOneOfTwo = 233472 / 3, kBesideNone = 233472 - kOneOfTwo - 2048;
constexpr int pow2_cols(int c) { return c <= 32 ? 32 : c <= 64 ? 64 : c <= 128 ? 128 : c <= 256 ? 256 : 512; }

template <bool FP4_, int NA_, int BN_, bool AMN_ = false>
struct Cfg {
    static constexpr bool FP4 = FP4_, AMN = AMN_;
    static constexpr int NA = NA_, BN = BN_;
    static constexpr int BK = FP4 ? 256 : 64;               // 128 bytes of a row
    static constexpr int A_BYTES = TM * 128, B_BYTES = BN * 128;
    static constexpr int SFA = FP4 ? 1024 : 0;              // scales of 128 rows x 256 elements
    static constexpr int STAGE = NA * A_BYTES + B_BYTES + (NA + 1) * SFA;
    static constexpr int PER_SM = BN < 128 ? 2 : 1;
    static constexpr int BUDGET = PER_SM == 2 ? 115712 - 1536 : 232448 - 1536;
    static constexpr int FIT = BUDGET / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int ACC = NA * BN;
    static constexpr int SF_COLS = FP4 ? NA * 8 + 8 : 0;   // one of two buffers
    static constexpr int BUFS = BN >= 128 && 2 * ACC + 2 * SF_COLS <= 512 ? 2 : 1;
    static constexpr int COLS = pow2_cols(BUFS * ACC + 2 * SF_COLS);
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 512;
    static_assert(STAGES >= 2 && PER_SM * COLS <= 512, "no room");
    static_assert(SMEM > (PER_SM == 2 ? kOneOfTwo : kBesideNone) && SMEM <= (PER_SM == 2 ? 115712 : 232448), "shares an SM with one block, or with none");
    static_assert(!FP4 || !AMN, "4-bit operands lie along K");
};

// Both activations are g / (1 + exp(-z)) with z = g (c0 + c1 g^2): silu has z = g, and v / 2 (1 + tanh(y)) = v / (1 + exp(-2 y)).  z has g's sign, so with
// e = exp(-|z|) = h^2, h = 2^(-|z| / (2 ln 2)), it is g / (1 + e), or (g / (1 + e)) h h where g is negative: the divisor is in [1, 2], and h is a normal
// number as far as h^2 is any, so that the two approximate instructions need no care for their ranges and results are right relative to their own size
// down to the least numbers.  (exp(-z) in the divisor made zeros of results below 1e-36.)  Off by 7.5 steps of 2^-23, and by |z| of them for the
// rounding of h's argument, as a rounding of g would cause.  expf(-|z|) was 8 to 27 % slower a call in 4-bit gated products of 256 to 4096 in K.
struct ActForm { float c0, c1; };  // over 2 ln 2
constexpr float kTwoLn2 = 1.3862943611198906f;
__device__ __forceinline__ ActForm act_form(int act) {
    constexpr float silu = 1.f / kTwoLn2, gelu = 1.5957691216057308f / kTwoLn2;
    return act == ACT_SILU ? ActForm{silu, 0.f} : ActForm{gelu, gelu * 0.044715f};
}
__device__ __forceinline__ float act_square(float g) { return fminf(g * g, 1e30f); }  // finite, so that 0 times it is 0
__device__ __forceinline__ float power_of_two(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float act_of(ActForm f, float g) {
    const float h = power_of_two(-fabsf(g * fmaf(f.c1, act_square(g), f.c0))), q = g * reciprocal(fmaf(h, h, 1.f)), s = g < 0.f ? h : 1.f;
    return q * s * s;
}

template <int OUT>
__device__ __forceinline__ void put(void* out, size_t at, float v) {
    if constexpr (OUT == T_F32) reinterpret_cast<float*>(out)[at] = v;
    else if constexpr (OUT == T_F16) reinterpret_cast<__half*>(out)[at] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
}

// Byte of scale j (of 32 elements) of row r in the tiles of a matrix with `kb` tiles a row.
__host__ __device__ __forceinline__ size_t scale_at(size_t r, int j, int kb) {
    return ((r >> 7) * kb + (j >> 2)) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4 + (j & 3);
}
// The scale byte of a block whose largest magnitude has these bits: floor(log2) - 2, at least 2^-127; 255 (NaN) where it is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const uint32_t ex = amax_bits >> 23;
    return ex == 255 ? 255u : ex > 2 ? ex - 2 : 0u;
}
__device__ __forceinline__ float scale_inverse(uint32_t e) { return __uint_as_float((254u - (e == 255 ? 254u : e)) << 23); }  // 0 where the scale is NaN
// Numbers as e2m1, the first in the lowest bits; nearest, ties to even, 6 beyond 6.
__device__ __forceinline__ uint32_t e2m1_pair(float a, float b) {
    uint16_t r;
    asm("{\n\t.reg .b8 c;\n\tcvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\tmov.b16 %0, {c, c};\n\t}" : "=h"(r) : "f"(a), "f"(b));
    return r & 0xffu;
}
__device__ __forceinline__ uint32_t e2m1_eight(const float (&v)[8], float by) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r) : "f"(v[0] * by), "f"(v[1] * by), "f"(v[2] * by), "f"(v[3] * by), "f"(v[4] * by), "f"(v[5] * by), "f"(v[6] * by), "f"(v[7] * by));
    return r;
}

// ---- tcgen05 of this file ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
        : "memory");
}
// 512 bytes of scales (32 x 16 bytes) to four TMEM columns of all four row quarters.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem) {
    const uint64_t desc = ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | ((smem >> 4) & 0x3FFFu);  // no swizzle, 8 rows of 16 bytes after 128
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(s32(dst)), "l"(src), "r"(bytes),
                 "r"(s32(bar))
                 : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_id() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same for reads alone: does not wait for this thread's stores.
__device__ __forceinline__ void cluster_leave() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 peer_floats(uint32_t smem, uint32_t rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem), "r"(rank) : "memory");
    return v;
}

// One column of results: feature m of this lane (beyond M: nothing stored), row n of the output.
template <class C, int OUT>
__device__ __forceinline__ void emit(const Params& p, int m, int n, float v0, float v1) {
    float v = v0;
    if constexpr (C::NA == 2) {
        v = act_of(act_form(p.act), v0) * v1;
        if (p.pre && m < p.M) {
            p.pre[(size_t)n * p.M + m] = v0;
            p.pre[((size_t)p.N + n) * p.M + m] = v1;
        }
    }
    if constexpr (OUT == T_MXFP4) {
        // The warp's 32 features are one block.
        const int lane = threadIdx.x & 31;
        const uint32_t e = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
        const float s = v * scale_inverse(e);
        const float other = __shfl_xor_sync(0xffffffffu, s, 1);
        uint32_t c = e == 255 ? 0u : (lane & 1) ? e2m1_pair(other, s) : e2m1_pair(s, other);
        c <<= 8 * ((lane >> 1) & 3);
        c |= __shfl_xor_sync(0xffffffffu, c, 2);
        c |= __shfl_xor_sync(0xffffffffu, c, 4);
        if (m < p.M && (lane & 7) == 0) *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out) + ((size_t)n * p.M + m) / 2) = c;
        if (lane == 0) p.out_scales[scale_at(n, m >> 5, (p.M + 127) >> 7)] = (uint8_t)(m < p.M ? e : 0u);
    } else {
        if (m < p.M) put<OUT>(p.out, (size_t)n * p.ldo + m, v);
    }
}

template <class C, int OUT>
__device__ __forceinline__ void tile_out(const Params& p, int tile, uint32_t tacc, int quad, int half, int lane) {
    const int m = tile * TM + quad * 32 + lane;
    const uint32_t ta = tacc + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
    for (int g = half; 16 * g < p.N; g += 2) {
        uint32_t v0[16], v1[16];
        tmem_ld16(ta + 16 * g, v0);
        if constexpr (C::NA == 2) tmem_ld16(ta + C::BN + 16 * g, v1);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int n = 16 * g + j;
            if (n < p.N) emit<C, OUT>(p, m, n, __uint_as_float(v0[j]), C::NA == 2 ? __uint_as_float(v1[j]) : 0.f);
        }
    }
}

// Four neighbouring results, of which `left` exist; whole: 8- or 16-byte stores are aligned.
template <int OUT>
__device__ __forceinline__ void put4(void* out, size_t at, const float (&o)[4], int left, bool whole) {
    if (whole && left >= 4) {
        if constexpr (OUT == T_F32) {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = make_float4(o[0], o[1], o[2], o[3]);
        } else {
            uint16_t h[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) put<OUT>(h, i, o[i]);
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + at) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) put<OUT>(out, at + i, o[i]);
}
// The sums of columns' shares, in rank order: a warp two columns at a time, four neighbouring features a lane, all shares asked for at once.  One column where two
// accumulators meet the 96 registers of two blocks an SM: with two, 588 bytes went to local memory (452 in 16 bits).  us a call with two / one: 4-bit gated 2048 -> 8192
// of 1, 8, 33 tokens 5.3 / 4.9, 6.0 / 4.9, 7.8 / 6.8; bf16 gated 4 tokens, 4096 -> 10240 31.1 / 29.0, 64 tokens, 2048 -> 5632 18.0 / 16.2.
template <class C, int OUT>
__device__ __forceinline__ void split_out(const Params& p, int tile, uint32_t red, uint32_t rank, int warp, int lane) {
    const int m = tile * TM + 4 * lane, left = p.M - m;
    const ActForm act = act_form(p.act);
    const bool whole = ((p.ldo | (reinterpret_cast<uintptr_t>(p.out) / (OUT == T_F32 ? 4 : 2))) & 3) == 0;
    const int step = EPI_WARPS * p.splits;
    constexpr int COLUMNS = C::NA == 2 && C::PER_SM == 2 ? 1 : 2;
#pragma unroll 1
    for (int c0 = (int)rank + p.splits * warp; c0 < p.N; c0 += COLUMNS * step) {
        float4 s[COLUMNS][C::NA];
        for (int r = 0; r < p.splits; r += 4) {
            float4 v[COLUMNS][C::NA][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r + i < p.splits) {
#pragma unroll
                    for (int j = 0; j < COLUMNS; ++j)
#pragma unroll
                        for (int a = 0; a < C::NA; ++a)  // a second column beyond the last reads where the ring was
                            v[j][a][i] = peer_floats(red + 4u * (uint32_t)((a * C::BN + min(c0 + j * step, C::BN - 1)) * TM + 4 * lane), r + i);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r + i < p.splits) {
#pragma unroll
                    for (int j = 0; j < COLUMNS; ++j)
#pragma unroll
                        for (int a = 0; a < C::NA; ++a) {
                            float4& d = s[j][a];
                            const float4 t = v[j][a][i];
                            if (r + i == 0) d = t;
                            else d.x += t.x, d.y += t.y, d.z += t.z, d.w += t.w;
                        }
                }
        }
#pragma unroll
        for (int j = 0; j < COLUMNS; ++j) {
            const int c = c0 + j * step;
            if (c >= p.N) break;
            float o[4] = {s[j][0].x, s[j][0].y, s[j][0].z, s[j][0].w};
            if constexpr (C::NA == 2) {
                const float u[4] = {s[j][1].x, s[j][1].y, s[j][1].z, s[j][1].w};
                if (p.pre) {  // M is a multiple of eight
                    put4<T_F32>(p.pre, (size_t)c * p.M + m, o, left, true);
                    put4<T_F32>(p.pre, ((size_t)p.N + c) * p.M + m, u, left, true);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = act_of(act, o[i]) * u[i];
            }
            if constexpr (OUT == T_MXFP4) {  // a block is eight lanes
                uint32_t mx = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = max(mx, __float_as_uint(o[i]) & 0x7fffffffu);
#pragma unroll
                for (int d = 1; d < 8; d <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                const uint32_t e = scale_byte(mx);
                const float by = scale_inverse(e);
                const uint32_t code = e2m1_pair(o[0] * by, o[1] * by) | e2m1_pair(o[2] * by, o[3] * by) << 8;
                if (left > 0) *reinterpret_cast<uint16_t*>(reinterpret_cast<uint8_t*>(p.out) + ((size_t)c * p.M + m) / 2) = (uint16_t)(e == 255 ? 0u : code);
                if ((lane & 7) == 0) p.out_scales[scale_at(c, m >> 5, (p.M + 127) >> 7)] = (uint8_t)(left > 0 ? e : 0u);
            } else {
                put4<OUT>(p.out, (size_t)c * p.ldo + m, o, left, whole);
            }
        }
    }
}

template <class C>
__global__ void __launch_bounds__(NTHREADS, C::PER_SM) dense_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE);
    uint64_t* empty = full + C::STAGES;
    uint64_t* tfull = empty + C::STAGES;
    uint64_t* tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mb_init(&full[i], 1);
            mb_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mb_init(&tfull[i], 1);
            mb_init(&tempty[i], EPI_WARPS);
        }
        fence_mbarrier_init();
    }
    if (warp == 0 && lane < 4) prefetch_map(lane < 2 ? &p.a[lane & (C::NA == 2 ? 1 : p.passes - 1)] : &p.b[lane & (p.passes - 1)]);
    if (warp == 1) tmem_alloc<C::COLS>(tmem_slot);
    const int rank = p.splits > 1 ? (int)cluster_rank() : 0, c0 = p.share[rank], c1 = p.share[rank + 1], kch = p.passes == 2 ? p.chunks >> 1 : p.chunks;
    const int tiles = (p.M + TM - 1) / TM, first = p.splits > 1 ? (int)cluster_id() : blockIdx.x, step = p.splits > 1 ? tiles : gridDim.x;
    const int nkb = (p.K + 127) >> 7;  // scale tiles along K
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    bool ok = true;

    if (warp == 0) {
        // ---------------- TMA ----------------
        int it = 0;
        for (int t = first; t < tiles && ok; t += step) {
            const int m0 = t * TM;
            for (int c = c0; c < c1; ++c, ++it) {
                const int st = it % C::STAGES, n = it / C::STAGES;
                if (n > 0) ok = warp_all(mb_wait(&empty[st], (uint32_t)(n - 1) & 1u, p.status, kWaitStage));
                if (!ok) break;
                if (elect_one()) {
                    uint8_t* s = smem + st * C::STAGE;
                    const int pass = c >= kch, kc = pass ? c - kch : c;
                    const int kbs = C::FP4 ? min(2, nkb - 2 * kc) : 0;
                    mb_expect_tx(&full[st], (uint32_t)(C::NA * C::A_BYTES + p.bn * 128 + (C::NA + 1) * kbs * 512));
#pragma unroll
                    for (int a = 0; a < C::NA; ++a) {
                        const CUtensorMap* map = &p.a[C::NA == 2 ? a : pass];
                        if constexpr (C::AMN) {
#pragma unroll
                            for (int i = 0; i < TM / 64; ++i) tma_load_2d(s + a * C::A_BYTES + i * 8192, map, m0 + 64 * i, kc * 64, &full[st]);
                        } else {
                            tma_load_2d(s + a * C::A_BYTES, map, kc * (C::FP4 ? 128 : 64), m0, &full[st]);
                        }
                    }
                    uint8_t* sb = s + C::NA * C::A_BYTES;
                    tma_load_2d(sb, &p.b[pass], kc * (C::FP4 ? 128 : 64), 0, &full[st]);
                    if constexpr (C::FP4) {
                        uint8_t* sf = sb + C::B_BYTES;
                        for (int a = 0; a < C::NA; ++a)
                            bulk_load(sf + a * 1024, p.sa[a] + ((size_t)t * nkb + 2 * kc) * 512, kbs * 512, &full[st]);
                        bulk_load(sf + C::NA * 1024, p.sb + (size_t)2 * kc * 512, kbs * 512, &full[st]);
                    }
                }
                __syncwarp();
            }
        }
        if (!ok)  // copies in flight end before their shared memory is given up
            for (int i = max(0, it - C::STAGES); i < it; ++i) mb_wait(&full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, p.status, kWaitStage);
    } else if (warp == 1) {
        // ---------------- MMA issue ----------------
        const uint32_t smem_lo = (s32(smem) & 0x3FFFFu) >> 4;  // in a cluster an address has its CTA's rank above
        constexpr uint32_t LA = (C::AMN ? (8192u >> 4) : 1u) << 16, LB = 1u << 16;
        constexpr uint32_t KA = C::AMN ? 128 : 2, KB = 2;  // bytes / 16 from one K step of an MMA to the next
        const uint32_t sf_tmem = tmem + C::BUFS * C::ACC;
        uint32_t idesc;
        if constexpr (C::FP4)  // e2m1 operands, 2^x scales
            idesc = (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | (1u << 23) | (1u << 27);
        else
            idesc = (1u << 4) | ((uint32_t)p.idesc_type << 7) | ((uint32_t)p.idesc_type << 10) | ((uint32_t)C::AMN << 15) | ((uint32_t)(p.bn >> 3) << 17) |
                    ((uint32_t)(TM >> 4) << 24);
        int it = 0, nt = 0;
        for (int t = first; t < tiles && ok; t += step, ++nt) {
            const int buf = nt % C::BUFS, use = nt / C::BUFS;
            if (use > 0) ok = warp_all(mb_wait(&tempty[buf], (uint32_t)(use - 1) & 1u, p.status, kWaitDrain));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem + buf * C::ACC;
            for (int c = c0; c < c1; ++c, ++it) {
                const int st = it % C::STAGES, n = it / C::STAGES;
                ok = warp_all(mb_wait(&full[st], (uint32_t)n & 1u, p.status, kWaitStage));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t a0 = smem_lo + (uint32_t)(st * (C::STAGE >> 4)), b0 = a0 + ((C::NA * C::A_BYTES) >> 4);
                    if constexpr (C::FP4) {
                        const uint32_t sf = b0 + (C::B_BYTES >> 4), ts = sf_tmem + (it & 1) * C::SF_COLS;
                        const int left = p.K - c * C::BK, kbs = left > 128 ? 2 : 1, steps = left >= C::BK ? 4 : (left + 63) >> 6;
                        // TMEM: A's scales 4 columns per (A, 128 of K), B's 4 per 128 of K
                        for (int kb = 0; kb < kbs; ++kb) {
#pragma unroll
                            for (int a = 0; a < C::NA; ++a) scales_to_tmem(ts + a * 8 + kb * 4, (sf + a * 64 + kb * 32) << 4);
                            scales_to_tmem(ts + C::NA * 8 + kb * 4, (sf + C::NA * 64 + kb * 32) << 4);
                        }
                        for (int ks = 0; ks < steps; ++ks) {
                            const uint32_t id = idesc | ((uint32_t)(ks & 1) << 30) | ((uint32_t)(ks & 1) << 5);  // scales 0, 1 or 2, 3 of a word
                            const uint32_t tb = ts + C::NA * 8 + (ks >> 1) * 4;
#pragma unroll
                            for (int a = 0; a < C::NA; ++a)
                                mma_mxf4(d + a * C::BN, desc_of(a0 + a * (C::A_BYTES >> 4) + ks * KA | LA), desc_of(b0 + ks * KB | LB), id,
                                         ts + a * 8 + (ks >> 1) * 4, tb, c > c0 || ks > 0);
                        }
                    } else {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                            for (int a = 0; a < C::NA; ++a)
                                mma_bf16(d + a * C::BN, desc_of(a0 + a * (C::A_BYTES >> 4) + ks * KA | LA), desc_of(b0 + ks * KB | LB), idesc,
                                         c > c0 || ks > 0);
                    }
                    mma_commit(&empty[st]);
                    if (c == c1 - 1) mma_commit(&tfull[buf]);
                }
                __syncwarp();
            }
        }
    } else {
        // ---------------- epilogue ----------------
        const int quad = warp & 3, half = (warp - 2) >> 2;
        int nt = 0;
        for (int t = first; t < tiles && ok; t += step, ++nt) {
            const int buf = nt % C::BUFS, use = nt / C::BUFS;
            ok = warp_all(mb_wait(&tfull[buf], (uint32_t)use & 1u, p.status, kWaitAcc));
            if (!ok) break;
            tc_fence_after();
            const uint32_t tacc = tmem + buf * C::ACC;
            if (p.splits == 1) {
                switch (p.out_type) {
                    case T_F32: tile_out<C, T_F32>(p, t, tacc, quad, half, lane); break;
                    case T_F16: tile_out<C, T_F16>(p, t, tacc, quad, half, lane); break;
                    case T_BF16: tile_out<C, T_BF16>(p, t, tacc, quad, half, lane); break;
                    default: if constexpr (C::FP4 && C::NA == 2) tile_out<C, T_MXFP4>(p, t, tacc, quad, half, lane);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mb_arrive(&tempty[buf]);
            } else {
                // This CTA's share of the sum, into the ring's memory: all copies have landed and been read.
                float* red = reinterpret_cast<float*>(smem);
                const uint32_t ta = tacc + ((uint32_t)(quad * 32) << 16);
                for (int g = half; g < C::ACC / 16; g += 2) {
                    if (g * 16 % C::BN >= p.N) continue;
                    uint32_t v[16];
                    tmem_ld16(ta + 16 * g, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) red[(16 * g + j) * TM + quad * 32 + lane] = __uint_as_float(v[j]);
                }
            }
        }
    }
    __syncwarp();
    if (p.splits > 1) {
        cluster_sync();
        if (warp >= 2) {
            const uint32_t red = s32(smem);
            switch (p.out_type) {
                case T_F32: split_out<C, T_F32>(p, first, red, rank, warp - 2, lane); break;
                case T_F16: split_out<C, T_F16>(p, first, red, rank, warp - 2, lane); break;
                case T_BF16: split_out<C, T_BF16>(p, first, red, rank, warp - 2, lane); break;
                default: if constexpr (C::FP4 && C::NA == 2) split_out<C, T_MXFP4>(p, first, red, rank, warp - 2, lane);
            }
        }
        __syncwarp();
        cluster_leave();  // nobody leaves while its sums are being read
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<C::COLS>(tmem);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
struct Operand {  // a matrix in memory
    const void* data;
    uint64_t rows, cols, pitch;  // pitch: bytes between rows
};
// Boxes of 128 bytes a row, of which L2 fetches 256: a row's next box comes from the same page of memory.  8 % where the weights' bytes count: 4-bit 65536 x
// 4096, 8 tokens, 29.2 us with 128 and 27.4 with 256; gated bf16, 4 tokens, 4096 -> 10240 34.0 and 31.2; no difference elsewhere.
template <bool FP4>
int operand_map(CUtensorMap* m, const Operand& o, int box_rows, int type) {
    const CUtensorMapDataType t = FP4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return tiled_map(m, t, FP4 ? 1 : 2, o.data, o.rows, FP4 ? o.cols / 2 : o.cols, o.pitch, box_rows, 0, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

template <class C>
cudaLaunchConfig_t launch_config(dnb_ctx* c, cudaLaunchAttribute (&at)[2], unsigned grid, int splits) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(NTHREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = c->stream;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = c->use_pdl;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = splits;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    return cfg;
}

// How many clusters the device holds at once, 0: none, or it did not say (which is asked again).  Blocks of a cluster share a GPC, whose SMs they may not
// fill (15 clusters of eight blocks that each want an SM, where 148 SMs could hold 18).  Asked once a device.
template <class K>
int clusters_at_once(std::atomic<int>& known, K kernel, const cudaLaunchConfig_t& cfg) {
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        known.store(n > 0 ? n : -1, std::memory_order_relaxed);
    }
    return n > 0 ? n : 0;
}

// p: everything but the maps, the operands' type and the splits.  a, b: C::NA or p.passes operands of A, p.passes of B.
template <class C>
int launch_dense(dnb_ctx* c, Params& p, const Operand* a, int na, const Operand* b, int nb, int type, const char* name) {
    int rc;
    p.bn = (p.N + 15) / 16 * 16;
    for (int i = 0; i < na; ++i)
        if ((rc = operand_map<C::FP4>(&p.a[i], a[i], C::AMN ? 64 : TM, type))) return rc;
    for (int i = 0; i < nb; ++i)
        if ((rc = operand_map<C::FP4>(&p.b[i], b[i], p.bn, type))) return rc;
    p.idesc_type = type == T_BF16;
    p.status = c->status;
    const int tiles = (p.M + TM - 1) / TM, chunks = (p.K + C::BK - 1) / C::BK * p.passes;
    static_assert(C::ACC * TM * 4 <= C::STAGES * C::STAGE, "the partial sums of a split lie in the ring");
    static SmemGrant grant;
    DNB_CUDA(grant_smem(grant, c->device, dense_kernel<C>, C::SMEM));
    static std::atomic<int> known[64][9];
    int at_once[9] = {0, c->sm_count * C::PER_SM};
    cudaLaunchAttribute at[2];
    for (int s = 2; s <= 8 && s <= chunks; ++s) at_once[s] = clusters_at_once(known[c->device][s], dense_kernel<C>, launch_config<C>(c, at, s, s));
    p.splits = best_splits(at_once, c->sm_count, C::STAGE, tiles, chunks);
    p.chunks = chunks;
    for (int i = 0; i <= p.splits; ++i) p.share[i] = (int)((int64_t)chunks * i / p.splits);
    const int slots = c->sm_count * C::PER_SM;
    const unsigned grid = p.splits > 1 ? (unsigned)tiles * p.splits : (unsigned)(tiles < slots ? tiles : slots);
    ProfScope prof_(c, c->stream, name);
    const cudaLaunchConfig_t cfg = launch_config<C>(c, at, grid, p.splits);
    DNB_CUDA(cudaLaunchKernelEx(&cfg, dense_kernel<C>, p));
    c->launches++;
    return DNB_OK;
}

}  // namespace dt
}  // namespace dnb
