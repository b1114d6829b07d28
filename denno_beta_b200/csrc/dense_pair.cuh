// Dense products of many rows on tcgen05, two SMs a tile (cta_group::2): D[m][n] = sum_k A[m][k] B[n][k], out[m][n] with n contiguous.
//
// Tiles of 256 x 256: each CTA of a pair holds 128 rows of A and 128 of B, the MMA (M 256, N 256) reads B from both, and a CTA's
// tensor memory gets its 128 rows of D: half the operand bytes of two separate 128 x 256 tiles, through L2 as well as into the MMAs.
// Gated: the B tile is 128 rows of gate in one CTA and the same 128 of up in the other, so that a thread that reads a row of D has g and u
// of the same features: 256 x 128 results from one MMA.
// Operands as in dense_tc.cuh: 4 bits with scales in tensor memory, or 16 bits with rows along K or along m / n.
//
// Tiles go to the pairs in turn.  What is left over when every pair has had as many, or all of them where there are few, one tile a cluster of
// two to four pairs: these divide K, and each CTA adds up some pieces of it, the pairs' shares in ascending order, through distributed shared memory.
//
// A CTA: warp 0 brings its halves by TMA (every copy reports to the leader's barrier), warp 1 of the leader issues the MMAs of both, eight warps
// read the accumulators: a thread a row, its 128 columns at once, then 64 (16 bits) or 32 at a time through 4 KB of shared memory a warp and out by TMA
// stores (rows that do not start or end at multiples of 16 bytes: by plain stores, a row a warp).  16 bits: two accumulators; 4 bits, where the scales
// take the room: one, in registers before the next tile's MMAs need it.
//
// What bounds it.  A chunk (64 of K in 16 bits, 256 in 4) takes 615 and 650 cycles where its MMAs alone take 512: the copies that come in and what the
// MMAs read are 107 bytes a clock of shared memory's 128; the scales' way to tensor memory is 4 % of a chunk.  Two tiles that share a B (three quarters
// of the copies) were 1.5 to 5 % faster on long runs, no faster on short ones, and are not kept.  Long runs are bound by the power limit: bf16 4096 tokens,
// 4096 -> 10240, 1.57 PFLOP/s for some milliseconds (0.93 of the measured peak), 1.36 at 1.2 to 1.35 GHz; 4 bits, 8192 tokens, 4096 -> 8192, 104 us
// (5.3 PFLOP/s), 118 to 123 at 1.5 GHz.  Short ones: about 5 us of launch, set-up and first copies, and a first tile's epilogue of 2,500 cycles (1,100
// once its code is in the instruction cache); and this one width of tile, which leaves pairs idle where their number and the tiles' do not meet.
#pragma once
#include <type_traits>

#include "dense_tc.cuh"

namespace dnb {
namespace dp {
using namespace dt;

// Quotients of numbers below 2^31 by a multiplication: integer divisions took 400 of a small tile's 2,000 cycles.
struct Divisor {
    int d;
    uint32_t mul, shift;
    __device__ __forceinline__ int div(int x) const { return d == 1 ? x : (int)(__umulhi((uint32_t)x, mul) >> shift); }
};
inline Divisor divisor(int d) {  // mul = ceil(2^(32 + shift) / d), with 2^shift the largest power of two below d: exact for x < 2^31
    Divisor r = {d, 0, 0};
    while (d > 1 && (2 << r.shift) < d) ++r.shift;
    if (d > 1) r.mul = (uint32_t)(((1ull << (32 + r.shift)) + d - 1) / d);
    return r;
}

struct Params {
    CUtensorMap a[2], b[2];         // operands
    CUtensorMap sa, sb[2];          // scale tiles, 512 bytes a row (4 bit)
    CUtensorMap out[2], pre[2];     // results
    CUtensorMap narrow[2];          // 16-bit results of split tiles, in boxes of 32 columns
    int M, N, K;                    // N: columns of the output
    int passes;                     // 2: the sum goes on over a[1], b[1]
    int both;                       // 2: twice the tiles, the second half with a[1] to the second output
    int tiles_m, per_output;        // rows of tiles; tiles of one output
    Divisor group, last_group;      // tiles of eight rows of tiles; rows of the last group
    int parts, whole, tiles;        // pairs a cluster; tiles that are not split (the rest: one a cluster); all
    int each, more;                 // whole tiles a pair, one more for the first `more` pairs
    int chunks, share[5];           // of K; the parts' first chunks of a split tile
    int idesc_type, out_type, act;
    bool tma_out, keep;             // keep: g and u to pre
    void* outp[2];
    uint8_t* out_scales;
    size_t ldo;
    int* status;
};

constexpr int PAIR_THREADS = 384;   // a warpgroup for copies and MMAs (two of its warps idle), two for the results
// Registers after the split, of the 168 a thread that 384 threads start with: 128 x 56 + 256 x 216 = 62,464 of 64,512.
constexpr int kFewRegs = 56, kManyRegs = 216;

template <bool FP4_, bool GATED_, bool AMN_ = false, bool BMN_ = false>
struct Cfg {
    static constexpr bool FP4 = FP4_, GATED = GATED_, AMN = AMN_, BMN = BMN_;
    static constexpr int BK = FP4 ? 256 : 64;
    static constexpr int HALF = 128 * 128;                     // a CTA's half of an operand's tile
    static constexpr int SF = FP4 ? 3 * 1024 : 0;              // scales: 128 rows of A, 256 of B, 256 of K
    static constexpr int STAGE = 2 * HALF + SF;
    static constexpr int STAGES = 5;
    static constexpr int BOXES = FP4 ? 1 : 2;                  // 4 KB of results a warp may have on their way
    static constexpr int STAGING = EPI_WARPS * BOXES * 4096;
    static constexpr int ACC = 256, BUFS = FP4 ? 1 : 2;
    static constexpr int SF_COLS = 24;                         // 8 of A, 16 of B
    static constexpr int COLS = 512;
    static constexpr int NOUT = GATED ? 128 : 256;             // columns of the output a tile
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + STAGING + 1024 + 256;
    static_assert(SMEM > kBesideNone && SMEM <= 232448, "alone on its SM");
};

// ---- PTX of pairs ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t in_cta(uint32_t smem, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(rank));
    return a;
}
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(s32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int MORE>
__device__ __forceinline__ void store_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(MORE) : "memory"); }
// Says that tensor memory has been read (tcgen05's wait and fence stand before it).  Released at the cluster's scope it would wait 1,300 cycles for
// the stores of the last tile, which nobody has to see.
__device__ __forceinline__ void remote_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void pair_commit(uint64_t* bar, uint16_t pair) {  // the barrier of both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(s32(bar)), "h"(pair) : "memory");
}
__device__ __forceinline__ void pair_mma16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void pair_mma4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void pair_scales(uint32_t taddr, uint32_t smem) {  // each CTA's own 512 bytes to its own tensor memory
    const uint64_t desc = ((uint64_t)((128u >> 4) | (1u << 14)) << 32) | ((smem >> 4) & 0x3FFFu);
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
__device__ __forceinline__ void pair_alloc(uint32_t* slot) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_free(uint32_t base) { asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory"); }
// 32 columns of this thread's row.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// ---- results ----------------------------------------------------------------------------------------------------------------------
template <int OUT>
__device__ __forceinline__ uint32_t two(float a, float b) {
    if constexpr (OUT == T_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
// A warp's 32 rows x 128 bytes of results, a row a lane, in its 4 KB of shared memory, 16 bytes swizzled as in the tensor map (which keeps the
// stores of eight lanes apart), and out as one box: rows of 128 bytes, as TMA's stores go by the row.
__device__ __forceinline__ void chunk_put(uint8_t* buf, int lane, const float (&v)[32]) {
    uint8_t* row = buf + lane * 128;
#pragma unroll
    for (int c = 0; c < 8; ++c) *reinterpret_cast<float4*>(row + ((c ^ (lane & 7)) << 4)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}
__device__ __forceinline__ void chunk_put(uint8_t* buf, int lane, const uint32_t (&h)[16]) {  // a row of 64 bytes
    uint8_t* row = buf + lane * 64;
#pragma unroll
    for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(row + ((c ^ (lane >> 1 & 3)) << 4)) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
}
__device__ __forceinline__ void chunk_put(uint8_t* buf, int lane, int part, const uint32_t (&h)[16]) {  // 16 bits: one of two halves of a row
    uint8_t* row = buf + lane * 128;
#pragma unroll
    for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4*>(row + (((c + 4 * part) ^ (lane & 7)) << 4)) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
}
template <int OUT>
__device__ __forceinline__ void halves(const float (&v)[32], uint32_t (&h)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) h[i] = two<OUT>(v[2 * i], v[2 * i + 1]);
}
// A warp's boxes take turns: one is written when all groups of stores but the last have been read.  So every chunk is a group, stored by TMA or not.
struct Boxes {
    uint8_t* base;
    uint32_t at;  // 0 or 4096
};
template <class C>
__device__ __forceinline__ uint8_t* chunk_begin(int lane, Boxes& b) {
    if constexpr (C::BOXES == 2) b.at ^= 4096;
    if (lane == 0) store_read<C::BOXES - 1>();
    __syncwarp();
    return b.base + b.at;
}
// From (row0, col0) of a [M][N] matrix, rows of BYTES.
template <int OUT, int BYTES = 128>
__device__ __forceinline__ void chunk_end(const CUtensorMap* map, bool tma, void* out, size_t ldo, int M, int N, int row0, int col0, const uint8_t* buf, int lane) {
    if (tma) fence_async_smem();
    __syncwarp();
    if (lane == 0) {
        if (tma && row0 < M && col0 < N) store_2d(map, col0, row0, s32(buf));
        store_commit();
    }
    if (tma) return;
    const int rows = min(32, M - row0);
    constexpr int SIZE = OUT == T_F32 ? 4 : 2;
    using W = typename std::conditional<OUT == T_F32, float, uint16_t>::type;
#pragma unroll
    for (int i = 0; i < BYTES / SIZE / 32; ++i) {
        const int c = 32 * i + lane;
        if (col0 + c >= N) break;
        W* to = reinterpret_cast<W*>(out) + (size_t)row0 * ldo + col0 + c;
#pragma unroll 8
        for (int r = 0; r < rows; ++r) to[r * ldo] = *reinterpret_cast<const W*>(buf + r * BYTES + (((c * SIZE >> 4) ^ (BYTES == 128 ? r & 7 : r >> 1 & 3)) << 4) + (c * SIZE & 15));
    }
    __syncwarp();
}
// 32 features of a row as one 4-bit block.
__device__ __forceinline__ void block_out(const Params& p, int row, int col, const float (&v)[32]) {
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t e = scale_byte(mx);
    const float by = scale_inverse(e);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float w[8] = {v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3], v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]};
        c[i] = e == 255 ? 0u : e2m1_eight(w, by);
    }
    if (row >= p.M) return;
    if (col < p.N) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.outp[0]) + ((size_t)row * p.N + col) / 2) = make_uint4(c[0], c[1], c[2], c[3]);
    p.out_scales[scale_at(row, col >> 5, (p.N + 127) >> 7)] = (uint8_t)(col < p.N ? e : 0u);
}

// 32 columns of g and u: kept, and g becomes the output.
template <class C>
__device__ __forceinline__ void gated_chunk(const Params& p, ActForm act, int row0, int col, float (&g)[32], float (&u)[32], Boxes& boxes, int lane) {
    if (p.keep) {
        uint8_t* buf = chunk_begin<C>(lane, boxes);
        chunk_put(buf, lane, g);
        chunk_end<T_F32>(&p.pre[0], true, nullptr, 0, p.M, p.N, row0, col, buf, lane);
        buf = chunk_begin<C>(lane, boxes);
        chunk_put(buf, lane, u);
        chunk_end<T_F32>(&p.pre[1], true, nullptr, 0, p.M, p.N, row0, col, buf, lane);
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) g[j] = act_of(act, g[j]) * u[j];
}
// What a thread does with 32 columns (gated: of g and of u) from `col`: chunk c of its row.
template <class C, int OUT>
__device__ __forceinline__ void chunk_of(const Params& p, ActForm act, int which, int c, int row0, int col, float (&g)[32], float (&u)[32], Boxes& boxes, int lane,
                                         uint32_t (&first)[16]) {
    if constexpr (C::GATED) gated_chunk<C>(p, act, row0, col, g, u, boxes, lane);
    if constexpr (OUT == T_MXFP4) {
        block_out(p, row0 + lane, col, g);
    } else if constexpr (OUT == T_F32) {
        uint8_t* buf = chunk_begin<C>(lane, boxes);
        chunk_put(buf, lane, g);
        chunk_end<OUT>(&p.out[which], p.tma_out, p.outp[which], p.ldo, p.M, p.N, row0, col, buf, lane);
    } else {
        // two chunks make a row of 128 bytes; the buffer may be wanted for pre between them
        if ((c & 1) == 0) return halves<OUT>(g, first);
        uint32_t h[16];
        halves<OUT>(g, h);
        uint8_t* buf = chunk_begin<C>(lane, boxes);
        chunk_put(buf, lane, 0, first);
        chunk_put(buf, lane, 1, h);
        chunk_end<OUT>(&p.out[which], p.tma_out, p.outp[which], p.ldo, p.M, p.N, row0, col - 32, buf, lane);
    }
}

// This thread's part of a tile, 128 columns (gated: 64 of g and of u), in registers: every element by a constant index, so the chunks are unrolled.
template <class C, int OUT>
__device__ __forceinline__ void results(const Params& p, int which, int row0, int n0, int half, Boxes& boxes, int lane, float (&v)[4][32]) {
    constexpr int CHUNKS = C::GATED ? 2 : 4;
    const ActForm act = act_form(p.act);
    uint32_t first[16];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        chunk_of<C, OUT>(p, act, which, c, row0, n0 + 32 * (half * CHUNKS + c), v[c], v[C::GATED ? 2 + c : c], boxes, lane, first);
}

// A split tile.  This CTA's sums in the ring's memory, four columns of all rows after another: what a warp reads of another CTA's is 512 bytes in a
// row (16 bytes a row apart took twice as long).
__device__ __forceinline__ uint32_t share_at(int row, int unit) { return (uint32_t)(unit * 128 + row) * 16; }
// The output of this CTA's 128 rows in pieces of 32 rows x 32 columns, a row a lane, summed over the cluster's pairs.  Neighbouring pieces go to
// different pairs: all SMs read, with as many warps as there are pieces for; each asks another CTA first (all the same one: 7 % of a call) and
// adds in ascending order.
template <class C, int OUT>
__device__ __forceinline__ void joined(const Params& p, int which, int part, int warp, int row0, int n0, uint32_t share, uint32_t rank, Boxes& boxes, int lane) {
    const ActForm act = act_form(p.act);
#pragma unroll 1
    for (int piece = part + p.parts * warp; piece < C::NOUT / 8; piece += p.parts * EPI_WARPS) {
        const int r32 = (piece & 3) * 32, left = 32 * (piece >> 2), row = row0 + r32, col = n0 + left;
        float v[C::GATED ? 2 : 1][32];
#pragma unroll
        for (int a = 0; a < (C::GATED ? 2 : 1); ++a) {
            float t[4][32];
#pragma unroll 1
            for (int j = 0, r = part; j < p.parts; ++j, r = r + 1 < p.parts ? r + 1 : 0)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    if (r == s) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(&t[s][4 * i]) = peer_floats(share + share_at(r32 + lane, (a * 128 + left) / 4 + i), 2 * s + rank);
                    }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                v[a][i] = t[0][i] + t[1][i];
                if (p.parts > 2) v[a][i] += t[2][i];
                if (p.parts > 3) v[a][i] += t[3][i];
            }
        }
        if constexpr (OUT == T_F16 || OUT == T_BF16) {
            if constexpr (C::GATED) gated_chunk<C>(p, act, row, col, v[0], v[1], boxes, lane);
            uint32_t h[16];
            halves<OUT>(v[0], h);
            uint8_t* buf = chunk_begin<C>(lane, boxes);
            chunk_put(buf, lane, h);
            chunk_end<OUT, 64>(&p.narrow[which], p.tma_out, p.outp[which], p.ldo, p.M, p.N, row, col, buf, lane);
        } else {
            uint32_t unused[16];
            chunk_of<C, OUT>(p, act, which, 0, row, col, v[0], v[C::GATED ? 1 : 0], boxes, lane, unused);
        }
    }
}

// Groups of eight rows of tiles, column by column: 8 x 256 rows of A by about as many of B are in flight.
__device__ __forceinline__ void pair_tile(const Params& p, int t, int& m, int& n, int& which) {
    which = t >= p.per_output;
    if (which) t -= p.per_output;
    const int g = p.group.div(t), in = t - g * p.group.d;
    if (8 * g + 8 <= p.tiles_m) {
        m = 8 * g + (in & 7);
        n = in >> 3;
    } else {
        n = p.last_group.div(in);
        m = 8 * g + in - n * p.last_group.d;
    }
}

template <class C>
__global__ void __launch_bounds__(PAIR_THREADS, 1) pair_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* staging = smem + C::STAGES * C::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);
    uint64_t* empty = full + C::STAGES;
    uint64_t* tfull = empty + C::STAGES;
    uint64_t* tempty = tfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t in_cluster = cluster_rank(), rank = in_cluster & 1, part = in_cluster >> 1, leader = in_cluster & ~1u;
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mb_init(&full[i], 1);   // the leader's: its own expect_tx; bytes of both CTAs
            mb_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mb_init(&tfull[i], 1);
            mb_init(&tempty[i], 2 * EPI_WARPS);  // the leader's: both CTAs' warps
        }
        fence_mbarrier_init();
    }
    if (warp == 0 && lane < 4) prefetch_map(lane < 2 ? &p.a[lane & ((p.passes | p.both) >> 1)] : &p.b[lane & (C::GATED ? 1 : p.passes >> 1)]);
    if (warp == 1) pair_alloc(tmem_slot);
    // Turn i of this pair: a tile of its own, or its share of the cluster's tile, which is the last.  Worked out while the barriers are under way; the
    // quotients come with the launch.
    const int first = blockIdx.x >> 1, step = gridDim.x >> 1, chunks = p.chunks;
    const int own = p.each + (first < p.more), split = p.whole + (int)cluster_id();
    const bool shares = split < p.tiles;
    const int turns = own + shares, s0 = p.share[part], s1 = p.share[part + 1];
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    bool ok = true;
    int m, n, which;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegs));
        if (warp == 0) {
            // ---------------- TMA ----------------
            const int nkb = (p.K + 127) >> 7, kch = p.passes == 2 ? chunks >> 1 : chunks;
            int it = 0;
            for (int i = 0; i < turns && ok; ++i) {
                pair_tile(p, i < own ? first + i * step : split, m, n, which);
                const int c0 = i < own ? 0 : s0, c1 = i < own ? chunks : s1;
                const int m0 = m * 256 + (int)rank * 128, n0 = C::GATED ? n * 128 : n * 256 + (int)rank * 128;
                for (int c = c0; c < c1; ++c, ++it) {
                    const int st = it % C::STAGES, use = it / C::STAGES;
                    if (use > 0) ok = warp_all(mb_wait(&empty[st], (uint32_t)(use - 1) & 1u, p.status, kWaitStage));
                    if (!ok) break;
                    if (elect_one()) {
                        uint8_t *sa = smem + st * C::STAGE, *sb = sa + C::HALF;
                        const int pass = c >= kch, kc = pass ? c - kch : c;
                        const uint32_t bar = in_cta(s32(&full[st]), leader);
                        if (rank == 0) mb_expect_tx(&full[st], 2u * C::STAGE);
                        const CUtensorMap *ma = &p.a[pass | which], *mb = &p.b[C::GATED ? (int)rank : pass];
                        if constexpr (C::AMN) {
                            pair_load_2d(sa, ma, m0, kc * 64, bar);
                            pair_load_2d(sa + 8192, ma, m0 + 64, kc * 64, bar);
                        } else {
                            pair_load_2d(sa, ma, kc * (C::FP4 ? 128 : 64), m0, bar);
                        }
                        if constexpr (C::BMN) {
                            pair_load_2d(sb, mb, n0, kc * 64, bar);
                            pair_load_2d(sb + 8192, mb, n0 + 64, kc * 64, bar);
                        } else {
                            pair_load_2d(sb, mb, kc * (C::FP4 ? 128 : 64), n0, bar);
                        }
                        if constexpr (C::FP4) {
                            uint8_t* sf = sb + C::HALF;
                            pair_load_2d(sf, &p.sa, 0, (m0 >> 7) * nkb + 2 * kc, bar);
                            pair_load_2d(sf + 1024, &p.sb[0], 0, (C::GATED ? n : 2 * n) * nkb + 2 * kc, bar);
                            pair_load_2d(sf + 2048, &p.sb[C::GATED], 0, (C::GATED ? n : 2 * n + 1) * nkb + 2 * kc, bar);
                        }
                    }
                    __syncwarp();
                }
            }
            // The last stages' arrivals, from the leader, come before the barriers that they arrive at go; if a wait gave up: the copies in flight, of both CTAs.
            for (int i = max(0, it - C::STAGES); i < it && (ok || rank == 0); ++i)
                mb_wait(ok ? &empty[i % C::STAGES] : &full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1u, p.status, kWaitStage);
        } else if (warp == 1) {
            // ---------------- MMA issue: the leader's thread for both ----------------
            if (rank == 0) {
                const uint32_t smem_lo = (s32(smem) & 0x3FFFFu) >> 4;  // in a cluster an address has its CTA's rank above
                constexpr uint32_t LA = (C::AMN ? (8192u >> 4) : 1u) << 16, LB = (C::BMN ? (8192u >> 4) : 1u) << 16;
                constexpr uint32_t KA = C::AMN ? 128 : 2, KB = C::BMN ? 128 : 2;
                const uint32_t sf_tmem = tmem + C::BUFS * C::ACC;
                const uint32_t idesc = C::FP4 ? (1u << 7) | (1u << 10) | ((256u >> 3) << 17) | (1u << 23) | ((256u >> 7) << 27)
                                              : (1u << 4) | ((uint32_t)p.idesc_type << 7) | ((uint32_t)p.idesc_type << 10) | ((uint32_t)C::AMN << 15) |
                                                    ((uint32_t)C::BMN << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
                const uint16_t pair = (uint16_t)(3u << leader);
                int it = 0;
                for (int nt = 0; nt < turns && ok; ++nt) {
                    const int c0 = nt < own ? 0 : s0, c1 = nt < own ? chunks : s1;
                    const int buf = nt % C::BUFS, use = nt / C::BUFS;
                    if (use > 0) ok = warp_all(mb_wait(&tempty[buf], (uint32_t)(use - 1) & 1u, p.status, kWaitDrain));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + buf * C::ACC;
                    for (int c = c0; c < c1; ++c, ++it) {
                        const int st = it % C::STAGES;
                        ok = warp_all(mb_wait(&full[st], (uint32_t)(it / C::STAGES) & 1u, p.status, kWaitStage));
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint32_t a0 = smem_lo + (uint32_t)(st * (C::STAGE >> 4)), b0 = a0 + (C::HALF >> 4);
                            if constexpr (C::FP4) {
                                const uint32_t sf = b0 + (C::HALF >> 4), ts = sf_tmem + (it & 1) * C::SF_COLS;
                                const int left = p.K - c * C::BK, kbs = left > 128 ? 2 : 1, steps = left >= C::BK ? 4 : (left + 63) >> 6;
                                for (int kb = 0; kb < kbs; ++kb) {
                                    pair_scales(ts + kb * 4, (sf + kb * 32) << 4);
                                    pair_scales(ts + 8 + kb * 8, (sf + 64 + kb * 32) << 4);
                                    pair_scales(ts + 12 + kb * 8, (sf + 128 + kb * 32) << 4);
                                }
                                for (int ks = 0; ks < steps; ++ks)
                                    pair_mma4(d, desc_of(a0 + ks * KA | LA), desc_of(b0 + ks * KB | LB), idesc | ((uint32_t)(ks & 1) << 30) | ((uint32_t)(ks & 1) << 5),
                                              ts + (ks >> 1) * 4, ts + 8 + (ks >> 1) * 8, c > c0 || ks > 0);
                            } else {
#pragma unroll
                                for (int ks = 0; ks < 4; ++ks)
                                    pair_mma16(d, desc_of(a0 + ks * KA | LA), desc_of(b0 + ks * KB | LB), idesc, c > c0 || ks > 0);
                            }
                            pair_commit(&empty[st], pair);
                            if (c == c1 - 1) pair_commit(&tfull[buf], pair);
                        }
                        __syncwarp();
                    }
                }
            }
        }
        __syncwarp();
        if (shares) cluster_sync();  // the shares are written
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        // ---------------- results ----------------
        const int quad = warp & 3, half = (warp - 4) >> 2;
        Boxes boxes = {staging + (warp - 4) * C::BOXES * 4096, 0};
        for (int nt = 0; nt < turns && ok; ++nt) {
            const int buf = nt % C::BUFS, use = nt / C::BUFS;
            // Where to is worked out before the wait: with one accumulator the next tile's MMAs wait for what is between it and the arrival.  All of a
            // thread's columns are read at once, with two accumulators, too: 32 at a time, each waited for, took 2.6 times as long a tile.
            const uint32_t ta = tmem + buf * C::ACC + ((uint32_t)(quad * 32) << 16), drained = in_cta(s32(&tempty[buf]), leader);
            pair_tile(p, nt < own ? first + nt * step : split, m, n, which);
            const int row0 = m * 256 + (int)rank * 128 + quad * 32, n0 = n * C::NOUT;
            ok = warp_all(mb_wait(&tfull[buf], (uint32_t)use & 1u, p.status, kWaitAcc));
            if (!ok) break;
            tc_fence_after();
            float v[4][32];
            if (nt < own) {
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(ta + (C::GATED ? (c & 2 ? 128 : 0) + half * 64 + 32 * (c & 1) : half * 128 + 32 * c), v[c]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && nt + C::BUFS < turns) remote_arrive(drained);  // where a later tile waits for it
            }
            if (nt == own) {  // the ring is empty: every copy has landed and been read
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    tmem_ld32(ta + half * 128 + 32 * c, v[0]);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<float4*>(smem + share_at(quad * 32 + lane, half * 32 + c * 8 + i)) =
                            make_float4(v[0][4 * i], v[0][4 * i + 1], v[0][4 * i + 2], v[0][4 * i + 3]);
                }
                break;
            }
            switch (p.out_type) {
                case T_F16: results<C, T_F16>(p, which, row0, n0, half, boxes, lane, v); break;
                case T_BF16: results<C, T_BF16>(p, which, row0, n0, half, boxes, lane, v); break;
                case T_F32: if constexpr (C::FP4) results<C, T_F32>(p, which, row0, n0, half, boxes, lane, v); break;
                default: if constexpr (C::FP4 && C::GATED) results<C, T_MXFP4>(p, which, row0, n0, half, boxes, lane, v);
            }
        }
        __syncwarp();
        if (shares) {  // the whole cluster: those of the other warps wait below
            cluster_sync();
            pair_tile(p, split, m, n, which);
            const int row0 = m * 256 + (int)rank * 128, n0 = n * C::NOUT;
            const uint32_t sums = s32(smem);
            switch (p.out_type) {
                case T_F16: joined<C, T_F16>(p, which, part, warp - 4, row0, n0, sums, rank, boxes, lane); break;
                case T_BF16: joined<C, T_BF16>(p, which, part, warp - 4, row0, n0, sums, rank, boxes, lane); break;
                case T_F32: if constexpr (C::FP4) joined<C, T_F32>(p, which, part, warp - 4, row0, n0, sums, rank, boxes, lane); break;
                default: if constexpr (C::FP4 && C::GATED) joined<C, T_MXFP4>(p, which, part, warp - 4, row0, n0, sums, rank, boxes, lane);
            }
        }
        if (lane == 0) store_read<0>();  // the boxes have been read
    }
    __syncwarp();
    tc_fence_before();
    // Nobody's shared or tensor memory goes while another may still use it: reads are over, and every arrival at another CTA's barrier has been waited for.
    cluster_leave();
    if (warp == 1) {
        tc_fence_after();
        pair_free(tmem);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------------
// Scale tiles of `rows` rows, as a matrix of 512-byte rows; boxes of two.
inline int scale_map(CUtensorMap* m, const void* scales, uint64_t rows, uint64_t k) {
    return tiled_map(m, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, scales, (rows + 127) / 128 * ((k + 127) / 128), 128, 512, 2, 128, CU_TENSOR_MAP_SWIZZLE_NONE);
}
// Results [rows][cols] of `type`, in the epilogue's boxes, rows of 128 bytes or (16-bit ones) 64.
inline int result_map(CUtensorMap* m, int type, const void* out, uint64_t rows, uint64_t cols, uint64_t ld, int bytes = 128) {
    const bool f32 = type == T_F32;
    return tiled_map(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, f32 ? 4 : 2, out, rows,
                     cols, ld * (f32 ? 4 : 2), 32, bytes / (f32 ? 4 : 2), bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

template <class C>
cudaLaunchConfig_t pair_config(dnb_ctx* c, cudaLaunchAttribute (&at)[2], unsigned grid, int parts) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(PAIR_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = c->stream;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2 * parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = c->use_pdl;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cfg;
}
// p: M, N, K, passes, both, type, act, outp, out_scales, ldo; maps of scales and pre where there are any.
template <class C>
int launch_pair(dnb_ctx* c, Params& p, const Operand* a, int na, const Operand* b, int nb, int type, const char* name) {
    int rc;
    for (int i = 0; i < na; ++i)
        if ((rc = operand_map<C::FP4>(&p.a[i], a[i], C::AMN ? 64 : 128, type))) return rc;
    for (int i = 0; i < nb; ++i)
        if ((rc = operand_map<C::FP4>(&p.b[i], b[i], C::BMN ? 64 : 128, type))) return rc;
    const int es = p.out_type == T_F32 ? 4 : 2;
    // Rows that end inside 16 bytes would be written to their end.
    p.tma_out = p.out_type != T_MXFP4 && p.ldo * es % 16 == 0 && (size_t)p.N * es % 16 == 0;
    for (int i = 0; i < p.both; ++i) p.tma_out = p.tma_out && ((uintptr_t)p.outp[i] & 15) == 0;
    if (p.tma_out)
        for (int i = 0; i < p.both; ++i)
            if ((rc = result_map(&p.out[i], p.out_type, p.outp[i], p.M, p.N, p.ldo))) return rc;
    p.idesc_type = type == T_BF16;
    p.status = c->status;
    p.tiles_m = (p.M + 255) / 256;
    const int tiles_n = (p.N + C::NOUT - 1) / C::NOUT;
    const int64_t tiles = (int64_t)p.tiles_m * tiles_n * p.both;
    if (tiles > 0x3fffffff) {
        set_error("%s: %d x %d results are more than one launch takes", name, p.M, p.N);
        return DNB_DECLINED;
    }
    p.per_output = p.tiles_m * tiles_n;
    p.tiles = (int)tiles;
    p.chunks = (p.K + C::BK - 1) / C::BK * p.passes;
    p.group = divisor(8 * tiles_n);
    p.last_group = divisor(p.tiles_m % 8 ? p.tiles_m % 8 : 8);
    static SmemGrant grant;
    DNB_CUDA(grant_smem(grant, c->device, pair_kernel<C>, C::SMEM));
    static std::atomic<int> known[64][5];
    int at_once[5];
    cudaLaunchAttribute at[2];
    for (int s = 1; s <= 4; ++s) at_once[s] = clusters_at_once(known[c->device][s], pair_kernel<C>, pair_config<C>(c, at, 2 * s, s));
    if (at_once[1] < 1) at_once[1] = 1;  // one pair takes the tiles in turn, if any can be launched
    const PairPlan plan = pair_plan(at_once, p.tiles, p.chunks);
    p.parts = plan.parts;
    p.whole = plan.whole;
    p.each = plan.each;
    p.more = plan.more;
    for (int i = 0; i < p.both; ++i)
        if (p.parts > 1 && p.tma_out && p.out_type != T_F32 && (rc = result_map(&p.narrow[i], p.out_type, p.outp[i], p.M, p.N, p.ldo, 64))) return rc;
    for (int i = 0; i <= p.parts; ++i) p.share[i] = (int)((int64_t)p.chunks * i / p.parts);
    ProfScope prof_(c, c->stream, name);
    const cudaLaunchConfig_t cfg = pair_config<C>(c, at, 2u * (unsigned)plan.pairs, p.parts);
    DNB_CUDA(cudaLaunchKernelEx(&cfg, pair_kernel<C>, p));
    c->launches++;
    return DNB_OK;
}

}  // namespace dp
}  // namespace dnb
