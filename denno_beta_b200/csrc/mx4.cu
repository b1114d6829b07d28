// Microscaled 4-bit matrices: rows to 4 bits and back, and products of two of them on the tensor cores (dense_tc.cuh).
//
// A matrix is two arrays.  codes [rows][k / 2]: e2m1 numbers, element 2 i in the low half of byte i: the order in which tcgen05 takes them
// from swizzled shared memory, so that TMA moves them as they are.  scales: a byte for each 32 elements of a row, 2^(byte - 127), in tiles of
// 128 rows x 4 scales of 512 bytes: the order in which tcgen05.cp puts them into tensor memory.  (A GGUF file has both in one block of 17
// bytes, which neither could take.)
#include "dense_pair.cuh"

namespace dnb {
namespace mx {
using namespace dt;
using dt::Cfg;
using dt::Params;

// A thread takes 8 elements of the rows r, r + 32, r + 64 and r + 96 of a tile of scales, 16 threads (half a warp) its 128 columns: four independent
// 16- or 32-byte loads in flight a thread, and the 16 bytes of scales that these rows have next to each other are one store.  A block of 32 is four
// neighbouring lanes.  Bound by memory: 14018 x 4096, fp32 to 4 bits 40 us (6.5 TB/s), bf16 26.1 (5.6) and back 23.5 (6.2; a row a thread at a time, 64-bit
// divisions and a branch at each load, which waited for it: 47 and 37).  A file's blocks, whose 17 bytes start anywhere, 23 (2.6): nine
// loads of a byte a piece bound it; weights go through it once, as they are loaded.
constexpr int THREADS = 256, UNITS = THREADS / 16;

// Where a thread is: unit u = folded row * nkb + kb, a folded row being 32 * tile + r.  Advanced without a division.  Fewer than 2^31 units (check_units).
struct Walk {
    uint32_t u, units;
    size_t row;  // the first of the four
    int kb, nkb, dkb;
    uint32_t dq, q;
    __device__ Walk(uint32_t folded, int nkb_) : u(blockIdx.x * UNITS + (threadIdx.x >> 4)), units(folded * nkb_), nkb(nkb_) {
        const uint32_t step = gridDim.x * UNITS;
        q = u / (uint32_t)nkb; kb = (int)(u - q * nkb); dq = step / (uint32_t)nkb; dkb = (int)(step - dq * nkb);
        place();
    }
    __device__ void place() { row = (size_t)(q >> 5) * 128 + (q & 31); }
    __device__ bool warp_in() const { return u - ((threadIdx.x >> 4) & 1) < units; }  // the first of the warp's two units
    __device__ void next() {
        u += gridDim.x * UNITS;
        q += dq;
        kb += dkb;
        if (kb >= nkb) kb -= nkb, ++q;
        place();
    }
};
static int tiles_along(int k) { return (k - 1) / 128 + 1; }  // of scales
static size_t folded_rows(int rows) { return (size_t)(rows / 128) * 32 + (rows % 128 < 32 ? rows % 128 : 32); }

template <int T> struct Num { using type = float; };
template <> struct Num<T_F16> { using type = __half; };
template <> struct Num<T_BF16> { using type = __nv_bfloat16; };

// Eight elements as loaded (rows may start anywhere; WHOLE: at multiples of 16 bytes), and as numbers.
template <int T> struct Raw { uint32_t w[T == T_F32 ? 8 : 4]; };
template <int T, bool WHOLE>
__device__ __forceinline__ Raw<T> load8(const void* x, size_t at) {
    Raw<T> r;
    if constexpr (WHOLE) {
        const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const typename Num<T>::type*>(x) + at);
#pragma unroll
        for (int i = 0; i < (T == T_F32 ? 2 : 1); ++i) {
            const uint4 v = s[i];
            r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (T == T_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(x)[at + i];
    } else {
        const uint16_t* s = reinterpret_cast<const uint16_t*>(x) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
    }
    return r;
}
template <int T>
__device__ __forceinline__ void numbers(const Raw<T>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == T_F32) {
            v[2 * i] = __uint_as_float(r.w[2 * i]);
            v[2 * i + 1] = __uint_as_float(r.w[2 * i + 1]);
        } else if constexpr (T == T_BF16) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
// Bits, as fp32, of the largest magnitudes of four rows' blocks (four neighbouring lanes).  16-bit magnitudes are compared two rows a word.
template <int T>
__device__ __forceinline__ void block_max(const Raw<T> (&r)[4], uint32_t (&mx)[4]) {
    if constexpr (T == T_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mx[i] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) mx[i] = max(mx[i], r[i].w[j] & 0x7fffffffu);
            mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        }
    } else {
        uint32_t m[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = __vmaxu2(__vmaxu2(r[i].w[0] & 0x7fff7fffu, r[i].w[1] & 0x7fff7fffu), __vmaxu2(r[i].w[2] & 0x7fff7fffu, r[i].w[3] & 0x7fff7fffu));
            m[i] = max(a & 0xffffu, a >> 16);
        }
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            uint32_t two = m[i] | m[i + 1] << 16;
            two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 1));
            two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 2));
            if constexpr (T == T_BF16) {
                mx[i] = two << 16;
                mx[i + 1] = two & 0xffff0000u;
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
                mx[i] = __float_as_uint(f.x);
                mx[i + 1] = __float_as_uint(f.y);
            }
        }
    }
}

// Eight elements as they lie in a GGUF file's blocks: the scale's byte, then 16 bytes with elements 0 to 15 in their low halves and 16 to 31 in the
// high ones.
__device__ __forceinline__ void file_piece(const uint8_t* b, int at, uint32_t& code, uint32_t& e) {
    const int first = at & 15, high = at & 16 ? 4 : 0;
    e = b[0];
    code = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) code |= (uint32_t)((b[1 + first + i] >> high) & 15) << (4 * i);
}

template <int T, bool WHOLE>
__global__ void __launch_bounds__(THREADS)
quantize_kernel(const void* __restrict__ x, size_t ldx, int rows, uint32_t folded, int k, int nkb, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 15;
    const size_t apart = (size_t)16 * k;  // bytes of codes from one of the four rows to the next
    for (Walk w(folded, nkb); w.warp_in(); w.next()) {
        const int at = w.kb * 128 + lane * 8;
        const bool col = w.u < w.units && at < k;
        const int here = col ? (int)min((size_t)4, ((size_t)rows - w.row + 31) / 32) : 0;  // of the four rows
        uint32_t code[4], e[4];
        if constexpr (T == T_MXFP4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                code[i] = e[i] = 0;
                if (i < here) file_piece(reinterpret_cast<const uint8_t*>(x) + ((w.row + 32 * i) * ldx + at) / 32 * 17, at, code[i], e[i]);
            }
        } else {
            Raw<T> r[4] = {};
            const size_t first = w.row * ldx + at;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < here) r[i] = load8<T, WHOLE>(x, first + (size_t)(32 * i) * ldx);
            block_max<T>(r, e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[8];
                numbers<T>(r[i], v);
                e[i] = scale_byte(e[i]);
                code[i] = e2m1_eight(v, scale_inverse(e[i]));
                if (e[i] == 255) code[i] = 0;
                if (!col) e[i] = 0;
            }
        }
        uint8_t* to = codes + (w.row * k + at) / 2;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < here) *reinterpret_cast<uint32_t*>(to + i * apart) = code[i];
        // Four lanes' bytes of four rows to a word a row.
        const uint32_t b0 = e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24, b1 = __shfl_down_sync(0xffffffffu, b0, 4, 16),
                       b2 = __shfl_down_sync(0xffffffffu, b0, 8, 16), b3 = __shfl_down_sync(0xffffffffu, b0, 12, 16);
        if (lane == 0 && here > 0) {
            const uint32_t p = __byte_perm(b0, b1, 0x5140), q = __byte_perm(b2, b3, 0x5140), r = __byte_perm(b0, b1, 0x7362), t = __byte_perm(b2, b3, 0x7362);
            const uint32_t word[4] = {__byte_perm(p, q, 0x5410), __byte_perm(p, q, 0x7632), __byte_perm(r, t, 0x5410), __byte_perm(r, t, 0x7632)};
            uint32_t* s = reinterpret_cast<uint32_t*>(scales + scale_at(w.row, 4 * w.kb, nkb));
            if (here == 4) {
                *reinterpret_cast<uint4*>(s) = make_uint4(word[0], word[1], word[2], word[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (i < here) s[i] = word[i];
            }
        }
    }
}

// Four codes (16 bits) as numbers.
__device__ __forceinline__ void four_values(uint32_t code, float s, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h2;
        asm("{\n\t.reg .b8 b, z;\n\tmov.b16 {b, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h2) : "h"((uint16_t)((code >> (8 * i)) & 0xff)));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        v[2 * i] = f.x * s;
        v[2 * i + 1] = f.y * s;
    }
}

// 16 bytes of results a store, neighbouring lanes next to each other: 8 elements a lane, or (F32) 4 of each half of the 128 columns.
template <int T, bool WHOLE>
__global__ void __launch_bounds__(THREADS)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, uint32_t folded, int k, int nkb, void* __restrict__ out, size_t ldo) {
    pdl_wait();
    pdl_launch_dependents();
    using N = typename Num<T>::type;
    constexpr int EACH = T == T_F32 ? 4 : 8, PIECES = 8 / EACH;
    const int lane = threadIdx.x & 15;
    const size_t apart = (size_t)16 * k;
    for (Walk w(folded, nkb); w.u < w.units; w.next()) {
        const int here = (int)min((size_t)4, ((size_t)rows - w.row + 31) / 32);
        uint32_t code[PIECES][4];
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
            const int at = w.kb * 128 + 64 * h + lane * EACH;
            const uint8_t* from = codes + (w.row * k + at) / 2;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= here || at >= k) code[h][i] = 0;
                else if constexpr (T == T_F32) code[h][i] = *reinterpret_cast<const uint16_t*>(from + i * apart);
                else code[h][i] = *reinterpret_cast<const uint32_t*>(from + i * apart);
            }
        }
        const uint4 s4 = *reinterpret_cast<const uint4*>(scales + scale_at(w.row, 4 * w.kb, nkb));  // rows past the last: read, not used
        const uint32_t word[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int h = 0; h < PIECES; ++h) {
            const int in = 64 * h + lane * EACH, at = w.kb * 128 + in;
            N* to = reinterpret_cast<N*>(out) + w.row * ldo + at;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (r >= here || at >= k) continue;
                const uint32_t e = (word[r] >> (8 * (in >> 5))) & 255u;
                const float s = __uint_as_float(e == 255 ? 0x7fc00000u : e ? e << 23 : 0x00400000u);
                N* d = to + (size_t)(32 * r) * ldo;
                alignas(16) N v[EACH];
#pragma unroll
                for (int i = 0; i < EACH / 4; ++i) {
                    float f[4];
                    four_values(code[h][r] >> (16 * i), s, f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) put<T>(v, 4 * i + j, f[j]);
                }
                if constexpr (WHOLE) {
                    *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(v);
                } else {
#pragma unroll
                    for (int i = 0; i < EACH; ++i) d[i] = v[i];
                }
            }
        }
    }
}

// Blocks an SM, more than fit at once (5 and 8), so that the SMs end together; us for 14018 x 4096 bf16 with 4, 8, 16, 48 an SM: to 4 bits 31.2, 26.7, 26.1,
// 28.3, back 27.1, 27.7, 26.0, 23.5.
constexpr int TO_FOUR_BITS = 16, BACK = 48;
static unsigned grid_of(const dnb_ctx* c, size_t units, int an_sm) {
    const size_t want = (units + UNITS - 1) / UNITS, most = (size_t)c->sm_count * an_sm;
    return (unsigned)(want < most ? want : most);
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static int elem_size(int type) { return type == T_F32 ? 4 : type == T_F16 || type == T_BF16 ? 2 : 0; }
static bool float_type(int type) { return elem_size(type) != 0; }

// What the checks of all entry points of this file have in common.
static int check_matrix(const char* what, const void* codes, const void* scales, int rows, int k) {
    if (rows < 0 || k < 1 || (rows > 0 && (!codes || !scales))) {
        set_error("%s: bad argument (rows %d, k %d)", what, rows, k);
        return DNB_ERR_ARG;
    }
    if (k % 32) {
        set_error("%s: k=%d is not a whole number of blocks of 32", what, k);
        return DNB_DECLINED;
    }
    if (!aligned16(codes) || !aligned16(scales)) {
        set_error("%s: codes and scales start at multiples of 16 bytes", what);
        return DNB_DECLINED;
    }
    return DNB_OK;
}

// Sizes that tiles are counted for in 32 bits, and sums that a wait outlasts.
static int check_sizes(const char* what, int nt, int k, int n) {
    if (nt <= 1 << 30 && k <= kMostChunks * 256 && n <= 1 << 30) return DNB_OK;
    set_error("%s: %d x %d x %d is more than one launch takes (k up to 2^27)", what, nt, k, n);
    return DNB_DECLINED;
}

// Units that Walk counts: a launch's worth of rows (half a terabyte of codes and more).
static int check_units(const char* what, int rows, int k) {
    if (folded_rows(rows) * tiles_along(k) < (size_t)1 << 31) return DNB_OK;
    set_error("%s: %d rows of %d are more than one launch takes", what, rows, k);
    return DNB_DECLINED;
}

// One product (NA 1) or the gated one (2).  Up to 128 tokens: narrow tiles of tokens under the weights' rows (dense_tc.cuh); beyond, tiles of
// 256 tokens (dense_pair.cuh).
template <int NA>
static int product(dnb_ctx* c, const void* xc, const void* xs, const void* const* wc, const void* const* ws, int nt, int k, int n, int act, int type, void* out,
                   uint8_t* out_scales, size_t ldo, const char* name) {
    const uint64_t K = k, N = n;
    const Operand w[2] = {{wc[0], N, K, K / 2}, {wc[NA - 1], N, K, K / 2}}, x = {xc, (uint64_t)nt, K, K / 2};
    if (nt <= 128) {
        Params p = {};
        p.M = n; p.N = nt; p.K = k;
        p.passes = 1;
        p.sa[0] = (const uint8_t*)ws[0];
        p.sa[1] = (const uint8_t*)ws[NA - 1];
        p.sb = (const uint8_t*)xs;
        p.out = out;
        p.out_scales = out_scales;
        p.out_type = type;
        p.ldo = ldo;
        p.act = act;
        if (nt <= 16) return launch_dense<Cfg<true, NA, 16>>(c, p, w, NA, &x, 1, 0, name);
        if (nt <= 32) return launch_dense<Cfg<true, NA, 32>>(c, p, w, NA, &x, 1, 0, name);
        if (nt <= 64) return launch_dense<Cfg<true, NA, 64>>(c, p, w, NA, &x, 1, 0, name);
        return launch_dense<Cfg<true, NA, 128>>(c, p, w, NA, &x, 1, 0, name);
    }
    dp::Params p = {};
    p.M = nt; p.N = n; p.K = k;
    p.passes = p.both = 1;
    p.outp[0] = out;
    p.out_scales = out_scales;
    p.out_type = type;
    p.ldo = ldo;
    p.act = act;
    int rc = dp::scale_map(&p.sa, xs, nt, k);
    for (int i = 0; i < 2 && !rc; ++i) rc = dp::scale_map(&p.sb[i], ws[i < NA ? i : 0], n, k);
    return rc ? rc : dp::launch_pair<dp::Cfg<true, NA == 2>>(c, p, &x, 1, w, NA, 0, name);
}

}  // namespace mx
}  // namespace dnb

using namespace dnb;
using namespace dnb::mx;

extern "C" {

int dnb_mx4_bytes(int rows, int k, size_t* codes, size_t* scales) {
    if (rows < 0 || k < 1 || !codes || !scales) return DNB_ERR_ARG;
    if (k % 32) {
        set_error("mx4_bytes: k=%d is not a whole number of blocks of 32", k);
        return DNB_DECLINED;
    }
    *codes = (size_t)rows * k / 2;
    *scales = ((size_t)rows + 127) / 128 * tiles_along(k) * 512;
    return DNB_OK;
}

int dnb_mx4_quantize_dev(dnb_ctx* c, int type, const void* x_dev, size_t ldx, int rows, int k, void* codes_dev, void* scales_dev) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_matrix("mx4_quantize", codes_dev, scales_dev, rows, k);
    if (rc) return rc;
    if ((rows > 0 && !x_dev) || ldx < (size_t)k) {
        set_error("mx4_quantize: bad argument (x %p, ldx %zu, k %d)", x_dev, ldx, k);
        return DNB_ERR_ARG;
    }
    const int es = elem_size(type);
    if ((!es && type != T_MXFP4) || (type == T_MXFP4 && ldx % 32) || (es && (uintptr_t)x_dev % es)) {
        set_error("mx4_quantize: rows of ggml type %d, %zu elements apart, are not handled", type, ldx);
        return DNB_DECLINED;
    }
    if ((rc = check_units("mx4_quantize", rows, k)) || rows == 0) return rc;
    DNB_CUDA(cudaSetDevice(c->device));
    const int nkb = tiles_along(k);
    const size_t folded = folded_rows(rows);
    const dim3 grid(grid_of(c, folded * nkb, TO_FOUR_BITS)), block(THREADS);
    const bool whole = aligned16(x_dev) && ldx * es % 16 == 0;
    uint8_t *codes = (uint8_t*)codes_dev, *scales = (uint8_t*)scales_dev;
    ProfScope prof_(c, c->stream, "mx4_quantize");
#define QUANTIZE(T) (whole ? launch_k(quantize_kernel<T, true>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, rows, folded, k, nkb, codes, scales) \
                           : launch_k(quantize_kernel<T, false>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, rows, folded, k, nkb, codes, scales))
    DNB_CUDA(type == T_F32 ? QUANTIZE(T_F32) : type == T_F16 ? QUANTIZE(T_F16) : type == T_BF16 ? QUANTIZE(T_BF16)
             : launch_k(quantize_kernel<T_MXFP4, false>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, rows, folded, k, nkb, codes, scales));
#undef QUANTIZE
    c->launches++;
    return DNB_OK;
}

int dnb_mx4_dequantize_dev(dnb_ctx* c, const void* codes_dev, const void* scales_dev, int rows, int k, int type, void* out_dev, size_t ldo) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_matrix("mx4_dequantize", codes_dev, scales_dev, rows, k);
    if (rc) return rc;
    if ((rows > 0 && !out_dev) || ldo < (size_t)k) {
        set_error("mx4_dequantize: bad argument (out %p, ldo %zu, k %d)", out_dev, ldo, k);
        return DNB_ERR_ARG;
    }
    const int es = elem_size(type);
    if (!es || (uintptr_t)out_dev % es) {
        set_error("mx4_dequantize: results of ggml type %d are not handled", type);
        return DNB_DECLINED;
    }
    if ((rc = check_units("mx4_dequantize", rows, k)) || rows == 0) return rc;
    DNB_CUDA(cudaSetDevice(c->device));
    const int nkb = tiles_along(k);
    const size_t folded = folded_rows(rows);
    const dim3 grid(grid_of(c, folded * nkb, BACK)), block(THREADS);
    const bool whole = aligned16(out_dev) && ldo * es % 16 == 0;
    const uint8_t *codes = (const uint8_t*)codes_dev, *scales = (const uint8_t*)scales_dev;
    ProfScope prof_(c, c->stream, "mx4_dequantize");
#define DEQUANTIZE(T) (whole ? launch_k(dequantize_kernel<T, true>, grid, block, 0, c->stream, c->use_pdl, codes, scales, rows, folded, k, nkb, out_dev, ldo) \
                             : launch_k(dequantize_kernel<T, false>, grid, block, 0, c->stream, c->use_pdl, codes, scales, rows, folded, k, nkb, out_dev, ldo))
    DNB_CUDA(type == T_F32 ? DEQUANTIZE(T_F32) : type == T_F16 ? DEQUANTIZE(T_F16) : DEQUANTIZE(T_BF16));
#undef DEQUANTIZE
    c->launches++;
    return DNB_OK;
}

int dnb_mx4_gemm_dev(dnb_ctx* c, const void* xc, const void* xs, const void* wc, const void* ws, int nt, int k, int n, int type, void* out_dev, size_t ldo) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_matrix("mx4_gemm", xc, xs, nt, k);
    if (!rc) rc = check_matrix("mx4_gemm", wc, ws, n, k);
    if (rc) return rc;
    if (n < 1 || (nt > 0 && !out_dev) || ldo < (size_t)n) {
        set_error("mx4_gemm: bad argument (out %p, ldo %zu, n %d)", out_dev, ldo, n);
        return DNB_ERR_ARG;
    }
    if (!float_type(type) || (uintptr_t)out_dev % elem_size(type)) {
        set_error("mx4_gemm: results of ggml type %d are not handled", type);
        return DNB_DECLINED;
    }
    if ((rc = check_sizes("mx4_gemm", nt, k, n)) || nt == 0) return rc;
    DNB_CUDA(cudaSetDevice(c->device));
    return product<1>(c, xc, xs, &wc, &ws, nt, k, n, ACT_NONE, type, out_dev, nullptr, ldo, "mx4_gemm");
}

int dnb_mx4_gated_dev(dnb_ctx* c, int act, const void* xc, const void* xs, const void* gc, const void* gs, const void* uc, const void* us, int nt, int k,
                      int n, int type, void* out_dev, void* out_scales_dev, size_t ldo) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_matrix("mx4_gated", xc, xs, nt, k);
    if (!rc) rc = check_matrix("mx4_gated", gc, gs, n, k);
    if (!rc) rc = check_matrix("mx4_gated", uc, us, n, k);
    if (rc) return rc;
    const bool four = type == T_MXFP4;
    if (n < 1 || (act != ACT_SILU && act != ACT_GELU) || (nt > 0 && !out_dev) || (nt > 0 && four && !out_scales_dev) || (!four && ldo < (size_t)n)) {
        set_error("mx4_gated: bad argument (activation %d, out %p, ldo %zu, n %d)", act, out_dev, ldo, n);
        return DNB_ERR_ARG;
    }
    if (four ? n % 32 || !aligned16(out_dev) || !aligned16(out_scales_dev) : !float_type(type) || (uintptr_t)out_dev % elem_size(type)) {
        set_error("mx4_gated: results of ggml type %d, %d a row, are not handled", type, n);
        return DNB_DECLINED;
    }
    if ((rc = check_sizes("mx4_gated", nt, k, n)) || nt == 0) return rc;
    DNB_CUDA(cudaSetDevice(c->device));
    const void *wc[2] = {gc, uc}, *ws[2] = {gs, us};
    return product<2>(c, xc, xs, wc, ws, nt, k, n, act, type, out_dev, (uint8_t*)out_scales_dev, ldo, "mx4_gated");
}

}  // extern "C"
