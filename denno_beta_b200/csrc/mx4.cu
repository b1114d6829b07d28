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

// 16 threads a unit of 128 elements of a row (a scale tile's width), 8 elements a thread; a block of 32 is four neighbouring lanes.
constexpr int UNIT_THREADS = 16, THREADS = 256, UNITS = THREADS / UNIT_THREADS;

template <int T> struct Num { using type = float; };
template <> struct Num<T_F16> { using type = __half; };
template <> struct Num<T_BF16> { using type = __nv_bfloat16; };

// Eight elements from `at`; whole says that the pointer is 16-byte aligned (rows may start anywhere).
template <int T>
__device__ __forceinline__ void load8(const void* x, size_t at, bool whole, float (&v)[8]) {
    if constexpr (T == T_F32) {
        const float* s = reinterpret_cast<const float*>(x) + at;
        if (whole) {
            const float4 a = reinterpret_cast<const float4*>(s)[0], b = reinterpret_cast<const float4*>(s)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = s[i];
        }
    } else {
        using N = typename Num<T>::type;
        N s[8];
        const N* src = reinterpret_cast<const N*>(x) + at;
        if (whole) {
            *reinterpret_cast<uint4*>(s) = *reinterpret_cast<const uint4*>(src);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = src[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)s[i];
    }
}

// Units u = row * nkb + kb.
template <int T>
__global__ void __launch_bounds__(THREADS)
quantize_kernel(const void* __restrict__ x, size_t ldx, bool whole, size_t units, int k, int nkb, uint8_t* __restrict__ codes,
                uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & (UNIT_THREADS - 1);
    // whole warps stay in the loop: a warp's two units are neighbours
    for (size_t u0 = (size_t)blockIdx.x * UNITS + (threadIdx.x >> 5) * 2; u0 < units; u0 += (size_t)gridDim.x * UNITS) {
        const size_t u = u0 + ((threadIdx.x >> 4) & 1);
        const size_t row = u / nkb;
        const int kb = (int)(u - row * nkb), at = kb * 128 + lane * 8;
        const bool in = u < units && at < k;
        float v[8] = {};
        if (in) load8<T>(x, row * ldx + at, whole, v);
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const uint32_t e = scale_byte(mx);
        const uint32_t code = e2m1_eight(v, scale_inverse(e));
        if (in) *reinterpret_cast<uint32_t*>(codes + (row * k + at) / 2) = e == 255 ? 0u : code;
        uint32_t s = in ? e << (8 * (lane >> 2)) : 0u;
        s |= __shfl_xor_sync(0xffffffffu, s, 4);
        s |= __shfl_xor_sync(0xffffffffu, s, 8);
        if (lane == 0 && u < units) *reinterpret_cast<uint32_t*>(scales + scale_at(row, 4 * kb, nkb)) = s;
    }
}

// Blocks of a GGUF file: the scale's byte, then 16 bytes with elements 0 to 15 in their low halves and 16 to 31 in the high ones.
__global__ void __launch_bounds__(THREADS)
relay_kernel(const uint8_t* __restrict__ blocks, size_t ldx, size_t units, int k, int nkb, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & (UNIT_THREADS - 1);
    for (size_t u0 = (size_t)blockIdx.x * UNITS + (threadIdx.x >> 5) * 2; u0 < units; u0 += (size_t)gridDim.x * UNITS) {
        const size_t u = u0 + ((threadIdx.x >> 4) & 1);
        const size_t row = u / nkb;
        const int kb = (int)(u - row * nkb), at = kb * 128 + lane * 8;
        const bool in = u < units && at < k;
        uint32_t code = 0, e = 0;
        if (in) {
            const uint8_t* b = blocks + (row * ldx + at) / 32 * 17;
            const int first = at & 15, high = at & 16 ? 4 : 0;
            e = b[0];
#pragma unroll
            for (int i = 0; i < 8; ++i) code |= (uint32_t)((b[1 + first + i] >> high) & 15) << (4 * i);
            *reinterpret_cast<uint32_t*>(codes + (row * k + at) / 2) = code;
        }
        uint32_t s = e << (8 * (lane >> 2));
        s |= __shfl_xor_sync(0xffffffffu, s, 4);
        s |= __shfl_xor_sync(0xffffffffu, s, 8);
        if (lane == 0 && u < units) *reinterpret_cast<uint32_t*>(scales + scale_at(row, 4 * kb, nkb)) = s;
    }
}

template <int T>
__global__ void __launch_bounds__(THREADS)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, size_t units, int k, int nkb, void* __restrict__ out, size_t ldo,
                  bool whole) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & (UNIT_THREADS - 1);
    for (size_t u = (size_t)blockIdx.x * UNITS + (threadIdx.x >> 4); u < units; u += (size_t)gridDim.x * UNITS) {
        const size_t row = u / nkb;
        const int kb = (int)(u - row * nkb), at = kb * 128 + lane * 8;
        if (at >= k) continue;
        const uint32_t code = *reinterpret_cast<const uint32_t*>(codes + (row * k + at) / 2);
        const uint32_t e = scales[scale_at(row, at >> 5, nkb)];
        const float s = __uint_as_float(e == 255 ? 0x7fc00000u : e ? e << 23 : 0x00400000u);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t h2;
            asm("{\n\t.reg .b8 b, z;\n\tmov.b16 {b, z}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h2) : "h"((uint16_t)((code >> (8 * i)) & 0xff)));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
            v[2 * i] = f.x * s;
            v[2 * i + 1] = f.y * s;
        }
        const size_t o = row * ldo + at;
        if constexpr (T == T_F32) {
            float* d = reinterpret_cast<float*>(out) + o;
            if (whole) {
                reinterpret_cast<float4*>(d)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(d)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = v[i];
            }
        } else {
            using N = typename Num<T>::type;
            N h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) put<T>(h, i, v[i]);
            N* d = reinterpret_cast<N*>(out) + o;
            if (whole) *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(h);
            else {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = h[i];
            }
        }
    }
}

static unsigned grid_of(const dnb_ctx* c, size_t units) {
    const size_t want = (units + UNITS - 1) / UNITS, most = (size_t)c->sm_count * 8;
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
    *scales = ((size_t)rows + 127) / 128 * ((k + 127) / 128) * 512;
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
    if (rows == 0) return DNB_OK;
    DNB_CUDA(cudaSetDevice(c->device));
    const int nkb = (k + 127) / 128;
    const size_t units = (size_t)rows * nkb;
    const dim3 grid(grid_of(c, units)), block(THREADS);
    const bool whole = aligned16(x_dev) && ldx * es % 16 == 0;
    uint8_t *codes = (uint8_t*)codes_dev, *scales = (uint8_t*)scales_dev;
    ProfScope prof_(c, c->stream, "mx4_quantize");
    switch (type) {
        case T_F32: DNB_CUDA(launch_k(quantize_kernel<T_F32>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, whole, units, k, nkb, codes, scales)); break;
        case T_F16: DNB_CUDA(launch_k(quantize_kernel<T_F16>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, whole, units, k, nkb, codes, scales)); break;
        case T_BF16: DNB_CUDA(launch_k(quantize_kernel<T_BF16>, grid, block, 0, c->stream, c->use_pdl, x_dev, ldx, whole, units, k, nkb, codes, scales)); break;
        default: DNB_CUDA(launch_k(relay_kernel, grid, block, 0, c->stream, c->use_pdl, (const uint8_t*)x_dev, ldx, units, k, nkb, codes, scales));
    }
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
    if (rows == 0) return DNB_OK;
    DNB_CUDA(cudaSetDevice(c->device));
    const int nkb = (k + 127) / 128;
    const size_t units = (size_t)rows * nkb;
    const dim3 grid(grid_of(c, units)), block(THREADS);
    const bool whole = aligned16(out_dev) && ldo * es % 16 == 0;
    const uint8_t *codes = (const uint8_t*)codes_dev, *scales = (const uint8_t*)scales_dev;
    ProfScope prof_(c, c->stream, "mx4_dequantize");
    switch (type) {
        case T_F32: DNB_CUDA(launch_k(dequantize_kernel<T_F32>, grid, block, 0, c->stream, c->use_pdl, codes, scales, units, k, nkb, out_dev, ldo, whole)); break;
        case T_F16: DNB_CUDA(launch_k(dequantize_kernel<T_F16>, grid, block, 0, c->stream, c->use_pdl, codes, scales, units, k, nkb, out_dev, ldo, whole)); break;
        default: DNB_CUDA(launch_k(dequantize_kernel<T_BF16>, grid, block, 0, c->stream, c->use_pdl, codes, scales, units, k, nkb, out_dev, ldo, whole));
    }
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
    if (nt == 0) return DNB_OK;
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
    if (nt == 0) return DNB_OK;
    DNB_CUDA(cudaSetDevice(c->device));
    const void *wc[2] = {gc, uc}, *ws[2] = {gs, us};
    return product<2>(c, xc, xs, wc, ws, nt, k, n, act, type, out_dev, (uint8_t*)out_scales_dev, ldo, "mx4_gated");
}

}  // extern "C"
