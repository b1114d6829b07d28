// The gated feed-forward block on 16-bit operands: out = act(x G^T) * (x U^T), both projections, the activation and the product in one
// kernel, and its backward pass (dense_tc.cuh).
//
//   g = x G^T, u = x U^T, out = act(g) u
//   du = dout act(g),  dg = dout u act'(g)                      gradients_kernel
//   dx = dg G + du U                                            one launch: the sum over features goes on from gate to up
//   dG = dg^T x,  dU = du^T x                                   one launch: two outputs
// No operand is transposed in memory: the tensor core takes G, U, x, dg and du from shared memory with either index innermost.
// Kept from the forward pass are g and u, in 32 bits: rounded to 16, dg and du would be off by twice their own rounding.
// dg and du are rounded to the operands' type, as the tensor cores take them; all sums are 32 bits.
#include "dense_pair.cuh"

namespace dnb {
namespace gt {
using namespace dt;
using dt::Cfg;
using dt::Params;

// With p = 1 / (1 + exp(-z)): act = g p, act' = p + g p (1 - p) z'.  p and 1 - p from h (act_of), so that neither cancels nor vanishes.
__device__ __forceinline__ void act_and_slope(ActForm f, float g, float& a, float& slope) {
    const float s = act_square(g), h = power_of_two(-fabsf(g * fmaf(f.c1, s, f.c0))), big = reciprocal(fmaf(h, h, 1.f)), small = big * h * h;
    const float p = g < 0.f ? small : big, rest = g < 0.f ? big : small;
    a = g * p;
    slope = fmaf(a * rest, fmaf(3.f * f.c1, s, f.c0) * kTwoLn2, p);
}

// Eight features a thread: pre [2][nt][n] fp32, dout rows ldd apart, dpre [2][nt][n].  Memory: 4096 x 10240 in bf16, 587 MB, 84 us,
// 7.0 TB/s: 420 MB read and 137 written while it runs, the last 31 stay in L2; that is 6.7 of DRAM, above a copy's 6.5, as three quarters are reads.
// 1024 x 5632 8.2, 77 x 5640 2.2.  With 8 blocks an SM that go on in strides a tenth longer (95 and 12.6 where this form took 84 and 10.9).
template <int T>
__global__ void __launch_bounds__(256)
gradients_kernel(int act_id, const float* __restrict__ pre, const void* __restrict__ dout, size_t ldd, int nt, int n, void* __restrict__ dpre) {
    pdl_wait();
    pdl_launch_dependents();
    const ActForm act = act_form(act_id);
    const size_t per = n / 8, all = per * nt, plane = (size_t)nt * n;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= all) return;
    const size_t t = i / per, at = (i - t * per) * 8;
    float g[8], u[8];
    const float4* gp = reinterpret_cast<const float4*>(pre + t * n + at);
    const float4* up = reinterpret_cast<const float4*>(pre + plane + t * n + at);
    *reinterpret_cast<float4*>(g) = gp[0];
    *reinterpret_cast<float4*>(g + 4) = gp[1];
    *reinterpret_cast<float4*>(u) = up[0];
    *reinterpret_cast<float4*>(u + 4) = up[1];
    const uint4 raw = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(dout) + t * ldd + at);
    uint4 og, ou;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint16_t b = reinterpret_cast<const uint16_t*>(&raw)[j];
        const float d = T == T_BF16 ? __bfloat162float(__ushort_as_bfloat16(b)) : __half2float(__ushort_as_half(b));
        float a, slope;
        act_and_slope(act, g[j], a, slope);
        put<T>(&og, j, d * u[j] * slope);
        put<T>(&ou, j, d * a);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dpre) + t * n + at) = og;
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(dpre) + plane + t * n + at) = ou;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The checks that both directions share: type, activation, sizes.
static int check_shape(const char* what, int act, int type, int nt, int k, int n) {
    if (nt < 0 || k < 1 || n < 1 || (act != ACT_SILU && act != ACT_GELU)) {
        set_error("%s: bad argument (activation %d, tokens %d, k %d, n %d)", what, act, nt, k, n);
        return DNB_ERR_ARG;
    }
    if ((type != T_F16 && type != T_BF16) || k % 8 || n % 8 || nt > 1 << 30 || k > 1 << 30 || n > 1 << 30) {
        set_error("%s: ggml type %d with %d tokens, k=%d, n=%d is not handled (F16 or BF16, k and n multiples of 8, up to 2^30)", what, type, nt, k, n);
        return DNB_DECLINED;
    }
    return DNB_OK;
}
// A sum that a wait outlasts (64 a chunk).
static int check_sum(const char* what, const char* over, int64_t terms) {
    if (terms <= (int64_t)kMostChunks * 64) return DNB_OK;
    set_error("%s: a sum over %lld %s is more than one launch takes (2^25)", what, (long long)terms, over);
    return DNB_DECLINED;
}
// Rows of a matrix that TMA or 16-byte loads take.
static int check_rows(const char* what, const char* name, const void* p, size_t ld, int cols) {
    if (!p || ld < (size_t)cols) {
        set_error("%s: %s is missing, or its rows of %d are %zu apart", what, name, cols, ld);
        return DNB_ERR_ARG;
    }
    if (!aligned16(p) || ld % 8) {
        set_error("%s: rows of %s start at multiples of 16 bytes", what, name);
        return DNB_DECLINED;
    }
    return DNB_OK;
}

}  // namespace gt
}  // namespace dnb

using namespace dnb;
using namespace dnb::gt;

extern "C" {

int dnb_gated_dev(dnb_ctx* c, int act, int type, const void* x_dev, size_t ldx, const void* gate_dev, const void* up_dev, int nt, int k, int n, void* out_dev,
                  size_t ldo, float* pre_dev) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_shape("gated", act, type, nt, k, n);
    if (rc || (rc = check_sum("gated", "elements of a row", k)) || nt == 0) return rc;
    if ((rc = check_rows("gated", "x", x_dev, ldx, k))) return rc;
    if ((rc = check_rows("gated", "gate", gate_dev, k, k))) return rc;
    if ((rc = check_rows("gated", "up", up_dev, k, k))) return rc;
    if (!out_dev || ldo < (size_t)n) {
        set_error("gated: out is missing, or its rows of %d are %zu apart", n, ldo);
        return DNB_ERR_ARG;
    }
    if ((uintptr_t)out_dev % 2 || !aligned16(pre_dev)) {
        set_error("gated: misaligned out or pre");
        return DNB_DECLINED;
    }
    DNB_CUDA(cudaSetDevice(c->device));
    const uint64_t N = n, K = k, T = nt;
    const Operand w[2] = {{gate_dev, N, K, K * 2}, {up_dev, N, K, K * 2}}, x = {x_dev, T, K, (uint64_t)ldx * 2};
    if (nt > 128) {
        dp::Params p = {};
        p.M = nt; p.N = n; p.K = k;
        p.passes = p.both = 1;
        p.outp[0] = out_dev;
        p.out_type = type;
        p.ldo = ldo;
        p.act = act;
        p.keep = pre_dev != nullptr;
        for (int i = 0; i < 2 && p.keep; ++i)
            if ((rc = dp::result_map(&p.pre[i], T_F32, pre_dev + i * T * N, T, N, N))) return rc;
        return dp::launch_pair<dp::Cfg<false, true>>(c, p, &x, 1, w, 2, type, "gated");
    }
    Params p = {};
    p.M = n; p.N = nt; p.K = k;
    p.passes = 1;
    p.out = out_dev;
    p.out_type = type;
    p.ldo = ldo;
    p.act = act;
    p.pre = pre_dev;
    if (nt <= 16) return launch_dense<Cfg<false, 2, 16>>(c, p, w, 2, &x, 1, type, "gated");
    if (nt <= 32) return launch_dense<Cfg<false, 2, 32>>(c, p, w, 2, &x, 1, type, "gated");
    if (nt <= 64) return launch_dense<Cfg<false, 2, 64>>(c, p, w, 2, &x, 1, type, "gated");
    return launch_dense<Cfg<false, 2, 128>>(c, p, w, 2, &x, 1, type, "gated");
}

int dnb_gated_backward_dev(dnb_ctx* c, int act, int type, const void* x_dev, size_t ldx, const void* gate_dev, const void* up_dev, const float* pre_dev,
                           const void* dout_dev, size_t ldd, int nt, int k, int n, void* dpre_dev, void* dx_dev, size_t lddx, void* dgate_dev, void* dup_dev) {
    if (!c) return DNB_ERR_ARG;
    int rc = check_shape("gated_backward", act, type, nt, k, n);
    if (rc) return rc;
    const size_t blocks = ((size_t)nt * n / 8 + 255) / 256;
    if (blocks > 0x7fffffff) {
        set_error("gated_backward: %d x %d is more than one launch takes", nt, n);
        return DNB_DECLINED;
    }
    const bool weights = dgate_dev || dup_dev;
    if (weights && (!dgate_dev || !dup_dev)) {
        set_error("gated_backward: gradients of both weights, or of none");
        return DNB_ERR_ARG;
    }
    if (dx_dev && (rc = check_sum("gated_backward", "features of gate and up", 2 * (int64_t)n))) return rc;
    if (weights && (rc = check_sum("gated_backward", "tokens", nt))) return rc;
    if ((uintptr_t)dgate_dev % 2 || (uintptr_t)dup_dev % 2 || (uintptr_t)dx_dev % 2) {
        set_error("gated_backward: misaligned result");
        return DNB_DECLINED;
    }
    if (nt > 0) {
        if ((rc = check_rows("gated_backward", "dout", dout_dev, ldd, n))) return rc;
        if ((rc = check_rows("gated_backward", "pre", pre_dev, n, n))) return rc;
        if ((rc = check_rows("gated_backward", "dpre", dpre_dev, n, n))) return rc;
        if (weights && (rc = check_rows("gated_backward", "x", x_dev, ldx, k))) return rc;
        if (dx_dev && ((rc = check_rows("gated_backward", "gate", gate_dev, k, k)) || (rc = check_rows("gated_backward", "up", up_dev, k, k)))) return rc;
        if (dx_dev && lddx < (size_t)k) {
            set_error("gated_backward: rows of %d of dx are %zu apart", k, lddx);
            return DNB_ERR_ARG;
        }
    }
    DNB_CUDA(cudaSetDevice(c->device));
    if (nt == 0) {  // sums of nothing
        if (weights) {
            DNB_CUDA(cudaMemsetAsync(dgate_dev, 0, (size_t)n * k * 2, c->stream));
            DNB_CUDA(cudaMemsetAsync(dup_dev, 0, (size_t)n * k * 2, c->stream));
        }
        return DNB_OK;
    }
    {
        ProfScope prof_(c, c->stream, "gated_gradients");
        const dim3 grid((unsigned)blocks);
        if (type == T_BF16) DNB_CUDA(launch_k(gradients_kernel<T_BF16>, grid, dim3(256), 0, c->stream, c->use_pdl, act, pre_dev, dout_dev, ldd, nt, n, dpre_dev));
        else DNB_CUDA(launch_k(gradients_kernel<T_F16>, grid, dim3(256), 0, c->stream, c->use_pdl, act, pre_dev, dout_dev, ldd, nt, n, dpre_dev));
        c->launches++;
    }
    const uint8_t* dpre = (const uint8_t*)dpre_dev;
    const uint64_t N = n, K = k, T = nt;
    const Operand d[2] = {{dpre, T, N, N * 2}, {dpre + T * N * 2, T, N, N * 2}};
    if (dx_dev) {
        const Operand w[2] = {{gate_dev, N, K, K * 2}, {up_dev, N, K, K * 2}};
        if (nt <= 128) {
            Params p = {};
            p.M = k; p.N = nt; p.K = n;
            p.passes = 2;
            p.out = dx_dev;
            p.out_type = type;
            p.ldo = lddx;
            if (nt <= 16) rc = launch_dense<Cfg<false, 1, 16, true>>(c, p, w, 2, d, 2, type, "gated_dx");
            else if (nt <= 32) rc = launch_dense<Cfg<false, 1, 32, true>>(c, p, w, 2, d, 2, type, "gated_dx");
            else if (nt <= 64) rc = launch_dense<Cfg<false, 1, 64, true>>(c, p, w, 2, d, 2, type, "gated_dx");
            else rc = launch_dense<Cfg<false, 1, 128, true>>(c, p, w, 2, d, 2, type, "gated_dx");
        } else {
            dp::Params p = {};
            p.M = nt; p.N = k; p.K = n;
            p.passes = 2;
            p.both = 1;
            p.outp[0] = dx_dev;
            p.out_type = type;
            p.ldo = lddx;
            rc = dp::launch_pair<dp::Cfg<false, false, false, true>>(c, p, d, 2, w, 2, type, "gated_dx");
        }
        if (rc) return rc;
    }
    if (weights) {
        dp::Params p = {};
        p.M = n; p.N = k; p.K = nt;
        p.passes = 1;
        p.both = 2;
        p.outp[0] = dgate_dev;
        p.outp[1] = dup_dev;
        p.out_type = type;
        p.ldo = k;
        const Operand x = {x_dev, T, K, (uint64_t)ldx * 2};
        if ((rc = dp::launch_pair<dp::Cfg<false, false, true, true>>(c, p, d, 2, &x, 1, type, "gated_dw"))) return rc;
    }
    return DNB_OK;
}

}  // extern "C"
