// linear_i8.cu -- the 8-bit linear layer: out[m][n] = act(s(m, n) * (xs[m] * ws[n]) + bias[n]),
// s(m, n) = sum_k x[m][k] w[n][k] in 32-bit integers, act the identity or the tanh form of GELU.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ss {
namespace lin {

struct Params {
    const int8_t *x;
    const int8_t *w;
    int64_t x_ld, w_ld;
    const float *xs, *ws;
    const void *bias;
    int bias_dtype, gelu, out_dtype;
    int M, N, K;
    void *out;
    int64_t out_ld;
};

__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
    if (dtype == SS_F32) return static_cast<const float *>(p)[i];
    if (dtype == SS_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v) {
    if (dtype == SS_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == SS_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// tanh form of GELU, 0.5 v (1 + tanh(u)) = v / (1 + exp(-2u)), u = sqrt(2/pi) (v + 0.044715 v^3):
// no cancellation for negative v, and an exponential that overflows gives -0
__device__ __forceinline__ float gelu_tanh(float v) {
    const float u2 = 1.5957691216057308f * v * (1.f + 0.044715f * v * v);
    return v / (1.f + __expf(-u2));
}

constexpr int BM = 64, BN = 64, BK = 64;

// 64 x 64 tile of 256 threads, 4 x 4 outputs each, four products an instruction (dp4a)
__global__ void __launch_bounds__(256) linear_kernel(const Params p) {
    __shared__ int xt[BK / 4][BM + 1], wt[BK / 4][BN + 1];
    const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * BM, n0 = (int64_t)blockIdx.x * BN;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += BK) {
        // thread t stages 16 bytes of row t / 4 of each operand, zero outside
        const int r = t >> 2, c = (t & 3) * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t a = 0u, b = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = k0 + c + 4 * j + i;
                if (k < p.K && m0 + r < p.M) a |= (uint32_t)(uint8_t)p.x[(m0 + r) * p.x_ld + k] << (8 * i);
                if (k < p.K && n0 + r < p.N) b |= (uint32_t)(uint8_t)p.w[(n0 + r) * p.w_ld + k] << (8 * i);
            }
            xt[c / 4 + j][r] = (int)a;
            wt[c / 4 + j][r] = (int)b;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK / 4; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xt[k][ty + 16 * i], wt[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= p.M || n >= p.N) continue;
            float v = __fmul_rn((float)acc[i][j], __fmul_rn(p.xs[m], p.ws[n]));
            if (p.bias) v = __fadd_rn(v, load_any(p.bias, p.bias_dtype, n));
            if (p.gelu) v = gelu_tanh(v);
            store_any(p.out, p.out_dtype, m * p.out_ld + n, v);
        }
}

static bool off(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
static size_t type_bytes(int dtype) { return dtype == SS_F32 ? 4 : 2; }
static bool known(int dtype) { return dtype == SS_BF16 || dtype == SS_F32 || dtype == SS_F16; }

}  // namespace lin
}  // namespace ss

extern "C" int ss_linear_i8(const int8_t *x, int64_t x_ld, const float *xs, const int8_t *w, int64_t w_ld,
                            const float *ws, const void *bias, int bias_dtype, int gelu, int M, int N, int K,
                            void *out, int64_t out_ld, int out_dtype, int *status, void *stream) {
    using namespace ss;
    if (M < 0 || N <= 0 || K <= 0 || K > SS_LINEAR_I8_MAX_K || x_ld < K || w_ld < K || out_ld < N || (x_ld % 16) ||
        (w_ld % 16) || !lin::known(out_dtype) || (bias && !lin::known(bias_dtype)))
        return SS_ERR_SHAPE;
    if (M == 0) return 0;   // buffers without rows may have no address
    if (!x || !xs || !w || !ws || !out) return SS_ERR_POINTER;
    if (lin::off(x, 16) || lin::off(w, 16) || lin::off(xs, 4) || lin::off(ws, 4) || lin::off(status, 4) ||
        lin::off(out, lin::type_bytes(out_dtype)) || (bias && lin::off(bias, lin::type_bytes(bias_dtype))))
        return SS_ERR_POINTER;
    lin::Params p = {x, w, x_ld, w_ld, xs, ws, bias, bias_dtype, gelu, out_dtype, M, N, K, out, out_ld};
    const dim3 grid((unsigned)((N + lin::BN - 1) / lin::BN), (unsigned)((M + lin::BM - 1) / lin::BM));
    if (grid.y > 65535) return SS_ERR_SHAPE;
    lin::linear_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return (int)cudaGetLastError();
}
