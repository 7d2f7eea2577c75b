// Matrix product with its epilogue:  C = act(A B + bias) + residual,  fp32 accumulation and epilogue, one rounding.
//
// A plain FMA kernel: 64 x 64 tiles of C through shared memory.
#include "common.cuh"

namespace tl {

struct EpilogueArgs {
  const void* bias;       // [n] or nullptr
  const void* residual;   // [m, n] or nullptr; may be C itself (every element is read by the thread that writes it)
  int act;
};

__device__ __forceinline__ float activate(float x, int act) {
  switch (act) {
    case TL_B200_ACT_RELU: return x < 0.f ? 0.f : x;                                            // NaN stays NaN
    case TL_B200_ACT_GELU: return 0.5f * x * (1.f + erff(x * 0.70710678118654752f));
    case TL_B200_ACT_GELU_TANH: return 0.5f * x * (1.f + tanhf(0.79788456080286536f * fmaf(0.044715f * x * x, x, x)));
    case TL_B200_ACT_SILU: return x / (1.f + expf(-x));
    default: return x;
  }
}

template <typename TIn, typename TOut, bool TRANS_B>
__global__ void __launch_bounds__(256)
gemm_epilogue_fma_kernel(const TIn* __restrict__ a, const TIn* __restrict__ b, TOut* c, int m, int n, int k, const EpilogueArgs ep) {
  constexpr int T = 64, KT = 16;
  __shared__ float sa[KT][T + 1];
  __shared__ float sb[KT][T + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int n0 = blockIdx.x * T;
  for (int m0 = blockIdx.y * T; m0 < m; m0 += gridDim.y * T) {
    float acc[4][4] = {};
    for (int k0 = 0; k0 < k; k0 += KT) {
      for (int i = threadIdx.x; i < T * KT; i += 256) {
        const int r = i / KT, kk = i % KT, gm = m0 + r, gk = k0 + kk;
        sa[kk][r] = (gm < m && gk < k) ? to_f32(a[(int64_t)gm * k + gk]) : 0.f;
      }
      for (int i = threadIdx.x; i < T * KT; i += 256) {
        const int kk = TRANS_B ? i % KT : i / T, col = TRANS_B ? i / KT : i % T, gn = n0 + col, gk = k0 + kk;
        sb[kk][col] = (gn < n && gk < k) ? to_f32(TRANS_B ? b[(int64_t)gn * k + gk] : b[(int64_t)gk * n + gn]) : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < KT; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ty * 4 + i], sb[kk][tx * 4 + j], acc[i][j]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int gm = m0 + ty * 4 + i, gn = n0 + tx * 4 + j;
        if (gm < m && gn < n) {
          float x = acc[i][j];
          if (ep.bias) x += to_f32(reinterpret_cast<const TIn*>(ep.bias)[gn]);
          x = activate(x, ep.act);
          if (ep.residual) x += to_f32(reinterpret_cast<const TIn*>(ep.residual)[(int64_t)gm * n + gn]);
          c[(int64_t)gm * n + gn] = from_f32<TOut>(x);
        }
      }
  }
}

template <typename TIn, typename TOut>
static int launch_epilogue_fma(const void* a, const void* b, void* c, int m, int n, int k, bool trans_b, const EpilogueArgs& ep,
                               cudaStream_t s) {
  const int rows = (m + 63) / 64;
  const dim3 grid((n + 63) / 64, rows < 65535 ? rows : 65535);
  if (trans_b) gemm_epilogue_fma_kernel<TIn, TOut, true><<<grid, 256, 0, s>>>((const TIn*)a, (const TIn*)b, (TOut*)c, m, n, k, ep);
  else gemm_epilogue_fma_kernel<TIn, TOut, false><<<grid, 256, 0, s>>>((const TIn*)a, (const TIn*)b, (TOut*)c, m, n, k, ep);
  TL_LAUNCH_CHECK("gemm_epilogue_fma_kernel");
  return TL_B200_OK;
}

}  // namespace tl

using namespace tl;

extern "C" int tl_b200_gemm_epilogue(const void* a, const void* b, const void* bias, const void* residual, void* c, int64_t m, int64_t n,
                                     int64_t k, int trans_b, int act, int in_dtype, int out_dtype, void* stream) {
  TL_REQUIRE(m >= 0 && n >= 0 && k >= 0, "gemm_epilogue: negative size");
  TL_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "gemm_epilogue: dimension exceeds 2^31");
  TL_REQUIRE(act >= TL_B200_ACT_NONE && act <= TL_B200_ACT_SILU, "gemm_epilogue: unknown activation %d", act);
  TL_REQUIRE(in_dtype == TL_F32 || in_dtype == TL_F16 || in_dtype == TL_BF16, "gemm_epilogue: unsupported input dtype %d", in_dtype);
  TL_REQUIRE(out_dtype == in_dtype || out_dtype == TL_F32, "gemm_epilogue: output must be the input type or float32");
  if (m == 0 || n == 0) return TL_B200_OK;
  TL_REQUIRE(a && b && c, "gemm_epilogue: null tensor pointer");
  TL_REQUIRE(k > 0, "gemm_epilogue: K must be positive");
  TL_REQUIRE(residual != c || out_dtype == in_dtype, "gemm_epilogue: a residual that is the output has the output's type");
  const EpilogueArgs ep{bias, residual, act};
  const bool tb = trans_b != 0;
  const int M = (int)m, N = (int)n, K = (int)k;
  cudaStream_t s = (cudaStream_t)stream;
  if (in_dtype == TL_F32) return launch_epilogue_fma<float, float>(a, b, c, M, N, K, tb, ep, s);
  if (in_dtype == TL_BF16)
    return out_dtype == TL_F32 ? launch_epilogue_fma<__nv_bfloat16, float>(a, b, c, M, N, K, tb, ep, s)
                               : launch_epilogue_fma<__nv_bfloat16, __nv_bfloat16>(a, b, c, M, N, K, tb, ep, s);
  return out_dtype == TL_F32 ? launch_epilogue_fma<__half, float>(a, b, c, M, N, K, tb, ep, s)
                             : launch_epilogue_fma<__half, __half>(a, b, c, M, N, K, tb, ep, s);
}
