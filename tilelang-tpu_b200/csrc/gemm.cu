// Dense GEMM  C[M,N] = A[M,K] * B  with fp32 accumulation.
//
// Large products run on CTA pairs (`gemm_pair_kernel`: 256 x 256 tiles, cta_group::2); smaller ones on the one-CTA
// kernel described first.  Both live in gemm_kernels.cuh, which the product with an epilogue shares.
//
// The 16-bit path is a persistent, warp-specialised tcgen05 kernel: TMA brings 128xBK tiles of A
// and BNxBK tiles of B into a shared-memory ring (128-byte swizzle), one thread issues
// tcgen05.mma into a double-buffered fp32 accumulator in tensor memory, and four epilogue warps
// drain the other accumulator (tcgen05.ld -> round -> global stores) while the next tile's main
// loop already runs.  B may be [K,N] row-major (MN-major operand, the layout of the reference
// matmul program) or [N,K] row-major (K-major, `transpose_B=True` of ppl_gemm).
// e4m3 operands (the plain, un-scaled FP8 form of ppl_gemm, src/target/codegen_ppl.cc:775-790) run the same
// kernel with `kind::f8f6f4`: every byte offset is the same, a stage simply holds twice the K elements.
// fp32 inputs and shapes TMA cannot describe use a plain shared-memory-tiled FMA kernel.
#include "gemm_kernels.cuh"

namespace tl {

// =================================================================================
// Plain FMA kernel: any of fp32 / fp16 / bf16, any size and alignment.
// =================================================================================
template <typename TIn, typename TOut, bool TRANS_B>
__global__ void __launch_bounds__(256)
gemm_simt_kernel(const TIn* __restrict__ a, const TIn* __restrict__ b, TOut* __restrict__ c, int m, int n, int k) {
  constexpr int T = 64, KT = 16;
  __shared__ float sa[KT][T + 1];
  __shared__ float sb[KT][T + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int m0 = blockIdx.y * T, n0 = blockIdx.x * T;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < k; k0 += KT) {
    for (int i = threadIdx.x; i < T * KT; i += 256) {
      int r = i / KT, kk = i % KT;             // A tile: rows of M, K contiguous
      int gm = m0 + r, gk = k0 + kk;
      sa[kk][r] = (gm < m && gk < k) ? to_f32(a[(int64_t)gm * k + gk]) : 0.f;
    }
    for (int i = threadIdx.x; i < T * KT; i += 256) {
      int kk, cidx;
      if (TRANS_B) { cidx = i / KT; kk = i % KT; } else { kk = i / T; cidx = i % T; }
      int gn = n0 + cidx, gk = k0 + kk;
      float v = 0.f;
      if (gn < n && gk < k) v = TRANS_B ? to_f32(b[(int64_t)gn * k + gk]) : to_f32(b[(int64_t)gk * n + gn]);
      sb[kk][cidx] = v;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < KT; ++kk) {
      float av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { av[i] = sa[kk][ty * 4 + i]; bv[i] = sb[kk][tx * 4 + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(av[i], bv[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int gm = m0 + ty * 4 + i, gn = n0 + tx * 4 + j;
      if (gm < m && gn < n) c[(int64_t)gm * n + gn] = from_f32<TOut>(acc[i][j]);
    }
}

template <typename TIn, typename TOut>
static int launch_simt(const void* a, const void* b, void* c, int m, int n, int k, bool trans_b, cudaStream_t s) {
  dim3 grid((n + 63) / 64, (m + 63) / 64);
  if (trans_b)
    gemm_simt_kernel<TIn, TOut, true><<<grid, 256, 0, s>>>((const TIn*)a, (const TIn*)b, (TOut*)c, m, n, k);
  else
    gemm_simt_kernel<TIn, TOut, false><<<grid, 256, 0, s>>>((const TIn*)a, (const TIn*)b, (TOut*)c, m, n, k);
  TL_LAUNCH_CHECK("gemm_simt_kernel");
  return TL_B200_OK;
}

}  // namespace tl

using namespace tl;

extern "C" int tl_b200_gemm(const void* a, const void* b, void* c, int64_t m, int64_t n, int64_t k, int trans_b,
                            int in_dtype, int out_dtype, void* stream) {
  return tl_b200_gemm_tiled(a, b, c, m, n, k, trans_b, in_dtype, out_dtype, 0, stream);
}

extern "C" int tl_b200_gemm_tiled(const void* a, const void* b, void* c, int64_t m, int64_t n, int64_t k, int trans_b,
                                  int in_dtype, int out_dtype, int tile_n, void* stream) {
  TL_REQUIRE(tile_n == 0 || tile_n == 64 || tile_n == 128 || tile_n == 256 || tile_n == kTilePair,
             "gemm: tile_n must be 0, 64, 128, 256 or 512 (a 256 x 256 tile on a CTA pair)");
  TL_REQUIRE(m >= 0 && n >= 0 && k >= 0, "gemm: negative size");
  TL_REQUIRE(m < (1ll << 31) && n < (1ll << 31) && k < (1ll << 31), "gemm: dimension exceeds 2^31");
  if (m == 0 || n == 0) return TL_B200_OK;
  TL_REQUIRE(a && b && c, "gemm: null tensor pointer");
  TL_REQUIRE(k > 0, "gemm: K must be positive");
  TL_REQUIRE(out_dtype == in_dtype || out_dtype == TL_F32 ||
                 (in_dtype == TL_E4M3 && (out_dtype == TL_BF16 || out_dtype == TL_F16)),
             "gemm: output must be the input type or float32 (e4m3 operands: float32, bfloat16 or float16)");
  TL_REQUIRE(!(in_dtype == TL_E4M3 && out_dtype == TL_E4M3), "gemm: e4m3 operands need a float32, bfloat16 or float16 output");
  cudaStream_t s = (cudaStream_t)stream;
  const bool tb = trans_b != 0;
  const int M = (int)m, N = (int)n, K = (int)k;
  if (in_dtype == TL_F32) return launch_simt<float, float>(a, b, c, M, N, K, tb, s);
  if (in_dtype == TL_E4M3) {
    // plain (un-scaled) FP8 product: tensor cores only; TMA needs 16-byte aligned bases and row strides
    TL_REQUIRE(aligned16(a) && aligned16(b) && K % 16 == 0 && (tb || N % 16 == 0),
               "gemm: e4m3 operands need 16-byte aligned tensors, K %% 16 == 0 and (transposed B or N %% 16 == 0)");
    const int out_kind = out_dtype == TL_F32 ? 0 : (out_dtype == TL_BF16 ? 1 : 2);
    return gemm_tc<uint8_t>(a, b, c, M, N, K, tb, out_dtype == TL_F32, s, out_kind, tile_n);
  }
  TL_REQUIRE(in_dtype == TL_F16 || in_dtype == TL_BF16, "gemm: unsupported input dtype %d", in_dtype);
  // TMA needs 16-byte aligned bases and row strides
  const bool tma_ok = aligned16(a) && aligned16(b) && K % 8 == 0 && (tb || N % 8 == 0);
  if (tma_ok) {
    if (in_dtype == TL_BF16) return gemm_tc<__nv_bfloat16>(a, b, c, M, N, K, tb, out_dtype == TL_F32, s, 0, tile_n);
    return gemm_tc<__half>(a, b, c, M, N, K, tb, out_dtype == TL_F32, s, 0, tile_n);
  }
  if (in_dtype == TL_BF16) {
    if (out_dtype == TL_F32) return launch_simt<__nv_bfloat16, float>(a, b, c, M, N, K, tb, s);
    return launch_simt<__nv_bfloat16, __nv_bfloat16>(a, b, c, M, N, K, tb, s);
  }
  if (out_dtype == TL_F32) return launch_simt<__half, float>(a, b, c, M, N, K, tb, s);
  return launch_simt<__half, __half>(a, b, c, M, N, K, tb, s);
}
