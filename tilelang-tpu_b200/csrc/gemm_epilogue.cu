// Matrix product with its epilogue:  C = act(A B + bias) + residual,  fp32 accumulation and epilogue, one rounding.
//
// Three kernels:
//   many rows the GEMM's tcgen05 kernels (gemm_kernels.cuh) with the epilogue applied to the accumulator columns a thread
//             holds, before they are rounded: bound by the tensor core, the epilogue runs under the next tile's MMAs
//             (8192 x 14336 x 4096: 0.71 to 0.76 ms without bias and GELU, 0.72 to 0.78 with them, as the power cap allows).
//   few rows  the product has to stream the weights once, 2 n k bytes: bound by HBM.  The weights are the 128-row operand
//             and the rows of A (rounded up to 16, 32, 64 or 128) the columns, D = W A^T, so no tile is mostly padding;
//             K is cut over the CTAs of a cluster until two CTAs per SM have a share, each with its own ring of TMA loads,
//             and the cluster adds its partial tiles up through distributed shared memory in a fixed order: no scratch, no
//             atomics, one launch.  The main loop runs at 6.3 to 6.9 TB/s; set-up, the joining of the tiles and the launch
//             take about 5 us (16 x 6144 x 4096: 12.7 us for 50 MB).
//   else      (fp32, or rows that TMA cannot describe) a plain FMA kernel through shared memory: right for every size and
//             alignment, and no more (1024^3 in fp32 196 us, 11 TFLOP/s; 256 x 4096 x 4095 in bf16 0.83 ms).
#include "gemm_kernels.cuh"

namespace tl {

struct EpilogueArgs {
  const void* bias;       // [n] or nullptr
  const void* residual;   // [m, n] or nullptr; may be C itself (every element is read by the thread that writes it)
  int act;
};

// x / (1 + exp(-z)), by the exponential that does not overflow: values far below zero keep their precision, down to fp32's
// smallest normal numbers, and the divisor is in [1, 2].
__device__ __forceinline__ float gated(float x, float z) {
  const float t = expf(-fabsf(z));
  return __fdividef(z >= 0.f ? x : x * t, 1.f + t);
}
// x erfc(-x / sqrt 2) / 2.  For y = |x|, erfc(y / sqrt 2) / 2 = (1/2 - y G(1 / (1 + y/4))) exp(-y^2 / 2) with a smooth G: the
// polynomial is the one whose relative error, over 1 + y^2 as the exponent's own, is least (2.8e-8 up to y = 14); with the
// roundings it is 4 (1 + y^2) 2^-24.  (1 + erf is off by 4% at -5 and zero below -5.5.  8192 x 8192 x 256, where the epilogue
// decides: 136 us; 149 us by erff, 259 us by erfcf.)
__device__ __forceinline__ float gelu(float x) {
  const float y = fminf(fabsf(x), 16.f);                          // exp(-128) is zero; NaN comes back by the last product
  const float u = __fdividef(1.f, fmaf(y, 0.25f, 1.f));
  float g = fmaf(u, -0.024126967f, 0.06715658f);
  g = fmaf(g, u, -0.011316363f);
  g = fmaf(g, u, 0.071484454f);
  g = fmaf(g, u, 0.07005878f);
  g = fmaf(g, u, 0.100706294f);
  g = fmaf(g, u, 0.12498111f);
  g = fmaf(g, u, -2.1028713e-06f);
  const float tail = fmaf(-y, g, 0.5f) * sm100::ex2_approx(y * y * -0.72134752044448170f);
  return x * (x < 0.f ? tail : 1.f - tail);
}
__device__ __forceinline__ float activate(float x, int act) {
  switch (act) {
    case TL_B200_ACT_RELU: return x < 0.f ? 0.f : x;                                            // NaN stays NaN
    case TL_B200_ACT_GELU: return gelu(x);
    // 1 + tanh u = 2 / (1 + exp(-2 u)): no difference of near numbers
    case TL_B200_ACT_GELU_TANH: return gated(x, 1.59576912160573071f * fmaf(0.044715f * x * x, x, x));
    case TL_B200_ACT_SILU: return gated(x, x);
    default: return x;
  }
}

// 32 accumulator columns of one row (tcgen05 kernels of gemm_kernels.cuh).
template <typename T> struct RowEpilogue {
  const T* bias;
  const T* residual;
  int64_t ld;
  int act;
  int vec;                // rows of the residual and the bias are 16-byte aligned
  __device__ __forceinline__ void add(uint32_t (&v)[32], const T* src, int valid) const {
    if (vec && valid == 32) {
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        Vec16<T> x;
        x.raw = *reinterpret_cast<const uint4*>(src + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j + e] = __float_as_uint(__uint_as_float(v[j + e]) + to_f32(x.e[e]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < valid) v[j] = __float_as_uint(__uint_as_float(v[j]) + to_f32(src[j]));
    }
  }
  __device__ __forceinline__ void operator()(uint32_t (&v)[32], int row, int col, int valid) const {
    if (bias) add(v, bias + col, valid);
    if (act != TL_B200_ACT_NONE) {
      switch (act) {      // the switch outside the loop: one copy of each function
        case TL_B200_ACT_RELU:
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(activate(__uint_as_float(v[j]), TL_B200_ACT_RELU));
          break;
        case TL_B200_ACT_GELU:
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(activate(__uint_as_float(v[j]), TL_B200_ACT_GELU));
          break;
        case TL_B200_ACT_GELU_TANH:
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(activate(__uint_as_float(v[j]), TL_B200_ACT_GELU_TANH));
          break;
        default:
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(activate(__uint_as_float(v[j]), TL_B200_ACT_SILU));
      }
    }
    if (residual) add(v, residual + (int64_t)row * ld + col, valid);
  }
};

// =================================================================================
// Few rows: D[128 weight rows, MT rows of A] per CTA, K split over a cluster
// =================================================================================
template <int MT> struct SkinnyCfg {
  static constexpr int kStageW = kBM * kRowBytes;               // 128 weight rows (or 64 k rows of 2 x 64 weight columns)
  static constexpr int kStageX = MT * kRowBytes;
  static constexpr int kStage = kStageW + kStageX;
  static constexpr int kStages = (113 * 1024 - 1024 - 256) / kStage;             // two CTAs per SM
  static constexpr int kPitch = kBM + 4;                        // floats of a row (one row of A) of the partial tile
  static constexpr int kSmemBytes = kStages * kStage + 1024 + 256;
  static constexpr int kTmemCols = MT < 32 ? 32 : MT;
  static_assert(MT * kPitch * 4 <= kStages * kStage, "the partial tile reuses the ring");
};

struct SkinnyParams {
  void* c;
  int m, n, k, splits, in_fmt;
  int vec;                 // rows of C, the residual and the bias allow vectors of four
  int* status;
};

template <int MT, bool W_MN_MAJOR, typename T, typename TOut>
__global__ void __launch_bounds__(128, 2)
gemm_skinny_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const SkinnyParams p,
                   const EpilogueArgs ep) {
  using Cfg = SkinnyCfg<MT>;
  constexpr int STAGES = Cfg::kStages, kBK = kRowBytes / 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw_addr);
  uint8_t* tail = base_ptr + STAGES * Cfg::kStage;
  const uint32_t bar_full = smem_u32(tail), bar_empty = bar_full + 8 * STAGES, bar_done = bar_empty + 8 * STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8 * (2 * STAGES + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int tile = blockIdx.x / p.splits, split = blockIdx.x % p.splits;         // the splits of a tile are one cluster
  const int row0 = blockIdx.y * MT, rows = min(MT, p.m - row0);                  // rows of A
  const int num_kb = (p.k + kBK - 1) / kBK;
  // K blocks split, split + splits, ...: together the cluster reads a contiguous piece of every weight row
  const int mine = (num_kb - split + p.splits - 1) / p.splits;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_done, 1);
    mbar_fence_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_slot), Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  dependency_wait();            // what came before runs under the set-up above
  dependency_release();

  if (warp == 0) {
    if (elect_one()) {
      for (int i = 0; i < mine; ++i) {
        const int stage = i % STAGES, kb = split + i * p.splits;
        if (!mbar_wait(bar_empty + 8 * stage, ((i / STAGES) & 1) ^ 1, abort_flag)) break;
        const uint32_t full = bar_full + 8 * stage, dst = base + stage * Cfg::kStage;
        mbar_expect_tx(full, Cfg::kStage);
        if constexpr (W_MN_MAJOR) {          // weights [k, n]: two slabs of 64 columns x 64 k rows
          tma_load_2d(dst, &tm_w, full, tile * kBM, kb * kBK);
          tma_load_2d(dst + kBK * kRowBytes, &tm_w, full, tile * kBM + 64, kb * kBK);
        } else {
          tma_load_2d(dst, &tm_w, full, kb * kBK, tile * kBM);
        }
        tma_load_2d(dst + Cfg::kStageW, &tm_x, full, kb * kBK, row0);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc(p.in_fmt, p.in_fmt, W_MN_MAJOR, false, kBM, MT);
      bool ok = true;
      for (int i = 0; i < mine; ++i) {
        const int stage = i % STAGES;
        if (!(ok = mbar_wait(bar_full + 8 * stage, (i / STAGES) & 1, abort_flag))) break;
        tc_fence_after_sync();
        const uint32_t w = base + stage * Cfg::kStage, x = w + Cfg::kStageW;
#pragma unroll
        for (int kk = 0; kk < kRowBytes / kUmmaBytes; ++kk) {
          const uint64_t a = W_MN_MAJOR ? smem_desc_sw128(w + kk * 16 * kRowBytes, kBK * kRowBytes, 1024)
                                        : smem_desc_sw128(w + kk * kUmmaBytes, 16, 1024);
          mma_f16_ss(tmem_base, a, smem_desc_sw128(x + kk * kUmmaBytes, 16, 1024), idesc, (i | kk) ? 1u : 0u);
        }
        mma_commit(bar_empty + 8 * stage);
      }
      if (ok) mma_commit(bar_done);
    }
  }
  __syncwarp();
  // ---- the tile: each warp's 32 weight rows (columns of C) to shared memory, row by row of A ----------------------------
  bool ok = mbar_wait(bar_done, 0, abort_flag);
  ok = __all_sync(0xffffffffu, ok);
  tc_fence_after_sync();
  const uint32_t t_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
  float* part = reinterpret_cast<float*>(base_ptr);               // [MT][kPitch]: every MMA that read the ring has retired
  if (ok) {
#pragma unroll 1
    for (int c0 = 0; c0 < rows; c0 += 16) {
      uint32_t v[16];
      tmem_ld_32x16(t_addr + c0, v);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e) part[(c0 + e) * Cfg::kPitch + warp * 32 + lane] = __uint_as_float(v[e]);
    }
  }
  if (p.splits > 1) cluster_sync_all();                           // the cluster's partial tiles are there
  else __syncthreads();
  if (ok) {
    // this CTA's share of the tile, four neighbouring columns a thread; all the partial sums of an element at once
    const int items = rows * (kBM / 4);
    const int i0 = (int)((int64_t)split * items / p.splits), i1 = (int)((int64_t)(split + 1) * items / p.splits);
    const T *bias = reinterpret_cast<const T*>(ep.bias), *residual = reinterpret_cast<const T*>(ep.residual);
    TOut* c = reinterpret_cast<TOut*>(p.c);
    for (int i = i0 + threadIdx.x; i < i1; i += 128) {
      const int r = i / (kBM / 4), in_tile = i % (kBM / 4) * 4, n0 = tile * kBM + in_tile;
      const int valid = min(4, p.n - n0);
      if (valid <= 0) continue;
      const int64_t at = (int64_t)(row0 + r) * p.n + n0;
      union { uint2 raw; T e[4]; } b, res;
      b.raw = res.raw = make_uint2(0, 0);
      if (p.vec && valid == 4) {
        if (bias) b.raw = *reinterpret_cast<const uint2*>(bias + n0);
        if (residual) res.raw = *reinterpret_cast<const uint2*>(residual + at);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < valid) {
            if (bias) b.e[e] = bias[n0 + e];
            if (residual) res.e[e] = residual[at + e];
          }
      }
      const uint32_t mine_at = smem_u32(part + r * Cfg::kPitch + in_tile);
      float y[8][4];
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < p.splits)
          asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y[s][0]), "=f"(y[s][1]), "=f"(y[s][2]), "=f"(y[s][3])
                       : "r"(map_to_cta(mine_at, s)) : "memory");
        else
          y[s][0] = y[s][1] = y[s][2] = y[s][3] = 0.f;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = y[0][e];
#pragma unroll
        for (int s = 1; s < 8; ++s) x[e] += y[s][e];
        if (bias) x[e] += to_f32(b.e[e]);
      }
      if (ep.act != TL_B200_ACT_NONE) {
        switch (ep.act) {      // outside the loop: one copy of each function
          case TL_B200_ACT_RELU:
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = activate(x[e], TL_B200_ACT_RELU);
            break;
          case TL_B200_ACT_GELU:
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = activate(x[e], TL_B200_ACT_GELU);
            break;
          case TL_B200_ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = activate(x[e], TL_B200_ACT_GELU_TANH);
            break;
          default:
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = activate(x[e], TL_B200_ACT_SILU);
        }
      }
      union { uint4 raw16; uint2 raw8; TOut e[4]; } o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o.e[e] = from_f32<TOut>(residual ? x[e] + to_f32(res.e[e]) : x[e]);
      if (p.vec && valid == 4) {
        if constexpr (sizeof(TOut) == 4) *reinterpret_cast<uint4*>(c + at) = o.raw16;
        else *reinterpret_cast<uint2*>(c + at) = o.raw8;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < valid) c[at + e] = o.e[e];
      }
    }
  }

  // ---- teardown -------------------------------------------------------------------------------------------------------
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(20000);
    if (threadIdx.x == 0 && p.status) *p.status = *abort_flag;
    __syncthreads();
  }
  if (p.splits > 1) cluster_sync_all();                           // nobody leaves while its partial tile is being read
  if (warp == 2) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

template <int MT, bool W_MN_MAJOR, typename T, typename TOut>
static int launch_skinny(const CUtensorMap& tw, const CUtensorMap& tx, const SkinnyParams& p, const EpilogueArgs& ep, cudaStream_t s) {
  auto kernel = gemm_skinny_kernel<MT, W_MN_MAJOR, T, TOut>;
  TL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SkinnyCfg<MT>::kSmemBytes));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.n + kBM - 1) / kBM * p.splits), (unsigned)((p.m + MT - 1) / MT));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = SkinnyCfg<MT>::kSmemBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits > 1 ? 2 : 1;
  TL_CUDA(cudaLaunchKernelEx(&cfg, kernel, tw, tx, p, ep));
  TL_LAUNCH_CHECK("gemm_skinny_kernel");
  return TL_B200_OK;
}

template <int MT, typename T>
static int launch_skinny_out(const CUtensorMap& tw, const CUtensorMap& tx, const SkinnyParams& p, const EpilogueArgs& ep, bool mn, bool f32,
                             cudaStream_t s) {
  if (f32) return mn ? launch_skinny<MT, true, T, float>(tw, tx, p, ep, s) : launch_skinny<MT, false, T, float>(tw, tx, p, ep, s);
  return mn ? launch_skinny<MT, true, T, T>(tw, tx, p, ep, s) : launch_skinny<MT, false, T, T>(tw, tx, p, ep, s);
}

constexpr int kSkinnyTile = 128;
// Few rows, or a product whose narrowest tiles (128 x 64) would leave SMs without one.  Measured, this kernel and the GEMM's:
// 128 x 4096 x 4096 15.5 and 16.4 us, 256 x 4096 x 14336 38 and 44 us, 256 x 1024 x 4096 12.4 and 16.8 us; and where every SM
// has a tile, 128 x 14336 x 4096 39 and 32 us, 256 x 14336 x 4096 50 and 43 us.
static bool is_skinny(int m, int n) {
  return m <= 64 || (m <= 512 && (int64_t)((m + kBM - 1) / kBM) * ((n + 63) / 64) < sm_count());
}

template <typename T>
static int gemm_skinny(const void* a, const void* b, void* c, int m, int n, int k, bool trans_b, bool c_f32, const EpilogueArgs& ep,
                       cudaStream_t s) {
  const bool bf = std::is_same<T, __nv_bfloat16>::value;
  const CUtensorMapDataType dt = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int row_tiles = (m + kSkinnyTile - 1) / kSkinnyTile, mt = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
  CUtensorMap tw, tx;
  {
    uint64_t dims[2] = {(uint64_t)k, (uint64_t)m};
    uint64_t strides[1] = {(uint64_t)k * 2};
    uint32_t box[2] = {64u, (uint32_t)mt};
    if (int rc = make_tensor_map(&tx, dt, 2, a, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  {
    uint64_t dims[2] = {(uint64_t)(trans_b ? k : n), (uint64_t)(trans_b ? n : k)};
    uint64_t strides[1] = {dims[0] * 2};
    uint32_t box[2] = {64u, trans_b ? (uint32_t)kBM : 64u};
    if (int rc = make_tensor_map(&tw, dt, 2, b, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  SkinnyParams p;
  p.c = c; p.m = m; p.n = n; p.k = k;
  p.in_fmt = bf ? kFmtBF16 : kFmtF16;
  p.vec = n % 4 == 0 && aligned16(c) && aligned16(ep.bias) && aligned16(ep.residual);
  p.status = device_status_word();
  // as many splits of K (1, 2, 4, 8: a portable cluster) as two CTAs per SM have room for, with at least four K blocks each
  const int tiles = (n + kBM - 1) / kBM, num_kb = (k + 63) / 64;
  p.splits = 1;
  while (p.splits < 8 && (int64_t)tiles * row_tiles * p.splits * 2 <= 2 * sm_count() && num_kb >= p.splits * 2 * 4) p.splits *= 2;
  const bool mn = !trans_b;
  switch (mt) {
    case 16: return launch_skinny_out<16, T>(tw, tx, p, ep, mn, c_f32, s);
    case 32: return launch_skinny_out<32, T>(tw, tx, p, ep, mn, c_f32, s);
    case 64: return launch_skinny_out<64, T>(tw, tx, p, ep, mn, c_f32, s);
    default: return launch_skinny_out<128, T>(tw, tx, p, ep, mn, c_f32, s);
  }
}

template <typename T>
static int gemm_epilogue_tc(const void* a, const void* b, void* c, int m, int n, int k, bool trans_b, bool c_f32, const EpilogueArgs& ep,
                            cudaStream_t s) {
  if (is_skinny(m, n)) return gemm_skinny<T>(a, b, c, m, n, k, trans_b, c_f32, ep, s);
  RowEpilogue<T> e;
  e.bias = (const T*)ep.bias;
  e.residual = (const T*)ep.residual;
  e.ld = n;
  e.act = ep.act;
  e.vec = n % 8 == 0 && aligned16(ep.bias) && aligned16(ep.residual);
  return gemm_tc<T, RowEpilogue<T>>(a, b, c, m, n, k, trans_b, c_f32, s, 0, 0, e);
}

// =================================================================================
// Plain FMA kernel: fp32, and 16-bit shapes without a tensor map; 64 x 64 tiles of C through shared memory
// =================================================================================
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
  constexpr int64_t kMost = (1ll << 31) - (1 << 23);              // sizes rounded up to tiles and grid strides stay below 2^31
  TL_REQUIRE(m <= kMost && n <= kMost && k <= kMost, "gemm_epilogue: dimension exceeds 2^31 - 2^23");
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
  // TMA needs 16-byte aligned bases and row strides
  if (aligned16(a) && aligned16(b) && K % 8 == 0 && (tb || N % 8 == 0))
    return in_dtype == TL_BF16 ? gemm_epilogue_tc<__nv_bfloat16>(a, b, c, M, N, K, tb, out_dtype == TL_F32, ep, s)
                               : gemm_epilogue_tc<__half>(a, b, c, M, N, K, tb, out_dtype == TL_F32, ep, s);
  if (in_dtype == TL_BF16)
    return out_dtype == TL_F32 ? launch_epilogue_fma<__nv_bfloat16, float>(a, b, c, M, N, K, tb, ep, s)
                               : launch_epilogue_fma<__nv_bfloat16, __nv_bfloat16>(a, b, c, M, N, K, tb, ep, s);
  return out_dtype == TL_F32 ? launch_epilogue_fma<__half, float>(a, b, c, M, N, K, tb, ep, s)
                             : launch_epilogue_fma<__half, __half>(a, b, c, M, N, K, tb, ep, s);
}
