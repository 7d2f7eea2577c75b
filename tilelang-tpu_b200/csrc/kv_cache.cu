// A paged key/value cache held in fewer bits: rows are quantised as they are written and widened as they are read back.
//
// Two formats, each the one an attention kernel of this library reads:
//   TL_U4G  codes [pages, heads, page, dim/2] (the even column in the low four bits of a byte) and, per group of `group`
//           columns, two values of the model's 16-bit type [pages, heads, page, dim/group, 2]: step s and minimum lo;
//           lo = min x, s = (max x - lo) / 15 rounded once, code = round((x - lo) / s) cut to 0..15 (0 where s is 0),
//           value = s * code + lo.  s and lo are kept in the 16-bit type because the inputs are no finer than that.
//   TL_E4M3 rows [pages, page, dim] with an fp32 scale each [pages, page]: s = max(amax |x|, 1e-4) / 448,
//           byte = e4m3(x / s), value = s * byte  (mla_decode_paged).
// A group (a row, for e4m3) that holds a NaN or an infinity reads back as NaN: the minima and maxima propagate NaN, and
// an infinite step turns 0 * s into NaN.
// `slots[t]` is page * page_size + position for token t; tokens whose slot is outside the cache (negative: padding) are
// skipped, and nothing else in the cache or in the output is touched.
//
// HBM-bound: a 16-bit row is read (written) once and its codes written (read) once.  Measured at a copy rate of 6.55 TB/s:
// 8192 tokens of 8 heads of 128 written to 4 bits, keys and values, 10.9 us (3.9 TB/s) and read back 9.6 us (4.5 TB/s), in turn
// 18.9 us; 65500 e4m3 rows of 576 read back 19.5 us (5.8 TB/s).  Of the short ones a few us are the launch and the drain.
// The 4-bit write has a row a thread in flight and much integer work: at 32768 tokens its issue slots are 69% taken, and a warp
// waits 6.0 of its 18 cycles an instruction for its row, 4.5 for its turn and 2.4 for a busy pipe, at 42% of the memory's rate.
#include "sm100.cuh"

#include <type_traits>

namespace tl {

struct Side {
  void* x;                    // 16-bit rows
  int64_t stride;             // elements from one token to the next
  void *cache, *scale;
};
struct CacheArgs {
  const int64_t* slots;
  uint32_t tokens, rows;      // rows = tokens * heads
  Side k, v;                  // v only with gridDim.y == 2
  int heads, page_size;
  FastDiv head_div, page_div, vec_div;
  int64_t total_slots;
  int wide;                   // rows are 32-byte aligned: one 256-bit access for 16 columns
};

// NaN-propagating minimum and maximum of two packed 16-bit values.
__device__ __forceinline__ __nv_bfloat162 min2_nan(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2_nan(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 min2_nan(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 max2_nan(__half2 a, __half2 b) { return __hmax2_nan(a, b); }

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr float kTiny = 0x1p-100f;       // smallest step of the quick division below
};
template <> struct Pair<__half> {
  using type = __half2;
  static constexpr float kTiny = 0x1p-14f;        // steps below are subnormal: coarser than 2^-9, a code can pass 15
};

__device__ __forceinline__ float2 widen2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 widen2(__half2 v) { return __half22float2(v); }
template <typename T> __device__ __forceinline__ uint32_t narrow2(float2 f) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __float22bfloat162_rn(f);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __float22half2_rn(f);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename P> __device__ __forceinline__ P shfl_xor_pair(P v, int o) {
  uint32_t w = *reinterpret_cast<uint32_t*>(&v);
  w = __shfl_xor_sync(0xffffffffu, w, o);
  return *reinterpret_cast<P*>(&w);
}

// a / s for two values at once, correctly rounded, given y = rn(1 / s): Markstein's theorem (IBM J. Res. Dev. 34, 1990) -
// q = rn(a y), then rn(q + (a - q s) y) is rn(a / s) as long as nothing leaves the normal range.  The codes have to be those
// of the IEEE division of the definition, ties included; a division per element would cost three times the memory traffic.
__device__ __forceinline__ float2 div2(float2 a, float2 neg_s, float2 y) {
  const float2 q = sm100::mul2(a, y);
  return sm100::fma2(sm100::fma2(q, neg_s, a), y, q);
}

// ---- 4 bits: a thread holds 16 columns (32 bytes in, 8 bytes of codes out); GROUP/16 neighbouring lanes own a group -----
template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(256)
kv_write_u4g_kernel(const CacheArgs p) {
  using P = typename Pair<T>::type;
  constexpr int kLanes = DIM / 16, kGroupLanes = GROUP / 16;
  dependency_wait();
  dependency_release();
  const Side side = blockIdx.y ? p.v : p.k;
  const uint32_t row = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int part = threadIdx.x % kLanes;
  const uint32_t t = p.head_div(row);
  const int h = (int)(row - t * p.heads);
  const int64_t slot = row < p.rows ? p.slots[t] : -1;
  const bool live = slot >= 0 && slot < p.total_slots;
  union { uint4 raw[2]; P v[8]; } in;
  in.raw[0] = in.raw[1] = make_uint4(0, 0, 0, 0);
  if (row < p.rows) {                 // whatever the slot: the two loads need not wait for each other
    const T* src = reinterpret_cast<const T*>(side.x) + t * side.stride + h * DIM + part * 16;
    if (p.wide) {                     // two 16-byte loads would each fetch every sector
      const Vec32<T> v = ld_fresh32<T>(src);
      in.raw[0] = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
      in.raw[1] = make_uint4(v.w[4], v.w[5], v.w[6], v.w[7]);
    } else {
      in.raw[0] = ld_fresh16(src);
      in.raw[1] = ld_fresh16(src + 8);
    }
  }
  P lo2 = in.v[0], hi2 = in.v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) { lo2 = min2_nan(lo2, in.v[i]); hi2 = max2_nan(hi2, in.v[i]); }
#pragma unroll
  for (int o = 1; o < kGroupLanes; o *= 2) {
    lo2 = min2_nan(lo2, shfl_xor_pair(lo2, o));
    hi2 = max2_nan(hi2, shfl_xor_pair(hi2, o));
  }
  if (!live) return;
  const T lo16 = __hmin_nan(lo2.x, lo2.y), hi16 = __hmax_nan(hi2.x, hi2.y);
  const float lo = to_f32(lo16);
  const T step16 = from_f32<T>((to_f32(hi16) - lo) / 15.0f);
  const float step = to_f32(step16);
  uint32_t w[2] = {0, 0};
  if (step >= Pair<T>::kTiny && step <= 0x1p100f) {
    // (x - lo) / step < 15.5 here, since the step is within 2^-8 of a fifteenth of the range: no clamp.  Adding 1.5 * 2^23
    // rounds to the nearest even integer and leaves the code in the low bits; eight of them are joined by shifts and adds,
    // and the eight exponent fields taken off at the end.
    const float y = __frcp_rn(step);
    const float2 y2 = make_float2(y, y), s2 = make_float2(-step, -step), l2 = make_float2(-lo, -lo), magic = make_float2(12582912.f, 12582912.f);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t acc = 0;
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        const float2 r = sm100::add2(div2(sm100::add2(widen2(in.v[half * 4 + i]), l2), s2, y2), magic);
        acc = (acc << 4) + __float_as_uint(r.y);
        acc = (acc << 4) + __float_as_uint(r.x);
      }
      w[half] = acc - 0x4b400000u * 0x11111111u;
    }
  } else if (step > 0.f) {            // steps near the ends of the range, and NaN and infinity, whose codes do not matter
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = widen2(in.v[i]);
      const uint32_t ca = (uint32_t)fminf(fmaxf(rintf((f.x - lo) / step), 0.f), 15.f);
      const uint32_t cb = (uint32_t)fminf(fmaxf(rintf((f.y - lo) / step), 0.f), 15.f);
      w[i / 4] |= (ca | (cb << 4)) << (8 * (i & 3));
    }
  }
  const uint32_t s32 = (uint32_t)slot, page = p.page_div(s32), off = s32 - page * (uint32_t)p.page_size;
  const int64_t dst = ((int64_t)page * p.heads + h) * p.page_size + off;
  *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(side.cache) + dst * (DIM / 2) + part * 8) = make_uint2(w[0], w[1]);
  if (part % kGroupLanes == 0) {
    P sc;
    sc.x = step16;
    sc.y = lo16;
    reinterpret_cast<P*>(side.scale)[dst * (DIM / GROUP) + part / kGroupLanes] = sc;
  }
}

// A thread widens 16 columns of two rows; both rows' slots, then both rows' codes are on their way at once.
template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(256)
kv_read_u4g_kernel(const CacheArgs p) {
  using P = typename Pair<T>::type;
  constexpr int kLanes = DIM / 16, kGroupLanes = GROUP / 16, kRows = 256 / kLanes;
  dependency_wait();
  dependency_release();
  const Side side = blockIdx.y ? p.v : p.k;
  const int part = threadIdx.x % kLanes;
  uint32_t t[2];
  int h[2];
  int64_t slot[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t row = (blockIdx.x * 2 + k) * kRows + threadIdx.x / kLanes;
    t[k] = p.head_div(row);
    h[k] = (int)(row - t[k] * p.heads);
    slot[k] = row < p.rows ? p.slots[t[k]] : -1;
  }
  uint2 codes[2];
  P scale[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (slot[k] >= 0 && slot[k] < p.total_slots) {
      const uint32_t s32 = (uint32_t)slot[k], page = p.page_div(s32), off = s32 - page * (uint32_t)p.page_size;
      const int64_t src = ((int64_t)page * p.heads + h[k]) * p.page_size + off;
      codes[k] = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(side.cache) + src * (DIM / 2) + part * 8);
      scale[k] = reinterpret_cast<const P*>(side.scale)[src * (DIM / GROUP) + part / kGroupLanes];
    }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (slot[k] >= 0 && slot[k] < p.total_slots) {
      const float2 sc = widen2(scale[k]);
      const float2 s2 = make_float2(sc.x, sc.x), l2 = make_float2(sc.y, sc.y), m128 = make_float2(-128.f, -128.f);
      Vec32<T> out;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w = half ? codes[k].y : codes[k].x;
        float2 f[4];                  // columns i and i + 4 of the word
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;        // bf16 pair of 128 + code
          const float2 c = sm100::add2(make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)), m128);
          f[i] = sm100::fma2(s2, c, l2);      // s * code is exact in fp32, so this is one rounding; then the output's
        }
        out.w[half * 4 + 0] = narrow2<T>(make_float2(f[0].x, f[1].x));
        out.w[half * 4 + 1] = narrow2<T>(make_float2(f[2].x, f[3].x));
        out.w[half * 4 + 2] = narrow2<T>(make_float2(f[0].y, f[1].y));
        out.w[half * 4 + 3] = narrow2<T>(make_float2(f[2].y, f[3].y));
      }
      T* dst = reinterpret_cast<T*>(side.x) + t[k] * side.stride + h[k] * DIM + part * 16;
      if (p.wide) {
        st_stream32(dst, out);
      } else {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(out.w[0], out.w[1], out.w[2], out.w[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(out.w[4], out.w[5], out.w[6], out.w[7]);
      }
    }
}

// ---- e4m3: a warp owns a row and keeps it in registers, 8 columns (16 bytes) a lane and pass ----------------------------
template <typename T, int PASSES>
__global__ void __launch_bounds__(256)
kv_write_e4m3_kernel(const CacheArgs p, const int dim) {
  using P = typename Pair<T>::type;
  dependency_wait();
  dependency_release();
  const Side side = blockIdx.y ? p.v : p.k;
  const int lane = threadIdx.x % 32;
  const uint32_t t = blockIdx.x * 8 + threadIdx.x / 32;
  if (t >= p.tokens) return;                                   // the whole warp
  const int64_t slot = p.slots[t];
  const T* src = reinterpret_cast<const T*>(side.x) + t * side.stride;
  union { uint4 raw; P v[4]; } in[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int c = (i * 32 + lane) * 8;
    in[i].raw = c < dim ? ld_fresh16(src + c) : make_uint4(0, 0, 0, 0);
  }
  P top = __habs2(in[0].v[0]);
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max2_nan(top, __habs2(in[i].v[e]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max2_nan(top, shfl_xor_pair(top, o));
  if (slot < 0 || slot >= p.total_slots) return;
  float amax = to_f32(__hmax_nan(top.x, top.y));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(1e-4f));
  const float s = amax / 448.0f;
  // The quick quotient is that by -s, and the bytes' signs are turned over: so the correction, whose remainder of an exact
  // quotient is +0, leaves both zeros their sign (by s, -0 would come out as +0).
  const float y = -__frcp_rn(s);
  const float2 y2 = make_float2(y, y), s2 = make_float2(s, s);
  const bool quick = s <= 0x1p100f;                            // s >= 2^-23 always
  const uint32_t turn = quick ? 0x80808080u : 0u;
  uint8_t* dst = reinterpret_cast<uint8_t*>(side.cache) + slot * dim;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int c = (i * 32 + lane) * 8;
    if (c < dim) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a = widen2(in[i].v[e]);
        const float2 q = quick ? div2(a, s2, y2) : make_float2(a.x / s, a.y / s);
        w[e / 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(q, __NV_SATFINITE, __NV_E4M3) << (16 * (e & 1));
      }
      *reinterpret_cast<uint2*>(dst + c) = make_uint2(w[0] ^ turn, w[1] ^ turn);
    }
  }
  if (lane == 0) reinterpret_cast<float*>(side.scale)[slot] = s;
}

// COLS columns a thread and item; a block takes `per_block` tokens, at most two items a thread, both on their way at once.
template <typename T, int COLS>
__global__ void __launch_bounds__(256)
kv_read_e4m3_kernel(const CacheArgs p, const int dim, const int per_block) {
  dependency_wait();
  dependency_release();
  const Side side = blockIdx.y ? p.v : p.k;
  const int vecs = dim / COLS;
  const uint32_t t0 = blockIdx.x * (uint32_t)per_block;
  const int items = (int)min((uint32_t)per_block, p.tokens - t0) * vecs;
  uint32_t t[2];
  int col[2];
  int64_t slot[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = threadIdx.x + 256 * k;
    const uint32_t in_block = p.vec_div((uint32_t)i);
    t[k] = t0 + in_block;
    col[k] = (i - (int)in_block * vecs) * COLS;
    slot[k] = i < items ? p.slots[t[k]] : -1;
  }
  uint32_t codes[2][COLS / 4];
  float s[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (slot[k] >= 0 && slot[k] < p.total_slots) {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(side.cache) + slot[k] * dim + col[k];
      if constexpr (COLS == 16) {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        codes[k][0] = w.x; codes[k][1] = w.y; codes[k][2] = w.z; codes[k][3] = w.w;
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        codes[k][0] = w.x; codes[k][1] = w.y;
      }
      s[k] = reinterpret_cast<const float*>(side.scale)[slot[k]];
    }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (slot[k] >= 0 && slot[k] < p.total_slots) {
      uint32_t out[COLS / 2];
#pragma unroll
      for (int e = 0; e < COLS / 2; ++e) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes[k][e / 2] >> (16 * (e & 1))), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));    // e4m3 -> fp16 is exact
        out[e] = narrow2<T>(make_float2(f.x * s[k], f.y * s[k]));
      }
      T* dst = reinterpret_cast<T*>(side.x) + t[k] * side.stride + col[k];
      if constexpr (COLS == 16) {
        Vec32<T> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.w[e] = out[e];
        st_stream32(dst, v);
      } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
      }
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------
template <typename T, int DIM>
static int launch_u4g(const CacheArgs& a, int group, int sides, bool write, cudaStream_t s) {
  const unsigned rows_per_block = 256 / (DIM / 16) * (write ? 1 : 2);
  const dim3 grid((a.rows + rows_per_block - 1) / rows_per_block, (unsigned)sides);
  cudaError_t rc = cudaSuccess;
  auto go = [&](auto g) {
    constexpr int G = decltype(g)::value;
    if constexpr (G <= DIM) {
      rc = launch_overlapped(write ? kv_write_u4g_kernel<T, DIM, G> : kv_read_u4g_kernel<T, DIM, G>, grid, dim3(256), 0, s, a);
    }
  };
  if (group == 32) go(std::integral_constant<int, 32>());
  else if (group == 64) go(std::integral_constant<int, 64>());
  else go(std::integral_constant<int, 128>());
  TL_CUDA(rc);
  TL_LAUNCH_CHECK(write ? "kv_write_u4g_kernel" : "kv_read_u4g_kernel");
  return TL_B200_OK;
}

template <typename T>
static int launch_cache(const CacheArgs& a, int64_t dim, int64_t group, int format, int sides, bool write, cudaStream_t s) {
  if (format == TL_U4G) {
    if (dim == 64) return launch_u4g<T, 64>(a, (int)group, sides, write, s);
    if (dim == 128) return launch_u4g<T, 128>(a, (int)group, sides, write, s);
    return launch_u4g<T, 256>(a, (int)group, sides, write, s);
  }
  if (write) {
    const dim3 grid((unsigned)((a.tokens + 7) / 8), (unsigned)sides);
    auto kernel = dim <= 256 ? kv_write_e4m3_kernel<T, 1> : dim <= 512 ? kv_write_e4m3_kernel<T, 2>
                : dim <= 768 ? kv_write_e4m3_kernel<T, 3> : kv_write_e4m3_kernel<T, 4>;
    TL_CUDA(launch_overlapped(kernel, grid, dim3(256), 0, s, a, (int)dim));
    TL_LAUNCH_CHECK("kv_write_e4m3_kernel");
  } else {
    const bool sixteen = dim % 16 == 0 && a.wide;
    const int vecs = (int)dim / (sixteen ? 16 : 8), per_block = 512 / vecs;      // at most 1024 columns: 4 tokens or more
    CacheArgs b = a;
    b.vec_div = FastDiv((uint32_t)vecs);
    const dim3 grid((a.tokens + per_block - 1) / per_block, (unsigned)sides);
    TL_CUDA(launch_overlapped(sixteen ? kv_read_e4m3_kernel<T, 16> : kv_read_e4m3_kernel<T, 8>, grid, dim3(256), 0, s, b, (int)dim, per_block));
    TL_LAUNCH_CHECK("kv_read_e4m3_kernel");
  }
  return TL_B200_OK;
}

static int cache_call(const char* who, const int64_t* slots, int64_t tokens, const void* k, int64_t k_stride, const void* k_cache,
                      const void* k_scale, const void* v, int64_t v_stride, const void* v_cache, const void* v_scale, int64_t heads,
                      int64_t dim, int64_t group, int64_t num_pages, int64_t page_size, int format, int dtype, bool write, void* stream) {
  TL_REQUIRE(tokens >= 0 && heads >= 1 && dim >= 1 && num_pages >= 0 && page_size >= 1, "%s: bad size", who);
  TL_REQUIRE(dtype == TL_BF16 || dtype == TL_F16, "%s: rows must be bfloat16 or float16", who);
  TL_REQUIRE(format == TL_U4G || format == TL_E4M3, "%s: unknown cache format %d", who, format);
  if (format == TL_U4G) {
    TL_REQUIRE(dim == 64 || dim == 128 || dim == 256, "%s: a 4-bit cache has 64, 128 or 256 columns, not %lld", who, (long long)dim);
    TL_REQUIRE((group == 32 || group == 64 || group == 128) && group <= dim, "%s: groups of 32, 64 or 128 columns, at most the row", who);
  } else {
    TL_REQUIRE(heads == 1, "%s: an e4m3 cache has a single kv head", who);
    TL_REQUIRE(dim % 8 == 0 && dim <= 1024, "%s: e4m3 rows have a multiple of 8 columns, at most 1024", who);
  }
  TL_REQUIRE(num_pages < (1ll << 31) && page_size < (1ll << 31) && num_pages * page_size < (1ll << 31), "%s: cache too large", who);
  TL_REQUIRE(heads <= 65536 && tokens < (1ll << 31) && tokens * heads < (1ll << 31) - 256, "%s: size too large", who);
  if (tokens == 0 || num_pages == 0) return TL_B200_OK;        // no slot is inside a cache without pages
  const bool both = v != nullptr || v_cache != nullptr || v_scale != nullptr;
  TL_REQUIRE(slots && k && k_cache && k_scale, "%s: null tensor pointer", who);
  TL_REQUIRE(!both || (v && v_cache && v_scale), "%s: null tensor pointer", who);
  TL_REQUIRE(aligned16(k) && aligned16(k_cache) && k_stride % 8 == 0 && (!both || (aligned16(v) && aligned16(v_cache) && v_stride % 8 == 0)),
             "%s: rows and caches must be 16-byte aligned", who);
  TL_REQUIRE((reinterpret_cast<uintptr_t>(k_scale) & 3u) == 0 && (!both || (reinterpret_cast<uintptr_t>(v_scale) & 3u) == 0) &&
                 (reinterpret_cast<uintptr_t>(slots) & 7u) == 0, "%s: scales or slots not aligned", who);
  if (!write) TL_REQUIRE(tokens == 1 || (k_stride >= heads * dim && (!both || v_stride >= heads * dim)), "%s: output rows overlap", who);
  CacheArgs a;
  a.slots = slots;
  a.tokens = (uint32_t)tokens;
  a.rows = (uint32_t)(tokens * heads);
  a.k = Side{const_cast<void*>(k), k_stride, const_cast<void*>(k_cache), const_cast<void*>(k_scale)};
  a.v = Side{const_cast<void*>(v), v_stride, const_cast<void*>(v_cache), const_cast<void*>(v_scale)};
  a.heads = (int)heads;
  a.page_size = (int)page_size;
  a.total_slots = num_pages * page_size;
  a.head_div = FastDiv((uint32_t)heads);
  a.page_div = FastDiv((uint32_t)page_size);
  a.wide = aligned32(k) && k_stride % 16 == 0 && (!both || (aligned32(v) && v_stride % 16 == 0));
  cudaStream_t s = (cudaStream_t)stream;
  const int sides = both ? 2 : 1;
  return dtype == TL_BF16 ? launch_cache<__nv_bfloat16>(a, dim, group, format, sides, write, s)
                          : launch_cache<__half>(a, dim, group, format, sides, write, s);
}

}  // namespace tl

extern "C" int tl_b200_kv_cache_write(const int64_t* slots, const void* k, void* k_cache, void* k_scale, const void* v, void* v_cache,
                                      void* v_scale, int64_t tokens, int64_t k_stride, int64_t v_stride, int64_t heads, int64_t dim,
                                      int64_t group, int64_t num_pages, int64_t page_size, int format, int dtype, void* stream) {
  return tl::cache_call("kv_cache_write", slots, tokens, k, k_stride, k_cache, k_scale, v, v_stride, v_cache, v_scale, heads, dim, group,
                        num_pages, page_size, format, dtype, true, stream);
}

extern "C" int tl_b200_kv_cache_read(const int64_t* slots, const void* k_cache, const void* k_scale, void* k, const void* v_cache,
                                     const void* v_scale, void* v, int64_t tokens, int64_t k_stride, int64_t v_stride, int64_t heads,
                                     int64_t dim, int64_t group, int64_t num_pages, int64_t page_size, int format, int dtype, void* stream) {
  return tl::cache_call("kv_cache_read", slots, tokens, k, k_stride, k_cache, k_scale, v, v_stride, v_cache, v_scale, heads, dim, group,
                        num_pages, page_size, format, dtype, false, stream);
}
