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
// HBM-bound: a 16-bit row is read (written) once and its codes written (read) once.
#include "common.cuh"

#include <type_traits>

namespace tl {

struct CacheArgs {
  const int64_t* slots;
  int64_t tokens;
  void* x[2];                 // rows of keys and of values (x[1] only with gridDim.y == 2)
  int64_t x_stride[2];        // elements from one token to the next
  void* cache[2];
  void* scale[2];
  int heads, page_size;
  int64_t total_slots;
};

// NaN-propagating minimum and maximum of two packed 16-bit values.
__device__ __forceinline__ __nv_bfloat162 min2_nan(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2_nan(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 min2_nan(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 max2_nan(__half2 a, __half2 b) { return __hmax2_nan(a, b); }

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

__device__ __forceinline__ float2 widen2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 widen2(__half2 v) { return __half22float2(v); }

template <typename P> __device__ __forceinline__ P shfl_xor_pair(P v, int o) {
  uint32_t w = *reinterpret_cast<uint32_t*>(&v);
  w = __shfl_xor_sync(0xffffffffu, w, o);
  return *reinterpret_cast<P*>(&w);
}

// ---- 4 bits: a thread holds 16 columns (32 bytes in, 8 bytes of codes out); GROUP/16 neighbouring lanes own a group -----
template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(256)
kv_write_u4g_kernel(const CacheArgs p) {
  using P = typename Pair<T>::type;
  constexpr int kLanes = DIM / 16, kGroupLanes = GROUP / 16;
  const int which = blockIdx.y;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / kLanes;
  const int part = (int)(idx % kLanes);
  const int64_t t = row / p.heads;
  const int h = (int)(row - t * p.heads);
  const int64_t slot = t < p.tokens ? __ldg(p.slots + t) : -1;
  const bool live = slot >= 0 && slot < p.total_slots;
  union { uint4 raw[2]; P v[8]; } in;
  in.raw[0] = in.raw[1] = make_uint4(0, 0, 0, 0);
  if (live) {
    const T* src = reinterpret_cast<const T*>(p.x[which]) + t * p.x_stride[which] + h * DIM + part * 16;
    in.raw[0] = ld_stream16(src);
    in.raw[1] = ld_stream16(src + 8);
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
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = widen2(in.v[i]);
    // the same fp32 subtraction, IEEE division and round-to-even as the definition: codes agree bit for bit
    const float a = step > 0.f ? rintf((f.x - lo) / step) : 0.f, b = step > 0.f ? rintf((f.y - lo) / step) : 0.f;
    const uint32_t ca = (uint32_t)fminf(fmaxf(a, 0.f), 15.f), cb = (uint32_t)fminf(fmaxf(b, 0.f), 15.f);
    w[i / 4] |= (ca | (cb << 4)) << (8 * (i & 3));
  }
  const uint32_t s32 = (uint32_t)slot, page = s32 / (uint32_t)p.page_size, off = s32 - page * (uint32_t)p.page_size;
  const int64_t dst = ((int64_t)page * p.heads + h) * p.page_size + off;
  *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(p.cache[which]) + dst * (DIM / 2) + part * 8) = make_uint2(w[0], w[1]);
  if (part % kGroupLanes == 0) {
    P sc;
    sc.x = step16;
    sc.y = lo16;
    reinterpret_cast<P*>(p.scale[which])[dst * (DIM / GROUP) + part / kGroupLanes] = sc;
  }
}

template <typename T, int DIM, int GROUP>
__global__ void __launch_bounds__(256)
kv_read_u4g_kernel(const CacheArgs p) {
  using P = typename Pair<T>::type;
  constexpr int kLanes = DIM / 16, kGroupLanes = GROUP / 16;
  const int which = blockIdx.y;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = idx / kLanes;
  const int part = (int)(idx % kLanes);
  const int64_t t = row / p.heads;
  const int h = (int)(row - t * p.heads);
  const int64_t slot = t < p.tokens ? __ldg(p.slots + t) : -1;
  if (slot < 0 || slot >= p.total_slots) return;
  const uint32_t s32 = (uint32_t)slot, page = s32 / (uint32_t)p.page_size, off = s32 - page * (uint32_t)p.page_size;
  const int64_t src = ((int64_t)page * p.heads + h) * p.page_size + off;
  const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(p.cache[which]) + src * (DIM / 2) + part * 8);
  const float2 sc = widen2(reinterpret_cast<const P*>(p.scale[which])[src * (DIM / GROUP) + part / kGroupLanes]);
  union { uint4 raw[2]; T e[16]; } out;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t c = ((i < 8 ? w.x : w.y) >> (4 * (i & 7))) & 15u;
    out.e[i] = from_f32<T>(fmaf(sc.x, (float)c, sc.y));      // s * code is exact in fp32, so this is one rounding, then the output's
  }
  T* dst = reinterpret_cast<T*>(p.x[which]) + t * p.x_stride[which] + h * DIM + part * 16;
  reinterpret_cast<uint4*>(dst)[0] = out.raw[0];
  reinterpret_cast<uint4*>(dst)[1] = out.raw[1];
}

// ---- e4m3: a warp owns a row and keeps it in registers, 8 columns (16 bytes) a lane and pass ----------------------------
template <typename T, int PASSES>
__global__ void __launch_bounds__(256)
kv_write_e4m3_kernel(const CacheArgs p, const int dim) {
  const int which = blockIdx.y;
  const int lane = threadIdx.x % 32;
  const int64_t t = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t slot = t < p.tokens ? __ldg(p.slots + t) : -1;
  if (slot < 0 || slot >= p.total_slots) return;               // the whole warp
  const T* src = reinterpret_cast<const T*>(p.x[which]) + t * p.x_stride[which];
  Vec16<T> v[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int c = (i * 32 + lane) * 8;
    v[i].raw = c < dim ? ld_stream16(src + c) : make_uint4(0, 0, 0, 0);
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(to_f32(v[i].e[e]));
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(a));
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, amax, o);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(a));
  }
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(1e-4f));
  const float s = amax / 448.0f;
  uint8_t* dst = reinterpret_cast<uint8_t*>(p.cache[which]) + slot * dim;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int c = (i * 32 + lane) * 8;
    if (c < dim) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const __nv_fp8x2_storage_t two =
            __nv_cvt_float2_to_fp8x2(make_float2(to_f32(v[i].e[e]) / s, to_f32(v[i].e[e + 1]) / s), __NV_SATFINITE, __NV_E4M3);
        w[e / 4] |= (uint32_t)two << (8 * (e & 3));
      }
      *reinterpret_cast<uint2*>(dst + c) = make_uint2(w[0], w[1]);
    }
  }
  if (lane == 0) reinterpret_cast<float*>(p.scale[which])[slot] = s;
}

template <typename T>
__global__ void __launch_bounds__(256)
kv_read_e4m3_kernel(const CacheArgs p, const int dim) {
  const int which = blockIdx.y;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int vecs = dim / 8;
  const int64_t t = idx / vecs;
  const int c = (int)(idx - t * vecs) * 8;
  const int64_t slot = t < p.tokens ? __ldg(p.slots + t) : -1;
  if (slot < 0 || slot >= p.total_slots) return;
  const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(p.cache[which]) + slot * dim + c);
  const float s = reinterpret_cast<const float*>(p.scale[which])[slot];
  Vec16<T> out;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));      // e4m3 -> fp16 is exact
    out.e[e] = from_f32<T>(f.x * s);
    out.e[e + 1] = from_f32<T>(f.y * s);
  }
  *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.x[which]) + t * p.x_stride[which] + c) = out.raw;
}

// ---- host --------------------------------------------------------------------------------------------------------------
template <typename T, int DIM>
static int launch_u4g(const CacheArgs& a, int group, int sides, bool write, cudaStream_t s) {
  const int64_t threads = a.tokens * a.heads * (DIM / 16);
  const dim3 grid((unsigned)((threads + 255) / 256), (unsigned)sides);
  auto go = [&](auto g) {
    constexpr int G = decltype(g)::value;
    if constexpr (G <= DIM) {
      if (write) kv_write_u4g_kernel<T, DIM, G><<<grid, 256, 0, s>>>(a);
      else kv_read_u4g_kernel<T, DIM, G><<<grid, 256, 0, s>>>(a);
    }
  };
  if (group == 32) go(std::integral_constant<int, 32>());
  else if (group == 64) go(std::integral_constant<int, 64>());
  else go(std::integral_constant<int, 128>());
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
    const int d = (int)dim;
    if (dim <= 256) kv_write_e4m3_kernel<T, 1><<<grid, 256, 0, s>>>(a, d);
    else if (dim <= 512) kv_write_e4m3_kernel<T, 2><<<grid, 256, 0, s>>>(a, d);
    else if (dim <= 768) kv_write_e4m3_kernel<T, 3><<<grid, 256, 0, s>>>(a, d);
    else kv_write_e4m3_kernel<T, 4><<<grid, 256, 0, s>>>(a, d);
    TL_LAUNCH_CHECK("kv_write_e4m3_kernel");
  } else {
    const int64_t threads = a.tokens * (dim / 8);
    kv_read_e4m3_kernel<T><<<dim3((unsigned)((threads + 255) / 256), (unsigned)sides), 256, 0, s>>>(a, (int)dim);
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
  TL_REQUIRE(num_pages <= (1ll << 31) && page_size <= (1ll << 31) && num_pages * page_size < (1ll << 31), "%s: cache too large", who);
  // grid.x < 2^31 blocks of 256 threads of at least 8 columns; the products below cannot overflow
  TL_REQUIRE(heads <= 65536 && tokens < (1ll << 31) && tokens * heads * dim < (1ll << 41), "%s: size too large", who);
  if (tokens == 0) return TL_B200_OK;
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
  a.tokens = tokens;
  a.x[0] = const_cast<void*>(k); a.x[1] = const_cast<void*>(v);
  a.x_stride[0] = k_stride; a.x_stride[1] = v_stride;
  a.cache[0] = const_cast<void*>(k_cache); a.cache[1] = const_cast<void*>(v_cache);
  a.scale[0] = const_cast<void*>(k_scale); a.scale[1] = const_cast<void*>(v_scale);
  a.heads = (int)heads;
  a.page_size = (int)page_size;
  a.total_slots = num_pages * page_size;
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
