// Attention over a paged cache held in 4 bits (TL_U4G, see kv_cache.cu), grouped query heads, s_q query tokens a sequence.
//
//   out[b,i,h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q[b,i,h] . k_t),  t < len_b - s_q + i + 1,
//   k_t = s c + lo per group (likewise v_t); a row that sees no key is zero.
//
// One warp per (sequence, query token, head): lanes share the columns, keys one after the other with a running maximum.
#include "sm100.cuh"
#include "mla_common.cuh"

#include <type_traits>

namespace tl {
using namespace sm100;

struct AttnInt4Params {
  const void* q;
  int64_t q_sb, q_ss;                  // elements from one sequence / query token to the next
  const uint8_t *k_codes, *v_codes;
  const void *k_scale, *v_scale;
  const int *table, *lens;
  void* out;
  int batch, s_q, h_q, h_kv, page_size, max_pages, num_pages, len_cap;
  float scale;
};

template <typename T> __device__ __forceinline__ float2 scale_pair(const void* base, int64_t i) {
  const T* p = reinterpret_cast<const T*>(base) + 2 * i;
  return make_float2(to_f32(p[0]), to_f32(p[1]));
}

template <typename T, int DIM>
__global__ void __launch_bounds__(128)
attn_int4_rows_kernel(const AttnInt4Params p, const int group) {
  constexpr int E = DIM / 32;                      // columns a lane holds: lane * E ..
  const int lane = threadIdx.x % 32;
  const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= (int64_t)p.batch * p.s_q * p.h_q) return;
  const int h = (int)(row % p.h_q), i = (int)(row / p.h_q % p.s_q), b = (int)(row / ((int64_t)p.h_q * p.s_q));
  const int kvh = h / (p.h_q / p.h_kv), groups = DIM / group, g = lane * E / group;
  const int len = mla_len(p.lens, b, p.len_cap), seen = len - p.s_q + i + 1;
  float q[E], acc[E];
  const T* qp = reinterpret_cast<const T*>(p.q) + b * p.q_sb + i * p.q_ss + (int64_t)h * DIM + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) { q[e] = to_f32(qp[e]); acc[e] = 0.f; }
  float m = -INFINITY, l = 0.f;
  for (int t = 0; t < seen; ++t) {
    const int page = __ldg(p.table + (int64_t)b * p.max_pages + t / p.page_size);
    if (!mla_page_ok(page, p.num_pages)) continue;
    const int64_t r = ((int64_t)page * p.h_kv + kvh) * p.page_size + t % p.page_size;
    const float2 ks = scale_pair<T>(p.k_scale, r * groups + g), vs = scale_pair<T>(p.v_scale, r * groups + g);
    float dot = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint32_t kc = p.k_codes[r * (DIM / 2) + (lane * E + e) / 2], vc = p.v_codes[r * (DIM / 2) + (lane * E + e) / 2];
      dot = fmaf(q[e], fmaf(ks.x, (float)(kc & 15u), ks.y), dot);
      dot = fmaf(q[e + 1], fmaf(ks.x, (float)(kc >> 4), ks.y), dot);
      v[e] = fmaf(vs.x, (float)(vc & 15u), vs.y);
      v[e + 1] = fmaf(vs.x, (float)(vc >> 4), vs.y);
    }
    const float s = warp_sum(dot) * p.scale;
    const float m_new = fmaxf(m, s);
    const float alpha = m == -INFINITY ? 0.f : expf(m - m_new), w = expf(s - m_new);
    l = fmaf(l, alpha, w);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(acc[e], alpha, w * v[e]);
    m = m_new;
  }
  T* o = reinterpret_cast<T*>(p.out) + row * DIM + lane * E;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = from_f32<T>(acc[e] * inv);
}

template <typename T>
static int launch_int4(const AttnInt4Params& p, int64_t dim, int64_t group, cudaStream_t s) {
  const int64_t rows = (int64_t)p.batch * p.s_q * p.h_q;
  const unsigned grid = (unsigned)((rows + 3) / 4);
  if (dim == 64) attn_int4_rows_kernel<T, 64><<<grid, 128, 0, s>>>(p, (int)group);
  else if (dim == 128) attn_int4_rows_kernel<T, 128><<<grid, 128, 0, s>>>(p, (int)group);
  else attn_int4_rows_kernel<T, 256><<<grid, 128, 0, s>>>(p, (int)group);
  TL_LAUNCH_CHECK("attn_int4_rows_kernel");
  return TL_B200_OK;
}

}  // namespace tl

using namespace tl;

extern "C" int64_t tl_b200_attn_decode_paged_int4_workspace_bytes(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  (void)batch; (void)s_q; (void)h_q; (void)h_kv; (void)dim;
  return 0;
}

extern "C" int64_t tl_b200_attn_decode_paged_int4_zero_bytes(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  (void)batch; (void)s_q; (void)h_q; (void)h_kv; (void)dim;
  return 0;
}

extern "C" int tl_b200_attn_decode_paged_int4(const void* q, const void* k_cache, const void* k_scale, const void* v_cache,
                                              const void* v_scale, const int32_t* block_table, const int32_t* cache_seqlens, void* out,
                                              int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim, int64_t group,
                                              int64_t q_stride_batch, int64_t q_stride_token, int64_t page_size,
                                              int64_t max_pages_per_seq, int64_t num_pages, float softmax_scale, int dtype,
                                              void* workspace, int64_t workspace_bytes, void* stream) {
  TL_REQUIRE(batch >= 0 && s_q >= 0 && h_q >= 1 && h_kv >= 1 && page_size >= 1 && max_pages_per_seq >= 0 && num_pages >= 0,
             "attn_decode_paged_int4: bad size");
  TL_REQUIRE(dtype == TL_BF16 || dtype == TL_F16, "attn_decode_paged_int4: q must be bfloat16 or float16");
  TL_REQUIRE(dim == 64 || dim == 128 || dim == 256, "attn_decode_paged_int4: head dim must be 64, 128 or 256, not %lld", (long long)dim);
  TL_REQUIRE((group == 32 || group == 64 || group == 128) && group <= dim,
             "attn_decode_paged_int4: groups of 32, 64 or 128 columns, at most the row");
  TL_REQUIRE(h_q % h_kv == 0, "attn_decode_paged_int4: h_q must be a multiple of h_kv");
  TL_REQUIRE(batch < (1 << 24) && s_q < (1 << 24) && h_q <= 65536 && batch * s_q * h_q < (1ll << 31),
             "attn_decode_paged_int4: size too large");
  TL_REQUIRE(num_pages < (1ll << 31) && page_size < (1ll << 31) && num_pages * page_size < (1ll << 31) && max_pages_per_seq < (1ll << 31),
             "attn_decode_paged_int4: cache too large");
  if (batch == 0 || s_q == 0) return TL_B200_OK;
  const bool keys = num_pages > 0 && max_pages_per_seq > 0;
  TL_REQUIRE(q && cache_seqlens && out && (!keys || (k_cache && k_scale && v_cache && v_scale && block_table)),
             "attn_decode_paged_int4: null tensor pointer");
  TL_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache) && aligned16(v_cache) && aligned16(k_scale) && aligned16(v_scale) &&
                 q_stride_batch % 8 == 0 && q_stride_token % 8 == 0, "attn_decode_paged_int4: tensors and rows of q must be 16-byte aligned");
  AttnInt4Params p;
  p.q = q; p.q_sb = q_stride_batch; p.q_ss = q_stride_token;
  p.k_codes = (const uint8_t*)k_cache; p.v_codes = (const uint8_t*)v_cache;
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.table = block_table; p.lens = cache_seqlens; p.out = out;
  p.batch = (int)batch; p.s_q = (int)s_q; p.h_q = (int)h_q; p.h_kv = (int)h_kv;
  p.page_size = (int)page_size; p.max_pages = (int)max_pages_per_seq; p.num_pages = (int)num_pages;
  const int64_t cap = max_pages_per_seq * page_size;           // a sequence may name a page more than once
  p.len_cap = (int)(cap < 0x7fffff00ll ? cap : 0x7fffff00ll);
  if (num_pages == 0) p.len_cap = 0;
  p.scale = softmax_scale;
  (void)workspace; (void)workspace_bytes;
  return dtype == TL_BF16 ? launch_int4<__nv_bfloat16>(p, dim, group, (cudaStream_t)stream)
                          : launch_int4<__half>(p, dim, group, (cudaStream_t)stream);
}
