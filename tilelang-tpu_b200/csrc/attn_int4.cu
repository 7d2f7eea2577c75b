// Attention over a paged cache held in 4 bits (TL_U4G, see kv_cache.cu): grouped query heads, s_q query tokens a sequence.
//
//   out[b,i,h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q[b,i,h] . k_t),  t < len_b - s_q + i + 1,
//   k_t = s c + lo per group of columns (likewise v_t); a row that sees no key is zero.
//
// What bounds it.  A key of one kv head is dim/2 + 4 groups bytes, twice with its value (136 bytes at dim 128 and one
// group), against 4 dim flop for each of the few query heads that share it: HBM, if the codes can be widened fast enough.
// At the measured copy rate an SM receives 43 codes a clock, so every instruction spent on eight codes counts; a score
// costs next to nothing beside that.
//
// Layout.  The MMAs are the warp-level m16n8k16 ones: at most 8 or 16 query rows share a key, so a 128-row tensor-memory
// tile would be 90% padding, and codes have to pass through registers to be widened anyway.  Keys (and columns of V) are
// the 16 rows, queries the 8 columns:  S^T = K Q^T  and  O^T = V^T P^T, both in fp16.  Widening is one AND per pair of
// codes: a nibble in the low bits of an fp16 number is the subnormal c 2^-24 (the next nibble 16 c 2^-24), which the tensor
// core multiplies exactly; the powers of two are taken back outside the loop.
//   * K: a lane holds whole 32-bit words of a key; word & 0x000f000f are columns 0 and 4 of the word, one register of the A
//     operand.  The columns of Q are permuted (and those of odd nibbles divided by 16) when they are loaded, once a
//     sequence; a power of two per query tile brings Q into fp16's range, and what falls below it is 2^-35 of its largest.
//   * V: a register of the A operand is one column of two neighbouring tokens: one byte permute joins half words of the two.
//   * Steps and minima never touch the codes:  q . k = s (q . c) + lo sum(q) per group, and the value's step multiplies p
//     (rounded to fp16 with a power-of-two factor per warp that keeps p s in range: 2^-12 of each weight), its minimum
//     adds p lo in fp32.  The weights' rounding should meet c - 8, not c, so 8 times the sum of the ROUNDED weights, from an
//     MMA with ones, is taken off, and 8 s goes to the minimum.
// Every group of columns has its own MMAs, so a group's step can multiply the score or the weight.
//
// Work.  Sequences are cut into units of 128 tokens; the list of all (sequence, kv head, query tile, unit) is dealt out in
// equal contiguous ranges to the CTAs, whatever the lengths.  A unit is a stage of a ring that bulk copies fill, page by
// page, across the ends of sequences; the warps take turns to issue them, so that no warp falls behind and none is idle.
// Each of the eight warps takes 16 tokens of a unit.  Their results are joined in shared memory,
// a few rows at a time, at the end of a segment; a segment that CTAs share leaves fp32 partial sums, and the CTA that arrives last adds them up in
// their fixed order, so the result does not depend on who that is.
#include "sm100.cuh"
#include "mla_common.cuh"

#include <cfloat>
#include <type_traits>

namespace tl {
using namespace sm100;

struct AttnInt4Params {
  const void* q;
  int64_t q_sb, q_ss;                  // elements from one sequence / query token to the next
  const uint8_t *k_codes, *v_codes;
  const uint8_t *k_scale, *v_scale;    // (step, minimum) pairs of the 16-bit type
  const int *table, *lens;
  void* out;
  int batch, s_q, h_q, h_kv, per, page_size, max_pages, num_pages, len_cap;
  int rows, q_tiles;                   // query rows of a kv head (s_q * per), tiles of them
  FastDiv page_div;                    // t / page_size
  float scale_log2;
  int* counters;                       // one per CTA, zero between calls
  float* partial;                      // [2 * gridDim.x][kRows * (dim + 2)]
  int* status;
};

constexpr int kWarps = 8, kUnit = 16 * kWarps;

template <int DIM, int GROUP, int NT> struct I4Cfg {
  static constexpr int kGroups = DIM / GROUP;
  static constexpr int kCodes = kUnit * DIM / 2;                        // a stage: codes of K and of V, their scales,
  static constexpr int kScales = kUnit * 4 * kGroups;                   // a word of 16 live bits per warp
  static constexpr int kMask = 2 * kCodes + 2 * kScales;
  static constexpr int kStage = kMask + 4 * kWarps;
  static constexpr int kRows = 8 * NT;
  static constexpr int kJoinRows = 4 * NT;                              // rows joined at a time
  static constexpr int kPitch = DIM + 4;                                // floats of a row of the join buffer
  static constexpr int kJoin = kWarps * (kJoinRows * kPitch + 2 * kRows) * 4;   // partial rows, maxima and sums of the eight warps
  static constexpr int kCtas = DIM * NT <= 128 ? 2 : 1;                 // resident per SM: registers and shared memory
  static constexpr int kFit = ((227 * 1024 / kCtas) - 1024 - kJoin - 384) / kStage;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kAhead = kStages - 2;                            // units in flight while one is worked on
  static constexpr int kSmem = kStages * kStage + kJoin + 384;
  static_assert(kStages >= 3 && kAhead <= kWarps, "ring");
  static_assert(kStage % 16 == 0, "bulk copies are 16-byte aligned");
  static_assert(kWarps * kJoinRows * kPitch >= 5 * 32 * kWarps, "the join buffer serves the merge of partial sums too");
};

// Plain loads and non-volatile MMAs: the compiler may move them (never across the barriers, which clobber memory).
template <int WORDS> __device__ __forceinline__ void lds_words(const uint8_t* at, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  }
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Four nibbles of each half of `r` as fp16 pairs: c, 16 c, c, 16 c, each times 2^-24 (subnormal, exact).
__device__ __forceinline__ void widen4(uint32_t r, uint32_t (&u)[4]) {
  const uint32_t h = r >> 8;
  u[0] = r & 0x000f000fu;
  u[1] = r & 0x00f000f0u;
  u[2] = h & 0x000f000fu;
  u[3] = h & 0x00f000f0u;
}
template <typename T> __device__ __forceinline__ float2 widen_scale(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where a warp is in the list of units.  Units of a sequence: max(1, ceil(len / 128)), so an empty sequence still has its
// zero rows written.
struct UnitIter {
  int b, h, qt, u, units, len;
};
__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnit - 1) / kUnit : 1; }
__device__ __forceinline__ bool advance(UnitIter& it, const AttnInt4Params& p) {      // true: a new segment begins
  if (++it.u < it.units) return false;
  it.u = 0;
  if (++it.qt == p.q_tiles) {
    it.qt = 0;
    if (++it.h == p.h_kv) {
      it.h = 0;
      if (++it.b < p.batch) {
        it.len = mla_len(p.lens, it.b, p.len_cap);
        it.units = units_of(it.len);
      }
    }
  }
  return true;
}

template <typename T, int DIM, int GROUP, int NT>
__global__ void __launch_bounds__(32 * kWarps, I4Cfg<DIM, GROUP, NT>::kCtas)
attn_int4_kernel(const AttnInt4Params p) {
  using Cfg = I4Cfg<DIM, GROUP, NT>;
  constexpr int NG = Cfg::kGroups, ST = Cfg::kStages, MT = DIM / 16, MG = GROUP / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4;
  uint8_t* tail = smem + ST * Cfg::kStage;
  float* join = reinterpret_cast<float*>(tail);                  // [warps][join rows][pitch]
  float* join_m = join + kWarps * Cfg::kJoinRows * Cfg::kPitch;  // [warps][rows]
  float* join_l = join_m + kWarps * Cfg::kRows;
  // what only the ends of segments need stays in shared memory
  struct Shared {
    int64_t sums[kWarps];
    int64_t total, ctas, start, end, seq_base;         // seq_base: first unit of sequence it.b
    uint64_t full[ST], empty[ST];                      // a unit has landed; all warps have left it
    int first_b, last, abort;
  };
  Shared& sh = *reinterpret_cast<Shared*>(join_l + kWarps * Cfg::kRows);
  const uint32_t ring = smem_u32(smem), bar_full = smem_u32(sh.full), bar_empty = smem_u32(sh.empty);
  // Row r of the 16-row operands is token r ^ (r >> 1 & 1) of the tile: with unswizzled rows of 64 bytes K is then read
  // without bank conflicts and V with two-way ones.
  const int tok = g ^ (g >> 1 & 1);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(bar_full + 8 * i, 1);
      mbar_init(bar_empty + 8 * i, kWarps);
    }
    sh.abort = 0;
    mbar_fence_init();
  }

  // ---- this CTA's range of the list --------------------------------------------------------------------------------
  UnitIter it;
  int left;                                            // units of this CTA still to do
  {
    const int64_t per_unit = (int64_t)p.h_kv * p.q_tiles;
    const int chunk = (p.batch + 32 * kWarps - 1) / (32 * kWarps);
    const int b0 = min((int)threadIdx.x * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(mla_len(p.lens, b, p.len_cap));
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh.sums[warp] = incl;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.sums[w];
      total += sh.sums[w];
    }
    total *= per_unit;
    const int64_t ctas = total < gridDim.x ? total : gridDim.x;          // every one of them has a unit
    if (blockIdx.x >= ctas) return;                                      // the whole CTA
    const int64_t start = (int64_t)blockIdx.x * total / ctas, end = ((int64_t)blockIdx.x + 1) * total / ctas;
    int64_t base = before + incl - mine;
    if (base * per_unit <= start && start < (base + mine) * per_unit) {  // exactly one thread
      int b = b0, units = 0;
      for (; b < b1; ++b) {
        units = units_of(mla_len(p.lens, b, p.len_cap));
        if (start < (base + units) * per_unit) break;
        base += units;
      }
      sh.first_b = b;
      sh.seq_base = base * per_unit;
      sh.total = total;
      sh.ctas = ctas;
      sh.start = start;
      sh.end = end;
    }
    __syncthreads();
    left = (int)(end - start);                                           // the host checks that it fits
    it.b = sh.first_b;
    it.len = mla_len(p.lens, it.b, p.len_cap);
    it.units = units_of(it.len);
    const int64_t off = start - sh.seq_base;
    const int seg = (int)(off / it.units);
    it.u = (int)(off - (int64_t)seg * it.units);
    it.h = seg / p.q_tiles;
    it.qt = seg - it.h * p.q_tiles;
  }

  // ---- loads: one warp fills a stage with a unit, a lane per page ------------------------------------------------------
  const bool whole_rows = p.page_size % 4 == 0;         // pieces of pages are multiples of four rows: of 16 bytes of scales
  auto issue = [&](const UnitIter& w, int stage) {
    const uint32_t at = ring + stage * Cfg::kStage, full = bar_full + 8 * stage;
    const int t0 = w.u * kUnit, t1 = min(t0 + kUnit, w.len);
    const int* table = p.table + (int64_t)w.b * p.max_pages;
    uint32_t* masks = reinterpret_cast<uint32_t*>(smem + stage * Cfg::kStage + Cfg::kMask);
    if (whole_rows) {
      const int first = (int)p.page_div((uint32_t)t0);                    // at most 32 pages: they hold four tokens or more
      const int64_t edge = (int64_t)(first + lane) * p.page_size;         // first token of this lane's page
      const int begin = (int)max((int64_t)t0, min(edge, (int64_t)t1)), end = (int)min((int64_t)t1, edge + p.page_size);
      int page = -1;
      if (begin < end) page = __ldg(table + first + lane);
      const bool have = begin < end && mla_page_ok(page, p.num_pages);
      const int rows = have ? (end - begin + 3) / 4 * 4 : 0;              // up to three rows behind the last token, of the same page
      if (__all_sync(0xffffffffu, have || begin >= end) && t1 == t0 + kUnit) {
        if (lane < kWarps) masks[lane] = 0xffffu;
      } else {
        if (lane < kWarps) masks[lane] = 0;
        __syncwarp();
        if (have)
          for (int i = (begin - t0) / 16; i * 16 < end - t0; ++i) {
            const int lo = max(begin - t0 - i * 16, 0), hi = min(end - t0 - i * 16, 16);
            atomicOr(masks + i, (1u << hi) - (1u << lo));
          }
      }
      const uint32_t all = __reduce_add_sync(0xffffffffu, (uint32_t)rows);
      __syncwarp();
      if (lane == 0) mbar_expect_tx(full, all * (DIM + 8 * NG));
      __syncwarp();
      if (have) {
        // rows of the cache are fewer than 2^32
        const uint32_t row = ((uint32_t)page * p.h_kv + w.h) * (uint32_t)p.page_size + (uint32_t)(begin - (int)edge);
        const uint32_t n = (uint32_t)rows, to = (uint32_t)(begin - t0);
        bulk_load(at + to * (DIM / 2), p.k_codes + (uint64_t)row * (DIM / 2), n * (DIM / 2), full);
        bulk_load(at + 2 * Cfg::kCodes + to * (4 * NG), p.k_scale + (uint64_t)row * (4 * NG), n * (4 * NG), full);
        bulk_load(at + Cfg::kCodes + to * (DIM / 2), p.v_codes + (uint64_t)row * (DIM / 2), n * (DIM / 2), full);
        bulk_load(at + 2 * Cfg::kCodes + Cfg::kScales + to * (4 * NG), p.v_scale + (uint64_t)row * (4 * NG), n * (4 * NG), full);
      }
    } else {                                              // any page size: a lane per token, by plain loads and stores
      uint8_t* stage_ptr = smem + stage * Cfg::kStage;
#pragma unroll 1
      for (int i = 0; i < kUnit / 32; ++i) {
        const int to = i * 32 + lane, t = t0 + to;
        bool have = t < t1;
        uint32_t row = 0;
        if (have) {
          const uint32_t pg = p.page_div((uint32_t)t);
          const int page = __ldg(table + pg);
          have = mla_page_ok(page, p.num_pages);
          row = ((uint32_t)page * p.h_kv + w.h) * (uint32_t)p.page_size + ((uint32_t)t - pg * (uint32_t)p.page_size);
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, have);
        if (lane < 2) masks[2 * i + lane] = mask >> (16 * lane) & 0xffffu;
        if (have) {
          const uint4 *k = reinterpret_cast<const uint4*>(p.k_codes + (uint64_t)row * (DIM / 2)),
                      *v = reinterpret_cast<const uint4*>(p.v_codes + (uint64_t)row * (DIM / 2));
          for (int c = 0; c < DIM / 32; ++c) {
            reinterpret_cast<uint4*>(stage_ptr + to * (DIM / 2))[c] = __ldg(k + c);
            reinterpret_cast<uint4*>(stage_ptr + Cfg::kCodes + to * (DIM / 2))[c] = __ldg(v + c);
          }
          for (int c = 0; c < NG; ++c) {
            reinterpret_cast<uint32_t*>(stage_ptr + 2 * Cfg::kCodes)[to * NG + c] = __ldg(reinterpret_cast<const uint32_t*>(p.k_scale) + (uint64_t)row * NG + c);
            reinterpret_cast<uint32_t*>(stage_ptr + 2 * Cfg::kCodes + Cfg::kScales)[to * NG + c] =
                __ldg(reinterpret_cast<const uint32_t*>(p.v_scale) + (uint64_t)row * NG + c);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
  };
  // the unit `by` behind `it`
  auto ahead_of = [&](UnitIter w, int by) {
    w.u += by;
    while (w.u >= w.units) {
      const int over = w.u - w.units;
      w.u = w.units - 1;
      advance(w, p);
      w.u = over;
    }
    return w;
  };
  volatile int* abort_flag = &sh.abort;
  const int count = left;
  if (warp < Cfg::kAhead && warp < count) issue(ahead_of(it, warp), warp);       // the ring is fresh: no wait

  // ---- segments -------------------------------------------------------------------------------------------------------
  int stage = 0;
  uint32_t phase = 0;                                  // of the full barriers
  int next_stage = Cfg::kAhead, next_phase = 1;        // where the unit kAhead further on goes, and the parity its empty barrier has by then
  bool ok = true;
  while (left > 0) {
    const int rows = min(Cfg::kRows, p.rows - it.qt * Cfg::kRows);
    // the columns of Q as the B operand: permuted like the columns of the widened keys, times a power of two that brings the
    // largest (finite) one to 2^14, odd nibbles' columns divided by 16
    uint32_t qf[NT][DIM / 16][2];
    float qsum[NG][NT][2], to_score;                  // scale * sum of q over the group for queries 2j, 2j + 1; scale of the dot products
    int limit[NT][2];                                 // keys that queries 2j and 2j + 1 see
    {
      uint4 raw[NT][DIM / 32];
      float big = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g, row = it.qt * Cfg::kRows + r;
        const bool ok = r < rows;
        const int qi = ok ? row / p.per : 0;
        const T* src = reinterpret_cast<const T*>(p.q) + it.b * p.q_sb + qi * p.q_ss + ((int64_t)it.h * p.per + (ok ? row - qi * p.per : 0)) * DIM;
#pragma unroll
        for (int x = 0; x < DIM / 32; ++x) {
          const int col = x / (GROUP / 32) * GROUP + (j * (GROUP / 32) + x % (GROUP / 32)) * 8;
          raw[nt][x] = ok ? __ldg(reinterpret_cast<const uint4*>(src + col)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) limit[nt][e] = it.len - p.s_q + (it.qt * Cfg::kRows + nt * 8 + 2 * j + e) / p.per + 1;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < DIM / 32; ++x) {
          const uint32_t w[4] = {raw[nt][x].x, raw[nt][x].y, raw[nt][x].z, raw[nt][x].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = widen_scale<T>(w[e]);
            big = fmaxf(big, fabsf(f.x) < INFINITY ? fabsf(f.x) : 0.f);
            big = fmaxf(big, fabsf(f.y) < INFINITY ? fabsf(f.y) : 0.f);
          }
        }
      big = warp_max(big);
      const int up = min(14 - ((int)(__float_as_uint(big) >> 23) - 127), 120);         // big < 2^128, so up >= -113
      const float mul = __uint_as_float((uint32_t)(127 + up) << 23), mul16 = mul * 0.0625f;
      to_score = p.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23) * 0x1p24f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < DIM / 32; ++x) {
          const float2 e01 = widen_scale<T>(raw[nt][x].x), e23 = widen_scale<T>(raw[nt][x].y), e45 = widen_scale<T>(raw[nt][x].z),
                       e67 = widen_scale<T>(raw[nt][x].w);
          qf[nt][2 * x][0] = pack_f16(e01.x * mul, e45.x * mul);
          qf[nt][2 * x][1] = pack_f16(e01.y * mul16, e45.y * mul16);
          qf[nt][2 * x + 1][0] = pack_f16(e23.x * mul, e67.x * mul);
          qf[nt][2 * x + 1][1] = pack_f16(e23.y * mul16, e67.y * mul16);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {             // sums of q: an MMA with keys whose widened codes are 1 and 16
          const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u};
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < MG; ++ks) mma16816(d, ones, qf[nt][gg * MG + ks][0], qf[nt][gg * MG + ks][1]);
          qsum[gg][nt][0] = d[0] * (to_score * 0x1p-24f);
          qsum[gg][nt][1] = d[1] * (to_score * 0x1p-24f);
        }
    }
    const int all_see = it.len - p.s_q + 1;           // tokens before this one are seen by every query

    float acc[MT][NT][4], wsum[NG][NT][4], low[NG][NT][2], m[NT][2], l[NT][2];
    float f = 0.f, most = 0.f;                        // the weights are p * step * f, steps up to `most`; 0: none seen yet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = -FLT_MAX;                          // finite, so that a score of -inf weighs 0 and not NaN
        l[nt][e] = 0.f;
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) low[gg][nt][e] = wsum[gg][nt][e] = wsum[gg][nt][2 + e] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][nt][e] = 0.f;
    }

    const int first_u = it.u;                         // the first unit of this CTA's share of the segment
    while (true) {
      if (left > Cfg::kAhead && (count - left + Cfg::kAhead) % kWarps == warp) {          // this warp's turn
        ok = mbar_wait(bar_empty + 8 * next_stage, next_phase, abort_flag);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        issue(ahead_of(it, Cfg::kAhead), next_stage);
      }
      if (++next_stage == ST) { next_stage = 0; next_phase ^= 1; }
      ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      const uint8_t* at = smem + stage * Cfg::kStage + warp * 16 * (DIM / 2);
      const uint8_t* at_scale = smem + stage * Cfg::kStage + 2 * Cfg::kCodes + warp * 16 * (4 * NG);
      const int t0 = it.u * kUnit + warp * 16;
      uint32_t mask[1];
      lds_words(smem + stage * Cfg::kStage + Cfg::kMask + 4 * warp, mask);
      if (mask[0]) {                                  // uniform in the warp, like `full`
        const bool full = mask[0] == 0xffffu && t0 + 16 <= all_see;       // every query sees every token
        // ---- S^T = K Q^T, log2 domain -------------------------------------------------------------------------------------
        float sc[NT][4];
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          constexpr int W = GROUP / 32;
          uint32_t w0[W], w1[W];
          {
            const int b = gg * (GROUP / 2) + j * (GROUP / 8);
            lds_words(at + tok * (DIM / 2) + b, w0);
            lds_words(at + (tok + 8) * (DIM / 2) + b, w1);
          }
          float d[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[nt][e] = 0.f;
#pragma unroll
          for (int x = 0; x < W; ++x) {
            uint32_t u0[4], u1[4];
            widen4(w0[x], u0);
            widen4(w1[x], u1);
            const uint32_t a0[4] = {u0[0], u1[0], u0[1], u1[1]}, a1[4] = {u0[2], u1[2], u0[3], u1[3]};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816(d[nt], a0, qf[nt][gg * MG + 2 * x][0], qf[nt][gg * MG + 2 * x][1]);
              mma16816(d[nt], a1, qf[nt][gg * MG + 2 * x + 1][0], qf[nt][gg * MG + 2 * x + 1][1]);
            }
          }
          uint32_t s0[1], s1[1];
          lds_words(at_scale + (tok * NG + gg) * 4, s0);
          lds_words(at_scale + ((tok + 8) * NG + gg) * 4, s1);
          const float2 k0 = widen_scale<T>(s0[0]), k1 = widen_scale<T>(s1[0]);
          const float a0 = k0.x * to_score, a1 = k1.x * to_score;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float lo0 = k0.y * qsum[gg][nt][e], lo1 = k1.y * qsum[gg][nt][e];
              sc[nt][e] = fmaf(a0, d[nt][e], gg ? sc[nt][e] + lo0 : lo0);
              sc[nt][2 + e] = fmaf(a1, d[nt][2 + e], gg ? sc[nt][2 + e] + lo1 : lo1);
            }
        }
        // ---- the values' steps and minima; what is not seen --------------------------------------------------------------
        float2 v0[NG], v1[NG];
        float big = 0.f;
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          uint32_t s0[1], s1[1];
          lds_words(at_scale + Cfg::kScales + (tok * NG + gg) * 4, s0);
          lds_words(at_scale + Cfg::kScales + ((tok + 8) * NG + gg) * 4, s1);
          v0[gg] = widen_scale<T>(s0[0]);
          v1[gg] = widen_scale<T>(s1[0]);
        }
        uint32_t see = 0xffffffffu;                   // bit 4 nt + e: query 2j + (e & 1) sees token tok + 8 (e >> 1)
        if (!full) {
          const bool live0 = mask[0] >> tok & 1, live1 = mask[0] >> (tok + 8) & 1;
          see = 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool ok = (e < 2 ? live0 : live1) && t0 + tok + (e < 2 ? 0 : 8) < limit[nt][e & 1];
              sc[nt][e] = ok ? sc[nt][e] : -INFINITY;
              see |= (ok ? 1u : 0u) << (4 * nt + e);
            }
#pragma unroll
          for (int gg = 0; gg < NG; ++gg) {           // rows behind the last token hold anything
            v0[gg] = live0 ? v0[gg] : make_float2(0.f, 0.f);
            v1[gg] = live1 ? v1[gg] : make_float2(0.f, 0.f);
          }
        }
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          big = fmaxf(big, fmaxf(fabsf(v0[gg].x), fabsf(v1[gg].x)));
          v0[gg].y = fmaf(8.f, v0[gg].x, v0[gg].y);   // the middle of the range: the weights' rounding meets c - 8
          v1[gg].y = fmaf(8.f, v1[gg].x, v1[gg].y);
        }
        // ---- whether the running maximum or the factor f has to move -----------------------------------------------------
        // the maximum may lag by 2^8: p stays below 256, and sums are exact whatever the reference is
        float over = 0.f, rel[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            rel[nt][e] = sc[nt][e] - m[nt][e & 1];
            over = fmaxf(over, rel[nt][e]);
          }
        if (__any_sync(0xffffffffu, over > 8.f || big > most)) {
          float top[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(sc[nt][e], sc[nt][2 + e]);
#pragma unroll
          for (int o = 4; o < 32; o *= 2) {
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], o));
          }
          float ratio = 1.f;                          // what the factor f changes by
          if (big > most) {
            // f = 2^(4 - exponent): the largest step times f lies in [16, 32), and steps up to four times as large need no
            // change; exponents of f stay normal
            const int ex = max((int)(__float_as_uint(big) >> 23) - 127, -112);
            const float f_new = __uint_as_float((uint32_t)(127 + 4 - min(ex, 127)) << 23);
            ratio = f == 0.f ? 0.f : f_new / f;
            f = f_new;
            most = 64.f / f_new;                      // infinity at the upper end
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float m_new = fmaxf(m[nt][e], top[nt][e]), alpha = ex2_approx(m[nt][e] - m_new), both = alpha * ratio;
              m[nt][e] = m_new;
              l[nt][e] *= alpha;
#pragma unroll
              for (int gg = 0; gg < NG; ++gg) {
                low[gg][nt][e] *= alpha;
                wsum[gg][nt][e] *= both;
                wsum[gg][nt][2 + e] *= both;
              }
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                acc[t][nt][e] *= both;
                acc[t][nt][2 + e] *= both;
              }
              rel[nt][e] = sc[nt][e] - m_new;
              rel[nt][2 + e] = sc[nt][2 + e] - m_new;
            }
        }
        // ---- p and its sum ---------------------------------------------------------------------------------------------------
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] = ex2_approx(rel[nt][e]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) l[nt][e] += sc[nt][e] + sc[nt][2 + e];
        // ---- O^T += V^T P^T, group by group ----------------------------------------------------------------------------------
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          uint32_t pb[NT][2];
          const float f0 = v0[gg].x * f, f1 = v1[gg].x * f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4] = {sc[nt][0] * f0, sc[nt][1] * f0, sc[nt][2] * f1, sc[nt][3] * f1};
            if (full) {
#pragma unroll
              for (int e = 0; e < 2; ++e) low[gg][nt][e] = fmaf(sc[nt][e], v0[gg].y, fmaf(sc[nt][2 + e], v1[gg].y, low[gg][nt][e]));
            } else {                                  // a value that a query does not see may be NaN, which 0 does not cancel
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool ok = see >> (4 * nt + e) & 1;
                w[e] = ok ? w[e] : 0.f;
                low[gg][nt][e & 1] += ok ? sc[nt][e] * (e < 2 ? v0[gg].y : v1[gg].y) : 0.f;
              }
            }
            pb[nt][0] = movmatrix_trans(pack_f16(w[0], w[1]));
            pb[nt][1] = movmatrix_trans(pack_f16(w[2], w[3]));
            const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
            mma16816(wsum[gg][nt], ones, pb[nt][0], pb[nt][1]);
          }
          // words of the tokens of operand rows 2j, 2j + 1, 2j + 8, 2j + 9
          constexpr int W = GROUP >= 64 ? GROUP / 64 : 1;
          uint32_t w[4][W];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = ((2 * j + (i & 1)) ^ (j & 1)) + 8 * (i >> 1);
            lds_words(at + Cfg::kCodes + row * (DIM / 2) + gg * (GROUP / 2) + (GROUP >= 64 ? g * (GROUP / 16) : (g >> 1) * 4), w[i]);
          }
#pragma unroll
          for (int x = 0; x < W; ++x)
#pragma unroll
            for (int half = 0; half < (GROUP >= 64 ? 2 : 1); ++half) {
              const uint32_t sel = GROUP >= 64 ? (half ? 0x7632u : 0x5410u) : ((g & 1) ? 0x7632u : 0x5410u);
              uint32_t ua[4], ub[4];
              widen4(__byte_perm(w[0][x], w[1][x], sel), ua);
              widen4(__byte_perm(w[2][x], w[3][x], sel), ub);
              const int t = gg * MG + (GROUP >= 64 ? 4 * x + 2 * half : 0);
              const uint32_t a0[4] = {ua[0], ua[1], ub[0], ub[1]}, a1[4] = {ua[2], ua[3], ub[2], ub[3]};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816(acc[t][nt], a0, pb[nt][0], pb[nt][1]);
                mma16816(acc[t + 1][nt], a1, pb[nt][0], pb[nt][1]);
              }
            }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_empty + 8 * stage);
      if (++stage == ST) { stage = 0; phase ^= 1; }
      --left;
      if (left == 0 || it.u + 1 == it.units) break;
      ++it.u;
    }
    if (!ok) {
      // a wait gave up: let the copies in flight land before the shared memory is released, report, leave
      for (int i = 0; i < 64; ++i) __nanosleep(20000);
      if (lane == 0 && p.status) *p.status = *abort_flag;
      return;
    }

    // ---- join the warps ---------------------------------------------------------------------------------------------------
#pragma unroll
    for (int o = 4; o < 32; o *= 2)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], o);
#pragma unroll
          for (int gg = 0; gg < NG; ++gg) low[gg][nt][e] += __shfl_xor_sync(0xffffffffu, low[gg][nt][e], o);
        }
    if (g == 0)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) join_m[warp * Cfg::kRows + nt * 8 + 2 * j + e] = m[nt][e];
    __syncthreads();
    const float inv_f = f == 0.f ? 0.f : 1.f / f;
    float part[NT][2];                                // this warp's weight in the joint result
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + 2 * j + e;
        float top = join_m[r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, join_m[w * Cfg::kRows + r]);
        part[nt][e] = ex2_approx(m[nt][e] - top);
        if (g == 0) join_l[warp * Cfg::kRows + r] = l[nt][e] * part[nt][e];
      }
    const int64_t seg_first = sh.seq_base + ((int64_t)it.h * p.q_tiles + it.qt) * it.units, seg_end = seg_first + it.units;
    const bool whole = seg_first >= sh.start && seg_end <= sh.end;
    auto store_out = [&](int r, int d, float4 v) {
      const int row = it.qt * Cfg::kRows + r, qi = row / p.per;
      T* dst = reinterpret_cast<T*>(p.out) + (((int64_t)it.b * p.s_q + qi) * p.h_q + (int64_t)it.h * p.per + (row - qi * p.per)) * DIM + d;
      union { uint2 raw; T e[4]; } o;
      o.e[0] = from_f32<T>(v.x); o.e[1] = from_f32<T>(v.y); o.e[2] = from_f32<T>(v.z); o.e[3] = from_f32<T>(v.w);
      *reinterpret_cast<uint2*>(dst) = o.raw;
    };
    constexpr int kSlot = Cfg::kRows * (DIM + 2);      // floats of one partial result: rows, maxima, sums
    float* slot = p.partial + ((int64_t)blockIdx.x * 2 + (seg_first + first_u > sh.start ? 1 : 0)) * kSlot;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += Cfg::kJoinRows) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * j + e - r0;
          if (r >= 0 && r < Cfg::kJoinRows) {
            float* dst = join + (warp * Cfg::kJoinRows + r) * Cfg::kPitch;
#pragma unroll
            for (int gg = 0; gg < NG; ++gg)
#pragma unroll
              for (int t = 0; t < MG; ++t) {
                const int d = gg * GROUP + g * (GROUP / 8) + 2 * t;
                const float a0 = fmaf(acc[gg * MG + t][nt][e], 0x1p24f, -8.f * wsum[gg][nt][e]);
                const float a1 = fmaf(acc[gg * MG + t][nt][2 + e], 0x1p20f, -8.f * wsum[gg][nt][e]);
                *reinterpret_cast<float2*>(dst + d) =
                    make_float2(fmaf(a0, inv_f, low[gg][nt][e]) * part[nt][e], fmaf(a1, inv_f, low[gg][nt][e]) * part[nt][e]);
              }
          }
        }
      __syncthreads();
      // the segment's rows: to the output, or to the partial sums
      for (int i = threadIdx.x; i < min(rows - r0, Cfg::kJoinRows) * (DIM / 4); i += 32 * kWarps) {
        const int rj = i / (DIM / 4), r = r0 + rj, d = i % (DIM / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f, top = join_m[r];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 a = *reinterpret_cast<const float4*>(join + (w * Cfg::kJoinRows + rj) * Cfg::kPitch + d);
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
          sum += join_l[w * Cfg::kRows + r];
          top = fmaxf(top, join_m[w * Cfg::kRows + r]);
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          store_out(r, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        } else {
          __stcg(reinterpret_cast<float4*>(slot + r * DIM + d), v);
          if (d == 0) {
            __stcg(slot + Cfg::kRows * DIM + r, top);
            __stcg(slot + Cfg::kRows * (DIM + 1) + r, sum);
          }
        }
      }
      __syncthreads();                                 // the join buffer is free again
    }
    if (!whole) {
      // CTAs c0 .. c1 share the segment; the last to arrive adds up their partial sums
      const int64_t total = sh.total, ctas = sh.ctas;
      const int c0 = (int)(((seg_first + 1) * ctas - 1) / total), c1 = (int)((seg_end * ctas - 1) / total);
      int* counter = p.counters + c0;                // only one shared segment begins in a CTA's range: its last
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) sh.last = atomicAdd(counter, 1) == c1 - c0;
      __syncthreads();
      if (sh.last) {
        __threadfence();
        if (threadIdx.x == 0) *counter = 0;            // ready for the next call
        // the segment is the last of CTA c0 (slot 1 unless it is its first as well) and the first of all others (slot 0)
        const float* slots = p.partial + (int64_t)c0 * 2 * kSlot;
        const int in_c0 = seg_first > (int64_t)c0 * total / ctas ? kSlot : 0, count = c1 - c0 + 1;
        auto slot_of = [&](int c) { return slots + (c == 0 ? in_c0 : (int64_t)c * 2 * kSlot); };
        constexpr int kRowThreads = DIM / 4 < 32 ? DIM / 4 : 32;         // neighbouring lanes with one row
        const int items = rows * (DIM / 4), teams = 32 * kWarps > items ? 32 * kWarps / items : 1;
        float4* team_v = reinterpret_cast<float4*>(join);               // [teams][items], at most 256
        float* team_l = join + 4 * 32 * kWarps;
        for (int i0 = 0; i0 < items; i0 += 32 * kWarps) {                // one round, unless a tile has more than 256 items
          const int team = items < 32 * kWarps ? threadIdx.x / items : 0, i = items < 32 * kWarps ? threadIdx.x % items : i0 + threadIdx.x;
          const bool on = team < teams && i < items;
          const int r = on ? i / (DIM / 4) : 0, d = i % (DIM / 4) * 4;
          float top = -FLT_MAX;
          for (int c = lane % kRowThreads; c < count; c += kRowThreads) top = fmaxf(top, __ldcg(slot_of(c) + Cfg::kRows * DIM + r));
#pragma unroll
          for (int o = 1; o < kRowThreads; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          float sum = 0.f;
          if (on) {
#pragma unroll 8
            for (int c = team; c < count; c += teams) {
              const float* s = slot_of(c);
              const float mc = __ldcg(s + Cfg::kRows * DIM + r), lc = __ldcg(s + Cfg::kRows * (DIM + 1) + r);
              const float4 x = __ldcg(reinterpret_cast<const float4*>(s + r * DIM + d));
              const float a = ex2_approx(mc - top);
              v.x = fmaf(x.x, a, v.x); v.y = fmaf(x.y, a, v.y); v.z = fmaf(x.z, a, v.z); v.w = fmaf(x.w, a, v.w);
              sum = fmaf(lc, a, sum);
            }
          }
          if (teams > 1) {                             // in a fixed order
            if (on) {
              team_v[team * items + i] = v;
              team_l[team * items + i] = sum;
            }
            __syncthreads();
            if (on && team == 0)
              for (int t = 1; t < teams; ++t) {
                const float4 x = team_v[t * items + i];
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
                sum += team_l[t * items + i];
              }
          }
          if (on && team == 0) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            store_out(r, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
          }
        }
      }
    }
    __syncthreads();                                   // sh, the maxima and the join buffer are free again
    if (left > 0) {
      const int b = it.b;
      const int64_t next = (int64_t)it.units * p.h_kv * p.q_tiles;
      advance(it, p);
      if (it.b != b) {                                 // read again only behind the barriers of the next segment's end
        if (threadIdx.x == 0) sh.seq_base += next;
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
// Query rows of a kv head go in tiles of 8; from 9 rows on of 16 (dim 64, 128), where a widened key serves twice as many.
static int q_tile_rows(int64_t rows, int64_t dim) { return rows > 8 && dim <= 128 ? 16 : 8; }
static int ctas_per_sm(int64_t dim, int tile_rows) { return dim * (tile_rows / 8) <= 128 ? 2 : 1; }

struct I4Plan {
  int tile_rows, q_tiles, grid;
  int64_t bytes;
};
static I4Plan i4_plan(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  I4Plan r;
  const int64_t rows = s_q * (h_q / h_kv);
  r.tile_rows = q_tile_rows(rows, dim);
  r.q_tiles = (int)((rows + r.tile_rows - 1) / r.tile_rows);
  r.grid = sm_count() * ctas_per_sm(dim, r.tile_rows);
  r.bytes = TL_B200_ATTN_INT4_ZERO_BYTES + (int64_t)r.grid * 2 * r.tile_rows * (dim + 2) * 4;
  return r;
}

template <typename T, int DIM, int GROUP, int NT>
static int launch_i4(const AttnInt4Params& p, int grid, cudaStream_t s) {
  auto kernel = attn_int4_kernel<T, DIM, GROUP, NT>;
  constexpr int smem = I4Cfg<DIM, GROUP, NT>::kSmem;
  TL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<grid, 32 * kWarps, smem, s>>>(p);
  TL_LAUNCH_CHECK("attn_int4_kernel");
  return TL_B200_OK;
}
template <typename T, int DIM, int GROUP>
static int launch_i4_tile(const AttnInt4Params& p, const I4Plan& plan, cudaStream_t s) {
  if constexpr (DIM <= 128)
    if (plan.tile_rows == 16) return launch_i4<T, DIM, GROUP, 2>(p, plan.grid, s);
  return launch_i4<T, DIM, GROUP, 1>(p, plan.grid, s);
}
template <typename T>
static int launch_i4_dim(const AttnInt4Params& p, const I4Plan& plan, int64_t dim, int64_t group, cudaStream_t s) {
  if (dim == 64) return group == 32 ? launch_i4_tile<T, 64, 32>(p, plan, s) : launch_i4_tile<T, 64, 64>(p, plan, s);
  if (dim == 128) {
    if (group == 32) return launch_i4_tile<T, 128, 32>(p, plan, s);
    return group == 64 ? launch_i4_tile<T, 128, 64>(p, plan, s) : launch_i4_tile<T, 128, 128>(p, plan, s);
  }
  if (group == 32) return launch_i4_tile<T, 256, 32>(p, plan, s);
  return group == 64 ? launch_i4_tile<T, 256, 64>(p, plan, s) : launch_i4_tile<T, 256, 128>(p, plan, s);
}

static bool i4_sizes_ok(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  return batch >= 0 && s_q >= 0 && h_q >= 1 && h_kv >= 1 && h_q % h_kv == 0 && batch < (1 << 24) && s_q < (1 << 24) && h_q <= 65536 &&
         batch * s_q * h_q < (1ll << 31) && (dim == 64 || dim == 128 || dim == 256);
}

}  // namespace tl

using namespace tl;

extern "C" int64_t tl_b200_attn_decode_paged_int4_workspace_bytes(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  return i4_sizes_ok(batch, s_q, h_q, h_kv, dim) ? i4_plan(batch, s_q, h_q, h_kv, dim).bytes : 0;
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
  TL_REQUIRE(num_pages < (1ll << 31) && page_size < (1ll << 31) && num_pages * page_size < (1ll << 31) && max_pages_per_seq < (1ll << 31) &&
                 num_pages * page_size * h_kv < (1ll << 32),            // 2^32 rows of 32 bytes and their values are over 256 GB
             "attn_decode_paged_int4: cache too large");
  if (batch == 0 || s_q == 0) return TL_B200_OK;
  const bool keys = num_pages > 0 && max_pages_per_seq > 0;
  TL_REQUIRE(q && cache_seqlens && out && (!keys || (k_cache && k_scale && v_cache && v_scale && block_table)),
             "attn_decode_paged_int4: null tensor pointer");
  TL_REQUIRE(aligned16(q) && aligned16(out) && aligned16(k_cache) && aligned16(v_cache) && aligned16(k_scale) && aligned16(v_scale) &&
                 q_stride_batch % 8 == 0 && q_stride_token % 8 == 0, "attn_decode_paged_int4: tensors and rows of q must be 16-byte aligned");
  const I4Plan plan = i4_plan(batch, s_q, h_q, h_kv, dim);
  TL_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= plan.bytes,
             "attn_decode_paged_int4: needs a 16-byte aligned workspace of %lld bytes, got %lld", (long long)plan.bytes,
             (long long)workspace_bytes);
  AttnInt4Params p;
  p.q = q; p.q_sb = q_stride_batch; p.q_ss = q_stride_token;
  p.k_codes = (const uint8_t*)k_cache; p.v_codes = (const uint8_t*)v_cache;
  p.k_scale = (const uint8_t*)k_scale; p.v_scale = (const uint8_t*)v_scale;
  p.table = block_table; p.lens = cache_seqlens; p.out = out;
  p.batch = (int)batch; p.s_q = (int)s_q; p.h_q = (int)h_q; p.h_kv = (int)h_kv; p.per = (int)(h_q / h_kv);
  p.page_size = (int)page_size; p.max_pages = (int)max_pages_per_seq; p.num_pages = (int)num_pages;
  const int64_t cap = max_pages_per_seq * page_size;           // a sequence may name a page more than once
  p.len_cap = num_pages == 0 ? 0 : (int)(cap < 0x7fff0000ll ? cap : 0x7fff0000ll);
  p.rows = (int)(s_q * (h_q / h_kv)); p.q_tiles = plan.q_tiles;
  p.page_div = FastDiv((uint32_t)page_size);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.status = device_status_word();
  TL_REQUIRE((batch * h_kv * plan.q_tiles) / plan.grid + 1 < (1ll << 31) / (p.len_cap / kUnit + 1),
             "attn_decode_paged_int4: more units of work than a CTA counts");
  TL_REQUIRE(plan.grid * 4 <= TL_B200_ATTN_INT4_ZERO_BYTES, "attn_decode_paged_int4: more SMs than counters");
  p.counters = (int*)workspace;
  p.partial = (float*)((uint8_t*)workspace + TL_B200_ATTN_INT4_ZERO_BYTES);
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == TL_BF16 ? launch_i4_dim<__nv_bfloat16>(p, plan, dim, group, s) : launch_i4_dim<__half>(p, plan, dim, group, s);
}
