// Attention over a paged cache held in 4 bits (TL_U4G, see kv_cache.cu): grouped query heads, s_q query tokens a sequence.
//
//   out[b,i,h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q[b,i,h] . k_t),  t < len_b - s_q + i + 1,
//   k_t = s c + lo per group of columns (likewise v_t); a row that sees no key is zero.
//
// What bounds it.  A key of one kv head is dim/2 + 4 groups bytes, twice with its value (136 bytes at dim 128 and one
// group), against 4 dim flop for each of the few query heads that share it: HBM, if the codes can be widened fast enough.
// At the measured copy rate an SM receives 43 codes a clock, so every instruction spent on eight codes counts.  As it stands
// neither memory nor any one unit is full: a warp's steps depend on one another, and the registers and the rings leave four
// warps a scheduler to hide that (figures below).
//
// Layout.  The MMAs are the warp-level m16n8k16 ones: at most 8 or 16 query rows share a key, so a 128-row tensor-memory
// tile would be 90% padding, and codes have to pass through registers to be widened anyway.  Keys (and columns of V) are
// the 16 rows, queries the 8 columns:  S^T = K Q^T  and  O^T = V^T P^T, both in fp16.  Widening is one AND per pair of
// codes: a nibble in the low bits of an fp16 number is the subnormal c 2^-24 (the next nibble 16 c 2^-24), which the tensor
// core multiplies exactly; the powers of two are taken back outside the loop.
//   * K: a lane holds whole 32-bit words of a key; word & 0x000f000f are columns 0 and 4 of the word, one register of the A
//     operand.  The columns of Q are permuted (and those of odd nibbles divided by 16) when they are loaded, once a
//     sequence; a power of two per query brings Q into fp16's range, and what falls below it is 2^-35 of its largest.
//   * V: a register of the A operand is one column of two neighbouring tokens: one byte permute joins half words of the two.
//   * Steps and minima never touch the codes:  q . k = s (q . c) + lo sum(q) per group, and the value's step multiplies p
//     (rounded to fp16: half a step, 2^-11 of each weight, or 2^-29 of the query's largest where that is more, for every query
//     has a power of two per group of columns that keeps its p s in range, whatever other queries and groups meet), its
//     minimum adds p lo in fp32.  The codes of V become c - 8 (an addition per pair of codes) and 8 s goes to the
//     minimum: the weights' rounding then meets numbers about zero, and so do the sums, which with codes of one sign are
//     hundreds of times the output of a long sequence and carry the tensor core's truncation into it (error against 64 bits,
//     60 sequences of 100000 tokens, fp16: 2.6e-4 of the output, of which 2.1e-4 is its own rounding; 1.1e-3 without, 4.7e-4
//     with 8 times the sum of the weights taken off at the end; bf16 1.68e-3, all of it rounding, and up to 2.3e-3 without).
//     It cost 5% when it was made: 64 sequences of 2048 to 12288 tokens 108.6 and 114 us.
// Every group of columns has its own MMAs, so a group's step can multiply the score or the weight.
//
// Work.  Sequences are cut into units of 128 tokens; the list of all (sequence, kv head, query tile, unit) is dealt out in
// equal contiguous ranges to teams of four warps, whatever the lengths.  Each warp takes two tiles of 16 tokens of a unit, through a
// ring of cp.async stages of its own that runs ahead across the ends of sequences: no warp waits for another inside a
// segment (a ring of bulk copies shared by the warps was 40% slower: whoever refills a stage waits for the slowest).  Two
// tiles at a time halve what control costs a token and give a warp two chains of MMAs to interleave; the teams of an SM
// cover each other's ends.  The warps' results are joined in shared memory,
// a few rows at a time, at the end of a segment; a segment that teams share leaves fp32 partial sums, and the team that arrives
// last adds them up in their fixed order, so the result does not depend on who that is.
//
// Measured (bf16, dim 128, one group, 32 query and 8 kv heads, at a copy rate of 6.55 TB/s): 64 sequences of 2048 to 12288
// tokens 115.5 us, 4.3 TB/s of cache; one of 131077 tokens (groups of 64) 52 us, 2.9 TB/s; one of 777 tokens 9.0 us.  Counters of
// 32 sequences of 8192: 662 instructions a round of 32 tokens, all told; while an SM is busy its issue slots are 61% taken and the
// integer pipe 53%, memory 45%; in 39% of the cycles none of a scheduler's four warps can issue.  A warp's 6.6 cycles an
// instruction are 1.3 waiting for its turn, 1.3 for results of fixed latency, 1.0 for a busy pipe, 0.5 for shared memory and
// shuffles, hardly any for global loads.  Launch, first loads and joins take 15% of that call.  Each integer or IEEE
// division between segments is felt: without those by run-time sizes 200 sequences of 40 to 300 tokens took 32.4 us instead
// of 36.4 us, in an earlier form.
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
  FastDiv page_div, per_div, tile_div, team_div;     // t / page_size, row / per, tile / q_tiles, unit / teams
  float scale_log2;
  int* counters;                       // three per team, zero between calls
  float* partial;                      // [2 * teams][kRows * (dim + 2)]
};

constexpr int kWarps = 4, kHalf = 16 * kWarps, kUnit = 2 * kHalf;      // a warp's two tiles of a unit lie kHalf tokens apart

// Teams per SM, by the registers a thread needs: 128 (four teams), 168 with four groups' steps and sums (32 x 4096 tokens, in an
// earlier form: 59 us, 73 us with four teams that spill), 255 with twice the accumulators (24 sequences of 4 tokens, dim 64, likewise: 39 us, 42 us).
__host__ __device__ constexpr int i4_teams(int dim, int groups, int nt) {
  return nt == 2 || dim == 256 ? 2 : dim == 128 && groups == 4 ? 3 : 4;
}

template <int DIM, int GROUP, int NT> struct I4Cfg {
  static constexpr int kGroups = DIM / GROUP;
  static constexpr int kCodes = 16 * DIM / 2;                           // a stage, 16 tokens: codes of K and of V, their scales,
  static constexpr int kScales = 16 * 4 * kGroups;                      // a word of 16 live bits
  static constexpr int kMask = 2 * kCodes + 2 * kScales;
  static constexpr int kStage = kMask + 16;
  static constexpr int kRows = 8 * NT;
  static constexpr int kJoinRows = (DIM == 64 ? 4 : 2) * NT;            // rows joined at a time
  static constexpr int kJoin = kWarps * (kJoinRows * DIM + 2 * kRows) * 4;      // partial rows, maxima and sums of the warps
  static constexpr int kTeams = i4_teams(DIM, kGroups, NT);             // of four warps, on an SM
  static constexpr int kFit = (228 * 1024 / kTeams - 1024 - kJoin - 256) / (kWarps * kStage);
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kSmem = (kWarps * kStages * kStage + kJoin + 128 + 127) / 128 * 128;             // of a team
  static_assert(kStages >= 4, "two stages are worked on while two are on their way");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // onto zeros
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// The same of c - 8 (exact: multiples of 2^-24 below 2^-16).
__device__ __forceinline__ void centre4(uint32_t (&u)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t minus8 = i & 1 ? 0x80808080u : 0x80088008u;
    const __half2 c = __hadd2(*reinterpret_cast<const __half2*>(&u[i]), *reinterpret_cast<const __half2*>(&minus8));
    u[i] = *reinterpret_cast<const uint32_t*>(&c);
  }
}
template <typename T> __device__ __forceinline__ float2 widen_scale(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float inverse_pow2(float f) {        // 1 / f for a power of two of 2^-126 to 2^126
  return __uint_as_float((254u << 23) - __float_as_uint(f));
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
// Lengths, page table and queries are read by ordinary loads: the kernel before may write them while this one is resident.
__device__ __forceinline__ int length_of(const AttnInt4Params& p, int b) { return min(max(p.lens[b], 0), p.len_cap); }
__device__ __forceinline__ int units_of(int len) { return len > 0 ? (len + kUnit - 1) / kUnit : 1; }
__device__ __forceinline__ bool advance(UnitIter& it, const AttnInt4Params& p) {      // true: a new segment begins
  if (++it.u < it.units) return false;
  it.u = 0;
  if (++it.qt == p.q_tiles) {
    it.qt = 0;
    if (++it.h == p.h_kv) {
      it.h = 0;
      if (++it.b < p.batch) {
        it.len = length_of(p, it.b);
        it.units = units_of(it.len);
      }
    }
  }
  return true;
}

template <typename T, int DIM, int GROUP, int NT, int TEAMS>
__global__ void __launch_bounds__(32 * kWarps * TEAMS, I4Cfg<DIM, GROUP, NT>::kTeams / TEAMS)
attn_int4_kernel(const AttnInt4Params p) {
  using Cfg = I4Cfg<DIM, GROUP, NT>;
  constexpr int NG = Cfg::kGroups, ST = Cfg::kStages, MT = DIM / 16, MG = GROUP / 16;
  extern __shared__ __align__(128) uint8_t all_smem[];
  // With TEAMS > 1, warp w of the block runs on scheduler w % 4 and is the (w / 4)-th oldest there; a team has one warp on each scheduler,
  // each of another age.
  const int scheduler = threadIdx.x / 32 % 4, team = TEAMS == 1 ? 0 : (threadIdx.x / 128 + scheduler) % TEAMS;
  const int warp = scheduler, lane = threadIdx.x % 32, g = lane / 4, j = lane % 4, tid = warp * 32 + lane;
  const int me = team * gridDim.x + blockIdx.x, all_teams = gridDim.x * TEAMS;      // few of them go to SMs of their own
  uint8_t* const smem = all_smem + team * Cfg::kSmem;
  auto team_sync = [&]() {
    if constexpr (TEAMS == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(32 * kWarps) : "memory");
  };
  dependency_wait();
  dependency_release();
  uint8_t* tail = smem + kWarps * ST * Cfg::kStage;
  float* join = reinterpret_cast<float*>(tail);                  // [warps][join rows][pitch]
  float* join_m = join + kWarps * Cfg::kJoinRows * DIM;  // [warps][rows]
  float* join_l = join_m + kWarps * Cfg::kRows;
  // what only the ends of segments need stays in shared memory
  struct Shared {
    int64_t sums[kWarps];
    int64_t total, quot, start, end, seq_base;         // seq_base: first unit of sequence it.b
    int ctas, first_b, last;
    uint32_t rest;
  };
  Shared& sh = *reinterpret_cast<Shared*>(join_l + kWarps * Cfg::kRows);
  uint8_t* const ring = smem + warp * ST * Cfg::kStage;                    // this warp's stages

  // ---- this team's range of the list --------------------------------------------------------------------------------
  UnitIter it;
  int left;                                            // units of this team still to do
  {
    const int64_t per_unit = (int64_t)p.h_kv * p.q_tiles;
    const int chunk = (p.batch + 32 * kWarps - 1) / (32 * kWarps);
    const int b0 = min((int)tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(length_of(p, b));
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh.sums[warp] = incl;
    team_sync();
    int64_t before = 0, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.sums[w];
      total += sh.sums[w];
    }
    total *= per_unit;
    const int64_t ctas = total < all_teams ? total : all_teams;          // every one of them has a unit
    if (me >= ctas) return;                                              // the whole team
    // team i begins at floor(i * total / ctas)
    const int64_t quot = total <= all_teams ? 1 : total >> 31 ? total / all_teams : (int64_t)p.team_div((uint32_t)total);
    const uint32_t rest = (uint32_t)(total - quot * ctas);               // times a team's number: below 2^31
    const int64_t start = me * quot + p.team_div(me * rest);
    const int64_t end = (me + 1) * quot + p.team_div((me + 1) * rest);
    int64_t base = before + incl - mine;
    if (base * per_unit <= start && start < (base + mine) * per_unit) {  // exactly one thread
      int b = b0, units = 0;
      for (; b < b1; ++b) {
        units = units_of(length_of(p, b));
        if (start < (base + units) * per_unit) break;
        base += units;
      }
      sh.first_b = b;
      sh.seq_base = base * per_unit;
      sh.total = total;
      sh.ctas = (int)ctas;
      sh.quot = quot;
      sh.rest = rest;
      sh.start = start;
      sh.end = end;
    }
    team_sync();
    left = (int)(end - start);                                           // the host checks that it fits
    it.b = sh.first_b;
    it.len = length_of(p, it.b);
    it.units = units_of(it.len);
    const int64_t off = start - sh.seq_base;
    const int seg = off >> 32 ? (int)(off / it.units) : (int)((uint32_t)off / (uint32_t)it.units);
    it.u = (int)(off - (int64_t)seg * it.units);
    it.h = (int)p.tile_div((uint32_t)seg);
    it.qt = seg - it.h * p.q_tiles;
  }

  // ---- loads: the 16 tokens of a warp in a unit go into a stage; one commit group each, empty ones included -------------
  constexpr int kLines = 256 / DIM, kChunks = DIM / 32;                     // rows per 128 bytes of shared memory, 16-byte chunks per row
  const bool tile_in_page = p.page_size % 16 == 0;
  const uint8_t* k_lane = p.k_codes + lane * 16;                            // the codes of 16 tokens of a page are contiguous
  const uint8_t* v_lane = p.v_codes + lane * 16;
  const uint8_t* s_lane = (lane < 16 ? p.k_scale : p.v_scale) + lane % 16 * (4 * NG);
  // Rows of a stage are swizzled by 16-byte chunks, K in the tokens' order and V with tokens 2j, 2j + 1, 2j + 8, 2j + 9 in
  // rows j, j + 4, j + 8, j + 12, so that neither operand's reads conflict.
  auto k_place = [&](int row, int c) { return row * (DIM / 2) + (c ^ (row / kLines * (GROUP / 32)) % kChunks) * 16; };
  auto v_place = [&](int rho, int c) { return Cfg::kCodes + rho * (DIM / 2) + (c ^ (rho / kLines * 2) % kChunks) * 16; };
  uint32_t k_dst[DIM / 64], v_dst[DIM / 64];          // where chunk lane + 32 i of a tile goes
#pragma unroll
  for (int i = 0; i < DIM / 64; ++i) {
    const int row = (lane + 32 * i) / kChunks, c = lane % kChunks;
    k_dst[i] = k_place(row, c);
    v_dst[i] = v_place((row >> 1 & 3) | (row & 1) << 2 | (row & 8), c);
    asm("" : "+r"(k_dst[i]), "+r"(v_dst[i]));         // kept, not computed again for every tile
  }
  auto copy_scales = [&](uint32_t at, const uint8_t* from) {
    const uint32_t to = at + 2 * Cfg::kCodes + lane * (4 * NG);
    if constexpr (NG <= 2) cp_async_small<4 * NG>(to, from);
    else
#pragma unroll
      for (int i = 0; i < NG / 4; ++i) cp_async16(to + 16 * i, from + 16 * i);
  };
  // a tile that lies in one page and is all there: `row0` is its first row of the cache
  auto load_whole = [&](int stage, uint32_t row0) {
    uint8_t* const stage_ptr = ring + stage * Cfg::kStage;
    const uint32_t at = smem_u32(stage_ptr);
    const uint8_t *k = k_lane + (uint64_t)row0 * (DIM / 2), *v = v_lane + (uint64_t)row0 * (DIM / 2);
#pragma unroll
    for (int i = 0; i < DIM / 64; ++i) cp_async16(at + k_dst[i], k + 512 * i);
    copy_scales(at, s_lane + (uint64_t)row0 * (4 * NG));
#pragma unroll
    for (int i = 0; i < DIM / 64; ++i) cp_async16(at + v_dst[i], v + 512 * i);
    *reinterpret_cast<uint32_t*>(stage_ptr + Cfg::kMask) = 0xffffu;          // every lane, the same word
  };
  auto row_of = [&](int page, int h, int t0) {        // rows of the cache are fewer than 2^32
    const uint32_t off = (uint32_t)t0 - p.page_div((uint32_t)t0) * (uint32_t)p.page_size;
    return ((uint32_t)page * p.h_kv + h) * (uint32_t)p.page_size + off;
  };
  // tile `half` of the unit; page: of its first token, where tiles lie in one
  auto load = [&](const UnitIter& w, int half, int stage, int page) {
    uint8_t* const stage_ptr = ring + stage * Cfg::kStage;
    const uint32_t at = smem_u32(stage_ptr);
    const int t0 = w.u * kUnit + half * kHalf + warp * 16;
    uint32_t mask = 0;
    if (tile_in_page) {
      const int live = mla_page_ok(page, p.num_pages) ? min(w.len - t0, 16) : 0;
      const uint32_t row0 = row_of(page, w.h, t0);
      if (live == 16) {
        load_whole(stage, row0);
        return;
      }
      mask = (1u << live) - 1u;
      const uint8_t *k = k_lane + (uint64_t)row0 * (DIM / 2), *v = v_lane + (uint64_t)row0 * (DIM / 2);
#pragma unroll
      for (int i = 0; i < DIM / 64; ++i)
        if ((lane + 32 * i) / kChunks < live) {
          cp_async16(at + k_dst[i], k + 512 * i);
          cp_async16(at + v_dst[i], v + 512 * i);
        }
      if (lane % 16 < live) copy_scales(at, s_lane + (uint64_t)row0 * (4 * NG));
    } else {                                          // pages end inside the tile: a table entry per token
      const int my = t0 + lane % 16;
      bool live = my < w.len;
      uint32_t row = 0;
      if (live) {
        const int id = p.table[(int64_t)w.b * p.max_pages + p.page_div((uint32_t)my)];
        live = mla_page_ok(id, p.num_pages);
        row = row_of(id, w.h, my);
      }
      mask = __ballot_sync(0xffffffffu, live) & 0xffffu;
#pragma unroll
      for (int i = 0; i < DIM / 64; ++i) {
        const int r = (lane + 32 * i) / kChunks;      // k_lane points at this lane's chunk of row lane / kChunks
        const uint32_t from = __shfl_sync(0xffffffffu, row, r);
        const int64_t o = (int64_t)from * (DIM / 2) - (lane / kChunks) * (DIM / 2);
        if (mask >> r & 1) {
          cp_async16(at + k_dst[i], k_lane + o);
          cp_async16(at + v_dst[i], v_lane + o);
        }
      }
      if (live) copy_scales(at, s_lane + (int64_t)row * (4 * NG) - lane % 16 * (4 * NG));
    }
    *reinterpret_cast<uint32_t*>(stage_ptr + Cfg::kMask) = mask;             // every lane, the same word
  };
  auto page_at = [&](const UnitIter& w, int half) {
    const int t0 = w.u * kUnit + half * kHalf + warp * 16;
    return tile_in_page && t0 < w.len ? p.table[(int64_t)w.b * p.max_pages + p.page_div((uint32_t)t0)] : -1;
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
  // ---- segments -------------------------------------------------------------------------------------------------------
  int stage = 0;
  bool first = true;
  while (left > 0) {
    const int rows = min(Cfg::kRows, p.rows - it.qt * Cfg::kRows);
    // the columns of Q as the B operand: permuted like the columns of the widened keys, times a power of two that brings the
    // query's largest (finite) one to 2^14, odd nibbles' columns divided by 16
    uint32_t qf[NT][DIM / 16][2];
    float qsum[NG][NT][2], to_score[NT][2];           // for queries 2j, 2j + 1: scale * sum of q over the group; scale of the dot products
    int limit[NT][2];                                 // keys that queries 2j and 2j + 1 see
    bool huge = false;                                // a query above 2^74: its to_score could pass fp32, so scores are 2^-24 of theirs
    {
      uint4 raw[NT][DIM / 32];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g, row = it.qt * Cfg::kRows + r;
        const bool ok = r < rows;
        const int qi = ok ? (int)p.per_div((uint32_t)row) : 0;
        const T* src = reinterpret_cast<const T*>(p.q) + it.b * p.q_sb + qi * p.q_ss + ((int64_t)it.h * p.per + (ok ? row - qi * p.per : 0)) * DIM;
#pragma unroll
        for (int x = 0; x < DIM / 32; ++x) {
          const int col = x / (GROUP / 32) * GROUP + (j * (GROUP / 32) + x % (GROUP / 32)) * 8;
          raw[nt][x] = ok ? *reinterpret_cast<const uint4*>(src + col) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) limit[nt][e] = it.len - p.s_q + (int)p.per_div((uint32_t)(it.qt * Cfg::kRows + nt * 8 + 2 * j + e)) + 1;
      }
      if (first) {                                    // fill the ring: lane k looks up the page of tile k, all at once
        first = false;
        const int page = lane < min(ST, 2 * left) ? page_at(ahead_of(it, lane / 2), lane % 2) : -1;
#pragma unroll 1
        for (int k = 0; k < ST; ++k) {
          const int pg = __shfl_sync(0xffffffffu, page, k);
          if (k < 2 * left) load(ahead_of(it, k / 2), k % 2, k, pg);
          cp_async_commit();
        }
      }
      if (lane < 2 * NT && it.units - it.u < left) {  // the queries of the next segment here: on their way to L2 by then
        const UnitIter n = ahead_of(it, it.units - it.u);
        const int row = n.qt * Cfg::kRows + (warp * 2 * NT + lane), qi = (int)p.per_div((uint32_t)row);
        if (row < p.rows) {
          const T* at = reinterpret_cast<const T*>(p.q) + n.b * p.q_sb + qi * p.q_ss + ((int64_t)n.h * p.per + (row - qi * p.per)) * DIM;
#pragma unroll
          for (int i = 0; i < DIM; i += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + i));
        }
      }
      int up[NT];                                     // query g of the tile (and g + 8) goes times 2^up
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float big = 0.f;
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
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        up[nt] = min(14 - ((int)(__float_as_uint(big) >> 23) - 127), 120);             // big < 2^128, so up >= -113
        if constexpr (std::is_same<T, __nv_bfloat16>::value) huge |= up[nt] < -60;
      }
      huge = __any_sync(0xffffffffu, huge);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float mul = __uint_as_float((uint32_t)(127 + up[nt]) << 23), mul16 = mul * 0.0625f;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          to_score[nt][e] = p.scale_log2 * (__uint_as_float((uint32_t)(127 - __shfl_sync(0xffffffffu, up[nt], (2 * j + e) * 4)) << 23) *
                                            (huge ? 1.f : 0x1p24f));
#pragma unroll
        for (int x = 0; x < DIM / 32; ++x) {
          const float2 e01 = widen_scale<T>(raw[nt][x].x), e23 = widen_scale<T>(raw[nt][x].y), e45 = widen_scale<T>(raw[nt][x].z),
                       e67 = widen_scale<T>(raw[nt][x].w);
          qf[nt][2 * x][0] = pack_f16(e01.x * mul, e45.x * mul);
          qf[nt][2 * x][1] = pack_f16(e01.y * mul16, e45.y * mul16);
          qf[nt][2 * x + 1][0] = pack_f16(e23.x * mul, e67.x * mul);
          qf[nt][2 * x + 1][1] = pack_f16(e23.y * mul16, e67.y * mul16);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {             // sums of q: an MMA with keys whose widened codes are 1 and 16
          const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u};
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < MG; ++ks) mma16816(d, ones, qf[nt][gg * MG + ks][0], qf[nt][gg * MG + ks][1]);
          qsum[gg][nt][0] = d[0] * (to_score[nt][0] * 0x1p-24f);
          qsum[gg][nt][1] = d[1] * (to_score[nt][1] * 0x1p-24f);
        }
    }
    const int all_see = it.len - p.s_q + 1;           // tokens before this one are seen by every query

    float acc[MT][NT][4], low[NG][NT][2], m[NT][2], l[NT][2];
    float2 f[NG][NT];                                 // the weights of queries 2j, 2j + 1 are p * step * f, a power of two
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int gg = 0; gg < NG; ++gg) f[gg][nt] = make_float2(0x1p120f, 0x1p120f);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = -FLT_MAX;                          // finite, so that a score of -inf weighs 0 and not NaN
        l[nt][e] = 0.f;
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) low[gg][nt][e] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][nt][e] = 0.f;
    }

    const int first_u = it.u;                         // the first unit of this team's share of the segment
    while (true) {
      const int stage1 = stage + 1 == ST ? 0 : stage + 1;
      // Usually the two tiles ST further on belong to the segment, whole and in a page each: their pages are looked up here,
      // for the loads at the end of this round.
      const int next0 = it.u * kUnit + ST * kHalf + warp * 16, next1 = next0 + kHalf;
      const bool easy = 2 * left > ST + 1 && tile_in_page && next1 + 16 <= it.len;
      int page0 = 0, page1 = 0;
      if (easy) {
        const int* table = p.table + (int64_t)it.b * p.max_pages;
        page0 = table[p.page_div((uint32_t)next0)];
        page1 = table[p.page_div((uint32_t)next1)];
      }
      cp_async_wait<ST - 2>();
      __syncwarp();                                           // every lane's copies have landed
      const uint8_t* base[2] = {ring + stage * Cfg::kStage, ring + stage1 * Cfg::kStage};
      const int t0 = it.u * kUnit + warp * 16;                // tokens t0 .. t0 + 15 and t0 + kHalf ..
      uint32_t mask[2];
      mask[0] = *reinterpret_cast<const uint32_t*>(base[0] + Cfg::kMask);
      mask[1] = *reinterpret_cast<const uint32_t*>(base[1] + Cfg::kMask);
      if (mask[0] | mask[1]) {                        // uniform in the warp, like `full`
        const bool full = (mask[0] & mask[1]) == 0xffffu && t0 + kHalf + 16 <= all_see;       // every query sees every token
        // ---- S^T = K Q^T, log2 domain -------------------------------------------------------------------------------------
        float sc[2][NT][4];
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          constexpr int W = GROUP / 32;
          uint32_t w0[2][W], w1[2][W];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int in_row = gg * (GROUP / 2) + j * (GROUP / 8);
            lds_words(base[t] + k_place(g, in_row / 16) + in_row % 16, w0[t]);
            lds_words(base[t] + k_place(g + 8, in_row / 16) + in_row % 16, w1[t]);
          }
          float d[2][NT][4];
#pragma unroll
          for (int x = 0; x < W; ++x)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                const uint32_t r0 = half ? w0[t][x] >> 8 : w0[t][x], r1 = half ? w1[t][x] >> 8 : w1[t][x];
                const uint32_t a[4] = {r0 & 0x000f000fu, r1 & 0x000f000fu, r0 & 0x00f000f0u, r1 & 0x00f000f0u};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const uint32_t(&q)[2] = qf[nt][gg * MG + 2 * x + half];
                  if (x == 0 && half == 0) mma16816_zero(d[t][nt], a, q[0], q[1]);
                  else mma16816(d[t][nt], a, q[0], q[1]);
                }
              }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint8_t* at = base[t] + 2 * Cfg::kCodes + (g * NG + gg) * 4;
            const float2 k0 = widen_scale<T>(*reinterpret_cast<const uint32_t*>(at)), k1 = widen_scale<T>(*reinterpret_cast<const uint32_t*>(at + 32 * NG));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float lo0 = k0.y * qsum[gg][nt][e], lo1 = k1.y * qsum[gg][nt][e];
                sc[t][nt][e] = fmaf(k0.x, d[t][nt][e] * to_score[nt][e], gg ? sc[t][nt][e] + lo0 : lo0);
                sc[t][nt][2 + e] = fmaf(k1.x, d[t][nt][2 + e] * to_score[nt][e], gg ? sc[t][nt][2 + e] + lo1 : lo1);
              }
          }
        }
        if (std::is_same<T, __nv_bfloat16>::value && huge) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[t][nt][e] *= 0x1p24f;
        }
        // ---- the values' steps and minima; what is not seen --------------------------------------------------------------
        float2 v0[2][NG], v1[2][NG];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int gg = 0; gg < NG; ++gg) {
            const uint8_t* at = base[t] + 2 * Cfg::kCodes + Cfg::kScales + (g * NG + gg) * 4;
            v0[t][gg] = widen_scale<T>(*reinterpret_cast<const uint32_t*>(at));
            v1[t][gg] = widen_scale<T>(*reinterpret_cast<const uint32_t*>(at + 32 * NG));
          }
        uint32_t see = 0xffffffffu;                   // bit 8 t + 4 nt + e: query 2j + (e & 1) sees token g + 8 (e >> 1) of tile t
        if (!full) {
          see = 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bool live0 = mask[t] >> g & 1, live1 = mask[t] >> (g + 8) & 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool ok2 = (e < 2 ? live0 : live1) && t0 + t * kHalf + g + (e < 2 ? 0 : 8) < limit[nt][e & 1];
                sc[t][nt][e] = ok2 ? sc[t][nt][e] : -INFINITY;
                see |= (ok2 ? 1u : 0u) << (4 * NT * t + 4 * nt + e);
              }
#pragma unroll
            for (int gg = 0; gg < NG; ++gg) {         // rows behind the last token hold anything; NaN counts for nothing below
              v0[t][gg].x = live0 ? v0[t][gg].x : __uint_as_float(0x7fffffffu);
              v1[t][gg].x = live1 ? v1[t][gg].x : __uint_as_float(0x7fffffffu);
            }
          }
        }
        // ---- whether the running maximum or a factor f has to move -------------------------------------------------------
        // the maximum may lag by 2^4: p stays below 16, and sums are exact whatever the reference is
        float over = 0.f, rel[2][NT][4];
        bool coarse = false;                          // a step times f above 2^11: its weight could pass fp16's range
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          const float big = fmaxf(fmaxf(fabsf(v0[0][gg].x), fabsf(v1[0][gg].x)), fmaxf(fabsf(v0[1][gg].x), fabsf(v1[1][gg].x)));
          float finest = fmaxf(f[gg][0].x, f[gg][0].y);
          if constexpr (NT == 2) finest = fmaxf(finest, fmaxf(f[gg][1].x, f[gg][1].y));
          coarse |= big * finest > 0x1p11f;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            v0[t][gg].y = fmaf(8.f, v0[t][gg].x, v0[t][gg].y);       // the middle of the range
            v1[t][gg].y = fmaf(8.f, v1[t][gg].x, v1[t][gg].y);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              rel[t][nt][e] = sc[t][nt][e] - m[nt][e & 1];
              over = fmaxf(over, rel[t][nt][e]);
            }
        if (__any_sync(0xffffffffu, over > 4.f || coarse)) {
          float top[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][2 + e]), fmaxf(sc[1][nt][e], sc[1][nt][2 + e]));
#pragma unroll
          for (int o = 4; o < 32; o *= 2)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], o));
          float alpha[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float m_new = fmaxf(m[nt][e], top[nt][e]);
              alpha[nt][e] = ex2_approx(m[nt][e] - m_new);
              m[nt][e] = m_new;
              l[nt][e] *= alpha[nt][e];
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                rel[t][nt][e] = sc[t][nt][e] - m_new;
                rel[t][nt][2 + e] = sc[t][nt][2 + e] - m_new;
              }
            }
          // A query's factor f for a group of columns: 2^4 over its largest weight so far (to a power of two), so that what
          // falls below fp16's range is 2^-29 of that, and a step may be 2^6 times it before this place is come to again.  By
          // the weights and not the steps: a step may be huge, or infinite, and hardly weigh, or be hidden from this query.
          // Of the weights before, f has what is needed: they lost alpha since.  Where nothing has weighed f stays at 2^120.
          // (Straight on: with votes and branches around what is seldom needed, 16 x 4096 tokens at dim 256 and groups of 32 took
          // 80.4 us where this takes 78.4, and 24 sequences of 4 tokens 29.6 us where this takes 28.9.)
          float p_now[2][NT][4];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) p_now[t][nt][e] = ex2_approx(rel[t][nt][e]);
#pragma unroll
          for (int gg = 0; gg < NG; ++gg)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t heavy[2];                      // bits of the largest weight of the round (NaN, 0 times infinity, aside)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                heavy[e] = __float_as_uint(fmaxf(fmaxf(fmaxf(0.f, p_now[0][nt][e] * fabsf(v0[0][gg].x)), fmaxf(p_now[0][nt][2 + e] * fabsf(v1[0][gg].x),
                                                       p_now[1][nt][e] * fabsf(v0[1][gg].x))), p_now[1][nt][2 + e] * fabsf(v1[1][gg].x)));
              uint32_t both16 = __byte_perm(heavy[0], heavy[1], 0x7632);       // the upper halves of the two are ordered like them
#pragma unroll
              for (int o = 4; o < 32; o *= 2) both16 = __vmaxu2(both16, __shfl_xor_sync(0xffffffffu, both16, o));
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& fe = e ? f[gg][nt].y : f[gg][nt].x;
                const float old = fe, a = alpha[nt][e];
                const int by_new = 254 + 4 - (int)(both16 >> (e ? 23 : 7) & 0xff);
                const int by_old = (int)(__float_as_uint(old) >> 23) + 127 - (int)(__float_as_uint(a) >> 23);
                fe = __uint_as_float((uint32_t)min(min(by_new, by_old), 247) << 23);
                const float both = a > 0.f ? a * (inverse_pow2(old) * fe) : 0.f;         // 2 at most
                low[gg][nt][e] *= a;
#pragma unroll
                for (int t = 0; t < MG; ++t) {
                  acc[gg * MG + t][nt][e] *= both;
                  acc[gg * MG + t][nt][2 + e] *= both;
                }
              }
            }
        }
        // ---- p and its sum ---------------------------------------------------------------------------------------------------
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][nt][e] = ex2_approx(rel[t][nt][e]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) l[nt][e] += (sc[0][nt][e] + sc[0][nt][2 + e]) + (sc[1][nt][e] + sc[1][nt][2 + e]);
        // ---- O^T += V^T P^T, group by group ----------------------------------------------------------------------------------
#pragma unroll
        for (int gg = 0; gg < NG; ++gg) {
          uint32_t pb[2][NT][2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float2 s0 = make_float2(v0[t][gg].x, v0[t][gg].x), s1 = make_float2(v1[t][gg].x, v1[t][gg].x);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const float(&pr)[4] = sc[t][nt];
              // p f first: f may be as small as a step is large
              float2 w01 = sm100::mul2(sm100::mul2(make_float2(pr[0], pr[1]), f[gg][nt]), s0);
              float2 w23 = sm100::mul2(sm100::mul2(make_float2(pr[2], pr[3]), f[gg][nt]), s1);
              if (full) {
#pragma unroll
                for (int e = 0; e < 2; ++e) low[gg][nt][e] = fmaf(pr[e], v0[t][gg].y, fmaf(pr[2 + e], v1[t][gg].y, low[gg][nt][e]));
              } else {                                // a value that a query does not see may be NaN, which 0 does not cancel
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const bool ok2 = see >> (4 * NT * t + 4 * nt + e) & 1;
                  float& w = e == 0 ? w01.x : e == 1 ? w01.y : e == 2 ? w23.x : w23.y;
                  w = ok2 ? w : 0.f;
                  low[gg][nt][e & 1] += ok2 ? pr[e] * (e < 2 ? v0[t][gg].y : v1[t][gg].y) : 0.f;
                }
              }
              pb[t][nt][0] = movmatrix_trans(pack_f16(w01.x, w01.y));
              pb[t][nt][1] = movmatrix_trans(pack_f16(w23.x, w23.y));
            }
          }
          // words of the tokens of operand rows 2j, 2j + 1, 2j + 8, 2j + 9
          constexpr int W = GROUP >= 64 ? GROUP / 64 : 1;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            uint32_t w[4][W];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int in_row = gg * (GROUP / 2) + (GROUP >= 64 ? g * (GROUP / 16) : (g >> 1) * 4);
              lds_words(base[t] + v_place(j + 4 * i, in_row / 16) + in_row % 16, w[i]);
            }
#pragma unroll
            for (int x = 0; x < W; ++x)
#pragma unroll
              for (int half = 0; half < (GROUP >= 64 ? 2 : 1); ++half) {
                const uint32_t sel = GROUP >= 64 ? (half ? 0x7632u : 0x5410u) : ((g & 1) ? 0x7632u : 0x5410u);
                uint32_t ua[4], ub[4];
                widen4(__byte_perm(w[0][x], w[1][x], sel), ua);
                widen4(__byte_perm(w[2][x], w[3][x], sel), ub);
                centre4(ua);
                centre4(ub);
                const int mt = gg * MG + (GROUP >= 64 ? 4 * x + 2 * half : 0);
                const uint32_t a0[4] = {ua[0], ua[1], ub[0], ub[1]}, a1[4] = {ua[2], ua[3], ub[2], ub[3]};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  mma16816(acc[mt][nt], a0, pb[t][nt][0], pb[t][nt][1]);
                  mma16816(acc[mt + 1][nt], a1, pb[t][nt][0], pb[t][nt][1]);
                }
              }
          }
        }
      }
      __syncwarp();                                   // every lane has left the stages: the tiles ST further on go there
      if (easy && mla_page_ok(page0, p.num_pages) && mla_page_ok(page1, p.num_pages)) {
        load_whole(stage, row_of(page0, it.h, next0));
        cp_async_commit();
        load_whole(stage1, row_of(page1, it.h, next1));
        cp_async_commit();
      } else {
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          if (ST + k < 2 * left) {
            const UnitIter w = ahead_of(it, (ST + k) / 2);
            load(w, (ST + k) % 2, k ? stage1 : stage, page_at(w, (ST + k) % 2));
          }
          cp_async_commit();
        }
      }
      stage = stage1 + 1 == ST ? 0 : stage1 + 1;
      --left;
      ++it.u;
      if (left == 0 || it.u == it.units) break;
    }
    --it.u;                                           // the segment's last unit here

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
    team_sync();
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
      const int row = it.qt * Cfg::kRows + r, qi = (int)p.per_div((uint32_t)row);
      T* dst = reinterpret_cast<T*>(p.out) + (((int64_t)it.b * p.s_q + qi) * p.h_q + (int64_t)it.h * p.per + (row - qi * p.per)) * DIM + d;
      union { uint2 raw; T e[4]; } o;
      o.e[0] = from_f32<T>(v.x); o.e[1] = from_f32<T>(v.y); o.e[2] = from_f32<T>(v.z); o.e[3] = from_f32<T>(v.w);
      *reinterpret_cast<uint2*>(dst) = o.raw;
    };
    constexpr int kSlot = Cfg::kRows * (DIM + 2);      // floats of one partial result: rows, maxima, sums
    float* slot = p.partial + ((int64_t)me * 2 + (seg_first + first_u > sh.start ? 1 : 0)) * kSlot;
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += Cfg::kJoinRows) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * j + e - r0;
          if (r >= 0 && r < Cfg::kJoinRows) {
            float* dst = join + (warp * Cfg::kJoinRows + r) * DIM;
#pragma unroll
            for (int gg = 0; gg < NG; ++gg) {
              const float inv_f = inverse_pow2(e ? f[gg][nt].y : f[gg][nt].x);
#pragma unroll
              for (int t = 0; t < MG; ++t) {
                const int d = gg * GROUP + g * (GROUP / 8) + 2 * t;
                const float a0 = acc[gg * MG + t][nt][e] * 0x1p24f, a1 = acc[gg * MG + t][nt][2 + e] * 0x1p20f;
                *reinterpret_cast<float2*>(dst + d) =
                    make_float2(fmaf(a0, inv_f, low[gg][nt][e]) * part[nt][e], fmaf(a1, inv_f, low[gg][nt][e]) * part[nt][e]);
              }
            }
          }
        }
      team_sync();
      // the segment's rows: to the output, or to the partial sums
      for (int i = tid; i < min(rows - r0, Cfg::kJoinRows) * (DIM / 4); i += 32 * kWarps) {
        const int rj = i / (DIM / 4), r = r0 + rj, d = i % (DIM / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f, top = join_m[r];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 a = *reinterpret_cast<const float4*>(join + (w * Cfg::kJoinRows + rj) * DIM + d);
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
          sum += join_l[w * Cfg::kRows + r];
          top = fmaxf(top, join_m[w * Cfg::kRows + r]);
        }
        if (whole) {
          const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);      // two steps of fp32; the sum is below 2^40
          store_out(r, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        } else {
          __stcg(reinterpret_cast<float4*>(slot + r * DIM + d), v);
          if (d == 0) {
            __stcg(slot + Cfg::kRows * DIM + r, top);
            __stcg(slot + Cfg::kRows * (DIM + 1) + r, sum);
          }
        }
      }
      team_sync();                                 // the join buffer is free again
    }
    if (!whole) {
      // Teams c0 .. c1 share the segment.  They are taken in groups of twelve neighbours: the last of a group to arrive adds
      // its partial results up into the slot of the group's first team, the last group to be done adds up the groups'.  (One
      // team adding up 74 takes 12 us.)
      const int64_t total = sh.total, ctas = sh.ctas;
      auto team_of = [&](int64_t unit) {               // the last team that begins at or before a unit
        const int64_t a = (unit + 1) * ctas - 1;
        return (a | total) >> 32 ? (int)(a / total) : (int)((uint32_t)a / (uint32_t)total);
      };
      const int c0 = seg_first >= sh.start ? me : team_of(seg_first), c1 = seg_end <= sh.end ? me : team_of(seg_end - 1);
      // the segment is the last of team c0 (slot 1 unless it is its first as well) and the first of all others (slot 0)
      const int in_c0 = seg_first > c0 * sh.quot + p.team_div(c0 * sh.rest) ? 1 : 0;
      auto slot_of = [&](int c) { return p.partial + ((int64_t)c * 2 + (c == c0 ? in_c0 : 0)) * kSlot; };
      constexpr int kGroup = 12;
      const int lead = c0 + (me - c0) / kGroup * kGroup, tail = min(c1, lead + kGroup - 1);
      const int groups = (c1 - c0) / kGroup + 1;
      // Three counters a team.  Only one shared segment begins in a team's range (its last), and a group of another segment
      // that begins with this team goes by the counter of those that only pass through.
      int* const group_counter = p.counters + 3 * lead + (lead == c0 ? 1 : 0);
      int* const seg_counter = p.counters + 3 * c0 + 2;
      auto arrive = [&](int* counter, int others) {    // behind a barrier, so it speaks for every thread's stores
        if (tid == 0) {
          int seen;                                    // releases this team's stores, acquires those of the teams before
          asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
          sh.last = seen == others;
          if (sh.last) *counter = 0;                   // ready for the next call
        }
        team_sync();
        return sh.last;
      };
      // Adds up `many` partial results in their order; `emit(r, d, sums, sum, top)` takes four columns of a row.
      auto add_up = [&](int many, auto slot_at, auto emit) {
        // Four at a time, all on their way at once, in the last batch too; most segments are shared by two or three (16 at a
        // time: 1 x 777 tokens 12.3 us where this takes 10.8, and the registers make the loop above spill)
        constexpr int kBatch = 4;
        const int items = rows * (DIM / 4), rounds = (items + 32 * kWarps - 1) / (32 * kWarps);
        for (int k = 0; k < rounds; ++k) {
          const int i = k * 32 * kWarps + tid;
          const bool on = i < items;
          const int r = on ? i / (DIM / 4) : 0, d = i % (DIM / 4) * 4;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          float sum = 0.f, top = -FLT_MAX;
          for (int c = 0; c < many; c += kBatch) {
            float4 x[kBatch];
            float mc[kBatch], lc[kBatch];
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
              const float* s = slot_at(min(c + q, many - 1));
              mc[q] = __ldcg(s + Cfg::kRows * DIM + r);
              lc[q] = __ldcg(s + Cfg::kRows * (DIM + 1) + r);
              x[q] = __ldcg(reinterpret_cast<const float4*>(s + r * DIM + d));
            }
            float higher = top;
#pragma unroll
            for (int q = 0; q < kBatch; ++q) higher = fmaxf(higher, mc[q]);
            const float keep = ex2_approx(top - higher);
            top = higher;
            v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
            sum *= keep;
#pragma unroll
            for (int q = 0; q < kBatch; ++q)
              if (c + q < many) {
                const float w = ex2_approx(mc[q] - top);
                v.x = fmaf(x[q].x, w, v.x); v.y = fmaf(x[q].y, w, v.y); v.z = fmaf(x[q].z, w, v.z); v.w = fmaf(x[q].w, w, v.w);
                sum = fmaf(lc[q], w, sum);
              }
          }
          if (on) emit(r, d, v, sum, top);
        }
      };
      auto to_out = [&](int r, int d, float4 v, float sum, float) {
        const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);      // two steps of fp32; the sum is below 2^40
        store_out(r, d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
      };
      if (arrive(group_counter, tail - lead)) {
        auto member = [&](int i) { return slot_of(lead + i); };
        if (groups == 1) {
          add_up(tail - lead + 1, member, to_out);
        } else {
          float* const into = slot_of(lead);
          // a thread reads all it needs of a row's columns before it writes them; the maxima and sums, which the threads of a
          // row share, are written behind a barrier
          add_up(tail - lead + 1, member, [&](int r, int d, float4 v, float sum, float top) {
            __stcg(reinterpret_cast<float4*>(into + r * DIM + d), v);
            if (d == 0) {
              join_l[r] = sum;                         // free since the rows were joined
              join_m[r] = top;
            }
          });
          team_sync();
          if (tid < rows) {
            __stcg(into + Cfg::kRows * DIM + tid, join_m[tid]);
            __stcg(into + Cfg::kRows * (DIM + 1) + tid, join_l[tid]);
          }
          team_sync();
          if (arrive(seg_counter, groups - 1))
            add_up(groups, [&](int i) { return slot_of(c0 + i * kGroup); }, to_out);
        }
      }
    }
    team_sync();                                   // sh, the maxima and the join buffer are free again
    if (left > 0) {
      const int b = it.b;
      const int64_t next = (int64_t)it.units * p.h_kv * p.q_tiles;
      advance(it, p);
      if (it.b != b) {                                 // read again only behind the barriers of the next segment's end
        if (tid == 0) sh.seq_base += next;
      }
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
// Query rows of a kv head go in tiles of 8; from 9 rows on of 16 (dim 64, 128), where a widened key serves twice as many.
static int q_tile_rows(int64_t rows, int64_t dim) { return rows > 8 && dim <= 128 ? 16 : 8; }

struct I4Plan {
  int tile_rows, q_tiles, grid;
  int64_t bytes;
};
static I4Plan i4_plan(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim, int64_t group) {
  I4Plan r;
  const int64_t rows = s_q * (h_q / h_kv);
  r.tile_rows = q_tile_rows(rows, dim);
  r.q_tiles = (int)((rows + r.tile_rows - 1) / r.tile_rows);
  r.grid = sm_count() * i4_teams((int)dim, (int)(dim / group), r.tile_rows / 8);
  r.bytes = TL_B200_ATTN_INT4_ZERO_BYTES + (int64_t)r.grid * 2 * r.tile_rows * (dim + 2) * 4;
  return r;
}

template <typename T, int DIM, int GROUP, int NT>
static int launch_i4(const AttnInt4Params& p, int grid, cudaStream_t s) {
  // Four small teams to an SM are one CTA: the schedulers favour the oldest warps, and as CTAs of their own the teams end at 80,
  // 92, 105 and 118 us (64 sequences of 2048 to 12288 tokens: 112.7 us; 107.8 us as one CTA, whose teams have a warp of every
  // age; 32 x 4096 tokens 44.8 and 44.0 us, one sequence of 131077 49.2 and 49.7 us; all before V's codes were taken about zero, like
  // what follows).  Two and three teams an SM:
  // 47.6 us as CTAs and 49.5 us as one (16 x 4096 tokens, dim 256), 60.5 and 63.4 us (32 x 4096, 16 rows).
  using Cfg = I4Cfg<DIM, GROUP, NT>;
  constexpr int teams = Cfg::kTeams == 4 ? 4 : 1, smem = teams * Cfg::kSmem;
  auto kernel = attn_int4_kernel<T, DIM, GROUP, NT, teams>;
  TL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  TL_CUDA(launch_overlapped(kernel, dim3(grid / teams), dim3(32 * kWarps * teams), smem, s, p));
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
         batch * s_q < (1ll << 31) && batch * s_q * h_q < (1ll << 31) && (dim == 64 || dim == 128 || dim == 256);
}

}  // namespace tl

using namespace tl;

extern "C" int64_t tl_b200_attn_decode_paged_int4_workspace_bytes(int64_t batch, int64_t s_q, int64_t h_q, int64_t h_kv, int64_t dim) {
  return i4_sizes_ok(batch, s_q, h_q, h_kv, dim) ? i4_plan(batch, s_q, h_q, h_kv, dim, dim).bytes : 0;
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
  TL_REQUIRE(batch < (1 << 24) && s_q < (1 << 24) && h_q <= 65536 && batch * s_q < (1ll << 31) && batch * s_q * h_q < (1ll << 31),
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
  const I4Plan plan = i4_plan(batch, s_q, h_q, h_kv, dim, group);
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
  p.per_div = FastDiv((uint32_t)p.per);
  p.tile_div = FastDiv((uint32_t)p.q_tiles);
  p.team_div = FastDiv((uint32_t)plan.grid);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  TL_REQUIRE((batch * h_kv * plan.q_tiles) / plan.grid + 1 < (1ll << 31) / (p.len_cap / kUnit + 1),
             "attn_decode_paged_int4: more units of work than a CTA counts");
  TL_REQUIRE(plan.grid * 12 <= TL_B200_ATTN_INT4_ZERO_BYTES, "attn_decode_paged_int4: more SMs than counters");
  p.counters = (int*)workspace;
  p.partial = (float*)((uint8_t*)workspace + TL_B200_ATTN_INT4_ZERO_BYTES);
  cudaStream_t s = (cudaStream_t)stream;
  return dtype == TL_BF16 ? launch_i4_dim<__nv_bfloat16>(p, plan, dim, group, s) : launch_i4_dim<__half>(p, plan, dim, group, s);
}
