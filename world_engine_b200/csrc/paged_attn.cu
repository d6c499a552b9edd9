// Attention of one new token per session over the paged KV cache (sm_100a).
//
//   x_gj = scale q_g . k_j,   p_gj = 2^(x_gj log2 e - m_g) / l_g,   o_g = sum_j p_gj v_j,   weight_j += sum_g p_gj
//
// Every K and V row is used for the few query heads that share its kv head, once: the work is reading the cache, and
// the kernel is built so that nothing but TMA touches it on the way to the tensor cores.  The products are turned
// around: 128 tokens are the M rows of S^T = K Q^T and the head dim is M of O^T = V^T P^T, the query heads are the N
// columns, so K (K-major) and V (MN-major) are read as they lie in shared memory.
//
// Work is cut by tokens, not by heads: the tokens of all (session, kv head, chunk of 16 query heads) units are laid end
// to end in granules of 16 or 32 tokens and cut into equal runs, one per CTA, whatever the sessions' lengths.  The SMs
// do not read equally fast (runs of one length end up to 12% apart), so of long runs a part is cut off into small
// pieces that the CTAs which finish first take one by one.  A run crosses units: each part is a segment, with its own
// softmax statistics.  A unit that lies in one run is finished there; of one that lies in several each leaves
// (m, l, O) in the workspace and paged_join_kernel puts them together, in the order of the tokens.
//
// One CTA per SM, 416 threads:
//   warps 0-7  softmax, two groups of 128 threads that take tiles in turn, each with statistics and an accumulator of
//              its own (put together at the end of a segment).  Thread t of a group owns token t of a tile (TMEM
//              lane t): its logits of the G heads are G columns.  The reference m_g is raised only when a logit
//              exceeds it by more than 8 (then O is rescaled in tensor memory), so a tile costs one vote among the
//              128 threads and no reduction.  P goes to shared memory as the sum of two 16-bit numbers in two
//              columns: the second column costs nothing (N is at least 16) and leaves the weights accurate to 2^-16
//              instead of 2^-8 (fp16: 2^-22 instead of 2^-11, down to 2^-43 of the largest weight: its exponents end
//              soon, so the reference lies 7 below the largest logit and the second number is held times 2^12; without
//              that, tokens of less than 2^-25 of the largest weight counted for nothing, however many they were).
//              A token's columns lie next to each other (P is an MN-major operand): one or two
//              16-byte stores per token.
//   warp 8     walks the run and publishes the segments, one ahead of the one being loaded: what to read, its first
//              pages, its Q rows; takes further runs
//   warp 11    loads the K tiles, warp 12 the V tiles (a ring each; issuing a copy takes a warp about 0.1 us, and a tile
//              is four to eight: one warp for both held up the tiles of head dim 64)
//   warp 9     issues S^T, warp 10 issues O^T (one thread each)
// Tensor memory (128 columns): four S buffers of 16, O of either group (high and low parts of up to 16 heads: 32).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace we {

constexpr int kPagedThreads = 416;
constexpr int kPagedWarps = kPagedThreads / 32;
constexpr int kTile = 128;                 // tokens per tile
constexpr int kSegs = 3;                   // segments in flight
constexpr int kBufs = 4;                   // S buffers
constexpr uint32_t kTmemColumns = 128;
constexpr uint32_t kColO = 64;             // + 32 per group
constexpr float kFloor = -3.4028234e38f;   // the reference before the first logit: no finite one lies below
constexpr int kMaxGroup = 16;              // query heads per unit
constexpr float kRaise = 8.0f;             // log2 units by which a logit may exceed the largest so far
// fp16: weights are held times 2^7 (2^15 at most, after a rise that is not followed), what is left of them by the first
// rounding (8 at most) times 2^12 (2^15 at most)
template <bool BF16>
constexpr float kAbove = BF16 ? 0.f : 7.f;
template <bool BF16>
constexpr float kLowScale = BF16 ? 1.f : 4096.f;
constexpr int kJoinThreads = 256;
constexpr int kJoinTokens = 4 * kJoinThreads;
constexpr int kWholeUnitTokens = 128;      // sessions this short are never split

struct PagedAttnParams {
  PagedView v;
  const uint16_t* q;
  uint16_t* out;
  int64_t qs[2], os[2];
  const int32_t* lens;
  float* weights;
  float* lse;
  // workspace
  int32_t* ws_prefix;        // [units + 1] granules before a unit; then the number of small runs handed out
  float2* ws_ml;             // [2 runs][GP] statistics of the segments of shared units
  float* ws_o;               // [2 runs][GP][DH]
  float* ws_lse;             // [units][GP] log2 of the softmax sum of units one CTA finished
  float* ws_x;               // [units][GP][cap] logits (log2 units)
  int64_t x_stride;          // max_pages * page
  int64_t unit_plane, unit_page, unit_head;   // tensor map coordinates of the V plane, of a page, of a head
  int32_t Hq, group, chunks; // query heads, per kv head, units per kv head
  int32_t units, grid;
  int32_t gran_shift;        // log2 of the tokens per granule
  int32_t whole;             // 1: every unit belongs to one CTA (no join)
  int32_t min_share;         // granules of a tile: what a CTA gets at least, and what beginning a unit counts
  int32_t dynamic;           // 1: long runs are shortened, and the rest handed out
  int32_t out_blocks;        // join: CTAs that join outputs (the others give the tokens their weights)
  int32_t out_by_warp;       // join: 1: a head per warp
  float scale_log2;
};

struct Segment {
  int32_t unit, tok0, ntok;  // ntok 0: the end of the run
  int32_t slot;              // workspace slot, or -1: the segment is the whole unit
};

template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else return __half_as_ushort(__float2half_rn(x));
}
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t x) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  else return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {           // a in the low half
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// Sums of N values over a warp, N shuffles and log2(32 / N) more in place of 5 N: at each step a lane keeps one half of
// its values and gives the other away.  Lane i ends with the sum number i / (32 / N) in v[0].
template <int N>
__device__ __forceinline__ void warp_sums(float (&v)[N], int lane) {
  int d = 16;
#pragma unroll
  for (int n = N / 2; n >= 1; n /= 2, d /= 2) {
    const bool up = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = up ? v[i + n] : v[i], give = up ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
    }
  }
#pragma unroll
  for (int k = 32 / N / 2; k >= 1; k /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], k);
}
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ bool bar_any(int id, int n, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t"
      ".reg .pred p, q;\n\t"
      "setp.ne.u32 q, %3, 0;\n\t"
      "bar.red.or.pred p, %1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(x ? 1u : 0u)
      : "memory");
  return r != 0;
}

template <int DH, int GP>
struct PagedCfg {
  static constexpr int kChunks = DH / 64;
  static constexpr int kRowGroup = kChunks * 1024;           // 8 tokens: [chunk][8 rows][128 bytes]
  static constexpr int kTileBytes = 16 * kRowGroup;
  static constexpr int kStages = DH == 128 ? 3 : 6;
  static constexpr int kNP = 2 * GP <= 16 ? 16 : 32;         // columns of O^T
  static constexpr int kQBytes = 16 * DH * 2;                // [chunk][16 rows][128 bytes]
  static constexpr int kPRow = 2 * kNP;                      // a token's columns: 32 or 64 bytes, swizzled as such
  static constexpr int kPBytes = kTile * kPRow;
  static_assert(GP * 128 * 4 <= kPBytes, "a group's O passes through its P buffer");
  static constexpr int kOffV = kStages * kTileBytes;
  static constexpr int kOffQ = 2 * kStages * kTileBytes;
  static constexpr int kOffP = kOffQ + kSegs * kQBytes;
  static constexpr int kOffAux = kOffP + 2 * kPBytes;
  static constexpr int kAux = 384 + 2 * 512 + 192 + 128 + kSegs * (16 + 128);
  static_assert((4 * kStages + 2 * kSegs + 2 * kBufs + 5) * 8 <= 384, "barriers");
  static constexpr int kSmem = kOffAux + kAux + 1024;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

// The heads of a unit.
struct UnitHeads {
  int s, h, hq0, n;          // session, kv head, first query head, query heads
};
// (integer divisions cost some fifty cycles each: one unit per kv head is the rule)
__device__ __forceinline__ int kv_head_of(const PagedAttnParams& p, int u) { return p.chunks == 1 ? u : u / p.chunks; }
__device__ __forceinline__ UnitHeads unit_heads(const PagedAttnParams& p, int u) {
  UnitHeads r;
  const int sh = kv_head_of(p, u), c = u - sh * p.chunks;
  r.s = static_cast<int>(static_cast<uint32_t>(sh) / static_cast<uint32_t>(p.v.Hkv));
  r.h = sh - r.s * p.v.Hkv;
  r.hq0 = r.h * p.group + c * kMaxGroup;
  r.n = min(p.group - c * kMaxGroup, kMaxGroup);
  return r;
}

// A unit that holds nothing, or sits out.
__device__ void write_empty(const PagedAttnParams& p, int u, int dh) {
  const UnitHeads w = unit_heads(p, u);
  for (int g = 0; g < w.n; ++g) {
    uint4* dst = reinterpret_cast<uint4*>(p.out + w.s * p.os[0] + (w.hq0 + g) * p.os[1]);
    for (int i = 0; i < dh / 8; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr) p.lse[static_cast<int64_t>(w.s) * p.Hq + w.hq0 + g] = -INFINITY;
  }
}

// How the granules are cut into runs: `grid` of `first` granules (run i belongs to CTA i), the rest in runs of `later`.
// Beginning a segment costs a CTA about what a tile does, so every unit that holds something counts one tile more
// (its head): without it a CTA that is given a dozen short sessions ends long after the others.
struct Cut {
  int first, later, border, runs;
  __device__ __forceinline__ Cut(const PagedAttnParams& p, int total) {
    const int share = max(static_cast<int>(static_cast<uint32_t>(total + p.grid - 1) / static_cast<uint32_t>(p.grid)), p.min_share);
    first = share;
    later = 1;
    border = total;
    runs = p.grid;
    // (a run of fewer than 32 tiles ends too soon for the difference to be worth the joins of small ones)
    if (p.dynamic && share >= 32 * p.min_share) {
      first = share - 3 * (share >> 4);
      later = max(share >> 5, 6 * p.min_share);
      border = static_cast<int>(min(static_cast<int64_t>(first) * p.grid, static_cast<int64_t>(total)));
      runs += (total - border + later - 1) / later;
    }
  }
  __device__ __forceinline__ int run_of(int granule, int grid) const {
    return granule < border ? static_cast<int>(static_cast<uint32_t>(granule) / static_cast<uint32_t>(first))
                            : grid + (granule - border) / later;
  }
  __device__ __forceinline__ int64_t begin(int run, int grid) const {
    return run < grid ? static_cast<int64_t>(run) * first : border + static_cast<int64_t>(run - grid) * later;
  }
};
// Runs there can be at most, per CTA: its own and 3/16 of a share in pieces of 1/32 of it (six of them, rounded down by
// 1 in 24 at most).
constexpr int kRunsPerCta = 8;

// The pages of a segment's granules, for the warp that loads tiles: 32 granules (four or eight tiles) per look-up of the
// table, the next 32 under way while these are used.
struct PageWalk {
  const int32_t* row;        // the session's table row
  int next, end, here, ahead;

  // (unchecked: the check waits for the value)
  __device__ __forceinline__ static int fetch(const PagedAttnParams& p, const int32_t* row, int tok, int end, int lane) {
    const int t = tok + (lane << p.gran_shift);
    return t < end ? row[t >> p.v.page_shift] : 0;
  }
  __device__ __forceinline__ void advance(const PagedAttnParams& p, int lane) {
    ahead = fetch(p, row, next, end, lane);
    next += 32 << p.gran_shift;
  }
  __device__ __forceinline__ void begin(const PagedAttnParams& p, int s, int tok0, int tok1, int first, int lane) {
    row = p.v.table + s * p.v.table_stride;
    next = tok0 + (32 << p.gran_shift);
    end = tok1;
    here = first;
    advance(p, lane);
  }
  // The page of granule `lane` of the segment's tile `i`.
  __device__ __forceinline__ int page(const PagedAttnParams& p, int i, int lane) {
    const int per = kTile >> p.gran_shift, first = (i * per) & 31;
    if (first == 0 && i > 0) {
      here = ahead;
      advance(p, lane);
    }
    int pg = __shfl_sync(0xffffffffu, here, first + (lane & (per - 1)));
    if (pg < 0 || pg >= p.v.n_pages) {
      paged_report(p.v);
      pg = 0;
    }
    return pg;
  }
};

template <int DH, bool BF16, int GP>
__global__ void __launch_bounds__(kPagedThreads, 1)
paged_attn_kernel(const __grid_constant__ CUtensorMap tm, const PagedAttnParams p) {
  using C = PagedCfg<DH, GP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sK = smem;
  uint8_t* sV = smem + C::kOffV;
  uint8_t* sQ = smem + C::kOffQ;
  uint8_t* sP = smem + C::kOffP;
  uint8_t* aux = smem + C::kOffAux;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(aux);
  uint64_t* k_empty = k_full + C::kStages;
  uint64_t* v_full = k_empty + C::kStages;
  uint64_t* v_empty = v_full + C::kStages;
  uint64_t* q_full = v_empty + C::kStages;
  uint64_t* q_empty = q_full + kSegs;
  uint64_t* s_full = q_empty + kSegs;
  uint64_t* p_full = s_full + kBufs;
  uint64_t* pv_done = p_full + kBufs;
  uint64_t* taken = pv_done + 2;
  uint64_t* half_full = taken + 1;       // group 1's part of a segment is in shared memory ...
  uint64_t* half_read = taken + 2;       // ... and group 0 has it
  float* s_max = reinterpret_cast<float*>(aux + 384);                 // [2 groups][4 warps][16]
  float* s_sum = s_max + 128;                                         // [2 groups][4 warps][16]
  float* s_join = s_sum + 128;                                        // group 1's m and l: [2][16]
  int* s_plan = reinterpret_cast<int*>(aux + 1600);                   // 0 unit, 1 granule, 2 run, 3 held, 4.. scan
  int* s_pre = s_plan + 4 + kPagedWarps;                              // [warps] granules before the units of a warp
  static_assert(4 + 2 * kPagedWarps <= 30, "the set-up's words");
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_plan + 30);
  Segment* segs = reinterpret_cast<Segment*>(aux + 1728);
  int* s_pages = reinterpret_cast<int*>(aux + 1728 + kSegs * 16);     // [segments][32]
  volatile int* s_abort = s_plan + 31;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  if (warp == 9) {
    tmem_alloc(s_tmem, kTmemColumns);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kSegs; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 12);        // eight softmax warps, both issuers, both loaders
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    mbar_init(taken, 1);
    mbar_init(half_full, 128);
    mbar_init(half_read, 128);
    *s_abort = 0;
    fence_mbar_init();
  }
  if (tid == 128) prefetch_tensormap(&tm);
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ------------------------------------------------------------------ this CTA's run of granules
  auto held = [&](int u) { return paged_count(p.v, p.lens[kv_head_of(p, u)]); };
  const int gs = p.gran_shift;
  auto granules = [&](int n) { return (n + (1 << gs) - 1) >> gs; };
  auto cost = [&](int n) { return n > 0 ? granules(n) + p.min_share : 0; };
  int end_unit = p.units;
  const int per = (p.units + kPagedThreads - 1) / kPagedThreads;
  int total = 0;
  if (p.whole) {
    const int u0 = static_cast<int>(static_cast<int64_t>(p.units) * cta / p.grid);
    end_unit = static_cast<int>(static_cast<int64_t>(p.units) * (cta + 1) / p.grid);
    if (tid == 0) {
      s_plan[0] = u0;
      s_plan[1] = 0;
      s_plan[2] = 0x7FFFFFFF;
      s_plan[3] = u0 < end_unit ? held(u0) : 0;
    }
    for (int u = u0 + tid; u < end_unit; u += kPagedThreads)
      if (held(u) == 0) write_empty(p, u, DH);
  } else {
    const int first = min(tid * per, p.units), last = min(first + per, p.units);
    int sum = 0;
    for (int u = first; u < last; ++u) {
      const int n = held(u);
      sum += cost(n);
      if (n == 0 && u % p.grid == cta) write_empty(p, u, DH);
    }
    int pre = sum;
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, pre, d);
      if (lane >= d) pre += y;
    }
    if (lane == 31) s_plan[4 + warp] = pre;
    __syncthreads();
    const int y = lane < kPagedWarps ? s_plan[4 + lane] : 0;
    total = __reduce_add_sync(0xffffffffu, y);
    pre += __reduce_add_sync(0xffffffffu, lane < warp ? y : 0);
    pre -= sum;
    if (lane == 0) s_pre[warp] = pre;
    const Cut cut(p, total);
    const int64_t g0 = cut.begin(cta, p.grid);
    if (tid == 0) s_plan[2] = g0 < cut.border ? static_cast<int>(min(static_cast<int64_t>(cut.first), cut.border - g0)) : 0;
    if (g0 >= pre && g0 < pre + sum) {
      int u = first, at = pre;
      for (int n = cost(held(u)); at + n <= g0 && u + 1 < last; n = cost(held(++u))) at += n;
      s_plan[0] = u;
      s_plan[1] = static_cast<int>(g0) - at;
      s_plan[3] = held(u);
    }
    if (cta == 0) {                      // for the join
      int at = pre;
      for (int u = first; u < last; ++u) {
        p.ws_prefix[u] = at;
        at += cost(held(u));
      }
      if (tid == 0) p.ws_prefix[p.units] = total;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = *s_tmem;
  if (warp == 8) {
    // ---------------------------------------------------------------- segments
    int u = s_plan[0], at = s_plan[1], left = s_plan[2], n = s_plan[3];
    int seg = 0, run = cta, run_segs = 0;
    const Cut cut(p, total);
    bool ok = true;
    // Takes the next of the runs that are handed out, and finds the unit it starts in.
    auto take_run = [&]() {
      int k = 0;
      if (lane == 0) k = atomicAdd(p.ws_prefix + p.units + 1, 1);
      run = min(p.grid + __shfl_sync(0xffffffffu, k, 0), cut.runs);
      run_segs = 0;
      const int g0 = static_cast<int>(cut.begin(run, p.grid));
      left = run < cut.runs ? min(cut.later, total - g0) : 0;
      if (left == 0) return;
      // as at the set-up each lane takes `per` units of the warp that had the place, then walks its own
      const uint32_t from = __ballot_sync(0xffffffffu, lane < kPagedWarps && s_pre[lane < kPagedWarps ? lane : 0] <= g0);
      const int w = 31 - __clz(from), first = min((w * 32 + lane) * per, p.units), last = min(first + per, p.units);
      int sum = 0;
      for (int i = first; i < last; ++i) sum += cost(held(i));
      int upto = sum;
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      upto += s_pre[w];
      const uint32_t hit = __ballot_sync(0xffffffffu, upto > g0);
      const int l = hit != 0 ? __ffs(hit) - 1 : 0;
      int i = first, before = upto - sum, mine = 0;
      for (; i < last; ++i) {
        mine = held(i);
        if (before + cost(mine) > g0) break;
        before += cost(mine);
      }
      u = __shfl_sync(0xffffffffu, i, l);
      n = __shfl_sync(0xffffffffu, mine, l);
      at = __shfl_sync(0xffffffffu, g0 - before, l);
      if (hit == 0) left = 0;                              // (the counts changed under us)
    };
    while (true) {
      // one segment ahead of the loader: further ahead, runs would be taken that another CTA could begin sooner
      if (seg > 0) ok = __all_sync(0xffffffffu, mbar_wait(taken, (seg - 1) & 1, s_abort));
      if (!ok) break;
      int n_next = 0, tok0 = 0, ntok = 0;
      while (true) {
        if (left <= 0 && cut.runs > p.grid && run < cut.runs) take_run();
        if (left <= 0 || u >= end_unit) break;
        n_next = u + 1 < end_unit ? p.lens[kv_head_of(p, u + 1)] : 0;        // (clamped when its turn comes)
        const int head = n > 0 ? max(p.min_share - at, 0) : 0;             // of the unit's head, in this run
        tok0 = max(at - p.min_share, 0) << gs;
        ntok = n - tok0;
        if (!p.whole) {
          ntok = static_cast<int>(min(static_cast<int64_t>(ntok), static_cast<int64_t>(left - head) << gs));
          left -= head;
        }
        if (ntok > 0) break;
        ++u;
        at = 0;
        n = paged_count(p.v, n_next);
      }
      const int qslot = seg % kSegs;
      if (ntok <= 0) {                                     // the end
        if (mbar_wait(&q_empty[qslot], ((seg / kSegs) & 1) ^ 1, s_abort) && lane == 0) {
          segs[qslot].ntok = 0;
          mbar_arrive(&q_full[qslot]);
        }
        break;
      }
      const UnitHeads w = unit_heads(p, u);
      const int first_pages = PageWalk::fetch(p, p.v.table + w.s * p.v.table_stride, tok0, tok0 + ntok, lane);
      constexpr int kVecs = DH / 8, kLoads = (GP * kVecs + 31) / 32;
      uint4 q[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int e = lane + 32 * i, row = e / kVecs, vec = e % kVecs;
        q[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < w.n && row < GP)
          q[i] = *reinterpret_cast<const uint4*>(p.q + w.s * p.qs[0] + (w.hq0 + row) * p.qs[1] + 8 * vec);
      }
      ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[qslot], ((seg / kSegs) & 1) ^ 1, s_abort));
      if (!ok) break;
      s_pages[qslot * 32 + lane] = first_pages;
      // the query rows: [chunk][16 rows][128 bytes], 128-byte swizzle
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int e = lane + 32 * i, row = e / kVecs, vec = e % kVecs;
        if (row < GP)
          *reinterpret_cast<uint4*>(sQ + qslot * C::kQBytes + (vec >> 3) * 2048 + row * 128 +
                                    (((vec & 7) ^ (row & 7)) << 4)) = q[i];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        Segment d;
        d.unit = u;
        d.tok0 = tok0;
        d.ntok = ntok;
        d.slot = (tok0 == 0 && ntok == n) ? -1 : 2 * run + (run_segs == 0 ? 0 : 1);
        segs[qslot] = d;
        mbar_arrive(&q_full[qslot]);
      }
      ++seg;
      ++run_segs;
      if (!p.whole) left -= granules(ntok);
      ++u;
      at = 0;
      n = paged_count(p.v, n_next);
    }
  } else if (warp >= 11) {
    // ---------------------------------------------------------------- K tiles (warp 11) and V tiles (warp 12)
    const bool is_k = warp == 11;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    const uint32_t ring = smem_u32(is_k ? sK : sV);
    const int x_plane = is_k ? 0 : static_cast<int>(p.unit_plane);
    const uint64_t policy = p.chunks == 1 ? l2_evict_first() : l2_evict_normal();
    int it = 0;
    // The first segment is plain from the set-up: its first tiles are asked for while warp 8 still gathers its queries.
    Segment d;
    d.unit = s_plan[0];
    d.tok0 = max(s_plan[1] - p.min_share, 0) << gs;
    d.ntok = s_plan[2] > 0 && d.unit < end_unit ? s_plan[3] - d.tok0 : 0;
    if (!p.whole && d.ntok > 0)
      d.ntok = static_cast<int>(min(static_cast<int64_t>(d.ntok),
                                    static_cast<int64_t>(s_plan[2] - max(p.min_share - s_plan[1], 0)) << gs));
    bool early = d.ntok > 0;
    for (int seg = 0;; ++seg) {
      const int qslot = seg % kSegs;
      int first_pages = 0;
      bool ok = true;
      auto receive = [&]() {                               // the segment as warp 8 published it
        ok = __all_sync(0xffffffffu, mbar_wait(&q_full[qslot], (seg / kSegs) & 1, s_abort));
        if (!ok) return;
        d = segs[qslot];
        first_pages = s_pages[qslot * 32 + lane];
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&q_empty[qslot]);
          if (is_k) mbar_arrive(taken);
        }
      };
      if (!early) {
        receive();
        if (!ok || d.ntok == 0) break;
      } else {
        const int32_t* row = p.v.table + unit_heads(p, d.unit).s * p.v.table_stride;
        first_pages = PageWalk::fetch(p, row, d.tok0, d.tok0 + d.ntok, lane);
      }
      const UnitHeads w = unit_heads(p, d.unit);
      const int end = d.tok0 + d.ntok, x_head = w.h * static_cast<int>(p.unit_head) + x_plane;
      PageWalk walk;
      walk.begin(p, w.s, d.tok0, end, first_pages, lane);
      for (int t0 = d.tok0; t0 < end; t0 += kTile, ++it) {
        const int st = it % C::kStages, ng = (min(kTile, end - t0) + (1 << gs) - 1) >> gs;
        const int pg = walk.page(p, (t0 - d.tok0) / kTile, lane);
        ok = mbar_wait(&empty[st], ((it / C::kStages) & 1) ^ 1, s_abort);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], (ng << gs) * DH * 2);
        __syncwarp();
        if (lane < ng)
          tma_load_5d(ring + st * C::kTileBytes + lane * ((DH * 2) << gs), &tm, &full[st], 0, 0, 0,
                      ((t0 + (lane << gs)) & (p.v.page - 1)) >> 3, pg * static_cast<int>(p.unit_page) + x_head, policy);
        if (early) {
          early = false;
          receive();
          if (!ok) break;
        }
      }
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- S^T = K Q^T: 128 tokens x 16 heads
    if (lane == 0) {
      constexpr uint32_t kIdesc = umma_idesc(BF16 ? 1u : 0u, 0u, kTile, 16);
      constexpr uint32_t kHiK = umma_desc_hi(C::kRowGroup), kHiQ = umma_desc_hi(1024);
      int it = 0;
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int qslot = seg % kSegs;
        if (!mbar_wait(&q_full[qslot], (seg / kSegs) & 1, s_abort)) break;
        const int ntok = segs[qslot].ntok;
        if (ntok == 0) break;
        const uint32_t q_lo = umma_desc_lo(smem_u32(sQ + qslot * C::kQBytes), 16);
        for (int t0 = 0; t0 < ntok && ok; t0 += kTile, ++it) {
          const int st = it % C::kStages;
          ok = mbar_wait(&k_full[st], (it / C::kStages) & 1, s_abort);
          if (it >= kBufs) ok = mbar_wait(&p_full[it % kBufs], ((it / kBufs) - 1) & 1, s_abort) && ok;   // the buffer was read
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_lo = umma_desc_lo(smem_u32(sK + st * C::kTileBytes), 16);
#pragma unroll
          for (int kk = 0; kk < DH / 16; ++kk)
            umma_ss(tmem + 16 * (it % kBufs), k_lo + (kk >> 2) * 64 + (kk & 3) * 2, kHiK, q_lo + (kk >> 2) * 128 + (kk & 3) * 2,
                    kHiQ, kIdesc, kk > 0);
          tc_commit(&s_full[it % kBufs]);
          tc_commit(&k_empty[st]);
        }
        tc_commit(&q_empty[qslot]);
      }
    }
  } else if (warp == 10) {
    // ---------------------------------------------------------------- O^T += V^T P^T: 128 rows (of the head dim) x heads
    if (lane == 0) {
      constexpr uint32_t kIdesc = umma_idesc(BF16 ? 1u : 0u, 1u, 128, C::kNP) | (1u << 15);     // both MN-major
      constexpr uint32_t kHiV = umma_desc_hi(C::kRowGroup), kHiP = umma_desc_hi(8 * C::kPRow, C::kPRow == 32 ? 6 : 4);
      int it = 0;
      bool ok = true;
      for (int seg = 0; ok; ++seg) {
        const int qslot = seg % kSegs;
        if (!mbar_wait(&q_full[qslot], (seg / kSegs) & 1, s_abort)) break;
        const int ntok = segs[qslot].ntok;
        mbar_arrive(&q_empty[qslot]);
        if (ntok == 0) break;
        for (int t0 = 0; t0 < ntok && ok; t0 += kTile, ++it) {
          const int st = it % C::kStages, steps = (min(kTile, ntok - t0) + 15) >> 4;
          ok = mbar_wait(&v_full[st], (it / C::kStages) & 1, s_abort);
          ok = mbar_wait(&p_full[it % kBufs], (it / kBufs) & 1, s_abort) && ok;
          if (!ok) break;
          tc_fence_after();
          // (head dim 64: rows 64.. of the product read the next eight tokens in place of a second column chunk;
          // nobody reads what they give)
          const uint32_t v_lo = umma_desc_lo(smem_u32(sV + st * C::kTileBytes), 1024);
          const uint32_t p_lo = umma_desc_lo(smem_u32(sP + (it & 1) * C::kPBytes), 16);
          for (int kk = 0; kk < steps; ++kk)
            umma_ss(tmem + kColO + 32 * (it & 1), v_lo + kk * (2 * C::kRowGroup >> 4), kHiV, p_lo + kk * C::kPRow, kHiP,
                    kIdesc, t0 >= 2 * kTile || kk > 0);
          tc_commit(&v_empty[st]);
          tc_commit(&pv_done[it & 1]);
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    const int grp = warp >> 2, row = tid & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_col = tmem + lanes + kColO + 32 * grp;
    float* my_max = s_max + 64 * grp;
    float* my_sum = s_sum + 64 * grp;
    float* other_o = reinterpret_cast<float*>(sP + C::kPBytes);         // [GP][128], in group 1's P buffer
    uint8_t* p_row = sP + grp * C::kPBytes + row * C::kPRow;
    const uint32_t swz = C::kPRow == 32 ? (row >> 2) & 1 : (row >> 1) & 3;
    int it = 0, halves = 0;
    bool given = false;                                    // group 1: its part has not been collected yet
    // (the groups meet nowhere but in segments of several tiles, through barriers with a limit: short segments go to
    // either group in turn, two at a time)
    for (int seg = 0;; ++seg) {
      const int qslot = seg % kSegs;
      const bool ok = mbar_wait(&q_full[qslot], (seg / kSegs) & 1, s_abort);
      __syncwarp();
      if (bar_any(2 + grp, 128, !ok)) break;
      const Segment d = segs[qslot];
      if (d.ntok == 0) break;
      const UnitHeads w = unit_heads(p, d.unit);
      float m[GP], l[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) m[g] = kFloor, l[g] = 0.f;
      float* xs = p.weights != nullptr ? p.ws_x + static_cast<int64_t>(d.unit) * GP * p.x_stride + d.tok0 : nullptr;
      // (the first store to a page the SM has not translated yet holds up everything behind it: ask for it early)
      if (xs != nullptr && row < w.n) asm volatile("prefetch.global.L2 [%0];" ::"l"(xs + row * p.x_stride));
      int last = -1;                                       // this group's last tile
      for (int t0 = 0; t0 < d.ntok; t0 += kTile, ++it) {
        if ((it & 1) != grp) continue;
        const int nv = min(kTile, d.ntok - t0);
        mbar_wait(&s_full[it % kBufs], (it / kBufs) & 1, s_abort);
        __syncwarp();
        tc_fence_after();
        uint32_t raw[GP];
        tmem_ld_n<GP>(tmem + lanes + 16 * (it % kBufs), raw);
        tmem_ld_wait();
        float x[GP], e[GP];
#pragma unroll
        for (int g = 0; g < GP; ++g) x[g] = __uint_as_float(raw[g]) * p.scale_log2;
        if (w.n < GP) {
#pragma unroll
          for (int g = 1; g < GP; ++g)
            if (g >= w.n) x[g] = -INFINITY;
        }
        if (row >= nv) {
#pragma unroll
          for (int g = 0; g < GP; ++g) x[g] = -INFINITY;
        } else if (xs != nullptr) {
#pragma unroll
          for (int g = 0; g < GP; ++g)
            if (g < w.n) xs[g * p.x_stride + t0 + row] = x[g];
        }
        float over = -INFINITY;
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          e[g] = x[g] - m[g];
          over = fmaxf(over, e[g]);
        }
        if (bar_any(2 + grp, 128, over > kRaise + kAbove<BF16>)) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float t = warp_max(x[g]);
            if (lane == 0) my_max[(warp & 3) * 16 + g] = t;
          }
          bar_sync(2 + grp, 128);
          float f[GP];
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            const float top = fmaxf(fmaxf(my_max[g], my_max[16 + g]), fmaxf(my_max[32 + g], my_max[48 + g]));
            const float t = fmaxf(top - kAbove<BF16>, m[g]);
            f[g] = t == m[g] ? 1.f : exp2_fast(m[g] - t);
            m[g] = t;
            l[g] *= f[g];
            e[g] = x[g] - t;
          }
          if (last >= 0) {
            mbar_wait(&pv_done[grp], (last >> 1) & 1, s_abort);
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              uint32_t o[GP];
              tmem_ld_n<GP>(o_col + part * GP, o);
              tmem_ld_wait();
#pragma unroll
              for (int g = 0; g < GP; ++g) o[g] = __float_as_uint(__uint_as_float(o[g]) * f[g]);
              tmem_st_n<GP>(o_col + part * GP, o);
            }
            tmem_st_wait();
          }
        }
        uint32_t words[GP == 1 ? 1 : GP];                  // GP high parts, then GP low parts
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          e[g] = exp2_fast(e[g]);
          l[g] += e[g];
        }
        if constexpr (GP == 1) {
          const uint16_t hi = narrow<BF16>(e[0]);
          words[0] = hi | (static_cast<uint32_t>(narrow<BF16>((e[0] - widen<BF16>(hi)) * kLowScale<BF16>)) << 16);
        } else {
#pragma unroll
          for (int g = 0; g < GP; g += 2) {
            const uint32_t hi = narrow2<BF16>(e[g], e[g + 1]);
            words[g / 2] = hi;
            words[(GP + g) / 2] = narrow2<BF16>((e[g] - widen<BF16>(static_cast<uint16_t>(hi))) * kLowScale<BF16>,
                                                (e[g + 1] - widen<BF16>(static_cast<uint16_t>(hi >> 16))) * kLowScale<BF16>);
          }
        }
        if (it >= 2) mbar_wait(&pv_done[grp], ((it - 2) >> 1) & 1, s_abort);      // the P before was read
        if (given) {
          mbar_wait(half_read, (halves - 1) & 1, s_abort);
          given = false;
        }
        if constexpr (GP == 1) {
          *reinterpret_cast<uint32_t*>(p_row + (swz << 4)) = words[0];
        } else if constexpr (GP == 2) {
          *reinterpret_cast<uint2*>(p_row + (swz << 4)) = make_uint2(words[0], words[1]);
        } else {
#pragma unroll
          for (int c = 0; c < GP / 4; ++c)
            *reinterpret_cast<uint4*>(p_row + ((c ^ swz) << 4)) =
                make_uint4(words[4 * c], words[4 * c + 1], words[4 * c + 2], words[4 * c + 3]);
        }
        if (row >= nv && row < ((nv + 15) & ~15)) {
          // rows behind the last token: whatever the page holds there must not meet a weight of zero
          const int st = it % C::kStages;
          mbar_wait(&v_full[st], (it / C::kStages) & 1, s_abort);
          uint8_t* v_row = sV + st * C::kTileBytes + (row >> 3) * C::kRowGroup + (row & 7) * 128;
#pragma unroll
          for (int c = 0; c < C::kChunks; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v_row + c * 1024 + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[it % kBufs]);
        last = it;
      }
      if (last < 0) {                                      // one tile, and the other group had it
        if (lane == 0) mbar_arrive(&q_empty[qslot]);
        continue;
      }
      // ---- the segment's sums: of either group, then of both
      warp_sums<GP>(l, lane);
      if (lane % (32 / GP) == 0) my_sum[(warp & 3) * 16 + lane / (32 / GP)] = l[0];
      bar_sync(2 + grp, 128);
#pragma unroll
      for (int g = 0; g < GP; ++g) l[g] = (my_sum[g] + my_sum[16 + g]) + (my_sum[32 + g] + my_sum[48 + g]);
      mbar_wait(&pv_done[grp], (last >> 1) & 1, s_abort);
      __syncwarp();
      tc_fence_after();
      uint32_t hi[GP], lo[GP];
      tmem_ld_n<GP>(o_col, hi);
      tmem_ld_n<GP>(o_col + GP, lo);
      tmem_ld_wait();
      float o[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        // (an infinite value times a low part, which may be 0 or negative, is none of the formula's terms)
        const float y = __uint_as_float(lo[g]) * (1.f / kLowScale<BF16>);
        o[g] = __uint_as_float(hi[g]) + (fabsf(y) < INFINITY ? y : 0.f);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_empty[qslot]);
      if (d.ntok > kTile) {                                // both groups had tiles: group 0 finishes
        ++halves;
        if (grp == 1) {
#pragma unroll
          for (int g = 0; g < GP; ++g) {
            other_o[g * 128 + row] = o[g];
            if (row == g) s_join[g] = m[g], s_join[16 + g] = l[g];
          }
          mbar_arrive(half_full);
          given = true;                                    // (its P buffer, where O lies, is not written until then)
          continue;
        }
        mbar_wait(half_full, (halves - 1) & 1, s_abort);
#pragma unroll
        for (int g = 0; g < GP; ++g) {
          const float m1 = s_join[g], top = fmaxf(m[g], m1);
          const float f0 = exp2_fast(m[g] - top), f1 = exp2_fast(m1 - top);
          m[g] = top;
          // (which group had the first tile depends on what the CTA did before: the sum must not, so no fused multiply-add)
          l[g] = __fadd_rn(__fmul_rn(l[g], f0), __fmul_rn(s_join[16 + g], f1));
          o[g] = __fadd_rn(__fmul_rn(o[g], f0), __fmul_rn(other_o[g * 128 + row], f1));
        }
        mbar_arrive(half_read);
      }
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        if (g >= w.n) continue;
        if (d.slot >= 0) {
          if (row < DH) p.ws_o[(static_cast<int64_t>(d.slot) * GP + g) * DH + row] = o[g];
          if (row == g) p.ws_ml[d.slot * GP + g] = make_float2(m[g], l[g]);
        } else {
          if (row < DH) p.out[w.s * p.os[0] + (w.hq0 + g) * p.os[1] + row] = narrow<BF16>(o[g] / l[g]);
          if (row == g && (p.lse != nullptr || xs != nullptr)) {
            const float lse = m[g] + log2f(l[g]);
            if (p.lse != nullptr) p.lse[static_cast<int64_t>(w.s) * p.Hq + w.hq0 + g] = lse * 0.6931471805599453f;
            if (xs != nullptr) p.ws_lse[static_cast<int64_t>(d.unit) * GP + g] = lse;
          }
        }
      }
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (*s_abort != 0) {
    if (tid == 0 && p.v.status != nullptr) atomicExch(p.v.status, WE_B200_ST_WAIT_EXPIRED);
    __nanosleep(1000000);  // let copies and products that are still in flight land before the CTA goes away
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

// ------------------------------------------------------------------ units that several CTAs share
// Where the pieces of a unit lie: in n runs from `run` on, and the workspace slot of each.
struct Pieces {
  int run, n, slot0;
};
// (a unit at [a, b) of the granules, its head the first `head` of them)
__device__ __forceinline__ Pieces pieces_of(const Cut& cut, int a, int b, int head, int grid) {
  Pieces r;
  r.run = cut.run_of(a + head, grid);
  r.n = cut.run_of(b - 1, grid) - r.run + 1;
  r.slot0 = 2 * r.run + (cut.begin(r.run, grid) >= a ? 0 : 1);
  return r;
}
__device__ __forceinline__ int slot_of_piece(const Pieces& r, int k) { return k == 0 ? r.slot0 : 2 * (r.run + k); }

// Softmax statistics of a head over the pieces of its unit, by one warp: maximum and sum, in every lane.
template <int GP>
__device__ __forceinline__ float2 join_ml(const PagedAttnParams& p, const Pieces& r, int g, int lane) {
  float top = -INFINITY;
  for (int k = lane; k < r.n; k += 32) top = fmaxf(top, p.ws_ml[slot_of_piece(r, k) * GP + g].x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f;
  for (int k = lane; k < r.n; k += 32) {
    const float2 ml = p.ws_ml[slot_of_piece(r, k) * GP + g];
    sum += ml.y * exp2_fast(ml.x - top);
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return make_float2(top, sum);
}

template <int DH, bool BF16, int GP>
__global__ void __launch_bounds__(kJoinThreads, 4) paged_join_kernel(const PagedAttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kWarps = kJoinThreads / 32, kPer = DH / 32;
  __shared__ float s_o[kWarps][DH];
  __shared__ float s_lse[kMaxGroup];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // ---- outputs: a head per block, its pieces dealt out to the warps, or where there are many heads one per warp
  if (blockIdx.x < p.out_blocks) {
    const int heads = min(p.group, kMaxGroup);
    const int64_t items = static_cast<int64_t>(p.units) * heads;
    const int64_t step = static_cast<int64_t>(p.out_blocks) * (p.out_by_warp ? kWarps : 1);
    const int first = p.out_by_warp ? 0 : warp, stride = p.out_by_warp ? 1 : kWarps;
    for (int64_t item = p.out_by_warp ? blockIdx.x * kWarps + warp : blockIdx.x; item < items; item += step) {
      const int u = static_cast<int>(item / heads), g = static_cast<int>(item - static_cast<int64_t>(u) * heads);
      const int a = p.ws_prefix[u], b = p.ws_prefix[u + 1], total = p.ws_prefix[p.units];   // (loads that go out together)
      if (a == b) continue;
      const Cut cut(p, total);
      const Pieces r = pieces_of(cut, a, b, p.min_share, p.grid);
      const UnitHeads w = unit_heads(p, u);
      if (r.n == 1 || g >= w.n) continue;
      const float* ws_o = p.ws_o + static_cast<int64_t>(g) * DH + lane;
      float o[kPer], here[kPer];                           // (the first piece is on its way while the statistics are)
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        o[i] = 0.f;
        here[i] = first < r.n ? ws_o[static_cast<int64_t>(slot_of_piece(r, first)) * GP * DH + 32 * i] : 0.f;
      }
      const float2 ml = join_ml<GP>(p, r, g, lane);
#pragma unroll 2
      for (int k = first; k < r.n; k += stride) {
        const float f = exp2_fast(p.ws_ml[slot_of_piece(r, k) * GP + g].x - ml.x);
        const int next = k + stride;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          o[i] += f * here[i];
          here[i] = next < r.n ? ws_o[static_cast<int64_t>(slot_of_piece(r, next)) * GP * DH + 32 * i] : 0.f;
        }
      }
      uint16_t* out = p.out + w.s * p.os[0] + (w.hq0 + g) * p.os[1];
      if (p.out_by_warp) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) out[32 * i + lane] = narrow<BF16>(o[i] / ml.y);
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) s_o[warp][32 * i + lane] = o[i];
        __syncthreads();
        if (tid < DH) {
          float x = 0.f;
#pragma unroll
          for (int k = 0; k < kWarps; ++k) x += s_o[k][tid];
          out[tid] = narrow<BF16>(x / ml.y);
        }
        __syncthreads();
      }
      if ((p.out_by_warp ? lane : tid) == 0 && p.lse != nullptr)
        p.lse[static_cast<int64_t>(w.s) * p.Hq + w.hq0 + g] = (ml.x + log2f(ml.y)) * 0.6931471805599453f;
    }
    return;
  }
  // ---- weights: 1024 tokens of a kv head at a time, four neighbours per thread (they lie in one page).  The logits come
  // through shared memory, all heads at once: with loads to registers an SM has half as many bytes on their way.
  // Where a kv head has several units, their shares of a token's weight are added up before they go to memory, in the
  // order of the heads.
  extern __shared__ __align__(128) float s_x[];        // [GP][kJoinTokens]
  __shared__ uint64_t s_full;
  __shared__ int s_abort;
  if (tid == 0) {
    mbar_init(&s_full, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  uint32_t phase = 0;
  const int kv_heads = p.units / p.chunks;
  const int64_t items = static_cast<int64_t>(kv_heads) * ((p.x_stride + kJoinTokens - 1) / kJoinTokens);
  for (int64_t item = blockIdx.x - p.out_blocks; item < items; item += gridDim.x - p.out_blocks) {
    const int part = static_cast<int>(item / kv_heads), kvh = static_cast<int>(item - static_cast<int64_t>(part) * kv_heads);
    const int t0 = part * kJoinTokens, t = t0 + 4 * tid;
    const int total = p.ws_prefix[p.units], held = p.lens[kvh];
    const int n = paged_count(p.v, held);
    if (t0 >= n) continue;
    const Cut cut(p, total);
    const int s = kvh / p.v.Hkv, h = kvh - s * p.v.Hkv;
    const int pg = t < n ? p.v.table[s * p.v.table_stride + (t >> p.v.page_shift)] : 0;
    float add[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < p.chunks; ++c) {
      const int u = kvh * p.chunks + c, nh = unit_heads(p, u).n;
      if (warp == 0) {
        // (whole rows of pages: what lies behind the last token is not used)
        const uint32_t bytes = static_cast<uint32_t>((min(n - t0, kJoinTokens) + 3) & ~3) * 4;
        if (lane == 0) mbar_arrive_expect_tx(&s_full, bytes * nh);
        __syncwarp();
        if (lane < nh)
          bulk_load(s_x + lane * kJoinTokens, p.ws_x + (static_cast<int64_t>(u) * GP + lane) * p.x_stride + t0, bytes, &s_full);
      }
      const Pieces r = pieces_of(cut, p.ws_prefix[u], p.ws_prefix[u + 1], p.min_share, p.grid);
      for (int g = warp; g < nh; g += kWarps) {
        float lse;
        if (r.n == 1) {
          lse = p.ws_lse[static_cast<int64_t>(u) * GP + g];
        } else {
          const float2 ml = join_ml<GP>(p, r, g, lane);
          lse = ml.x + log2f(ml.y);
        }
        if (lane == 0) s_lse[g] = lse;
      }
      mbar_wait(&s_full, phase & 1, &s_abort);
      ++phase;
      __syncthreads();
      if (t < n) {
#pragma unroll 4
        for (int g = 0; g < nh; ++g) {
          const float4 x = *reinterpret_cast<const float4*>(s_x + g * kJoinTokens + 4 * tid);
          const float le = s_lse[g];
          add[0] += exp2_fast(x.x - le);
          add[1] += exp2_fast(x.y - le);
          add[2] += exp2_fast(x.z - le);
          add[3] += exp2_fast(x.w - le);
        }
      }
      __syncthreads();                                   // before the logits and sums of the next unit
    }
    if (t >= n) continue;
    if (pg < 0 || pg >= p.v.n_pages) {
      paged_report(p.v);
      continue;
    }
    float* dst = p.weights + ((static_cast<int64_t>(pg) * p.v.Hkv + h) << p.v.page_shift) + (t & (p.v.page - 1));
    if (t + 3 < n) {
      atomicAdd(reinterpret_cast<float4*>(dst), make_float4(add[0], add[1], add[2], add[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (t + k < n) atomicAdd(dst + k, add[k]);
    }
  }
  if (s_abort != 0) {
    if (tid == 0 && p.v.status != nullptr) atomicExch(p.v.status, WE_B200_ST_WAIT_EXPIRED);
    __nanosleep(1000000);  // let copies that are still in flight land before the CTA goes away
  }
}

// In front of the others, where one of the two is needed: the number of runs handed out is 0, and sessions without a new
// token hold nothing as far as the others see.  (Asking for n_new wherever they look at a count made small batches 5 %
// slower that have no n_new.)
__global__ void paged_prepare_kernel(int32_t* counter, const int32_t* lens, const int32_t* n_new, int32_t* seen, int heads,
                                     int Hkv) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i == 0 && counter != nullptr) *counter = 0;
  if (n_new != nullptr && i < heads) seen[i] = n_new[i / Hkv] > 0 ? lens[i] : 0;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ------------------------------------------------------------------ host
struct PagedPlan {
  int chunks, gp, units, gran_shift, grid, whole, min_share, dynamic;
  int64_t cap;
  size_t off_ml, off_o, off_lse, off_x, off_seen, bytes;
};

static int paged_plan(const we_b200_paged_geom& g, int Hq, bool accumulate, bool padded, PagedPlan* r) {
  const int group = Hq / g.Hkv;
  r->chunks = (group + kMaxGroup - 1) / kMaxGroup;
  const int n = group < kMaxGroup ? group : kMaxGroup;
  r->gp = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16;
  const int64_t units = static_cast<int64_t>(g.S) * g.Hkv * r->chunks;
  r->gran_shift = g.page == 16 ? 4 : 5;
  r->cap = static_cast<int64_t>(g.max_pages) * g.page;
  r->min_share = kTile >> r->gran_shift;
  // granules and heads, counted in 32 bits by the kernels
  const int64_t most = units * ((r->cap >> r->gran_shift) + r->min_share);
  if (units > (1 << 24) || most > 0x3FFFFFFF) return WE_B200_E_LIMIT;
  r->units = static_cast<int>(units);
  r->whole = r->cap <= kWholeUnitTokens && !accumulate;
  const int64_t want = r->whole ? units : (most + r->min_share - 1) / r->min_share;
  const int sms = sm_count();
  r->grid = static_cast<int>(want < sms ? want : sms);
  // (decided by the room the sessions have: what they hold is known on the device only)
  r->dynamic = !r->whole && r->grid == sms && most / sms >= 32 * r->min_share;
  const size_t runs = static_cast<size_t>(r->grid) * (r->dynamic ? kRunsPerCta : 1);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  r->off_ml = up(sizeof(int32_t) * (r->units + 2));
  r->off_o = r->off_ml + up(sizeof(float2) * 2 * runs * r->gp);
  r->off_lse = r->off_o + sizeof(float) * 2 * runs * r->gp * g.Dh;
  r->off_x = r->off_lse + up(sizeof(float) * r->units * r->gp);
  r->bytes = r->whole ? 0 : r->off_x;
  if (accumulate) r->bytes += sizeof(float) * static_cast<size_t>(r->units) * r->gp * r->cap;
  r->off_seen = r->bytes;
  if (padded) r->bytes += sizeof(int32_t) * static_cast<size_t>(g.S) * g.Hkv;
  return WE_B200_OK;
}

// One map for both planes: (64 columns, 8 rows, column chunks, groups of 8 rows, pages and heads).  The last axis steps
// by the greatest common divisor of the plane, page and head strides, so any of them can lie anywhere.
static int paged_map(CUtensorMap* m, const void* kv, const we_b200_paged_geom& g, int gran, PagedAttnParams* p) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return WE_B200_E_DRIVER;
  auto gcd = [](int64_t a, int64_t b) {
    while (b != 0) {
      const int64_t t = a % b;
      a = b;
      b = t;
    }
    return a;
  };
  const int64_t page_s = g.n_pages > 1 ? g.page_stride : 0, head_s = g.Hkv > 1 ? g.head_stride : 0;
  int64_t step = gcd(gcd(g.plane_stride, page_s), head_s);
  if (step == 0) step = g.token_stride;
  p->unit_plane = g.plane_stride / step;
  p->unit_page = page_s / step;
  p->unit_head = head_s / step;
  const int64_t top = p->unit_plane + (g.n_pages - 1) * p->unit_page + (g.Hkv - 1) * p->unit_head;
  if (top >= 0x7FFFFFFF || step * 2 >= (1ll << 40) || g.token_stride * 16 >= (1ll << 40)) return WE_B200_E_LIMIT;
  const cuuint32_t chunks = static_cast<cuuint32_t>(g.Dh / 64);
  const cuuint64_t dims[5] = {64, 8, chunks, static_cast<cuuint64_t>(g.page / 8), static_cast<cuuint64_t>(top + 1)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(g.token_stride * 2), 128,
                                 static_cast<cuuint64_t>(g.token_stride * 16), static_cast<cuuint64_t>(step * 2)};
  const cuuint32_t box[5] = {64, 8, chunks, static_cast<cuuint32_t>(gran / 8), 1};
  const cuuint32_t one[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType dt =
      g.dtype == WE_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult rc = fn(m, dt, 5, const_cast<void*>(kv), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? WE_B200_OK : WE_B200_E_DRIVER;
}

template <int DH, bool BF16, int GP>
static int launch_paged(const CUtensorMap& tm, const PagedAttnParams& given, const int32_t* n_new, int32_t* seen, int weight_blocks,
                        cudaStream_t stream) {
  using C = PagedCfg<DH, GP>;
  PagedAttnParams p = given;
  if (n_new != nullptr) p.lens = seen;
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return WE_B200_E_LIMIT;
  if (!done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(paged_attn_kernel<DH, BF16, GP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(paged_join_kernel<DH, BF16, GP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               GP * kJoinTokens * static_cast<int>(sizeof(float)));
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return static_cast<int>(e);
    }
    done[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.grid), 1, 1);
  cfg.blockDim = dim3(kPagedThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.dynamic || n_new != nullptr) {
    const int heads = p.units / p.chunks;
    cudaLaunchConfig_t prepare = cfg;
    prepare.blockDim = dim3(n_new != nullptr ? 256u : 1u, 1, 1);
    prepare.gridDim = dim3(n_new != nullptr ? static_cast<unsigned>(heads + 255) / 256u : 1u, 1, 1);
    prepare.dynamicSmemBytes = 0;
    int32_t* counter = p.dynamic ? p.ws_prefix + p.units + 1 : nullptr;
    e = cudaLaunchKernelEx(&prepare, paged_prepare_kernel, counter, given.lens, n_new, seen, heads, static_cast<int>(p.v.Hkv));
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) {
    e = cudaLaunchKernelEx(&cfg, paged_attn_kernel<DH, BF16, GP>, tm, p);
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  if (e == cudaSuccess && !p.whole) {
    cfg.gridDim = dim3(static_cast<unsigned>(p.out_blocks + weight_blocks), 1, 1);
    cfg.blockDim = dim3(kJoinThreads, 1, 1);
    cfg.dynamicSmemBytes = weight_blocks > 0 ? GP * kJoinTokens * sizeof(float) : 0;
    e = cudaLaunchKernelEx(&cfg, paged_join_kernel<DH, BF16, GP>, p);
    g_launches.fetch_add(1, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return static_cast<int>(e);
  const cudaError_t e2 = cudaGetLastError();
  return e2 == cudaSuccess ? WE_B200_OK : static_cast<int>(e2);
}

template <int DH, bool BF16>
static int launch_group(int gp, const CUtensorMap& tm, const PagedAttnParams& p, const int32_t* n_new, int32_t* seen, int weight_blocks,
                        cudaStream_t stream) {
  switch (gp) {
    case 1: return launch_paged<DH, BF16, 1>(tm, p, n_new, seen, weight_blocks, stream);
    case 2: return launch_paged<DH, BF16, 2>(tm, p, n_new, seen, weight_blocks, stream);
    case 4: return launch_paged<DH, BF16, 4>(tm, p, n_new, seen, weight_blocks, stream);
    case 8: return launch_paged<DH, BF16, 8>(tm, p, n_new, seen, weight_blocks, stream);
    default: return launch_paged<DH, BF16, 16>(tm, p, n_new, seen, weight_blocks, stream);
  }
}

}  // namespace we

extern "C" size_t we_b200_paged_attn_workspace_bytes(const we_b200_paged_geom* g, int32_t Hq, int uses) {
  we::PagedPlan plan;
  if (g == nullptr || we::check_paged_geom(*g) != WE_B200_OK || Hq < 1 || Hq % g->Hkv != 0) return 0;
  return we::paged_plan(*g, Hq, (uses & WE_B200_USES_WEIGHTS) != 0, (uses & WE_B200_USES_N_NEW) != 0, &plan) == WE_B200_OK ? plan.bytes : 0;
}

extern "C" int we_b200_paged_attn(const we_b200_paged_attn_args* a, int32_t* status, void* stream) {
  using namespace we;
  if (a == nullptr) return WE_B200_E_NULL;
  const we_b200_paged_geom& g = a->geom;
  int rc = check_paged_geom(g);
  if (rc != WE_B200_OK) return rc;
  if (!a->q || !a->out || !a->kv || !a->table || !a->lens) return WE_B200_E_NULL;
  if (a->Hq < 1 || a->Hq % g.Hkv != 0) return WE_B200_E_SHAPE;
  if (a->Hq > 65535) return WE_B200_E_LIMIT;
  for (int i = 0; i < 2; ++i) {
    if (a->q_strides[i] < 0 || a->out_strides[i] < 0) return WE_B200_E_SHAPE;
    if ((a->q_strides[i] | a->out_strides[i]) & 7) return WE_B200_E_ALIGN;
  }
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->kv) || !aligned16(a->weights)) return WE_B200_E_ALIGN;
  PagedPlan plan;
  if ((rc = paged_plan(g, a->Hq, a->weights != nullptr, a->n_new != nullptr, &plan)) != WE_B200_OK) return rc;
  if (plan.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < plan.bytes)) return WE_B200_E_WORKSPACE;
  if (!aligned16(a->workspace)) return WE_B200_E_ALIGN;
  PagedAttnParams p;
  p.v = paged_view(g, a->table, status);
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  for (int i = 0; i < 2; ++i) p.qs[i] = a->q_strides[i], p.os[i] = a->out_strides[i];
  p.lens = a->lens;
  p.weights = a->weights;
  p.lse = a->lse;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.ws_prefix = reinterpret_cast<int32_t*>(ws);
  p.ws_ml = reinterpret_cast<float2*>(ws + plan.off_ml);
  p.ws_o = reinterpret_cast<float*>(ws + plan.off_o);
  p.ws_lse = reinterpret_cast<float*>(ws + plan.off_lse);
  p.ws_x = reinterpret_cast<float*>(ws + plan.off_x);
  p.x_stride = plan.cap;
  p.Hq = a->Hq;
  p.group = a->Hq / g.Hkv;
  p.chunks = plan.chunks;
  p.units = plan.units;
  p.grid = plan.grid;
  p.gran_shift = plan.gran_shift;
  p.whole = plan.whole;
  p.min_share = plan.min_share;
  p.scale_log2 = (a->scale > 0.f ? a->scale : 1.0f / sqrtf(static_cast<float>(g.Dh))) * 1.4426950408889634f;
  p.dynamic = plan.dynamic;
  // join: a CTA per head to join, or a warp where those would not fit at once, and a CTA per 1024 tokens of a kv
  // head to give them their weights
  const int64_t items = static_cast<int64_t>(plan.units) * (p.group < kMaxGroup ? p.group : kMaxGroup);
  const int sms = sm_count();
  p.out_by_warp = items > 2 * sms;
  const int64_t out_blocks = p.out_by_warp ? (items + kJoinThreads / 32 - 1) / (kJoinThreads / 32) : items;
  p.out_blocks = static_cast<int>(out_blocks < 2 * sms ? out_blocks : (p.out_by_warp ? sms : 2 * sms));
  const int64_t blocks = static_cast<int64_t>(plan.units / plan.chunks) * ((plan.cap + kJoinTokens - 1) / kJoinTokens);
  const int weight_blocks = p.weights != nullptr ? static_cast<int>(blocks < 16 * sms ? blocks : 16 * sms) : 0;
  int32_t* seen = reinterpret_cast<int32_t*>(ws + plan.off_seen);
  CUtensorMap tm;
  if ((rc = paged_map(&tm, a->kv, g, 1 << plan.gran_shift, &p)) != WE_B200_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (g.Dh == 128)
    return g.dtype == WE_B200_BF16 ? launch_group<128, true>(plan.gp, tm, p, a->n_new, seen, weight_blocks, s)
                                   : launch_group<128, false>(plan.gp, tm, p, a->n_new, seen, weight_blocks, s);
  return g.dtype == WE_B200_BF16 ? launch_group<64, true>(plan.gp, tm, p, a->n_new, seen, weight_blocks, s)
                                 : launch_group<64, false>(plan.gp, tm, p, a->n_new, seen, weight_blocks, s);
}
