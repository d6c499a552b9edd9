// Append to the paged KV cache, without and with a budget (sm_100a).
//
// Both give every (session, kv head) to a thread-block cluster of 1 to 8 CTAs, which alone reads and writes its counts,
// so they can be updated in place.  The append is a copy of rows: 16 bytes per thread and plane.
//
// Under a budget the cluster first finds the key of the last token to keep: weights are mapped to unsigned numbers of
// the same order (shielded tokens above all) and the keep-th largest is found digit by digit, each CTA counting the
// digits of its slice of the candidates and adding up the other CTAs' counts through cluster shared memory.  Weights and
// positions are read once: the keys stay in registers (those of longer slices are read again for every digit).  Then
// each CTA lists, in the order of the indexes, the holes of its slice (indexes below the budget that are given up) and
// the movers (kept ones behind it), and the j-th mover goes to the j-th hole: as many rows are copied as tokens leave,
// not as many as stay.  Reading is a matter of 1 to 3 us; what bounds the kernel is the chain of its phases (11 to
// 20 us): counts -> table -> keys -> two or three digits -> lists -> table -> rows, with a barrier or two in each.
#include "paged.cuh"

namespace we {

constexpr int kAppendThreads = 256;
constexpr int kMaxCluster = 8;
// Candidates a CTA deals with before its (session, head) gets a cluster: a barrier of the cluster and the counts read
// through it cost 1 to 2 us a digit, 4096 more candidates in one CTA less (16 heads of 4097: 11.2 us in one CTA, 14.6
// in two; 16 heads of 17001: 18.3 us in four CTAs, 31.9 in eight, which do not all find room at once).
constexpr int kEvictPerCta = 8192;

struct PagedAppendParams {
  PagedView v;
  const uint16_t* k_new;
  const uint16_t* v_new;
  int64_t ks[3], vs[3], wns[3];
  uint16_t* kv;
  float* weights;
  int32_t* positions;
  const int32_t* lens;
  const int32_t* next_pos;
  int32_t* lens_out;
  int32_t* next_pos_out;
  const int32_t* n_new;
  const float* w_new;
  int32_t* ws;           // lists of slices that do not fit in shared memory
  int64_t ws_stride;     // entries of one list of one CTA
  int64_t ws_chunk;      // entries of everything of one CTA
  int32_t T, keep, sink, recent;
  int32_t vec_shift;     // log2 of 16-byte vectors per row
  int32_t cluster;       // CTAs per (session, head)
  int32_t fit;           // entries of a list that fit in shared memory
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// All threads of the (session, head).
__device__ __forceinline__ void unit_sync(const PagedAppendParams& p) {
  if (p.cluster == 1) __syncthreads();
  else cluster_sync();
}
// The address of CTA `rank`'s copy of a shared variable, for ordinary loads.
template <class T>
__device__ __forceinline__ T* of_rank(T* mine, int rank) {
  uint64_t r;
  asm("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(reinterpret_cast<uint64_t>(mine)), "r"(rank));
  return reinterpret_cast<T*>(r);
}

__device__ __forceinline__ int new_count(const PagedAppendParams& p, int s) {
  if (p.n_new == nullptr) return p.T;
  const int n = p.n_new[s];
  if (n < 0 || n > p.T) {
    paged_report(p.v);
    return n < 0 ? 0 : p.T;
  }
  return n;
}

__device__ __forceinline__ int64_t meta_index(const PagedAppendParams& p, int pg, int h, int row) {
  return ((static_cast<int64_t>(pg) * p.v.Hkv + h) << p.v.page_shift) + row;
}
__device__ __forceinline__ float new_weight(const PagedAppendParams& p, int s, int h, int t) {
  return p.w_new != nullptr ? p.w_new[s * p.wns[0] + h * p.wns[1] + t * p.wns[2]] : 0.f;
}

// How many of `want` tokens from slot `first` on (all of them within the table) can be held: up to the first one for which
// the table names no page.  Called by all threads of the CTA, with the same arguments; so is the answer.  Up to 32 pages
// are looked up by every warp for itself, one load; more by the CTA together.
__device__ __forceinline__ int with_a_page(const PagedView& v, int s, int first, int want, int* s_first_bad) {
  if (want <= 0) return 0;
  const int32_t* row = v.table + s * v.table_stride;
  const int b0 = first >> v.page_shift, b1 = (first + want - 1) >> v.page_shift, lane = threadIdx.x & 31;
  int bad = 0x7FFFFFFF;
  if (b1 - b0 < 32) {
    const int pg = b0 + lane <= b1 ? row[b0 + lane] : 0;
    const uint32_t none = __ballot_sync(0xffffffffu, pg < 0 || pg >= v.n_pages);
    if (none != 0) bad = b0 + __ffs(none) - 1;
  } else {
#pragma unroll 4
    for (int b = b0 + static_cast<int>(threadIdx.x); b <= b1; b += static_cast<int>(blockDim.x)) {
      const int pg = row[b];
      if (pg < 0 || pg >= v.n_pages) bad = min(bad, b);
    }
    bad = __reduce_min_sync(0xffffffffu, bad);
    if (lane == 0) s_first_bad[threadIdx.x >> 5] = bad;
    __syncthreads();
    const int warps = static_cast<int>(blockDim.x) >> 5;
    bad = __reduce_min_sync(0xffffffffu, lane < warps ? s_first_bad[lane] : 0x7FFFFFFF);
  }
  return bad > b1 ? want : max((bad << v.page_shift) - first, 0);
}

// `items` moves of a token, one 16-byte vector of its K and of its V row per thread and step, kDepth steps at a time.
// where(e, &src, &dst): src >= len is the new token src - len, anything else a slot.
template <int kDepth, class F>
__device__ __forceinline__ void move_tokens(const PagedAppendParams& p, int s, int h, int len, int pos0, int items,
                                            int first, int step, F where) {
  const int64_t total = static_cast<int64_t>(items) << p.vec_shift;
  const int vecs = 1 << p.vec_shift;
  for (int64_t i0 = first; i0 < total; i0 += static_cast<int64_t>(step) * kDepth) {
    uint4 k[kDepth], v[kDepth];
    float w[kDepth];
    int32_t pos[kDepth], to[kDepth], row[kDepth];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int64_t i = i0 + static_cast<int64_t>(step) * d;
      to[d] = -1;
      if (i >= total) continue;
      const int c = static_cast<int>(i) & (vecs - 1);
      int src, dst;
      where(static_cast<int>(i >> p.vec_shift), &src, &dst);
      to[d] = paged_page(p.v, s, dst >> p.v.page_shift);
      row[d] = dst & (p.v.page - 1);
      if (src >= len) {
        const int t = src - len;
        k[d] = *reinterpret_cast<const uint4*>(p.k_new + s * p.ks[0] + h * p.ks[1] + t * p.ks[2] + 8 * c);
        v[d] = *reinterpret_cast<const uint4*>(p.v_new + s * p.vs[0] + h * p.vs[1] + t * p.vs[2] + 8 * c);
        if (c == 0) w[d] = new_weight(p, s, h, t);
        pos[d] = pos0 + t;
      } else {
        const int pg = paged_page(p.v, s, src >> p.v.page_shift), r = src & (p.v.page - 1);
        if (pg < 0) {
          to[d] = -1;
          continue;
        }
        const uint16_t* a = p.kv + pg * p.v.page_s + h * p.v.head_s + r * p.v.token_s + 8 * c;
        k[d] = *reinterpret_cast<const uint4*>(a);
        v[d] = *reinterpret_cast<const uint4*>(a + p.v.plane_s);
        if (c == 0) {
          const int64_t m = meta_index(p, pg, h, r);
          w[d] = p.weights[m];
          pos[d] = p.positions[m];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (to[d] < 0) continue;
      const int c = static_cast<int>(i0 + static_cast<int64_t>(step) * d) & (vecs - 1);
      uint16_t* b = p.kv + to[d] * p.v.page_s + h * p.v.head_s + row[d] * p.v.token_s + 8 * c;
      *reinterpret_cast<uint4*>(b) = k[d];
      *reinterpret_cast<uint4*>(b + p.v.plane_s) = v[d];
      if (c == 0) {
        const int64_t m = meta_index(p, to[d], h, row[d]);
        if (p.weights != nullptr) p.weights[m] = w[d];
        if (p.positions != nullptr) p.positions[m] = pos[d];
      }
    }
  }
}

// 16-byte vectors of K and of V that a thread has under way (and the pages of its next ones).  Prompts of 142000 tokens
// (146 MB read and written), without the look at the pages: 28.1 us with two and six CTAs on an SM, 30.3 with five, 34.8 with one
// vector and eight CTAs, 30.9 with four and four.  With it 29.2 us, 5.0 TB/s or 0.76 of the measured copy.  Bound by the
// latency of the table's and the rows' loads.
constexpr int kRows = 2;

//
// kStep: one token per session (64 threads).  Its page is looked up once, while its row is on its way, and thread 0 of the
// unit, which copies a part of it, knows whether it had one: 64 sessions x 16 heads take 2.3 us, 2.75 with the general look.
// The general kernel looks at the pages of all its tokens first (1 us of the prompts' 29.2): what lies behind the first
// missing page is not to be written, however many pages follow it.
template <bool kStep>
__global__ void __launch_bounds__(kStep ? 64 : kAppendThreads, kStep ? 16 : 6) paged_append_kernel(const PagedAppendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int unit = blockIdx.x / p.cluster, rank = blockIdx.x - unit * p.cluster;
  const int s = unit / p.v.Hkv, h = unit - s * p.v.Hkv;
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  const int n = new_count(p, s);
  const int room = (p.v.max_pages << p.v.page_shift) - len;
  __shared__ int s_first_bad[kAppendThreads / 32];
  // (a token that is dropped is not held: the count ends where the pages do)
  const int want = n < room ? n : room;
  int take = kStep ? want : with_a_page(p.v, s, len, want, s_first_bad);
  if (!kStep && take < n && threadIdx.x == 0) paged_report(p.v);
  const int32_t* table = p.v.table + s * p.v.table_stride;
  const int c = threadIdx.x & ((1 << p.vec_shift) - 1);
  const uint16_t* k_new = p.k_new + s * p.ks[0] + h * p.ks[1] + 8 * c;
  const uint16_t* v_new = p.v_new + s * p.vs[0] + h * p.vs[1] + 8 * c;
  uint16_t* kv = p.kv + h * p.v.head_s + 8 * c;
  const int step = (p.cluster * static_cast<int>(blockDim.x)) >> p.vec_shift;            // tokens
  int t0 = (rank * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) >> p.vec_shift;
  auto page_of = [&](int t) { return t < take ? table[(len + t) >> p.v.page_shift] : -1; };
  int pg[kRows];
#pragma unroll
  for (int d = 0; d < kRows; ++d) pg[d] = page_of(t0 + step * d);
  const int first_page = pg[0];
  for (; t0 < take; t0 += step * kRows) {
    uint4 k[kRows], v[kRows];
    int next[kRows];
#pragma unroll
    for (int d = 0; d < kRows; ++d) {
      const int t = t0 + step * d;
      if (t >= take) continue;
      k[d] = *reinterpret_cast<const uint4*>(k_new + t * p.ks[2]);
      v[d] = *reinterpret_cast<const uint4*>(v_new + t * p.vs[2]);
    }
#pragma unroll
    for (int d = 0; d < kRows; ++d) next[d] = page_of(t0 + step * (kRows + d));
#pragma unroll
    for (int d = 0; d < kRows; ++d) {
      const int t = t0 + step * d, row = (len + t) & (p.v.page - 1);
      // (the general kernel has looked already, but the address goes by this look)
      if (t >= take || static_cast<uint32_t>(pg[d]) >= static_cast<uint32_t>(p.v.n_pages)) continue;
      uint16_t* dst = kv + pg[d] * p.v.page_s + row * p.v.token_s;
      *reinterpret_cast<uint4*>(dst) = k[d];
      *reinterpret_cast<uint4*>(dst + p.v.plane_s) = v[d];
      if (c == 0) {
        const int64_t m = meta_index(p, pg[d], h, row);
        if (p.weights != nullptr) p.weights[m] = new_weight(p, s, h, t);
        if (p.positions != nullptr) p.positions[m] = pos0 + t;
      }
    }
#pragma unroll
    for (int d = 0; d < kRows; ++d) pg[d] = next[d];
  }
  unit_sync(p);                          // every thread has read the counts before they are replaced
  if (threadIdx.x == 0 && rank == 0) {
    if (kStep) {
      if (static_cast<uint32_t>(first_page) >= static_cast<uint32_t>(p.v.n_pages)) take = 0;
      if (take < n) paged_report(p.v);
    }
    p.lens_out[unit] = len + take;
    p.next_pos_out[unit] = pos0 + n;
  }
}

// ------------------------------------------------------------------ under a budget
// Weights as unsigned numbers of the same order: NaN above every number, shielded tokens above NaN, -0 equal to 0.
// A held slot for which the table names no page holds nothing that could be kept or moved, and nothing can be put there.
// Below the budget it stays where it is, above everything (it can be neither a hole nor a mover, and the tokens with the
// least weight go for want of a slot); behind the budget it comes below everything, and is given up: there are always
// `keep` others, as all indexes below the budget are candidates.
constexpr uint32_t kKeyNan = 0xFFFFFFFDu, kKeyShielded = 0xFFFFFFFEu, kKeyFixed = 0xFFFFFFFFu, kKeyNothing = 0u;
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kKeyNan;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// In one CTA: three digits of 11, 11 and 10 bits.  In a cluster four of 8: every CTA reads the counts of all others
// through cluster shared memory, and with 2048 of them that took 3 to 5 us a digit (65536 candidates in eight CTAs).
constexpr int kHistWords = 3 * 2048;
struct Digits {
  int bits, passes;
  __device__ __forceinline__ explicit Digits(int cluster) : bits(cluster == 1 ? 11 : 8), passes(cluster == 1 ? 3 : 4) {}
  __device__ __forceinline__ int shift(int pass) const { return max(32 - bits * (pass + 1), 0); }
  __device__ __forceinline__ uint32_t mask(int pass) const { return (1u << min(bits, 32 - bits * pass)) - 1u; }
};

// Sum of x over the threads before this one; *all gets the sum over the block.  (One copy for all its uses: a call of
// this kernel is a few microseconds, and fetching code that runs once is a part of that.)
template <int kThreads, class T>
__device__ __noinline__ T block_scan(T x, uint64_t* s_warp, T* all) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  T upto = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += y;
  }
  __syncthreads();                                       // (s_warp may still be read from the call before)
  if (lane == 31) s_warp[wid] = upto;
  __syncthreads();
  T w = lane < kWarps ? static_cast<T>(s_warp[lane]) : 0;
  if constexpr (sizeof(T) == 4) {
    *all = __reduce_add_sync(0xffffffffu, w);
    return upto - x + __reduce_add_sync(0xffffffffu, lane < wid ? w : 0);
  } else {
#pragma unroll
    for (int d = 1; d < kWarps; d <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    *all = __shfl_sync(0xffffffffu, w, kWarps - 1);
    const T before = __shfl_sync(0xffffffffu, w, wid > 0 ? wid - 1 : 0);
    return upto - x + (wid > 0 ? before : 0);
  }
}

// Candidates a thread holds in registers: five times four neighbours.  A slice of up to kThreads * 20 is read once;
// a longer one (a session that held much more than its budget) is read again for every pass, a round at a time.
constexpr int kGroups = 5;

template <int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 256 ? 4 : 1) paged_append_evict_kernel(const PagedAppendParams p) {
  constexpr int kRound = kThreads * 4 * kGroups, kBatch = kThreads == 256 ? 2 : 3;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(16) int32_t s_lists_mem[];  // holes [fit], movers [fit], bits [fit / 32] twice
  __shared__ __align__(16) uint32_t s_hist[kHistWords];
  __shared__ uint64_t s_warp[32];
  __shared__ uint32_t s_found[3];                      // digit, how many of it are kept, how many there are
  __shared__ int s_equal, s_lists[3];                  // of this CTA: equal keys; holes, movers, new ones in place
  __shared__ int s_base[3][kMaxCluster + 1];
  const int unit = blockIdx.x / p.cluster, rank = blockIdx.x - unit * p.cluster;
  const int s = unit / p.v.Hkv, h = unit - s * p.v.Hkv;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const Digits digits(p.cluster);
  const int bins = 1 << digits.bits;
  for (int b = tid; b < digits.passes * bins / 4; b += kThreads) reinterpret_cast<uint4*>(s_hist)[b] = make_uint4(0u, 0u, 0u, 0u);
  // One CTA starts at the first token whatever the counts are: its pages are looked up while they are on their way.
  int early[kGroups];
  auto look_up = [&]() {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int b = (4 * (g * kThreads + tid)) >> p.v.page_shift;
      early[g] = p.cluster == 1 && b < p.v.max_pages ? p.v.table[s * p.v.table_stride + b] : 0;
    }
  };
  look_up();
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  int n = new_count(p, s);
  const int64_t end = static_cast<int64_t>(pos0) + n;
  __syncthreads();
  if (len < p.keep) {                                    // below the budget a token goes to the next slot, if it has a page
    const int have = with_a_page(p.v, s, len, min(n, p.keep - len), reinterpret_cast<int*>(s_warp));
    if (have < min(n, p.keep - len)) {                   // the rest is dropped
      n = have;
      if (tid == 0) paged_report(p.v);
    }
    look_up();                                           // (again: a session at its budget comes past here, in registers)
  }
  const int total = len + n;
  if (total <= p.keep) {
    move_tokens<2>(p, s, h, len, pos0, n, rank * kThreads + tid, p.cluster * kThreads,
                   [&](int e, int* src, int* dst) { *src = *dst = len + e; });
  } else {
    // ---- this CTA's slice of the candidates, in rounds; a thread has four neighbours at a time (they lie in one page)
    const int slice = ((total + p.cluster - 1) / p.cluster + 3) & ~3;
    const int lo = min(rank * slice, total), hi = min(lo + slice, total), mine = hi - lo;
    const int rounds = (mine + kRound - 1) / kRound;
    const bool fits = slice <= p.fit;
    auto key_of = [&](float w, int64_t pos) {
      return pos < p.sink || pos >= end - p.recent ? kKeyShielded : weight_key(w);
    };
    uint32_t key[kGroups][4];                            // (those behind the slice: unused)
    auto first_of = [&](int round, int g) { return lo + round * kRound + 4 * (g * kThreads + tid); };
    auto load = [&](int round) {
      int pg[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int i = first_of(round, g);
        if (p.cluster == 1 && round == 0) pg[g] = early[g];
        else pg[g] = i < hi && i < len ? p.v.table[s * p.v.table_stride + (i >> p.v.page_shift)] : 0;
      }
#pragma unroll
      for (int g0 = 0; g0 < kGroups; g0 += kBatch) {
        float4 w[kBatch];
        int4 pos[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch && g0 + b < kGroups; ++b) {
          const int g = g0 + b, i = first_of(round, g);
          w[b] = make_float4(0.f, 0.f, 0.f, 0.f);
          pos[b] = make_int4(0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF);
          if (i >= hi || i >= len) continue;
          if (pg[g] < 0 || pg[g] >= p.v.n_pages) {
            paged_report(p.v);
            continue;
          }
          const int64_t m = meta_index(p, pg[g], h, i & (p.v.page - 1));
          w[b] = *reinterpret_cast<const float4*>(p.weights + m);
          pos[b] = *reinterpret_cast<const int4*>(p.positions + m);
        }
#pragma unroll
        for (int b = 0; b < kBatch && g0 + b < kGroups; ++b) {
          const int g = g0 + b, i = first_of(round, g);
          if (i >= hi) continue;
          key[g][0] = key_of(w[b].x, pos[b].x);
          key[g][1] = key_of(w[b].y, pos[b].y);
          key[g][2] = key_of(w[b].z, pos[b].z);
          key[g][3] = key_of(w[b].w, pos[b].w);
          if (i < len && (pg[g] < 0 || pg[g] >= p.v.n_pages)) {
#pragma unroll
            for (int u = 0; u < 4; ++u) key[g][u] = i + u < p.keep ? kKeyFixed : kKeyNothing;
          }
          if (i + 3 < len) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i + u >= len)
              key[g][u] = i + u < hi ? key_of(new_weight(p, s, h, i + u - len), static_cast<int64_t>(pos0) + (i + u - len)) : 0u;
        }
      }
    };
    if (rounds == 1) load(0);
    // ---- the key of the last one kept (its leading digits, as far as they decide), how many of that key are kept
    uint32_t prefix = 0, mask = 0, need = static_cast<uint32_t>(p.keep), equals = 0;
#pragma unroll 1
    for (int pass = 0; pass < digits.passes; ++pass) {
      const int shift = digits.shift(pass);
      const uint32_t low = digits.mask(pass);
      uint32_t* hist = s_hist + pass * bins;
      for (int round = 0; round < rounds; ++round) {
        if (rounds > 1) load(round);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int i = first_of(round, g);
          if (i >= hi) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (i + u < hi && (key[g][u] & mask) == prefix) atomicAdd(&hist[(key[g][u] >> shift) & low], 1u);
        }
      }
      unit_sync(p);
      // the largest digits to thread 0; a scan over the block finds the one with the keep-th
      constexpr int kOwn = 2048 / kThreads;
      uint32_t c[kOwn], sum = 0;
      int bin0 = 0;
      if (p.cluster == 1) {
        bin0 = 2048 - kOwn * (tid + 1);
#pragma unroll
        for (int b = 0; b < kOwn; b += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(hist + bin0 + b);
          c[b] = x.x;
          c[b + 1] = x.y;
          c[b + 2] = x.z;
          c[b + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int b = 0; b < kOwn; ++b) c[b] = 0;
        if (tid < 256) {
          bin0 = 255 - tid;
#pragma unroll
          for (int r = 0; r < kMaxCluster; ++r)
            if (r < p.cluster) c[0] += *of_rank(hist + bin0, r);
        }
      }
#pragma unroll
      for (int b = 0; b < kOwn; ++b) sum += c[b];
      uint32_t all;
      const uint32_t before = block_scan<kThreads, uint32_t>(sum, s_warp, &all);
      if (before < need && before + sum >= need) {
        uint32_t at = before;
        bool found = false;
#pragma unroll
        for (int b = kOwn - 1; b >= 0; --b) {
          if (!found && at + c[b] >= need) {
            found = true;
            s_found[0] = bin0 + b;
            s_found[1] = need - at;
            s_found[2] = c[b];
          }
          at += c[b];
        }
      }
      __syncthreads();
      prefix |= s_found[0] << shift;
      mask |= low << shift;
      need = s_found[1];
      equals = s_found[2];
      if (equals == need) break;                         // everything with these digits stays
    }
    // ---- one bit per candidate: kept outright, or one of the equal keys of which only some are kept
    int32_t* holes = fits ? s_lists_mem : p.ws + blockIdx.x * p.ws_chunk;
    const int64_t room = fits ? p.fit : p.ws_stride;
    int32_t* movers = holes + room;
    uint32_t* bits_kept = reinterpret_cast<uint32_t*>(movers + room);
    uint32_t* bits_equal = bits_kept + ((room + 31) >> 5);
    const bool ties = equals != need;
    const int words = (mine + 31) >> 5;
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load(round);
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int i = first_of(round, g);
        if (i - 4 * lane >= hi) continue;                // (the same for the whole warp)
        uint32_t more = 0, same = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t k = key[g][u] & mask;
          more |= i + u < hi && k > prefix ? 1u << u : 0u;
          same |= i + u < hi && k == prefix ? 1u << u : 0u;
        }
        if (!ties) more |= same;
        const int at = 4 * (lane & 7);                   // eight lanes make a word
        more <<= at;
        same <<= at;
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
          more |= __shfl_xor_sync(0xffffffffu, more, d);
          same |= __shfl_xor_sync(0xffffffffu, same, d);
        }
        const int w = (i - lo) >> 5;
        if ((lane & 7) == 0 && w < words) {
          bits_kept[w] = more;
          bits_equal[w] = same;
        }
      }
    }
    __syncthreads();
    // a thread goes on with `per` neighbouring words
    const int per = (words + kThreads - 1) / kThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    if (ties) {                                          // the first `need` of them, in the order of the indexes
      uint32_t cnt = 0, all;
      for (int w = w0; w < w1; ++w) cnt += __popc(bits_equal[w]);
      int64_t left = need;
      left -= block_scan<kThreads, uint32_t>(cnt, s_warp, &all);
      if (p.cluster > 1) {
        if (tid == 0) s_equal = static_cast<int>(all);
        unit_sync(p);
        left -= __reduce_add_sync(0xffffffffu, lane < rank ? *of_rank(&s_equal, lane) : 0);
      }
      for (int w = w0; w < w1; ++w) {
        uint32_t e = bits_equal[w];
        const int have = __popc(e);
        for (int drop = have - static_cast<int>(left < 0 ? 0 : left < have ? left : have); drop > 0; --drop)
          e &= ~(0x80000000u >> __clz(e));
        bits_kept[w] |= e;
        left -= have;
      }
    }
    // ---- holes, movers and new tokens that lie below the budget already, listed in the order of the indexes
    auto bits_from = [&](int base, int from) {           // bits of the word at `base` whose index is >= from
      const int d = from - base;
      return d <= 0 ? 0xFFFFFFFFu : d >= 32 ? 0u : 0xFFFFFFFFu << d;
    };
    auto split = [&](int w, uint32_t* hole, uint32_t* mover, uint32_t* stay) {
      const int base = lo + 32 * w;
      const uint32_t kept = bits_kept[w], beyond = bits_from(base, p.keep);
      *hole = ~kept & ~bits_from(base, hi) & ~beyond;
      *mover = kept & beyond;
      *stay = kept & ~beyond & bits_from(base, len);
    };
    uint64_t sums = 0, all;                              // 21 bits each
    for (int w = w0; w < w1; ++w) {
      uint32_t b[3];
      split(w, &b[0], &b[1], &b[2]);
      sums += static_cast<uint64_t>(__popc(b[0])) | (static_cast<uint64_t>(__popc(b[1])) << 21) |
              (static_cast<uint64_t>(__popc(b[2])) << 42);
    }
    const uint64_t at = block_scan<kThreads, uint64_t>(sums, s_warp, &all);
    int64_t at_h = at & 0x1FFFFF, at_m = (at >> 21) & 0x1FFFFF, at_s = at >> 42;
    if (tid == 0) {
      s_lists[0] = static_cast<int>(all & 0x1FFFFF);
      s_lists[1] = static_cast<int>((all >> 21) & 0x1FFFFF);
      s_lists[2] = static_cast<int>(all >> 42);
    }
    for (int w = w0; sums != 0 && w < w1; ++w) {
      uint32_t b[3];
      split(w, &b[0], &b[1], &b[2]);
      const int base = lo + 32 * w;
      for (; b[0] != 0; b[0] &= b[0] - 1) holes[at_h++] = base + __ffs(b[0]) - 1;
      for (; b[1] != 0; b[1] &= b[1] - 1) movers[at_m++] = base + __ffs(b[1]) - 1;
      for (; b[2] != 0; b[2] &= b[2] - 1) holes[room - 1 - at_s++] = base + __ffs(b[2]) - 1;     // from the far end
    }
    unit_sync(p);
    if (wid < 3) {                                       // where each CTA's entries begin
      const int x = lane < p.cluster ? (p.cluster == 1 ? s_lists[wid] : *of_rank(&s_lists[wid], lane)) : 0;
      int upto = x;
      for (int d = 1; d < kMaxCluster; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      if (lane < kMaxCluster) s_base[wid][lane + 1] = upto;
      if (lane == 0) s_base[wid][0] = 0;
    }
    __syncthreads();
    // ---- the moves, spread over the cluster
    const int moves = s_base[1][kMaxCluster], stays = s_base[2][kMaxCluster];
    auto entry = [&](int q, int32_t* list, int64_t j) {
      int r = 0;
      while (r + 1 < p.cluster && j >= s_base[q][r + 1]) ++r;
      const int64_t k = q == 2 ? room - 1 - (j - s_base[q][r]) : j - s_base[q][r];
      if (fits) return p.cluster == 1 ? list[k] : of_rank(list, r)[k];
      return list[static_cast<int64_t>(r - rank) * p.ws_chunk + k];
    };
    move_tokens<2>(p, s, h, len, pos0, moves + stays, rank * kThreads + tid, p.cluster * kThreads,
                   [&](int e, int* src, int* dst) {
                     if (e < moves) {
                       *src = entry(1, movers, e);
                       *dst = entry(0, holes, e);
                     } else {
                       *src = *dst = entry(2, holes, e - moves);
                     }
                   });
  }
  unit_sync(p);                          // the counts have been read, and nobody needs this CTA's lists any more
  if (tid == 0 && rank == 0) {
    p.lens_out[unit] = total < p.keep ? total : p.keep;
    p.next_pos_out[unit] = static_cast<int32_t>(end);
  }
}

static int fill(const we_b200_paged_append_args* a, int32_t* status, PagedAppendParams* p) {
  if (a == nullptr) return WE_B200_E_NULL;
  const we_b200_paged_geom& g = a->geom;
  int rc = check_paged_geom(g);
  if (rc != WE_B200_OK) return rc;
  if ((a->T != 0 && (!a->k_new || !a->v_new)) || !a->kv || !a->table || !a->lens || !a->next_pos || !a->lens_out || !a->next_pos_out)
    return WE_B200_E_NULL;
  if (a->w_new != nullptr && a->weights == nullptr) return WE_B200_E_NULL;
  if (a->T < 0) return WE_B200_E_SHAPE;
  if (a->T > (1 << 26)) return WE_B200_E_LIMIT;
  if ((rc = check_strides(a->k_strides, 2)) != WE_B200_OK) return rc;
  if ((rc = check_strides(a->v_strides, 2)) != WE_B200_OK) return rc;
  for (int i = 0; i < 3; ++i)
    if (a->w_new != nullptr && a->w_strides[i] < 0) return WE_B200_E_SHAPE;
  if (!aligned16(a->k_new) || !aligned16(a->v_new) || !aligned16(a->kv)) return WE_B200_E_ALIGN;
  p->v = paged_view(g, a->table, status);
  p->k_new = static_cast<const uint16_t*>(a->k_new);
  p->v_new = static_cast<const uint16_t*>(a->v_new);
  for (int i = 0; i < 3; ++i) {
    p->ks[i] = a->k_strides[i];
    p->vs[i] = a->v_strides[i];
    p->wns[i] = a->w_strides[i];
  }
  p->kv = static_cast<uint16_t*>(a->kv);
  p->weights = a->weights;
  p->positions = a->positions;
  p->lens = a->lens;
  p->next_pos = a->next_pos;
  p->lens_out = a->lens_out;
  p->next_pos_out = a->next_pos_out;
  p->n_new = a->n_new;
  p->w_new = a->w_new;
  p->ws = nullptr;
  p->ws_stride = p->ws_chunk = 0;
  p->cluster = 1;
  p->fit = 0;
  p->T = a->T;
  p->keep = p->sink = p->recent = 0;
  p->vec_shift = g.Dh == 128 ? 4 : 3;
  return WE_B200_OK;
}

static int launch(void (*kernel)(PagedAppendParams), const PagedAppendParams& p, int threads, int smem,
                  cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.v.S) * p.v.Hkv * p.cluster, 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  if (e != cudaSuccess) return static_cast<int>(e);
  const cudaError_t e2 = cudaGetLastError();
  return e2 == cudaSuccess ? WE_B200_OK : static_cast<int>(e2);
}

// CTAs per (session, head): as few as give each at most `per_cta` of the work, unless there are so many sessions and
// heads that the SMs are busy with fewer.
static int cluster_for(int64_t units, int64_t work, int64_t per_cta, int64_t most_ctas) {
  int c = 1;
  while (c < kMaxCluster && work > per_cta * c && units * c * 2 <= most_ctas) c *= 2;
  return c;
}

struct EvictPlan {
  int threads, cluster, fit;
  int64_t list, chunk;     // entries of a list in the workspace (0: never needed) and of all a CTA has there
  size_t bytes;
};
constexpr int kMaxFit = 20480;
constexpr int evict_smem(int fit) { return 8 * fit + 2 * ((fit + 31) / 32) * 4; }
static_assert(evict_smem(kMaxFit) + kHistWords * 4 + 1024 <= 227 * 1024, "shared memory");

// (the counts are on the device: a session that holds more than its budget says, once, is found there)
static EvictPlan evict_plan(const we_b200_paged_geom& g, int32_t T, int32_t keep) {
  EvictPlan r;
  const int64_t units = static_cast<int64_t>(g.S) * g.Hkv, usual = static_cast<int64_t>(keep) + T;
  // four CTAs of 256 threads fit on an SM, or one of 512 has it to itself (16 heads of 4097: 15.5 us with 256 threads,
  // 12.9 with 512, 13.6 with 1024, whose scans over the block take longer; 512 heads of 2064: 12.5 us, 16.4 with 512)
  r.threads = units > 2 * sm_count() ? 256 : 512;
  r.cluster = cluster_for(units, usual, kEvictPerCta, sm_count());
  // (to the end of the budget's last page: a table that has no more pages needs no lists in the workspace)
  const int64_t most = static_cast<int64_t>(g.max_pages) * g.page + T;
  const int64_t whole = (static_cast<int64_t>(keep) + g.page - 1) / g.page * g.page + T;
  const int64_t fit = ((whole + r.cluster - 1) / r.cluster + 3) & ~3ll;
  r.fit = static_cast<int>(fit < kMaxFit ? fit : kMaxFit);
  const int64_t slice = ((most + r.cluster - 1) / r.cluster + 3) & ~3ll;
  r.list = slice <= r.fit ? 0 : slice;
  r.chunk = 2 * r.list + 2 * ((r.list + 31) >> 5);
  r.bytes = static_cast<size_t>(units) * r.cluster * r.chunk * sizeof(int32_t);
  return r;
}

template <int kThreads>
static int launch_evict(const PagedAppendParams& p, cudaStream_t stream) {
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= kMaxDevices) return WE_B200_E_LIMIT;
  if (!done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(paged_append_evict_kernel<kThreads>, cudaFuncAttributeMaxDynamicSharedMemorySize, evict_smem(kMaxFit));
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return static_cast<int>(e);
    }
    done[dev].store(true, std::memory_order_release);
  }
  return launch(paged_append_evict_kernel<kThreads>, p, kThreads, evict_smem(p.fit), stream);
}

}  // namespace we

extern "C" int we_b200_paged_append(const we_b200_paged_append_args* a, int32_t* status, void* stream) {
  we::PagedAppendParams p;
  const int rc = we::fill(a, status, &p);
  if (rc != WE_B200_OK) return rc;
  p.cluster = we::cluster_for(static_cast<int64_t>(p.v.S) * p.v.Hkv, static_cast<int64_t>(p.T) << p.vec_shift,
                              4 * we::kAppendThreads, 8 * we::sm_count());
  // (a decoding step has one row per plane, session and head: 16 threads of work)
  const int threads = (p.T << p.vec_shift) <= 64 ? 64 : we::kAppendThreads;
  return we::launch(p.T == 1 ? we::paged_append_kernel<true> : we::paged_append_kernel<false>, p, threads, 0,
                    static_cast<cudaStream_t>(stream));
}

extern "C" size_t we_b200_paged_evict_workspace_bytes(const we_b200_paged_geom* g, int32_t T, int32_t keep) {
  if (g == nullptr || we::check_paged_geom(*g) != WE_B200_OK || T < 0 || keep < 1) return 0;
  return we::evict_plan(*g, T, keep).bytes;
}

extern "C" int we_b200_paged_append_evict(const we_b200_paged_append_args* a, int32_t* status, void* stream) {
  we::PagedAppendParams p;
  const int rc = we::fill(a, status, &p);
  if (rc != WE_B200_OK) return rc;
  if (a->weights == nullptr || a->positions == nullptr) return WE_B200_E_NULL;
  if (a->keep < 1 || a->sink < 0 || a->recent < 0) return WE_B200_E_SHAPE;
  if (static_cast<int64_t>(a->sink) + a->recent > a->keep) return WE_B200_E_SHAPE;
  if (static_cast<int64_t>(a->geom.max_pages) * a->geom.page < a->keep) return WE_B200_E_SHAPE;
  // (a CTA counts its holes and movers in 21 bits)
  if (static_cast<int64_t>(a->geom.max_pages) * a->geom.page + a->T >= (1 << 21)) return WE_B200_E_LIMIT;
  const we::EvictPlan plan = we::evict_plan(a->geom, a->T, a->keep);
  if (plan.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < plan.bytes)) return WE_B200_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 3u) return WE_B200_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(a->weights) | reinterpret_cast<uintptr_t>(a->positions)) & 15u) return WE_B200_E_ALIGN;
  p.ws = static_cast<int32_t*>(a->workspace);
  p.ws_stride = plan.list;
  p.ws_chunk = plan.chunk;
  p.keep = a->keep;
  p.sink = a->sink;
  p.recent = a->recent;
  p.cluster = plan.cluster;
  p.fit = plan.fit;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return plan.threads == 256 ? we::launch_evict<256>(p, st) : we::launch_evict<512>(p, st);
}
