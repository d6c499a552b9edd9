// Append to the paged KV cache, without and with a budget (sm_100a).
//
// Both give every (session, kv head) to a thread-block cluster of 1 to 8 CTAs, which alone reads and writes its counts,
// so they can be updated in place.  The append is a copy of rows: 16 bytes per thread and plane, all loads of a thread
// under way before the first store.
//
// Under a budget the cluster first finds the key of the last token to keep: weights are mapped to unsigned numbers of
// the same order (shielded tokens above all) and the keep-th largest is found eight bits at a time, each CTA counting
// the digits of its slice of the candidates and adding up the other CTAs' counts through cluster shared memory.  One
// pass over weights and positions in global memory; the later passes read keys from shared memory (slices that do not
// fit are recomputed from global memory).  Then each CTA lists, in the order of the indexes, the holes of its slice
// (indexes below the budget that are given up) and the movers (kept ones behind it), and the j-th mover goes to the
// j-th hole: as many rows are copied as tokens leave, not as many as stay.
#include "paged.cuh"

namespace we {

constexpr int kAppendThreads = 256;
constexpr int kMaxCluster = 8;

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
  int32_t T, keep, sink, recent;
  int32_t vec_shift;     // log2 of 16-byte vectors per row
  int32_t cluster;       // CTAs per (session, head)
  int32_t fit;           // keys of a slice that fit in shared memory
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

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int unit = blockIdx.x / p.cluster, rank = blockIdx.x - unit * p.cluster;
  const int s = unit / p.v.Hkv, h = unit - s * p.v.Hkv;
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  const int n = new_count(p, s);
  const int room = (p.v.max_pages << p.v.page_shift) - len;
  const int take = n < room ? n : room;
  if (take < n && threadIdx.x == 0) paged_report(p.v);
  move_tokens<4>(p, s, h, len, pos0, take, rank * kAppendThreads + threadIdx.x, p.cluster * kAppendThreads,
                 [&](int e, int* src, int* dst) { *src = *dst = len + e; });
  unit_sync(p);                          // every thread has read the counts before they are replaced
  if (threadIdx.x == 0 && rank == 0) {
    p.lens_out[unit] = len + take;
    p.next_pos_out[unit] = pos0 + n;
  }
}

// ------------------------------------------------------------------ under a budget
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;

// Weights as unsigned numbers of the same order: NaN above every number, shielded tokens above NaN, -0 equal to 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__global__ void __launch_bounds__(kEvictThreads) paged_append_evict_kernel(const PagedAppendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint32_t s_keys[];                 // [fit] keys, [fit] holes, [fit] movers
  __shared__ uint32_t s_hist[4][256], s_bins[256];
  __shared__ int s_count[3][kEvictWarps];
  __shared__ int s_equal, s_lists[3];                  // of this CTA: equal keys; holes, movers, new ones in place
  __shared__ int s_base[3][kMaxCluster + 1];
  const int unit = blockIdx.x / p.cluster, rank = blockIdx.x - unit * p.cluster;
  const int s = unit / p.v.Hkv, h = unit - s * p.v.Hkv;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  for (int b = tid; b < 4 * 256; b += kEvictThreads) s_hist[0][b] = 0;
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  const int n = new_count(p, s);
  const int total = len + n;
  const int64_t end = static_cast<int64_t>(pos0) + n;
  __syncthreads();
  if (total <= p.keep) {
    move_tokens<2>(p, s, h, len, pos0, n, rank * kEvictThreads + tid, p.cluster * kEvictThreads,
                   [&](int e, int* src, int* dst) { *src = *dst = len + e; });
  } else {
    // ---- keys of this CTA's slice, four neighbours at a time (they lie in one page), with the first digit's counts
    const int slice = ((total + p.cluster - 1) / p.cluster + 3) & ~3;
    const int lo = min(rank * slice, total), hi = min(lo + slice, total), mine = hi - lo;
    const bool fits = slice <= p.fit;
    auto key_of = [&](float w, int64_t pos) {
      return pos < p.sink || pos >= end - p.recent ? 0xFFFFFFFFu : weight_key(w);
    };
    auto key_at = [&](int i) -> uint32_t {              // one candidate, from global memory
      if (i >= len) return key_of(new_weight(p, s, h, i - len), static_cast<int64_t>(pos0) + (i - len));
      const int pg = paged_page(p.v, s, i >> p.v.page_shift);
      if (pg < 0) return 0u;
      const int64_t m = meta_index(p, pg, h, i & (p.v.page - 1));
      return key_of(p.weights[m], p.positions[m]);
    };
    auto key = [&](int i) { return fits ? s_keys[i - lo] : key_at(i); };
    constexpr int kDepth = 4;
    for (int i0 = lo + 4 * tid; i0 < hi; i0 += 4 * kEvictThreads * kDepth) {
      int pg[kDepth];
      float4 w[kDepth];
      int4 pos[kDepth];
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int i = i0 + 4 * kEvictThreads * d;
        pg[d] = i < hi && i + 3 < len ? paged_page(p.v, s, i >> p.v.page_shift) : -1;
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        if (pg[d] < 0) continue;
        const int64_t m = meta_index(p, pg[d], h, (i0 + 4 * kEvictThreads * d) & (p.v.page - 1));
        w[d] = *reinterpret_cast<const float4*>(p.weights + m);
        pos[d] = *reinterpret_cast<const int4*>(p.positions + m);
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        const int i = i0 + 4 * kEvictThreads * d;
        if (i >= hi) continue;
        uint32_t k[4];
        if (pg[d] >= 0) {
          k[0] = key_of(w[d].x, pos[d].x);
          k[1] = key_of(w[d].y, pos[d].y);
          k[2] = key_of(w[d].z, pos[d].z);
          k[3] = key_of(w[d].w, pos[d].w);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) k[u] = i + u < hi ? key_at(i + u) : 0u;
        }
        if (fits) *reinterpret_cast<uint4*>(s_keys + (i - lo)) = make_uint4(k[0], k[1], k[2], k[3]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u < hi) atomicAdd(&s_hist[0][k[u] >> 24], 1u);
      }
    }
    // ---- the key of the last one kept (its leading digits, as far as they decide), how many of that key are kept
    uint32_t prefix = 0, mask = 0, need = static_cast<uint32_t>(p.keep), equals = 0;
    for (int pass = 0; pass < 4; ++pass) {
      const int shift = 24 - 8 * pass;
      if (pass > 0) {
        for (int i = lo + tid; i < hi; i += kEvictThreads) {
          const uint32_t k = key(i);
          if ((k & mask) == prefix) atomicAdd(&s_hist[pass][(k >> shift) & 255u], 1u);
        }
      }
      unit_sync(p);
      if (p.cluster > 1) {
        if (tid < 256) {
          uint32_t x = 0;
          for (int r = 0; r < p.cluster; ++r) x += of_rank(&s_hist[pass][tid], r)[0];
          s_bins[tid] = x;
        }
        __syncthreads();
      }
      // every warp finds the digit for itself: eight bins per lane, the largest digits in lane 0
      const uint32_t* bins = p.cluster > 1 ? s_bins : s_hist[pass];
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        c[b] = bins[255 - 8 * lane - b];
        sum += c[b];
      }
      uint32_t before = sum;
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += y;
      }
      before -= sum;
      const uint32_t who = __ballot_sync(0xffffffffu, before < need && before + sum >= need);
      uint32_t digit = 0, left = 0, same = 0;
      {
        uint32_t at = before;
        bool found = false;
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          if (!found && at + c[b] >= need) {
            found = true;
            digit = 255 - 8 * lane - b;
            left = need - at;
            same = c[b];
          }
          at += c[b];
        }
      }
      const int from = __ffs(who) - 1;
      digit = __shfl_sync(0xffffffffu, digit, from);
      need = __shfl_sync(0xffffffffu, left, from);
      equals = __shfl_sync(0xffffffffu, same, from);
      prefix |= digit << shift;
      mask |= 255u << shift;
      if (equals == need) break;                         // everything with these digits stays
      __syncthreads();                                   // (s_bins is read before the next pass writes it)
    }
    // ---- ranks among equal keys, where not all of them stay: in the order of the indexes
    const int sub = ((mine + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
    const int w_lo = min(lo + wid * sub, hi), w_hi = min(w_lo + sub, hi);
    const uint32_t below = (1u << lane) - 1u;
    uint32_t equal_base = 0;
    if (equals != need) {
      int cnt = 0;
      for (int i = w_lo; i < w_hi; i += 32)
        cnt += __popc(__ballot_sync(0xffffffffu, i + lane < w_hi && (key(i + lane) & mask) == prefix));
      if (lane == 0) s_count[0][wid] = cnt;
      __syncthreads();
      if (tid == 0) {
        int x = 0;
        for (int w = 0; w < kEvictWarps; ++w) x += s_count[0][w];
        s_equal = x;
      }
      unit_sync(p);
      for (int r = 0; r < rank; ++r) equal_base += *of_rank(&s_equal, r);
      for (int w = 0; w < wid; ++w) equal_base += s_count[0][w];
      __syncthreads();
    }
    // ---- holes, movers and new tokens that lie below the budget already: counted, then listed
    int32_t* holes = fits ? reinterpret_cast<int32_t*>(s_keys) + p.fit
                          : p.ws + (static_cast<int64_t>(blockIdx.x) * 2) * p.ws_stride;
    int32_t* movers = holes + (fits ? p.fit : p.ws_stride);
    const int64_t room = fits ? p.fit : p.ws_stride;
    int at[3] = {0, 0, 0};
    for (int round = 0; round < 2; ++round) {
      uint32_t rank_eq = equal_base;
      for (int i0 = w_lo; i0 < w_hi; i0 += 32) {
        const int i = i0 + lane;
        const bool in = i < w_hi;
        const uint32_t k = in ? key(i) & mask : 0u;
        const bool equal = in && k == prefix;
        bool kept = in && (k > prefix || equal);
        if (equals != need) {
          const uint32_t e = __ballot_sync(0xffffffffu, equal);
          if (equal && rank_eq + __popc(e & below) >= need) kept = false;
          rank_eq += __popc(e);
        }
        const bool hole = in && i < p.keep && !kept, mover = kept && i >= p.keep, stay = kept && i >= len && i < p.keep;
        const uint32_t b0 = __ballot_sync(0xffffffffu, hole), b1 = __ballot_sync(0xffffffffu, mover),
                       b2 = __ballot_sync(0xffffffffu, stay);
        if (round == 1) {
          if (hole) holes[at[0] + __popc(b0 & below)] = i;
          if (mover) movers[at[1] + __popc(b1 & below)] = i;
          if (stay) holes[room - 1 - (at[2] + __popc(b2 & below))] = i;      // from the far end
        }
        at[0] += __popc(b0);
        at[1] += __popc(b1);
        at[2] += __popc(b2);
      }
      if (round == 1) break;
      if (lane < 3) s_count[lane][wid] = lane == 0 ? at[0] : lane == 1 ? at[1] : at[2];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        int x = 0;
        for (int w = 0; w < wid; ++w) x += s_count[q][w];
        if (wid == kEvictWarps - 1 && lane == 0) s_lists[q] = x + at[q];
        at[q] = x;
      }
    }
    unit_sync(p);
    if (tid < 3) {
      int x = 0;
      for (int r = 0; r < p.cluster; ++r) {
        s_base[tid][r] = x;
        x += of_rank(&s_lists[tid], r)[0];
      }
      for (int r = p.cluster; r <= kMaxCluster; ++r) s_base[tid][r] = x;
    }
    __syncthreads();
    // ---- the moves, spread over the cluster
    const int moves = s_base[1][kMaxCluster], stays = s_base[2][kMaxCluster];
    auto entry = [&](int q, int32_t* list, int64_t j) {
      int r = 0;
      while (r + 1 < p.cluster && j >= s_base[q][r + 1]) ++r;
      const int64_t k = q == 2 ? room - 1 - (j - s_base[q][r]) : j - s_base[q][r];
      if (fits) return of_rank(list, r)[k];
      return list[static_cast<int64_t>(r - rank) * 2 * p.ws_stride + k];
    };
    move_tokens<2>(p, s, h, len, pos0, moves + stays, rank * kEvictThreads + tid, p.cluster * kEvictThreads,
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
  p->ws_stride = 0;
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
  int cluster, fit;
  int64_t list;            // entries of a list in the workspace, 0: never needed
  size_t bytes;
};
constexpr int kMaxFit = 16384;        // 12 bytes each of the 227 KB

// (the counts are on the device: a session that holds more than its budget says, once, is found there)
static EvictPlan evict_plan(const we_b200_paged_geom& g, int32_t T, int32_t keep) {
  EvictPlan r;
  const int64_t units = static_cast<int64_t>(g.S) * g.Hkv, usual = static_cast<int64_t>(keep) + T;
  r.cluster = cluster_for(units, usual, 1024, 4 * sm_count());
  const int64_t fit = ((usual + r.cluster - 1) / r.cluster + 1027) & ~3ll;
  r.fit = static_cast<int>(fit < kMaxFit ? fit : kMaxFit);
  const int64_t most = static_cast<int64_t>(g.max_pages) * g.page + T;
  const int64_t slice = ((most + r.cluster - 1) / r.cluster + 3) & ~3ll;
  r.list = slice <= r.fit ? 0 : slice;
  r.bytes = static_cast<size_t>(units) * r.cluster * 2 * r.list * sizeof(int32_t);
  return r;
}

}  // namespace we

extern "C" int we_b200_paged_append(const we_b200_paged_append_args* a, int32_t* status, void* stream) {
  we::PagedAppendParams p;
  const int rc = we::fill(a, status, &p);
  if (rc != WE_B200_OK) return rc;
  p.cluster = we::cluster_for(static_cast<int64_t>(p.v.S) * p.v.Hkv, static_cast<int64_t>(p.T) << p.vec_shift,
                              4 * we::kAppendThreads, 8 * we::sm_count());
  return we::launch(we::paged_append_kernel, p, we::kAppendThreads, 0, static_cast<cudaStream_t>(stream));
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
  const we::EvictPlan plan = we::evict_plan(a->geom, a->T, a->keep);
  if (plan.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < plan.bytes)) return WE_B200_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 3u) return WE_B200_E_ALIGN;
  if ((reinterpret_cast<uintptr_t>(a->weights) | reinterpret_cast<uintptr_t>(a->positions)) & 15u) return WE_B200_E_ALIGN;
  p.ws = static_cast<int32_t*>(a->workspace);
  p.ws_stride = plan.list;
  p.keep = a->keep;
  p.sink = a->sink;
  p.recent = a->recent;
  p.cluster = plan.cluster;
  p.fit = plan.fit;
  static std::atomic<bool> done[we::kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 0 || dev >= we::kMaxDevices) return WE_B200_E_LIMIT;
  if (!done[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(we::paged_append_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 12 * we::kMaxFit);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return static_cast<int>(e);
    }
    done[dev].store(true, std::memory_order_release);
  }
  return we::launch(we::paged_append_evict_kernel, p, we::kEvictThreads, 12 * plan.fit, static_cast<cudaStream_t>(stream));
}
