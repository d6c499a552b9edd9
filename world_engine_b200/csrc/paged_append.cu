// Append to the paged KV cache, without and with a budget (sm_100a).
#include "paged.cuh"

namespace we {

constexpr int kAppendThreads = 256;

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
  int32_t* ws;
  int64_t ws_stride;     // list entries of one (session, head)
  int32_t T, keep, sink, recent;
  int32_t vec_shift;     // log2 of 16-byte vectors per row
};

// One 16-byte vector `c` of the K and the V row of a token: from a new row, to a slot.
__device__ __forceinline__ void put_new(const PagedAppendParams& p, int s, int h, int t, int pg, int row, int c) {
  const uint4 k = *reinterpret_cast<const uint4*>(p.k_new + s * p.ks[0] + h * p.ks[1] + t * p.ks[2] + 8 * c);
  const uint4 v = *reinterpret_cast<const uint4*>(p.v_new + s * p.vs[0] + h * p.vs[1] + t * p.vs[2] + 8 * c);
  uint16_t* dst = p.kv + pg * p.v.page_s + h * p.v.head_s + row * p.v.token_s + 8 * c;
  *reinterpret_cast<uint4*>(dst) = k;
  *reinterpret_cast<uint4*>(dst + p.v.plane_s) = v;
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

__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const PagedAppendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.x, s = blockIdx.y, unit = s * p.v.Hkv + h;
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  const int n = new_count(p, s);
  const int room = (p.v.max_pages << p.v.page_shift) - len;
  const int take = n < room ? n : room;
  if (take < n && threadIdx.x == 0) paged_report(p.v);
  __syncthreads();                       // every thread has read the counts before they are replaced
  const int vecs = 1 << p.vec_shift;
  for (int i = threadIdx.x; i < (take << p.vec_shift); i += kAppendThreads) {
    const int t = i >> p.vec_shift, c = i & (vecs - 1), at = len + t, row = at & (p.v.page - 1);
    const int pg = paged_page(p.v, s, at >> p.v.page_shift);
    if (pg < 0) continue;
    put_new(p, s, h, t, pg, row, c);
    if (c == 0) {
      const int64_t m = (static_cast<int64_t>(pg) * p.v.Hkv + h) * p.v.page + row;
      if (p.weights != nullptr)
        p.weights[m] = p.w_new != nullptr ? p.w_new[s * p.wns[0] + h * p.wns[1] + t * p.wns[2]] : 0.f;
      if (p.positions != nullptr) p.positions[m] = pos0 + t;
    }
  }
  if (threadIdx.x == 0) {
    p.lens_out[unit] = len + take;
    p.next_pos_out[unit] = pos0 + n;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ------------------------------------------------------------------ under a budget
constexpr int kEvictThreads = 512;

// Weights as unsigned numbers of the same order: NaN above every number, shielded tokens above NaN, -0 equal to 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xFFFFFFFEu;
  const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct Candidate {
  uint32_t key;
  bool there;
};

__global__ void __launch_bounds__(kEvictThreads) paged_append_evict_kernel(const PagedAppendParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_need, s_sum[kEvictThreads / 32], s_base[3];
  const int h = blockIdx.x, s = blockIdx.y, unit = s * p.v.Hkv + h, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int len = paged_count(p.v, p.lens[unit]);
  const int pos0 = p.next_pos[unit];
  const int n = new_count(p, s);
  const int total = len + n;
  const int64_t end = static_cast<int64_t>(pos0) + n;
  int32_t* holes = p.ws + 2 * unit * p.ws_stride;
  int32_t* movers = holes + p.ws_stride;

  auto key_of = [&](int i) -> uint32_t {
    float w = 0.f;
    int64_t pos;
    if (i < len) {
      const int pg = paged_page(p.v, s, i >> p.v.page_shift);
      if (pg < 0) return 0u;
      const int64_t m = (static_cast<int64_t>(pg) * p.v.Hkv + h) * p.v.page + (i & (p.v.page - 1));
      w = p.weights[m];
      pos = p.positions[m];
    } else {
      if (p.w_new != nullptr) w = p.w_new[s * p.wns[0] + h * p.wns[1] + (i - len) * p.wns[2]];
      pos = static_cast<int64_t>(pos0) + (i - len);
    }
    if (pos < p.sink || pos >= end - p.recent) return 0xFFFFFFFFu;
    return weight_key(w);
  };

  // ---- the key of the last one kept, eight bits at a time, and how many of that key are kept
  uint32_t prefix = 0, need = 0;
  const bool over = total > p.keep;
  if (over) {
    if (tid == 0) s_need = static_cast<uint32_t>(p.keep);
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int b = tid; b < 256; b += kEvictThreads) hist[b] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
      for (int i = tid; i < total; i += kEvictThreads) {
        const uint32_t k = key_of(i);
        if ((k & mask) == (prefix & mask)) atomicAdd(&hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t want = s_need;
        int b = 255;
        for (; b > 0 && hist[b] < want; --b) want -= hist[b];
        s_prefix = prefix | (static_cast<uint32_t>(b) << shift);
        s_need = want;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
    }
  }

  // ---- who goes where, in the order of the indexes
  if (tid < 3) s_base[tid] = 0;                    // equals, holes and movers so far
  __syncthreads();
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = 0; over && i0 < total; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < total ? key_of(i) : 0u;
    const bool equal = i < total && k == prefix;
    uint32_t vote = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) s_sum[wid] = __popc(vote);
    __syncthreads();
    uint32_t rank = s_base[0] + __popc(vote & below);
    for (int w = 0; w < wid; ++w) rank += s_sum[w];
    const bool kept = i < total && (k > prefix || (equal && rank < need));
    const bool hole = i < p.keep && i < total && !kept, mover = kept && i >= p.keep;
    __syncthreads();
    if (tid == kEvictThreads - 1) s_base[0] = rank + (equal ? 1u : 0u);
    for (int pass = 0; pass < 2; ++pass) {
      const bool mine = pass == 0 ? hole : mover;
      vote = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) s_sum[wid] = __popc(vote);
      __syncthreads();
      uint32_t at = s_base[1 + pass] + __popc(vote & below);
      for (int w = 0; w < wid; ++w) at += s_sum[w];
      if (mine && at < p.ws_stride) (pass == 0 ? holes : movers)[at] = i;
      __syncthreads();
      if (tid == kEvictThreads - 1) s_base[1 + pass] = at + (mine ? 1u : 0u);
    }
    // a new token that stays below the budget is written where it comes to lie
    if (kept && i >= len && i < p.keep) {
      const int pg = paged_page(p.v, s, i >> p.v.page_shift);
      if (pg >= 0) {
        const int row = i & (p.v.page - 1), t = i - len;
        for (int c = 0; c < (1 << p.vec_shift); ++c) put_new(p, s, h, t, pg, row, c);
        const int64_t m = (static_cast<int64_t>(pg) * p.v.Hkv + h) * p.v.page + row;
        p.weights[m] = p.w_new != nullptr ? p.w_new[s * p.wns[0] + h * p.wns[1] + t * p.wns[2]] : 0.f;
        p.positions[m] = pos0 + t;
      }
    }
  }
  __syncthreads();
  const int moves = over ? static_cast<int>(s_base[2]) : n;
  for (int j = tid; j < (moves << p.vec_shift); j += kEvictThreads) {
    const int c = j & ((1 << p.vec_shift) - 1), e = j >> p.vec_shift;
    const int src = over ? movers[e] : len + e, dst = over ? holes[e] : len + e;
    const int to = paged_page(p.v, s, dst >> p.v.page_shift), to_row = dst & (p.v.page - 1);
    if (to < 0) continue;
    const int64_t mt = (static_cast<int64_t>(to) * p.v.Hkv + h) * p.v.page + to_row;
    if (src >= len) {
      const int t = src - len;
      put_new(p, s, h, t, to, to_row, c);
      if (c == 0) {
        p.weights[mt] = p.w_new != nullptr ? p.w_new[s * p.wns[0] + h * p.wns[1] + t * p.wns[2]] : 0.f;
        p.positions[mt] = pos0 + t;
      }
      continue;
    }
    const int from = paged_page(p.v, s, src >> p.v.page_shift), from_row = src & (p.v.page - 1);
    if (from < 0) continue;
    const uint16_t* a = p.kv + from * p.v.page_s + h * p.v.head_s + from_row * p.v.token_s + 8 * c;
    uint16_t* b = p.kv + to * p.v.page_s + h * p.v.head_s + to_row * p.v.token_s + 8 * c;
    *reinterpret_cast<uint4*>(b) = *reinterpret_cast<const uint4*>(a);
    *reinterpret_cast<uint4*>(b + p.v.plane_s) = *reinterpret_cast<const uint4*>(a + p.v.plane_s);
    if (c == 0) {
      const int64_t mf = (static_cast<int64_t>(from) * p.v.Hkv + h) * p.v.page + from_row;
      p.weights[mt] = p.weights[mf];
      p.positions[mt] = p.positions[mf];
    }
  }
  if (tid == 0) {
    p.lens_out[unit] = total < p.keep ? total : p.keep;
    p.next_pos_out[unit] = static_cast<int32_t>(end);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
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
  p->T = a->T;
  p->keep = p->sink = p->recent = 0;
  p->vec_shift = g.Dh == 128 ? 4 : 3;
  return WE_B200_OK;
}

static int launch(void (*kernel)(PagedAppendParams), const PagedAppendParams& p, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.v.Hkv), static_cast<unsigned>(p.v.S), 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  if (e != cudaSuccess) return static_cast<int>(e);
  const cudaError_t e2 = cudaGetLastError();
  return e2 == cudaSuccess ? WE_B200_OK : static_cast<int>(e2);
}

// Entries of a (session, head)'s list of moves: no more tokens can move than the budget has room for, nor than lie
// beyond it.
static int64_t list_entries(const we_b200_paged_geom& g, int32_t T, int32_t keep) {
  const int64_t beyond = static_cast<int64_t>(g.max_pages) * g.page + T - keep;
  return beyond < keep ? (beyond < 0 ? 0 : beyond) : keep;
}

}  // namespace we

extern "C" int we_b200_paged_append(const we_b200_paged_append_args* a, int32_t* status, void* stream) {
  we::PagedAppendParams p;
  const int rc = we::fill(a, status, &p);
  if (rc != WE_B200_OK) return rc;
  return we::launch(we::paged_append_kernel, p, we::kAppendThreads, static_cast<cudaStream_t>(stream));
}

extern "C" size_t we_b200_paged_evict_workspace_bytes(const we_b200_paged_geom* g, int32_t T, int32_t keep) {
  if (g == nullptr || we::check_paged_geom(*g) != WE_B200_OK || T < 0 || keep < 1) return 0;
  return static_cast<size_t>(g->S) * g->Hkv * 2 * we::list_entries(*g, T, keep) * sizeof(int32_t);
}

extern "C" int we_b200_paged_append_evict(const we_b200_paged_append_args* a, int32_t* status, void* stream) {
  we::PagedAppendParams p;
  const int rc = we::fill(a, status, &p);
  if (rc != WE_B200_OK) return rc;
  if (a->weights == nullptr || a->positions == nullptr) return WE_B200_E_NULL;
  if (a->keep < 1 || a->sink < 0 || a->recent < 0) return WE_B200_E_SHAPE;
  if (static_cast<int64_t>(a->sink) + a->recent > a->keep) return WE_B200_E_SHAPE;
  if (static_cast<int64_t>(a->geom.max_pages) * a->geom.page < a->keep) return WE_B200_E_SHAPE;
  const size_t need = we_b200_paged_evict_workspace_bytes(&a->geom, a->T, a->keep);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return WE_B200_E_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 3u) return WE_B200_E_ALIGN;
  p.ws = static_cast<int32_t*>(a->workspace);
  p.ws_stride = we::list_entries(a->geom, a->T, a->keep);
  p.keep = a->keep;
  p.sink = a->sink;
  p.recent = a->recent;
  return we::launch(we::paged_append_evict_kernel, p, we::kEvictThreads, static_cast<cudaStream_t>(stream));
}
