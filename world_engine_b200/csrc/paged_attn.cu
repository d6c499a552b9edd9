// Attention of one new token per session over the paged KV cache (sm_100a).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "paged.cuh"

namespace we {

constexpr int kPagedThreads = 256;

struct PagedAttnParams {
  PagedView v;
  const uint16_t* q;
  uint16_t* out;
  int64_t qs[2], os[2];
  const uint16_t* kv;
  const int32_t* lens;
  float* weights;
  float* lse;
  int32_t Hq, group;
  float scale_log2;
};

template <bool BF16>
__device__ __forceinline__ float to_float(uint16_t x) {
  if constexpr (BF16) return __bfloat162float(__ushort_as_bfloat16(x));
  else return __half2float(__ushort_as_half(x));
}
template <bool BF16>
__device__ __forceinline__ uint16_t from_float(float x) {
  if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  else return __half_as_ushort(__float2half_rn(x));
}

template <bool BF16, int DH>
__global__ void __launch_bounds__(kPagedThreads) paged_attn_kernel(const PagedAttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int kWarps = kPagedThreads / 32, kPer = DH / 32;
  __shared__ float s_m[kWarps], s_l[kWarps], s_o[kWarps][DH];
  const int h = blockIdx.x, s = blockIdx.y, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int len = paged_count(p.v, p.lens[s * p.v.Hkv + h]);
  for (int g = 0; g < p.group; ++g) {
    const int hq = h * p.group + g;
    float q[kPer], o[kPer];
    for (int u = 0; u < kPer; ++u) {
      q[u] = to_float<BF16>(p.q[s * p.qs[0] + hq * p.qs[1] + kPer * lane + u]);
      o[u] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    auto row_of = [&](int j) {
      int pg = paged_page(p.v, s, j >> p.v.page_shift);
      if (pg < 0) pg = 0;
      return p.kv + pg * p.v.page_s + h * p.v.head_s + (j & (p.v.page - 1)) * p.v.token_s + kPer * lane;
    };
    auto score = [&](const uint16_t* k) {
      float x = 0.f;
      for (int u = 0; u < kPer; ++u) x = fmaf(q[u], to_float<BF16>(k[u]), x);
      for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
      return x * p.scale_log2;
    };
    for (int j = wid; j < len; j += kWarps) {
      const uint16_t* k = row_of(j);
      const float x = score(k);
      const float mn = fmaxf(m, x);
      const float a = mn == m ? 1.f : exp2f(m - mn), w = exp2f(x - mn);
      l = l * a + w;
      for (int u = 0; u < kPer; ++u) o[u] = o[u] * a + w * to_float<BF16>(k[p.v.plane_s + u]);
      m = mn;
    }
    __syncthreads();
    if (lane == 0) s_m[wid] = m, s_l[wid] = l;
    for (int u = 0; u < kPer; ++u) s_o[wid][kPer * lane + u] = o[u];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w]);
    for (int w = 0; w < kWarps && w < len; ++w) sum += s_m[w] == top ? s_l[w] : s_l[w] * exp2f(s_m[w] - top);
    const float lse2 = top + log2f(sum);
    for (int d = threadIdx.x; d < DH; d += kPagedThreads) {
      float x = 0.f;
      for (int w = 0; w < kWarps && w < len; ++w) x += s_m[w] == top ? s_o[w][d] : s_o[w][d] * exp2f(s_m[w] - top);
      p.out[s * p.os[0] + hq * p.os[1] + d] = from_float<BF16>(len > 0 ? x / sum : 0.f);
    }
    if (threadIdx.x == 0 && p.lse != nullptr) p.lse[s * p.Hq + hq] = len > 0 ? lse2 * 0.6931471805599453f : -INFINITY;
    if (p.weights != nullptr) {
      for (int j = wid; j < len; j += kWarps) {
        const float x = score(row_of(j));
        const int pg = paged_page(p.v, s, j >> p.v.page_shift);
        if (lane == 0 && pg >= 0)
          atomicAdd(p.weights + (static_cast<int64_t>(pg) * p.v.Hkv + h) * p.v.page + (j & (p.v.page - 1)), exp2f(x - top) / sum);
      }
    }
    __syncthreads();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace we

extern "C" size_t we_b200_paged_attn_workspace_bytes(const we_b200_paged_geom* g, int32_t Hq, int accumulate) {
  (void)g;
  (void)Hq;
  (void)accumulate;
  return 0;
}

extern "C" int we_b200_paged_attn(const we_b200_paged_attn_args* a, int32_t* status, void* stream) {
  using namespace we;
  if (a == nullptr) return WE_B200_E_NULL;
  const we_b200_paged_geom& g = a->geom;
  const int rc = check_paged_geom(g);
  if (rc != WE_B200_OK) return rc;
  if (!a->q || !a->out || !a->kv || !a->table || !a->lens) return WE_B200_E_NULL;
  if (a->Hq < 1 || a->Hq % g.Hkv != 0) return WE_B200_E_SHAPE;
  if (a->Hq > 65535) return WE_B200_E_LIMIT;
  for (int i = 0; i < 2; ++i) {
    if (a->q_strides[i] < 0 || a->out_strides[i] < 0) return WE_B200_E_SHAPE;
    if ((a->q_strides[i] | a->out_strides[i]) & 7) return WE_B200_E_ALIGN;
  }
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->kv)) return WE_B200_E_ALIGN;
  PagedAttnParams p;
  p.v = paged_view(g, a->table, status);
  p.q = static_cast<const uint16_t*>(a->q);
  p.out = static_cast<uint16_t*>(a->out);
  for (int i = 0; i < 2; ++i) p.qs[i] = a->q_strides[i], p.os[i] = a->out_strides[i];
  p.kv = static_cast<const uint16_t*>(a->kv);
  p.lens = a->lens;
  p.weights = a->weights;
  p.lse = a->lse;
  p.Hq = a->Hq;
  p.group = a->Hq / g.Hkv;
  p.scale_log2 = (a->scale > 0.f ? a->scale : 1.0f / sqrtf(static_cast<float>(g.Dh))) * 1.4426950408889634f;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.Hkv), static_cast<unsigned>(g.S), 1);
  cfg.blockDim = dim3(kPagedThreads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e;
  const bool bf16 = g.dtype == WE_B200_BF16;
  if (g.Dh == 128) e = bf16 ? cudaLaunchKernelEx(&cfg, paged_attn_kernel<true, 128>, p) : cudaLaunchKernelEx(&cfg, paged_attn_kernel<false, 128>, p);
  else e = bf16 ? cudaLaunchKernelEx(&cfg, paged_attn_kernel<true, 64>, p) : cudaLaunchKernelEx(&cfg, paged_attn_kernel<false, 64>, p);
  g_launches.fetch_add(1, std::memory_order_relaxed);
  if (e != cudaSuccess) return static_cast<int>(e);
  const cudaError_t e2 = cudaGetLastError();
  return e2 == cudaSuccess ? WE_B200_OK : static_cast<int>(e2);
}
