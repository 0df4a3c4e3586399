// Balance loss of a router with per-expert counts, and the gradient of its gates and of the balance loss with respect to its logits.
//
// Over N counted tokens (all, or those whose mask is set) with k choices each among E experts, c_e = choices of e and
// S_e = sum of the probabilities of e:
//   loss = E sum_e (c_e / (N k)) (S_e / N),   d loss / d p[t, e] = E c_e / (N^2 k) on counted tokens, 0 on the others;  N = 0: 0.
// The gates are the chosen probabilities divided by their sum s, so with the gates' gradient dg
//   d p = scatter((dg_j - sum_j dg_j gate_j) / s) + w d loss / d p,    d logit_e = p_e (d p_e - sum_e d p_e p_e).
//
// Sums run in a fixed order (per thread, per CTA, over the CTAs of a cluster, over clusters), so two calls give the same bits; counts are
// integers.
#include <cuda_runtime.h>
#include <stdint.h>

#include "api.h"
#include "ptx.cuh"
#include "tmap.h"

namespace dh {

constexpr int BT = 256;              // threads per CTA
constexpr int B_CLUSTER = 8;
constexpr int B_MAX_E = 1024;
constexpr int B_MAX_K = 32;
constexpr int B_ROWS = 4;            // rows of a thread's column in flight

struct BalArgs {
  const float* probs;
  const void* ids;
  const uint8_t* mask;
  int64_t p_stride, id_stride;
  int id64, T, E, k;
};

__device__ __forceinline__ int bal_id(const BalArgs& a, int64_t t, int j) {
  const int64_t i = t * a.id_stride + j;
  const int64_t v = a.id64 ? reinterpret_cast<const int64_t*>(a.ids)[i] : (int64_t)reinterpret_cast<const int*>(a.ids)[i];
  return v < 0 || v >= a.E ? -1 : (int)v;
}
__device__ __forceinline__ uint32_t bal_at(const void* mine, int cta) { return mapa_u32(smem_u32(mine), cta); }
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

template <int W> struct BalVec { float v[W]; };
template <int W>
__device__ __forceinline__ BalVec<W> bal_load(const float* p) {
  BalVec<W> r;
  if constexpr (W == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    r.v[0] = f.x; r.v[1] = f.y; r.v[2] = f.z; r.v[3] = f.w;
  } else {
    r.v[0] = *p;
  }
  return r;
}

// Sums of the probabilities and counts of the choices over a share of the tokens.  A CTA's threads stand for columns of W experts and,
// as far as that leaves threads over, for several rows; a cluster joins what its CTAs have, each CTA a share of the experts.  One cluster
// finishes by itself, several leave psum [clusters, E] and pcount [clusters, E + 1] (last: counted tokens) for the kernel below.
template <int W>
__global__ void __launch_bounds__(BT) balance_kernel(const BalArgs a, float* __restrict__ psum, int* __restrict__ pcount, float* __restrict__ loss,
                                                     int* __restrict__ counts, float* __restrict__ coef) {
  __shared__ int cnt[B_MAX_E + 1];
  __shared__ float csum[B_MAX_E];
  __shared__ float part[8 * 32 * 4];
  __shared__ float losses[B_CLUSTER];
  __shared__ float red[BT / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= a.E; e += BT) cnt[e] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)a.T * blockIdx.x / gridDim.x, t1 = (int64_t)a.T * (blockIdx.x + 1) / gridDim.x;
  const int n = (int)(t1 - t0);
  for (int i = threadIdx.x; i < n * a.k; i += BT) {
    const int r = i / a.k, j = i - r * a.k;
    const int e = bal_id(a, t0 + r, j);
    if (a.mask == nullptr || a.mask[t0 + r]) {
      if (e >= 0) atomicAdd(&cnt[e], 1);
      if (j == 0) atomicAdd(&cnt[a.E], 1);
    }
  }
  // columns: the next power of two of E / W, at most BT
  const int groups = (a.E + W - 1) / W;
  int cols = 1;
  while (cols < groups && cols < BT) cols <<= 1;
  const int c = threadIdx.x & (cols - 1), r0 = threadIdx.x / cols, rows = BT / cols;
  for (int first = 0; first < groups; first += cols) {
    const int g = first + c;
    float s[W];
#pragma unroll
    for (int q = 0; q < W; ++q) s[q] = 0.f;
    if (g < groups) {
      const float* p = a.probs + t0 * a.p_stride + g * W;
      for (int r = r0; r < n; r += rows * B_ROWS) {
        BalVec<W> v[B_ROWS];
        bool in[B_ROWS];
#pragma unroll
        for (int b = 0; b < B_ROWS; ++b) {
          const int q = r + b * rows;
          in[b] = q < n;
          if (in[b]) {
            v[b] = bal_load<W>(p + q * a.p_stride);
            if (a.mask != nullptr) in[b] = a.mask[t0 + q] != 0;
          }
        }
#pragma unroll
        for (int b = 0; b < B_ROWS; ++b)
          if (in[b]) {
#pragma unroll
            for (int q = 0; q < W; ++q) s[q] += v[b].v[q];
          }
      }
    }
    // over the rows of a warp, then over what the warps have
    for (int o = cols; o < 32; o <<= 1) {
#pragma unroll
      for (int q = 0; q < W; ++q) s[q] += __shfl_xor_sync(0xffffffffu, s[q], o);
    }
    const int parts = cols < 32 ? BT / 32 : rows, mine = cols < 32 ? warp : r0;
    __syncthreads();
    if (cols >= 32 || lane < cols) {
#pragma unroll
      for (int q = 0; q < W; ++q) part[(mine * cols + c) * W + q] = s[q];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cols * W; e += BT) {
      if (first * W + e >= a.E) continue;
      float t = part[e];
      for (int q = 1; q < parts; ++q) t += part[q * cols * W + e];
      csum[first * W + e] = t;
    }
  }
  __syncthreads();
  cluster_sync_all();
  const int me = (int)cluster_ctarank(), cluster = blockIdx.x / B_CLUSTER;
  const bool alone = gridDim.x == B_CLUSTER;
  int counted = 0;
#pragma unroll
  for (int r = 0; r < B_CLUSTER; ++r) counted += (int)ld_cluster_u32(bal_at(&cnt[a.E], r));
  const float inv = counted > 0 ? 1.f / (float)counted : 0.f;
  float l = 0.f;
  for (int e = me + (int)threadIdx.x * B_CLUSTER; e < a.E; e += B_CLUSTER * BT) {
    float s = 0.f;
    int n_e = 0;
#pragma unroll
    for (int r = 0; r < B_CLUSTER; ++r) {
      s += __uint_as_float(ld_cluster_u32(bal_at(&csum[e], r)));
      n_e += (int)ld_cluster_u32(bal_at(&cnt[e], r));
    }
    if (alone) {
      const float w = (float)n_e * inv * inv * ((float)a.E / (float)a.k);
      counts[e] = n_e;
      coef[e] = w;
      l += w * s;
    } else {
      psum[(size_t)cluster * a.E + e] = s;
      pcount[(size_t)cluster * (a.E + 1) + e] = n_e;
    }
  }
  if (!alone) {
    if (me == 0 && threadIdx.x == 0) pcount[(size_t)cluster * (a.E + 1) + a.E] = counted;
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) red[warp] = l;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int q = 1; q < BT / 32; ++q) l += red[q];
      st_cluster_f32(bal_at(&losses[me], 0), l);
    }
  }
  __syncthreads();
  cluster_sync_all();                 // nobody leaves while another reads its sums
  if (alone && me == 0 && threadIdx.x == 0) {
    float t = losses[0];
    for (int q = 1; q < B_CLUSTER; ++q) t += losses[q];
    *loss = t;
  }
}

__global__ void __launch_bounds__(1024) balance_finish_kernel(const float* __restrict__ psum, const int* __restrict__ pcount, int parts, int E, int k,
                                                              float* __restrict__ loss, int* __restrict__ counts, float* __restrict__ coef) {
  __shared__ float red[32];
  int n = 0;
  for (int p = threadIdx.x & 31; p < parts; p += 32) n += pcount[(size_t)p * (E + 1) + E];
  n = __reduce_add_sync(0xffffffffu, n);
  const float inv = n > 0 ? 1.f / (float)n : 0.f;
  float l = 0.f;
  if ((int)threadIdx.x < E) {
    float s = 0.f;
    int c = 0;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      s += psum[(size_t)p * E + threadIdx.x];
      c += pcount[(size_t)p * (E + 1) + threadIdx.x];
    }
    const float w = (float)c * inv * inv * ((float)E / (float)k);
    counts[threadIdx.x] = c;
    coef[threadIdx.x] = w;
    l = w * s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) l += red[w];
    *loss = l;
  }
}

struct RouterArgs {
  const float *gates, *d_gates, *coef;       // coef null: no balance term
  float* out;
  int64_t g_stride, dg_stride;
  float weight;
  int lanes;                                 // threads of a row: a power of two, at least k
};

// `lanes` threads per token, each with NV vectors of W experts; thread j of them also has the j-th choice.  The row is written with the
// balance term alone and its k chosen experts once more behind that (the few that were chosen need no search by the others).
template <int W, int NV>
__global__ void __launch_bounds__(BT) router_bwd_kernel(const BalArgs a, const RouterArgs b) {
  const int lane = threadIdx.x & 31, L = b.lanes, l = lane & (L - 1);
  const int per_warp = 32 / L;
  float co[NV][W];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const int e = (i * L + l) * W + q;
      co[i][q] = b.coef != nullptr && e < a.E ? b.weight * b.coef[e] : 0.f;
    }
  const int64_t step = (int64_t)gridDim.x * (BT / 32) * per_warp;
  for (int64_t base = ((int64_t)blockIdx.x * (BT / 32) + (threadIdx.x >> 5)) * per_warp; base < a.T; base += step) {
    const int64_t t = base + lane / L;
    const bool row = t < a.T;
    const float* p = a.probs + (row ? t : 0) * a.p_stride;
    BalVec<W> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * L + l) * W;
#pragma unroll
      for (int q = 0; q < W; ++q) v[i].v[q] = 0.f;
      if (row && e < a.E) v[i] = bal_load<W>(p + e);
    }
    int id = -1;
    float dg = 0.f, g = 0.f, pj = 0.f;
    if (row && l < a.k) {
      id = bal_id(a, t, l);
      dg = b.d_gates[t * b.dg_stride + l];
      g = b.gates[t * b.g_stride + l];
    }
    const bool counts = row && (a.mask == nullptr || a.mask[t] != 0);
    if (id >= 0) pj = p[id];
    float dot = id >= 0 ? dg * g : 0.f, sel = pj;
    for (int o = L >> 1; o > 0; o >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
      sel += __shfl_xor_sync(0xffffffffu, sel, o);
    }
    float u = id >= 0 && sel != 0.f ? (dg - dot) / sel : 0.f;
    float all = u * pj;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const int e = (i * L + l) * W + q;
        if (counts && e < a.E) all += co[i][q] * v[i].v[q];
      }
    for (int o = L >> 1; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    float* o = b.out + (row ? t : 0) * a.E;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * L + l) * W;
      if (!row || e >= a.E) continue;
      float r[W];
#pragma unroll
      for (int q = 0; q < W; ++q) r[q] = v[i].v[q] * ((counts ? co[i][q] : 0.f) - all);
      if constexpr (W == 4) *reinterpret_cast<float4*>(o + e) = make_float4(r[0], r[1], r[2], r[3]);
      else o[e] = r[0];
    }
    // an expert that was chosen twice gets both choices' gradients, in the order of the choices
    const unsigned int twins = __match_any_sync(0xffffffffu, id >= 0 ? (lane / L) * B_MAX_E + id : -1 - lane);
    if (__any_sync(0xffffffffu, (twins & (twins - 1)) != 0)) {
      float sum = 0.f;
      for (int q = 0; q < 32; ++q) {
        const float other = __shfl_sync(0xffffffffu, u, q);
        if (twins >> q & 1) sum += other;
      }
      u = sum;
    }
    __syncwarp();
    if (id >= 0) o[id] = pj * ((counts && b.coef != nullptr ? b.weight * b.coef[id] : 0.f) - all + u);
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------- host
// All fields 8 bytes wide, as the Python layer packs them.
struct BalCall {
  int64_t probs, p_stride, ids, id_stride, id64, mask, T, E, k, budget, stream;
};

static int bal_refuse(const char* what, const BalCall& c) {
  if (c.T >= 0 && c.E > 0 && c.E <= B_MAX_E && c.k > 0 && c.k <= B_MAX_K && c.T * c.k < INT32_MAX) return 0;
  set_last_error_c(what, "1 to 1024 experts, 1 to 32 choices, fewer than 2^31 choices in all");
  return (int)cudaErrorInvalidValue;
}
static int bal_rc(const char* what, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c(what, cudaGetErrorString(e));
  return (int)e;
}
static BalArgs bal_args(const BalCall& c) {
  return BalArgs{(const float*)c.probs, (const void*)c.ids, (const uint8_t*)c.mask, c.p_stride, c.id_stride, (int)c.id64, (int)c.T, (int)c.E, (int)c.k};
}
static int bal_budget(const BalCall& c) {
  const int sms = dh_sm_count();
  return (c.budget <= 0 || c.budget > sms) ? sms : (int)c.budget;
}
static bool bal_wide(const BalCall& c) { return c.E % 4 == 0 && c.p_stride % 4 == 0 && (c.probs & 15) == 0; }
// Clusters of the forward: one (a single launch) up to B_ALONE probabilities, beyond it up to two CTAs per SM.
constexpr int64_t B_ALONE = 1 << 19;
static int bal_clusters(const BalCall& c) {
  if (c.T * c.E <= B_ALONE) return 1;
  const int64_t want = c.T * c.E / (1 << 16) / B_CLUSTER, most = 2 * bal_budget(c) / B_CLUSTER;
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

template <int W>
static void router_launch(const BalCall& c, const RouterArgs& r, int vecs, cudaStream_t s) {
  const int64_t warps = (c.T + 32 / r.lanes - 1) / (32 / r.lanes), blocks = (warps + BT / 32 - 1) / (BT / 32);
  const int64_t most = 8ll * bal_budget(c);
  const unsigned int grid = (unsigned int)(blocks < most ? blocks : most);
  const BalArgs a = bal_args(c);
  if (vecs <= 1) router_bwd_kernel<W, 1><<<grid, BT, 0, s>>>(a, r);
  else if (vecs <= 2) router_bwd_kernel<W, 2><<<grid, BT, 0, s>>>(a, r);
  else if (vecs <= 4) router_bwd_kernel<W, 4><<<grid, BT, 0, s>>>(a, r);
  else if (vecs <= 8) router_bwd_kernel<W, 8><<<grid, BT, 0, s>>>(a, r);
  else if (W == 1 && vecs <= 16) router_bwd_kernel<W, W == 1 ? 16 : 1><<<grid, BT, 0, s>>>(a, r);
  else router_bwd_kernel<W, W == 1 ? 32 : 1><<<grid, BT, 0, s>>>(a, r);
}

}  // namespace dh

using namespace dh;

extern "C" {

// Words of 4 bytes that the forward needs as scratch (0: none).
int64_t dh_balance_scratch(const void* call) {
  const BalCall& c = *(const BalCall*)call;
  const int n = bal_clusters(c);
  return n > 1 ? n * (2 * c.E + 1) : 0;
}
// loss [1] fp32, counts [E] int32, coef [E] fp32 = d loss / d p of a counted token.
int dh_balance_fwd(const void* call, void* scratch, void* loss, void* counts, void* coef) {
  const BalCall& c = *(const BalCall*)call;
  if (int rc = bal_refuse("dh_balance_fwd", c)) return rc;
  const int n = bal_clusters(c);
  if (n > 1 && scratch == nullptr) {
    set_last_error_c("dh_balance_fwd", "no scratch");
    return (int)cudaErrorInvalidValue;
  }
  float* psum = (float*)scratch;
  int* pcount = n > 1 ? (int*)(psum + (size_t)n * c.E) : nullptr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * B_CLUSTER);
  cfg.blockDim = dim3(BT);
  cfg.stream = (cudaStream_t)c.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = B_CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = bal_wide(c) ? cudaLaunchKernelEx(&cfg, balance_kernel<4>, bal_args(c), psum, pcount, (float*)loss, (int*)counts, (float*)coef)
                                    : cudaLaunchKernelEx(&cfg, balance_kernel<1>, bal_args(c), psum, pcount, (float*)loss, (int*)counts, (float*)coef);
  if (e == cudaSuccess && n > 1)
    balance_finish_kernel<<<1, 1024, 0, cfg.stream>>>(psum, pcount, n, (int)c.E, (int)c.k, (float*)loss, (int*)counts, (float*)coef);
  return bal_rc("dh_balance_fwd", e);
}
// out [T, E] fp32 contiguous, 16-byte aligned.  coef may be null (no balance term).
int dh_router_bwd(const void* call, const void* gates, int64_t g_stride, const void* d_gates, int64_t dg_stride, const void* coef, float weight,
                  void* out) {
  const BalCall& c = *(const BalCall*)call;
  if (int rc = bal_refuse("dh_router_bwd", c)) return rc;
  if (c.T == 0) return 0;
  RouterArgs r{(const float*)gates, (const float*)d_gates, (const float*)coef, (float*)out, g_stride, dg_stride, weight, 1};
  const bool wide = bal_wide(c) && ((uintptr_t)out & 15) == 0;
  const int groups = (int)(wide ? c.E / 4 : c.E);
  while (r.lanes < 32 && (r.lanes < groups || r.lanes < c.k)) r.lanes *= 2;
  const int vecs = (groups + r.lanes - 1) / r.lanes;
  if (wide) router_launch<4>(c, r, vecs, (cudaStream_t)c.stream);
  else router_launch<1>(c, r, vecs, (cudaStream_t)c.stream);
  return bal_rc("dh_router_bwd", cudaSuccess);
}

}  // extern "C"
