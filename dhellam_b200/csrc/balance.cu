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

constexpr int BT = 256;              // threads per CTA of the backward
constexpr int B_CLUSTER = 8;
constexpr int B_MAX_E = 1024;
constexpr int B_MAX_K = 32;
constexpr int B_ROWS = 8;            // rows of a thread's column in flight

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

__device__ __forceinline__ float bal_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int W> struct BalVec { float v[W]; };
template <int W>
__device__ __forceinline__ BalVec<W> bal_load(const float* p) {
  BalVec<W> r;
  if constexpr (W == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    r.v[0] = f.x; r.v[1] = f.y; r.v[2] = f.z; r.v[3] = f.w;
  } else if constexpr (W == 2) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    r.v[0] = f.x; r.v[1] = f.y;
  } else {
    r.v[0] = *p;
  }
  return r;
}

// Sums of the probabilities and counts of the choices over a share of the tokens.  A CTA's threads stand for columns of W experts and,
// as far as that leaves threads over, for several rows; a cluster joins what its CTAs have, each CTA a share of the experts.  One cluster
// finishes by itself, several leave psum [clusters, E] and pcount [clusters, E + 1] (last: counted tokens) for the kernel below.
template <int W, int BF>
__global__ void __launch_bounds__(BF, 1024 / BF) balance_kernel(const BalArgs a, float* __restrict__ psum, int* __restrict__ pcount, float* __restrict__ loss,
                                                     int* __restrict__ counts, float* __restrict__ coef) {
  __shared__ int cnt[B_MAX_E + 1];
  __shared__ float csum[B_MAX_E];
  __shared__ float part[BF * W];
  __shared__ float losses[B_CLUSTER];
  __shared__ float red[BF / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= a.E; e += BF) cnt[e] = 0;
  __syncthreads();
  const int64_t t0 = (int64_t)a.T * blockIdx.x / gridDim.x, t1 = (int64_t)a.T * (blockIdx.x + 1) / gridDim.x;
  const int n = (int)(t1 - t0);
  int tokens = 0;
  for (int r = threadIdx.x; r < n; r += BF) {
    if (a.mask != nullptr && !a.mask[t0 + r]) continue;
    ++tokens;
#pragma unroll 4
    for (int j = 0; j < a.k; ++j) {
      const int e = bal_id(a, t0 + r, j);
      if (e >= 0) atomicAdd(&cnt[e], 1);
    }
  }
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  if (lane == 0) atomicAdd(&cnt[a.E], tokens);
  // columns: the next power of two of E / W, at most BF
  const int groups = (a.E + W - 1) / W;
  int cols = 1;
  while (cols < groups && cols < BF) cols <<= 1;
  const int c = threadIdx.x & (cols - 1), r0 = threadIdx.x / cols, rows = BF / cols;
  for (int first = 0; first < groups; first += cols) {
    const int g = first + c;
    float s[W];
#pragma unroll
    for (int q = 0; q < W; ++q) s[q] = 0.f;
    if (g < groups) {
      const float* p = a.probs + t0 * a.p_stride + g * W;
      int r = r0;
      // Narrow loads in batches without a question per row first (65536 x 134: 29 -> 20 us, x 255: 36 -> 26; loads of four are slower so
      // where they come from HBM, 65536 x 256: 29 -> 34 us).
      if constexpr (W < 4) {
        for (; r + (B_ROWS - 1) * rows < n; r += rows * B_ROWS) {
          BalVec<W> v[B_ROWS];
#pragma unroll
          for (int b = 0; b < B_ROWS; ++b) v[b] = bal_load<W>(p + (r + b * rows) * a.p_stride);
          if (a.mask != nullptr) {
            uint8_t in[B_ROWS];
#pragma unroll
            for (int b = 0; b < B_ROWS; ++b) in[b] = a.mask[t0 + r + b * rows];
#pragma unroll
            for (int b = 0; b < B_ROWS; ++b)
#pragma unroll
              for (int q = 0; q < W; ++q) s[q] += in[b] ? v[b].v[q] : 0.f;
          } else {
#pragma unroll
            for (int b = 0; b < B_ROWS; ++b)
#pragma unroll
              for (int q = 0; q < W; ++q) s[q] += v[b].v[q];
          }
        }
      }
      for (; r < n; r += rows * B_ROWS) {
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
    const int parts = cols < 32 ? BF / 32 : rows, mine = cols < 32 ? warp : r0;
    __syncthreads();
    if (cols >= 32 || lane < cols) {
#pragma unroll
      for (int q = 0; q < W; ++q) part[(mine * cols + c) * W + q] = s[q];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cols * W; e += BF) {
      if (first * W + e >= a.E) continue;
      float t = part[e];
      for (int q = 1; q < parts; ++q) t += part[q * cols * W + e];
      csum[first * W + e] = t;
    }
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");       // the kernel below may be put in place
  __syncthreads();
  cluster_sync_all();
  const int me = (int)cluster_ctarank(), cluster = blockIdx.x / B_CLUSTER;
  const bool alone = gridDim.x == B_CLUSTER;
  int counted = 0;
#pragma unroll
  for (int r = 0; r < B_CLUSTER; ++r) counted += (int)ld_cluster_u32(bal_at(&cnt[a.E], r));
  const float inv = counted > 0 ? 1.f / (float)counted : 0.f;
  float l = 0.f;
  for (int e = me + (int)threadIdx.x * B_CLUSTER; e < a.E; e += B_CLUSTER * BF) {
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
    l = bal_warp_sum(l);
    if (lane == 0) red[warp] = l;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int q = 1; q < BF / 32; ++q) l += red[q];
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

// What the clusters have: 1024 threads, as many of them for an expert as that leaves.
__global__ void __launch_bounds__(1024) balance_finish_kernel(const float* __restrict__ psum, const int* __restrict__ pcount, int parts, int E, int k,
                                                              float* __restrict__ loss, int* __restrict__ counts, float* __restrict__ coef) {
  __shared__ float sums[1024];
  __shared__ int cnts[1024];
  __shared__ float red[32];
  __shared__ int counted;
  if (threadIdx.x == 0) counted = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)threadIdx.x < parts) atomicAdd(&counted, pcount[(size_t)threadIdx.x * (E + 1) + E]);
  int cols = 32;
  while (cols < E) cols <<= 1;
  const int e = threadIdx.x & (cols - 1), step = 1024 / cols;
  float s = 0.f;
  int c = 0;
  if (e < E) {
#pragma unroll 8
    for (int p = threadIdx.x / cols; p < parts; p += step) {
      s += psum[(size_t)p * E + e];
      c += pcount[(size_t)p * (E + 1) + e];
    }
  }
  sums[threadIdx.x] = s;
  cnts[threadIdx.x] = c;
  __syncthreads();
  float l = 0.f;
  if ((int)threadIdx.x < E) {
    for (int q = 1; q < step; ++q) {
      s += sums[q * cols + e];
      c += cnts[q * cols + e];
    }
    const float inv = counted > 0 ? 1.f / (float)counted : 0.f;
    const float w = (float)c * inv * inv * ((float)E / (float)k);
    counts[e] = c;
    coef[e] = w;
    l = w * s;
  }
  l = bal_warp_sum(l);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = l;
  __syncthreads();
  if (threadIdx.x < 32) {
    l = bal_warp_sum(red[threadIdx.x]);
    if (threadIdx.x == 0) *loss = l;
  }
}

struct RouterArgs {
  const float *gates, *d_gates, *coef;       // coef null: no balance term
  float* out;
  int64_t g_stride, dg_stride;
  float weight;
};

template <int L>
__device__ __forceinline__ void bal_group_sum(float& a, float& b) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
}

// L threads per token (a power of two, at least k), each with NV vectors of W experts; thread j of them also has the j-th choice.  The row
// is written with the balance term alone and its k chosen experts once more behind that (no search for the few that were chosen).
template <int W, int L, int NV>
__global__ void __launch_bounds__(BT) router_bwd_kernel(const BalArgs a, const RouterArgs b) {
  const int lane = threadIdx.x & 31, l = lane & (L - 1);
  constexpr int PER_WARP = 32 / L;
  float co[NV][W];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const int e = (i * L + l) * W + q;
      co[i][q] = b.coef != nullptr && e < a.E ? b.weight * b.coef[e] : 0.f;
    }
  const int step = gridDim.x * (BT / 32) * PER_WARP;
  for (int base = (blockIdx.x * (BT / 32) + (threadIdx.x >> 5)) * PER_WARP; base < a.T; base += step) {
    const int64_t t = base + lane / L;
    const bool row = t < a.T;
    const float* p = a.probs + (row ? t : 0) * a.p_stride;
    int id = -1;
    float dg = 0.f, g = 0.f;
    if (row && l < a.k) {
      id = bal_id(a, t, l);
      dg = b.d_gates[t * b.dg_stride + l];
      g = b.gates[t * b.g_stride + l];
    }
    const bool counts = row && (a.mask == nullptr || a.mask[t] != 0);
    BalVec<W> v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * L + l) * W;
#pragma unroll
      for (int q = 0; q < W; ++q) v[i].v[q] = 0.f;
      if (row && e < a.E) v[i] = bal_load<W>(p + e);
    }
    float dot = 0.f, pj = 0.f;
    if (id >= 0) { pj = p[id]; dot = dg * g; }
    float sel = pj;
    bal_group_sum<L>(dot, sel);
    float u = id >= 0 ? (dg - dot) / sel : 0.f;          // a sum of 0 has no finite gradient: it shows
    float all = u * pj, bal = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int q = 0; q < W; ++q) bal = fmaf(co[i][q], v[i].v[q], bal);
    bal_group_sum<L>(all, bal);
    if (counts) all += bal;
    const float on = counts ? 1.f : 0.f;
    float* o = b.out + (row ? t : 0) * a.E;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * L + l) * W;
      if (!row || e >= a.E) continue;
      float r[W];
#pragma unroll
      for (int q = 0; q < W; ++q) r[q] = v[i].v[q] * fmaf(co[i][q], on, -all);
      if constexpr (W == 4) *reinterpret_cast<float4*>(o + e) = make_float4(r[0], r[1], r[2], r[3]);
      else o[e] = r[0];
    }
    // an expert that was chosen twice gets both choices' gradients, in the order of the choices
    bool twice = false;
#pragma unroll
    for (int q = 1; q <= L / 2; ++q) {
      const int other = __shfl_sync(0xffffffffu, id, (l + q) & (L - 1), L);
      twice |= id >= 0 && other == id;
    }
    if (__any_sync(0xffffffffu, twice)) {
      float sum = 0.f;
#pragma unroll 1
      for (int q = 0; q < L; ++q) {
        const float x = __shfl_sync(0xffffffffu, u, q, L);
        const int other = __shfl_sync(0xffffffffu, id, q, L);
        if (other == id) sum += x;
      }
      u = sum;
    }
    __syncwarp();
    if (id >= 0) o[id] = pj * (fmaf(b.coef != nullptr ? b.weight * b.coef[id] : 0.f, on, -all) + u);
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------- host
// All fields 8 bytes wide, as the Python layer packs them.
struct BalCall {
  int64_t probs, p_stride, ids, id_stride, id64, mask, T, E, k, budget, stream;
};

static int bal_refuse(const char* what, const BalCall& c) {
  if (c.T >= 0 && c.E > 0 && c.E <= B_MAX_E && c.k > 0 && c.k <= B_MAX_K && c.T * c.k <= (1 << 30)) return 0;
  set_last_error_c(what, "1 to 1024 experts, 1 to 32 choices, at most 2^30 choices in all");
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
static bool bal_aligned(const BalCall& c, int w) { return c.E % w == 0 && c.p_stride % w == 0 && c.probs % (4 * w) == 0; }
// Clusters of the forward: one (a single launch) up to B_ALONE probabilities and choices (65536 x 8 with 8 choices alone 21 us, in several
// 12; 5003 x 61 12 us either way, with a launch and an allocation fewer), beyond it two CTAs of 256 threads per SM (65536 x 256: 21 us, with four of them 25, with one of
// 1024 threads 34).  A budget of fewer SMs than a cluster's CTAs still takes one cluster.
constexpr int64_t B_ALONE = 1 << 19;
static int bal_clusters(const BalCall& c) {
  const int64_t work = c.T * (c.E + c.k);
  if (work <= B_ALONE) return 1;
  const int64_t want = work / (1 << 14) / B_CLUSTER, most = 2 * bal_budget(c) / B_CLUSTER;
  const int64_t n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

template <int W, int L, int NV>
static void router_launch(const BalCall& c, const RouterArgs& r) {
  const int64_t warps = (c.T + 32 / L - 1) / (32 / L), blocks = (warps + BT / 32 - 1) / (BT / 32), most = 8ll * bal_budget(c);
  router_bwd_kernel<W, L, NV><<<(unsigned int)(blocks < most ? blocks : most), BT, 0, (cudaStream_t)c.stream>>>(bal_args(c), r);
}
// Vectors of a thread: up to MOST of them.
template <int W, int L, int MOST>
static void router_launch_lanes(const BalCall& c, const RouterArgs& r, int vecs) {
  if (vecs <= 1) router_launch<W, L, 1>(c, r);
  else if (vecs <= 2) router_launch<W, L, 2>(c, r);
  else if (vecs <= 4) router_launch<W, L, 4>(c, r);
  else if (MOST <= 8 || vecs <= 8) router_launch<W, L, MOST < 8 ? MOST : 8>(c, r);
  else if (MOST <= 16 || vecs <= 16) router_launch<W, L, MOST < 16 ? MOST : 16>(c, r);
  else router_launch<W, L, MOST>(c, r);
}
// Threads of a token: as few as hold its row in MOST vectors each and have a choice each; 32 with up to LAST vectors where MOST are too few.
// MOST: 65536 x 256 with vectors of four 46, 32 and 37 us for 2, 4 and 8 of them, 65536 x 255 one by one 55 and 33 us for 8 and 16.
template <int W, int MOST, int LAST>
static void router_launch_wide(const BalCall& c, const RouterArgs& r) {
  const int groups = (int)((c.E + W - 1) / W);
  int lanes = 1;
  while (lanes < 32 && (lanes * MOST < groups || lanes < c.k)) lanes *= 2;
  const int vecs = (groups + lanes - 1) / lanes;
  switch (lanes) {
    case 1: return router_launch_lanes<W, 1, MOST>(c, r, vecs);
    case 2: return router_launch_lanes<W, 2, MOST>(c, r, vecs);
    case 4: return router_launch_lanes<W, 4, MOST>(c, r, vecs);
    case 8: return router_launch_lanes<W, 8, MOST>(c, r, vecs);
    case 16: return router_launch_lanes<W, 16, MOST>(c, r, vecs);
    default: return router_launch_lanes<W, 32, LAST>(c, r, vecs);
  }
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
  // one cluster alone asks for everything itself: with 256 threads each its CTAs took 24 us for 5003 x 61, with 1024 14
  void (*const kernels[2][3])(const BalArgs, float*, int*, float*, int*, float*) = {
      {balance_kernel<1, 1024>, balance_kernel<2, 1024>, balance_kernel<4, 1024>}, {balance_kernel<1, 256>, balance_kernel<2, 256>, balance_kernel<4, 256>}};
  const int width = bal_aligned(c, 4) ? 2 : bal_aligned(c, 2) ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * B_CLUSTER);
  cfg.blockDim = dim3(n > 1 ? 256 : 1024);
  cfg.stream = (cudaStream_t)c.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = B_CLUSTER;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernels[n > 1][width], bal_args(c), psum, pcount, (float*)loss, (int*)counts, (float*)coef);
  if (e == cudaSuccess && n > 1) {
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(1024);
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    e = cudaLaunchKernelEx(&cfg, balance_finish_kernel, (const float*)psum, (const int*)pcount, n, (int)c.E, (int)c.k, (float*)loss, (int*)counts,
                           (float*)coef);
  }
  return bal_rc("dh_balance_fwd", e);
}
// out [T, E] fp32 contiguous, 16-byte aligned.  coef may be null (no balance term).
int dh_router_bwd(const void* call, const void* gates, int64_t g_stride, const void* d_gates, int64_t dg_stride, const void* coef, float weight,
                  void* out) {
  const BalCall& c = *(const BalCall*)call;
  if (int rc = bal_refuse("dh_router_bwd", c)) return rc;
  if (c.T == 0) return 0;
  const RouterArgs r{(const float*)gates, (const float*)d_gates, (const float*)coef, (float*)out, g_stride, dg_stride, weight};
  if (bal_aligned(c, 4) && ((uintptr_t)out & 15) == 0) router_launch_wide<4, 4, 8>(c, r);
  else router_launch_wide<1, 16, 32>(c, r);
  return bal_rc("dh_router_bwd", cudaSuccess);
}

}  // extern "C"
