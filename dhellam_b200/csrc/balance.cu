// Balance loss of a router with per-expert counts, and the gradient of its gates and of the balance loss with respect to its logits.
//
// Over N counted tokens (all, or those whose mask is set) with k choices each among E experts, c_e = choices of e and
// S_e = sum of the probabilities of e:
//   loss = E sum_e (c_e / (N k)) (S_e / N),   d loss / d p[t, e] = E c_e / (N^2 k) on counted tokens, 0 on the others;  N = 0: 0.
// The gates are the chosen probabilities divided by their sum s, so with the gates' gradient dg
//   d p = scatter((dg_j - sum_j dg_j gate_j) / s) + w d loss / d p,    d logit_e = p_e (d p_e - sum_e d p_e p_e).
//
// Sums run in a fixed order (per thread, per CTA, over CTAs), so two calls give the same bits; counts are integers.
#include <cuda_runtime.h>
#include <stdint.h>

#include "api.h"
#include "ptx.cuh"
#include "tmap.h"

namespace dh {

constexpr int BT = 256;              // threads per CTA
constexpr int B_MAX_E = 1024;

__device__ __forceinline__ float bal_warp_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct BalArgs {
  const float* probs;
  long long p_stride;
  const void* ids;
  long long id_stride;
  int id64;
  const uint8_t* mask;
  int T, E, k;
};

__device__ __forceinline__ int bal_id(const BalArgs& a, long long t, int j) {
  if (a.id64) {
    const long long v = reinterpret_cast<const long long*>(a.ids)[t * a.id_stride + j];
    return v < 0 || v >= a.E ? -1 : (int)v;
  }
  const int v = reinterpret_cast<const int*>(a.ids)[t * a.id_stride + j];
  return v < 0 || v >= a.E ? -1 : v;
}

// Partial sums of one CTA's rows: psum [grid, E], pcount [grid, E + 1] (the last one: counted tokens).
__global__ void __launch_bounds__(BT) balance_partial_kernel(const BalArgs a, float* __restrict__ psum, int* __restrict__ pcount) {
  __shared__ int cnt[B_MAX_E + 1];
  __shared__ float red[BT];
  for (int e = threadIdx.x; e <= a.E; e += BT) cnt[e] = 0;
  __syncthreads();
  const int per = (a.T + gridDim.x - 1) / gridDim.x;
  const int t0 = min(a.T, (int)blockIdx.x * per), t1 = min(a.T, t0 + per);
  for (int i = threadIdx.x; i < (t1 - t0) * a.k; i += BT) {
    const int t = t0 + i / a.k, j = i % a.k;
    if (a.mask == nullptr || a.mask[t]) {
      const int e = bal_id(a, t, j);
      if (e >= 0) atomicAdd(&cnt[e], 1);
      if (j == 0) atomicAdd(&cnt[a.E], 1);
    }
  }
  // columns over the threads (as many as the next power of two of E, at most BT), rows over what is left of them
  int cols = 1;
  while (cols < a.E && cols < BT) cols <<= 1;
  const int c = threadIdx.x & (cols - 1), r = threadIdx.x / cols, rows = BT / cols;
  for (int e0 = 0; e0 < a.E; e0 += cols) {
    const int e = e0 + c;
    float s = 0.f;
    if (e < a.E) {
      for (int t = t0 + r; t < t1; t += rows)
        if (a.mask == nullptr || a.mask[t]) s += a.probs[t * a.p_stride + e];
    }
    __syncthreads();
    red[threadIdx.x] = s;
    __syncthreads();
    if (r == 0 && e < a.E) {
      for (int q = 1; q < rows; ++q) s += red[q * cols + c];
      psum[(size_t)blockIdx.x * a.E + e] = s;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= a.E; e += BT) pcount[(size_t)blockIdx.x * (a.E + 1) + e] = cnt[e];
}

__global__ void __launch_bounds__(BT) balance_finish_kernel(const float* __restrict__ psum, const int* __restrict__ pcount, int parts, int E, int k,
                                                            float* __restrict__ loss, int* __restrict__ counts, float* __restrict__ coef) {
  __shared__ float red[BT / 32];
  int n = 0;
  for (int p = 0; p < parts; ++p) n += pcount[(size_t)p * (E + 1) + E];
  const float inv = n > 0 ? 1.f / (float)n : 0.f;
  float part = 0.f;
  for (int e = threadIdx.x; e < E; e += BT) {
    float s = 0.f;
    int c = 0;
    for (int p = 0; p < parts; ++p) {
      s += psum[(size_t)p * E + e];
      c += pcount[(size_t)p * (E + 1) + e];
    }
    const float w = (float)c * inv * inv * ((float)E / (float)k);
    counts[e] = c;
    coef[e] = w;
    part += w * s;
  }
  part = bal_warp_sum(part, 32);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = part;
  __syncthreads();
  if (threadIdx.x == 0) {
    float l = 0.f;
    for (int w = 0; w < BT / 32; ++w) l += red[w];
    *loss = l;
  }
}

// One warp per token.
__global__ void __launch_bounds__(BT) router_bwd_kernel(const BalArgs a, const float* __restrict__ gates, long long g_stride,
                                                        const float* __restrict__ d_gates, long long dg_stride, const float* __restrict__ coef,
                                                        float weight, float* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  for (long long t = (long long)blockIdx.x * (BT / 32) + (threadIdx.x >> 5); t < a.T; t += (long long)gridDim.x * (BT / 32)) {
    const float* p = a.probs + t * a.p_stride;
    const float w = coef != nullptr && (a.mask == nullptr || a.mask[t]) ? weight : 0.f;
    float dot = 0.f, sel = 0.f;
    for (int j = 0; j < a.k; ++j) {
      const int e = bal_id(a, t, j);
      if (e >= 0) {
        dot += d_gates[t * dg_stride + j] * gates[t * g_stride + j];
        sel += p[e];
      }
    }
    const float inv = sel == 0.f ? 0.f : 1.f / sel;
    float all = 0.f;
    for (int e = lane; e < a.E; e += 32) {
      float d = coef != nullptr ? w * coef[e] : 0.f;
      for (int j = 0; j < a.k; ++j)
        if (bal_id(a, t, j) == e) d += (d_gates[t * dg_stride + j] - dot) * inv;
      all += d * p[e];
    }
    all = bal_warp_sum(all, 32);
    for (int e = lane; e < a.E; e += 32) {
      float d = coef != nullptr ? w * coef[e] : 0.f;
      for (int j = 0; j < a.k; ++j)
        if (bal_id(a, t, j) == e) d += (d_gates[t * dg_stride + j] - dot) * inv;
      out[t * a.E + e] = p[e] * (d - all);
    }
  }
}

static int bal_refuse(const char* what, int T, int E, int k) {
  if (T >= 0 && E > 0 && E <= B_MAX_E && k > 0 && (int64_t)T * k < INT32_MAX) return 0;
  set_last_error_c(what, "1 to 1024 experts, at least one choice, fewer than 2^31 choices in all");
  return (int)cudaErrorInvalidValue;
}
static int bal_rc(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c(what, cudaGetErrorString(e));
  return (int)e;
}

}  // namespace dh

using namespace dh;

extern "C" {

// CTAs of the forward over T tokens: rows of its scratch, each E floats and E + 1 ints.
int dh_balance_parts(int T, int E, int sm_budget) {
  const int sms = dh_sm_count();
  const int budget = (sm_budget <= 0 || sm_budget > sms) ? sms : sm_budget;
  const int64_t want = ((int64_t)T * E + 4095) / 4096;
  return want < 1 ? 1 : want < budget ? (int)want : budget;
}
// loss [1] fp32, counts [E] int32, coef [E] fp32 = d loss / d p of a counted token.  scratch: parts * (2 E + 1) words of 4 bytes.
int dh_balance_fwd(const void* probs, int64_t p_stride, const void* ids, int64_t id_stride, int id64, const void* mask, int T, int E, int k,
                   void* scratch, int parts, void* loss, void* counts, void* coef, cudaStream_t s) {
  if (int rc = bal_refuse("dh_balance_fwd", T, E, k)) return rc;
  if (parts <= 0) {
    set_last_error_c("dh_balance_fwd", "no scratch");
    return (int)cudaErrorInvalidValue;
  }
  const BalArgs a{(const float*)probs, p_stride, ids, id_stride, id64, (const uint8_t*)mask, T, E, k};
  float* psum = (float*)scratch;
  int* pcount = (int*)(psum + (size_t)parts * E);
  balance_partial_kernel<<<parts, BT, 0, s>>>(a, psum, pcount);
  balance_finish_kernel<<<1, BT, 0, s>>>(psum, pcount, parts, E, k, (float*)loss, (int*)counts, (float*)coef);
  return bal_rc("dh_balance_fwd");
}
// out [T, E] fp32 contiguous.  coef may be null (no balance term).
int dh_router_bwd(const void* probs, int64_t p_stride, const void* ids, int64_t id_stride, int id64, const void* mask, const void* gates,
                  int64_t g_stride, const void* d_gates, int64_t dg_stride, const void* coef, float weight, void* out, int T, int E, int k,
                  int sm_budget, cudaStream_t s) {
  if (int rc = bal_refuse("dh_router_bwd", T, E, k)) return rc;
  if (T == 0) return 0;
  const BalArgs a{(const float*)probs, p_stride, ids, id_stride, id64, (const uint8_t*)mask, T, E, k};
  const int sms = dh_sm_count();
  const int budget = (sm_budget <= 0 || sm_budget > sms) ? sms : sm_budget;
  const int64_t blocks = ((int64_t)T + BT / 32 - 1) / (BT / 32);
  const int grid = (int)(blocks < (int64_t)budget * 8 ? blocks : (int64_t)budget * 8);
  router_bwd_kernel<<<grid, BT, 0, s>>>(a, (const float*)gates, g_stride, (const float*)d_gates, dg_stride, (const float*)coef, weight, (float*)out);
  return bal_rc("dh_router_bwd");
}

}  // extern "C"
