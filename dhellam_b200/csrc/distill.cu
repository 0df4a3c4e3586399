// Cross entropy and distillation from a teacher's top logits over vocabulary shards, forward statistics and gradient.
//
// A row has student logits z over V entries (a shard of them here), a label (or none) and the teacher's best K entries: ids and
// logits t.  With temperature tau, q = softmax(t / tau) over the row's entries (an id outside [0, V) is padding, without weight) and
// p = softmax(z / tau) over the whole vocabulary,
//   ce = lse(z) - z_label,     kd = tau^2 (sum_j q_j log q_j - sum_j q_j z_{id_j} / tau + lse(z / tau)),
//   d z = g_ce (softmax(z) - onehot(label)) + g_kd tau (p - sum_j q_j onehot(id_j)).
// A label outside [0, V) gives ce = 0 and no gradient, a row without entries kd = 0 and none, a row whose logits are all -inf neither
// loss nor gradient.  An id may stand twice; its weights add.
//
// Forward: one pass over the shard gives per row the maximum m, sum exp(z - m), sum exp((z - m) / tau), the label's and the chosen
// entries' logits relative to m: eight numbers that the ranks exchange at once and one small kernel combines.  Sums are fp32.
// Backward: one pass computes every element from (m, lse, lse at tau) and the few entries with a label or a teacher's weight are
// written once more behind it, from logits read before it, so that each element is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "api.h"
#include "ptx.cuh"
#include "tmap.h"

namespace dh {

constexpr int DT = 256;
constexpr int D_MAX_K = 1024;
constexpr float D_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float d_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float d_max(float a, float b) { return (a > b || a != a) ? a : b; }      // a NaN stays
__device__ __forceinline__ float d_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = d_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// Over the CTA; every thread gets the result.  `red`: 32 floats, free again behind the next barrier.
__device__ __forceinline__ float d_block_sum(float v, float* red) {
  v = d_warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return d_warp_sum((threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f);
}
__device__ __forceinline__ float d_block_max(float v, float* red) {
  v = d_warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return d_warp_max((threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : -INFINITY);
}

struct DistillArgs {
  const void* z;                   // [T, Vl], row stride ld
  long long ld;
  const int* labels;               // nullable
  const void* ids;                 // [T, K] int32 or int64
  long long id_stride;
  const void* t;                   // [T, K]
  long long t_stride;
  int id64, t_type;                // t_type: 0 bf16, 1 fp32, 2 fp16
  int T, Vl, K, v0, V;
  float inv_tau;
};

__device__ __forceinline__ float d_load(const float* p) { return *p; }
__device__ __forceinline__ float d_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void d_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void d_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float d_teacher(const DistillArgs& a, long long row, int j) {
  const long long i = row * a.t_stride + j;
  if (a.t_type == 1) return reinterpret_cast<const float*>(a.t)[i];
  if (a.t_type == 0) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.t)[i]);
  return __half2float(reinterpret_cast<const __half*>(a.t)[i]);
}
// The vocabulary entry of the teacher's j-th logit, -1 for padding.
__device__ __forceinline__ int d_id(const DistillArgs& a, long long row, int j) {
  const long long i = row * a.id_stride + j;
  const long long v = a.id64 ? reinterpret_cast<const long long*>(a.ids)[i] : (long long)reinterpret_cast<const int*>(a.ids)[i];
  return v < 0 || v >= a.V ? -1 : (int)v;
}

// Eight numbers per row: m, sum exp(z - m), sum exp((z - m) / tau), z_label - m (0: not in this shard), sum q (z_id - m) and sum q over
// the entries in this shard, sum q log q (+inf: the row has no entries), 1 if the label is in this shard.
template <typename T>
__global__ void __launch_bounds__(DT) distill_stats_kernel(const DistillArgs a, float* __restrict__ stats, float* __restrict__ teacher_lse) {
  __shared__ float red[32];
  for (int row = blockIdx.x; row < a.T; row += gridDim.x) {
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
    float m = -FLT_MAX, s = 0.f, st = 0.f;
    for (int c = threadIdx.x; c < a.Vl; c += DT) {
      const float v = d_load(z + c);
      if (v > m) {
        s *= exp2f((m - v) * D_LOG2E);
        st *= exp2f((m - v) * D_LOG2E * a.inv_tau);
        m = v;
      }
      const float x = (v - m) * D_LOG2E;
      s += exp2f(x);
      st += exp2f(x * a.inv_tau);
    }
    const float gm = d_block_max(m, red);
    s = d_block_sum(s * exp2f((m - gm) * D_LOG2E), red);
    st = d_block_sum(st * exp2f((m - gm) * D_LOG2E * a.inv_tau), red);
    // the teacher's distribution over the row's entries
    float tm = -INFINITY;
    for (int j = threadIdx.x; j < a.K; j += DT)
      if (d_id(a, row, j) >= 0) tm = d_max(tm, d_teacher(a, row, j));
    tm = d_block_max(tm, red);
    const bool some = tm != -INFINITY;
    float w = 0.f;
    if (some)
      for (int j = threadIdx.x; j < a.K; j += DT)
        if (d_id(a, row, j) >= 0) w += expf((d_teacher(a, row, j) - tm) * a.inv_tau);
    w = d_block_sum(w, red);
    const float lw = logf(w);
    float dot = 0.f, own = 0.f, ent = 0.f;
    if (some)
      for (int j = threadIdx.x; j < a.K; j += DT) {
        const int id = d_id(a, row, j);
        if (id < 0) continue;
        const float lq = (d_teacher(a, row, j) - tm) * a.inv_tau - lw;
        const float q = expf(lq);
        if (q == 0.f) continue;                          // no weight: its logit may be infinite
        ent += q * lq;
        const int loc = id - a.v0;
        if (loc >= 0 && loc < a.Vl) {
          dot += q * (d_load(z + loc) - gm);
          own += q;
        }
      }
    dot = d_block_sum(dot, red);
    own = d_block_sum(own, red);
    ent = d_block_sum(ent, red);
    if (threadIdx.x == 0) {
      const int lab = a.labels != nullptr ? a.labels[row] : -1;
      const int loc = lab >= 0 && lab < a.V ? lab - a.v0 : -1;
      const bool in = loc >= 0 && loc < a.Vl;
      float4* o = reinterpret_cast<float4*>(stats + (size_t)row * 8);
      o[0] = make_float4(gm, s, st, in ? d_load(z + loc) - gm : 0.f);
      o[1] = make_float4(dot, own, some ? ent : INFINITY, in ? 1.f : 0.f);
      teacher_lse[row] = some ? tm * a.inv_tau + lw : INFINITY;
    }
  }
}

// stats [R, T, 8] of the ranks -> ce [T] (nullable), kd [T], saved [T, 4] = (m, lse(z) or +inf where ce has no gradient, lse(z / tau),
// the teacher's lse at tau or +inf where kd has none).
__global__ void __launch_bounds__(DT) distill_combine_kernel(const float4* __restrict__ stats, const float* __restrict__ teacher_lse, int R, int T,
                                                             float tau, float* __restrict__ ce, float* __restrict__ kd, float4* __restrict__ saved) {
  const int t = blockIdx.x * DT + threadIdx.x;
  if (t >= T) return;
  float m = stats[(size_t)t * 2].x;
  for (int r = 1; r < R; ++r) m = d_max(m, stats[((size_t)r * T + t) * 2].x);
  const float it = 1.f / tau;
  float s = 0.f, st = 0.f, target = 0.f, has = 0.f, dot = 0.f, ent = 0.f;
  for (int r = 0; r < R; ++r) {
    const float4 u = stats[((size_t)r * T + t) * 2], v = stats[((size_t)r * T + t) * 2 + 1];
    const float d = u.x - m;
    s += u.y * expf(d);
    st += u.z * expf(d * it);
    if (v.w != 0.f) { target += u.w + d; has = 1.f; }
    if (v.y != 0.f) dot += v.x + v.y * d;
    ent = v.z;
  }
  const float l = logf(s), lt = logf(st);
  const bool hard = has != 0.f && s != 0.f, soft = ent != INFINITY && s != 0.f;      // s = 0: all logits are -inf
  if (ce != nullptr) ce[t] = hard ? l - target : 0.f;
  kd[t] = soft ? tau * tau * (ent - dot * it + lt) : 0.f;
  saved[t] = make_float4(m, hard ? l + m : INFINITY, lt + m * it, soft ? teacher_lse[t] : INFINITY);
}

// out = d loss / d z; out may be z.  One CTA per row.
template <typename T>
__global__ void __launch_bounds__(DT) distill_grad_kernel(const DistillArgs a, const float4* __restrict__ saved, const float* __restrict__ g_ce,
                                                          const float* __restrict__ g_kd, float tau, void* out, long long out_ld) {
  __shared__ int ids[D_MAX_K + 1];          // entries of this shard that get more than the softmax: the teacher's, then the label
  __shared__ float add[D_MAX_K + 1], at[D_MAX_K + 1];
  for (int row = blockIdx.x; row < a.T; row += gridDim.x) {
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
    T* o = reinterpret_cast<T*>(out) + row * out_ld;
    const float4 sv = saved[row];
    const bool some = sv.w != INFINITY;
    const int lab = a.labels != nullptr ? a.labels[row] : -1;
    const bool hard = a.labels != nullptr && sv.y != INFINITY;
    const float gc = hard ? g_ce[row] : 0.f, gk = some ? g_kd[row] * tau : 0.f;
    __syncthreads();
    for (int j = threadIdx.x; j <= a.K; j += DT) {
      int loc = -1;
      float w = 0.f;
      if (j == a.K) {
        if (hard) { loc = lab - a.v0; w = gc; }
      } else if (gk != 0.f) {
        const int id = d_id(a, row, j);
        if (id >= 0) { loc = id - a.v0; w = gk * expf(d_teacher(a, row, j) * a.inv_tau - sv.w); }
      }
      const bool in = loc >= 0 && loc < a.Vl;
      ids[j] = in ? loc : -1;
      add[j] = w;
      at[j] = in ? d_load(z + loc) : 0.f;
    }
    __syncthreads();
    if (gc == 0.f && gk == 0.f) {             // a token without loss: zeros, whatever its logits
      for (int c = threadIdx.x; c < a.Vl; c += DT) d_store(o + c, 0.f);
      continue;
    }
    auto soft = [&](float v) {
      float g = 0.f;
      if (gc != 0.f) g += gc * expf(v - sv.y);
      if (gk != 0.f) g += gk * expf(v * a.inv_tau - sv.z);
      return g;
    };
    for (int c = threadIdx.x; c < a.Vl; c += DT) d_store(o + c, soft(d_load(z + c)));
    __syncthreads();
    for (int j = threadIdx.x; j <= a.K; j += DT) {
      const int id = ids[j];
      if (id < 0) continue;
      bool first = true;
      float w = add[j];
      for (int i = 0; i <= a.K; ++i) {
        if (i == j || ids[i] != id) continue;
        if (i < j) first = false;
        else w += add[i];
      }
      if (first) d_store(o + id, soft(at[j]) - w);
    }
  }
}

static int d_refuse(const char* what, int T, int Vl, int K, int v0, int V, float inv_tau) {
  if (T >= 0 && Vl > 0 && K >= 0 && K <= D_MAX_K && v0 >= 0 && V >= v0 + (int64_t)Vl && inv_tau > 0.f && inv_tau <= FLT_MAX) return 0;
  set_last_error_c(what, "a shard inside the vocabulary, at most 1024 teacher's entries, a positive temperature");
  return (int)cudaErrorInvalidValue;
}
static int d_rc(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c(what, cudaGetErrorString(e));
  return (int)e;
}
static int d_grid(int64_t rows, int sm_budget) {
  const int sms = dh_sm_count();
  const int budget = (sm_budget <= 0 || sm_budget > sms) ? sms : sm_budget;
  return (int)(rows < (int64_t)budget * 8 ? rows : (int64_t)budget * 8);
}

}  // namespace dh

using namespace dh;

extern "C" {

// stats [T, 8] and teacher_lse [T], fp32; logits bf16 or fp32 (f32).
int dh_distill_stats(const void* z, int64_t ld, int f32, const void* labels, const void* ids, int64_t id_stride, int id64, const void* t,
                     int64_t t_stride, int t_type, int T, int Vl, int K, int v0, int V, float tau, void* stats, void* teacher_lse, int sm_budget,
                     cudaStream_t s) {
  if (int rc = d_refuse("dh_distill_stats", T, Vl, K, v0, V, 1.f / tau)) return rc;
  if (T == 0) return 0;
  const DistillArgs a{z, ld, (const int*)labels, ids, id_stride, t, t_stride, id64, t_type, T, Vl, K, v0, V, 1.f / tau};
  if (f32) distill_stats_kernel<float><<<d_grid(T, sm_budget), DT, 0, s>>>(a, (float*)stats, (float*)teacher_lse);
  else distill_stats_kernel<__nv_bfloat16><<<d_grid(T, sm_budget), DT, 0, s>>>(a, (float*)stats, (float*)teacher_lse);
  return d_rc("dh_distill_stats");
}
int dh_distill_combine(const void* stats, const void* teacher_lse, int R, int T, float tau, void* ce, void* kd, void* saved, cudaStream_t s) {
  if (R <= 0 || T <= 0) return 0;
  distill_combine_kernel<<<(T + DT - 1) / DT, DT, 0, s>>>((const float4*)stats, (const float*)teacher_lse, R, T, tau, (float*)ce, (float*)kd,
                                                          (float4*)saved);
  return d_rc("dh_distill_combine");
}
int dh_distill_grad(const void* z, int64_t ld, int f32, const void* labels, const void* ids, int64_t id_stride, int id64, const void* t,
                    int64_t t_stride, int t_type, int T, int Vl, int K, int v0, int V, float tau, const void* saved, const void* g_ce,
                    const void* g_kd, void* out, int64_t out_ld, int sm_budget, cudaStream_t s) {
  if (int rc = d_refuse("dh_distill_grad", T, Vl, K, v0, V, 1.f / tau)) return rc;
  if (T == 0) return 0;
  const DistillArgs a{z, ld, (const int*)labels, ids, id_stride, t, t_stride, id64, t_type, T, Vl, K, v0, V, 1.f / tau};
  if (f32) distill_grad_kernel<float><<<d_grid(T, sm_budget), DT, 0, s>>>(a, (const float4*)saved, (const float*)g_ce, (const float*)g_kd, tau, out, out_ld);
  else distill_grad_kernel<__nv_bfloat16><<<d_grid(T, sm_budget), DT, 0, s>>>(a, (const float4*)saved, (const float*)g_ce, (const float*)g_kd, tau, out, out_ld);
  return d_rc("dh_distill_grad");
}

}  // extern "C"
