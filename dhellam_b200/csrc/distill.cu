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
// Forward: one pass over the shard.  A thread's sums of exponentials are relative to a reference m that is the maximum of what it has
// seen or up to D_RISE / log2 e below it: it moves only when an element rises further, so the rescaling leaves the loop and no term is
// below what its own rounding loses.  Exponentials are 2^(z c - R) in one fma, with c = log2 e or log2 e / tau and R = m c rounded; the
// rounding of R is taken out of the sum when the thread is done.  A row whose maximum is
// beyond D_FAR powers of two (the type's lowest value everywhere) has a slow form, the difference first.  The teacher's sums are linear in
// exp(t / tau), so a row needs two rounds of reductions in all; CTAs that share a row join their maxima in the first.  Sums are fp32.
// Backward: one pass computes every element from m, 1 / sum and 1 / sum at tau, and the few entries with a label or a teacher's weight are
// written once more behind it, from logits read before it, so that each element is rounded once.
//
// With both losses an element costs two exponentials, unless tau is 1 (they are the same) or 2 or 4 (exp(x) is a power of exp(x / tau):
// one or two products).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "api.h"
#include "ptx.cuh"
#include "tmap.h"

namespace dh {

constexpr int D_MAX_K = 1024;
constexpr int D_AHEAD = 2;               // entries of a thread that the forward asks for at a time
constexpr int D_BATCH = 4;               // 16-byte loads of a thread at a time
constexpr float D_LOG2E = 1.4426950408889634f;
constexpr float D_LN2 = 0.6931471805599453f;
constexpr float D_FAR = 2097152.f;       // references of the fast form are that far from zero at most, in powers of two: 1/8 is what R is off by
constexpr float D_RISE = 8.f;            // in powers of two; 2^-24 of it is what an exponent loses at most by a reference that is too low

// Which exponentials an element needs: ONE (a single sum), TWO (both, on their own), SQUARE and FOURTH (tau = 2, 4).
enum { D_ONE = 0, D_TWO = 1, D_SQUARE = 2, D_FOURTH = 3 };

struct DistillArgs {
  const void* z;                   // [T, Vl], row stride ld
  const int* labels;               // nullable
  const void* ids;                 // [T, K] int32 or int64
  const void* t;                   // [T, K]
  int64_t ld, id_stride, t_stride;
  int id64, t_type;                // t_type: 0 bf16, 1 fp32, 2 fp16
  int T, Vl, K, v0, V;
  float tau, inv_tau;
};

__device__ __forceinline__ void d_copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ float d_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float d_max(float a, float b) { return (a > b || a != a) ? a : b; }      // a NaN stays
__device__ __forceinline__ float d_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float d_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = d_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Two fp32 in one register pair: the packed forms of add, multiply and fma need one issue slot for two elements.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_get(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 f2_ex2(F2 a) {
  const float2 x = f2_get(a);
  return f2(d_ex2(x.x), d_ex2(x.y));
}

// 2^x on the FMA pipe, for x up to 127 and (as 2^-126) below -126: x = n + f with |f| <= 1/2 by adding 1.5 x 2^23 (+ 127, so that the sum's
// low bits are the exponent field of 2^n), and a polynomial of degree 5 for 2^f (own minimax fit by Remez' exchange, relative error
// 2.1e-7 in fp32; the special function's bound is 2.4e-7).  A NaN stays.
__device__ __forceinline__ float d_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2_ex2_fma(F2 a) {
  const float2 x = f2_get(a);
  const F2 c = f2(d_max_nan(x.x, -126.f), d_max_nan(x.y, -126.f));
  const F2 t = c + f2(12583039.f, 12583039.f);
  const F2 f = f2_fma(t + f2(-12583039.f, -12583039.f), f2(-1.f, -1.f), c);
  F2 p = f2_fma(f, f2(0.0013277939287945628f, 0.0013277939287945628f), f2(0.009675757959485054f, 0.009675757959485054f));
  p = f2_fma(p, f, f2(0.05550709739327431f, 0.05550709739327431f));
  p = f2_fma(p, f, f2(0.24022114276885986f, 0.24022114276885986f));
  p = f2_fma(p, f, f2(0.6931469440460205f, 0.6931469440460205f));
  p = f2_fma(p, f, f2(1.0000001192092896f, 1.0000001192092896f));
  const float2 n = f2_get(t);
  return p * f2(__int_as_float(__float_as_int(n.x) << 23), __int_as_float(__float_as_int(n.y) << 23));
}

// 16 bytes of logits as pairs of fp32, and their largest.
template <typename T> struct DVec;
template <> struct DVec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static __forceinline__ void unpack(const uint4& u, F2 (&x)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ static __forceinline__ uint4 pack(const F2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = f2_get(x[i]); w[i] = pack_bf16x2(f.x, f.y); }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static __forceinline__ float largest(const uint4 (&u)[D_BATCH]) {
    __nv_bfloat162 m = __hmax2(as2(u[0].x), as2(u[0].y));
    m = __hmax2(m, __hmax2(as2(u[0].z), as2(u[0].w)));
#pragma unroll
    for (int i = 1; i < D_BATCH; ++i) {
      m = __hmax2(m, __hmax2(as2(u[i].x), as2(u[i].y)));
      m = __hmax2(m, __hmax2(as2(u[i].z), as2(u[i].w)));
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ static __forceinline__ __nv_bfloat162 as2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
};
template <> struct DVec<float> {
  static constexpr int N = 4;
  __device__ static __forceinline__ void unpack(const uint4& u, F2 (&x)[2]) {
    x[0] = f2(__uint_as_float(u.x), __uint_as_float(u.y));
    x[1] = f2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  __device__ static __forceinline__ uint4 pack(const F2 (&x)[2]) {
    const float2 a = f2_get(x[0]), b = f2_get(x[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  }
  __device__ static __forceinline__ float largest(const uint4 (&u)[D_BATCH]) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < D_BATCH; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u[i].x), __uint_as_float(u[i].y)), fmaxf(__uint_as_float(u[i].z), __uint_as_float(u[i].w))));
    return m;
  }
};

__device__ __forceinline__ float d_load(const float* p) { return *p; }
__device__ __forceinline__ float d_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void d_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void d_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }

__device__ __forceinline__ float d_teacher(const DistillArgs& a, int64_t row, int j) {
  const int64_t i = row * a.t_stride + j;
  if (a.t_type == 1) return reinterpret_cast<const float*>(a.t)[i];
  if (a.t_type == 0) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.t)[i]);
  return __half2float(reinterpret_cast<const __half*>(a.t)[i]);
}
// The vocabulary entry of the teacher's j-th logit, -1 for padding.
__device__ __forceinline__ int d_id(const DistillArgs& a, int64_t row, int j) {
  const int64_t i = row * a.id_stride + j;
  const int64_t v = a.id64 ? reinterpret_cast<const int64_t*>(a.ids)[i] : (int64_t)reinterpret_cast<const int*>(a.ids)[i];
  return v < 0 || v >= a.V ? -1 : (int)v;
}

// Entries j, j + DT, ... of a row: ids (-1: padding or none) and logits.
template <int DT, int N>
__device__ __forceinline__ void d_entries(const DistillArgs& a, int64_t row, int j, int (&id)[N], float (&t)[N]) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    id[u] = -1;
    t[u] = 0.f;
    if (j + u * DT < a.K) { id[u] = d_id(a, row, j + u * DT); t[u] = d_teacher(a, row, j + u * DT); }
  }
}

// A row's elements in 16-byte vectors of the memory they lie in: `lead` elements before the first, then `vecs`, the rest behind them.
// Part p of n: vectors [v0, v1), the lead with the first part, the rest with the last.
struct DSpan {
  int lead, vecs, v0, v1, c0, c1;        // c0, c1: this part's elements
};
template <typename T>
__device__ __forceinline__ DSpan d_span(const T* row, int n, int part, int parts) {
  constexpr int N = DVec<T>::N;
  DSpan s;
  s.lead = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
  s.vecs = (n - s.lead) / N;
  s.v0 = (int)((int64_t)s.vecs * part / parts);
  s.v1 = (int)((int64_t)s.vecs * (part + 1) / parts);
  s.c0 = part == 0 ? 0 : s.lead + s.v0 * N;
  s.c1 = part == parts - 1 ? n : s.lead + s.v1 * N;
  return s;
}

// Sums of one thread relative to its reference.
template <int MODE>
struct DSums {
  float m, r1, rt;                                 // reference, rounded m c1 and m ct
  F2 s1 = f2(0.f, 0.f), st = f2(0.f, 0.f);         // ONE: st alone
  __device__ __forceinline__ void refer(float to, float c1, float ct) {
    m = to;
    rt = to * ct;
    r1 = MODE == D_SQUARE ? 2.f * rt : MODE == D_FOURTH ? 4.f * rt : to * c1;
  }
  __device__ __forceinline__ void raise(float to, float c1, float ct) {
    const float o1 = r1, ot = rt;
    refer(to, c1, ct);
    const float f = d_ex2(ot - rt);
    st = st * f2(f, f);
    if (MODE != D_ONE) {
      const float g = d_ex2(o1 - r1);
      s1 = s1 * f2(g, g);
    }
  }
  // F1: a second exponential of its own on the FMA pipe
  template <bool F1>
  __device__ __forceinline__ void add(F2 z, F2 n1, F2 nt, F2 c1, F2 ct) {
    const F2 e = f2_ex2(f2_fma(z, ct, nt));
    st = st + e;
    if (MODE == D_TWO) {
      const F2 x = f2_fma(z, c1, n1);
      s1 = s1 + (F1 ? f2_ex2_fma(x) : f2_ex2(x));
    }
    if (MODE == D_SQUARE) s1 = f2_fma(e, e, s1);
    if (MODE == D_FOURTH) { const F2 q = e * e; s1 = f2_fma(q, q, s1); }
  }
  // The sums relative to m itself.
  __device__ __forceinline__ void finish(float c1, float ct, float& a1, float& at) const {
    const float2 p = f2_get(s1), q = f2_get(st);
    at = (q.x + q.y) * d_ex2(-fmaf(m, ct, -rt));
    a1 = MODE == D_ONE ? 0.f : (p.x + p.y) * d_ex2(-fmaf(m, c1, -r1));
  }
};

// What a row's sums give.  m: reference; s1, st: sums; target: z_label - m (+inf: no label here); dot, own: sums of q (z_id - m) and of q
// over the entries here; ent: sum of q log q (+inf: the row has no entries); tm, lv: the teacher's largest logit and log of its sum relative
// to that.  Differences of logits carry no factor: they may be as large as the type's lowest value.
// saved [4] pairs: (m, 0), (1 / s1 or 0 where ce has no gradient, 0), (1 / st, 0), (lv or +inf where kd has no gradient, tm).  tm / tau + lv
// in one number would lose lv where a row's logits are far from zero.
__device__ __forceinline__ void d_finish(float m, float s1, float st, float target, float dot, float ent, float lv, float tm, float tau, float* ce,
                                         float* kd, float4* saved) {
  const bool hard = target != INFINITY && s1 != 0.f, soft = ent != INFINITY && st != 0.f;      // a sum of 0: all logits are -inf
  if (ce != nullptr) *ce = hard ? D_LN2 * log2f(s1) - target : 0.f;
  *kd = soft ? tau * (tau * (ent + D_LN2 * log2f(st)) - dot) : 0.f;
  saved[0] = make_float4(m, 0.f, hard ? 1.f / s1 : 0.f, 0.f);
  saved[1] = make_float4(soft ? 1.f / st : 0.f, 0.f, soft ? lv : INFINITY, tm);
}

// One cluster of CTAs per row (one CTA where there are rows enough); they share its vectors and the first one joins their sums.  CTAs
// that stay and ask for the next row's logits while they reduce are slower (4096 x 128256: 182 us, 207 so): SMs are not equally far from
// the memory, and whoever is done takes the next row.  Bound by memory: 180 us without the exponentials.
// Where `stats` is given (the vocabulary is divided among ranks) a row's numbers go there: m, s1, st, target, dot, own, ent, 0; and what is the
// same on every rank, lv and tm, to `saved`.
template <typename T, int MODE, int DT>
__global__ void __launch_bounds__(DT, 1024 / DT) distill_fwd_kernel(const DistillArgs a, int parts, float* __restrict__ ce, float* __restrict__ kd,
                                                            float4* __restrict__ saved, float4* __restrict__ stats) {
  constexpr int N = DVec<T>::N, DW = DT / 32, STAGE = D_BATCH * DT;
  extern __shared__ __align__(16) uint4 d_ring[];          // [2][D_BATCH][DT]: a thread's vectors pass through its own slots
  __shared__ float red[2][DW];
  __shared__ float sums[DW][6];
  __shared__ float join[4];                          // for the cluster: this CTA's maximum (fast and slow form), s1, st
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % parts;
  const float ct = D_LOG2E * a.inv_tau, c1 = D_LOG2E;
  const float cr = MODE == D_ONE ? ct : fmaxf(c1, ct), far = D_FAR / cr;
  const F2 c1p = f2(c1, c1), ctp = f2(ct, ct);
  uint4* const ring = d_ring + threadIdx.x;

  const uint4* src;                                  // this thread's next vector to ask for
  int full, left;                                    // batches of which every thread has all vectors, this thread's vectors behind them
  auto fetch = [&](int k, int stage) {
    if (k < full) {
#pragma unroll
      for (int b = 0; b < D_BATCH; ++b) d_copy16(ring + stage + b * DT, src + b * DT);
    } else if (k == full) {
#pragma unroll
      for (int b = 0; b < D_BATCH; ++b)
        if (b < left) d_copy16(ring + stage + b * DT, src + b * DT);
    }
    src += STAGE;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int row = blockIdx.x / parts; row < a.T; row += gridDim.x / parts) {
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
    const DSpan sp = d_span(z, a.Vl, part, parts);
    full = (sp.v1 - sp.v0) / STAGE;
    left = (sp.v1 - (sp.v0 + full * STAGE + (int)threadIdx.x) + DT - 1) / DT;
    src = reinterpret_cast<const uint4*>(z + sp.lead) + sp.v0 + threadIdx.x;
    fetch(0, 0);
    fetch(1, STAGE);
    // what a row's end needs is on its way before its logits are added up
    int id0 = -1, lab = -1;
    float t0 = 0.f;
    if (part == 0) {
      if ((int)threadIdx.x < a.K) { id0 = d_id(a, row, threadIdx.x); t0 = d_teacher(a, row, threadIdx.x); }
      if (threadIdx.x == 0 && a.labels != nullptr) lab = a.labels[row];
    }
    DSums<MODE> acc;
    acc.refer(-far, c1, ct);               // what lies below counts only where nothing lies above: the slow form
    auto batch = [&](int stage, int count) {
      uint4 u[D_BATCH];
#pragma unroll
      for (int b = 0; b < D_BATCH; ++b) u[b] = ring[stage + (b < count ? b : 0) * DT];
      const float lm = DVec<T>::largest(u);
      if ((lm - acc.m) * cr > D_RISE) acc.raise(lm, c1, ct);
      const F2 n1 = f2(-acc.r1, -acc.r1), nt = f2(-acc.rt, -acc.rt);
#pragma unroll
      for (int b = 0; b < D_BATCH; ++b) {
        if (b >= count) continue;
        F2 x[N / 2];
        DVec<T>::unpack(u[b], x);
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
          // of two exponentials of their own a quarter goes to the FMA pipe: none, 1/8, 1/4, 3/8 of them 264, 246, 238, 256 us
          // (4096 x 128256, tau 1.5); of a single one none (a quarter: 182 -> 195 us)
          if (N == 8 && j < 2) acc.template add<true>(x[j], n1, nt, c1p, ctp);
          else acc.template add<false>(x[j], n1, nt, c1p, ctp);
        }
      }
    };
    int stage = 0;
    for (int k = 0; k < full; ++k, stage = STAGE - stage) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      batch(stage, D_BATCH);
      fetch(k + 2, stage);
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (left > 0) batch(stage, left);
    const float z0 = id0 - a.v0 >= 0 && id0 - a.v0 < a.Vl ? d_load(z + (id0 - a.v0)) : 0.f;
    const int lloc = lab >= 0 && lab < a.V ? lab - a.v0 : -1;
    const bool lin = lloc >= 0 && lloc < a.Vl;
    const float zl = lin ? d_load(z + lloc) : 0.f;
    float s1, st;
    acc.finish(c1, ct, s1, st);
    // elements one by one: before the first and behind the last vector
    auto single = [&](int c) {
      const float v = d_load(z + c);
      if ((v - acc.m) * cr > D_RISE) {
        s1 *= d_ex2((acc.m - v) * c1);
        st *= d_ex2((acc.m - v) * ct);
        acc.m = v;
      }
      st += d_ex2((v - acc.m) * ct);
      if (MODE != D_ONE) s1 += d_ex2((v - acc.m) * c1);
    };
    const int tail = sp.lead + sp.vecs * N + (int)threadIdx.x;
    if (part == 0 && (int)threadIdx.x < sp.lead) single(threadIdx.x);
    if (part == parts - 1 && tail < a.Vl) single(tail);
    // first round: the row's reference, which all CTAs that share the row take before they form anything relative to it (their own
    // shares may lie far below: a masked part of the vocabulary; the exchange takes 0.3 to 0.8 us, 17 x 128256: 7.3 -> 7.8 us), and the
    // teacher's largest logit
    float tm = -INFINITY;
    if (id0 >= 0) tm = t0;
    if (part == 0)
      for (int j = threadIdx.x + DT; j < a.K; j += D_AHEAD * DT) {
        int id[D_AHEAD];
        float t[D_AHEAD];
        d_entries<DT>(a, row, j, id, t);
#pragma unroll
        for (int u = 0; u < D_AHEAD; ++u)
          if (id[u] >= 0) tm = d_max(tm, t[u]);
      }
    float m, top;
    auto round = [&](int slot) {
      const float wm = d_warp_max(acc.m), wt = d_warp_max(tm);
      if (lane == 0) { red[0][w] = wm; red[1][w] = wt; }
      __syncthreads();
      m = red[0][0];
      top = red[1][0];
#pragma unroll
      for (int q = 1; q < DW; ++q) { m = d_max(m, red[0][q]); top = d_max(top, red[1][q]); }
      if (parts > 1) {
        if (threadIdx.x == 0) join[slot] = m;
        __syncwarp();
        cluster_sync_all();
        m = d_warp_max(lane < parts ? __uint_as_float(ld_cluster_u32(mapa_u32(smem_u32(join + slot), lane))) : -INFINITY);
      }
    };
    round(0);
    if (!(m > -far && m < far)) {
      acc.m = -FLT_MAX;
      s1 = st = 0.f;
      for (int c = sp.c0 + threadIdx.x; c < sp.c1; c += DT) single(c);
      __syncthreads();
      round(1);
    }
    tm = top;
    // second round: the sums; the teacher's relative to its largest
    float v[6] = {s1 * d_ex2((acc.m - m) * c1), st * d_ex2((acc.m - m) * ct), 0.f, 0.f, 0.f, 0.f};
    if (part == 0 && tm != -INFINITY) {
      auto entry = [&](int id, float t, float zj) {
        if (id < 0) return;
        const float lt = (t - tm) * a.inv_tau, q = expf(lt);
        if (q == 0.f) return;                            // no weight: its logit may be infinite
        v[2] += q;
        v[3] += q * lt;
        if (id - a.v0 >= 0 && id - a.v0 < a.Vl) {
          v[4] += q * ((zj - m) * (1.f / D_MAX_K));        // a power of two: the sum of all entries stays finite
          v[5] += q;
        }
      };
      entry(id0, t0, z0);
      for (int j = threadIdx.x + DT; j < a.K; j += D_AHEAD * DT) {
        int id[D_AHEAD];
        float t[D_AHEAD], zj[D_AHEAD];
        d_entries<DT>(a, row, j, id, t);
#pragma unroll
        for (int u = 0; u < D_AHEAD; ++u) zj[u] = id[u] - a.v0 >= 0 && id[u] - a.v0 < a.Vl ? d_load(z + (id[u] - a.v0)) : 0.f;
#pragma unroll
        for (int u = 0; u < D_AHEAD; ++u) entry(id[u], t[u], zj[u]);
      }
    }
#pragma unroll
    for (int q = 0; q < 6; ++q) v[q] = d_warp_sum(v[q]);
    if (lane == 0) {
#pragma unroll
      for (int q = 0; q < 6; ++q) sums[w][q] = v[q];
    }
    __syncthreads();
    if (w == 0) {
      float t = 0.f;
      if (lane < 6) {
#pragma unroll
        for (int q = 0; q < DW; ++q) t += sums[q][lane];
      }
#pragma unroll
      for (int q = 0; q < 6; ++q) v[q] = __shfl_sync(0xffffffffu, t, q);
      if (lane == 0 && parts > 1) { join[2] = v[0]; join[3] = v[1]; }
    }
    __syncwarp();
    if (parts > 1) cluster_sync_all();
    if (part == 0 && threadIdx.x == 0) {
      float dot = v[4], own = v[5];
      const float target = lin ? zl - m : INFINITY;
      for (int r = 1; r < parts; ++r) {
        const uint32_t at = mapa_u32(smem_u32(join), r);
        v[0] += __uint_as_float(ld_cluster_u32(at + 8));
        v[1] += __uint_as_float(ld_cluster_u32(at + 12));
      }
      if (MODE == D_ONE) v[0] = v[1];
      const float lv = tm != -INFINITY ? logf(v[2]) : INFINITY, ent = tm != -INFINITY ? v[3] / v[2] - lv : INFINITY;
      if (own != 0.f) { dot = dot / v[2] * D_MAX_K; own /= v[2]; }
      if (stats != nullptr) {
        stats[(size_t)row * 2] = make_float4(m, v[0], v[1], target);
        stats[(size_t)row * 2 + 1] = make_float4(dot, own, ent, 0.f);
        saved[(size_t)row * 2 + 1] = make_float4(0.f, 0.f, lv, tm);
      } else {
        d_finish(m, v[0], v[1], target, dot, ent, lv, tm, a.tau, ce != nullptr ? ce + row : nullptr, kd + row, saved + (size_t)row * 2);
      }
    }
    __syncwarp();
    if (parts > 1) cluster_sync_all();               // nobody leaves or writes anew while the first CTA reads
  }
}

// stats [R, T, 8] of the ranks, and lv and tm in saved -> ce [T] (nullable), kd [T], saved.
__global__ void __launch_bounds__(256) distill_combine_kernel(const float4* __restrict__ stats, int R, int T, float tau, float* __restrict__ ce,
                                                             float* __restrict__ kd, float4* saved) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const float ct = D_LOG2E / tau;
  float m = stats[(size_t)t * 2].x;
  for (int r = 1; r < R; ++r) m = d_max(m, stats[((size_t)r * T + t) * 2].x);
  float s1 = 0.f, st = 0.f, target = INFINITY, dot = 0.f, ent = 0.f;
  for (int r = 0; r < R; ++r) {
    const float4 u = stats[((size_t)r * T + t) * 2], v = stats[((size_t)r * T + t) * 2 + 1];
    const float d = u.x - m;
    s1 += u.y * d_ex2(d * D_LOG2E);
    st += u.z * d_ex2(d * ct);
    if (u.w != INFINITY) target = u.w + d;
    if (v.y != 0.f) dot += v.x + v.y * d;
    ent = v.z;
  }
  const float4 teacher = saved[(size_t)t * 2 + 1];
  d_finish(m, s1, st, target, dot, ent, teacher.z, teacher.w, tau, ce != nullptr ? ce + t : nullptr, kd + t, saved + (size_t)t * 2);
}

__device__ __forceinline__ int d_slot(int id, int slots) { return (int)(((unsigned int)id * 2654435761u) >> 16) & (slots - 1); }

// out = d loss / d z; out may be z.  One CTA per part of a row, last rows first: where the backward follows the forward, the L2 still
// holds the rows that it read last, and the stores ask not to be kept there (a pass over 4096 x 128256: 512 -> 503 us).
template <typename T, int MODE, int DT>
__global__ void __launch_bounds__(DT, 1024 / DT) distill_bwd_kernel(const DistillArgs a, int parts, const float4* __restrict__ saved,
                                                            const float* __restrict__ g_ce, const float* __restrict__ g_kd, void* out,
                                                            int64_t out_ld, int slots) {
  constexpr int N = DVec<T>::N;
  // Entries of this part that get more than the softmax: the teacher's, then the label.  An id may stand twice (often the label among the
  // teacher's), so one entry of an id writes for all: the one that gets the id's place in a table, half of which stays empty.  Only
  // entries with twins look through the list, and add up in its order (K^2 steps without the table: 256 entries took 113 of 457 us at
  // 4096 x 128256).
  extern __shared__ __align__(16) int d_shared[];
  int* table = d_shared;                    // [slots] entries, -1: empty
  int* ids = table + slots;                 // [K + 1], -1: not in this part
  float* add = reinterpret_cast<float*>(ids + a.K + 1);
  float* at = add + a.K + 1;
  uint8_t* twins = reinterpret_cast<uint8_t*>(at + a.K + 1);      // 1: writes for others too, 2: another one writes
  const int part = blockIdx.x % parts;
  const float ct = D_LOG2E * a.inv_tau, c1 = D_LOG2E;
  for (int back = blockIdx.x / parts; back < a.T; back += gridDim.x / parts) {
    const int row = a.T - 1 - back;
    const T* z = reinterpret_cast<const T*>(a.z) + row * a.ld;
    T* o = reinterpret_cast<T*>(out) + row * out_ld;
    const DSpan sp = d_span(z, a.Vl, part, parts);
    const float4 sv = saved[(size_t)row * 2], teacher = saved[(size_t)row * 2 + 1];
    const float gc = a.labels != nullptr && sv.z != 0.f ? g_ce[row] : 0.f, gk = teacher.z != INFINITY ? g_kd[row] * a.tau : 0.f;
    const float A = gc != 0.f ? gc * sv.z : 0.f, B = gk != 0.f ? gk * teacher.x : 0.f;
    const bool same = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0;
    const bool zero = gc == 0.f && gk == 0.f;        // a token without loss: zeros, whatever its logits
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.lead);
    uint4* ov = reinterpret_cast<uint4*>(o + sp.lead);
    // the first logits are on their way before the entries are
    int i = sp.v0 + threadIdx.x;
    uint4 u[D_BATCH];
    const bool ahead = same && !zero && i + (D_BATCH - 1) * DT < sp.v1;
    if (ahead) {
#pragma unroll
      for (int b = 0; b < D_BATCH; ++b) u[b] = zv[i + b * DT];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < slots / 4; j += DT) reinterpret_cast<int4*>(table)[j] = make_int4(-1, -1, -1, -1);
    for (int j = threadIdx.x; j <= a.K; j += DT) {
      int loc = -1;
      float g = 0.f;
      if (j == a.K) {
        if (gc != 0.f) { loc = a.labels[row] - a.v0; g = gc; }
      } else if (gk != 0.f) {
        const int id = d_id(a, row, j);
        if (id >= 0) { loc = id - a.v0; g = gk * expf((d_teacher(a, row, j) - teacher.w) * a.inv_tau - teacher.z); }
      }
      const bool in = loc >= sp.c0 && loc < sp.c1;
      ids[j] = in ? loc : -1;
      add[j] = g;
      at[j] = in ? d_load(z + loc) : 0.f;
      twins[j] = 0;
    }
    __syncthreads();
    for (int j = threadIdx.x; j <= a.K; j += DT) {
      const int id = ids[j];
      if (id < 0) continue;
      for (int s = d_slot(id, slots);; s = (s + 1) & (slots - 1)) {        // ends: half of the slots stay empty
        const int other = atomicCAS(table + s, -1, j);
        if (other < 0) break;
        if (ids[other] == id) {
          twins[other] = 1;
          twins[j] = 2;
          break;
        }
      }
    }
    const F2 nm = f2(-sv.x, -sv.x), c1p = f2(c1, c1), ctp = f2(ct, ct), Ap = f2(A, A), Bp = f2(B, B);
    auto soft2 = [&](F2 v) {
      const F2 x = v + nm;
      const F2 e = f2_ex2(x * ctp);
      if (MODE == D_ONE) return e * (Ap + Bp);
      if (MODE == D_TWO) return f2_fma(f2_ex2(x * c1p), Ap, e * Bp);
      const F2 q = e * e;
      return f2_fma(MODE == D_SQUARE ? q : q * q, Ap, e * Bp);
    };
    auto soft = [&](float v) { return f2_get(soft2(f2(v, v))).x; };
    auto single = [&](int c) { d_store(o + c, zero ? 0.f : soft(d_load(z + c))); };
    if (!same) {
      for (int c = sp.c0 + threadIdx.x; c < sp.c1; c += DT) single(c);      // rows that are aligned differently
    } else {
      if (part == 0 && (int)threadIdx.x < sp.lead) single(threadIdx.x);
      if (part == parts - 1 && sp.lead + sp.vecs * N + (int)threadIdx.x < a.Vl) single(sp.lead + sp.vecs * N + threadIdx.x);
      if (zero) {
        for (; i < sp.v1; i += DT) __stcs(ov + i, make_uint4(0, 0, 0, 0));
      } else {
        auto vec = [&](const uint4& r) {
          F2 x[N / 2];
          DVec<T>::unpack(r, x);
#pragma unroll
          for (int j = 0; j < N / 2; ++j) x[j] = soft2(x[j]);
          return DVec<T>::pack(x);
        };
        if (ahead) {
          while (true) {
#pragma unroll
            for (int b = 0; b < D_BATCH; ++b) __stcs(ov + i + b * DT, vec(u[b]));
            i += D_BATCH * DT;
            if (i + (D_BATCH - 1) * DT >= sp.v1) break;
#pragma unroll
            for (int b = 0; b < D_BATCH; ++b) u[b] = zv[i + b * DT];
          }
        }
        for (; i < sp.v1; i += DT) __stcs(ov + i, vec(zv[i]));
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j <= a.K; j += DT) {
      const int id = ids[j];
      if (id < 0 || zero) continue;
      const int twin = twins[j];
      if (twin == 2) continue;
      float g = add[j];
      if (twin == 1) {
        g = 0.f;
        for (int q = 0; q <= a.K; ++q)
          if (ids[q] == id) g += add[q];
      }
      d_store(o + id, soft(at[j]) - g);
    }
  }
}

// ---------------------------------------------------------------------------- host
// All fields 8 bytes wide, as the Python layer packs them.
struct DistillCall {
  int64_t z, ld, f32, labels, ids, id_stride, id64, t, t_stride, t_type, T, Vl, K, v0, V, budget, stream;
  double tau;
};

static int d_refuse(const char* what, const DistillCall& c) {
  // 2^30: a row's or an element's number plus one step of a loop stays in 31 bits
  if (c.T >= 0 && c.T <= (1 << 30) && c.Vl > 0 && c.Vl <= (1 << 30) && c.K >= 0 && c.K <= D_MAX_K && c.v0 >= 0 && c.V >= c.v0 + c.Vl && c.V <= INT32_MAX &&
      c.tau >= FLT_MIN && c.tau <= FLT_MAX)
    return 0;
  set_last_error_c(what, "a shard inside a vocabulary of at most 2^31 - 1 entries, at most 2^30 rows and entries a shard, 1024 teacher's entries, a temperature that is a normal fp32 number");
  return (int)cudaErrorInvalidValue;
}
// The statistics of a row are read and written as vectors.
static int d_refuse_unaligned(const char* what, const void* a, const void* b) {
  if ((((uintptr_t)a | (uintptr_t)b) & 15) == 0) return 0;
  set_last_error_c(what, "statistics that start on 16 bytes");
  return (int)cudaErrorInvalidValue;
}
static int d_rc(const char* what, cudaError_t e) {
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c(what, cudaGetErrorString(e));
  return (int)e;
}
static DistillArgs d_args(const DistillCall& c) {
  DistillArgs a;
  a.z = (const void*)c.z;
  a.labels = (const int*)c.labels;
  a.ids = (const void*)c.ids;
  a.t = (const void*)c.t;
  a.ld = c.ld;
  a.id_stride = c.id_stride;
  a.t_stride = c.t_stride;
  a.id64 = (int)c.id64;
  a.t_type = (int)c.t_type;
  a.T = (int)c.T;
  a.Vl = (int)c.Vl;
  a.K = (int)c.K;
  a.v0 = (int)c.v0;
  a.V = (int)c.V;
  a.tau = (float)c.tau;
  a.inv_tau = (float)(1. / c.tau);
  return a;
}
static int d_mode(const DistillCall& c) {
  if (c.labels == 0 || c.tau == 1.) return D_ONE;
  return c.tau == 2. ? D_SQUARE : c.tau == 4. ? D_FOURTH : D_TWO;
}
// Threads of a CTA: four batches of loads each, as far as 32 to 256 threads give that.  A row has some microseconds of its own (the
// entries, two rounds of reductions), so short rows take small CTAs and the SM holds more of them.  Forward / backward with 256, 64 and 32
// threads at 16384 x 4000: 160 / 172, 66 / 76 and 54 / 68 us; with 128 and 64 at 16384 x 8000: 91 / 113 and 76 / 109 us.  Where there are
// fewer rows than the GPU holds such CTAs, larger ones (2000 x 2000 forward: 23 us in clusters of two CTAs of 32, 8 with 64 threads).
static int d_threads(const DistillCall& c, int per_vec) {
  const int sms = dh_sm_count();
  const int64_t vecs = c.Vl / per_vec, room = 1024ll * ((c.budget <= 0 || c.budget > sms) ? sms : c.budget);
  int threads = vecs >= 16 * 256 ? 256 : vecs >= 16 * 128 ? 128 : vecs >= 16 * 64 ? 64 : 32;
  while (threads < 256 && c.T * threads * 2 <= room && vecs >= threads) threads *= 2;
  return threads;
}
// CTAs that share a row: where there are fewer rows than the GPU holds CTAs, as long as each thread still has a vector; `waves` > 1 (the
// backward, whose parts need not be joined): up to that many times what the GPU holds while each thread has four batches, so that
// the last rows do not run alone (700 x 128256: 84 -> 74 us, 1500 rows 139 -> 133; the forward's clusters only lose by it, 59 -> 66 us).
static int d_parts(const DistillCall& c, int threads, int per_vec, int most, int waves) {
  const int sms = dh_sm_count();
  const int64_t room = 1024 / threads * ((c.budget <= 0 || c.budget > sms) ? sms : c.budget), vecs = c.Vl / per_vec;
  int parts = 1;
  while (parts < most) {
    const int64_t ctas = c.T * parts * 2, each = vecs / (threads * parts * 2);
    if (!(ctas <= room ? each >= 1 : ctas <= room * waves && each >= 4 * D_BATCH)) break;
    parts *= 2;
  }
  return parts;
}
// CTAs of a launch: one per row and part; as many as fit on the SMs of a budget, which then walk over the rows.
static unsigned int d_grid(const DistillCall& c, int threads, int parts) {
  const int sms = dh_sm_count();
  int64_t fit = INT32_MAX / parts;
  if (c.budget > 0 && c.budget < sms) fit = 1024 / threads * c.budget / parts;
  if (fit < 1) fit = 1;
  return (unsigned int)((c.T < fit ? c.T : fit) * parts);
}

template <typename T, int DT>
static cudaError_t d_launch_fwd_as(const DistillCall& c, float* ce, float* kd, float4* saved, float4* stats) {
  void (*const kernels[4])(const DistillArgs, int, float*, float*, float4*, float4*) = {
      distill_fwd_kernel<T, D_ONE, DT>, distill_fwd_kernel<T, D_TWO, DT>, distill_fwd_kernel<T, D_SQUARE, DT>, distill_fwd_kernel<T, D_FOURTH, DT>};
  const int parts = d_parts(c, DT, DVec<T>::N, 8, 1);       // the largest cluster that every GPU runs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(d_grid(c, DT, parts));
  cfg.blockDim = dim3(DT);
  cfg.dynamicSmemBytes = sizeof(uint4) * 2 * D_BATCH * DT;
  cfg.stream = (cudaStream_t)c.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernels[d_mode(c)], d_args(c), parts, ce, kd, saved, stats);
}
template <typename T>
static cudaError_t d_launch_fwd(const DistillCall& c, float* ce, float* kd, float4* saved, float4* stats) {
  const int threads = d_threads(c, DVec<T>::N);
  if (threads == 256) return d_launch_fwd_as<T, 256>(c, ce, kd, saved, stats);
  if (threads == 128) return d_launch_fwd_as<T, 128>(c, ce, kd, saved, stats);
  return threads == 64 ? d_launch_fwd_as<T, 64>(c, ce, kd, saved, stats) : d_launch_fwd_as<T, 32>(c, ce, kd, saved, stats);
}
template <typename T, int DT>
static void d_launch_bwd_as(const DistillCall& c, const float4* saved, const float* g_ce, const float* g_kd, void* out, int64_t out_ld) {
  void (*const kernels[4])(const DistillArgs, int, const float4*, const float*, const float*, void*, int64_t, int) = {
      distill_bwd_kernel<T, D_ONE, DT>, distill_bwd_kernel<T, D_TWO, DT>, distill_bwd_kernel<T, D_SQUARE, DT>, distill_bwd_kernel<T, D_FOURTH, DT>};
  const int parts = d_parts(c, DT, DVec<T>::N, 64, 8);
  int slots = 64;
  while (slots < 2 * (c.K + 1)) slots *= 2;
  const size_t shared = sizeof(int) * (slots + 3 * (size_t)(c.K + 1)) + c.K + 1;       // at most 30 KB
  kernels[d_mode(c)]<<<d_grid(c, DT, parts), DT, shared, (cudaStream_t)c.stream>>>(d_args(c), parts, saved, g_ce, g_kd, out, out_ld, slots);
}
template <typename T>
static void d_launch_bwd(const DistillCall& c, const float4* saved, const float* g_ce, const float* g_kd, void* out, int64_t out_ld) {
  const int threads = d_threads(c, DVec<T>::N);
  if (threads == 256) d_launch_bwd_as<T, 256>(c, saved, g_ce, g_kd, out, out_ld);
  else if (threads == 128) d_launch_bwd_as<T, 128>(c, saved, g_ce, g_kd, out, out_ld);
  else if (threads == 64) d_launch_bwd_as<T, 64>(c, saved, g_ce, g_kd, out, out_ld);
  else d_launch_bwd_as<T, 32>(c, saved, g_ce, g_kd, out, out_ld);
}

}  // namespace dh

using namespace dh;

extern "C" {

// ce [T] (null without labels), kd [T], saved [T, 4] pairs of fp32; or, for a shard of a divided vocabulary, stats [T, 8] and the teacher's
// part of saved.
int dh_distill_fwd(const void* call, void* ce, void* kd, void* saved, void* stats) {
  const DistillCall& c = *(const DistillCall*)call;
  if (int rc = d_refuse("dh_distill_fwd", c)) return rc;
  if (int rc = d_refuse_unaligned("dh_distill_fwd", saved, stats)) return rc;
  if (c.T == 0) return 0;
  if (saved == nullptr || (kd == nullptr && stats == nullptr)) {
    set_last_error_c("dh_distill_fwd", "no place for what a row gives");
    return (int)cudaErrorInvalidValue;
  }
  const cudaError_t e = c.f32 ? d_launch_fwd<float>(c, (float*)ce, (float*)kd, (float4*)saved, (float4*)stats)
                              : d_launch_fwd<__nv_bfloat16>(c, (float*)ce, (float*)kd, (float4*)saved, (float4*)stats);
  return d_rc("dh_distill_fwd", e);
}
int dh_distill_combine(const void* stats, int R, int T, float tau, void* ce, void* kd, void* saved, cudaStream_t s) {
  if (R <= 0 || T <= 0) return 0;
  if (int rc = d_refuse_unaligned("dh_distill_combine", stats, saved)) return rc;
  distill_combine_kernel<<<(T + 255) / 256, 256, 0, s>>>((const float4*)stats, R, T, tau, (float*)ce, (float*)kd, (float4*)saved);
  return d_rc("dh_distill_combine", cudaSuccess);
}
int dh_distill_bwd(const void* call, const void* saved, const void* g_ce, const void* g_kd, void* out, int64_t out_ld) {
  const DistillCall& c = *(const DistillCall*)call;
  if (int rc = d_refuse("dh_distill_bwd", c)) return rc;
  if (int rc = d_refuse_unaligned("dh_distill_bwd", saved, nullptr)) return rc;
  if (c.T == 0) return 0;
  if (saved == nullptr || g_kd == nullptr || out == nullptr || (c.labels != 0 && g_ce == nullptr)) {
    set_last_error_c("dh_distill_bwd", "no statistics, gradients or output");
    return (int)cudaErrorInvalidValue;
  }
  if (c.f32) d_launch_bwd<float>(c, (const float4*)saved, (const float*)g_ce, (const float*)g_kd, out, out_ld);
  else d_launch_bwd<__nv_bfloat16>(c, (const float4*)saved, (const float*)g_ce, (const float*)g_kd, out, out_ld);
  return d_rc("dh_distill_bwd", cudaSuccess);
}

}  // extern "C"
