// Rotary positions of separate query and key heads for sm_100a, out of place or in place, forward and backward.
//
// Pair i of a head (i < r/2 of the r rotated elements: (i, i + r/2) or, interleaved, (2i, 2i + 1)) at position p is turned by the
// angle p f_i and scaled by m:  (x, y) -> m (x cos - y sin, y cos + x sin).  The backward is the transposed rotation (sin -> -sin).
// Elements from r on are copied.
//
// The angles are computed here, from r/2 frequencies in 64 bits, and not read from a table of all positions: a table for a million
// positions is 512 MB, has an end that a position can pass, and costs as many bytes per row as a head.  p f_i is formed in
// turns in 64 bits and reduced to [-1/2, 1/2] before it is rounded to 32, so far positions lose nothing (a 32-bit product is off
// by 0.03 rad at position 10^6).
//
// One thread holds the cosines and sines of V pairs of one row in registers and walks over heads with them, several in flight: two 16-byte
// loads and stores per head.  Bound by memory: 65536 x 40 heads of 128, 214 us (6.3 TB/s).  A table of a CTA's angles in shared memory, so
// that threads that share a row do not compute them anew, was slower (225 us; 65536 x 3 heads 39 against 27), and so was one head at a
// time (243 us).
//
// Interleaved, a vector may hold pairs that are turned and pairs that stay, so V follows from addresses and strides alone.  In halves it has
// to divide half the rotated elements too; where that leaves little of a vector, whole heads pass through shared memory (second kernel).
// Elements that are only copied stay with the pairs of their head: as work items behind all pairs they tore the lines of memory apart
// (3799 x 80 heads of 128, 64 rotated: 37 against 51 us).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "api.h"
#include "ptx.cuh"
#include "tmap.h"

namespace dh {

constexpr int RT = 256;

struct RopeTensor {
  const void* in;
  void* out;
  long long is0, is1, ish, os0, os1, osh;     // strides in elements of the two row dimensions and of the heads
};
struct RopeArgs {
  RopeTensor t[2];                            // queries, keys
  int heads[2];
  const void* pos;
  const double* freq;
  float scale, sign;
  int pos64, inner;                           // rows = outer x inner
  int rot_units, units, half, d, groups;      // units of V pairs (or 2 V copied elements) per head, threads that share a row's heads
  long long row0, rows;
};

// V elements as they are loaded and stored, and as fp32.
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };
template <typename T, int V> using RopeRaw = typename RawOf<sizeof(T) * V>::type;

template <typename T, int V>
__device__ __forceinline__ void rope_unpack(const RopeRaw<T, V>& r, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = __uint_as_float(w[j]);
  } else if constexpr (V == 1) {
    f[0] = __uint_as_float((uint32_t)r << 16);
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) { const float2 p = unpack_bf16x2(w[j]); f[2 * j] = p.x; f[2 * j + 1] = p.y; }
  }
}
template <typename T, int V>
__device__ __forceinline__ RopeRaw<T, V> rope_pack(const float (&f)[V]) {
  RopeRaw<T, V> r;
  if constexpr (sizeof(T) == 4) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = __float_as_uint(f[j]);
  } else if constexpr (V == 1) {
    r = __bfloat16_as_ushort(__float2bfloat16(f[0]));
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
  }
  return r;
}
// One pair, the same bits wherever it is turned: the results of a row do not depend on what shares the call with it.
__device__ __forceinline__ void rope_pair(float& x, float& y, float c, float s) {
  const float u = __fmul_rn(y, s), w = __fmul_rn(x, s);
  x = fmaf(x, c, -u);
  y = fmaf(y, c, w);
}
// Turns V pairs: x the first, y the second elements; interleaved, x has the first V/2 pairs, y the others, and those from n on stay.
template <typename T, int V, bool INTERLEAVED>
__device__ __forceinline__ void rope_turn(RopeRaw<T, V>& x, RopeRaw<T, V>& y, const float (&cs)[V], const float (&sn)[V], int n) {
  float p[V], q[V];
  rope_unpack<T, V>(x, p);
  rope_unpack<T, V>(y, q);
  if constexpr (INTERLEAVED && V > 1) {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const int f = j / 2, s = V / 2 + j / 2;
      if (f < n) rope_pair(p[j], p[j + 1], cs[f], sn[f]);
      if (s < n) rope_pair(q[j], q[j + 1], cs[s], sn[s]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) rope_pair(p[j], q[j], cs[j], sn[j]);
  }
  RopeRaw<T, V> rx = rope_pack<T, V>(p), ry = rope_pack<T, V>(q);
  if constexpr (INTERLEAVED && V > 1 && sizeof(T) == 2) {       // what stays, stays bit by bit: a NaN's bits do not survive the conversion
    const uint32_t *x0 = reinterpret_cast<const uint32_t*>(&x), *y0 = reinterpret_cast<const uint32_t*>(&y);
#pragma unroll
    for (int f = 0; f < V / 2; ++f) {
      if (f >= n) reinterpret_cast<uint32_t*>(&rx)[f] = x0[f];
      if (V / 2 + f >= n) reinterpret_cast<uint32_t*>(&ry)[f] = y0[f];
    }
  }
  x = rx;
  y = ry;
}

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(RT, 3) rope_heads_kernel(const RopeArgs a) {
  constexpr int R_HEADS = sizeof(T) * V >= 8 ? 4 : 8;        // heads in flight
  const unsigned int total = (unsigned int)(a.rows * a.units * a.groups);
  for (unsigned int i = blockIdx.x * RT + threadIdx.x; i < total; i += gridDim.x * RT) {
    const unsigned int g = i / a.units, unit = i - g * a.units;
    const unsigned int r = g / a.groups, group = g - r * a.groups;
    const long long row = a.row0 + r;
    const long long outer = row / a.inner, inner = row - outer * a.inner;
    const bool rotates = (int)unit < a.rot_units;
    // element offsets of the two vectors of this unit inside a head; `two`: the second one is there; n: pairs that are turned
    const int c = (int)unit * V, n = min(V, a.half - c);
    int e0, e1;
    if (rotates) {
      e0 = INTERLEAVED ? 2 * c : c;
      e1 = INTERLEAVED ? 2 * c + V : c + a.half;
    } else {
      e0 = (INTERLEAVED ? 2 * V * a.rot_units : 2 * a.half) + 2 * V * ((int)unit - a.rot_units);
      e1 = e0 + V;
    }
    const bool two = e1 < a.d;
    if (!two) e1 = e0;
    float cs[V], sn[V];
    if (rotates) {
      const double p = a.pos64 ? (double)reinterpret_cast<const long long*>(a.pos)[row] : (double)reinterpret_cast<const int*>(a.pos)[row];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double turns = p * a.freq[min(c + j, a.half - 1)] * 0.15915494309189533577;      // 1 / (2 pi)
        float s, k;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &k);
        cs[j] = k * a.scale;
        sn[j] = s * a.scale * a.sign;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) { cs[j] = 1.f; sn[j] = 0.f; }
    }
    const int all = a.heads[0] + a.heads[1];
    for (int first = (int)group; first < all; first += R_HEADS * a.groups) {
      RopeRaw<T, V> x[R_HEADS], y[R_HEADS];
#pragma unroll
      for (int u = 0; u < R_HEADS; ++u) {
        const int h = first + u * a.groups;
        if (h >= all) continue;
        const int w = h >= a.heads[0];
        const RopeTensor& t = a.t[w];
        const T* src = reinterpret_cast<const T*>(t.in) + outer * t.is0 + inner * t.is1 + (w ? h - a.heads[0] : h) * t.ish;
        x[u] = *reinterpret_cast<const RopeRaw<T, V>*>(src + e0);
        y[u] = *reinterpret_cast<const RopeRaw<T, V>*>(src + e1);
      }
#pragma unroll
      for (int u = 0; u < R_HEADS; ++u) {
        const int h = first + u * a.groups;
        if (h >= all) continue;
        const int w = h >= a.heads[0];
        const RopeTensor& t = a.t[w];
        T* dst = reinterpret_cast<T*>(t.out) + outer * t.os0 + inner * t.os1 + (w ? h - a.heads[0] : h) * t.osh;
        if (rotates) rope_turn<T, V, INTERLEAVED>(x[u], y[u], cs, sn, n);
        *reinterpret_cast<RopeRaw<T, V>*>(dst + e0) = x[u];
        if (two) *reinterpret_cast<RopeRaw<T, V>*>(dst + e1) = y[u];
      }
    }
  }
}

// Pairs in halves whose half is an odd number of elements, or of pairs of bf16: a warp brings whole heads of a row into shared memory by
// vectors, turns them there, W pairs of a lane side by side, and sends them out by vectors.  Where half a head's pairs need 16 lanes or
// fewer, 2, 4, ... heads are turned at a time.  NP: times that a lane has W pairs of a head.  Bound by the instructions around the
// vectors: the addresses of a row's heads are kept over its steps (16384 x 80 heads of 96, 38 rotated: 109 -> 92 us), and the next
// step's vectors are asked for before this one's are turned (114 -> 109 us).  Three CTAs per SM: with four a few registers spill, 158 us.
constexpr int RS = 4;                         // vectors of a lane at a time: 2 KB a warp
template <typename T, int W> struct RopeWords;
template <> struct RopeWords<float, 1> {
  using type = float;
  __device__ static __forceinline__ void get(float w, float (&f)[1]) { f[0] = w; }
  __device__ static __forceinline__ float put(const float (&f)[1]) { return f[0]; }
};
template <> struct RopeWords<__nv_bfloat16, 1> {
  using type = __nv_bfloat16;
  __device__ static __forceinline__ void get(__nv_bfloat16 w, float (&f)[1]) { f[0] = __bfloat162float(w); }
  __device__ static __forceinline__ __nv_bfloat16 put(const float (&f)[1]) { return __float2bfloat16(f[0]); }
};
template <> struct RopeWords<__nv_bfloat16, 2> {
  using type = uint32_t;
  __device__ static __forceinline__ void get(uint32_t w, float (&f)[2]) { const float2 p = unpack_bf16x2(w); f[0] = p.x; f[1] = p.y; }
  __device__ static __forceinline__ uint32_t put(const float (&f)[2]) { return pack_bf16x2(f[0], f[1]); }
};

template <typename T, int W, int LANES, int NP>
__global__ void __launch_bounds__(RT, 3) rope_staged_kernel(const RopeArgs a) {
  constexpr int BATCH = 4 / W, SUBS = 32 / LANES;         // heads of a lane at a time, lanes' groups
  using Words = RopeWords<T, W>;
  using Word = typename Words::type;
  __shared__ uint4 stage[RT / 32][RS * 32];
  const int lane = threadIdx.x & 31, sub = lane / LANES, li = lane % LANES;
  uint4* const mine = stage[threadIdx.x >> 5];
  const int vecs = a.units, per = RS * 32 / vecs, all = a.heads[0] + a.heads[1];      // vectors of a head, heads of a step
  int head[RS];
#pragma unroll
  for (int s = 0; s < RS; ++s) head[s] = min((s * 32 + lane) / vecs, per);
  const auto offset = [&](int s) { return s * 32 + lane - head[s] * vecs; };
  const auto there = [&](int s, int first) { return head[s] < per && first + head[s] < all; };
  const unsigned int total = (unsigned int)(a.rows * a.groups), step = gridDim.x * (RT / 32);
  for (unsigned int i = blockIdx.x * (RT / 32) + (threadIdx.x >> 5); i < total; i += step) {
    const unsigned int r = i / a.groups, group = i - r * a.groups;
    const long long row = a.row0 + r;
    const long long outer = row / a.inner, inner = row - outer * a.inner;
    const T* const in0 = reinterpret_cast<const T*>(a.t[0].in) + outer * a.t[0].is0 + inner * a.t[0].is1;
    const T* const in1 = reinterpret_cast<const T*>(a.t[1].in) + outer * a.t[1].is0 + inner * a.t[1].is1 - a.heads[0] * a.t[1].ish;
    T* const out0 = reinterpret_cast<T*>(a.t[0].out) + outer * a.t[0].os0 + inner * a.t[0].os1;
    T* const out1 = reinterpret_cast<T*>(a.t[1].out) + outer * a.t[1].os0 + inner * a.t[1].os1 - a.heads[0] * a.t[1].osh;
    uint4 v[RS];
    const auto fetch = [&](int first) {
#pragma unroll
      for (int s = 0; s < RS; ++s) {
        const int h = first + head[s];
        if (!there(s, first)) continue;
        const T* src = h < a.heads[0] ? in0 + h * a.t[0].ish : in1 + h * a.t[1].ish;
        v[s] = reinterpret_cast<const uint4*>(src)[offset(s)];
      }
    };
    fetch((int)group * per);
    const double p = a.pos64 ? (double)reinterpret_cast<const long long*>(a.pos)[row] : (double)reinterpret_cast<const int*>(a.pos)[row];
    float cs[NP][W], sn[NP][W];
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const double turns = p * a.freq[min((li + LANES * j) * W + q, a.half - 1)] * 0.15915494309189533577;
        float s, k;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &k);
        cs[j][q] = k * a.scale;
        sn[j][q] = s * a.scale * a.sign;
      }
    for (int first = (int)group * per; first < all; first += a.groups * per) {
#pragma unroll
      for (int s = 0; s < RS; ++s)
        if (there(s, first)) mine[s * 32 + lane] = v[s];
      fetch(first + a.groups * per);
      __syncwarp();
      const int count = min(per, all - first);
      for (int g = sub; g < count; g += BATCH * SUBS) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if ((li + LANES * j) * W >= a.half) continue;
          T* const e = reinterpret_cast<T*>(mine) + g * a.d + (li + LANES * j) * W;
          Word x[BATCH], y[BATCH];
#pragma unroll
          for (int u = 0; u < BATCH; ++u)
            if (g + u * SUBS < count) {
              x[u] = *reinterpret_cast<const Word*>(e + u * SUBS * a.d);
              y[u] = *reinterpret_cast<const Word*>(e + u * SUBS * a.d + a.half);
            }
#pragma unroll
          for (int u = 0; u < BATCH; ++u)
            if (g + u * SUBS < count) {
              float f[W], t[W];
              Words::get(x[u], f);
              Words::get(y[u], t);
#pragma unroll
              for (int q = 0; q < W; ++q) rope_pair(f[q], t[q], cs[j][q], sn[j][q]);
              *reinterpret_cast<Word*>(e + u * SUBS * a.d) = Words::put(f);
              *reinterpret_cast<Word*>(e + u * SUBS * a.d + a.half) = Words::put(t);
            }
        }
      }
      __syncwarp();
#pragma unroll
      for (int s = 0; s < RS; ++s) {
        const int h = first + head[s];
        if (!there(s, first)) continue;
        T* dst = h < a.heads[0] ? out0 + h * a.t[0].osh : out1 + h * a.t[1].osh;
        reinterpret_cast<uint4*>(dst)[offset(s)] = mine[s * 32 + lane];
      }
      __syncwarp();
    }
  }
}

// All fields 8 bytes wide, as the Python layer packs them.  ptrs: q in, q out, k in, k out; strides (elements): for each of them the outer
// row, inner row and head stride; rows are outer x inner.
struct RopeCall {
  int64_t ptrs[4], strides[12], heads_q, heads_k, pos, pos64, freq, rows, inner, d, rotated, interleaved, f32, transposed, budget, stream;
  double scale;
};

template <typename T, int V>
static void rope_launch(const RopeArgs& a, int interleaved, int grid, cudaStream_t s) {
  if (interleaved) rope_heads_kernel<T, V, true><<<grid, RT, 0, s>>>(a);
  else rope_heads_kernel<T, V, false><<<grid, RT, 0, s>>>(a);
}

template <typename T, int W>
static void rope_launch_staged(const RopeArgs& a, int words, int grid, cudaStream_t s) {
  if (words <= 8) rope_staged_kernel<T, W, 8, 1><<<grid, RT, 0, s>>>(a);
  else if (words <= 16) rope_staged_kernel<T, W, 16, 1><<<grid, RT, 0, s>>>(a);
  else if (words <= 32) rope_staged_kernel<T, W, 32, 1><<<grid, RT, 0, s>>>(a);
  else if (words <= 64) rope_staged_kernel<T, W, 32, 2><<<grid, RT, 0, s>>>(a);
  else rope_staged_kernel<T, W, 32, 4><<<grid, RT, 0, s>>>(a);
}
static int rope_rc() {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c("dh_rope_heads", cudaGetErrorString(e));
  return (int)e;
}

}  // namespace dh

using namespace dh;

extern "C" {

// Rotates the heads of q (and of k, unless heads_k is 0); in == out (with equal strides) works in place.
int dh_rope_heads(const void* call) {
  const RopeCall& c = *(const RopeCall*)call;
  const int64_t rows = c.rows, inner = c.inner;
  const int heads_q = (int)c.heads_q, heads_k = (int)c.heads_k, d = (int)c.d, rotated = (int)c.rotated;
  const int64_t* ptrs = c.ptrs;
  if (c.heads_q < 0 || c.heads_k < 0 || c.heads_q > (1 << 28) || c.heads_k > (1 << 28) || c.d <= 0 || c.d > 65536 || c.rotated <= 0 || c.rotated > c.d ||
      (c.rotated & 1) || rows < 0 || inner <= 0 || inner > INT32_MAX) {
    set_last_error_c("dh_rope_heads", "sizes out of range (an even number of rotated elements, at most the head size; at most 2^28 heads each)");
    return (int)cudaErrorInvalidValue;
  }
  if (rows == 0 || heads_q + heads_k == 0) return 0;
  const int size = c.f32 ? 4 : 2;
  const bool in_place = (heads_q == 0 || ptrs[0] == ptrs[1]) && (heads_k == 0 || ptrs[2] == ptrs[3]);
  const int interleaved = (int)c.interleaved;
  // the widest vector that divides every address and stride, and a head (interleaved) or half the rotated part and the rest (in halves)
  uint64_t wide = 0;
  for (int i = 0; i < 4; ++i) {
    if ((i < 2 ? heads_q : heads_k) == 0) continue;
    wide |= (uint64_t)ptrs[i];
    for (int j = 0; j < 3; ++j) wide |= (uint64_t)(c.strides[3 * i + j] * size);
  }
  const uint64_t odd = wide | (uint64_t)(interleaved ? d : rotated / 2) * size | (interleaved || in_place ? 0 : (uint64_t)(d - rotated) * size);
  const int bytes = (odd & 15) == 0 ? 16 : (odd & 7) == 0 ? 8 : (odd & 3) == 0 ? 4 : 2;
  const int V = bytes / size;
  if (V == 0) {
    set_last_error_c("dh_rope_heads", "fp32 operands must be aligned to their elements");
    return (int)cudaErrorInvalidValue;
  }
  RopeArgs a;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = c.strides + 6 * i;
    a.t[i] = RopeTensor{(const void*)ptrs[2 * i], (void*)ptrs[2 * i + 1], st[0], st[1], st[2], st[3], st[4], st[5]};
  }
  a.heads[0] = heads_q;
  a.heads[1] = heads_k;
  a.pos = (const void*)c.pos;
  a.freq = (const double*)c.freq;
  a.scale = (float)c.scale;
  a.sign = c.transposed ? -1.f : 1.f;
  a.pos64 = (int)c.pos64;
  a.inner = (int)inner;
  a.half = rotated / 2;
  a.d = d;
  const int sms = dh_sm_count();
  const int budget = (c.budget <= 0 || c.budget > sms) ? sms : (int)c.budget;
  const cudaStream_t s = (cudaStream_t)c.stream;
  // CTAs of a launch; beyond them they walk on.  On the whole GPU 8, 16, 32 per SM and as many as there are: 200000 x 40 heads of 128 661,
  // 637, 631 and 632 us, 500000 x 3 155, 153, 152 and 160 us.
  const int64_t cap = (int64_t)budget * (budget < sms ? 8 : 32);
  // Through shared memory, where the pairs alone keep a vector at 4 bytes or fewer.  By the kernel above / so: 16384 x 80 heads of 96, 38
  // rotated 212 / 92 us, 16384 x 40 of 128, 50 rotated 144 / 60, 16384 x 80 of 80, 20 rotated 109 / 76, fp32 16384 x 40 of 96, 38 rotated
  // 110 / 88.  Not for small calls (30 x 40 heads of 96: 4.3 / 5.3 us, 100 x 40: 6.4 / 5.5), nor where 8 lanes' angles are for less than a
  // step (65536 x 8 heads of 80, 20 rotated: 53 / 58 us; x 16: 91 / 85); at 8 bytes the kernel above has the fewer instructions.
  const int all = heads_q + heads_k, words = !c.f32 && bytes == 4 ? a.half / 2 : a.half;
  const int vecs = d * size / 16, per = vecs > 0 ? 32 * RS / vecs : 0;
  if (bytes <= 4 && !interleaved && ((wide | (uint64_t)d * size) & 15) == 0 && per > 0 && a.half <= 128 && rows * all >= 4096 &&
      (words > 8 || all >= per)) {
    a.units = vecs;
    a.groups = 1;
    while (a.groups * 2 * per <= all && rows * a.groups < (int64_t)budget * 64) a.groups *= 2;
    const int64_t most = INT32_MAX / a.groups;
    for (int64_t r = 0; r < rows; r += most) {
      a.row0 = r;
      a.rows = rows - r < most ? rows - r : most;
      const int64_t blocks = (a.rows * a.groups + RT / 32 - 1) / (RT / 32);
      const int grid = (int)(blocks < cap ? blocks : cap);
      if (c.f32) rope_launch_staged<float, 1>(a, words, grid, s);
      else if (bytes == 4) rope_launch_staged<__nv_bfloat16, 2>(a, words, grid, s);
      else rope_launch_staged<__nv_bfloat16, 1>(a, words, grid, s);
    }
    return rope_rc();
  }
  a.rot_units = (a.half + V - 1) / V;
  const int rest = interleaved ? d - 2 * V * a.rot_units : d - rotated;
  a.units = a.rot_units + (in_place || rest <= 0 ? 0 : (rest + 2 * V - 1) / (2 * V));
  // threads that share the heads of a row: enough of them to fill half of the GPU's threads, where there are that few rows
  a.groups = 1;
  while (a.groups * 2 <= all && rows * a.units * a.groups < (int64_t)budget * 1024) a.groups *= 2;
  const int64_t most = INT32_MAX / ((int64_t)a.units * a.groups);      // rows of one launch: item numbers stay in 31 bits
  for (int64_t r = 0; r < rows; r += most) {
    a.row0 = r;
    a.rows = rows - r < most ? rows - r : most;
    const int64_t blocks = (a.rows * a.units * a.groups + RT - 1) / RT;
    const int grid = (int)(blocks < cap ? blocks : cap);
    if (c.f32) {
      if (V == 4) rope_launch<float, 4>(a, interleaved, grid, s);
      else if (V == 2) rope_launch<float, 2>(a, interleaved, grid, s);
      else rope_launch<float, 1>(a, interleaved, grid, s);
    } else {
      if (V == 8) rope_launch<__nv_bfloat16, 8>(a, interleaved, grid, s);
      else if (V == 4) rope_launch<__nv_bfloat16, 4>(a, interleaved, grid, s);
      else if (V == 2) rope_launch<__nv_bfloat16, 2>(a, interleaved, grid, s);
      else rope_launch<__nv_bfloat16, 1>(a, interleaved, grid, s);
    }
  }
  return rope_rc();
}

}  // extern "C"
