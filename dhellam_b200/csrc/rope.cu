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
// One thread holds the cosines and sines of V pairs of one row in registers and walks over heads with them: two 16-byte loads and
// stores per head.  Bound by memory.
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

template <int BYTES> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };
template <> struct RawOf<2> { using type = uint16_t; };

template <typename T, int V>
struct alignas(sizeof(T) * V) RopeVec {
  T e[V];
};

__device__ __forceinline__ float rope_f(float x) { return x; }
__device__ __forceinline__ float rope_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rope_t(float x);
template <> __device__ __forceinline__ float rope_t<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 rope_t<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

template <typename T, int V>
__device__ __forceinline__ RopeVec<T, V> rope_load(const T* p) {
  using R = typename RawOf<sizeof(T) * V>::type;
  union { R r; RopeVec<T, V> v; } u;
  u.r = *reinterpret_cast<const R*>(p);
  return u.v;
}
template <typename T, int V>
__device__ __forceinline__ void rope_store(T* p, const RopeVec<T, V>& v) {
  using R = typename RawOf<sizeof(T) * V>::type;
  union { R r; RopeVec<T, V> v; } u;
  u.v = v;
  *reinterpret_cast<R*>(p) = u.r;
}

template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(RT) rope_heads_kernel(const RopeArgs a) {
  const unsigned int total = (unsigned int)(a.rows * a.units * a.groups);
  for (unsigned int i = blockIdx.x * RT + threadIdx.x; i < total; i += gridDim.x * RT) {
    const unsigned int g = i / a.units, unit = i - g * a.units;
    const unsigned int r = g / a.groups, group = g - r * a.groups;
    const long long row = a.row0 + r;
    const long long outer = row / a.inner, inner = row - outer * a.inner;
    const bool rotates = (int)unit < a.rot_units;
    // element offsets of the two vectors of this unit inside a head; `two`: the second one is there
    const int c = (int)unit * V;
    int e0, e1;
    bool two = true;
    if (rotates) {
      e0 = INTERLEAVED ? 2 * c : c;
      e1 = INTERLEAVED ? 2 * c + V : c + a.half;
    } else {
      e0 = 2 * a.half + 2 * V * ((int)unit - a.rot_units);
      e1 = e0 + V;
      two = e1 < a.d;
      if (!two) e1 = e0;
    }
    float cs[V], sn[V];
    if (rotates) {
      const double p = a.pos64 ? (double)reinterpret_cast<const long long*>(a.pos)[row] : (double)reinterpret_cast<const int*>(a.pos)[row];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double turns = p * a.freq[c + j] * 0.15915494309189533577;      // 1 / (2 pi)
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
    for (int h = (int)group; h < all; h += a.groups) {
      const int w = h >= a.heads[0];
      const int hh = w ? h - a.heads[0] : h;
      const RopeTensor& t = a.t[w];
      const T* src = reinterpret_cast<const T*>(t.in) + outer * t.is0 + inner * t.is1 + hh * t.ish;
      T* dst = reinterpret_cast<T*>(t.out) + outer * t.os0 + inner * t.os1 + hh * t.osh;
      const RopeVec<T, V> x = rope_load<T, V>(src + e0), y = rope_load<T, V>(src + e1);
      RopeVec<T, V> ox = x, oy = y;
      if (rotates) {
        if (INTERLEAVED && V > 1) {
#pragma unroll
          for (int j = 0; j < V; j += 2) {        // x holds the first V/2 pairs, y the others
            const float p0 = rope_f(x.e[j]), p1 = rope_f(x.e[(j + 1) % V]), q0 = rope_f(y.e[j]), q1 = rope_f(y.e[(j + 1) % V]);
            const int f = j / 2, s = V / 2 + j / 2;
            ox.e[j] = rope_t<T>(p0 * cs[f] - p1 * sn[f]);
            ox.e[(j + 1) % V] = rope_t<T>(p1 * cs[f] + p0 * sn[f]);
            oy.e[j] = rope_t<T>(q0 * cs[s] - q1 * sn[s]);
            oy.e[(j + 1) % V] = rope_t<T>(q1 * cs[s] + q0 * sn[s]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float p = rope_f(x.e[j]), q = rope_f(y.e[j]);
            ox.e[j] = rope_t<T>(p * cs[j] - q * sn[j]);
            oy.e[j] = rope_t<T>(q * cs[j] + p * sn[j]);
          }
        }
      }
      rope_store<T, V>(dst + e0, ox);
      if (two) rope_store<T, V>(dst + e1, oy);
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

}  // namespace dh

using namespace dh;

extern "C" {

// Rotates the heads of q (and of k, unless heads_k is 0); in == out (with equal strides) works in place.
int dh_rope_heads(const void* call) {
  const RopeCall& c = *(const RopeCall*)call;
  const int64_t rows = c.rows, inner = c.inner;
  const int heads_q = (int)c.heads_q, heads_k = (int)c.heads_k, d = (int)c.d, rotated = (int)c.rotated;
  const int64_t* ptrs = c.ptrs;
  if (c.heads_q < 0 || c.heads_k < 0 || c.heads_q + c.heads_k > INT32_MAX || c.d <= 0 || c.d > 65536 || c.rotated <= 0 || c.rotated > c.d ||
      (c.rotated & 1) || rows < 0 || inner <= 0 || inner > INT32_MAX) {
    set_last_error_c("dh_rope_heads", "sizes out of range (an even number of rotated elements, at most the head size)");
    return (int)cudaErrorInvalidValue;
  }
  if (rows == 0 || heads_q + heads_k == 0) return 0;
  const int size = c.f32 ? 4 : 2;
  const bool in_place = (heads_q == 0 || ptrs[0] == ptrs[1]) && (heads_k == 0 || ptrs[2] == ptrs[3]);
  // the widest vector that divides half the rotated part, the rest, every address and every stride
  uint64_t odd = (uint64_t)(rotated / 2) * size;
  if (!in_place) odd |= (uint64_t)(d - rotated) * size;
  for (int i = 0; i < 4; ++i) {
    if ((i < 2 ? heads_q : heads_k) == 0) continue;
    odd |= (uint64_t)ptrs[i];
    for (int j = 0; j < 3; ++j) odd |= (uint64_t)(c.strides[3 * i + j] * size);
  }
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
  a.rot_units = a.half / V;
  a.units = a.rot_units + (in_place ? 0 : (d - rotated + 2 * V - 1) / (2 * V));
  const int sms = dh_sm_count();
  const int budget = (c.budget <= 0 || c.budget > sms) ? sms : (int)c.budget;
  const int interleaved = (int)c.interleaved;
  const cudaStream_t s = (cudaStream_t)c.stream;
  // threads that share the heads of a row: enough of them to fill half of the GPU's threads, where there are that few rows
  a.groups = 1;
  while (a.groups * 2 <= heads_q + heads_k && rows * a.units * a.groups < (int64_t)budget * 1024) a.groups *= 2;
  const int64_t most = INT32_MAX / ((int64_t)a.units * a.groups);      // rows of one launch: item numbers stay in 31 bits
  for (int64_t r = 0; r < rows; r += most) {
    a.row0 = r;
    a.rows = rows - r < most ? rows - r : most;
    const int64_t blocks = (a.rows * a.units * a.groups + RT - 1) / RT;
    const int grid = (int)(blocks < (int64_t)budget * 8 ? blocks : (int64_t)budget * 8);
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
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) set_last_error_c("dh_rope_heads", cudaGetErrorString(e));
  return (int)e;
}

}  // extern "C"
