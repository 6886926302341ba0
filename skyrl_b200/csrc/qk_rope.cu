// Rotary positions on the heads of packed projection rows, with the RMS norm of every query and key head in the same
// pass, forward and backward, and the serving form that also writes key and value heads to their paged-cache slots.
//
//   n = x * rsqrt(mean(x^2) + eps) * w            (per head; skipped without norm weights)
//   (a, b) -> (a c - b s, b c + a s)              c, s = cos | sin halves of table[pos], pairs (i, i + R/2) or (2i, 2i+1)
//
// Elements R.. of a head and the heads behind the rotated ones pass unchanged.  Backward, with dn the rotated-back
// gradient and xh = x * rstd:  dw = sum dn * xh,  dx = rstd * (dn * w - xh * mean(dn * w * xh)).
//
// Bound by HBM: every row is read and written once (backward: gradient and input in, gradient out).  A thread owns 16
// elements of a head as two 16-byte vectors, placed so that both members of its eight pairs are its own: rotation needs
// no exchange, the norm only a shuffle over the D/16 lanes of a head.  A warp takes several heads of one token, so the
// angles are loaded once and stay in registers.  Statistics, products and sums are fp32; rows are rounded once on store.
// Positions outside the table give NaN in the rotated elements instead of a read outside it.
#include <cuda_fp16.h>

#include "host_common.h"
#include "ptx.cuh"

namespace sb {
namespace qkr {

struct Args {
  const void* src;       // [T, heads * D] rows, stride src_stride (elements); or fp32 partial sums [n_part][T][heads * D]
  const void* x;         // backward: the forward's input rows (src is the gradient)
  void* dst;             // [T, heads * D], stride dst_stride
  const void* qw;
  const void* kw;
  const int* pos;
  const float* table;    // [max_pos, R]
  const int* slots;
  void* kc;
  void* vc;
  float* dw_part;        // backward: [gridDim.x][2][D]
  long long src_stride, x_stride, dst_stride, part_stride;
  long long n_slots;
  int n_part, max_pos, T, nq, nk, heads, store_heads, D, R;
  int log_group;         // lanes of a head: 1 << log_group >= D / 16
  int blocks_per_row;    // head blocks a token's heads are split into
  float eps, sign;
};

template <typename T>
struct Vec8;  // eight elements: raw registers, to and from fp32
template <>
struct Vec8<__nv_bfloat16> {
  uint4 r;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void get(float* f) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __bfloat1622float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  }
};
template <>
struct Vec8<__half> {
  uint4 r;
  __device__ __forceinline__ void load(const __half* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void store(__half* p) const { *reinterpret_cast<uint4*>(p) = r; }
  __device__ __forceinline__ void get(float* f) const {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(h[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  }
};
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
  __device__ __forceinline__ void get(float* f) const {
    *reinterpret_cast<float4*>(f) = a;
    *reinterpret_cast<float4*>(f + 4) = b;
  }
  __device__ __forceinline__ void set(const float* f) {
    a = *reinterpret_cast<const float4*>(f);
    b = *reinterpret_cast<const float4*>(f + 4);
  }
};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sum over the 1 << lg consecutive lanes of a head.
__device__ __forceinline__ float group_sum(float v, int lg) {
  for (int o = (1 << lg) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rotate the 16 elements of a unit; e[0..7] and e[8..15] are its two vectors.  Half layout: pairs (e[i], e[8 + i]);
// interleaved: (e[2i], e[2i + 1]).
template <bool kInter>
__device__ __forceinline__ void rotate16(float (&e)[16], const float (&c)[8], const float (&s)[8], float sign) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : 8 + i;
    const float a = e[ia], b = e[ib], sn = s[i] * sign;
    e[ia] = a * c[i] - b * sn;
    e[ib] = b * c[i] + a * sn;
  }
}

struct Unit {
  int lo, hi;   // element offsets of the two vectors in the head
  bool live;    // this lane has a unit
  bool rot;     // its elements are rotated
};
template <bool kInter>
__device__ __forceinline__ Unit unit_of(int c, int D, int R) {
  Unit u;
  u.live = c * 16 < D;
  u.rot = c * 16 < R;
  if (kInter || !u.rot) {
    u.lo = 16 * c;
    u.hi = 16 * c + 8;
  } else {
    u.lo = 8 * c;
    u.hi = (R >> 1) + 8 * c;
  }
  return u;
}

__device__ __forceinline__ void load_angles(const float* table, int p, int max_pos, int R, int c, float (&cs)[8], float (&sn)[8]) {
  if (p < 0 || p >= max_pos) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __int_as_float(0x7fffffff);
    return;
  }
  const float* t = table + static_cast<size_t>(p) * R + 8 * c;
  *reinterpret_cast<float4*>(cs) = __ldg(reinterpret_cast<const float4*>(t));
  *reinterpret_cast<float4*>(cs + 4) = __ldg(reinterpret_cast<const float4*>(t + 4));
  *reinterpret_cast<float4*>(sn) = __ldg(reinterpret_cast<const float4*>(t + (R >> 1)));
  *reinterpret_cast<float4*>(sn + 4) = __ldg(reinterpret_cast<const float4*>(t + (R >> 1) + 4));
}

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// One warp per (token, head block) of kIter x (32 / group) heads.  All rows of the block are requested before the first
// is used.
template <typename T, bool kInter, bool kNorm, bool kPart, int kIter>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(a.T) * a.blocks_per_row) return;
  const int t = static_cast<int>(item / a.blocks_per_row);
  const int blk = static_cast<int>(item - static_cast<long long>(t) * a.blocks_per_row);
  const int hpw = 32 >> a.log_group;
  const int c = lane & ((1 << a.log_group) - 1);
  const int head0 = blk * (kIter * hpw) + (lane >> a.log_group);
  const Unit u = unit_of<kInter>(c, a.D, a.R);
  Vec8<T> vlo[kIter], vhi[kIter];
#pragma unroll
  for (int it = 0; it < kIter; ++it) {
    const int h = head0 + it * hpw;
    if (u.live && h < a.heads) {
      if (kPart) {
        float lo[8] = {}, hi[8] = {};
        const float* p = static_cast<const float*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
        for (int i = 0; i < a.n_part; ++i, p += a.part_stride) {
          Vec8<float> l, r;
          l.load(p + u.lo);
          r.load(p + u.hi);
          float fl[8], fr[8];
          l.get(fl);
          r.get(fr);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            lo[j] += fl[j];
            hi[j] += fr[j];
          }
        }
        // the unsplit projection stores its rows in this type: keep that rounding, so that both paths agree
        vlo[it].set(lo);
        vhi[it].set(hi);
      } else {
        const T* p = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
        vlo[it].load(p + u.lo);
        vhi[it].load(p + u.hi);
      }
    }
  }
  float cs[8], sn[8];
  if (u.rot) load_angles(a.table, __ldg(a.pos + t), a.max_pos, a.R, c, cs, sn);
  long long slot = a.slots ? __ldg(a.slots + t) : -1;
  if (slot >= a.n_slots) slot = -1;
#pragma unroll
  for (int it = 0; it < kIter; ++it) {
    const int h = head0 + it * hpw;
    const bool on = u.live && h < a.heads;
    const bool turned = h < a.nq + a.nk;
    float e[16];
    float ss = 0.f;
    if (on && turned) {
      vlo[it].get(e);
      vhi[it].get(e + 8);
      if (kNorm) {
#pragma unroll
        for (int j = 0; j < 16; ++j) ss += e[j] * e[j];
      }
    }
    if (kNorm) ss = group_sum(ss, a.log_group);
    if (!on) continue;
    if (turned) {
      if (kNorm) {
        const float r = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
        const T* w = static_cast<const T*>(h < a.nq ? a.qw : a.kw);
        Vec8<T> wl, wh;
        wl.load(w + u.lo);
        wh.load(w + u.hi);
        float f[16];
        wl.get(f);
        wh.get(f + 8);
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] = e[j] * r * f[j];
      }
      if (u.rot) rotate16<kInter>(e, cs, sn, a.sign);
      if (kNorm || u.rot) {
        vlo[it].set(e);
        vhi[it].set(e + 8);
      }
    }
    if (h < a.store_heads) {
      T* d = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D;
      vlo[it].store(d + u.lo);
      vhi[it].store(d + u.hi);
    }
    if (slot >= 0 && h >= a.nq) {
      T* base = static_cast<T*>(turned ? a.kc : a.vc);
      T* d = base + (static_cast<size_t>(slot) * a.nk + (turned ? h - a.nq : h - a.nq - a.nk)) * a.D;
      vlo[it].store(d + u.lo);
      vhi[it].store(d + u.hi);
    }
  }
}

// Backward of norm + rotation.  Warps walk over (token, head block) items; a lane's 16 elements are the same in every
// head, so it carries the gradient of its query and key weights in registers.  Each CTA leaves one row of partial sums
// for reduce_dw_kernel: no atomics, the result does not change from run to run.
template <typename T, bool kInter, int kIter>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const Args a) {
  extern __shared__ float sdw[];  // [kWarps][2 * D]
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hpw = 32 >> a.log_group;
  const int c = lane & ((1 << a.log_group) - 1);
  const Unit u = unit_of<kInter>(c, a.D, a.R);
  float aq[16], ak[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) aq[j] = ak[j] = 0.f;
  const long long items = static_cast<long long>(a.T) * a.blocks_per_row;
  for (long long item = static_cast<long long>(blockIdx.x) * kWarps + warp; item < items;
       item += static_cast<long long>(gridDim.x) * kWarps) {
    const int t = static_cast<int>(item / a.blocks_per_row);
    const int blk = static_cast<int>(item - static_cast<long long>(t) * a.blocks_per_row);
    const int head0 = blk * (kIter * hpw) + (lane >> a.log_group);
    Vec8<T> dlo[kIter], dhi[kIter], xlo[kIter], xhi[kIter];
#pragma unroll
    for (int it = 0; it < kIter; ++it) {
      const int h = head0 + it * hpw;
      if (u.live && h < a.heads) {
        const T* p = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
        dlo[it].load(p + u.lo);
        dhi[it].load(p + u.hi);
        if (h < a.nq + a.nk) {
          const T* q = static_cast<const T*>(a.x) + static_cast<size_t>(t) * a.x_stride + h * a.D;
          xlo[it].load(q + u.lo);
          xhi[it].load(q + u.hi);
        }
      }
    }
    float cs[8], sn[8];
    if (u.rot) load_angles(a.table, __ldg(a.pos + t), a.max_pos, a.R, c, cs, sn);
#pragma unroll
    for (int it = 0; it < kIter; ++it) {
      const int h = head0 + it * hpw;
      const bool on = u.live && h < a.heads;
      const bool turned = h < a.nq + a.nk;
      float g[16], x[16], w[16];
      float ss = 0.f, dot = 0.f;
      if (on && turned) {
        dlo[it].get(g);
        dhi[it].get(g + 8);
        xlo[it].get(x);
        xhi[it].get(x + 8);
        const T* wp = static_cast<const T*>(h < a.nq ? a.qw : a.kw);
        Vec8<T> wl, wh;
        wl.load(wp + u.lo);
        wh.load(wp + u.hi);
        wl.get(w);
        wh.get(w + 8);
        if (u.rot) rotate16<kInter>(g, cs, sn, -1.f);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          ss += x[j] * x[j];
          dot += g[j] * w[j] * x[j];
        }
      }
      ss = group_sum(ss, a.log_group);
      dot = group_sum(dot, a.log_group);
      if (!on) continue;
      if (turned) {
        const float inv_d = 1.f / static_cast<float>(a.D);
        const float r = rsqrtf(ss * inv_d + a.eps);
        const float m = dot * r * r * inv_d;  // mean(dn w xh) * rstd
        const bool is_q = h < a.nq;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float xg = g[j] * x[j] * r;
          aq[j] += is_q ? xg : 0.f;
          ak[j] += is_q ? 0.f : xg;
          g[j] = r * (g[j] * w[j] - x[j] * m);
        }
        dlo[it].set(g);
        dhi[it].set(g + 8);
      }
      T* d = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D;
      dlo[it].store(d + u.lo);
      dhi[it].store(d + u.hi);
    }
  }
  if (!a.dw_part) return;
  for (int o = 16; o >= (1 << a.log_group); o >>= 1) {  // lanes that own the same elements of different heads
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      aq[j] += __shfl_xor_sync(0xffffffffu, aq[j], o);
      ak[j] += __shfl_xor_sync(0xffffffffu, ak[j], o);
    }
  }
  if ((lane >> a.log_group) == 0 && u.live) {
    float* s = sdw + warp * 2 * a.D;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = j < 8 ? u.lo + j : u.hi + j - 8;
      s[e] = aq[j];
      s[a.D + e] = ak[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sdw[w * 2 * a.D + i];
    a.dw_part[static_cast<size_t>(blockIdx.x) * 2 * a.D + i] = v;
  }
}

// Any head size, rotated width, stride or alignment: one warp per (token, head), element by element.  A lane reads and
// writes the same elements, so rows may be rotated in place.
template <typename T, bool kPart>
__device__ __forceinline__ float elem(const Args& a, int t, int h, int e) {
  if (kPart) {
    const float* p = static_cast<const float*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D + e;
    float v = 0.f;
    for (int i = 0; i < a.n_part; ++i) v += p[static_cast<size_t>(i) * a.part_stride];
    return to_f(from_f<T>(v));
  }
  return to_f(static_cast<const T*>(a.src)[static_cast<size_t>(t) * a.src_stride + h * a.D + e]);
}

template <typename T, bool kInter, bool kNorm, bool kPart>
__global__ void __launch_bounds__(kThreads) fwd_any_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(a.T) * a.heads) return;
  const int t = static_cast<int>(item / a.heads), h = static_cast<int>(item - static_cast<long long>(t) * a.heads);
  const bool turned = h < a.nq + a.nk;
  long long slot = a.slots ? a.slots[t] : -1;
  if (slot >= a.n_slots) slot = -1;
  T* d = h < a.store_heads ? static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D : nullptr;
  T* cd = nullptr;
  if (slot >= 0 && h >= a.nq)
    cd = static_cast<T*>(turned ? a.kc : a.vc) +
         (static_cast<size_t>(slot) * a.nk + (turned ? h - a.nq : h - a.nq - a.nk)) * a.D;
  float r = 1.f;
  const T* w = static_cast<const T*>(h < a.nq ? a.qw : a.kw);
  if (kNorm && turned) {
    float ss = 0.f;
    for (int e = lane; e < a.D; e += 32) {
      const float v = elem<T, kPart>(a, t, h, e);
      ss += v * v;
    }
    r = rsqrtf(warp_sum(ss) / static_cast<float>(a.D) + a.eps);
  }
  auto put = [&](int e, float v) {
    const T o = from_f<T>(v);
    if (d) d[e] = o;
    if (cd) cd[e] = o;
  };
  const int half = turned ? a.R >> 1 : 0;
  const int p = a.pos[t];
  const bool known = p >= 0 && p < a.max_pos;
  for (int i = lane; i < half; i += 32) {
    const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : half + i;
    float va = elem<T, kPart>(a, t, h, ia), vb = elem<T, kPart>(a, t, h, ib);
    if (kNorm) {
      va = va * r * to_f(w[ia]);
      vb = vb * r * to_f(w[ib]);
    }
    const float nan = __int_as_float(0x7fffffff);
    const float c = known ? a.table[static_cast<size_t>(p) * a.R + i] : nan;
    const float s = (known ? a.table[static_cast<size_t>(p) * a.R + half + i] : nan) * a.sign;
    put(ia, va * c - vb * s);
    put(ib, vb * c + va * s);
  }
  for (int e = 2 * half + lane; e < a.D; e += 32) {
    float v = elem<T, kPart>(a, t, h, e);
    if (kNorm && turned) v = v * r * to_f(w[e]);
    put(e, v);
  }
}

template <typename T, bool kInter>
__global__ void __launch_bounds__(kThreads) bwd_any_kernel(const Args a) {
  extern __shared__ float sdw[];  // [kWarps][2 * D], a row of its own for every warp
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* acc = sdw + warp * 2 * a.D;
  for (int i = lane; i < 2 * a.D; i += 32) acc[i] = 0.f;
  __syncwarp();
  const long long items = static_cast<long long>(a.T) * a.heads;
  const int half = a.R >> 1;
  for (long long item = static_cast<long long>(blockIdx.x) * kWarps + warp; item < items;
       item += static_cast<long long>(gridDim.x) * kWarps) {
    const int t = static_cast<int>(item / a.heads), h = static_cast<int>(item - static_cast<long long>(t) * a.heads);
    const T* g = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
    T* d = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D;
    if (h >= a.nq + a.nk) {
      for (int e = lane; e < a.D; e += 32) d[e] = g[e];
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + static_cast<size_t>(t) * a.x_stride + h * a.D;
    const T* w = static_cast<const T*>(h < a.nq ? a.qw : a.kw);
    float* dw = acc + (h < a.nq ? 0 : a.D);
    const int p = a.pos[t];
    const bool known = p >= 0 && p < a.max_pos;
    const float nan = __int_as_float(0x7fffffff);
    auto back = [&](int i, float& ga, float& gb) {  // gradient of pair i before the rotation
      const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : half + i;
      const float c = known ? a.table[static_cast<size_t>(p) * a.R + i] : nan;
      const float s = known ? a.table[static_cast<size_t>(p) * a.R + half + i] : nan;
      const float va = to_f(g[ia]), vb = to_f(g[ib]);
      ga = va * c + vb * s;
      gb = vb * c - va * s;
    };
    float ss = 0.f, dot = 0.f;
    for (int e = lane; e < a.D; e += 32) {
      const float v = to_f(x[e]);
      ss += v * v;
    }
    for (int i = lane; i < half; i += 32) {
      const int ia = kInter ? 2 * i : i, ib = kInter ? 2 * i + 1 : half + i;
      float ga, gb;
      back(i, ga, gb);
      dot += ga * to_f(w[ia]) * to_f(x[ia]) + gb * to_f(w[ib]) * to_f(x[ib]);
    }
    for (int e = a.R + lane; e < a.D; e += 32) dot += to_f(g[e]) * to_f(w[e]) * to_f(x[e]);
    ss = warp_sum(ss);
    dot = warp_sum(dot);
    const float r = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
    const float m = dot * r * r / static_cast<float>(a.D);
    auto put = [&](int e, float ge) {
      const float xe = to_f(x[e]);
      dw[e] += ge * xe * r;
      d[e] = from_f<T>(r * (ge * to_f(w[e]) - xe * m));
    };
    for (int i = lane; i < half; i += 32) {
      float ga, gb;
      back(i, ga, gb);
      put(kInter ? 2 * i : i, ga);
      put(kInter ? 2 * i + 1 : half + i, gb);
    }
    for (int e = a.R + lane; e < a.D; e += 32) put(e, to_f(g[e]));  // an element falls to the same lane in every head
  }
  if (!a.dw_part) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.D; i += kThreads) {
    float v = 0.f;
    for (int k = 0; k < kWarps; ++k) v += sdw[k * 2 * a.D + i];
    a.dw_part[static_cast<size_t>(blockIdx.x) * 2 * a.D + i] = v;
  }
}

// Sum of the CTAs' partial rows, 32 columns a CTA, always in the same order.  Columns [0, D) are the query weight's
// gradient, [D, 2D) the key's; each is added to an fp32 buffer or stored in the rows' type.
constexpr int kReduceRows = 32;
template <typename T>
__global__ void __launch_bounds__(32 * kReduceRows)
reduce_dw_kernel(const float* part, int rows, int D, void* dq, void* dk, int accumulate) {
  __shared__ float s[kReduceRows][33];
  pdl_launch_dependents();
  pdl_wait();
  const int col = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (col < 2 * D)
    for (int r = threadIdx.y; r < rows; r += kReduceRows) v += part[static_cast<size_t>(r) * 2 * D + col];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = warp_sum(s[threadIdx.x][threadIdx.y]);  // warp y sums column y
  const int out = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x != 0 || out >= 2 * D) return;
  void* base = out < D ? dq : dk;
  const int e = out < D ? out : out - D;
  if (!base) return;
  if (accumulate)
    static_cast<float*>(base)[e] += v;
  else
    static_cast<T*>(base)[e] = from_f<T>(v);
}

bool vectorised(const Args& a, size_t elt) {
  const auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const long long per = 16 / static_cast<long long>(elt);
  const bool strides = a.n_part ? (a.src_stride % 4 == 0 && a.part_stride % 4 == 0) : a.src_stride % per == 0;
  return a.D % 16 == 0 && a.R % 16 == 0 && strides && a.x_stride % per == 0 && a.dst_stride % per == 0 && al(a.src) &&
         al(a.x) && al(a.dst) && al(a.qw) && al(a.kw) && al(a.table) && al(a.kc) && al(a.vc);
}

int log2_ceil(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

template <typename T, bool kInter, bool kNorm, bool kPart>
cudaError_t launch_fwd(Args a, cudaStream_t st) {
  if (!vectorised(a, sizeof(T))) {
    const long long ctas = (static_cast<long long>(a.T) * a.heads + kWarps - 1) / kWarps;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_pdl(fwd_any_kernel<T, kInter, kNorm, kPart>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, st, a);
  }
  a.log_group = log2_ceil(a.D / 16);
  const int hpw = 32 >> a.log_group;
  const int passes = (a.heads + hpw - 1) / hpw;
  // few rows: every head on a warp of its own, so that the whole call is one round of loads; many: four at a time share
  // the token's angles and keep eight loads a thread in flight
  const bool wide = static_cast<long long>(a.T) * passes >= 8LL * kWarps * sm_count() * 4;
  a.blocks_per_row = wide ? (passes + 3) / 4 : passes;
  const long long ctas = (static_cast<long long>(a.T) * a.blocks_per_row + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  if (wide) return launch_pdl(fwd_kernel<T, kInter, kNorm, kPart, 4>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, st, a);
  return launch_pdl(fwd_kernel<T, kInter, kNorm, kPart, 1>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, st, a);
}

template <typename T>
cudaError_t pick_fwd(const Args& a, bool inter, cudaStream_t st) {
  const bool norm = a.qw != nullptr;
  if (a.n_part) {
    if (inter) return norm ? launch_fwd<T, true, true, true>(a, st) : launch_fwd<T, true, false, true>(a, st);
    return norm ? launch_fwd<T, false, true, true>(a, st) : launch_fwd<T, false, false, true>(a, st);
  }
  if (inter) return norm ? launch_fwd<T, true, true, false>(a, st) : launch_fwd<T, true, false, false>(a, st);
  return norm ? launch_fwd<T, false, true, false>(a, st) : launch_fwd<T, false, false, false>(a, st);
}

constexpr int kBwdIter = 2;
int bwd_ctas(long long items) {
  const long long want = (items + kWarps - 1) / kWarps, cap = 4LL * sm_count();
  return static_cast<int>(want < cap ? want : cap);
}

template <typename T, bool kInter>
cudaError_t launch_bwd(Args a, int ctas, cudaStream_t st) {
  const size_t smem = sizeof(float) * kWarps * 2 * a.D;  // at most 32 KB (D <= 512)
  if (!vectorised(a, sizeof(T)))
    return launch_pdl(bwd_any_kernel<T, kInter>, dim3(ctas), dim3(kThreads), smem, st, a);
  a.log_group = log2_ceil(a.D / 16);
  const int hpw = 32 >> a.log_group;
  a.blocks_per_row = (a.heads + kBwdIter * hpw - 1) / (kBwdIter * hpw);
  return launch_pdl(bwd_kernel<T, kInter, kBwdIter>, dim3(ctas), dim3(kThreads), smem, st, a);
}

bool shape_ok(int T, int nq, int nk, int heads, int D, int R, int max_pos) {
  return T > 0 && nq >= 0 && nk >= 0 && nq + nk > 0 && heads >= nq + nk && D > 0 && D <= 512 && R > 0 && R <= D &&
         (R & 1) == 0 && max_pos > 0 && static_cast<long long>(heads) * D < (1LL << 30);
}

}  // namespace qkr
}  // namespace sb

extern "C" {

// dtype: 0 bf16, 1 fp16, 2 fp32.  dst may be src (rows in place; strides equal), then heads behind nq + nk are not
// stored again.  n_part > 0: src holds fp32 partial sums.  qw / kw: both or neither.  slots / k_cache / v_cache: all or
// none; with them the rows are nq query, nk key and nk value heads.
int sb_qk_rope_fwd(const void* src, void* dst, const void* qw, const void* kw, const int* pos, const float* table,
                   const int* slots, void* kc, void* vc, long long n_slots, long long src_stride, long long dst_stride,
                   long long part_stride, int n_part, int max_pos, int T, int nq, int nk, int heads, int D, int R, int dtype,
                   int interleaved, float eps, float sign, void* stream) {
  if (!sb::qkr::shape_ok(T, nq, nk, heads, D, R, max_pos) || n_part < 0 || (!qw) != (!kw)) return SB_ERR_ARG;
  if (slots && (!kc || !vc || heads != nq + 2 * nk)) return SB_ERR_ARG;
  if (dst == src && (n_part || src_stride != dst_stride)) return SB_ERR_ARG;
  sb::qkr::Args a = {};
  a.src = src;
  a.dst = dst;
  a.qw = qw;
  a.kw = kw;
  a.pos = pos;
  a.table = table;
  a.slots = slots;
  a.kc = kc;
  a.vc = vc;
  a.n_slots = n_slots;
  a.src_stride = src_stride;
  a.dst_stride = dst_stride;
  a.part_stride = part_stride;
  a.n_part = n_part;
  a.max_pos = max_pos;
  a.T = T;
  a.nq = nq;
  a.nk = nk;
  a.store_heads = dst == src ? nq + nk : heads;
  a.heads = slots ? heads : a.store_heads;
  a.D = D;
  a.R = R;
  a.eps = eps;
  a.sign = sign;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == 0)
    e = sb::qkr::pick_fwd<__nv_bfloat16>(a, interleaved, st);
  else if (dtype == 1)
    e = sb::qkr::pick_fwd<__half>(a, interleaved, st);
  else if (dtype == 2)
    e = sb::qkr::pick_fwd<float>(a, interleaved, st);
  else
    return SB_ERR_ARG;
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

// Rows of partial sums [2 * D] floats that sb_qk_norm_rope_bwd needs for T rows of `heads` heads of size D.
int sb_qk_norm_rope_bwd_parts(int T, int heads, int D) {
  if (T <= 0 || heads <= 0 || D <= 0 || D > 512) return 0;
  // every variant has at least this many (token, head block) items of work and at most heads of them a token
  return sb::qkr::bwd_ctas(static_cast<long long>(T) * heads);
}

// dy, x, dx: [T, heads * D] rows.  dqw / dkw: gradients of the norm weights (null: not wanted), added to fp32 buffers when
// accumulate is set, else stored in the rows' type.  part: n_parts x 2 D floats of scratch, not read before it is written.
int sb_qk_norm_rope_bwd(const void* dy, const void* x, void* dx, const void* qw, const void* kw, const int* pos,
                        const float* table, void* dqw, void* dkw, float* part, int n_parts, long long dy_stride,
                        long long x_stride, long long dx_stride, int max_pos, int T, int nq, int nk, int heads, int D, int R,
                        int dtype, int interleaved, int accumulate, float eps, void* stream) {
  if (!sb::qkr::shape_ok(T, nq, nk, heads, D, R, max_pos) || !qw || !kw || n_parts <= 0) return SB_ERR_ARG;
  if ((dqw || dkw) && !part) return SB_ERR_ARG;
  sb::qkr::Args a = {};
  a.src = dy;
  a.x = x;
  a.dst = dx;
  a.qw = qw;
  a.kw = kw;
  a.pos = pos;
  a.table = table;
  a.dw_part = (dqw || dkw) ? part : nullptr;
  a.src_stride = dy_stride;
  a.x_stride = x_stride;
  a.dst_stride = dx_stride;
  a.max_pos = max_pos;
  a.T = T;
  a.nq = nq;
  a.nk = nk;
  a.heads = a.store_heads = heads;
  a.D = D;
  a.R = R;
  a.eps = eps;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 rg((2 * D + 31) / 32), rb(32, sb::qkr::kReduceRows);
  cudaError_t e;
  if (dtype == 0)
    e = interleaved ? sb::qkr::launch_bwd<__nv_bfloat16, true>(a, n_parts, st) : sb::qkr::launch_bwd<__nv_bfloat16, false>(a, n_parts, st);
  else if (dtype == 1)
    e = interleaved ? sb::qkr::launch_bwd<__half, true>(a, n_parts, st) : sb::qkr::launch_bwd<__half, false>(a, n_parts, st);
  else if (dtype == 2)
    e = interleaved ? sb::qkr::launch_bwd<float, true>(a, n_parts, st) : sb::qkr::launch_bwd<float, false>(a, n_parts, st);
  else
    return SB_ERR_ARG;
  if (e != cudaSuccess) return SB_ERR_CUDA;
  if (!a.dw_part) return SB_OK;
  if (dtype == 0)
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<__nv_bfloat16>, rg, rb, 0, st, part, n_parts, D, dqw, dkw, accumulate);
  else if (dtype == 1)
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<__half>, rg, rb, 0, st, part, n_parts, D, dqw, dkw, accumulate);
  else
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<float>, rg, rb, 0, st, part, n_parts, D, dqw, dkw, accumulate);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

}  // extern "C"
