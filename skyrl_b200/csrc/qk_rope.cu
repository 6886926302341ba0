// Rotary positions on the heads of packed projection rows, with the RMS norm of every query and key head in the same
// pass, forward and backward, and the serving form that also writes key and value heads to their paged-cache slots.
//
//   n = x * rsqrt(mean(x^2) + eps) * w            (per head; skipped without norm weights)
//   (a, b) -> (a c - b s, b c + a s)              c, s = cos | sin halves of table[pos], pairs (i, i + R/2) or (2i, 2i+1)
//
// Elements R.. of a head and the heads behind the rotated ones pass unchanged.  Backward, with dn the rotated-back
// gradient and xh = x * rstd:  dw = sum dn * xh,  dx = rstd * (dn * w - xh * mean(dn * w * xh)).
//
// Bound by HBM: every row is read and written once (backward: gradient and input in, gradient out).  A lane owns whole
// pairs of a head (16 elements, 8 in the pipeline for many rows), so that rotation needs no exchange and the norm only a
// shuffle over a head's lanes; a warp holds several heads of one token at a time and loads the angles once for all.
// Statistics, products and sums are fp32; rows are rounded once on store.  Variants: plain loads for few rows (16 or 8
// elements a lane), a pipeline of bulk copies through shared memory for many, element by element for any size and alignment.
// Positions outside the table give NaN in the rotated elements instead of a read outside it.
// 16384 rows of 32 + 4 + 4 heads of 128 in bf16: forward 60 us, 88% of the measured copy bandwidth; backward 90 us, 84%.
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
  int log_group;         // lanes of a head: 1 << log_group >= D / 16 (fwd_kernel, bwd_kernel) or D / 8
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

// Partial sums are added up in two fp32 words, rounded to fp32 and then, as an unsplit projection's sum would be, to the
// rows' type: the result does not depend on how many parts it came in.
struct Sum {
  float hi = 0.f, lo = 0.f;
  __device__ __forceinline__ void add(float v) {
    const float s = hi + v, b = s - hi;
    lo += (hi - (s - b)) + (v - b);  // what the addition rounded away
    hi = s;
  }
  // an infinite sum has no finite remainder (inf - inf)
  __device__ __forceinline__ float get() const { return lo == lo ? hi + lo : hi; }
};

// Sum over the 1 << lg consecutive lanes of a head.
__device__ __forceinline__ float group_sum(float v, int lg) {
#pragma unroll
  for (int o = 4; o >= 0; --o)
    if (o < lg) v += __shfl_xor_sync(0xffffffffu, v, 1 << o);
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

// Few rows: a warp takes as many neighbouring heads of a token as fit its lanes, so that the call is one round of loads.
template <typename T, bool kInter, bool kNorm>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(a.T) * a.blocks_per_row) return;
  const int t = static_cast<int>(item / a.blocks_per_row);
  const int blk = static_cast<int>(item - static_cast<long long>(t) * a.blocks_per_row);
  const int c = lane & ((1 << a.log_group) - 1);
  const int h = (blk << (5 - a.log_group)) + (lane >> a.log_group);
  const Unit u = unit_of<kInter>(c, a.D, a.R);
  const bool on = u.live && h < a.heads, turned = h < a.nq + a.nk;
  Vec8<T> vlo, vhi;
  if (on) {
    const T* p = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
    vlo.load(p + u.lo);
    vhi.load(p + u.hi);
  }
  float cs[8], sn[8];
  if (u.rot) load_angles(a.table, a.pos[t], a.max_pos, a.R, c, cs, sn);
  long long slot = a.slots ? a.slots[t] : -1;
  if (slot >= a.n_slots) slot = -1;
  float e[16];
  float ss = 0.f;
  if (on && turned) {
    vlo.get(e);
    vhi.get(e + 8);
    if (kNorm) {
#pragma unroll
      for (int j = 0; j < 16; ++j) ss += e[j] * e[j];
    }
  }
  if (kNorm) ss = group_sum(ss, a.log_group);
  if (!on) return;
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
      vlo.set(e);
      vhi.set(e + 8);
    }
  }
  if (h < a.store_heads) {
    T* d = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D;
    vlo.store(d + u.lo);
    vhi.store(d + u.hi);
  }
  if (slot >= 0 && h >= a.nq) {
    T* base = static_cast<T*>(turned ? a.kc : a.vc);
    T* d = base + (static_cast<size_t>(slot) * a.nk + (turned ? h - a.nq : h - a.nq - a.nk)) * a.D;
    vlo.store(d + u.lo);
    vhi.store(d + u.hi);
  }
}

// Backward of norm + rotation for few rows.  A lane's 16 elements are the same in every head, so it carries the gradient
// of its query and key weights in registers.  Each CTA leaves one row of partial sums for reduce_dw_kernel: no atomics, the
// result does not change from run to run.
template <typename T, bool kInter>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const Args a) {
  extern __shared__ float sdw[];  // [kWarps][2 * D]
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = lane & ((1 << a.log_group) - 1);
  const Unit u = unit_of<kInter>(c, a.D, a.R);
  const float inv_d = 1.f / static_cast<float>(a.D);
  float aq[16], ak[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) aq[j] = ak[j] = 0.f;
  const long long items = static_cast<long long>(a.T) * a.blocks_per_row;
  for (long long item = static_cast<long long>(blockIdx.x) * kWarps + warp; item < items;
       item += static_cast<long long>(gridDim.x) * kWarps) {
    const int t = static_cast<int>(item / a.blocks_per_row);
    const int blk = static_cast<int>(item - static_cast<long long>(t) * a.blocks_per_row);
    const int h = (blk << (5 - a.log_group)) + (lane >> a.log_group);
    const bool on = u.live && h < a.heads, turned = h < a.nq + a.nk;
    Vec8<T> dlo, dhi;
    float g[16], x[16], w[16];
    float ss = 0.f, dot = 0.f;
    if (on) {
      const T* p = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D;
      dlo.load(p + u.lo);
      dhi.load(p + u.hi);
      if (turned) {
        const T* q = static_cast<const T*>(a.x) + static_cast<size_t>(t) * a.x_stride + h * a.D;
        const T* wp = static_cast<const T*>(h < a.nq ? a.qw : a.kw);
        Vec8<T> l, r;
        l.load(q + u.lo);
        r.load(q + u.hi);
        l.get(x);
        r.get(x + 8);
        l.load(wp + u.lo);
        r.load(wp + u.hi);
        l.get(w);
        r.get(w + 8);
        dlo.get(g);
        dhi.get(g + 8);
        if (u.rot) {
          float cs[8], sn[8];
          load_angles(a.table, a.pos[t], a.max_pos, a.R, c, cs, sn);
          rotate16<kInter>(g, cs, sn, -1.f);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          ss += x[j] * x[j];
          dot += g[j] * w[j] * x[j];
        }
      }
    }
    ss = group_sum(ss, a.log_group);
    dot = group_sum(dot, a.log_group);
    if (!on) continue;
    if (turned) {
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
      dlo.set(g);
      dhi.set(g + 8);
    }
    T* d = static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D;
    dlo.store(d + u.lo);
    dhi.store(d + u.hi);
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

// ---------------------------------------------------------------------------
// Many rows: every warp runs its own pipeline over row pieces (kStages buffers in shared memory, filled and emptied by
// bulk copies), so that the loads of the next pieces, the arithmetic of this one and the stores of the last are under way
// at once and no register waits for memory.  A piece is `block_heads` neighbouring heads of one token, one copy each way.
// A lane owns eight elements of a head, four pairs, which keeps 16 warps within 128 registers: 16 elements, or two heads at
// a time, spill there, and what 12 warps gain in registers they lose in latency.  The norm weights are multiplied into the
// angles once a piece, and products are two fp32 at a time (f32x2).
// ---------------------------------------------------------------------------
typedef unsigned long long f2;  // two fp32
__device__ __forceinline__ f2 pack2(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float sum2(f2 v) {
  float x, y;
  unpack2(v, x, y);
  return x + y;
}

// Four neighbouring elements.
__device__ __forceinline__ void get4(const __nv_bfloat16* p, float (&e)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  e[0] = __uint_as_float(v.x << 16);
  e[1] = __uint_as_float(v.x & 0xffff0000u);
  e[2] = __uint_as_float(v.y << 16);
  e[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void get4(const __half* p, float (&e)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  e[0] = a.x;
  e[1] = a.y;
  e[2] = b.x;
  e[3] = b.y;
}
__device__ __forceinline__ void get4(const float* p, float (&e)[4]) { *reinterpret_cast<float4*>(e) = *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ void put4(__nv_bfloat16* p, const float (&e)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]));
}
__device__ __forceinline__ void put4(__half* p, const float (&e)[4]) {
  const __half2 a = __floats2half2_rn(e[0], e[1]), b = __floats2half2_rn(e[2], e[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void put4(float* p, const float (&e)[4]) { *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(e); }

// Two neighbouring elements.
__device__ __forceinline__ f2 get2(const __nv_bfloat16* p) {
  const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
  return pack2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ f2 get2(const __half* p) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(p));
  return pack2(v.x, v.y);
}
__device__ __forceinline__ f2 get2(const float* p) { return *reinterpret_cast<const f2*>(p); }
__device__ __forceinline__ void put2(__nv_bfloat16* p, f2 v) {
  float x, y;
  unpack2(v, x, y);
  *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(x, y);
}
__device__ __forceinline__ void put2(__half* p, f2 v) {
  float x, y;
  unpack2(v, x, y);
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
}
__device__ __forceinline__ void put2(float* p, f2 v) { *reinterpret_cast<f2*>(p) = v; }

// The first (a) and second (b) members of a lane's four pairs, two at a time.
struct Pairs {
  f2 a[2], b[2];
};
// Eight neighbouring elements; 16 bytes at once where they are that.
template <typename T>
__device__ __forceinline__ void get8(const T* p, float (&l)[4], float (&r)[4]) {
  if constexpr (sizeof(T) == 2) {
    uint4 v = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
    get4(e, l);
    get4(e + 4, r);
  } else {
    get4(p, l);
    get4(p + 4, r);
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&l)[4], const float (&r)[4]) {
  if constexpr (sizeof(T) == 2) {
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
    put4(e, l);
    put4(e + 4, r);
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    put4(p, l);
    put4(p + 4, r);
  }
}
// Where a lane's elements lie in a head: its four first members, or its first two pairs' and its last two pairs'.
struct Spot {
  int lo, hi;    // first and second members of pairs 0 and 1; without kFine of all four
  int lo2, hi2;  // of pairs 2 and 3
};
template <bool kInter, bool kFine>
__device__ __forceinline__ Spot spot_of(int c, int half, bool live, bool rot, bool rot2) {
  Spot at;
  at.lo = !live ? 0 : kInter || !rot ? 8 * c : 4 * c;
  if (kFine) {
    at.hi = rot ? half + 4 * c : at.lo + 2;
    at.lo2 = !live ? 4 : rot2 ? 4 * c + 2 : 8 * c + 4;
    at.hi2 = rot2 ? half + 4 * c + 2 : at.lo2 + 2;
  } else {
    at.hi = kInter || !rot ? at.lo + 4 : half + 4 * c;
  }
  return at;
}
template <typename T, bool kInter, bool kFine>
__device__ __forceinline__ Pairs get_pairs(const T* p, const Spot& at) {
  Pairs v;
  if (kFine && !kInter) {
    v.a[0] = get2(p + at.lo);
    v.b[0] = get2(p + at.hi);
    v.a[1] = get2(p + at.lo2);
    v.b[1] = get2(p + at.hi2);
    return v;
  }
  float l[4], r[4];
  if (kInter) {
    get8(p + at.lo, l, r);
    v.a[0] = pack2(l[0], l[2]);
    v.b[0] = pack2(l[1], l[3]);
    v.a[1] = pack2(r[0], r[2]);
    v.b[1] = pack2(r[1], r[3]);
  } else {
    get4(p + at.lo, l);
    get4(p + at.hi, r);
    v.a[0] = pack2(l[0], l[1]);
    v.a[1] = pack2(l[2], l[3]);
    v.b[0] = pack2(r[0], r[1]);
    v.b[1] = pack2(r[2], r[3]);
  }
  return v;
}
template <typename T, bool kInter, bool kFine>
__device__ __forceinline__ void put_pairs(T* p, const Spot& at, const Pairs& v) {
  if (kFine && !kInter) {
    put2(p + at.lo, v.a[0]);
    put2(p + at.hi, v.b[0]);
    put2(p + at.lo2, v.a[1]);
    put2(p + at.hi2, v.b[1]);
    return;
  }
  float l[4], r[4];
  if (kInter) {
    unpack2(v.a[0], l[0], l[2]);
    unpack2(v.b[0], l[1], l[3]);
    unpack2(v.a[1], r[0], r[2]);
    unpack2(v.b[1], r[1], r[3]);
    put8(p + at.lo, l, r);
  } else {
    unpack2(v.a[0], l[0], l[1]);
    unpack2(v.a[1], l[2], l[3]);
    unpack2(v.b[0], r[0], r[1]);
    unpack2(v.b[1], r[2], r[3]);
    put4(p + at.lo, l);
    put4(p + at.hi, r);
  }
}

__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}

// Angles of a rotating lane's four pairs at position p; 1 and 0 for pairs that do not rotate.
template <bool kFine>
__device__ __forceinline__ void load_angles4(const Args& a, int p, int c, bool rot2, float4& cs, float4& sn) {
  if (p < 0 || p >= a.max_pos) {
    const float nan = __int_as_float(0x7fffffff);
    cs = rot2 ? make_float4(nan, nan, nan, nan) : make_float4(nan, nan, 1.f, 1.f);
    sn = rot2 ? make_float4(nan, nan, nan, nan) : make_float4(nan, nan, 0.f, 0.f);
    return;
  }
  const float* t = a.table + static_cast<size_t>(p) * a.R + 4 * c;
  const float* u = t + (a.R >> 1);
  if (kFine) {
    const float2 c0 = __ldg(reinterpret_cast<const float2*>(t)), s0 = __ldg(reinterpret_cast<const float2*>(u));
    float2 c1 = make_float2(1.f, 1.f), s1 = make_float2(0.f, 0.f);
    if (rot2) {
      c1 = __ldg(reinterpret_cast<const float2*>(t + 2));
      s1 = __ldg(reinterpret_cast<const float2*>(u + 2));
    }
    cs = make_float4(c0.x, c0.y, c1.x, c1.y);
    sn = make_float4(s0.x, s0.y, s1.x, s1.y);
  } else {
    cs = __ldg(reinterpret_cast<const float4*>(t));
    sn = __ldg(reinterpret_cast<const float4*>(u));
  }
}

// Few rows as in fwd_kernel, with eight elements a lane: for sizes that are no multiples of 16, for fp32 rows, where that
// is 32 bytes, and for partial sums, where twice the lanes have the loads of twice the parts under way.
template <typename T, bool kInter, bool kFine, bool kNorm, bool kPart>
__global__ void __launch_bounds__(kThreads) fwd8_kernel(const Args a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(a.T) * a.blocks_per_row) return;
  const int t = static_cast<int>(item / a.blocks_per_row);
  const int blk = static_cast<int>(item - static_cast<long long>(t) * a.blocks_per_row);
  const int c = lane & ((1 << a.log_group) - 1);
  const int h = (blk << (5 - a.log_group)) + (lane >> a.log_group);
  const int half = a.R >> 1;
  const bool live = c * 8 < a.D, on = live && h < a.heads, turned = h < a.nq + a.nk;
  const bool rot = c * 8 < a.R, rot2 = kFine ? 4 * c + 2 < half : rot;
  const Spot at = spot_of<kInter, kFine>(c, half, live, rot, rot2);
  Pairs v = {};
  if (on) {
    const size_t from = static_cast<size_t>(t) * a.src_stride + h * a.D;
    if (kPart) {
      Sum sum[8];
      const float* p = static_cast<const float*>(a.src) + from;
      for (int i = 0; i < a.n_part; ++i, p += a.part_stride) {
        const Pairs q = get_pairs<float, kInter, kFine>(p, at);
        float e[8];
        unpack2(q.a[0], e[0], e[1]);
        unpack2(q.a[1], e[2], e[3]);
        unpack2(q.b[0], e[4], e[5]);
        unpack2(q.b[1], e[6], e[7]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j].add(e[j]);
      }
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = to_f(from_f<T>(sum[j].get()));
      v.a[0] = pack2(e[0], e[1]);
      v.a[1] = pack2(e[2], e[3]);
      v.b[0] = pack2(e[4], e[5]);
      v.b[1] = pack2(e[6], e[7]);
    } else {
      v = get_pairs<T, kInter, kFine>(static_cast<const T*>(a.src) + from, at);
    }
  }
  float4 cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
  if (rot) load_angles4<kFine>(a, a.pos[t], c, rot2, cs, sn);
  long long slot = a.slots ? a.slots[t] : -1;
  if (slot >= a.n_slots) slot = -1;
  if (kNorm) {
    f2 s2 = mul2(v.a[0], v.a[0]);
    s2 = fma2(v.b[0], v.b[0], s2);
    s2 = fma2(v.a[1], v.a[1], s2);
    s2 = fma2(v.b[1], v.b[1], s2);
    const float ss = group_sum(on ? sum2(s2) : 0.f, a.log_group);
    if (on && turned) {
      const float r = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
      const f2 r2 = pack2(r, r);
      const Pairs w = get_pairs<T, kInter, kFine>(static_cast<const T*>(h < a.nq ? a.qw : a.kw), at);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v.a[j] = mul2(mul2(v.a[j], r2), w.a[j]);
        v.b[j] = mul2(mul2(v.b[j], r2), w.b[j]);
      }
    }
  }
  if (!on) return;
  if (turned && rot) {
    const f2 cc[2] = {pack2(cs.x, cs.y), pack2(cs.z, cs.w)};
    const f2 ss[2] = {pack2(sn.x * a.sign, sn.y * a.sign), pack2(sn.z * a.sign, sn.w * a.sign)};
    const f2 ns[2] = {pack2(sn.x * -a.sign, sn.y * -a.sign), pack2(sn.z * -a.sign, sn.w * -a.sign)};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (j == 1 && !rot2) continue;  // not times 1 plus 0: there may be infinities
      const f2 va = fma2(v.b[j], ns[j], mul2(v.a[j], cc[j]));
      v.b[j] = fma2(v.a[j], ss[j], mul2(v.b[j], cc[j]));
      v.a[j] = va;
    }
  }
  if (h < a.store_heads)
    put_pairs<T, kInter, kFine>(static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h * a.D, at, v);
  if (slot >= 0 && h >= a.nq)
    put_pairs<T, kInter, kFine>(
        static_cast<T*>(turned ? a.kc : a.vc) + (static_cast<size_t>(slot) * a.nk + (turned ? h - a.nq : h - a.nq - a.nk)) * a.D, at, v);
}

constexpr int kStages = 3;
constexpr int kRowWarps = 16;

enum Mode { kRotate, kNormRotate, kNormBack };

// kFine: the rotated width is a multiple of 4, not of 8, so that a lane may own two pairs that rotate and two that do not.
// kPart (with norms): heads are rotated in part.  Elements that do not rotate go through times 1 plus 0 times their
// neighbour; where that may be infinite, which shows in the head's sum, they are made again without it.  16384 rows of 32 + 4
// + 4 heads of 128, with kPart / without: forward 62 / 59 us, backward 94 / 89.
template <typename T, bool kInter, bool kFine, Mode kMode, bool kPart>
__global__ void __launch_bounds__(kRowWarps * 32, 1) rows_kernel(const Args a, int piece_bytes, int* status) {
  constexpr bool kBack = kMode == kNormBack;
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t full[kRowWarps * kStages];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int stage_bytes = piece_bytes * (kBack ? 2 : 1);
  char* mine = smem + static_cast<size_t>(warp) * kStages * stage_bytes;
  uint64_t* bar = full + warp * kStages;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bar[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  const int hpw = 32 >> a.log_group;
  const int c = lane & ((1 << a.log_group) - 1), sub = lane >> a.log_group;
  const bool live = c * 8 < a.D, rot = c * 8 < a.R;  // a lane without elements goes along with the first one's
  const int half = a.R >> 1;
  const bool rot2 = kFine ? 4 * c + 2 < half : rot;  // pairs 2 and 3
  const Spot at = spot_of<kInter, kFine>(c, half, live, rot, rot2);
  const int turned = a.nq + a.nk;
  const int head_bytes = a.D * static_cast<int>(sizeof(T));
  const int block_heads = piece_bytes / head_bytes;
  const long long items = static_cast<long long>(a.T) * a.blocks_per_row;
  const int step = gridDim.x * kRowWarps, first = blockIdx.x * kRowWarps + warp;
  const int count = first < items ? static_cast<int>((items - first + step - 1) / step) : 0;
  struct Place {  // of a piece: token and block of heads
    int t, blk;
  };
  const int step_t = step / a.blocks_per_row, step_blk = step - step_t * a.blocks_per_row;
  auto advance = [&](Place& p) {
    p.t += step_t;
    p.blk += step_blk;
    if (p.blk >= a.blocks_per_row) {
      p.blk -= a.blocks_per_row;
      ++p.t;
    }
  };
  auto fill = [&](const Place& p, int stage) {  // lane 0
    const int h0 = p.blk * block_heads, h1 = min(a.heads, h0 + block_heads);
    const uint32_t n = (h1 - h0) * head_bytes, nx = kBack ? max(0, min(h1, turned) - h0) * head_bytes : 0;
    char* dst = mine + stage * stage_bytes;
    mbar_arrive_expect_tx(&bar[stage], n + nx);
    bulk_load(dst, static_cast<const T*>(a.src) + static_cast<size_t>(p.t) * a.src_stride + h0 * a.D, n, &bar[stage]);
    if (kBack && nx > 0)
      bulk_load(dst + piece_bytes, static_cast<const T*>(a.x) + static_cast<size_t>(p.t) * a.x_stride + h0 * a.D, nx, &bar[stage]);
  };
  Place now, ahead, next;  // the piece in work, the one to be loaded next, the one whose position is read next
  now.t = first / a.blocks_per_row;
  now.blk = first - now.t * a.blocks_per_row;
  ahead = next = now;
  const int p_first = count > 0 ? a.pos[next.t] : 0;
  advance(next);
  int p_next = count > 1 ? a.pos[next.t] : 0;
  advance(next);
  for (int i = 0; i < kStages - 1; ++i) {
    if (lane == 0 && i < count) fill(ahead, i);
    advance(ahead);
  }
  // angles of the next piece and the position of the one after it are under way while a piece is in work
  float4 cos_next = make_float4(1.f, 1.f, 1.f, 1.f), sin_next = make_float4(0.f, 0.f, 0.f, 0.f);
  auto angles = [&](int p) {
    if (!rot) return;
    load_angles4<kFine>(a, p, c, rot2, cos_next, sin_next);
  };
  if (count > 0) angles(p_first);

  f2 acc_q[4] = {0ull, 0ull, 0ull, 0ull}, acc_k[4] = {0ull, 0ull, 0ull, 0ull};  // weight gradients: a's, then b's
  const float inv_d = 1.f / static_cast<float>(a.D);
  int stage = 0;
  uint32_t parity = 0;
  bool ok = true;
  float least = 1.f;  // of a piece's factors r: 0 where a head's sum is infinite
  int i = 0;
  for (; i < count; ++i) {
    // forward: a -> a c - b s, b -> b c + a s; backwards with -s
    const float sg = kBack ? -1.f : a.sign;
    const f2 cc[2] = {pack2(cos_next.x, cos_next.y), pack2(cos_next.z, cos_next.w)};
    const f2 ss[2] = {pack2(sin_next.x * sg, sin_next.y * sg), pack2(sin_next.z * sg, sin_next.w * sg)};
    const f2 ns[2] = {pack2(sin_next.x * -sg, sin_next.y * -sg), pack2(sin_next.z * -sg, sin_next.w * -sg)};
    if (i + 1 < count) angles(p_next);
    if (i + 2 < count) p_next = a.pos[next.t];
    advance(next);
    const int t = now.t, h0 = now.blk * block_heads, h1 = min(a.heads, h0 + block_heads);
    advance(now);
    long long slot = -1;
    if (!kBack && a.slots) slot = a.slots[t];
    char* piece = mine + stage * stage_bytes;
    if (!__all_sync(0xffffffffu, mbar_wait(&bar[stage], parity, status, 0x4d10))) {  // the warp gives up as one
      ok = false;
      break;
    }
    auto heads = [&](int from, int to, const T* w, f2 (&acc)[4]) {
      if (from >= to) return;
      Pairs wt, ca, sa;
      if (kMode != kRotate) wt = get_pairs<T, kInter, kFine>(w, at);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ca.a[j] = kMode == kNormRotate ? mul2(cc[j], wt.a[j]) : cc[j];
        ca.b[j] = kMode == kNormRotate ? mul2(cc[j], wt.b[j]) : cc[j];
        sa.a[j] = kMode == kNormRotate ? mul2(ss[j], wt.a[j]) : ss[j];
        sa.b[j] = kMode == kNormRotate ? mul2(ns[j], wt.b[j]) : ns[j];
      }
      T* base = reinterpret_cast<T*>(piece) - h0 * a.D;
      for (int h = from + sub; h - sub < to; h += hpw) {
        T* row = base + min(h, to - 1) * a.D;  // a lane behind the last head goes along with the last one's
        const bool on = live && h < to;
        Pairs v = get_pairs<T, kInter, kFine>(row, at), x;
        if (kBack) x = get_pairs<T, kInter, kFine>(row + piece_bytes / static_cast<int>(sizeof(T)), at);
        float r = 1.f, m = 0.f;
        if (kMode != kRotate) {
          const Pairs& y = kBack ? x : v;
          f2 s2 = mul2(y.a[0], y.a[0]);
          s2 = fma2(y.b[0], y.b[0], s2);
          s2 = fma2(y.a[1], y.a[1], s2);
          s2 = fma2(y.b[1], y.b[1], s2);
          r = live ? sum2(s2) : 0.f;
          if (kBack) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const f2 ga = fma2(v.b[j], ns[j], mul2(v.a[j], cc[j]));
              v.b[j] = fma2(v.a[j], ss[j], mul2(v.b[j], cc[j]));
              v.a[j] = ga;
            }
            f2 d2 = mul2(mul2(v.a[0], wt.a[0]), x.a[0]);
            d2 = fma2(mul2(v.b[0], wt.b[0]), x.b[0], d2);
            d2 = fma2(mul2(v.a[1], wt.a[1]), x.a[1], d2);
            d2 = fma2(mul2(v.b[1], wt.b[1]), x.b[1], d2);
            m = live ? sum2(d2) : 0.f;
          }
#pragma unroll
          for (int o = 4; o >= 0; --o) {
            if (o >= a.log_group) continue;
            r += __shfl_xor_sync(0xffffffffu, r, 1 << o);
            if (kBack) m += __shfl_xor_sync(0xffffffffu, m, 1 << o);
          }
          r = rsqrtf(r * inv_d + a.eps);
          if (kPart && kBack && !rot2 && !(fabsf(m) < __int_as_float(0x7f800000))) {
            const Pairs u = get_pairs<T, kInter, kFine>(row, at);
            if (!rot) {
              v.a[0] = u.a[0];
              v.b[0] = u.b[0];
            }
            v.a[1] = u.a[1];
            v.b[1] = u.b[1];
          }
          if (kPart && !kBack) least = fminf(least, r);
        }
        const f2 r2 = pack2(r, r);
        __syncwarp();  // every lane has read its elements before one that goes along with it writes them
        if (kBack) {
          const float back = -m * inv_d * r * r;  // - mean(dn w xh) * rstd
          const f2 b2 = pack2(back, back);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const f2 xa = mul2(x.a[j], r2), xb = mul2(x.b[j], r2);  // xh
            if (on) {
              acc[j] = fma2(v.a[j], xa, acc[j]);
              acc[2 + j] = fma2(v.b[j], xb, acc[2 + j]);
            }
            v.a[j] = fma2(xa, b2, mul2(mul2(v.a[j], wt.a[j]), r2));
            v.b[j] = fma2(xb, b2, mul2(mul2(v.b[j], wt.b[j]), r2));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (kFine && kMode == kRotate && j == 1 && !rot2) continue;  // not times 1 plus 0: there may be infinities
            const f2 va = fma2(v.b[j], sa.b[j], mul2(v.a[j], ca.a[j]));
            const f2 vb = fma2(v.a[j], sa.a[j], mul2(v.b[j], ca.b[j]));
            v.a[j] = kMode == kNormRotate ? mul2(va, r2) : va;
            v.b[j] = kMode == kNormRotate ? mul2(vb, r2) : vb;
          }
        }
        if (on && (kMode != kRotate || rot)) put_pairs<T, kInter, kFine>(row, at, v);
      }
    };
    heads(h0, min(h1, a.nq), static_cast<const T*>(a.qw), acc_q);
    heads(max(h0, a.nq), min(h1, turned), static_cast<const T*>(a.kw), acc_k);
    if (kPart && !kBack && __any_sync(0xffffffffu, least == 0.f)) {  // from the row, whose own memory is not written yet
      least = 1.f;
      __syncwarp();  // every lane has written its elements
      for (int h = h0 + sub; h - sub < min(h1, turned); h += hpw) {
        const bool on = live && h < min(h1, turned);
        const int hh = on ? h : h0;
        const T* src = static_cast<const T*>(a.src) + static_cast<size_t>(t) * a.src_stride + hh * a.D;
        const T* w = static_cast<const T*>(hh < a.nq ? a.qw : a.kw);
        float ss = 0.f;
        if (on)
          for (int e = c * 8; e < c * 8 + 8; ++e) ss += to_f(src[e]) * to_f(src[e]);
        ss = group_sum(ss, a.log_group);
        if (!on || rsqrtf(ss * inv_d + a.eps) != 0.f) continue;
        T* row = reinterpret_cast<T*>(piece) + (h - h0) * a.D;
        for (int e = max(a.R, c * 8); e < c * 8 + 8; ++e) row[e] = from_f<T>(to_f(src[e]) * 0.f * to_f(w[e]));
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      const int stored = min(h1, a.store_heads);
      if (stored > h0)
        bulk_store(static_cast<T*>(a.dst) + static_cast<size_t>(t) * a.dst_stride + h0 * a.D, piece, (stored - h0) * head_bytes);
      if (!kBack && slot >= 0 && slot < a.n_slots) {
        const int k0 = max(h0, a.nq), k1 = min(h1, turned), v0 = max(h0, turned);
        if (k1 > k0)
          bulk_store(static_cast<T*>(a.kc) + (static_cast<size_t>(slot) * a.nk + k0 - a.nq) * a.D, piece + (k0 - h0) * head_bytes,
                     (k1 - k0) * head_bytes);
        if (h1 > v0)
          bulk_store(static_cast<T*>(a.vc) + (static_cast<size_t>(slot) * a.nk + v0 - turned) * a.D, piece + (v0 - h0) * head_bytes,
                     (h1 - v0) * head_bytes);
      }
      tma_store_commit();
      // the buffer of the piece before is free once its stores have read it
      if (i + kStages - 1 < count) {
        tma_store_wait_read<1>();
        fill(ahead, stage == 0 ? kStages - 1 : stage - 1);
      }
    }
    advance(ahead);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1;
    }
  }
  if (lane == 0) {
    if (!ok) {  // loads that are still under way, piece i's and those behind it, land before the buffers are given back
      const unsigned long long t0 = globaltimer_ns();
      for (int j = i; j < min(count, i + kStages - 1); ++j) {
        while (!mbar_try_wait(&bar[stage], parity))
          if (globaltimer_ns() - t0 > kWaitTimeoutNs) break;
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1;
        }
      }
    }
    tma_store_wait_read<0>();  // the buffers have been read; the writes end with the kernel
  }
  if (!kBack || !a.dw_part) return;
  // lanes that own the same elements of different heads, then the warps, in a fixed order
  float aq[8], ak[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unpack2(acc_q[j], aq[2 * j], aq[2 * j + 1]);
    unpack2(acc_k[j], ak[2 * j], ak[2 * j + 1]);
  }
  for (int o = 16; o >= (1 << a.log_group); o >>= 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      aq[j] += __shfl_xor_sync(0xffffffffu, aq[j], o);
      ak[j] += __shfl_xor_sync(0xffffffffu, ak[j], o);
    }
  }
  __syncthreads();  // every warp's buffers are done with
  float* sdw = reinterpret_cast<float*>(smem);  // [kRowWarps][2 * D]
  if (sub == 0 && live) {
    float* s = sdw + warp * 2 * a.D;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // pair j: interleaved pairs 0, 1 lie at lo, pairs 2, 3 behind them
      const int first_at = kFine && j > 1 ? at.lo2 + j - 2 : at.lo + j, second_at = kFine && j > 1 ? at.hi2 + j - 2 : at.hi + j;
      const int ea = kInter ? at.lo + 2 * j : first_at, eb = kInter ? ea + 1 : second_at;
      s[ea] = aq[j];
      s[eb] = aq[4 + j];
      s[a.D + ea] = ak[j];
      s[a.D + eb] = ak[4 + j];
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * a.D; j += kRowWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) v += sdw[w * 2 * a.D + j];
    a.dw_part[static_cast<size_t>(blockIdx.x) * 2 * a.D + j] = v;
  }
}

// Any head size, rotated width, stride or alignment: one warp per (token, head), element by element.  A lane reads and
// writes the same elements, so rows may be rotated in place.
template <typename T, bool kPart>
__device__ __forceinline__ float elem(const Args& a, int t, int h, int e) {
  if (kPart) {
    const float* p = static_cast<const float*>(a.src) + static_cast<size_t>(t) * a.src_stride + h * a.D + e;
    Sum v;
    for (int i = 0; i < a.n_part; ++i) v.add(p[static_cast<size_t>(i) * a.part_stride]);
    return to_f(from_f<T>(v.get()));
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
#pragma unroll 8
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

// Whether rows, weights, tables and caches can be read 16 bytes at a time by lanes that own `unit` elements of a head and
// `rot_unit` of its rotated part.
bool vectorised(const Args& a, size_t elt, int unit, int rot_unit) {
  const auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const long long per = 16 / static_cast<long long>(elt);
  const bool strides = a.n_part ? (a.src_stride % 4 == 0 && a.part_stride % 4 == 0) : a.src_stride % per == 0;
  return a.D % unit == 0 && a.R % rot_unit == 0 && strides && a.x_stride % per == 0 && a.dst_stride % per == 0 && al(a.src) &&
         al(a.x) && al(a.dst) && al(a.qw) && al(a.kw) && al(a.table) && al(a.kc) && al(a.vc);
}

int log2_ceil(int v) {
  int l = 0;
  while ((1 << l) < v) ++l;
  return l;
}

// The row pipeline: heads of a piece so that a CTA's buffers fill at most kRowSmem.
constexpr int kRowSmem = 200 * 1024;

template <typename T, bool kInter, bool kFine, Mode kMode, bool kPart>
cudaError_t launch_rows_as(Args a, int ctas, cudaStream_t st) {
  const int head = a.D * static_cast<int>(sizeof(T)), per_head = kRowWarps * kStages * head * (kMode == kNormBack ? 2 : 1);
  int block = kRowSmem / per_head;  // as large as the buffers allow, and alike
  a.blocks_per_row = (a.heads + block - 1) / block;
  block = (a.heads + a.blocks_per_row - 1) / a.blocks_per_row;
  const size_t sums = kMode == kNormBack ? sizeof(float) * kRowWarps * 2 * a.D : 0;
  size_t smem = static_cast<size_t>(block) * per_head;
  if (smem < sums) smem = sums;
  static bool attr_dev[64] = {};
  bool& attr = attr_dev[device_index()];
  if (!attr) {
    const cudaError_t e = cudaFuncSetAttribute(rows_kernel<T, kInter, kFine, kMode, kPart>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem);
    if (e != cudaSuccess) return e;
    attr = true;
  }
  int* status = device_status_ptr();
  if (!status) return cudaErrorUnknown;
  a.log_group = log2_ceil(a.D / 8);
  return launch_pdl(rows_kernel<T, kInter, kFine, kMode, kPart>, dim3(ctas), dim3(kRowWarps * 32), smem, st, a, block * head, status);
}

template <typename T, bool kInter, Mode kMode>
cudaError_t launch_rows(const Args& a, int ctas, cudaStream_t st) {
  constexpr bool kNorm = kMode != kRotate;
  if (a.R % 8) return launch_rows_as<T, kInter, true, kMode, kNorm>(a, ctas, st);
  return kNorm && a.R < a.D ? launch_rows_as<T, kInter, false, kMode, kNorm>(a, ctas, st)
                            : launch_rows_as<T, kInter, false, kMode, false>(a, ctas, st);
}

// From how many bytes of rows on the pipeline is taken.  Below, its start (4 us against 2) costs more than it gains, and
// rows that lie in L2 come fast enough through plain loads.  bf16, 40 heads of 128, plain kernel / pipeline in us: forward
// of 23 MB 12.1 / 13.5, of 47 MB 28.3 / 23.5, of 160 MB 89.7 / 60.0; backward of 0.6 MB 6.2 / 6.8, of 1.5 MB 8.7 / 7.0, of
// 160 MB 144 / 90.  Head sizes and widths that are no multiples of 16: 8 + 2 + 2 heads of 80, 40 rotated, plain / pipeline,
// forward of 1 M elements 3.4 / 4.8, of 2 M 5.4 / 4.9, of 16 M 33 / 20, in fp32 of 2 M 5.2 / 5.9, of 4 M 9.0 / 8.9; backward,
// element by element / pipeline, of 0.25 M 7.8 / 8.5, of 0.5 M 10.3 / 8.7, of 16 M 146 / 30.
constexpr long long kForwardFrom = 28LL << 20, kBackwardFrom = 640LL << 10;
constexpr long long kForwardFromElements = 1LL << 20, kBackwardFromElements = 175LL << 10;  // per byte of an element
bool row_pipeline(const Args& a, size_t elt, long long from, long long from_elements) {
  if (a.D > 256 || !vectorised(a, elt, 8, 4)) return false;
  const long long e = static_cast<long long>(elt), elements = static_cast<long long>(a.T) * a.heads * a.D;
  return vectorised(a, elt, 16, 16) ? elements * e > from : elements > from_elements * e;
}

template <typename T, bool kInter, bool kNorm, bool kPart>
cudaError_t launch_fwd(Args a, cudaStream_t st) {
  if (!kPart && row_pipeline(a, sizeof(T), kForwardFrom, kForwardFromElements))
    return launch_rows<T, kInter, kNorm ? kNormRotate : kRotate>(a, sm_count(), st);
  // 16 elements a lane where that is the faster form (us, 16 / 8 elements a lane, 32 + 4 + 4 heads of 128): bf16 rows, 64
  // 2.5 / 2.4, 1024 6.4 / 8.1, 2048 10.5 / 14.3; fp32 rows of 8 + 4 + 4 heads of 256, 256 4.4 / 3.6, 2048 13.9 / 13.3; four
  // partial sums, 64 rows 4.4 / 3.7, 512 rows 11.7 / 9.3.
  const bool wide = !kPart && vectorised(a, sizeof(T), 16, 16) && (sizeof(T) == 2 || a.D > 256);
  if (!wide && (a.D > 256 || !vectorised(a, sizeof(T), 8, 4))) {
    const long long ctas = (static_cast<long long>(a.T) * a.heads + kWarps - 1) / kWarps;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
    return launch_pdl(fwd_any_kernel<T, kInter, kNorm, kPart>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), 0, st, a);
  }
  a.log_group = log2_ceil(wide ? a.D / 16 : a.D / 8);
  const int hpw = 32 >> a.log_group;
  a.blocks_per_row = (a.heads + hpw - 1) / hpw;  // every pass over heads on a warp of its own: the call is one round of loads
  const long long ctas = (static_cast<long long>(a.T) * a.blocks_per_row + kWarps - 1) / kWarps;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(ctas));
  if constexpr (!kPart) {
    if (wide) return launch_pdl(fwd_kernel<T, kInter, kNorm>, grid, dim3(kThreads), 0, st, a);
  }
  if (a.R % 8) return launch_pdl(fwd8_kernel<T, kInter, true, kNorm, kPart>, grid, dim3(kThreads), 0, st, a);
  return launch_pdl(fwd8_kernel<T, kInter, false, kNorm, kPart>, grid, dim3(kThreads), 0, st, a);
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

int bwd_ctas(long long items) {
  const long long want = (items + kWarps - 1) / kWarps, cap = 4LL * sm_count();
  return static_cast<int>(want < cap ? want : cap);
}

// Returns in `ctas` how many rows of partial sums were written (at most as many as were given).
template <typename T, bool kInter>
cudaError_t launch_bwd(Args a, int& ctas, cudaStream_t st) {
  const size_t smem = sizeof(float) * kWarps * 2 * a.D;  // at most 32 KB (D <= 512)
  if (row_pipeline(a, sizeof(T), kBackwardFrom, kBackwardFromElements)) {
    if (ctas > sm_count()) ctas = sm_count();
    return launch_rows<T, kInter, kNormBack>(a, ctas, st);
  }
  if (!vectorised(a, sizeof(T), 16, 16))
    return launch_pdl(bwd_any_kernel<T, kInter>, dim3(ctas), dim3(kThreads), smem, st, a);
  a.log_group = log2_ceil(a.D / 16);
  const int hpw = 32 >> a.log_group;
  a.blocks_per_row = (a.heads + hpw - 1) / hpw;
  return launch_pdl(bwd_kernel<T, kInter>, dim3(ctas), dim3(kThreads), smem, st, a);
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
  int rows = n_parts;
  if (dtype == 0)
    e = interleaved ? sb::qkr::launch_bwd<__nv_bfloat16, true>(a, rows, st) : sb::qkr::launch_bwd<__nv_bfloat16, false>(a, rows, st);
  else if (dtype == 1)
    e = interleaved ? sb::qkr::launch_bwd<__half, true>(a, rows, st) : sb::qkr::launch_bwd<__half, false>(a, rows, st);
  else if (dtype == 2)
    e = interleaved ? sb::qkr::launch_bwd<float, true>(a, rows, st) : sb::qkr::launch_bwd<float, false>(a, rows, st);
  else
    return SB_ERR_ARG;
  if (e != cudaSuccess) return SB_ERR_CUDA;
  if (!a.dw_part) return SB_OK;
  if (dtype == 0)
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<__nv_bfloat16>, rg, rb, 0, st, part, rows, D, dqw, dkw, accumulate);
  else if (dtype == 1)
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<__half>, rg, rb, 0, st, part, rows, D, dqw, dkw, accumulate);
  else
    e = sb::launch_pdl(sb::qkr::reduce_dw_kernel<float>, rg, rb, 0, st, part, rows, D, dqw, dkw, accumulate);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

}  // extern "C"
