// A mixture-of-experts layer for a few tokens, in three launches:
//   route_kernel    z = h R^T, the k largest experts of every token, their softmax weights
//   gate_up_kernel  act[t, s] = silu(Wg h_t) * (Wu h_t)  for the expert e of (t, s)
//   down_kernel     out[t] = sum_s w[t, s] * Wd act[t, s]
//
// Bound by HBM: with few rows an expert, a layer reads the weights of the experts that some token picked, once, and
// little else (6 F H bytes an expert).  Rows are not padded or gathered: an expert's rows are a list of (token, slot)
// entries that every CTA derives from the routing table in shared memory.  The weights stream from global memory into
// registers as the A operand of m16n8k16 products, eight rows of an expert as its N side.  Such a product is far from
// bound by the tensor pipe (8 rows: 16 FLOP per weight byte), so what counts is that the operand needs no staging: a
// lane's 16-byte load of eight consecutive k is used as the fragments of two products whose k order is permuted the
// same way in both operands, which a sum over k does not see.
// Every result is summed in a fixed order, without atomics on floats.
#include <cooperative_groups.h>

#include "host_common.h"
#include "ptx.cuh"

namespace sb {
namespace mf {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = 1024;
constexpr int kMaxEntries = 2048;
constexpr int kMaxTopK = 16;

// ---------------------------------------------------------------------------
// Router.  A cluster of eight CTAs takes kTok tokens and an eighth of the experts each; the logits of token i meet in
// CTA i's shared memory.  Products of bf16 are exact in fp32; eight of them are summed there and the rest in fp64, so
// that experts whose logits lie next to one another are ordered by the values and not by the order of the sum.
// ---------------------------------------------------------------------------
constexpr int kCluster = 8;

__device__ __forceinline__ float dot8(const uint4& a, const uint4& b) {
  const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&a);
  const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&b);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __bfloat1622float2(x[i]), q = __bfloat1622float2(y[i]);
    s = fmaf(p.x, q.x, s);
    s = fmaf(p.y, q.y, s);
  }
  return s;
}

template <int kTok>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
route_kernel(const __nv_bfloat16* __restrict__ h, long long h_stride, const __nv_bfloat16* __restrict__ rw,
             const int* __restrict__ live, float* __restrict__ w, int* __restrict__ idx, int T, int E, int H, int k, int norm) {
  extern __shared__ double logits[];  // [E], of token t0 + rank
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = static_cast<int>(blockIdx.x / kCluster) * kTok;
  pdl_launch_dependents();
  pdl_wait();
  cluster.sync();  // every CTA of the cluster runs before its shared memory is written
  const int per = (E + kCluster - 1) / kCluster;
  const int e_hi = min(E, (rank + 1) * per);
  for (int e = rank * per + warp; e < e_hi; e += kWarps) {
    const uint4* r = reinterpret_cast<const uint4*>(rw + static_cast<size_t>(e) * H);
    double acc[kTok];
#pragma unroll
    for (int i = 0; i < kTok; ++i) acc[i] = 0.0;
#pragma unroll 4
    for (int v = lane; v < (H >> 3); v += 32) {
      const uint4 a = __ldg(r + v);
#pragma unroll
      for (int i = 0; i < kTok; ++i)
        if (t0 + i < T)
          acc[i] += static_cast<double>(
              dot8(a, __ldg(reinterpret_cast<const uint4*>(h + static_cast<size_t>(t0 + i) * h_stride) + v)));
    }
#pragma unroll
    for (int i = 0; i < kTok; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
      if (lane == 0) cluster.map_shared_rank(logits, i)[e] = acc[i];
    }
  }
  cluster.sync();
  const int t = t0 + rank;
  if (rank >= kTok || t >= T || warp != 0) return;
  if (live && live[t] == 0) {
    if (lane < k) {
      w[static_cast<size_t>(t) * k + lane] = 0.f;
      idx[static_cast<size_t>(t) * k + lane] = -1;
    }
    return;
  }
  // k rounds of a warp-wide maximum; ties go to the lower expert.  A NaN counts as the smallest value, so that the
  // indices stay in range, and makes the row's weights NaN.
  const double inf = __longlong_as_double(0x7ff0000000000000ll);
  uint32_t taken = 0;  // expert lane + 32 j: bit j
  bool bad = false;
  double top = 0.0;
  float mine = 0.f, sel = 0.f;
  int my_e = 0;
  for (int s = 0; s < k; ++s) {
    double best = -inf;
    int best_e = 0x7fffffff;
    for (int j = 0, e = lane; e < E; ++j, e += 32) {
      if (taken >> j & 1) continue;
      double v = logits[e];
      if (v != v) {
        bad = true;
        v = -inf;
      }
      if (v > best || best_e == 0x7fffffff) {
        best = v;
        best_e = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
      if (oe != 0x7fffffff && (best_e == 0x7fffffff || ov > best || (ov == best && oe < best_e))) {
        best = ov;
        best_e = oe;
      }
    }
    if ((best_e & 31) == lane) taken |= 1u << (best_e >> 5);
    if (s == 0) top = best;
    const float p = expf(static_cast<float>(best - top));
    sel += p;
    if (lane == s) {
      mine = p;
      my_e = best_e;
    }
  }
  float all = sel;
  if (!norm) {
    all = 0.f;
    for (int e = lane; e < E; e += 32) all += expf(static_cast<float>(logits[e] - top));
    all = warp_sum(all);
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane < k) {
    w[static_cast<size_t>(t) * k + lane] = bad ? __int_as_float(0x7fffffff) : mine / all;
    idx[static_cast<size_t>(t) * k + lane] = my_e;
  }
}

// ---------------------------------------------------------------------------
// Rows of every expert, in shared memory: entry = token * k + slot.  The order of an expert's entries does not matter
// (an entry's result does not depend on its neighbours).
// ---------------------------------------------------------------------------
struct Lists {
  int first[kMaxExperts + 1];         // first entry of each expert
  int cursor[kMaxExperts];
  unsigned short used[kMaxExperts];   // experts that have entries, ascending
  unsigned short entry[kMaxEntries];
  int n_used;
};

__device__ __forceinline__ void build_lists(Lists& L, const int* __restrict__ idx, int n, int E) {
  for (int e = threadIdx.x; e < E; e += kThreads) L.cursor[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int e = idx[i];
    if (e >= 0 && e < E) atomicAdd(&L.cursor[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int run = 0, used = 0;
    for (int base = 0; base < E; base += 32) {
      const int e = base + threadIdx.x;
      const int c = e < E ? L.cursor[e] : 0;
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (threadIdx.x >= o) inc += v;
      }
      const unsigned int has = __ballot_sync(0xffffffffu, c > 0);
      if (e < E) {
        L.first[e] = L.cursor[e] = run + inc - c;
        if (c > 0) L.used[used + __popc(has & ((1u << threadIdx.x) - 1u))] = static_cast<unsigned short>(e);
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
      used += __popc(has);
    }
    if (threadIdx.x == 0) {
      L.first[E] = run;
      L.n_used = used;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int e = idx[i];
    if (e >= 0 && e < E) L.entry[atomicAdd(&L.cursor[e], 1)] = static_cast<unsigned short>(i);
  }
  __syncthreads();
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// weights are read once: keep them from displacing the rows in L1
__device__ __forceinline__ uint4 ld_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// acc[n] (+)= 16 weight rows x 8 kNt operand rows over the k steps [s0, s1) of 32.  top / low: this lane's two weight
// rows (g and g + 8, null outside the matrix) at k = 8 (lane % 4); x[n]: its operand row of column group n.
template <int kNt, int kUnroll>
__device__ __forceinline__ void products(float (&acc)[kNt][4], const __nv_bfloat16* top, const __nv_bfloat16* low,
                                         const __nv_bfloat16* const (&x)[kNt], int s0, int s1, int K, int t4) {
  for (int s = s0; s < s1; s += kUnroll) {
    uint4 a[kUnroll], b[kUnroll], v[kUnroll][kNt];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int col = (s + j) * 32;
      const bool ok = s + j < s1 && col + 8 * t4 < K;
      const uint4 z = make_uint4(0, 0, 0, 0);
      a[j] = ok && top ? ld_stream(top + col) : z;
      b[j] = ok && low ? ld_stream(low + col) : z;
#pragma unroll
      for (int n = 0; n < kNt; ++n) v[j][n] = ok && x[n] ? *reinterpret_cast<const uint4*>(x[n] + col) : z;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        mma_bf16(acc[n], a[j].x, b[j].x, a[j].y, b[j].y, v[j][n].x, v[j][n].y);
        mma_bf16(acc[n], a[j].z, b[j].z, a[j].w, b[j].w, v[j][n].z, v[j][n].w);
      }
  }
}

// ---------------------------------------------------------------------------
// Gate and up projections.  An item is eight gate rows and the eight up rows beside them of one expert: a lane then
// holds both factors of an activation.  The CTA's warps split K; their sums meet in shared memory.
// ---------------------------------------------------------------------------
constexpr int kMaxNt = 4;

template <int kNt, int kUnroll>
__device__ __forceinline__ void gate_up_tile(const Lists& L, float4* red, const __nv_bfloat16* h, long long h_stride,
                                             const __nv_bfloat16* wgu, __nv_bfloat16* act, int e, int f0, int r0, int r1, int k,
                                             int H, int F) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int steps = (H + 31) >> 5;
  const int s0 = warp * steps / kWarps, s1 = (warp + 1) * steps / kWarps;
  const __nv_bfloat16* top = f0 + g < F ? wgu + (static_cast<size_t>(e) * 2 * F + f0 + g) * H + 8 * t4 : nullptr;
  const __nv_bfloat16* low = top ? top + static_cast<size_t>(F) * H : nullptr;
  const __nv_bfloat16* x[kNt];
  float acc[kNt][4];
#pragma unroll
  for (int n = 0; n < kNt; ++n) {
    const int r = r0 + n * 8 + g;
    x[n] = r < r1 ? h + static_cast<size_t>(L.entry[r] / k) * h_stride + 8 * t4 : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  }
  products<kNt, kUnroll>(acc, top, low, x, s0, s1, H, t4);
#pragma unroll
  for (int n = 0; n < kNt; ++n) red[(warp * kNt + n) * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
  __syncthreads();
  // thread -> (column group, lane of the fragment, one of its two columns)
  for (int i = threadIdx.x; i < kNt * 64; i += kThreads) {
    const int n = i >> 6, l = (i >> 1) & 31, col = i & 1;
    const int r = r0 + n * 8 + 2 * (l & 3) + col, f = f0 + (l >> 2);
    if (r >= r1 || f >= F) continue;
    float gate = 0.f, up = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* p = reinterpret_cast<const float*>(&red[(w * kNt + n) * 32 + l]);
      gate += p[col];
      up += p[2 + col];
    }
    // the activation is the down product's bf16 operand, rounded here as on the path for many tokens
    act[static_cast<size_t>(L.entry[r]) * F + f] = __float2bfloat16_rn(gate / (1.f + __expf(-gate)) * up);
  }
}

__global__ void __launch_bounds__(kThreads, 2)
gate_up_kernel(const __nv_bfloat16* __restrict__ h, long long h_stride, const int* __restrict__ idx,
               const __nv_bfloat16* __restrict__ wgu, __nv_bfloat16* __restrict__ act, int n, int k, int E, int H, int F) {
  __shared__ Lists L;
  __shared__ float4 red[2][kWarps * kMaxNt * 32];
  pdl_launch_dependents();
  pdl_wait();
  build_lists(L, idx, n, E);
  const int tiles = (F + 7) >> 3;
  const long long items = static_cast<long long>(L.n_used) * tiles;
  const int lo = static_cast<int>(items * blockIdx.x / gridDim.x), hi = static_cast<int>(items * (blockIdx.x + 1) / gridDim.x);
  int flip = 0;
  for (int i = lo; i < hi; ++i) {
    const int e = L.used[i / tiles], f0 = (i % tiles) * 8;
    const int r1 = L.first[e + 1];
    for (int r0 = L.first[e]; r0 < r1; r0 += 8 * kMaxNt, flip ^= 1) {
      const int m = r1 - r0;
      if (m <= 8)
        gate_up_tile<1, 8>(L, red[flip], h, h_stride, wgu, act, e, f0, r0, r1, k, H, F);
      else if (m <= 16)
        gate_up_tile<2, 4>(L, red[flip], h, h_stride, wgu, act, e, f0, r0, r1, k, H, F);
      else
        gate_up_tile<4, 2>(L, red[flip], h, h_stride, wgu, act, e, f0, r0, min(r1, r0 + 32), k, H, F);
    }
  }
}

// ---------------------------------------------------------------------------
// Down projection and combination.  A CTA owns 16 columns of the output for all tokens and walks over the used experts,
// one expert a warp at a time; the entries' results stay in shared memory until all are there and are then added up
// slot by slot, so no sum crosses a CTA.
// ---------------------------------------------------------------------------
template <int kNt, int kUnroll>
__device__ __forceinline__ void down_tile(const Lists& L, float* y, const __nv_bfloat16* act, const __nv_bfloat16* wd, int e,
                                          int n0, int r0, int r1, int H, int F) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const __nv_bfloat16* base = wd + (static_cast<size_t>(e) * H + n0) * F + 8 * t4;
  const __nv_bfloat16* top = n0 + g < H ? base + static_cast<size_t>(g) * F : nullptr;
  const __nv_bfloat16* low = n0 + g + 8 < H ? base + static_cast<size_t>(g + 8) * F : nullptr;
  const __nv_bfloat16* x[kNt];
  float acc[kNt][4];
#pragma unroll
  for (int n = 0; n < kNt; ++n) {
    const int r = r0 + n * 8 + g;
    x[n] = r < r1 ? act + static_cast<size_t>(L.entry[r]) * F + 8 * t4 : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  }
  products<kNt, kUnroll>(acc, top, low, x, 0, (F + 31) >> 5, F, t4);
#pragma unroll
  for (int n = 0; n < kNt; ++n)
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      const int r = r0 + n * 8 + 2 * t4 + col;
      if (r < r1) {
        float* o = y + L.entry[r] * 16;
        o[g] = acc[n][col];
        o[g + 8] = acc[n][2 + col];
      }
    }
}

__global__ void __launch_bounds__(kThreads)
down_kernel(const __nv_bfloat16* __restrict__ act, const int* __restrict__ idx, const float* __restrict__ w,
            const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* __restrict__ out, int T, int k, int E, int H, int F) {
  __shared__ Lists L;
  extern __shared__ float y[];  // [T * k][16]
  pdl_launch_dependents();
  pdl_wait();
  const int n = T * k;
  build_lists(L, idx, n, E);
  const int n0 = blockIdx.x * 16;
  for (int a = threadIdx.x >> 5; a < L.n_used; a += kWarps) {
    const int e = L.used[a], r1 = L.first[e + 1];
    for (int r0 = L.first[e]; r0 < r1; r0 += 8 * kMaxNt) {
      const int m = r1 - r0;
      if (m <= 8)
        down_tile<1, 8>(L, y, act, wd, e, n0, r0, r1, H, F);
      else if (m <= 16)
        down_tile<2, 4>(L, y, act, wd, e, n0, r0, r1, H, F);
      else
        down_tile<4, 2>(L, y, act, wd, e, n0, r0, min(r1, r0 + 32), H, F);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < T * 16; i += kThreads) {
    const int t = i >> 4, c = i & 15;
    if (n0 + c >= H) continue;
    float v = 0.f;
    for (int s = 0; s < k; ++s) {
      const int e = idx[t * k + s];
      if (e >= 0 && e < E) v = fmaf(w[t * k + s], y[(t * k + s) * 16 + c], v);
    }
    out[static_cast<size_t>(t) * H + n0 + c] = __float2bfloat16_rn(v);
  }
}

}  // namespace mf
}  // namespace sb

extern "C" {

// h [T, H] rows of stride h_stride, router [E, H]; w fp32 / idx int32 [T, k]; live [T] or null.
int sb_moe_few_route(const void* h, long long h_stride, const void* router, const int* live, float* w, int* idx, int T, int E,
                     int H, int k, int norm, void* stream) {
  if (T <= 0 || E <= 0 || E > sb::mf::kMaxExperts || H <= 0 || (H & 7) || k <= 0 || k > sb::mf::kMaxTopK || k > E || (h_stride & 7))
    return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(router)) & 15) return SB_ERR_ARG;
  const size_t smem = sizeof(double) * E;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto* hp = static_cast<const __nv_bfloat16*>(h);
  const auto* rp = static_cast<const __nv_bfloat16*>(router);
  // a token a cluster while the clusters fit the SMs side by side; beyond that four share the router's rows
  cudaError_t e;
  if (T * sb::mf::kCluster <= sb::sm_count())
    e = sb::launch_pdl(sb::mf::route_kernel<1>, dim3(T * sb::mf::kCluster), dim3(sb::mf::kThreads), smem, st, hp, h_stride, rp, live,
                       w, idx, T, E, H, k, norm);
  else
    e = sb::launch_pdl(sb::mf::route_kernel<4>, dim3((T + 3) / 4 * sb::mf::kCluster), dim3(sb::mf::kThreads), smem, st, hp, h_stride,
                       rp, live, w, idx, T, E, H, k, norm);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

// h [T, H], idx int32 / w fp32 [T, k] (idx outside [0, E): the slot contributes nothing), wgu [E, 2F, H], wd [E, H, F];
// act: [T * k, F] scratch; out [T, H].
int sb_moe_few_experts(const void* h, long long h_stride, const float* w, const int* idx, const void* wgu, const void* wd,
                       void* act, void* out, int T, int k, int E, int H, int F, void* stream) {
  if (T <= 0 || k <= 0 || static_cast<long long>(T) * k > sb::mf::kMaxEntries || E <= 0 || E > sb::mf::kMaxExperts || H <= 0 ||
      (H & 7) || F <= 0 || (F & 7) || (h_stride & 7))
    return SB_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(h) | reinterpret_cast<uintptr_t>(wgu) | reinterpret_cast<uintptr_t>(wd) |
       reinterpret_cast<uintptr_t>(act)) & 15)
    return SB_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  static bool attr_dev[64] = {};
  bool& attr = attr_dev[sb::device_index()];
  const size_t most = sizeof(float) * 16 * sb::mf::kMaxEntries;
  if (!attr) {
    if (cudaFuncSetAttribute(sb::mf::down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)) != cudaSuccess)
      return SB_ERR_CUDA;
    attr = true;
  }
  const int n = T * k;
  const auto* a = static_cast<__nv_bfloat16*>(act);
  cudaError_t e = sb::launch_pdl(sb::mf::gate_up_kernel, dim3(2 * sb::sm_count()), dim3(sb::mf::kThreads), 0, st,
                                 static_cast<const __nv_bfloat16*>(h), h_stride, idx, static_cast<const __nv_bfloat16*>(wgu),
                                 static_cast<__nv_bfloat16*>(act), n, k, E, H, F);
  if (e != cudaSuccess) return SB_ERR_CUDA;
  e = sb::launch_pdl(sb::mf::down_kernel, dim3((H + 15) / 16), dim3(sb::mf::kThreads), sizeof(float) * 16 * n, st, a, idx, w,
                     static_cast<const __nv_bfloat16*>(wd), static_cast<__nv_bfloat16*>(out), T, k, E, H, F);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

}  // extern "C"
