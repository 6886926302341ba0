// A mixture-of-experts layer for a few tokens, in three launches:
//   route_kernel    z = h R^T, the k largest experts of every token, their softmax weights
//   gate_up_kernel  act[t, s] = silu(Wg h_t) * (Wu h_t)  for the expert e of (t, s)
//   down_kernel     out[t] = sum_s w[t, s] * Wd act[t, s]
//
// Bound by HBM: with few rows an expert, a layer reads the weights of the experts that some token picked, once, and
// little else (6 F H bytes an expert).  Rows are not padded or gathered: an expert's rows are a list of (token, slot)
// entries that every CTA derives from the routing table in shared memory.  The weights are the A operand of m16n8k16
// products, eight rows of an expert the N side.  Such a product is far from bound by the tensor pipe (8 rows: 16 FLOP
// per weight byte), so what counts is that the operand needs no rearranging: a lane's 16 bytes of eight consecutive k are
// used as the fragments of two products whose k order is permuted the same way in both operands, which a sum over k does
// not see.  Gate and up weights come through a ring of bulk copies in shared memory, down weights straight from global
// memory into registers.  Every result is summed in a fixed order, without atomics on floats.
// 128 experts of 2048 x 768, top 8, bf16, all three launches replayed one behind the other, without a profiler: 185 to 190 us
// for 64 tokens, 97 to 99% of the measured copy bandwidth over the whole layer (alone, gate and up take 120 to 124 and down
// 64), 91 for nine, 25 for one, of which 12 are its weights and the rest starts and routing.
#include <cooperative_groups.h>

#include <type_traits>

#include "host_common.h"
#include "ptx.cuh"

namespace sb {
namespace mf {

namespace cg = cooperative_groups;

constexpr int kMaxExperts = 1024;
constexpr int kMaxEntries = 2048;
constexpr int kMaxTopK = 16;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---------------------------------------------------------------------------
// Router.  A cluster of eight CTAs takes eight tokens and an eighth of the experts each, 16 experts at a time; the CTA's
// warps split the columns, and the logits of token i meet in CTA i's shared memory.  Products of bf16 are exact in the
// matrix unit; its fp32 sums are taken out every 32 columns and carried on in two fp32 words, and where the order still
// hangs on their error (one row in 140 at 128 experts) the logits in question are summed again in fp64: experts are ordered
// by the values, equal ones by their number.  128 experts, rows of 2048: 4.6 us for one token, 4.9 for 64, of which 0.3 are
// that check; a call with a row whose logits are in question takes 3 more.
// The k largest are found by rank, the number of experts that come before one: all are compared with one another at once,
// where k rounds of a maximum would wait for one another.  Beyond kRankGroup experts, passes over groups leave k
// candidates each, and a last pass ranks those.
// ---------------------------------------------------------------------------
constexpr int kCluster = 8;  // CTAs, and tokens
constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRankGroup = 128;  // entries ranked in a pass, two lanes each
// Logits that lie closer than this share of the largest sum of magnitudes are compared in fp64.  Each of the 16 addends of
// a product is cut off at 2^-24 of the largest one, its result at 2^-23, and two results are added in fp32: 19 * 2^-24 of
// the 32 columns' sum of magnitudes, however one of them dominates.  Two logits: 38 * 2^-24, below 2^-18.  (A product that
// starts from another's result cuts off at that: such a chain would need twice as much.)
constexpr double kLogitError = 1.0 / (1 << 18);
constexpr int kExactBatch = 4;

// Order-preserving key of a logit, unique: the lowest ten bits hold the expert, the lower one first among equals.  A NaN
// comes last.
__device__ __forceinline__ unsigned long long logit_key(double v, int e) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
  const unsigned long long k = v != v ? 0ull : (b >> 63 ? ~b : b | 0x8000000000000000ull);
  return (k & ~1023ull) | static_cast<unsigned long long>(1023 - e);
}
__device__ __forceinline__ int key_expert(unsigned long long k) { return 1023 - static_cast<int>(k & 1023); }

// z + the products of eight bf16 pairs, in fp64
__device__ __forceinline__ double dot8(const uint4& a, const uint4& b, double z) {
  const uint32_t p[4] = {a.x, a.y, a.z, a.w}, q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    z = fma(static_cast<double>(__uint_as_float(p[j] << 16)), static_cast<double>(__uint_as_float(q[j] << 16)), z);
    z = fma(static_cast<double>(__uint_as_float(p[j] & 0xffff0000u)), static_cast<double>(__uint_as_float(q[j] & 0xffff0000u)), z);
  }
  return z;
}

// Entries of key[0..n) above `mine`, counted by two neighbouring lanes.
__device__ __forceinline__ int rank_of(const unsigned long long* key, int n, unsigned long long mine) {
  int before = 0;
#pragma unroll 8
  for (int j = threadIdx.x & 1; j < n; j += 2) before += key[j] > mine;
  return before + __shfl_xor_sync(0xffffffffu, before, 1);
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kRouteThreads, 1)
route_kernel(const __nv_bfloat16* __restrict__ h, long long h_stride, const __nv_bfloat16* __restrict__ rw,
             const int* __restrict__ live, float* __restrict__ w, int* __restrict__ idx, int T, int E, int H, int k, int norm) {
  __shared__ float2 part[kRouteWarps][4][32];
  __shared__ float part_mag[kRouteWarps][4][32], warp_mag[kRouteWarps];
  __shared__ unsigned long long key[kMaxExperts], cand[kRankGroup];
  __shared__ int n_cand, n_close, chosen[kMaxTopK];
  __shared__ unsigned short near[kMaxExperts];
  __shared__ double exact_part[kExactBatch][kRouteWarps];
  extern __shared__ double logits[];  // [E], of token t0 + rank
  float* mags = reinterpret_cast<float*>(logits + E);  // [E] sums of the products' magnitudes
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = static_cast<int>(blockIdx.x / kCluster) * kCluster;
  cluster.barrier_arrive();
  pdl_launch_dependents();
  if (threadIdx.x == 0) n_cand = 0;
  const int per = (E + kCluster - 1) / kCluster;
  const int e_hi = min(E, (rank + 1) * per);
  const int g = lane >> 2, t4 = lane & 3;
  const int steps = (H + 31) >> 5, s0 = warp * steps / kRouteWarps, s1 = (warp + 1) * steps / kRouteWarps;
  const __nv_bfloat16* x = h + static_cast<size_t>(min(t0 + g, T - 1)) * h_stride + 8 * t4;  // rows behind the last: not used
  bool waited = false;
  for (int e0 = rank * per; e0 < e_hi; e0 += 16) {
    const __nv_bfloat16* top = rw + static_cast<size_t>(min(e0 + g, e_hi - 1)) * H + 8 * t4;
    const __nv_bfloat16* low = rw + static_cast<size_t>(min(e0 + g + 8, e_hi - 1)) * H + 8 * t4;
    float hi[4] = {0.f, 0.f, 0.f, 0.f}, lo[4] = {0.f, 0.f, 0.f, 0.f}, mag[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int kUnroll = 8;
    for (int s = s0; s < s1; s += kUnroll) {
      uint4 a[kUnroll], b[kUnroll], v[kUnroll];
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        const int col = (s + j) * 32;
        const bool ok = s + j < s1 && col + 8 * t4 < H;
        const uint4 z = make_uint4(0, 0, 0, 0);
        a[j] = ok ? __ldg(reinterpret_cast<const uint4*>(top + col)) : z;
        b[j] = ok ? __ldg(reinterpret_cast<const uint4*>(low + col)) : z;
        v[j] = ok ? __ldg(reinterpret_cast<const uint4*>(x + col)) : z;
      }
#pragma unroll
      for (int j = 0; j < kUnroll; ++j) {
        float d[4] = {0.f, 0.f, 0.f, 0.f}, d2[4] = {0.f, 0.f, 0.f, 0.f};
        mma_bf16(d, a[j].x, b[j].x, a[j].y, b[j].y, v[j].x, v[j].y);
        mma_bf16(d2, a[j].z, b[j].z, a[j].w, b[j].w, v[j].z, v[j].w);
        constexpr uint32_t kAbs = 0x7fff7fffu;
        mma_bf16(mag, a[j].x & kAbs, b[j].x & kAbs, a[j].y & kAbs, b[j].y & kAbs, v[j].x & kAbs, v[j].y & kAbs);
        mma_bf16(mag, a[j].z & kAbs, b[j].z & kAbs, a[j].w & kAbs, b[j].w & kAbs, v[j].z & kAbs, v[j].w & kAbs);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float both = d[c] + d2[c], sum = hi[c] + both, back = sum - hi[c];
          lo[c] += (hi[c] - (sum - back)) + (both - back);  // what the addition rounded away
          hi[c] = sum;
        }
      }
    }
    if (waited) __syncthreads();  // the sums of the 16 experts before have been read
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      part[warp][c][lane] = make_float2(hi[c], lo[c]);
      part_mag[warp][c][lane] = mag[c];
    }
    __syncthreads();
    if (!waited) cluster.barrier_wait();  // every CTA of the cluster runs before its shared memory is written
    waited = true;
    if (threadIdx.x < 128) {
      const int c = threadIdx.x >> 5;  // fragment component: expert g + 8 (c / 2), token 2 t4 + c % 2
      double v = 0.0;
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < kRouteWarps; ++i) {
        const float2 s = part[i][c][lane];
        v += s.y == s.y ? static_cast<double>(s.x) + static_cast<double>(s.y) : static_cast<double>(s.x);  // infinite: no remainder
        m += part_mag[i][c][lane];
      }
      const int e = e0 + g + 8 * (c >> 1), to = 2 * t4 + (c & 1);
      if (e < e_hi) {
        cluster.map_shared_rank(logits, to)[e] = v + 0.0;  // -0 counts as +0
        cluster.map_shared_rank(mags, to)[e] = m;
      }
    }
  }
  if (!waited) cluster.barrier_wait();
  cluster.sync();
  const int t = t0 + rank;
  if (t >= T) return;
  if (live && live[t] == 0) {
    if (threadIdx.x < k) {
      w[static_cast<size_t>(t) * k + threadIdx.x] = 0.f;
      idx[static_cast<size_t>(t) * k + threadIdx.x] = -1;
    }
    return;
  }
  int bad = 0;
  float top_mag = 0.f;
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    const double v = logits[e];
    bad |= v != v;
    key[e] = logit_key(v, e);
    top_mag = fmaxf(top_mag, mags[e]);
  }
  top_mag = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_mag)));  // none is negative
  if (lane == 0) warp_mag[warp] = top_mag;
  bad = __syncthreads_or(bad);
#pragma unroll
  for (int i = 0; i < kRouteWarps; ++i) top_mag = fmaxf(top_mag, warp_mag[i]);
  const double tol = static_cast<double>(top_mag) * kLogitError;
  for (bool exact = false;; exact = true) {
    const int slot = threadIdx.x >> 1;
    const unsigned long long* of = key;
    int n = E;
    if (E > kRankGroup) {  // at most eight groups, with k <= 16 candidates each
      for (int g0 = 0; g0 < E; g0 += kRankGroup) {
        const int gn = min(kRankGroup, E - g0);
        const unsigned long long mine = key[g0 + min(slot, gn - 1)];
        const int before = rank_of(key + g0, gn, mine);
        if (slot < gn && !(threadIdx.x & 1) && before < k) cand[atomicAdd(&n_cand, 1)] = mine;
      }
      __syncthreads();
      n = n_cand;
      of = cand;
    }
    const unsigned long long mine = of[min(slot, n - 1)];
    const int before = rank_of(of, n, mine);
    if (slot < n && !(threadIdx.x & 1) && before < k) chosen[before] = key_expert(mine);
    __syncthreads();
    int close = 0;
    if (warp == 0) {
      const int my_e = lane < k ? chosen[lane] : chosen[0];
      const double top = logits[chosen[0]];
      const float p = expf(static_cast<float>(logits[my_e] - top));
      float all = 0.f;
      if (norm)
        all = lane < k ? p : 0.f;
      else
        for (int e = lane; e < E; e += 32) all += expf(static_cast<float>(logits[e] - top));
      all = warp_sum(all);
      if (lane < k) {
        w[static_cast<size_t>(t) * k + lane] = bad ? __int_as_float(0x7fffffff) : p / all;
        idx[static_cast<size_t>(t) * k + lane] = my_e;
      }
    } else if (!exact) {  // whether the error of the sums could have made this order
      const int i = threadIdx.x - 32;
      const double last = logits[chosen[k - 1]];
      const unsigned long long last_key = key[chosen[k - 1]];
      close = i + 1 < k && logits[chosen[i]] - logits[chosen[i + 1]] <= tol;
      for (int e = i; e < E; e += kRouteThreads - 32) close |= key[e] < last_key && logits[e] >= last - tol;
    }
    if (!__syncthreads_or(close)) return;
    // the logits in question again in fp64, and once more: chosen ones beside a neighbour or the last one, others beside it
    const double last = logits[chosen[k - 1]];
    const unsigned long long last_key = key[chosen[k - 1]];
    if (threadIdx.x == 0) n_cand = n_close = 0;
    __syncthreads();
    const int r = threadIdx.x;
    if (r < k) {
      const double z = logits[chosen[r]];
      if (z - last <= tol || (r > 0 && logits[chosen[r - 1]] - z <= tol) || z - logits[chosen[min(r + 1, k - 1)]] <= tol)
        near[atomicAdd(&n_close, 1)] = static_cast<unsigned short>(chosen[r]);
    }
    for (int e = threadIdx.x; e < E; e += kRouteThreads)
      if (key[e] < last_key && logits[e] >= last - tol) near[atomicAdd(&n_close, 1)] = static_cast<unsigned short>(e);
    __syncthreads();
    const int n_near = n_close;
    for (int c0 = 0; c0 < n_near; c0 += kExactBatch) {  // every thread takes eight columns of a batch of experts
      double z[kExactBatch];
      const __nv_bfloat16* row[kExactBatch];
#pragma unroll
      for (int j = 0; j < kExactBatch; ++j) {
        z[j] = 0.0;
        row[j] = rw + static_cast<size_t>(near[min(c0 + j, n_near - 1)]) * H;
      }
      for (int i = threadIdx.x * 8; i < H; i += 8 * kRouteThreads) {
        const uint4 x8 = *reinterpret_cast<const uint4*>(h + static_cast<size_t>(t) * h_stride + i);
        uint4 w8[kExactBatch];
#pragma unroll
        for (int j = 0; j < kExactBatch; ++j) w8[j] = __ldg(reinterpret_cast<const uint4*>(row[j] + i));
#pragma unroll
        for (int j = 0; j < kExactBatch; ++j) z[j] = dot8(x8, w8[j], z[j]);
      }
#pragma unroll
      for (int j = 0; j < kExactBatch; ++j) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z[j] += __shfl_xor_sync(0xffffffffu, z[j], o);
        if (lane == 0) exact_part[j][warp] = z[j];
      }
      __syncthreads();
      if (threadIdx.x < kExactBatch && c0 + static_cast<int>(threadIdx.x) < n_near) {
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < kRouteWarps; ++i) v += exact_part[threadIdx.x][i];
        const int e = near[c0 + threadIdx.x];
        logits[e] = v + 0.0;
        key[e] = logit_key(v + 0.0, e);
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of every expert, in shared memory: entry = token * k + slot.  An expert's rows are taken in units of at most
// kUnitRows.  An entry's result does not depend on its neighbours, so the order of an expert's entries matters only where
// they are cut into units, which all CTAs have to cut alike.
// ---------------------------------------------------------------------------
constexpr int kUnitRows = 16;

struct Lists {
  int* cursor;              // [E] scratch of the construction
  unsigned short* first;    // [E + 1] first entry of each expert
  unsigned short* used;     // [E] experts that have entries, ascending
  unsigned short* unit0;    // [E + 1] first unit of the i-th used expert
  unsigned short* entry;    // [n]
  int* count;               // per 32 experts: rows | units << 16, used experts, rows of the largest expert
  int n_used, n_units, most;
};

__host__ __device__ constexpr int lists_bytes(int n, int E) {
  return (4 * 3 * 32 + 4 * E + 2 * (E + 1) * 2 + 2 * E + 2 * n + 127) / 128 * 128;
}

__device__ __forceinline__ Lists build_lists(char* smem, const int* idx, int n, int E) {
  Lists L;
  L.count = reinterpret_cast<int*>(smem);
  L.cursor = L.count + 3 * 32;
  L.first = reinterpret_cast<unsigned short*>(L.cursor + E);
  L.unit0 = L.first + E + 1;
  L.used = L.unit0 + E + 1;
  L.entry = L.used + E;
  const int lane = threadIdx.x & 31;
  const int held = threadIdx.x < n ? idx[threadIdx.x] : -1;  // this thread's first entry
  for (int e = threadIdx.x; e < E; e += blockDim.x) L.cursor[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int e = i == threadIdx.x ? held : idx[i];
    if (e >= 0 && e < E) atomicAdd(&L.cursor[e], 1);
  }
  __syncthreads();
  // a warp takes 32 experts at a time: totals first, then offsets from the totals before.  Rows in the low half, units in
  // the high half: neither passes 16 bits (at most kMaxEntries of each).
  const int chunks = (E + 31) >> 5, warps = blockDim.x >> 5;
  for (int c = threadIdx.x >> 5; c < chunks; c += warps) {
    const int e = c * 32 + lane;
    const int rows = e < E ? L.cursor[e] : 0;
    const int sum = __reduce_add_sync(0xffffffffu, rows | ((rows + kUnitRows - 1) / kUnitRows) << 16);
    const int most = __reduce_max_sync(0xffffffffu, rows);
    const unsigned int has = __ballot_sync(0xffffffffu, rows > 0);
    if (lane == 0) {
      L.count[c] = sum;
      L.count[32 + c] = __popc(has);
      L.count[64 + c] = most;
    }
  }
  __syncthreads();
  {
    const bool on = lane < chunks;
    const int sum = __reduce_add_sync(0xffffffffu, on ? L.count[lane] : 0);
    L.n_units = sum >> 16;
    L.n_used = __reduce_add_sync(0xffffffffu, on ? L.count[32 + lane] : 0);
    L.most = min(kUnitRows, __reduce_max_sync(0xffffffffu, on ? L.count[64 + lane] : 0));
    if (threadIdx.x == 0) {
      L.first[E] = static_cast<unsigned short>(sum & 0xffff);
      L.unit0[L.n_used] = static_cast<unsigned short>(sum >> 16);
    }
  }
  for (int c = threadIdx.x >> 5; c < chunks; c += warps) {
    const int e = c * 32 + lane;
    const int rows = e < E ? L.cursor[e] : 0;
    const int own = rows | ((rows + kUnitRows - 1) / kUnitRows) << 16;
    int inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const int at = __reduce_add_sync(0xffffffffu, lane < c ? L.count[lane] : 0) + inc - own;
    const int a = __reduce_add_sync(0xffffffffu, lane < c ? L.count[32 + lane] : 0) +
                  __popc(__ballot_sync(0xffffffffu, rows > 0) & ((1u << lane) - 1u));
    if (e < E) {
      L.cursor[e] = at & 0xffff;
      L.first[e] = static_cast<unsigned short>(at & 0xffff);
      if (rows > 0) {
        L.used[a] = static_cast<unsigned short>(e);
        L.unit0[a] = static_cast<unsigned short>(at >> 16);
      }
    }
  }
  __syncthreads();
  if (L.n_units == L.n_used) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int e = i == threadIdx.x ? held : idx[i];
      if (e >= 0 && e < E) L.entry[atomicAdd(&L.cursor[e], 1)] = static_cast<unsigned short>(i);
    }
  } else if (threadIdx.x < 32) {  // in the entries' order, 32 at a time
    for (int base = 0; base < n; base += 32) {
      const int i = base + lane;
      int e = i < n ? idx[i] : -1;
      const bool on = e >= 0 && e < E;
      if (!on) e = -1 - lane;
      const unsigned int peers = __match_any_sync(0xffffffffu, e);
      const int rank = __popc(peers & ((1u << lane) - 1u));
      if (on) L.entry[L.cursor[e] + rank] = static_cast<unsigned short>(i);
      __syncwarp();
      if (on && rank == 0) L.cursor[e] += __popc(peers);
      __syncwarp();
    }
  }
  __syncthreads();
  return L;
}

struct Unit {
  int e, r0, r1;  // expert and its entries [r0, r1)
};
__device__ __forceinline__ Unit unit_at(const Lists& L, int unit) {
  int lo = 0, hi = L.n_used - 1;  // last used expert whose first unit is not behind `unit`
  if (L.n_units == L.n_used) lo = hi = unit;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.unit0[mid] <= unit)
      lo = mid;
    else
      hi = mid - 1;
  }
  Unit u;
  u.e = L.used[lo];
  u.r0 = L.first[u.e] + (unit - L.unit0[lo]) * kUnitRows;
  u.r1 = min(static_cast<int>(L.first[u.e + 1]), u.r0 + kUnitRows);
  return u;
}

// ---------------------------------------------------------------------------
// The weight stream.  An item is 16 weight rows of one unit, in two blocks of eight rows that lie one behind the other in
// memory.  A ring of stages takes a block each (or a piece of at most kMaxPiece columns of it); one lane fills it with
// bulk copies as far ahead as the ring is long, a whole block in a copy where it fits: a copy costs the engine about 90
// cycles whatever its size: rows of 1.5 KB one by one came at 4.8 TB/s, blocks of 16 to 32 KB come at 6.7 to 6.9.
// The consumers are groups of kGroup warps; each group takes the next item on, its warps a share of the columns each, and
// their sums meet in shared memory at the end of the item.  A warp's share stays in registers, so that wide rows need all
// eight warps; narrow ones leave groups that hide one another's barriers (gate, up and down of 64 tokens, 128 experts of
// 1024 x 512, top 8: 89 us with one group, 74 with two; of 28 tokens, 159 experts of 1288 x 728: 133 and 120; of 64 tokens,
// 128 experts of 256 x 256: 35 with one, 31 with eight).
// A stage always returns to the group that used it last: the ring's length is a multiple of the blocks that a round of all
// groups takes.  Copies may land in any order, and a group that met a stage for the first time could find the other group's
// copy still under way; the parity it waits for would then name the phase before that copy, which is complete, and the wait
// would end at once.
// ---------------------------------------------------------------------------
constexpr int kConsumers = 8;
constexpr int kConsumerThreads = 32 * kConsumers;
constexpr int kRingThreads = kConsumerThreads + 32;
constexpr int kMaxStages = 32;
constexpr int kMaxPiece = 2048;  // columns
// k steps of 32 columns, at most, of a warp's share: more than twelve spill with 16 rows a unit
__host__ __device__ constexpr int max_steps(int group) { return group == kConsumers ? kMaxPiece / 32 / kConsumers : 12; }
constexpr int kMaxNt = kUnitRows / 8;
constexpr int kRedBytes = 2 * kConsumers * kMaxNt * 32 * 16;  // sums of two items

struct Ring {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
};

struct Shape {
  int stages, pieces, piece, K;  // piece: columns of a stage's rows
};

struct Turn {  // place in the ring
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step(int stages) {
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
};

// Weights that other kernels wrote through ordinary stores are read by bulk copies.
__device__ __forceinline__ void fence_proxy_async_global() { asm volatile("fence.proxy.async.global;" ::: "memory"); }
template <int kGroup>
__device__ __forceinline__ void group_sync(int group) {
  if (kGroup == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(32 * kGroup) : "memory");
}

// Fill the stages of one item (called by a whole warp): blocks of rows_a rows at a and rows_b rows at b.  Returns false
// when a wait gave up.  `filled` counts the stages filled.
__device__ __forceinline__ bool produce_item(Ring& ring, char* buf, const Shape& s, Turn& turn, long long& filled, const __nv_bfloat16* a,
                                             int rows_a, const __nv_bfloat16* b, int rows_b, int* status) {
  const int lane = threadIdx.x & 31;
  for (int q = 0; q < s.pieces; ++q)
    for (int half = 0; half < 2; ++half, ++filled, turn.step(s.stages)) {
      const __nv_bfloat16* src = half ? b : a;
      const int rows = half ? rows_b : rows_a;
      // the warp gives up as one: no lane copies to a stage that another did not announce
      if (!__all_sync(0xffffffffu, mbar_wait(&ring.empty[turn.stage], turn.parity ^ 1, status, 0x4d01))) return false;
      const uint32_t bytes = 2u * min(s.piece, s.K - q * s.piece);
      char* dst = buf + static_cast<size_t>(turn.stage) * 16 * s.piece;
      if (lane == 0) mbar_arrive_expect_tx(&ring.full[turn.stage], bytes * rows);
      __syncwarp();
      if (s.pieces == 1) {
        if (lane == 0 && rows > 0) bulk_load(dst, src, bytes * rows, &ring.full[turn.stage]);
      } else if (lane < rows) {
        bulk_load(dst + lane * 2 * s.piece, src + static_cast<size_t>(lane) * s.K + q * s.piece, bytes, &ring.full[turn.stage]);
      }
    }
  return true;
}

// A group's loop over its items, every (kConsumers / kGroup)-th of `items`.  unit_of() gives the unit of its next item,
// row_ptr(r) the operand row of entry r, finish(unit, sums) takes the warps' sums [warp][column group][lane] of an item.  A warp's share of the operand rows
// stays in registers from item to item of a unit (rows of more than one piece: from L1 or L2 again).
template <int kNt, int kGroup, class UnitOf, class RowPtr, class Finish>
__device__ __forceinline__ void consume(Ring& ring, const char* buf, float4* red, const Shape& s, int items, int* status,
                                        UnitOf unit_of, RowPtr row_ptr, Finish finish) {
  constexpr int kGroups = kConsumers / kGroup, kSteps = max_steps(kGroup);
  const int lane = threadIdx.x & 31, group = threadIdx.x / (32 * kGroup), warp = (threadIdx.x >> 5) % kGroup;
  const int g = lane >> 2, t4 = lane & 3;
  // k steps of piece q that fall to this warp: `mine` from `lo`; the first `some` of them have columns for this lane
  int lo = 0, mine = 0, some = 0;
  auto share = [&](int q) {
    const int cols = min(s.piece, s.K - q * s.piece);
    const int steps = (cols + 31) >> 5;
    lo = warp * steps / kGroup;
    mine = (warp + 1) * steps / kGroup - lo;
    some = min(mine, max(0, (cols - lo * 32 - 8 * t4 + 31) >> 5));
  };
  share(0);
  const __nv_bfloat16* x[kNt];
  uint4 v[kSteps][kNt];
  auto request = [&](int q) {
    const int at = q * s.piece + lo * 32;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int n = 0; n < kNt; ++n)
        v[j][n] = j < some && x[n] ? *reinterpret_cast<const uint4*>(x[n] + at + j * 32) : make_uint4(0, 0, 0, 0);
  };
  Turn turn;
  for (int i = 0; i < 2 * group; ++i) turn.step(s.stages);  // more than one group: rows of one piece
  int r0 = -1;
  // After a wait gave up, the items are run through without waiting: every warp still meets the others.  It gives no stage
  // back any more, so that none is filled over a copy that has not landed: the producer's wait ends too, as the status is set.
  bool ok = true;
  float4* sums = red + group * (2 * kGroup * kNt * 32);
  for (int i = group; i < items; i += kGroups) {
    const Unit u = unit_of();
    float acc[kNt][4];
#pragma unroll
    for (int n = 0; n < kNt; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
    const bool changed = u.r0 != r0;
    if (changed) {
      r0 = u.r0;
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        const int r = r0 + n * 8 + g;
        x[n] = r < u.r1 ? row_ptr(r) + 8 * t4 : nullptr;
      }
    }
    for (int q = 0; q < s.pieces; ++q) {
      if (s.pieces > 1) share(q);
      if (changed || s.pieces > 1) request(q);
      const int off = g * 2 * s.piece + lo * 64 + 16 * t4;
      const char* top = buf + static_cast<size_t>(turn.stage) * 16 * s.piece + off;
      uint64_t* free_a = &ring.empty[turn.stage];
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&ring.full[turn.stage], turn.parity, status, 0x4d02));
      turn.step(s.stages);
      const char* low = buf + static_cast<size_t>(turn.stage) * 16 * s.piece + off;
      uint64_t* free_b = &ring.empty[turn.stage];
      ok = ok && __all_sync(0xffffffffu, mbar_wait(&ring.full[turn.stage], turn.parity, status, 0x4d03));
      turn.step(s.stages);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        if (j >= mine) break;
        uint4 a = make_uint4(0, 0, 0, 0), b = a;
        if (j < some) {  // what lies behind a row in a stage belongs to other rows
          a = *reinterpret_cast<const uint4*>(top + j * 64);
          b = *reinterpret_cast<const uint4*>(low + j * 64);
        }
#pragma unroll
        for (int n = 0; n < kNt; ++n) {
          mma_bf16(acc[n], a.x, b.x, a.y, b.y, v[j][n].x, v[j][n].y);
          mma_bf16(acc[n], a.z, b.z, a.w, b.w, v[j][n].z, v[j][n].w);
        }
      }
      __syncwarp();
      if (lane == 0 && ok) {
        mbar_arrive(free_a);
        mbar_arrive(free_b);
      }
    }
#pragma unroll
    for (int skip = 0; skip < 2 * (kGroups - 1); ++skip) turn.step(s.stages);
    // two buffers: an item's sums are read while the next item's are not yet all written, so one barrier an item is enough
#pragma unroll
    for (int n = 0; n < kNt; ++n) sums[(warp * kNt + n) * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
    group_sync<kGroup>(group);
    finish(u, sums);
    sums = red + group * (2 * kGroup * kNt * 32) + (sums == red + group * (2 * kGroup * kNt * 32) ? kGroup * kNt * 32 : 0);
  }
}

// Sum over the warps of component c of column group n's fragment in lane l.
template <int kNt, int kGroup>
__device__ __forceinline__ float warp_total(const float4* sums, int n, int l, int c) {
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < kGroup; ++w) v += reinterpret_cast<const float*>(&sums[(w * kNt + n) * 32 + l])[c];
  return v;
}

__device__ __forceinline__ void ring_init(Ring& ring, int stages, int group_warps) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], group_warps);
    }
    fence_mbar_init();
  }
}
// The producer's end: copies that are still under way land before the CTA's shared memory is given back.  The consumers
// wait for them too, but one that gave up does not.  `filled`: stages filled in all, the last of them before `turn`.
__device__ __forceinline__ void ring_drain(Ring& ring, const Shape& s, Turn turn, long long filled) {
  Turn oldest;  // of the last s.stages fills
  if (filled >= s.stages) {
    oldest = turn;
    oldest.parity ^= 1;
  }
  const int n = filled < s.stages ? static_cast<int>(filled) : s.stages;
  const unsigned long long t0 = globaltimer_ns();
  for (int i = 0; i < n; ++i, oldest.step(s.stages)) {
    while (!mbar_try_wait(&ring.full[oldest.stage], oldest.parity))
      if (globaltimer_ns() - t0 > kWaitTimeoutNs) break;
  }
}

// ---------------------------------------------------------------------------
// Gate and up projections: an item is eight gate rows and the eight up rows beside them, so that a lane holds both
// factors of an activation.
// ---------------------------------------------------------------------------
template <int kGroup>
__global__ void __launch_bounds__(kRingThreads, 1)
gate_up_kernel(const __nv_bfloat16* h, long long h_stride, const int* idx, const __nv_bfloat16* __restrict__ wgu,
               __nv_bfloat16* act, int n, int k, int E, int H, int F, Shape s, int* status) {
  __shared__ Ring ring;
  extern __shared__ __align__(128) char smem[];
  float4* red = reinterpret_cast<float4*>(smem);
  char* buf = smem + kRedBytes;
  ring_init(ring, s.stages, kGroup);
  pdl_wait();
  pdl_launch_dependents();
  const Lists L = build_lists(buf + static_cast<size_t>(s.stages) * 16 * s.piece, idx, n, E);
  const int tiles = (F + 7) >> 3;
  const long long items = static_cast<long long>(L.n_units) * tiles;
  const int lo = static_cast<int>(items * blockIdx.x / gridDim.x), hi = static_cast<int>(items * (blockIdx.x + 1) / gridDim.x);
  if (threadIdx.x >= kConsumerThreads) {
    Turn turn;
    int unit = lo / tiles, tile = lo - unit * tiles;
    long long filled = 0;
    bool ok = true;
    fence_proxy_async_global();
    for (int i = lo; ok && i < hi; ++unit, tile = 0) {
      const Unit u = unit_at(L, unit);
      for (; ok && tile < tiles && i < hi; ++tile, ++i) {
        const int f0 = tile * 8, rows = min(8, F - f0);
        const __nv_bfloat16* w = wgu + (static_cast<size_t>(u.e) * 2 * F + f0) * H;
        ok = produce_item(ring, buf, s, turn, filled, w, rows, w + static_cast<size_t>(F) * H, rows, status);
      }
    }
    ring_drain(ring, s, turn, filled);
    return;
  }
  auto run = [&](auto nt) {
    constexpr int kNt = decltype(nt)::value;
    constexpr int kGroups = kConsumers / kGroup;
    const int group = threadIdx.x / (32 * kGroup), first = lo + group;
    int unit = first / tiles, tile = first - unit * tiles - kGroups, f0 = 0;
    Unit u = {};
    if (first < hi) u = unit_at(L, unit);
    auto unit_of = [&]() {
      tile += kGroups;
      if (tile >= tiles) {
        do {
          tile -= tiles;
          ++unit;
        } while (tile >= tiles);
        u = unit_at(L, unit);
      }
      f0 = tile * 8;
      return u;
    };
    auto row_ptr = [&](int r) { return h + static_cast<size_t>(L.entry[r] / k) * h_stride; };
    auto finish = [&](const Unit& v, const float4* sums) {
      // (column group, lane of the fragment, one of its two columns)
      for (int o = threadIdx.x % (32 * kGroup); o < kNt * 64; o += 32 * kGroup) {
        const int c = o & 1, l = (o >> 1) & 31, grp = o >> 6;
        const int r = v.r0 + grp * 8 + 2 * (l & 3) + c, f = f0 + (l >> 2);
        if (r >= v.r1 || f >= F) continue;
        const float gate = warp_total<kNt, kGroup>(sums, grp, l, c), up = warp_total<kNt, kGroup>(sums, grp, l, 2 + c);
        // the activation is the down product's bf16 operand, rounded here as on the path for many tokens
        act[static_cast<size_t>(L.entry[r]) * F + f] = __float2bfloat16_rn(gate / (1.f + __expf(-gate)) * up);
      }
    };
    consume<kNt, kGroup>(ring, buf, red, s, hi - lo, status, unit_of, row_ptr, finish);
  };
  if (L.most <= 8)
    run(std::integral_constant<int, 1>());
  else
    run(std::integral_constant<int, 2>());
}

// ---------------------------------------------------------------------------
// Down projection and combination.  A CTA owns 16 columns of the output for all tokens; where there are fewer such columns
// than SMs, the CTAs of a cluster share them, each with a part of the units and, at the end, of the tokens (34 tokens, 104
// experts of 552 x 560, top 7: 33 us with a CTA for 16 columns, 18 with three).  Its warps take the units in turn,
// one each, with the weights straight from global memory into fragments: 16 warps with 16 loads a lane keep 128 KB a SM
// under way, and no warp waits for another.  The entries' results stay in shared memory until all are there and are then
// added up slot by slot, so no sum crosses a CTA.
// ---------------------------------------------------------------------------
constexpr int kDownThreads = 512;

// weights are read once: keep them from displacing the operand rows in L1
__device__ __forceinline__ uint4 ld_stream(const __nv_bfloat16* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int kNt>
__device__ __forceinline__ void down_unit(const Lists& L, float* y, const __nv_bfloat16* act, const __nv_bfloat16* wd, const Unit& u,
                                          int n0, int H, int F, int k, int size) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  constexpr int kUnroll = kNt == 1 ? 8 : 4;
  const __nv_bfloat16* base = wd + (static_cast<size_t>(u.e) * H + n0) * F + 8 * t4;
  // rows behind the last are read as the last one; their results are not stored
  const __nv_bfloat16* top = base + static_cast<size_t>(min(g, H - 1 - n0)) * F;
  const __nv_bfloat16* low = base + static_cast<size_t>(min(g + 8, H - 1 - n0)) * F;
  const __nv_bfloat16* x[kNt];
  float acc[kNt][4];
#pragma unroll
  for (int n = 0; n < kNt; ++n) {
    const int r = u.r0 + n * 8 + g;
    x[n] = r < u.r1 ? act + static_cast<size_t>(L.entry[r]) * F + 8 * t4 : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  }
  const int steps = (F - 8 * t4 + 31) >> 5;  // of this lane; lane t4 = 0 has the most
  const int all = (F + 31) >> 5;
  for (int s = 0; s < all; s += kUnroll) {
    uint4 a[kUnroll], b[kUnroll], v[kUnroll][kNt];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      const bool ok = s + j < steps;
      a[j] = ok ? ld_stream(top + (s + j) * 32) : z;
      b[j] = ok ? ld_stream(low + (s + j) * 32) : z;
#pragma unroll
      for (int n = 0; n < kNt; ++n) v[j][n] = ok && x[n] ? *reinterpret_cast<const uint4*>(x[n] + (s + j) * 32) : z;
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j)
#pragma unroll
      for (int n = 0; n < kNt; ++n) {
        mma_bf16(acc[n], a[j].x, b[j].x, a[j].y, b[j].y, v[j][n].x, v[j][n].y);
        mma_bf16(acc[n], a[j].z, b[j].z, a[j].w, b[j].w, v[j][n].z, v[j][n].w);
      }
  }
#pragma unroll
  for (int n = 0; n < kNt; ++n)
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      const int r = u.r0 + n * 8 + 2 * t4 + col;
      if (r < u.r1) {
        const int entry = L.entry[r];
        float* o = y + entry * 16;
        if (size > 1) o = cg::this_cluster().map_shared_rank(o, entry / k % size);  // the CTA that combines this token
        o[g] = acc[n][col];
        o[g + 8] = acc[n][2 + col];
      }
    }
}

// The combination of a CTA's 16 columns from y [T * k][16], for every `of`-th token from `first` on: slot by slot, so that
// the order is always the same.
__device__ __forceinline__ void combine(const float* y, const int* idx, const float* w, __nv_bfloat16* out, int n0, int T, int k,
                                        int E, int H, int first, int of) {
  for (int i = threadIdx.x;; i += kDownThreads) {
    const int t = (i >> 4) * of + first, c = i & 15;
    if (t >= T) break;
    if (n0 + c >= H) continue;
    float v = 0.f;
    for (int j = 0; j < k; ++j) {
      const int e = idx[t * k + j];
      if (e >= 0 && e < E) v = fmaf(w[t * k + j], y[(t * k + j) * 16 + c], v);
    }
    out[static_cast<size_t>(t) * H + n0 + c] = __float2bfloat16_rn(v);
  }
}

__global__ void __launch_bounds__(kDownThreads, 1)
down_kernel(const __nv_bfloat16* act, const int* __restrict__ idx, const float* w, const __nv_bfloat16* __restrict__ wd,
            __nv_bfloat16* __restrict__ out, int T, int k, int E, int H, int F) {
  extern __shared__ __align__(128) char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int size = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  if (size > 1) cluster.barrier_arrive();
  const int n = T * k;
  float* y = reinterpret_cast<float*>(smem);  // [n][16]; of the tokens that fall to this CTA
  const Lists L = build_lists(smem + sizeof(float) * 16 * static_cast<size_t>(n), idx, n, E);
  const int n0 = static_cast<int>(blockIdx.x) / size * 16;
  if (size > 1) cluster.barrier_wait();  // every CTA of the cluster runs before its shared memory is written
  for (int i = (threadIdx.x >> 5) * size + rank; i < L.n_units; i += kDownThreads / 32 * size) {
    const Unit u = unit_at(L, i);
    if (u.r1 - u.r0 <= 8)
      down_unit<1>(L, y, act, wd, u, n0, H, F, k, size);
    else
      down_unit<2>(L, y, act, wd, u, n0, H, F, k, size);
  }
  if (size > 1)
    cluster.sync();
  else
    __syncthreads();
  combine(y, idx, w, out, n0, T, k, E, H, rank, size);
}

// The same for so few entries that all weights a CTA needs fit into its shared memory at once (one token with eight experts
// of width 768).  A CTA starts when the first kernel's CTA on its SM ends, fetches its weights (a unit's 16 rows lie one
// behind the other: one bulk copy) while others of that kernel still run, and only then waits for the activations.  The
// routing table is complete by then: the kernel before waits for it before it lets this one start.  Both expert kernels
// for that token: 19.4 us, 22.9 with the kernel above in its place.
constexpr int kOnceUnits = 32;

template <int kNt>
__device__ __forceinline__ void once_unit(const Lists& L, float* y, const char* wgt, const char* act, const Unit& u, int rows, int F) {
  const int lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const char* top = wgt + static_cast<size_t>(min(g, rows - 1)) * 2 * F + 16 * t4;
  const char* low = wgt + static_cast<size_t>(min(g + 8, rows - 1)) * 2 * F + 16 * t4;
  const char* x[kNt];
  float acc[kNt][4];
#pragma unroll
  for (int n = 0; n < kNt; ++n) {
    const int r = u.r0 + n * 8 + g;
    x[n] = r < u.r1 ? act + static_cast<size_t>(r) * 2 * F + 16 * t4 : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  }
  const int steps = (F - 8 * t4 + 31) >> 5, all = (F + 31) >> 5;  // of this lane; lane t4 = 0 has the most
  const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll 4
  for (int s = 0; s < all; ++s) {
    const bool ok = s < steps;
    const uint4 a = ok ? *reinterpret_cast<const uint4*>(top + s * 64) : z;
    const uint4 b = ok ? *reinterpret_cast<const uint4*>(low + s * 64) : z;
#pragma unroll
    for (int n = 0; n < kNt; ++n) {
      const uint4 v = ok && x[n] ? *reinterpret_cast<const uint4*>(x[n] + s * 64) : z;
      mma_bf16(acc[n], a.x, b.x, a.y, b.y, v.x, v.y);
      mma_bf16(acc[n], a.z, b.z, a.w, b.w, v.z, v.w);
    }
  }
#pragma unroll
  for (int n = 0; n < kNt; ++n)
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      const int r = u.r0 + n * 8 + 2 * t4 + col;
      if (r < u.r1) {
        float* o = y + L.entry[r] * 16;
        o[g] = acc[n][col];
        o[g + 8] = acc[n][2 + col];
      }
    }
}

__host__ __device__ constexpr size_t once_bytes(int n, int F) { return static_cast<size_t>(n) * (34 * F + 64); }

__global__ void __launch_bounds__(kDownThreads, 1)
down_once_kernel(const __nv_bfloat16* act, const int* idx, const float* w, const __nv_bfloat16* __restrict__ wd, __nv_bfloat16* out,
                 int T, int k, int E, int H, int F, int* status) {
  extern __shared__ __align__(128) char smem[];
  __shared__ uint64_t full[kOnceUnits];
  const int n = T * k, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kDownThreads / 32;
  char* wgt = smem;                                     // [units][16][F]
  char* rows = smem + static_cast<size_t>(n) * 32 * F;  // [n][F], by place in the lists
  float* y = reinterpret_cast<float*>(rows + static_cast<size_t>(n) * 2 * F);
  if (threadIdx.x < n) mbar_init(&full[threadIdx.x], 1);
  if (threadIdx.x < 32) fence_mbar_init();
  const Lists L = build_lists(smem + once_bytes(n, F), idx, n, E);  // its barriers also order the lines above
  const int n0 = blockIdx.x * 16, n_rows = min(16, H - n0);
  if (lane == 0) {
    fence_proxy_async_global();
    for (int i = warp; i < L.n_units; i += kWarps) {
      const uint32_t bytes = 2u * F * n_rows;
      mbar_arrive_expect_tx(&full[i], bytes);
      bulk_load(wgt + static_cast<size_t>(i) * 32 * F, wd + (static_cast<size_t>(unit_at(L, i).e) * H + n0) * F, bytes, &full[i]);
    }
  }
  __syncwarp();
  pdl_wait();
  for (int i = warp; i < L.n_units; i += kWarps) {
    const Unit u = unit_at(L, i);
    for (int r = u.r0; r < u.r1; ++r) {
      const uint4* from = reinterpret_cast<const uint4*>(act + static_cast<size_t>(L.entry[r]) * F);
      uint4* to = reinterpret_cast<uint4*>(rows + static_cast<size_t>(r) * 2 * F);
#pragma unroll 4
      for (int c = lane; c < F / 8; c += 32) to[c] = from[c];
    }
  }
  __syncwarp();
  for (int i = warp; i < L.n_units; i += kWarps) {
    // the warp gives up as one, and its copy still lands before the buffer is given back
    if (!__all_sync(0xffffffffu, mbar_wait(&full[i], 0, status, 0x4d04))) {
      const unsigned long long t0 = globaltimer_ns();
      while (!mbar_try_wait(&full[i], 0))
        if (globaltimer_ns() - t0 > kWaitTimeoutNs) break;
      __syncwarp();
      continue;
    }
    const Unit u = unit_at(L, i);
    const char* mine = wgt + static_cast<size_t>(i) * 32 * F;
    if (u.r1 - u.r0 <= 8)
      once_unit<1>(L, y, mine, rows, u, n_rows, F);
    else
      once_unit<2>(L, y, mine, rows, u, n_rows, F);
  }
  __syncthreads();
  combine(y, idx, w, out, n0, T, k, E, H, 0, 1);
}

// The gate and up kernel's ring for rows of K columns beside the lists of n entries over E experts: stages of eight rows
// (or of pieces of them, equal ones, where a row has more than kMaxPiece columns), and as few warps a group as the columns
// allow.
struct RingPlan {
  Shape s;
  int group;    // warps of a consumer group
  size_t smem;  // dynamic shared memory
};
constexpr size_t kMostSmem = 227 * 1024 - sizeof(Ring) - 128;  // dynamic shared memory that a CTA may have beside its Ring
inline bool plan_ring(int n, int E, int K, RingPlan& plan) {
  const size_t fixed = kRedBytes + static_cast<size_t>(lists_bytes(n, E));
  Shape& s = plan.s;
  s.K = K;
  s.pieces = (K + kMaxPiece - 1) / kMaxPiece;
  s.piece = s.pieces == 1 ? K : ((K + s.pieces - 1) / s.pieces + 31) / 32 * 32;
  const size_t fit = (kMostSmem - fixed) / (16 * static_cast<size_t>(s.piece));
  const int most = static_cast<int>(fit < kMaxStages ? fit : kMaxStages), steps = (s.piece + 31) / 32;
  for (plan.group = s.pieces > 1 ? kConsumers : 1; plan.group <= kConsumers; plan.group *= 2) {
    const int round = 2 * kConsumers / plan.group;  // stages that an item of every group takes
    if (steps > plan.group * max_steps(plan.group)) continue;
    // one group meets every stage: any length will do
    s.stages = plan.group == kConsumers ? most : most / round * round;
    if (s.stages < round) continue;
    plan.smem = fixed + static_cast<size_t>(s.stages) * 16 * s.piece;
    return true;
  }
  return false;
}

template <int kGroup>
cudaError_t launch_gate_up(const void* h, long long h_stride, const int* idx, const void* wgu, void* act, int T, int k, int E, int H,
                           int F, const Shape& s, size_t smem, size_t smem_most, int* status, cudaStream_t st) {
  static bool attr_dev[64] = {};
  bool& attr = attr_dev[device_index()];
  if (!attr) {
    const cudaError_t e = cudaFuncSetAttribute(gate_up_kernel<kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_most));
    if (e != cudaSuccess) return e;
    attr = true;
  }
  return launch_pdl(gate_up_kernel<kGroup>, dim3(sm_count()), dim3(kRingThreads), smem, st, static_cast<const __nv_bfloat16*>(h), h_stride,
                    idx, static_cast<const __nv_bfloat16*>(wgu), static_cast<__nv_bfloat16*>(act), T * k, k, E, H, F, s, status);
}

cudaError_t launch_down(const void* act, const int* idx, const float* w, const void* wd, void* out, int T, int k, int E, int H, int F,
                        size_t smem, size_t smem_most, cudaStream_t st) {
  static bool attr_dev[64] = {};
  bool& attr = attr_dev[device_index()];
  if (!attr) {
    const cudaError_t e = cudaFuncSetAttribute(down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_most));
    if (e != cudaSuccess) return e;
    attr = true;
  }
  constexpr int kMaxCluster = 8;
  static int most_dev[64][kMaxCluster] = {};
  int* clusters = most_dev[device_index()];  // of 1 to 8 CTAs that run at once
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kDownThreads);
  cfg.dynamicSmemBytes = smem_most;
  cudaLaunchAttribute shape[1];
  shape[0].id = cudaLaunchAttributeClusterDimension;
  cfg.attrs = shape;
  cfg.numAttrs = 1;
  for (unsigned i = 1; i <= kMaxCluster && clusters[kMaxCluster - 1] == 0; ++i) {
    shape[0].val.clusterDim = {i, 1, 1};
    cfg.gridDim = dim3(i);
    int fit = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&fit, down_kernel, &cfg);
    if (e != cudaSuccess) return e;
    clusters[i - 1] = fit > 0 ? fit : 1;
  }
  const int tiles = (H + 15) / 16;
  unsigned size = 1;  // as many CTAs as run in one wave
  while (size < kMaxCluster && tiles <= clusters[size]) ++size;
  shape[0].val.clusterDim = {size, 1, 1};
  cfg.gridDim = dim3(tiles * size);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, down_kernel, static_cast<const __nv_bfloat16*>(act), idx, w, static_cast<const __nv_bfloat16*>(wd),
                            static_cast<__nv_bfloat16*>(out), T, k, E, H, F);
}

cudaError_t launch_down_once(const void* act, const int* idx, const float* w, const void* wd, void* out, int T, int k, int E, int H,
                             int F, size_t smem, size_t smem_most, int* status, cudaStream_t st) {
  static bool attr_dev[64] = {};
  bool& attr = attr_dev[device_index()];
  if (!attr) {
    const cudaError_t e = cudaFuncSetAttribute(down_once_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_most));
    if (e != cudaSuccess) return e;
    attr = true;
  }
  return launch_pdl(down_once_kernel, dim3((H + 15) / 16), dim3(kDownThreads), smem, st, static_cast<const __nv_bfloat16*>(act), idx, w,
                    static_cast<const __nv_bfloat16*>(wd), static_cast<__nv_bfloat16*>(out), T, k, E, H, F, status);
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
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  sb::mf::route_kernel<<<(T + sb::mf::kCluster - 1) / sb::mf::kCluster * sb::mf::kCluster, sb::mf::kRouteThreads, (sizeof(double) + sizeof(float)) * E, st>>>(
      static_cast<const __nv_bfloat16*>(h), h_stride, static_cast<const __nv_bfloat16*>(router), live, w, idx, T, E, H, k, norm);
  return cudaGetLastError() == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

// The ring that sb_moe_few_experts takes for n = T * k entries over E experts of rows of H columns: stages, pieces a row,
// columns a piece, consumer groups, bytes of dynamic shared memory.  Host only.
int sb_moe_few_ring(int n, int E, int H, int* stages, int* pieces, int* piece, int* groups, int* smem) {
  sb::mf::RingPlan p;
  if (n <= 0 || n > sb::mf::kMaxEntries || E <= 0 || E > sb::mf::kMaxExperts || H <= 0 || (H & 7)) return SB_ERR_ARG;
  if (!sb::mf::plan_ring(n, E, H, p)) return SB_ERR_TOO_LARGE;
  *stages = p.s.stages;
  *pieces = p.s.pieces;
  *piece = p.s.piece;
  *groups = sb::mf::kConsumers / p.group;
  *smem = static_cast<int>(p.smem);
  return SB_OK;
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
  int* status = sb::device_status_ptr();
  if (!status) return SB_ERR_CUDA;
  const int n = T * k;
  const size_t most = sb::mf::kMostSmem, lists = sb::mf::lists_bytes(n, E);
  sb::mf::RingPlan gu;
  if (!sb::mf::plan_ring(n, E, H, gu)) return SB_ERR_TOO_LARGE;
  const auto launch = gu.group == 8   ? sb::mf::launch_gate_up<8>
                      : gu.group == 4 ? sb::mf::launch_gate_up<4>
                      : gu.group == 2 ? sb::mf::launch_gate_up<2>
                                      : sb::mf::launch_gate_up<1>;
  cudaError_t e = launch(h, h_stride, idx, wgu, act, T, k, E, H, F, gu.s, gu.smem, most, status, st);
  if (e != cudaSuccess) return SB_ERR_CUDA;
  const size_t once = sb::mf::once_bytes(n, F) + lists;
  if (n <= sb::mf::kOnceUnits && once <= most)
    e = sb::mf::launch_down_once(act, idx, w, wd, out, T, k, E, H, F, once, most, status, st);
  else
    e = sb::mf::launch_down(act, idx, w, wd, out, T, k, E, H, F, sizeof(float) * 16 * static_cast<size_t>(n) + lists, most, st);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

}  // extern "C"
