// Row layout of a packed prefill batch from request lengths and block tables: sequence offsets, positions and cache slots.
//
// Sequence b contributes its tokens start_b .. len_b - 1, one row each, in order:
//   cu[b + 1] = cu[b] + max(len_b - start_b, 0)
//   row r of sequence b:  pos = start_b + (r - cu[b]),  slot = table[b][pos / bs] * bs + pos % bs,
//                         whole = sum of the lengths before b + pos   (its row in the layout of the whole sequences)
// Rows behind the last sequence get pos 0, slot -1, whole -1.
//
// 12 bytes written a row, a table entry read per block: bound by launch and latency at serving sizes.  One launch: a CTA
// belongs to one sequence and sums the lengths before it itself (the lengths of a batch are a few KB and stay in L2),
// so no scan kernel, workspace or flag is needed; more CTAs share a sequence when the rows are many.
#include "host_common.h"
#include "ptx.cuh"

namespace sb {

constexpr int kLayoutThreads = 256;

__device__ __forceinline__ long long layout_block_sum(long long v, long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  long long t = 0;
#pragma unroll
  for (int i = 0; i < kLayoutThreads / 32; ++i) t += red[i];
  __syncthreads();
  return t;
}

__global__ void __launch_bounds__(kLayoutThreads)
paged_layout_kernel(const int* tables, long long table_stride, int width, const int* starts, const int* lens, int B, int bs,
                    int total, int* __restrict__ cu, int* __restrict__ pos, int* __restrict__ slots, int* __restrict__ whole) {
  __shared__ long long red[kLayoutThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;  // B: the rows behind the last sequence
  long long rows = 0, tokens = 0;
  for (int i = threadIdx.x; i < b; i += kLayoutThreads) {
    const int n = max(lens[i], 0), s = starts ? min(max(starts[i], 0), n) : 0;
    rows += n - s;
    tokens += n;
  }
  rows = layout_block_sum(rows, red);
  if (threadIdx.x == 0 && blockIdx.y == 0) cu[b] = static_cast<int>(rows);
  const long long step = static_cast<long long>(gridDim.y) * kLayoutThreads;
  const long long first = static_cast<long long>(blockIdx.y) * kLayoutThreads + threadIdx.x;
  if (b == B) {
    for (long long r = rows + first; r < total; r += step) {
      pos[r] = 0;
      slots[r] = -1;
      whole[r] = -1;
    }
    return;
  }
  tokens = layout_block_sum(tokens, red);
  const int n = max(lens[b], 0), s = starts ? min(max(starts[b], 0), n) : 0;
  const int* table = tables + b * table_stride;
  for (long long r = first; r < n - s; r += step) {
    if (rows + r >= total) break;
    const int p = s + static_cast<int>(r);
    const int blk = p / bs;
    const int e = blk < width ? table[blk] : -1;
    const long long slot = e >= 0 ? static_cast<long long>(e) * bs + (p - blk * bs) : -1;
    pos[rows + r] = p;
    slots[rows + r] = slot > 0x7fffffffLL ? -1 : static_cast<int>(slot);
    whole[rows + r] = static_cast<int>(tokens + p);
  }
}

}  // namespace sb

extern "C" {

// tables [B, width] with row stride table_stride; starts may be null (all zero); cu [B + 1]; pos, slots, whole [total].
int sb_paged_layout(const int* tables, long long table_stride, int width, const int* starts, const int* lens, int B, int bs,
                    int total, int* cu, int* pos, int* slots, int* whole, void* stream) {
  if (B < 0 || bs <= 0 || total < 0 || width < 0) return SB_ERR_ARG;
  // about 1024 rows a CTA when the lengths are even; a single long sequence among short ones gets at most 64 CTAs
  long long y = 1 + 2LL * total / (1024LL * (B + 1));
  if (y > 64) y = 64;
  const cudaError_t e = sb::launch_pdl(sb::paged_layout_kernel, dim3(B + 1, static_cast<unsigned>(y)), dim3(sb::kLayoutThreads), 0,
                                       reinterpret_cast<cudaStream_t>(stream), tables, table_stride, width, starts, lens, B, bs,
                                       total, cu, pos, slots, whole);
  return e == cudaSuccess ? SB_OK : SB_ERR_CUDA;
}

}  // extern "C"
