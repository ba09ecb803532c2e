// Pages of a key-value cache copied to other places, every layer's keys and values in one launch, with the tables that
// name them rewritten beside: page dst[i] := page src[i], table entries equal to src[i] become dst[i].
//
// Bound by memory: each byte once in and once out. A wave copies 4 pieces of 2 KB, all loads before the first store; pieces
// are counted over (layer, keys or values, page), so that few pages are spread over all CUs. The workgroups past the
// copy's do the tables: each holds up to 1024 of the sources at a time in LDS and compares its entries with all of
// them (n comparisons an entry; entries are few beside the bytes of a page).
// 151 MB read and written (48 pages of 64 KB, 12 layers) take 27 us, 1.57 GB 338 us: 5.6 and 4.65 TB/s, where a copy of 2 GiB
// reaches 4.87.
#include <hip/hip_runtime.h>

#include "ss_common.hpp"
#include "ss_launch.hpp"
#include "ss_rope.hpp"

namespace ss {

namespace {

constexpr int kPieces = 4;  // pieces of a wave, of 2 KB (1 KB where a page of bytes has an odd number of them)

// H: KB of a piece. Pages with exponents have workgroups for these behind the tables', a wave for a page and layer.
template <int H>
__global__ __launch_bounds__(256) void move_pages_kernel(MoveArgs a) {
  __shared__ int32_t from[1024], to[1024];
  const int tid = threadIdx.x, lane = tid & 63;
  if (blockIdx.x < a.copy_blocks) {
    // Piece numbers fit 31 bits (the entry point's bound); one division each for a wave's four.
    const uint32_t per = (uint32_t)(a.page_bytes / (1024 * H)), one = per * a.n, all = 2 * one * a.layers;
    const uint32_t first = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(tid >> 6)) * kPieces;
    uint32_t lk = first / one, i = (first - lk * one) / per, in = first - lk * one - i * per;
    uint4 x[kPieces][H];
    uint8_t* dst[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      if (j > 0 && ++in == per) {
        in = 0;
        if (++i == (uint32_t)a.n) {
          i = 0;
          ++lk;
        }
      }
      dst[j] = nullptr;
      if (first + j >= all) continue;
      const int64_t off = (int64_t)in * (1024 * H) + 16 * lane;
      const int32_t s = gp(a.src)[i], d = gp(a.dst)[i];
      if ((uint32_t)s >= (uint64_t)a.n_pages || (uint32_t)d >= (uint64_t)a.n_pages) {
        if (lane == 0) ss_raise(a.err, SS_ERR_PAGE);
        continue;
      }
      uint8_t* base = (lk % 2 ? a.v : a.k) + (lk / 2) * a.n_pages * a.page_bytes + off;
      dst[j] = base + d * a.page_bytes;
      x[j][0] = ldg16(base + s * a.page_bytes);
      if constexpr (H == 2) x[j][H - 1] = ldg16(base + s * a.page_bytes + 1024);
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
      if (dst[j]) {
        stg16(dst[j], x[j][0]);
        if constexpr (H == 2) stg16(dst[j] + 1024, x[j][H - 1]);
      }
    return;
  }
  if (H == 1 && blockIdx.x >= a.copy_blocks + a.table_blocks) {
    const uint32_t at = (blockIdx.x - a.copy_blocks - a.table_blocks) * 4 + (tid >> 6), layer = at / (uint32_t)a.n, i = at - layer * a.n;
    if (layer >= (uint32_t)a.layers) return;
    const int32_t s = gp(a.src)[i], d = gp(a.dst)[i];  // raised by the copy where they are no pages
    if ((uint32_t)s >= (uint64_t)a.n_pages || (uint32_t)d >= (uint64_t)a.n_pages) return;
    uint8_t* base = a.scales + (int64_t)layer * a.n_pages * a.scale_bytes;
    for (int64_t o = 16 * lane; o < a.scale_bytes; o += 1024) stg16(base + d * a.scale_bytes + o, ldg16(base + s * a.scale_bytes + o));
    return;
  }
  const int64_t e = (int64_t)(blockIdx.x - a.copy_blocks) * 256 + tid;
  const bool in = e < a.entries;
  const int32_t old = in ? a.table[e] : -1;
  int32_t now = old;
  bool done = false;
  for (int i0 = 0; i0 < a.n; i0 += 1024) {
    const int m = min(a.n - i0, 1024);
    __syncthreads();
    for (int i = tid; i < m; i += 256) {
      from[i] = gp(a.src)[i0 + i];
      to[i] = gp(a.dst)[i0 + i];
    }
    __syncthreads();
    for (int i = 0; i < m; ++i) {
      const bool hit = !done && from[i] == old;
      now = hit ? to[i] : now;
      done |= hit;
    }
  }
  // an entry of -1 holds no page; a move out of the cache was raised by the copy and is not followed
  if (in && done && (uint32_t)old < (uint64_t)a.n_pages && (uint32_t)now < (uint64_t)a.n_pages) a.table[e] = now;
}

}  // namespace

hipError_t launch_move_pages(MoveArgs a, hipStream_t st) {
  const int64_t pieces = 2 * (a.page_bytes / (a.scales ? 1024 : 2048)) * a.n * a.layers;
  a.copy_blocks = (unsigned)((pieces + 4 * kPieces - 1) / (4 * kPieces));
  a.table_blocks = a.table ? (unsigned)((a.entries + 255) / 256) : 0;
  a.scale_blocks = a.scales ? (unsigned)(((int64_t)a.n * a.layers + 3) / 4) : 0;
  const dim3 grid(a.copy_blocks + a.table_blocks + a.scale_blocks);
  if (grid.x == 0) return hipSuccess;
  if (a.scales)
    hipLaunchKernelGGL(move_pages_kernel<1>, grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL(move_pages_kernel<2>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ss
