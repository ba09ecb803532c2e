// Rotary positions with several axes, and the cache write of the rows they turn.
//
// Row r, frequency i (of rot / 2): angle = positions[axis[i]][r] * inv_freq[i]; the elements (i, i + rot / 2) of a head, or
// (2 i, 2 i + 1) with `adjacent`, are turned by it: (a cos - b sin, b cos + a sin). Elements from rot on stay. Angles are
// reduced to a part of a turn in 64 bits: a position of 100,000 at inv_freq 1 leaves 7 bits of a turn's fraction in 32.
//
// A workgroup has 8 positions (from a multiple of 8) of one sequence and some of the heads. Its threads work the angles out once,
// into LDS, and each wave turns its heads, a thread 8 frequencies of a row in each; the value rows are read as 8
// rows by 8 dimensions and transposed in registers into the cache's token-contiguous order, 16 bytes per dimension where
// all 8 tokens are the call's, single values at the ends.
//
// Bound by memory on prompts: 8,190 rows of 16 + 2 + 2 heads of 256 dimensions, a quarter of them turned by three axes, 168 MB
// in 39 us from memory (4.3 TB/s; a copy reaches 4.9); 64 single tokens of 32 + 4 + 4 heads of 128 take 6 to 7 us, most of it
// the chain of a row's place, its page, its angles and its rows. With every wave working out its own angles 8.8.
#include <hip/hip_runtime.h>

#include "ss_attn.hpp"
#include "ss_launch.hpp"
#include "ss_rope.hpp"

namespace ss {

namespace {

template <class T>
__global__ __launch_bounds__(256) void rope_append_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cs_of[8 * 128], sn_of[8 * 128];  // [8 positions][rot / 2]
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups are dealt to the 8 XCDs in turn; each XCD takes a run of neighbours, whose 16-byte parts of a line of values then
  // meet in one L2 (8,190 rows of 40 heads of 128: 53 us in launch order, 49 so; 64 sequences of 4 rows 10.2 and 9.3; 8,190 rows
  // of 18 heads of 256 38 and 38).
  const uint32_t xcd = blockIdx.x % 8, even = gridDim.x / 8, more = gridDim.x % 8;
  uint32_t b = xcd * even + min(xcd, more) + blockIdx.x / 8;
  const int hg = b % (uint32_t)a.head_groups;
  b /= (uint32_t)a.head_groups;
  const int tile = b % (uint32_t)a.tiles, s = b / (uint32_t)a.tiles;
  const int page = 1 << a.page_shift;
  const int64_t cap = (int64_t)a.width * page;
  const SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, cap, a.err);
  // Positions [first, first + 8) of the cache; rows that the cache is too short for begin below 0.
  const int base = sr.pos0 >= 0 ? sr.pos0 & ~7 : -((-sr.pos0 + 7) & ~7);
  const int first = base + 8 * tile;
  if (first >= sr.pos0 + sr.n) return;
  const int half = a.rot / 2, chunks = a.rot / 16;
  const int D = a.dim;

  // Where each of the 8 positions' tokens go; all 8 share a page (a page is a multiple of 8).
  int id = -1;
  if (first >= 0 && first < cap) {
    id = gp(a.table)[(int64_t)s * a.width + (first >> a.page_shift)];
    if ((uint32_t)id >= (uint64_t)a.n_pages) {
      id = -1;
      if (tid == 0) raise_bit(a.err, SS_ERR_PAGE);
    }
  }
  const int off = first & (page - 1);
  const int stride = 4 * a.head_groups, h0 = 4 * hg + w;  // this wave's heads: h0, h0 + stride, ...

  for (int it = tid; it < 8 * half; it += 256) {
    const int rr = (uint32_t)it / (uint32_t)half, f = it - rr * half, row = first + rr - sr.pos0;
    if (row < 0 || row >= sr.n) continue;
    const int ax = a.axis ? gp(a.axis)[f] : 0;
    int p = 0;
    if ((uint32_t)ax < (uint32_t)a.axes)
      p = gp(a.positions)[ax * a.pos_stride + sr.r0 + row];
    else
      raise_bit(a.err, SS_ERR_BATCH);
    const double turns = (double)p * (gp(a.inv_freq)[f] * 0.15915494309189533577);
    float sn, cs;
    sincospif(2.f * (float)(turns - __builtin_rint(turns)), &sn, &cs);
    cs_of[it] = cs * a.factor;
    sn_of[it] = sn * a.factor;
  }
  __syncthreads();

  // Query heads, then key heads; a thread's loads for some of its heads go out together.
  const int hs = a.heads + a.kv_heads;
  auto from = [&](int64_t r, int h) {
    return h < a.heads ? a.q + r * a.q_row + h * a.q_head : a.k + r * a.k_row + (h - a.heads) * a.k_head;
  };
  auto to = [&](int64_t r, int h, int rr) {
    return h < a.heads ? a.out + (r * a.heads + h) * D
                       : a.k_pages + (((int64_t)id * a.kv_heads + (h - a.heads)) * page + off + rr) * D;
  };
  // Turned elements: items of (row, 8 frequencies).
  for (int it = lane; it < 8 * chunks; it += 64) {
    const int rr = (uint32_t)it / (uint32_t)chunks, j = it - rr * chunks, row = first + rr - sr.pos0;
    if (row < 0 || row >= sr.n) continue;
    const int64_t r = sr.r0 + row;
    ss_f32x4 cv[2], sv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      cv[e] = *reinterpret_cast<const ss_f32x4*>(&cs_of[8 * it + 4 * e]);
      sv[e] = *reinterpret_cast<const ss_f32x4*>(&sn_of[8 * it + 4 * e]);
    }
    float cs[8], sn[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      cs[e] = cv[e / 4][e % 4];
      sn[e] = sv[e / 4][e % 4];
    }
    const int o0 = a.adjacent ? 16 * j : 8 * j, o1 = a.adjacent ? 16 * j + 8 : half + 8 * j;
    for (int ha = h0; ha < hs; ha += 2 * stride) {
      ss_u32x4 x0[2], x1[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (ha + u * stride < hs) {
          const uint16_t* src = from(r, ha + u * stride);
          x0[u] = *(const SS_G ss_u32x4*)(src + o0);
          x1[u] = *(const SS_G ss_u32x4*)(src + o1);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int h = ha + u * stride;
        if (h >= hs || (h >= a.heads && id < 0)) break;
        ss_u32x4 y0, y1;
        if (a.adjacent) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = T::widen(x0[u][e] & 0xFFFFu), p1 = T::widen(x0[u][e] >> 16);
            const float q0 = T::widen(x1[u][e] & 0xFFFFu), q1 = T::widen(x1[u][e] >> 16);
            y0[e] = T::pack(p0 * cs[e] - p1 * sn[e], p1 * cs[e] + p0 * sn[e]);
            y1[e] = T::pack(q0 * cs[4 + e] - q1 * sn[4 + e], q1 * cs[4 + e] + q0 * sn[4 + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = T::widen(x0[u][e] & 0xFFFFu), p1 = T::widen(x0[u][e] >> 16);
            const float q0 = T::widen(x1[u][e] & 0xFFFFu), q1 = T::widen(x1[u][e] >> 16);
            y0[e] = T::pack(p0 * cs[2 * e] - q0 * sn[2 * e], p1 * cs[2 * e + 1] - q1 * sn[2 * e + 1]);
            y1[e] = T::pack(q0 * cs[2 * e] + p0 * sn[2 * e], q1 * cs[2 * e + 1] + p1 * sn[2 * e + 1]);
          }
        }
        uint16_t* dst = to(r, h, rr);
        *(SS_G ss_u32x4*)(dst + o0) = y0;
        *(SS_G ss_u32x4*)(dst + o1) = y1;
      }
    }
  }
  // Elements past rot, as they are.
  const int rest = (D - a.rot) / 8;
  for (int it = lane; it < 8 * rest; it += 64) {
    const int rr = (uint32_t)it / (uint32_t)rest, o = a.rot + 8 * (it - rr * rest), row = first + rr - sr.pos0;
    if (row < 0 || row >= sr.n) continue;
    const int64_t r = sr.r0 + row;
    for (int ha = h0; ha < hs; ha += 4 * stride) {
      ss_u32x4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (ha + u * stride < hs) x[u] = *(const SS_G ss_u32x4*)(from(r, ha + u * stride) + o);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int h = ha + u * stride;
        if (h >= hs || (h >= a.heads && id < 0)) break;
        *(SS_G ss_u32x4*)(to(r, h, rr) + o) = x[u];
      }
    }
  }
  // Value rows.
  if (id < 0) return;
  const int lo = max(sr.pos0 - first, 0), hi = min(sr.pos0 + sr.n - first, 8);  // the call's tokens of the 8
  const int per = D / 8;
  for (int it = 64 * h0 + lane; it < per * a.kv_heads; it += 64 * stride) {
    const int h = it / per, d = 8 * (it - h * per);
    ss_u32x4 x[8];
#pragma unroll
    for (int rr = 0; rr < 8; ++rr) {
      x[rr] = ss_u32x4{0u, 0u, 0u, 0u};
      if (rr >= lo && rr < hi)
        x[rr] = *(const SS_G ss_u32x4*)(a.v + (int64_t)(sr.r0 + first + rr - sr.pos0) * a.v_row + h * a.v_head + d);
    }
    uint16_t* dst = a.v_pages + (((int64_t)id * a.kv_heads + h) * D + d) * page + off;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ss_u32x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u0 = x[2 * i][e / 2], u1 = x[2 * i + 1][e / 2];
        y[i] = e % 2 ? (u0 >> 16) | (u1 & 0xFFFF0000u) : (u0 & 0xFFFFu) | (u1 << 16);
      }
      if (lo == 0 && hi == 8) {
        *(SS_G ss_u32x4*)(dst + (int64_t)e * page) = y;
      } else {
#pragma unroll
        for (int rr = 0; rr < 8; ++rr)
          if (rr >= lo && rr < hi) gp(dst)[(int64_t)e * page + rr] = (uint16_t)(rr % 2 ? y[rr / 2] >> 16 : y[rr / 2]);
      }
    }
  }
}

}  // namespace

hipError_t launch_rope_append(const RopeArgs& a, bool fp16, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.seqs * a.tiles * a.head_groups));
  if (fp16)
    hipLaunchKernelGGL((rope_append_kernel<Fp16>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((rope_append_kernel<Bf16>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ss
