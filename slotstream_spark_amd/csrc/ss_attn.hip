// Attention of few rows: the kernels over 16-bit pages with causal rows, the launch that joins chunks and the choice of the
// packed rows. The kernel itself is in ss_attn_few.hpp.
#include <hip/hip_runtime.h>

#include "ss_attn_few.hpp"

namespace ss {

namespace {

// Joins the chunks of a row: o = sum_k o_k 2^(m_k - m) / sum_k l_k 2^(m_k - m), m the largest m_k. A row and head is read by
// groups of dim / 4 threads, 16 bytes each. WIDE: its workgroup's groups take the chunks by their number modulo the
// number of groups, each with a running maximum, and the groups' sums are added in order; else one group takes all its
// chunks and a workgroup has as many rows. Either way the order goes by the chunks' numbers alone.
// EXT: calls of trees or with shared chunks. DEEP: a group's loads of eight chunks go out together, those past its last one anew.
template <class T, int D, bool WIDE, bool EXT, bool DEEP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  constexpr int TD = D / 4, GROUPS = 256 / TD, STEP = WIDE ? GROUPS : 1;
  __shared__ __attribute__((aligned(16))) float part[WIDE ? GROUPS : 1][D];
  __shared__ float part_l[GROUPS], part_m[GROUPS];
  const int tid = threadIdx.x, d4 = 4 * (tid % TD), k = tid / TD;
  const uint32_t all = (uint32_t)a.seqs * a.max_rows * a.heads;  // below 2^31
  uint32_t b = WIDE ? blockIdx.x : blockIdx.x * GROUPS + k;
  if (b >= all) return;
  const int head = (int)(b % (uint32_t)a.heads);
  b /= (uint32_t)a.heads;
  const int i = (int)(b % (uint32_t)a.max_rows), s = (int)(b / (uint32_t)a.max_rows);
  const SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, (int64_t)a.width << a.page_shift, nullptr);
  if (i >= sr.n) return;
  // The slots of the workgroup that had this row, as it counted them.
  const int tile = (i * a.group + head % a.group) / a.packed, p0 = tile * a.packed, np = sr.n * a.group;
  const bool tree = EXT && a.tree, share = EXT && a.share > 0;
  const int lo = tree ? 0 : p0 / a.group, hi = tree ? sr.n - 1 : (min(p0 + a.packed, np) - 1) / a.group;
  const Seen sn = seen_tokens(sr.pos0 + lo, sr.pos0 + hi, sr.end, a.window, a.sinks);
  const int chunk = share ? 64 * gp(a.meta)[0] : a.chunk;
  const int sc = (sn.s_end + chunk - 1) / chunk, wc = max(sn.w_begin / chunk, sc);
  const int used = sc + max((EXT ? (int)(((int64_t)sn.end + chunk - 1) / chunk) : (sn.end + chunk - 1) / chunk) - wc, 0);
  const int64_t row = (int64_t)(sr.r0 + i) * a.heads + head;
  // Where the row's partial sums begin and how far those of the next chunk are.
  const int64_t rows = share ? (int64_t)((np + 127) / 128) * a.kv_heads * 128 : (int64_t)a.rows * a.heads;
  int64_t first = row;
  if (share)
    first = ((int64_t)(gp(a.meta)[1 + s] + tile) * a.kv_heads + head / a.group) * 128 + (i * a.group + head % a.group) % 128;
  ss_f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float m = kNegInf, l = 0.f;
  auto add = [&](const ss_f32x4& x, float mk, float lk) {
    const float mn = fmaxf(m, mk), mu = mn == kNegInf ? 0.f : mn;
    const float f = m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - mu), fk = mk == kNegInf ? 1.f : __builtin_amdgcn_exp2f(mk - mu);
    m = mn;
    l = l * f + lk * fk;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * f + x[e] * fk;
  };
  auto take = [&](int from, int to) {
#pragma unroll 4
    for (int j = from; j < to; j += STEP) {
      const int64_t at = j * rows + first;
      const float mk = gp(a.pml)[2 * at], lk = gp(a.pml)[2 * at + 1];
      const ss_f32x4 x = *reinterpret_cast<const SS_G ss_f32x4*>(gp(a.po) + at * D + d4);
      add(x, mk, lk);
    }
  };
  if constexpr (WIDE) {
    // Slot j holds chunk j (first tokens) or chunk wc + j - sc: group k takes the chunks k, k + GROUPS, ...
    take(k, sc);
    take(sc + (k + GROUPS - wc % GROUPS) % GROUPS, used);
    *reinterpret_cast<ss_f32x4*>(&part[k][d4]) = o;
    if (d4 == 0) {
      part_m[k] = m;
      part_l[k] = l;
    }
    __syncthreads();
    if (k > 0) return;
    m = kNegInf;
    l = 0.f;
    o = ss_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) add(*reinterpret_cast<const ss_f32x4*>(&part[j][d4]), part_m[j], part_l[j]);
  } else if constexpr (DEEP) {
    constexpr int U = 8;
    for (int j = 0; j < used; j += U) {
      float mk[U], lk[U];
      ss_f32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = min(j + u, used - 1) * rows + first;
        mk[u] = gp(a.pml)[2 * at];
        lk[u] = gp(a.pml)[2 * at + 1];
        x[u] = *reinterpret_cast<const SS_G ss_f32x4*>(gp(a.po) + at * D + d4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (j + u < used) add(x[u], mk[u], lk[u]);
    }
  } else {
    take(0, used);
  }
  const float r = l == 0.f ? 0.f : 1.f / l;
  uint2 word;
  word.x = T::pack(o[0] * r, o[1] * r);
  word.y = T::pack(o[2] * r, o[3] * r);
  *reinterpret_cast<uint2*>(a.out + row * D + d4) = word;
  if (a.lse && d4 == 0) a.lse[row] = l == 0.f ? kNegInf : (m + __log2f(l)) * 0.693147180559945309f;
}

// More than 16 chunks are joined by a workgroup a row: one row and 32 heads over 12,000 tokens 12.3 us a call with it, 18.9
// without, over 51,000 24.4 and 39.8. Up to 16, where a batch brings the rows, by a group of threads a row: 32 sequences of 4
// rows and 32 heads 186 us a call, 191 with a workgroup each.
// Where those are at most a wave for each SIMD of 256 CUs, eight chunks are loaded at a time: then no other wave's loads fill the time. A call in us,
// so and without: one token after 777 8.8 and 9.2, a tree of 12 rows over 777 14.8 and 15.2, 8 sequences of 3 rows of 256 dimensions
// 24.4 and 24.8; but 3 prompts of 333 rows 84.5 and 82.6, 16 trees of 26 rows 64.1 and 63.6.
template <class T, int D, bool EXT>
hipError_t launch_join(const AttnArgs& a, hipStream_t st) {
  const int64_t all = (int64_t)a.seqs * a.max_rows * a.heads;
  constexpr int GROUPS = 256 / (D / 4);
  const dim3 rows((unsigned)((all + GROUPS - 1) / GROUPS));
  if ((a.share > 0 ? a.slots / ((int64_t)a.seqs * a.tiles) : a.slots) > 16)  // of shared chunks as many as a row has if all are alike
    hipLaunchKernelGGL((attn_join_kernel<T, D, true, EXT, false>), dim3((unsigned)all), dim3(256), 0, st, a);
  else if (rows.x <= 256)
    hipLaunchKernelGGL((attn_join_kernel<T, D, false, EXT, true>), rows, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_join_kernel<T, D, false, EXT, false>), rows, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <class T, bool EXT>
hipError_t launch_join_of(const AttnArgs& a, int dim, hipStream_t st) {
  return dim == 64 ? launch_join<T, 64, EXT>(a, st) : dim == 128 ? launch_join<T, 128, EXT>(a, st) : launch_join<T, 256, EXT>(a, st);
}

}  // namespace

// Packed rows of a workgroup: as few tiles of 16 as hold them all, up to 4 (2 of 256 dimensions, whose sums of four tiles
// would take every register, and of 128 in e4m3, whose tiles have twice the tokens).
int attn_few_packed(int dim, int packed, bool e4m3) {
  if (packed <= 16) return 16;
  return packed <= 32 || dim == 256 || (e4m3 && dim == 128) ? 32 : 64;
}

hipError_t launch_attn_few(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_few_of<Fp16, false, false>(a, dim, st) : launch_few_of<Bf16, false, false>(a, dim, st);
}

hipError_t launch_attn_join(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  if (a.tree || a.share > 0) return fp16 ? launch_join_of<Fp16, true>(a, dim, st) : launch_join_of<Bf16, true>(a, dim, st);
  return fp16 ? launch_join_of<Fp16, false>(a, dim, st) : launch_join_of<Bf16, false>(a, dim, st);
}

}  // namespace ss
