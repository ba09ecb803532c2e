// Around a tree of drafted tokens: which rows a row sees, how far the target's choices go along it, and the accepted branch's
// keys and values moved to where the next round expects them.
//
// A sequence's tree is its rows of the call, row 0 the pending token, every other row behind its parent. At most 64 rows, so
// that a set of rows is a 64-bit word.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ss_attn.hpp"
#include "ss_common.hpp"
#include "ss_launch.hpp"
#include "ss_tree.hpp"

namespace ss {

namespace {

// Rows [r0, r0 + n) of sequence s, cut to the arguments (raised).
struct TreeRows {
  int r0, n;
};
SS_DEV TreeRows tree_rows(const int32_t* cu, int s, int rows, int max_rows, int* err) {
  const int a = gp(cu)[s], b = gp(cu)[s + 1];
  TreeRows r;
  r.r0 = min(max(a, 0), rows);
  const int e = min(b, rows);
  r.n = min(e > r.r0 ? e - r.r0 : 0, max_rows);
  if ((a < 0 || b < a || b > rows || b - a > max_rows) && threadIdx.x == 0) raise_bit(err, SS_ERR_BATCH);
  return r;
}

// A wave a sequence, a lane a row. mask_i = 2^i | mask_parent: by doubling, a row's word first has itself, then itself and its
// parent, then four ... (rows never reach past 2^6 steps). A parent that is not a row before it is none, and raised.
__global__ __launch_bounds__(64) void tree_masks_kernel(TreeMaskArgs a) {
  __shared__ uint64_t word[kTreeRows];
  __shared__ int up[kTreeRows];
  const int i = threadIdx.x, s = blockIdx.x;
  const TreeRows r = tree_rows(a.cu, s, a.rows, a.max_rows, a.err);
  int p = -1;
  if (i > 0 && i < r.n) {
    p = gp(a.parents)[r.r0 + i];
    if (p < 0 || p >= i) {
      p = -1;
      raise_bit(a.err, SS_ERR_BATCH);
    }
  }
  uint64_t m = 1ull << i;
  for (int step = 0; step < 6; ++step) {
    word[i] = m;
    up[i] = p;
    __syncthreads();
    if (p >= 0) {
      m |= word[p];
      p = up[p];
    }
    __syncthreads();
  }
  if (i < r.n) {
    a.masks[r.r0 + i] = m;
    if (a.positions) {
      const int len = max(gp(a.kv_len)[s], 0), all = max(gp(a.cu)[s + 1] - gp(a.cu)[s], 0);
      a.positions[r.r0 + i] = len - all + __builtin_popcountll(m) - 1;
    }
  }
}

// The largest value of a span of a row: the higher word its key, the lower one the complement of its place, so that the maximum
// of such words is the largest value's first place; all ones where the span has a value that is not finite.
// Bound by memory: each logit is read once, 16 bytes a lane, four loads in flight; rows are cut in spans so that few of them fill the chip.
// 261 rows of 248,320 logits (259 MB) take 48 us, 5.4 TB/s; 12 of 151,936 3.9.
__global__ __launch_bounds__(256) void tree_argmax_kernel(TreeAcceptArgs a) {
  __shared__ uint64_t best[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / (uint32_t)a.splits, sp = blockIdx.x - row * a.splits;
  const float* x = a.target + (int64_t)row * a.vocab;
  const int from = sp * a.span, to = min(from + a.span, a.vocab);
  uint32_t top = 0, bad = 0;  // every value's key is above 0 but NaN's
  int at = 0;
  auto take = [&](float v, int i) {
    const uint32_t k = ss_key(v + 0.f);  // -0 is as large as 0
    bad |= (ss_fu(v) & 0x7F800000u) == 0x7F800000u;
    if (k > top) {
      top = k;
      at = i;
    }
  };
  // up to three values before the first 16-byte place, then whole pieces, then the rest
  const int skew = (int)((0 - (reinterpret_cast<uintptr_t>(x + from) >> 2)) & 3u), body = from + min(skew, to - from);
  if (from + tid < body) take(gp(x)[from + tid], from + tid);
  const int pieces = (to - body) / 4;
  int p = tid;
  for (; p + 768 < pieces; p += 1024) {
    ss_f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *(const SS_G ss_f32x4*)(x + body + 4 * (p + 256 * u));
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) take(v[u][e], body + 4 * (p + 256 * u) + e);
  }
  for (; p < pieces; p += 256) {
    const ss_f32x4 v = *(const SS_G ss_f32x4*)(x + body + 4 * p);
#pragma unroll
    for (int e = 0; e < 4; ++e) take(v[e], body + 4 * p + e);
  }
  const int tail = body + 4 * pieces + tid;
  if (tail < to) take(gp(x)[tail], tail);
  uint64_t word = bad ? ~0ull : (uint64_t)top << 32 | (uint32_t)~at;
  word = ss_wave_max_u64(word);
  if (lane == 0) best[w] = word;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < 4; ++i) word = word > best[i] ? word : best[i];
    a.part[(int64_t)row * a.splits + sp] = word;
  }
}

// A workgroup a sequence: sixteen threads a row join its spans, then one wave walks the tree: from row 0, to the first row behind the
// present one whose token is the present one's choice.
// Bound by latency, a turn of the walk is a ballot and some 20 instructions: 2.6 us for a sequence, 4.6 for 16 of up to 26 rows.
__global__ __launch_bounds__(1024) void tree_walk_kernel(TreeAcceptArgs a) {
  __shared__ uint64_t best[kTreeRows];
  const int tid = threadIdx.x, s = blockIdx.x;
  const TreeRows r = tree_rows(a.cu, s, a.rows, a.max_rows, a.err);
  int p = -1, tok = -1;
  if (tid > 0 && tid < r.n) {
    p = gp(a.parents)[r.r0 + tid];
    tok = gp(a.tokens)[r.r0 + tid];
  }
  {
    const int i = tid / 16;
    uint64_t word = 0;
    if (i < r.n) {
      const uint64_t* part = a.part + (int64_t)(r.r0 + i) * a.splits;
      for (int j = tid % 16; j < a.splits; j += 64) {  // four loads at a time; a span that is none is the first one again
        uint64_t o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) o[u] = gp(part)[j + 16 * u < a.splits ? j + 16 * u : 0];
#pragma unroll
        for (int u = 0; u < 4; ++u) word = o[u] > word ? o[u] : word;
      }
    }
    auto other = [&](uint64_t v, uint32_t hi, uint32_t lo) {
      const uint64_t o = (uint64_t)hi << 32 | lo;
      return o > v ? o : v;
    };
    word = other(word, ss_xor_lane<1>((uint32_t)(word >> 32)), ss_xor_lane<1>((uint32_t)word));
    word = other(word, ss_xor_lane<2>((uint32_t)(word >> 32)), ss_xor_lane<2>((uint32_t)word));
    word = other(word, ss_xor_lane<4>((uint32_t)(word >> 32)), ss_xor_lane<4>((uint32_t)word));
    word = other(word, ss_xor_lane<8>((uint32_t)(word >> 32)), ss_xor_lane<8>((uint32_t)word));
    if (tid % 16 == 0) best[i] = word;
  }
  __syncthreads();
  if (tid >= 64) return;
  const int i = tid;
  if (i > 0 && i < r.n && (p < 0 || p >= i)) {
    p = -1;
    raise_bit(a.err, SS_ERR_BATCH);
  }
  const uint64_t mine = i < r.n ? best[i] : 0;
  const bool fine = mine != ~0ull;
  const int choice = (int)~(uint32_t)mine;
  int cur = 0, depth = 0, emit = 0, flags = 0, my_tok = -1, my_row = -1;
  while (depth < r.n) {  // every turn goes to a later row
    if (i == depth) my_row = cur;
    const int t = __builtin_amdgcn_readlane(choice, cur);
    if (!__builtin_amdgcn_readlane((int)fine, cur)) {
      flags = 1;
      break;
    }
    if (i == depth) my_tok = t;
    ++emit;
    const uint64_t next = __ballot(p == cur && tok == t);
    if (!next) break;
    cur = __builtin_ctzll(next);
    ++depth;
  }
  int32_t* out = a.out + (int64_t)s * (4 + 2 * a.max_rows);
  if (i < 4) out[i] = i == 0 ? depth : i == 1 ? emit : i == 2 ? 0 : flags;
  if (i < a.max_rows) {
    out[4 + i] = my_tok;
    out[4 + a.max_rows + i] = my_row;
  }
}

// Token base + d takes the row path[d]. Paths rise, so every source lies at or behind its place. A thread has one of three kinds of
// parts of a layer and key head, and no two share any:
//   a dimension of the values: 8 tokens at multiples of 8 are a piece of 8 or 16 bytes, which is read whole, gets the moved tokens'
//     elements and is written whole (the others as they were): stores of single elements are as many requests as elements;
//   16 bytes of the keys, or a byte of the exponents, of each token: eight loads before eight stores.
// Either way pieces and tokens go by their order, so nothing is written over that is yet to be read. A workgroup works a sequence's
// branch out once and takes parts of all layers and key heads; a wave's parts are of one kind.
// Bound by latency for one sequence (48 layers of 4 key heads 4.5 us), and by the lines of the values, of which an element a token is
// moved: 32 sequences of 48 layers, 8 key heads, 128 dimensions of e4m3 and pages of 64 tokens read 119 MB of lines and write 56 MB, of
// 32 bytes at least each, in 50 us (stored an element at a time 57).
template <class V, bool E8>
__global__ __launch_bounds__(256) void keep_rows_kernel(KeepArgs a) {
  constexpr int EV = 16 / sizeof(V), W = 2 * sizeof(V);  // elements of 16 bytes; words of 8 elements
  constexpr int kPieces = kTreeRows / 8 + 1;
  __shared__ int64_t src[kTreeRows], dst[kTreeRows];  // page and token in it: page << 8 | token
  // Of the values' pieces that hold the branch: element places in a dimension's pages of what their tokens take (-1: stay), the
  // pieces' own and the bits of the tokens that move.
  __shared__ __attribute__((aligned(16))) int64_t take[8 * kPieces], into[kPieces];
  __shared__ uint32_t moved[kPieces][W];
  __shared__ int count;
  const int tid = threadIdx.x, page = 1 << a.page_shift;
  const int s = blockIdx.x / (uint32_t)a.blocks, block = blockIdx.x - s * a.blocks;
  const int64_t cap = (int64_t)a.width * page, one = (int64_t)a.kv_heads * page * a.dim;  // `one`: elements of a page
  const SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, cap, a.err);
  const int32_t* took = a.took + (int64_t)s * (4 + 2 * a.max_rows);
  const int skew = sr.pos0 & 7;  // of the first row in its piece
  if (tid < 8 * kPieces) take[tid] = -1;
  if (tid < kPieces) {
    into[tid] = -1;
    for (int i = 0; i < W; ++i) moved[tid][i] = 0;
  }
  __syncthreads();
  if (tid < 64) {
    const int kept = gp(took)[0] + 1;
    int at = tid < a.max_rows ? gp(took)[4 + a.max_rows + tid] : -1;
    if (tid >= kept) at = -1;
    int before = __shfl_up(at, 1);
    if (tid == 0) before = -1;
    // the branch as far as its rows rise and exist
    const bool good = tid < kept && at > before && at < sr.n;
    const uint64_t all = __ballot(good);
    const int n = all == ~0ull ? 64 : __builtin_ctzll(~all);
    if (tid == 0) {
      count = n;
      if (sr.n > 0 && n < kept) raise_bit(a.err, SS_ERR_BATCH);
    }
    if (tid < n) {
      auto place = [&](int t) {
        int id = -1;
        if (t >= 0 && t < cap) {
          id = gp(a.table)[(int64_t)s * a.width + (t >> a.page_shift)];
          if ((uint32_t)id >= (uint64_t)a.n_pages) {
            id = -1;
            raise_bit(a.err, SS_ERR_PAGE);
          }
        }
        return id < 0 ? (int64_t)-1 : (int64_t)id << 8 | (t & (page - 1));
      };
      const int64_t x = at == tid ? -1 : place(sr.pos0 + at), y = at == tid ? -1 : place(sr.pos0 + tid);
      const bool moves = x >= 0 && y >= 0;  // rows in their places, or without one, stay
      src[tid] = moves ? x : -1;
      dst[tid] = y;
      if (moves) {
        const int j = skew + tid;
        take[j] = (x >> 8) * one + (x & 255);
        into[j / 8] = (y >> 8) * one + (y & 255 & ~7);  // the same of every token of the piece
        atomicOr(&moved[j / 8][j % 8 * sizeof(V) / 4], (E8 ? 0xFFu : 0xFFFFu) << (8 * (j * sizeof(V) % 4)));
      }
    }
  }
  __syncthreads();
  const int n = __builtin_amdgcn_readfirstlane(count), last = n > 0 ? (skew + n - 1) / 8 : -1;
  auto values = [&](V* base) {
    for (int b = 0; b <= last; ++b) {
      const int64_t to = into[b];
      if (__builtin_amdgcn_readfirstlane((int)(to >> 32)) < 0) continue;
      uint32_t x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t from = take[8 * b + u];
        x[u] = 0;
        if (__builtin_amdgcn_readfirstlane((int)(from >> 32)) >= 0) x[u] = gp(base)[from];
      }
      typedef uint32_t Piece __attribute__((ext_vector_type(W)));
      SS_G Piece* const at = (SS_G Piece*)(base + to);
      Piece w = *at;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint32_t m = moved[b][i];
        const uint32_t v = E8 ? x[4 * i % 8] | x[(4 * i + 1) % 8] << 8 | x[(4 * i + 2) % 8] << 16 | x[(4 * i + 3) % 8] << 24
                              : x[2 * i % 8] | x[(2 * i + 1) % 8] << 16;
        w[i] = (w[i] & ~m) | v;
      }
      *at = w;
    }
  };
  // `base`: the part's first element in the layer; elements of a page and of a token of its kind
  auto move = [&](auto* base, int64_t per_page, int64_t per_token) {
    typedef typename std::remove_reference<decltype(*base)>::type E;
    for (int d0 = 0; d0 < n; d0 += 8) {
      E x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (d0 + u < n && src[d0 + u] >= 0) x[u] = *(const SS_G E*)(base + (src[d0 + u] >> 8) * per_page + (src[d0 + u] & 255) * per_token);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (d0 + u < n && src[d0 + u] >= 0) *(SS_G E*)(base + (dst[d0 + u] >> 8) * per_page + (dst[d0 + u] & 255) * per_token) = x[u];
    }
  };
  // Numbers of parts fit 31 bits (the entry point's bound).
  const uint32_t units = (uint32_t)(a.layers * a.kv_heads), nv = units * a.dim, kpieces = a.dim / EV, nk = units * kpieces;
  const uint32_t all = nv + (nk + 63) / 64 * 64 + (E8 ? 2 * units : 0);
  auto first = [&](uint32_t unit) {  // element of the unit's first page
    const uint32_t layer = unit / (uint32_t)a.kv_heads, h = unit - layer * a.kv_heads;
    return (int64_t)layer * a.n_pages * one + (int64_t)(h * (uint32_t)page) * a.dim;
  };
  const int dsh = 31 - __builtin_clz(a.dim), ksh = 31 - __builtin_clz(kpieces);
  for (uint32_t it = block * 256 + tid; it < all; it += a.blocks * 256) {
    if (it < nv) {
      values(reinterpret_cast<V*>(a.v) + first(it >> dsh) + (int64_t)(it & (a.dim - 1)) * page);
    } else if (it - nv < (nk + 63) / 64 * 64) {
      const uint32_t i = it - nv;
      if (i < nk) move(reinterpret_cast<ss_u32x4*>(reinterpret_cast<V*>(a.k) + first(i >> ksh)) + (i & (kpieces - 1)), one / EV, kpieces);
    } else {
      const uint32_t i = it - nv - (nk + 63) / 64 * 64, layer = (i >> 1) / (uint32_t)a.kv_heads, h = (i >> 1) - layer * a.kv_heads;
      move(a.scales + (((int64_t)layer * a.n_pages * a.kv_heads + h) * 2 + (i & 1)) * page, (int64_t)a.kv_heads * 2 * page, 1);
    }
  }
}

}  // namespace

hipError_t launch_tree_masks(const TreeMaskArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(tree_masks_kernel, dim3((unsigned)a.seqs), dim3(64), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_tree_accept(const TreeAcceptArgs& a, hipStream_t st) {
  if (a.rows > 0) {
    hipLaunchKernelGGL(tree_argmax_kernel, dim3((unsigned)((int64_t)a.rows * a.splits)), dim3(256), 0, st, a);
    if (const hipError_t e = hipGetLastError()) return e;
  }
  hipLaunchKernelGGL(tree_walk_kernel, dim3((unsigned)a.seqs), dim3(1024), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_keep_rows(KeepArgs a, hipStream_t st) {
  // A part a thread up to 8,192 workgroups, past which more of them change nothing: 32 sequences of 48 layers and 8 key heads of e4m3 take
  // 54 us so and with 16,384, 57 with 4,096, 62 with 2,048, 60 with 512.
  const int64_t parts = (int64_t)(a.dim + a.dim * a.size / 16 + (a.size == 1 ? 2 : 0)) * a.kv_heads * a.layers + 63;
  a.blocks = (int)std::min<int64_t>((parts + 255) / 256, std::max<int64_t>(8192 / a.seqs, 1));
  const dim3 grid((unsigned)(a.blocks * a.seqs));
  if (a.size == 1)
    hipLaunchKernelGGL((keep_rows_kernel<uint8_t, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((keep_rows_kernel<uint16_t, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ss
