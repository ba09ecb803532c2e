// What the attention kernels over a paged key-value cache share: their arguments, the two element types and a
// sequence's place in the batch.
//
// Cache of a layer: keys [n_pages][kv_heads][page][dim], values [n_pages][kv_heads][dim][page]. Values are kept token
// by token along each dimension because the product with the probabilities sums over tokens: eight consecutive tokens
// of one dimension are one 16-byte MFMA operand, so neither kernel transposes anything.
#pragma once
#include "ss_common.hpp"

namespace ss {

struct AttnArgs {
  const uint16_t* q;  // [rows][heads][dim], strides in elements
  int64_t q_row, q_head;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* cu;      // [seqs + 1]
  const int32_t* kv_len;  // [seqs]
  const int32_t* table;   // [seqs][width]
  uint16_t* out;          // [rows][heads][dim]
  float* lse;             // [rows][heads] or null
  float* po;              // partial sums [slots][rows][heads][dim] and ...
  float* pml;             // ... their maxima and weights [slots][rows][heads][2]; unused with one slot
  int* err;
  int64_t n_pages;
  int rows, seqs, max_rows, heads, kv_heads, group, page_shift, width;
  int window;  // keys a row sees counted back from its own; INT_MAX / 2 for all
  int sinks;   // first tokens that stay visible under a window
  int slots;   // chunks of one sequence that the grid covers
  int chunk;   // tokens of a chunk, a multiple of 128; at most 4096 with few rows, up to the whole table with many
  int packed;  // packed rows (rows times heads of a key head) of a workgroup
  int tiles;   // workgroups over the packed rows of one sequence and key head
  int rising;  // many rows: the tiles at the end of the launch that go up
  float scale; // of the scores, times log2(e)
  const uint8_t* scales;  // [n_pages][kv_heads][2][page] exponents of e4m3 keys and values (k, v then hold bytes), or null
  const uint64_t* tree;   // [rows] which of its sequence's rows a row sees, or null (causal)
  // Shared chunks (many rows over e4m3 pages or of trees): `share` > 0 of them for the row tiles of all sequences together, of one size,
  // by how many tiles and tokens each has; `slots` then counts them over all, po and pml are [slots][kv_heads][128 packed rows], and
  int share;
  int32_t* meta;  // [1 + seqs] has the size in units of 64 tokens and each sequence's first chunk, for the join
};

// ss_raise through a global pointer (a flat atomic would make every later wait of the wave one for all its LDS reads).
SS_DEV void raise_bit(int* err, int bit) {
  if (err) __hip_atomic_fetch_or(gp(err), bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

typedef _Float16 ss_f16x8 __attribute__((ext_vector_type(8)));

// The element types. kShift: probabilities are kept 2^kShift times as large, the running maximum that much lower. fp16
// has no exponents below 2^-14 with full precision, so a probability of 2^-14 of the row's largest would lose bits;
// with the factor they are whole to 2^-24, and at most 2^10 leaves room for fp32 sums. bf16 has fp32's exponents.
// kLazy: a running maximum is raised only when a score passes it by 2^kLazy; until then weights are up to 2^(kShift + kLazy),
// at most 2^14 in fp16.
struct Bf16 {
  static constexpr float kShift = 0.f, kLazy = 8.f;
  static constexpr uint32_t kExp = 0x7F80u, kOne = 0x3F80u;
  SS_DEV static ss_f32x4 mfma16(const ss_u32x4& a, const ss_u32x4& b, const ss_f32x4& c) { return ss_mfma(a, b, c); }
  // One v_cvt_pk_bf16_f32 (of two conversions and an or, the compiler makes four instructions).
  SS_DEV static uint32_t pack(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), b2));
  }
  SS_DEV static float widen(uint32_t u) { return ss_bf16_to_f32(u); }
};
struct Fp16 {
  static constexpr float kShift = 10.f, kLazy = 4.f;
  static constexpr uint32_t kExp = 0x7C00u, kOne = 0x3C00u;
  SS_DEV static ss_f32x4 mfma16(const ss_u32x4& a, const ss_u32x4& b, const ss_f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ss_f16x8, a), __builtin_bit_cast(ss_f16x8, b), c, 0,
                                                  0, 0);
  }
  SS_DEV static uint32_t pack(float lo, float hi) {
    return (uint32_t)__builtin_bit_cast(uint16_t, static_cast<_Float16>(lo)) |
           ((uint32_t)__builtin_bit_cast(uint16_t, static_cast<_Float16>(hi)) << 16);
  }
  SS_DEV static float widen(uint32_t u) { return (float)__builtin_bit_cast(_Float16, (uint16_t)u); }
};

// Whether either half of a word is an infinity or NaN.
template <class T>
SS_DEV bool nonfinite2(uint32_t w) {
  return (w & T::kExp) == T::kExp || (w & (T::kExp << 16)) == (T::kExp << 16);
}
// One 16-bit value: the value to multiply with, or with `kind` 0, 1, 2 a one where it is +inf, -inf, NaN.
template <class T>
SS_DEV uint32_t part_of(uint32_t x, int kind) {
  const bool nf = (x & T::kExp) == T::kExp, nan = nf && (x & (T::kExp ^ 0x7FFFu)) != 0;
  if (kind < 0) return nf ? 0u : x;
  const bool hit = kind == 2 ? nan : (nf && !nan && (x >> 15) == (uint32_t)kind);
  return hit ? T::kOne : 0u;
}
template <class T>
SS_DEV ss_u32x4 parts_of(const ss_u32x4& v, int kind) {
  ss_u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = part_of<T>(v[i] & 0xFFFFu, kind) | (part_of<T>(v[i] >> 16, kind) << 16);
  return r;
}

// Rows [r0, r0 + n) of sequence s, the position of its first row (negative where the cache is said to hold fewer tokens
// than the call has rows) and the end of its tokens. What contradicts the arguments is cut to them and raised.
struct SeqRows {
  int r0, n, pos0, end;
};
SS_DEV SeqRows seq_rows(const int32_t* cu, const int32_t* kv_len, int s, int rows, int max_rows, int64_t cap, int* err) {
  int a = gp(cu)[s], b = gp(cu)[s + 1], len = gp(kv_len)[s];
  bool bad = a < 0 || b < a || b > rows || b - a > max_rows || len < 0 || (int64_t)len > cap;
  SeqRows r;
  r.r0 = a < 0 ? 0 : (a > rows ? rows : a);
  int e = b > rows ? rows : b;
  r.n = e > r.r0 ? e - r.r0 : 0;
  if (r.n > max_rows) r.n = max_rows;
  len = len < 0 ? 0 : len;
  // The rows' positions go by the row count the caller gave; a row that was cut away keeps its place behind the others.
  const int64_t p0 = (int64_t)len - (b > a ? (int64_t)b - a : 0) + (r.r0 - a);
  r.pos0 = (int)(p0 < -(1 << 30) ? -(1 << 30) : p0);
  r.end = (int64_t)len > cap ? (int)cap : len;
  if (bad && (threadIdx.x & 63) == 0) raise_bit(err, SS_ERR_BATCH);
  return r;
}

// The parts of a sequence's tokens that rows at positions [pos_a, pos_b] see: [0, s_end) (the first tokens) and
// [w_begin, end), both empty or apart.
struct Seen {
  int s_end, w_begin, end;
};
SS_DEV Seen seen_tokens(int pos_a, int pos_b, int end, int window, int sinks) {
  Seen r;
  r.end = pos_b + 1 < end ? pos_b + 1 : end;
  if (r.end < 0) r.end = 0;
  const int w = pos_a - window + 1;
  r.w_begin = w > 0 ? (w < r.end ? w : r.end) : 0;
  r.s_end = sinks < r.w_begin ? sinks : r.w_begin;
  return r;
}

// ---------------------------------------------------------------- shared chunks
// Chunk g of a call whose row tiles share at most `a.share` chunks: units of 64 tokens, `size` of them a chunk, two or more. (More than
// the CUs have places for would wait for the first to end: with 150 in the place of 126 sixteen trees of up to 26 rows took 96 us, not 65.) A
// sequence's chunks go by their place, the tiles of one place side by side. A wave works it out from all lengths. With `write` (one
// wave of the launch) the sequences' first chunks go to a.meta.
//
// A chunk has `per` workgroups (key heads, parts of the dimensions). Workgroups are dealt to the 8 XCDs in turn; each XCD takes a run of
// neighbours, so that the row tiles that read one chunk of the cache do so through one L2.
struct Share {
  int s, tile, slot, size;  // the sequence, the row tile, the chunk of its tokens; s < 0: nothing for this workgroup
  int g, part;              // the chunk, the workgroup's number in it
};
SS_DEV Share find_share(const AttnArgs& a, int block, int per, bool write) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)a.width << a.page_shift;
  struct Size {
    uint32_t units, tiles;
  };
  auto size_of = [&](int s) {
    Size r = {0, 0};
    if (s >= a.seqs) return r;
    const int from = gp(a.cu)[s], to = gp(a.cu)[s + 1], len = max(gp(a.kv_len)[s], 0);
    const int n = min(min(to, a.rows) - min(max(from, 0), a.rows), a.max_rows);  // as seq_rows cuts them
    if (n <= 0) return r;
    r.units = (uint32_t)(((int64_t)len < cap ? len : cap) + 63) / 64;
    r.tiles = (uint32_t)(n * a.group + 127) / 128;
    return r;
  };
  auto sum = [](uint32_t x) {  // over the lanes; in a scalar register, as all that follows from it
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)ss_butterfly(x, [](uint32_t p, uint32_t q) { return p + q; }));
  };
  // One sequence: no sums over the lanes (a tree of 12 rows over 777 tokens 16.2 -> 15.6 us).
  if (a.seqs == 1) {
    const Size z = size_of(0);
    const uint32_t units = __builtin_amdgcn_readfirstlane(z.units), tiles = max(__builtin_amdgcn_readfirstlane(z.tiles), 1);
    const uint32_t most = (uint32_t)a.share / tiles;  // chunks of a tile
    const uint32_t size = max((units + most - 1) / most, 2u), chunks = (units + size - 1) / size;
    const int all = (int)(chunks * tiles) * per, run = (all + 7) / 8, id = block % 8 * run + block / 8;
    if (write && lane == 0) {
      a.meta[0] = (int)size;
      a.meta[1] = 0;
    }
    Share r = {-1, 0, 0, (int)size, -1, 0};
    if (block / 8 < run && id < all) {
      r.g = id / per;
      r.part = id - r.g * per;
      r.s = 0;
      r.slot = r.g / (int)tiles;
      r.tile = r.g - r.slot * (int)tiles;
    }
    return r;
  }
  const Size first = size_of(lane);
  uint64_t total = 0;
  uint32_t tiles = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const Size z = s0 ? size_of(s0 + lane) : first;
    total += sum(z.units * z.tiles);
    tiles += sum(z.tiles);
  }
  // No size below total / share is enough, and total / (share - tiles) is, whatever the tiles' last chunks are (tiles are at most
  // half of share). Between them the least one is looked for; of more than 64 sequences the latter is taken.
  uint32_t size = max((uint32_t)((total + a.share - tiles - 1) / (a.share - tiles)), 2u);
  if (a.seqs <= 64) {
    uint32_t lo = max((uint32_t)((total + a.share - 1) / a.share), 2u);
    while (lo < size) {
      const uint32_t mid = (lo + size) / 2;
      if (sum((first.units + mid - 1) / mid * first.tiles) <= (uint32_t)a.share)
        size = mid;
      else
        lo = mid + 1;
    }
  }
  uint32_t chunks = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const Size z = s0 ? size_of(s0 + lane) : first;
    chunks += sum((z.units + size - 1) / size * z.tiles);
  }
  const int all = (int)chunks * per, run = (all + 7) / 8, id = block % 8 * run + block / 8;
  Share r = {-1, 0, 0, (int)size, -1, 0};
  if (block / 8 < run && id < all) {
    r.g = id / per;
    r.part = id - r.g * per;
  }
  const int g = r.g;
  if (g < 0 && !write) return r;
  int before = 0;
  for (int s0 = 0; s0 < a.seqs && (write || r.s < 0); s0 += 64) {
    const Size z = s0 ? size_of(s0 + lane) : first;
    const int mine = (int)((z.units + size - 1) / size * z.tiles);
    int upto = mine;
    for (int d = 1; d < min(a.seqs, 64); d *= 2) {
      const int o = __shfl_up(upto, d);
      upto += lane >= d ? o : 0;
    }
    if (write && s0 + lane < a.seqs) a.meta[1 + s0 + lane] = before + upto - mine;
    const uint64_t hit = g < 0 ? 0 : __ballot(before + upto > g);
    if (r.s < 0 && hit) {
      const int l = __builtin_ctzll(hit);  // past the last sequence `upto` may be short: only a lane of one can be hit
      r.s = s0 + l;
      const int local = g - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l));
      const int tiles = __builtin_amdgcn_readlane((int)z.tiles, l);
      r.slot = local / tiles;
      r.tile = local - r.slot * tiles;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (write && lane == 0) a.meta[0] = (int)size;
  r.s = __builtin_amdgcn_readfirstlane(r.s);
  r.slot = __builtin_amdgcn_readfirstlane(r.slot);
  r.tile = __builtin_amdgcn_readfirstlane(r.tile);
  r.size = __builtin_amdgcn_readfirstlane(r.size);
  return r;
}

// ---------------------------------------------------------------- pages of e4m3 numbers
// A token's keys (its values) are its e4m3 numbers times 2^(s - 127), s a byte of 1 to 247: a power of two, so that a key
// times its scale is a bfloat16 as it is (3 bits of mantissa), and the conversion instruction applies it on the way. 255 is read
// as 254: what an unseen place holds stays finite.
SS_DEV float scale_of(uint32_t s) { return ss_uf(min(s, 254u) << 23); }
// 8 e4m3 numbers, two words, times `scale` (a power of two) as bfloat16.
SS_DEV ss_u32x4 widen8(uint32_t lo, uint32_t hi, float scale) {
  ss_u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return r;
}
// A word of four e4m3 numbers without its NaN (all but the sign set).
SS_DEV uint32_t without_nan8(uint32_t w) {
  uint32_t r = w;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (((w >> (8 * i)) & 0x7Fu) == 0x7Fu) r &= ~(0xFFu << (8 * i));
  return r;
}

// ---------------------------------------------------------------- rows of a tree
// Which of the 8 tokens from `first` on a row of a tree sees, a bit each: tokens before `base` (the place of the sequence's first
// row) that its window `pos - window` or the first tokens let it, and from base on those of its mask.
SS_DEV uint32_t tree_sees(int first, int base, int end, uint64_t mask, int pos, int window, int sinks) {
  const int off = base - first;  // tokens of the 8 before base
  uint32_t r = off >= 8 ? 0xFFu : off <= 0 ? 0u : (1u << off) - 1;
  const int w = pos - window + 1 - first, k = sinks - first;  // below w only those below k
  const uint32_t far = w >= 8 ? 0xFFu : w <= 0 ? 0u : (1u << w) - 1, kept = k >= 8 ? 0xFFu : k <= 0 ? 0u : (1u << k) - 1;
  r &= ~far | kept;
  if (off < 8 && off > -64) r |= (uint32_t)(off >= 0 ? mask << off : mask >> -off) & 0xFFu;
  const int left = end - first;
  return r & (left >= 8 ? 0xFFu : left <= 0 ? 0u : (1u << left) - 1);
}

int attn_prompt_parts(int dim, int page_shift, bool e4m3);
hipError_t launch_attn_prompt(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
hipError_t launch_attn_prompt_tree(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
hipError_t launch_attn_prompt_e4m3(const AttnArgs& a, int dim, hipStream_t st);
hipError_t launch_attn_few(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
hipError_t launch_attn_few_tree(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
hipError_t launch_attn_few_e4m3(const AttnArgs& a, int dim, hipStream_t st);
int attn_few_packed(int dim, int packed, bool e4m3);
hipError_t launch_attn_join(const AttnArgs& a, int dim, bool fp16, hipStream_t st);

}  // namespace ss
