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

int attn_prompt_parts(int dim, int page_shift);
hipError_t launch_attn_prompt(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
hipError_t launch_attn_few(const AttnArgs& a, int dim, bool fp16, hipStream_t st);
int attn_few_packed(int dim, int packed);
hipError_t launch_attn_join(const AttnArgs& a, int dim, bool fp16, hipStream_t st);

}  // namespace ss
