// Attention of prompt chunks over a paged cache: many rows of a sequence, so that the work is the two matrix products,
// 4 dim FLOP per (row, token) and head.
//
// The rows of a sequence times the heads of a key head are one packed axis, as in ss_attn.hip: a chunk's tiles hold
// rows of nearly one position, and a key head's tokens are read once for all its heads. A workgroup has 128 packed rows,
// 32 a wave as the columns of v_mfma_f32_32x32x16, and goes over the tokens in tiles of TK:
//   S^T = K Q^T, queries in registers; A row m = 8 b + 4 h + r of a 32-token tile is token 16 (b / 2) + 8 h + 4 (b % 2) + r, so
//     lane (c, h) = (lane % 32, lane / 32) ends with column c's scores at tokens 16 s + 8 h + 0..7 (s = 0, 1), and its
//     probabilities are, as they are, the B operands of
//   O^T = V^T P^T, whose A operand is 8 consecutive tokens of a dimension: the cache's own order.
// A column's maximum and weight need one exchange between lanes c and c + 32.
//
// Keys and values go from memory to LDS without registers, two stages, the next tile's loads issued before the present
// tile's products. In LDS the 16-byte piece c of a row lies at c ^ swizzle(row), so that 16 rows read at one place
// touch all banks; the loads put it there by which piece each lane fetches.
//
// The running maximum is raised only when a score passes it by 2^kLazy: until then probabilities are up to 2^kLazy, exact
// all the same, and the sums are not touched. Masks are worked out only in tiles that some row of the wave does not see
// whole, where values at unseen places are also kept out of the products (as in ss_attn.hip).
//
// Bound by the matrix units and what runs beside them: a tile of 64 tokens and 128 dimensions is 32 products (1,024 cycles of a
// SIMD) beside some 290 other instructions, 32 exponentials among them. 8,191 rows of 32 heads under a window of 4,096 (551
// GFLOP) take 560-620 us, 0.89 to 0.98 PFLOP/s; an 8,192^3 bf16 product of the library reaches 1.23 on this card.
#include <hip/hip_runtime.h>

#include "ss_attn.hpp"
#include "ss_launch.hpp"

namespace ss {

namespace {

constexpr float kNegInf = -__builtin_inff();
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

SS_DEV void dma16(const void* src, void* lds) { __builtin_amdgcn_global_load_lds(src, (lds_void*)lds, 16, 0, 0); }

template <class T>
SS_DEV f32x16 mfma32(const ss_u32x4& a, const ss_u32x4& b, const f32x16& c) {
  if constexpr (std::is_same<T, Bf16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(ss_bf16x8, a), __builtin_bit_cast(ss_bf16x8, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(ss_f16x8, a), __builtin_bit_cast(ss_f16x8, b), c, 0,
                                                  0, 0);
}

SS_DEV void local_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

SS_DEV float other_half(float v, bool upper) {
  uint32_t lo, hi;
  ss_pair<32>(ss_fu(v), lo, hi);
  return ss_uf(upper ? lo : hi);
}

// Where the 16-byte piece c of row r lies in LDS: at c ^ swizzle(r). A row has D / 8 pieces (keys) or TK / 8 (values), and 16
// rows that one read touches at the same piece fall on 16 different places of the 256 bytes that the banks cover.
template <int D>
SS_DEV constexpr int kswizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int TK>
SS_DEV constexpr int vswizzle(int row) {
  return TK == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// D: dimensions; DV: those of the output that one workgroup has (of 256 it has half, and its scores are computed twice: the
// sums of all of them beside the queries would leave no registers).
// ONE: a tile lies in one page (page >= TK).
template <class T, int D, int DV, int TK, bool ONE>
__global__ __launch_bounds__(256, 2) void attn_prompt_kernel(AttnArgs a) {
  constexpr int KS = D / 16, DT = DV / 32, ST = TK / 32;        // products per score tile, output tiles, score tiles
  constexpr int KROW = D * 2, VROW = TK * 2;                   // bytes of a row in LDS
  constexpr int KC = D / 8, VC = TK / 8;                       // 16-byte pieces of a row
  constexpr int KI = TK * KROW / 4096, VI = DV * VROW / 4096;   // 1 KB load instructions a wave
  __shared__ __attribute__((aligned(1024))) uint8_t k0[TK * KROW];
  __shared__ __attribute__((aligned(1024))) uint8_t k1[TK * KROW];
  __shared__ __attribute__((aligned(1024))) uint8_t v0[DV * VROW];
  __shared__ __attribute__((aligned(1024))) uint8_t v1[DV * VROW];
  __shared__ int odd;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  int b = blockIdx.x;
  const int dv = b % (D / DV) * DV;  // first output dimension
  b /= D / DV;
  const int kh = b % a.kv_heads;
  b /= a.kv_heads;
  const int slot = b % a.slots;
  b /= a.slots;
  const int s = b % a.seqs, turn = b / a.seqs;
  // The tiles that see most first; the last `a.rising` turns, which share CUs with the first ones, from the other end.
  const int tile = turn < a.tiles - a.rising ? a.tiles - 1 - turn : turn - (a.tiles - a.rising);
  const int page = 1 << a.page_shift;
  SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, (int64_t)a.width * page, a.err);
  sr.r0 = __builtin_amdgcn_readfirstlane(sr.r0);
  sr.n = __builtin_amdgcn_readfirstlane(sr.n);
  sr.pos0 = __builtin_amdgcn_readfirstlane(sr.pos0);
  sr.end = __builtin_amdgcn_readfirstlane(sr.end);
  const int p0 = tile * 128, np = sr.n * a.group;
  if (p0 >= np) return;
  const Seen sn = seen_tokens(sr.pos0 + p0 / a.group, sr.pos0 + (min(p0 + 128, np) - 1) / a.group, sr.end, a.window,
                              a.sinks);
  const int sc = (sn.s_end + a.chunk - 1) / a.chunk, wc = max(sn.w_begin / a.chunk, sc);
  int t_begin = 0, t_end = sn.end;
  if (a.slots > 1) {
    const int ch = slot < sc ? slot : wc + slot - sc;
    t_begin = ch * a.chunk;
    t_end = min(t_begin + a.chunk, sn.end);
    if (t_begin >= t_end) return;
  }
  // The tiles of [t_begin, t_end) that some row sees: up to the first tokens' end, then from the window's begin on.
  const int gap_a = (sn.s_end + TK - 1) / TK * TK, gap_b = max(sn.w_begin / TK * TK, gap_a);
  auto next_tile = [&](int t) { return t >= gap_a && t < gap_b ? gap_b : t; };

  // This lane's column.
  const int p = p0 + 32 * w + c, i = p / a.group;
  const bool in = p < np;
  const int qpos = in ? sr.pos0 + i : -1;
  ss_u32x4 qf[KS];
  {
    const uint16_t* qp = a.q + (int64_t)(sr.r0 + (in ? i : 0)) * a.q_row +
                         (int64_t)(kh * a.group + (in ? p - i * a.group : 0)) * a.q_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const SS_G ss_u32x4*)(qp + 16 * ks);
  }
  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
  float m = kNegInf, l = 0.f, top = kNegInf;

  // Pages of a tile's 16-token groups (one where the tile lies in one page), -1 where there is none: the table's entries 64 at
  // a time in one register, an entry a lane. (Scalar loads of single entries cost some 500 cycles of every tile.)
  constexpr int NP = ONE ? 1 : TK / 16;
  const int32_t* tab = a.table + (int64_t)s * a.width;
  int first_entry = -64, entries = -1;
  auto page_id = [&](int t, int j) {
    const int at = (t + 16 * j) >> a.page_shift;
    if (__builtin_expect((uint32_t)(at - first_entry) >= 64u, 0)) {
      first_entry = at;
      entries = at + lane < a.width ? gp(tab)[at + lane] : -1;
      entries = (uint32_t)entries < (uint32_t)a.n_pages ? entries : -1;
    }
    return __builtin_amdgcn_readlane(entries, at - first_entry);
  };
  const int64_t page_bytes = (int64_t)a.kv_heads * page * D * 2;
  const char* kbase = reinterpret_cast<const char*>(a.k) + (int64_t)kh * page * D * 2;
  const char* vbase = reinterpret_cast<const char*>(a.v) + (int64_t)(kh * D + dv) * page * 2;
  // What this lane fetches in its first load of a stage, as bytes from the place of the tile (K without ONE: of the load's
  // 16-token group) in its page; K rows are tokens, V rows dimensions. Load n is RK (RV) rows on, and its piece differs in
  // the swizzle bits of those rows.
  constexpr int RK = 64 / KC, RV = 64 / VC;
  const int krow0 = w * KI * RK + lane / KC, vrow0 = w * VI * RV + lane / VC;
  const uint32_t koff0 = (ONE ? krow0 : krow0 % 16) * KROW + 16 * ((lane % KC) ^ kswizzle<D>(krow0));
  const int vpiece0 = (lane % VC) ^ vswizzle<TK>(vrow0);
  const uint32_t voff0 = (uint32_t)vrow0 * page * 2 + 16 * (ONE ? vpiece0 : vpiece0 & 1);
  struct Tile {
    int t;          // its first token
    int ids[NP];    // its pages, 0 where there is none
    uint32_t held;  // bit j: page j is there
  };
  auto tile_at = [&](int t) {
    Tile r;
    r.t = t;
    r.held = 0;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int id = page_id(t, j);
      r.held |= id >= 0 ? 1u << j : 0u;
      r.ids[j] = max(id, 0);
    }
    return r;
  };
  auto load_k = [&](const Tile& r, uint8_t* kl, int n) {
    {
      const int j = ONE ? 0 : (w * KI + n) * (64 / KC) / 16;  // the load's 16-token group
      int id = r.ids[0];
#pragma unroll
      for (int q = 1; q < NP; ++q) id = j == q ? r.ids[q] : id;
      const char* at = kbase + id * page_bytes + (((r.t + 16 * j) & (page - 1)) + n * RK) * KROW;
      dma16(at + (koff0 ^ (16 * kswizzle<D>(n * RK))), kl + (w * KI + n) * 1024);
    }
  };
  auto load_v = [&](const Tile& r, uint8_t* vl, int n) {
    {
      if constexpr (ONE) {
        const char* at = vbase + r.ids[0] * page_bytes + ((r.t & (page - 1)) + n * RV * page) * 2;
        dma16(at + (voff0 ^ (16 * vswizzle<TK>(n * RV))), vl + (w * VI + n) * 1024);
      } else {
        const int j = (vpiece0 ^ vswizzle<TK>(n * RV)) / 2;
        int id = r.ids[0];
#pragma unroll
        for (int q = 1; q < NP; ++q) id = j == q ? r.ids[q] : id;
        dma16(vbase + id * page_bytes + ((r.t + 16 * j) & (page - 1)) * 2 + n * RV * page * 2 + voff0,
              vl + (w * VI + n) * 1024);
      }
    }
  };
  constexpr uint32_t kAll = (1u << NP) - 1;
  auto has = [&](uint32_t held, int group) { return ((held >> (ONE ? 0 : group)) & 1u) != 0; };

  // Where this lane reads: K row of score row c, V row of dimension c.
  const int krow = 16 * (c / 16) + 8 * ((c / 4) % 2) + 4 * ((c / 8) % 2) + c % 4;
  const int kswz = kswizzle<D>(krow), vswz = vswizzle<TK>(c);

  auto sees = [&](int tok, bool held) { return held && tok <= qpos && (tok > qpos - a.window || tok < a.sinks); };
  // A plain tile: every row of the workgroup sees all of it. The tiles that hold first tokens only are taken as not plain.
  const int blk_lo = sr.pos0 + p0 / a.group, blk_hi = sr.pos0 + (min(p0 + 128, np) - 1) / a.group;
  const int plain_a = blk_hi - a.window + 1, plain_b = blk_lo - TK + 1;
  auto plain = [&](const Tile& r) { return r.t >= plain_a && r.t <= plain_b && r.held == kAll; };
  auto kread = [&](const uint8_t* kl, int f) {
    return *reinterpret_cast<const ss_u32x4*>(kl + (krow + 32 * (f / KS)) * KROW + 16 * ((2 * (f % KS) + h) ^ kswz));
  };
  auto vread = [&](const uint8_t* vl, int d, int nk) {
    return *reinterpret_cast<const ss_u32x4*>(vl + (c + 32 * d) * VROW + 16 * ((2 * nk + h) ^ vswz));
  };
  auto scores = [&](const uint8_t* kl, f32x16 (&y)[ST]) {
#pragma unroll
    for (int n = 0; n < ST; ++n) y[n] = f32x16{};
#pragma unroll
    for (int f = 0; f < ST * KS; ++f) y[f / KS] = mfma32<T>(kread(kl, f), qf[f % KS], y[f / KS]);
  };
  auto mask = [&](const Tile& r, f32x16 (&x)[ST]) {
    const int t = r.t;
    const uint32_t held = r.held;
    // This lane's token e of score tile n is seen where lo < 32 n + 16 (e / 8) + e % 8 <= hi. The comparisons are kept in
    // small groups: all at once they would take more scalar registers than there are.
    const int hi = qpos - t - 8 * h, lo = hi - a.window;
    if (t >= a.sinks && held == kAll) {
#pragma unroll
      for (int n = 0; n < ST; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int off = 32 * n + 16 * (e / 8) + e % 8;
          x[n][e] = off <= hi && off > lo ? x[n][e] : kNegInf;
          if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    } else {
#pragma unroll
      for (int n = 0; n < ST; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int off = 32 * n + 16 * (e / 8) + e % 8;
          const bool see = has(held, 2 * n + e / 8) && off <= hi && (off > lo || off < a.sinks - t - 8 * h);
          x[n][e] = see ? x[n][e] : kNegInf;
          if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (held != kAll) {
      // a page that is missing where a row of the wave sees a token
      bool miss = false;
#pragma unroll
      for (int j = 0; j < TK / 16; ++j) {
        const int first = t + 16 * j;
        miss |= !has(held, j) && first <= qpos && (first + 15 > qpos - a.window || first < a.sinks);
      }
      if (miss) raise_bit(a.err, SS_ERR_PAGE);
    }
  };
  // In a tile that is not plain non-finite values are taken out of the stage before any
  // wave uses it; `odd` says that there were any, and they are dealt with after the last tile.
  auto clean = [&](uint8_t* vl) {
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      ss_u32x4* at = reinterpret_cast<ss_u32x4*>(vl + (n * 256 + tid) * 16);
      const ss_u32x4 x = *at;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) bad |= nonfinite2<T>(x[j]);
      if (bad) {
        *at = parts_of<T>(x, -1);
        odd = 1;
      }
    }
    local_barrier();
  };
  auto max_of = [&](const f32x16 (&y)[ST]) {
    float v = y[0][0];
#pragma unroll
    for (int n = 0; n < ST; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) v = fmaxf(v, y[n][e]);
    return v;
  };
  // The softmax and value product of tile r, whose scores are x with the lane's largest one in `top`; between, the scores of
  // the next tile (in kl) are worked out into y: the matrix unit has them while the exponentials take the vector unit.
  // The loads of the keys of rk (to kn) and the values of rv (to vn) go out one at a time beside the products: all at once
  // they hold up the wave for as long as the memory path takes them in.
  auto step = [&](const Tile& r, const uint8_t* kl, uint8_t* vl, f32x16 (&x)[ST], f32x16 (&y)[ST], const Tile& rk,
                  uint8_t* kn, const Tile& rv, uint8_t* vn) {
    if (__builtin_expect(!plain(r), 0)) {
      clean(vl);
      mask(r, x);
      top = max_of(x);
    }
    const float mx = fmaxf(top, other_half(top, h)) * a.scale - T::kShift;
    if (__builtin_expect(__any(mx > m + T::kLazy || (m == kNegInf && mx > kNegInf)), 0)) {
      const float mn = fmaxf(m, mx);
      const float f = m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - mn);  // nothing summed yet (or NaN) where m is -inf
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] *= f;
      m = mn;
    }
    const float mu = m == kNegInf ? 0.f : m;
    ss_u32x4 pf[ST][2];
    float part[2] = {0.f, 0.f};
    // The operands of a product are read AHEAD products before it, those of the first value products beside the last of
    // the scores; PER scores of x are worked on beside each product of y.
    constexpr int NK = ST * KS, PER = 16 * ST / NK, NV = DT * 2 * ST, AHEAD = 4, RING = AHEAD + 1;
    ss_u32x4 fr[RING];
    auto fetch = [&](int f) {
      if (f < NK)
        fr[f % RING] = kread(kl, f);
      else if (f < NK + NV)
        fr[f % RING] = vread(vl, (f - NK) / (2 * ST), (f - NK) % (2 * ST));
    };
#pragma unroll
    for (int f = 0; f < AHEAD; ++f) fetch(f);
#pragma unroll
    for (int n = 0; n < ST; ++n) y[n] = f32x16{};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int f = 0; f < NK; ++f) {
      fetch(f + AHEAD);
      y[f / KS] = mfma32<T>(fr[f % RING], qf[f % KS], y[f / KS]);
      if (PER > 1 || f % 2 == 0) {
#pragma unroll
        for (int q = f * PER; q < f * PER + (PER > 1 ? PER : 2); q += 2) {
          const int n = q / 16, e = q % 16;
          const float q0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][e], a.scale, -mu));
          const float q1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[n][e + 1], a.scale, -mu));
          part[q / 2 % 2] += q0;
          part[q / 2 % 2] += q1;  // the sum has the weights as they are, the product rounded once to the element type
          pf[n][e / 8][(e % 8) / 2] = T::pack(q0, q1);
        }
      }
      constexpr int EVERY = NK / (KI + VI) < 1 ? 1 : NK / (KI + VI);
      if (f % EVERY == EVERY - 1) {
        if (f / EVERY < KI)
          load_k(rk, kn, f / EVERY);
        else if (f / EVERY < KI + VI)
          load_v(rv, vn, f / EVERY - KI);
      }
      if (f % 2) __builtin_amdgcn_sched_barrier(0);
    }
    l += part[0] + part[1];
    top = y[0][0];
#pragma unroll
    for (int f = NK; f < NK + NV; ++f) {
      const int d = (f - NK) / (2 * ST), nk = (f - NK) % (2 * ST);
      fetch(f + AHEAD);
      acc[d] = mfma32<T>(fr[f % RING], pf[nk / 2][nk % 2], acc[d]);
#pragma unroll
      for (int q = (f - NK) * 16 * ST / NV; q < (f - NK + 1) * 16 * ST / NV; ++q) top = fmaxf(top, y[q / 16][q % 16]);
      if (f % 2) __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto sync = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of the stage have landed
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  if (tid == 0) odd = 0;  // before the first tile's barrier
  // Tile i: keys in stage i % 2 from two steps before its softmax, values from one. Loads for tiles past the last one are
  // issued too (of page 0 where there is none): what they bring is not read.
  f32x16 x[ST], y[ST];
  Tile r0 = tile_at(next_tile(t_begin)), r1 = tile_at(next_tile(r0.t + TK));
  if (r0.t < t_end) {
#pragma unroll
    for (int n = 0; n < KI; ++n) load_k(r0, k0, n);
#pragma unroll
    for (int n = 0; n < KI; ++n) load_k(r1, k1, n);
#pragma unroll
    for (int n = 0; n < VI; ++n) load_v(r0, v0, n);
    sync();
    scores(k0, x);
    top = max_of(x);
  }
  while (r0.t < t_end) {
    sync();  // keys of r1 and values of r0 are there, the other stages free: every wave has finished with them
    const Tile r2 = tile_at(next_tile(r1.t + TK));
    step(r0, k1, v0, x, y, r2, k0, r1, v1);
    if (r1.t >= t_end) break;
    sync();
    const Tile r3 = tile_at(next_tile(r2.t + TK));
    step(r1, k0, v1, y, x, r3, k1, r2, v0);
    r0 = r2;
    r1 = r3;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no load into LDS outlives the wave
  __syncthreads();
  const bool fix = odd;
  l += other_half(l, h);
  const int64_t at = (int64_t)(sr.r0 + i) * a.heads + kh * a.group + (p - i * a.group);
  const int64_t pa = (int64_t)slot * a.rows * a.heads + at;
  if (in && a.slots > 1) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b4 = 0; b4 < 4; ++b4) {
        ss_f32x4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = acc[d][4 * b4 + r];
        *reinterpret_cast<SS_G ss_f32x4*>(gp(a.po) + pa * D + dv + 32 * d + 8 * b4 + 4 * h) = o;
      }
    if (h == 0 && dv == 0) {
      gp(a.pml)[2 * pa] = m;
      gp(a.pml)[2 * pa + 1] = l;
    }
  } else if (in) {
    const float r = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int b4 = 0; b4 < 4; ++b4) {
        uint2 word;
        word.x = T::pack(acc[d][4 * b4] * r, acc[d][4 * b4 + 1] * r);
        word.y = T::pack(acc[d][4 * b4 + 2] * r, acc[d][4 * b4 + 3] * r);
        *reinterpret_cast<uint2*>(a.out + at * D + dv + 32 * d + 8 * b4 + 4 * h) = word;
      }
    if (a.lse && h == 0 && dv == 0) a.lse[at] = l == 0.f ? kNegInf : (m + __log2f(l)) * 0.693147180559945309f;
  }
  if (!fix) return;
  // Infinities and NaN that were taken out go to the columns that see them, by a product of ones in their places with ones
  // for the tokens seen; each lane adds to what it wrote itself.
#pragma unroll 1
  for (int t = next_tile(t_begin); t < t_end; t = next_tile(t + TK)) {
    if (plain(tile_at(t))) continue;
#pragma unroll 1
    for (int nk = 0; nk < 2 * ST; ++nk) {
      const int first = t + 16 * nk + 8 * h, id = page_id(t, nk);
      const uint16_t* vp = reinterpret_cast<const uint16_t*>(vbase + max(id, 0) * page_bytes) + (int64_t)c * page +
                           (first & (page - 1));
      ss_u32x4 ones;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        ones[j] = (sees(first + 2 * j, id >= 0) ? T::kOne : 0u) | (sees(first + 2 * j + 1, id >= 0) ? T::kOne << 16 : 0u);
#pragma unroll 1
      for (int d = 0; d < DT; ++d) {
        const ss_u32x4 vf = *(const SS_G ss_u32x4*)(vp + (int64_t)32 * d * page);
#pragma unroll 1
        for (int kind = 0; kind < 3; ++kind) {
          const float add = kind == 0 ? -kNegInf : kind == 1 ? kNegInf : __builtin_nanf("");
          const f32x16 hits = mfma32<T>(parts_of<T>(vf, kind), ones, f32x16{});
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (!in || !(hits[e] > 0.f)) continue;
            const int od = dv + 32 * d + 8 * (e / 4) + 4 * h + e % 4;
            if (a.slots > 1)
              gp(a.po)[pa * D + od] += add;
            else
              a.out[at * D + od] = (uint16_t)T::pack(T::widen(a.out[at * D + od]) + add, 0.f);
          }
        }
      }
    }
  }
}

// Tiles of 64 tokens where a page holds them, else of 32 (and of 256 dimensions always: registers).
template <class T, int D, int DV>
void launch_prompt(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.slots * a.tiles * a.kv_heads * a.seqs * attn_prompt_parts(D, a.page_shift)));
  if (a.page_shift >= 6 && D < 256)
    hipLaunchKernelGGL((attn_prompt_kernel<T, D, DV, D < 256 ? 64 : 32, true>), grid, dim3(256), 0, st, a);
  else if (a.page_shift >= 5)
    hipLaunchKernelGGL((attn_prompt_kernel<T, D, DV, 32, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_prompt_kernel<T, D, D < 256 ? DV : 64, 32, false>), grid, dim3(256), 0, st, a);
}

template <class T>
hipError_t launch_prompt_of(const AttnArgs& a, int dim, hipStream_t st) {
  if (dim == 64)
    launch_prompt<T, 64, 64>(a, st);
  else if (dim == 128)
    launch_prompt<T, 128, 128>(a, st);
  else
    launch_prompt<T, 256, 128>(a, st);
  return hipGetLastError();
}

}  // namespace

// Workgroups that share the output dimensions of a row tile (a quarter each where pages of 16 tokens take more registers).
int attn_prompt_parts(int dim, int page_shift) { return dim < 256 ? 1 : page_shift >= 5 ? 2 : 4; }

hipError_t launch_attn_prompt(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_prompt_of<Fp16>(a, dim, st) : launch_prompt_of<Bf16>(a, dim, st);
}

}  // namespace ss
