// Attention of a batch's few new rows (a decoded token, the rows of a verify round) over a paged cache.
//
// For row i at position p, o_i = sum_j softmax_j(scale q_i k_j) v_j over the tokens j <= p, under a window those with
// p - j < window or j < sinks. Every key and value is used by the few rows of a sequence and the heads that share its key
// head, so the work is reading the cache once: 4 dim bytes per token and key head, 2 dim + 2 of e4m3 numbers.
//
// The rows of a sequence times the heads of a key head are one "packed" axis: NT tiles of 16, the columns of
// v_mfma_f32_16x16x32. A workgroup takes one chunk of the tokens of one (sequence, key head, NT tiles); its four waves
// take the chunk's 32-token tiles in turn:
//   S^T = K Q^T: A row m of S tile t (0, 1) is token 8 (m / 4) + 4 t + m % 4, so lane (c, g) = (lane % 16, lane / 16) ends
//     with the scores of column c at tokens 8 g + 0..7: its probabilities are, as they are, the B operand of
//   O^T = V^T P^T, whose A operand is 8 consecutive tokens 8 g.. of dimension 16 d + c.
// The running maximum is one value per column, equal in its four lanes; the sum of the weights stays per lane to the end.
//
// Each wave has a slot of LDS for a tile's keys and one for its values, filled by direct loads: the next tile's keys go out
// when this one's scores are done, its values after the products, and nothing waits for another wave. (Operands straight from
// memory into registers touch 16 rows with every load, 16 bytes of a row by lanes 16 apart, which the memory path takes as 64
// accesses where rows of adjacent lanes are 16.) In LDS the 16-byte piece p of a row lies at p ^ swizzle(row), so that
// the 16 rows of one operand read fall on different banks.
//
// A chunk begins at a multiple of its size from the sequence's first token and its tiles go to waves by their place in
// it, and masked tokens add exact zeros: the bits of a row do not depend on the other rows of the call. The
// chunks' partial sums are joined by a second launch (attn_join_kernel); a grid of one chunk writes the result itself.
//
// Values at places that a row does not see must not reach it, whatever they hold: a probability of 0 times an infinity is
// not 0. Only tiles that some row does not see whole can hold such places. There the operand is searched for non-finite
// values; where any are, they are taken out of the product and added at the join, by three more products with ones in their
// places and ones for the tokens seen, to the rows that see them.
//
// Pages of e4m3 numbers (E8): k_j = c_j 2^(s_j), v_j likewise, a power of two for each token and key head. A tile has 64 tokens, so that
// slots and loads are those of the 16-bit kernel. Keys are widened to bfloat16 by the instruction that multiplies by their power
// of two (exact: 3 bits of mantissa); a value's token is the product's inner index, so its power of two goes to the weight
// instead (exact, before the weight's rounding), and the sum of the weights leaves it out. A NaN code is dealt with as a non-finite
// value of 16 bits is, and there are no infinities.
//
// Trees (TREE): the rows of a sequence see its tokens before them and those rows whose bits their masks have. Only tiles that reach into
// the rows look at the masks, which lie in LDS: a lane's 8 tokens are 8 bits of its column's word. Under a window a row's position is its depth.
//
// Measured, kernel alone: 64 sequences of up to 16,384 tokens (32 heads on 8, 128 dimensions, 2.7 GB) 478 us, 5.7 TB/s, where a
// streaming read reaches 5.3; one of 131,072 tokens (268 MB) 42 us; one of 777 5.2 us, the chain of a sequence's place, its
// pages, its keys and the columns' sums. Operands straight from memory into registers took 8 % longer for the first.
// Of e4m3 the first (1.37 GB) takes 247 us, 5.6 TB/s of what is fetched; 8 sequences of up to 6,145 tokens, 3 rows of 256 dimensions (31 MB)
// 18.9 us, as of 16 bits: a chunk's fixed part. Tiles of 32 tokens, half of a slot, would load as many bytes with twice the instructions.
#pragma once
#include <hip/hip_runtime.h>

#include "ss_attn.hpp"
#include "ss_launch.hpp"

namespace ss {

namespace {

constexpr float kNegInf = -__builtin_inff();

SS_DEV float max_over_quads(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  uint32_t lo, hi;
  ss_pair<16>(ss_fu(v), lo, hi);
  v = fmaxf(ss_uf(lo), ss_uf(hi));
  ss_pair<32>(ss_fu(v), lo, hi);
  return fmaxf(ss_uf(lo), ss_uf(hi));
}

typedef __attribute__((address_space(3))) void lds_void;
SS_DEV void dma4(const void* src, void* lds) { __builtin_amdgcn_global_load_lds(src, (lds_void*)lds, 4, 0, 0); }
template <int OFF>  // bytes added to both addresses
SS_DEV void dma16(const void* src, void* lds) { __builtin_amdgcn_global_load_lds(src, (lds_void*)lds, 16, OFF, 0); }

// The same from a place that all lanes have and a lane's own offset.
template <int OFF>
SS_DEV void dma16_at(const void* src, uint32_t off, void* lds) {
  __builtin_amdgcn_global_load_lds((const SS_G void*)((const SS_G char*)src + off), (lds_void*)lds, 16, OFF, 0);
}

// A barrier over LDS alone: it waits for no load or store in flight.
SS_DEV void local_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// s_waitcnt for all but the last `n` vector-memory operations (vmcnt in bits 3:0 and 15:14, the other counts at their maxima).
template <int N>
SS_DEV void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  asm volatile("" ::: "memory");
}

// This lane's number, worked out anew: what a kernel derives from it then takes no register up to there.
SS_DEV int fresh_lane() {
  uint32_t none = 0;
  asm volatile("" : "+v"(none));
  return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
}

// Where the 16-byte piece p of a key row lies: at p ^ key_swizzle(row). The 16 rows of an operand read differ in bits 0, 1, 3
// and 4; a row of 64 dimensions is half of the 256 bytes that the banks cover (bit 0 says which), the others cover them.
template <int D>
SS_DEV constexpr int key_swizzle(int row) {
  return D == 64 ? ((row >> 1) & 1) | ((row >> 3) & 3) << 1 : (row & 3) | ((row >> 3) & 3) << 2;
}
// The same of e4m3 rows, which are half as long and whose operand reads differ in bits 0, 1, 4 and 5.
template <int D>
SS_DEV constexpr int key_swizzle8(int row) {
  return D == 64 ? (row >> 4) & 3 : D == 128 ? ((row >> 1) & 1) | ((row >> 4) & 3) << 1 : (row & 3) | ((row >> 4) & 3) << 2;
}

// E8: pages of e4m3 numbers with scales (T is Bf16). TREE: rows see what their masks say.
template <class T, int D, int NT, bool E8, bool TREE>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(AttnArgs a) {
  constexpr int W = 4, KS = D / 32, DT = D / 16, EB = E8 ? 1 : 2;  // EB: bytes of an element
  constexpr bool kQLds = NT * KS > 8;  // more than 32 registers of queries stay in LDS, one copy for the waves
  // A tile is U units of 32 tokens, so that the slots hold as many bytes of either kind; G tokens of a 16-byte piece of values.
  constexpr int U = E8 ? 2 : 1, TT = 32 * U, G = 8 * U;
  constexpr int KROW = D * EB, KC = KROW / 16, SLOT = TT * KROW;  // bytes of a key row, its pieces; bytes of a slot
  constexpr int LI = SLOT / 1024;                            // load instructions of a slot
  // Column tiles whose scores are worked out at once: of four of e4m3, or two of 256 dimensions, the scores would take the registers
  // that there are, so the keys are read (and widened) once for each half.
  constexpr int NB = E8 && (NT == 4 || (TREE && D == 256 && NT == 2)) ? NT / 2 : NT;
  constexpr int RK = 64 / KC;                                // key rows of one (of values 16: a row is 64 bytes)
  constexpr int JH = 2, JD = D / JH;  // the waves' sums are joined in two halves of the dimensions, one where the keys were
  // Keys and queries in dynamic LDS: where all of it is static and leaves room for one workgroup a CU, the compiler takes 512
  // registers a wave and moves sums between their halves for every product (8 sequences of up to 6,145 tokens, 3 rows, 256
  // dimensions: 22.4 us; so 21.2).
  extern __shared__ __attribute__((aligned(1024))) uint8_t dyn_lds[];
  __shared__ __attribute__((aligned(1024))) uint8_t v_slot[W][SLOT];
  uint8_t* const k_slot = dyn_lds;
  ss_u32x4(*const q_lds)[64] = reinterpret_cast<ss_u32x4(*)[64]>(dyn_lds + W * SLOT);
  __shared__ __attribute__((aligned(16))) int32_t page_of[512];  // page of each G-token group of the chunk, -1: none
  __shared__ __attribute__((aligned(16))) uint8_t exp_slot[E8 ? W : 1][E8 ? 256 : 16];  // exponents of a tile's keys, of its values
  __shared__ uint64_t qmask[TREE ? NT * 16 : 1];  // masks of the columns' rows
  __shared__ float join_m[W][NT][16], join_l[W][NT][16];
  __shared__ ss_f32x4 join_f[NT * 16];
  __shared__ int64_t join_at[NT * 16];
  __shared__ int32_t qpos[NT * 16];  // positions of the columns' rows, -1: none
  typedef float JoinRow[16][JD + 4];
  JoinRow* const join_o[JH] = {reinterpret_cast<JoinRow*>(k_slot), reinterpret_cast<JoinRow*>(&v_slot[0][0])};
  static_assert(sizeof(JoinRow) <= SLOT, "the waves' sums fit the slots");
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  // Slot by slot, so that those which have work are neighbours: of a table wider than its sequences they are the first ones. (Workgroups
  // are dealt to the 8 XCDs and their CUs in turn: with a sequence's slots side by side every 32nd had work on a table of 32 slots,
  // all on one XCD. 64 sequences of up to 2,000 tokens and 8 key heads on tables of 2,112 / 8,192 / 32,768 / 131,072 tokens: 63 / 67 /
  // 68 / 85 us, so 63 / 98 / 283 / 902; of up to 16,384 on 16,448 and 131,072 483 and 486, so 539 and 2,950.)
  const uint32_t units = (uint32_t)(a.tiles * a.kv_heads) * (uint32_t)a.seqs;
  const int slot = blockIdx.x / units;
  uint32_t b = blockIdx.x - slot * units;
  const int tile = b % (uint32_t)a.tiles;
  b /= (uint32_t)a.tiles;
  const int h = b % (uint32_t)a.kv_heads, s = b / (uint32_t)a.kv_heads;
  const int page = 1 << a.page_shift;
  // Without a window the chunk is the slot, and its pages are asked for before the sequence's length is known.
  const bool all = a.window >= (1 << 30);
  const int32_t* tab = a.table + (int64_t)s * a.width;
  auto entry = [&](int t) { return gp(tab)[min(t >> a.page_shift, a.width - 1)]; };
  int early = -1;
  if (all && G * tid < a.chunk) early = entry(slot * a.chunk + G * tid);
  const SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, (int64_t)a.width * page, a.err);
  const int p0 = tile * NT * 16, np = sr.n * a.group;  // packed rows [p0, min(p0 + 16 NT, np))
  if (p0 >= np) return;                                // whole workgroup, before any barrier
  const uint32_t group = a.group;
  const int i0 = p0 / group, i1 = (min(p0 + NT * 16, np) - 1) / group;
  // The positions that the workgroup's rows have (a tree's rows lie anywhere among the sequence's new ones).
  const int pos_lo = TREE ? sr.pos0 : sr.pos0 + i0, pos_hi = TREE ? sr.pos0 + sr.n - 1 : sr.pos0 + i1;
  const Seen sn = seen_tokens(pos_lo, pos_hi, sr.end, a.window, a.sinks);
  // Slots cover the chunks that hold first tokens, then those from the window's on.
  const int sc = (sn.s_end + a.chunk - 1) / a.chunk;
  const int wc = max(sn.w_begin / a.chunk, sc);
  const int ch = slot < sc ? slot : wc + slot - sc;
  const int t_begin = ch * a.chunk, t_end = min(t_begin + a.chunk, sn.end);
  if (t_begin >= t_end && a.slots > 1) return;  // the join reads no further than the last token's chunk

  for (int j = tid; j < a.chunk / G; j += 64 * W) {
    const int t = t_begin + G * j;
    int id = -1;
    if (t < t_end) {
      id = all && j == tid ? early : entry(t);
      if ((uint32_t)id >= (uint32_t)a.n_pages) {
        id = -1;
        if (t < sn.s_end || t + G > sn.w_begin) raise_bit(a.err, SS_ERR_PAGE);
      }
    }
    page_of[j] = id;
  }
  // Queries: the four waves share the loads where they stay in LDS. They are not waited for before the tiles' first loads.
  ss_u32x4 qf[kQLds ? 1 : NT][KS];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int p = p0 + 16 * n + c, i = p / group;
    const bool in = p < np;
    if constexpr (TREE) {
      if (w == 0 && g == 0) {  // a row's position: as many rows behind the cache as it sees, one at least
        const uint64_t mine = in ? gp(a.tree)[sr.r0 + i] & (~0ull >> (64 - sr.n)) : 0;
        qmask[16 * n + c] = mine;
        qpos[16 * n + c] = in ? sr.pos0 + max(__builtin_popcountll(mine), 1) - 1 : -1;
      }
    } else {
      if (w == 0) qpos[16 * n + c] = in ? sr.pos0 + i : -1;
    }
    // Of e4m3 a 16-byte piece of a key has 16 dimensions, for two products: lane g's of the products 2 k and 2 k + 1 are 64 k + 16 g ...
    const uint16_t* qp = a.q + (int64_t)(sr.r0 + (in ? i : 0)) * a.q_row +
                         (int64_t)(h * a.group + (in ? p - i * a.group : 0)) * a.q_head + 8 * U * g;
    auto dim_of = [](int ks) { return E8 ? 64 * (ks / 2) + 8 * (ks % 2) : 32 * ks; };
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (kQLds) {
        if ((n * KS + ks) % W == w) dma16<0>(qp + dim_of(ks), &q_lds[n * KS + ks][0]);
      } else {
        qf[n][ks] = *(const SS_G ss_u32x4*)(qp + dim_of(ks));
      }
    }
  }
  ss_f32x4 acc[NT][DT];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = kNegInf;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[n][d] = ss_f32x4{0.f, 0.f, 0.f, 0.f};
  }
  local_barrier();

  const int nt = (t_end - t_begin + TT - 1) / TT;
  // The wave's tiles: w, w + W, ... but those that no row sees, from the first tokens' end to the window's begin.
  constexpr int TSH = E8 ? 6 : 5;  // log2 of TT
  const int gap_a = (sn.s_end - t_begin + TT - 1) >> TSH, gap_b = (sn.w_begin - t_begin) >> TSH;
  auto next_tile = [&](int tt) {
    if (tt >= gap_a && tt < gap_b) tt = gap_b + ((tt - gap_b) & (W - 1));
    return tt;
  };
  // Whether every row of the workgroup sees all tokens of a tile (of a tree, whose rows may see none, in the cache before it).
  auto whole = [&](int t0, int idv) {
    return t0 + TT - 1 <= (TREE ? pos_lo - 1 : pos_lo) && (t0 > pos_hi - a.window || t0 + TT <= a.sinks) && __all(idv >= 0);
  };
  auto sees = [&](int tok, int pos, int idv) {
    return idv >= 0 && tok <= pos && (tok > pos - a.window || tok < a.sinks);
  };
  // Of the tokens first .. first + 7, in a page `idv`, those that column `col` sees, a bit each (trees).
  auto tree_bits = [&](int first, int col, int idv) {
    return idv < 0 ? 0u : tree_sees(first, sr.pos0, sr.end, qmask[TREE ? col : 0], qpos[col], a.window, a.sinks);
  };
  const uint32_t page_bytes = (uint32_t)a.kv_heads * page * D * EB;
  const char* kbase = reinterpret_cast<const char*>(a.k) + (int64_t)h * page * D * EB;
  const char* vbase = reinterpret_cast<const char*>(a.v) + (int64_t)h * page * D * EB;
  uint8_t* kl = k_slot + w * SLOT;
  uint8_t* vl = v_slot[w];
  // What this lane fetches: in its n-th load of keys row n RK + lane / KC, of values row (dimension) 16 n + lane / 4. The rows
  // of G keys lie as close in a page as in the slot, so one address serves them with a constant added to both.
  constexpr auto swizzle = [](int row) { return E8 ? key_swizzle8<D>(row) : key_swizzle<D>(row); };
  const uint32_t koff = (lane / KC) * KROW + 16 * ((lane % KC) ^ swizzle(lane / KC));
  const int vpiece0 = (lane & 3) ^ ((lane >> 4) & 3);
  auto load_k = [&](int tt) {
    const int4 ids = *reinterpret_cast<const int4*>(&page_of[4 * tt]);
    const int id[4] = {ids.x, ids.y, ids.z, ids.w};
    uint32_t ko = koff;
    if constexpr (E8) {
      const int ln = fresh_lane();
      ko = (ln / KC) * KROW + 16 * ((ln % KC) ^ swizzle(ln / KC));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = __builtin_amdgcn_readfirstlane(max(id[j], 0));
      const uint32_t tok = (t_begin + TT * tt + G * j) & (page - 1);
      const char* from = kbase + ((uint64_t)at * page_bytes + tok * KROW);
      uint8_t* to = kl + G * KROW * j;
      if constexpr (E8) {
        // The places go by one register (kept for every row group they would take 16).
        dma16_at<0>(from, ko ^ (16 * swizzle(G * j)), to);
        if constexpr (LI >= 8) dma16_at<1024>(from, ko ^ (16 * swizzle(G * j + RK)), to);
        if constexpr (LI >= 16) {
          dma16_at<2048>(from, ko ^ (16 * swizzle(G * j + 2 * RK)), to);
          dma16_at<3 * 1024>(from, ko ^ (16 * swizzle(G * j + 3 * RK)), to);
        }
        continue;
      }
      dma16<0>(from + (koff ^ (16 * swizzle(G * j))), to);
      if constexpr (LI >= 8) dma16<1024>(from + (koff ^ (16 * swizzle(G * j + RK))), to);
      if constexpr (LI >= 16) {
        dma16<2048>(from + (koff ^ (16 * swizzle(G * j + 2 * RK))), to);
        dma16<3 * 1024>(from + (koff ^ (16 * swizzle(G * j + 3 * RK))), to);
      }
    }
    if constexpr (E8) {  // the exponents of 4 tokens a lane, keys' and values' (the upper 32 lanes do the same again)
      const int ln = fresh_lane(), q = ln & 15, id = page_of[4 * tt + q / 4];
      const int64_t at = ((int64_t)max(id, 0) * a.kv_heads + h) * 2 + ((ln >> 4) & 1);
      dma4(a.scales + at * page + ((t_begin + TT * tt + 4 * q) & (page - 1)), exp_slot[w]);
    }
  };
  auto load_v = [&](int tt) {
    const int ln = E8 ? fresh_lane() : lane, vpiece = E8 ? (ln & 3) ^ ((ln >> 4) & 3) : vpiece0;
    const int id = page_of[4 * tt + vpiece], tok = (t_begin + TT * tt + G * vpiece) & (page - 1);
    const char* at = vbase + ((uint64_t)(uint32_t)max(id, 0) * page_bytes + ((ln >> 2) * page + tok) * EB);
    const int64_t step = 16 * EB * page;
#pragma unroll
    for (int n = 0; n < LI; n += 4) {
      dma16<0>(at, vl + 1024 * n);
      dma16<1024>(at += step - 1024, vl + 1024 * n);
      dma16<2048>(at += step - 1024, vl + 1024 * n);
      dma16<3 * 1024>(at += step - 1024, vl + 1024 * n);
      at += step + 3 * 1024;
    }
  };
  auto kread = [&](int t, int ks) {
    const int row = 8 * (c >> 2) + 4 * t + (c & 3);
    return *reinterpret_cast<const ss_u32x4*>(kl + row * KROW + 16 * ((4 * ks + g) ^ key_swizzle<D>(row)));
  };
  // The 16 bytes of a lane's tokens of dimension 16 d + c: of e4m3 those of both units.
  auto vread = [&](int d) {
    return *reinterpret_cast<const ss_u32x4*>(vl + (16 * d + c) * 64 + 16 * (g ^ ((c >> 2) & 3)));
  };
  // Row m of the score tile t of unit u is token 16 (m / 4) + 8 u + 4 t + m % 4 of e4m3, so that a lane ends with tokens G g + 8 u + 4 t + 0..3.
  // The swizzle is that of the row with u = t = 0, so all places are one (kat0) by exclusive or and a constant.
  const int krow0 = 16 * (c >> 2) + (c & 3);
  const uint32_t kat0 = krow0 * KROW + 16 * (g ^ swizzle(krow0));
  auto kread8 = [&](uint32_t kat, int u, int t, int kp) {
    return *reinterpret_cast<const ss_u32x4*>(kl + (kat ^ (64 * kp)) + (8 * u + 4 * t) * KROW);
  };
  bool any_odd = false;
  // The loop's first turn has no tile yet and only loads. A wave issues an instruction in some 5 cycles, so short calls go by
  // how many they execute: with the first loads in the loop, one address for 8 keys, the columns' factors worked out
  // once and the maximum raised lazily, a sequence of 32 tokens takes 8.4 us at 256 dimensions and two column tiles (12.5
  // without), 4.2 at 128 and one (4.5).
  int tt = nt > 0 ? -1 : 0, tn = next_tile(w);
#pragma unroll 1
  while (tt < nt) {
    const int t0 = t_begin + TT * tt, idv = page_of[4 * max(tt, 0) + g];
    const bool more = tn < nt;
    const bool part_seen = !whole(t0, idv);
    ss_u32x4 pf[NT][U];
    ss_f32x4 sv[NB][2 * U];
    ss_u32x4 vexp;  // exponents of the lane's values
    auto scores = [&](int n0) {  // of the column tiles n0 .. n0 + NB - 1
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int t = 0; t < 2 * U; ++t) sv[n][t] = ss_f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (E8) {
        const ss_u32x4 kexp = *reinterpret_cast<const ss_u32x4*>(&exp_slot[w][16 * (c >> 2)]);
        float by[4];
        uint32_t kat = kat0;
        asm volatile("" : "+v"(kat));
#pragma unroll
        for (int t = 0; t < 4; ++t) by[t] = scale_of((kexp[t] >> (8 * (c & 3))) & 0xFFu);
#pragma unroll
        for (int kp = 0; kp < KS / 2; ++kp) {
          if constexpr (NT * D >= 256) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const ss_u32x4 k8 = kread8(kat, t / 2, t % 2, kp);
            const ss_u32x4 k0 = widen8(k8[0], k8[1], by[t]), k1 = widen8(k8[2], k8[3], by[t]);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              const int q = (n0 + n) * KS + 2 * kp;
              sv[n][t] = T::mfma16(k0, kQLds ? q_lds[q][lane] : qf[kQLds ? 0 : n0 + n][2 * kp], sv[n][t]);
              sv[n][t] = T::mfma16(k1, kQLds ? q_lds[q + 1][lane] : qf[kQLds ? 0 : n0 + n][2 * kp + 1], sv[n][t]);
            }
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const ss_u32x4 kf = kread(t, ks);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              sv[n][t] = T::mfma16(kf, kQLds ? q_lds[n * KS + ks][lane] : qf[kQLds ? 0 : n][ks], sv[n][t]);
          }
      }
    };
    auto vby = [&](int e) {  // the power of two of the values of the lane's token e
      const uint32_t word = vexp[e / 4], at = 8 * (e % 4);
      return ss_uf((at < 23 ? word << (23 - at) : word >> (at - 23)) & 0x7F800000u);
    };
    auto weights = [&](int n0) {
#pragma unroll
      for (int n = n0; n < n0 + NB; ++n) {
        float x[8 * U];
#pragma unroll
        for (int e = 0; e < 8 * U; ++e) x[e] = sv[n - n0][e / 4][e % 4];
        if (part_seen) {
          if constexpr (TREE) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const uint32_t see = tree_bits(t0 + G * g + 8 * u, 16 * n + c, idv);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[8 * u + e] = (see >> e) & 1u ? x[8 * u + e] : kNegInf;
            }
          } else {
            const int pos = qpos[16 * n + c];
#pragma unroll
            for (int e = 0; e < 8 * U; ++e) x[e] = sees(t0 + G * g + e, pos, idv) ? x[e] : kNegInf;
          }
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 8 * U; ++e) mx = fmaxf(mx, x[e]);
        mx = max_over_quads(mx) * a.scale - T::kShift;
        // The maximum is raised where it is passed by more than kLazy: the weights are at most 2^kLazy until then.
        const float mn = mx > m[n] + T::kLazy ? mx : m[n];
        const float mu = mn == kNegInf ? 0.f : mn;
        if (__any(mn > m[n] && m[n] != kNegInf)) {
          const float f = __builtin_amdgcn_exp2f(m[n] - mu);
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][d][i] *= f;
        }
        m[n] = mn;
        float p[8 * U];
#pragma unroll
        for (int e = 0; e < 8 * U; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale, -mu));
          l[n] += p[e];
          if constexpr (E8) p[e] *= vby(e);
        }
        // A weight is rounded to the element type here, once, as the matrix unit takes it (a half step of it, as much as the result's
        // own rounding); the row's sum has the weights before that.
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) pf[n][u][i] = T::pack(p[8 * u + 2 * i], p[8 * u + 2 * i + 1]);
        if constexpr (E8) __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (tt >= 0) {
      wait_loads<LI>();  // this tile's keys are there, its values may be on their way
      if constexpr (E8) {
        vexp = *reinterpret_cast<const ss_u32x4*>(&exp_slot[w][64 + 16 * g]);
        if (part_seen) {  // a place that no row sees may hold 255: 254 is finite
#pragma unroll
          for (int e = 0; e < 4; ++e) vexp[e] &= ~((((vexp[e] & 0x7F7F7F7Fu) + 0x01010101u) & vexp[e] & 0x80808080u) >> 7);
        }
      }
#pragma unroll
      for (int n0 = 0; n0 < NT - NB; n0 += NB) {
        scores(n0);
        weights(n0);
      }
      scores(NT - NB);
    }
    __builtin_amdgcn_sched_barrier(0);  // the reads above have been used, so the slot may be filled again
    if (more) load_k(tn);
    if (tt >= 0) {
      weights(NT - NB);
      // This tile's values are there, the next one's keys may be on their way.
      if (more)
        wait_loads<E8 ? LI + 1 : LI>();
      else
        wait_loads<0>();
      bool odd = false;
      if (part_seen) {  // zero times the values is zero where all are finite
        ss_f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const ss_u32x4 vf = vread(d);
          if constexpr (E8) {
            z = T::mfma16(widen8(vf[0], vf[1], 1.f), ss_u32x4{0u, 0u, 0u, 0u}, z);
            z = T::mfma16(widen8(vf[2], vf[3], 1.f), ss_u32x4{0u, 0u, 0u, 0u}, z);
          } else {
            z = T::mfma16(vf, ss_u32x4{0u, 0u, 0u, 0u}, z);
          }
        }
        odd = __any(z[0] != 0.f || z[1] != 0.f || z[2] != 0.f || z[3] != 0.f);
        any_odd |= odd;
      }
      if (odd) {  // the wave's own slot: cleaned in place
#pragma unroll 1
        for (int d = 0; d < DT; ++d) {
          const ss_u32x4 vf = vread(d);
          *reinterpret_cast<ss_u32x4*>(vl + (16 * d + c) * 64 + 16 * (g ^ ((c >> 2) & 3))) =
              E8 ? ss_u32x4{without_nan8(vf[0]), without_nan8(vf[1]), without_nan8(vf[2]), without_nan8(vf[3])} : parts_of<T>(vf, -1);
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const ss_u32x4 vf = vread(d);
        if constexpr (E8) {
          const ss_u32x4 v0 = widen8(vf[0], vf[1], 1.f), v1 = widen8(vf[2], vf[3], 1.f);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n][d] = T::mfma16(v0, pf[n][0], acc[n][d]);
            acc[n][d] = T::mfma16(v1, pf[n][U - 1], acc[n][d]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[n][d] = T::mfma16(vf, pf[n][0], acc[n][d]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_v(tn);
    if constexpr (kQLds)
      if (tt < 0) {
        if (more)
          wait_loads<E8 ? 2 * LI + 1 : 2 * LI>();  // the queries are older than the tile
        else
          wait_loads<0>();
        local_barrier();
      }
    tt = tn;
    tn = next_tile(tt + W);
  }
  wait_loads<0>();  // no load into LDS outlives the tiles (without tiles the queries are on their way)

  const int lane_was = lane;
  {
  const int lane = E8 ? fresh_lane() : lane_was, c = lane & 15, g = lane >> 4, tid = 64 * w + lane;
  // The waves' sums, weighted by how far each wave's maximum is below the largest.
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = ss_rows_sum(l[n]);
    if (g == 0) {
      join_m[w][n][c] = m[n];
      join_l[w][n][c] = l[n];
    }
  }
  local_barrier();  // all waves are done with their tiles as well
  const float* const jm = &join_m[0][0][0];
  const float* const jl = &join_l[0][0][0];
  if (tid < 16 * NT && p0 + tid < np) {
    // A column: the waves' factors, and where its row and head lie.
    constexpr int WS = 16 * NT;
    float big = kNegInf, sum = 0.f;
    ss_f32x4 f;
#pragma unroll
    for (int k = 0; k < W; ++k) big = fmaxf(big, jm[WS * k + tid]);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float mk = jm[WS * k + tid];
      f[k] = mk == kNegInf ? 1.f : __builtin_amdgcn_exp2f(mk - big);
      sum += jl[WS * k + tid] * f[k];
    }
    uint32_t group = a.group;
    if constexpr (E8) asm volatile("" : "+s"(group));  // else the reciprocal of the queries' division is kept over the tiles
    const int p = p0 + tid, i = p / group;
    int64_t at = (int64_t)(sr.r0 + i) * a.heads + h * a.group + (p - i * a.group);
    if (a.slots > 1) {
      at += (int64_t)slot * a.rows * a.heads;
      gp(a.pml)[2 * at] = big;
      gp(a.pml)[2 * at + 1] = sum;
    } else {
      const float r = sum == 0.f ? 0.f : 1.f / sum;
      if (a.lse) a.lse[at] = sum == 0.f ? kNegInf : (big + __log2f(sum)) * 0.693147180559945309f;
#pragma unroll
      for (int k = 0; k < W; ++k) f[k] *= r;
    }
    join_f[tid] = f;
    join_at[tid] = at * D;
  }
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    if (n) local_barrier();  // the last columns are read
#pragma unroll
    for (int k = 0; k < NT; ++k)
      if (k == n) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<ss_f32x4*>(&join_o[d / (DT / JH)][w][c][16 * (d % (DT / JH)) + 4 * g]) = acc[k][d];
      }
    if (any_odd) {
      // Infinities and NaN that were taken out of the wave's tiles, to the columns that see them.
      const int pos = qpos[16 * n + c];
#pragma unroll 1
      for (int tt = next_tile(w); tt < nt; tt = next_tile(tt + W)) {
        const int t0 = t_begin + TT * tt, idv = page_of[4 * tt + g];
        if (whole(t0, idv)) continue;
#pragma unroll 1
        for (int du = 0; du < DT * U; ++du) {
          const int d = du / U, first = t0 + G * g + 8 * (du % U);
          const char* vp = vbase + (uint64_t)max(idv, 0) * page_bytes + ((int64_t)(16 * d + c) * page + (first & (page - 1))) * EB;
          ss_u32x4 ones, v;
          if constexpr (E8)
            v = widen8(gp((const uint32_t*)vp)[0], gp((const uint32_t*)vp)[1], 1.f);
          else
            v = *(const SS_G ss_u32x4*)vp;
          uint32_t see = 0;
          if constexpr (TREE) see = tree_bits(first, 16 * n + c, idv);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = first + 2 * i;
            const bool s0 = TREE ? (see >> (2 * i)) & 1u : sees(tok, pos, idv);
            const bool s1 = TREE ? (see >> (2 * i + 1)) & 1u : sees(tok + 1, pos, idv);
            ones[i] = (s0 ? T::kOne : 0u) | (s1 ? T::kOne << 16 : 0u);
          }
          float* o = &(d < DT / JH ? join_o[0] : join_o[1])[w][c][16 * (d % (DT / JH)) + 4 * g];
#pragma unroll 1
          for (int kind = E8 ? 2 : 0; kind < 3; ++kind) {
            const float add = kind == 0 ? -kNegInf : kind == 1 ? kNegInf : __builtin_nanf("");
            const ss_f32x4 hits = T::mfma16(parts_of<T>(v, kind), ones, ss_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (hits[i] > 0.f) o[i] += add;
          }
        }
      }
    }
    local_barrier();
    const int d4 = 4 * (tid % (D / 4));
    const JoinRow* jo = d4 < JD ? join_o[0] : join_o[1];
#pragma unroll 1
    for (int col = tid / (D / 4); col < min(16, np - p0 - 16 * n); col += 1024 / D) {
      const ss_f32x4 f = join_f[16 * n + col];
      ss_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const ss_f32x4 x = *reinterpret_cast<const ss_f32x4*>(&jo[k][col][d4 % JD]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += x[i] * f[k];
      }
      const int64_t at = join_at[16 * n + col] + d4;
      if (a.slots > 1) {
        *reinterpret_cast<SS_G ss_f32x4*>(gp(a.po) + at) = o;
      } else {
        uint2 word;
        word.x = T::pack(o[0], o[1]);
        word.y = T::pack(o[2], o[3]);
        *reinterpret_cast<uint2*>(a.out + at) = word;
      }
    }
  }
  }
}

template <class T, int D, int NT, bool E8, bool TREE>
hipError_t launch_few(const AttnArgs& a, hipStream_t st) {
  constexpr size_t kDyn = 4 * 32 * D * 2 + (NT * D / 32 > 8 ? NT * (D / 32) * 1024 : 0);  // key slots, queries
  const auto kern = attn_few_kernel<T, D, NT, E8, TREE>;
  KernelCfg cfg;
  const hipError_t e = kernel_cfg(reinterpret_cast<const void*>(kern), 256, kDyn, &cfg);  // raises the kernel's LDS limit
  if (e != hipSuccess) return e;
  const unsigned grid = (unsigned)((int64_t)a.slots * a.tiles * a.kv_heads * a.seqs);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), kDyn, st, a);
  return hipGetLastError();
}

template <class T, bool E8, bool TREE>
hipError_t launch_few_of(const AttnArgs& a, int dim, hipStream_t st) {
  const int nt = a.packed / 16;
  if (dim == 64)
    return nt == 1   ? launch_few<T, 64, 1, E8, TREE>(a, st)
           : nt == 2 ? launch_few<T, 64, 2, E8, TREE>(a, st)
                     : launch_few<T, 64, 4, E8, TREE>(a, st);
  if constexpr (!E8)
    if (dim == 128 && nt == 4) return launch_few<T, 128, 4, E8, TREE>(a, st);
  if (dim == 128) return nt == 1 ? launch_few<T, 128, 1, E8, TREE>(a, st) : launch_few<T, 128, 2, E8, TREE>(a, st);
  return nt == 1 ? launch_few<T, 256, 1, E8, TREE>(a, st) : launch_few<T, 256, 2, E8, TREE>(a, st);
}

}  // namespace

}  // namespace ss
