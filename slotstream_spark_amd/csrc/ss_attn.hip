// Attention of a batch's few new rows (a decoded token, the rows of a verify round) over a paged cache.
//
// For row i at position p, o_i = sum_j softmax_j(scale q_i k_j) v_j over the tokens j <= p, under a window those with
// p - j < window or j < sinks. Every key and value is used by the few rows of a sequence and the heads that share its key
// head, so the work is reading the cache once: 4 dim bytes per token and key head.
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
// Measured, kernel alone: 64 sequences of up to 16,384 tokens (32 heads on 8, 128 dimensions, 2.7 GB) 478 us, 5.7 TB/s, where a
// streaming read reaches 5.3; one of 131,072 tokens (268 MB) 42 us; one of 777 5.2 us, the chain of a sequence's place, its
// pages, its keys and the columns' sums. Operands straight from memory into registers took 8 % longer for the first.
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
template <int OFF>  // bytes added to both addresses
SS_DEV void dma16(const void* src, void* lds) { __builtin_amdgcn_global_load_lds(src, (lds_void*)lds, 16, OFF, 0); }

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

// Where the 16-byte piece p of a key row lies: at p ^ key_swizzle(row). The 16 rows of an operand read differ in bits 0, 1, 3
// and 4; a row of 64 dimensions is half of the 256 bytes that the banks cover (bit 0 says which), the others cover them.
template <int D>
SS_DEV constexpr int key_swizzle(int row) {
  return D == 64 ? ((row >> 1) & 1) | ((row >> 3) & 3) << 1 : (row & 3) | ((row >> 3) & 3) << 2;
}

template <class T, int D, int NT>
__global__ __launch_bounds__(256, 2) void attn_few_kernel(AttnArgs a) {
  constexpr int W = 4, KS = D / 32, DT = D / 16;
  constexpr bool kQLds = NT * KS > 8;  // more than 32 registers of queries stay in LDS, one copy for the waves
  constexpr int KROW = D * 2, KC = D / 8, SLOT = 32 * KROW;  // bytes of a key row, its pieces; bytes of a slot
  constexpr int LI = SLOT / 1024;                            // load instructions of a slot
  constexpr int RK = 64 / KC;                                // key rows of one (of values 16: a row is 64 bytes)
  constexpr int JH = 2, JD = D / JH;  // the waves' sums are joined in two halves of the dimensions, one where the keys were
  // Keys and queries in dynamic LDS: where all of it is static and leaves room for one workgroup a CU, the compiler takes 512
  // registers a wave and moves sums between their halves for every product (8 sequences of up to 6,145 tokens, 3 rows, 256
  // dimensions: 22.4 us; so 21.2).
  extern __shared__ __attribute__((aligned(1024))) uint8_t dyn_lds[];
  __shared__ __attribute__((aligned(1024))) uint8_t v_slot[W][SLOT];
  uint8_t* const k_slot = dyn_lds;
  ss_u32x4(*const q_lds)[64] = reinterpret_cast<ss_u32x4(*)[64]>(dyn_lds + W * SLOT);
  __shared__ __attribute__((aligned(16))) int32_t page_of[512];  // page of each 8-token group of the chunk, -1: none
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
  if (all && 8 * tid < a.chunk) early = entry(slot * a.chunk + 8 * tid);
  const SeqRows sr = seq_rows(a.cu, a.kv_len, s, a.rows, a.max_rows, (int64_t)a.width * page, a.err);
  const int p0 = tile * NT * 16, np = sr.n * a.group;  // packed rows [p0, min(p0 + 16 NT, np))
  if (p0 >= np) return;                                // whole workgroup, before any barrier
  const uint32_t group = a.group;
  const int i0 = p0 / group, i1 = (min(p0 + NT * 16, np) - 1) / group;
  const int pos_lo = sr.pos0 + i0, pos_hi = sr.pos0 + i1;
  const Seen sn = seen_tokens(pos_lo, pos_hi, sr.end, a.window, a.sinks);
  // Slots cover the chunks that hold first tokens, then those from the window's on.
  const int sc = (sn.s_end + a.chunk - 1) / a.chunk;
  const int wc = max(sn.w_begin / a.chunk, sc);
  const int ch = slot < sc ? slot : wc + slot - sc;
  const int t_begin = ch * a.chunk, t_end = min(t_begin + a.chunk, sn.end);
  if (t_begin >= t_end && a.slots > 1) return;  // the join reads no further than the last token's chunk

  for (int j = tid; j < a.chunk / 8; j += 64 * W) {
    const int t = t_begin + 8 * j;
    int id = -1;
    if (t < t_end) {
      id = all && j == tid ? early : entry(t);
      if ((uint32_t)id >= (uint32_t)a.n_pages) {
        id = -1;
        if (t < sn.s_end || t + 8 > sn.w_begin) raise_bit(a.err, SS_ERR_PAGE);
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
    if (w == 0) qpos[16 * n + c] = in ? sr.pos0 + i : -1;
    const uint16_t* qp = a.q + (int64_t)(sr.r0 + (in ? i : 0)) * a.q_row +
                         (int64_t)(h * a.group + (in ? p - i * a.group : 0)) * a.q_head + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (kQLds) {
        if ((n * KS + ks) % W == w) dma16<0>(qp + 32 * ks, &q_lds[n * KS + ks][0]);
      } else {
        qf[n][ks] = *(const SS_G ss_u32x4*)(qp + 32 * ks);
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

  const int nt = (t_end - t_begin + 31) / 32;
  // The wave's tiles: w, w + W, ... but those that no row sees, from the first tokens' end to the window's begin.
  const int gap_a = (sn.s_end - t_begin + 31) >> 5, gap_b = (sn.w_begin - t_begin) >> 5;
  auto next_tile = [&](int tt) {
    if (tt >= gap_a && tt < gap_b) tt = gap_b + ((tt - gap_b) & (W - 1));
    return tt;
  };
  // Whether every row of the workgroup sees all 32 tokens.
  auto whole = [&](int t0, int idv) {
    return t0 + 31 <= pos_lo && (t0 > pos_hi - a.window || t0 + 32 <= a.sinks) && __all(idv >= 0);
  };
  auto sees = [&](int tok, int pos, int idv) {
    return idv >= 0 && tok <= pos && (tok > pos - a.window || tok < a.sinks);
  };
  const uint32_t page_bytes = (uint32_t)a.kv_heads * page * D * 2;
  const char* kbase = reinterpret_cast<const char*>(a.k) + (int64_t)h * page * D * 2;
  const char* vbase = reinterpret_cast<const char*>(a.v) + (int64_t)h * page * D * 2;
  uint8_t* kl = k_slot + w * SLOT;
  uint8_t* vl = v_slot[w];
  // What this lane fetches: in its n-th load of keys row n RK + lane / KC, of values row (dimension) 16 n + lane / 4. The rows
  // of 8 keys lie as close in a page as in the slot, so one address serves them with a constant added to both.
  const uint32_t koff = (lane / KC) * KROW + 16 * ((lane % KC) ^ key_swizzle<D>(lane / KC));
  const int vpiece = (lane & 3) ^ ((lane >> 4) & 3);
  auto load_k = [&](int tt) {
    const int4 ids = *reinterpret_cast<const int4*>(&page_of[4 * tt]);
    const int id[4] = {ids.x, ids.y, ids.z, ids.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = __builtin_amdgcn_readfirstlane(max(id[j], 0));
      const uint32_t tok = (t_begin + 32 * tt + 8 * j) & (page - 1);
      const char* from = kbase + ((uint64_t)at * page_bytes + tok * KROW);
      uint8_t* to = kl + 8 * KROW * j;
      dma16<0>(from + (koff ^ (16 * key_swizzle<D>(8 * j))), to);
      if constexpr (LI >= 8) dma16<1024>(from + (koff ^ (16 * key_swizzle<D>(8 * j + RK))), to);
      if constexpr (LI >= 16) {
        dma16<2048>(from + (koff ^ (16 * key_swizzle<D>(8 * j + 2 * RK))), to);
        dma16<3 * 1024>(from + (koff ^ (16 * key_swizzle<D>(8 * j + 3 * RK))), to);
      }
    }
  };
  auto load_v = [&](int tt) {
    const int id = page_of[4 * tt + vpiece], tok = (t_begin + 32 * tt + 8 * vpiece) & (page - 1);
    const char* at = vbase + ((uint64_t)(uint32_t)max(id, 0) * page_bytes + ((lane >> 2) * page + tok) * 2);
    const int64_t step = 32 * page;
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
  auto vread = [&](int d) {
    return *reinterpret_cast<const ss_u32x4*>(vl + (16 * d + c) * 64 + 16 * (g ^ ((c >> 2) & 3)));
  };
  bool any_odd = false;
  // The loop's first turn has no tile yet and only loads. A wave issues an instruction in some 5 cycles, so short calls go by
  // how many they execute: with the first loads in the loop, one address for 8 keys, the columns' factors worked out
  // once and the maximum raised lazily, a sequence of 32 tokens takes 8.4 us at 256 dimensions and two column tiles (12.5
  // without), 4.2 at 128 and one (4.5).
  int tt = nt > 0 ? -1 : 0, tn = next_tile(w);
#pragma unroll 1
  while (tt < nt) {
    const int t0 = t_begin + 32 * tt, idv = page_of[4 * max(tt, 0) + g];
    const bool more = tn < nt;
    const bool part_seen = !whole(t0, idv);
    ss_f32x4 sv[NT][2];
    if (tt >= 0) {
      wait_loads<LI>();  // this tile's keys are there, its values may be on their way
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) sv[n][t] = ss_f32x4{0.f, 0.f, 0.f, 0.f};
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
    __builtin_amdgcn_sched_barrier(0);  // the reads above have been used, so the slot may be filled again
    if (more) load_k(tn);
    if (tt >= 0) {
      ss_u32x4 pf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = sv[n][e / 4][e % 4];
        if (part_seen) {
          const int pos = qpos[16 * n + c];
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = sees(t0 + 8 * g + e, pos, idv) ? x[e] : kNegInf;
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
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
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale, -mu));
          l[n] += p[e];
        }
        // A weight is rounded to the element type here, once, as the matrix unit takes it (a half step of it, as much as the result's
        // own rounding); the row's sum has the weights before that.
#pragma unroll
        for (int i = 0; i < 4; ++i) pf[n][i] = T::pack(p[2 * i], p[2 * i + 1]);
      }
      // This tile's values are there, the next one's keys may be on their way.
      if (more)
        wait_loads<LI>();
      else
        wait_loads<0>();
      bool odd = false;
      if (part_seen) {  // zero times the values is zero where all are finite
        ss_f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) z = T::mfma16(vread(d), ss_u32x4{0u, 0u, 0u, 0u}, z);
        odd = __any(z[0] != 0.f || z[1] != 0.f || z[2] != 0.f || z[3] != 0.f);
        any_odd |= odd;
      }
      if (odd) {  // the wave's own slot: cleaned in place
#pragma unroll 1
        for (int d = 0; d < DT; ++d) {
          const ss_u32x4 vf = vread(d);
          *reinterpret_cast<ss_u32x4*>(vl + (16 * d + c) * 64 + 16 * (g ^ ((c >> 2) & 3))) = parts_of<T>(vf, -1);
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const ss_u32x4 vf = vread(d);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][d] = T::mfma16(vf, pf[n], acc[n][d]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_v(tn);
    if constexpr (kQLds)
      if (tt < 0) {
        if (more)
          wait_loads<2 * LI>();  // the queries are older than the tile
        else
          wait_loads<0>();
        local_barrier();
      }
    tt = tn;
    tn = next_tile(tt + W);
  }
  wait_loads<0>();  // no load into LDS outlives the tiles (without tiles the queries are on their way)

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
        const int t0 = t_begin + 32 * tt, idv = page_of[4 * tt + g];
        if (whole(t0, idv)) continue;
        const uint16_t* vp = reinterpret_cast<const uint16_t*>(vbase + (uint64_t)max(idv, 0) * page_bytes) + (int64_t)c * page +
                             ((t0 + 8 * g) & (page - 1));
        ss_u32x4 ones;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = t0 + 8 * g + 2 * i;
          ones[i] = (sees(tok, pos, idv) ? T::kOne : 0u) | (sees(tok + 1, pos, idv) ? T::kOne << 16 : 0u);
        }
#pragma unroll 1
        for (int d = 0; d < DT; ++d) {
          const ss_u32x4 v = *(const SS_G ss_u32x4*)(vp + (int64_t)16 * d * page);
          float* o = &(d < DT / JH ? join_o[0] : join_o[1])[w][c][16 * (d % (DT / JH)) + 4 * g];
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind) {
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

// Joins the chunks of a row: o = sum_k o_k 2^(m_k - m) / sum_k l_k 2^(m_k - m), m the largest m_k. A row and head is read by
// groups of dim / 4 threads, 16 bytes each. WIDE: its workgroup's groups take the chunks by their number modulo the
// number of groups, each with a running maximum, and the groups' sums are added in order; else one group takes all its
// chunks and a workgroup has as many rows. Either way the order goes by the chunks' numbers alone.
template <class T, int D, bool WIDE>
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
  const Seen sn = seen_tokens(sr.pos0 + p0 / a.group, sr.pos0 + (min(p0 + a.packed, np) - 1) / a.group, sr.end, a.window,
                              a.sinks);
  const int sc = (sn.s_end + a.chunk - 1) / a.chunk, wc = max(sn.w_begin / a.chunk, sc);
  const int used = sc + max((sn.end + a.chunk - 1) / a.chunk - wc, 0);
  const int64_t row = (int64_t)(sr.r0 + i) * a.heads + head, rows = (int64_t)a.rows * a.heads;
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
      const int64_t at = j * rows + row;
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

template <class T, int D, int NT>
hipError_t launch_few(const AttnArgs& a, hipStream_t st) {
  constexpr size_t kDyn = 4 * 32 * D * 2 + (NT * D / 32 > 8 ? NT * (D / 32) * 1024 : 0);  // key slots, queries
  const auto kern = attn_few_kernel<T, D, NT>;
  KernelCfg cfg;
  const hipError_t e = kernel_cfg(reinterpret_cast<const void*>(kern), 256, kDyn, &cfg);  // raises the kernel's LDS limit
  if (e != hipSuccess) return e;
  const unsigned grid = (unsigned)((int64_t)a.slots * a.tiles * a.kv_heads * a.seqs);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), kDyn, st, a);
  return hipGetLastError();
}

template <class T>
hipError_t launch_few_of(const AttnArgs& a, int dim, hipStream_t st) {
  const int nt = a.packed / 16;
  if (dim == 64) return nt == 1 ? launch_few<T, 64, 1>(a, st) : nt == 2 ? launch_few<T, 64, 2>(a, st) : launch_few<T, 64, 4>(a, st);
  if (dim == 128)
    return nt == 1 ? launch_few<T, 128, 1>(a, st) : nt == 2 ? launch_few<T, 128, 2>(a, st) : launch_few<T, 128, 4>(a, st);
  return nt == 1 ? launch_few<T, 256, 1>(a, st) : launch_few<T, 256, 2>(a, st);
}

// More than 16 chunks are joined by a workgroup a row: one row and 32 heads over 12,000 tokens 12.3 us a call with it, 18.9
// without, over 51,000 24.4 and 39.8. Up to 16, where a batch brings the rows, by a group of threads a row: 32 sequences of 4
// rows and 32 heads 186 us a call, 191 with a workgroup each.
template <class T, int D>
hipError_t launch_join(const AttnArgs& a, hipStream_t st) {
  const int64_t all = (int64_t)a.seqs * a.max_rows * a.heads;
  constexpr int GROUPS = 256 / (D / 4);
  if (a.slots > 16)
    hipLaunchKernelGGL((attn_join_kernel<T, D, true>), dim3((unsigned)all), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_join_kernel<T, D, false>), dim3((unsigned)((all + GROUPS - 1) / GROUPS)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <class T>
hipError_t launch_join_of(const AttnArgs& a, int dim, hipStream_t st) {
  return dim == 64 ? launch_join<T, 64>(a, st) : dim == 128 ? launch_join<T, 128>(a, st) : launch_join<T, 256>(a, st);
}

}  // namespace

// Packed rows of a workgroup: as few tiles of 16 as hold them all, up to 4 (2 of 256 dimensions, whose sums of four tiles
// would take every register).
int attn_few_packed(int dim, int packed) {
  if (packed <= 16) return 16;
  return packed <= 32 || dim == 256 ? 32 : 64;
}

hipError_t launch_attn_few(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_few_of<Fp16>(a, dim, st) : launch_few_of<Bf16>(a, dim, st);
}

hipError_t launch_attn_join(const AttnArgs& a, int dim, bool fp16, hipStream_t st) {
  return fp16 ? launch_join_of<Fp16>(a, dim, st) : launch_join_of<Bf16>(a, dim, st);
}

}  // namespace ss
