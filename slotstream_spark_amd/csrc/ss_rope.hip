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
// Into pages of e4m3 numbers (E8) a row's largest magnitude is found first, over the lanes that have its elements in registers already, so each
// byte is still read and written once: the prompt writes 76 MB where 16 bits take 92 (160 MB both ways) in 34 to 36 us, the single
// tokens take 9.1, the maximum's exchanges one more link of the chain.
#include <hip/hip_runtime.h>

#include "ss_attn.hpp"
#include "ss_launch.hpp"
#include "ss_rope.hpp"

namespace ss {

namespace {

// ---------------------------------------------------------------- rows as e4m3 numbers
// A vector x of a token and head is kept as e4m3 numbers of x 2^-e, rounded once from fp32, and the byte e + 127: e the least exponent
// with max |x| <= 448 2^e, from -126 on, of a key turned in 64 bits. The numbers are of keys turned in fp32: off by 2^-20 of the largest,
// beside a code's half step of 2^-4. What is not finite is left out of the maximum and kept as NaN.
SS_DEV float finite_abs(float x) {
  const float y = fabsf(x);
  return y < __builtin_inff() ? y : 0.f;
}
// The byte of a vector whose largest magnitude is `top`: 448 is 1.75 2^8, so the mantissa says which exponent is enough.
SS_DEV uint32_t exponent8(float top) {
  const uint32_t u = ss_fu(top);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 1);
}
// How far an fp32 maximum of turned elements may be from the one in 64 bits, in units of its last place at 1.75 2^n. Where both of a pair
// are at most y, (|p| + |q|) factor <= 2 y. A cosine is off by 2 pi 2^-26 for its angle and 4 2^-24 for itself, times factor by 2^-24; the
// products and their sum by 2^-24 each: 2 (0.94 + 2.4 + 0.6) 10^-7 + 1.8 10^-7 = 9.7 10^-7 of y, 15 units.
constexpr uint32_t kNear = 32;
// x 2^-e for the byte of e, NaN where x is not finite.
SS_DEV float scaled8(float x, float by) { return fabsf(x) < __builtin_inff() ? x * by : __builtin_nanf(""); }
SS_DEV float inverse8(uint32_t byte) { return ss_uf((254u - byte) << 23); }
SS_DEV uint32_t pack8(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// Sine and cosine of a part of a turn in 64 bits: less its quarters it is at most pi / 4, where the series up to x^19 and x^18 are off by
// less than 10^-19. A loop over a table: as straight code (the library's sincospi) it takes more scalar registers than there are.
__constant__ const double kSeries[10][2] = {  // 1 / (2 n + 1)!, 1 / (2 n)!
    {1., 1.}, {1. / 6, 1. / 2}, {1. / 120, 1. / 24}, {1. / 5040, 1. / 720}, {1. / 362880, 1. / 40320},
    {1. / 39916800, 1. / 3628800}, {1. / 6227020800, 1. / 479001600}, {1. / 1307674368000, 1. / 87178291200},
    {1. / 355687428096000, 1. / 20922789888000}, {1. / 121645100408832000, 1. / 6402373705728000}};
SS_DEV void turn64(double part, double* sn, double* cs) {
  const double quarters = __builtin_rint(4. * part), x = (part - 0.25 * quarters) * 6.28318530717958647693, z = -x * x;
  double s = 0., c = 0.;
#pragma unroll 1
  for (int n = 9; n >= 0; --n) {
    s = __builtin_fma(s, z, kSeries[n][0]);
    c = __builtin_fma(c, z, kSeries[n][1]);
  }
  s *= x;
  const int k = (int)quarters & 3;  // of -2 .. 2
  *sn = k == 0 ? s : k == 1 ? c : k == 2 ? -s : -c;
  *cs = k == 0 ? c : k == 1 ? -s : k == 2 ? -c : s;
}
// The maximum over the lanes l ^ 1, ..., l ^ (n - 1), n = 4, 8, 16 or 32.
SS_DEV float max_over(float v, int n) {
  v = fmaxf(v, ss_uf(ss_xor_lane<1>(ss_fu(v))));
  v = fmaxf(v, ss_uf(ss_xor_lane<2>(ss_fu(v))));
  if (n > 4) v = fmaxf(v, ss_uf(ss_xor_lane<4>(ss_fu(v))));
  if (n > 8) v = fmaxf(v, ss_uf(ss_xor_lane<8>(ss_fu(v))));
  if (n > 16) {
    uint32_t lo, hi;
    ss_pair<16>(ss_fu(v), lo, hi);
    v = fmaxf(ss_uf(lo), ss_uf(hi));
  }
  return v;
}

// Key and value rows of the 8 positions from `first` on, into page `id` at `off`.
template <class T>
SS_DEV void append_e4m3(const RopeArgs& a, const SeqRows& sr, int first, int id, int off, int h0, int stride, const float* cs_of,
                        const float* sn_of, const double* turn_of) {
  if (id < 0) return;
  const int lane = threadIdx.x & 63, D = a.dim, page = 1 << a.page_shift, half = a.rot / 2, chunks = a.rot / 16;
  const int lo = max(sr.pos0 - first, 0), hi = min(sr.pos0 + sr.n - first, 8), rows = hi - lo;  // the call's tokens of the 8
  uint8_t* const kp = reinterpret_cast<uint8_t*>(a.k_pages) + (int64_t)id * a.kv_heads * page * D;
  uint8_t* const vp = reinterpret_cast<uint8_t*>(a.v_pages) + (int64_t)id * a.kv_heads * page * D;
  uint8_t* const ep = a.scales + (int64_t)id * a.kv_heads * 2 * page + off;
  // Keys: L lanes a row and head, lane j with the frequencies 8 j .. 8 j + 7 or 16 elements past rot.
  const int L = D / 16, keys = rows * a.kv_heads * L, kunits = (keys + 63) / 64;
  int unit = h0 + (a.heads > h0 ? (a.heads - h0 + stride - 1) / stride * stride : 0) - a.heads;  // this wave's first one past the queries
  for (; unit < kunits; unit += stride) {
    const int it = min(64 * unit + lane, keys - 1), j = it % L, rh = (uint32_t)it / (uint32_t)L;  // lanes past the last repeat it
    const int h = rh % a.kv_heads, rr = lo + rh / a.kv_heads;
    const uint16_t* src = a.k + (int64_t)(sr.r0 + first + rr - sr.pos0) * a.k_row + (int64_t)h * a.k_head;
    const bool turn = j < chunks;
    const int o0 = !turn || a.adjacent ? 16 * j : 8 * j, o1 = !turn || a.adjacent ? 16 * j + 8 : half + 8 * j;
    const ss_u32x4 x0 = *(const SS_G ss_u32x4*)(src + o0), x1 = *(const SS_G ss_u32x4*)(src + o1);
    float y[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = T::widen(e % 2 ? x0[e / 2] >> 16 : x0[e / 2] & 0xFFFFu);
      y[8 + e] = T::widen(e % 2 ? x1[e / 2] >> 16 : x1[e / 2] & 0xFFFFu);
    }
    if (turn) {
      const float *cs = cs_of + rr * half + 8 * j, *sn = sn_of + rr * half + 8 * j;
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        // frequency f turns elements (f, 8 + f), or (2 f, 2 f + 1) with adjacent
        const float p = a.adjacent ? y[2 * f] : y[f], q = a.adjacent ? y[2 * f + 1] : y[8 + f];
        const float u = p * cs[f] - q * sn[f], v = q * cs[f] + p * sn[f];
        if (a.adjacent) {
          y[2 * f] = u;
          y[2 * f + 1] = v;
        } else {
          y[f] = u;
          y[8 + f] = v;
        }
      }
    }
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, finite_abs(y[e]));
    top = max_over(top, L);
    uint32_t byte = exponent8(top);
    // The exponent is that of the rows turned in 64 bits. Where the maximum is that near to 448 2^n, the turned elements that may pass it are
    // turned again: elements of 448 2^n itself under small angles (27 of 39 million keys had the next smaller byte without).
    const uint32_t bits = ss_fu(top), edge = (bits & 0x7F800000u) | 0x600000u;
    const bool near = bits + kNear >= edge && bits <= edge + kNear;
    if (__builtin_expect(__any(near), 0)) {
      // The elements that may: all at once their comparisons would take more scalar registers than there are.
      const uint32_t least = near ? (turn ? edge - kNear : edge + 1) : ~0u;
      uint32_t which = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        which |= ss_fu(finite_abs(y[e])) >= least ? 1u << e : 0u;
        asm volatile("" : "+v"(which));
      }
      bool over = !turn && which;
      if (!turn) which = 0;
      which = a.adjacent ? which | which >> 1 : which | which >> 8;  // by frequencies, in the even bits of adjacent pairs
      which &= a.adjacent ? 0x5555u : 0xFFu;
#pragma unroll 1
      while (which) {
        const int f = __builtin_ctz(which) >> (a.adjacent ? 1 : 0), freq = 8 * j + f;
        which &= which - 1;
        double sn, cs;
        turn64(turn_of[rr * half + freq], &sn, &cs);
        sn *= a.factor;
        cs *= a.factor;
        const double p = T::widen(gp(src)[a.adjacent ? 2 * freq : freq]), q = T::widen(gp(src)[a.adjacent ? 2 * freq + 1 : half + freq]);
        over |= fmax(fabs(p * cs - q * sn), fabs(q * cs + p * sn)) > (double)ss_uf(edge);
      }
      const int e = (int)(bits >> 23) - 8 + (max_over(over ? 1.f : 0.f, L) > 0.f ? 1 : 0);
      if (near) byte = (uint32_t)max(e, 1);
    }
    const float by = inverse8(byte);
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = scaled8(y[e], by);
    if (64 * unit + lane >= keys) continue;
    uint8_t* dst = kp + ((int64_t)h * page + off + rr) * D;
    uint2 c0, c1;
    c0.x = pack8(y[0], y[1], y[2], y[3]);
    c0.y = pack8(y[4], y[5], y[6], y[7]);
    c1.x = pack8(y[8], y[9], y[10], y[11]);
    c1.y = pack8(y[12], y[13], y[14], y[15]);
    *reinterpret_cast<uint2*>(dst + o0) = c0;
    *reinterpret_cast<uint2*>(dst + o1) = c1;
    if (j == 0) gp(ep)[h * 2 * page + rr] = (uint8_t)byte;
  }
  // Values: 8 rows by 8 dimensions a lane, transposed on the way.
  const int per = D / 8, vals = per * a.kv_heads, vunits = (vals + 63) / 64;
  for (unit -= kunits; unit < vunits; unit += stride) {
    const int it = min(64 * unit + lane, vals - 1), h = (uint32_t)it / (uint32_t)per, d = 8 * (it - h * per);
    const bool mine = 64 * unit + lane < vals;
    ss_u32x4 x[8];
#pragma unroll
    for (int rr = 0; rr < 8; ++rr) {
      x[rr] = ss_u32x4{0u, 0u, 0u, 0u};
      if (rr >= lo && rr < hi)
        x[rr] = *(const SS_G ss_u32x4*)(a.v + (int64_t)(sr.r0 + first + rr - sr.pos0) * a.v_row + (int64_t)h * a.v_head + d);
    }
    float by[8];
#pragma unroll
    for (int rr = 0; rr < 8; ++rr) {
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_abs(T::widen(x[rr][e] & 0xFFFFu)), finite_abs(T::widen(x[rr][e] >> 16))));
      const uint32_t byte = exponent8(max_over(top, per));
      by[rr] = inverse8(byte);
      if (mine && d == 0 && rr >= lo && rr < hi) gp(ep)[(h * 2 + 1) * page + rr] = (uint8_t)byte;
    }
    if (!mine) continue;
    uint8_t* dst = vp + ((int64_t)h * D + d) * page + off;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y[8];
#pragma unroll
      for (int rr = 0; rr < 8; ++rr) y[rr] = scaled8(T::widen(e % 2 ? x[rr][e / 2] >> 16 : x[rr][e / 2] & 0xFFFFu), by[rr]);
      uint2 c;
      c.x = pack8(y[0], y[1], y[2], y[3]);
      c.y = pack8(y[4], y[5], y[6], y[7]);
      if (lo == 0 && hi == 8) {
        *reinterpret_cast<uint2*>(dst + (int64_t)e * page) = c;
      } else {
#pragma unroll
        for (int rr = 0; rr < 8; ++rr)
          if (rr >= lo && rr < hi) gp(dst)[(int64_t)e * page + rr] = (uint8_t)((rr < 4 ? c.x : c.y) >> (8 * (rr % 4)));
      }
    }
  }
}

// Five waves a SIMD with E8 (the compiler would take 99 registers and leave four: 8,190 rows 45.0 us a call for 44.5).
// E8: the cache's pages are e4m3 numbers with exponents; keys and values then go in two parts of their own, in units of a wave
// behind the query heads: of keys 16 elements of a row a lane, of values 8 rows by 8 dimensions.
template <class T, bool E8>
__global__ __launch_bounds__(256, E8 ? 5 : 1) void rope_append_kernel(RopeArgs a) {
  __shared__ __attribute__((aligned(16))) float cs_of[8 * 128], sn_of[8 * 128];  // [8 positions][rot / 2]
  __shared__ double turn_of[E8 ? 8 * 128 : 1];                                   // the angles' parts of a turn, as they are
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
    const double part = turns - __builtin_rint(turns);
    if constexpr (E8) turn_of[it] = part;
    float sn, cs;
    sincospif(2.f * (float)part, &sn, &cs);
    cs_of[it] = cs * a.factor;
    sn_of[it] = sn * a.factor;
  }
  __syncthreads();

  // Query heads, then key heads; a thread's loads for some of its heads go out together.
  const int hs = E8 ? a.heads : a.heads + a.kv_heads;
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
  if constexpr (E8) {
    append_e4m3<T>(a, sr, first, id, off, h0, stride, cs_of, sn_of, turn_of);
    return;
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
  if (a.scales)
    hipLaunchKernelGGL((rope_append_kernel<Bf16, true>), grid, dim3(256), 0, st, a);
  else if (fp16)
    hipLaunchKernelGGL((rope_append_kernel<Fp16, false>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((rope_append_kernel<Bf16, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ss
