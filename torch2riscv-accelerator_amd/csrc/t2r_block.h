// The block-scaled KV cache on gfx950: int8 codes in blocks of bs tokens (16 .. 128) with one fp32 scale per block
// and KV head, and a table that says which block of a pool holds which tokens of a sequence.
//
//   kc [blocks, Hk, bs, hd], vc [blocks, Hk, hd, bs]: a (block, head) tile is contiguous, K by token and V by channel,
//   so that both products of the attention read 16 codes along their summed axis in one load.
//   ks, vs [blocks, Hk]: value = F(code * scale).
//
// A scale is F(max|x| / 127) over the rows that entered the block, a code is x / scale rounded to the nearest integer,
// ties to even, as a real quotient (not as a rounded one: quant_code).
#pragma once
#include "t2r_device.h"

namespace t2r {

typedef _Float16 v2h_t __attribute__((ext_vector_type(2)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));
typedef float v16f_t __attribute__((ext_vector_type(16)));

// bfloat16 values as they lie in memory; loads widen, stores round to nearest even (a NaN stays one)
struct bf16_t { uint16_t b; };

T2R_DEV float widen(float x) { return x; }
T2R_DEV float widen(_Float16 x) { return (float)x; }
T2R_DEV float widen(bf16_t x) { return fv((uint32_t)x.b << 16); }
template <class E> T2R_DEV E narrow(float x);
template <> T2R_DEV float narrow<float>(float x) { return x; }
template <> T2R_DEV _Float16 narrow<_Float16>(float x) { return (_Float16)x; }
template <> T2R_DEV bf16_t narrow<bf16_t>(float x) {
  const uint32_t u = fb(x);
  return bf16_t{(uint16_t)(x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16)};
}

// 16 consecutive elements at any element's alignment (the rows of a split q | k | v matrix start anywhere): gfx950's
// global loads take it
template <class E> struct Row16 {
  static constexpr int kPer = 16 / sizeof(E), kN = 16 / kPer;
  struct __attribute__((packed, aligned(sizeof(E)))) V { v4i_t v; };
  static T2R_DEV void load(const E* p, float* x) {
    V w[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) w[i] = ((const V*)p)[i];
#pragma unroll
    for (int i = 0; i < kN; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = (uint32_t)w[i].v[j];
        if constexpr (sizeof(E) == 4) {
          x[i * 4 + j] = fv(u);
        } else {
          x[i * 8 + 2 * j] = widen(__builtin_bit_cast(E, (uint16_t)u));
          x[i * 8 + 2 * j + 1] = widen(__builtin_bit_cast(E, (uint16_t)(u >> 16)));
        }
      }
  }
  static T2R_DEV void store(E* p, const float* x) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      V w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(E) == 4) {
          w.v[j] = (int)fb(x[i * 4 + j]);
        } else {
          const uint16_t a = __builtin_bit_cast(uint16_t, narrow<E>(x[i * 8 + 2 * j]));
          const uint16_t b = __builtin_bit_cast(uint16_t, narrow<E>(x[i * 8 + 2 * j + 1]));
          w.v[j] = (int)((uint32_t)a | ((uint32_t)b << 16));
        }
      }
      ((V*)p)[i] = w;
    }
  }
};

// The cache and its table, as the kernels take them.
struct BlkCache {
  int8_t* kc;
  int8_t* vc;
  float* ks;
  float* vs;
  const int32_t* table;     // [B, width], rows `width` apart
  int n_blocks, Hk, hd, lbs, width;   // lbs = log2(bs)
  T2R_DEV int bs() const { return 1 << lbs; }
  T2R_DEV int tile_bytes() const { return hd << lbs; }
  // the pool's block of sequence b's j-th one; -1 where the table has none (outside it, or an entry outside the pool)
  T2R_DEV int block(int b, long long j) const {
    if (j < 0 || j >= width) return -1;
    const int t = table[(long long)b * width + j];
    return t >= 0 && t < n_blocks ? t : -1;
  }
};

// The ragged rows of a call: sequence b's are starts[b] .. starts[b + 1] - 1 and the last of them stands at position
// lens[b] - 1. starts and lens are device memory, which the host has not read: rows are clamped into [0, rows) here,
// and a sequence whose starts run backwards has none.
struct Ragged {
  const int32_t* starts;
  const int32_t* lens;
  int B, rows;
};
struct Seq {
  int b, r0, n;             // its rows r0 .. r0 + n - 1
  long long p0;             // position of row r0 (below zero where lens[b] < n)
};
T2R_DEV Seq seq_of(const Ragged& g, int b) {
  Seq s;
  s.b = b;
  s.r0 = min(max(g.starts[b], 0), g.rows);
  s.n = min(max(g.starts[b + 1], s.r0), g.rows) - s.r0;
  s.p0 = (long long)g.lens[b] - s.n;
  return s;
}

// The piece'th of all sequences' pieces, a sequence having count(Seq) of them; in order, from the last one backwards, or the
// later half backwards and then the earlier half forwards (a workgroup of the second round then does what its place in the
// first left over, where pieces grow evenly: the tiles of a long prompt). Every wave of a workgroup finds it by itself, 64
// sequences a step. Returns the piece's place in its sequence, -1 past the last one. A sequence has fewer than kMaxRows
// rows, so 64 of them count in 32 bits whatever `starts` holds; all of them may not.
constexpr int kMaxRows = 1 << 24;
enum { ORDER_FORWARDS = 0, ORDER_BACKWARDS = 1, ORDER_BOTH = 2 };
template <int CTRL, int ROWS = 0xF> T2R_DEV int dpp_or_0(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false); }
// sums over lanes 0 .. lane; the largest of a wave's lanes' values (none below 0), in every lane
T2R_DEV int wave_scan(int x) {
  x += dpp_or_0<0x111>(x);                    // from 1, 2, 4, 8 lanes before, within 16
  x += dpp_or_0<0x112>(x);
  x += dpp_or_0<0x114>(x);
  x += dpp_or_0<0x118>(x);
  x += dpp_or_0<0x142, 0xA>(x);               // the last of the 16 before, then of the 32 before
  return x + dpp_or_0<0x143, 0xC>(x);
}
T2R_DEV float wave_max0(float v) {
  auto up = [&](int y) { v = fmaxf(v, fv((uint32_t)y)); };
  up(dpp_or_0<0x111>((int)fb(v)));
  up(dpp_or_0<0x112>((int)fb(v)));
  up(dpp_or_0<0x114>((int)fb(v)));
  up(dpp_or_0<0x118>((int)fb(v)));
  up(dpp_or_0<0x142, 0xA>((int)fb(v)));
  up(dpp_or_0<0x143, 0xC>((int)fb(v)));
  return fv((uint32_t)__builtin_amdgcn_readlane((int)fb(v), 63));
}

template <class F>
T2R_DEV int find_piece(const Ragged& g, long long piece, int order, F count, Seq* out) {
  auto turn = [&](long long total) {
    if (order == ORDER_FORWARDS) return piece;
    if (piece >= total) return -1LL;
    const long long half = order == ORDER_BOTH ? (total + 1) / 2 : total;
    return piece < half ? total - 1 - piece : piece - half;
  };
  if (g.B == 1) {
    *out = seq_of(g, 0);
    const int total = count(*out), t = (int)turn(total);
    return t < total ? t : -1;
  }
  const int lane = threadIdx.x & 63;
  Seq q;
  int c, s;
  auto scan = [&](int b0) {                   // 64 sequences: each lane's, its pieces, and the sum up to it
    const int b = b0 + lane;
    q = seq_of(g, min(b, g.B - 1));
    c = b < g.B ? count(q) : 0;
    s = wave_scan(c);
    return __builtin_amdgcn_readlane(s, 63);
  };
  int total = scan(0);
  if (order != ORDER_FORWARDS) {
    long long sum = total;
    for (int b0 = 64; b0 < g.B; b0 += 64) sum += scan(b0);
    piece = turn(sum);
    if (piece < 0) return -1;
    if (g.B > 64) total = scan(0);
  }
  long long base = 0;
  for (int b0 = 0;;) {
    if (piece < base + total) {
      const int l = __builtin_ctzll(__ballot(s > (int)(piece - base)));
      auto of = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
      out->b = b0 + l;
      out->r0 = of(q.r0);
      out->n = of(q.n);
      out->p0 = (long long)(((unsigned long long)(uint32_t)of((int)(q.p0 >> 32)) << 32) | (uint32_t)of((int)q.p0));
      return (int)(piece - base) - (of(s) - of(c));
    }
    base += total;
    b0 += 64;
    if (b0 >= g.B) return -1;
    total = scan(b0);
  }
}

// ---------------------------------------------------------------- rows into the cache, and out of it
constexpr int kBlkThreads = 256;

// the blocks that a sequence's rows lie in (the places below position 0 and past the table among them)
T2R_DEV int blocks_touched(const Seq& s, int lbs) {
  return s.n > 0 ? (int)(((s.p0 + s.n - 1) >> lbs) - (s.p0 >> lbs)) + 1 : 0;
}

// x / s to the nearest integer, ties to even, of the real quotient; inv = 1 / s. The rounded product x inv is within one
// of it, and x - q s is exact in fp32 (a multiple of the smaller ulp and at most s in size), so comparing it with s / 2
// settles the sides and the ties. s is not subnormal here (quant_scaled). NaN gives 0, everything is kept in +-127.
T2R_DEV int quant_code(float x, float s, float inv) {
  float q = rintf(fminf(fmaxf(x * inv, -128.0f), 128.0f));
  const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (fabsf(r) > h || (fabsf(r) == h && odd)) q += r > 0 ? 1.0f : -1.0f;
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return x != x ? 0 : (int)q;
}
// The same where it is plain. y after its step (a quotient by a reciprocal and one fused remainder: Markstein's division) is the
// quotient rounded, and exact where that is a fp32 number, as ties are: so
// rintf settles them, and a remainder of at most half a step says that no other integer is nearer. *sure is cleared where it
// is not that (NaN, an infinity, and without FIX a quotient rounded past the middle): quant_code then. FIX is for 16-bit rows,
// where that is no rarity: half of the largest value is often among them, 63.5 steps but for the scale's rounding. (All by
// quant_code: 2032 rows of 8 heads of 128 took 11.4 us, fp32 9.2 so.)
template <bool FIX>
T2R_DEV int quant_plain(float x, float s, float inv, bool* sure) {
  float y = x * inv;
  y = __builtin_fmaf(__builtin_fmaf(-y, s, x), inv, y);
  float q = rintf(fminf(fmaxf(y, -127.0f), 127.0f));
  const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
  if (FIX) {
    *sure = *sure && fabsf(r) <= s;
    q += fabsf(r) > h ? copysignf(1.0f, r) : 0.0f;
  } else {
    *sure = *sure && fabsf(r) <= h;
  }
  return (int)q;
}
// an old code on the block's larger scale: code so / sn to the nearest integer, ties to even (the products are exact
// in 64 bits)
T2R_DEV int requant_code(int c, float so, float sn, float ratio) {
  float q = rintf((float)c * ratio);
  const double r = (double)c * (double)so - (double)q * (double)sn, h = 0.5 * (double)sn, a = r < 0 ? -r : r;
  if (a > h || (a == h && ((int)q & 1))) q += r > 0 ? 1.0f : -1.0f;
  return (int)q;
}

struct BlkRows {
  const void* k;
  const void* v;
  long long k_ld, v_ld;     // elements from row to row
};

// bytes [from, to) of word i of 16 bytes, as a mask
T2R_DEV uint32_t byte_mask(int i, int from, int to) {
  const int a = min(max(from - 4 * i, 0), 4), b = min(max(to - 4 * i, 0), 4);
  return (uint32_t)((1ull << (8 * b)) - (1ull << (8 * a)));
}

// Rows into the cache: a workgroup takes one (block, KV head) of K or of V that rows enter: their maximum, the block's
// new scale, the codes, and the block's older codes where the scale grew. No other workgroup needs that scale, so one pass and
// one launch do. A thread has NU units of 16 values, which stay in registers between the maximum and the codes: K (token,
// 16 channels), V (channel, 16 tokens: lanes along the channels, so that loads are whole lines and a store is 16 codes).
// Reads the rows, writes a byte a value. A call of few rows is a launch and one chain of loads (16 sequences of 8 heads of 64,
// a row each: 4.5 us, 3.3 of them an empty kernel's); a prompt of 2032 rows of 8 heads of 128 in fp32 takes 8.3 us (2.5 TB/s
// of 20.8 MB, 508 workgroups: loads, maximum, codes and stores follow each other in each, and all run at once).
template <class E, int NU>
__global__ __launch_bounds__(kBlkThreads) void k_blk_append(BlkRows x, Ragged g, BlkCache c) {
  __shared__ float red[kBlkThreads / 64];
  const int tid = threadIdx.x, head = blockIdx.y, hd = c.hd, lbs = c.lbs;
  const bool is_v = blockIdx.z != 0;
  Seq s;
  const int piece = find_piece(g, blockIdx.x, ORDER_FORWARDS, [&](const Seq& q) { return blocks_touched(q, lbs); }, &s);
  if (piece < 0) return;
  const long long j = (s.p0 >> lbs) + piece, base = j << lbs;      // the sequence's j-th block, its first position
  const int blk = c.block(s.b, j);
  if (blk < 0) return;
  const int lo = (int)max(s.p0 - base, 0LL), hi = (int)min(s.p0 + s.n - base, (long long)c.bs());
  const long long row = s.r0 + (base - s.p0);                      // of slot 0 (a row of this call from slot lo on)
  const long long at = (long long)blk * c.Hk + head;
  float* scale = (is_v ? c.vs : c.ks) + at;
  int8_t* tile = (is_v ? c.vc : c.kc) + at * c.tile_bytes();
  const long long ld = is_v ? x.v_ld : x.k_ld;
  const E* src = (const E*)(is_v ? x.v : x.k) + row * ld + (long long)head * hd;
  const float was = lo > 0 ? *scale : 0.0f;
  const int per = is_v ? hd : hd >> 4, units = is_v ? per << (lbs - 4) : per << lbs;
  float val[NU][16];
  float m = 0;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = min(tid + i * kBlkThreads, units - 1), a = u / per, b = u - a * per;
    // (what is no row of the call repeats one that is: its maximum counts anyway)
    if (is_v) {
#pragma unroll
      for (int t = 0; t < 16; ++t) val[i][t] = widen(src[min(max(a * 16 + t, lo), hi - 1) * ld + b]);
    } else {
      Row16<E>::load(src + min(max(a, lo), hi - 1) * ld + b * 16, val[i]);
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) m = fmaxf(m, fabsf(val[i][t]));      // (a NaN is left out)
  }
  m = wave_max0(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  m = fminf(m, 3.4028234663852886e38f);                            // an infinity counts as the largest number
  const float now = fmaxf(was, m / 127.0f);
  const bool grew = lo > 0 && now > was && was > 0;
  // small scales are worked with 2^64 times larger, which is exact, so that 1 / s exists
  const float up = now < 0x1p-64f ? 0x1p64f : 1.0f, sn = now * up, inv = now > 0 ? 1.0f / sn : 0.0f;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = tid + i * kBlkThreads;
    if (u >= units) break;
    const int a = u / per, b = u - a * per;
    int8_t* dst = tile + (is_v ? (b << lbs) + a * 16 : a * hd + b * 16);
    const int n_old = is_v ? min(max(lo - a * 16, 0), 16) : a < lo ? 16 : 0;     // values [0, n_old) are older ones,
    const int n_end = is_v ? min(max(hi - a * 16, 0), 16) : a < hi ? 16 : 0;     // [n_old, n_end) new ones
    if (n_end == 0 || (n_old == n_end && !grew)) continue;
    v4i_t w = {0, 0, 0, 0};
    if (n_old > 0 || n_end < 16) w = *(const v4i_t*)dst;
    if (grew && n_old > 0) {
      const float ratio = was / now;
      for (int t = 0; t < n_old; t += 4) {
        // (a word of w by its index, four codes; rare, so short rather than fast)
        const uint32_t o = (uint32_t)(t < 8 ? t < 4 ? w[0] : w[1] : t < 12 ? w[2] : w[3]);
        uint32_t r = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) r |= (uint32_t)(requant_code((int8_t)(o >> (8 * k)), was, now, ratio) & 0xFF) << (8 * k);
        const uint32_t keep = byte_mask(t >> 2, 0, n_old);
        r = (r & keep) | (o & ~keep);
        if (t == 0) w[0] = (int)r;
        else if (t == 4) w[1] = (int)r;
        else if (t == 8) w[2] = (int)r;
        else w[3] = (int)r;
      }
    }
    if (n_old < n_end) {
      int q[16];
      bool sure = true;
#pragma unroll
      for (int t = 0; t < 16; ++t) q[t] = quant_plain<sizeof(E) == 2>(val[i][t] * up, sn, inv, &sure);
      if (!sure) {
#pragma unroll
        for (int t = 0; t < 16; ++t) q[t] = now > 0 ? quant_code(val[i][t] * up, sn, inv) : 0;
      }
#pragma unroll
      for (int t = 0; t < 16; t += 4) {
        uint32_t r = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) r |= (uint32_t)(q[t + k] & 0xFF) << (8 * k);
        const uint32_t put = byte_mask(t >> 2, n_old, n_end);
        w[t >> 2] = (int)((r & put) | ((uint32_t)w[t >> 2] & ~put));
      }
    }
    *(v4i_t*)dst = w;
  }
  if (tid == 0) *scale = now;
}

// Rows out of the cache, as the values that the codes stand for; zeros where the table holds no such position. The same
// pieces as above, the other way. 2032 rows of 8 heads of 128 to fp32: 8.2 us in a row of calls, 9.7 from idle (20.8 MB, 2.1 to
// 2.5 TB/s: table, scale, codes and stores of 508 workgroups, once each); single rows 4.5 us.
template <class E>
__global__ __launch_bounds__(kBlkThreads) void k_blk_read(Ragged g, BlkCache c, E* k, E* v) {
  const int tid = threadIdx.x, head = blockIdx.y, hd = c.hd, lbs = c.lbs;
  const bool is_v = blockIdx.z != 0;
  Seq s;
  const int piece = find_piece(g, blockIdx.x, ORDER_FORWARDS, [&](const Seq& q) { return blocks_touched(q, lbs); }, &s);
  if (piece < 0) return;
  const long long j = (s.p0 >> lbs) + piece, base = j << lbs;
  const int blk = c.block(s.b, j);
  const int lo = (int)max(s.p0 - base, 0LL), hi = (int)min(s.p0 + s.n - base, (long long)c.bs());
  const long long row = s.r0 + (base - s.p0), ld = (long long)c.Hk * hd;
  const long long at = (long long)max(blk, 0) * c.Hk + head;
  const float scale = blk < 0 ? 0.0f : (is_v ? c.vs : c.ks)[at];
  const int8_t* tile = (is_v ? c.vc : c.kc) + at * c.tile_bytes();
  E* dst = (is_v ? v : k) + row * ld + (long long)head * hd;
  const int per = is_v ? hd : hd >> 4, units = is_v ? per << (lbs - 4) : per << lbs;
  for (int u = tid; u < units; u += kBlkThreads) {
    const int a = u / per, b = u - a * per;
    const int from = is_v ? max(lo - a * 16, 0) : a >= lo ? 0 : 16, to = is_v ? min(hi - a * 16, 16) : a < hi ? 16 : 0;
    if (from >= to) continue;
    v4i_t w = {0, 0, 0, 0};
    if (blk >= 0) w = *(const v4i_t*)(tile + (is_v ? (b << lbs) + a * 16 : a * hd + b * 16));
    float y[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) y[t] = (float)(int8_t)(w[t >> 2] >> (8 * (t & 3))) * scale;
    if (is_v) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
        if (t >= from && t < to) dst[(a * 16 + t) * ld + b] = narrow<E>(y[t]);
    } else {
      Row16<E>::store(dst + a * ld + b * 16, y);
    }
  }
}

}  // namespace t2r
