// Attention over the block-scaled int8 KV cache (t2r_block.h): out = softmax(scale q K^T) V for the heads of a KV head
// that share its K and V.
//
// Both products run on fp16 MFMA with the key axis as the rows: S^T = K Q^T and O^T = V^T P^T. The codes are exact in
// fp16, and so nothing of the cache is rounded. What is rounded to fp16:
//  - q, scaled by a power of two to [1, 2) per row: fp32 rows as the sum of two fp16 numbers (22 bits, 2^-25 of the
//    row's largest value), 16-bit rows as one (exact but for values below 2^-24 of it);
//  - p V's scale, again as two numbers with fp32 rows (the fp32 result then stays within a few 2^-22) and as one with
//    16-bit ones, whose result keeps 8 or 11 bits.
// Scores, maxima, sums and outputs are fp32. The scale of a K block multiplies the scores, that of a V block the
// probabilities: w = p vs / vref with vref the largest vs seen, so that w <= p fits fp16 whatever the scales are.
// A maximum is raised only where a score passes it by more than a factor 2^kSlack, so that most steps neither rescale nor
// exchange maxima between lanes. p is kept 2^kLift larger than the maximum says: it reaches 2^(kLift + kSlack), within
// fp16's range, and fp16's smallest step (2^-25 off) is 2^-36 of a row's largest probability times vref.
//
// The MFMA lane layouts meet without any exchange: a lane of S^T holds 4 rows of each 16 (or 4 of each 8 of 32), and
// which key a row stands for is free. Rows are assigned so that a lane ends up with 16 consecutive keys, which are
// what it needs of P as the second product's operand, against 16 consecutive codes of a V^T row (one 16-byte load).
#pragma once
#include "t2r_block.h"

namespace t2r {

constexpr int kBaThreads = 256, kBaWaves = 4;
constexpr int kBaSeg = 2048;                 // keys whose table entries and scales lie in LDS at a time
constexpr float kSlack = 4.0f, kLift = 11.0f;
constexpr float kNegInf = -__builtin_inff();

struct BlkAttn {
  const void* q;
  long long q_ld;
  void* out;
  long long out_ld;
  BlkCache c;
  Ragged g;                 // step form: row b is sequence b's (starts unused)
  int H, G;                 // heads, heads of a KV head
  float a;                  // softmax scale times log2(e)
  int chunk, nsplit;        // keys of a workgroup (a multiple of its waves' step, at most kBaSeg when nsplit > 1)
  float* ws_o;              // parts of long rows: [row's column, split, hd] sums, and [.., 2] maxima and weights
  float* ws_ml;
};

// 8 int8 codes (two words) as fp16: byte b + 128 is put under the exponent of 1024, then 1152 is subtracted (exact)
T2R_DEV v8h_t codes_h(int w0, int w1) {
  const uint32_t u0 = (uint32_t)w0 ^ 0x80808080u, u1 = (uint32_t)w1 ^ 0x80808080u;
  const v2h_t off = {(_Float16)1152.0f, (_Float16)1152.0f};
  v2h_t r[4];
  r[0] = __builtin_bit_cast(v2h_t, __builtin_amdgcn_perm(0x64646464u, u0, 0x04010400u)) - off;
  r[1] = __builtin_bit_cast(v2h_t, __builtin_amdgcn_perm(0x64646464u, u0, 0x04030402u)) - off;
  r[2] = __builtin_bit_cast(v2h_t, __builtin_amdgcn_perm(0x64646464u, u1, 0x04010400u)) - off;
  r[3] = __builtin_bit_cast(v2h_t, __builtin_amdgcn_perm(0x64646464u, u1, 0x04030402u)) - off;
  return __builtin_bit_cast(v8h_t, r);
}

// 2^-e of a row's largest magnitude (e kept where 2^-e is a float), and 2^e on request
T2R_DEV int row_exp(float amax) {
  const int e = (int)((fb(amax) >> 23) & 255u) - 127;
  return min(max(e, -126), 126);
}
T2R_DEV float pow2i(int e) { return fv((uint32_t)(e + 127) << 23); }

// x as a rounded fp32 number: a product that is split into two fp16 ones is taken apart as this number. (Without it the
// compiler rounds the exact product for the first one only, which at a tie is another fp16 number than the second is the
// remainder of.)
T2R_DEV float held(float x) {
  asm("" : "+v"(x));
  return x;
}

// what the products of codes and scaled q are worth; not below the smallest normal float, so that a masked score (-inf)
// times it stays -inf where the block or the row is zero
T2R_DEV float score_scale(float sq, float ks) { return fmaxf(sq * ks, 0x1p-126f); }

// x + (x of the lane 8 further in its row of 16): the two pieces of a q row lie 8 columns apart
T2R_DEV float add_ror8(float x) {
  return x + fv((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fb(x), 0x128, 0xF, 0xF, false));
}

// Fills the segment's LDS tables for keys key0 .. key0 + n - 1 (16 keys an entry; -1: no such block, its keys are left
// out) and returns the largest V scale among them.
struct BaSeg {
  int tb[kBaSeg / 16];
  float ks[kBaSeg / 16], vs[kBaSeg / 16];
  float red[kBaWaves];
};
T2R_DEV float seg_load(BaSeg& sg, const BlkCache& c, int b, int head, long long key0, int n) {
  const int tid = threadIdx.x;
  float m = 0;
  if (tid * 16 < n) {
    const int blk = c.block(b, (key0 + tid * 16) >> c.lbs);
    const long long at = (long long)max(blk, 0) * c.Hk + head;
    const float ks = c.ks[at], vs = c.vs[at];
    sg.tb[tid] = blk < 0 ? -1 : (int)at;
    sg.ks[tid] = ks;
    sg.vs[tid] = blk < 0 ? 0.0f : vs;
    m = blk < 0 ? 0.0f : fabsf(vs);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) sg.red[tid >> 6] = m;
  __syncthreads();
  return fmaxf(fmaxf(sg.red[0], sg.red[1]), fmaxf(sg.red[2], sg.red[3]));
}

// ---------------------------------------------------------------- one row a sequence
// A workgroup takes `chunk` keys of one (sequence, KV head) and up to HW of its query heads, its four waves every fourth
// 64 of them. 16 x 16 x 32 MFMA: columns 0 .. HW - 1 are the heads; with fp32 rows columns 8 .. 15 hold their low
// pieces, so that one product serves both and the columns are added afterwards.
template <class E> struct Pieces { static constexpr int kN = sizeof(E) == 4 ? 2 : 1, kHeads = 16 / kN; };

template <class E, int HD>
__global__ __launch_bounds__(kBaThreads) void k_blk_step(BlkAttn p) {
  constexpr int NP = Pieces<E>::kN, HW = Pieces<E>::kHeads, KU = HD / 64, DT = HD / 16;
  __shared__ BaSeg sg;
  __shared__ float s_m[kBaWaves][16], s_l[kBaWaves][16];
  __shared__ float s_o[kBaWaves][16][HD + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, c4 = lane >> 4;
  const int sets = (p.G + HW - 1) / HW;
  const int kvh = blockIdx.x / sets, h0 = (blockIdx.x - kvh * sets) * HW, b = blockIdx.z, split = blockIdx.y;
  const int hd = p.c.hd, lbs = p.c.lbs, bmask = (1 << lbs) - 1;
  const int nh = min(HW, p.G - h0);                       // heads of this workgroup
  const long long len = min((long long)p.g.lens[b], (long long)p.c.width << lbs), k0 = (long long)split * p.chunk;
  E* out = (E*)p.out + (long long)b * p.out_ld + (long long)(kvh * p.G + h0) * hd;
  if (k0 >= len) {
    if (split == 0)                                        // nothing to attend to
      for (int i = tid; i < nh * hd; i += kBaThreads) out[i] = narrow<E>(0.0f);
    return;
  }
  const int n = (int)min((long long)p.chunk, len - k0);
  const float vref = seg_load(sg, p.c, b, kvh, k0, n);
  const long long tile = p.c.tile_bytes();

  v4i_t kr[4][KU], vr[DT];
  // K rows: row m = 4 c' + r of the t-th 16 stands for key 16 c' + 4 t + r of the 64
  auto load_k = [&](int st) {
    const int ch = st * 4 + (col >> 2), t = max(sg.tb[ch], 0);
    const int8_t* base = p.c.kc + t * tile + (long long)(((ch * 16) & bmask) + (col & 3)) * hd;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int d = u * 64 + c4 * 16;
        kr[i][u] = *(const v4i_t*)(base + 4 * i * hd + (d < hd ? d : 0));   // (past hd q is zero)
      }
  };
  auto load_v = [&](int st) {
    const int ch = st * 4 + c4, t = max(sg.tb[ch], 0);
    const int8_t* base = p.c.vc + t * tile + ((ch * 16) & bmask);
#pragma unroll
    for (int i = 0; i < DT; ++i) vr[i] = *(const v4i_t*)(base + ((long long)min(i * 16 + col, hd - 1) << lbs));
  };
  // the table holds entries up to the segment's last 16 keys: whole steps of 64 read those past it as "no block"
  const int steps = (n + 63) >> 6;
  for (int i = (n + 15) / 16 + tid; i < steps * 4; i += kBaThreads) {
    sg.tb[i] = -1;
    sg.ks[i] = 0;
    sg.vs[i] = 0;
  }
  __syncthreads();
  int st = wave;
  if (st < steps) {
    load_k(st);
    load_v(st);
  }
  // q: the row's largest magnitude, then its pieces in the layout of K's rows
  v8h_t qf[KU][2];
  float sq;
  {
    const int hsel = col % HW;
    const E* q = (const E*)p.q + (long long)b * p.q_ld + (long long)(kvh * p.G + h0 + min(hsel, nh - 1)) * hd;
    float x[KU][16], am = 0;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int d = u * 64 + c4 * 16;
      Row16<E>::load(q + (d < hd ? d : 0), x[u]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[u][i] = d < hd && hsel < nh ? x[u][i] : 0.0f;
        am = fmaxf(am, fabsf(x[u][i]));
      }
    }
    am = fmaxf(am, __shfl_xor(am, 16));
    am = fmaxf(am, __shfl_xor(am, 32));
    const int e = row_exp(am);
    const float down = pow2i(-e);
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = held(x[u][i] * down);
        _Float16 h = (_Float16)y;
        if (NP == 2 && col >= 8) h = (_Float16)(y - (float)h);
        qf[u][i >> 3][i & 7] = h;
      }
    sq = p.a * pow2i(e);
  }
  float m = kNegInf, l = 0;
  v4f_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f_t{0, 0, 0, 0};
  for (; st < steps; st += kBaWaves) {
    v4f_t s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[t] = v4f_t{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h(kr[t][u][0], kr[t][u][1]), qf[u][0], s[t], 0, 0, 0);
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h(kr[t][u][2], kr[t][u][3]), qf[u][1], s[t], 0, 0, 0);
      }
    }
    const bool more = st + kBaWaves < steps;
    if (more) load_k(st + kBaWaves);
    // this lane's 16 keys: 16 c4 + 4 t + r of the 64
    const int ch = st * 4 + c4, left = sg.tb[ch] < 0 ? 0 : n - ch * 16;
    const float sk = score_scale(sq, sg.ks[ch]);
    float wv = 0;
    if (vref > 0) wv = sg.vs[ch] / vref;
    if (NP == 2) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = add_ror8(s[t][r]);
    }
    if (__any(left < 16)) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = 4 * t + r < left ? s[t][r] : kNegInf;
    }
    float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int t = 1; t < 4; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
    mx *= sk;
    if (__any(mx > m + kSlack)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      if (mx > m + kSlack) {
        const float al = __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= al;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] *= al;
      }
    }
    const float sub = (m == kNegInf ? 0.0f : m) - kLift;
    v8h_t pf[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], sk, -sub));
        l += e;
        const float w = NP == 2 ? held(e * wv) : e * wv;
        _Float16 h = (_Float16)w;
        if (NP == 2) {
          const _Float16 lo = (_Float16)(w - (float)h);
          h = col >= 8 ? lo : h;
        }
        pf[t >> 1][(t & 1) * 4 + r] = h;
      }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h(vr[i][0], vr[i][1]), pf[0], o[i], 0, 0, 0);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_h(vr[i][2], vr[i][3]), pf[1], o[i], 0, 0, 0);
    }
    if (more) load_v(st + kBaWaves);
  }
  // the four waves' parts
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = o[i][r];
      if (NP == 2) x = add_ror8(x);
      s_o[wave][col][i * 16 + c4 * 4 + r] = x;
    }
  if (c4 == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
  }
  __syncthreads();
  const bool whole = k0 == 0 && n == len;                 // the only part: the result itself
  for (int i = tid; i < nh * hd; i += kBaThreads) {
    const int h = i / hd, d = i - h * hd;
    float mm = kNegInf;
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) mm = fmaxf(mm, s_m[w][h]);
    const float mu = mm == kNegInf ? 0.0f : mm;
    float x = 0, ls = 0;
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][h] - mu);
      x += f * s_o[w][h][d];
      ls += f * s_l[w][h];
    }
    x *= vref;
    if (whole) {
      out[i] = narrow<E>(ls == 0 ? 0.0f : x / ls);
    } else {
      const long long at = ((long long)b * p.H + kvh * p.G + h0 + h) * p.nsplit + split;
      p.ws_o[at * hd + d] = x;
      if (d == 0) {
        p.ws_ml[2 * at] = mm;
        p.ws_ml[2 * at + 1] = ls;
      }
    }
  }
}

// Joins the parts of a long row: a workgroup per (head, sequence).
constexpr int kJoinThreads = 128;
template <class E>
T2R_DEV void join_row(const BlkAttn& p, long long at, int parts, E* out, int d, bool place) {
  float mm = kNegInf;
  for (int s = 0; s < parts; ++s) mm = fmaxf(mm, p.ws_ml[2 * (at + s)]);
  const float mu = mm == kNegInf ? 0.0f : mm;
  float x = 0, l = 0;
#pragma unroll 8
  for (int s = 0; s < parts; ++s) {
    const float f = __builtin_amdgcn_exp2f(p.ws_ml[2 * (at + s)] - mu);
    x += f * p.ws_o[(at + s) * p.c.hd + d];
    l += f * p.ws_ml[2 * (at + s) + 1];
  }
  *out = narrow<E>(!place ? fv(kQNaN) : l == 0 ? 0.0f : x / l);
}
template <class E>
__global__ __launch_bounds__(kJoinThreads) void k_blk_step_join(BlkAttn p) {
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const long long len = min((long long)p.g.lens[b], (long long)p.c.width << p.c.lbs);
  if (len <= p.chunk || d >= p.c.hd) return;              // one part (or none): written already
  const int parts = (int)((len + p.chunk - 1) / p.chunk);
  join_row<E>(p, ((long long)b * p.H + h) * p.nsplit, parts, (E*)p.out + (long long)b * p.out_ld + (long long)h * p.c.hd + d, d, true);
}

// ---------------------------------------------------------------- several rows a sequence
// A tile is up to 32 CT columns (row, head of the KV head) of one sequence, rows outermost; a workgroup takes one tile
// (and `chunk` of its keys where few rows meet long caches), its four waves every fourth 32 keys, 32 x 32 x 16 MFMA.
// Each wave converts the codes it loads by itself and uses them for all CT 32 columns: no barrier stands in the loop,
// and the q fragments, which the waves share, come from LDS.
template <class E, int HD, int CT> struct RowsLds {
  static constexpr int NP = Pieces<E>::kN, KU = HD / 32;
  static constexpr int kQ = KU * 2 * NP * CT * 64 * 16;              // q fragments, 16 bytes a lane
  static constexpr int kO = kBaWaves * CT * 32 * 33 * 4;             // 32 channels of every wave's sums (33: no bank conflicts)
  static constexpr int kBytes = kQ > kO ? kQ : kO;
};

struct Tile {
  Seq s;
  int t, i0, rows;          // tile t of sequence s: its rows i0 .. i0 + rows - 1
  long long end;            // keys that its last row sees
};
T2R_DEV bool find_tile(const BlkAttn& p, int cols, int w, Tile* t) {
  const int rt = cols / p.G;
  t->t = find_piece(p.g, w, true, [&](const Seq& q) { return (q.n + rt - 1) / rt; }, &t->s);
  if (t->t < 0) return false;
  t->i0 = t->t * rt;
  t->rows = min(rt, t->s.n - t->i0);
  t->end = min(t->s.p0 + t->i0 + t->rows, (long long)p.c.width << p.c.lbs);
  return true;
}

template <class E, int HD, int CT>
__global__ __launch_bounds__(kBaThreads, CT == 2 && HD == 128 ? 1 : 2) void k_blk_rows(BlkAttn p) {
  constexpr int NP = Pieces<E>::kN, KU = HD / 32, DT = HD / 32, COLS = 32 * CT;
  __shared__ BaSeg sg;
  __shared__ float s_m[kBaWaves][COLS], s_l[kBaWaves][COLS];
  __shared__ __align__(16) char s_big[RowsLds<E, HD, CT>::kBytes];
  __shared__ int s_exp[COLS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, c2 = lane >> 5;
  const int w_tile = blockIdx.x / p.c.Hk, kvh = blockIdx.x - w_tile * p.c.Hk, split = blockIdx.y;
  const int hd = p.c.hd, lbs = p.c.lbs, bmask = (1 << lbs) - 1, G = p.G;
  Tile t;
  if (!find_tile(p, COLS, w_tile, &t)) return;
  const long long k0 = p.nsplit > 1 ? (long long)split * p.chunk : 0;
  const int ncol = t.rows * G;
  if (k0 >= t.end) {
    if (split == 0)                                        // every row of the tile stands below position 0
      for (int i = tid; i < ncol * hd; i += kBaThreads) {
        const int c = i / hd, r = c / G;
        ((E*)p.out)[(t.s.r0 + t.i0 + r) * p.out_ld + (long long)(kvh * G + c - r * G) * hd + (i - c * hd)] = narrow<E>(fv(kQNaN));
      }
    return;
  }
  const long long kend = p.nsplit > 1 ? min(t.end, k0 + p.chunk) : t.end;
  const long long tile = p.c.tile_bytes();
  // q fragments into LDS: unit (column, 16 channels); a row's largest magnitude first
  v8h_t* qs = (v8h_t*)s_big;
  {
    constexpr int per = HD / 16, cols_at_once = kBaThreads / per;
    for (int cb = 0; cb < COLS; cb += cols_at_once) {
      const int cc = cb + tid / per, d = (tid % per) * 16, r = cc / G;
      const bool live = cc < ncol && d < hd;
      float x[16], am = 0;
      if (live) {
        Row16<E>::load((const E*)p.q + (t.s.r0 + t.i0 + r) * p.q_ld + (long long)(kvh * G + cc - r * G) * hd + d, x);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) am = fmaxf(am, fabsf(x[i]));
#pragma unroll
      for (int o = 1; o < per; o <<= 1) am = fmaxf(am, __shfl_xor(am, o));
      const int e = row_exp(am);
      const float down = pow2i(-e);
      v8h_t f[NP][2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = held(x[i] * down);
        const _Float16 h = (_Float16)y;
        f[0][i >> 3][i & 7] = h;
        if (NP == 2) f[NP - 1][i >> 3][i & 7] = (_Float16)(y - (float)h);
      }
      // channels 32 u + 16 c + 8 half of column cc: fragment [u][half][piece][cc / 32], lane 32 c + cc % 32
      const int u = d >> 5, ln = ((d >> 4) & 1) * 32 + (cc & 31);
      if (cc < COLS) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int q = 0; q < NP; ++q) qs[(((u * 2 + half) * NP + q) * CT + (cc >> 5)) * 64 + ln] = f[q][half];
        if (d == 0) s_exp[cc] = e;
      }
    }
  }
  // the last key that a lane's columns see (columns past the tile's: none of it matters)
  long long lim[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) lim[ct] = t.s.p0 + t.i0 + min(ct * 32 + col, ncol - 1) / G;
  const long long all_see = t.s.p0 + t.i0 + 1;              // keys below this are seen by every row
  float m[CT], l[CT], sq[CT], vref = 0;
  v16f_t o[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = kNegInf;
    l[ct] = 0;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[ct][i][r] = 0;
  }
  for (long long seg = k0; seg < kend; seg += kBaSeg) {
    const int n = (int)min((long long)kBaSeg, kend - seg);
    const float vmax = fmaxf(vref, seg_load(sg, p.c, t.s.b, kvh, seg, n));
    const int steps = (n + 31) >> 5;
    if ((n + 15) / 16 < steps * 2 && tid == 0) {
      sg.tb[steps * 2 - 1] = -1;
      sg.ks[steps * 2 - 1] = 0;
      sg.vs[steps * 2 - 1] = 0;
    }
    __syncthreads();
    if (seg == k0) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) sq[ct] = p.a * pow2i(s_exp[ct * 32 + col]);
    } else if (vmax > vref) {
      const float f = vref / vmax;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int i = 0; i < DT; ++i) o[ct][i] *= f;
    }
    vref = vmax;
    v4i_t kr[KU], vr[DT];
    // row 8 i + 4 c' + r of the 32 stands for key 16 c' + 4 i + r
    const int kc = (col >> 2) & 1, krow = 4 * (col >> 3) + (col & 3);
    auto load_k = [&](int st) {
      const int ch = st * 2 + kc, tb = max(sg.tb[ch], 0);
      const int8_t* base = p.c.kc + tb * tile + (long long)(((ch * 16) & bmask) + krow) * hd;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int d = u * 32 + c2 * 16;
        kr[u] = *(const v4i_t*)(base + (d < hd ? d : 0));
      }
    };
    auto load_v = [&](int st) {
      const int ch = st * 2 + c2, tb = max(sg.tb[ch], 0);
      const int8_t* base = p.c.vc + tb * tile + ((ch * 16) & bmask);
#pragma unroll
      for (int i = 0; i < DT; ++i) vr[i] = *(const v4i_t*)(base + ((long long)min(i * 32 + col, hd - 1) << lbs));
    };
    int st = wave;
    if (st < steps) {
      load_k(st);
      load_v(st);
    }
    for (; st < steps; st += kBaWaves) {
      v16f_t s[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[ct][r] = 0;
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const v8h_t kf = codes_h(kr[u][2 * half], kr[u][2 * half + 1]);
#pragma unroll
          for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              s[ct] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qs[(((u * 2 + half) * NP + q) * CT + ct) * 64 + lane], s[ct], 0, 0, 0);
        }
      const bool more = st + kBaWaves < steps;
      if (more) load_k(st + kBaWaves);
      const int ch = st * 2 + c2;
      const bool gone = sg.tb[ch] < 0;
      const float ksc = sg.ks[ch];
      float wv = 0;
      if (vref > 0) wv = sg.vs[ch] / vref;
      const bool edge = seg + st * 32 + 32 > all_see || __any(gone);
      v8h_t pf[CT][NP][2];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float sk = score_scale(sq[ct], ksc);
        if (edge) {
          // this lane's keys: seg + 32 st + 16 c2 + r
          const long long room = lim[ct] - (seg + ch * 16);
          const int left = gone || room < 0 ? 0 : room > 15 ? 16 : (int)room + 1;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[ct][r] = r < left ? s[ct][r] : kNegInf;
        }
        float mx = s[ct][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[ct][r]);
        mx *= sk;
        if (__any(mx > m[ct] + kSlack)) {
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          if (mx > m[ct] + kSlack) {
            const float al = __builtin_amdgcn_exp2f(m[ct] - mx);
            m[ct] = mx;
            l[ct] *= al;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[ct][i] *= al;
          }
        }
        const float sub = (m[ct] == kNegInf ? 0.0f : m[ct]) - kLift;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ct][r], sk, -sub));
          l[ct] += e;
          const float w = NP == 2 ? held(e * wv) : e * wv;
          const _Float16 h = (_Float16)w;
          pf[ct][0][r >> 3][r & 7] = h;
          if (NP == 2) pf[ct][NP - 1][r >> 3][r & 7] = (_Float16)(w - (float)h);
        }
      }
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const v8h_t vf = codes_h(vr[i][2 * half], vr[i][2 * half + 1]);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int q = 0; q < NP; ++q) o[ct][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[ct][q][half], o[ct][i], 0, 0, 0);
        }
      if (more) load_v(st + kBaWaves);
    }
    __syncthreads();                                        // the next segment's tables, or the sums below, reuse the LDS
  }
  // the four waves' parts, 32 channels at a time
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 32);
    if (c2 == 0) {
      s_m[wave][ct * 32 + col] = m[ct];
      s_l[wave][ct * 32 + col] = l[ct];
    }
  }
  __syncthreads();
  float f[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float mm = kNegInf;
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) mm = fmaxf(mm, s_m[w][ct * 32 + col]);
    f[ct] = __builtin_amdgcn_exp2f(m[ct] - (mm == kNegInf ? 0.0f : mm)) * vref;
  }
  const bool whole = k0 == 0 && kend == t.end;
  float* so = (float*)s_big;
#pragma unroll
  for (int i = 0; i < DT; ++i) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        so[(wave * COLS + ct * 32 + col) * 33 + 8 * (r >> 2) + 4 * c2 + (r & 3)] = o[ct][i][r] * f[ct];
    __syncthreads();
    for (int e = tid; e < ncol * 32; e += kBaThreads) {
      const int cc = e >> 5, d = i * 32 + (e & 31);
      if (d >= hd) continue;
      float x = 0, ls = 0, mm = kNegInf;
#pragma unroll
      for (int w = 0; w < kBaWaves; ++w) mm = fmaxf(mm, s_m[w][cc]);
      const float mu = mm == kNegInf ? 0.0f : mm;
#pragma unroll
      for (int w = 0; w < kBaWaves; ++w) {
        x += so[(w * COLS + cc) * 33 + (e & 31)];
        ls += __builtin_amdgcn_exp2f(s_m[w][cc] - mu) * s_l[w][cc];
      }
      if (whole) {
        const int r = cc / G;
        ((E*)p.out)[(t.s.r0 + t.i0 + r) * p.out_ld + (long long)(kvh * G + cc - r * G) * hd + d] =
            narrow<E>(t.s.p0 + t.i0 + r < 0 ? fv(kQNaN) : ls == 0 ? 0.0f : x / ls);
      } else {
        const long long at = ((long long)blockIdx.x * COLS + cc) * p.nsplit + split;
        p.ws_o[at * hd + d] = x;
        if (d == 0) {
          p.ws_ml[2 * at] = mm;
          p.ws_ml[2 * at + 1] = ls;
        }
      }
    }
    __syncthreads();
  }
}

// Joins the parts of a tile's columns: a workgroup per (KV head, tile, 4 columns)
template <class E, int CT>
__global__ __launch_bounds__(kBaThreads) void k_blk_rows_join(BlkAttn p) {
  constexpr int COLS = 32 * CT;
  const int w_tile = blockIdx.x / p.c.Hk, kvh = blockIdx.x - w_tile * p.c.Hk;
  Tile t;
  if (!find_tile(p, COLS, w_tile, &t) || t.end <= p.chunk) return;
  const int cc = blockIdx.y * 4 + (threadIdx.x >> 6), G = p.G;
  if (cc >= t.rows * G) return;
  const int parts = (int)((t.end + p.chunk - 1) / p.chunk), r = cc / G;
  const long long at = ((long long)blockIdx.x * COLS + cc) * p.nsplit;
  E* out = (E*)p.out + (t.s.r0 + t.i0 + r) * p.out_ld + (long long)(kvh * G + cc - r * G) * p.c.hd;
  for (int d = threadIdx.x & 63; d < p.c.hd; d += 64) join_row<E>(p, at, parts, out + d, d, t.s.p0 + t.i0 + r >= 0);
}

}  // namespace t2r
