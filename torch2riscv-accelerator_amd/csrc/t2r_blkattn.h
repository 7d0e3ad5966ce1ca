// Attention over the block-scaled int8 KV cache (t2r_block.h): out = softmax(scale q K^T) V for the heads of a KV head
// that share its K and V.
//
// Both products run on fp16 MFMA with the key axis as the rows: S^T = K Q^T and O^T = V^T P^T. The codes are exact in
// fp16, and so nothing of the cache is rounded. What is rounded to fp16:
//  - q, scaled by a power of two to [1, 2) per row: fp32 rows as the sum of two fp16 numbers (22 bits), 16-bit rows as one;
//    either way 2^-25 of the row's largest value is lost at most (nothing of fp16 values down to 2^-14 of it, of bf16 ones down
//    to 2^-17);
//  - the weights, p times V's scale, again as two numbers (the fp32 result then stays within a few 2^-22), but as one in the ragged
//    form's bf16 rows (Pieces).
// Scores, maxima, sums and outputs are fp32. The scale of a K block multiplies the scores, that of a V block the
// probabilities, as a power of two in their exponent: with t = log2(e) scale q . k and u = log2 vs a weight is 2^(t + u).
// The values' sums o run about a base M of the row's own that follows max (t + u), the weights' sum l about another one, m, that
// follows max t: out = 2^(M - m) o / l. A weight is so held against the largest one that the row itself sees, whatever the scales
// are, of blocks that it does not see among them; and nothing leaves fp32's range before the division, however large V is.
// Both bases are whole numbers, so that neither they nor a scale's exponent add a rounding: t is the only large term.
// M is raised only where a weight passes it by more than a factor 2^kSlack, so that most steps neither rescale nor exchange
// maxima between lanes. A weight is kept 2^kLift larger than its base says: it reaches 2^(kLift + kSlack), within fp16's range, and
// fp16's smallest step (2^-25 off) is 2^-36 of the row's largest weight.
//
// The MFMA lane layouts meet without any exchange: a lane of S^T holds 4 rows of each 16 (or 4 of each 8 of 32), and
// which key a row stands for is free. Rows are assigned so that a lane ends up with 16 consecutive keys, which are
// what it needs of P as the second product's operand, against 16 consecutive codes of a V^T row (one 16-byte load).
#pragma once
#include <type_traits>

#include "t2r_block.h"

namespace t2r {

constexpr int kBaThreads = 256, kBaWaves = 4;
constexpr int kBaSeg = 2048;                 // keys whose table entries and scales lie in LDS at a time
constexpr float kSlack = 4.0f, kLift = 11.0f;
constexpr float kFar = 40.0f;                // t above m at which m is raised: l has fp32's range
constexpr float kNegInf = -__builtin_inff();
constexpr float kNoBase = -1e30f;            // a base before the first key: any t lies far above it, and differences with it are numbers

T2R_DEV int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

struct BlkAttn {
  const void* q;
  long long q_ld;
  void* out;
  long long out_ld;
  BlkCache c;
  Ragged g;                 // step form: row b is sequence b's (starts unused)
  int H, G;                 // heads, heads of a KV head
  float a;                  // softmax scale times log2(e)
  int order;                // find_piece's, of the tiles
  int chunk, nsplit;        // keys of a workgroup (a multiple of 128 where there are several; the step form: at most kBaSeg)
  float* ws_o;              // parts of long rows: [row's column, split, hd] sums, and [.., 4] their bases M and m and weights
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

// What a segment's keys need, 16 keys an entry: where their codes begin in kc and in vc (0 where there is no block), how many
// of them there are, the K scale, and the V scale's u = log2 vs in two: the exponent, a whole number, and the rest in [0, 1).
struct BaSeg {
  long long k_at[kBaSeg / 16], v_at[kBaSeg / 16];
  int seen[kBaSeg / 16];                      // 16, or fewer at the end, or none
  float ks[kBaSeg / 16], ue[kBaSeg / 16], uf[kBaSeg / 16];
  int holes[kBaWaves];
};
constexpr float kNoScale = -512.0f;           // u of a scale of 0: such a block's weights count, its values are nothing
// The tables of the keys key0 .. key0 + n - 1, in whole steps of `step` keys, for the whole workgroup. In parts, so that what
// a kernel has to load meanwhile is asked for between them: seg_table asks for this thread's table entry; seg_blocks puts the
// places into LDS (a barrier: the codes can be asked for then); seg_scales the scales (a second one), and returns whether
// some of the n keys have no block.
T2R_DEV int seg_table(const BlkCache& c, int b, long long key0, int n) {
  const int tid = threadIdx.x;
  return tid * 16 < n ? c.block(b, (key0 + tid * 16) >> c.lbs) : -1;
}
T2R_DEV void seg_blocks(BaSeg& sg, const BlkCache& c, int blk, int head, int n, int step) {
  const int tid = threadIdx.x, entries = (n + step - 1) / step * (step >> 4);
  if (tid < entries) {
    const long long tile = (long long)(max(blk, 0) * c.Hk + (blk < 0 ? 0 : head)) * c.tile_bytes();
    const int in = (tid * 16) & (c.bs() - 1);             // (segments begin at whole blocks)
    sg.k_at[tid] = tile + in * c.hd;
    sg.v_at[tid] = tile + in;
    sg.seen[tid] = blk < 0 ? 0 : min(n - tid * 16, 16);
  }
  __syncthreads();
}
T2R_DEV bool seg_scales(BaSeg& sg, const BlkCache& c, int blk, int head, int n, int step) {
  const int tid = threadIdx.x, wave = wave_index(), entries = (n + step - 1) / step * (step >> 4);
  float ks = 0, vs = 0;
  if (blk >= 0) {
    const long long at = (long long)blk * c.Hk + head;
    ks = c.ks[at];
    vs = c.vs[at];
  }
  const bool hole = __any(tid * 16 < n && blk < 0);
  if ((tid & 63) == 0) sg.holes[wave] = hole;
  if (tid < entries) {
    sg.ks[tid] = ks;
    // (subnormal scales have an exponent, too)
    sg.ue[tid] = vs > 0 ? (float)(__builtin_amdgcn_frexp_expf(vs) - 1) : kNoScale;
    sg.uf[tid] = vs > 0 ? __builtin_amdgcn_logf(2.0f * __builtin_amdgcn_frexp_mantf(vs)) : 0.0f;
  }
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < kBaWaves; ++w) any |= sg.holes[w];
  return any != 0;
}

// The bases of a column, the same in each of its lanes.
struct Bases { float M, m; };
// A lane's 16 keys of one block, their largest t in tm (-inf: none is seen): raises the bases where needed, and o and l with
// them. `cols`: f(x) = the largest x of the column's lanes.
template <int DT, class V, class F> T2R_DEV void raise_bases(float tm, float u, Bases& b, float& l, V* o, F cols) {
  const float wm = tm + u;
  if (!__any(wm > b.M + (kLift + kSlack) || tm > b.m + kFar)) return;
  const float t = cols(tm), w = cols(wm);
  const float M = w > b.M + (kLift + kSlack) ? floorf(w) - kLift : b.M, m = t > b.m ? floorf(t) : b.m;
  l *= m == b.m ? 1.0f : __builtin_amdgcn_exp2f(b.m - m);
  const float f = M == b.M ? 1.0f : __builtin_amdgcn_exp2f(b.M - M);
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] *= f;
  b = Bases{M, m};
}
// What is added to those keys' t: u - M, but at least so much that their largest weight is 2^-60: below that the values add
// nothing to o (fp16 gives 0 either way), while the weights, with u taken out again, may be all there is to l. At most -kNoBase,
// where no key is seen.
T2R_DEV float weight_exponent(float tm, float ue, float uf, const Bases& b) {
  return __builtin_amdgcn_fmed3f(-60.0f - tm, ue - b.M, -kNoBase) + uf;
}
// l and those keys' weights, whose sum is ws: that exponent is taken out again, and m put in
T2R_DEV float add_weights(float l, float ws, float add, const Bases& b) {
  return __builtin_fmaf(ws, __builtin_amdgcn_exp2f(-add - b.m), l);
}
// 2^(M - m), as ldexp takes it
T2R_DEV int base_shift(const Bases& b) { return (int)(b.M - b.m); }

// ---------------------------------------------------------------- one row a sequence
// A workgroup takes `chunk` keys of one (sequence, KV head) and up to HW of its query heads, its four waves every fourth
// 64 of them. 16 x 16 x 32 MFMA: columns 0 .. HW - 1 are the heads; with fp32 rows columns 8 .. 15 hold their low
// pieces, so that one product serves both and the columns are added afterwards. 16-bit rows have 16 heads and a second product of
// the weights' low pieces.
//
// Every code is needed once, so the codes go from memory into the waves' registers, a step ahead, and never through LDS; the
// loads of a step are 64 tokens' whole rows. Long caches are bound by memory: 32 sequences of 8192 tokens, 8 KV heads of 128,
// 98 us (5.5 TB/s); of 1021 .. 8192 tokens 60 (5.0 TB/s: the longest sequences end alone), 58 for bf16 rows, and 4.4 for the join.
// Short ones are a chain of length, table, scales, codes and products: one sequence of 96 tokens 4.7 us, of 8101 5.9 and 4.7.
// Head dims between 64 and 128, and below 64, run as the next of these: their codes alone are read, but a wave's chain is as
// long, so the same lengths of 4 heads of 80 take 28 us (3.4 TB/s), of 5 of 96 30 (4.7), of 7 of 32 27 (2.4).
//
// fp16 pieces of an fp32 number: of q, of the weights of the ragged form. One piece of a weight is 2^-12 off, which fp16 results
// show (2-norm, 2.9e-4 off against 2.06e-4 of the rounded exact ones and of two pieces) and bf16's do not (1.67e-3, 1.65e-3,
// 1.65e-3). A second one costs the tiles 15 to 19% (2032 rows, 32 heads of 64: 39.7 and 45.9 us; 16 of 128: 40.4 and 46.5), so bf16
// rows have one there. The step form, bound by memory, always has two: 0 to 4%.
template <class E> struct Pieces { static constexpr int kQ = sizeof(E) == 4 ? 2 : 1, kW = std::is_same<E, bf16_t>::value ? 1 : 2; };

template <class E, int HD>
__global__ __launch_bounds__(kBaThreads, HD == 64 ? 3 : 2) void k_blk_step(BlkAttn p) {
  constexpr int NQ = Pieces<E>::kQ, NP = 3 - NQ, HW = 16 / NQ, KU = HD / 64, DT = HD / 16;     // NP: operands of weights
  __shared__ BaSeg sg;
  __shared__ Bases s_b[kBaWaves][16];
  __shared__ float s_l[kBaWaves][16];
  __shared__ float s_o[kBaWaves][16][HD + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), col = lane & 15, c4 = lane >> 4;
  const int sets = (p.G + HW - 1) / HW;
  const int kvh = blockIdx.x / sets, h0 = (blockIdx.x - kvh * sets) * HW, b = blockIdx.y, split = blockIdx.z;
  const int hd = p.c.hd, lbs = p.c.lbs;
  const int nh = min(HW, p.G - h0);                       // heads of this workgroup
  const long long k0 = (long long)split * p.chunk;
  // everything that needs nothing loaded is asked for at once: the length, the table and q
  const int blk = seg_table(p.c, b, k0, p.chunk);
  float x[KU][16];
  const int hsel = col % HW;
  {
    const E* q = (const E*)p.q + (long long)b * p.q_ld + (long long)(kvh * p.G + h0 + min(hsel, nh - 1)) * hd;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int d = u * 64 + c4 * 16;
      Row16<E>::load(q + (d < hd ? d : 0), x[u]);           // (channels past hd are made zero below)
    }
  }
  const long long len = min((long long)p.g.lens[b], (long long)p.c.width << lbs);
  E* out = (E*)p.out + (long long)b * p.out_ld + (long long)(kvh * p.G + h0) * hd;
  if (k0 >= len) {
    if (split == 0)                                        // nothing to attend to
      for (int i = tid; i < nh * hd; i += kBaThreads) out[i] = narrow<E>(0.0f);
    return;
  }
  const int n = (int)min((long long)p.chunk, len - k0), steps = (n + 63) >> 6;
  const int mine = tid * 16 < n ? blk : -1;
  v4i_t kr[4][KU], vr[DT];
  // K rows: row m = 4 c' + r of the t-th 16 stands for key 16 c' + 4 t + r of the 64
  auto load_k = [&](int st) {
    const int8_t* base = p.c.kc + sg.k_at[st * 4 + (col >> 2)] + (col & 3) * hd;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        const int d = u * 64 + c4 * 16;
        kr[i][u] = *(const v4i_t*)(base + 4 * i * hd + (d < hd ? d : 0));   // (past hd q is zero)
      }
  };
  auto load_v = [&](int st) {
    const int8_t* base = p.c.vc + sg.v_at[st * 4 + c4];
#pragma unroll
    for (int i = 0; i < DT; ++i) vr[i] = *(const v4i_t*)(base + (min(i * 16 + col, hd - 1) << lbs));
  };
  seg_blocks(sg, p.c, mine, kvh, n, 64);
  int st = wave;
  if (st < steps) {
    load_k(st);
    load_v(st);
  }
  const bool holes = seg_scales(sg, p.c, mine, kvh, n, 64);
  // q's pieces in the layout of K's rows, after the row's largest magnitude
  v8h_t qf[KU][2];
  float sq;
  {
    float am = 0;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) am = fmaxf(am, fabsf(x[u][i]));
    am = fmaxf(am, __shfl_xor(am, 16));
    am = fmaxf(am, __shfl_xor(am, 32));
    const int e = row_exp(am);
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const float down = u * 64 + c4 * 16 < hd ? pow2i(-e) : 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = held(x[u][i] * down);
        _Float16 h = (_Float16)y;
        if (NQ == 2 && col >= 8) h = (_Float16)(y - (float)h);
        qf[u][i >> 3][i & 7] = h;
      }
    }
    sq = p.a * pow2i(e);
  }
  Bases bs{kNoBase, kNoBase};
  float l = 0;
  v4f_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = v4f_t{0, 0, 0, 0};
  // a step of 64 keys; edge: not all of them are seen
  auto step = [&](auto edge) {
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
    const int ch = st * 4 + c4;
    const float sk = score_scale(sq, sg.ks[ch]), ue = sg.ue[ch], uf = sg.uf[ch];
    if (NQ == 2) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = add_ror8(s[t][r]);
    }
    if constexpr (edge.value) {
      const int left = sg.seen[ch];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][r] = 4 * t + r < left ? s[t][r] : kNegInf;
    }
    float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
    for (int t = 1; t < 4; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
    mx *= sk;
    raise_bases<DT>(mx, ue + uf, bs, l, o, [](float x) {
      x = fmaxf(x, __shfl_xor(x, 16));
      return fmaxf(x, __shfl_xor(x, 32));
    });
    const float add = weight_exponent(mx, ue, uf, bs);
    v8h_t pf[NP][2];
    float ls[4] = {0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], sk, add));
        ls[r] += w;
        const _Float16 h = (_Float16)w, lo = (_Float16)__builtin_fmaf((float)h, -1.0f, w);
        pf[0][t >> 1][(t & 1) * 4 + r] = NQ == 2 && col >= 8 ? lo : h;
        if (NP == 2) pf[NP - 1][t >> 1][(t & 1) * 4 + r] = lo;
      }
    l = add_weights(l, (ls[0] + ls[1]) + (ls[2] + ls[3]), add, bs);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const v8h_t vf = codes_h(vr[i][2 * half], vr[i][2 * half + 1]);
#pragma unroll
        for (int q = 0; q < NP; ++q) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[q][half], o[i], 0, 0, 0);
      }
    if (more) load_v(st + kBaWaves);
  };
  for (const int plain = holes ? 0 : n >> 6; st < plain; st += kBaWaves) step(std::false_type());
  for (; st < steps; st += kBaWaves) step(std::true_type());
  // the four waves' parts
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = o[i][r];
      if (NQ == 2) x = add_ror8(x);
      s_o[wave][col][i * 16 + c4 * 4 + r] = x;
    }
  if (c4 == 0) {
    s_b[wave][col] = bs;
    s_l[wave][col] = l;
  }
  __syncthreads();
  const bool whole = k0 == 0 && n == len;                 // the only part: the result itself
  for (int i = tid; i < nh * hd; i += kBaThreads) {
    const int h = i / hd, d = i - h * hd;
    Bases top{kNoBase, kNoBase};
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) top = Bases{fmaxf(top.M, s_b[w][h].M), fmaxf(top.m, s_b[w][h].m)};
    float x = 0, ls = 0;
#pragma unroll
    for (int w = 0; w < kBaWaves; ++w) {
      x += __builtin_amdgcn_exp2f(s_b[w][h].M - top.M) * s_o[w][h][d];
      ls += __builtin_amdgcn_exp2f(s_b[w][h].m - top.m) * s_l[w][h];
    }
    if (whole) {
      out[i] = narrow<E>(ls == 0 ? 0.0f : __builtin_amdgcn_ldexpf(x / ls, base_shift(top)));
    } else {
      const long long at = ((long long)b * p.H + kvh * p.G + h0 + h) * p.nsplit + split;
      p.ws_o[at * hd + d] = x;
      if (d == 0) *(v4f_t*)(p.ws_ml + 4 * at) = v4f_t{top.M, top.m, ls, 0};
    }
  }
}

// Joins the parts of a row: their sums, moved to the largest of their bases. NWV waves of the workgroup take every NWV-th part
// each, a lane two channels; what the row's first wave has in *x is the row (and the weights' sum and the bases, the same in every
// wave, come back). The parts' bases are read 64 at a time, a lane each; the sums' loads wait for nothing. A wave has eight parts' sums
// in flight, and eight more cost a memory's latency: from kJoinWide parts on a row is worth four waves (32 columns of 32
// heads in 13 / 32 parts: 6.5 / 9.4 us with a wave each).
constexpr int kJoinWide = 9;
template <int NWV>
T2R_DEV float join_parts(const BlkAttn& p, long long at, int parts, float (*x)[2], Bases* top) {
  __shared__ float s_x[NWV > 1 ? kBaWaves : 1][64][2];
  const int lane = threadIdx.x & 63, hd = p.c.hd, d = min(2 * lane, hd - 2), wave = NWV > 1 ? wave_index() : 0;
  typedef float v2f_t __attribute__((ext_vector_type(2)));
  const v4f_t* ml = (const v4f_t*)p.ws_ml + at;
  float M = kNoBase, m = kNoBase;
  for (int s = lane; s < parts; s += 64) {
    const v4f_t v = ml[s];
    M = fmaxf(M, v[0]);
    m = fmaxf(m, v[1]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    M = fmaxf(M, __shfl_xor(M, o));
    m = fmaxf(m, __shfl_xor(m, o));
  }
  *top = Bases{M, m};
  float l = 0;
  v2f_t y = {0, 0};
  for (int b = 0; b < parts; b += 64) {
    const int n = min(parts - b, 64);
    v4f_t v = {kNoBase, kNoBase, 0, 0};
    if (lane < n) v = ml[b + lane];
    const float f = __builtin_amdgcn_exp2f(v[0] - M);
    l += __builtin_amdgcn_exp2f(v[1] - m) * v[2];
    const float* o = p.ws_o + (at + b) * hd + d;
#pragma unroll 8
    for (int s = wave; s < n; s += NWV) y += fv((uint32_t)__builtin_amdgcn_readlane((int)fb(f), s)) * *(const v2f_t*)(o + s * hd);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  (*x)[0] = y[0];
  (*x)[1] = y[1];
  if constexpr (NWV > 1) {
    s_x[wave][lane][0] = y[0];
    s_x[wave][lane][1] = y[1];
    __syncthreads();
#pragma unroll
    for (int w = 1; w < NWV; ++w) {
      (*x)[0] += s_x[w][lane][0];
      (*x)[1] += s_x[w][lane][1];
    }
  }
  return l;
}
// Two channels of a joined row. (It has a place in its sequence: a tile in parts ends past 512 keys and has 128 rows at most.)
template <class E>
T2R_DEV void join_store(const BlkAttn& p, E* out, const float* x, float l, const Bases& top) {
  const int d = 2 * (threadIdx.x & 63);
  if (d >= p.c.hd) return;
  const float inv = l == 0 ? 0.0f : 1.0f / l;
  const int e = base_shift(top);
  out[d] = narrow<E>(__builtin_amdgcn_ldexpf(x[0] * inv, e));
  out[d + 1] = narrow<E>(__builtin_amdgcn_ldexpf(x[1] * inv, e));
}

// a workgroup per (head, sequence); 4.3 us, 3.3 of them an empty kernel's
template <class E>
__global__ __launch_bounds__(kBaThreads) void k_blk_step_join(BlkAttn p) {
  const int h = blockIdx.x, b = blockIdx.y;
  const long long len = min((long long)p.g.lens[b], (long long)p.c.width << p.c.lbs);
  if (len <= p.chunk) return;                             // one part (or none): written already
  const int parts = (int)((len + p.chunk - 1) / p.chunk);
  float x[2];
  Bases top;
  const float l = join_parts<kBaWaves>(p, ((long long)b * p.H + h) * p.nsplit, parts, &x, &top);
  if (wave_index() == 0) join_store<E>(p, (E*)p.out + (long long)b * p.out_ld + (long long)h * p.c.hd, x, l, top);
}

// ---------------------------------------------------------------- several rows a sequence
// A tile is up to `cols` columns (row, head of the KV head) of one sequence, rows outermost; a workgroup takes one tile (and
// `chunk` of its keys where few rows meet long caches). 32 x 32 x 16 MFMA.
//
// k_blk_few: 32 columns. The four waves take every fourth 32 keys, each loading and converting its codes by itself: nothing
// is shared but the columns, and no barrier stands in the loop. 8 rows of each of four sequences over 5003 .. 8100 positions,
// 32 heads of 64: 16 us in parts of 512 keys, of which a part's beginning and end are half, and 5.1 for the join.
// k_blk_tile: 64 CT columns, two groups of 32 CT for the waves; the two waves of a group take the stage's two times 32 keys. The
// workgroup loads a stage's codes together (a stage ahead), converts them once into LDS, in the MFMA operands' order, two
// stages in turn with one barrier each. The conversion is as much vector work as the softmax of 32 columns (80 instructions of
// 32 keys at head dim 128 where two waves share it, against 100), so the groups share it.
// Bound by issue: a product takes 32 cycles of its unit and a vector instruction 4, five where a SIMD has one wave, and beyond
// three a product they add up. At head dim 128 in fp32 a wave has 32 products and 200 other vector instructions a stage, in
// bf16 at 64 16 and 215. One prompt of 2032 rows, 16 heads of 128 in fp32: 49.8 us in a row of calls (340 TFLOP/s of the formula's,
// twice that of fp16 products, q and the weights being two pieces), some 1.2 us a stage where one workgroup is on a CU, 1.0 where
// two are, so each CU's 33 stages take about as long however tiles are cut or paired; 7 us a tile lie before and after them. Seven
// prompts and turns in bf16, 32 heads of 64, 37.2 GFLOP: 68.7 us (541 TFLOP/s). Slower, all measured: eight waves a workgroup, a
// second stage in flight in registers, tiles cut along their keys; four groups of 32 columns at head dim 128 gain 0 .. 10% past
// 8000 rows and lose before. Other head dims run as 64 or 128 with the products of the missing channels: the prompt of 2032 rows
// of 16 heads takes 45.5 us at head dim 80 and 48.8 at 96, 31.0 and 30.9 at 48 and 32 against 32.0 at 64.
struct Tile {
  Seq s;
  int t, i0, rows;          // tile t of sequence s: its rows i0 .. i0 + rows - 1
  long long end;            // keys that its last row sees
};
T2R_DEV bool find_tile(const BlkAttn& p, int cols, int w, Tile* t) {
  const int rt = cols / p.G;
  t->t = find_piece(p.g, w, p.order, [&](const Seq& q) { return (q.n + rt - 1) / rt; }, &t->s);
  if (t->t < 0) return false;
  t->i0 = t->t * rt;
  t->rows = min(rt, t->s.n - t->i0);
  t->end = min(t->s.p0 + t->i0 + t->rows, (long long)p.c.width << p.c.lbs);
  return true;
}
// where column cc of a tile reads and writes
T2R_DEV long long col_at(const Tile& t, int G, int hd, int kvh, int cc, long long ld) {
  const int r = cc / G;
  return (t.s.r0 + t.i0 + r) * ld + (long long)(kvh * G + cc - r * G) * hd;
}

// a lane's column of q: its channels 32 u + 16 (lane / 32) .. + 15 (those past hd repeat the first ones) ...
template <class E, int KU>
T2R_DEV void q_load(const E* q, int hd, float (*x)[16]) {
  const int c2 = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const int d = u * 32 + c2 * 16;
    Row16<E>::load(q + (d < hd ? d : 0), x[u]);
  }
}
// ... and as fp16 pieces (zero past hd), in the order of K's rows; returns 2^e of the power that was taken out
template <class E, int KU>
T2R_DEV float q_pieces(int hd, const float (*x)[16], v8h_t (*qf)[Pieces<E>::kQ][2]) {
  constexpr int NQ = Pieces<E>::kQ;
  const int c2 = (threadIdx.x & 63) >> 5;
  float am = 0;
#pragma unroll
  for (int u = 0; u < KU; ++u)
#pragma unroll
    for (int i = 0; i < 16; ++i) am = fmaxf(am, fabsf(x[u][i]));
  am = fmaxf(am, __shfl_xor(am, 32));
  const int e = row_exp(am);
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const float down = u * 32 + c2 * 16 < hd ? pow2i(-e) : 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float y = held(x[u][i] * down);
      const _Float16 h = (_Float16)y;
      qf[u][0][i >> 3][i & 7] = h;
      if (NQ == 2) qf[u][NQ - 1][i >> 3][i & 7] = (_Float16)__builtin_fmaf((float)h, -1.0f, y);
    }
  }
  return pow2i(e);
}

// The softmax of 32 keys' scores s for a lane's column: this lane's 16 keys are 16 (lane / 32) + r, `left` of them (below 16
// only if EDGE) are seen. First the bases, raised where needed (o and l with them); returns the weights' exponent ...
template <int DT, bool EDGE>
T2R_DEV float soft_max(v16f_t& s, float sk, int left, float ue, float uf, Bases& b, float& l, v16f_t* o) {
  if constexpr (EDGE) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = r < left ? s[r] : kNegInf;
  }
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
  mx *= sk;
  raise_bases<DT>(mx, ue + uf, b, l, o, [](float x) { return fmaxf(x, __shfl_xor(x, 32)); });
  return weight_exponent(mx, ue, uf, b);
}
// ... then the weights of keys r .. r + 3 as fp16 pieces, and their sum; ...
template <int NW>
T2R_DEV float soft_weights(const v16f_t& s, float sk, float add, v8h_t (*pf)[2], int r) {
  typedef float v2f_t __attribute__((ext_vector_type(2)));
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + i], sk, add));
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    v2h_t h = __builtin_convertvector((v2f_t{w[i], w[i + 1]}), v2h_t);
    // The low pieces in one mixed-precision step each, which reads the high ones where they are. (Both values are kept from the
    // compiler, which would convert anew and take h out of fp16 to subtract it.)
    float minus = -1.0f;
    asm("" : "+v"(h));
    asm("" : "+s"(minus));
    pf[0][r >> 3][(r & 7) + i] = h[0];
    pf[0][r >> 3][(r & 7) + i + 1] = h[1];
    if (NW == 2) {
      pf[NW - 1][r >> 3][(r & 7) + i] = (_Float16)__builtin_fmaf((float)h[0], minus, w[i]);
      pf[NW - 1][r >> 3][(r & 7) + i + 1] = (_Float16)__builtin_fmaf((float)h[1], minus, w[i + 1]);
    }
  }
  return (w[0] + w[1]) + (w[2] + w[3]);
}
// ... of all 16, and their sum into l.
template <int NW>
T2R_DEV void soft_exp(const v16f_t& s, float sk, float add, const Bases& b, float& l, v8h_t (*pf)[2]) {
  float ls = 0;
#pragma unroll
  for (int r = 0; r < 16; r += 4) ls += soft_weights<NW>(s, sk, add, pf, r);
  l = add_weights(l, ls, add, b);
}

// The end of a tile: its waves' sums (wave's column group cg of 32 CT, key group kg of KG) are joined through LDS (so: KG x COLS
// rows of HD + 4 floats, which keeps 16-byte accesses free of bank conflicts) and written as the result or, of a part of the
// keys, into the workspace.
template <int HD, int CT, int CG> struct TileEnd {
  static constexpr int KG = kBaWaves / CG, COLS = 32 * CT * CG, LD = HD + 4, kBytes = KG * COLS * LD * 4;
  struct Ml { Bases b[KG][COLS], top[COLS]; float l[KG][COLS], sum[COLS], inv[COLS]; };
};
// four values side by side, at any element's alignment
template <class E> T2R_DEV void store4(E* p, v4f_t x) {
  struct __attribute__((packed, aligned(sizeof(E)))) V { E e[4]; };
  *(V*)p = V{{narrow<E>(x[0]), narrow<E>(x[1]), narrow<E>(x[2]), narrow<E>(x[3])}};
}
template <class E, int HD, int CT, int CG>
T2R_DEV void tile_end(const BlkAttn& p, const Tile& t, int kvh, int split, bool whole, const Bases* b, float* l,
                      v16f_t (*o)[HD / 32], typename TileEnd<HD, CT, CG>::Ml& ml, float* so) {
  using T = TileEnd<HD, CT, CG>;
  constexpr int KG = T::KG, COLS = T::COLS, LD = T::LD, DT = HD / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), col = lane & 31, c2 = lane >> 5;
  const int cg = wave % CG, kg = wave / CG, hd = p.c.hd, G = p.G, ncol = t.rows * G;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 32);
    if (c2 == 0) {
      ml.b[kg][(cg * CT + ct) * 32 + col] = b[ct];
      ml.l[kg][(cg * CT + ct) * 32 + col] = l[ct];
    }
  }
  __syncthreads();
  // a column's largest bases over its key groups, and the weights' sum about them
  if (tid < COLS) {
    Bases top = ml.b[0][tid];
#pragma unroll
    for (int w = 1; w < KG; ++w) top = Bases{fmaxf(top.M, ml.b[w][tid].M), fmaxf(top.m, ml.b[w][tid].m)};
    float ls = 0;
#pragma unroll
    for (int w = 0; w < KG; ++w) ls += __builtin_amdgcn_exp2f(ml.b[w][tid].m - top.m) * ml.l[w][tid];
    ml.top[tid] = top;
    ml.sum[tid] = ls;
    ml.inv[tid] = t.s.p0 + t.i0 + min(tid, ncol - 1) / G < 0 ? fv(kQNaN) : ls == 0 ? 0.0f : 1.0f / ls;
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int cc = (cg * CT + ct) * 32 + col;
    float M = ml.b[0][cc].M;
#pragma unroll
    for (int w = 1; w < KG; ++w) M = fmaxf(M, ml.b[w][cc].M);
    const float f = __builtin_amdgcn_exp2f(b[ct].M - M);
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(v4f_t*)(so + (kg * COLS + cc) * LD + i * 32 + 2 * r + 4 * c2) =
            v4f_t{o[ct][i][r] * f, o[ct][i][r + 1] * f, o[ct][i][r + 2] * f, o[ct][i][r + 3] * f};
  }
  __syncthreads();
  // four channels a thread
  constexpr int PER = HD / 4;
  const int d = tid % PER * 4;
  if (d >= hd) return;
#pragma unroll 2
  for (int cc = tid / PER; cc < ncol; cc += kBaThreads / PER) {
    v4f_t x = *(const v4f_t*)(so + cc * LD + d);
#pragma unroll
    for (int w = 1; w < KG; ++w) x += *(const v4f_t*)(so + (w * COLS + cc) * LD + d);
    if (whole) {
      const int e = base_shift(ml.top[cc]);
      x *= ml.inv[cc];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ldexpf(x[i], e);
      store4((E*)p.out + col_at(t, G, hd, kvh, cc, p.out_ld) + d, x);
    } else {
      const long long at = ((long long)blockIdx.x * COLS + cc) * p.nsplit + split;
      *(v4f_t*)(p.ws_o + at * hd + d) = x;
      if (d == 0) *(v4f_t*)(p.ws_ml + 4 * at) = v4f_t{ml.top[cc].M, ml.top[cc].m, ml.sum[cc], 0};
    }
  }
}

// The tile of a workgroup and its keys [k0, kend), false where it has none (a tile whose rows all stand below position 0 is
// answered here).
template <class E>
T2R_DEV bool tile_of(const BlkAttn& p, int cols, Tile* t, int* kvh, long long* k0, long long* kend) {
  const int w = blockIdx.x / p.c.Hk;
  *kvh = blockIdx.x - w * p.c.Hk;
  if (!find_tile(p, cols, w, t)) return false;
  *k0 = p.nsplit > 1 ? (long long)blockIdx.y * p.chunk : 0;
  *kend = p.nsplit > 1 ? min(t->end, *k0 + p.chunk) : t->end;
  if (*k0 < t->end) return true;
  if (blockIdx.y == 0)
    for (int i = threadIdx.x; i < t->rows * p.G * p.c.hd; i += blockDim.x) {
      const int cc = i / p.c.hd;
      ((E*)p.out)[col_at(*t, p.G, p.c.hd, *kvh, cc, p.out_ld) + (i - cc * p.c.hd)] = narrow<E>(fv(kQNaN));
    }
  return false;
}

// how many of the 16 keys from `from` on a row at position `at` sees, `seen` of them there
T2R_DEV int keys_left(long long at, long long from, int seen) {
  const long long room = at - from;
  return room < 0 ? 0 : min(room > 15 ? 16 : (int)room + 1, seen);
}
// whole steps of `step` keys at a segment's start that every row sees all of
T2R_DEV int plain_steps(long long all_see, long long seg, int n, int step, bool holes) {
  return holes ? 0 : (int)max(min(all_see - seg, (long long)n), 0LL) / step;
}

template <class E, int HD>
__global__ __launch_bounds__(kBaThreads, HD == 64 ? 3 : 2) void k_blk_few(BlkAttn p) {
  constexpr int NQ = Pieces<E>::kQ, NW = Pieces<E>::kW, KU = HD / 32, DT = HD / 32;
  __shared__ BaSeg sg;
  using End = TileEnd<HD, 1, 1>;
  __shared__ typename End::Ml ml;
  __shared__ __align__(16) char s_o[End::kBytes];
  const int lane = threadIdx.x & 63, wave = wave_index(), col = lane & 31, c2 = lane >> 5;
  const int hd = p.c.hd, lbs = p.c.lbs, G = p.G;
  Tile t;
  int kvh;
  long long k0, kend;
  if (!tile_of<E>(p, 32, &t, &kvh, &k0, &kend)) return;
  const int cc = min(col, t.rows * G - 1);
  int blk = seg_table(p.c, t.s.b, k0, (int)min((long long)kBaSeg, kend - k0));
  float x[KU][16];
  q_load<E, KU>((const E*)p.q + col_at(t, G, hd, kvh, cc, p.q_ld), hd, x);
  v8h_t qf[KU][NQ][2];
  const long long at = t.s.p0 + t.i0 + cc / G, all_see = t.s.p0 + t.i0 + 1;   // (keys below all_see are seen by every row)
  // row 8 i + 4 c' + r of the 32 stands for key 16 c' + 4 i + r
  const int kc = (col >> 2) & 1, krow = 4 * (col >> 3) + (col & 3);
  Bases bs{kNoBase, kNoBase};
  float l = 0;
  v16f_t o[1][DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[0][i] = v16f_t{};
  v4i_t kr[KU], vr[DT];
  auto load_k = [&](int st) {
    const int8_t* base = p.c.kc + sg.k_at[st * 2 + kc] + krow * hd;
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int d = u * 32 + c2 * 16;
      kr[u] = *(const v4i_t*)(base + (d < hd ? d : 0));              // (past hd q is zero)
    }
  };
  auto load_v = [&](int st) {
    const int8_t* base = p.c.vc + sg.v_at[st * 2 + c2];
#pragma unroll
    for (int i = 0; i < DT; ++i) vr[i] = *(const v4i_t*)(base + (min(i * 32 + col, hd - 1) << lbs));
  };
  // a segment's blocks, and its first loads
  auto begin = [&](int n) {
    seg_blocks(sg, p.c, blk, kvh, n, 32);
    if (wave < (n + 31) >> 5) {
      load_k(wave);
      load_v(wave);
    }
  };
  begin((int)min((long long)kBaSeg, kend - k0));
  const float sq = p.a * q_pieces<E, KU>(hd, x, qf);
  for (long long seg = k0; seg < kend; seg += kBaSeg) {
    const int n = (int)min((long long)kBaSeg, kend - seg), steps = (n + 31) >> 5;
    const bool holes = seg_scales(sg, p.c, blk, kvh, n, 32);
    int st = wave;
    auto step = [&](auto edge) {
      v16f_t s = {};
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const v8h_t kf = codes_h(kr[u][2 * half], kr[u][2 * half + 1]);
#pragma unroll
          for (int q = 0; q < NQ; ++q) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[u][q][half], s, 0, 0, 0);
        }
      const bool more = st + kBaWaves < steps;
      if (more) load_k(st + kBaWaves);
      const int ch = st * 2 + c2;
      v8h_t pf[NW][2];
      const float sk = score_scale(sq, sg.ks[ch]);
      const float add = soft_max<DT, edge.value>(s, sk, edge.value ? keys_left(at, seg + ch * 16, sg.seen[ch]) : 16, sg.ue[ch],
                                                 sg.uf[ch], bs, l, o[0]);
      soft_exp<NW>(s, sk, add, bs, l, pf);
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const v8h_t vf = codes_h(vr[i][2 * half], vr[i][2 * half + 1]);
#pragma unroll
          for (int q = 0; q < NW; ++q) o[0][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[q][half], o[0][i], 0, 0, 0);
        }
      if (more) load_v(st + kBaWaves);
    };
    for (const int plain = plain_steps(all_see, seg, n, 32, holes); st < plain; st += kBaWaves) step(std::false_type());
    for (; st < steps; st += kBaWaves) step(std::true_type());
    __syncthreads();                                        // the next segment's tables take this one's place
    const long long next = seg + kBaSeg;
    if (next < kend) {
      const int m = (int)min((long long)kBaSeg, kend - next);
      blk = seg_table(p.c, t.s.b, next, m);
      begin(m);
    }
  }
  tile_end<E, HD, 1, 1>(p, t, kvh, blockIdx.y, k0 == 0 && kend == t.end, &bs, &l, o, ml, (float*)s_o);
}

// LDS of k_blk_tile, in 16-byte slots: a fragment (64 lanes' operand of one MFMA) is 64 slots. K's fragments of a stage are
// [kg][u][half], V's [kg][i][half]. The lane's slot is turned by the fragment's place, so that the loading threads, which
// hold neighbouring 16-byte pieces of a token or channel, write to different banks.
//
// What a wave has to wait for is kept off its path: a stage's codes are loaded a stage ahead, its V fragments are read from LDS
// before the softmax, and two buffers leave one barrier a stage.
template <class E, int HD, int CT>
__global__ __launch_bounds__(kBaThreads, 2) void k_blk_tile(BlkAttn p) {
  constexpr int NQ = Pieces<E>::kQ, NW = Pieces<E>::kW, KU = HD / 32, DT = HD / 32, CG = 2, KG = kBaWaves / CG, COLS = 32 * CT * CG;
  constexpr int STAGE = 32 * KG, FR = KG * KU * 2, PIECES = STAGE * HD / 16, PER = PIECES / kBaThreads;   // 16-byte pieces of K, of V
  using End = TileEnd<HD, CT, CG>;
  constexpr int kBufs = 4 * FR * 1024;
  static_assert(PER * kBaThreads == PIECES, "whole loads");
  __shared__ BaSeg sg;
  __shared__ typename End::Ml ml;
  __shared__ __align__(16) char s_big[kBufs > End::kBytes ? kBufs : End::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_index(), col = lane & 31, c2 = lane >> 5;
  const int cg = wave % CG, kg = wave / CG;
  const int hd = p.c.hd, lbs = p.c.lbs, G = p.G;
  Tile t;
  int kvh;
  long long k0, kend;
  if (!tile_of<E>(p, COLS, &t, &kvh, &k0, &kend)) return;
  const int ncol = t.rows * G;
  int blk = seg_table(p.c, t.s.b, k0, (int)min((long long)kBaSeg, kend - k0));
  v8h_t qf[CT][KU][NQ][2];
  float x[CT][KU][16], sq[CT], l[CT];
  Bases bs[CT];
  long long at[CT];
  v16f_t o[CT][DT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int cc = min((cg * CT + ct) * 32 + col, ncol - 1);
    q_load<E, KU>((const E*)p.q + col_at(t, G, hd, kvh, cc, p.q_ld), hd, x[ct]);
    at[ct] = t.s.p0 + t.i0 + cc / G;
    bs[ct] = Bases{kNoBase, kNoBase};
    l[ct] = 0;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[ct][i] = v16f_t{};
  }
  const long long all_see = t.s.p0 + t.i0 + 1;                // keys below this are seen by every row
  v4i_t kr[PER], vr[PER];
  // What this thread loads of a stage and where it puts it, in parts that no stage changes (an index worked out anew for each is
  // vector work, which the kernel is bound by). Piece j = tid + 256 i of K: token j / (HD / 16), channels 16 (j % (HD / 16)); of
  // V: channel j / (2 KG), tokens 16 (j % (2 KG)). The i'th piece lies KI tokens, VI channels after the first.
  constexpr int KI = kBaThreads / (HD / 16), VI = kBaThreads / (2 * KG);
  static_assert(PER == 1 || (KI % 32 == 0 && VI % 32 == 0), "whole fragments from piece to piece");
  const int8_t *k_from, *v_from[PER];
  int k_put, v_put;
  {
    const int key = tid / (HD / 16), dc = tid % (HD / 16), k16 = key & 15;
    k_from = p.c.kc + (k16 * hd + (dc * 16 < hd ? dc * 16 : 0));
    const int row = 8 * (k16 >> 2) + 4 * (key >> 4 & 1) + (k16 & 3);            // (the token's row of the 32)
    k_put = (((key >> 5) * KU * 2 + (dc >> 1) * 2) * 64 + (((dc & 1) * 32 + row) ^ (dc & 7))) * 16;
    const int ck = tid % (2 * KG), d = tid / (2 * KG);
#pragma unroll
    for (int i = 0; i < PER; ++i) v_from[i] = p.c.vc + (min(d + i * VI, hd - 1) << lbs);
    v_put = ((FR + (ck >> 1) * DT * 2 + (d >> 5) * 2) * 64 + (((ck & 1) * 32 + (d & 31)) ^ (2 * ck & 7))) * 16;
  }
  auto load_k = [&](int st) {
#pragma unroll
    for (int i = 0; i < PER; ++i) kr[i] = *(const v4i_t*)(k_from + sg.k_at[st * 2 * KG + (tid / (HD / 16) >> 4) + i * (KI / 16)]);
  };
  auto load_v = [&](int st) {
    const long long at = sg.v_at[st * 2 * KG + tid % (2 * KG)];
#pragma unroll
    for (int i = 0; i < PER; ++i) vr[i] = *(const v4i_t*)(v_from[i] + at);
  };
  // half of a loaded piece (K's PER, then V's) into its fragment of buffer 0 or 1
  auto put_half = [&](int buf, int h) {
    const int i = h >> 1, half = h & 1;
    char* to = s_big + buf * (2 * FR * 1024);
    if (i < PER) *(v8h_t*)(to + k_put + ((i * KI >> 5) * KU * 2 + half) * 1024) = codes_h(kr[i][2 * half], kr[i][2 * half + 1]);
    else *(v8h_t*)(to + v_put + (((i - PER) * VI >> 5) * 2 + half) * 1024) = codes_h(vr[i - PER][2 * half], vr[i - PER][2 * half + 1]);
  };
  // a segment's blocks, and its first loads
  auto begin = [&](int n) {
    seg_blocks(sg, p.c, blk, kvh, n, STAGE);
    load_k(0);
    load_v(0);
  };
  begin((int)min((long long)kBaSeg, kend - k0));
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) sq[ct] = p.a * q_pieces<E, KU>(hd, x[ct], qf[ct]);
  for (long long seg = k0; seg < kend; seg += kBaSeg) {
    const int n = (int)min((long long)kBaSeg, kend - seg), stages = (n + STAGE - 1) / STAGE, last = stages - 1;
    const bool holes = seg_scales(sg, p.c, blk, kvh, n, STAGE);
    // (past the last stage loads repeat it, and nobody reads what is put of them)
#pragma unroll
    for (int h = 0; h < 4 * PER; ++h) put_half(0, h);
    load_k(min(1, last));
    load_v(min(1, last));
    __syncthreads();
    auto stage = [&](int st, auto edge) {
      const v8h_t* buf = (const v8h_t*)s_big + (st & 1) * 2 * FR * 64;
      const int ch = ((st * STAGE + kg * 32) >> 4) + c2;
      v8h_t kf[KU][2], vf[DT][2];
      auto read_k = [&](int from, int to) {
#pragma unroll
        for (int u = from; u < to; ++u)
#pragma unroll
          for (int half = 0; half < 2; ++half) kf[u][half] = buf[((kg * KU + u) * 2 + half) * 64 + (lane ^ ((2 * u + c2) & 7))];
      };
      read_k(0, KU / 2);                                      // (the others follow while these are used)
      const float ks = sg.ks[ch], ue = sg.ue[ch], uf = sg.uf[ch];
      const int seen = edge.value ? sg.seen[ch] : 16;
      __builtin_amdgcn_sched_barrier(0);
      // The scores; between their products the next stage's codes are converted. (The order is pinned: left to itself the
      // compiler puts all of one before all of the other.)
      v16f_t s[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct] = v16f_t{};
      constexpr int GROUPS = KU * 2, EACH = 4 * PER / GROUPS;
      static_assert(EACH * GROUPS == 4 * PER, "the same number of pieces a group");
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) s[ct] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[g >> 1][g & 1], qf[ct][g >> 1][q][g & 1], s[ct], 0, 0, 0);
        if (g == 0) read_k(KU / 2, KU);
#pragma unroll
        for (int h = 0; h < EACH; ++h) put_half(~st & 1, g * EACH + h);
        __builtin_amdgcn_sched_barrier(0);
      }
      auto read_v = [&](int half) {
#pragma unroll
        for (int i = 0; i < DT; ++i) vf[i][half] = buf[(FR + (kg * DT + i) * 2 + half) * 64 + (lane ^ (2 * (2 * kg + c2) & 7))];
      };
      read_v(0);
      __builtin_amdgcn_sched_barrier(0);
      v8h_t pf[CT][NW][2];
      float sk[CT], add[CT], ls[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        sk[ct] = score_scale(sq[ct], ks);
        add[ct] = soft_max<DT, edge.value>(s[ct], sk[ct], edge.value ? keys_left(at[ct], seg + ch * 16, seen) : 16, ue, uf, bs[ct],
                                           l[ct], o[ct]);
        ls[ct] = 0;
      }
      // The probabilities of 8 keys, then their products; the other 8 keys' between those, the next loads between the last.
      auto weigh = [&](int r) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) ls[ct] += soft_weights<NW>(s[ct], sk[ct], add[ct], pf[ct], r);
      };
#pragma unroll
      for (int r = 0; r < 8; r += 4) weigh(r);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int g = 0; g < NW * DT; ++g) {
          const int q = g / DT, i = g % DT;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) o[ct][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[i][half], pf[ct][q][half], o[ct][i], 0, 0, 0);
          if (half == 0) {
            if (g == 0) read_v(1);
#pragma unroll
            for (int r = 2 + g * 2 / (NW * DT); r < 2 + (g + 1) * 2 / (NW * DT); ++r) weigh(4 * r);
          } else if (g == 0) {
            load_k(min(st + 2, last));
          } else if (g == 1) {
            load_v(min(st + 2, last));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) l[ct] = add_weights(l[ct], ls[ct], add[ct], bs[ct]);
      __syncthreads();                                        // this buffer is read, the other one whole
    };
    const int plain = plain_steps(all_see, seg, n, STAGE, holes);
    int st = 0;
    for (; st < plain; ++st) stage(st, std::false_type());
    for (; st < stages; ++st) stage(st, std::true_type());
    const long long next = seg + kBaSeg;
    if (next < kend) {
      const int m2 = (int)min((long long)kBaSeg, kend - next);
      blk = seg_table(p.c, t.s.b, next, m2);
      begin(m2);
    }
  }
  tile_end<E, HD, CT, CG>(p, t, kvh, blockIdx.y, k0 == 0 && kend == t.end, bs, l, o, ml, (float*)s_big);
}

// Joins the parts of a tile's columns, NWV waves a column
template <class E, int NWV>
__global__ __launch_bounds__(kBaThreads) void k_blk_rows_join(BlkAttn p, int cols) {
  const int w_tile = blockIdx.x / p.c.Hk, kvh = blockIdx.x - w_tile * p.c.Hk;
  Tile t;
  if (!find_tile(p, cols, w_tile, &t) || t.end <= p.chunk) return;
  const int cc = NWV > 1 ? (int)blockIdx.y : (int)blockIdx.y * kBaWaves + wave_index();
  if (cc >= t.rows * p.G) return;
  const int parts = (int)((t.end + p.chunk - 1) / p.chunk);
  float x[2];
  Bases top;
  const float l = join_parts<NWV>(p, ((long long)blockIdx.x * cols + cc) * p.nsplit, parts, &x, &top);
  if (NWV == 1 || wave_index() == 0)
    join_store<E>(p, (E*)p.out + col_at(t, p.G, p.c.hd, kvh, cc, p.out_ld), x, l, top);
}

}  // namespace t2r
