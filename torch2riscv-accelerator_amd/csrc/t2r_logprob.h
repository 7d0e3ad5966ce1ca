// Log probabilities of logits rows: for x[V] with m = max x and l = sum exp(x - m),
//   log p(t) = x[t] - (m + ln l),   entropy = ln l - sum (x - m) exp(x - m) / l,
// and the `top` largest values with their indices (descending, the lower index first on ties, a NaN before everything).
// The logits are read once: a workgroup takes spans of kLpSpan values of a row into registers, the next one's loads in flight,
// and works out their maxima and sums there; k_lp_join joins a row's parts.
//
// fp32 logits are bound by memory (1024 rows of 151936, top 20: 116 us, 5.4 TB/s), 16-bit ones by the vector units: six
// instructions a value, one of them an exponential that counts four times, and what a span needs besides. 2032 rows of 49155:
// 48 us with the top 5 (4.2 TB/s), 42 without; of 128256: 110 us with the top 20 (4.7), 101 without. Few rows: 16 of 128256
// 7.7 us and 6.3 for the join, an empty kernel taking 3.3. Small vocabularies with a large top are slow (the selection below).
#pragma once
#include "t2r_block.h"

namespace t2r {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64, kLpPer = 32, kLpSpan = kLpThreads * kLpPer;
constexpr int kLpMaxTop = 32;
// Loads with candidates that wait for the next spans, at most: more make the selections, whose work grows with the square, the
// dearer (24 / 64 / 200: 112 / 117 / 126 us for the top 20 of 2032 bf16 rows of 128256).
constexpr int kLpMany = 24;
constexpr int kLpKeys = 512;                 // keys that the quick selection holds
constexpr int kLpMaxParts = 64;              // parts of a row
constexpr float kLpNone = -__builtin_inff();
constexpr float kLpSlack = 4.0f;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;
// Sums run about c = F(m log2 e) in powers of two, l = sum 2^t and e = sum t 2^t with t = x log2 e - c, one fused step a
// value; past this size, where x log2 e or c may overflow, t = (x - m) log2 e instead and c stands for m log2 e exactly.
constexpr float kLpHuge = 1e37f;
// how far c lies below m log2 e: l is too large by 2^this
T2R_DEV float lp_low(float m) { return fabsf(m) < kLpHuge ? __builtin_fmaf(m, kLog2e, -(m * kLog2e)) : 0.0f; }
// sums about m moved to the larger maximum n
T2R_DEV void lp_move(float m, float n, float* l, float* e) {
  float d = (m - n) * kLog2e;
  if (fabsf(m) < kLpHuge && fabsf(n) < kLpHuge) d = m * kLog2e - n * kLog2e;
  if (*l == 0) return;                                                 // (d may be -inf)
  const float f = __builtin_amdgcn_exp2f(d);
  const float to = *l * f;                                             // (a NaN stays)
  *e = f == 0 ? to : (*e + d * *l) * f;
  *l = to;
}

struct LpArgs {
  const void* x;
  long long ld;
  const int32_t* tokens;
  int rows, V, top, spans, parts;            // spans of kLpSpan values a part takes, parts of a row
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_lp;
  unsigned long long* ws_key;                // [rows, parts, top]: a part's largest values as keys
  float* ws_sum;                             // [rows, parts, 4]: its (m, l, e)
};

// values in an order of unsigned numbers: -0 as +0, a NaN above +inf
constexpr uint32_t kOrderNone = 0x007FFFFFu;                           // of -inf, the least
T2R_DEV uint32_t order_of(float x) {
  const uint32_t u = fb(x + 0.0f);
  return x != x ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
T2R_DEV float order_value(uint32_t o) { return o == 0xFFFFFFFFu ? fv(kQNaN) : fv(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o); }
T2R_DEV unsigned long long lp_key(float x, uint32_t i) { return ((unsigned long long)order_of(x) << 32) | (uint32_t)~i; }
T2R_DEV float key_value(unsigned long long k) { return order_value((uint32_t)(k >> 32)); }
// f over the wave's values, to every lane (f needs no order)
template <class F> T2R_DEV float wave_all(float x, F f) {
  x = f(x, dpp_f<kDppXor1>(x));
  x = f(x, dpp_f<kDppXor2>(x));
  x = f(x, dpp_f<kDppHalfMirror>(x));
  x = f(x, dpp_f<kDppMirror>(x));
  auto of = [&](int lane) { return fv((uint32_t)__builtin_amdgcn_readlane((int)fb(x), lane)); };
  return f(f(of(0), of(16)), f(of(32), of(48)));
}
T2R_DEV float wave_top(float x) { return wave_all(x, [](float a, float b) { return fmaxf(a, b); }); }
T2R_DEV float wave_total(float x) { return wave_all(x, [](float a, float b) { return a + b; }); }
// the largest key of the wave, to every lane
template <int CTRL> T2R_DEV unsigned long long key_dpp(unsigned long long k) {
  const unsigned long long o = ((unsigned long long)(uint32_t)dpp_i<CTRL>((int)(k >> 32)) << 32) | (uint32_t)dpp_i<CTRL>((int)(uint32_t)k);
  return o > k ? o : k;
}
T2R_DEV unsigned long long wave_key(unsigned long long k) {
  k = key_dpp<kDppMirror>(key_dpp<kDppHalfMirror>(key_dpp<kDppXor2>(key_dpp<kDppXor1>(k))));
  auto of = [&](int lane) {
    return ((unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, lane);
  };
  const unsigned long long a = max(of(0), of(16)), b = max(of(32), of(48));
  return max(a, b);
}

struct LpLds {
  unsigned long long best[2][kLpMaxTop];     // the largest so far, in order (0: none), before and after a selection
  unsigned long long key[kLpKeys];
  int cand[kLpMany + kLpSpan / 4];           // loads with candidates: where they begin in the row
  float grp[kLpThreads / 4];
  unsigned long long redk[kLpWaves];
  float red[3][kLpWaves];
  int n[3];                                  // a span's loads with candidates, the next one's, those of the one before
  int keys;
};

// What is told of a row: from m, l and e, and its largest keys in order.
template <class E> T2R_DEV float lp_logit(const LpArgs& p, int row) {
  const int t = p.tokens[row];
  return t >= 0 && t < p.V ? widen(((const E*)p.x)[(long long)row * p.ld + t]) : fv(kQNaN);
}
T2R_DEV void lp_sums(const LpArgs& p, int row, float xt, float m, float l, float e, float* lse) {
  // a row with nothing above -inf has no distribution: every log p is -inf, the entropy 0
  const float ln = l == 0 ? 0.0f : logf(l);
  *lse = m == kLpNone ? ln : m + (ln - kLn2 * lp_low(m));
  if (threadIdx.x == 0) {
    if (p.logprob) p.logprob[row] = xt - *lse;
    if (p.entropy) p.entropy[row] = l == 0 ? 0.0f : ln - kLn2 * (e / l);
  }
}
T2R_DEV void lp_top(const LpArgs& p, int row, int place, unsigned long long k, float lse) {
  p.top_ids[(long long)row * p.top + place] = (int32_t)~(uint32_t)k;
  p.top_lp[(long long)row * p.top + place] = key_value(k) - lse;
}

template <class E>
__global__ __launch_bounds__(kLpThreads, 4) void k_lp_part(LpArgs p) {
  constexpr int PER = 16 / sizeof(E), NL = kLpPer / PER;              // values of a load, loads of a thread
  struct __attribute__((packed, aligned(sizeof(E)))) Vec { v4i_t v; };
  __shared__ LpLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts, top = p.top, V = p.V;
  const E* x = (const E*)p.x + (long long)row * p.ld;
  if (tid < 2 * kLpMaxTop) (&s.best[0][0])[tid] = 0;                   // (both rows: a part may hold fewer than top values)
  if (tid < 3) s.n[tid] = 0;
  if (tid == 0) s.keys = 0;
  int now = 0;                                                         // the row of s.best that holds
  // This thread's sums so far run about a value m of its own, no further than kLpSlack below its maximum: only the end brings
  // the threads together, and few spans move it.
  float m = kLpNone, l = 0, e = 0;
  // Load i of a thread begins at place (i kLpThreads + tid) PER of its span. Spans of long rows begin `off` values before the
  // row, so that whole ones are loaded at multiples of 16 bytes (odd rows of 49155 values took 46 us of loads and sums, 43
  // so). A load over the row's beginning or end is moved inside; the values that are another load's too count as -inf
  // then. Loads are issued a span ahead.
  v4i_t w[NL];
  const int off = V >= kLpSpan ? (int)((uintptr_t)x % 16 / sizeof(E)) : 0;
  auto start_of = [&](int sp) { return ((long long)part * p.spans + sp) * kLpSpan - off; };
  // the places of a span at i0 where the row begins, and where its last PER values do (before the span where few are left)
  auto first_of = [&](long long i0) { return (int)max(-i0, 0LL); };
  auto last_of = [&](long long i0) { return (int)min(V - PER - i0, (long long)kLpSpan); };
  auto fetch = [&](int sp) {
    const long long i0 = start_of(sp);
    if (sp >= p.spans || i0 >= V) return;
    if (i0 >= 0 && i0 + kLpSpan <= V) {
#pragma unroll
      for (int i = 0; i < NL; ++i) w[i] = ((const v4i_t*)(x + i0 + i * kLpThreads * PER))[tid];
    } else if (V >= PER) {
      const int first = first_of(i0), last = last_of(i0);
#pragma unroll
      for (int i = 0; i < NL; ++i) w[i] = ((const Vec*)(x + i0 + min(max((i * kLpThreads + tid) * PER, first), last)))->v;
    } else {
      // a row of fewer values than a load takes: thread 0's first load, by hand, its values at the end
      for (int i = 0; i < NL; ++i) w[i] = v4i_t{0, 0, 0, 0};
      E* e0 = (E*)&w[0];
      for (int j = 0; j < PER; ++j)
        if (j >= PER - V) e0[j] = x[j - (PER - V)];
    }
  };
  // The candidates in the first n noted loads, and what was best, into the best: a key's rank is the number of larger ones (keys
  // differ: their indices do; 0 is none).
  uint32_t bound = 0;                                                  // of a candidate's order from below
  auto value_key = [&](int c) {                                        // value c of the noted loads
    const int i = s.cand[c / PER] + c % PER;
    if (i < 0 || i >= V) return 0ull;
    const unsigned long long k = lp_key(widen(x[i]), (uint32_t)i);
    return (uint32_t)(k >> 32) >= bound ? k : 0ull;
  };
  auto settle = [&](int n) {
    if (n == 0) return;
    for (int c = tid; c < n * PER; c += kLpThreads) {
      const unsigned long long k = value_key(c);
      if (k == 0) continue;
      const int at = atomicAdd(&s.keys, 1);
      if (at < kLpKeys) s.key[at] = k;
    }
    __syncthreads();
    int nk = s.keys;
    if (nk > kLpKeys) {
      // Too many: the largest one by one. Equal values, or rows whose values lie with fewer threads than the first span's bound
      // has groups for, so that every value is a candidate: 513 to 608 values of 16 bits with the top 20, 513 to 992 with the top
      // 32. (2032 such rows of 600: 140 and 210 us; of 500, by rank among 500 keys, 87; of 1000 with the top 20, under a bound, 15.)
      unsigned long long below = ~0ull;
      for (nk = 0; nk < top; ++nk) {
        unsigned long long b = 0;
        for (int c = tid; c < n * PER; c += kLpThreads) {
          const unsigned long long k = value_key(c);
          b = k < below && k > b ? k : b;
        }
        b = wave_key(b);
        if (lane == 0) s.redk[wave] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) b = s.redk[w] > b ? s.redk[w] : b;
        below = b;
        if (tid == 0) s.key[nk] = b;
        __syncthreads();
      }
    }
    const unsigned long long* was = s.best[now];
    unsigned long long* next = s.best[now ^ 1];
    for (int i = tid; i < nk + top; i += kLpThreads) {
      const unsigned long long k = i < nk ? s.key[i] : was[i - nk];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < nk; ++j) r += s.key[j] > k;
#pragma unroll 4
      for (int j = 0; j < top; ++j) r += was[j] > k;
      if (k != 0 && r < top) next[r] = k;
    }
    now ^= 1;
    __syncthreads();
    if (tid == 0) s.keys = 0;                                          // (every thread has read it; the next span's barrier follows)
    bound = max(bound, (uint32_t)(s.best[now][top - 1] >> 32));
  };
  int noted = 0;                                                       // loads of earlier spans
  fetch(0);
  for (int sp = 0; sp < p.spans; ++sp) {
    const long long i0 = start_of(sp);
    if (i0 >= V) break;
    const int turn = sp % 3;
    const bool whole = i0 >= 0 && i0 + kLpSpan <= V;
    uint32_t mine = ~0u;                                               // the values of its loads that are this thread's
    if (!whole) {
      const int first = first_of(i0), last = last_of(i0);
      mine = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int at = (i * kLpThreads + tid) * PER, before = min(max(first - at, 0), PER), past = min(max(at - last, 0), PER);
        mine |= ((1u << PER) - 1) >> before >> past << past << (i * PER);
      }
    }
    const bool some = whole || __any(mine != 0);                       // (the row's last span may leave a wave nothing)
    float v[kLpPer], lm[NL], tm = kLpNone, ls = 0;                     // the maxima of the loads, and of all of them
    if (some) {
#pragma unroll
      for (int i = 0; i < kLpPer; ++i) {
        if constexpr (sizeof(E) == 4) v[i] = fv((uint32_t)w[i / PER][i % PER]);
        else v[i] = widen(__builtin_bit_cast(E, (uint16_t)((uint32_t)w[i / PER][i % PER >> 1] >> (16 * (i & 1)))));
      }
      fetch(sp + 1);
      if (!whole && __any(mine != ~0u)) {
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) v[i] = mine >> i & 1 ? v[i] : kLpNone;
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        lm[i] = v[i * PER];
#pragma unroll
        for (int j = 1; j < PER; ++j) lm[i] = fmaxf(lm[i], v[i * PER + j]);
        tm = fmaxf(tm, lm[i]);
      }
      if (tm > m + kLpSlack) {
        if (m != kLpNone) lp_move(m, tm, &l, &e);                      // (else both are 0, or NaN and stay that)
        m = tm;
      }
      const float mu = m == kLpNone ? 0.0f : m;
      if (fabsf(mu) < kLpHuge) {
        const float c = mu * kLog2e;
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) {
          const float t = __builtin_fmaf(v[i], kLog2e, -c), q = __builtin_amdgcn_exp2f(t);
          ls += q;
          e = __builtin_fmaf(q, fmaxf(t, -200.0f), e);                 // (q is 0 there: -inf adds nothing)
        }
      } else {
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) {
          const float t = (v[i] - mu) * kLog2e, q = __builtin_amdgcn_exp2f(t);
          ls += q;
          e = __builtin_fmaf(q, fmaxf(t, -200.0f), e);
        }
      }
      l += ls;
    }
    if (top == 0) continue;
    // A lower bound of the top-th largest value: the last of the best so far, or before the first selection the top-th largest
    // of the first span's maxima of 64 groups of 4 threads, to its upper 16 bits. Loads that hold something at or above it, a
    // dozen of a span's 1024 or 2048 as a rule, are noted, and selected from at the end or once they are many.
    if (sp == 0) {
      float gm = fmaxf(tm, dpp_f<kDppXor1>(tm));
      gm = fmaxf(gm, dpp_f<kDppXor2>(gm));
      if ((tid & 3) == 0) s.grp[tid >> 2] = gm;
      __syncthreads();
      const uint32_t og = order_of(s.grp[lane]);
#pragma unroll
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | (1u << bit);
        bound = __popcll(__ballot(og >= t)) >= top ? t : bound;
      }
      bound = max(bound, kOrderNone);
    }
    const float least = order_value(bound);
    if (tid == 0) s.n[(sp + 1) % 3] = 0;                               // (last read two spans ago)
    const bool nan = ls != ls;                                         // (a NaN among the values, or an infinity)
    if (some && (tm >= least || nan)) {
      int set = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) set |= lm[i] >= least || nan ? 1 << i : 0;
      // one place for all of a thread's (an atomic and its wait for each value took 90 us of 190 in 2032 rows of 49155)
      for (int c = noted + atomicAdd(&s.n[turn], __popc(set)); set != 0; set &= set - 1, ++c)
        s.cand[c] = (int)i0 + (__builtin_ctz(set) * kLpThreads + tid) * PER;
    }
    __syncthreads();
    noted += s.n[turn];
    if (noted > kLpMany || sp + 1 == p.spans || i0 + kLpSpan >= V) {
      settle(noted);
      noted = 0;
    }
  }
  // the sums over the threads, about the largest m
  float all = wave_top(m);
  if (lane == 0) s.red[0][wave] = all;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) all = fmaxf(all, s.red[0][w]);
  if (l == l) lp_move(m, all, &l, &e);
  m = all;
  l = wave_total(l);
  e = wave_total(e);
  if (lane == 0) {
    s.red[1][wave] = l;
    s.red[2][wave] = e;
  }
  __syncthreads();
  l = e = 0;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    l += s.red[1][w];
    e += s.red[2][w];
  }
  if (p.parts == 1) {
    float lse;
    lp_sums(p, row, p.logprob ? lp_logit<E>(p, row) : 0.0f, m, l, e, &lse);
    if (tid < top) lp_top(p, row, tid, s.best[now][tid], lse);
    return;
  }
  const long long at = (long long)row * p.parts + part;
  if (tid == 0) *(v4f_t*)(p.ws_sum + 4 * at) = v4f_t{m, l, e, 0};
  if (tid < top) p.ws_key[at * top + tid] = s.best[now][tid];
}

// A row's parts: the maximum and the sums, then the largest keys by rank. A part's last key bounds the row's from below (its
// part alone has `top` keys from it on), so few of the others are ranked.
template <class E>
__global__ __launch_bounds__(kLpThreads) void k_lp_join(LpArgs p) {
  __shared__ unsigned long long key[kLpMaxParts * kLpMaxTop];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x, top = p.top, parts = p.parts;
  v4f_t sum = {kLpNone, 0, 0, 0};
  unsigned long long last = 0;
  const unsigned long long* from = p.ws_key + (long long)row * parts * top;
  // (the token is waited for, for its range; then its logit, the keys and the sums are asked for together)
  float xt = fv(kQNaN);
  if (p.logprob) xt = lp_logit<E>(p, row);
  constexpr int KEYS = kLpMaxParts * kLpMaxTop / kLpThreads;
  unsigned long long mine[KEYS];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) mine[i] = tid + i * kLpThreads < parts * top ? from[tid + i * kLpThreads] : 0;
  if (lane < parts) {
    sum = *(const v4f_t*)(p.ws_sum + 4 * ((long long)row * parts + lane));
    if (top > 0) last = from[lane * top + top - 1];
  }
  if (tid == 0) s_n = 0;
  const float m = wave_top(sum[0]);
  last = wave_key(last);
  float l = sum[1], e = sum[2];
  if (l == l) lp_move(sum[0], m, &l, &e);
  l = wave_total(l);
  e = wave_total(e);
  float lse;
  lp_sums(p, row, xt, m, l, e, &lse);
  if (top == 0) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < KEYS; ++i)
    if (mine[i] != 0 && mine[i] >= last) key[atomicAdd(&s_n, 1)] = mine[i];
  __syncthreads();
  const int n = s_n;
  for (int i = tid; i < n; i += kLpThreads) {
    const unsigned long long k = key[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += key[j] > k;
    if (r < top) lp_top(p, row, r, k, lse);
  }
}

}  // namespace t2r
