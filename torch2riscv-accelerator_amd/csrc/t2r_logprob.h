// Log probabilities of logits rows: for x[V] with m = max x and l = sum exp(x - m),
//   log p(t) = x[t] - (m + ln l),   entropy = ln l - sum (x - m) exp(x - m) / l,
// and the `top` largest values with their indices (descending, the lower index first on ties, a NaN before everything).
// The logits are read once: a workgroup takes parts of kLpSpan values of a row into registers and works out their maximum,
// sums and largest values there; k_lp_join joins a row's parts.
#pragma once
#include "t2r_block.h"

namespace t2r {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64, kLpPer = 32, kLpSpan = kLpThreads * kLpPer;
constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 512;                 // candidates that a span's quick selection holds
constexpr int kLpMaxParts = 64;              // parts of a row
constexpr float kLpNone = -__builtin_inff();
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
  *e = (*e + d * *l) * f;
  *l *= f;
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
T2R_DEV unsigned long long shfl_key(unsigned long long k, int from_xor) {
  const uint32_t lo = __shfl_xor((int)(uint32_t)k, from_xor), hi = __shfl_xor((int)(uint32_t)(k >> 32), from_xor);
  return ((unsigned long long)hi << 32) | lo;
}
template <int CTRL> T2R_DEV float max_dpp(float x) {
  return fmaxf(x, fv((uint32_t)__builtin_amdgcn_update_dpp(0, (int)fb(x), CTRL, 0xF, 0xF, false)));
}

struct LpLds {
  unsigned long long best[2][kLpMaxTop];     // the largest so far, in order (0: none), before and after a span
  unsigned long long cand[kLpCand];
  float grp[2][kLpThreads / 4];
  unsigned long long redk[kLpWaves];
  float red[2][kLpWaves];
  int n[2];
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
  constexpr int PER = 16 / sizeof(E), NL = kLpPer / PER;              // elements of a load, loads of a thread
  struct __attribute__((packed, aligned(sizeof(E)))) Vec { v4i_t v; };
  __shared__ LpLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts, top = p.top, V = p.V;
  const E* x = (const E*)p.x + (long long)row * p.ld;
  if (tid < 2 * kLpMaxTop) (&s.best[0][0])[tid] = 0;                         // (both rows: a part may hold fewer than top values)
  if (tid == 0) s.n[0] = 0;
  int now = 0;                                                         // the row of s.best that holds
  float m = kLpNone, l = 0, e = 0;                                     // of the part so far; l and e this thread's
  Vec w[NL];
  // a whole span's loads, issued a span ahead
  auto fetch = [&](int sp) {
    const long long i0 = ((long long)part * p.spans + sp) * kLpSpan;
    if (sp < p.spans && i0 + kLpSpan <= V) {
#pragma unroll
      for (int i = 0; i < NL; ++i) w[i] = ((const Vec*)(x + i0 + i * kLpThreads * PER))[tid];
    }
  };
  fetch(0);
  for (int sp = 0; sp < p.spans; ++sp) {
    const long long i0 = ((long long)part * p.spans + sp) * kLpSpan;
    if (i0 >= V) break;
    const int n = (int)min((long long)kLpSpan, V - i0), odd = sp & 1;
    // Load i of a thread takes the PER values from place (i kLpThreads + tid) PER of the span on. In a span that the row's end
    // cuts, loads past it are moved back to the row's last PER values; of those the first skip(i) lie before the thread's
    // place (another load has them) and count as -inf.
    const int lastv = n - PER;
    // (the places are worked out anew in every span: kept over the loop they would take 60 registers more than there are)
    int tq = tid;
    asm volatile("" : "+v"(tq));
    auto place = [&](int i) { return (i * kLpThreads + tq) * PER; };
    auto skip = [&](int i) { return max(place(i) - lastv, 0); };
    float v[kLpPer];
    const bool whole = n == kLpSpan;
    if (whole) {
    } else if (V >= PER) {
#pragma unroll
      for (int i = 0; i < NL; ++i) w[i] = *(const Vec*)(x + (i0 + min(place(i), lastv)));
    } else {
      // a row of fewer values than a load takes: thread 0's first load, by hand, its values at the end
      for (int i = 0; i < NL; ++i) w[i].v = v4i_t{0, 0, 0, 0};
      E* e0 = (E*)&w[0];
      for (int j = 0; j < PER; ++j)
        if (j >= PER - V) e0[j] = x[j - (PER - V)];
    }
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) {
      if constexpr (sizeof(E) == 4) v[i] = fv((uint32_t)w[i / PER].v[i % PER]);
      else v[i] = widen(__builtin_bit_cast(E, (uint16_t)((uint32_t)w[i / PER].v[i % PER >> 1] >> (16 * (i & 1)))));
    }
    fetch(sp + 1);
    uint32_t mine = ~0u;                                               // the values of its loads that are this thread's
    if (!whole) {
      mine = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i) mine |= ((1u << PER) - 1) >> min(skip(i), PER) << min(skip(i), PER) << (i * PER);
#pragma unroll
      for (int i = 0; i < kLpPer; ++i) v[i] = mine >> i & 1 ? v[i] : kLpNone;
    }
    // value i again, from the cache: an index into registers would put them all into memory
    auto key = [&](int i) {
      const int at = place(i / PER) - (whole ? 0 : skip(i / PER)) + i % PER;
      return lp_key(widen(x[i0 + at]), (uint32_t)(i0 + at));
    };
    float lm[NL], tm = kLpNone;                                        // the maxima of the loads, and of all of them
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      lm[i] = v[i * PER];
#pragma unroll
      for (int j = 1; j < PER; ++j) lm[i] = fmaxf(lm[i], v[i * PER + j]);
      tm = fmaxf(tm, lm[i]);
    }
    // the maxima of the 64 groups of 4 threads, to every wave: the span's maximum, and below the bound of its largest
    const float gm = max_dpp<0x4E>(max_dpp<0xB1>(tm));
    if ((tid & 3) == 0) s.grp[odd][tid >> 2] = gm;
    __syncthreads();
    const float g = s.grp[odd][lane];
    float bm = max_dpp<0x121>(max_dpp<0x122>(max_dpp<0x124>(max_dpp<0x128>(g))));      // of 16 lanes
    bm = fmaxf(bm, __shfl_xor(bm, 16));
    bm = fmaxf(m, fmaxf(bm, __shfl_xor(bm, 32)));
    if (bm > m) {                                                      // (uniform)
      if (m != kLpNone) lp_move(m, bm, &l, &e);                        // (else both are 0, or NaN and stay that)
      m = bm;
    }
    const float mu = m == kLpNone ? 0.0f : m;
    float ls = 0;
    if (!whole && !__any(mine != 0)) {
      // (a wave that the row's last span leaves nothing)
    } else if (fabsf(mu) < kLpHuge) {
      const float c = mu * kLog2e;
#pragma unroll
      for (int i = 0; i < kLpPer; ++i) {
        const float t = __builtin_fmaf(v[i], kLog2e, -c), q = __builtin_amdgcn_exp2f(t);
        ls += q;
        e = __builtin_fmaf(q, fmaxf(t, -200.0f), e);                   // (q is 0 there: -inf adds nothing)
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
    if (top == 0) continue;
    // A lower bound of the top-th largest value: the last of the best so far, or in the first span the top-th largest of the
    // groups' maxima, to its upper 16 bits. What lies at or above it is a candidate: a few dozen of 8192 values as a rule.
    uint32_t bound = (uint32_t)(s.best[now][top - 1] >> 32);
    if (bound == 0) {
      const uint32_t og = order_of(g);
#pragma unroll
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = bound | (1u << bit);
        bound = __popcll(__ballot(og >= t)) >= top ? t : bound;
      }
    }
    const float least = order_value(max(bound, kOrderNone));
    if (tid == 0) s.n[odd ^ 1] = 0;
    const bool nan = ls != ls;                                         // (a NaN among the values, or an infinity)
    if (tm >= least || nan) {
      uint32_t set = 0;
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (lm[i] >= least) {
#pragma unroll
          for (int j = 0; j < PER; ++j) set |= v[i * PER + j] >= least ? 1u << (i * PER + j) : 0u;
        }
      if (nan) {
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) set |= v[i] != v[i] ? 1u << i : 0u;
      }
      set &= mine;
      // one place for all of a thread's (an atomic and its wait for each took 90 us of 190 in 2032 rows of 49155)
      int c = set ? atomicAdd(&s.n[odd], __popc(set)) : 0;
      for (; set != 0; set &= set - 1, ++c)
        if (c < kLpCand) s.cand[c] = key(__builtin_ctz(set));
    }
    __syncthreads();
    int nc = s.n[odd];
    if (nc > kLpCand) {
      // many equal values: the span's largest keys one by one
      unsigned long long below = ~0ull;
      for (int c = 0; c < top; ++c) {
        unsigned long long b = 0;
#pragma unroll 4
        for (int i = 0; i < kLpPer; ++i) {
          const unsigned long long k = mine >> i & 1 ? key(i) : 0;
          b = k < below && k > b ? k : b;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
          const unsigned long long k = shfl_key(b, o);
          b = k > b ? k : b;
        }
        if (lane == 0) s.redk[wave] = b;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) b = s.redk[w] > b ? s.redk[w] : b;
        below = b;
        if (tid == 0) s.cand[c] = b;
        __syncthreads();
      }
      nc = top;
    }
    if (nc > 0) {                                                      // (uniform)
      // each key's rank is the number of larger ones (keys differ: their indices do; 0 is none)
      const unsigned long long* was = s.best[now];
      unsigned long long* next = s.best[now ^ 1];
      for (int i = tid; i < nc + top; i += kLpThreads) {
        const unsigned long long k = i < nc ? s.cand[i] : was[i - nc];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < nc; ++j) r += s.cand[j] > k;
#pragma unroll 4
        for (int j = 0; j < top; ++j) r += was[j] > k;
        if (k != 0 && r < top) next[r] = k;
      }
      now ^= 1;
    }
  }
  // the sums over the threads
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o);
    e += __shfl_xor(e, o);
  }
  if (lane == 0) {
    s.red[0][wave] = l;
    s.red[1][wave] = e;
  }
  __syncthreads();
  l = e = 0;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    l += s.red[0][w];
    e += s.red[1][w];
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
  // (the token's logit and the keys are asked for before anything waits)
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
  float m = sum[0];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor(m, o));
    const unsigned long long k = shfl_key(last, o);
    last = k > last ? k : last;
  }
  float l = sum[1], e = sum[2];
  if (l == l) lp_move(sum[0], m, &l, &e);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o);
    e += __shfl_xor(e, o);
  }
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
