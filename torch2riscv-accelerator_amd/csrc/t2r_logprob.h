// Log probabilities of logits rows: for x[V] with m = max x and l = sum exp(x - m),
//   log p(t) = x[t] - m - ln l,   entropy = ln l - sum (x - m) exp(x - m) / l,
// and the `top` largest values with their indices (descending, the lower index first on ties, a NaN before everything).
// The logits are read once: a workgroup takes parts of kLpSpan values of a row into registers and works out their maximum,
// sums and largest values there; k_lp_join joins a row's parts.
#pragma once
#include "t2r_block.h"

namespace t2r {

constexpr int kLpThreads = 256, kLpPer = 32, kLpSpan = kLpThreads * kLpPer;
constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 512;                 // candidates that a part's quick selection holds
constexpr float kNegInfLp = -__builtin_inff();
// e^x
T2R_DEV float exp_lp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// what a part leaves: (m, l, e) and its largest values as keys
struct LpArgs {
  const void* x;
  long long ld;
  const int32_t* tokens;
  int rows, V, top, spans, parts;            // spans of kLpSpan values a part takes, parts of a row
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_lp;
  unsigned long long* ws_key;                // [rows, parts, top]
  float* ws_sum;                             // [rows, parts, 4]
};

// values in an order of unsigned numbers: -0 as +0, a NaN above +inf
T2R_DEV uint32_t order_of(float x) {
  const uint32_t u = fb(x + 0.0f);
  return x != x ? 0xFFFFFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
T2R_DEV unsigned long long lp_key(float x, uint32_t i) { return ((unsigned long long)order_of(x) << 32) | (uint32_t)~i; }
T2R_DEV float key_value(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return o == 0xFFFFFFFFu ? fv(kQNaN) : fv(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
T2R_DEV unsigned long long shfl_key(unsigned long long k, int from_xor) {
  const uint32_t lo = __shfl_xor((int)(uint32_t)k, from_xor), hi = __shfl_xor((int)(uint32_t)(k >> 32), from_xor);
  return ((unsigned long long)hi << 32) | lo;
}

struct LpLds {
  unsigned long long best[kLpMaxTop];        // the largest so far, in order (0: none)
  unsigned long long cand[kLpCand + kLpMaxTop];
  uint32_t grp[64];
  unsigned long long redk[kLpThreads / 64];
  float red[2][kLpThreads / 64];
  uint32_t least;
  int n;
};

// (two rows of s.red in turn: one barrier a call)
T2R_DEV float block_max(LpLds& s, float v, int turn) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  float* r = s.red[turn & 1];
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
}

// the `top` largest of n keys in s.cand into s.best, in order: each key's rank is the number of larger ones (keys differ:
// their indices do; empty places hold 0 and are not written)
T2R_DEV void rank_cand(LpLds& s, int n, int top) {
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const unsigned long long k = s.cand[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += s.cand[j] > k;
    if (k != 0 && r < top) s.best[r] = k;
  }
}

template <class E>
__global__ __launch_bounds__(kLpThreads) void k_lp_part(LpArgs p) {
  constexpr int PER = 16 / sizeof(E), NL = kLpPer / PER;              // elements of a load, loads of a thread
  struct __attribute__((packed, aligned(sizeof(E)))) Vec { v4i_t v; };
  __shared__ LpLds s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts, top = p.top, V = p.V;
  const E* x = (const E*)p.x + (long long)row * p.ld;
  if (tid < kLpMaxTop) s.best[tid] = 0;
  float m = kNegInfLp, l = 0, e = 0;                                   // of the part so far
  for (int sp = 0; sp < p.spans; ++sp) {
    const long long i0 = ((long long)part * p.spans + sp) * kLpSpan;
    if (i0 >= V) break;
    const int n = (int)min((long long)kLpSpan, V - i0);
    float v[kLpPer];
    // element of (load i, place j): (i * kLpThreads + tid) * PER + j
    if (n == kLpSpan) {
      Vec w[NL];
#pragma unroll
      for (int i = 0; i < NL; ++i) w[i] = *(const Vec*)(x + i0 + (i * kLpThreads + tid) * PER);
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if constexpr (sizeof(E) == 4) v[i * PER + j] = fv((uint32_t)w[i].v[j]);
          else v[i * PER + j] = widen(__builtin_bit_cast(E, (uint16_t)((uint32_t)w[i].v[j >> 1] >> (16 * (j & 1)))));
        }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int at = (i * kLpThreads + tid) * PER + j;
          v[i * PER + j] = at < n ? widen(x[i0 + at]) : kNegInfLp;
        }
    }
    float tm = kNegInfLp;
    bool tn = false;
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) {
      tm = fmaxf(tm, v[i]);
      tn |= v[i] != v[i];
    }
    const float bm = fmaxf(m, block_max(s, tm, sp));
    if (bm > m) {                                                      // (uniform)
      // sums kept about the old maximum move to the new one: exp(x - bm) = exp(x - m) exp(m - bm)
      if (m != kNegInfLp) {                                            // (else both are 0, or NaN and stay that)
        const float d = m - bm, f = exp_lp(d);
        e = (e + d * l) * f;
        l *= f;
      }
      m = bm;
    }
    const float mu = m == kNegInfLp ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < kLpPer; ++i) {
      const float d = v[i] - mu, q = exp_lp(d);
      l += q;
      e += q > 0 ? q * d : 0.0f;                                       // (a value of -inf adds nothing)
    }
    if (top > 0) {
      // A lower bound of the top-th largest value: that of the maxima of 64 groups of 4 threads. What lies at or above it
      // (and above the last of the best so far) is a candidate: a few dozen of the span's 8192 values as a rule.
      const uint32_t to = tn ? 0xFFFFFFFFu : order_of(tm);
      uint32_t gm = max(to, (uint32_t)__shfl_xor((int)to, 1));
      gm = max(gm, (uint32_t)__shfl_xor((int)gm, 2));
      if ((tid & 3) == 0) s.grp[tid >> 2] = gm;
      if (tid == 0) s.n = 0;
      __syncthreads();
      if (wave == 0) {
        const uint32_t g = s.grp[lane];
        int r = 0;
#pragma unroll 8
        for (int j = 0; j < 64; ++j) {
          const uint32_t h = (uint32_t)__builtin_amdgcn_readlane((int)g, j);
          r += h > g || (h == g && j < lane);
        }
        if (r == top - 1) s.least = g;
      }
      __syncthreads();
      const unsigned long long last = s.best[top - 1];
      const uint32_t least = max(s.least, (uint32_t)(last >> 32));
      if (to >= least) {
#pragma unroll
        for (int i = 0; i < kLpPer; ++i) {
          const int at = (i / PER * kLpThreads + tid) * PER + i % PER;
          if (at < n && order_of(v[i]) >= least) {
            const unsigned long long k = lp_key(v[i], (uint32_t)(i0 + at));
            if (k > last) {
              const int c = atomicAdd(&s.n, 1);
              if (c < kLpCand) s.cand[c] = k;
            }
          }
        }
      }
      __syncthreads();
      const int found = s.n;
      if (found > kLpCand) {
        // many equal values: the span's largest keys one by one
        unsigned long long below = ~0ull;
        for (int c = 0; c < top; ++c) {
          unsigned long long b = 0;
#pragma unroll
          for (int i = 0; i < kLpPer; ++i) {
            const int at = (i / PER * kLpThreads + tid) * PER + i % PER;
            const unsigned long long k = at < n ? lp_key(v[i], (uint32_t)(i0 + at)) : 0;
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
          for (int w = 0; w < kLpThreads / 64; ++w) b = s.redk[w] > b ? s.redk[w] : b;
          below = b;
          if (tid == 0) s.cand[c] = b;
          __syncthreads();
        }
      }
      const int nc = found > kLpCand ? top : found;
      if (nc > 0) {                                                    // (uniform)
        if (tid < top) s.cand[nc + tid] = s.best[tid];
        __syncthreads();
        rank_cand(s, nc + top, top);
      }
      __syncthreads();
    }
  }
  // the sums over the threads: every thread's are about the same m
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l += __shfl_xor(l, o);
    e += __shfl_xor(e, o);
  }
  __syncthreads();
  if (lane == 0) {
    s.red[0][wave] = l;
    s.red[1][wave] = e;
  }
  __syncthreads();
  const long long at = (long long)row * p.parts + part;
  if (tid == 0) {
    float L = 0, S = 0;
#pragma unroll
    for (int w = 0; w < kLpThreads / 64; ++w) {
      L += s.red[0][w];
      S += s.red[1][w];
    }
    *(v4f_t*)(p.ws_sum + 4 * at) = v4f_t{m, L, S, 0};
  }
  if (tid < top) p.ws_key[at * top + tid] = s.best[tid];
}

// A row's parts: the maximum and the sums, then the largest keys by rank.
template <class E>
__global__ __launch_bounds__(kLpThreads) void k_lp_join(LpArgs p) {
  __shared__ unsigned long long key[kLpCand];
  __shared__ unsigned long long best[kLpMaxTop];
  const int tid = threadIdx.x, row = blockIdx.x, top = p.top, parts = p.parts;
  const float* sum = p.ws_sum + 4LL * row * parts;
  float m = kNegInfLp;
  for (int i = 0; i < parts; ++i) m = fmaxf(m, sum[4 * i]);
  const float mu = m == kNegInfLp ? 0.0f : m;
  float l = 0, e = 0;
  for (int i = 0; i < parts; ++i) {
    const float pl = sum[4 * i + 1];
    if (pl > 0 || pl != pl) {
      const float d = sum[4 * i] - mu, f = exp_lp(d);
      l += pl * f;
      e += (sum[4 * i + 2] + d * pl) * f;
    }
  }
  // a row with nothing above -inf has no distribution: every log p is -inf, the entropy 0
  const float ln = l == 0 ? 0.0f : logf(l), lse = mu + ln;
  if (tid == 0) {
    if (p.logprob) {
      const int t = p.tokens[row];
      p.logprob[row] = t >= 0 && t < p.V ? widen(((const E*)p.x)[(long long)row * p.ld + t]) - lse : fv(kQNaN);
    }
    if (p.entropy) p.entropy[row] = l == 0 ? 0.0f : ln - e / l;
  }
  if (top == 0) return;
  // runs of keys, kLpCand - top new ones with the best so far
  if (tid < kLpMaxTop) best[tid] = 0;
  const unsigned long long* from = p.ws_key + (long long)row * parts * top;
  const long long total = (long long)parts * top;
  for (long long i0 = 0; i0 < total; i0 += kLpCand - kLpMaxTop) {
    const int n = (int)min((long long)(kLpCand - kLpMaxTop), total - i0);
    __syncthreads();
    for (int i = tid; i < n; i += kLpThreads) key[i] = from[i0 + i];
    if (tid < top) key[n + tid] = best[tid];
    __syncthreads();
    for (int i = tid; i < n + top; i += kLpThreads) {
      const unsigned long long k = key[i];
      int r = 0;
      for (int j = 0; j < n + top; ++j) r += key[j] > k;
      if (k != 0 && r < top) best[r] = k;
    }
  }
  __syncthreads();
  if (tid < top) {
    const unsigned long long k = best[tid];
    p.top_ids[(long long)row * top + tid] = (int32_t)(uint32_t)~(uint32_t)k;
    p.top_lp[(long long)row * top + tid] = key_value(k) - lse;
  }
}

}  // namespace t2r
