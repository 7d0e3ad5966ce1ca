// The block-scaled KV cache, the attention over it and the token log probabilities: the entry points of include/t2r.h.
// A unit of its own: its kernels' code lies apart from t2r.hip's.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>

#include "../../include/t2r.h"
#include "t2r_blkattn.h"
#include "t2r_block.h"
#include "t2r_logprob.h"

using namespace t2r;

namespace {

constexpr long long kMaxGroups = (1 << 24) - 1;      // workgroups of 256 along x: a launch's threads count in 32 bits there

inline int launched() { return hipGetLastError() == hipSuccess ? T2R_OK : T2R_EHIP; }
inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }
inline size_t elem_size(int dtype) { return dtype == T2R_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == T2R_F32 || dtype == T2R_BF16 || dtype == T2R_F16; }
inline bool misaligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) != 0; }

// f(an element of the type): one instantiation a type
template <class F>
int by_type(int dtype, F f) {
  switch (dtype) {
    case T2R_F32: return f(float());
    case T2R_BF16: return f(bf16_t());
    default: return f(_Float16());
  }
}

// the cache's sizes but for the pool's
bool cache_sizes_ok(int block, int Hk, int hd, int width) {
  if (block != 16 && block != 32 && block != 64 && block != 128) return false;
  return hd > 0 && hd <= 128 && hd % 16 == 0 && Hk > 0 && Hk <= 65535 && width > 0 && (long long)width * block <= INT32_MAX;
}
// the cache's description, checked; T2R_OK or a code
int cache_args(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, int n_blocks, int block, int Hk,
               int hd, const int32_t* table, int width, BlkCache* c) {
  if (!kc || !vc || !ks || !vs || !table) return T2R_EINVAL;
  if (misaligned(kc, 16) || misaligned(vc, 16) || misaligned(ks, 4) || misaligned(vs, 4) || misaligned(table, 4)) return T2R_EINVAL;
  if (!cache_sizes_ok(block, Hk, hd, width) || n_blocks <= 0 || (long long)n_blocks * Hk > INT32_MAX) return T2R_ESHAPE;
  c->kc = (int8_t*)kc; c->vc = (int8_t*)vc; c->ks = (float*)ks; c->vs = (float*)vs; c->table = table;
  c->n_blocks = n_blocks; c->Hk = Hk; c->hd = hd; c->lbs = __builtin_ctz((unsigned)block); c->width = width;
  return T2R_OK;
}

// (block, head) tiles that `rows` rows of B sequences enter at most: n rows enter up to 1 + ceil((n - 1) / block) blocks
long long blocks_entered(long long rows, long long B, int block) {
  const long long s = B < rows ? B : rows, x = rows - s;
  return s + (x < x / block + s ? x : x / block + s);
}

// units of 16 values that a thread of the append kernel has (1, 2 or 4): 128 x 128 values are the most
int units_of(int hd, int block) {
  const int n = hd * block;
  return n <= 16 * kBlkThreads ? 1 : n <= 32 * kBlkThreads ? 2 : 4;
}

// How the step form is cut: `chunk` keys a workgroup. The lengths are on the device: the table's width bounds them, and
// workgroups past a sequence's end return at once.
//  - A cache that one workgroup gets through in some 10 us stays whole, which saves the join's launch (3.3 us on the GPU, 3
//    on the host). One sequence of 32 heads of 64 in a 2048-token table: 96 / 700 / 2040 tokens 4.9 / 7.1 / 11.7 us (10.7 /
//    10.7 / 11.9 a call) whole, 8.7 / 9.1 / 9.2 (13.6 .. 13.8) in parts; at head dim 128 2040 tokens take 17 us whole.
//  - Otherwise some 2000 workgroups: fewer leave a ragged batch's longest sequences over at the end, more begin and end too
//    often. 32 sequences of 1021 .. 8192 tokens, 16 heads of 128: 66.6 us, 68.5 with half as many, 75 with twice; all of 8192:
//    98.8 us (5.4 TB/s), 96.7, 116.
struct Cut {
  int chunk, nsplit, tiles, cols;       // tiles and their columns: the ragged form
};
Cut step_cut(int B, int H, int Hk, int hd, int block, int width, int dtype) {
  const long long cap = (long long)width * block;
  const int heads = dtype == T2R_F32 ? 8 : 16, sets = (H / Hk + heads - 1) / heads;
  const long long units = (long long)B * Hk * sets;
  const bool whole = cap * (hd <= 64 ? 64 : 128) <= 2048 * 64;
  Cut c{256, 1, 0, 0};
  while (c.chunk < kBaSeg && c.chunk < cap && (whole || units * cdiv(cap, c.chunk) > 2048)) c.chunk *= 2;
  c.nsplit = (int)cdiv(cap, c.chunk);
  return c;
}
Cut rows_cut(int B, int rows, int H, int Hk, int hd, int block, int width) {
  const long long cap = (long long)width * block;
  const int G = H / Hk;
  Cut c;
  // Few rows: one tile of 32 columns a sequence. Else 64; 128, which a conversion of codes then serves, at head dims whose sums
  // leave a wave registers for two times 32, once 64 would be more than the chip has places for twice (1024). 32 heads of 64,
  // one prompt of 512 / 2032 / 4064 rows, us: fp32 13.2 / 51.1 / 162 in 64 columns and 22.6 / 51.8 / 153 in 128, bf16 12.3 /
  // 38.0 / 116 and 19.6 / 37.7 / 105, fp16 12.3 / 43.2 / 141 and 20.8 / 44.2 / 131. One rule for the whole call: a batch of a prompt
  // and single rows has the prompt's columns for all of them, a prompt among many idle sequences 32. 31 rows at 1000 .. 8192
  // positions and a prompt of 512 in bf16 take 95 us in one call, 32 and 16 in two (the rows by the step form); 2000 rows among
  // 256 slots 50, alone 38.
  c.cols = (long long)rows * G <= 32LL * B ? 32 : hd <= 64 && (long long)rows * H > 64 * 1024 ? 128 : 64;
  const int rt = c.cols / G;
  // every sequence's last tile may be a part of one
  const long long tiles = rows / rt + (B < rows ? B : rows);
  c.tiles = (int)tiles;
  c.chunk = (int)cap;
  c.nsplit = 1;
  // A part costs what a tile costs before and after its keys (7 us) and the join's launch (4 to 5 us); 64 keys of a tile take 1.3
  // us. So keys are cut only while workgroups leave half of the chip's places empty, and into parts of 512 at least: a
  // 1024-row prompt (256 workgroups) took 33 us in four parts and 26 whole, 8 rows at 8100 positions 16 in parts and 52 whole.
  // Few rows are one tile a sequence as a rule, three workgroups of which fit a CU: 8 rows of 16 sequences at 5000 .. 8100
  // positions, 32 heads of 64, took 52 / 41 / 35 / 38 / 48 us in parts of 4096 / 2048 / 1280 / 1024 / 512 keys; of 4
  // sequences 23 / 21 / 20 in parts of 2048 / 1024 / 512.
  // Turns of a few hundred rows late in long caches (tables past 2048 positions) gain from a second workgroup on every CU, in
  // parts of 1536 at least: 548 rows at 7127 positions, 32 heads of 64 in bf16 (280 workgroups), took 97 us whole and 79 / 77 /
  // 73 / 72 / 77 in parts of 4096 / 2688 / 2048 / 1536 / 1024; 1200 at 8000, 16 heads of 128 (304) in bf16, 151 and 143 / 128 / 128 /
  // 130 / 138; but 900 rows (456) 95 whole and 107 to 109 in parts. The lengths are on the device, so a first prompt of some hundred
  // rows in such a table pays for parts that it has not got: 512 rows 16.3 us, 12.4 whole (fp32 17.5 and 12.7).
  const bool few = c.cols == 32;
  const long long wgs = (few ? B : tiles) * Hk;
  const bool turns = !few && wgs > 128 && cap > 2048;
  const long long parts = few ? 768 : turns ? 1024 : 512, least = turns ? 1536 : 512;
  if (wgs <= (turns ? 432 : parts / 2)) {
    const long long want = parts / wgs, ch = cdiv(cdiv(cap, want), 128) * 128;
    c.chunk = (int)(ch < least ? least : ch);
    c.nsplit = (int)cdiv(cap, c.chunk);
  }
  return c;
}

// (the kernels take it times log2(e))
bool scale_ok(float scale) { return scale > 0 && scale * kLog2e <= 3.4028234663852886e38f; }
bool attn_shape_ok(int H, int Hk) { return Hk > 0 && H > 0 && H % Hk == 0 && H / Hk <= 32; }
// The two forms' sizes, of the calls and of the workspace query alike (the cuts are worked out for these only); the cut, or
// false where a launch cannot hold it
bool step_sizes(int B, int H, int Hk, int hd, int block, int width, int dtype, Cut* c) {
  if (!attn_shape_ok(H, Hk) || B <= 0 || B > 65535 || H > 65535) return false;
  *c = step_cut(B, H, Hk, hd, block, width, dtype);
  return c->nsplit <= 65535;
}
bool rows_sizes(int B, int rows, int H, int Hk, int hd, int block, int width, Cut* c) {
  if (!attn_shape_ok(H, Hk) || B <= 0 || rows <= 0 || rows >= kMaxRows) return false;
  *c = rows_cut(B, rows, H, Hk, hd, block, width);
  return c->nsplit <= 65535 && (long long)c->tiles * Hk <= kMaxGroups;
}
long long part_bytes(long long parts, int hd) { return parts * 4 * (hd + 4); }
long long step_ws(const Cut& c, int B, int H, int hd) { return c.nsplit > 1 ? part_bytes((long long)B * H * c.nsplit, hd) : 0; }
long long rows_ws(const Cut& c, int Hk, int hd) {
  return c.nsplit > 1 ? part_bytes((long long)c.tiles * Hk * c.cols * c.nsplit, hd) : 0;
}

// Parts of a logits row: as many as give the launch four workgroups a CU, each of whole spans
Cut lp_cut(int rows, int V) {             // chunk: spans a part takes; nsplit: parts
  const long long spans = cdiv(V + (V >= kLpSpan ? 7LL : 0), kLpSpan);      // (spans begin at 16 bytes, up to 7 values early)
  const long long want = cdiv(1024, rows) < kLpMaxParts ? cdiv(1024, rows) : kLpMaxParts;
  const long long per = cdiv(spans, want < spans ? want : spans);
  return Cut{(int)per, (int)cdiv(spans, per), 0, 0};
}
bool lp_sizes(int rows, int V, Cut* c) {
  if (rows <= 0 || V <= 0 || V > INT32_MAX - 2 * kLpSpan) return false;
  *c = lp_cut(rows, V);
  return (long long)rows * c->nsplit <= kMaxGroups;
}
long long lp_ws(const Cut& c, int rows, int top) { return c.nsplit > 1 ? (long long)rows * c.nsplit * (16 + 8LL * top) : 0; }

}  // namespace

extern "C" {

int t2r_kv_append_blk(const void* k, const void* v, int dtype, int64_t k_ld, int64_t v_ld, int8_t* kc, int8_t* vc, float* ks,
                      float* vs, int n_blocks, int block, int Hk, int hd, const int32_t* table, int width,
                      const int32_t* starts, const int32_t* lens, int B, int rows, void* stream) {
  if (!k || !v || !starts || !lens || !dtype_ok(dtype)) return T2R_EINVAL;
  if (misaligned(k, elem_size(dtype)) || misaligned(v, elem_size(dtype)) || misaligned(starts, 4) || misaligned(lens, 4)) return T2R_EINVAL;
  BlkCache c;
  if (int rc = cache_args(kc, vc, ks, vs, n_blocks, block, Hk, hd, table, width, &c)) return rc;
  if (B <= 0 || rows <= 0 || rows >= kMaxRows || k_ld < (int64_t)Hk * hd || v_ld < (int64_t)Hk * hd) return T2R_ESHAPE;
  const BlkRows x{k, v, k_ld, v_ld};
  const Ragged g{starts, lens, B, rows};
  const dim3 grid((unsigned)blocks_entered(rows, B, block), Hk, 2);
  return by_type(dtype, [&](auto e) {
    using E = decltype(e);
    const dim3 threads(kBlkThreads);
    const hipStream_t st = (hipStream_t)stream;
    switch (units_of(hd, block)) {
      case 1: launch((k_blk_append<E, 1>), grid, threads, 0, st, x, g, c); break;
      case 2: launch((k_blk_append<E, 2>), grid, threads, 0, st, x, g, c); break;
      default: launch((k_blk_append<E, 4>), grid, threads, 0, st, x, g, c); break;
    }
    return launched();
  });
}

int t2r_kv_read_blk(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, int n_blocks, int block, int Hk,
                    int hd, const int32_t* table, int width, const int32_t* starts, const int32_t* lens, int B, int rows,
                    int dtype, void* k, void* v, void* stream) {
  if (!k || !v || !starts || !lens || !dtype_ok(dtype)) return T2R_EINVAL;
  if (misaligned(k, elem_size(dtype)) || misaligned(v, elem_size(dtype)) || misaligned(starts, 4) || misaligned(lens, 4)) return T2R_EINVAL;
  BlkCache c;
  if (int rc = cache_args(kc, vc, ks, vs, n_blocks, block, Hk, hd, table, width, &c)) return rc;
  if (B <= 0 || rows <= 0 || rows >= kMaxRows) return T2R_ESHAPE;
  const Ragged g{starts, lens, B, rows};
  const dim3 grid((unsigned)blocks_entered(rows, B, block), Hk, 2);
  return by_type(dtype, [&](auto e) {
    using E = decltype(e);
    const dim3 threads(kBlkThreads);
    const hipStream_t st = (hipStream_t)stream;
    launch(k_blk_read<E>, grid, threads, 0, st, g, c, (E*)k, (E*)v);
    return launched();
  });
}

int64_t t2r_attn_blk_workspace_bytes(int B, int rows, int H, int Hk, int hd, int block, int width, int dtype) {
  if (!cache_sizes_ok(block, Hk, hd, width) || !dtype_ok(dtype)) return -1;
  Cut c;
  if (rows == 0) return step_sizes(B, H, Hk, hd, block, width, dtype, &c) ? step_ws(c, B, H, hd) : -1;
  return rows_sizes(B, rows, H, Hk, hd, block, width, &c) ? rows_ws(c, Hk, hd) : -1;
}

int t2r_attn_blk_decode(const void* q, int dtype, int64_t q_ld, const int8_t* kc, const int8_t* vc, const float* ks,
                        const float* vs, int n_blocks, int block, int Hk, int hd, const int32_t* table, int width,
                        const int32_t* lens, int B, int H, float scale, void* out, int64_t out_ld, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  if (!q || !out || !lens || !dtype_ok(dtype) || !scale_ok(scale)) return T2R_EINVAL;
  if (misaligned(q, elem_size(dtype)) || misaligned(out, elem_size(dtype)) || misaligned(lens, 4)) return T2R_EINVAL;
  BlkAttn p;
  std::memset(&p, 0, sizeof(p));
  if (int rc = cache_args(kc, vc, ks, vs, n_blocks, block, Hk, hd, table, width, &p.c)) return rc;
  Cut cut;
  if (!step_sizes(B, H, Hk, hd, block, width, dtype, &cut) || q_ld < (int64_t)H * hd || out_ld < (int64_t)H * hd) return T2R_ESHAPE;
  const long long need = step_ws(cut, B, H, hd);
  if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 16))) return T2R_ENOMEM;
  p.q = q; p.q_ld = q_ld; p.out = out; p.out_ld = out_ld;
  p.g = Ragged{nullptr, lens, B, B};
  p.H = H; p.G = H / Hk; p.a = scale * kLog2e;
  p.chunk = cut.chunk; p.nsplit = cut.nsplit;
  p.ws_o = (float*)workspace;
  p.ws_ml = p.ws_o + (long long)B * H * cut.nsplit * hd;
  const hipStream_t st = (hipStream_t)stream;
  return by_type(dtype, [&](auto e) {
    using E = decltype(e);
    const int heads = 16 / Pieces<E>::kQ, sets = (p.G + heads - 1) / heads;
    // later parts come last: those past their sequence's end, which return at once, then hold up nobody's place
    const dim3 grid(Hk * sets, B, cut.nsplit);
    if (hd <= 64) launch((k_blk_step<E, 64>), grid, dim3(kBaThreads), 0, st, p);
    else launch((k_blk_step<E, 128>), grid, dim3(kBaThreads), 0, st, p);
    if (cut.nsplit > 1) launch(k_blk_step_join<E>, dim3(H, B), dim3(kBaThreads), 0, st, p);
    return launched();
  });
}

int t2r_attn_blk_prefill(const void* q, int dtype, int64_t q_ld, const int8_t* kc, const int8_t* vc, const float* ks,
                         const float* vs, int n_blocks, int block, int Hk, int hd, const int32_t* table, int width,
                         const int32_t* starts, const int32_t* lens, int B, int rows, int H, float scale, void* out,
                         int64_t out_ld, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!q || !out || !starts || !lens || !dtype_ok(dtype) || !scale_ok(scale)) return T2R_EINVAL;
  if (misaligned(q, elem_size(dtype)) || misaligned(out, elem_size(dtype)) || misaligned(starts, 4) || misaligned(lens, 4)) return T2R_EINVAL;
  BlkAttn p;
  std::memset(&p, 0, sizeof(p));
  if (int rc = cache_args(kc, vc, ks, vs, n_blocks, block, Hk, hd, table, width, &p.c)) return rc;
  Cut cut;
  if (!rows_sizes(B, rows, H, Hk, hd, block, width, &cut) || q_ld < (int64_t)H * hd || out_ld < (int64_t)H * hd) return T2R_ESHAPE;
  const long long need = rows_ws(cut, Hk, hd);
  if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 16))) return T2R_ENOMEM;
  p.q = q; p.q_ld = q_ld; p.out = out; p.out_ld = out_ld;
  p.g = Ragged{starts, lens, B, rows};
  p.H = H; p.G = H / Hk; p.a = scale * kLog2e;
  p.chunk = cut.chunk; p.nsplit = cut.nsplit;
  p.order = (long long)cut.tiles * Hk <= 512 ? ORDER_BOTH : ORDER_BACKWARDS;
  p.ws_o = (float*)workspace;
  p.ws_ml = p.ws_o + (long long)cut.tiles * Hk * cut.cols * cut.nsplit * hd;
  const hipStream_t st = (hipStream_t)stream;
  return by_type(dtype, [&](auto e) {
    using E = decltype(e);
    const dim3 grid(cut.tiles * Hk, cut.nsplit), block(kBaThreads);
    if (cut.cols == 32) {
      if (hd <= 64) launch((k_blk_few<E, 64>), grid, block, 0, st, p);
      else launch((k_blk_few<E, 128>), grid, block, 0, st, p);
    } else if (cut.cols == 64) {
      if (hd <= 64) launch((k_blk_tile<E, 64, 1>), grid, block, 0, st, p);
      else launch((k_blk_tile<E, 128, 1>), grid, block, 0, st, p);
    } else {
      launch((k_blk_tile<E, 64, 2>), grid, block, 0, st, p);
    }
    if (cut.nsplit >= kJoinWide) launch((k_blk_rows_join<E, kBaWaves>), dim3(cut.tiles * Hk, cut.cols), block, 0, st, p, cut.cols);
    else if (cut.nsplit > 1) launch((k_blk_rows_join<E, 1>), dim3(cut.tiles * Hk, cut.cols / kBaWaves), block, 0, st, p, cut.cols);
    return launched();
  });
}

int64_t t2r_logprobs_workspace_bytes(int rows, int V, int top) {
  Cut cut;
  return top >= 0 && top <= kLpMaxTop && top <= V && lp_sizes(rows, V, &cut) ? lp_ws(cut, rows, top) : -1;
}

int t2r_logprobs(const void* logits, int dtype, int64_t ld, const int32_t* tokens, int rows, int V, int top,
                 float* logprob, float* entropy, int32_t* top_ids, float* top_logprob, void* workspace,
                 int64_t workspace_bytes, void* stream) {
  if (!logits || !dtype_ok(dtype) || (logprob && !tokens) || (top > 0 && (!top_ids || !top_logprob))) return T2R_EINVAL;
  if (misaligned(logits, elem_size(dtype)) || misaligned(tokens, 4) || misaligned(logprob, 4) || misaligned(entropy, 4) ||
      misaligned(top_ids, 4) || misaligned(top_logprob, 4))
    return T2R_EINVAL;
  Cut cut;
  if (!lp_sizes(rows, V, &cut) || ld < V) return T2R_ESHAPE;
  if (top < 0 || top > kLpMaxTop || top > V) return T2R_ERANGE;
  const long long need = lp_ws(cut, rows, top);
  if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 16))) return T2R_ENOMEM;
  LpArgs p;
  std::memset(&p, 0, sizeof(p));
  p.x = logits; p.ld = ld; p.tokens = tokens; p.rows = rows; p.V = V; p.top = top;
  p.spans = cut.chunk; p.parts = cut.nsplit;
  p.logprob = logprob; p.entropy = entropy; p.top_ids = top_ids; p.top_lp = top_logprob;
  p.ws_sum = (float*)workspace;
  p.ws_key = (unsigned long long*)(p.ws_sum + 4LL * rows * cut.nsplit);
  const hipStream_t st = (hipStream_t)stream;
  return by_type(dtype, [&](auto e) {
    using E = decltype(e);
    launch(k_lp_part<E>, dim3(rows * cut.nsplit), dim3(kLpThreads), 0, st, p);
    if (cut.nsplit > 1) launch(k_lp_join<E>, dim3(rows), dim3(kLpThreads), 0, st, p);
    return launched();
  });
}

}  // extern "C"
