// ragged.cuh — attention of ragged groups of query tokens to one paged key
// sequence per group: what the two ragged kernels and their merge share.
//
// Math, for query row (token t of group g, query head h, KV head h / grp):
//   s_j = scale * <q_th, K[g, j]>, j < kv_len[g],  m = max_j s_j,
//   out = sum_j e^(s_j - m) V[g, j] / l,  l = sum_j e^(s_j - m),
//   lse = m + ln l   (no causal mask: every query token sees every key).
// Cross attention is this with one group per request.  Decode over a shared
// prefix is this with the sequences of a group as its tokens, merged with
// each sequence's own tokens.
//
// Packing.  All grp query heads of a KV head read the same K and V, so a
// tile's rows are (token, head of the KV head) pairs: row r is token r / grp,
// head h * grp + r % grp.  A tile takes TS whole tokens, TS * grp <= its rows.
//
// Work split.  An item is one tile of one KV head of a group, or two that run
// side by side (pairs = 1, the tcgen05 kernel): two neighbouring tiles of a
// KV head, which share its K and V, and, for the odd last tile, the same
// tile of two neighbouring KV heads.  An item has ceil(kv_len / CH) chunks of
// CH keys.  The chunks of all items form one line, cut into equal ranges, one
// per CTA (as the decode kernel does), so few long items fill the GPU as well
// as many short ones.  Within a group the tiles of one KV head are neighbours
// on the line, so they read its K and V at about the same time, from L2.  An
// item inside one range is written directly; the pieces of a cut item go to
// the segments of their CTAs (a range cuts at most its first and its last
// item: two segments per CTA).
#pragma once

#include "common.cuh"
#include "gqa_kernel.cuh"

namespace b2d {

struct RaggedParams {
  const void* q;
  int64_t q_st, q_sh;           // token and head stride, elements
  const void* kc;
  const void* vc;
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  int64_t k_sg;                 // between 8-element groups of a K row (8, or P * 8 for vLLM)
  int64_t v_sd;                 // between the dims of a V row (1, or P for vLLM)
  const int32_t* starts;        // [G + 1] first token of each group, or null: uniform
  const int32_t* kv_lens;       // [G]
  const int32_t* block_table;
  int64_t bt_stride;
  const float* k_scale;
  const float* v_scale;
  void* out;                    // 16-bit output
  int64_t o_st, o_sh;
  float* lse;                   // natural log; may be null
  int64_t lse_st;
  float* out_f32;               // shared prefix: uncut items go here, [T, Hq, D] fp32, with
                                // lse2 [T, Hq] in log2 units; null: they go to out and lse
  float* lse2;
  float* seg_o;                 // [2 * CTAs][tile rows][D] fp32, normalised
  float* seg_lse;               // [2 * CTAs][tile rows], log2 units
  int32_t* table_g;             // [G + 1], written by CTA 0 for the merge
  int* status;
  unsigned long long wait_ns;
  int no_loads;
  int G, T, uniform, Hq, Hkv, grp, P, num_pages, max_pages;
  int TS, CH, rows;             // tokens of a tile, keys of a chunk, rows of a segment
  int pairs;                    // 1: items of two tiles
  float scale;                  // softmax_scale * log2(e)
};

// First token and token count of group g (clamped into [0, T]).
__device__ __forceinline__ int2 ragged_tokens(const RaggedParams& p, int g) {
  if (p.starts == nullptr) {
    const int64_t a = (int64_t)g * p.uniform;
    const int t0 = a < p.T ? (int)a : p.T;
    const int n = p.T - t0;
    return make_int2(t0, n < p.uniform ? n : p.uniform);
  }
  int a = __ldg(p.starts + g), b = __ldg(p.starts + g + 1);
  a = a < 0 ? 0 : (a > p.T ? p.T : a);
  b = b < a ? a : (b > p.T ? p.T : b);
  return make_int2(a, b - a);
}

__device__ __forceinline__ int ragged_kv_len(const RaggedParams& p, int g) {
  const int cap = p.max_pages * p.P;
  const int n = __ldg(p.kv_lens + g);
  return n < 0 ? 0 : (n > cap ? cap : n);
}

// Items of a group with n tokens.
__device__ __forceinline__ int ragged_items(const RaggedParams& p, int n) {
  const int tiles = (n + p.TS - 1) / p.TS;
  return p.pairs ? p.Hkv * (tiles >> 1) + (tiles & 1) * ((p.Hkv + 1) >> 1) : p.Hkv * tiles;
}

// table[g] = chunks of all items before group g (block-wide scan; ends with
// __syncthreads).  warp_tmp: 32 ints.
__device__ __forceinline__ void ragged_table(const RaggedParams& p, int32_t* table,
                                             int32_t* warp_tmp) {
  const int tid = threadIdx.x, nth = blockDim.x;
  const int lane = tid & 31, warp = tid >> 5, nwarps = nth >> 5;
  int carry = 0;
  for (int base = 0; base < p.G; base += nth) {
    const int g = base + tid;
    int n = 0;
    if (g < p.G) {
      n = ragged_items(p, ragged_tokens(p, g).y) * ((ragged_kv_len(p, g) + p.CH - 1) / p.CH);
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_tmp[warp] = x;
    __syncthreads();
    if (warp == 0) {
      int w = lane < nwarps ? warp_tmp[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      if (lane < nwarps) warp_tmp[lane] = w;
    }
    __syncthreads();
    if (g < p.G) table[g] = carry + (warp > 0 ? warp_tmp[warp - 1] : 0) + x - n;
    const int total = warp_tmp[nwarps - 1];
    __syncthreads();
    carry += total;
  }
  if (tid == 0) table[p.G] = carry;
  __syncthreads();
}

// The piece of an item that starts at line position x, inside a range that
// ends at x1: chunks [c0, c1) of nch.  Part s (0 or 1) of the item is the
// tile of TS tokens from tile + (tiles == 2 ? s : 0) on, of KV head h +
// (heads == 2 ? s : 0); it exists for s < tiles * heads.
struct RaggedPiece {
  int g, h, tile, tiles, heads, t0, n, len, c0, c1, nch;   // group's tokens: [t0, t0 + n)
  __device__ __forceinline__ int parts() const { return tiles * heads; }
  __device__ __forceinline__ int head(int s) const { return h + (heads == 2 ? s : 0); }
  __device__ __forceinline__ int first(int s, int TS) const { return (tile + (tiles == 2 ? s : 0)) * TS; }
};

__device__ __forceinline__ RaggedPiece ragged_piece(const RaggedParams& p, const int32_t* table,
                                                    int g, int x, int x1) {
  RaggedPiece w;
  w.g = g;
  const int2 tok = ragged_tokens(p, g);
  w.t0 = tok.x;
  w.n = tok.y;
  w.len = ragged_kv_len(p, g);
  w.nch = (w.len + p.CH - 1) / p.CH;
  const int tiles = (tok.y + p.TS - 1) / p.TS;
  const int rel = x - table[g];
  const int it = rel / w.nch;
  w.c0 = rel - it * w.nch;
  w.c1 = min(w.nch, w.c0 + (x1 - x));
  const int per = p.pairs ? tiles >> 1 : tiles;   // items of a KV head
  w.tiles = p.pairs ? 2 : 1;
  w.heads = 1;
  if (it < p.Hkv * per) {
    w.h = it / per;
    w.tile = (it - w.h * per) * w.tiles;
  } else {
    w.h = 2 * (it - p.Hkv * per);
    w.tile = tiles - 1;
    w.tiles = 1;
    w.heads = min(2, p.Hkv - w.h);
  }
  return w;
}

// Where token i of a group of n and query head h are: item and row of its
// segments.
__device__ __forceinline__ int2 ragged_row(const RaggedParams& p, int n, int i, int h) {
  const int tiles = (n + p.TS - 1) / p.TS, tile = i / p.TS, kvh = h / p.grp;
  const int r = (i - tile * p.TS) * p.grp + (h - kvh * p.grp);
  if (!p.pairs) return make_int2(kvh * tiles + tile, r);
  const int per = tiles >> 1;
  if (tile < 2 * per) return make_int2(kvh * per + (tile >> 1), (tile & 1) * p.TS * p.grp + r);
  return make_int2(p.Hkv * per + (kvh >> 1), (kvh & 1) * p.TS * p.grp + r);
}

__device__ __forceinline__ int range_begin(int64_t W, int ctas, int c) {
  return (int)((int64_t)c * W / ctas);
}

// Query rows of groups without keys: out = 0, lse = -inf.
template <int D, typename QT>
__device__ __forceinline__ void ragged_zero_rows(const RaggedParams& p) {
  for (int g = blockIdx.x; g < p.G; g += gridDim.x) {
    if (ragged_kv_len(p, g) > 0) continue;
    const int2 tok = ragged_tokens(p, g);
    const int64_t n = (int64_t)tok.y * p.Hq;
    for (int64_t i = threadIdx.x; i < n * (D / 8); i += blockDim.x) {
      const int64_t row = i / (D / 8);
      const int c = (int)(i - row * (D / 8)) * 8;
      const int t = tok.x + (int)(row / p.Hq), h = (int)(row % p.Hq);
      if (p.out_f32 == nullptr) {
        *reinterpret_cast<uint4*>(reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st +
                                  (int64_t)h * p.o_sh + c) = make_uint4(0, 0, 0, 0);
        if (p.lse != nullptr && c == 0) p.lse[(int64_t)t * p.lse_st + h] = -INFINITY;
      } else if (c == 0) {
        p.lse2[(int64_t)t * p.Hq + h] = -INFINITY;  // its out_f32 row is never read
      }
    }
  }
}

// Running merge of normalised partial outputs: (o, lse in log2 units), EPL
// elements per lane.  Parts with lse = -inf are not read.
template <int EPL>
struct StateMerge {
  float acc[EPL], mx, sum;
  __device__ __forceinline__ StateMerge() : mx(-INFINITY), sum(0.f) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
  }
  __device__ __forceinline__ void add(const float* o, float l2) {
    if (l2 == -INFINITY) return;
    const float nm = fmaxf(mx, l2);
    const float r = mx == -INFINITY ? 0.f : fast_exp2(mx - nm), w = fast_exp2(l2 - nm);
    sum = sum * r + w;
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = acc[e] * r + w * o[e];
    mx = nm;
  }
  __device__ __forceinline__ float inv() const { return sum > 0.f ? 1.f / sum : 0.f; }
  __device__ __forceinline__ float lse2() const { return mx + fast_log2(sum); }  // -inf when empty
};

template <int EPL, typename QT>
__device__ __forceinline__ void store_lane(QT* dst, const float* v, float s) {
#pragma unroll
  for (int e = 0; e < EPL; ++e) dst[e] = QT(v[e] * s);
}

template <int EPL>
__device__ __forceinline__ void load_lane(const float* src, float* v) {
#pragma unroll
  for (int e = 0; e < EPL; ++e) v[e] = src[e];
}

// Adds the segments of row r of the item at line positions [xs, xe) to m.
template <int D>
__device__ __forceinline__ void merge_segments(const RaggedParams& p, int64_t W, int ctas, int xs,
                                               int xe, int r, StateMerge<D / 32>& m) {
  constexpr int EPL = D / 32;
  const int lane = threadIdx.x & 31;
  const int cf = cta_of_chunk(xs, W, ctas), cl = cta_of_chunk(xe - 1, W, ctas);
  for (int c = cf; c <= cl; ++c) {
    const int slot = (c == cf && xs > range_begin(W, ctas, c)) ? 1 : 0;
    const int64_t at = (int64_t)(2 * c + slot) * p.rows + r;
    float o[EPL];
    load_lane<EPL>(p.seg_o + at * D + lane * EPL, o);
    m.add(o, p.seg_lse[at]);
  }
}

// Cross attention: writes the rows of items that a range boundary cut.  Block
// x looks at the boundary behind CTA x; the CTA in which the item starts
// owns it.  One warp per row.
template <int D, typename QT>
__global__ void __launch_bounds__(256) ragged_merge_kernel(const RaggedParams p, int ctas) {
  constexpr float kLn2 = 0.69314718055994530942f;
  constexpr int EPL = D / 32;
  const int W = p.table_g[p.G];
  if (W < ctas) ctas = W;
  const int c = blockIdx.x;
  if (c + 1 >= ctas) return;
  const int b = range_begin(W, ctas, c + 1);
  const int g = find_row(p.table_g, p.G, b);
  const RaggedPiece w = ragged_piece(p, p.table_g, g, b, b + 1);
  const int xs = b - w.c0;
  if (w.c0 == 0 || xs < range_begin(W, ctas, c)) return;  // not cut here, or owned by an earlier CTA
  const int lane = threadIdx.x & 31;
  const int per = p.TS * p.grp;   // rows of a part
  for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < w.parts() * per; r += gridDim.y * 8) {
    const int s = r / per, i = w.first(s, p.TS) + (r - s * per) / p.grp;
    if (i >= w.n) continue;
    StateMerge<EPL> m;
    merge_segments<D>(p, W, ctas, xs, xs + w.nch, r, m);
    const int t = w.t0 + i, h = w.head(s) * p.grp + r % p.grp;
    store_lane<EPL>(reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh +
                        lane * EPL, m.acc, m.inv());
    if (p.lse != nullptr && lane == 0) p.lse[(int64_t)t * p.lse_st + h] = m.lse2() * kLn2;
  }
}

// Shared prefix: joins each sequence's prefix part (direct or in segments)
// with its own tokens' part (own_o [T, Hq, D] fp32, own_lse [T, Hq] natural
// log).  One warp per (sequence, query head).
template <int D, typename QT>
__global__ void __launch_bounds__(256) shared_join_kernel(const RaggedParams p, int ctas,
                                                          const float* own_o,
                                                          const float* own_lse) {
  constexpr float kLn2 = 0.69314718055994530942f;
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int EPL = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)p.T * p.Hq) return;
  const int t = (int)(row / p.Hq), h = (int)(row - (int64_t)t * p.Hq);
  StateMerge<EPL> m;
  // The group that holds sequence t, if any: the last one that starts at or
  // before t (empty groups that start there too come before it).
  int lo = 0, hi = p.G - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ragged_tokens(p, mid).x <= t) lo = mid; else hi = mid - 1;
  }
  const int2 tok = ragged_tokens(p, lo);
  const int len = ragged_kv_len(p, lo);
  if (t >= tok.x && t < tok.x + tok.y && len > 0) {
    const int W = p.table_g[p.G];
    if (W < ctas) ctas = W;
    const int nch = (len + p.CH - 1) / p.CH;
    const int2 at = ragged_row(p, tok.y, t - tok.x, h);
    const int xs = p.table_g[lo] + at.x * nch;
    if (cta_of_chunk(xs, W, ctas) == cta_of_chunk(xs + nch - 1, W, ctas)) {
      float o[EPL];
      load_lane<EPL>(p.out_f32 + row * D + lane * EPL, o);
      m.add(o, p.lse2[row]);
    } else {
      merge_segments<D>(p, W, ctas, xs, xs + nch, at.y, m);
    }
  }
  float o[EPL];
  load_lane<EPL>(own_o + row * D + lane * EPL, o);
  m.add(o, own_lse[row] * kLog2e);
  store_lane<EPL>(reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh +
                      lane * EPL, m.acc, m.inv());
  if (p.lse != nullptr && lane == 0)
    p.lse[(int64_t)t * p.lse_st + h] = m.lse2() * kLn2;
}

}  // namespace b2d
