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
// as many short ones.  On the line an item is kItemCost chunks longer than it
// is: what its queries and outputs cost.  (48 ragged requests, 1 to 1500 keys:
// without it the slowest CTA took 2.1 times the median.)  An item inside one
// range is written directly; the pieces of a cut item go to the segments of
// their CTAs (a range cuts at most its first and its last item: segment 0 of a
// CTA is for an item that began before its range, segment 1 for one that goes on
// behind it).
//
// Order.  Tiles of one KV head should read its K and V at about the same time,
// from L2.  Where an item is cut over CTAs, or has one, neighbours on the line
// are neighbouring tiles.  Where a CTA has `step` > 1 items of a group, items
// `step` apart on the line are: the group's items (numbered head by head, tile
// by tile) are written into a matrix of `step` columns column by column, and the
// line reads its rows, so that neighbouring CTAs work on neighbouring tiles at
// the same time.  16 requests of up to 1024 tokens x 6500 keys: 835 us -> 812 us.
// For sequences of fewer than 16 chunks, which L2 holds anyway, the arithmetic
// costs more than it gives (48 ragged requests: 106 -> 111 us).
#pragma once

#include "common.cuh"
#include "gqa_kernel.cuh"

namespace b2d {

constexpr int kItemCost = 3;   // positions of an item on the line before its first chunk

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
  const float* own_o;           // shared prefix: the part over each sequence's own tokens, [T, Hq, D]
  const float* own_lse;         // fp32 and [T, Hq] natural log, to be joined with; else null
  int beside;                   // 1: start while the kernel that writes the own parts still runs
  float* seg_o;                 // [2 * CTAs][tile rows][D] fp32, normalised
  float* seg_lse;               // [2 * CTAs][tile rows], log2 units
  int32_t* cuts;                // [CTAs][8]: the item that each CTA begins and does not finish
  int* status;
  unsigned long long wait_ns;
  int no_loads;
  int G, T, uniform, Hq, Hkv, grp, P, num_pages, max_pages;
  int TS, CH, rows;             // tokens of a tile, keys of a chunk, rows of a segment
  int pairs;                    // 1: items of two tiles
  int spread;                   // 1: there are at least two items per CTA
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

// The groups in shared memory: table[g] = line positions of all items before
// group g, [G + 1]; 32 ints of scratch; and, for up to kCachedGroups groups,
// first token, tokens and keys of each, so that finding a piece waits for no
// global load.
constexpr int kCachedGroups = 1024;
__host__ __device__ constexpr size_t ragged_table_bytes(int groups) {
  return ((size_t)groups + 1 + 32 + (groups <= kCachedGroups ? 3 * (size_t)groups : 0)) * 4;
}

// Set when the starts descend somewhere.  Tokens would then belong to several
// groups, whose rows race, and the work line could pass 32 bits (the host's
// bound counts every token once): the table is one of no work, and no row is
// written.  It lies in the last int of the scratch, of which a block's warps use
// at most 16.  (As a variable that lives across the kernel it cost 2 % on long
// calls: 838 -> 857 us for 16 requests of up to 1024 x 6500 tokens.)
__device__ __forceinline__ int32_t& ragged_descends(const RaggedParams& p, int32_t* table) {
  return table[p.G + 32];
}

// Fills the table (block-wide scan; ends with __syncthreads).
__device__ __forceinline__ void ragged_table(const RaggedParams& p, int32_t* table) {
  int32_t* warp_tmp = table + p.G + 1;
  int32_t* cache = p.G <= kCachedGroups ? warp_tmp + 32 : nullptr;
  const int tid = threadIdx.x, nth = blockDim.x;
  const int lane = tid & 31, warp = tid >> 5, nwarps = nth >> 5;
  if (tid == 0) ragged_descends(p, table) = 0;
  __syncthreads();
  int carry = 0;
  for (int base = 0; base < p.G; base += nth) {
    const int g = base + tid;
    int n = 0;
    if (g < p.G) {
      if (p.starts != nullptr && __ldg(p.starts + g + 1) < __ldg(p.starts + g)) ragged_descends(p, table) = 1;
      const int2 tok = ragged_tokens(p, g);
      const int len = ragged_kv_len(p, g), nch = (len + p.CH - 1) / p.CH;
      n = nch > 0 ? ragged_items(p, tok.y) * (nch + kItemCost) : 0;
      if (cache != nullptr) {
        cache[g] = tok.x;
        cache[p.G + g] = tok.y;
        cache[2 * p.G + g] = len;
      }
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
  if (tid == 0) {
    const bool descends = ragged_descends(p, table) != 0;
    table[p.G] = descends ? 0 : carry;
    if (descends && blockIdx.x == 0) record_status(p.status, kStatusBounds);
  }
  __syncthreads();
}

// A piece of an item, inside one range: chunks [c0, c1) of nch.  Part s (0 or
// 1) of the item is the tile of TS tokens from tile + (tiles == 2 ? s : 0) on,
// of KV head h + (heads == 2 ? s : 0); it exists for s < tiles * heads.
struct RaggedPiece {
  int g, h, tile, tiles, heads, t0, n, len, c0, c1, nch;   // group's tokens: [t0, t0 + n)
  int last;                                                // line position of the item's last chunk
  __device__ __forceinline__ int parts() const { return tiles * heads; }
  __device__ __forceinline__ int head(int s) const { return h + (heads == 2 ? s : 0); }
  __device__ __forceinline__ int first(int s, int TS) const { return (tile + (tiles == 2 ? s : 0)) * TS; }
  __device__ __forceinline__ bool whole() const { return c0 == 0 && c1 == nch; }
  __device__ __forceinline__ int segment(int cta) const { return 2 * cta + (c0 == 0 ? 1 : 0); }
};

// The next piece with a chunk in line positions [x, x1); moves x behind it and
// g to its group.  False: none is left.
__device__ __forceinline__ bool ragged_next(const RaggedParams& p, const int32_t* table, int x1,
                                            int& g, int& x, RaggedPiece& w) {
  while (x < x1) {
    while (x >= table[g + 1]) ++g;
    w.g = g;
    if (p.G <= kCachedGroups) {
      const int32_t* cache = table + p.G + 1 + 32 + g;
      w.t0 = cache[0];
      w.n = cache[p.G];
      w.len = cache[2 * p.G];
    } else {
      const int2 tok = ragged_tokens(p, g);
      w.t0 = tok.x;
      w.n = tok.y;
      w.len = ragged_kv_len(p, g);
    }
    w.nch = (w.len + p.CH - 1) / p.CH;
    const int tiles = (w.n + p.TS - 1) / p.TS;
    const int rel = x - table[g], size = w.nch + kItemCost;
    int it = rel / size;
    const int pos = rel - it * size, end = min(size, pos + (x1 - x));
    w.c0 = max(0, pos - kItemCost);
    w.c1 = max(0, end - kItemCost);
    w.last = x - pos + size - 1;
    x += end - pos;
    if (p.spread && w.nch >= 16) {   // (see "Order" above)
      const int step = (table[p.G] / (int)gridDim.x + (size >> 1)) / size, items = ragged_items(p, w.n);
      if (step > 1 && step < items) {
        const int a = it / step, b = it - a * step, runs = (items + step - 1) / step;
        const int full = items - (runs - 1) * step;
        it = b < full ? b * runs + a : full * runs + (b - full) * (runs - 1) + a;
      }
    }
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
    if (w.c1 > w.c0) return true;
  }
  return false;
}

__device__ __forceinline__ int range_begin(int64_t W, int ctas, int c) {
  return (int)((int64_t)c * W / ctas);
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

template <typename QT>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (std::is_same<QT, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <int EPL, typename QT>
__device__ __forceinline__ void store_lane(QT* dst, const float* v, float s) {
#pragma unroll
  for (int e = 0; e < EPL; e += 2) {   // EPL is even: 4-byte stores
    const uint32_t w = pack_pair<QT>(v[e] * s, v[e + 1] * s);
    *reinterpret_cast<uint32_t*>(dst + e) = w;
  }
}

template <int EPL>
__device__ __forceinline__ void load_lane(const float* src, float* v) {
#pragma unroll
  for (int e = 0; e < EPL; e += 2) {
    const float2 f = *reinterpret_cast<const float2*>(src + e);
    v[e] = f.x;
    v[e + 1] = f.y;
  }
}

// Weights of a normalised part (log2 sum a2) and the own part (natural log
// sum) in their join, and the join's log2 sum.  A part without mass gets 0.
__device__ __forceinline__ float2 join_weights(float a2, float own, float& lse2) {
  const float b2 = own * 1.4426950408889634f, mx = fmaxf(a2, b2);
  if (mx == -INFINITY) {   // no mass, or NaN beside none (fmaxf leaves a NaN out)
    lse2 = a2 + b2;
    return make_float2(lse2 == -INFINITY ? 1.f : lse2, 0.f);
  }
  const float wa = fast_exp2(a2 - mx), wb = fast_exp2(b2 - mx), inv = 1.f / (wa + wb);
  lse2 = mx + fast_log2(wa + wb);
  return make_float2(wa * inv, wb * inv);
}

// A row without keys of its group: its own part alone, or out = 0, lse = -inf.
// One warp.
template <int D, typename QT>
__device__ __forceinline__ void ragged_row_without_keys(const RaggedParams& p, int t, int h) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994530942f;
  constexpr int EPL = D / 32;
  const int lane = threadIdx.x & 31;
  StateMerge<EPL> m;
  if (p.own_o != nullptr) {
    griddep_wait();
    const int64_t row = (int64_t)t * p.Hq + h;
    float o[EPL];
    load_lane<EPL>(p.own_o + row * D + lane * EPL, o);
    m.add(o, p.own_lse[row] * kLog2e);
  }
  store_lane<EPL>(reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + lane * EPL,
                  m.acc, m.inv());
  if (p.lse != nullptr && lane == 0) p.lse[(int64_t)t * p.lse_st + h] = m.lse2() * kLn2;
}

// All rows of groups without keys, and (shared prefix) of tokens outside every
// group, spread over the blocks and their warps.
template <int D, typename QT>
__device__ __forceinline__ void ragged_rows_without_keys(const RaggedParams& p, int32_t* table) {
  if (ragged_descends(p, table) != 0) return;
  const int warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  auto rows = [&](int t0, int n, int first, int step) {
    for (int64_t i = first; i < (int64_t)n * p.Hq; i += step)
      ragged_row_without_keys<D, QT>(p, t0 + (int)(i / p.Hq), (int)(i % p.Hq));
  };
  for (int g = blockIdx.x; g < p.G; g += gridDim.x)
    if (ragged_kv_len(p, g) == 0) {
      const int2 tok = ragged_tokens(p, g);
      rows(tok.x, tok.y, warp, nwarps);
    }
  if (p.own_o != nullptr && p.starts != nullptr) {
    const int first = blockIdx.x * nwarps + warp, step = gridDim.x * nwarps;
    rows(0, ragged_tokens(p, 0).x, first, step);
    const int2 tok = ragged_tokens(p, p.G - 1);
    rows(tok.x + tok.y, p.T - tok.x - tok.y, first, step);
  }
}

// What CTA c leaves for the merge: nothing, or the item that it begins and
// does not finish.
__device__ __forceinline__ void ragged_note_cut(const RaggedParams& p, int c, const RaggedPiece* w,
                                                int64_t W, int ctas) {
  int v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (w != nullptr) {
    v[0] = cta_of_chunk(w->last, W, ctas) - c + 1;
    for (int s = 0; s < w->parts(); ++s) {
      v[2 + 3 * s] = w->t0 + w->first(s, p.TS);
      v[3 + 3 * s] = min(p.TS, w->n - w->first(s, p.TS));
      v[4 + 3 * s] = w->head(s);
    }
  }
  for (int i = 0; i < 8; ++i) p.cuts[8 * c + i] = v[i];
}

// Joins the segments of every cut item (and its rows' own parts) into out and
// lse.  Block x takes the item that CTA x begins; one warp per row.  The
// weights of up to 32 segments are computed side by side by the lanes; then
// the segments' values are loaded U at a time.
template <int D, typename QT>
__global__ void __launch_bounds__(256) ragged_merge_kernel(const RaggedParams p) {
  constexpr float kLn2 = 0.69314718055994530942f;
  constexpr float kLog2e = 1.4426950408889634f;
  constexpr int EPL = D / 32, U = 8;
  griddep_wait();
  const int c = blockIdx.x, lane = threadIdx.x & 31;
  const int4 a = *reinterpret_cast<const int4*>(p.cuts + 8 * c);
  if (a.x == 0) return;
  const int4 b = *reinterpret_cast<const int4*>(p.cuts + 8 * c + 4);
  const int per = p.TS * p.grp;   // rows of a part
  for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < 2 * per; r += gridDim.y * 8) {
    const int s = r >= per ? 1 : 0, rr = r - s * per, i = rr / p.grp;
    if (i >= (s ? b.z : a.w)) continue;
    const int t = (s ? b.y : a.z) + i, h = (s ? b.w : b.x) * p.grp + rr - i * p.grp;
    auto seg_at = [&](int j) { return (int64_t)(2 * (c + j) + (j == 0 ? 1 : 0)) * p.rows + r; };
    float acc[EPL], mx = -INFINITY, sum = 0.f, own[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = own[e] = 0.f;
    if (p.own_o != nullptr) {
      const int64_t row = (int64_t)t * p.Hq + h;
      load_lane<EPL>(p.own_o + row * D + lane * EPL, own);
      mx = p.own_lse[row] * kLog2e;
      sum = mx == -INFINITY ? 0.f : 1.f;
      if (sum != 0.f) {
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = own[e];
      }
    }
    for (int j0 = 0; j0 < a.x; j0 += 32) {
      const float l = j0 + lane < a.x ? p.seg_lse[seg_at(j0 + lane)] : -INFINITY;
      float nm = l;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, o));
      nm = fmaxf(nm, mx);
      const float w = l == -INFINITY ? 0.f : fast_exp2(l - nm);
      const float old = mx == -INFINITY ? 0.f : fast_exp2(mx - nm);
      sum *= old;
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] *= old;
      mx = nm;
      const int n = min(32, a.x - j0);
      for (int j = 0; j < n; j += U) {
        float v[U][EPL];
#pragma unroll
        for (int u = 0; u < U; ++u)
          load_lane<EPL>(p.seg_o + seg_at(j0 + min(j + u, n - 1)) * D + lane * EPL, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float wj = __shfl_sync(0xffffffffu, w, (j + u) & 31);
          if (j + u >= n || wj == 0.f) continue;   // (a segment without mass may hold anything)
          sum += wj;
#pragma unroll
          for (int e = 0; e < EPL; ++e) acc[e] += wj * v[u][e];
        }
      }
    }
    store_lane<EPL>(reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh +
                        lane * EPL, acc, sum == 0.f ? 0.f : 1.f / sum);
    if (p.lse != nullptr && lane == 0) p.lse[(int64_t)t * p.lse_st + h] = (mx + fast_log2(sum)) * kLn2;
  }
}

}  // namespace b2d
