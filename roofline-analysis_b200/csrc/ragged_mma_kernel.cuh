// ragged_mma_kernel.cuh — ragged attention (ragged.cuh) on warp-level
// tensor-core tiles: the kernel for every cache that the tcgen05 kernel does
// not take (page sizes that are not multiples of 16, head_dim 192 and 256,
// vLLM's layout).
//
// A block of 4 warps takes 64 query rows; warp w owns rows 16w .. 16w + 15.
// Per chunk of CH keys: S = Q.K^T (m16n8k16, fp32), the running maximum and
// sum of the softmax in registers (4 lanes per row), O += P.V with P straight
// from the score registers (the C layout of the first product is the A
// layout of the second).  K and V come in with plain 16-byte loads through
// the block table, one token at a time, so a page may end anywhere; e4m3 is
// converted to fp16 (exact) on the way.  Keys past the end are zero-filled
// and masked.  Weights in fp16 are 2^15 as large as they are, so that small ones
// keep their bits (ragged_tc_kernel.cuh).  Rows in shared memory are padded by
// 16 bytes, so the 8 row addresses of an ldmatrix fall into different banks.
//
// Bound by the loads, which nothing overlaps: 16 requests of 64 - 256 x 500 -
// 2000 tokens, 32 query heads on 8, head_dim 128, pages of 8: 766 us, 69
// TFLOP/s; vLLM's layout, whose V is read 2 bytes at a time, 1148 us.
#pragma once

#include "gqa_mma_kernel.cuh"
#include "ragged.cuh"

namespace b2d {

// 8 consecutive cache elements as four packed 16-bit pairs (e4m3 -> fp16).
template <int KIND>
__device__ __forceinline__ uint4 load_cache8(const void* base, int64_t at, int64_t stride) {
  if constexpr (KIND == kKvFp8) {
    const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + at);
    return make_uint4(e4m3x2_to_f16x2_cvt(w.x), e4m3x2_to_f16x2_cvt(w.x >> 16),
                      e4m3x2_to_f16x2_cvt(w.y), e4m3x2_to_f16x2_cvt(w.y >> 16));
  } else {
    const uint16_t* src = static_cast<const uint16_t*>(base) + at;
    if (stride == 1) return *reinterpret_cast<const uint4*>(src);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = (uint32_t)src[2 * i * stride] | ((uint32_t)src[(2 * i + 1) * stride] << 16);
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
}

template <int D>
struct RaggedMma {
  static constexpr int kRows = 64, kThreads = 128;
  static constexpr int kCH = D <= 128 ? 64 : 32;   // keys per chunk
  static constexpr int kLd = D + 8;                // padded row, elements
};

template <int D, int KIND, typename QT>
__global__ void __launch_bounds__(128) ragged_mma_kernel(const RaggedParams p) {
  using C = RaggedMma<D>;
  constexpr bool BF = KIND == kKvBf16;             // e4m3 and fp16 caches: fp16 products
  constexpr int CH = C::kCH, LD = C::kLd, NT = CH / 8, KS = D / 16;
  constexpr float kLn2 = 0.69314718055994530942f, kUp = BF ? 0.f : 15.f;
  extern __shared__ __align__(16) uint8_t smem[];
  uint16_t* sq = reinterpret_cast<uint16_t*>(smem);
  uint16_t* sk = sq + C::kRows * LD;
  uint16_t* sv = sk + CH * LD;
  int32_t* table = reinterpret_cast<int32_t*>(sv + CH * LD);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, tq = lane & 3;

  griddep_wait();
  griddep_launch();
  ragged_table(p, table);
  ragged_rows_without_keys<D, QT>(p, table);
  const int W = table[p.G];
  const int ctas = W < (int)gridDim.x ? W : (int)gridDim.x;
  if (tid == 0) ragged_note_cut(p, blockIdx.x, nullptr, W, ctas);   // nothing yet
  if ((int)blockIdx.x >= ctas) return;
  const int x0 = range_begin(W, ctas, blockIdx.x), x1 = range_begin(W, ctas, blockIdx.x + 1);
  const uint32_t q32 = smem_u32(sq), k32 = smem_u32(sk), v32 = smem_u32(sv);
  const int mtx = lane >> 3, rr = lane & 7;

  int g = find_row(table, p.G, x0);
  RaggedPiece w;
  for (int x = x0; ragged_next(p, table, x1, g, x, w);) {
    const int t0 = w.t0 + w.first(0, p.TS), nrows = min(p.TS, w.n - w.first(0, p.TS)) * p.grp;
    __syncthreads();
    for (int i = tid; i < C::kRows * (D / 8); i += 128) {
      const int r = i / (D / 8), c = (i - r * (D / 8)) * 8;
      uint32_t o[4] = {0, 0, 0, 0};
      if (r < nrows) {
        const QT* src = reinterpret_cast<const QT*>(p.q) + (int64_t)(t0 + r / p.grp) * p.q_st +
                        (int64_t)(w.h * p.grp + r % p.grp) * p.q_sh + c;
        float f[8];
        load_q8<QT>(src, f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2<BF>(f[2 * e], f[2 * e + 1]);
      }
      *reinterpret_cast<uint4*>(sq + r * LD + c) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    float sc = p.scale, vscale = 1.f;
    if constexpr (KIND == kKvFp8) {
      sc *= p.k_scale ? __ldg(p.k_scale + w.h) : 1.f;
      vscale = p.v_scale ? __ldg(p.v_scale + w.h) : 1.f;
    }
    float acc[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;

    for (int ch = w.c0; ch < w.c1; ++ch) {
      const int tok0 = ch * CH, nvalid = min(CH, w.len - tok0);
      __syncthreads();
      for (int i = tid; i < CH * (D / 8); i += 128) {
        const int tk = i / (D / 8), c = i - tk * (D / 8);
        uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
        if (tk < nvalid) {
          const int pos = tok0 + tk, pi = pos / p.P, off = pos - pi * p.P;
          int pg = __ldg(p.block_table + (int64_t)w.g * p.bt_stride + pi);
          if (pg < 0 || pg >= p.num_pages) {
            if (c == 0) record_status(p.status, kStatusBounds);
            pg = 0;
          }
          kw = load_cache8<KIND>(p.kc, pg * p.k_sp + off * p.k_st + w.h * p.k_sh + c * p.k_sg, 1);
          vw = load_cache8<KIND>(p.vc, pg * p.v_sp + off * p.v_st + w.h * p.v_sh + c * 8 * p.v_sd,
                                 p.v_sd);
        }
        *reinterpret_cast<uint4*>(sk + tk * LD + c * 8) = kw;
        *reinterpret_cast<uint4*>(sv + tk * LD + c * 8) = vw;
      }
      __syncthreads();

      float s[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t a[4];
        ldsm_x4(q32 + (uint32_t)(((16 * warp + (mtx & 1) * 8 + rr) * LD + 16 * ks + (mtx >> 1) * 8) * 2), a);
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t b[4];   // two key tiles x two halves of the 16 dims
          ldsm_x4(k32 + (uint32_t)(((8 * (j + (mtx >> 1)) + rr) * LD + 16 * ks + (mtx & 1) * 8) * 2), b);
          mma16816<BF>(s[j], a, b[0], b[1]);
          mma16816<BF>(s[j + 1], a, b[2], b[3]);
        }
      }
      float mx[2] = {m[0], m[1]};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = 8 * j + 2 * tq + (e & 1) < nvalid ? s[j][e] * sc : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
        }
      float mz[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        mz[r] = mx[r] == -INFINITY ? 0.f : mx[r];   // a row of -inf scores so far
        const float al = fast_exp2(m[r] - mz[r]);
        m[r] = mx[r];
        l[r] *= al;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          acc[i][2 * r] *= al;
          acc[i][2 * r + 1] *= al;
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][e] = fast_exp2(s[j][e] - (mz[e >> 1] - kUp));
          l[e >> 1] += s[j][e];
        }
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        const uint32_t a[4] = {pack2<BF>(s[j][0], s[j][1]), pack2<BF>(s[j][2], s[j][3]),
                               pack2<BF>(s[j + 1][0], s[j + 1][1]), pack2<BF>(s[j + 1][2], s[j + 1][3])};
#pragma unroll
        for (int i = 0; i < D / 8; i += 2) {
          uint32_t b[4];   // keys 0-7 | 8-15 of the step x two dim tiles
          ldsm_x4_t(v32 + (uint32_t)(((8 * j + (mtx & 1) * 8 + rr) * LD + 8 * i + (mtx >> 1) * 8) * 2), b);
          mma16816<BF>(acc[i], a, b[0], b[1]);
          mma16816<BF>(acc[i + 1], a, b[2], b[3]);
        }
      }
    }

    const bool whole = w.whole();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      const int row = 16 * warp + gq + 8 * r;
      if (row >= nrows) continue;
      float inv = l[r] > 0.f ? vscale / l[r] : l[r];   // no mass at all: 0; NaN stays
      float lse2 = m[r] + (fast_log2(l[r]) - kUp);
      const int t = t0 + row / p.grp, h = w.h * p.grp + row % p.grp;
      if (whole) {
        if (p.own_o != nullptr) {   // join with the sequence's own part
          const int64_t at = (int64_t)t * p.Hq + h;
          const float2 jw = join_weights(lse2, p.own_lse[at], lse2);
          inv *= jw.x;
          if (jw.y != 0.f) {
            const float* own = p.own_o + at * D + 2 * tq;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              acc[i][2 * r] = acc[i][2 * r] * inv + own[8 * i] * jw.y;
              acc[i][2 * r + 1] = acc[i][2 * r + 1] * inv + own[8 * i + 1] * jw.y;
            }
            inv = 1.f;
          }
        }
        QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + 2 * tq;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          dst[8 * i] = QT(acc[i][2 * r] * inv);
          dst[8 * i + 1] = QT(acc[i][2 * r + 1] * inv);
        }
        if (p.lse != nullptr && tq == 0) p.lse[(int64_t)t * p.lse_st + h] = lse2 * kLn2;
      } else {
        const int64_t at = (int64_t)w.segment(blockIdx.x) * p.rows + row;
        float* dst = p.seg_o + at * D + 2 * tq;
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
          *reinterpret_cast<float2*>(dst + 8 * i) =
              make_float2(acc[i][2 * r] * inv, acc[i][2 * r + 1] * inv);
        if (tq == 0) p.seg_lse[at] = lse2;
      }
    }
    if (tid == 0 && w.c0 == 0 && !whole) ragged_note_cut(p, blockIdx.x, &w, W, ctas);
  }
}

}  // namespace b2d
