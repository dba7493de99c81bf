// ragged_tc_kernel.cuh — ragged attention (ragged.cuh) on tcgen05: head_dim 64
// and 128, page sizes that are multiples of 16, NHD / HND caches of every
// type.
//
// One block per SM works on an item of up to 256 query rows: two tiles of 128
// rows, each with its own stream of
//   S = Q.K^T   (128 x 128 keys, Q and K in shared memory, S in TMEM)
//   P = 2^(scale S - m)   (one thread per row; P goes back to TMEM, 16 bits,
//                          over the columns of S that were read already)
//   O += P.V    (A from TMEM, V in shared memory, O in TMEM)
// The two streams take turns on the tensor cores: while one is in its
// softmax, the products of the other run.  With both tiles in use every K and
// V chunk that is loaded serves 256 rows.  An item with one tile (few query
// rows) gives its even chunks to stream 0 and its odd ones to stream 1, which
// share the rows; the two halves are merged through shared memory at the end.
//
// Warps 0-3 and 4-7: softmax and output of stream 0 and 1 (thread = row =
// TMEM lane, so maximum, sum and rescaling need no other thread).  Warp 8:
// TMEM allocation and all MMAs.  Warp 9: TMA.  e4m3 caches: warps 10-13
// convert each raw tile to fp16 (exact) into the swizzled layout the MMAs
// read; q and P are then fp16 too.
//
// The maximum is lazy: it moves only when a score exceeds it by 2^8, so P <=
// 256 and O is rescaled (a TMEM round trip) rarely.  Keys past the end:
// their pages are not loaded, their scores are masked, and the MMA warp zeroes
// their V rows, which may hold anything, even NaN, before P.V reads them.
#pragma once

#include <type_traits>

#include "gqa_mma_kernel.cuh"
#include "ragged.cuh"
#include "tcgen05.cuh"

namespace b2d {

template <int D, int KIND>
struct RaggedTc {
  static constexpr bool kFp8 = KIND == kKvFp8;
  static constexpr int kCH = 128;                    // keys per chunk
  static constexpr int kBlk = D / 64;                // 128-byte column blocks of a tile
  static constexpr uint32_t kTile = kBlk * 16384;    // [block][128 rows][128 bytes], swizzled
  static constexpr uint32_t kRaw = 128 * D;          // e4m3 tile [128 keys][D]
  static constexpr int kSlots = (kFp8 ? 98304 : 131072) / kTile;   // K and V alternate
  static constexpr int kRawSlots = kFp8 ? 49152 / kRaw : 0;
  static constexpr int kThreads = kFp8 ? 448 : 320;
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffRing = 2 * kTile;
  static constexpr uint32_t kOffRaw = kOffRing + kSlots * kTile;
  static constexpr uint32_t kOffX = kOffRaw + kRawSlots * kRaw;    // m, l of stream 1: 2 x 128 floats
  static constexpr uint32_t kOffBar = kOffX + 1024;
  // full, empty [slots]; raw full, empty; q, s, p, o full [2]; exchange [3]; drain
  static constexpr int kBars = 2 * kSlots + 2 * kRawSlots + 8 + 3 + 1;
  static constexpr uint32_t kOffTmem = kOffBar + kBars * 8;
  static constexpr uint32_t kOffTable = kOffTmem + 16;
  static constexpr size_t smem(int groups) { return kOffTable + (size_t)(groups + 1 + 32) * 4 + 1024; }
};

// 32 lanes x 32 columns: register j of thread t is lane t (of the warp's
// quadrant), column j.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
      "%29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y),
               "r"(v.z), "r"(v.w)
               : "memory");
}

// kind::f16 instruction descriptor, fp32 accumulators, A K-major.
__host__ __device__ constexpr uint32_t umma_idesc_16(bool bf16, int M, int N, bool b_mn_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

template <int D, int KIND, typename QT>
__global__ void __launch_bounds__(RaggedTc<D, KIND>::kThreads, 1)
    ragged_tc_kernel(const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const RaggedParams p, int granule) {
  using C = RaggedTc<D, KIND>;
  constexpr bool BF = KIND == kKvBf16;
  constexpr bool F8 = C::kFp8;
  constexpr int CH = C::kCH, NS = C::kSlots, NR = C::kRawSlots;
  constexpr float kLazy = 8.f;
  constexpr float kLn2 = 0.69314718055994530942f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + NS;
  uint64_t* raw_full = empty + NS;
  uint64_t* raw_empty = raw_full + NR;
  uint64_t* q_full = raw_empty + NR;
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* xch = o_full + 2;
  uint64_t* drain = xch + 3;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffTmem);
  int32_t* table = reinterpret_cast<int32_t*>(smem + C::kOffTable);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, F8 ? 128 : 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < NR; ++i) {
      mbar_init(raw_full + i, 1);
      mbar_init(raw_empty + i, 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(q_full + s, 128);
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 128);
      mbar_init(o_full + s, 1);
    }
    for (int i = 0; i < 3; ++i) mbar_init(xch + i, 256);
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 9 && lane == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  tc_fence_before();
  ragged_table(p, table, table + p.G + 1);   // ends with __syncthreads
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= p.G; i += blockDim.x) p.table_g[i] = table[i];
  ragged_zero_rows<D, QT>(p);
  const int W = table[p.G];
  const int ctas = W < (int)gridDim.x ? W : (int)gridDim.x;
  const bool active = (int)blockIdx.x < ctas;
  const int x0 = active ? range_begin(W, ctas, blockIdx.x) : 0;
  const int x1 = active ? range_begin(W, ctas, blockIdx.x + 1) : 0;
  const int S = p.TS >> 1;                       // tokens of a tile
  const int g_first = active ? find_row(table, p.G, x0) : 0;
  // All lanes of a warp see the same answer: one that ran out of time stops all.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mla_wait(bar, parity, p.status, p.wait_ns));
  };

  if (warp < 8) {
    // ---------------- softmax and output ----------------
    const int st = warp >> 2;                    // stream
    const int r = threadIdx.x & 127;             // row of the tile
    const uint32_t t_row = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t t_s = t_row + (uint32_t)(st * 128);
    const uint32_t t_o = t_row + 256u + (uint32_t)(st * D);
    const uint32_t q_base = sbase + C::kOffQ + (uint32_t)st * C::kTile;
    float* xml = reinterpret_cast<float*>(smem + C::kOffX);
    uint32_t ns_all = 0, pieces = 0, nx = 0;     // steps, pieces and exchanges so far
    int g = g_first;
    bool ok = true;
    for (int x = x0; x < x1 && ok;) {
      while (x >= table[g + 1]) ++g;
      const RaggedPiece w = ragged_piece(p, table, g, x, x1);
      const int nc = w.c1 - w.c0;
      const bool dual = w.ntok > S;
      const int steps = dual ? nc : (nc - st + 1) >> 1;
      const int tile0 = dual ? st * S : 0;       // first token of this tile
      const int nrows = min(S, w.ntok - tile0) * p.grp;
      const bool whole = w.c0 == 0 && w.c1 == w.nch;
      const int slot = (w.c0 == 0 && x > x0) ? 1 : 0;
      x += nc;
      if (steps == 0) continue;
      float sl = p.scale, vscale = 1.f;
      if constexpr (F8) {
        sl *= p.k_scale ? __ldg(p.k_scale + w.h) : 1.f;
        vscale = p.v_scale ? __ldg(p.v_scale + w.h) : 1.f;
      }
      // A negative scale turns into the sign of q, so that the largest product
      // is always the largest score.
      const uint32_t flip = sl < 0.f ? 0x80008000u : 0u;
      sl = fabsf(sl);
      const int tok = w.t0 + tile0 + r / p.grp, head = w.h * p.grp + r % p.grp;
      {
        const QT* src = reinterpret_cast<const QT*>(p.q) + (int64_t)tok * p.q_st + (int64_t)head * p.q_sh;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < nrows) {
            v = *reinterpret_cast<const uint4*>(src + 8 * c);
            if constexpr (F8 && std::is_same<QT, __nv_bfloat16>::value) {
              uint32_t* e = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = bf16x2_to_f2(e[i]);
                e[i] = pack2<false>(f.x, f.y);
              }
            }
            v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
          }
          sts128(swz(q_base + (uint32_t)(c >> 3) * 16384u, r, c & 7), v);
        }
        fence_async_smem();
        mbar_arrive(q_full + st);
      }
      const bool live = 32 * (warp & 3) < nrows;  // this warp has query rows
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < steps; ++i) {
        const int nvalid = min(CH, w.len - (w.c0 + (dual ? i : 2 * i + st)) * CH);
        if (!wait(s_full + st, ns_all & 1u)) { ok = false; break; }
        ++ns_all;
        tc_fence_after();
        if (live) {
          float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < CH; c += 32) {
            uint32_t v[32];
            tmem_ld32(t_s + (uint32_t)c, v);
            tmem_wait_ld();
            if (nvalid == CH) {
#pragma unroll
              for (int j = 0; j < 32; ++j) mc[j & 3] = fmaxf(mc[j & 3], __uint_as_float(v[j]));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c + j < nvalid) mc[j & 3] = fmaxf(mc[j & 3], __uint_as_float(v[j]));
            }
          }
          const float cm = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3]));
          float alpha = 1.f;
          if (cm != -INFINITY && (m == -INFINITY || (cm - m) * sl > kLazy)) {
            alpha = m == -INFINITY ? 0.f : fast_exp2((m - cm) * sl);
            m = cm;
          }
          if (__any_sync(0xffffffffu, alpha != 1.f) && i > 0) {
            // S of this step was issued behind P.V of the last one, so O is
            // complete; P.V of this step waits for this warp.
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t v[32];
              tmem_ld32(t_o + (uint32_t)c, v);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
              tmem_st32(t_o + (uint32_t)c, v);
            }
          }
          const float off = m == -INFINITY ? 0.f : -m * sl;
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < CH; c += 32) {
            uint32_t v[32], pk[16];
            tmem_ld32(t_s + (uint32_t)c, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float a = fast_exp2(fmaf(__uint_as_float(v[j]), sl, off));
              float b = fast_exp2(fmaf(__uint_as_float(v[j + 1]), sl, off));
              if (nvalid != CH) {
                a = c + j < nvalid ? a : 0.f;
                b = c + j + 1 < nvalid ? b : 0.f;
              }
              ls[j & 3] += a;
              ls[(j & 3) + 1] += b;
              pk[j >> 1] = pack2<BF>(a, b);
            }
            tmem_st16(t_s + (uint32_t)(c >> 1), pk);
          }
          l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(p_full + st);
      }
      if (!ok) break;
      if (!wait(o_full + st, pieces & 1u)) { ok = false; break; }
      ++pieces;
      tc_fence_after();

      float own = 1.f, other = 0.f;              // weights of the two streams' halves
      const bool exchange = !dual && nc > 1;
      float* xo = reinterpret_cast<float*>(smem + C::kOffQ);
      // Row r of stream 1's half: 16-byte groups, permuted by the row so that
      // neighbouring rows use different banks.
      auto xat = [&](int c4) { return xo + r * D + ((c4 ^ (r & (D / 4 - 1))) << 2); };
      if (exchange) {
        // Every Q.K^T of both streams is done once both are here: Q is free.
        mbar_arrive(xch);
        if (!wait(xch, nx & 1u)) { ok = false; break; }
        if (st == 1) {
          xml[r] = m;
          xml[128 + r] = l;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld32(t_o + (uint32_t)c, v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<uint4*>(xat((c + j) >> 2)) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          }
        }
        mbar_arrive(xch + 1);
        if (!wait(xch + 1, nx & 1u)) { ok = false; break; }
        if (st == 0) {
          const float m1 = xml[r], l1 = xml[128 + r];
          if (m1 != -INFINITY) {
            const float mm = fmaxf(m, m1);
            own = m == -INFINITY ? 0.f : fast_exp2((m - mm) * sl);
            other = fast_exp2((m1 - mm) * sl);
            m = mm;
            l = l * own + l1 * other;
          } else {
            l += l1;                             // 0, or NaN
          }
        }
      }
      if (st == 0 || !exchange) {
        const float inv = l > 0.f ? vscale / l : l;
        const float lse2 = l == 0.f ? -INFINITY : m * sl + fast_log2(l);
        const bool direct = whole && p.out_f32 == nullptr;
        const int64_t at = whole ? (int64_t)tok * p.Hq + head
                                 : (int64_t)(2 * blockIdx.x + slot) * p.rows + tile0 * p.grp + r;
        float* fdst = (whole ? p.out_f32 : p.seg_o) + at * D;
        QT* dst = reinterpret_cast<QT*>(p.out) + (int64_t)tok * p.o_st + (int64_t)head * p.o_sh;
        if (live) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            tmem_ld32(t_o + (uint32_t)c, v);
            tmem_wait_ld();
            if (r < nrows) {
              float f[32];
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]) * own;
              if (exchange && other != 0.f) {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                  const float4 y = *reinterpret_cast<const float4*>(xat((c + j) >> 2));
                  f[j] += y.x * other;
                  f[j + 1] += y.y * other;
                  f[j + 2] += y.z * other;
                  f[j + 3] += y.w * other;
                }
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] *= inv;
              if (direct) {
#pragma unroll
                for (int j = 0; j < 32; j += 8) store_out8<QT>(dst + c + j, f + j);
              } else {
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                  *reinterpret_cast<float4*>(fdst + c + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
              }
            }
          }
        }
        if (r < nrows) {
          if (!direct) (whole ? p.lse2 : p.seg_lse)[at] = lse2;
          else if (p.lse != nullptr) p.lse[(int64_t)tok * p.lse_st + head] = lse2 * kLn2;
        }
        tc_fence_before();
      }
      if (exchange) {
        mbar_arrive(xch + 2);                    // the halves are read: Q may be written again
        if (!wait(xch + 2, nx & 1u)) { ok = false; break; }
        ++nx;
      }
    }
  } else if (warp == 8) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t idesc_qk = umma_idesc_16(BF, 128, CH, false);
    constexpr uint32_t idesc_pv = umma_idesc_16(BF, 128, D, true);
    uint32_t ring = 0;                           // ring position of the piece's first K
    uint32_t np[2] = {0, 0}, nq[2] = {0, 0};
    int g = g_first;
    bool ok = true;
    for (int x = x0; x < x1 && ok;) {
      while (x >= table[g + 1]) ++g;
      const RaggedPiece w = ragged_piece(p, table, g, x, x1);
      const int nc = w.c1 - w.c0;
      const bool dual = w.ntok > S;
      x += nc;
      // S of stream st for chunk j (of this piece)
      auto qk = [&](int st, int j, bool last_use) -> bool {
        const uint32_t n = ring + 2u * (uint32_t)j, slot = n % NS;
        if (!wait(full + slot, (n / NS) & 1u)) return false;
        tc_fence_after();
        if (lane == 0) {
          const uint64_t ad0 = umma_desc_sw128(sbase + C::kOffQ + (uint32_t)st * C::kTile, 16, 1024);
          const uint64_t bd0 = umma_desc_sw128(sbase + C::kOffRing + slot * C::kTile, 16, 1024);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t o = (uint64_t)(((k >> 2) * 16384 + (k & 3) * 32) >> 4);
            umma_bf16(tmem + (uint32_t)(st * 128), ad0 + o, bd0 + o, idesc_qk, k > 0);
          }
          umma_commit(s_full + st);
          if (last_use) umma_commit(empty + slot);
        }
        __syncwarp();
        return true;
      };
      auto pv = [&](int st, int j, bool first, bool first_use, bool last_use) -> bool {
        if (!wait(p_full + st, np[st] & 1u)) return false;
        ++np[st];
        const uint32_t n = ring + 2u * (uint32_t)j + 1u, slot = n % NS;
        if (!wait(full + slot, (n / NS) & 1u)) return false;
        if constexpr (!F8) {
          const int nvalid = w.len - (w.c0 + j) * CH;
          if (nvalid < CH && first_use) {
            const int rows = CH - nvalid;
            for (int i = lane; i < rows * 8 * C::kBlk; i += 32) {
              const int b = i / (rows * 8), rest = i - b * (rows * 8);
              sts128(sbase + C::kOffRing + slot * C::kTile + (uint32_t)(b * 16384 + nvalid * 128 + rest * 16),
                     make_uint4(0, 0, 0, 0));
            }
            fence_async_smem();
            __syncwarp();
          }
        }
        tc_fence_after();
        if (lane == 0) {
          const uint64_t vd0 = umma_desc_sw128(sbase + C::kOffRing + slot * C::kTile, 16384, 1024);
#pragma unroll
          for (int k = 0; k < CH / 16; ++k)
            umma_bf16_ts(tmem + 256u + (uint32_t)(st * D), tmem + (uint32_t)(st * 128 + 8 * k),
                         vd0 + (uint64_t)((k * 2048) >> 4), idesc_pv, !(first && k == 0));
          if (last_use) umma_commit(empty + slot);
        }
        __syncwarp();
        return true;
      };
      auto done = [&](int st) {
        if (lane == 0) umma_commit(o_full + st);
        __syncwarp();
      };
      for (int st = 0; st < 2 && ok; ++st) {
        if (!dual && st >= nc) break;
        ok = wait(q_full + st, nq[st] & 1u);
        ++nq[st];
        ok = ok && qk(st, dual ? 0 : st, !dual || st == 1);
      }
      if (dual) {
        for (int j = 0; j < nc && ok; ++j)
          for (int st = 0; st < 2 && ok; ++st) {
            ok = pv(st, j, j == 0, st == 0, st == 1);
            if (ok && j + 1 < nc) ok = qk(st, j + 1, st == 1);
            else if (ok) done(st);
          }
      } else {
        for (int j = 0; j < nc && ok; ++j) {
          ok = pv(j & 1, j, j < 2, true, true);
          if (ok && j + 2 < nc) ok = qk(j & 1, j + 2, true);
          else if (ok) done(j & 1);
        }
      }
      ring += 2u * (uint32_t)nc;
    }
    // Nothing of this warp is in flight when tensor memory is freed.
    if (lane == 0) umma_commit(drain);
    __syncwarp();
    wait(drain, 0);
  } else if (warp == 9) {
    // ---------------- TMA producer ----------------
    if (!p.no_loads) {
      constexpr int N = F8 ? NR : NS;
      constexpr int PB = F8 ? 1 : C::kBlk;       // boxes per granule
      constexpr uint32_t kBox = F8 ? D : 128;    // bytes per key of a box
      uint64_t* fb = F8 ? raw_full : full;
      uint64_t* eb = F8 ? raw_empty : empty;
      const uint32_t base = C::kOffRaw * (F8 ? 1 : 0) + C::kOffRing * (F8 ? 0 : 1);
      constexpr uint32_t bytes = F8 ? C::kRaw : C::kTile;
      uint64_t policy;
      asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
      const int gr = lane / PB, blk = lane - gr * PB;   // this lane's box: granule and column block
      const int granules = CH / granule;
      uint32_t n = 0;
      int g = g_first;
      bool ok = true;
      for (int x = x0; x < x1 && ok;) {
        while (x >= table[g + 1]) ++g;
        const RaggedPiece w = ragged_piece(p, table, g, x, x1);
        const int32_t* row = p.block_table + (int64_t)w.g * p.bt_stride;
        auto page_of = [&](int c) -> int {
          const int t = c * CH + gr * granule;
          return gr < granules && c < w.c1 && t < w.len ? __ldg(row + t / p.P) : 0;
        };
        int page = page_of(w.c0);
        for (int c = w.c0; c < w.c1 && ok; ++c) {
          const int t = c * CH + gr * granule;
          const bool load = gr < granules && t < w.len;
          if (page < 0 || page >= p.num_pages) {
            record_status(p.status, kStatusBounds);
            page = 0;
          }
          const int left = min(CH, w.len - c * CH);
          const uint32_t tx = (uint32_t)((left + granule - 1) / granule * granule) * kBox * PB;
          const int next = page_of(c + 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const uint32_t slot = n % N;
            if (!wait(eb + slot, ((n / N) & 1u) ^ 1u)) { ok = false; break; }
            if (lane == 0) mbar_arrive_expect_tx(fb + slot, tx);
            __syncwarp();
            if (load)
              tma_load_4d(smem + base + slot * bytes + (uint32_t)(blk * 16384 + gr * granule * (int)kBox),
                          kv ? &tmap_v : &tmap_k, fb + slot, blk * 64, t % p.P, w.h, page, policy);
          }
          page = next;
        }
        x += w.c1 - w.c0;
      }
      // Copies still in flight land before the block ends.
      for (uint32_t i = n > (uint32_t)N ? n - N : 0; i < n; ++i)
        if (!mbar_wait(fb + i % N, (i / N) & 1u, p.wait_ns)) break;
    }
  } else if (F8) {
    // ---------------- e4m3 -> fp16 ----------------
    constexpr int LPK = D / 16;                  // lanes per key, 16 values each
    const int ct = threadIdx.x - 320;
    const int c = ct % LPK;
    uint32_t n = 0;
    int g = g_first;
    bool ok = true;
    for (int x = x0; x < x1 && ok;) {
      while (x >= table[g + 1]) ++g;
      const RaggedPiece w = ragged_piece(p, table, g, x, x1);
      for (int ch = w.c0; ch < w.c1 && ok; ++ch) {
        const int nvalid = min(CH, w.len - ch * CH);
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t rs = n % (NR > 0 ? NR : 1), slot = n % NS;
          if (!wait(raw_full + rs, (n / (NR > 0 ? NR : 1)) & 1u) ||
              !wait(empty + slot, ((n / NS) & 1u) ^ 1u)) {
            ok = false;
            break;
          }
          const uint32_t src = sbase + C::kOffRaw + rs * C::kRaw, dst = sbase + C::kOffRing + slot * C::kTile;
#pragma unroll 4
          for (int k = ct / LPK; k < CH; k += 128 / LPK) {
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (k < nvalid) {
              const uint4 v = lds128(src + (uint32_t)(k * D + c * 16));
              lo = make_uint4(e4m3x2_to_f16x2_cvt(v.x), e4m3x2_to_f16x2_cvt(v.x >> 16),
                              e4m3x2_to_f16x2_cvt(v.y), e4m3x2_to_f16x2_cvt(v.y >> 16));
              hi = make_uint4(e4m3x2_to_f16x2_cvt(v.z), e4m3x2_to_f16x2_cvt(v.z >> 16),
                              e4m3x2_to_f16x2_cvt(v.w), e4m3x2_to_f16x2_cvt(v.w >> 16));
            }
            // Lanes of the second column block store their halves in the other
            // order, so the 8 lanes of a key use 8 different bank groups.
            const uint32_t b = dst + (uint32_t)(c >> 2) * 16384u;
            const int c2 = 2 * (c & 3), sw = (c >> 2) & 1;
            sts128(swz(b, k, c2 + sw), sw ? hi : lo);
            sts128(swz(b, k, c2 + 1 - sw), sw ? lo : hi);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(raw_empty + rs);
          fence_async_smem();
          mbar_arrive(full + slot);
        }
      }
      x += w.c1 - w.c0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

}  // namespace b2d
