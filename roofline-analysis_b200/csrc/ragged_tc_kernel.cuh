// ragged_tc_kernel.cuh — ragged attention (ragged.cuh) on tcgen05: head_dim 64
// and 128, page sizes that are multiples of 16, NHD / HND caches of every
// type.
//
// One block per SM works on an item of two parts of up to 128 query rows, each
// with its own stream of
//   S = Q.K^T   (128 x 128 keys, Q and K in shared memory, S in TMEM)
//   P = 2^(scale S - m)   (one thread per row; P goes back to TMEM, 16 bits,
//                          over the columns of S that were read already)
//   O += P.V    (A from TMEM, V in shared memory, O in TMEM)
// While one stream is in its softmax, the products of the other run.  The two
// parts are tiles of the same KV head, so that every K and V chunk that is
// loaded serves 256 rows, or (few query rows) two KV heads with chunks of
// their own.
//
// Warps 0-3 and 4-7: softmax and output of stream 0 and 1 (thread = row =
// TMEM lane, so maximum, sum and rescaling need no other thread).  Warp 8:
// one thread issues the MMAs of both streams in turn, which keeps one stream's
// products beside the other's softmax.  Warp 10: TMA (head_dim 128, 16 bits: K
// only, and warp 9 V).  Warp 11: the last V tile of a sequence, see below.
// e4m3 caches: warps 12-15 convert each raw tile to fp16 (exact) into the
// swizzled layout the MMAs read; q and P are then fp16 too.  The softmax warps
// get registers of the others (setmaxnreg).
//
// The maximum is lazy: it moves only when a score exceeds it by 2^8, so P <=
// 256 and O is rescaled (a TMEM round trip) rarely: a chunk that leaves it, or
// sets it first, goes from S to P in registers, any other takes the general
// step.  In fp16, whose smallest number is 2^-24, P is 2^7 as large (at most
// 2^15): of a long sequence beside a dominant key, the many weights far below
// it keep their bits (20000 of 2^-24.3 each were 27 % off, of 2^-26 all lost).
// The sum is of the same scaled weights, so only lse has to take the 7 back.
//
// Keys past the end: their pages are not loaded, their scores are masked, and
// warp 11 (e4m3: the conversion) zeroes their V rows, which may hold anything,
// even NaN, before P.V reads them.
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
  static constexpr int kRawSlots = kFp8 ? 32768 / kRaw : 0;
  // K and V loads from a warp each: 866 -> 832 us for 16 requests of up to 1024 x
  // 6500 tokens at head_dim 128; at head_dim 64, whose tiles are half as large, it
  // cost 5 %.
  static constexpr bool kTwoLoaders = D == 128 && !kFp8;
  static constexpr uint32_t kStage = 2048;           // output staging of a softmax warp
  static constexpr int kThreads = kFp8 ? 512 : 384;
  // Registers per thread, softmax and others: 256 x kRegSm + (kThreads - 256) x
  // kRegOther is at most what the block starts with (168 or 128 a thread).
  static constexpr int kRegSm = kFp8 ? 184 : 208, kRegOther = kFp8 ? 72 : 80;
  static_assert(256 * kRegSm + (kThreads - 256) * kRegOther <= kThreads * (kFp8 ? 128 : 168), "");
  static constexpr uint32_t kOffQ = 0;
  static constexpr uint32_t kOffRing = 2 * kTile;
  static constexpr uint32_t kOffRaw = kOffRing + kSlots * kTile;
  static constexpr uint32_t kOffStage = kOffRaw + kRawSlots * kRaw;
  static constexpr uint32_t kOffBar = kOffStage + 8 * kStage;
  // full, empty, tail [slots]; raw full, empty; q, s, p, o full [2]; drain
  static constexpr int kBars = 3 * kSlots + 2 * kRawSlots + 9;
  static constexpr uint32_t kOffTmem = kOffBar + kBars * 8;
  static constexpr uint32_t kOffTable = kOffTmem + 16;   // (TMEM address, failure flag)
  static constexpr size_t smem(int groups) { return kOffTable + ragged_table_bytes(groups) + 1024; }
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
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

// Largest of three; NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D, int KIND, typename QT>
__global__ void __launch_bounds__(RaggedTc<D, KIND>::kThreads, 1)
    ragged_tc_kernel(const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ CUtensorMap tmap_v, const RaggedParams p, int granule) {
  using C = RaggedTc<D, KIND>;
  constexpr bool BF = KIND == kKvBf16;
  constexpr bool F8 = C::kFp8;
  constexpr int CH = C::kCH, NS = C::kSlots, NR = C::kRawSlots;
  constexpr float kLazy = 8.f, kUp = BF ? 0.f : 7.f;
  constexpr float kLn2 = 0.69314718055994530942f;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + NS;
  uint64_t* tail = empty + NS;     // a V tile that warp 11 completes
  uint64_t* raw_full = tail + NS;
  uint64_t* raw_empty = raw_full + NR;
  uint64_t* q_full = raw_empty + NR;
  uint64_t* s_full = q_full + 2;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* drain = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffTmem);
  int32_t* table = reinterpret_cast<int32_t*>(smem + C::kOffTable);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  volatile int* failed = reinterpret_cast<int*>(tmem_slot + 1);   // a wait ran out of time
  if (threadIdx.x == 0) {
    *failed = 0;
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, F8 ? 4 : 1);
      mbar_init(empty + i, 1);
      mbar_init(tail + i, 1);
    }
    for (int i = 0; i < NR; ++i) {
      mbar_init(raw_full + i, 1);
      mbar_init(raw_empty + i, 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(q_full + s, 4);
      mbar_init(s_full + s, 1);
      mbar_init(p_full + s, 4);
      mbar_init(o_full + s, 1);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 10 && lane == 0) {
    prefetch_tmap(&tmap_k);
    prefetch_tmap(&tmap_v);
  }
  tc_fence_before();
  // Everything above overlaps the kernel before.  Shared prefix: that one is the
  // own-token decode, all of whose blocks have seen its inputs complete before
  // they let this kernel start, so only its outputs are waited for, where they
  // are read (and before the block ends, for the merge).
  if (!p.beside) griddep_wait();
  griddep_launch();
  ragged_table(p, table);                    // ends with __syncthreads
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ragged_rows_without_keys<D, QT>(p, table);
  const int W = table[p.G];
  const int ctas = W < (int)gridDim.x ? W : (int)gridDim.x;
  const bool active = (int)blockIdx.x < ctas;
  const int x0 = active ? range_begin(W, ctas, blockIdx.x) : 0;
  const int x1 = active ? range_begin(W, ctas, blockIdx.x + 1) : 0;
  const int g_first = active ? find_row(table, p.G, x0) : 0;
  if (threadIdx.x == 0) ragged_note_cut(p, blockIdx.x, nullptr, W, ctas);   // nothing yet
  // All lanes of a warp see the same answer: one that ran out of time stops all.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    for (int i = 0; i < 64; ++i)   // the clock is read only after some polls
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const bool done = __all_sync(0xffffffffu, mla_wait(bar, parity, p.status, p.wait_ns));
    if (!done) *failed = 1;
    return done;
  };
  // One arrival per warp, behind what all its lanes did.
  auto arrive = [&](uint64_t* bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };

  // (one setmaxnreg per warpgroup: warps 8-11 and 12-15 give, 0-7 take)
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegSm));
    // ---------------- softmax and output ----------------
    const int st = warp >> 2;                    // stream
    const int r = threadIdx.x & 127, r0 = r & ~31;   // row of the part, first of the warp
    const uint32_t t_row = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const uint32_t t_s = t_row + (uint32_t)(st * 128);
    const uint32_t t_o = t_row + 256u + (uint32_t)(st * D);
    const uint32_t q_base = sbase + C::kOffQ + (uint32_t)st * C::kTile;
    const uint32_t stage = sbase + C::kOffStage + (uint32_t)warp * C::kStage;
    constexpr int kCpr = D / 8, kRpi = 32 / kCpr;  // 16-byte pieces of a row; rows per warp access
    const int tq = r / p.grp, hq = r - tq * p.grp; // this row's token of the part and query head

    auto rows_of = [&](const RaggedPiece& w) { return min(p.TS, w.n - w.first(st, p.TS)) * p.grp; };
    // Score scale of the part's KV head; a negative one turns into the sign of
    // q, so that the largest product is always the largest score.
    auto scale_of = [&](const RaggedPiece& w) {
      if constexpr (F8) return p.scale * (p.k_scale ? __ldg(p.k_scale + w.head(st)) : 1.f);
      else return p.scale;
    };
    // The part's query rows, loaded by whole rows, into the swizzled Q tile.
    auto load_q = [&](const RaggedPiece& w) {
      if (st >= w.parts()) return;
      const int nrows = rows_of(w);
      const uint32_t flip = scale_of(w) < 0.f ? 0x80008000u : 0u;
      const int64_t mine = (int64_t)(w.t0 + w.first(st, p.TS) + tq) * p.q_st +
                           (int64_t)(w.head(st) * p.grp + hq) * p.q_sh;
#pragma unroll 1
      for (int i0 = 0; i0 < kCpr; i0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rl = (i0 + i) * kRpi + lane / kCpr;
          const int64_t at = __shfl_sync(0xffffffffu, mine, rl);
          v[i] = make_uint4(0, 0, 0, 0);
          if (r0 + rl < nrows)
            v[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const QT*>(p.q) + at + 8 * (lane % kCpr));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rl = (i0 + i) * kRpi + lane / kCpr, c = lane % kCpr;
          if constexpr (F8 && std::is_same<QT, __nv_bfloat16>::value) {
            uint32_t* e = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = bf16x2_to_f2(e[j]);
              e[j] = pack2<false>(f.x, f.y);
            }
          }
          v[i].x ^= flip; v[i].y ^= flip; v[i].z ^= flip; v[i].w ^= flip;
          sts128(swz(q_base + (uint32_t)(c >> 3) * 16384u, r0 + rl, c & 7), v[i]);
        }
      }
      fence_async_smem();
      arrive(q_full + st);
    };

    uint32_t ns_all = 0, outs = 0;               // steps and outputs so far
    int g = g_first;
    bool ok = true;
    RaggedPiece w, d;                            // the next piece and the one before it
    int x = x0, nrows = 0;
    bool mine = false, live = false;             // d has this part; this warp has rows of it
    float sl = 0.f, m = 0.f, l = 0.f;
    for (;;) {
      // Q of the next piece first, so that its first product runs beside the
      // output of the last.
      const bool more = ragged_next(p, table, x1, g, x, w);
      if (more) load_q(w);
      if (mine) {
        const bool whole = d.whole();
        if (!wait(o_full + st, outs & 1u)) { ok = false; break; }
        ++outs;
        tc_fence_after();
        if (live) {
          float vscale = 1.f;
          if constexpr (F8) vscale = p.v_scale ? __ldg(p.v_scale + d.head(st)) : 1.f;
          float inv = l > 0.f ? vscale / l : l;
          float lse2 = l == 0.f ? -INFINITY : m * sl + (fast_log2(l) - kUp);
          const int tok = d.t0 + d.first(st, p.TS) + tq, head = d.head(st) * p.grp + hq;
          const bool join = whole && p.own_o != nullptr;
          float own = 0.f;                         // weight of the sequence's own part
          if (join) griddep_wait();
          if (join && r < nrows) {
            const float2 jw = join_weights(lse2, p.own_lse[(int64_t)tok * p.Hq + head], lse2);
            inv *= jw.x;
            own = jw.y;
          }
          // Through shared memory, 16 fp32 columns of each row at a time, so that a
          // warp stores whole sectors; 16-byte pieces are permuted by the row
          // against bank conflicts.  Lane k copies piece k % 4 of rows 8i + k / 4.
          // (Rolled and with few registers: it must not cost the softmax any.)
          const int64_t at = whole ? (int64_t)tok * p.o_st + (int64_t)head * p.o_sh
                                   : (int64_t)d.segment(blockIdx.x) * p.rows + st * p.TS * p.grp + r;
          const int64_t my_row = (int64_t)tok * p.Hq + head;
          const int piece = lane & 3, row4 = lane >> 2;
          auto piece_at = [&](int row, int q) {
            return stage + (uint32_t)(row * 64 + ((q ^ ((row >> 1) & 3)) << 4));
          };
          uint32_t v[16];
          float4 z[4];                             // own parts of the next columns
          auto load_own = [&](int c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float ow = __shfl_sync(0xffffffffu, own, 8 * i + row4);
              const int64_t orow = __shfl_sync(0xffffffffu, my_row, 8 * i + row4);
              z[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (ow != 0.f) {
                z[i] = *reinterpret_cast<const float4*>(p.own_o + orow * D + c + 4 * piece);
                z[i].x *= ow;
                z[i].y *= ow;
                z[i].z *= ow;
                z[i].w *= ow;
              }
            }
          };
          tmem_ld16(t_o, v);
          if (join) load_own(0);
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float f[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(v[4 * q + e]) * inv;
              sts128(piece_at(lane, q), make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]),
                                                   __float_as_uint(f[2]), __float_as_uint(f[3])));
            }
            if (c + 16 < D) tmem_ld16(t_o + (uint32_t)(c + 16), v);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rl = 8 * i + row4, cc = c + 4 * piece;
              uint4 y = lds128(piece_at(rl, piece));
              const int64_t dst = __shfl_sync(0xffffffffu, at, rl);
              if (join) {
                y.x = __float_as_uint(__uint_as_float(y.x) + z[i].x);
                y.y = __float_as_uint(__uint_as_float(y.y) + z[i].y);
                y.z = __float_as_uint(__uint_as_float(y.z) + z[i].z);
                y.w = __float_as_uint(__uint_as_float(y.w) + z[i].w);
              }
              if (r0 + rl < nrows) {
                if (whole)
                  *reinterpret_cast<uint2*>(reinterpret_cast<QT*>(p.out) + dst + cc) =
                      make_uint2(pack_pair<QT>(__uint_as_float(y.x), __uint_as_float(y.y)),
                                 pack_pair<QT>(__uint_as_float(y.z), __uint_as_float(y.w)));
                else
                  *reinterpret_cast<uint4*>(p.seg_o + dst * D + cc) = y;
              }
            }
            if (join && c + 16 < D) load_own(c + 16);
            __syncwarp();
          }
          tc_fence_before();
          if (r < nrows) {
            if (!whole) p.seg_lse[at] = lse2;
            else if (p.lse != nullptr) p.lse[(int64_t)tok * p.lse_st + head] = lse2 * kLn2;
          }
        }
        if (threadIdx.x == 0 && d.c0 == 0 && !whole) ragged_note_cut(p, blockIdx.x, &d, W, ctas);
      }
      if (!more) break;
      d = w;
      mine = st < d.parts();
      nrows = mine ? rows_of(d) : 0;
      live = r0 < nrows;
      sl = fabsf(scale_of(d));
      m = -INFINITY;
      l = 0.f;
      const float2 sl2 = make_float2(sl, sl);
      // P of 32 scores with offset off, and their sum; with a limit, P is 0 from
      // that score on.
      auto weights = [&](const uint32_t* v, float off, uint32_t* pk, float2& sum, int limit = 32) {
        const float2 off2 = make_float2(off, off);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float2 e = __ffma2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), sl2, off2);
          e.x = fast_exp2(e.x);
          e.y = fast_exp2(e.y);
          if (j >= limit) e.x = 0.f;
          if (j + 1 >= limit) e.y = 0.f;
          sum = __fadd2_rn(sum, e);
          pk[j >> 1] = pack2<BF>(e.x, e.y);
        }
      };
      // The general step: any state, keys from nvalid on masked.
      auto full_step = [&](int i, int nvalid) {
        float cm = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < CH; c += 32) {
          uint32_t v[32];
          tmem_ld32(t_s + (uint32_t)c, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            cm = max3_nan(cm, c + j < nvalid ? __uint_as_float(v[j]) : -INFINITY,
                          c + j + 1 < nvalid ? __uint_as_float(v[j + 1]) : -INFINITY);
        }
        float alpha = 1.f;
        if (cm != -INFINITY && (m == -INFINITY || (cm - m) * sl > kLazy)) {
          alpha = m == -INFINITY ? 0.f : fast_exp2((m - cm) * sl);
          m = cm;
        }
        if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // S of this step was issued behind P.V of the last one, so O is
          // complete; P.V of this step waits for this warp.
          l *= alpha;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(t_o + (uint32_t)c, o);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
            tmem_st16(t_o + (uint32_t)c, o);
          }
        }
        // A score of NaN or +inf makes the whole row NaN, by way of l.
        const float off = !(cm < INFINITY) ? NAN : m == -INFINITY ? 0.f : fmaf(-m, sl, kUp);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < CH; c += 32) {
          uint32_t v[32], pk[16];
          tmem_ld32(t_s + (uint32_t)c, v);
          tmem_wait_ld();
          weights(v, off, pk, sum, nvalid - c);
          tmem_st16(t_s + (uint32_t)(c >> 1), pk);
        }
        l += sum.x + sum.y;
      };
      // The usual step: the first of a piece, which sets the maximum, or one that
      // leaves it.  False: nothing was done.
      auto fast_step = [&](bool first, int nvalid) -> bool {
        uint32_t v[CH];
#pragma unroll
        for (int c = 0; c < CH; c += 32) tmem_ld32(t_s + (uint32_t)c, v + c);
        tmem_wait_ld();
        if (nvalid < CH) {
          if (sl == 0.f) return false;           // (a score of -inf times 0 is no weight of 0)
#pragma unroll
          for (int j = 0; j < CH; ++j)
            if (j >= nvalid) v[j] = 0xff800000u;
        }
        float mc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < CH; j += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mc[k] = max3_nan(mc[k], __uint_as_float(v[j + 2 * k]), __uint_as_float(v[j + 2 * k + 1]));
        const float cm = max3_nan(mc[0], mc[1], max3_nan(mc[2], mc[3], -INFINITY));
        const float mn = first ? cm : m;
        // (a NaN, an infinite maximum, or +inf against a finite one fail this)
        if (!__all_sync(0xffffffffu, (cm - mn) * sl <= kLazy && fabsf(mn) < INFINITY)) return false;
        m = mn;
        const float off = fmaf(-m, sl, kUp);
        float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
        for (int c = 0; c < CH; c += 32) {
          uint32_t pk[16];
          weights(v + c, off, pk, (c & 32) ? s1 : s0);
          tmem_st16(t_s + (uint32_t)(c >> 1), pk);
        }
        l += (s0.x + s0.y) + (s1.x + s1.y);
        return true;
      };
      const int steps = mine ? d.c1 - d.c0 : 0;
      for (int i = 0; i < steps; ++i) {
        const int nvalid = min(CH, d.len - (d.c0 + i) * CH);
        if (!wait(s_full + st, ns_all & 1u)) { ok = false; break; }
        ++ns_all;
        tc_fence_after();
        if (live) {
          if (!fast_step(i == 0, nvalid)) full_step(i, nvalid);
          tmem_wait_st();
        }                                        // (rows that do not exist: P is never used)
        tc_fence_before();
        arrive(p_full + st);
      }
      if (!ok) break;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegOther));
  }
  // The ring holds, for each chunk of a piece, K of each KV head of its item
  // and then V of each: a K slot is free again long before its V is.
  if (warp == 8) {
    // ---------------- MMAs (one thread) ----------------
    if (lane == 0) {
      constexpr uint32_t idesc_qk = umma_idesc_16(BF, 128, CH, false);
      constexpr uint32_t idesc_pv = umma_idesc_16(BF, 128, D, true);
      auto wait1 = [&](uint64_t* bar, uint32_t parity) -> bool {
        for (int i = 0; i < 64; ++i)
          if (mbar_try_wait(bar, parity)) return true;
        const bool done = mla_wait(bar, parity, p.status, p.wait_ns);
        if (!done) *failed = 1;
        return done;
      };
      uint32_t ring = 0;                         // ring position of the piece's first K
      uint32_t np[2] = {0, 0}, nq[2] = {0, 0};
      int g = g_first;
      bool ok = true;
      RaggedPiece w;
      for (int x = x0; ok && ragged_next(p, table, x1, g, x, w);) {
        const int nc = w.c1 - w.c0, parts = w.parts();
        // Ring position of stream st's K (its V: `heads` further) of chunk i;
        // whether the stream is the tile's last reader.
        auto k_at = [&](int st, int i) { return ring + (uint32_t)(2 * w.heads * i + (w.heads == 2 ? st : 0)); };
        auto last = [&](int st) { return w.heads == 2 || st == parts - 1; };
        auto qk = [&](int st, int i) -> bool {   // S of step i
          const uint32_t n = k_at(st, i), slot = n % NS;
          if (!wait1(full + slot, (n / NS) & 1u)) return false;
          tc_fence_after();
          const uint64_t qd = umma_desc_sw128(sbase + C::kOffQ + (uint32_t)st * C::kTile, 16, 1024);
          const uint64_t kd = umma_desc_sw128(sbase + C::kOffRing + slot * C::kTile, 16, 1024);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t o = (uint64_t)(((k >> 2) * 16384 + (k & 3) * 32) >> 4);
            umma_bf16(tmem + (uint32_t)(st * 128), qd + o, kd + o, idesc_qk, k > 0);
          }
          umma_commit(s_full + st);
          if (last(st)) umma_commit(empty + slot);
          return true;
        };
        auto pv = [&](int st, int i) -> bool {   // O += P.V of step i
          const uint32_t n = k_at(st, i) + (uint32_t)w.heads, slot = n % NS;
          if (!wait1(full + slot, (n / NS) & 1u) || !wait1(p_full + st, np[st]++ & 1u)) return false;
          tc_fence_after();
          const uint32_t ts = tmem + (uint32_t)(st * 128), to = tmem + 256u + (uint32_t)(st * D);
          const uint64_t vd = umma_desc_sw128(sbase + C::kOffRing + slot * C::kTile, 16384, 1024);
#pragma unroll
          for (int k = 0; k < CH / 16; ++k)
            umma_bf16_ts(to, ts + 8u * k, vd + (uint64_t)((k * 2048) >> 4), idesc_pv, i > 0 || k > 0);
          if (last(st)) umma_commit(empty + slot);
          if (i + 1 == nc) umma_commit(o_full + st);
          return true;
        };
        for (int st = 0; st < parts && ok; ++st) ok = wait1(q_full + st, nq[st]++ & 1u) && qk(st, 0);
        for (int i = 0; i < nc && ok; ++i)
          for (int st = 0; st < parts && ok; ++st) ok = pv(st, i) && (i + 1 >= nc || qk(st, i + 1));
        ring += (uint32_t)(2 * w.heads * nc);
      }
      // Nothing of this thread is in flight when tensor memory is freed.
      umma_commit(drain);
      wait1(drain, 0);
    }
    __syncwarp();
  } else if (warp == 10 || (warp == 9 && C::kTwoLoaders)) {
    // ---------------- TMA producer(s) ----------------
    // Two of them both walk the whole ring.  Neither can be two phases of a
    // slot's barrier ahead: the tile that it loaded last waited for one that is
    // consumed after those.
    if (!p.no_loads) {
      constexpr int N = F8 ? NR : NS;
      constexpr int PB = F8 ? 1 : C::kBlk;       // boxes per granule
      constexpr uint32_t kBox = F8 ? D : 128;    // bytes per key of a box
      constexpr uint32_t base = F8 ? C::kOffRaw : C::kOffRing, bytes = F8 ? C::kRaw : C::kTile;
      uint64_t* fb = F8 ? raw_full : full;
      uint64_t* eb = F8 ? raw_empty : empty;
      uint64_t policy;
      asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
      const int gr = lane / PB, blk = lane - gr * PB;   // this lane's box: granule and column block
      const int granules = CH / granule;
      uint32_t n = 0;
      int g = g_first;
      bool ok = true;
      RaggedPiece w;
      for (int x = x0; ok && ragged_next(p, table, x1, g, x, w);) {
        const int32_t* row = p.block_table + (int64_t)w.g * p.bt_stride;
        auto page_of = [&](int c) -> int {
          const int t = c * CH + gr * granule;
          int pg = 0;   // (volatile: loaded a chunk ahead of its use, not at it)
          if (gr < granules && c < w.c1 && t < w.len)
            asm volatile("ld.global.nc.b32 %0, [%1];" : "=r"(pg) : "l"(row + t / p.P));
          return pg;
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
          const int next = page_of(c + 1), off = t % p.P;
          for (int u = 0; u < 2 * w.heads; ++u, ++n) {   // K of each head, V of each head
            const uint32_t slot = n % N;
            const bool is_v = u >= w.heads;
            if (C::kTwoLoaders && is_v != (warp == 9)) continue;
            if (!wait(eb + slot, ((n / N) & 1u) ^ 1u)) { ok = false; break; }
            uint64_t* bar = !F8 && is_v && left < CH ? tail + slot : fb + slot;
            if (lane == 0) mbar_arrive_expect_tx(bar, tx);
            __syncwarp();
            if (load)
              tma_load_4d(smem + base + slot * bytes + (uint32_t)(blk * 16384 + gr * granule * (int)kBox),
                          is_v ? &tmap_v : &tmap_k, bar, blk * 64, off, w.h + (is_v ? u - w.heads : u), page, policy);
          }
          page = next;
        }
      }
    }
  } else if (warp == 11) {
    // ---------------- last V tile of a sequence: zero the rows behind it ----------------
    if (!F8) {
      uint32_t ring = 0, seen = 0;               // seen: bit s = parity of tail[s]
      int g = g_first;
      bool ok = true;
      RaggedPiece w;
      for (int x = x0; ok && ragged_next(p, table, x1, g, x, w);) {
        const int nc = w.c1 - w.c0;
        const int nvalid = w.len - (w.c1 - 1) * CH;
        ring += (uint32_t)(2 * w.heads * nc);
        if (nvalid >= CH) continue;
        const int per = (CH - nvalid) * 8;       // 16-byte pieces of a column block
        for (int h = w.heads; h > 0 && ok; --h) {
          const uint32_t slot = (ring - (uint32_t)h) % NS;
          if (!(ok = wait(tail + slot, (seen >> slot) & 1u))) break;
          seen ^= 1u << slot;
          for (int i = lane; i < per * C::kBlk; i += 32) {
            const int b = i / per, rest = i - b * per;
            sts128(sbase + C::kOffRing + slot * C::kTile + (uint32_t)(b * 16384 + nvalid * 128 + rest * 16),
                   make_uint4(0, 0, 0, 0));
          }
          fence_async_smem();
          arrive(full + slot);
        }
      }
    }
  } else if (F8 && warp >= 12) {
    // ---------------- e4m3 -> fp16 ----------------
    constexpr int LPK = D / 16;                  // lanes per key, 16 values each
    constexpr uint32_t kNr = NR > 0 ? NR : 1;
    const int ct = threadIdx.x - 384;
    const int c = ct % LPK;
    uint32_t n = 0;
    int g = g_first;
    bool ok = true;
    RaggedPiece w;
    for (int x = x0; ok && ragged_next(p, table, x1, g, x, w);) {
      for (int ch = w.c0; ch < w.c1 && ok; ++ch) {
        const int nvalid = min(CH, w.len - ch * CH);
        for (int u = 0; u < 2 * w.heads; ++u, ++n) {
          const uint32_t rs = n % kNr, slot = n % NS;
          if (!wait(raw_full + rs, (n / kNr) & 1u) || !wait(empty + slot, ((n / NS) & 1u) ^ 1u)) {
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
          fence_async_smem();
          arrive(raw_empty + rs);
          if (lane == 0) mbar_arrive(full + slot);
        }
      }
    }
  }
  if (p.own_o != nullptr) griddep_wait();
  tc_fence_before();
  __syncthreads();
  if (*failed) {
    // Every copy of a block that came through has been consumed; of one that
    // gave up, those in flight land now.
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {}
  }
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

}  // namespace b2d
