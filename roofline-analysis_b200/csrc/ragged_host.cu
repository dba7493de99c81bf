// ragged_host.cu — host side of cross attention and shared-prefix decode:
// argument checks, the choice of kernel, workspace layout and launches.
#include <algorithm>

#include "b2d_decode.h"
#include "host_common.h"
#include "ragged.cuh"
#include "ragged_mma_kernel.cuh"
#include "ragged_tc_kernel.cuh"

namespace b2d {

// Groups per launch: the chunk table of all of them sits in shared memory
// (16 KB).  Cross attention runs longer lists in slices.
constexpr int kMaxGroups = 4096;

struct RaggedPlan {
  bool tc;       // tcgen05 kernel; else warp-level tiles
  int granule;   // tc: keys per TMA box
  int TS, CH, rows, ctas;
  size_t smem;
  size_t off_cuts, off_seg_lse, off_seg_o, bytes;  // offsets from the plan's part of the workspace
};

static int check_sizes(const b2d_cross_args* a) {
  if (a == nullptr) return B2D_ERR_INVALID_ARG;
  if (a->num_tokens < 0 || a->num_groups < 0 || a->query_len < 0 || a->num_q_heads <= 0 ||
      a->num_kv_heads <= 0 || a->page_size <= 0 || a->max_pages_per_seq <= 0)
    return B2D_ERR_INVALID_ARG;
  if (a->num_q_heads % a->num_kv_heads != 0) return B2D_ERR_INVALID_ARG;
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 192 && a->head_dim != 256)
    return B2D_ERR_UNSUPPORTED;
  if (a->q_dtype != B2D_BF16 && a->q_dtype != B2D_FP16) return B2D_ERR_UNSUPPORTED;
  if (a->kv_dtype != a->q_dtype && a->kv_dtype != B2D_FP8_E4M3) return B2D_ERR_UNSUPPORTED;
  if (a->num_q_heads / a->num_kv_heads > 32) return B2D_ERR_UNSUPPORTED;
  if (a->page_size > (1 << 24)) return B2D_ERR_TOO_LARGE;
  // (a chunk's last position stays a 32-bit number)
  if ((int64_t)a->max_pages_per_seq * a->page_size > (int64_t)INT32_MAX - 256) return B2D_ERR_TOO_LARGE;
  if (a->wait_limit_us < 0 || (a->flags & ~B2D_FLAG_TEST_NO_LOADS)) return B2D_ERR_INVALID_ARG;
  if (a->kv_layout != B2D_KV_STRIDED && a->kv_layout != B2D_KV_VLLM) return B2D_ERR_INVALID_ARG;
  if (a->kv_layout == B2D_KV_VLLM && (a->kv_dtype == B2D_FP8_E4M3 || a->page_size % 16 != 0))
    return B2D_ERR_UNSUPPORTED;
  return B2D_OK;
}

static int check_pointers(const b2d_cross_args* a) {
  if (!a->q || !a->k_cache || !a->v_cache || !a->kv_lens || !a->block_table || !a->out)
    return B2D_ERR_INVALID_ARG;
  if (a->num_pages <= 0 || a->num_pages > (int64_t)INT32_MAX) return B2D_ERR_INVALID_ARG;
  if (!a->query_starts && (int64_t)a->num_groups * a->query_len != a->num_tokens)
    return B2D_ERR_INVALID_ARG;
  const int es = a->kv_dtype == B2D_FP8_E4M3 ? 1 : 2;
  if (((uintptr_t)a->k_cache & 15) || ((uintptr_t)a->v_cache & 15) || ((uintptr_t)a->q & 15) ||
      ((uintptr_t)a->out & 15))
    return B2D_ERR_ALIGNMENT;
  const int64_t strides[6] = {a->k_stride_page, a->k_stride_tok, a->k_stride_head,
                              a->v_stride_page, a->v_stride_tok, a->v_stride_head};
  for (int i = 0; i < 6; ++i) {
    if (a->kv_layout == B2D_KV_VLLM && (i == 1 || i == 4)) continue;  // token strides implied
    if (strides[i] <= 0 || (strides[i] * es) % 16 != 0) return B2D_ERR_ALIGNMENT;
  }
  if ((a->q_stride_t * 2) % 16 || (a->q_stride_h * 2) % 16 || (a->out_stride_t * 2) % 16 ||
      (a->out_stride_h * 2) % 16)
    return B2D_ERR_ALIGNMENT;
  return B2D_OK;
}

static int make_plan(const b2d_cross_args* a, RaggedPlan* pl) {
  const int grp = a->num_q_heads / a->num_kv_heads;
  const int groups = std::min(a->num_groups, kMaxGroups);
  pl->tc = (a->head_dim == 64 || a->head_dim == 128) && a->page_size % 16 == 0 &&
           a->kv_layout == B2D_KV_STRIDED;
  if (pl->tc) {
    pl->granule = 16;   // the largest power of two up to 128 that divides a page
    while (pl->granule < 128 && a->page_size % (2 * pl->granule) == 0) pl->granule *= 2;
    pl->rows = 256;
    pl->CH = 128;
    pl->TS = 128 / grp;
  } else {
    pl->rows = 64;
    pl->CH = a->head_dim <= 128 ? 64 : 32;
    pl->TS = pl->rows / grp;
    pl->smem = (size_t)(pl->rows + 2 * pl->CH) * (a->head_dim + 8) * 2 + ragged_table_bytes(groups);
  }
  pl->ctas = a->num_ctas;
  if (pl->ctas <= 0) {
    int sms = 0;
    if (device_sm_count(&sms) != 0) return B2D_ERR_CUDA;
    pl->ctas = pl->tc ? sms : 2 * sms;
  }
  // Positions on the chunk line are 32-bit in the kernels.
  const int64_t chunks = ((int64_t)a->max_pages_per_seq * a->page_size + pl->CH - 1) / pl->CH + kItemCost;
  const int64_t tiles = (int64_t)a->num_tokens / pl->TS + groups;
  if (tiles * a->num_kv_heads > (int64_t)INT32_MAX / chunks) return B2D_ERR_TOO_LARGE;
  const size_t seg_rows = (size_t)2 * pl->ctas * pl->rows;
  pl->off_cuts = 0;
  pl->off_seg_lse = align_up((size_t)pl->ctas * 32, 256);
  pl->off_seg_o = align_up(pl->off_seg_lse + seg_rows * 4, 256);
  pl->bytes = align_up(pl->off_seg_o + seg_rows * a->head_dim * 4, 256);
  return B2D_OK;
}

static RaggedParams params_of(const b2d_cross_args* a, const RaggedPlan& pl, uint8_t* part) {
  RaggedParams p{};
  p.q = a->q;
  p.q_st = a->q_stride_t;
  p.q_sh = a->q_stride_h;
  p.kc = a->k_cache;
  p.vc = a->v_cache;
  p.k_sp = a->k_stride_page;
  p.k_st = a->k_stride_tok;
  p.k_sh = a->k_stride_head;
  p.v_sp = a->v_stride_page;
  p.v_st = a->v_stride_tok;
  p.v_sh = a->v_stride_head;
  p.k_sg = 8;
  p.v_sd = 1;
  if (a->kv_layout == B2D_KV_VLLM) {  // K [blocks, Hkv, D/8, P, 8], V [blocks, Hkv, D, P]
    p.k_st = 8;
    p.k_sg = (int64_t)a->page_size * 8;
    p.v_st = 1;
    p.v_sd = a->page_size;
  }
  p.starts = a->query_starts;
  p.kv_lens = a->kv_lens;
  p.block_table = a->block_table;
  p.bt_stride = a->block_table_stride;
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.out = a->out;
  p.o_st = a->out_stride_t;
  p.o_sh = a->out_stride_h;
  p.lse = a->lse;
  p.lse_st = a->lse_stride_t;
  p.cuts = reinterpret_cast<int32_t*>(part + pl.off_cuts);
  p.seg_lse = reinterpret_cast<float*>(part + pl.off_seg_lse);
  p.seg_o = reinterpret_cast<float*>(part + pl.off_seg_o);
  p.status = static_cast<int*>(a->workspace);
  p.wait_ns = a->wait_limit_us > 0 ? (unsigned long long)a->wait_limit_us * 1000ull : kWaitLimitNs;
  p.no_loads = (a->flags & B2D_FLAG_TEST_NO_LOADS) ? 1 : 0;
  p.G = a->num_groups;
  p.T = a->num_tokens;
  p.uniform = a->query_len;
  p.Hq = a->num_q_heads;
  p.Hkv = a->num_kv_heads;
  p.grp = a->num_q_heads / a->num_kv_heads;
  p.P = a->page_size;
  p.num_pages = (int)a->num_pages;
  p.max_pages = a->max_pages_per_seq;
  p.TS = pl.TS;
  p.CH = pl.CH;
  p.rows = pl.rows;
  p.pairs = pl.tc ? 1 : 0;
  p.spread = (int64_t)a->num_tokens / pl.TS * a->num_kv_heads >> p.pairs >= 2 * (int64_t)pl.ctas;
  p.scale = a->softmax_scale * 1.4426950408889634f;
  return p;
}

// Launch whose start may overlap the kernel before it on the stream (the kernel
// itself waits for that one's end before it reads what it wrote).
template <typename... P, typename... A>
static int launch_overlapped(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                             A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess && cudaGetLastError() == cudaSuccess
             ? B2D_OK : B2D_ERR_CUDA;
}

template <int D, int KIND, typename QT>
static int launch_mma(const RaggedPlan& pl, const RaggedParams& p, cudaStream_t st) {
  auto kern = ragged_mma_kernel<D, KIND, QT>;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), pl.smem)) return B2D_ERR_CUDA;
  return launch_overlapped(kern, dim3(pl.ctas), 128, pl.smem, st, p);
}

// {column, key of the page, head, page}: a box is `granule` keys of 128 bytes
// (one column block, 128-byte swizzle), or of a whole e4m3 row (no swizzle;
// the conversion writes the swizzled tile).
static int encode_cache(CUtensorMap* map, const void* base, const b2d_cross_args* a, int granule,
                        int64_t s_page, int64_t s_tok, int64_t s_head) {
  const bool f8 = a->kv_dtype == B2D_FP8_E4M3;
  const uint64_t es = f8 ? 1 : 2;
  const uint64_t dims[4] = {(uint64_t)a->head_dim, (uint64_t)a->page_size, (uint64_t)a->num_kv_heads,
                            (uint64_t)a->num_pages};
  const uint64_t strides[3] = {(uint64_t)s_tok * es, (uint64_t)s_head * es, (uint64_t)s_page * es};
  const uint32_t box[4] = {f8 ? (uint32_t)a->head_dim : 64u, (uint32_t)granule, 1u, 1u};
  return encode_tiled_map(map, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 4,
                          base, dims, strides, box,
                          f8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, int KIND, typename QT>
static int launch_tc(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                     cudaStream_t st) {
  using C = RaggedTc<D, KIND>;
  CUtensorMap tk, tv;
  if (encode_cache(&tk, a->k_cache, a, pl.granule, a->k_stride_page, a->k_stride_tok, a->k_stride_head) ||
      encode_cache(&tv, a->v_cache, a, pl.granule, a->v_stride_page, a->v_stride_tok, a->v_stride_head))
    return B2D_ERR_CUDA;
  auto kern = ragged_tc_kernel<D, KIND, QT>;
  const size_t smem = C::smem(p.G);
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(kern), smem)) return B2D_ERR_CUDA;
  return launch_overlapped(kern, dim3(pl.ctas), C::kThreads, smem, st, tk, tv, p, pl.granule);
}

template <int D, int KIND, typename QT>
static int launch_one(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                      cudaStream_t st) {
  if constexpr (D <= 128) {
    if (pl.tc) return launch_tc<D, KIND, QT>(a, pl, p, st);
  }
  return launch_mma<D, KIND, QT>(pl, p, st);
}

template <int D>
static int launch_attention(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                            cudaStream_t st) {
  const bool bf = a->q_dtype == B2D_BF16;
  if (a->kv_dtype == B2D_FP8_E4M3)
    return bf ? launch_one<D, kKvFp8, __nv_bfloat16>(a, pl, p, st)
              : launch_one<D, kKvFp8, __half>(a, pl, p, st);
  return bf ? launch_one<D, kKvBf16, __nv_bfloat16>(a, pl, p, st)
            : launch_one<D, kKvFp16, __half>(a, pl, p, st);
}

static int launch_attention(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                            cudaStream_t st) {
  switch (a->head_dim) {
    case 64: return launch_attention<64>(a, pl, p, st);
    case 128: return launch_attention<128>(a, pl, p, st);
    case 192: return launch_attention<192>(a, pl, p, st);
    default: return launch_attention<256>(a, pl, p, st);
  }
}

template <int D>
static int launch_merge(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                        cudaStream_t st) {
  if (pl.ctas < 2) return B2D_OK;
  const dim3 grid(pl.ctas - 1, (unsigned)((pl.rows + 15) / 16));
  return a->q_dtype == B2D_BF16
             ? launch_overlapped(ragged_merge_kernel<D, __nv_bfloat16>, grid, 256, 0, st, p)
             : launch_overlapped(ragged_merge_kernel<D, __half>, grid, 256, 0, st, p);
}

// The attention kernel and the merge of the items that its ranges cut.
static int launch_both(const b2d_cross_args* a, const RaggedPlan& pl, const RaggedParams& p,
                       cudaStream_t st) {
  const int rc = launch_attention(a, pl, p, st);
  if (rc) return rc;
  switch (a->head_dim) {
    case 64: return launch_merge<64>(a, pl, p, st);
    case 128: return launch_merge<128>(a, pl, p, st);
    case 192: return launch_merge<192>(a, pl, p, st);
    default: return launch_merge<256>(a, pl, p, st);
  }
}

// The prefix half of a shared-prefix decode as a ragged problem: the
// sequences of a group are the tokens that read its prefix.
static b2d_cross_args prefix_of(const b2d_shared_prefix_args* a) {
  const b2d_gqa_args& o = a->own;
  b2d_cross_args c{};
  c.q = o.q;
  c.q_stride_t = o.q_stride_b;
  c.q_stride_h = o.q_stride_h;
  c.k_cache = o.k_cache;
  c.v_cache = o.v_cache;
  c.k_stride_page = o.k_stride_page;
  c.k_stride_tok = o.k_stride_tok;
  c.k_stride_head = o.k_stride_head;
  c.v_stride_page = o.v_stride_page;
  c.v_stride_tok = o.v_stride_tok;
  c.v_stride_head = o.v_stride_head;
  c.num_pages = o.num_pages;
  c.query_starts = a->group_starts;
  c.kv_lens = a->prefix_lens;
  c.block_table = a->prefix_block_table;
  c.block_table_stride = a->prefix_block_table_stride;
  c.k_scale = o.k_scale;
  c.v_scale = o.v_scale;
  c.out = o.out;
  c.out_stride_t = o.out_stride_b;
  c.out_stride_h = o.out_stride_h;
  c.lse = o.lse;
  c.lse_stride_t = o.lse_stride_b;
  c.num_tokens = o.batch;
  c.num_groups = a->num_groups;
  c.query_len = o.batch;
  c.num_q_heads = o.num_q_heads;
  c.num_kv_heads = o.num_kv_heads;
  c.head_dim = o.head_dim;
  c.page_size = o.page_size;
  c.max_pages_per_seq = a->prefix_max_pages;
  c.q_dtype = o.q_dtype;
  c.kv_dtype = o.kv_dtype;
  c.softmax_scale = o.softmax_scale;
  c.workspace = o.workspace;
  c.workspace_bytes = o.workspace_bytes;
  c.num_ctas = o.num_ctas;
  c.flags = o.flags & B2D_FLAG_TEST_NO_LOADS;
  c.kv_layout = o.kv_layout;
  c.wait_limit_us = o.wait_limit_us;
  return c;
}

struct SharedLayout {
  size_t gqa, off_part, off_own_o, off_own_lse, bytes;
};

static int shared_layout(const b2d_shared_prefix_args* a, const b2d_cross_args* c,
                         RaggedPlan* pl, SharedLayout* lay) {
  int rc = b2d_gqa_workspace_bytes(&a->own, &lay->gqa);
  if (rc) return rc;
  if (a->num_groups > kMaxGroups) return B2D_ERR_TOO_LARGE;
  if ((rc = check_sizes(c)) || (rc = make_plan(c, pl))) return rc;
  const size_t rows = (size_t)a->own.batch * a->own.num_q_heads;
  lay->off_part = align_up(lay->gqa, 256);
  lay->off_own_lse = align_up(lay->off_part + pl->bytes, 256);
  lay->off_own_o = align_up(lay->off_own_lse + rows * 4, 256);
  lay->bytes = align_up(lay->off_own_o + rows * a->own.head_dim * 4, 256);
  return B2D_OK;
}

}  // namespace b2d

using namespace b2d;

extern "C" int b2d_cross_workspace_bytes(const b2d_cross_args* a, size_t* bytes) {
  int rc = check_sizes(a);
  if (rc) return rc;
  if (!bytes) return B2D_ERR_INVALID_ARG;
  RaggedPlan pl{};
  if ((rc = make_plan(a, &pl))) return rc;
  *bytes = kWsHeaderBytes + pl.bytes;
  return B2D_OK;
}

extern "C" int b2d_cross_attention(const b2d_cross_args* a, void* stream) {
  int rc = check_sizes(a);
  if (rc) return rc;
  if (a->num_tokens == 0 || a->num_groups == 0) return B2D_OK;
  RaggedPlan pl{};
  if ((rc = make_plan(a, &pl))) return rc;
  if ((rc = check_pointers(a))) return rc;
  if (!a->workspace || a->workspace_bytes < kWsHeaderBytes + pl.bytes) return B2D_ERR_WORKSPACE;
  if ((uintptr_t)a->workspace & 255) return B2D_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* part = static_cast<uint8_t*>(a->workspace) + kWsHeaderBytes;
  for (int g0 = 0; g0 < a->num_groups; g0 += kMaxGroups) {
    b2d_cross_args s = *a;
    s.num_groups = std::min(a->num_groups - g0, kMaxGroups);
    s.kv_lens = a->kv_lens + g0;
    s.block_table = a->block_table + (int64_t)g0 * a->block_table_stride;
    if (a->query_starts) {
      s.query_starts = a->query_starts + g0;
    } else {
      const int64_t t0 = (int64_t)g0 * a->query_len;
      s.q = static_cast<const uint8_t*>(a->q) + t0 * a->q_stride_t * 2;
      s.out = static_cast<uint8_t*>(a->out) + t0 * a->out_stride_t * 2;
      s.lse = a->lse ? a->lse + t0 * a->lse_stride_t : nullptr;
      s.num_tokens = s.num_groups * a->query_len;
    }
    const RaggedParams p = params_of(&s, pl, part);
    if ((rc = launch_both(&s, pl, p, st))) return rc;
  }
  return B2D_OK;
}

extern "C" int b2d_shared_prefix_workspace_bytes(const b2d_shared_prefix_args* a, size_t* bytes) {
  if (!a || !bytes || a->num_groups < 0 || a->prefix_max_pages <= 0) return B2D_ERR_INVALID_ARG;
  const b2d_cross_args c = prefix_of(a);
  RaggedPlan pl{};
  SharedLayout lay{};
  const int rc = shared_layout(a, &c, &pl, &lay);
  if (rc) return rc;
  *bytes = lay.bytes;
  return B2D_OK;
}

extern "C" int b2d_decode_shared_prefix(const b2d_shared_prefix_args* a, void* stream) {
  if (!a || a->num_groups < 0 || a->prefix_max_pages <= 0) return B2D_ERR_INVALID_ARG;
  if (a->own.flags & ~B2D_FLAG_TEST_NO_LOADS) return B2D_ERR_INVALID_ARG;
  if (!a->group_starts && a->num_groups > 1) return B2D_ERR_INVALID_ARG;
  const b2d_cross_args c = prefix_of(a);
  RaggedPlan pl{};
  SharedLayout lay{};
  int rc = shared_layout(a, &c, &pl, &lay);
  if (rc) return rc;
  if (a->own.batch == 0) return B2D_OK;
  if (a->num_groups == 0) return b2d_decode_gqa(&a->own, stream);
  if ((rc = check_pointers(&c))) return rc;
  if (!a->own.workspace || a->own.workspace_bytes < lay.bytes) return B2D_ERR_WORKSPACE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(a->own.workspace);
  float* own_o = reinterpret_cast<float*>(ws + lay.off_own_o);
  float* own_lse = reinterpret_cast<float*>(ws + lay.off_own_lse);
  // Own tokens first: that call checks the rest of the arguments before it
  // enqueues anything.  Its part stays in fp32; the prefix kernel joins the two
  // and rounds once.
  b2d_gqa_args own = a->own;
  own.out = own_o;
  own.out_stride_b = (int64_t)own.num_q_heads * own.head_dim;
  own.out_stride_h = own.head_dim;
  own.lse = own_lse;
  own.lse_stride_b = own.num_q_heads;
  own.workspace_bytes = lay.gqa;
  if ((rc = gqa_decode_f32(&own, own_o, stream))) return rc;
  RaggedParams p = params_of(&c, pl, ws + lay.off_part);
  p.own_o = own_o;
  p.own_lse = own_lse;
  // (a wait with a short limit must not run while the own-token decode does)
  p.beside = p.wait_ns >= kWaitLimitNs;
  return launch_both(&c, pl, p, st);
}
