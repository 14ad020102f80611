// C ABI for the paged verification attention over INT8 caches with per-token scales and over int8 /
// e4m3 caches with block scales: validation, grid, workspace and launch.
#include <algorithm>
#include <atomic>

#include "api_common.hpp"
#include "paged_attn_block.hpp"

namespace specq {

// Workgroups the split length aims at (0 = the device's CUs), set through
// specq_set_option("attn_target_wgs", v); eager and plan-mode calls that are compared bit for
// bit must run with the same value.
std::atomic<int> g_attn_target{0};

const void* attn_plan_fn_d64(int rb_max, int fp32);   // attn_plan_d64.hip
const void* attn_plan_fn_d128(int rb_max, int fp32);  // attn_plan_d128.hip
const void* attn_block_fn_d64(int rb, int f8, int plan);   // attn_block_d64.hip
const void* attn_block_fn_d128(int rb, int f8, int plan);  // attn_block_d128.hip
const void* attn_merge_fn_d64();
const void* attn_merge_fn_d128();

namespace {

template <int D>
const void* attn_fn_d(int rb, int fp32) {
  switch (rb * 2 + fp32) {
    case 2: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 1, _Float16>);
    case 3: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 1, float>);
    case 4: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 2, _Float16>);
    case 5: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 2, float>);
    case 6: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 3, _Float16>);
    case 7: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 3, float>);
    case 8: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 4, _Float16>);
    case 9: return reinterpret_cast<const void*>(&paged_attn_kernel<D, 4, float>);
  }
  return nullptr;
}

// Cache kinds: per-token fp16 / fp32 scales on int8, block scales on int8 / e4m3.
enum { kTokF16 = 0, kTokF32 = 1, kBlkI8 = 2, kBlkF8 = 3 };

// The eager kernel of rb row blocks, or (plan) the one that takes its row blocks from the active q_len.
const void* attn_fn(int D, int rb, int kind, bool plan) {
  if (D != 64 && D != 128) return nullptr;
  if (kind >= kBlkI8) return D == 128 ? attn_block_fn_d128(rb, kind - kBlkI8, plan) : attn_block_fn_d64(rb, kind - kBlkI8, plan);
  if (plan) return D == 128 ? attn_plan_fn_d128(rb, kind) : attn_plan_fn_d64(rb, kind);
  return D == 128 ? attn_fn_d<128>(rb, kind) : attn_fn_d<64>(rb, kind);
}

// grid.x: the splits of a block table of max_pages * PAGE tokens when at least `pairs_min`
// (sequence, KV head) pairs are active (fewer pairs never means fewer splits).
int n_splits_for(bool blk, int max_pages, int PAGE, int pairs_min, int target) {
  const int cap = max_pages * PAGE;
  const int per = blk ? kBlkUnit * blk_split_units(cap, pairs_min, target) : kAttnUnit * attn_split_units(cap, pairs_min, target);
  return std::max(1, ceil_div(cap, per));
}

// Splits, and the one-dimensional grid of program x split (the kernel derives both from the active count): the
// exact count for an eager call, the most any active count needs in plan mode.
struct AttnGrid {
  int ns;
  int64_t wgs;
};
AttnGrid attn_grid(bool blk, bool plan, int B_grid, int n_seqs, int q_len, int n_qc, int H_KV, int G, int max_pages,
                   int PAGE, int target) {
  // Eager calls know the active sequences; a plan may activate as few as one.
  const int ns = n_splits_for(blk, max_pages, PAGE,
                              plan ? H_KV : std::max(n_seqs, 1) * H_KV * attn_row_programs(q_len, G), target);
  int64_t wgs = (int64_t)n_seqs * H_KV * n_qc * ns;
  if (plan) {
    // Active query tokens that fill one program cut a sequence finest; past that the cut gets coarser.
    wgs = 0;
    for (int s = 1; s <= B_grid; ++s)
      wgs = std::max(wgs, (int64_t)s * H_KV * n_qc * n_splits_for(blk, max_pages, PAGE, s * H_KV, target));
  }
  return {ns, wgs};
}

}  // namespace

// `variant` is the head dim, | kAttrsScaleFp32 for fp32 K/V scales, | kAttrsBlockI8 / kAttrsBlockF8 for
// block-scaled caches.
int attn_attrs(int variant, int rows, specq_kernel_attrs* out) {
  const int kind = (variant & kAttrsBlockI8) ? kBlkI8 : (variant & kAttrsBlockF8) ? kBlkF8
                   : (variant & kAttrsScaleFp32) ? kTokF32 : kTokF16;
  const int D = variant & ~(kAttrsScaleFp32 | kAttrsBlockI8 | kAttrsBlockF8);
  SPECQ_REQUIRE(rows >= 1 && rows <= 64, SPECQ_ENOTSUP, "paged_attn: %d packed rows (1..64 supported)", rows);
  const int rb = ceil_div(rows, 16);
  const void* fn = attn_fn(D, rb, kind, false);
  SPECQ_REQUIRE(fn != nullptr, SPECQ_ENOTSUP, "paged_attn: head_dim %d not supported", D);
  hipFuncAttributes fa;
  if (hipFuncGetAttributes(&fa, fn) != hipSuccess) return fail(SPECQ_EIO, "paged_attn: hipFuncGetAttributes failed");
  static const char* const kNames[] = {"paged_attn_kernel<%d, %d, _Float16>", "paged_attn_kernel<%d, %d, float>",
                                       "attn_block_kernel<%d, %d, false>", "attn_block_kernel<%d, %d, true>"};
  // The name carries the template arguments exactly as profilers print the kernel symbol.
  char name[64];
  snprintf(name, sizeof(name), kNames[kind], D, rb);
  snprintf(out->name, sizeof(out->name), "specq::%s", name);
  out->num_regs = fa.numRegs;
  out->lds_bytes = (int)fa.sharedSizeBytes;
  out->scratch_bytes = (int)fa.localSizeBytes;
  out->threads = kAttnThreads;
  out->block_m = rb * 16;
  return SPECQ_OK;
}

}  // namespace specq

using namespace specq;

extern "C" size_t specq_paged_attn_workspace_size(int B_grid, int H, int H_KV, int ql_grid, int QPP, int max_pages,
                                                  int PAGE) {
  if (B_grid <= 0 || H_KV <= 0 || H % H_KV != 0 || QPP <= 0 || ql_grid <= 0 || max_pages <= 0 || PAGE <= 0) return 0;
  const int G = H / H_KV;
  const int rows = ceil_div(QPP * G, 16) * 16;
  const int n_qc = ceil_div(ql_grid, QPP);
  const int64_t progs = (int64_t)B_grid * H_KV * n_qc;
  if ((int64_t)max_pages * PAGE > kAttnMaxTokens) return 0;
  // Plan-mode bound: at least one active sequence.
  const int tgt = g_attn_target.load();
  const int ns = n_splits_for(false, max_pages, PAGE, H_KV, tgt > 0 ? tgt : device_cus());
  if (ns <= 1) return 0;
  // Sized for D = 128 (the largest supported head dimension).
  const size_t part = (size_t)progs * ns * rows * (128 + 2) * 4;
  return kCounterBytes + align_up(part, 256);
}

static size_t attn_block_bytes(const AttnGrid& g, int rows, int D) {
  return g.ns <= 1 || g.wgs == 0 ? 0 : kCounterBytes + align_up((size_t)g.wgs * rows * (D + 2) * 4, 256);
}

extern "C" size_t specq_paged_attn_block_workspace_size(int B_grid, int H, int H_KV, int ql_grid, int QPP, int D,
                                                        int max_pages, int PAGE, int plan) {
  if (B_grid <= 0 || H_KV <= 0 || H % H_KV != 0 || QPP <= 0 || ql_grid <= 0 || max_pages <= 0 || PAGE <= 0) return 0;
  const int G = H / H_KV, tgt = g_attn_target.load();
  if ((int64_t)max_pages * PAGE > kBlkMaxTokens || (int64_t)QPP * G > 64) return 0;
  return attn_block_bytes(attn_grid(true, plan != 0, B_grid, B_grid, ql_grid, ceil_div(ql_grid, QPP), H_KV, G, max_pages,
                                    PAGE, tgt > 0 ? tgt : device_cus()),
                          ceil_div(QPP * G, 16) * 16, D);
}

// Both entry points: `kind` is the cache's, `sb` its tokens per scale block (block scales only).
static int attn_call(int kind, const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const void* kc, const void* vc,
                     int64_t s_kp, int64_t s_ko, int64_t s_kh, const void* ks, const void* vs, int64_t s_sp,
                     int64_t s_so, int64_t s_sh, int sb, const int32_t* block_tbl, int64_t s_bt, int max_pages,
                     int n_pages, const int32_t* ctx_len, void* out, int64_t s_ob, int64_t s_ot, int64_t s_oh,
                     int B_grid, int n_seqs, int q_len, int ql_grid, int H, int H_KV, int D, int PAGE, int QPP,
                     float sm_scale, const int32_t* plan, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  SPECQ_REQUIRE(q && kc && vc && ks && vs && block_tbl && ctx_len && out, SPECQ_EINVAL,
                "paged_attn: null tensor pointer");
  SPECQ_REQUIRE(B_grid >= 0 && ql_grid > 0 && H > 0 && H_KV > 0 && H % H_KV == 0, SPECQ_EINVAL,
                "paged_attn: bad sizes B=%d ql=%d H=%d H_KV=%d", B_grid, ql_grid, H, H_KV);
  SPECQ_REQUIRE(D == 64 || D == 128, SPECQ_ENOTSUP, "paged_attn: head_dim %d (64 or 128 supported)", D);
  SPECQ_REQUIRE(PAGE > 0 && PAGE % 16 == 0, SPECQ_ENOTSUP, "paged_attn: PAGE=%d must be a multiple of 16", PAGE);
  SPECQ_REQUIRE(max_pages > 0, SPECQ_EINVAL, "paged_attn: empty block table");
  SPECQ_REQUIRE(n_pages > 0, SPECQ_EINVAL, "paged_attn: empty K/V pool (n_pages=%d)", n_pages);
  const bool blk = kind >= kBlkI8;
  const int64_t most = blk ? kBlkMaxTokens : kAttnMaxTokens;
  SPECQ_REQUIRE((int64_t)max_pages * PAGE <= most, SPECQ_ENOTSUP, "paged_attn: block table of %lld tokens exceeds %lld",
                (long long)max_pages * PAGE, (long long)most);
  SPECQ_REQUIRE(QPP > 0, SPECQ_EINVAL, "paged_attn: QPP=%d", QPP);
  const int G = H / H_KV;
  SPECQ_REQUIRE((int64_t)QPP * G <= 64, SPECQ_ENOTSUP, "paged_attn: QPP*G=%lld packed rows exceed 64",
                (long long)QPP * G);
  if (plan == nullptr) {
    SPECQ_REQUIRE(n_seqs >= 0 && n_seqs <= B_grid && q_len >= 0 && q_len <= ql_grid, SPECQ_EINVAL,
                  "paged_attn: n_seqs=%d q_len=%d outside the grid (%d, %d)", n_seqs, q_len, B_grid, ql_grid);
  }
  SPECQ_REQUIRE((uintptr_t)q % 16 == 0 && s_qb % 8 == 0 && s_qt % 8 == 0 && s_qh % 8 == 0, SPECQ_ENOTSUP,
                "paged_attn: q rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)out % 16 == 0 && s_ob % 8 == 0 && s_ot % 8 == 0 && s_oh % 8 == 0, SPECQ_ENOTSUP,
                "paged_attn: out rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)kc % 16 == 0 && (uintptr_t)vc % 16 == 0 && s_kp % 16 == 0 && s_ko % 16 == 0 &&
                    s_kh % 16 == 0,
                SPECQ_ENOTSUP, "paged_attn: K/V cache rows must be 16-byte aligned");
  SPECQ_REQUIRE(!blk || s_ko >= D, SPECQ_ENOTSUP, "paged_attn: rows of the K/V cache overlap (token stride %lld)",
                (long long)s_ko);
  SPECQ_REQUIRE(!blk || (lie_apart(plan ? B_grid : n_seqs, s_ob, D) && lie_apart(plan ? ql_grid : q_len, s_ot, D) &&
                         lie_apart(H, s_oh, D)),
                SPECQ_ENOTSUP, "paged_attn: rows of the output overlap");
  SPECQ_REQUIRE(s_ko > 0 && 16 * s_ko + D < ((int64_t)1 << 31), SPECQ_ENOTSUP,
                "paged_attn: token stride %lld of the K/V cache outside (0, 2^27)", (long long)s_ko);
  if (B_grid == 0) return SPECQ_OK;
  const int rb = ceil_div(QPP * G, 16);
  // Plan mode with more than one row block runs the launch that sizes its programs to the
  // active q_len on the device (the rows of a program whose queries are inactive do nothing).
  const void* fn = attn_fn(D, rb, kind, plan != nullptr && rb > 1);
  SPECQ_REQUIRE(fn != nullptr, SPECQ_ENOTSUP, "paged_attn: no kernel for D=%d rows=%d", D, QPP * G);
  const int n_qc = ceil_div(plan ? ql_grid : q_len, QPP);
  if (n_qc == 0) return SPECQ_OK;
  const int target = g_attn_target.load() > 0 ? g_attn_target.load() : device_cus();
  const AttnGrid grid = attn_grid(blk, plan != nullptr, B_grid, n_seqs, q_len, n_qc, H_KV, G, max_pages, PAGE, target);
  const int ns = grid.ns;
  const int64_t progs = (int64_t)B_grid * H_KV * n_qc;
  const bool defer = blk && (ns > kBlkMergeIn || (ns > 1 && progs > kMaxCounters));
  const int rows = rb * 16;
  size_t need = 0;
  if (ns > 1) {
    SPECQ_REQUIRE(defer || progs <= kMaxCounters, SPECQ_ENOTSUP, "paged_attn: %lld programs exceed the counter region",
                  (long long)progs);
    need = blk ? attn_block_bytes(grid, rows, D)
               : kCounterBytes + align_up((size_t)progs * ns * rows * (D + 2) * 4, 256);
  }
  SPECQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), SPECQ_ENOSPC,
                "paged_attn: workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : 0);
  const int64_t wgs = grid.wgs;
  if (wgs == 0) return SPECQ_OK;
  SPECQ_REQUIRE(wgs <= INT32_MAX, SPECQ_ENOTSUP, "paged_attn: grid too large");
  AttnBlockParams p;  // the per-token kernels take its AttnParams
  p.q = (const _Float16*)q; p.s_qb = s_qb; p.s_qt = s_qt; p.s_qh = s_qh;
  p.kc = (const int8_t*)kc; p.vc = (const int8_t*)vc; p.s_kp = s_kp; p.s_ko = s_ko; p.s_kh = s_kh;
  p.ks = ks; p.vs = vs; p.s_sp = s_sp; p.s_so = s_so; p.s_sh = s_sh;
  p.bt = block_tbl; p.s_bt = s_bt; p.max_pages = max_pages; p.n_pages = n_pages; p.ctx_len = ctx_len;
  p.out = (_Float16*)out; p.s_ob = s_ob; p.s_ot = s_ot; p.s_oh = s_oh;
  p.plan = plan; p.B_grid = B_grid; p.n_seqs = plan ? B_grid : n_seqs; p.q_len = plan ? ql_grid : q_len;
  p.ql_grid = ql_grid; p.G = G; p.QPP = QPP; p.n_qc = n_qc; p.H_KV = H_KV; p.PAGE = PAGE; p.n_splits = ns;
  p.target_wgs = target;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.counters = need ? (int32_t*)workspace : nullptr;
  p.part = need ? (float*)((char*)workspace + kCounterBytes) : nullptr;
  p.sb = sb;
  p.defer = defer;
  p.n_part = wgs;
  diag_timeline(&p.tl, &p.tl_cap);
  void* args[] = {&p};
  hipError_t e = hipLaunchKernel(fn, dim3((unsigned)wgs), dim3(kAttnThreads), args, 0, (hipStream_t)stream);
  if (e != hipSuccess) {
    set_error("paged_attn: hipLaunchKernel failed: %s", hipGetErrorString(e));
    return SPECQ_EIO;
  }
  if (!defer) return SPECQ_OK;
  const int64_t merge = (int64_t)(plan ? B_grid : n_seqs) * H_KV * n_qc * QPP * G;
  SPECQ_REQUIRE(merge <= INT32_MAX, SPECQ_ENOTSUP, "paged_attn: grid too large");
  return launch(D == 128 ? attn_merge_fn_d128() : attn_merge_fn_d64(), (int)merge, 256, 0, (hipStream_t)stream, &p);
}

extern "C" int specq_paged_attn(const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const int8_t* kc,
                                const int8_t* vc, int64_t s_kp, int64_t s_ko, int64_t s_kh, const void* ks,
                                const void* vs, int64_t s_sp, int64_t s_so, int64_t s_sh, int scale_fp32,
                                const int32_t* block_tbl, int64_t s_bt, int max_pages, int n_pages,
                                const int32_t* ctx_len,
                                void* out, int64_t s_ob, int64_t s_ot, int64_t s_oh, int B_grid, int n_seqs,
                                int q_len, int ql_grid, int H, int H_KV, int D, int PAGE, int QPP, float sm_scale,
                                const int32_t* plan, void* workspace, size_t workspace_bytes, void* stream) {
  return attn_call(scale_fp32 ? kTokF32 : kTokF16, q, s_qb, s_qt, s_qh, kc, vc, s_kp, s_ko, s_kh, ks, vs, s_sp, s_so,
                   s_sh, 0, block_tbl, s_bt, max_pages, n_pages, ctx_len, out, s_ob, s_ot, s_oh, B_grid, n_seqs, q_len,
                   ql_grid, H, H_KV, D, PAGE, QPP, sm_scale, plan, workspace, workspace_bytes, stream);
}

extern "C" int specq_paged_attn_block(const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const void* kc,
                                      const void* vc, int code_fp8, int64_t s_kp, int64_t s_ko, int64_t s_kh,
                                      const float* ks, const float* vs, int64_t s_sp, int64_t s_sb, int64_t s_sh,
                                      int block, const int32_t* block_tbl, int64_t s_bt, int max_pages, int n_pages,
                                      const int32_t* ctx_len, void* out, int64_t s_ob, int64_t s_ot, int64_t s_oh,
                                      int B_grid, int n_seqs, int q_len, int ql_grid, int H, int H_KV, int D, int PAGE,
                                      int QPP, float sm_scale, const int32_t* plan, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  clear_error();
  SPECQ_REQUIRE(block > 0 && block % 16 == 0 && PAGE > 0 && PAGE % block == 0, SPECQ_ENOTSUP,
                "paged_attn_block: block=%d must be a multiple of 16 that divides PAGE=%d", block, PAGE);
  SPECQ_REQUIRE((uintptr_t)ks % 4 == 0 && (uintptr_t)vs % 4 == 0 && s_sp >= 0 && s_sb >= 0 && s_sh >= 0, SPECQ_EINVAL,
                "paged_attn_block: bad scale pointer or strides");
  return attn_call(code_fp8 ? kBlkF8 : kBlkI8, q, s_qb, s_qt, s_qh, kc, vc, s_kp, s_ko, s_kh, ks, vs, s_sp, s_sb, s_sh,
                   block, block_tbl, s_bt, max_pages, n_pages, ctx_len, out, s_ob, s_ot, s_oh, B_grid, n_seqs, q_len,
                   ql_grid, H, H_KV, D, PAGE, QPP, sm_scale, plan, workspace, workspace_bytes, stream);
}
