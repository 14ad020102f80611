// Verification attention over a paged K/V cache with block scales, for gfx950.
//
// The cache holds int8 or e4m3 codes [pages, PAGE, H_KV, D] and one fp32 scale for each (block of SB
// tokens, KV head), [pages, PAGE / SB, H_KV], SB a multiple of 16 that divides PAGE.  For every active
// sequence b, KV head h, query token i (of the q_len appended to the context) and query head of the group:
//   s_t = (q . k_t) * ks_blk(t) * sm_scale   for t <= L - q_len + i
//   o   = (sum_t p_t * vs_blk(t) * v_t) / sum_t p_t,   p_t = exp(s_t - max s);  0 where no token is seen.
// Tokens on a page whose id lies outside [0, pages) are masked.
//
// Programs, splits, the grid and the plan are those of the attention over per-token scales
// (paged_attn.hpp): a workgroup is a (KV split, KV head, query chunk, sequence), its QPP * G rows packed
// into RB blocks of 16, with the page ids of a split fetched ahead of the sequence's length.  The
// loop is built for what bounds it: HBM for few rows, instructions for many.  A wave issues at most one
// VALU instruction in 8 cycles here and two waves of a SIMD one in 4 (measured with loops of one
// instruction), so a chunk costs its instruction count, and everything below is there to have fewer of
// them for each token; 64 rows share what it takes to read and convert K and V.
//  * Eight waves take interleaved chunks of 32 tokens, two page sub-tiles of 16, through a
//    wave-private LDS ring filled by LDS DMA.  A slot is refilled as soon as its chunk has been read
//    into registers, so NS chunks a wave are in flight or in use.
//  * A sub-tile lies in one block: its scales are wave-uniform, fetched once with the split's page
//    ids (lane j holds those of the wave's sub-tile j) and picked with v_readlane.
//  * S^T = K . Q^T on v_mfma_f32_16x16x32_f16, one product per sub-tile, so lane (r, g) gets query row r,
//    tokens 4g .. 4g + 3 of both; that is the B operand of O^T = V^T . P^T on 16x16x32 with k-slot
//    8g + j = token 4g + j of sub-tile 0 (j < 4) or 4g + j - 4 of sub-tile 1.  V^T comes out of LDS
//    transposed by ds_read_b64_tr_b8: in a group of 16 lanes, lanes 2j and 2j + 1 name 16 bytes of a
//    row j and lane i receives byte i of the eight rows.  K/V granules are swizzled so that a
//    half-wave's reads of either kind touch all banks (blk_key).
//  * The V scale goes into the exponent: P' = exp2(s + log2 vs - m) is what the product takes, rounded to
//    fp16 once, with m a running max of s + log2 vs -- of what the tokens contribute, so that P' stays
//    a normal fp16 for everything down to 2^-22 of a row's largest contribution, whatever the scales' size.
//    The row sum is that of P' / vs, one FMA a sub-tile.  Sub-tiles whose V scale is not in
//    (2^-100, 2^100) (zero, negative, not finite) count as 1 there and multiply theirs onto P'.
//  * The running max is lazy: m lies 8 below the row's largest s + log2 vs when it moves, which it does
//    where P' passes 2^14; so P' fits fp16, and most chunks leave the accumulator alone.  A wave's first
//    chunk takes its max before its exponentials.
//  * The waves merge through the ring, every wave writing its rows once and all threads summing eight,
//    two row blocks at a time.  Up to kBlkMergeIn splits are merged by the program's last workgroup to
//    arrive, more by attn_merge_kernel behind the launch.
// Measured in a graph over distinct inputs, 32 / 8 heads, D = 128, codes read per second: 32 sequences of one token,
// contexts up to 8192, int8 85.8 us = 3.8 TB/s; 8 and 32 sequences of 9 tokens, context 4096, e4m3 26.1 us = 2.6
// TB/s and 63.2 us = 4.3 TB/s (of the 26.1, 14 are the loop, the rest start, first loads and merges); 2 x 256
// tokens, contexts up to 4096, int8 48.3 us, e4m3 45.4, one prompt of 4096 int8 245 us, e4m3 233, bound by
// instructions; one sequence of 5 tokens, context 131072, 16 / 2 heads, D = 64, e4m3 22.2 us, 4.9 of them the merge
// launch.  64-row programs at D = 128 have no register left; the e4m3 ones spill 23 (plan mode 26).
// A row's result does not depend on the rows packed with it: split boundaries, chunks and merge orders are
// fixed, so QPP = 1, fused, eager and plan calls agree bit for bit.
//
// e4m3 codes become fp16 exactly (NaN codes NaN).  A NaN in V must not reach the rows that do not see
// its token (0 * NaN): chunks with masked tokens multiply V with its NaNs cleared, and where there are any a
// product of the two indicators (token seen, code NaN) says which outputs are NaN.
#pragma once
#include "paged_attn.hpp"

namespace specq {

struct AttnBlockParams : AttnParams {
  int sb;     // tokens per scale block
  int defer;  // splits are merged by attn_merge_kernel behind this launch
  // Partials, (program, split) of the active count: part holds [n_part][rows][D] of O, then [n_part][rows][2] of
  // (m, l).
  int64_t n_part;
};

constexpr int kBlkSub = 16;                                  // tokens of a sub-tile
constexpr int kBlkChunk = 2 * kBlkSub;                       // tokens per wave iteration
constexpr int kBlkUnit = kBlkChunk * kAttnWaves;             // 256 tokens: one chunk of every wave
constexpr int kBlkMaxUnits = 64 / 2;                         // longest split: the 64 sub-tiles a wave's lanes hold
constexpr int kBlkOneSplit = 2;                              // tables of up to 512 tokens are one split
constexpr int kBlkRegion = 16384;                            // LDS ring bytes of a wave
// Up to kBlkMergeIn splits are merged by the program's last workgroup, more (and those of more programs than
// the workspace has counters) by a launch of their own, a workgroup to each row (at most kBlkMergeMax, one
// per thread there).  In a graph, 5 tokens, 32 / 8 heads,
// D = 128, e4m3: 8 splits in place and by a launch 23.8 and 26.1 us (B = 4, context 8192), 14.5 and 16.2
// (context 2048); 16 splits 25.1 and 25.5 (B = 2, context 16384), 17.2 and 15.8 (context 4096).
constexpr int kBlkMergeIn = 8;
constexpr int kBlkMergeMax = 256;
constexpr float kBlkRoom = 8.f, kBlkLazyP = 16384.f;         // m below the max when it moves; the P' that moves it
constexpr int64_t kBlkMaxTokens = (int64_t)kBlkUnit * kBlkMaxUnits * kBlkMergeMax;  // 2097152

// 256-token units per split for a table of L tokens when `pairs` (sequence, KV head) pairs (times their
// row programs) are active: as many splits as bring the workgroups to `target`, evened out.
// A second unit of a split costs 1.3 us, the merge of two splits 2.9 (B = 1, 8 heads, D = 64, table of
// 304 tokens: 8.5 us as one split, 10.1 as two; B = 8, context 1024: 11.4 as four, 12.7 as two).
__host__ __device__ inline int blk_split_units(int L, int pairs, int target) {
  const int n = L > 0 ? (L + kBlkUnit - 1) / kBlkUnit : 1;
  const int pr = pairs > 0 ? pairs : 1;
  const int want = pr >= target ? 1 : (target + pr - 1) / pr;
  int u = (n + want - 1) / want;
  const int u_min = (n + kBlkMergeMax - 1) / kBlkMergeMax;
  if (u < u_min) u = u_min;
  if (n <= kBlkOneSplit) u = n;
  if (u > kBlkMaxUnits) u = kBlkMaxUnits;
  const int ns = (n + u - 1) / u;
  return (n + ns - 1) / ns;
}

// Swizzle key of chunk token T (0..31), GR 16-byte granules per row: granule q of the row is stored in
// slot q ^ key.  256 bytes of LDS (all banks) hold 16 / GR rows; the 16 rows that a half-wave's
// transposed V read names (tokens 8h .. 8h + 7 of both sub-tiles), and the 16 rows of a K read (one
// sub-tile), differ in (row mod 16 / GR, key).
template <int GR>
__device__ __forceinline__ int blk_key(int T) { return (T / (16 / GR) + (GR / 2) * (T >> 4)) & (GR - 1); }

// Four codes in a dword -> two packed half2, eight -> v8h (int8 or e4m3; both exact).
template <bool F8>
__device__ __forceinline__ v8h code8_to_h8(uint32_t x0, uint32_t x1) {
  if constexpr (F8) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x0, 1.0f, false);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x0, 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x1, 1.0f, false);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)x1, 1.0f, true);
    return v8h{(_Float16)a[0], (_Float16)a[1], (_Float16)b[0], (_Float16)b[1],
               (_Float16)c[0], (_Float16)c[1], (_Float16)d[0], (_Float16)d[1]};
  } else {
    return i8x8_to_h8(x0, x1);
  }
}
// Bit 7 of every byte of x that is an e4m3 NaN (0x7f, 0xff).
__device__ __forceinline__ uint32_t f8_nan_bits(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// Eight bytes whose bit 7 is set or not -> 1.0 or 0.0.
__device__ __forceinline__ v8h bits_to_h8(v2i x) {
  v8h r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (_Float16)((((uint32_t)x[j >> 2] >> (8 * (j & 3) + 7)) & 1) ? 1.f : 0.f);
  return r;
}
// Two floats to packed fp16, each rounded to nearest even.
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  uint32_t r;
  asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float readlane_f(float v, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
typedef __attribute__((address_space(3))) v2i* lds_v2i;
typedef const __attribute__((address_space(3))) v4i* lds_v4i;
typedef const __attribute__((address_space(3))) v8h* lds_v8h;

template <int RBL, int D>
struct AttnBlockLds {
  uint8_t ring[kAttnWaves][kBlkRegion];
  float scales[kAttnWaves][2][64];  // K then V scale of the wave's sub-tile `lane`
  v8h q[RBL][D / 32][64];           // Q fragments, MFMA B-operand order
  float ml[kAttnWaves][2][RBL * 16];
  float row[2][RBL * 16];
  int last;
};

// The kernel body for RB 16-row query blocks, on LDS arrays sized for RBL >= RB blocks.
template <int D, int RB, bool F8, int RBL>
__device__ __forceinline__ void attn_block_body(const AttnBlockParams& p, AttnBlockLds<RBL, D>& lds) {
  constexpr int NU = D / 32;                // MFMA K-steps over the head dimension
  constexpr int ND = D / 16;                // 16-row d blocks of O^T
  constexpr int GR = D / 16;                // 16-byte granules per K/V row
  constexpr int KV4 = D / 64;               // 16-byte K granules per lane per token
  constexpr int DS = D / 4;                 // head-dim values per lane of Q
  constexpr int ROWS = RB * 16;
  constexpr int NT = kAttnThreads;
  constexpr int SB_ = kBlkSub * D;          // K (or V) bytes of a sub-tile
  constexpr int SLOT = 4 * SB_;             // K of both sub-tiles, then V
  constexpr int NS = kBlkRegion / SLOT;     // ring slots: 2 (D = 128), 4 (D = 64)
  constexpr int NDMA = SB_ / 1024;          // 1 KB DMAs for K of a sub-tile, and again for V
  constexpr int NVM = 4 * NDMA;             // DMAs per chunk
  constexpr int QPR = D / 4;                // 4-float granules per row
  static_assert(D == 64 || D == 128, "head dim");
  static_assert(RB >= 1 && RB <= 4 && RB <= RBL, "row blocks");
  tl_mark(p.tl, p.tl_cap, 0);  // diagnostics build: workgroup start

  int n_seqs = p.n_seqs, q_len = p.q_len;
  if (p.plan != nullptr) {
    n_seqs = min(max(p.plan[0], 0), p.B_grid);
    q_len = min(max(p.plan[1], 0), p.ql_grid);
  }
  n_seqs = uniform(n_seqs);
  q_len = uniform(q_len);
  const int cap = p.max_pages * p.PAGE;
  const int split_tokens = kBlkUnit * blk_split_units(cap, n_seqs * p.H_KV * attn_row_programs(q_len, p.G), p.target_wgs);
  // Workgroup order as in paged_attn.hpp: program-major, and where several query chunks read a range of at
  // most two splits, those 8 workgroups apart (one XCD, at the same time).
  const int ns_act = (cap + split_tokens - 1) / split_tokens;
  int prog, split;
  if (p.n_qc == 1 || p.plan != nullptr || ns_act > 2) {
    prog = (int)blockIdx.x / ns_act;
    split = (int)blockIdx.x - prog * ns_act;
  } else {
    const int nr = n_seqs * p.H_KV * ns_act;  // (sequence, KV head, split) ranges
    const int id = (int)blockIdx.x, nq = p.n_qc;
    const int full = (nr / 8) * 8;
    int range, qc;
    if (id < full * nq) {
      const int blk = id / (8 * nq), rem = id - blk * (8 * nq);
      qc = rem / 8;
      range = blk * 8 + rem % 8;
    } else {
      const int rem = id - full * nq, tail = nr - full;
      if (tail <= 0 || rem >= tail * nq) return;
      qc = rem / tail;
      range = full + rem % tail;
    }
    split = range % ns_act;
    prog = (range / ns_act) * nq + qc;
  }
  if (prog >= n_seqs * p.H_KV * p.n_qc) return;
  const int qc = prog % p.n_qc, kvh = (prog / p.n_qc) % p.H_KV, b = prog / (p.n_qc * p.H_KV);
  if (qc * p.QPP >= q_len) return;
  const int s0 = split * split_tokens;
  const int L_raw = p.ctx_len[b];

  const int lane = lane_id(), w = uniform(wave_id()), g = lane >> 4, r = lane & 15;
  const int G = p.G;
  float m_run[RB], l_run[RB];
  v4f acc[RB][ND];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m_run[rb] = -INFINITY;
    l_run[rb] = 0.f;
#pragma unroll
    for (int db = 0; db < ND; ++db) acc[rb][db] = v4f{0.f, 0.f, 0.f, 0.f};
  }

  // The wave's chunk `it` is the 32 tokens from s0 + 32 (w + 8 it); its sub-tile j the 16 from sub_t0(j).
  auto sub_t0 = [&](int j) { return s0 + kBlkChunk * (w + kAttnWaves * (j >> 1)) + kBlkSub * (j & 1); };
  const int32_t* bt_row = p.bt + (int64_t)b * p.s_bt;
  const int my_t0 = sub_t0(lane);
  int page_v = -1;  // page of the wave's sub-tile `lane`
  if (my_t0 < s0 + split_tokens && my_t0 < cap) page_v = bt_row[my_t0 / p.PAGE];
  // Q fragments: thread t stages fragments t, t + NT, ... of [rb][u][lane].
  constexpr int QF = (RB * NU * 64 + NT - 1) / NT;
  v8h qtmp[QF];
#pragma unroll
  for (int i = 0; i < QF; ++i) {
    const int f = threadIdx.x + NT * i;
    const int rb = f / (NU * 64), u = (f / 64) % NU, ln = f % 64;
    const int row = rb * 16 + (ln & 15);
    const int qi = qc * p.QPP + row / G;
    const bool ok = f < RB * NU * 64 && row < p.QPP * G && qi < q_len;
    const int head = kvh * G + row % G;
    const _Float16* src = ok ? p.q + (int64_t)b * p.s_qb + (int64_t)qi * p.s_qt + (int64_t)head * p.s_qh + DS * (ln >> 4) + 8 * u
                             : p.q;
    const v8h x = *reinterpret_cast<const v8h*>(src);
    qtmp[i] = ok ? x : v8h{0, 0, 0, 0, 0, 0, 0, 0};
  }

  const int L = uniform(max(min(L_raw, cap), 0));
  const int kv_end = L - q_len + min(qc * p.QPP + p.QPP, q_len);
  // Split 0 always runs, so rows with no visible key still get their zero output.
  if (split > 0 && s0 >= kv_end) return;
  const int n_active = kv_end > split_tokens ? (kv_end + split_tokens - 1) / split_tokens : 1;
  const int s1 = min(s0 + split_tokens, kv_end);
  const int w0 = s0 + kBlkChunk * w;
  const int n_it = uniform(s1 > w0 ? (s1 - w0 + kBlkUnit - 1) / kBlkUnit : 0);
  int qpos[RB];  // absolute position of the query row this lane holds in each row block
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = rb * 16 + r;
    const int qi = qc * p.QPP + row / G;
    const bool valid = (row < p.QPP * G) && (qi < q_len);
    qpos[rb] = valid ? (L - q_len + qi) : -1;
  }

  // Page ids and Q arrive together; Q goes to LDS before any DMA is issued.
  wait_vmcnt<0>();
  tl_mark(p.tl, p.tl_cap, 1);  // diagnostics build: page ids, Q and the length have landed
#pragma unroll
  for (int i = 0; i < QF; ++i) {
    const int f = threadIdx.x + NT * i;
    if (f < RB * NU * 64) (&lds.q[0][0][0])[f] = qtmp[i];
  }

  // Lane j's sub-tile: whether it is on a page of the pool, where its codes and scales are.  Sub-tiles off
  // the pool or behind the sequence stand for page 0's (their DMAs read nothing; their scales are unused).
  const bool page_ok = (uint32_t)page_v < (uint32_t)p.n_pages;
  const uint64_t bad_subs = __builtin_amdgcn_ballot_w64(!page_ok);
  int64_t kv_base_v;
  {
    const int pg = page_ok ? page_v : 0;
    const int tk = my_t0 % p.PAGE;
    kv_base_v = (int64_t)pg * p.s_kp + (int64_t)tk * p.s_ko + (int64_t)kvh * p.s_kh;
    const int64_t sc = ((int64_t)pg * p.s_sp + (int64_t)(tk / p.sb) * p.s_so + (int64_t)kvh * p.s_sh) * 4;
    dma4_global(static_cast<const uint8_t*>(p.ks) + sc, reinterpret_cast<uint8_t*>(lds.scales[w][0]));
    dma4_global(static_cast<const uint8_t*>(p.vs) + sc, reinterpret_cast<uint8_t*>(lds.scales[w][1]));
  }
  uint8_t* ring = lds.ring[w];
  // Byte offset of the lane's granule within a sub-tile, for DMA i of sub-tile s.
  uint32_t kvoff[2][NDMA];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int gi = 64 * i + lane, T = gi / GR, sl = gi % GR;
      kvoff[s][i] = (uint32_t)((int64_t)T * p.s_ko + 16 * (sl ^ blk_key<GR>(kBlkSub * s + T)));
    }
  // One query chunk and D = 128: no other program reads these lines, and they are not kept in L2.
  const bool read_once = D == 128 && p.n_qc == 1;
  // The DMAs of chunk `it` into the ring slot at `slot`.  Sub-tiles off the pool, chunks past the wave's
  // last and tokens at or past kv_end are behind the end of their buffers (zeros).
  auto issue = [&](uint32_t slot, int it) __attribute__((always_inline)) {
    uint8_t* dst = ring + slot;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int j = min(2 * it + s, 63), n = kv_end - sub_t0(2 * it + s);
      const bool real = it < n_it && ((bad_subs >> j) & 1) == 0;
      const int64_t kb = readlane64(kv_base_v, j);
      v4i rk = attn_rsrc(p.kc + kb), rv = attn_rsrc(p.vc + kb);
      rk.z = rv.z = !real || n <= 0 ? 0 : n >= kBlkSub ? (int)kOOB : (int)(n * p.s_ko);
      uint8_t* dk = dst + s * SB_;
      uint8_t* dv = dst + 2 * SB_ + s * SB_;
      if (read_once) {
#pragma unroll
        for (int i = 0; i < NDMA; ++i) dma16_rs<true>(rk, kvoff[s][i], dk + 1024 * i);
#pragma unroll
        for (int i = 0; i < NDMA; ++i) dma16_rs<true>(rv, kvoff[s][i], dv + 1024 * i);
      } else {
#pragma unroll
        for (int i = 0; i < NDMA; ++i) dma16_rs<false>(rk, kvoff[s][i], dk + 1024 * i);
#pragma unroll
        for (int i = 0; i < NDMA; ++i) dma16_rs<false>(rv, kvoff[s][i], dv + 1024 * i);
      }
    }
  };
#pragma unroll 1
  for (int i = 0; i < NS; ++i) issue(i * SLOT, i);
  wg_barrier_lds();
  constexpr bool QREG = RB <= 2;  // Q fragments in registers; deeper packings read them from LDS per chunk
  v8h qreg[QREG ? RB : 1][NU];
  if constexpr (QREG) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int u = 0; u < NU; ++u) qreg[rb][u] = lds.q[rb][u][lane];
  }
  uint32_t q_at = lds_addr(&lds.q[0][0][lane]);
  auto qfrag = [&](int rb, int u) -> v8h {
    if constexpr (QREG) return qreg[rb][u];
    else return *(lds_v8h)(q_at + (rb * NU + u) * 1024);
  };
  wait_vmcnt<NS * NVM>();  // the scales have landed
  // Lane j: the K scale * sm_scale * log2(e) of sub-tile j; its V scale, that scale's log2 and reciprocal;
  // odd_subs: sub-tiles that multiply the V scale onto P' (for those log2 0, reciprocal 1).
  const float sub_k = lds.scales[w][0][lane] * p.scale_log2, sub_v = lds.scales[w][1][lane];
  const bool odd = !(sub_v > 0x1p-100f && sub_v < 0x1p100f);
  const uint64_t odd_subs = __builtin_amdgcn_ballot_w64(page_ok && odd);
  const float sub_lv = odd ? 0.f : __builtin_amdgcn_logf(sub_v);
  const float sub_iv = odd ? 1.f : 1.f / sub_v;

  // LDS addresses of the lane's operand reads in slot 0.  K: granule g KV4 + h of token r of sub-tile s,
  // which differs from that of (0, 0) in granule bits alone: h flips the lowest, s the highest.  V: lanes 2j,
  // 2j + 1 of group g name the halves of granule db of the token of k-slot 8g + j; db flips its bits.
  // (A wave's ring starts on a multiple of a row.)
  uint32_t k_at = lds_addr(ring) + r * D + 16 * ((g * KV4) ^ blk_key<GR>(r)), v_at;
  {
    const int j = r >> 1, T = kBlkSub * (j >> 2) + 4 * g + (j & 3);
    v_at = lds_addr(ring) + 2 * SB_ + T * D + 16 * blk_key<GR>(T) + 8 * (r & 1);
  }

  // S^T of a slot's chunk, both sub-tiles, before the scales, for the row blocks [RB0, RB1).
  auto scores = [&](auto rb0c, auto rb1c, uint32_t k_s, v4f (&cs)[RB][2]) __attribute__((always_inline)) {
    constexpr int RB0 = decltype(rb0c)::value, RB1 = decltype(rb1c)::value;
#pragma unroll
    for (int rb = RB0; rb < RB1; ++rb) cs[rb][0] = cs[rb][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < KV4; ++h) {
      v4i kx[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) kx[s] = *(lds_v4i)((k_s ^ (16 * h + 8 * GR * s)) + s * SB_);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v8h kf[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) kf[s] = code8_to_h8<F8>((uint32_t)kx[s][2 * i], (uint32_t)kx[s][2 * i + 1]);
#pragma unroll
        for (int rb = RB0; rb < RB1; ++rb) {
          const v8h q = qfrag(rb, 2 * h + i);
#pragma unroll
          for (int s = 0; s < 2; ++s) cs[rb][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[s], q, cs[rb][s], 0, 0, 0);
        }
      }
    }
  };
  // Programs of 48 and 64 rows at D = 128 have no registers for the chunk's V and its scores next to the
  // accumulator: they read V behind the softmax, refill the slot then, and form the scores again in the
  // rare case that a row's max moves behind the first chunk.
  constexpr bool LATE = RB >= 3 && D == 128;
  // A wave between its matrix instructions goes before the SIMD's other wave in its softmax, which fills the gaps
  // (2 x 256 tokens, context 4096, D = 128: int8 51.9 -> 50.3 us, e4m3 46.2 -> 45.4; nothing at 16 or 32 rows).
  constexpr bool PRIO = RB >= 3;
  auto chunk = [&](uint32_t slot, int it) __attribute__((always_inline)) {
    const uint32_t k_s = k_at + slot, v_s = v_at + slot;
    if constexpr (LATE) asm volatile("" : "+v"(q_at));  // Q's addresses are formed here, not kept
    v2i vx[ND];
    v4f cs[RB][2];
    auto read_v = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < ND; ++db) vx[db] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i)(v_s ^ (16 * db)));
    };
    if constexpr (!LATE) read_v();
    if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
    scores(std::integral_constant<int, 0>{}, std::integral_constant<int, RB>{}, k_s, cs);
    if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
    if constexpr (!LATE) {  // the slot has been read: its next chunk may come
      wait_lgkm0();
      issue(slot, it + NS);
    }

    // ---- Softmax.  P' = exp2(s_raw ks + log2 vs - m), masked tokens 0.
    const int t0 = sub_t0(2 * it), j0 = min(2 * it, 62);
    const uint32_t bad = (uint32_t)(bad_subs >> j0) & 3u;  // sub-tiles off the pool
    // Every row of the program sees every token of the chunk: no mask needed.
    const bool full = bad == 0 && t0 + kBlkChunk - 1 <= L - q_len + qc * p.QPP;
    // Row block rb sees tokens e <= limit of the lane's four in sub-tile s.
    auto limit = [&](int rb, int s) { return ((bad >> s) & 1) != 0 ? -1 : qpos[rb] - (t0 + kBlkSub * s + 4 * g); };
    const float kb[2] = {readlane_f(sub_k, j0), readlane_f(sub_k, j0 + 1)};
    const float lv[2] = {readlane_f(sub_lv, j0), readlane_f(sub_lv, j0 + 1)};
    const float iv[2] = {readlane_f(sub_iv, j0), readlane_f(sub_iv, j0 + 1)};
    // Row block rb's largest score of the chunk, less kBlkRoom; sc: its scores, -inf where hidden.
    auto top_score = [&](int rb, float (&sc)[2][4]) __attribute__((always_inline)) {
      float mx = -INFINITY;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int lim = full ? 4 : limit(rb, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[s][e] = fmaf(cs[rb][s][e], kb[s], lv[s]);
          sc[s][e] = e > lim ? -INFINITY : sc[s][e];
          mx = fmaxf(mx, sc[s][e]);
        }
      }
      return group_max4(mx) - kBlkRoom;
    };
    if (it == 0) {  // the max moves there for certain
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float sc[2][4];
        m_run[rb] = top_score(rb, sc);
      }
    }
    float pr[RB][2][4], big = 0.f;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float a = lv[s] - m_run[rb];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[rb][s][e] = fast_exp2(fmaf(cs[rb][s][e], kb[s], a));
        if (!full) {
          const int lim = limit(rb, s);
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[rb][s][e] = e > lim ? 0.f : pr[rb][s][e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) big = fmaxf(big, pr[rb][s][e]);
      }
    // Lazy running max.  After a row's first chunk it rarely moves, so one wave-wide test guards it; which
    // rows move is read off the same comparison, row by row.
    if (__builtin_amdgcn_ballot_w64(big > kBlkLazyP) != 0) {
      static_for<0, RB>([&](auto rbc) __attribute__((always_inline)) {
        constexpr int rb = decltype(rbc)::value;
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(pr[rb][0][e], pr[rb][1][e]));
        uint64_t rows = __builtin_amdgcn_ballot_w64(top > kBlkLazyP);
        rows |= rows >> 32;
        rows |= rows >> 16;
        if constexpr (LATE) {
          asm volatile("" ::: "memory");  // formed again, not kept
          scores(rbc, std::integral_constant<int, rb + 1>{}, k_s, cs);
        }
        float sc[2][4];
        const float mx = top_score(rb, sc);
        if ((rows >> r) & 1) {
          const float alpha = fast_exp2(m_run[rb] - mx);  // 0 from m = -inf
          m_run[rb] = mx;
          l_run[rb] *= alpha;
#pragma unroll
          for (int db = 0; db < ND; ++db) acc[rb][db] *= alpha;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const float a = lv[s] - mx;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              pr[rb][s][e] = sc[s][e] == -INFINITY ? 0.f : fast_exp2(fmaf(cs[rb][s][e], kb[s], a));
          }
        }
      });
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        l_run[rb] = fmaf((pr[rb][s][0] + pr[rb][s][1]) + (pr[rb][s][2] + pr[rb][s][3]), iv[s], l_run[rb]);
    if (((odd_subs >> j0) & 3) != 0) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if ((odd_subs >> (j0 + s)) & 1) {
          const float vb = readlane_f(lds.scales[w][1][lane], j0 + s);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int e = 0; e < 4; ++e) pr[rb][s][e] = pr[rb][s][e] == 0.f ? 0.f : pr[rb][s][e] * vb;
        }
    }
    // ---- O^T += V^T . P'^T.
    if constexpr (LATE) {
      read_v();
      wait_lgkm0();
      issue(slot, it + NS);
    }
    v8h pf[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      typedef uint32_t v4u __attribute__((ext_vector_type(4)));
      pf[rb] = __builtin_bit_cast(v8h, v4u{pack_h2(pr[rb][0][0], pr[rb][0][1]), pack_h2(pr[rb][0][2], pr[rb][0][3]),
                                           pack_h2(pr[rb][1][0], pr[rb][1][1]), pack_h2(pr[rb][1][2], pr[rb][1][3])});
    }
    if constexpr (F8) {  // NaN codes of V in a chunk with masked tokens
      if (!full) {
        uint32_t any = 0;
#pragma unroll
        for (int db = 0; db < ND; ++db) any |= f8_nan_bits((uint32_t)vx[db].x) | f8_nan_bits((uint32_t)vx[db].y);
        if (__builtin_amdgcn_ballot_w64(any != 0) != 0) {
#pragma unroll
          for (int db = 0; db < ND; ++db) {
            const v2i nb = {(int)f8_nan_bits((uint32_t)vx[db].x), (int)f8_nan_bits((uint32_t)vx[db].y)};
            const v8h isnan = bits_to_h8(nb);
            int at = t0 + 4 * g;  // the indicators are formed for each db, not kept in registers
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
              v8h seen;
#pragma unroll
              for (int j = 0; j < 8; ++j) seen[j] = (_Float16)(((bad >> (j >> 2)) & 1) != 0 || at + kBlkSub * (j >> 2) + (j & 3) > qpos[rb] ? 0.f : 1.f);
              const v4f hits = __builtin_amdgcn_mfma_f32_16x16x32_f16(isnan, seen, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (hits[j] > 0.f) acc[rb][db][j] = __builtin_nanf("");
            }
            vx[db].x &= ~(int)(((uint32_t)nb.x >> 7) * 0xffu);
            vx[db].y &= ~(int)(((uint32_t)nb.y >> 7) * 0xffu);
          }
        }
      }
    }
    if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int db = 0; db < ND; ++db) {
      const v8h vf = code8_to_h8<F8>((uint32_t)vx[db].x, (uint32_t)vx[db].y);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) acc[rb][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rb], acc[rb][db], 0, 0, 0);
    }
    if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
  };
  // One copy of the loop's code serves all slots: a launch finds the instruction cache cold, and most calls
  // go around a few times only.
#pragma unroll 1
  for (int it = 0, slot = 0; it < n_it; ++it) {
    wait_vmcnt<(NS - 1) * NVM>();  // chunk `it` has landed
    chunk(slot, it);
    slot = slot == (NS - 1) * SLOT ? 0 : slot + SLOT;
  }
  // Every DMA has landed before the ring is reused for the merge.
  wait_vmcnt<0>();
  tl_mark(p.tl, p.tl_cap, 3);       // diagnostics build: chunk loop done (wave 0)
  tl_mark_wave(p.tl, p.tl_cap, 8);  // ... and per wave (marks 8..15)

  // ---- Merge the eight waves: row statistics, then O scaled to the workgroup's row max, two row blocks
  // at a time.  A wave's region holds [2][16][D] floats, granule c of row n at c ^ n.
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float lr = l_run[rb];
    lr += __shfl_xor(lr, 16);
    lr += __shfl_xor(lr, 32);
    if (g == 0) {
      lds.ml[w][0][rb * 16 + r] = m_run[rb];
      lds.ml[w][1][rb * 16 + r] = lr;
    }
  }
  __syncthreads();
  tl_mark(p.tl, p.tl_cap, 7);  // diagnostics build: every wave's chunk loop done
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = rb * 16 + r;
    float mv[kAttnWaves];
#pragma unroll
    for (int ww = 0; ww < kAttnWaves; ++ww) mv[ww] = lds.ml[ww][0][row];
    float mx = mv[0];
#pragma unroll
    for (int ww = 1; ww < kAttnWaves; ++ww) mx = fmaxf(mx, mv[ww]);
    const float ms = (mx == -INFINITY) ? 0.f : mx;
    const float wsc = fast_exp2(m_run[rb] - ms);
    if (w == 0 && g == 0) {
      float l = 0.f;
#pragma unroll
      for (int ww = 0; ww < kAttnWaves; ++ww) l += fast_exp2(mv[ww] - ms) * lds.ml[ww][1][row];
      lds.row[0][row] = mx;
      lds.row[1][row] = l;
    }
#pragma unroll
    for (int db = 0; db < ND; ++db) acc[rb][db] *= wsc;
  }
  constexpr int ITEMS = (ROWS * QPR + NT - 1) / NT;
  constexpr int RPI = NT / QPR;  // rows one pass of all threads covers: 16 (D = 128) or 32
  v4f o[ITEMS];
  bool ivalid[ITEMS];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const int row = (int)threadIdx.x / QPR + RPI * it;
    const int qi = qc * p.QPP + row / G;
    ivalid[it] = row < ROWS && row < p.QPP * G && qi < q_len;
    o[it] = v4f{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int r0 = 0; r0 < RB; r0 += 2) {
    if (r0 > 0) __syncthreads();
#pragma unroll
    for (int rb = r0; rb < RB && rb < r0 + 2; ++rb)
#pragma unroll
      for (int db = 0; db < ND; ++db)
        *reinterpret_cast<v4f*>(ring + (rb - r0) * 64 * D + r * 4 * D + 16 * ((4 * db + g) ^ r)) = acc[rb][db];
    __syncthreads();
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      const int row = (int)threadIdx.x / QPR + RPI * it, c = (int)threadIdx.x % QPR;
      if (row >= 16 * r0 && row < 16 * r0 + 32 && ivalid[it]) {
        const int at = (row - 16 * r0) * 4 * D + 16 * (c ^ (row & 15));
#pragma unroll
        for (int ww = 0; ww < kAttnWaves; ++ww) o[it] += *reinterpret_cast<const v4f*>(lds.ring[ww] + at);
      }
    }
  }
  auto store_row4 = [&](int it, v4f v) {
    const int row = (int)threadIdx.x / QPR + RPI * it, d0 = ((int)threadIdx.x % QPR) * 4;
    const int qi = qc * p.QPP + row / G;
    const int head = kvh * G + row % G;
    *reinterpret_cast<v2i*>(p.out + (int64_t)b * p.s_ob + (int64_t)qi * p.s_ot + (int64_t)head * p.s_oh + d0) =
        v2i{(int)pack_h2(v.x, v.y), (int)pack_h2(v.z, v.w)};
  };
  tl_mark(p.tl, p.tl_cap, 4);  // diagnostics build: waves merged
  if (n_active == 1) {
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
      if (!ivalid[it]) continue;
      const float l = lds.row[1][(int)threadIdx.x / QPR + RPI * it];
      store_row4(it, o[it] * (l == 0.f ? 0.f : 1.f / l));
    }
    tl_mark_drained(p.tl, p.tl_cap, 6);  // diagnostics build: output stored
    return;
  }

  // ---- Splits: publish this split's valid rows, 16 bytes per lane.
  const int64_t prog_base = (int64_t)prog * ns_act;
  const int64_t n_o = p.n_part * ROWS * D;  // floats of the O region
  const rsrc_t ors = make_rsrc(p.part + prog_base * ROWS * D, (uint32_t)(ns_act * ROWS * D * 4));
  float* mlpart = p.part + n_o;
#pragma unroll
  for (int it = 0; it < ITEMS; ++it)
    if (ivalid[it]) publish16(ors, (uint32_t)((split * ROWS * QPR + (int)threadIdx.x + NT * it) * 16), __builtin_bit_cast(v4i, o[it]));
  if (threadIdx.x < ROWS) {
    float* mlp = mlpart + ((prog_base + split) * ROWS + threadIdx.x) * 2;
    publish(mlp, lds.row[0][threadIdx.x]);
    publish(mlp + 1, lds.row[1][threadIdx.x]);
  }
  tl_mark(p.tl, p.tl_cap, 5);  // diagnostics build: partials issued
  if (p.defer) return;
  if (!arrive_last(p.counters + prog, n_active, &lds.last, p.tl, p.tl_cap)) return;
  // The last split to arrive sums the program's, in split order: weights exp2(m_s - max) / l first (one
  // thread a row and all pairs in flight together), then the rows.  A plan-mode call may merge the same
  // splits by attn_merge_kernel, and both take the same steps: products rounded on their own, l summed as
  // a butterfly over lanes sums it, the weighted rows in split order.
  float* wts = reinterpret_cast<float*>(lds.ring[0]);  // [ROWS][kBlkMergeIn]
  if (threadIdx.x < ROWS) {
#pragma clang fp contract(off)
    float mv[kBlkMergeIn], lv[kBlkMergeIn], mx = -INFINITY;
#pragma unroll
    for (int sp = 0; sp < kBlkMergeIn; ++sp) {
      const float* src = mlpart + ((prog_base + min(sp, n_active - 1)) * ROWS + threadIdx.x) * 2;
      mv[sp] = collect(src);
      lv[sp] = collect(src + 1);
    }
#pragma unroll
    for (int sp = 0; sp < kBlkMergeIn; ++sp)
      if (sp < n_active) mx = fmaxf(mx, mv[sp]);
    const float mxs = (mx == -INFINITY) ? 0.f : mx;
#pragma unroll
    for (int sp = 0; sp < kBlkMergeIn; ++sp) {
      if (sp < n_active) {
        mv[sp] = fast_exp2(mv[sp] - mxs);
        lv[sp] = mv[sp] * lv[sp];
      } else {
        mv[sp] = lv[sp] = 0.f;
      }
    }
#pragma unroll
    for (int h = kBlkMergeIn / 2; h >= 1; h /= 2)
#pragma unroll
      for (int sp = 0; sp < h; ++sp) lv[sp] += lv[sp + h];
    const float inv = lv[0] == 0.f ? 0.f : 1.f / lv[0];
#pragma unroll
    for (int sp = 0; sp < kBlkMergeIn; ++sp) wts[threadIdx.x * kBlkMergeIn + sp] = mv[sp] * inv;
  }
  v4i part[ITEMS <= 2 ? kBlkMergeIn : kBlkMergeIn / 2][ITEMS];
  constexpr int SBT = ITEMS <= 2 ? kBlkMergeIn : kBlkMergeIn / 2;  // splits whose rows are in flight together
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) o[it] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int sp0 = 0; sp0 < n_active; sp0 += SBT) {
#pragma unroll
    for (int u = 0; u < SBT; ++u)
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
        part[u][it] = collect16(ors, oob_unless(ivalid[it] && sp0 + u < n_active,
                                                (uint32_t)(((sp0 + u) * ROWS * QPR + (int)threadIdx.x + NT * it) * 16)));
    if (sp0 == 0) __syncthreads();  // the weights
#pragma unroll
    for (int u = 0; u < SBT; ++u)
#pragma unroll
      for (int it = 0; it < ITEMS; ++it)
        if (ivalid[it] && sp0 + u < n_active) {
#pragma clang fp contract(off)
          o[it] += wts[((int)threadIdx.x / QPR + RPI * it) * kBlkMergeIn + sp0 + u] * __builtin_bit_cast(v4f, part[u][it]);
        }
  }
#pragma unroll
  for (int it = 0; it < ITEMS; ++it)
    if (ivalid[it]) store_row4(it, o[it]);
  tl_mark_drained(p.tl, p.tl_cap, 6);  // diagnostics build: splits merged and stored
}

template <int D, int RB, bool F8>
__global__ __launch_bounds__(kAttnThreads) void attn_block_kernel(AttnBlockParams p) {
  __shared__ __attribute__((aligned(1024))) AttnBlockLds<RB, D> lds;
  attn_block_body<D, RB, F8, RB>(p, lds);
}

// Plan-mode launch captured for programs of up to RBMAX row blocks: the body of the active q_len's blocks.
template <int D, int RBMAX, bool F8>
__global__ __launch_bounds__(kAttnThreads) void attn_block_plan_kernel(AttnBlockParams p) {
  __shared__ __attribute__((aligned(1024))) AttnBlockLds<RBMAX, D> lds;
  const int q_len = min(max(p.plan[1], 0), p.ql_grid);
  const int rb = uniform(min(max((min(q_len, p.QPP) * p.G + 15) / 16, 1), RBMAX));
  if (rb == 1) {
    attn_block_body<D, 1, F8, RBMAX>(p, lds);
  } else if (rb == 2) {
    attn_block_body<D, 2, F8, RBMAX>(p, lds);
  } else if (rb == 3) {
    if constexpr (RBMAX >= 3) attn_block_body<D, 3, F8, RBMAX>(p, lds);
  } else {
    if constexpr (RBMAX >= 4) attn_block_body<D, 4, F8, RBMAX>(p, lds);
  }
}

// Merge of launches with many splits: workgroup (program, packed row).  Thread t holds
// split t's (m, l); the row's weights exp2(m - max) / l go to LDS, and the 256 / (D / 4) thread groups
// sum every such-th split's row, the groups then in order.  The sum's order depends on nothing but
// the number of splits, and splits in which the row sees nothing add zeros.  Bound by latency: three
// dependent round trips (length, statistics, rows), the rows' loads eight in flight.
template <int D>
__global__ __launch_bounds__(256) void attn_merge_kernel(AttnBlockParams p) {
  constexpr int LN = D / 4, NG = 256 / LN, IN_FLIGHT = 8;
  int n_seqs = p.n_seqs, q_len = p.q_len;
  if (p.plan != nullptr) {
    n_seqs = min(max(p.plan[0], 0), p.B_grid);
    q_len = min(max(p.plan[1], 0), p.ql_grid);
  }
  n_seqs = uniform(n_seqs);
  q_len = uniform(q_len);
  // Rows of a program's partials: those of the row blocks it ran with, in plan mode the active q_len's.
  const int per = p.QPP * p.G, rows = ((p.plan != nullptr ? min(q_len, p.QPP) * p.G : per) + 15) / 16 * 16;
  const int prog = (int)blockIdx.x / per, row = (int)blockIdx.x - prog * per;
  const int qc = prog % p.n_qc, kvh = (prog / p.n_qc) % p.H_KV, b = prog / (p.n_qc * p.H_KV);
  const int qi = qc * p.QPP + row / p.G;
  if (b >= n_seqs || qi >= q_len) return;
  const int cap = p.max_pages * p.PAGE;
  const int split_tokens = kBlkUnit * blk_split_units(cap, n_seqs * p.H_KV * attn_row_programs(q_len, p.G), p.target_wgs);
  const int L = uniform(max(min(p.ctx_len[b], cap), 0));
  const int kv_end = L - q_len + min(qc * p.QPP + p.QPP, q_len);
  const int n = kv_end > split_tokens ? (kv_end + split_tokens - 1) / split_tokens : 1;
  if (n == 1) return;  // the row's only split has stored it
  const int ns_act = (cap + split_tokens - 1) / split_tokens;
  const int64_t base = (int64_t)prog * ns_act * rows + row;  // the row in split 0, in rows
  const float* ml = p.part + p.n_part * rows * D;
  const int t = threadIdx.x;
  __shared__ float wt[kBlkMergeMax], red[2][4];
  __shared__ v4f sum[NG][LN];
  float m = -INFINITY, l = 0.f;
  if (t < n) {
    m = ml[(base + (int64_t)t * rows) * 2];
    l = ml[(base + (int64_t)t * rows) * 2 + 1];
  }
  float mx = m;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
  if (lane_id() == 0) red[0][wave_id()] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float w = fast_exp2(m - (mx == -INFINITY ? 0.f : mx));
  float ls;
  {
#pragma clang fp contract(off)
    ls = t < n ? w * l : 0.f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) ls += __shfl_xor(ls, o);
  }
  if (lane_id() == 0) red[1][wave_id()] = ls;
  wt[t] = t < n ? w : 0.f;
  __syncthreads();
  ls = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const float inv = ls == 0.f ? 0.f : 1.f / ls;
  const int g = t / LN, c = t % LN;
  const v4f* o_part = reinterpret_cast<const v4f*>(p.part) + base * LN + c;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < n; s0 += NG * IN_FLIGHT) {
    v4f x[IN_FLIGHT];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u) x[u] = o_part[(int64_t)min(s0 + u * NG, n - 1) * rows * LN];
#pragma unroll
    for (int u = 0; u < IN_FLIGHT; ++u)
      if (s0 + u * NG < n) {
#pragma clang fp contract(off)
        o += wt[s0 + u * NG] * inv * x[u];
      }
  }
  sum[g][c] = o;
  __syncthreads();
  if (g == 0) {
    for (int i = 1; i < NG; ++i) o += sum[i][c];
    const int head = kvh * p.G + row % p.G;
    *reinterpret_cast<v2i*>(p.out + (int64_t)b * p.s_ob + (int64_t)qi * p.s_ot + (int64_t)head * p.s_oh + 4 * c) =
        v2i{(int)pack_h2(o.x, o.y), (int)pack_h2(o.z, o.w)};
  }
}

}  // namespace specq
