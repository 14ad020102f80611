// Attention weights gathered by the cached tokens, and its C ABI.
//
// For every active sequence b, KV head h and token t < L of the paged int8 cache:
//   s_r,t = (q_r . k_t) ks_t sm_scale       over the rows r = (new token i, query head of the group),
//                                           seen where t <= L - q_len + i and t's page is in the pool
//   p_r,t = softmax_t(s_r)                  a row that sees nothing gives 0
//   w[b, h, t] = (t >= L - q_len ? 0 : w[b, h, t]) + sum_r p_r,t
// K alone is read, V is not needed.  A softmax has to know its whole row before any of its values can be added up over
// the rows, so the work is two launches over the same tiles of 256 tokens:
//   1  scores, and (max, sum of exponentials) of each row within the tile; the last workgroup of a (sequence, head)
//      joins them to each row's max and the reciprocal of its sum over all tiles
//   2  p = exp2(s - max) / sum, summed over the rows, and the update of w
// Max and sum stay apart: in one number, max + log2(sum), the sum's part would be rounded to the steps of the max, the same way in
// all of a row's probabilities (2^-21 of them at scores of 10, 2^-10 at 16000).
// The scores of up to 16 rows (kAwStoreRows: plain decoding) go from 1 to 2 through the workspace; more rows compute them
// again.  Both ways add a token's rows in one order (16 lanes; in each the blocks of 16 rows of either parity, then both; then
// pairs of lanes; then units of 512 rows one after another) and join the rows' statistics in one (64 tokens, 256, all), so they
// give the same bits, and a plan-mode call those of an eager one.  Workgroups take one or two units each, and the last of a
// tile's adds theirs up.
//
// K stays: a wave holds 64 tokens, converts their codes to fp16 matrix operands once and walks the rows 16 at a time
// (K . Q^T on v_mfma_f32_16x16x32_f16: a lane's results are four tokens of one row).  Everything behind the products is
// fp32; log2(e) is folded into the scale.
// 8 KV heads of 128 (us): a new token of 32 sequences of up to 8192, stored scores, 51 + 7, codes and scores at 3.4 TB/s (loads
// alone 5.2; the CUs are busy 60 % of the time, since spans of tiles are cut from the table and not from the lengths); 9 of 8
// sequences of 4096, formed twice, 20 + 14, half of it fixed phases; 256 of 2 of up to 4096, 43 + 34, bound by vector instructions
// at two waves a SIMD.
#include <algorithm>

#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kAwTile = 256;       // tokens of a workgroup: 4 waves of 4 sub-tiles of 16
constexpr int kAwStoreRows = 16;   // rows whose scores go through the workspace
constexpr int kAwFewRows = 64;     // rows whose queries a workgroup keeps in LDS
constexpr int kAwSpan = 8;         // most tiles such a workgroup walks (its waves' lanes hold their pages, and one tile's more)
constexpr int kAwUnitRows = 512;   // rows whose sums are added to the weights in one piece
constexpr int kAwSegUnits = 2;     // most units of a workgroup
constexpr int kAwSegs = 8;         // most such segments of a launch
constexpr int kAwFill = 256;       // workgroups that fill the GPU: fewer take a unit each
constexpr int kAwSeg = 32;         // row blocks of 16 whose statistics are joined at a time
constexpr int kAwSumTile = 1024;   // tokens of a workgroup that adds up stored scores
// Most workgroups a CU of a launch of 256 threads, of 512, and of the one that sums stored scores; they come back for more.
constexpr int kAwFewGrid = 8, kAwManyGrid = 4, kAwSumGrid = 16;
// Bytes that scores, statistics and sums of a launch take at most, unless one sequence needs more: they are as wide as the table, however
// short the contexts, so a large batch is taken some sequences at a time.  A further pair of launches takes some 8 us, where the
// scores alone of 256 MiB take more than 50 each way.
constexpr int64_t kAwMost = 256 << 20;

struct AwParams {
  const _Float16* q; int64_t s_qb, s_qt, s_qh;
  const int8_t* kc; int64_t s_kp, s_ko, s_kh;
  const void* ks; int64_t s_sp, s_so, s_sh;
  const int32_t* bt; int64_t s_bt; int max_pages, n_pages;
  const int32_t* ctx_len; const int32_t* q_lens;
  float* w; int64_t s_wb, s_wh; int w_vec;  // w_vec: its rows are 16-byte aligned
  const int32_t* plan;
  int b0;  // the launch's first sequence in a plan's count; tensors and sizes are those from it on
  int n_seqs, q_len, B_grid, ql_grid, G, H_KV, PAGE;
  int cap;      // tokens a row of the table holds
  int tiles;    // of cap
  int span;     // tiles of a workgroup of few rows, at most
  int rows;     // of a program and segment at most
  int row0;     // the launch's first row: more than segs * seg_rows have several pairs of launches one after another
  int seg_rows, segs;  // rows of a workgroup's segment (a unit or more), segments of a launch
  uint32_t g_magic;  // ceil(2^32 / G): row / G is its product's high word (rows below 2^20, G below 2^12); 0 for G = 1
  float scale_log2;
  // Workspace: scores [prog][rows][tiles * 256]; (max, sum) [prog][seg][tiles][rows]; the rows' (max, 1 / sum) [prog][seg][rows];
  // sums of a unit's rows [prog][unit][tiles * 256], two tokens a word.
  float* scores; uint64_t* stats; uint64_t* norms; uint64_t* sums;
  int32_t* counters;  // [prog][seg], then [prog][tile]
};

// Program number `i` of the launch order.  The heads of a sequence read the same lines of scales: in blocks of eight
// sequences they come eight workgroups apart, which puts them on one XCD, whose L2 serves them.
__device__ __forceinline__ int aw_order(const AwParams& p, int i) {
  const int full = p.B_grid / 8 * 8 * p.H_KV;
  if (i >= full) return i;
  const int blk = i / (8 * p.H_KV), rem = i - blk * (8 * p.H_KV);
  return (blk * 8 + rem % 8) * p.H_KV + rem / 8;
}
// The new token of a row.
__device__ __forceinline__ int aw_token(const AwParams& p, int row) {
  return p.g_magic != 0 ? (int)__umulhi((uint32_t)row, p.g_magic) : row;
}
// A program (sequence b, KV head h): its rows from row0 on, of a segment at most, its tokens and active tiles.
struct AwProg {
  int b, h, ql, rows, L, tiles;
};
__device__ __forceinline__ bool aw_prog(const AwParams& p, int prog, AwProg& x, int row0 = 0) {
  int n_seqs = p.n_seqs, q_len = p.q_len;
  if (p.plan != nullptr) {
    n_seqs = min(max(p.plan[0] - p.b0, 0), p.B_grid);
    q_len = min(max(p.plan[1], 0), p.ql_grid);
  }
  x.b = prog / p.H_KV;
  x.h = prog - x.b * p.H_KV;
  if (x.b >= n_seqs) return false;
  x.ql = p.q_lens != nullptr ? min(max(p.q_lens[x.b], 0), q_len) : q_len;
  x.rows = min(x.ql * p.G - row0, p.rows);
  x.L = min(max(p.ctx_len[x.b], 0), p.cap);
  x.tiles = (x.L + kAwTile - 1) / kAwTile;
  return x.rows > 0 && x.L > 0;
}

// Tables are often much wider than the contexts, and an empty workgroup takes its turn as well: a prompt of 4096 tokens in a table of
// 131072 took 1200 us where one of 4096 takes 405, 9 tokens of 32 sequences of 1000 110 us and 33.  So a workgroup that comes back
// for its second item looks how long the longest sequence is, and items behind that are none: `live`, with `per` items to every
// `step` tiles (these: 370 and 42 us; calls without a second item 0 to 1 % longer).
__device__ __forceinline__ int64_t aw_live(const AwParams& p, int64_t item, int64_t live, int64_t per, int step) {
  if (item >= live || item != (int64_t)blockIdx.x + gridDim.x) return live;
  const int n = p.plan != nullptr ? min(max(p.plan[0] - p.b0, 0), p.B_grid) : p.n_seqs;
  int longest = 0;
  for (int b = lane_id(); b < n; b += kWave) longest = max(longest, p.ctx_len[b]);
  for (int o = 1; o < kWave; o *= 2) longest = max(longest, __shfl_xor(longest, o));
  const int tiles = (min(uniform(longest), p.cap) + kAwTile - 1) / kAwTile;
  return min(live, per * ((tiles + step - 1) / step));
}

__device__ __forceinline__ float aw_max4(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const int u = __builtin_bit_cast(int, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const int v = __builtin_bit_cast(int, fmaxf(__builtin_bit_cast(float, (int)a[0]), __builtin_bit_cast(float, (int)a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__builtin_bit_cast(float, (int)b[0]), __builtin_bit_cast(float, (int)b[1]));
}
__device__ __forceinline__ float aw_sum4(float x) {
  const int u = __builtin_bit_cast(int, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const int v = __builtin_bit_cast(int, __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_bit_cast(float, (int)b[0]) + __builtin_bit_cast(float, (int)b[1]);
}
// Sum over the 16 lanes of a row of lanes: lanes 2k and 2k + 1, pairs, fours (mirrored), eights (mirrored).
__device__ __forceinline__ float aw_sum16(float v) {
  auto add = [&](auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), c, 0xf, 0xf, false));
  };
  add(std::integral_constant<int, 0xB1>{});
  add(std::integral_constant<int, 0x4E>{});
  add(std::integral_constant<int, 0x141>{});
  add(std::integral_constant<int, 0x140>{});
  return v;
}
__device__ __forceinline__ uint64_t aw_pack(float m, float l) {
  return (uint64_t)__builtin_bit_cast(uint32_t, m) | ((uint64_t)__builtin_bit_cast(uint32_t, l) << 32);
}
__device__ __forceinline__ float aw_m(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }
__device__ __forceinline__ float aw_l(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)(x >> 32)); }
// (m, l) joined with (m2, l2): sums of exp2 relative to their maxima.  An empty one is (-inf, 0).
__device__ __forceinline__ void aw_join(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
  l = l * fast_exp2(m - ref) + l2 * fast_exp2(m2 - ref);
  m = top;
}

// The weights of tokens t..t + 3; new ones start from nothing (`start`: unless an earlier launch has set them).
__device__ __forceinline__ v4f aw_get(const AwParams& p, const AwProg& x, int t, bool start) {
  const float* w = p.w + x.b * p.s_wb + x.h * p.s_wh + t;
  v4f v = {0.f, 0.f, 0.f, 0.f};
  if (p.w_vec && t + 4 <= x.L) {
    v = *reinterpret_cast<const v4f*>(w);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t + i < x.L) v[i] = w[i];
  }
  const int fresh = start ? x.L - x.ql : x.L;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t + i >= fresh) v[i] = 0.f;
  return v;
}
__device__ __forceinline__ void aw_put(const AwParams& p, const AwProg& x, int t, const v4f& v) {
  float* w = p.w + x.b * p.s_wb + x.h * p.s_wh + t;
  if (p.w_vec && t + 4 <= x.L) {
    *reinterpret_cast<v4f*>(w) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t + i < x.L) w[i] = v[i];
  }
}

enum { kAwStats, kAwSums };  // pass 1, and pass 2 from K

// Where a wave's sub-tiles lie: lane l holds those of sub-tile l (four to a tile).  A sub-tile lies in one page.  One past the
// context or on no page of the pool is not `ok`: its codes read as nothing, its scales are the pool's first.
struct AwPages {
  int64_t kv, sc;  // of its first token: bytes to the codes, scales ahead
  uint64_t ok;     // bit l: sub-tile l
};
__device__ __forceinline__ AwPages aw_pages(const AwParams& p, const AwProg& x, int t, int page, bool in) {
  const bool ok = in && t < x.L && (uint32_t)page < (uint32_t)p.n_pages;
  const int pg = ok ? page : 0, slot = ok ? t % p.PAGE : 0;
  return {pg * p.s_kp + slot * p.s_ko + x.h * p.s_kh, pg * p.s_sp + slot * p.s_so + x.h * p.s_sh, __builtin_amdgcn_ballot_w64(ok)};
}
__device__ __forceinline__ int64_t aw_lane64(int64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)v >> 32), l);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// Codes and scales of sub-tiles l0..l0 + 3.  Always the same loads, so that the waits on them are counted, not drained.  An
// access takes whole rows (D / 16 lanes a row): lanes that take matrix operands directly touch half of each 128-byte line
// twice, 3.7 TB/s instead of 4.1 over a long cache; NT, the lines not kept in L2: 5.2 (loads alone).
template <int D, bool NT, typename ST>
__device__ __forceinline__ void aw_load(const AwParams& p, const AwPages& at, int l0, v4i (&raw)[4][D / 64], ST& scale) {
  constexpr int GR = D / 16, NI = D / 64;
  const int lane = lane_id(), r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const rsrc_t rs = make_rsrc(p.kc + aw_lane64(at.kv, l0 + s), kOOB);
    const uint32_t off = oob_unless((at.ok >> (l0 + s)) & 1, (uint32_t)(lane / GR * (int)p.s_ko + 16 * (lane % GR)));
#pragma unroll
    for (int i = 0; i < NI; ++i)
      raw[s][i] = __builtin_amdgcn_raw_buffer_load_b128(rs, off, i * (64 / GR) * (int)p.s_ko, NT ? 2 : 0);
  }
  const int64_t sc = (int64_t)(((uint64_t)(uint32_t)__shfl((int)(uint32_t)((uint64_t)at.sc >> 32), l0 + g) << 32) |
                               (uint32_t)__shfl((int)(uint32_t)at.sc, l0 + g));
  scale = static_cast<const ST*>(p.ks)[sc + r * p.s_so];
}

// A wave's codes change hands through LDS: granule q of token T lies in slot q ^ key(T) of its row, so that neither side's
// accesses meet in a bank.
template <int D>
struct AwStage {
  v4i x[4][16][D / 16];
  static __device__ __forceinline__ int key(int t) { return D == 128 ? t & 7 : (t >> 1) & 3; }
  __device__ __forceinline__ void put(const v4i (&raw)[4][D / 64]) {
    constexpr int GR = D / 16;
    const int lane = lane_id();
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const int t = i * (64 / GR) + lane / GR;
        x[s][t][(lane % GR) ^ key(t)] = raw[s][i];
      }
  }
  // fp16 operands of sub-tile s.  Values of matrix step u = 2 i + half: d = 64 i + 16 g + 8 half + j, for K and Q alike.
  __device__ __forceinline__ void get(int s, v8h (&kh)[D / 32]) const {
    const int r = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const v4i v = x[s][r][(4 * i + g) ^ key(r)];
      kh[2 * i] = i8x8_to_h8((uint32_t)v[0], (uint32_t)v[1]);
      kh[2 * i + 1] = i8x8_to_h8((uint32_t)v[2], (uint32_t)v[3]);
    }
  }
};

// -inf where the lane's row does not see the token.
__device__ __forceinline__ void aw_hide(int t0, int last, uint32_t seen, v4f (&acc)[4]) {
  const int g = lane_id() >> 4;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!(((seen >> s) & 1) && t0 + 16 * s + 4 * g + i <= last)) acc[s][i] = -INFINITY;
}
// A product's scale and, SUB, the row's max off it: not one instruction, since stored scores, and those of the row's sum, are
// rounded between the two.
template <bool SUB>
__device__ __forceinline__ float aw_scaled(float acc, float ksc, float top) {
#pragma clang fp contract(off)
  acc *= ksc;
  return SUB ? acc - top : acc;
}
template <bool SUB>
__device__ __forceinline__ void aw_scale(const v4f (&ksc)[4], float top, v4f (&acc)[4]) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[s][i] = aw_scaled<SUB>(acc[s][i], ksc[s][i], top);
}
// Scores (in log2; SUB, less the row's max) of the wave's tokens with the row of lane % 16.
template <int D, bool SUB>
__device__ __forceinline__ void aw_scores(const v8h (&kh)[4][D / 32], const v8h (&qf)[D / 32], const v4f (&ksc)[4], int t0, int last,
                                          bool all, uint32_t seen, float top, v4f (&acc)[4]) {
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    acc[s] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < D / 32; ++u) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[s][u], qf[u], acc[s], 0, 0, 0);
  }
  aw_scale<SUB>(ksc, top, acc);
  if (!all) aw_hide(t0, last, seen, acc);  // all: every row sees all
}
// (max, sum) of a row over the wave's tokens, in all lanes of the row.
__device__ __forceinline__ uint64_t aw_stat(const v4f (&acc)[4]) {
  float m = -INFINITY;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, acc[s][i]);
  m = aw_max4(m);
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) l += fast_exp2(acc[s][i] - ref);
  return aw_pack(m, aw_sum4(l));
}
// The rows' sums over the lanes: lanes 0..3 of each 16 have four tokens each, from aw_first(t0) on.
__device__ __forceinline__ int aw_first(int t0) { return t0 + 16 * (lane_id() & 15) + 4 * (lane_id() >> 4); }
__device__ __forceinline__ v4f aw_rows(const v4f (&sums)[4]) {
  const int r = lane_id() & 15;
  v4f got = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = aw_sum16(sums[s][i]);
      got[i] = r == s ? v : got[i];
    }
  return got;
}
// The last workgroup of a program joins its rows' tiles: many rows a thread each, few a group of lanes each (as many as
// there are tiles, at most a wave).
__device__ __forceinline__ void aw_norms(const AwParams& p, const AwProg& x, int at) {  // at: of [prog][seg]
  const int threads = blockDim.x;
  const uint64_t* st = p.stats + (int64_t)at * p.tiles * p.rows;
  uint64_t* out = p.norms + (int64_t)at * p.rows;
  // Of a row that sees nothing an infinite max, so that it gives 0; a maximum knows no NaN, the sum does, and makes the max one.
  auto done = [&](int row, float m, float l) {
    out[row] = !(l == l) ? aw_pack(l, 1.f) : m == -INFINITY ? aw_pack(INFINITY, 0.f) : aw_pack(m, 1.f / l);
  };
  // Tiles k0, k0 + step, ...: eight loads in flight.
  auto walk = [&](int row, int k0, int step, float& m, float& l) {
    constexpr int U = 8;
    for (int k = k0; k < x.tiles; k += U * step) {
      uint64_t v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = k + u * step < x.tiles ? collect(st + (int64_t)(k + u * step) * p.rows + row) : aw_pack(-INFINITY, 0.f);
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) top = fmaxf(top, aw_m(v[u]));
      const float ref = top == -INFINITY ? 0.f : top;
      l *= fast_exp2(m - ref);
#pragma unroll
      for (int u = 0; u < U; ++u) l += aw_l(v[u]) * fast_exp2(aw_m(v[u]) - ref);
      m = top;
    }
  };
  if (x.ql * p.G > kAwFewRows) {  // of the program, not of a segment: a row's order is the same in any
    for (int row = threadIdx.x; row < x.rows; row += threads) {
      float m = -INFINITY, l = 0.f;
      walk(row, 0, 1, m, l);
      done(row, m, l);
    }
    return;
  }
  int lanes = 1;
  while (lanes < x.tiles && lanes < kWave) lanes *= 2;
  for (int i = threadIdx.x; i / kWave * kWave < x.rows * lanes; i += threads) {  // whole waves
    const int row = min(i / lanes, x.rows - 1);
    float m = -INFINITY, l = 0.f;
    walk(row, i % lanes, lanes, m, l);
    float top = m;
    for (int o = 1; o < lanes; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    l *= fast_exp2(m - (top == -INFINITY ? 0.f : top));
    for (int o = 1; o < lanes; o *= 2) l += __shfl_xor(l, o);
    if (i % lanes == 0 && i / lanes < x.rows) done(row, top, l);
  }
}

// The statistics of a workgroup's `tiles` tiles, `step` apart, each of its four waves' joined.
template <int ROWS, int N>
__device__ __forceinline__ void aw_publish(const AwParams& p, const AwProg& x, int prog, int tile0, int step, int tiles,
                                           const uint64_t (&st)[N][4][ROWS]) {
  for (int i = threadIdx.x; i < tiles * x.rows; i += 256) {
    const int tile = i / x.rows, row = i - tile * x.rows;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) aw_join(m, l, aw_m(st[tile][v][row]), aw_l(st[tile][v][row]));
    publish(p.stats + ((int64_t)prog * p.tiles + tile0 + tile * step) * p.rows + row, aw_pack(m, l));
  }
}

// Up to 64 rows.  A workgroup walks up to `span` tiles of a program, a wave 64 tokens of each, with the next tile's codes on
// their way while one is multiplied; all rows' queries wait in LDS.  The tiles lie as far apart as the program has workgroups, so
// that a context shorter than the table is shared out to all of them and their pages can be looked up before its length is known:
// 9 tokens at 4096 in a table of 131072, 8 sequences: 42 us (side by side 50), one: 19 (45).  Stored scores are written side by
// side: tiles apart took 55 us for 53 where the workgroups are many enough.
template <int D, typename ST, int MODE>
__global__ __launch_bounds__(256, 2) void aw_few_kernel(AwParams p) {
  constexpr int NU = D / 32, RB = kAwFewRows / 16;
  __shared__ v8h s_q[RB][NU][64];
  __shared__ AwStage<D> s_k[4];
  __shared__ float s_scale[4][64];
  __shared__ uint64_t s_stat[MODE == kAwSums ? 1 : kAwSpan][4][MODE == kAwSums ? 1 : kAwFewRows];
  __shared__ int s_last;
  const int lane = lane_id(), w = uniform(wave_id()), r = lane & 15, g = lane >> 4;
  const int progs = p.B_grid * p.H_KV, spans = (p.tiles + p.span - 1) / p.span;
  int64_t live = (int64_t)progs * spans;
  for (int64_t item = blockIdx.x; item < live; item += gridDim.x, live = aw_live(p, item, live, progs, 1)) {
    const int tile0 = (int)(item / progs), prog = aw_order(p, (int)(item % progs));
    // The wave's sub-tile `lane` and its page, whose load does not wait for the context's length.
    const int sub_t = (tile0 + min(lane / 4, p.span - 1) * spans) * kAwTile + 64 * w + 16 * (lane & 3);
    int page = -1;
    if (lane < 4 * p.span && sub_t < p.cap) page = p.bt[(int64_t)(prog / p.H_KV) * p.s_bt + sub_t / p.PAGE];
    AwProg x;
    if (!aw_prog(p, prog, x) || tile0 >= x.tiles) continue;
    const int blocks = (x.rows + 15) / 16;
    __syncthreads();  // the last item's queries have been read
    for (int f = threadIdx.x; f < blocks * NU * 64; f += 256) {
      const int l = f % 64, u = (f / 64) % NU, row = min(f / (64 * NU) * 16 + (l & 15), x.rows - 1);
      const int qi = aw_token(p, row), head = x.h * p.G + row - qi * p.G;
      s_q[0][0][f] = *reinterpret_cast<const v8h*>(p.q + x.b * p.s_qb + qi * p.s_qt + head * p.s_qh + 64 * (u / 2) + 16 * (l >> 4) +
                                                   8 * (u & 1));
    }
    const int fresh = x.L - x.ql;  // a row of new token i sees t <= fresh + i
    const AwPages at = aw_pages(p, x, sub_t, page, lane < 4 * p.span);
    v4i raw[4][D / 64];
    ST scale;
    aw_load<D, false, ST>(p, at, 0, raw, scale);
    uint64_t norm[MODE == kAwSums ? RB : 1];
    if constexpr (MODE == kAwSums) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        norm[rb] = aw_pack(INFINITY, 0.f);
        if (rb * 16 + r < x.rows) norm[rb] = p.norms[(int64_t)prog * p.rows + rb * 16 + r];
      }
    }
    __syncthreads();
    for (int n = 0, tile = tile0; tile < x.tiles; ++n, tile += spans) {
      const int t0 = tile * kAwTile + 64 * w;
      const uint32_t seen = (uint32_t)(at.ok >> (4 * n)) & 0xf;
      // Lane (r, g) holds the scale of token t0 + 16 g + r; it needs those of tokens 16 s + 4 g + i.
      s_k[w].put(raw);
      s_scale[w][lane] = (float)scale * p.scale_log2;
      aw_load<D, false, ST>(p, at, 4 * (n + 1), raw, scale);
      wait_lgkm0();
      v8h kh[4][NU];
#pragma unroll
      for (int s = 0; s < 4; ++s) s_k[w].get(s, kh[s]);
      v4f ksc[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) ksc[s] = *reinterpret_cast<const v4f*>(&s_scale[w][16 * s + 4 * g]);
      v4f even[4], odd[4];  // sums over the blocks of either parity
#pragma unroll
      for (int s = 0; s < 4; ++s) even[s] = odd[s] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (rb >= blocks) break;
        const int row = rb * 16 + r;
        v8h qf[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) qf[u] = s_q[rb][u][lane];
        v4f acc[4];
        // Rows past the last add nothing: their statistics go nowhere, their max is infinite.
        aw_scores<D, MODE == kAwSums>(kh, qf, ksc, t0, fresh + aw_token(p, row), t0 + 63 <= fresh && seen == 0xf, seen,
                                      MODE == kAwSums ? aw_m(norm[rb]) : 0.f, acc);
        if constexpr (MODE == kAwSums) {
#pragma unroll
          for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v4f& sum = (rb & 1 ? odd : even)[s];
              sum[i] = fmaf(fast_exp2(acc[s][i]), aw_l(norm[rb]), sum[i]);
            }
        } else {
          const uint64_t st = aw_stat(acc);
          if (g == 0) s_stat[n][w][row] = st;
        }
      }
      if constexpr (MODE == kAwSums) {
#pragma unroll
        for (int s = 0; s < 4; ++s) even[s] += odd[s];
        const v4f got = aw_rows(even);
        if (const int t = aw_first(t0); r < 4 && t < x.L) aw_put(p, x, t, aw_get(p, x, t, true) + got);
      }
    }
    if constexpr (MODE != kAwSums) {
      __syncthreads();
      aw_publish(p, x, prog, tile0, spans, (x.tiles - tile0 + spans - 1) / spans, s_stat);
      if (arrive_last(p.counters + prog, min(spans, x.tiles), &s_last)) aw_norms(p, x, prog);
    }
  }
}

// Up to 16 rows, whose scores are stored: one block of rows, so a sub-tile's operands are made where they are used.
template <int D, typename ST>
__global__ __launch_bounds__(256) void aw_store_kernel(AwParams p) {
  constexpr int NU = D / 32;
  constexpr bool kOnce = D == 128;  // nothing reads the lines again; at D = 64 the next head does
  __shared__ AwStage<D> s_k[4];
  __shared__ float s_scale[4][64];
  __shared__ uint64_t s_stat[kAwSpan][4][16];
  __shared__ int s_last;
  const int lane = lane_id(), w = uniform(wave_id()), r = lane & 15, g = lane >> 4;
  const int progs = p.B_grid * p.H_KV, spans = (p.tiles + p.span - 1) / p.span;
  int64_t live = (int64_t)progs * spans;
  for (int64_t item = blockIdx.x; item < live; item += gridDim.x, live = aw_live(p, item, live, progs, p.span)) {
    const int tile0 = (int)(item / progs) * p.span, prog = aw_order(p, (int)(item % progs));
    const int sub_t = (tile0 + lane / 4) * kAwTile + 64 * w + 16 * (lane & 3);
    int page = -1;
    if (lane < 4 * p.span && sub_t < p.cap) page = p.bt[(int64_t)(prog / p.H_KV) * p.s_bt + sub_t / p.PAGE];
    AwProg x;
    if (!aw_prog(p, prog, x) || tile0 >= x.tiles) continue;
    const int tile1 = min(tile0 + p.span, x.tiles), fresh = x.L - x.ql;
    v8h qf[NU];
    {
      const int row = min(r, x.rows - 1), qi = aw_token(p, row), head = x.h * p.G + row - qi * p.G;
      const _Float16* src = p.q + x.b * p.s_qb + qi * p.s_qt + head * p.s_qh + 16 * g;
#pragma unroll
      for (int u = 0; u < NU; ++u) qf[u] = *reinterpret_cast<const v8h*>(src + 64 * (u / 2) + 8 * (u & 1));
    }
    const int last = fresh + aw_token(p, r);  // the last token the lane's row sees
    const AwPages at = aw_pages(p, x, sub_t, page, lane < 4 * p.span);
    const rsrc_t out = make_rsrc(p.scores + (int64_t)prog * p.rows * p.tiles * kAwTile, kOOB);
    const uint32_t out_row = oob_unless(r < x.rows, (uint32_t)(r * p.tiles * kAwTile + 4 * g) * 4);
    v4i raw[4][D / 64];
    ST scale;
    aw_load<D, kOnce, ST>(p, at, 0, raw, scale);
    for (int tile = tile0; tile < tile1; ++tile) {
      const int t0 = tile * kAwTile + 64 * w;
      const uint32_t seen = (uint32_t)(at.ok >> (4 * (tile - tile0))) & 0xf;
      s_k[w].put(raw);
      s_scale[w][lane] = (float)scale * p.scale_log2;
      aw_load<D, kOnce, ST>(p, at, 4 * (tile + 1 - tile0), raw, scale);
      wait_lgkm0();
      v4f acc[4], ksc[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        v8h kh[NU];
        s_k[w].get(s, kh);
        acc[s] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < NU; ++u) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[u], qf[u], acc[s], 0, 0, 0);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) ksc[s] = *reinterpret_cast<const v4f*>(&s_scale[w][16 * s + 4 * g]);
      aw_scale<false>(ksc, 0.f, acc);
      const bool all = t0 + 63 <= fresh && seen == 0xf;
      if (!all) aw_hide(t0, last, seen, acc);  // rows past the last go nowhere
      const uint64_t st = aw_stat(acc);
      // What is seen is stored as finite, what is not as -inf, which adds nothing even to a row whose max is NaN.
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[s][i] = fmaxf(acc[s][i], -3.402823466e38f);
      if (!all) aw_hide(t0, last, seen, acc);
      // Always the same stores, too; those of tokens behind the context lie in the row's last tile.
#pragma unroll
      for (int s = 0; s < 4; ++s)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, acc[s]), out, out_row + 4u * (uint32_t)(t0 + 16 * s), 0, 0);
      if (g == 0) s_stat[tile - tile0][w][r] = st;
    }
    __syncthreads();
    aw_publish(p, x, prog, tile0, 1, tile1 - tile0, s_stat);
    if (arrive_last(p.counters + prog, (x.tiles + p.span - 1) / p.span, &s_last)) aw_norms(p, x, prog);
  }
}

// More rows: a workgroup owns a tile, its waves 64 tokens and the row blocks of one parity each.  64 rows' queries at a time
// come through LDS, whole rows a load, while the 64 before are multiplied.  Loaded by each wave as its matrix operands,
// nearly every lane's 16 bytes were an access of their own: 2 x 256 tokens, 32 / 8 heads of 128, contexts of 4096 and less
// took 77 us in both launches instead of 69.  At two waves a SIMD (K's operands are 64 registers, and the shared memory has room
// for one workgroup a CU) the vector instructions have 61 % of a busy CU's cycles and the matrix ones 25 %, 30 % of which have
// vector ones beside them.  Put between one another by hand, 45 % had, and the sums took 35 us where they had taken 31.
template <int D, typename ST, int MODE>
__global__ __launch_bounds__(512) void aw_many_kernel(AwParams p) {
  constexpr int NU = D / 32, GQ = D / 8, kLoads = 64 * GQ / 512;  // 16-byte granules of a query row; loads of a thread
  __shared__ AwStage<D> s_k[8];
  __shared__ v8h s_q[2][64][GQ];
  __shared__ float s_scale[8][64];
  __shared__ uint64_t s_stat[MODE == kAwSums ? 1 : 4][MODE == kAwSums ? 1 : kAwSeg * 16];
  __shared__ v4f s_sums[MODE == kAwSums ? 4 : 1][4][64];
  __shared__ int s_last;
  const int lane = lane_id(), w = uniform(wave_id()) & 3, odd = uniform(wave_id()) >> 2, r = lane & 15, g = lane >> 4;
  // Granule q of row t lies in slot q ^ key(t): 16 rows' granules meet in no bank.
  auto key = [](int t) { return D == 128 ? t & 15 : (t >> 1) & 7; };
  const int progs = p.B_grid * p.H_KV, per = p.segs * progs;
  int64_t live = (int64_t)per * p.tiles;
  for (int64_t item = blockIdx.x; item < live; item += gridDim.x, live = aw_live(p, item, live, per, 1)) {
    const int tile = (int)(item / per), some = (int)(item % per), seg_i = some / progs, row0 = p.row0 + seg_i * p.seg_rows;
    const int prog = aw_order(p, some - seg_i * progs), index = prog * p.segs + seg_i, t0 = tile * kAwTile + 64 * w;
    AwProg x;
    if (!aw_prog(p, prog, x, row0) || tile >= x.tiles) continue;
    // The segment's last row sees its tiles up to this one.
    const int last_t = x.L - x.ql + aw_token(p, row0 + x.rows - 1);
    x.tiles = last_t < 0 ? 0 : last_t / kAwTile + 1;
    if (tile >= x.tiles) continue;
    const int sub_t = t0 + 16 * (lane & 3);
    const AwPages at = aw_pages(p, x, sub_t, sub_t < x.L ? p.bt[x.b * p.s_bt + sub_t / p.PAGE] : -1, lane < 4);
    const uint32_t seen = (uint32_t)at.ok;
    v4i raw[4][D / 64];
    ST scale;
    aw_load<D, false, ST>(p, at, 0, raw, scale);
    s_k[4 * odd + w].put(raw);
    s_scale[4 * odd + w][lane] = (float)scale * p.scale_log2;
    wait_lgkm0();
    v8h kh[4][NU];
#pragma unroll
    for (int s = 0; s < 4; ++s) s_k[4 * odd + w].get(s, kh[s]);
    v4f ksc[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) ksc[s] = *reinterpret_cast<const v4f*>(&s_scale[4 * odd + w][16 * s + 4 * g]);
    const int fresh = x.L - x.ql, blocks = (x.rows + 15) / 16;
    v4f sums[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) sums[s] = v4f{0.f, 0.f, 0.f, 0.f};
    // Segments of this launch that have rows which see the tile, from the first such row on; the weights so far of the lane's
    // tokens, where no other workgroup adds to them.
    const int first_row = max(tile * kAwTile - fresh, 0) * p.G, seg0 = max(first_row - p.row0, 0) / p.seg_rows;
    const int seg1 = min(p.segs, (x.ql * p.G - p.row0 + p.seg_rows - 1) / p.seg_rows), my_t = aw_first(t0);
    const bool alone = seg1 - seg0 == 1, start = first_row >= p.row0, mine = !odd && r < 4 && my_t < x.L;
    auto words = [&](int unit, int t) {  // of the launch
      return p.sums + (((int64_t)prog * (p.segs * p.seg_rows / kAwUnitRows) + unit) * p.tiles * kAwTile + t) / 2;
    };
    v4f weight = {0.f, 0.f, 0.f, 0.f};
    if (MODE == kAwSums && alone && mine) weight = aw_get(p, x, my_t, start);
    // The first row block that sees token t.
    auto first_of = [&](int t) { return t > fresh ? min(max((t - fresh) * p.G - row0, 0) / 16, blocks) : 0; };
    int rb = first_of(tile * kAwTile) & ~3;  // four blocks at a time, from the first that sees the tile's first token
    // A thread's rows of the blocks to be fetched.  Their places go on by 64 rows: products for each cost 1 us of 32.
    const int step_q = 64 / p.G, step_h = 64 - step_q * p.G;
    const _Float16* const q0 = p.q + x.b * p.s_qb + x.h * p.G * p.s_qh + 8 * (threadIdx.x % GQ);
    auto place = [&](int row, int& head) {
      const int qi = aw_token(p, row0 + row);
      head = row0 + row - qi * p.G;
      return q0 + qi * p.s_qt + head * p.s_qh;
    };
    int head[kLoads], row[kLoads], last_head;
    const _Float16 *from[kLoads], *const end = place(x.rows - 1, last_head);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      row[n] = rb * 16 + ((int)threadIdx.x + 512 * n) / GQ;
      from[n] = place(row[n], head[n]);
    }
    v8h next[kLoads];
    uint64_t next_norm[2] = {0, 0};
    auto fetch = [&](int b) {  // what four blocks need; past the last row, that row
#pragma unroll
      for (int n = 0; n < kLoads; ++n) {
        next[n] = *reinterpret_cast<const v8h*>(row[n] < x.rows ? from[n] : end);
        row[n] += 64;
        head[n] += step_h;
        from[n] += step_q * p.s_qt + step_h * p.s_qh;
        if (head[n] >= p.G) {
          head[n] -= p.G;
          from[n] += p.s_qt - p.G * p.s_qh;
        }
      }
      if constexpr (MODE == kAwSums) {
#pragma unroll
        for (int k = 0; k < 2; ++k) next_norm[k] = p.norms[(int64_t)index * p.rows + min((b + odd + 2 * k) * 16 + r, x.rows - 1)];
      }
    };
    int slot = 0;
    auto stage = [&] {
#pragma unroll
      for (int n = 0; n < kLoads; ++n) {
        const int i = (int)threadIdx.x + 512 * n, t = i / GQ;
        s_q[slot][t][(i % GQ) ^ key(t)] = next[n];
      }
    };
    constexpr int kSeg = MODE == kAwSums ? 1 << 30 : kAwSeg;  // sums need no segments
    int seg = 0, seg_end = 0;
    auto keep = [&](int b, uint64_t st) {
      if constexpr (MODE != kAwSums)
        if (g == 0 && b < seg_end) s_stat[w][(b - seg) * 16 + r] = st;
    };
    if (rb < blocks) fetch(rb);
    for (; seg < blocks; seg += kSeg) {
      seg_end = min(seg + kSeg, blocks);
      if constexpr (MODE != kAwSums)
        for (int b = seg + odd; b < min(rb, seg_end); b += 2) keep(b, aw_pack(-INFINITY, 0.f));
      for (; rb < seg_end; rb += 4, slot ^= 1) {
        stage();
        const uint64_t norm[2] = {next_norm[0], next_norm[1]};
        fetch(rb + 4);
        wg_barrier_lds();  // the other slot has been read, and is written next
        v4f acc[2][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int b = rb + odd + 2 * k, at = b * 16 + r;  // rows past the last see nothing
          v8h qf[NU];
#pragma unroll
          for (int u = 0; u < NU; ++u) qf[u] = s_q[slot][(odd + 2 * k) * 16 + r][(8 * (u / 2) + 2 * g + (u & 1)) ^ key(r)];
          aw_scores<D, MODE == kAwSums>(kh, qf, ksc, t0, at < x.rows ? fresh + aw_token(p, row0 + at) : -1,
                                        t0 + 63 <= fresh && seen == 0xf && b * 16 + 16 <= x.rows, seen, aw_m(norm[k]), acc[k]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if constexpr (MODE == kAwSums) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i) sums[s][i] = fmaf(fast_exp2(acc[k][s][i]), aw_l(norm[k]), sums[s][i]);
          } else {
            keep(rb + odd + 2 * k, aw_stat(acc[k]));
          }
        }
        if constexpr (MODE == kAwSums) {
          if (rb + 4 >= blocks || (rb + 4) % (kAwUnitRows / 16) == 0) {  // a unit ends: both parities, then the lanes
            if (odd) {
#pragma unroll
              for (int s = 0; s < 4; ++s) s_sums[w][s][lane] = sums[s];
            }
            wg_barrier_lds();
            if (!odd) {
#pragma unroll
              for (int s = 0; s < 4; ++s) sums[s] += s_sums[w][s][lane];
              const v4f got = aw_rows(sums);
              weight += got;
              if (r < 4 && !alone) {
                uint64_t* to = words((row0 - p.row0 + rb * 16) / kAwUnitRows, my_t);
                publish(to, aw_pack(got[0], got[1]));
                publish(to + 1, aw_pack(got[2], got[3]));
              }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) sums[s] = v4f{0.f, 0.f, 0.f, 0.f};
          }
        }
      }
      if constexpr (MODE != kAwSums) {
        __syncthreads();
        const int n = min((seg_end - seg) * 16, x.rows - seg * 16);
        for (int i = threadIdx.x; i < n; i += 512) {
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) aw_join(m, l, aw_m(s_stat[v][i]), aw_l(s_stat[v][i]));
          publish(p.stats + ((int64_t)index * p.tiles + tile) * p.rows + seg * 16 + i, aw_pack(m, l));
        }
        __syncthreads();
      }
    }
    if constexpr (MODE == kAwSums) {
      if (alone) {
        if (mine) aw_put(p, x, my_t, weight);
        __syncthreads();
      } else if (arrive_last(p.counters + per + (int64_t)prog * p.tiles + tile, seg1 - seg0, &s_last)) {
        // The last of the tile's workgroups adds the units up in their order.
        const int unit1 = (min(x.ql * p.G - p.row0, p.segs * p.seg_rows) + kAwUnitRows - 1) / kAwUnitRows;
        const int t = tile * kAwTile + 4 * (int)threadIdx.x;
        if (threadIdx.x < kAwTile / 4 && t < x.L) {
          v4f v = aw_get(p, x, t, start);
          for (int unit = max(first_row - p.row0, 0) / kAwUnitRows; unit < unit1; ++unit) {
            const uint64_t a = collect(words(unit, t)), b = collect(words(unit, t) + 1);
            v += v4f{aw_m(a), aw_l(a), aw_m(b), aw_l(b)};
          }
          aw_put(p, x, t, v);
        }
      }
    } else if (arrive_last(p.counters + index, x.tiles, &s_last)) {
      aw_norms(p, x, index);
    }
  }
}

// Pass 2 from stored scores of up to R rows: a thread owns four tokens, and adds their rows in the order of the lanes above.  32
// sequences of up to 8192, 4 rows: 7.6 us with R = 4, 12 with 16.
template <int R>
__device__ __forceinline__ void aw_sum(const AwParams& p, const AwProg& x, int prog, int t) {
#pragma clang fp contract(off)  // a probability is rounded before it is added, as the first addition to nothing does it above
  const float* sc = p.scores + (int64_t)prog * p.rows * p.tiles * kAwTile + t;
  v4f e[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    e[k] = v4f{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (k < x.rows) e[k] = *reinterpret_cast<const v4f*>(sc + (int64_t)k * p.tiles * kAwTile);
  }
  float top[R], inv[R];
  bool nan = false;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const uint64_t norm = k < x.rows ? p.norms[(int64_t)prog * p.rows + k] : aw_pack(INFINITY, 0.f);
    top[k] = aw_m(norm), inv[k] = aw_l(norm);
    nan |= !(top[k] == top[k]);
  }
  if (uniform((int)nan)) {  // a row gives its NaN to what it sees alone
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(top[k] == top[k]) && !(e[k][i] == -INFINITY)) e[k][i] = top[k];
#pragma unroll
    for (int k = 0; k < R; ++k)
      if (!(top[k] == top[k])) top[k] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < R; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) e[k][i] = fast_exp2(e[k][i] - top[k]) * inv[k];
  // Pairs, pairs of these, and the fours.
#pragma unroll
  for (int o = 1; o < R; o *= 2)
#pragma unroll
    for (int k = 0; k + o < R; k += 2 * o) e[k] += e[k + o];
  aw_put(p, x, t, aw_get(p, x, t, true) + e[0]);
}

template <int R>
__global__ __launch_bounds__(256, 4) void aw_sum_kernel(AwParams p) {
  const int progs = p.B_grid * p.H_KV, tiles = (p.cap + kAwSumTile - 1) / kAwSumTile;
  int64_t live = (int64_t)progs * tiles;
  for (int64_t item = blockIdx.x; item < live; item += gridDim.x, live = aw_live(p, item, live, progs, kAwSumTile / kAwTile)) {
    const int tile = (int)(item / progs), prog = (int)(item - (int64_t)tile * progs);
    AwProg x;
    const int t = tile * kAwSumTile + 4 * (int)threadIdx.x;
    if (!aw_prog(p, prog, x)) continue;
    if (t < x.L) aw_sum<R>(p, x, prog, t);
  }
}

template <int MODE>
static const void* aw_fn(int D, bool f32, bool few) {
  if (D == 64) {
    if (f32) return few ? reinterpret_cast<const void*>(&aw_few_kernel<64, float, MODE>)
                        : reinterpret_cast<const void*>(&aw_many_kernel<64, float, MODE>);
    return few ? reinterpret_cast<const void*>(&aw_few_kernel<64, _Float16, MODE>)
               : reinterpret_cast<const void*>(&aw_many_kernel<64, _Float16, MODE>);
  }
  if (f32) return few ? reinterpret_cast<const void*>(&aw_few_kernel<128, float, MODE>)
                      : reinterpret_cast<const void*>(&aw_many_kernel<128, float, MODE>);
  return few ? reinterpret_cast<const void*>(&aw_few_kernel<128, _Float16, MODE>)
             : reinterpret_cast<const void*>(&aw_many_kernel<128, _Float16, MODE>);
}
static const void* aw_sum_fn(int64_t rows) {
  if (rows <= 4) return reinterpret_cast<const void*>(&aw_sum_kernel<4>);
  return rows <= 8 ? reinterpret_cast<const void*>(&aw_sum_kernel<8>) : reinterpret_cast<const void*>(&aw_sum_kernel<16>);
}
static const void* aw_store_fn(int D, bool f32) {
  if (D == 64) return f32 ? reinterpret_cast<const void*>(&aw_store_kernel<64, float>)
                          : reinterpret_cast<const void*>(&aw_store_kernel<64, _Float16>);
  return f32 ? reinterpret_cast<const void*>(&aw_store_kernel<128, float>)
             : reinterpret_cast<const void*>(&aw_store_kernel<128, _Float16>);
}

// Whether scores are stored, the sequences of a launch, rows and segments as in AwParams, bytes.
struct AwSpace { bool store; int64_t seqs, seg_rows, segs, rows; size_t scores, stats, norms, sums; };
static AwSpace aw_space(int64_t B, int64_t H_KV, int64_t rows, int64_t tiles) {
  AwSpace a = {};
  // Two units a workgroup, or one where that fills no more than the GPU.  256 tokens at 4096, 8 heads of 4 queries, one sequence:
  // 68 us, 45; two (twice as many workgroups as CUs): 78, 83.
  a.seg_rows = kAwUnitRows * (B * H_KV * tiles * ceil_div64(rows, kAwUnitRows) <= kAwFill ? 1 : kAwSegUnits);
  a.rows = rows < a.seg_rows ? rows : a.seg_rows;
  // Scores of one sequence, where they are stored (those of a program lie within a buffer's offsets by that), and all it needs.
  const int64_t norms = H_KV * a.rows * (tiles + 1) * 8, scores = H_KV * rows * tiles * kAwTile * 4;
  a.store = rows <= kAwStoreRows && norms + scores <= kAwMost;
  const int64_t one = norms + (a.store ? scores : 0), most = one < kAwMost ? kAwMost / one : 1;
  a.seqs = ceil_div64(B, ceil_div64(B, most));  // turns of much the same size
  const int64_t progs = a.seqs * H_KV;
  a.scores = a.store ? align_up((size_t)(a.seqs * scores), 256) : 0;
  // As many segments as there are, where their counters, and they, find room.
  const int64_t segs = ceil_div64(rows, a.seg_rows);
  for (a.segs = segs < kAwSegs ? segs : kAwSegs;; --a.segs) {
    a.stats = align_up((size_t)(a.segs * progs * tiles * a.rows * 8), 256);
    a.norms = align_up((size_t)(a.segs * progs * a.rows * 8), 256);
    a.sums = a.segs > 1 ? (size_t)(a.segs * (a.seg_rows / kAwUnitRows) * progs * tiles * kAwTile * 4) : 0;
    if (a.segs <= 1 || (progs * (a.segs + tiles) * 4 <= (int64_t)kCounterBytes && a.stats + a.norms + a.sums <= (size_t)kAwMost)) return a;
  }
}

}  // namespace specq

using namespace specq;

extern "C" size_t specq_paged_attn_weights_workspace_size(int B_grid, int H, int H_KV, int ql_grid, int max_pages,
                                                          int PAGE) {
  if (B_grid <= 0 || H <= 0 || H_KV <= 0 || H % H_KV != 0 || ql_grid <= 0 || max_pages <= 0 || PAGE <= 0) return 0;
  const AwSpace s = aw_space(B_grid, H_KV, (int64_t)ql_grid * (H / H_KV), ceil_div64((int64_t)max_pages * PAGE, kAwTile));
  return kCounterBytes + s.scores + s.stats + s.norms + s.sums;
}

extern "C" int specq_paged_attn_weights(const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const int8_t* kc,
                                        int64_t s_kp, int64_t s_ko, int64_t s_kh, const void* ks, int64_t s_sp,
                                        int64_t s_so, int64_t s_sh, int scale_fp32, const int32_t* block_tbl,
                                        int64_t s_bt, int max_pages, int n_pages, const int32_t* ctx_len,
                                        const int32_t* q_lens, float* weights, int64_t s_wb, int64_t s_wh, int B_grid,
                                        int n_seqs, int q_len, int ql_grid, int H, int H_KV, int D, int PAGE,
                                        float sm_scale, const int32_t* plan, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  clear_error();
  SPECQ_REQUIRE(q && kc && ks && block_tbl && ctx_len && weights, SPECQ_EINVAL, "paged_attn_weights: null tensor pointer");
  SPECQ_REQUIRE(B_grid >= 0 && ql_grid >= 0 && n_seqs >= 0 && n_seqs <= B_grid && q_len >= 0 && q_len <= ql_grid,
                SPECQ_EINVAL, "paged_attn_weights: need 0 <= n_seqs <= B_grid and 0 <= q_len <= ql_grid");
  SPECQ_REQUIRE(H > 0 && H_KV > 0 && H % H_KV == 0, SPECQ_EINVAL, "paged_attn_weights: %d heads do not fit %d KV heads", H, H_KV);
  SPECQ_REQUIRE(max_pages > 0 && n_pages > 0 && PAGE > 0 && s_bt >= max_pages, SPECQ_EINVAL, "paged_attn_weights: bad sizes");
  SPECQ_REQUIRE(D == 64 || D == 128, SPECQ_ENOTSUP, "paged_attn_weights: head_dim %d must be 64 or 128", D);
  SPECQ_REQUIRE(PAGE % 16 == 0, SPECQ_ENOTSUP, "paged_attn_weights: PAGE %d must be a multiple of 16", PAGE);
  const int64_t cap = (int64_t)max_pages * PAGE, progs = (int64_t)B_grid * H_KV, rows = (int64_t)ql_grid * (H / H_KV);
  SPECQ_REQUIRE(cap <= (1 << 30), SPECQ_ENOTSUP, "paged_attn_weights: a table of %lld tokens is too long", (long long)cap);
  SPECQ_REQUIRE(H / H_KV < 4096, SPECQ_ENOTSUP, "paged_attn_weights: %d query heads to a KV head", H / H_KV);
  SPECQ_REQUIRE(rows <= (1 << 20) && ql_grid <= (1 << 20), SPECQ_ENOTSUP, "paged_attn_weights: too many query rows");
  SPECQ_REQUIRE(progs <= kMaxCounters, SPECQ_ENOTSUP, "paged_attn_weights: more than %lld sequences x KV heads",
                (long long)kMaxCounters);
  SPECQ_REQUIRE((uintptr_t)q % 16 == 0 && s_qb % 8 == 0 && s_qt % 8 == 0 && s_qh % 8 == 0, SPECQ_ENOTSUP,
                "paged_attn_weights: q rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)kc % 16 == 0 && s_kp % 16 == 0 && s_ko % 16 == 0 && s_kh % 16 == 0, SPECQ_ENOTSUP,
                "paged_attn_weights: cache rows must be 16-byte aligned");
  SPECQ_REQUIRE(s_ko < (1ll << 27) && s_ko >= 0, SPECQ_ENOTSUP, "paged_attn_weights: tokens %lld bytes apart", (long long)s_ko);
  SPECQ_REQUIRE((uintptr_t)ks % (scale_fp32 ? 4 : 2) == 0 && (uintptr_t)weights % 4 == 0, SPECQ_EINVAL,
                "paged_attn_weights: scales and weights must be aligned to their type");
  SPECQ_REQUIRE(nest_apart({{B_grid, s_wb}, {H_KV, s_wh}}, cap), SPECQ_ENOTSUP,
                "paged_attn_weights: rows of the weights overlap or are shorter than the table's %lld tokens", (long long)cap);
  if (B_grid == 0 || ql_grid == 0) return SPECQ_OK;
  AwParams p = {};
  p.q = (const _Float16*)q; p.s_qb = s_qb; p.s_qt = s_qt; p.s_qh = s_qh;
  p.kc = kc; p.s_kp = s_kp; p.s_ko = s_ko; p.s_kh = s_kh;
  p.ks = ks; p.s_sp = s_sp; p.s_so = s_so; p.s_sh = s_sh;
  p.bt = block_tbl; p.s_bt = s_bt; p.max_pages = max_pages; p.n_pages = n_pages;
  p.ctx_len = ctx_len; p.q_lens = q_lens;
  p.w = weights; p.s_wb = s_wb; p.s_wh = s_wh;
  p.w_vec = (uintptr_t)weights % 16 == 0 && s_wb % 4 == 0 && s_wh % 4 == 0;
  p.plan = plan; p.q_len = q_len; p.ql_grid = ql_grid;
  p.G = H / H_KV; p.g_magic = p.G > 1 ? (uint32_t)(((1ull << 32) + p.G - 1) / p.G) : 0;
  p.H_KV = H_KV; p.PAGE = PAGE;
  p.cap = (int)cap; p.tiles = (int)ceil_div64(cap, kAwTile);
  p.scale_log2 = sm_scale * 1.44269504088896340736f;
  const AwSpace space = aw_space(B_grid, H_KV, rows, p.tiles);
  p.rows = (int)space.rows;
  p.seg_rows = (int)space.seg_rows;
  p.segs = (int)space.segs;
  const size_t need = kCounterBytes + space.scores + space.stats + space.norms + space.sums;
  SPECQ_REQUIRE(workspace && workspace_bytes >= need, SPECQ_ENOSPC,
                "paged_attn_weights: workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  char* at = static_cast<char*>(workspace);
  p.counters = reinterpret_cast<int32_t*>(at);
  p.scores = reinterpret_cast<float*>(at + kCounterBytes);
  p.stats = reinterpret_cast<uint64_t*>(at + kCounterBytes + space.scores);
  p.norms = reinterpret_cast<uint64_t*>(at + kCounterBytes + space.scores + space.stats);
  p.sums = reinterpret_cast<uint64_t*>(at + kCounterBytes + space.scores + space.stats + space.norms);
  // Stored scores against scores formed twice (us, 8 KV heads of 128, tables as wide as the contexts):
  //           8 x 4096      32 x 8192     1 x 32768     32 x 1024
  //    4 rows 17.7, 23.3    81.5, 111.5   19.7, 29.1    17.2, 21.9
  //   12      24.1, 23.4    103, 114      25.1, 31.5    24.4, 22.8
  //   16      27.4, 23.2    122, 114      27.9, 32.5    25.1, 22.4
  // At 16 either gains as often as it loses, by as much; one sequence gains the most.
  // Queries in LDS for the whole call against 64 rows at a time: 20 rows, 8 of 4096: 28.7, 58.6; 64 rows: 37.7, 58.5; one of
  // 32768: 54, 69.
  const bool store = space.store, few = rows <= kAwFewRows, f32 = scale_fp32 != 0;
  for (; p.b0 < B_grid; p.b0 += (int)space.seqs) {
    p.B_grid = (int)(B_grid - p.b0 < space.seqs ? B_grid - p.b0 : space.seqs);
    p.n_seqs = n_seqs < p.b0 ? 0 : n_seqs - p.b0 < p.B_grid ? n_seqs - p.b0 : p.B_grid;
    const int64_t some = (int64_t)p.B_grid * H_KV;
    // Tiles of a workgroup of few rows: as many as leave two workgroups to a CU.
    const int64_t tiles = some * p.tiles, span = tiles / (2 * device_cus());
    p.span = few ? (int)(span < 1 ? 1 : span > kAwSpan ? kAwSpan : span) : 1;
    const int64_t items = some * ceil_div(p.tiles, p.span) * p.segs, sums = some * ceil_div64(cap, kAwSumTile);
    const int threads = few ? 256 : 512, cus = device_cus();
    const int grid = (int)std::min<int64_t>(items, (few ? kAwFewGrid : kAwManyGrid) * cus);
    for (p.row0 = 0; p.row0 < rows; p.row0 += p.segs * p.seg_rows) {
      if (int rc = launch(store ? aw_store_fn(D, f32) : aw_fn<kAwStats>(D, f32, few), grid, threads, 0, (hipStream_t)stream, &p))
        return rc;
      const int rc = store ? launch(aw_sum_fn(rows), (int)std::min<int64_t>(sums, kAwSumGrid * cus), 256, 0, (hipStream_t)stream, &p)
                           : launch(aw_fn<kAwSums>(D, f32, few), grid, threads, 0, (hipStream_t)stream, &p);
      if (rc != SPECQ_OK) return rc;
    }
    p.q += space.seqs * s_qb;
    p.bt += space.seqs * s_bt;
    p.ctx_len += space.seqs;
    if (p.q_lens != nullptr) p.q_lens += space.seqs;
    p.w += space.seqs * s_wb;
  }
  return SPECQ_OK;
}
