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
//      joins them to log2 of each row's sum over all tiles
//   2  p = exp2(s - that), summed over the rows, and the update of w
// The scores of up to 16 rows (kAwStoreRows: plain decoding) go from 1 to 2 through the workspace; more rows compute them again.  Both ways
// add a token's rows in one order (16 lanes, rows 16 apart in each lane, then pairs of lanes), so they give the same
// bits, and a plan-mode call those of an eager one.
//
// K stays: a wave owns 64 tokens, converts their codes to fp16 matrix operands once and walks the rows 16 at a time
// (K . Q^T on v_mfma_f32_16x16x32_f16: a lane's results are four tokens of one row).  Everything behind the products is
// fp32; log2(e) is folded into the scale.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kAwTile = 256;       // tokens of a workgroup: 4 waves of 4 sub-tiles of 16
constexpr int kAwStoreRows = 16;   // rows whose scores go through the workspace
constexpr int kAwSeg = 32;         // row blocks of 16 whose statistics are joined at a time
constexpr int kAwSumTile = 1024;   // tokens of a workgroup that adds up stored scores
constexpr int kAwMaxGrid = 1 << 16;

struct AwParams {
  const _Float16* q; int64_t s_qb, s_qt, s_qh;
  const int8_t* kc; int64_t s_kp, s_ko, s_kh;
  const void* ks; int64_t s_sp, s_so, s_sh;
  const int32_t* bt; int64_t s_bt; int max_pages, n_pages;
  const int32_t* ctx_len; const int32_t* q_lens;
  float* w; int64_t s_wb, s_wh; int w_vec;  // w_vec: its rows are 16-byte aligned
  const int32_t* plan;
  int n_seqs, q_len, B_grid, ql_grid, G, H_KV, PAGE;
  int cap;      // tokens a row of the table holds
  int tiles;    // of cap
  int rows;     // of a program at most: ql_grid * G
  float scale_log2;
  // Workspace: scores [prog][rows][tiles * 256]; (max, sum) [prog][tiles][rows]; log2 of the rows' sums [prog][rows].
  float* scores; uint64_t* stats; float* lse;
  int32_t* counters;  // [prog]
};

// A program (sequence b, KV head h): its rows, tokens and active tiles.
struct AwProg {
  int b, h, ql, rows, L, tiles;
};
__device__ __forceinline__ bool aw_prog(const AwParams& p, int prog, AwProg& x) {
  int n_seqs = p.n_seqs, q_len = p.q_len;
  if (p.plan != nullptr) {
    n_seqs = min(max(p.plan[0], 0), p.B_grid);
    q_len = min(max(p.plan[1], 0), p.ql_grid);
  }
  x.b = prog / p.H_KV;
  x.h = prog - x.b * p.H_KV;
  if (x.b >= n_seqs) return false;
  x.ql = p.q_lens != nullptr ? min(max(p.q_lens[x.b], 0), q_len) : q_len;
  x.rows = x.ql * p.G;
  x.L = min(max(p.ctx_len[x.b], 0), p.cap);
  x.tiles = (x.L + kAwTile - 1) / kAwTile;
  return x.rows > 0 && x.L > 0;
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

// What tokens gather is added to what they have; new ones start from nothing.
__device__ __forceinline__ void aw_update(const AwParams& p, const AwProg& x, int t, const v4f& got) {
  float* w = p.w + x.b * p.s_wb + x.h * p.s_wh + t;
  const int fresh = x.L - x.ql;
  if (p.w_vec && t + 4 <= x.L) {
    v4f old = *reinterpret_cast<const v4f*>(w);
#pragma unroll
    for (int i = 0; i < 4; ++i) old[i] = (t + i >= fresh ? 0.f : old[i]) + got[i];
    *reinterpret_cast<v4f*>(w) = old;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (t + i < x.L) w[i] = (t + i >= fresh ? 0.f : w[i]) + got[i];
  }
}

enum { kAwScores, kAwStats, kAwSums };  // pass 1 with and without storing the scores, pass 2 from K

template <int D, typename ST, int MODE>
__global__ __launch_bounds__(256) void aw_tile_kernel(AwParams p) {
  constexpr int NU = D / 32;  // matrix steps over the head dimension
  constexpr int NI = D / 64;  // 16-byte loads of a lane's token
  constexpr int NB = 4;       // sub-tiles of 16 tokens of a wave
  __shared__ float s_scale[4][64];
  __shared__ uint64_t s_stat[MODE == kAwSums ? 1 : 4][MODE == kAwSums ? 1 : kAwSeg * 16];
  __shared__ int s_last;
  const int lane = lane_id(), w = uniform(wave_id()), r = lane & 15, g = lane >> 4;
  const int progs = p.B_grid * p.H_KV;
  for (int64_t item = blockIdx.x; item < (int64_t)progs * p.tiles; item += gridDim.x) {
    const int tile = (int)(item / progs), prog = (int)(item - (int64_t)tile * progs);
    AwProg x;
    if (!aw_prog(p, prog, x) || tile >= x.tiles) continue;
    const int t0 = tile * kAwTile + 64 * w;  // the wave's first token
    // Codes and scales.  A sub-tile lies in one page; one past the context or on no page reads nothing and is not seen.
    v4i raw[NB][NI];
    uint32_t seen_sub = 0;
    float scale = 0.f;
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const int t = t0 + 16 * s;
#pragma unroll
      for (int i = 0; i < NI; ++i) raw[s][i] = v4i{0, 0, 0, 0};
      if (t >= x.L) continue;
      const int page = uniform(p.bt[x.b * p.s_bt + t / p.PAGE]), slot = t % p.PAGE;
      if ((uint32_t)page >= (uint32_t)p.n_pages) continue;
      seen_sub |= 1u << s;
      const int8_t* src = p.kc + page * p.s_kp + (int64_t)(slot + r) * p.s_ko + x.h * p.s_kh + 16 * g;
#pragma unroll
      for (int i = 0; i < NI; ++i) raw[s][i] = *reinterpret_cast<const v4i*>(src + 64 * i);
      if (g == s)
        scale = (float)static_cast<const ST*>(p.ks)[page * p.s_sp + (int64_t)(slot + r) * p.s_so + x.h * p.s_sh];
    }
    // Lane (r, g) holds the scale of token t0 + 16 g + r; it needs those of tokens 16 s + 4 g + i.
    s_scale[w][lane] = scale * p.scale_log2;
    wait_lgkm0();
    v4f ksc[NB];
#pragma unroll
    for (int s = 0; s < NB; ++s) ksc[s] = *reinterpret_cast<const v4f*>(&s_scale[w][16 * s + 4 * g]);
    // Operand bytes of matrix step u = 2 i + half: d = 64 i + 16 g + 8 half + j, for K and Q alike.
    v8h kh[NB][NU];
#pragma unroll
    for (int s = 0; s < NB; ++s)
#pragma unroll
      for (int u = 0; u < NU; ++u)
        kh[s][u] = i8x8_to_h8((uint32_t)raw[s][u / 2][2 * (u & 1)], (uint32_t)raw[s][u / 2][2 * (u & 1) + 1]);

    const int fresh = x.L - x.ql;  // a row of new token i sees t <= fresh + i
    const int blocks = (x.rows + 15) / 16;
    v4f sums[NB];
#pragma unroll
    for (int s = 0; s < NB; ++s) sums[s] = v4f{0.f, 0.f, 0.f, 0.f};
    auto load_q = [&](int rb, v8h (&qf)[NU]) {
      const int row = min(rb * 16 + r, x.rows - 1), qi = row / p.G, head = x.h * p.G + row - qi * p.G;
      const _Float16* src = p.q + x.b * p.s_qb + qi * p.s_qt + head * p.s_qh + 16 * g;
#pragma unroll
      for (int u = 0; u < NU; ++u) qf[u] = *reinterpret_cast<const v8h*>(src + 64 * (u / 2) + 8 * (u & 1));
    };
    // The first block with a row that sees the wave's first token.
    const int first = t0 > fresh ? min((t0 - fresh) * p.G / 16, blocks) : 0;
    for (int seg = 0; seg < blocks; seg += kAwSeg) {
      const int seg_end = min(seg + kAwSeg, blocks);
      for (int rb = seg; rb < seg_end; ++rb) {
        const int row = rb * 16 + r;
        if (seen_sub == 0 || rb < first) {
          if constexpr (MODE != kAwSums)
            if (g == 0) s_stat[w][row - seg * 16] = aw_pack(-INFINITY, 0.f);
          if constexpr (MODE == kAwScores) {
#pragma unroll
            for (int s = 0; s < NB; ++s)
              if (row < x.rows && t0 + 16 * s < x.L)
                *reinterpret_cast<v4f*>(p.scores + ((int64_t)prog * p.rows + row) * p.tiles * kAwTile + t0 + 16 * s + 4 * g) =
                    v4f{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          }
          continue;
        }
        v8h qf[NU];
        load_q(rb, qf);
        float lse = INFINITY;
        if constexpr (MODE == kAwSums)
          if (row < x.rows) lse = p.lse[(int64_t)prog * p.rows + row];
        v4f acc[NB];
#pragma unroll
        for (int s = 0; s < NB; ++s) {
          acc[s] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < NU; ++u) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[s][u], qf[u], acc[s], 0, 0, 0);
        }
        const int last = row < x.rows ? fresh + row / p.G : -1;  // the last token the lane's row sees
        const bool all = t0 + 63 <= fresh && seen_sub == 0xf && rb * 16 + 16 <= x.rows;
#pragma unroll
        for (int s = 0; s < NB; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[s][i] *= ksc[s][i];
            if (!all && !(((seen_sub >> s) & 1) && t0 + 16 * s + 4 * g + i <= last)) acc[s][i] = -INFINITY;
          }
        if constexpr (MODE == kAwSums) {
#pragma unroll
          for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[s][i] += fast_exp2(acc[s][i] - lse);
        } else {
          if constexpr (MODE == kAwScores) {
#pragma unroll
            for (int s = 0; s < NB; ++s)
              if (row < x.rows && t0 + 16 * s < x.L)
                *reinterpret_cast<v4f*>(p.scores + ((int64_t)prog * p.rows + row) * p.tiles * kAwTile + t0 + 16 * s + 4 * g) =
                    acc[s];
          }
          float m = -INFINITY;
#pragma unroll
          for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, acc[s][i]);
          m = aw_max4(m);
          const float ref = m == -INFINITY ? 0.f : m;
          float l = 0.f;
#pragma unroll
          for (int s = 0; s < NB; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) l += fast_exp2(acc[s][i] - ref);
          l = aw_sum4(l);
          if (g == 0) s_stat[w][row - seg * 16] = aw_pack(m, l);
        }
      }
      if constexpr (MODE != kAwSums) {
        __syncthreads();
        const int n = min((seg_end - seg) * 16, x.rows - seg * 16);
        for (int i = threadIdx.x; i < n; i += 256) {
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) aw_join(m, l, aw_m(s_stat[v][i]), aw_l(s_stat[v][i]));
          publish(p.stats + ((int64_t)prog * p.tiles + tile) * p.rows + seg * 16 + i, aw_pack(m, l));
        }
        __syncthreads();
      }
    }
    if constexpr (MODE == kAwSums) {
      // Lanes 0..3 of each 16 update four tokens each.
      v4f got = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = aw_sum16(sums[s][i]);
          got[i] = r == s ? v : got[i];
        }
      if (r < NB && t0 + 16 * r + 4 * g < x.L) aw_update(p, x, t0 + 16 * r + 4 * g, got);
    } else if (arrive_last(p.counters + prog, x.tiles, &s_last)) {
      // The rows' tiles joined: many rows a thread each, few a wave each.
      const uint64_t* st = p.stats + (int64_t)prog * p.tiles * p.rows;
      float* out = p.lse + (int64_t)prog * p.rows;
      auto done = [&](int row, float m, float l) { out[row] = m == -INFINITY ? INFINITY : m + __builtin_amdgcn_logf(l); };
      if (x.rows >= 64) {
        for (int row = threadIdx.x; row < x.rows; row += 256) {
          float m = -INFINITY, l = 0.f;
#pragma unroll 4
          for (int k = 0; k < x.tiles; ++k) {
            const uint64_t v = collect(st + (int64_t)k * p.rows + row);
            aw_join(m, l, aw_m(v), aw_l(v));
          }
          done(row, m, l);
        }
      } else {
        for (int row = w; row < x.rows; row += 4) {
          float m = -INFINITY, l = 0.f;
#pragma unroll 4
          for (int k = lane; k < x.tiles; k += kWave) {
            const uint64_t v = collect(st + (int64_t)k * p.rows + row);
            aw_join(m, l, aw_m(v), aw_l(v));
          }
#pragma unroll
          for (int o = 1; o < kWave; o *= 2) aw_join(m, l, __shfl_xor(m, o), __shfl_xor(l, o));
          if (lane == 0) done(row, m, l);
        }
      }
    }
  }
}

// Pass 2 from stored scores: a thread owns four tokens, and adds their rows in the order of the lanes above.
__global__ __launch_bounds__(256) void aw_sum_kernel(AwParams p) {
  const int progs = p.B_grid * p.H_KV, tiles = (p.cap + kAwSumTile - 1) / kAwSumTile;
  for (int64_t item = blockIdx.x; item < (int64_t)progs * tiles; item += gridDim.x) {
    const int tile = (int)(item / progs), prog = (int)(item - (int64_t)tile * progs);
    AwProg x;
    const int t = tile * kAwSumTile + 4 * (int)threadIdx.x;
    if (!aw_prog(p, prog, x) || t >= x.L) continue;
    const float* sc = p.scores + (int64_t)prog * p.rows * p.tiles * kAwTile + t;
    v4f e[kAwStoreRows];
#pragma unroll
    for (int k = 0; k < kAwStoreRows; ++k) {
      e[k] = v4f{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (k < x.rows) e[k] = *reinterpret_cast<const v4f*>(sc + (int64_t)k * p.tiles * kAwTile);
    }
#pragma unroll
    for (int k = 0; k < kAwStoreRows; ++k) {
      const float lse = k < x.rows ? p.lse[(int64_t)prog * p.rows + k] : INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) e[k][i] = fast_exp2(e[k][i] - lse);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int k = 0; k < 16; k += 2) e[k][i] += e[k + 1][i];
#pragma unroll
      for (int k = 0; k < 16; k += 4) e[k][i] += e[k + 2][i];
      e[0][i] = (e[0][i] + e[4][i]) + (e[8][i] + e[12][i]);
    }
    aw_update(p, x, t, e[0]);
  }
}

template <int D, int MODE>
static const void* aw_tile_fn(bool f32) {
  return f32 ? reinterpret_cast<const void*>(&aw_tile_kernel<D, float, MODE>)
             : reinterpret_cast<const void*>(&aw_tile_kernel<D, _Float16, MODE>);
}

struct AwSpace { size_t scores, stats, lse; };  // bytes
static AwSpace aw_space(int64_t progs, int64_t rows, int64_t tiles) {
  return {rows <= kAwStoreRows ? align_up((size_t)(progs * rows * tiles * kAwTile * 4), 256) : 0,
          align_up((size_t)(progs * tiles * rows * 8), 256), align_up((size_t)(progs * rows * 4), 256)};
}

}  // namespace specq

using namespace specq;

extern "C" size_t specq_paged_attn_weights_workspace_size(int B_grid, int H, int H_KV, int ql_grid, int max_pages,
                                                          int PAGE) {
  if (B_grid <= 0 || H <= 0 || H_KV <= 0 || H % H_KV != 0 || ql_grid <= 0 || max_pages <= 0 || PAGE <= 0) return 0;
  const AwSpace s = aw_space((int64_t)B_grid * H_KV, (int64_t)ql_grid * (H / H_KV),
                             ceil_div64((int64_t)max_pages * PAGE, kAwTile));
  return kCounterBytes + s.scores + s.stats + s.lse;
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
  SPECQ_REQUIRE(rows <= (1 << 20) && ql_grid <= (1 << 20), SPECQ_ENOTSUP, "paged_attn_weights: too many query rows");
  SPECQ_REQUIRE(progs <= kMaxCounters, SPECQ_ENOTSUP, "paged_attn_weights: more than %lld sequences x KV heads",
                (long long)kMaxCounters);
  SPECQ_REQUIRE((uintptr_t)q % 16 == 0 && s_qb % 8 == 0 && s_qt % 8 == 0 && s_qh % 8 == 0, SPECQ_ENOTSUP,
                "paged_attn_weights: q rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)kc % 16 == 0 && s_kp % 16 == 0 && s_ko % 16 == 0 && s_kh % 16 == 0, SPECQ_ENOTSUP,
                "paged_attn_weights: cache rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)ks % (scale_fp32 ? 4 : 2) == 0 && (uintptr_t)weights % 4 == 0, SPECQ_EINVAL,
                "paged_attn_weights: scales and weights must be aligned to their type");
  SPECQ_REQUIRE(lie_apart(B_grid, s_wb, cap) && lie_apart(H_KV, s_wh, cap), SPECQ_ENOTSUP,
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
  p.plan = plan; p.n_seqs = n_seqs; p.q_len = q_len; p.B_grid = B_grid; p.ql_grid = ql_grid;
  p.G = H / H_KV; p.H_KV = H_KV; p.PAGE = PAGE;
  p.cap = (int)cap; p.tiles = (int)ceil_div64(cap, kAwTile); p.rows = (int)rows;
  p.scale_log2 = sm_scale * 1.44269504088896340736f;
  const AwSpace space = aw_space(progs, rows, p.tiles);
  const size_t need = kCounterBytes + space.scores + space.stats + space.lse;
  SPECQ_REQUIRE(workspace && workspace_bytes >= need, SPECQ_ENOSPC,
                "paged_attn_weights: workspace of %zu bytes required, %zu given", need, workspace ? workspace_bytes : (size_t)0);
  char* at = static_cast<char*>(workspace);
  p.counters = reinterpret_cast<int32_t*>(at);
  p.scores = reinterpret_cast<float*>(at + kCounterBytes);
  p.stats = reinterpret_cast<uint64_t*>(at + kCounterBytes + space.scores);
  p.lse = reinterpret_cast<float*>(at + kCounterBytes + space.scores + space.stats);
  const bool store = rows <= kAwStoreRows, f32 = scale_fp32 != 0;
  const int64_t items = progs * p.tiles, sums = progs * ceil_div64(cap, kAwSumTile);
  const int grid = (int)(items < kAwMaxGrid ? items : kAwMaxGrid);
  const void* one = D == 64 ? (store ? aw_tile_fn<64, kAwScores>(f32) : aw_tile_fn<64, kAwStats>(f32))
                            : (store ? aw_tile_fn<128, kAwScores>(f32) : aw_tile_fn<128, kAwStats>(f32));
  if (int rc = launch(one, grid, 256, 0, (hipStream_t)stream, &p)) return rc;
  if (store)
    return launch(reinterpret_cast<const void*>(&aw_sum_kernel), (int)(sums < kAwMaxGrid ? sums : kAwMaxGrid), 256, 0,
                  (hipStream_t)stream, &p);
  return launch(D == 64 ? aw_tile_fn<64, kAwSums>(f32) : aw_tile_fn<128, kAwSums>(f32), grid, 256, 0, (hipStream_t)stream, &p);
}
