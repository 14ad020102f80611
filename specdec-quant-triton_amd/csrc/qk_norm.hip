// Norms of q and k for each head with their rotary positions in the same pass, and its C ABI.
//
// A head's row x of D values becomes
//   y = x rsqrt(mean(x^2) + eps) w,
// and the first R dimensions of y are turned by the token's position as rotary.hip turns them.  fp32 with one
// rounding to fp16; angles in fp64 turns.  w is [D] or [heads, D], fp16 or fp32, or absent (1).
//
// A group of UP lanes owns a row, a lane one unit of it -- 8 pairs (half layout, two 16-byte vectors), 4 pairs
// (interleaved, one vector) or 8 values that are not turned -- so the row is read once, stays in registers over the sum
// of its squares (a few lane exchanges) and is written once.  The lanes make their angles once for the heads they walk.
// In place works: every value of a row is an operand of the sum that each store waits for.
// Prompts are bound by HBM (2 x 4096 tokens, 32 / 8 heads of 128: 168 MB in 33.7 us, the rate of a copy), steps by the launch
// (one token 4.6 us; 51 tokens of 12 / 3 heads of 80, which the vector kernel does not take, 5.1).
#include "api_common.hpp"
#include "rotary.hpp"

namespace specq {

struct QkNormParams {
  RotaryParams r;
  const void* wq; const void* wk; int64_t s_wq, s_wk;  // elements from head to head, 0 for one row of weights
  int w_fp32;
  float eps, inv_d;
};

// Sum over the UP lanes of an aligned group; every lane of the group gets it.
template <int UP>
__device__ __forceinline__ float group_sum(float v) {
  auto add = [&](auto ctrl) {
    constexpr int c = decltype(ctrl)::value;
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), c, 0xf, 0xf, false));
  };
  if constexpr (UP >= 2) add(std::integral_constant<int, 0xB1>{});   // lane ^ 1
  if constexpr (UP >= 4) add(std::integral_constant<int, 0x4E>{});   // lane ^ 2
  if constexpr (UP >= 8) add(std::integral_constant<int, 0x141>{});  // mirrored in 8, whose halves agree
  if constexpr (UP >= 16) add(std::integral_constant<int, 0x140>{}); // mirrored in 16
  if constexpr (UP >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
  }
  if constexpr (UP >= 64) {
    const auto a = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), false, false);
    v = __builtin_bit_cast(float, (int)a[0]) + __builtin_bit_cast(float, (int)a[1]);
  }
  return v;
}

// The weights of head h: their row, or null where there are none.
struct NormWeights {
  const void* row;
  bool fp32;
  __device__ __forceinline__ float at(int i) const {
    if (row == nullptr) return 1.f;
    return fp32 ? static_cast<const float*>(row)[i] : (float)static_cast<const _Float16*>(row)[i];
  }
  __device__ __forceinline__ void at8(int i, float (&w)[8]) const {
    if (row == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = 1.f;
    } else if (fp32) {
      const v4f a = *reinterpret_cast<const v4f*>(static_cast<const float*>(row) + i);
      const v4f b = *reinterpret_cast<const v4f*>(static_cast<const float*>(row) + i + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = e < 4 ? a[e & 3] : b[e & 3];
    } else {
      const v8h a = *reinterpret_cast<const v8h*>(static_cast<const _Float16*>(row) + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = (float)a[e];
    }
  }
};
__device__ __forceinline__ NormWeights norm_weights(const QkNormParams& p, int h) {
  const bool is_q = h < p.r.H;
  const void* base = is_q ? p.wq : p.wk;
  if (base == nullptr) return {nullptr, false};
  const int64_t off = is_q ? h * p.s_wq : (h - p.r.H) * p.s_wk;
  return {static_cast<const char*>(base) + off * (p.w_fp32 ? 4 : 2), p.w_fp32 != 0};
}

// 16-byte aligned rows and weights, D a multiple of 8, R of 16 (half) or 8 (interleaved).
template <bool IL, int UP>
__global__ __launch_bounds__(256) void qk_norm_vec_kernel(QkNormParams p) {
  const RotaryParams& rp = p.r;
  int b, i, pos;
  if (!rotary_token(rp, (int)blockIdx.x * (256 / rp.tpt) + (int)threadIdx.x / rp.tpt, b, i, pos)) return;
  constexpr int NP = IL ? 4 : 8;  // pairs per unit
  const int t = threadIdx.x % rp.tpt;
  const int rot = rp.R / (2 * NP), units = rot + rp.tail / 8;
  const int heads = rp.H + rp.H_KV, lanes = rp.tpt / UP;  // heads side by side
  const int u = t % UP, hl = t / UP;
  const bool turned = u < rot, some = u < units;
  const int at = turned ? 8 * u : rp.R + 8 * (u - rot);
  float c[NP], s[NP];
  if (turned) {
#pragma unroll
    for (int e = 0; e < NP; ++e) rotary_angle(rotary_freq(rp, NP * u + e), pos, rp.mscale, c[e], s[e]);
  }
  // Weights and turns in one: with (x, y) a pair, its new values are scale (x cx - y sy) and scale (y cy + x sx); a value that
  // is not turned becomes scale x cx.  Made anew where q's heads end, and for each head where each has its weights.
  constexpr int NC = IL ? 4 : 8;
  float cx[8], sx[NC], cy[NC], sy[NC];
  int have = -1;
  // A head at a time: with the loads of four or five ahead the registers leave fewer waves (2 x 4096 tokens, 32 / 8 heads of
  // 128: 42 us against 38).
  for (int h = hl; h < heads; h += lanes) {
    const RotaryHead r = rotary_head(rp, b, i, h);
    v8h x = {}, y = {};
    if (some) x = *reinterpret_cast<const v8h*>(r.src + at);
    if (!IL && turned) y = *reinterpret_cast<const v8h*>(r.src + at + rp.R / 2);
    const int kind = h >= rp.H;
    if (some && (kind != have || (kind ? p.s_wk : p.s_wq) != 0)) {
      have = kind;
      const NormWeights w = norm_weights(p, h);
      float wx[8], wy[8];
      w.at8(at, wx);
      if (!turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) cx[e] = wx[e];
      } else {
        if constexpr (!IL) w.at8(at + rp.R / 2, wy);
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const float a = IL ? wx[(2 * e) & 7] : wx[e & 7], o = IL ? wx[(2 * e + 1) & 7] : wy[e & 7];
          cx[e] = a * c[e], sx[e] = a * s[e], cy[e] = o * c[e], sy[e] = o * s[e];
        }
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum = fmaf((float)x[e], (float)x[e], sum);
      if (!IL) sum = fmaf((float)y[e], (float)y[e], sum);
    }
    const float scale = rsqrtf(fmaf(group_sum<UP>(sum), p.inv_d, p.eps));
    if (!some) continue;
    if (!turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (_Float16)((float)x[e] * scale * cx[e]);
    } else if constexpr (IL) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = (float)x[2 * e] * scale, o = (float)x[2 * e + 1] * scale;
        x[2 * e] = (_Float16)(a * cx[e] - o * sy[e]);
        x[2 * e + 1] = (_Float16)(o * cy[e] + a * sx[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = (float)x[e] * scale, o = (float)y[e] * scale;
        x[e] = (_Float16)(a * cx[e] - o * sy[e]);
        y[e] = (_Float16)(o * cy[e] + a * sx[e]);
      }
      *reinterpret_cast<v8h*>(r.dst + at + rp.R / 2) = y;
    }
    *reinterpret_cast<v8h*>(r.dst + at) = x;
  }
}

// Any R, D and alignment, 2 bytes an access: a wave owns a row, a lane every 64th of its pairs and single values, and
// walks the heads with the workgroup's other waves: 16 of them where there are few tokens, so that few rows follow one
// another (51 tokens, 12 / 3 heads of 80: 8.3 us with four).  Prompts are bound by its narrow accesses: 2 x 4096 tokens of
// such heads, 39 MB, 51 us.
constexpr int kNormItems = 8;  // pairs and values a lane has at most: D <= 512
template <bool IL>
__global__ __launch_bounds__(1024) void qk_norm_any_kernel(QkNormParams p) {
  const RotaryParams& rp = p.r;
  int b, i, pos;
  if (!rotary_token(rp, blockIdx.x, b, i, pos)) return;
  const int np = rp.R / 2, items = np + rp.tail, heads = rp.H + rp.H_KV, lane = lane_id();
  float c[kNormItems], s[kNormItems];
  int i0[kNormItems], i1[kNormItems];  // i1 < 0: a single value; i0 < 0: nothing
#pragma unroll
  for (int e = 0; e < kNormItems; ++e) {
    const int u = lane + kWave * e;
    c[e] = 1.f, s[e] = 0.f, i0[e] = -1, i1[e] = -1;
    if (u < np) {
      i0[e] = IL ? 2 * u : u;
      i1[e] = IL ? 2 * u + 1 : u + np;
      rotary_angle(rotary_freq(rp, u), pos, rp.mscale, c[e], s[e]);
    } else if (u < items) {
      i0[e] = rp.R + u - np;
    }
  }
  for (int h = wave_id(); h < heads; h += (int)blockDim.x / kWave) {
    const RotaryHead r = rotary_head(rp, b, i, h);
    const NormWeights w = norm_weights(p, h);
    float x[kNormItems], y[kNormItems], sum = 0.f;
#pragma unroll
    for (int e = 0; e < kNormItems; ++e) {
      x[e] = i0[e] >= 0 ? (float)r.src[i0[e]] : 0.f;
      y[e] = i1[e] >= 0 ? (float)r.src[i1[e]] : 0.f;
      sum = fmaf(x[e], x[e], sum);
      sum = fmaf(y[e], y[e], sum);
    }
    const float scale = rsqrtf(fmaf(group_sum<kWave>(sum), p.inv_d, p.eps));
#pragma unroll
    for (int e = 0; e < kNormItems; ++e) {
      if (i0[e] < 0) continue;
      const float a0 = x[e] * scale * w.at(i0[e]);
      if (i1[e] < 0) {
        r.dst[i0[e]] = (_Float16)a0;
        continue;
      }
      const float a1 = y[e] * scale * w.at(i1[e]);
      r.dst[i0[e]] = (_Float16)(a0 * c[e] - a1 * s[e]);
      r.dst[i1[e]] = (_Float16)(a1 * c[e] + a0 * s[e]);
    }
  }
}

template <bool IL>
static const void* qk_norm_vec_fn(int units) {
  if (units <= 4) return reinterpret_cast<const void*>(&qk_norm_vec_kernel<IL, 4>);
  if (units <= 8) return reinterpret_cast<const void*>(&qk_norm_vec_kernel<IL, 8>);
  if (units <= 16) return reinterpret_cast<const void*>(&qk_norm_vec_kernel<IL, 16>);
  if (units <= 32) return reinterpret_cast<const void*>(&qk_norm_vec_kernel<IL, 32>);
  return reinterpret_cast<const void*>(&qk_norm_vec_kernel<IL, 64>);
}

}  // namespace specq

using namespace specq;

extern "C" int specq_qk_norm_rotary(const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const void* k, int64_t s_kb,
                                    int64_t s_kt, int64_t s_kh, void* q_out, int64_t s_qob, int64_t s_qot, int64_t s_qoh,
                                    void* k_out, int64_t s_kob, int64_t s_kot, int64_t s_koh, const void* q_weight,
                                    int64_t s_wq, const void* k_weight, int64_t s_wk, int weight_fp32, float eps,
                                    const void* inv_freq, int freq_fp64, float mscale, const int32_t* ctx_len,
                                    const int32_t* positions, int64_t s_pb, int B_grid, int n_seqs, int q_len, int ql_grid,
                                    int H, int H_KV, int D, int R, int interleaved, const int32_t* plan, void* stream) {
  clear_error();
  SPECQ_REQUIRE(q && q_out && inv_freq && (H_KV == 0 || (k && k_out)), SPECQ_EINVAL, "qk_norm_rotary: null tensor pointer");
  SPECQ_REQUIRE(ctx_len || positions, SPECQ_EINVAL, "qk_norm_rotary: neither ctx_len nor positions given");
  SPECQ_REQUIRE(B_grid >= 0 && ql_grid >= 0 && n_seqs >= 0 && n_seqs <= B_grid && q_len >= 0 && q_len <= ql_grid,
                SPECQ_EINVAL, "qk_norm_rotary: need 0 <= n_seqs <= B_grid and 0 <= q_len <= ql_grid");
  SPECQ_REQUIRE(H > 0 && H_KV >= 0 && D > 0 && R > 0 && R <= D && R % 2 == 0, SPECQ_EINVAL,
                "qk_norm_rotary: need an even number R=%d of rotated dimensions, at most head_dim %d", R, D);
  SPECQ_REQUIRE(D <= 512, SPECQ_ENOTSUP, "qk_norm_rotary: head_dim %d (at most 512 supported)", D);
  SPECQ_REQUIRE(eps >= 0.f && eps < INFINITY, SPECQ_EINVAL, "qk_norm_rotary: eps must be finite and not negative");
  const int64_t tokens = (int64_t)B_grid * ql_grid;
  SPECQ_REQUIRE(tokens <= INT32_MAX - 4, SPECQ_EINVAL, "qk_norm_rotary: grid too large");
  SPECQ_REQUIRE(nest_apart({{B_grid, s_qob}, {ql_grid, s_qot}, {H, s_qoh}}, D) &&
                    (H_KV == 0 || nest_apart({{B_grid, s_kob}, {ql_grid, s_kot}, {H_KV, s_koh}}, D)),
                SPECQ_ENOTSUP, "qk_norm_rotary: rows of an output overlap");
  if (tokens == 0) return SPECQ_OK;
  QkNormParams p = {};
  RotaryParams& r = p.r;
  r.q = (const _Float16*)q; r.s_qb = s_qb; r.s_qt = s_qt; r.s_qh = s_qh;
  r.k = (const _Float16*)k; r.s_kb = s_kb; r.s_kt = s_kt; r.s_kh = s_kh;
  r.qo = (_Float16*)q_out; r.s_qob = s_qob; r.s_qot = s_qot; r.s_qoh = s_qoh;
  r.ko = (_Float16*)k_out; r.s_kob = s_kob; r.s_kot = s_kot; r.s_koh = s_koh;
  r.inv_freq = inv_freq; r.freq64 = freq_fp64; r.mscale = mscale;
  r.ctx_len = ctx_len; r.positions = positions; r.s_pb = s_pb; r.plan = plan;
  r.n_seqs = n_seqs; r.q_len = q_len; r.ql_grid = ql_grid; r.B_grid = B_grid; r.H = H; r.H_KV = H_KV; r.D = D; r.R = R;
  r.tail = D - R;
  p.wq = q_weight; p.s_wq = s_wq; p.wk = H_KV ? k_weight : nullptr; p.s_wk = s_wk; p.w_fp32 = weight_fp32;
  p.eps = eps; p.inv_d = 1.f / (float)D;
  uint64_t bits = (uintptr_t)q | (uintptr_t)q_out | 2 * (uint64_t)(s_qb | s_qt | s_qh | s_qob | s_qot | s_qoh);
  if (H_KV) bits |= (uintptr_t)k | (uintptr_t)k_out | 2 * (uint64_t)(s_kb | s_kt | s_kh | s_kob | s_kot | s_koh);
  const uint64_t ws = weight_fp32 ? 4 : 2;
  if (p.wq) bits |= (uintptr_t)p.wq | ws * (uint64_t)s_wq;
  if (p.wk) bits |= (uintptr_t)p.wk | ws * (uint64_t)s_wk;
  const int per = interleaved ? 8 : 16;  // dimensions of a unit of pairs
  if (bits % 16 != 0 || D % 8 != 0 || R % per != 0) {
    const void* fn = interleaved ? reinterpret_cast<const void*>(&qk_norm_any_kernel<true>)
                                 : reinterpret_cast<const void*>(&qk_norm_any_kernel<false>);
    return launch(fn, (int)tokens, tokens <= 1024 ? 1024 : 256, 0, (hipStream_t)stream, &p);
  }
  // As the rotary kernel: few tokens have a workgroup each, many a wave each.
  r.tpt = tokens <= 1024 ? 256 : 64;
  const int units = R / per + r.tail / 8;
  return launch(interleaved ? qk_norm_vec_fn<true>(units) : qk_norm_vec_fn<false>(units),
                (int)ceil_div64(tokens, 256 / r.tpt), 256, 0, (hipStream_t)stream, &p);
}
