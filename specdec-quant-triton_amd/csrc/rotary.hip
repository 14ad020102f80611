// Rotary positions of the new tokens' q and k, and its C ABI.
//
// Pair j of a head's first R dimensions -- (j, j + R/2) or, interleaved, (2j, 2j + 1) -- is turned by
// pos * f_j and scaled by m:
//   a' = m (a cos - b sin),   b' = m (b cos + a sin);   dimensions R.. are copied.
// pos is ctx_len[b] - q_len + i (the position the K/V append and the attention give token i), or
// positions[b, i].
//
// The angle is formed in fp64 turns, pos * (f_j / 2 pi), and its fractional part goes to the hardware
// sine and cosine, whose argument is in turns: at position 2^20 an fp32 product would be off by 0.06
// radians.  Everything else is fp32 with one rounding to fp16.
//
// A thread owns one unit of a token -- 8 pairs (half layout, two 16-byte vectors), 4 pairs (interleaved,
// one vector) or 8 copied values -- and walks the heads, so the fp64 products and the sines are made
// once for the heads it covers.  Bound by HBM for prompts (4 bytes a value) and by launch and load
// latency for a step.  In place works: both halves of a pair are read before either is written, by
// one thread.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

struct RotaryParams {
  const _Float16* q; int64_t s_qb, s_qt, s_qh;
  const _Float16* k; int64_t s_kb, s_kt, s_kh;
  _Float16* qo; int64_t s_qob, s_qot, s_qoh;
  _Float16* ko; int64_t s_kob, s_kot, s_koh;
  const void* inv_freq; int freq64;
  const int32_t* ctx_len; const int32_t* positions; int64_t s_pb;
  const int32_t* plan;
  float mscale;
  int n_seqs, q_len, ql_grid, B_grid, H, H_KV, D, R;
  int tail;  // dimensions copied behind the rotated ones: D - R, or none where the call is in place
  int tpt;   // threads per token (vector kernel): a power of two, at least 64
};

__device__ __forceinline__ double rotary_freq(const RotaryParams& p, int j) {
  return p.freq64 ? static_cast<const double*>(p.inv_freq)[j] : (double)static_cast<const float*>(p.inv_freq)[j];
}
__device__ __forceinline__ void rotary_angle(double f, int pos, float m, float& c, float& s) {
  const double turns = (double)pos * (f * 0.15915494309189533577);
  const float x = (float)(turns - rint(turns));
  c = m * __builtin_amdgcn_cosf(x);
  s = m * __builtin_amdgcn_sinf(x);
}

// Token `tok` of the grid: its sequence and index, and its position; false where it is not active.
__device__ __forceinline__ bool rotary_token(const RotaryParams& p, int tok, int& b, int& i, int& pos) {
  b = tok / p.ql_grid;
  i = tok - b * p.ql_grid;
  if (b >= p.B_grid) return false;
  pos = p.positions != nullptr ? p.positions[(int64_t)b * p.s_pb + i] : p.ctx_len[b];
  int nb = p.n_seqs, ql = p.q_len;
  if (p.plan != nullptr) {
    nb = min(max(p.plan[0], 0), p.B_grid);
    ql = min(max(p.plan[1], 0), p.ql_grid);
  }
  if (b >= nb || i >= ql) return false;
  if (p.positions == nullptr) pos += i - ql;
  return true;
}

struct RotaryHead { const _Float16* src; _Float16* dst; };
__device__ __forceinline__ RotaryHead rotary_head(const RotaryParams& p, int b, int i, int h) {
  if (h < p.H)
    return {p.q + (int64_t)b * p.s_qb + (int64_t)i * p.s_qt + (int64_t)h * p.s_qh,
            p.qo + (int64_t)b * p.s_qob + (int64_t)i * p.s_qot + (int64_t)h * p.s_qoh};
  h -= p.H;
  return {p.k + (int64_t)b * p.s_kb + (int64_t)i * p.s_kt + (int64_t)h * p.s_kh,
          p.ko + (int64_t)b * p.s_kob + (int64_t)i * p.s_kot + (int64_t)h * p.s_koh};
}

// 16-byte aligned rows, D a multiple of 8, R of 16 (half) or 8 (interleaved).
template <bool IL>
__global__ __launch_bounds__(256) void rotary_vec_kernel(RotaryParams p) {
  const int t = threadIdx.x % p.tpt;
  int b, i, pos;
  if (!rotary_token(p, (int)blockIdx.x * (256 / p.tpt) + (int)threadIdx.x / p.tpt, b, i, pos)) return;
  constexpr int NP = IL ? 4 : 8;  // pairs per unit
  const int rot = p.R / (2 * NP), units = rot + p.tail / 8;
  const int heads = p.H + p.H_KV;
  const int lanes = p.tpt / units;  // heads side by side; units <= 64 <= tpt
  const int u = t % units, hl = t / units;
  if (hl >= lanes) return;
  float c[NP], s[NP];
  if (u < rot) {
#pragma unroll
    for (int e = 0; e < NP; ++e) rotary_angle(rotary_freq(p, NP * u + e), pos, p.mscale, c[e], s[e]);
  }
  const int at = u < rot ? 8 * u : p.R + 8 * (u - rot);
#pragma unroll 4
  for (int h = hl; h < heads; h += lanes) {
    const RotaryHead r = rotary_head(p, b, i, h);
    v8h x = *reinterpret_cast<const v8h*>(r.src + at);
    if (u < rot) {
      if constexpr (IL) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = (float)x[2 * e], x1 = (float)x[2 * e + 1];
          x[2 * e] = (_Float16)(x0 * c[e] - x1 * s[e]);
          x[2 * e + 1] = (_Float16)(x1 * c[e] + x0 * s[e]);
        }
      } else {
        v8h y = *reinterpret_cast<const v8h*>(r.src + at + p.R / 2);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x0 = (float)x[e], x1 = (float)y[e];
          x[e] = (_Float16)(x0 * c[e] - x1 * s[e]);
          y[e] = (_Float16)(x1 * c[e] + x0 * s[e]);
        }
        *reinterpret_cast<v8h*>(r.dst + at + p.R / 2) = y;
      }
    }
    *reinterpret_cast<v8h*>(r.dst + at) = x;
  }
}

// Any R, D and alignment: a thread owns pairs and copied values one by one, 2 bytes an access.  2 x 4096 tokens, 32 / 8
// heads, D = 80, in a graph: R = 20 here 80.6 us = 1.3 TB/s, R = 80 in the vector kernel 30.8.
template <bool IL>
__global__ __launch_bounds__(256) void rotary_any_kernel(RotaryParams p) {
  int b, i, pos;
  if (!rotary_token(p, blockIdx.x, b, i, pos)) return;
  const int np = p.R / 2, items = np + p.tail, heads = p.H + p.H_KV;
  const int width = min(items, 256), lanes = 256 / width;  // heads side by side
  const int hl = (int)threadIdx.x / width;
  if (hl >= lanes) return;
  for (int u = (int)threadIdx.x % width; u < items; u += width) {
    if (u < np) {
      float c, s;
      rotary_angle(rotary_freq(p, u), pos, p.mscale, c, s);
      const int a0 = IL ? 2 * u : u, a1 = IL ? 2 * u + 1 : u + np;
      for (int h = hl; h < heads; h += lanes) {
        const RotaryHead r = rotary_head(p, b, i, h);
        const float x0 = (float)r.src[a0], x1 = (float)r.src[a1];
        r.dst[a0] = (_Float16)(x0 * c - x1 * s);
        r.dst[a1] = (_Float16)(x1 * c + x0 * s);
      }
    } else {
      const int a = p.R + u - np;
      for (int h = hl; h < heads; h += lanes) {
        const RotaryHead r = rotary_head(p, b, i, h);
        r.dst[a] = r.src[a];
      }
    }
  }
}

}  // namespace specq

using namespace specq;

extern "C" int specq_rotary(const void* q, int64_t s_qb, int64_t s_qt, int64_t s_qh, const void* k, int64_t s_kb,
                            int64_t s_kt, int64_t s_kh, void* q_out, int64_t s_qob, int64_t s_qot, int64_t s_qoh,
                            void* k_out, int64_t s_kob, int64_t s_kot, int64_t s_koh, const void* inv_freq,
                            int freq_fp64, float mscale, const int32_t* ctx_len, const int32_t* positions,
                            int64_t s_pb, int B_grid, int n_seqs, int q_len, int ql_grid, int H, int H_KV, int D,
                            int R, int interleaved, const int32_t* plan, void* stream) {
  clear_error();
  SPECQ_REQUIRE(q && q_out && inv_freq && (H_KV == 0 || (k && k_out)), SPECQ_EINVAL, "rotary: null tensor pointer");
  SPECQ_REQUIRE(ctx_len || positions, SPECQ_EINVAL, "rotary: neither ctx_len nor positions given");
  SPECQ_REQUIRE(B_grid >= 0 && ql_grid >= 0 && n_seqs >= 0 && n_seqs <= B_grid && q_len >= 0 && q_len <= ql_grid,
                SPECQ_EINVAL, "rotary: need 0 <= n_seqs <= B_grid and 0 <= q_len <= ql_grid");
  SPECQ_REQUIRE(H > 0 && H_KV >= 0 && D > 0 && R > 0 && R <= D && R % 2 == 0, SPECQ_EINVAL,
                "rotary: need an even number R=%d of rotated dimensions, at most head_dim %d", R, D);
  SPECQ_REQUIRE(D <= 512, SPECQ_ENOTSUP, "rotary: head_dim %d (at most 512 supported)", D);
  SPECQ_REQUIRE(lie_apart(B_grid, s_qob, D) && lie_apart(ql_grid, s_qot, D) && lie_apart(H, s_qoh, D) &&
                    (H_KV == 0 || (lie_apart(B_grid, s_kob, D) && lie_apart(ql_grid, s_kot, D) && lie_apart(H_KV, s_koh, D))),
                SPECQ_ENOTSUP, "rotary: rows of an output overlap");
  const int64_t tokens = (int64_t)B_grid * ql_grid;
  SPECQ_REQUIRE(tokens <= INT32_MAX - 4, SPECQ_EINVAL, "rotary: grid too large");
  if (tokens == 0) return SPECQ_OK;
  RotaryParams p = {};
  p.q = (const _Float16*)q; p.s_qb = s_qb; p.s_qt = s_qt; p.s_qh = s_qh;
  p.k = (const _Float16*)k; p.s_kb = s_kb; p.s_kt = s_kt; p.s_kh = s_kh;
  p.qo = (_Float16*)q_out; p.s_qob = s_qob; p.s_qot = s_qot; p.s_qoh = s_qoh;
  p.ko = (_Float16*)k_out; p.s_kob = s_kob; p.s_kot = s_kot; p.s_koh = s_koh;
  p.inv_freq = inv_freq; p.freq64 = freq_fp64; p.mscale = mscale;
  p.ctx_len = ctx_len; p.positions = positions; p.s_pb = s_pb; p.plan = plan;
  p.n_seqs = n_seqs; p.q_len = q_len; p.ql_grid = ql_grid; p.B_grid = B_grid; p.H = H; p.H_KV = H_KV; p.D = D; p.R = R;
  const bool in_place = q == q_out && s_qb == s_qob && s_qt == s_qot && s_qh == s_qoh &&
                        (H_KV == 0 || (k == k_out && s_kb == s_kob && s_kt == s_kot && s_kh == s_koh));
  p.tail = in_place ? 0 : D - R;
  uint64_t bits = (uintptr_t)q | (uintptr_t)q_out | 2 * (uint64_t)(s_qb | s_qt | s_qh | s_qob | s_qot | s_qoh);
  if (H_KV) bits |= (uintptr_t)k | (uintptr_t)k_out | 2 * (uint64_t)(s_kb | s_kt | s_kh | s_kob | s_kot | s_koh);
  const bool vec = bits % 16 == 0 && D % 8 == 0 && R % (interleaved ? 8 : 16) == 0;
  if (!vec) {
    const void* fn = interleaved ? reinterpret_cast<const void*>(&rotary_any_kernel<true>)
                                 : reinterpret_cast<const void*>(&rotary_any_kernel<false>);
    return launch(fn, (int)tokens, 256, 0, (hipStream_t)stream, &p);
  }
  // Few tokens: a workgroup each, so that the heads' loads go out at once; many: a wave each, whose
  // lanes make the angles once for five heads of 40.
  p.tpt = tokens <= 1024 ? 256 : 64;
  const void* fn = interleaved ? reinterpret_cast<const void*>(&rotary_vec_kernel<true>)
                               : reinterpret_cast<const void*>(&rotary_vec_kernel<false>);
  return launch(fn, (int)ceil_div64(tokens, 256 / p.tpt), 256, 0, (hipStream_t)stream, &p);
}
