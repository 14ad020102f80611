// Positions of the rotary kernels (rotary.hip, qk_norm.hip): their parameters, and a token's angles and head rows.
#pragma once
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

}  // namespace specq
