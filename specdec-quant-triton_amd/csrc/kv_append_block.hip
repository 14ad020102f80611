// Append to a paged K/V cache with block scales, and its C ABI.
//
// The cache holds int8 or e4m3 codes [pages, PAGE, H_KV, D] and one fp32 scale for each (block of SB
// tokens, KV head), [pages, PAGE / SB, H_KV].  Token i of sequence b goes to position
// pos = ctx_len[b] - q_len + i (ctx_len counts the new tokens).  For each block that new tokens reach,
// with Q = 127 (int8) or 448 (e4m3) and x the new tokens' values in the block:
//   s' = max(amax |x|, 1e-8) / Q;  where the block holds earlier tokens of the sequence (its positions
//        below the first new one), s' = max(s', s) with s its scale so far;
//   new codes      rne(x / s');
//   earlier codes  rne(c * s / s'), clamped to +-Q, where s' > s, untouched otherwise; e4m3 NaN stays NaN.
// fp32, the quotients rounded as IEEE division rounds them.  Infinities count as +-65504 and NaN as 0, so
// that one bad value does not take the block's other tokens with it.  Slots past the last new token are
// not touched.
//
// One workgroup per (sequence, block, K or V, head): SB * D values, eight to a thread and pass, held in
// registers between the amax and the codes (up to 16384 values; larger blocks are read twice).  The
// block's earlier codes and its scale are fetched together with the new values' amax pass, so that
// the requantisation adds no round trip.  Bound by the latency of its three dependent loads (context
// length, page id, codes) for a verification step (B = 8, 9 tokens, 8 heads of 128, int8, blocks of 16:
// 4.1 us) and for a prompt by that and the instructions of the conversion (2 x 2048 tokens, e4m3, blocks
// of 32, 25 MB: 10.2 us = 2.5 TB/s on one set of inputs, 11.2 over distinct ones (int8 10.9), and 12.9 with a division
// and a clamp for each value).
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

struct KvAppendBlockParams {
  const _Float16* k; const _Float16* v; int64_t s_nb, s_nt, s_nh;  // new K/V [B, ql, H_KV, D]
  uint8_t* kc; uint8_t* vc; int64_t s_kp, s_ko, s_kh;              // codes [pages, PAGE, H_KV, D]
  float* ks; float* vs; int64_t s_sp, s_so, s_sh;                  // scales [pages, PAGE / SB, H_KV]
  const int32_t* bt; int64_t s_bt; int max_pages, n_pages;
  const int32_t* ctx_len;
  const int32_t* plan;
  int n_seqs, q_len, ql_grid, B_grid, H_KV, PAGE, SB, blocks;  // blocks: the most one sequence's tokens reach
  int log_dv;                                                  // log2(D / 8)
};

typedef uint16_t v2u16 __attribute__((ext_vector_type(2)));
typedef uint16_t v8u16 __attribute__((ext_vector_type(8)));

// Largest magnitude of eight fp16 values as fp16 bits, which order as the magnitudes do (not finite: 0x7c00
// and above).
__device__ __forceinline__ uint32_t top16(v8h x) {
  const v8u16 a = __builtin_bit_cast(v8u16, x) & (uint16_t)0x7fff;
  const v2u16 m = __builtin_elementwise_max(__builtin_elementwise_max(v2u16{a[0], a[1]}, v2u16{a[2], a[3]}),
                                            __builtin_elementwise_max(v2u16{a[4], a[5]}, v2u16{a[6], a[7]}));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}
// New values as they are quantised: NaN as 0, infinities as the largest finite fp16.  Returns top16 of that.
__device__ __forceinline__ uint32_t clean16(v8h& x) {
  const uint32_t m = top16(x);
  if (m < 0x7c00) return m;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float f = (float)x[e];
    x[e] = (_Float16)(f != f ? 0.f : fminf(fmaxf(f, -65504.f), 65504.f));
  }
  return top16(x);
}

// Codes of eight values over the scale s, clamped to the largest; NaN stays NaN where there is a code for it.
template <bool F8>
__device__ __forceinline__ v2i encode8(const float (&x)[8], float s) {
  int w[2] = {0, 0};
  if constexpr (F8) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = x[j] / s;
      q[j] = f != f ? f : fminf(fmaxf(f, -448.f), 448.f);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], w[h], false);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w[h], true);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = fminf(fmaxf(rintf(x[j] / s), -127.f), 127.f);
      w[j >> 2] |= ((int)q & 0xff) << (8 * (j & 3));
    }
  }
  return v2i{w[0], w[1]};
}
// The same for |x| <= Q s with s in [2^-60, 2^60] and y = 1 / s rounded to nearest.  x / s comes out as the
// division rounds it: q0 = x y is within an ulp or two, its remainder x - q0 s is exact in one FMA, and
// q0 plus remainder times a correctly rounded reciprocal is the rounded quotient (Markstein; equal to the
// division for every finite fp16 x and every scale max(amax, 1e-8) / Q above it).  It is at most
// Q (1 + 2^-23), whose code is Q's, so nothing is clamped; adding 1.5 * 2^23 rounds to an integer, ties to
// even, in the low bits.
template <bool F8>
__device__ __forceinline__ v2i encode8_by(v8h x, float s, float y) {
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = (float)x[j], q0 = f * y;
    q[j] = fmaf(fmaf(-q0, s, f), y, q0);
    if constexpr (F8) q[j] = __builtin_copysignf(q[j], f);  // -0 stays -0
  }
  int w[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (F8) {
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], w[h], false);
      w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], w[h], true);
    } else {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(uint32_t, q[4 * h + e] + 12582912.f);
      const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u);
      w[h] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    }
  }
  return v2i{w[0], w[1]};
}

template <bool F8>
__device__ __forceinline__ void decode8(v2i c, float (&x)[8]) {
  if constexpr (F8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x[4 * h] = __builtin_amdgcn_cvt_f32_fp8(c[h], 0);
      x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(c[h], 1);
      x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(c[h], 2);
      x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(c[h], 3);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int word = j < 4 ? c[0] : c[1];
      x[j] = (float)(int8_t)((uint32_t)word >> (8 * (j & 3)));
    }
  }
}

// VPT > 0: the block has at most 256 * VPT vectors of 8, held in registers; 0: any number, read twice.
template <bool F8, int VPT>
__global__ __launch_bounds__(256) void kv_append_block_kernel(KvAppendBlockParams p) {
  const int t = threadIdx.x;
  int id = blockIdx.x;
  const int h = id % p.H_KV;
  id /= p.H_KV;
  const bool is_v = id & 1;
  id >>= 1;
  const int b = id / p.blocks, j = id % p.blocks;
  const int L = p.ctx_len[b];
  int nb = p.n_seqs, ql = p.q_len;
  if (p.plan != nullptr) {
    nb = min(max(p.plan[0], 0), p.B_grid);
    ql = min(max(p.plan[1], 0), p.ql_grid);
  }
  nb = uniform(nb);
  ql = uniform(ql);
  if (b >= nb || ql == 0 || L <= 0) return;
  const int pos0 = uniform(L) - ql;  // position of the first new token (negative ones are skipped)
  const int64_t first = ((int64_t)(max(pos0, 0) / p.SB) + j) * p.SB;
  if (first / p.PAGE >= p.max_pages) return;
  const int lo = (int)first;  // first position of this workgroup's block
  const int n_old = max(pos0 - lo, 0), n_all = min(pos0 + ql - lo, p.SB);  // slots held before, and after
  if (n_all <= n_old) return;

  const int dv = 1 << p.log_dv, n_vec = n_all << p.log_dv;
  const _Float16* src = (is_v ? p.v : p.k) + (int64_t)b * p.s_nb + (int64_t)h * p.s_nh;
  auto load_new = [&](int i) -> v8h {
    return *reinterpret_cast<const v8h*>(src + (int64_t)(lo + (i >> p.log_dv) - pos0) * p.s_nt + 8 * (i & (dv - 1)));
  };
  auto is_new = [&](int i) { return i < n_vec && (i >> p.log_dv) >= n_old; };
  auto is_old = [&](int i) { return i < n_vec && (i >> p.log_dv) < n_old; };
  constexpr int R = VPT > 0 ? VPT : 1;
  v8h x[R];
  v2i c[R];
  if constexpr (VPT > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (is_new(t + 256 * i)) x[i] = load_new(t + 256 * i);
  }
  const int page = uniform(p.bt[(int64_t)b * p.s_bt + lo / p.PAGE]);
  if ((uint32_t)page >= (uint32_t)p.n_pages) return;
  const int slot = lo % p.PAGE;
  uint8_t* codes = (is_v ? p.vc : p.kc) + (int64_t)page * p.s_kp + (int64_t)slot * p.s_ko + (int64_t)h * p.s_kh;
  auto code_at = [&](int i) { return reinterpret_cast<v2i*>(codes + (int64_t)(i >> p.log_dv) * p.s_ko + 8 * (i & (dv - 1))); };
  float* scale = (is_v ? p.vs : p.ks) + (int64_t)page * p.s_sp + (int64_t)(slot / p.SB) * p.s_so + (int64_t)h * p.s_sh;
  float s_old = 0.f;
  if (n_old > 0) s_old = *scale;
  if constexpr (VPT > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (is_old(t + 256 * i)) c[i] = *code_at(t + 256 * i);
  }

  uint32_t top = 0;
  if constexpr (VPT > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (is_new(t + 256 * i)) top = max(top, clean16(x[i]));
  } else {
    for (int i = t; i < n_vec; i += 256)
      if (is_new(i)) {
        v8h v = load_new(i);
        top = max(top, clean16(v));
      }
  }
  __shared__ uint32_t red[4];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  if (lane_id() == 0) red[wave_id()] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  const float amax = (float)__builtin_bit_cast(_Float16, (uint16_t)top);
  constexpr float Q = F8 ? 448.f : 127.f;
  const float s_new = fmaxf(amax, 1e-8f) / Q;
  const float s = n_old > 0 ? fmaxf(s_old, s_new) : s_new;
  const bool grew = n_old > 0 && !(s <= s_old);

  const bool plain = s >= 0x1p-60f && s <= 0x1p60f;  // always, but for a scale of the cache's that was not written here
  const float y = 1.f / s;
  auto put_new = [&](int i, v8h v) {
    if (plain) {
      *code_at(i) = encode8_by<F8>(v, s, y);
    } else {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
      *code_at(i) = encode8<F8>(f, s);
    }
  };
  auto put_old = [&](int i, v2i v) {
    float f[8];
    decode8<F8>(v, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s_old;
    *code_at(i) = encode8<F8>(f, s);
  };
  if constexpr (VPT > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = t + 256 * i;
      if (is_new(v)) put_new(v, x[i]);
    }
    if (grew) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = t + 256 * i;
        if (is_old(v)) put_old(v, c[i]);
      }
    }
  } else {
    for (int v = t; v < n_vec; v += 256) {
      if (is_new(v)) {
        v8h xv = load_new(v);
        clean16(xv);
        put_new(v, xv);
      } else if (grew) {
        put_old(v, *code_at(v));
      }
    }
  }
  if (t == 0) *scale = s;
}

template <bool F8>
static const void* kv_append_block_fn(int per_thread) {
  if (per_thread <= 1) return reinterpret_cast<const void*>(&kv_append_block_kernel<F8, 1>);
  if (per_thread <= 2) return reinterpret_cast<const void*>(&kv_append_block_kernel<F8, 2>);
  if (per_thread <= 4) return reinterpret_cast<const void*>(&kv_append_block_kernel<F8, 4>);
  if (per_thread <= 8) return reinterpret_cast<const void*>(&kv_append_block_kernel<F8, 8>);
  return reinterpret_cast<const void*>(&kv_append_block_kernel<F8, 0>);
}

}  // namespace specq

using namespace specq;

extern "C" int specq_kv_append_block(const void* k_new, const void* v_new, int64_t s_nb, int64_t s_nt, int64_t s_nh,
                                     void* kc, void* vc, int code_fp8, int64_t s_kp, int64_t s_ko, int64_t s_kh,
                                     float* ks, float* vs, int64_t s_sp, int64_t s_sb, int64_t s_sh, int block,
                                     const int32_t* block_tbl, int64_t s_bt, int max_pages, int n_pages,
                                     const int32_t* ctx_len, int B_grid, int n_seqs, int q_len, int ql_grid, int H_KV,
                                     int D, int PAGE, const int32_t* plan, void* stream) {
  clear_error();
  SPECQ_REQUIRE(k_new && v_new && kc && vc && ks && vs && block_tbl && ctx_len, SPECQ_EINVAL,
                "kv_append_block: null tensor pointer");
  SPECQ_REQUIRE(B_grid >= 0 && ql_grid >= 0 && n_seqs >= 0 && n_seqs <= B_grid && q_len >= 0 && q_len <= ql_grid,
                SPECQ_EINVAL, "kv_append_block: need 0 <= n_seqs <= B_grid and 0 <= q_len <= ql_grid");
  SPECQ_REQUIRE(H_KV > 0 && PAGE > 0 && max_pages > 0 && n_pages > 0, SPECQ_EINVAL, "kv_append_block: bad sizes");
  SPECQ_REQUIRE(D == 64 || D == 128 || D == 256, SPECQ_ENOTSUP, "kv_append_block: head_dim %d must be 64, 128 or 256",
                D);
  SPECQ_REQUIRE(block > 0 && block % 16 == 0 && PAGE % block == 0, SPECQ_ENOTSUP,
                "kv_append_block: block=%d must be a multiple of 16 that divides PAGE=%d", block, PAGE);
  SPECQ_REQUIRE((int64_t)max_pages * PAGE <= INT32_MAX - PAGE, SPECQ_ENOTSUP,
                "kv_append_block: block table of %lld tokens is too long", (long long)max_pages * PAGE);
  SPECQ_REQUIRE((uintptr_t)k_new % 16 == 0 && (uintptr_t)v_new % 16 == 0 && s_nb % 8 == 0 && s_nt % 8 == 0 &&
                    s_nh % 8 == 0,
                SPECQ_ENOTSUP, "kv_append_block: new K/V rows must be 16-byte aligned");
  SPECQ_REQUIRE((uintptr_t)kc % 8 == 0 && (uintptr_t)vc % 8 == 0 && s_kp % 8 == 0 && s_ko % 8 == 0 && s_kh % 8 == 0,
                SPECQ_ENOTSUP, "kv_append_block: cache rows must be 8-byte aligned");
  SPECQ_REQUIRE((uintptr_t)ks % 4 == 0 && (uintptr_t)vs % 4 == 0, SPECQ_ENOTSUP,
                "kv_append_block: scales must be 4-byte aligned");
  SPECQ_REQUIRE(lie_apart(n_pages, s_kp, D) && lie_apart(PAGE, s_ko, D) && lie_apart(H_KV, s_kh, D), SPECQ_ENOTSUP,
                "kv_append_block: cache rows overlap");
  SPECQ_REQUIRE(lie_apart(n_pages, s_sp, 1) && lie_apart(PAGE / block, s_sb, 1) && lie_apart(H_KV, s_sh, 1), SPECQ_ENOTSUP,
                "kv_append_block: scales overlap");
  const int tokens = plan ? ql_grid : q_len, seqs = plan ? B_grid : n_seqs;
  if (seqs == 0 || tokens == 0) return SPECQ_OK;
  KvAppendBlockParams p = {};
  p.k = (const _Float16*)k_new; p.v = (const _Float16*)v_new; p.s_nb = s_nb; p.s_nt = s_nt; p.s_nh = s_nh;
  p.kc = (uint8_t*)kc; p.vc = (uint8_t*)vc; p.s_kp = s_kp; p.s_ko = s_ko; p.s_kh = s_kh;
  p.ks = ks; p.vs = vs; p.s_sp = s_sp; p.s_so = s_sb; p.s_sh = s_sh;
  p.bt = block_tbl; p.s_bt = s_bt; p.max_pages = max_pages; p.n_pages = n_pages;
  p.ctx_len = ctx_len; p.plan = plan;
  p.n_seqs = n_seqs; p.q_len = q_len; p.ql_grid = ql_grid; p.B_grid = B_grid; p.H_KV = H_KV; p.PAGE = PAGE;
  p.SB = block;
  p.blocks = ceil_div(tokens - 1, block) + 1;  // tokens in a row reach one block more where they start inside one
  p.log_dv = D == 64 ? 3 : D == 128 ? 4 : 5;
  const int64_t wgs = (int64_t)seqs * p.blocks * 2 * H_KV;
  SPECQ_REQUIRE(wgs <= INT32_MAX, SPECQ_EINVAL, "kv_append_block: grid too large");
  const int64_t vecs = (int64_t)block * D / 8;
  const int per_thread = (int)((vecs + 255) / 256 > 1000 ? 1000 : (vecs + 255) / 256);
  const void* fn = code_fp8 ? kv_append_block_fn<true>(per_thread) : kv_append_block_fn<false>(per_thread);
  return launch(fn, (int)wgs, 256, 0, (hipStream_t)stream, &p);
}
