// Beam search: the selection over beams and vocabulary, and the reordering of the batch's states.  C ABI.
//
// Selection, for each sequence b of W beams with scores c_w (log-probabilities so far) and logits x_w over V tokens:
//   c_w,v = c_w + x_w,v - log sum_u exp(x_w,u);   a finished beam has one candidate, its eos, with the score it has
// and the best n of the W V candidates, ties to the lower beam, then the lower token.  A candidate whose score is NaN or
// -infinity is none; where there are fewer than n the rest is (-inf, -1, -1).
//
// One pass over the logits, which is what bounds it.  A wave owns a segment of a row and keeps it in registers: its
// maximum and sum of exponentials, and its candidates.  The n-th largest of the 64 lanes' maxima is a value that at least n
// of the segment's reach, so what reaches it holds the segment's best n and few more; these go to the workspace, up to 64.
// Where more reach it (rows of equal values) the best n are taken one by one.
// The last workgroup of a sequence joins the segments: each row's sum, in fp64, then the candidates' scores, in fp64 too,
// since beams whose scores lie closer than an fp32 step apart are to be told apart as the formula does; the same
// two steps -- a value that n reach, then the few that do, ranked against one another -- give the selection.  Neither the
// order of arrival nor that of the list has a part in the result.
//
// Reordering: row r of every state becomes row parents[r] of the same group of rows.  In place: a thread owns one column of
// up to 16 bytes of a group's rows, reads what changes and then writes it.  Bound by HBM.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / kWave;
constexpr int kBeamMax = 64;    // beams of a sequence, and candidates selected
constexpr int kBeamSlots = 64;  // candidates of a segment
constexpr int kBeamList = 768;  // candidates ranked against one another

struct BeamParams {
  const void* x; int64_t s_xb, s_xw;
  const float* scores; int64_t s_sb;
  const uint8_t* done; int64_t s_db; int eos;
  float* out_score; int32_t* out_token; int32_t* out_parent;
  int W, V, n;
  int segs;  // of a row
  int wgs;   // of a sequence: ceil(W segs / 4)
  // Workspace, of each segment: (max, sum), the number of candidates, and they: (value, token).
  uint64_t* stats; int32_t* counts; uint64_t* cands;
  int32_t* counters;  // [B]
};

__device__ __forceinline__ uint64_t beam_pack(float a, uint32_t b) {
  return (uint64_t)__builtin_bit_cast(uint32_t, a) | ((uint64_t)b << 32);
}
__device__ __forceinline__ float beam_lo(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }
__device__ __forceinline__ float beam_hi(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)(x >> 32)); }

// The n-th largest (1 <= n <= 64) of the lanes' values, no NaN among them: its key bit by bit.
__device__ __forceinline__ float beam_nth(float v, int n) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v), key = (u >> 31) ? ~u : u | 0x80000000u;
  uint32_t at = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t up = at | (1u << bit);
    if (__popcll(__builtin_amdgcn_ballot_w64(key >= up)) >= n) at = up;
  }
  return __builtin_bit_cast(float, (at >> 31) ? at & 0x7FFFFFFFu : ~at);
}

// Whether (a, i) comes before (b, j).
template <typename T, typename I>
__device__ __forceinline__ bool beam_before(T a, I i, T b, I j) { return a > b || (a == b && i < j); }

// NV 16-byte vectors of a lane: the wave's segment is 64 NV of them.  They count from the row's start, wherever that lies (a
// load need only be aligned to its elements): equal rows have equal sums, to the bit, and their candidates tie.
template <typename T, int NV>
__device__ __forceinline__ void beam_segment(const BeamParams& p, int b, int f, uint64_t (&slots)[kBeamSlots]) {
  constexpr int VE = 16 / sizeof(T), E = NV * VE;
  const int w = f / p.segs, seg = f - w * p.segs, lane = lane_id();
  const int64_t at = (int64_t)b * p.W * p.segs + f;
  if (p.done != nullptr && p.done[b * p.s_db + w] != 0) {
    // One candidate of value 0 in a row whose sum is exp(0).
    if (lane == 0) {
      publish(p.stats + at, seg == 0 ? beam_pack(0.f, __builtin_bit_cast(uint32_t, 1.f)) : beam_pack(-INFINITY, 0));
      publish(p.counts + at, seg == 0 ? 1 : 0);
      if (seg == 0) publish(p.cands + at * kBeamSlots, beam_pack(0.f, (uint32_t)p.eos));
    }
    return;
  }
  const T* row = static_cast<const T*>(p.x) + b * p.s_xb + w * p.s_xw;
  const int first = (seg * NV * kWave + lane) * VE;  // the lane's first token; vector k is 64 vectors on
  float x[E];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int t = first + k * kWave * VE;
    if (t + VE <= p.V) {
      typedef T vec __attribute__((ext_vector_type(VE), aligned(sizeof(T))));
      const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec*>(row + t));
#pragma unroll
      for (int e = 0; e < VE; ++e) x[k * VE + e] = (float)v[e];
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) x[k * VE + e] = t + e < p.V ? (float)row[t + e] : -INFINITY;
    }
  }
  float mine = -INFINITY;
#pragma unroll
  for (int k = 0; k < E; ++k) mine = fmaxf(mine, x[k]);
  float m = mine;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) sum += fast_exp2((x[k] - ref) * 1.44269504088896340736f);
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) sum += __shfl_xor(sum, o);
  const float least = fmaxf(beam_nth(mine, p.n), -3.402823466e38f);
  auto token = [&](int k) { return first + (k / VE) * kWave * VE + k % VE; };
  int count = 0;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const bool in = x[k] >= least;
    const uint64_t who = __builtin_amdgcn_ballot_w64(in);
    if (who == 0) continue;
    const int slot = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (in && slot < kBeamSlots) slots[slot] = beam_pack(x[k], (uint32_t)token(k));
    count += __popcll(who);
  }
  if (count > kBeamSlots) {
    // One by one: the best behind the last taken.
    float last = INFINITY;
    int last_t = -1;
    count = 0;
    for (int i = 0; i < p.n; ++i) {
      float best = -INFINITY;
      int best_t = INT32_MAX;
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (x[k] > best && beam_before(last, last_t, x[k], token(k))) best = x[k], best_t = token(k);
#pragma unroll
      for (int o = 1; o < kWave; o *= 2) {
        const float v = __shfl_xor(best, o);
        const int t = __shfl_xor(best_t, o);
        if (beam_before(v, t, best, best_t)) best = v, best_t = t;
      }
      if (best == -INFINITY) break;
      if (lane == 0) slots[i] = beam_pack(best, (uint32_t)best_t);
      last = best, last_t = best_t;
      ++count;
    }
  }
  wait_lgkm0();
  if (lane == 0) {
    publish(p.stats + at, beam_pack(m, __builtin_bit_cast(uint32_t, sum)));
    publish(p.counts + at, count);
  }
  if (lane < count) publish(p.cands + at * kBeamSlots + lane, slots[lane]);
}

__device__ __forceinline__ double beam_shfl(double v, int o) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor((uint32_t)u, o), hi = __shfl_xor((uint32_t)(u >> 32), o);
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

template <typename T, int NV>
__global__ __launch_bounds__(kBeamThreads) void beam_select_kernel(BeamParams p) {
  __shared__ uint64_t slots[kBeamWaves][kBeamSlots];
  __shared__ double s_lse[kBeamMax], s_score[kBeamMax], s_key[kBeamList], s_best[kBeamWaves];
  __shared__ uint64_t s_at[kBeamList], s_best_at[kBeamWaves];
  __shared__ float s_least[kBeamWaves];
  __shared__ int s_last, s_count;
  const int b = (int)blockIdx.x / p.wgs, wave = uniform(wave_id()), lane = lane_id();
  const int f = ((int)blockIdx.x - b * p.wgs) * kBeamWaves + wave, all = p.W * p.segs;
  if (f < all) beam_segment<T, NV>(p, b, f, slots[wave]);
  if (!arrive_last(p.counters + b, p.wgs, &s_last)) return;

  // The rows' sums.
  const int64_t base = (int64_t)b * all;
  for (int w = wave; w < p.W; w += kBeamWaves) {
    float m = -INFINITY;
    for (int k = lane; k < p.segs; k += kWave) m = fmaxf(m, beam_lo(collect(p.stats + base + w * p.segs + k)));
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    double sum = 0;
    for (int k = lane; k < p.segs; k += kWave) {
      const uint64_t v = collect(p.stats + base + w * p.segs + k);
      if (beam_lo(v) > -INFINITY || !(beam_hi(v) == 0.f)) sum += (double)beam_hi(v) * exp((double)beam_lo(v) - (double)m);
    }
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) sum += beam_shfl(sum, o);
    if (lane == 0) {
      s_lse[w] = (double)m + log(sum);
      s_score[w] = (double)p.scores[b * p.s_sb + w];
    }
  }
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  // f(score, (beam, token)) of the candidates a lane has; a segment's go to other lanes than the next one's.
  auto each = [&](auto&& g) {
    for (int f0 = kWave * wave; f0 < all; f0 += kWave * kBeamWaves) {
      const int mine = f0 + lane < all ? collect(p.counts + base + f0 + lane) : 0;
      const int fs = min(kWave, all - f0);
#pragma unroll 4
      for (int k = 0; k < fs; ++k) {
        const int n = __builtin_amdgcn_readlane(mine, k), i = (lane + 11 * k) & (kWave - 1);
        if (i >= n) continue;
        const int w = (f0 + k) / p.segs;
        const uint64_t c = collect(p.cands + (base + f0 + k) * kBeamSlots + i);
        const double key = ((double)beam_lo(c) - s_lse[w]) + s_score[w];
        if (key > -(double)INFINITY) g(key, ((uint64_t)w << 32) | (c >> 32));
      }
    }
  };
  // A score that n candidates reach, as a float (rounding keeps the order).
  float best = -INFINITY;
  each([&](double key, uint64_t) { best = fmaxf(best, (float)key); });
  const float reach = beam_nth(best, p.n);
  if (lane == 0) s_least[wave] = reach;
  __syncthreads();
  float least = s_least[0];
#pragma unroll
  for (int v = 1; v < kBeamWaves; ++v) least = fmaxf(least, s_least[v]);
  each([&](double key, uint64_t at) {
    if ((float)key < least) return;
    const int i = atomicAdd(&s_count, 1);
    if (i < kBeamList) s_key[i] = key, s_at[i] = at;
  });
  __syncthreads();
  const int count = s_count;
  auto put = [&](int i, double key, uint64_t at) {
    const int64_t o = (int64_t)b * p.n + i;
    p.out_score[o] = (float)key;
    p.out_token[o] = (int32_t)(uint32_t)at;
    p.out_parent[o] = b * p.W + (int)(at >> 32);
  };
  auto none = [&](int i) {
    const int64_t o = (int64_t)b * p.n + i;
    p.out_score[o] = -INFINITY;
    p.out_token[o] = p.out_parent[o] = -1;
  };
  if (count <= kBeamList) {
    for (int i = threadIdx.x; i < count; i += kBeamThreads) {
      const double key = s_key[i];
      const uint64_t at = s_at[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += beam_before(s_key[j], s_at[j], key, at);
      if (rank < p.n) put(rank, key, at);
    }
    for (int i = count + (int)threadIdx.x; i < p.n; i += kBeamThreads) none(i);
    return;
  }
  // More than the list holds reach it (equal rows): one by one.
  double last = INFINITY;
  uint64_t last_at = 0;
  for (int i = 0; i < p.n; ++i) {
    double top = -INFINITY;
    uint64_t top_at = ~0ull;
    each([&](double key, uint64_t at) {
      const bool behind = i == 0 || beam_before(last, last_at, key, at);
      if (behind && beam_before(key, at, top, top_at)) top = key, top_at = at;
    });
#pragma unroll
    for (int o = 1; o < kWave; o *= 2) {
      const double v = beam_shfl(top, o);
      const uint64_t a = __builtin_bit_cast(uint64_t, beam_shfl(__builtin_bit_cast(double, top_at), o));
      if (beam_before(v, a, top, top_at)) top = v, top_at = a;
    }
    if (lane == 0) s_best[wave] = top, s_best_at[wave] = top_at;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kBeamWaves; ++v)
      if (beam_before(s_best[v], s_best_at[v], top, top_at)) top = s_best[v], top_at = s_best_at[v];
    __syncthreads();
    if (threadIdx.x == 0) {
      if (top > -(double)INFINITY) put(i, top, top_at);
      else none(i);
    }
    last = top, last_at = top_at;
  }
}

// ---- Reordering.
constexpr int kReorderTensors = 64;
constexpr int kReorderMax = 32;  // rows of a group

struct ReorderParams {
  uint8_t* base[kReorderTensors];
  int64_t stride[kReorderTensors], bytes[kReorderTensors];  // bytes from row to row, and of a row
  int32_t first[kReorderTensors + 1];                       // workgroups of a group before this tensor's
  uint8_t vec[kReorderTensors];                             // bytes of an access
  const int32_t* parents;
  int W, tensors;
};

template <typename T, int WB>
__device__ __forceinline__ void reorder_column(uint8_t* at, int64_t stride, const int32_t* parents, int W, int row0) {
  T x[WB];
  int from[WB];
#pragma unroll
  for (int i = 0; i < WB; ++i) {
    from[i] = i < W ? uniform(parents[i]) - row0 : i;
    const bool moves = (uint32_t)from[i] < (uint32_t)W && from[i] != i;
    if (!moves) from[i] = -1;
    x[i] = T{};
    if (moves) x[i] = *reinterpret_cast<const T*>(at + from[i] * stride);
  }
#pragma unroll
  for (int i = 0; i < WB; ++i)
    if (from[i] >= 0) *reinterpret_cast<T*>(at + i * stride) = x[i];
}

template <int WB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderParams p) {
  const int per = p.first[p.tensors], g = (int)blockIdx.x / per, u = (int)blockIdx.x - g * per;
  int i = 0;
  while (u >= p.first[i + 1]) ++i;
  const int vec = p.vec[i], row0 = g * p.W;
  const int64_t off = ((int64_t)(u - p.first[i]) * 256 + threadIdx.x) * vec;
  if (off >= p.bytes[i]) return;
  uint8_t* at = p.base[i] + row0 * p.stride[i] + off;
  const int32_t* parents = p.parents + row0;
  if (vec == 16) reorder_column<v4i, WB>(at, p.stride[i], parents, p.W, row0);
  else if (vec == 4) reorder_column<int32_t, WB>(at, p.stride[i], parents, p.W, row0);
  else reorder_column<uint8_t, WB>(at, p.stride[i], parents, p.W, row0);
}

// Vectors of a lane: 8, and 2 where 8 would give fewer than four waves to a CU.
static int beam_vectors(int64_t rows, int V, int size, int cus) {
  return rows * ceil_div64((int64_t)V * size, 16 * kWave * 8) < 4 * cus ? 2 : 8;
}
static int64_t beam_segs(int V, int size, int nv) {
  return ceil_div64((int64_t)V * size, 16 * kWave * nv);
}

}  // namespace specq

using namespace specq;

extern "C" size_t specq_beam_select_workspace_size(int B, int W, int V, int logits_fp32) {
  if (B <= 0 || W <= 0 || V <= 0) return 0;
  const int size = logits_fp32 ? 4 : 2;
  const size_t segs = (size_t)B * W * beam_segs(V, size, beam_vectors((int64_t)B * W, V, size, device_cus()));
  return kCounterBytes + align_up(segs * 4, 256) + segs * (8 + 8 * kBeamSlots);
}

extern "C" int specq_beam_select(const void* logits, int logits_fp32, int64_t s_lb, int64_t s_lw, const float* scores,
                                 int64_t s_sb, const uint8_t* finished, int64_t s_fb, int eos, float* out_scores,
                                 int32_t* out_tokens, int32_t* out_parents, int B, int W, int V, int n, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  clear_error();
  SPECQ_REQUIRE(logits && scores && out_scores && out_tokens && out_parents, SPECQ_EINVAL, "beam_select: null tensor pointer");
  SPECQ_REQUIRE(B >= 0 && W > 0 && V > 0 && n > 0, SPECQ_EINVAL, "beam_select: bad sizes B=%d W=%d V=%d n=%d", B, W, V, n);
  SPECQ_REQUIRE(W <= kBeamMax && n <= kBeamMax, SPECQ_ENOTSUP, "beam_select: %d beams, %d candidates (at most %d supported)", W,
                n, kBeamMax);
  SPECQ_REQUIRE(V <= (1 << 28) && B <= kMaxCounters && (int64_t)B * W <= INT32_MAX, SPECQ_ENOTSUP,
                "beam_select: vocabulary or batch too large");
  SPECQ_REQUIRE(!finished || (eos >= 0 && eos < V), SPECQ_EINVAL, "beam_select: eos %d is no token of %d", eos, V);
  SPECQ_REQUIRE((uintptr_t)logits % (logits_fp32 ? 4 : 2) == 0 && (uintptr_t)scores % 4 == 0, SPECQ_EINVAL,
                "beam_select: logits and scores must be aligned to their type");
  if (B == 0) return SPECQ_OK;
  const int size = logits_fp32 ? 4 : 2, nv = beam_vectors((int64_t)B * W, V, size, device_cus());
  const int64_t segs = beam_segs(V, size, nv), wgs = ceil_div64(W * segs, kBeamWaves);
  SPECQ_REQUIRE(B * wgs <= INT32_MAX, SPECQ_ENOTSUP, "beam_select: grid too large");
  const size_t need = specq_beam_select_workspace_size(B, W, V, logits_fp32);
  SPECQ_REQUIRE(workspace && workspace_bytes >= need, SPECQ_ENOSPC, "beam_select: workspace of %zu bytes required, %zu given",
                need, workspace ? workspace_bytes : (size_t)0);
  BeamParams p = {};
  p.x = logits; p.s_xb = s_lb; p.s_xw = s_lw; p.scores = scores; p.s_sb = s_sb;
  p.done = finished; p.s_db = s_fb; p.eos = eos;
  p.out_score = out_scores; p.out_token = out_tokens; p.out_parent = out_parents;
  p.W = W; p.V = V; p.n = n; p.segs = (int)segs; p.wgs = (int)wgs;
  const size_t count = (size_t)B * W * segs;
  char* at = static_cast<char*>(workspace);
  p.counters = reinterpret_cast<int32_t*>(at);
  p.counts = reinterpret_cast<int32_t*>(at + kCounterBytes);
  p.stats = reinterpret_cast<uint64_t*>(at + kCounterBytes + align_up(count * 4, 256));
  p.cands = p.stats + count;
  const void* fn = logits_fp32 ? (nv == 8 ? reinterpret_cast<const void*>(&beam_select_kernel<float, 8>)
                                          : reinterpret_cast<const void*>(&beam_select_kernel<float, 2>))
                               : (nv == 8 ? reinterpret_cast<const void*>(&beam_select_kernel<_Float16, 8>)
                                          : reinterpret_cast<const void*>(&beam_select_kernel<_Float16, 2>));
  return launch(fn, (int)(B * wgs), kBeamThreads, 0, (hipStream_t)stream, &p);
}

extern "C" int specq_beam_reorder(const int32_t* parents, int rows, int group, int n_tensors, void* const* base,
                                  const int64_t* row_stride, const int64_t* row_bytes, void* stream) {
  clear_error();
  SPECQ_REQUIRE(rows >= 0 && group > 0 && rows % group == 0, SPECQ_EINVAL, "beam_reorder: %d rows are no groups of %d", rows, group);
  SPECQ_REQUIRE(group <= kReorderMax, SPECQ_ENOTSUP, "beam_reorder: groups of %d rows (at most %d supported)", group, kReorderMax);
  SPECQ_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || (base && row_stride && row_bytes)), SPECQ_EINVAL,
                "beam_reorder: bad tensor list");
  SPECQ_REQUIRE(parents || rows == 0, SPECQ_EINVAL, "beam_reorder: null tensor pointer");
  for (int i = 0; i < n_tensors; ++i) {
    SPECQ_REQUIRE(base[i] && row_bytes[i] > 0 && (rows <= 1 || row_stride[i] >= row_bytes[i]), SPECQ_EINVAL,
                  "beam_reorder: state %d is null, empty or overlaps its own rows", i);
    for (int j = 0; j < i; ++j) SPECQ_REQUIRE(base[j] != base[i], SPECQ_EINVAL, "beam_reorder: states %d and %d are one", j, i);
  }
  if (rows == 0 || group == 1) return SPECQ_OK;
  const void* fn = group <= 4 ? reinterpret_cast<const void*>(&beam_reorder_kernel<4>)
                   : group <= 8 ? reinterpret_cast<const void*>(&beam_reorder_kernel<8>)
                   : group <= 16 ? reinterpret_cast<const void*>(&beam_reorder_kernel<16>)
                                 : reinterpret_cast<const void*>(&beam_reorder_kernel<32>);
  for (int t0 = 0; t0 < n_tensors; t0 += kReorderTensors) {
    ReorderParams p = {};
    p.parents = parents;
    p.W = group;
    int64_t per = 0;
    for (int t = t0; t < n_tensors && t < t0 + kReorderTensors; ++t) {
      const int i = p.tensors++;
      p.base[i] = static_cast<uint8_t*>(base[t]);
      p.stride[i] = row_stride[t];
      p.bytes[i] = row_bytes[t];
      const uint64_t bits = (uintptr_t)base[t] | (uint64_t)row_stride[t] | (uint64_t)row_bytes[t];
      p.vec[i] = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
      per += ceil_div64(row_bytes[t], 256 * p.vec[i]);
      SPECQ_REQUIRE(per <= INT32_MAX / (rows / group), SPECQ_ENOTSUP, "beam_reorder: states too large");
      p.first[i + 1] = (int32_t)per;
    }
    if (int rc = launch(fn, (int)(per * (rows / group)), 256, 0, (hipStream_t)stream, &p)) return rc;
  }
  return SPECQ_OK;
}
