// Beam search: the selection over beams and vocabulary, and the reordering of the batch's states.  C ABI.
//
// Selection, for each sequence b of W beams with scores c_w (log-probabilities so far) and logits x_w over V tokens:
//   c_w,v = c_w + x_w,v - log sum_u exp(x_w,u);   a finished beam has one candidate, its eos, with the score it has
// and the best n of the W V candidates, ties to the lower beam, then the lower token.  A candidate whose score, rounded to fp32, is
// NaN or -infinity is none; where there are fewer than n the rest is (-inf, -1, -1).
//
// One pass over the logits, which is what bounds it, and a second launch over what it leaves.
//   1  A workgroup owns a part of a row and keeps it in registers: its maximum and sum of exponentials, and its
//      candidates.  If k of the 64 lanes' maxima reach a value in each of the four waves, 4 k values of the part do; with k the
//      fourth part of n, what reaches the least such value of a wave holds the part's best n and few more.  These are left
//      for 2, at most kBeamSlots of them; where more reach it (equal values) the best n are taken one by one.
//   2  A workgroup to a sequence joins each row's sums and forms the candidates' scores.  Again a value that n reach, then the
//      few that do, ranked against one another.  The order in which lists are filled has no part in the result.
// Exponentials (within 2^-34 of themselves), sums, logarithms and scores are fp64, so beams are told apart as the formula does
// where their scores lie closer than fp32 steps: fp32 sums put a row's log-sum off by 2^-23, and with it all of its beam.
//
// 16 x 8 rows of 128257 fp32 logits, a quarter of them finished: 21.4 us (50 MB; with fp32 exponentials 17.1) and 9.0; 4 of 32000
// fp16: 5.9 and 5.8.  An exponential is 16 fp64 instructions of the rate of fp32 ones, and vector instructions have 58 % of a busy
// CU's cycles: they follow the loads of a wave instead of running beside them.  Fewer vectors a lane, for more waves, leave the first
// launch as it is and give the second more parts to join (4: 13 us); sums that start with the first loads keep more registers (1 us
// more).  The second launch waits for memory three times over, whatever its size.
//
// Reordering: row r of every state becomes row parents[r] of the same group of rows.  In place: a thread owns one column of
// up to 16 bytes of a group's rows, reads what changes and then writes it.  16 x 8 rows of 418 KB, 57 MB: 16.2 us from HBM (3.5
// TB/s), 11.7 where the last-level cache holds them from one call to the next.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / kWave;
constexpr int kBeamJoin = 1024, kBeamJoinWaves = kBeamJoin / kWave;  // threads of the second launch
constexpr int kBeamMax = 64;     // beams of a sequence, and candidates selected
constexpr int kBeamSlots = 128;  // candidates of a part
constexpr int kBeamList = 1024;  // candidates ranked against one another
// Threads of the second launch that share a part.  32 (and two slots, or a slot of four parts, read ahead): 11.7 us instead of 8.8 for
// 16 x 8 rows of 16 parts; 16: 10.3.
constexpr int kBeamGroup = 8;
constexpr int kBeamNear = 3;     // slots of a thread read ahead

struct BeamParams {
  const void* x; int64_t s_xb, s_xw;
  const float* scores; int64_t s_sb;
  const uint8_t* done; int64_t s_db; int eos;
  float* out_score; int32_t* out_token; int32_t* out_parent;
  int W, V, n;
  int parts;  // of a row
  // Workspace, of each part: maximum, sum, the number of candidates, and they: (value, token).
  float* tops; double* sums; int32_t* counts; uint64_t* cands;
};

__device__ __forceinline__ uint64_t beam_pack(float a, uint32_t b) {
  return (uint64_t)__builtin_bit_cast(uint32_t, a) | ((uint64_t)b << 32);
}
__device__ __forceinline__ float beam_lo(uint64_t x) { return __builtin_bit_cast(float, (uint32_t)x); }

// exp(x - ref), ref >= x.  The difference comes first, exact where it counts whatever the logits' size; then 2^n of the nearest whole
// number n, which adding 1.5 * 2^52 leaves in the lower bits, and a polynomial that meets 2^f on |f| <= 1/2 in the Chebyshev points
// of degree 7, off by at most 2^-34 of itself.  What is below 2^-1000 counts as that; -infinity too, and NaN.
__device__ __forceinline__ double beam_exp(float x, double ref) {
  constexpr double kWhole = 6755399441055744.;
  const double t = fmax(((double)x - ref) * 1.4426950408889634074, -1000.), w = t + kWhole, f = t - (w - kWhole);
  double e = 1.5303699001378845e-05;
  e = fma(e, f, 1.5469729140704658e-04);
  e = fma(e, f, 1.3333478480888061e-03);
  e = fma(e, f, 9.618025613598036e-03);
  e = fma(e, f, 5.550410906317715e-02);
  e = fma(e, f, 2.4022651213495422e-01);
  e = fma(e, f, 6.931471805568341e-01);
  e = fma(e, f, 9.999999999595622e-01);
  v2i u = __builtin_bit_cast(v2i, e);
  u[1] += __builtin_bit_cast(v2i, w)[0] << 20;
  return __builtin_bit_cast(double, u);
}
__device__ __forceinline__ double beam_shfl(double v, int o) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor((uint32_t)u, o), hi = __shfl_xor((uint32_t)(u >> 32), o);
  return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// Values that at least i and j (1..64) of the lanes' values reach, no NaN among them: the i-th and the j-th largest with the
// lower half of their keys cut off (found bit by bit; all 32 would take twice the time and spare few candidates).
struct BeamNth { float i, j; };
__device__ __forceinline__ BeamNth beam_nth(float v, int i, int j) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v), key = ((u >> 31) ? ~u : u | 0x80000000u) >> 16;
  uint32_t a = 0, b = 0;
#pragma unroll 4
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t up_a = a | (1u << bit), up_b = b | (1u << bit);
    if (__popcll(__builtin_amdgcn_ballot_w64(key >= up_a)) >= i) a = up_a;
    if (__popcll(__builtin_amdgcn_ballot_w64(key >= up_b)) >= j) b = up_b;
  }
  // The least value of the key's upper half; that of -infinity's holds NaN as well, and is -infinity.
  auto value = [](uint32_t k) {
    return (k >> 15) ? __builtin_bit_cast(float, (k << 16) & 0x7FFFFFFFu) : k <= 0x007Fu ? -INFINITY : __builtin_bit_cast(float, ~(k << 16));
  };
  return {value(a), value(b)};
}

// Whether (a, i) comes before (b, j).
template <typename T, typename I>
__device__ __forceinline__ bool beam_before(T a, I i, T b, I j) { return a > b || (a == b && i < j); }

// NV 16-byte vectors of a lane.  They count from the row's start, wherever that lies (a load need only be aligned to its
// elements): equal rows have equal sums, to the bit, and their candidates tie.
template <typename T, int NV>
__global__ __launch_bounds__(kBeamThreads) void beam_part_kernel(BeamParams p) {
  constexpr int VE = 16 / sizeof(T), E = NV * VE;
  __shared__ uint64_t slots[kBeamSlots];
  __shared__ double s_sum[kBeamWaves];
  __shared__ float s_max[kBeamWaves], s_some[kBeamWaves], s_all[kBeamWaves];
  __shared__ int s_token[kBeamWaves], s_count;
  const int64_t at = blockIdx.x;
  const int part = (int)(at % p.parts), row_id = (int)(at / p.parts), b = row_id / p.W, w = row_id - b * p.W;
  const int wave = uniform(wave_id()), lane = lane_id();
  if (p.done != nullptr && p.done[b * p.s_db + w] != 0) {
    // One candidate of value 0 in a row whose sum is exp(0).
    if (threadIdx.x == 0) {
      p.tops[at] = part == 0 ? 0.f : -INFINITY;
      p.sums[at] = part == 0 ? 1. : 0.;
      p.counts[at] = part == 0 ? 1 : 0;
      if (part == 0) p.cands[at * kBeamSlots] = beam_pack(0.f, (uint32_t)p.eos);
    }
    return;
  }
  const T* row = static_cast<const T*>(p.x) + b * p.s_xb + w * p.s_xw;
  const int first = ((part * kBeamWaves + wave) * NV * kWave + lane) * VE;  // the lane's first token; vector k is 64 vectors on
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
  if (threadIdx.x == 0) s_count = 0;
  float mine = -INFINITY;
#pragma unroll
  for (int k = 0; k < E; ++k) mine = fmaxf(mine, x[k]);
  float m = mine;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
  const double ref = m == -INFINITY ? 0. : (double)m;
  double sum = 0;
  bool nan = m == INFINITY;
#pragma unroll
  for (int k = 0; k < E; k += 2) {
    nan |= __builtin_isunordered(x[k], x[k + 1]);
    sum += beam_exp(x[k], ref);
    sum += beam_exp(x[k + 1], ref);
  }
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) sum += beam_shfl(sum, o);
  // Nothing, where there is no value; a row that holds NaN or +infinity has no sum.
  if (m == -INFINITY) sum = 0;
  if (__builtin_amdgcn_ballot_w64(nan) != 0) sum = __builtin_nan("");
  const BeamNth nth = beam_nth(mine, (p.n + kBeamWaves - 1) / kBeamWaves, p.n);
  if (lane == 0) s_max[wave] = m, s_sum[wave] = sum, s_some[wave] = nth.i, s_all[wave] = nth.j;
  __syncthreads();
  float least = -3.402823466e38f, low = INFINITY, top = -INFINITY;
#pragma unroll
  for (int v = 0; v < kBeamWaves; ++v) {
    least = fmaxf(least, s_all[v]);
    low = fminf(low, s_some[v]);
    top = fmaxf(top, s_max[v]);
  }
  least = fmaxf(least, low);
  auto token = [&](int k) { return first + (k / VE) * kWave * VE + k % VE; };
  if (m >= least) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const bool in = x[k] >= least;
      if (__builtin_amdgcn_ballot_w64(in) == 0) continue;
      if (in) {
        const int slot = atomicAdd(&s_count, 1);
        if (slot < kBeamSlots) slots[slot] = beam_pack(x[k], (uint32_t)token(k));
      }
    }
  }
  __syncthreads();
  int count = s_count;
  if (count > kBeamSlots) {
    // One by one: the best behind the last taken.
    float last = INFINITY;
    int last_t = -1;
    for (count = 0; count < p.n; ++count) {
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
      if (lane == 0) s_some[wave] = best, s_token[wave] = best_t;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < kBeamWaves; ++v)
        if (beam_before(s_some[v], s_token[v], best, best_t)) best = s_some[v], best_t = s_token[v];
      __syncthreads();
      if (best == -INFINITY) break;
      if (threadIdx.x == 0) slots[count] = beam_pack(best, (uint32_t)best_t);
      last = best, last_t = best_t;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < count; i += kBeamThreads) p.cands[at * kBeamSlots + i] = slots[i];
  // The waves' sums, a lane each.
  double all = threadIdx.x < kBeamWaves ? s_sum[threadIdx.x] : 0.;
  // A NaN sum stays one, whatever its wave's maximum.
  if (threadIdx.x < kBeamWaves && all != 0.) all *= beam_exp(s_max[threadIdx.x], top);
#pragma unroll
  for (int o = 1; o < kBeamWaves; o *= 2) all += beam_shfl(all, o);
  if (threadIdx.x == 0) {
    p.tops[at] = top;
    p.sums[at] = all;
    p.counts[at] = count;
  }
}

// One workgroup runs it once, so the time its instructions take to arrive counts: every step stands in the code once, the
// passes over the candidates among them.
__global__ __launch_bounds__(kBeamJoin) void beam_join_kernel(BeamParams p) {
  __shared__ double s_lse[kBeamMax], s_score[kBeamMax], s_key[kBeamList], s_best[kBeamJoinWaves];
  __shared__ uint64_t s_at[kBeamList], s_best_at[kBeamJoinWaves];
  __shared__ float s_some[kBeamJoinWaves], s_whole[kBeamJoinWaves];
  __shared__ int s_count;
  const int b = blockIdx.x, wave = uniform(wave_id()), lane = lane_id(), all = p.W * p.parts;
  const int64_t base = (int64_t)b * all;
  // A thread has every kBeamGroup-th candidate slot of every kStep-th part; the first kBeamNear of its first part are read at
  // once, before the part's count is known (what lies behind it is not looked at), others where they are used.
  const int slot = threadIdx.x % kBeamGroup, part0 = (int)threadIdx.x / kBeamGroup;
  constexpr int kStep = kBeamJoin / kBeamGroup;
  uint64_t near[kBeamNear];
  const int count0 = part0 < all ? p.counts[base + part0] : 0;
#pragma unroll
  for (int k = 0; k < kBeamNear; ++k) near[k] = p.cands[(base + min(part0, all - 1)) * kBeamSlots + slot + k * kBeamGroup];
  // The rows' sums.
  for (int w = wave; w < p.W; w += kBeamJoinWaves) {
    const float* tops = p.tops + base + w * p.parts;
    const double* sums = p.sums + base + w * p.parts;
    const float top0 = lane < p.parts ? tops[lane] : -INFINITY;
    const double sum0 = lane < p.parts ? sums[lane] : 0.;
    const float score = p.scores[b * p.s_sb + w];
    float m = top0;
    for (int k = lane + kWave; k < p.parts; k += kWave) m = fmaxf(m, tops[k]);
    for (int o = 1; o < kWave; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    double sum = 0;
    for (int k = lane; k < p.parts; k += kWave) {
      const float t = k == lane ? top0 : tops[k];
      const double v = k == lane ? sum0 : sums[k];
      if (v != 0.) sum += v * beam_exp(t, m);
    }
    for (int o = 1; o < kWave; o *= 2) sum += beam_shfl(sum, o);
    if (lane == 0) {
      s_lse[w] = (double)m + log(sum);
      s_score[w] = (double)score;
    }
  }
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  // Pass 0 finds a score that n candidates reach, as a float (rounding keeps the order), as in the first launch; pass 1
  // lists those that do; where they are more than the list holds (equal rows), pass 2 + i finds the i-th best.
  float best = -INFINITY, least = -INFINITY;
  double last = INFINITY;
  uint64_t last_at = 0;
  for (int pass = 0;; ++pass) {
    double top = -INFINITY;
    uint64_t top_at = ~0ull;
    for (int part = part0; part < all; part += kStep) {
      const bool first = part == part0;
      const int n = first ? count0 : p.counts[base + part];
      const int w = part / p.parts;
      for (int i = slot, k = 0; i < n; i += kBeamGroup, ++k) {
        uint64_t c = near[0];
#pragma unroll
        for (int j = 1; j < kBeamNear; ++j)
          if (k == j) c = near[j];
        if (!first || k >= kBeamNear) c = p.cands[(base + part) * kBeamSlots + i];
        const double key = ((double)beam_lo(c) - s_lse[w]) + s_score[w];
        const uint64_t at = ((uint64_t)w << 32) | (c >> 32);
        if ((float)key > -INFINITY) {  // as it is given out: one that fp32 has no number for is none
          if (pass == 0) {
            best = fmaxf(best, (float)key);
          } else if (pass == 1) {
            if ((float)key >= least) {
              const int to = atomicAdd(&s_count, 1);
              if (to < kBeamList) s_key[to] = key, s_at[to] = at;
            }
          } else if ((pass == 2 || beam_before(last, last_at, key, at)) && beam_before(key, at, top, top_at)) {
            top = key, top_at = at;
          }
        }
      }
    }
    auto put = [&](int i, double key, uint64_t at) {
      const int64_t o = (int64_t)b * p.n + i;
      const bool some = (float)key > -INFINITY;
      p.out_score[o] = (float)key;
      p.out_token[o] = some ? (int32_t)(uint32_t)at : -1;
      p.out_parent[o] = some ? b * p.W + (int)(at >> 32) : -1;
    };
    if (pass == 0) {
      const BeamNth nth = beam_nth(best, (p.n + kBeamJoinWaves - 1) / kBeamJoinWaves, p.n);
      if (lane == 0) s_some[wave] = nth.i, s_whole[wave] = nth.j;
      __syncthreads();
      float low = INFINITY;
      for (int v = 0; v < kBeamJoinWaves; ++v) {
        least = fmaxf(least, s_whole[v]);
        low = fminf(low, s_some[v]);
      }
      least = fmaxf(least, low);
    } else if (pass == 1) {
      __syncthreads();
      const int count = s_count;
      if (count > kBeamList) continue;
      // Eight lanes rank a candidate.  Places behind the candidates are empty.
      for (int i = threadIdx.x / 8; i < max(count, p.n); i += kBeamJoin / 8) {
        const double key = i < count ? s_key[i] : -INFINITY;
        const uint64_t at = i < count ? s_at[i] : 0;
        int rank = 0;
        if (i < count)
          for (int j = threadIdx.x % 8; j < count; j += 8) rank += beam_before(s_key[j], s_at[j], key, at);
        for (int o = 1; o < 8; o *= 2) rank += __shfl_xor(rank, o);
        if (i >= count) rank = i;
        if (threadIdx.x % 8 == 0 && rank < p.n) put(rank, key, at);
      }
      return;
    } else {
      for (int o = 1; o < kWave; o *= 2) {
        const double v = beam_shfl(top, o);
        const uint64_t a = __builtin_bit_cast(uint64_t, beam_shfl(__builtin_bit_cast(double, top_at), o));
        if (beam_before(v, a, top, top_at)) top = v, top_at = a;
      }
      if (lane == 0) s_best[wave] = top, s_best_at[wave] = top_at;
      __syncthreads();
      for (int v = 0; v < kBeamJoinWaves; ++v)
        if (beam_before(s_best[v], s_best_at[v], top, top_at)) top = s_best[v], top_at = s_best_at[v];
      __syncthreads();
      if (threadIdx.x == 0) put(pass - 2, top, top_at);
      last = top, last_at = top_at;
      if (pass == p.n + 1) return;
    }
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

// Vectors of a lane: 8, and 2 where 8 would give less than a workgroup to a CU.
static int beam_vectors(int64_t rows, int V, int size, int cus) {
  return rows * ceil_div64((int64_t)V * size, 16 * kBeamThreads * 8) < cus ? 2 : 8;
}
static int64_t beam_parts(int V, int size, int nv) { return ceil_div64((int64_t)V * size, 16 * kBeamThreads * nv); }

}  // namespace specq

using namespace specq;

extern "C" size_t specq_beam_select_workspace_size(int B, int W, int V, int logits_fp32) {
  if (B <= 0 || W <= 0 || V <= 0) return 0;
  const int size = logits_fp32 ? 4 : 2;
  const size_t parts = (size_t)B * W * beam_parts(V, size, beam_vectors((int64_t)B * W, V, size, device_cus()));
  return kCounterBytes + align_up(parts * 4, 256) + parts * (8 + 8 * kBeamSlots + 4);
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
  SPECQ_REQUIRE(V <= (1 << 28) && (int64_t)B * W <= INT32_MAX, SPECQ_ENOTSUP,
                "beam_select: vocabulary or batch too large");
  SPECQ_REQUIRE(!finished || (eos >= 0 && eos < V), SPECQ_EINVAL, "beam_select: eos %d is no token of %d", eos, V);
  SPECQ_REQUIRE((uintptr_t)logits % (logits_fp32 ? 4 : 2) == 0 && (uintptr_t)scores % 4 == 0, SPECQ_EINVAL,
                "beam_select: logits and scores must be aligned to their type");
  if (B == 0) return SPECQ_OK;
  const int size = logits_fp32 ? 4 : 2, nv = beam_vectors((int64_t)B * W, V, size, device_cus());
  const int64_t parts = beam_parts(V, size, nv), count = (int64_t)B * W * parts;
  SPECQ_REQUIRE(count <= INT32_MAX, SPECQ_ENOTSUP, "beam_select: grid too large");
  const size_t need = specq_beam_select_workspace_size(B, W, V, logits_fp32);
  SPECQ_REQUIRE(workspace && workspace_bytes >= need, SPECQ_ENOSPC, "beam_select: workspace of %zu bytes required, %zu given",
                need, workspace ? workspace_bytes : (size_t)0);
  BeamParams p = {};
  p.x = logits; p.s_xb = s_lb; p.s_xw = s_lw; p.scores = scores; p.s_sb = s_sb;
  p.done = finished; p.s_db = s_fb; p.eos = eos;
  p.out_score = out_scores; p.out_token = out_tokens; p.out_parent = out_parents;
  p.W = W; p.V = V; p.n = n; p.parts = (int)parts;
  char* at = static_cast<char*>(workspace) + kCounterBytes;
  p.counts = reinterpret_cast<int32_t*>(at);
  p.sums = reinterpret_cast<double*>(at + align_up((size_t)count * 4, 256));
  p.cands = reinterpret_cast<uint64_t*>(p.sums + count);
  p.tops = reinterpret_cast<float*>(p.cands + count * kBeamSlots);
  const void* fn = logits_fp32 ? (nv == 8 ? reinterpret_cast<const void*>(&beam_part_kernel<float, 8>)
                                          : reinterpret_cast<const void*>(&beam_part_kernel<float, 2>))
                               : (nv == 8 ? reinterpret_cast<const void*>(&beam_part_kernel<_Float16, 8>)
                                          : reinterpret_cast<const void*>(&beam_part_kernel<_Float16, 2>));
  if (int rc = launch(fn, (int)count, kBeamThreads, 0, (hipStream_t)stream, &p)) return rc;
  return launch(reinterpret_cast<const void*>(&beam_join_kernel), B, kBeamJoin, 0, (hipStream_t)stream, &p);
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
    SPECQ_REQUIRE(base[i] != parents, SPECQ_EINVAL, "beam_reorder: the parents are no state");
    for (int j = 0; j < i; ++j) SPECQ_REQUIRE(base[j] != base[i], SPECQ_EINVAL, "beam_reorder: states %d and %d are one", j, i);
  }
  if (rows == 0 || group == 1) return SPECQ_OK;
  const void* fn = group <= 4 ? reinterpret_cast<const void*>(&beam_reorder_kernel<4>)
                   : group <= 8 ? reinterpret_cast<const void*>(&beam_reorder_kernel<8>)
                   : group <= 16 ? reinterpret_cast<const void*>(&beam_reorder_kernel<16>)
                                 : reinterpret_cast<const void*>(&beam_reorder_kernel<32>);
  auto access = [&](int t) {
    const uint64_t bits = (uintptr_t)base[t] | (uint64_t)row_stride[t] | (uint64_t)row_bytes[t];
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  };
  // No launch of a call is too large: one that is refused has changed nothing.
  const int64_t most = UINT32_MAX / 256 / (rows / group);
  int64_t per = 0;
  for (int t = 0; t < n_tensors; ++t) {
    if (t % kReorderTensors == 0) per = 0;
    per += ceil_div64(row_bytes[t], 256 * access(t));
    SPECQ_REQUIRE(per <= most, SPECQ_ENOTSUP, "beam_reorder: states too large");
  }
  for (int t0 = 0; t0 < n_tensors; t0 += kReorderTensors) {
    ReorderParams p = {};
    p.parents = parents;
    p.W = group;
    per = 0;
    for (int t = t0; t < n_tensors && t < t0 + kReorderTensors; ++t) {
      const int i = p.tensors++;
      p.base[i] = static_cast<uint8_t*>(base[t]);
      p.stride[i] = row_stride[t];
      p.bytes[i] = row_bytes[t];
      p.vec[i] = access(t);
      per += ceil_div64(row_bytes[t], 256 * p.vec[i]);
      p.first[i + 1] = (int32_t)per;
    }
    if (int rc = launch(fn, (int)(per * (rows / group)), 256, 0, (hipStream_t)stream, &p)) return rc;
  }
  return SPECQ_OK;
}
