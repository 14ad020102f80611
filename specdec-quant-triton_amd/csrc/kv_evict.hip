// Eviction from a paged K/V cache by gathered attention weight, and its C ABI.
//
// A sequence b of L = ctx_len[b] > limit tokens is cut back to `budget`: for each KV head h stay its first `sinks` tokens,
// its last `recent` ones, and of the others those of greatest weights[b, h, t], ties to the lower position.  What stays
// keeps its order and moves together: token j of the `budget` comes from position kept[b, h, j], in every cache tensor
// and in the weights.  ctx_len[b] becomes budget.  A sequence whose table names a page outside the pool, or, with page
// counts given, a page that other rows name too, stays as it is.
//
// Selection, one workgroup a (sequence, head): the weights as unsigned keys of the same order (tokens that stay in any
// case have the largest key); the budget-th largest by counting digits of 11, 11 and 10 bits from the top, the lower
// ones over a list of the keys that share the upper one (over all keys where they are too many for it); then one pass in
// the order of the positions that ranks what is above it and the first of what equals it.  Three passes over the weights,
// 16384 at a time, the first 16384 in registers.  One workgroup for a row, so it is bound by latency: the code stands
// in few places (unrolled, it took longer to arrive than to run: 4096 tokens 8 -> 15 us).
//
// Moving is in place.  Token j goes to a place at or below its own, and everything behind it starts above, so it is
// enough that a tile of tokens has been read by all its threads before any of them writes it.  One workgroup walks one
// byte range of the rows of one (sequence, head) of one tensor; ranges are independent, so narrow ranges make more
// workgroups where there are few sequences and heads.  Bound by that walk, one tile after another with a barrier each, in few
// workgroups: 8 sequences of up to 4096 tokens to 2048, 8 heads of 128: 11 us to choose, 24 to move (28 MB read, 26 written; the
// CUs are busy 48 % of the time, since only sequences that are cut have work, and their waves wait in 58 % of it; eight accesses of
// a thread in flight instead of four change nothing); one of 65536 to 8191, two heads of 64: 25 and 25, by 22 workgroups.  By way
// of the workspace, with as many workgroups as there is work, the latter took 10 us less and shorter rows 4 us more.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kEvMove = 512;  // threads that move
constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvBins = 2048;
constexpr int kEvStep = 4 * kEvThreads;  // positions of a chunk, four consecutive ones a thread
constexpr int kEvGroup = 4;              // chunks that are loaded, and ranked, together
constexpr int kEvCopies = 4;             // histograms that lanes take in turn, since many weights share a digit
constexpr int kEvList = 8192;            // keys of one upper digit
constexpr int kEvSlices = 64;            // most slices of a row
constexpr int kEvTensors = 16;  // cache tensors of a call
constexpr int kEvUnits = 256;   // byte ranges of a call
constexpr int kEvPages = 4096;  // table entries whose pages' places are kept in LDS
constexpr int kEvBatch = 4;     // accesses of a thread in flight

struct EvictParams {
  const int32_t* bt; int64_t s_bt; int C, P;
  const int32_t* ref;      // page counts, or null
  int32_t* ctx_len;
  float* w; int64_t s_wb, s_wh; int w_vec;
  int32_t* kept;           // [B, H][budget]
  int32_t* flag;           // workspace, [B, H]: whether the sequence is cut back
  int H, PAGE, cap, budget, recent, sinks, limit;
  // Long rows: slices of slice_len positions (1 to 4 chunks).  Workspace, for each slice: a histogram, whether its pages may be
  // written, its keys above the upper digit and its keys of that digit; for each row that digit and what lies above it.
  int slices, slice_len;
  int32_t* hist; int32_t* slice_ok; int32_t* slice_above; int32_t* slice_n; uint32_t* list; int32_t* digit;
};

struct EvictMoveParams {
  EvictParams e;
  uint8_t* base[kEvTensors];
  int64_t s_p[kEvTensors], s_o[kEvTensors], s_h[kEvTensors];  // bytes from page to page, token to token, head to head
  // Range u: its tensor (kEvTensors: the weights), first byte, bytes and bytes of one access.
  uint8_t tensor[kEvUnits], vec[kEvUnits]; int16_t bytes[kEvUnits]; int32_t first[kEvUnits];
  int units, progs;
  uint32_t page_magic; int page_shift;  // t / PAGE = (t * magic >> 32) >> shift for t below 2^30; magic 0: PAGE = 1
};

// Exclusive prefixes of N values over the workgroup, and their sums.
template <int N>
__device__ __forceinline__ void ev_prefix(int (&x)[N], int (&total)[N], int (&part)[kEvGroup][kEvWaves]) {
  int v[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = x[n];
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x112, 0xf, 0xf, false);
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x114, 0xf, 0xf, false);
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x118, 0xf, 0xf, false);
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
    v[n] += __builtin_amdgcn_update_dpp(0, v[n], 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
  }
  __syncthreads();  // the last call's readers of part are done
  if (lane_id() == kWave - 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) part[n][wave_id()] = v[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    int w = part[n][lane_id() % kEvWaves];  // the waves' sums, then theirs up to each
    w += __builtin_amdgcn_update_dpp(0, w, 0x111, 0xf, 0xf, false);
    w += __builtin_amdgcn_update_dpp(0, w, 0x112, 0xf, 0xf, false);
    w += __builtin_amdgcn_update_dpp(0, w, 0x114, 0xf, 0xf, false);
    w += __builtin_amdgcn_update_dpp(0, w, 0x118, 0xf, 0xf, false);
    const int wave = uniform(wave_id());
    total[n] = __builtin_amdgcn_readlane(w, kEvWaves - 1);
    x[n] = (wave > 0 ? __builtin_amdgcn_readlane(w, max(wave - 1, 0)) : 0) + v[n] - x[n];
  }
}

// A key of the order of the weights; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t ev_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const int u = __builtin_bit_cast(int, w + 0.f);
  return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}

constexpr int kEvSpan = kEvGroup * kEvStep;  // positions of a group
typedef uint32_t EvKeys[kEvGroup][4];

// A (sequence, head)'s row of weights.
struct EvRow {
  const float* w;
  int L, sinks, recent, vec;
  // Whether all of a chunk's tokens compete.
  __device__ __forceinline__ bool inner(int at) const { return at >= sinks && at + kEvStep <= L - recent; }
  // Keys of the thread's positions of the group from g0 on; behind the context 0, which no weight has and none is found to be.
  __device__ __forceinline__ void load(int g0, EvKeys& k) const {
#pragma unroll
    for (int c = 0; c < kEvGroup; ++c) {
      const int t = g0 + c * kEvStep + 4 * (int)threadIdx.x;
      v4f x = {0.f, 0.f, 0.f, 0.f};
      if (vec && t + 4 <= L) {
        x = *reinterpret_cast<const v4f*>(w + t);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < L) x[i] = w[t + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) k[c][i] = ev_key(x[i]);
      if (!inner(g0 + c * kEvStep)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          k[c][i] = t + i >= L ? 0u : t + i < sinks || t + i >= L - recent ? 0xFFFFFFFFu : k[c][i];
      }
    }
  }
};
__device__ __forceinline__ EvRow ev_row(const EvictParams& p, int b, int h, int L) {
  return {p.w + b * p.s_wb + h * p.s_wh, L, p.sinks, p.recent, p.w_vec};
}
// Whether the table's columns c0..c1 - 1 of row b name pages of the pool that no other row names (as far as counts are given).
__device__ __forceinline__ int ev_pages_ok(const EvictParams& p, int b, int c0, int c1) {
  int ok = 1;
  for (int c = c0 + (int)threadIdx.x; c < c1; c += kEvThreads) {
    const int id = p.bt[b * p.s_bt + c];
    if ((uint32_t)id >= (uint32_t)p.P || (p.ref != nullptr && p.ref[id] > 1)) ok = 0;
  }
  return ok;
}

// One digit of the key that is looked for.
struct EvDigit {
  int bin, above, in;  // it, the keys with larger ones, and with it
};
typedef int EvHist[kEvCopies][kEvBins];
// The digit of the want-th largest key, from its histogram (which is cleared).
__device__ __forceinline__ EvDigit ev_digit(EvHist& hist, int want, int (&part)[kEvGroup][kEvWaves], EvDigit& shared) {
  // Thread i has bins 2047 - 2 i and 2046 - 2 i: the prefix runs from the largest digit down.
  const int hi = kEvBins - 1 - 2 * (int)threadIdx.x;
  int n1 = 0, n0 = 0;
#pragma unroll
  for (int c = 0; c < kEvCopies; ++c) {
    v2i* at = reinterpret_cast<v2i*>(&hist[c][hi - 1]);
    const v2i n = *at;
    *at = v2i{0, 0};
    n0 += n[0], n1 += n[1];
  }
  int sum[1] = {n1 + n0}, total[1];
  ev_prefix(sum, total, part);
  const int above = sum[0];
  if (above < want && above + n1 + n0 >= want) {
    const bool first = above + n1 >= want;
    shared = {first ? hi : hi - 1, first ? above : above + n1, first ? n1 : n0};
  }
  __syncthreads();
  return shared;
}

// What is known of the budget-th largest key: the keys from `larger` on stay, and of those that equal `found` the first `want`.
struct EvCut {
  uint32_t found, larger;
  int want;
  bool ties;  // some equal ones do not stay (else they count as larger; the largest key's tokens all stay)
};
__device__ __forceinline__ EvCut ev_cut(uint32_t found, int want, int in) {
  return {found, in == want ? found : found + 1, want, in != want};
}
// Ranks a group's tokens that stay, `above` larger and `equal` equal ones before them.
__device__ __forceinline__ void ev_rank(const EvCut& cut, const EvKeys& k, int g0, int L, int& above, int& equal, int32_t* kept,
                                        int (&part)[kEvGroup][kEvWaves]) {
  int count[kEvGroup], total[kEvGroup];  // larger keys of a chunk, and equal ones above bit 16
#pragma unroll
  for (int c = 0; c < kEvGroup; ++c) {
    count[c] = 0;
    if (g0 + c * kEvStep >= L) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) count[c] += k[c][i] >= cut.larger;
    if (cut.ties) {
#pragma unroll
      for (int i = 0; i < 4; ++i) count[c] += (k[c][i] == cut.found) << 16;
    }
  }
  ev_prefix(count, total, part);
#pragma unroll
  for (int c = 0; c < kEvGroup; ++c) {
    if (g0 + c * kEvStep >= L) break;
    const int t = g0 + c * kEvStep + 4 * (int)threadIdx.x;
    int a = above + (count[c] & 0xFFFF), e = equal + (count[c] >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool gt = k[c][i] >= cut.larger, eq = cut.ties && k[c][i] == cut.found;
      if (gt || (eq && e < cut.want)) kept[a + min(e, cut.want)] = t + i;
      a += gt;
      e += eq;
    }
    above += total[c] & 0xFFFF;
    equal += total[c] >> 16;
  }
}
// A sequence that stays as it is.
__device__ __forceinline__ void ev_stays(const EvictParams& p, int L, int32_t* kept) {
  for (int j = threadIdx.x; j < p.budget; j += kEvThreads) kept[j] = j < L ? j : -1;
}

__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictParams p) {
  __shared__ EvHist hist;
  __shared__ int part[kEvGroup][kEvWaves], s_list_n;
  __shared__ EvDigit s_digit;
  __shared__ uint32_t s_list[kEvList];
  const int prog = blockIdx.x, b = prog / p.H, h = prog - b * p.H, tid = threadIdx.x;
  const int L = min(max(p.ctx_len[b], 0), p.cap);
  int32_t* kept = p.kept + (int64_t)prog * p.budget;
  const EvRow row = ev_row(p, b, h, L);
  for (int i = tid; i < kEvCopies * kEvBins; i += kEvThreads) hist[0][i] = 0;
  int ok = L > p.limit;
  EvKeys near;
  if (ok) {
    row.load(0, near);
    ok = __syncthreads_and(ev_pages_ok(p, b, 0, (L + p.PAGE - 1) / p.PAGE));
  }
  if (tid == 0) p.flag[prog] = ok;
  if (!ok) return ev_stays(p, L, kept);
  auto each = [&](auto&& f) {  // f(first position, keys) of each group
#pragma unroll 1
    for (int g0 = 0; g0 < L; g0 += kEvSpan) {
      EvKeys k;
      if (g0 == 0) {
#pragma unroll
        for (int c = 0; c < kEvGroup; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) k[c][i] = near[c][i];
      } else {
        row.load(g0, k);
      }
      f(g0, k);
    }
  };
  auto keys = [&](auto&& f) {  // f(key) of each key, and of some 0
    each([&](int g0, const EvKeys& k) {
#pragma unroll
      for (int c = 0; c < kEvGroup; ++c) {
        if (g0 + c * kEvStep >= L) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) f(k[c][i]);
      }
    });
  };
  // The budget-th largest key, from its top digit down: `want` of those under the digits found so far.
  uint32_t found = 0, known = 0;  // its digits, and a mask of them
  int want = p.budget, in = 0;
  bool listed = false;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    int* mine = hist[tid % kEvCopies];
    auto count = [&](uint32_t k) {
      if (((k ^ found) & known) == 0) atomicAdd(&mine[(k >> low) & (bins - 1)], 1);
    };
    if (pass == 0) keys([&](uint32_t k) { atomicAdd(&mine[k >> 21], 1); });
    else if (listed) for (int i = tid; i < s_list_n; i += kEvThreads) count(s_list[i]);
    else keys(count);
    if (tid == 0 && pass == 0) s_list_n = 0;
    __syncthreads();
    const EvDigit d = ev_digit(hist, want, part, s_digit);
    found |= (uint32_t)d.bin << low;
    known |= (uint32_t)(bins - 1) << low;
    want -= d.above;
    in = d.in;
    if (pass == 0 && in <= kEvList) {
      listed = true;
      keys([&](uint32_t k) {
        if (((k ^ found) & known) == 0) s_list[atomicAdd(&s_list_n, 1)] = k;
      });
    }
    __syncthreads();
  }
  const EvCut cut = ev_cut(found, want, in);
  int above = 0, equal = 0;
  each([&](int g0, const EvKeys& k) { ev_rank(cut, k, g0, L, above, equal, kept, part); });
}

// ---- The same over slices of long rows, a workgroup each, in three launches: the upper digit's histograms; the digit, from
// all slices' (each workgroup for itself), and the slice's keys that have it, listed; the other digits, from the lists,
// and the ranks, behind those of the slices before.  Plain stores and loads between them.
struct EvSlice {
  int prog, slice, b, h, L, live, g0;  // live: slices with tokens; g0: the slice's first position
  int64_t at;                          // the slice's place among all
};
__device__ __forceinline__ bool ev_slice(const EvictParams& p, EvSlice& s) {
  s.prog = (int)blockIdx.x / p.slices;
  s.slice = (int)blockIdx.x - s.prog * p.slices;
  s.b = s.prog / p.H;
  s.h = s.prog - s.b * p.H;
  s.L = min(max(p.ctx_len[s.b], 0), p.cap);
  s.live = (s.L + p.slice_len - 1) / p.slice_len;
  s.g0 = s.slice * p.slice_len;
  s.at = (int64_t)s.prog * p.slices + s.slice;
  return s.L > p.limit && s.slice < s.live;
}
// Keys of the slice alone: those of later ones in the group are 0.
__device__ __forceinline__ void ev_slice_keys(const EvictParams& p, const EvSlice& s, EvKeys& k) {
  ev_row(p, s.b, s.h, s.L).load(s.g0, k);
#pragma unroll
  for (int c = 0; c < kEvGroup; ++c)
    if (c * kEvStep >= p.slice_len) {
#pragma unroll
      for (int i = 0; i < 4; ++i) k[c][i] = 0;
    }
}

__global__ __launch_bounds__(kEvThreads) void evict_slice_count_kernel(EvictParams p) {
  __shared__ EvHist hist;
  EvSlice s;
  if (!ev_slice(p, s)) return;
  EvKeys k;
  ev_slice_keys(p, s, k);
  for (int i = threadIdx.x; i < kEvCopies * kEvBins; i += kEvThreads) hist[0][i] = 0;
  const int end = min(s.g0 + p.slice_len, s.L);
  const int ok = __syncthreads_and(ev_pages_ok(p, s.b, s.g0 / p.PAGE, (end + p.PAGE - 1) / p.PAGE));
  int* mine = hist[threadIdx.x % kEvCopies];
#pragma unroll
  for (int c = 0; c < kEvGroup; ++c) {
    if (c * kEvStep >= p.slice_len || s.g0 + c * kEvStep >= s.L) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) atomicAdd(&mine[k[c][i] >> 21], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kEvBins; i += kEvThreads) {
    int n = 0;
#pragma unroll
    for (int c = 0; c < kEvCopies; ++c) n += hist[c][i];
    p.hist[s.at * kEvBins + i] = n;
  }
  if (threadIdx.x == 0) p.slice_ok[s.at] = ok;
}

__global__ __launch_bounds__(kEvThreads) void evict_slice_list_kernel(EvictParams p) {
  __shared__ EvHist hist;
  __shared__ int part[kEvGroup][kEvWaves], s_n;
  __shared__ EvDigit s_digit;
  EvSlice s;
  if (!ev_slice(p, s)) return;
  EvKeys k;
  ev_slice_keys(p, s, k);
  const int tid = threadIdx.x;
  v2i sum = {0, 0};
  const int32_t* counts = p.hist + (int64_t)s.prog * p.slices * kEvBins + 2 * tid;
#pragma unroll 8
  for (int i = 0; i < s.live; ++i) sum += *reinterpret_cast<const v2i*>(counts + (int64_t)i * kEvBins);
#pragma unroll
  for (int c = 0; c < kEvCopies; ++c) *reinterpret_cast<v2i*>(&hist[c][2 * tid]) = c == 0 ? sum : v2i{0, 0};
  if (tid == 0) s_n = 0;
  __syncthreads();
  const EvDigit d = ev_digit(hist, p.budget, part, s_digit);
  int above[1] = {0}, total[1];
  uint32_t* list = p.list + s.at * p.slice_len;
#pragma unroll
  for (int c = 0; c < kEvGroup; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int digit = (int)(k[c][i] >> 21);  // 0 is no key's, and not the one found
      above[0] += digit > d.bin;
      if (digit == d.bin) list[atomicAdd(&s_n, 1)] = k[c][i];
    }
  ev_prefix(above, total, part);
  if (tid == 0) {
    p.slice_n[s.at] = s_n;
    p.slice_above[s.at] = total[0];
    if (s.slice == 0) p.digit[2 * s.prog] = d.bin, p.digit[2 * s.prog + 1] = d.above;
  }
}

__global__ __launch_bounds__(kEvThreads) void evict_slice_rank_kernel(EvictParams p) {
  __shared__ EvHist hist;
  __shared__ int part[kEvGroup][kEvWaves];
  __shared__ EvDigit s_digit;
  __shared__ int s_n[kEvSlices], s_before[2];
  EvSlice s;
  const bool some = ev_slice(p, s);
  int32_t* kept = p.kept + (int64_t)s.prog * p.budget;
  const int64_t first = (int64_t)s.prog * p.slices;
  const int tid = threadIdx.x, wave = uniform(wave_id()), lane = lane_id();
  int ok = s.L > p.limit;
  if (ok) {
    ok = __syncthreads_and(tid < s.live ? p.slice_ok[first + tid] : 1);
  }
  if (s.slice == 0) {
    if (tid == 0) p.flag[s.prog] = ok;
    if (!ok) ev_stays(p, s.L, kept);
  }
  if (!ok || !some) return;
  EvKeys k;
  ev_slice_keys(p, s, k);
  for (int i = tid; i < kEvCopies * kEvBins; i += kEvThreads) hist[0][i] = 0;
  if (tid < s.live) s_n[tid] = p.slice_n[first + tid];
  if (tid < 2) s_before[tid] = 0;
  __syncthreads();
  uint32_t found = (uint32_t)p.digit[2 * s.prog] << 21, known = 0x7FFu << 21;
  int want = p.budget - p.digit[2 * s.prog + 1], in = 0;
  auto lists = [&](auto&& f) {  // f(slice, key); a wave takes every 16th slice's
    for (int i = wave; i < s.live; i += kEvWaves) {
      const uint32_t* list = p.list + (first + i) * p.slice_len;
      const int n = s_n[i];
#pragma unroll 4
      for (int j = lane; j < n; j += kWave) f(i, list[j]);
    }
  };
#pragma unroll 1
  for (int pass = 1; pass < 3; ++pass) {
    const int low = pass == 1 ? 10 : 0, bins = pass == 1 ? 2048 : 1024;
    int* mine = hist[tid % kEvCopies];
    lists([&](int, uint32_t k) {
      if (((k ^ found) & known) == 0) atomicAdd(&mine[(k >> low) & (bins - 1)], 1);
    });
    __syncthreads();
    const EvDigit d = ev_digit(hist, want, part, s_digit);
    found |= (uint32_t)d.bin << low;
    known |= (uint32_t)(bins - 1) << low;
    want -= d.above;
    in = d.in;
    __syncthreads();
  }
  const EvCut cut = ev_cut(found, want, in);
  // What stays of the slices before: their keys of larger digits, and of their lists.
  int above = tid < s.slice ? p.slice_above[first + tid] : 0, equal = 0;
  lists([&](int i, uint32_t k) {
    if (i >= s.slice) return;
    above += k >= cut.larger;
    equal += cut.ties && k == cut.found;
  });
  if (above != 0) atomicAdd(&s_before[0], above);
  if (equal != 0) atomicAdd(&s_before[1], equal);
  __syncthreads();
  above = s_before[0], equal = s_before[1];
  ev_rank(cut, k, s.g0, s.L, above, equal, kept, part);
}

// One byte range of one (sequence, head): accesses of sizeof(T) bytes, `lanes` of them a token.
template <typename T, typename F>
__device__ __forceinline__ void evict_walk(const int32_t* kept, int budget, int lanes, F&& place) {
  const int per = kEvMove / lanes, sub = (int)threadIdx.x % lanes, mine = (int)threadIdx.x / lanes;
  const bool on = mine < per;
  auto source = [&](int j) { return on && j < budget ? kept[j] : -1; };
  auto take = [&](int j0, T (&x)[kEvBatch], int (&src)[kEvBatch]) {
#pragma unroll
    for (int k = 0; k < kEvBatch; ++k) {
      const int j = j0 + k * per + mine, s = src[k];
      if (s > j) x[k] = *reinterpret_cast<const T*>(place(s) + sub * sizeof(T));
    }
  };
  int src[kEvBatch], next[kEvBatch];
  T x[kEvBatch], y[kEvBatch];
#pragma unroll
  for (int k = 0; k < kEvBatch; ++k) x[k] = T{}, y[k] = T{}, src[k] = source(k * per + mine);
  take(0, x, src);
  const int step = kEvBatch * per;
#pragma unroll
  for (int k = 0; k < kEvBatch; ++k) next[k] = source(step + k * per + mine);
  for (int j0 = 0; j0 < budget; j0 += step) {
    take(j0 + step, y, next);
    int after[kEvBatch];
#pragma unroll
    for (int k = 0; k < kEvBatch; ++k) after[k] = source(j0 + 2 * step + k * per + mine);
    // The tile has been read, by every thread, before anything of it is written.
#pragma unroll
    for (int k = 0; k < kEvBatch; ++k) {
      if constexpr (sizeof(T) >= 4) asm volatile("" ::"v"(x[k]));
      else asm volatile("" ::"v"((int)x[k]));
    }
    wg_barrier();
#pragma unroll
    for (int k = 0; k < kEvBatch; ++k) {
      const int j = j0 + k * per + mine;
      if (src[k] > j) *reinterpret_cast<T*>(place(j) + sub * sizeof(T)) = x[k];
      x[k] = y[k];
      src[k] = next[k];
      next[k] = after[k];
    }
  }
}

__global__ __launch_bounds__(kEvMove) void evict_move_kernel(EvictMoveParams p) {
  __shared__ int64_t pages[kEvPages];
  const EvictParams& e = p.e;
  // The ranges of one (sequence, head) run eight workgroups apart, on one XCD, whose L2 holds the lines they share.
  const int u = (int)(blockIdx.x / 8) % p.units, prog = (int)(blockIdx.x / 8) / p.units * 8 + (int)blockIdx.x % 8;
  if (prog >= p.progs) return;
  const int b = prog / e.H, h = prog - b * e.H;
  const int flag = e.flag[prog];
  const int32_t* kept = e.kept + (int64_t)prog * e.budget;
  const int tensor = p.tensor[u], vec = p.vec[u], lanes = p.bytes[u] / vec;
  if (tensor == kEvTensors) {
    if (!uniform(flag)) return;
    if (h == 0 && threadIdx.x == 0) e.ctx_len[b] = e.budget;  // the selection is over, and this launch does not read it
    float* w = e.w + b * e.s_wb + h * e.s_wh;
    evict_walk<float>(kept, e.budget, 1, [&](int t) { return reinterpret_cast<uint8_t*>(w + t); });
    return;
  }
  const int32_t* row = e.bt + b * e.s_bt;
  const int64_t s_p = p.s_p[tensor], s_o = p.s_o[tensor];
  const bool near = e.C <= kEvPages;
  if (near)
    for (int c = threadIdx.x; c < e.C; c += kEvMove) pages[c] = row[c] * s_p;
  __syncthreads();
  if (!uniform(flag)) return;
  uint8_t* base = p.base[tensor] + h * p.s_h[tensor] + p.first[u];
  auto place = [&](int t) {
    const int c = p.page_magic != 0 ? (int)(__umulhi((uint32_t)t, p.page_magic) >> p.page_shift) : t;
    return base + (near ? pages[c] : row[c] * s_p) + (t - c * e.PAGE) * s_o;
  };
  if (vec == 16) evict_walk<v4i>(kept, e.budget, lanes, place);
  else if (vec == 4) evict_walk<int32_t>(kept, e.budget, lanes, place);
  else if (vec == 2) evict_walk<uint16_t>(kept, e.budget, lanes, place);
  else evict_walk<uint8_t>(kept, e.budget, lanes, place);
}

}  // namespace specq

using namespace specq;

namespace specq {
namespace {

// Slices of a row of `cap` positions, where it is cut: long rows, few enough to leave half of the CUs idle.  One workgroup takes
// some 9 us and 2 more for each 4096 positions (65536 of two heads: 37 us), the three launches 25.
struct EvSpace { int slices, slice_len; size_t words; };  // words of the workspace behind the flags
EvSpace ev_space(int64_t progs, int64_t cap, int64_t cus) {
  const int64_t chunks = ceil_div64(cap, kEvStep), per = ceil_div64(chunks, kEvSlices);
  if (chunks <= 8 || per > kEvGroup || 2 * progs > cus) return {0, 0, 0};
  const int slices = (int)ceil_div64(chunks, per), len = (int)per * kEvStep;
  return {slices, len, (size_t)progs * (2 + (size_t)slices * (kEvBins + 3 + len))};
}
size_t ev_workspace(int64_t progs, const EvSpace& s) { return kCounterBytes + align_up((size_t)progs * 4, 256) + s.words * 4; }

}  // namespace
}  // namespace specq

extern "C" size_t specq_kv_evict_workspace_size(int B, int H_KV, int max_pages, int PAGE) {
  if (B <= 0 || H_KV <= 0 || max_pages <= 0 || PAGE <= 0) return 0;
  const int64_t progs = (int64_t)B * H_KV;
  return ev_workspace(progs, ev_space(progs, (int64_t)max_pages * PAGE, device_cus()));
}

extern "C" int specq_kv_evict(const int32_t* block_tbl, int64_t s_bt, int B, int max_pages, const int32_t* ref, int n_pages,
                              int32_t* ctx_len, float* weights, int64_t s_wb, int64_t s_wh, int H_KV, int PAGE,
                              int n_tensors, void* const* base, const int64_t* page_stride, const int64_t* token_stride,
                              const int64_t* head_stride, const int64_t* row_bytes, int budget, int recent, int sinks,
                              int limit, int32_t* kept, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  SPECQ_REQUIRE(block_tbl && ctx_len && weights && kept, SPECQ_EINVAL, "kv_evict: null tensor pointer");
  SPECQ_REQUIRE(B > 0 && H_KV > 0 && max_pages > 0 && n_pages > 0 && PAGE > 0 && s_bt >= max_pages, SPECQ_EINVAL,
                "kv_evict: bad sizes B=%d H_KV=%d columns=%d pages=%d PAGE=%d", B, H_KV, max_pages, n_pages, PAGE);
  const int64_t cap = (int64_t)max_pages * PAGE, progs = (int64_t)B * H_KV;
  SPECQ_REQUIRE(cap <= (1 << 30) && progs <= (1 << 22), SPECQ_ENOTSUP, "kv_evict: a table of %lld tokens or %lld rows is too large",
                (long long)cap, (long long)progs);
  // Either launch is of fewer than 2^32 threads, or neither is made.
  SPECQ_REQUIRE(progs * kEvThreads <= UINT32_MAX, SPECQ_ENOTSUP, "kv_evict: %lld sequences x heads to choose from", (long long)progs);
  SPECQ_REQUIRE(budget > 0 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget && limit >= budget, SPECQ_EINVAL,
                "kv_evict: need 0 <= recent + sinks <= budget <= limit and budget > 0 (recent=%d sinks=%d budget=%d limit=%d)",
                recent, sinks, budget, limit);
  SPECQ_REQUIRE(budget <= (1 << 30), SPECQ_ENOTSUP, "kv_evict: a budget of %d tokens", budget);
  SPECQ_REQUIRE((uintptr_t)weights % 4 == 0 && nest_apart({{B, s_wb}, {H_KV, s_wh}}, cap), SPECQ_ENOTSUP,
                "kv_evict: rows of the weights overlap or are shorter than the table's %lld tokens", (long long)cap);
  SPECQ_REQUIRE(n_tensors >= 0 && n_tensors <= kEvTensors, SPECQ_ENOTSUP, "kv_evict: %d cache tensors (at most %d)", n_tensors,
                kEvTensors);
  SPECQ_REQUIRE(n_tensors == 0 || (base && page_stride && token_stride && head_stride && row_bytes), SPECQ_EINVAL,
                "kv_evict: bad tensor list");
  EvictMoveParams m = {};
  EvictParams& p = m.e;
  for (int i = 0; i < n_tensors; ++i) {
    SPECQ_REQUIRE(base[i] && row_bytes[i] > 0 && row_bytes[i] <= 4096, SPECQ_EINVAL,
                  "kv_evict: cache tensor %d is null, or its rows of %lld bytes are not 1 to 4096", i, (long long)row_bytes[i]);
    for (int j = 0; j < i; ++j)
      SPECQ_REQUIRE(base[j] != base[i], SPECQ_EINVAL, "kv_evict: cache tensors %d and %d are one", j, i);
    SPECQ_REQUIRE(nest_apart({{n_pages, page_stride[i]}, {PAGE, token_stride[i]}, {H_KV, head_stride[i]}}, row_bytes[i]),
                  SPECQ_ENOTSUP, "kv_evict: rows of cache tensor %d overlap", i);
    m.base[i] = static_cast<uint8_t*>(base[i]);
    m.s_p[i] = page_stride[i]; m.s_o[i] = token_stride[i]; m.s_h[i] = head_stride[i];
  }
  const EvSpace space = ev_space(progs, cap, device_cus());
  const size_t need = ev_workspace(progs, space);
  SPECQ_REQUIRE(workspace && workspace_bytes >= need, SPECQ_ENOSPC, "kv_evict: workspace of %zu bytes required, %zu given", need,
                workspace ? workspace_bytes : (size_t)0);
  p.bt = block_tbl; p.s_bt = s_bt; p.C = max_pages; p.P = n_pages; p.ref = ref; p.ctx_len = ctx_len;
  p.w = weights; p.s_wb = s_wb; p.s_wh = s_wh;
  p.w_vec = (uintptr_t)weights % 16 == 0 && s_wb % 4 == 0 && s_wh % 4 == 0;
  p.kept = kept;
  p.flag = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + kCounterBytes);
  p.H = H_KV; p.PAGE = PAGE; p.cap = (int)cap; p.budget = budget; p.recent = recent; p.sinks = sinks; p.limit = limit;
  // Byte ranges: pieces of 128 bytes, or of less, down to 16, until there are three workgroups for two CUs.
  const int64_t cus = device_cus();
  int64_t piece = 128;
  auto ranges = [&](int64_t size) {
    int64_t n = 1;
    for (int i = 0; i < n_tensors; ++i) n += ceil_div64(row_bytes[i], size);
    return n;
  };
  while (piece > 16 && 2 * progs * ranges(piece) < 3 * cus) piece /= 2;
  while (ranges(piece) > kEvUnits) piece *= 2;
  for (int i = 0; i < n_tensors; ++i) {
    const uint64_t bits = (uintptr_t)base[i] | (uint64_t)page_stride[i] | (uint64_t)token_stride[i] | (uint64_t)head_stride[i] |
                          (uint64_t)row_bytes[i];
    const int vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    for (int64_t at = 0; at < row_bytes[i]; at += piece) {
      const int u = m.units++;
      m.tensor[u] = (uint8_t)i;
      m.vec[u] = (uint8_t)vec;
      m.first[u] = (int32_t)at;
      m.bytes[u] = (int16_t)(row_bytes[i] - at < piece ? row_bytes[i] - at : piece);
    }
  }
  m.tensor[m.units] = kEvTensors; m.vec[m.units] = 4; m.bytes[m.units] = 4;
  ++m.units;
  m.progs = (int)progs;
  const int64_t moves = (int64_t)align_up(progs, 8) * m.units;
  SPECQ_REQUIRE(moves * kEvMove <= UINT32_MAX, SPECQ_ENOTSUP, "kv_evict: %lld sequences x heads of %d byte ranges each are too many",
                (long long)progs, m.units);
  if (PAGE > 1) {
    int bits = 0;  // ceil(log2(PAGE))
    while ((1ll << bits) < PAGE) ++bits;
    // ceil(2^k / PAGE), k = 30 + bits, is off by less than PAGE <= 2^bits in 2^k, so its products with t < 2^30 by less than one.
    const uint64_t magic = ((1ull << (30 + bits)) + PAGE - 1) / PAGE;
    m.page_magic = (uint32_t)(bits < 2 ? magic << (2 - bits) : magic);
    m.page_shift = bits < 2 ? 0 : bits - 2;
  }
  hipStream_t st = (hipStream_t)stream;
  if (space.slices == 0) {
    if (int rc = launch(reinterpret_cast<const void*>(&evict_select_kernel), (int)progs, kEvThreads, 0, st, &p)) return rc;
  } else {
    const int64_t n = progs * space.slices;
    p.slices = space.slices;
    p.slice_len = space.slice_len;
    p.hist = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + kCounterBytes + align_up((size_t)progs * 4, 256));
    p.list = reinterpret_cast<uint32_t*>(p.hist + n * kEvBins);
    p.slice_ok = p.hist + n * (kEvBins + space.slice_len);
    p.slice_above = p.slice_ok + n;
    p.slice_n = p.slice_above + n;
    p.digit = p.slice_n + n;
    for (const void* fn : {reinterpret_cast<const void*>(&evict_slice_count_kernel),
                           reinterpret_cast<const void*>(&evict_slice_list_kernel),
                           reinterpret_cast<const void*>(&evict_slice_rank_kernel)})
      if (int rc = launch(fn, (int)n, kEvThreads, 0, st, &p)) return rc;
  }
  return launch(reinterpret_cast<const void*>(&evict_move_kernel), (int)moves, kEvMove, 0, st, &m);
}
