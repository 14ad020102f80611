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
// workgroups where there are few sequences and heads.
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

__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int hist[kEvCopies][kEvBins], part[kEvGroup][kEvWaves], s_bin, s_above, s_in, s_list_n;
  __shared__ uint32_t s_list[kEvList];
  const int prog = blockIdx.x, b = prog / p.H, h = prog - b * p.H, tid = threadIdx.x;
  const int L = min(max(p.ctx_len[b], 0), p.cap);
  int32_t* kept = p.kept + (int64_t)prog * p.budget;
  const float* wr = p.w + b * p.s_wb + h * p.s_wh;
  constexpr int kSpan = kEvGroup * kEvStep;
  // Whether all of a chunk's tokens compete.
  auto inner = [&](int at) { return at >= p.sinks && at + kEvStep <= L - p.recent; };
  // Keys of the thread's positions of the group from g0 on; behind the context 0, which no weight has and none is found to be.
  auto load = [&](int g0, uint32_t (&k)[kEvGroup][4]) {
#pragma unroll
    for (int c = 0; c < kEvGroup; ++c) {
      const int t = g0 + c * kEvStep + 4 * tid;
      v4f x = {0.f, 0.f, 0.f, 0.f};
      if (p.w_vec && t + 4 <= L) {
        x = *reinterpret_cast<const v4f*>(wr + t);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t + i < L) x[i] = wr[t + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) k[c][i] = ev_key(x[i]);
      if (!inner(g0 + c * kEvStep)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          k[c][i] = t + i >= L ? 0u : t + i < p.sinks || t + i >= L - p.recent ? 0xFFFFFFFFu : k[c][i];
      }
    }
  };
  for (int i = tid; i < kEvCopies * kEvBins; i += kEvThreads) hist[0][i] = 0;
  int ok = L > p.limit;
  uint32_t near[kEvGroup][4];
  if (ok) {
    load(0, near);
    const int32_t* row = p.bt + b * p.s_bt;
    for (int c = tid; c < (L + p.PAGE - 1) / p.PAGE; c += kEvThreads) {
      const int id = row[c];
      if ((uint32_t)id >= (uint32_t)p.P || (p.ref != nullptr && p.ref[id] > 1)) ok = 0;
    }
    ok = __syncthreads_and(ok);
  }
  if (tid == 0) p.flag[prog] = ok;
  if (!ok) {
    for (int j = tid; j < p.budget; j += kEvThreads) kept[j] = j < L ? j : -1;
    return;
  }
  // f(chunk of the group, the thread's four keys) of each chunk with tokens; `group` behind each four.
  auto each = [&](auto&& f, auto&& group) {
#pragma unroll 1
    for (int g0 = 0; g0 < L; g0 += kSpan) {
      uint32_t k[kEvGroup][4];
      if (g0 == 0) {
#pragma unroll
        for (int c = 0; c < kEvGroup; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) k[c][i] = near[c][i];
      } else {
        load(g0, k);
      }
#pragma unroll
      for (int c = 0; c < kEvGroup; ++c) {
        const int at = g0 + c * kEvStep;
        if (at < L) f(c, k[c]);
      }
      group(g0, k);
    }
  };
  auto nothing = [](int, const uint32_t (&)[kEvGroup][4]) {};
  // The budget-th largest key, from its top digit down: `want` of those under the digits found so far.
  uint32_t found = 0, known = 0;  // its digits, and a mask of them
  int want = p.budget;
  bool listed = false;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass < 2 ? 2048 : 1024;
    int* mine = hist[tid % kEvCopies];
    if (pass == 0) {
      each([&](int, const uint32_t (&k)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) atomicAdd(&mine[k[i] >> 21], 1);
      }, nothing);
    } else if (listed) {
      for (int i = tid; i < s_list_n; i += kEvThreads)
        if (((s_list[i] ^ found) & known) == 0) atomicAdd(&mine[(s_list[i] >> low) & (bins - 1)], 1);
    } else {
      each([&](int, const uint32_t (&k)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (((k[i] ^ found) & known) == 0) atomicAdd(&mine[(k[i] >> low) & (bins - 1)], 1);
      }, nothing);
    }
    __syncthreads();
    // Thread i has bins 2047 - 2 i and 2046 - 2 i, and clears them: the prefix runs from the largest digit down.
    const int hi = kEvBins - 1 - 2 * tid;
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
      s_bin = first ? hi : hi - 1;
      s_above = first ? above : above + n1;
      s_in = first ? n1 : n0;
    }
    if (tid == 0 && pass == 0) s_list_n = 0;
    __syncthreads();
    found |= (uint32_t)s_bin << low;
    known |= (uint32_t)(bins - 1) << low;
    want -= s_above;
    if (pass == 0 && s_in <= kEvList) {
      listed = true;
      each([&](int, const uint32_t (&k)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (((k[i] ^ found) & known) == 0) s_list[atomicAdd(&s_list_n, 1)] = k[i];
      }, nothing);
    }
    __syncthreads();
  }
  // `want` keys equal to `found` stay, the lowest positions; everything larger stays.  Counts of a chunk: larger keys, and equal
  // ones above bit 16; where all equal ones stay, they count as larger.
  const uint32_t larger = s_in == want ? found : found + 1;  // (the largest key's tokens all stay)
  const bool ties = s_in != want;
  int above = 0, equal = 0, count[kEvGroup] = {0, 0, 0, 0};
  each([&](int c, const uint32_t (&k)[4]) {
    int x = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) x += k[i] >= larger;
    if (ties) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x += (k[i] == found) << 16;
    }
    count[c] = x;
  }, [&](int g0, const uint32_t (&k)[kEvGroup][4]) {
    int total[kEvGroup];
    ev_prefix(count, total, part);
#pragma unroll
    for (int c = 0; c < kEvGroup; ++c) {
      if (g0 + c * kEvStep >= L) break;
      const int t = g0 + c * kEvStep + 4 * tid;
      int a = above + (count[c] & 0xFFFF), e = equal + (count[c] >> 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool gt = k[c][i] >= larger, eq = ties && k[c][i] == found;
        if (gt || (eq && e < want)) kept[a + min(e, want)] = t + i;
        a += gt;
        e += eq;
      }
      above += total[c] & 0xFFFF;
      equal += total[c] >> 16;
      count[c] = 0;
    }
  });
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

extern "C" size_t specq_kv_evict_workspace_size(int B, int H_KV) {
  if (B <= 0 || H_KV <= 0) return 0;
  return kCounterBytes + align_up((size_t)B * H_KV * 4, 256);
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
  SPECQ_REQUIRE(budget > 0 && recent >= 0 && sinks >= 0 && (int64_t)recent + sinks <= budget && limit >= budget, SPECQ_EINVAL,
                "kv_evict: need 0 <= recent + sinks <= budget <= limit and budget > 0 (recent=%d sinks=%d budget=%d limit=%d)",
                recent, sinks, budget, limit);
  SPECQ_REQUIRE((uintptr_t)weights % 4 == 0 && lie_apart(B, s_wb, cap) && lie_apart(H_KV, s_wh, cap), SPECQ_ENOTSUP,
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
    SPECQ_REQUIRE(lie_apart(n_pages, page_stride[i], row_bytes[i]) && lie_apart(PAGE, token_stride[i], row_bytes[i]) &&
                      lie_apart(H_KV, head_stride[i], row_bytes[i]),
                  SPECQ_ENOTSUP, "kv_evict: rows of cache tensor %d overlap", i);
    m.base[i] = static_cast<uint8_t*>(base[i]);
    m.s_p[i] = page_stride[i]; m.s_o[i] = token_stride[i]; m.s_h[i] = head_stride[i];
  }
  const size_t need = specq_kv_evict_workspace_size(B, H_KV);
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
  if (PAGE > 1) {
    int bits = 0;  // ceil(log2(PAGE))
    while ((1ll << bits) < PAGE) ++bits;
    // ceil(2^k / PAGE), k = 30 + bits, is off by less than PAGE <= 2^bits in 2^k, so its products with t < 2^30 by less than one.
    const uint64_t magic = ((1ull << (30 + bits)) + PAGE - 1) / PAGE;
    m.page_magic = (uint32_t)(bits < 2 ? magic << (2 - bits) : magic);
    m.page_shift = bits < 2 ? 0 : bits - 2;
  }
  hipStream_t st = (hipStream_t)stream;
  if (int rc = launch(reinterpret_cast<const void*>(&evict_select_kernel), (int)progs, kEvThreads, 0, st, &p)) return rc;
  return launch(reinterpret_cast<const void*>(&evict_move_kernel), (int)(align_up(progs, 8) * m.units), kEvMove, 0, st, &m);
}
