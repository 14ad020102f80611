// Eviction from a paged K/V cache by gathered attention weight, and its C ABI.
//
// A sequence b of L = ctx_len[b] > limit tokens is cut back to `budget`: for each KV head h stay its first `sinks` tokens,
// its last `recent` ones, and of the others those of greatest weights[b, h, t], ties to the lower position.  What stays
// keeps its order and moves together: token j of the `budget` comes from position kept[b, h, j], in every cache tensor
// and in the weights.  ctx_len[b] becomes budget.  A sequence whose table names a page outside the pool, or, with page
// counts given, a page that other rows name too, stays as it is.
//
// Selection, one workgroup a (sequence, head): the weights as unsigned keys of the same order (tokens that stay in any
// case have the largest key), the budget-th largest found by three passes of counting digits of 11, 11 and 10 bits from
// the top, then one pass in the order of the positions that ranks what is above it and the first of what equals it.  Keys
// of the first kEvKeys * 1024 tokens stay in registers, further ones are read again from L2.
//
// Moving is in place.  Token j goes to a place at or below its own, and everything behind it starts above, so it is
// enough that a tile of tokens has been read by all its threads before any of them writes it.  One workgroup walks one
// byte range of the rows of one (sequence, head) of one tensor; ranges are independent, so narrow ranges make more
// workgroups where there are few sequences and heads.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / kWave;
constexpr int kEvBins = 2048;
constexpr int kEvKeys = 8;      // keys of a thread in registers: positions 4 (tid + 1024 c) + 0..3, c < 2
constexpr int kEvTensors = 16;  // cache tensors of a call
constexpr int kEvUnits = 256;   // byte ranges of a call
constexpr int kEvPages = 8192;  // table entries kept in LDS
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
  int units;
};

// Exclusive prefix of x over the workgroup; `total` is the sum.
__device__ __forceinline__ int ev_prefix(int x, int& total, int (&part)[kEvWaves]) {
  int v = x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
  __syncthreads();  // the last call's readers of part are done
  if (lane_id() == kWave - 1) part[wave_id()] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kEvWaves; ++w) {
    const int y = part[w];
    before += w < wave_id() ? y : 0;
    all += y;
  }
  total = all;
  return before + v - x;
}

// A key of the order of the weights; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t ev_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.f);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kEvThreads) void evict_select_kernel(EvictParams p) {
  __shared__ int hist[kEvBins], part[kEvWaves], s_bin, s_above;
  const int prog = blockIdx.x, b = prog / p.H, h = prog - b * p.H, tid = threadIdx.x;
  const int L = min(max(p.ctx_len[b], 0), p.cap);
  int32_t* kept = p.kept + (int64_t)prog * p.budget;
  int ok = L > p.limit;
  if (ok) {
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
  const float* wr = p.w + b * p.s_wb + h * p.s_wh;
  auto load = [&](int t, uint32_t (&k)[4]) {  // keys of positions t..t+3, 0 past the context
    v4f x = {0.f, 0.f, 0.f, 0.f};
    if (p.w_vec && t + 4 <= L) {
      x = *reinterpret_cast<const v4f*>(wr + t);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < L) x[i] = wr[t + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = t + i;
      k[i] = at >= L ? 0u : (at < p.sinks || at >= L - p.recent) ? 0xFFFFFFFFu : ev_key(x[i]);
    }
  };
  constexpr int kStep = 4 * kEvThreads;
  uint32_t near[kEvKeys / 4][4];
#pragma unroll
  for (int c = 0; c < kEvKeys / 4; ++c) load(c * kStep + 4 * tid, near[c]);
  const int chunks = (L + kStep - 1) / kStep;
  auto each = [&](auto&& f) {  // f(first position, keys), a chunk of 4096 positions at a time
#pragma unroll
    for (int c = 0; c < kEvKeys / 4; ++c)
      if (c < chunks) f(c * kStep + 4 * tid, near[c]);
    for (int c = kEvKeys / 4; c < chunks; ++c) {
      uint32_t k[4];
      load(c * kStep + 4 * tid, k);
      f(c * kStep + 4 * tid, k);
    }
  };
  // The budget-th largest key, from its top digit down: `want` of those under the digits found so far.
  uint32_t found = 0;
  int want = p.budget;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass < 2 ? 11 : 10, bins = 1 << bits;
    hist[2 * tid] = hist[2 * tid + 1] = 0;
    __syncthreads();
    each([&](int t, const uint32_t (&k)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < L && (pass == 0 || (k[i] >> (low + bits)) == (found >> (low + bits))))
          atomicAdd(&hist[(k[i] >> low) & (bins - 1)], 1);
    });
    __syncthreads();
    // Thread i has bins 2047 - 2 i and 2046 - 2 i: the prefix runs from the largest digit down.
    const int hi = kEvBins - 1 - 2 * tid, n1 = hist[hi], n0 = hist[hi - 1];
    int total;
    const int above = ev_prefix(n1 + n0, total, part);
    if (above < want && above + n1 + n0 >= want) {
      const bool first = above + n1 >= want;
      s_bin = first ? hi : hi - 1;
      s_above = first ? above : above + n1;
    }
    __syncthreads();
    found |= (uint32_t)s_bin << low;
    want -= s_above;
    __syncthreads();
  }
  // `want` keys equal to `found` stay, the lowest positions; everything larger stays.
  int above = 0, equal = 0;
  each([&](int t, const uint32_t (&k)[4]) {
    int gt[4], eq[4], n = 0;  // counts of a chunk fit 16 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      gt[i] = t + i < L && k[i] > found;
      eq[i] = t + i < L && k[i] == found;
      n += gt[i] + (eq[i] << 16);
    }
    int total;
    const int before = ev_prefix(n, total, part);
    int a = above + (before & 0xFFFF), e = equal + (before >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (gt[i] || (eq[i] && e < want)) kept[a + min(e, want)] = t + i;
      a += gt[i];
      e += eq[i];
    }
    above += total & 0xFFFF;
    equal += total >> 16;
  });
}

// One byte range of one (sequence, head): accesses of sizeof(T) bytes, `lanes` of them a token.
template <typename T, typename F>
__device__ __forceinline__ void evict_walk(const int32_t* kept, int budget, int lanes, F&& place) {
  const int per = kEvThreads / lanes, sub = (int)threadIdx.x % lanes, mine = (int)threadIdx.x / lanes;
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

__global__ __launch_bounds__(kEvThreads) void evict_move_kernel(EvictMoveParams p) {
  __shared__ int32_t pages[kEvPages];
  const EvictParams& e = p.e;
  const int u = (int)blockIdx.x % p.units, prog = (int)blockIdx.x / p.units, b = prog / e.H, h = prog - b * e.H;
  if (!uniform(e.flag[prog])) return;
  const int32_t* kept = e.kept + (int64_t)prog * e.budget;
  const int tensor = p.tensor[u], vec = p.vec[u], lanes = p.bytes[u] / vec;
  if (tensor == kEvTensors) {
    if (h == 0 && threadIdx.x == 0) e.ctx_len[b] = e.budget;  // the selection is over, and this launch does not read it
    float* w = e.w + b * e.s_wb + h * e.s_wh;
    evict_walk<float>(kept, e.budget, 1, [&](int t) { return reinterpret_cast<uint8_t*>(w + t); });
    return;
  }
  const int32_t* row = e.bt + b * e.s_bt;
  const int last = uniform(kept[e.budget - 1]) / e.PAGE;  // the highest page that is read or written
  const bool near = last < kEvPages;
  if (near)
    for (int c = threadIdx.x; c <= last; c += kEvThreads) pages[c] = row[c];
  __syncthreads();
  uint8_t* base = p.base[tensor] + h * p.s_h[tensor] + p.first[u];
  const int64_t s_p = p.s_p[tensor], s_o = p.s_o[tensor];
  auto place = [&](int t) {
    const int c = t / e.PAGE;
    return base + (near ? pages[c] : row[c]) * s_p + (t - c * e.PAGE) * s_o;
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
  // Byte ranges: rows whole, or in pieces of at least 16 bytes until there is a workgroup or two for every CU.
  const int64_t cus = device_cus();
  int64_t piece = 128;
  auto ranges = [&](int64_t size) {
    int64_t n = 1;
    for (int i = 0; i < n_tensors; ++i) n += ceil_div64(row_bytes[i], size);
    return n;
  };
  while (piece > 16 && progs * ranges(piece) < 2 * cus) piece /= 2;
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
  hipStream_t st = (hipStream_t)stream;
  if (int rc = launch(reinterpret_cast<const void*>(&evict_select_kernel), (int)progs, kEvThreads, 0, st, &p)) return rc;
  return launch(reinterpret_cast<const void*>(&evict_move_kernel), (int)(progs * m.units), kEvThreads, 0, st, &m);
}
