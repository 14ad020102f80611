// Page tables of a paged K/V cache -- reserve, free, fork, compact, copy -- and their C ABI.
//
// State, all int32 on the device and changed in place: a block table [B, C] whose entries name pages
// (an id outside [0, P) is no page), and ref[P], how often the tables name each page; a page with
// ref <= 0 is free.  Pages are handed out lowest id first, to the entries that want one in the
// table's order, so every result is a function of its inputs alone: counts change by atomic adds and
// subtractions (whose order leaves no trace), everything else by one thread.
//
//   reserve  entries of row b's first ceil(lens[b] / PAGE) columns that name no page get a free one.
//   free     entries past row b's first ceil(keep[b] / PAGE) columns let go of their page.
//   fork     row b becomes a copy of row parent[b]: it shares the full pages; of the rows with one
//            parent the lowest keeps its partly filled last page, the others get a copy of it.
//   compact  the pages in use move below their own number: the i-th used page at or past it goes to
//            the i-th free page below it.
//
// Handing out is a scan of ref by one workgroup of 1024 threads, 16 counts a thread and step, that ends
// when enough free pages are found.  Bound by latency: a few dependent round trips of about a
// microsecond each; the page copies behind fork and compact are bound by HBM.
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kPagesThreads = 1024, kPagesWaves = kPagesThreads / kWave;
constexpr int kPagesPer = 16;  // counts a thread scans per step
constexpr int kPagesTensors = 64;
constexpr int kPagesChunk = 16384;  // bytes of a page one workgroup copies at a time

struct PagesParams {
  int32_t* tbl; int64_t s_bt; int B, C;
  int32_t* ref; int P;
  int32_t* lens; const int32_t* parent; int PAGE;
  int32_t* shortage;  // [1]: pages that could not be given
  int32_t* map;       // compact: [P] the page's id afterwards
  // Workspace: rows [B] counts then offsets, list [P] free page ids; fork: the new rows [B * C], the
  // copies' sources and destinations [B] each; compact: moves [P] each, and their number.
  int32_t* rows; int32_t* list; int32_t* table; int32_t* src; int32_t* dst; int32_t* n_moves;
};

struct PagesCopyParams {
  uint8_t* base[kPagesTensors];
  int64_t stride[kPagesTensors], bytes[kPagesTensors];  // bytes from page to page, and of a page
  int32_t first[kPagesTensors + 1];                     // chunks of the tensors before this one
  const int32_t* src; const int32_t* dst; const int32_t* n_dev;
  int n, P, tensors, vec;  // vec: bytes of one access, 16, 4 or 1
};

// Columns of a row that n tokens fill.
__device__ __forceinline__ int pages_of(int n, int page, int C) {
  return n <= 0 ? 0 : min((n - 1) / page + 1, C);
}
__device__ __forceinline__ bool is_page(int id, int P) { return (uint32_t)id < (uint32_t)P; }

// Exclusive prefix of x over the workgroup; `total` is the sum.
__device__ __forceinline__ int block_prefix(int x, int& total, int (&part)[kPagesWaves]) {
  int v = x;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int y = __shfl_up(v, o);
    if (lane_id() >= o) v += y;
  }
  __syncthreads();  // the last call's readers of part are done
  if (lane_id() == kWave - 1) part[wave_id()] = v;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPagesWaves; ++w) {
    const int y = part[w];
    before += w < wave_id() ? y : 0;
    all += y;
  }
  total = all;
  return before + v - x;
}

// The lowest `need` ids with ref <= 0, in order, to list; returns how many there are (at most need).
__device__ __forceinline__ int find_free(const int32_t* ref, int P, int need, int32_t* list, int (&part)[kPagesWaves]) {
  int found = 0;
  for (int base = 0; base < P && found < need; base += kPagesThreads * kPagesPer) {
    const int at = base + (int)threadIdx.x * kPagesPer;
    uint32_t free_bits = 0;
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i)
      if (at + i < P && ref[at + i] <= 0) free_bits |= 1u << i;
    int total;
    int rank = found + block_prefix(__popc(free_bits), total, part);
    for (; free_bits != 0 && rank < need; free_bits &= free_bits - 1) list[rank++] = at + __ffs(free_bits) - 1;
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

__global__ __launch_bounds__(kPagesThreads) void pages_reserve_kernel(PagesParams p) {
  __shared__ int part[kPagesWaves];
  const int lane = lane_id(), w = uniform(wave_id());
  // A wave counts the entries that want a page, row by row; then the rows' offsets.
  for (int b = w; b < p.B; b += kPagesWaves) {
    const int np = pages_of(p.lens[b], p.PAGE, p.C);
    int n = 0;
    for (int c0 = 0; c0 < np; c0 += kWave) {
      const int c = c0 + lane;
      const bool want = c < np && !is_page(p.tbl[b * p.s_bt + c], p.P);
      n += __popcll(__builtin_amdgcn_ballot_w64(want));
    }
    if (lane == 0) p.rows[b] = n;
  }
  __syncthreads();
  int need = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPagesThreads) {
    const int b = b0 + (int)threadIdx.x;
    const int n = b < p.B ? p.rows[b] : 0;
    int total;
    const int off = need + block_prefix(n, total, part);
    if (b < p.B) p.rows[b] = n > 0 ? off : -1;
    need += total;
  }
  __syncthreads();
  const int found = find_free(p.ref, p.P, need, p.list, part);
  if (threadIdx.x == 0) *p.shortage = need - found;
  if (need == 0) return;
  for (int b = w; b < p.B; b += kPagesWaves) {
    int rank = p.rows[b];
    if (rank < 0) continue;
    const int np = pages_of(p.lens[b], p.PAGE, p.C);
    for (int c0 = 0; c0 < np; c0 += kWave) {
      const int c = c0 + lane;
      const bool want = c < np && !is_page(p.tbl[b * p.s_bt + c], p.P);
      const uint64_t m = __builtin_amdgcn_ballot_w64(want);
      if (want) {
        const int r = rank + __popcll(m & ((1ull << lane) - 1));
        const int id = r < found ? p.list[r] : -1;
        p.tbl[b * p.s_bt + c] = id;
        if (id >= 0) p.ref[id] = 1;
      }
      rank += __popcll(m);
    }
  }
}

// Workgroup (row, 1024 columns).
__global__ __launch_bounds__(256) void pages_free_kernel(PagesParams p) {
  const int chunks = (p.C + 1023) / 1024, b = blockIdx.x / chunks, c0 = (blockIdx.x % chunks) * 1024;
  const int keep = pages_of(p.lens[b], p.PAGE, p.C);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 256 * i + (int)threadIdx.x;
    if (c >= p.C || c < keep) continue;
    int32_t* e = p.tbl + b * p.s_bt + c;
    const int id = *e;
    if (id == -1) continue;
    *e = -1;
    if (is_page(id, p.P)) atomicSub(p.ref + id, 1);
  }
}

// Fork, first pass, workgroup (row, 1024 columns): the new row into the workspace, the counts of the
// pages the row gains and loses, and the page its copy comes from (-1: none needed).
__global__ __launch_bounds__(256) void pages_fork_rows_kernel(PagesParams p) {
  const int chunks = (p.C + 1023) / 1024, b = blockIdx.x / chunks, c0 = (blockIdx.x % chunks) * 1024;
  const int par = p.parent[b];
  const bool has = (uint32_t)par < (uint32_t)p.B;
  const int n = has ? min(max(p.lens[par], 0), p.C * p.PAGE) : 0;
  const int full = n / p.PAGE;
  const bool part = n % p.PAGE != 0;
  int first = 1;  // whether no row before b has this parent
  for (int i = threadIdx.x; i < b; i += 256)
    if (p.parent[i] == par) first = 0;
  first = __syncthreads_and(first);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = c0 + 256 * i + (int)threadIdx.x;
    if (c >= p.C) continue;
    const int old = p.tbl[b * p.s_bt + c];
    int src = has && (c < full || (c == full && part)) ? p.tbl[par * p.s_bt + c] : -1;
    if (!is_page(src, p.P)) src = -1;
    const bool copy = c == full && part && !first;
    const int id = copy ? -1 : src;
    p.table[(int64_t)b * p.C + c] = id;
    if (c == full) p.src[b] = copy ? src : -1;
    if (id != old) {
      if (is_page(old, p.P)) atomicSub(p.ref + old, 1);
      if (id >= 0) atomicAdd(p.ref + id, 1);
    }
  }
  if (c0 == 0 && threadIdx.x == 0) {
    p.rows[b] = n;
    if (full >= p.C) p.src[b] = -1;
  }
}

// Second pass: workgroup 0 gives the copies their pages, the others write the rows back.
__global__ __launch_bounds__(kPagesThreads) void pages_fork_assign_kernel(PagesParams p) {
  if (blockIdx.x > 0) {
    const int64_t n = (int64_t)p.B * p.C;
    for (int64_t e = (int64_t)(blockIdx.x - 1) * kPagesThreads + threadIdx.x; e < n;
         e += (int64_t)(gridDim.x - 1) * kPagesThreads) {
      const int b = (int)(e / p.C), c = (int)(e - (int64_t)b * p.C);
      const int len = p.rows[b];
      if (c == 0) p.lens[b] = len;
      if (p.src[b] < 0 || c != len / p.PAGE) p.tbl[b * p.s_bt + c] = p.table[e];
    }
    return;
  }
  __shared__ int part[kPagesWaves];
  int need = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPagesThreads) {
    const int b = b0 + (int)threadIdx.x;
    int total;
    const bool want = b < p.B && p.src[b] >= 0;
    const int r = need + block_prefix(want, total, part);
    if (b < p.B) p.dst[b] = want ? r : -1;
    need += total;
  }
  __syncthreads();
  const int found = find_free(p.ref, p.P, need, p.list, part);
  if (threadIdx.x == 0) *p.shortage = need - found;
  for (int b = threadIdx.x; b < p.B; b += kPagesThreads) {
    const int r = p.dst[b];
    if (r < 0) continue;
    const int id = r < found ? p.list[r] : -1;
    p.tbl[b * p.s_bt + p.rows[b] / p.PAGE] = id;
    p.dst[b] = id;
    if (id >= 0) p.ref[id] = 1;
  }
}

// Compact, the plan: the moves in order, every page's id afterwards, and the counts as they will be.
__global__ __launch_bounds__(kPagesThreads) void pages_compact_kernel(PagesParams p) {
  __shared__ int part[kPagesWaves];
  int used = 0;
  for (int base = 0; base < p.P; base += kPagesThreads * kPagesPer) {
    const int at = base + (int)threadIdx.x * kPagesPer;
    int n = 0, total;
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i) n += at + i < p.P && p.ref[at + i] > 0;
    block_prefix(n, total, part);
    used += total;
  }
  const int moves = find_free(p.ref, used, used, p.dst, part);  // the free pages below `used`
  int done = 0;
  for (int base = 0; base < p.P; base += kPagesThreads * kPagesPer) {
    const int at = base + (int)threadIdx.x * kPagesPer;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i)
      if (at + i < p.P && at + i >= used && p.ref[at + i] > 0) bits |= 1u << i;
    int total;
    int rank = done + block_prefix(__popc(bits), total, part);
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i) {
      if (at + i >= p.P) continue;
      int to = at + i;
      if ((bits >> i) & 1) {
        to = p.dst[rank];
        p.src[rank++] = at + i;
        p.ref[to] = p.ref[at + i];
        p.ref[at + i] = 0;
      }
      p.map[at + i] = to;
    }
    done += total;
  }
  if (threadIdx.x == 0) *p.n_moves = moves;
}

// The table under the new ids.
__global__ __launch_bounds__(256) void pages_remap_kernel(PagesParams p) {
  const int64_t n = (int64_t)p.B * p.C;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
    const int b = (int)(e / p.C);
    int32_t* at = p.tbl + b * p.s_bt + (e - (int64_t)b * p.C);
    const int id = *at;
    if (!is_page(id, p.P)) continue;
    const int to = p.map[id];
    if (to != id) *at = to;
  }
}

template <typename T>
__device__ __forceinline__ void copy_chunk(const uint8_t* src, uint8_t* dst, int bytes) {
  const T* s = reinterpret_cast<const T*>(src);
  T* d = reinterpret_cast<T*>(dst);
  const int n = bytes / (int)sizeof(T);
  constexpr int U = 4;
  int i = threadIdx.x;
  for (; i + 256 * (U - 1) < n; i += 256 * U) {
    T x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = s[i + 256 * u];
#pragma unroll
    for (int u = 0; u < U; ++u) d[i + 256 * u] = x[u];
  }
  for (; i < n; i += 256) d[i] = s[i];
}

// Pages src[i] -> dst[i] of every tensor; a pair with an id outside the pool is left out.
__global__ __launch_bounds__(256) void pages_copy_kernel(PagesCopyParams p) {
  const int pairs = p.n_dev != nullptr ? min(uniform(*p.n_dev), p.n) : p.n;
  const int per = p.first[p.tensors];
  for (int64_t u = blockIdx.x; u < (int64_t)pairs * per; u += gridDim.x) {
    const int pair = (int)(u / per), k = (int)(u - (int64_t)pair * per);
    const int from = uniform(p.src[pair]), to = uniform(p.dst[pair]);
    if (!is_page(from, p.P) || !is_page(to, p.P) || from == to) continue;
    int i = 0;
    while (k >= p.first[i + 1]) ++i;
    const int64_t off = (int64_t)(k - p.first[i]) * kPagesChunk;
    const uint8_t* s = p.base[i] + from * p.stride[i] + off;
    uint8_t* d = p.base[i] + to * p.stride[i] + off;
    const int64_t left = p.bytes[i] - off;
    const int bytes = left < kPagesChunk ? (int)left : kPagesChunk;
    if (p.vec == 16) copy_chunk<v4i>(s, d, bytes);
    else if (p.vec == 4) copy_chunk<int>(s, d, bytes);
    else copy_chunk<uint8_t>(s, d, bytes);
  }
}

static size_t pages_ints(int B, int C, int P) { return (size_t)B * C + 3 * (size_t)B + 3 * (size_t)P + 16; }

static int pages_setup(PagesParams& p, const char* who, int32_t* tbl, int64_t s_bt, int B, int C, int32_t* ref, int P,
                       int PAGE) {
  SPECQ_REQUIRE(tbl && ref, SPECQ_EINVAL, "%s: null tensor pointer", who);
  SPECQ_REQUIRE(B > 0 && C > 0 && P > 0 && PAGE > 0 && s_bt >= C, SPECQ_EINVAL,
                "%s: bad sizes B=%d columns=%d pages=%d PAGE=%d", who, B, C, P, PAGE);
  SPECQ_REQUIRE((int64_t)C * PAGE <= INT32_MAX && P <= INT32_MAX - kPagesThreads * kPagesPer, SPECQ_ENOTSUP,
                "%s: a row of %lld tokens or a pool of %d pages is too large", who, (long long)C * PAGE, P);
  SPECQ_REQUIRE((int64_t)B * ceil_div(C, 1024) <= INT32_MAX, SPECQ_ENOTSUP, "%s: block table too large", who);
  p = {};
  p.tbl = tbl; p.s_bt = s_bt; p.B = B; p.C = C; p.ref = ref; p.P = P; p.PAGE = PAGE;
  return SPECQ_OK;
}

static int pages_scratch(PagesParams& p, const char* who, void* workspace, size_t bytes) {
  const size_t need = kCounterBytes + align_up(pages_ints(p.B, p.C, p.P) * 4, 256);
  SPECQ_REQUIRE(workspace && bytes >= need, SPECQ_ENOSPC, "%s: workspace of %zu bytes required, %zu given", who, need,
                workspace ? bytes : (size_t)0);
  int32_t* at = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + kCounterBytes);
  p.n_moves = at;
  p.rows = at + 16;
  p.list = p.rows + p.B;
  p.src = p.list + p.P;
  p.dst = p.src + (p.B > p.P ? p.B : p.P);
  p.table = p.dst + (p.B > p.P ? p.B : p.P);
  return SPECQ_OK;
}

// Page tensors of a copy.
static int pages_tensors(const char* who, int n, void* const* base, const int64_t* stride, const int64_t* bytes) {
  SPECQ_REQUIRE(n >= 0 && (n == 0 || (base && stride && bytes)), SPECQ_EINVAL, "%s: bad tensor list", who);
  for (int i = 0; i < n; ++i)
    SPECQ_REQUIRE(base[i] && bytes[i] > 0 && stride[i] >= bytes[i] && ceil_div64(bytes[i], kPagesChunk) < (1 << 20),
                  SPECQ_EINVAL, "%s: page tensor %d is null, empty or overlaps its own pages", who, i);
  return SPECQ_OK;
}

static int pages_copy(int n_tensors, void* const* base, const int64_t* stride, const int64_t* bytes, const int32_t* src,
                      const int32_t* dst, int n, const int32_t* n_dev, int P, hipStream_t stream) {
  for (int t0 = 0; t0 < n_tensors; t0 += kPagesTensors) {
    PagesCopyParams c = {};
    c.tensors = n_tensors - t0 < kPagesTensors ? n_tensors - t0 : kPagesTensors;
    uint64_t bits = 0;
    for (int i = 0; i < c.tensors; ++i) {
      c.base[i] = static_cast<uint8_t*>(base[t0 + i]);
      c.stride[i] = stride[t0 + i];
      c.bytes[i] = bytes[t0 + i];
      c.first[i + 1] = c.first[i] + (int)ceil_div64(bytes[t0 + i], kPagesChunk);
      bits |= (uintptr_t)base[t0 + i] | (uint64_t)stride[t0 + i] | (uint64_t)bytes[t0 + i];
    }
    c.vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    c.src = src; c.dst = dst; c.n_dev = n_dev; c.n = n; c.P = P;
    // Eight workgroups of 256 threads to a CU, each walking its chunks.
    const int64_t units = (int64_t)n * c.first[c.tensors], most = 8ll * device_cus();
    const int rc = launch(reinterpret_cast<const void*>(&pages_copy_kernel), (int)(units < most ? units : most), 256, 0,
                          stream, &c);
    if (rc != SPECQ_OK) return rc;
  }
  return SPECQ_OK;
}

}  // namespace specq

using namespace specq;

extern "C" size_t specq_kv_pages_workspace_size(int B, int C, int P) {
  if (B <= 0 || C <= 0 || P <= 0) return 0;
  return kCounterBytes + align_up(pages_ints(B, C, P) * 4, 256);
}

extern "C" int specq_kv_pages_reserve(int32_t* block_tbl, int64_t s_bt, int B, int max_pages, int32_t* ref, int n_pages,
                                      const int32_t* lens, int PAGE, int32_t* shortage, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  clear_error();
  PagesParams p;
  if (int rc = pages_setup(p, "kv_pages_reserve", block_tbl, s_bt, B, max_pages, ref, n_pages, PAGE)) return rc;
  SPECQ_REQUIRE(lens && shortage, SPECQ_EINVAL, "kv_pages_reserve: null tensor pointer");
  if (int rc = pages_scratch(p, "kv_pages_reserve", workspace, workspace_bytes)) return rc;
  p.lens = const_cast<int32_t*>(lens);
  p.shortage = shortage;
  return launch(reinterpret_cast<const void*>(&pages_reserve_kernel), 1, kPagesThreads, 0, (hipStream_t)stream, &p);
}

extern "C" int specq_kv_pages_free(int32_t* block_tbl, int64_t s_bt, int B, int max_pages, int32_t* ref, int n_pages,
                                   const int32_t* keep, int PAGE, void* stream) {
  clear_error();
  PagesParams p;
  if (int rc = pages_setup(p, "kv_pages_free", block_tbl, s_bt, B, max_pages, ref, n_pages, PAGE)) return rc;
  SPECQ_REQUIRE(keep, SPECQ_EINVAL, "kv_pages_free: null tensor pointer");
  p.lens = const_cast<int32_t*>(keep);
  return launch(reinterpret_cast<const void*>(&pages_free_kernel), B * ceil_div(max_pages, 1024), 256, 0,
                (hipStream_t)stream, &p);
}

extern "C" int specq_kv_pages_fork(int32_t* block_tbl, int64_t s_bt, int B, int max_pages, int32_t* ref, int n_pages,
                                   int32_t* lens, const int32_t* parent, int PAGE, int n_tensors, void* const* base,
                                   const int64_t* page_stride, const int64_t* page_bytes, int32_t* shortage,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  PagesParams p;
  if (int rc = pages_setup(p, "kv_pages_fork", block_tbl, s_bt, B, max_pages, ref, n_pages, PAGE)) return rc;
  SPECQ_REQUIRE(lens && parent && shortage, SPECQ_EINVAL, "kv_pages_fork: null tensor pointer");
  if (int rc = pages_tensors("kv_pages_fork", n_tensors, base, page_stride, page_bytes)) return rc;
  if (int rc = pages_scratch(p, "kv_pages_fork", workspace, workspace_bytes)) return rc;
  p.lens = lens; p.parent = parent; p.shortage = shortage;
  hipStream_t st = (hipStream_t)stream;
  const int chunks = B * ceil_div(max_pages, 1024);
  if (int rc = launch(reinterpret_cast<const void*>(&pages_fork_rows_kernel), chunks, 256, 0, st, &p)) return rc;
  const int64_t back = ceil_div64((int64_t)B * max_pages, kPagesThreads);
  if (int rc = launch(reinterpret_cast<const void*>(&pages_fork_assign_kernel), 1 + (int)(back < 512 ? back : 512),
                      kPagesThreads, 0, st, &p))
    return rc;
  return pages_copy(n_tensors, base, page_stride, page_bytes, p.src, p.dst, B, nullptr, n_pages, st);
}

extern "C" int specq_kv_pages_compact(int32_t* block_tbl, int64_t s_bt, int B, int max_pages, int32_t* ref, int n_pages,
                                      int32_t* page_map, int n_tensors, void* const* base, const int64_t* page_stride,
                                      const int64_t* page_bytes, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  clear_error();
  PagesParams p;
  if (int rc = pages_setup(p, "kv_pages_compact", block_tbl, s_bt, B, max_pages, ref, n_pages, 1)) return rc;
  SPECQ_REQUIRE(page_map, SPECQ_EINVAL, "kv_pages_compact: null tensor pointer");
  if (int rc = pages_tensors("kv_pages_compact", n_tensors, base, page_stride, page_bytes)) return rc;
  if (int rc = pages_scratch(p, "kv_pages_compact", workspace, workspace_bytes)) return rc;
  p.map = page_map;
  hipStream_t st = (hipStream_t)stream;
  if (int rc = launch(reinterpret_cast<const void*>(&pages_compact_kernel), 1, kPagesThreads, 0, st, &p)) return rc;
  const int64_t wgs = ceil_div64((int64_t)B * max_pages, 1024);
  if (int rc = launch(reinterpret_cast<const void*>(&pages_remap_kernel), (int)(wgs < 2048 ? wgs : 2048), 256, 0, st, &p))
    return rc;
  return pages_copy(n_tensors, base, page_stride, page_bytes, p.src, p.dst, n_pages, p.n_moves, n_pages, st);
}

extern "C" int specq_kv_pages_copy(const int32_t* src, const int32_t* dst, int n, int n_pages, int n_tensors,
                                   void* const* base, const int64_t* page_stride, const int64_t* page_bytes,
                                   void* stream) {
  clear_error();
  SPECQ_REQUIRE(n >= 0 && n_pages > 0 && (n == 0 || (src && dst)), SPECQ_EINVAL, "kv_pages_copy: bad sizes or pointers");
  if (int rc = pages_tensors("kv_pages_copy", n_tensors, base, page_stride, page_bytes)) return rc;
  if (n == 0) return SPECQ_OK;
  return pages_copy(n_tensors, base, page_stride, page_bytes, src, dst, n, nullptr, n_pages, (hipStream_t)stream);
}
