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
// Handing out is a scan of ref by one workgroup of 1024 threads, eight counts a thread and step, that ends
// when enough free pages are found.  Bound by latency, a few dependent round trips of about a
// microsecond each, so the first step's counts are loaded ahead of everything else and what one part
// hands the next stays in LDS where it fits (the table's bits up to kPagesBits words, ids up to kPagesList;
// the workspace otherwise).  The page copies behind fork and compact are bound by HBM.  Kernel times:
// reserve 6.8 us (32 rows of 258 columns, one page each), free 2.5, fork 3.6 + 3.8 and 4.3 for the copies of 24
// pages of 128 KB, compact 6.0 (4104 pages) and 13.1 for the copies of a thousand pages of 32 KB (4.9 TB/s).
#include "api_common.hpp"
#include "common.hpp"

namespace specq {

constexpr int kPagesThreads = 1024, kPagesWaves = kPagesThreads / kWave;
// Counts a thread scans per step.  Compacting 512, 4104, 65536, 262144 pages, 70 % used, took (with the launch and
// no copies) 15.5, 18.1, 66, 237 us with 16, 13.9, 15.7, 57, 195 with 8 and 15.0, 17.1, 63, 217 with 4.
constexpr int kPagesPer = 8;
constexpr int kPagesTensors = 64;
constexpr int kPagesChunk = 16384;  // bytes of a page one workgroup copies at a time
constexpr int kPagesStep = kPagesThreads * kPagesPer;
constexpr int kPagesList = 8192;  // page ids kept in LDS
constexpr int kPagesBits = 4096;  // words of 64 table entries kept in LDS
constexpr int kPagesRows = 4096;  // rows whose lengths are kept in LDS

struct PagesParams {
  int32_t* tbl; int64_t s_bt; int B, C;
  int32_t* ref; int P;
  int32_t* lens; const int32_t* parent; int PAGE;
  int32_t* shortage;  // [1]: pages that could not be given
  int32_t* map;       // compact: [P] the page's id afterwards
  // Workspace: list [P] free page ids; reserve: a bit for each entry [B][ceil(C / 64)] and
  // (in table) each word's place; fork: the new rows
  // [B * C] and their lengths [B], the copies' sources and destinations [B] each; compact: moves [P] each, and
  // their number.
  uint64_t* bits; int32_t* rows; int32_t* list; int32_t* table; int32_t* src; int32_t* dst; int32_t* n_moves;
};

struct PagesCopyParams {
  uint8_t* base[kPagesTensors];
  int64_t stride[kPagesTensors], bytes[kPagesTensors];  // bytes from page to page, and of a page
  int32_t first[kPagesTensors + 1];                     // chunks of the tensors before this one
  const int32_t* src; const int32_t* dst; const int32_t* n_dev;
  int n, P, tensors, vec;  // vec: bytes of one access, 16, 4 or 1
  int large;               // tensors whose pages are cut into chunks; the others go with a page's first chunk
  // compact: the workgroups ahead of the copies' put the table under the new ids.
  int remap; int32_t* tbl; int64_t s_bt; int B, C; const int32_t* map;
};

// Columns of a row that n tokens fill.
__device__ __forceinline__ int pages_of(int n, int page, int C) {
  return n <= 0 ? 0 : min((n - 1) / page + 1, C);
}
__device__ __forceinline__ bool is_page(int id, int P) { return (uint32_t)id < (uint32_t)P; }

// Exclusive prefix of x over the workgroup; `total` is the sum.
__device__ __forceinline__ int block_prefix(int x, int& total, int (&part)[kPagesWaves]) {
  // Inclusive sums over the wave: within rows of 16 lanes, then the row before, then the two before.
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
  for (int w = 0; w < kPagesWaves; ++w) {
    const int y = part[w];
    before += w < wave_id() ? y : 0;
    all += y;
  }
  total = all;
  return before + v - x;
}

// The thread's kPagesPer counts from page `base` on; pages past the pool count as `past`.
struct PageCounts {
  v4i x[kPagesPer / 4];
  __device__ __forceinline__ uint32_t used() const {
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i) bits |= (uint32_t)(x[i / 4][i % 4] > 0) << i;
    return bits;
  }
};
__device__ __forceinline__ PageCounts load_counts(const int32_t* ref, int P, int base, int past) {
  const int at = base + (int)threadIdx.x * kPagesPer;
  PageCounts c;
  if (at + kPagesPer <= P && ((uintptr_t)ref & 15) == 0) {
#pragma unroll
    for (int i = 0; i < kPagesPer / 4; ++i) c.x[i] = reinterpret_cast<const v4i*>(ref + at)[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i) c.x[i / 4][i % 4] = at + i < P ? ref[at + i] : past;
  }
  return c;
}

// Page ids in order: the first kPagesList in LDS, the rest in the workspace.
struct PageList {
  int* near;
  int32_t* far;
  __device__ __forceinline__ void put(int i, int id) const {
    if (i < kPagesList) near[i] = id;
    else far[i] = id;
  }
  __device__ __forceinline__ int get(int i) const { return i < kPagesList ? near[i] : far[i]; }
};

// The lowest `need` free ids, in order, to list; returns how many there are (at most need).  `first`: the
// first step's used().
__device__ __forceinline__ int find_free(const int32_t* ref, int P, int need, uint32_t first, const PageList& list,
                                         int (&part)[kPagesWaves]) {
  int found = 0;
  for (int base = 0; base < P && found < need; base += kPagesStep) {
    uint32_t free_bits = ~(base == 0 ? first : load_counts(ref, P, base, 1).used()) & ((1u << kPagesPer) - 1);
    int total;
    int rank = found + block_prefix(__popc(free_bits), total, part);
    for (; free_bits != 0 && rank < need; free_bits &= free_bits - 1)
      list.put(rank++, base + (int)threadIdx.x * kPagesPer + __ffs(free_bits) - 1);
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

__global__ __launch_bounds__(kPagesThreads) void pages_reserve_kernel(PagesParams p) {
  __shared__ int part[kPagesWaves], near_list[kPagesList];
  __shared__ uint64_t near_bits[kPagesBits];
  __shared__ int near_at[kPagesBits];
  __shared__ int cols[kPagesRows];
  const int lane = lane_id(), w = uniform(wave_id());
  const PageCounts first = load_counts(p.ref, p.P, 0, 1);
  for (int b = threadIdx.x; b < min(p.B, kPagesRows); b += kPagesThreads) cols[b] = pages_of(p.lens[b], p.PAGE, p.C);
  __syncthreads();
  // A word for each 64 entries of a row, with the bits of those that want a page.  Of each 1024 words a wave has
  // one of every 16; which of them turns with their number, so that words a fixed step apart -- rows that
  // grow by a page each -- fall to different waves.  A wave looks at its 64 words at once, a lane to a word,
  // and then reads the entries of those that count, eight words in flight: tables are as wide as the longest
  // row may become (32 rows of 4096 columns, a page each, with the launch: 84 us when every entry was read).
  const int words = (p.C + kWave - 1) / kWave, units = p.B * words;
  uint64_t* bits = units <= kPagesBits ? near_bits : p.bits;
  int* at = units <= kPagesBits ? near_at : p.table;
  auto word = [&](int u0, int l) { return u0 + kPagesWaves * l + ((w + l + l / 4 + l / 16) & (kPagesWaves - 1)); };
  constexpr int U = 8;
  for (int u0 = 0; u0 < units; u0 += kPagesThreads) {
    const int mine = word(u0, lane), row = min(mine, units - 1) / words, k = mine - row * words;
    int count = 0;  // columns of the word that count
    if (mine < units) {
      count = (row < kPagesRows ? cols[row] : pages_of(p.lens[row], p.PAGE, p.C)) - k * kWave;
      if (count <= 0) bits[mine] = 0;
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(count > 0);
    while (todo != 0) {
      int id[U], l[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        l[i] = todo != 0 ? __ffsll((unsigned long long)todo) - 1 : -1;
        todo &= todo - 1;  // stays 0
        if (l[i] < 0) continue;
        const int c = __builtin_amdgcn_readlane(k, l[i]) * kWave + lane;
        id[i] = p.tbl[__builtin_amdgcn_readlane(row, l[i]) * p.s_bt + min(c, p.C - 1)];
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (l[i] < 0) continue;
        const uint64_t m = __builtin_amdgcn_ballot_w64(lane < __builtin_amdgcn_readlane(count, l[i]) && !is_page(id[i], p.P));
        if (lane == 0) bits[word(u0, l[i])] = m;
      }
    }
  }
  __syncthreads();
  // Each word's place among the wants, four words to a thread.
  constexpr int WPT = 4;
  int need = 0;
  for (int base = 0; base < units; base += kPagesThreads * WPT) {
    int n[WPT], all = 0, total;
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
      const int u = base + (int)threadIdx.x * WPT + i;
      n[i] = u < units ? __popcll(bits[u]) : 0;
      all += n[i];
    }
    int rank = need + block_prefix(all, total, part);
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
      const int u = base + (int)threadIdx.x * WPT + i;
      if (u < units) at[u] = rank;
      rank += n[i];
    }
    need += total;
  }
  const PageList list = {near_list, p.list};
  const int found = find_free(p.ref, p.P, need, first.used(), list, part);
  if (threadIdx.x == 0) *p.shortage = need - found;
  if (need == 0) return;
  // A wave hands out its words' wants, a lane to an entry.
  for (int u0 = 0; u0 < units; u0 += kPagesThreads) {
    const int mine = word(u0, lane);
    uint64_t todo = __builtin_amdgcn_ballot_w64(mine < units && bits[min(mine, units - 1)] != 0);
    for (; todo != 0; todo &= todo - 1) {
      const int u = uniform(word(u0, __ffsll((unsigned long long)todo) - 1)), b = u / words;
      const uint64_t m = bits[u];
      if (((m >> lane) & 1) == 0) continue;
      const int rank = at[u] + __popcll(m & ((1ull << lane) - 1));
      const int id = rank < found ? list.get(rank) : -1;
      p.tbl[b * p.s_bt + (u - b * words) * kWave + lane] = id;
      if (id >= 0) p.ref[id] = 1;
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
  __shared__ int part[kPagesWaves], near_list[kPagesList];
  const PageCounts first = load_counts(p.ref, p.P, 0, 1);
  int need = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPagesThreads) {
    const int b = b0 + (int)threadIdx.x;
    int total;
    const bool want = b < p.B && p.src[b] >= 0;
    const int r = need + block_prefix(want, total, part);
    if (b < p.B) p.dst[b] = want ? r : -1;
    need += total;
  }
  const PageList list = {near_list, p.list};
  const int found = find_free(p.ref, p.P, need, first.used(), list, part);
  if (threadIdx.x == 0) *p.shortage = need - found;
  for (int b = threadIdx.x; b < p.B; b += kPagesThreads) {  // the rows this thread ranked
    const int r = p.dst[b];
    if (r < 0) continue;
    const int id = r < found ? list.get(r) : -1;
    p.tbl[b * p.s_bt + p.rows[b] / p.PAGE] = id;
    p.dst[b] = id;
    if (id >= 0) p.ref[id] = 1;
  }
}

// Compact, the plan: the moves in order, every page's id afterwards, and the counts as they will be.
__global__ __launch_bounds__(kPagesThreads) void pages_compact_kernel(PagesParams p) {
  __shared__ int part[kPagesWaves], near_list[kPagesList];
  const PageCounts first = load_counts(p.ref, p.P, 0, 0);
  auto counts = [&](int base) { return base == 0 ? first : load_counts(p.ref, p.P, base, 0); };
  int used = 0;
  for (int base = 0; base < p.P; base += kPagesStep) {
    int total;
    block_prefix(__popc(counts(base).used()), total, part);
    used += total;
  }
  // The free pages below `used`, as many as there are used ones past it.
  const PageList holes = {near_list, p.list};
  int found = 0;
  for (int base = 0; base < used; base += kPagesStep) {
    const int at = base + (int)threadIdx.x * kPagesPer, below = min(max(used - at, 0), kPagesPer);
    uint32_t bits = ~counts(base).used() & ((1u << below) - 1);
    int total;
    int rank = found + block_prefix(__popc(bits), total, part);
    for (; bits != 0; bits &= bits - 1) holes.put(rank++, at + __ffs(bits) - 1);
    found += total;
  }
  __syncthreads();
  int done = 0;
  for (int base = 0; base < p.P; base += kPagesStep) {
    const int at = base + (int)threadIdx.x * kPagesPer, below = min(max(used - at, 0), kPagesPer);
    const PageCounts c = counts(base);
    const uint32_t bits = c.used() & ~((1u << below) - 1);
    int total;
    int rank = done + block_prefix(__popc(bits), total, part);
    v4i to[kPagesPer / 4];
#pragma unroll
    for (int i = 0; i < kPagesPer; ++i) {
      to[i / 4][i % 4] = at + i;
      if (((bits >> i) & 1) == 0) continue;
      const int hole = to[i / 4][i % 4] = holes.get(rank);
      p.src[rank] = at + i;
      p.dst[rank++] = hole;
      p.ref[hole] = c.x[i / 4][i % 4];
      p.ref[at + i] = 0;
    }
    if (at + kPagesPer <= p.P && ((uintptr_t)p.map & 15) == 0) {
#pragma unroll
      for (int i = 0; i < kPagesPer / 4; ++i) reinterpret_cast<v4i*>(p.map + at)[i] = to[i];
    } else {
#pragma unroll
      for (int i = 0; i < kPagesPer; ++i)
        if (at + i < p.P) p.map[at + i] = to[i / 4][i % 4];
    }
    done += total;
  }
  if (threadIdx.x == 0) *p.n_moves = found;
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

// Pages src[i] -> dst[i] of every tensor; a pair with an id outside the pool is left out.  A unit is a chunk of
// kPagesChunk bytes of a large tensor's page, four 16-byte loads a thread in flight; pages of at most a
// quarter of that (scales) would leave most of a unit idle, and are copied with their pair's first one.
// One access width for all tensors of a launch: next to scale pages of 4 or 8 bytes K and V go 4 bytes an access, which
// costs nothing measurable (2048 pairs, heads of 128, in a graph, against scale pages padded to 16 bytes: one head, pages
// of 16 tokens 7.8 and 7.7 us, of 64 tokens 12.9 and 12.8; two heads, 64 tokens 20.2 and 20.4).
__global__ __launch_bounds__(256) void pages_copy_kernel(PagesCopyParams p) {
  if ((int)blockIdx.x < p.remap) {
    const int64_t n = (int64_t)p.B * p.C;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)p.remap * 256) {
      const int b = (int)(e / p.C);
      int32_t* at = p.tbl + b * p.s_bt + (e - (int64_t)b * p.C);
      const int id = *at;
      if (!is_page(id, p.P)) continue;
      const int to = p.map[id];
      if (to != id) *at = to;
    }
    return;
  }
  const int pairs = p.n_dev != nullptr ? min(uniform(*p.n_dev), p.n) : p.n;
  const int per = max(p.first[p.large], 1);
  for (int64_t u = (int)blockIdx.x - p.remap; u < (int64_t)pairs * per; u += (int)gridDim.x - p.remap) {
    const int pair = (int)(u / per), k = (int)(u - (int64_t)pair * per);
    const int from = uniform(p.src[pair]), to = uniform(p.dst[pair]);
    if (!is_page(from, p.P) || !is_page(to, p.P) || from == to) continue;
    auto copy = [&](int i, int64_t off, int bytes) {
      const uint8_t* s = p.base[i] + from * p.stride[i] + off;
      uint8_t* d = p.base[i] + to * p.stride[i] + off;
      if (p.vec == 16) copy_chunk<v4i>(s, d, bytes);
      else if (p.vec == 4) copy_chunk<int>(s, d, bytes);
      else copy_chunk<uint8_t>(s, d, bytes);
    };
    if (k < p.first[p.large]) {
      int i = 0;
      while (k >= p.first[i + 1]) ++i;
      const int64_t off = (int64_t)(k - p.first[i]) * kPagesChunk, left = p.bytes[i] - off;
      copy(i, off, left < kPagesChunk ? (int)left : kPagesChunk);
    }
    if (k == 0)
      for (int i = p.large; i < p.tensors; ++i) copy(i, 0, (int)p.bytes[i]);
  }
}

static size_t pages_ints(int B, int C, int P) {
  return 2 * (size_t)B * ceil_div(C, 64) + (size_t)B * C + 3 * (size_t)B + 3 * (size_t)P + 16;
}

static int pages_setup(PagesParams& p, const char* who, int32_t* tbl, int64_t s_bt, int B, int C, int32_t* ref, int P,
                       int PAGE) {
  SPECQ_REQUIRE(tbl && ref, SPECQ_EINVAL, "%s: null tensor pointer", who);
  SPECQ_REQUIRE(B > 0 && C > 0 && P > 0 && PAGE > 0 && s_bt >= C, SPECQ_EINVAL,
                "%s: bad sizes B=%d columns=%d pages=%d PAGE=%d", who, B, C, P, PAGE);
  SPECQ_REQUIRE((int64_t)C * PAGE <= INT32_MAX && C <= (1 << 30) && P <= INT32_MAX - kPagesThreads * kPagesPer, SPECQ_ENOTSUP,
                "%s: a row of %lld tokens or a pool of %d pages is too large", who, (long long)C * PAGE, P);
  SPECQ_REQUIRE((int64_t)B * ceil_div(C, 64) <= INT32_MAX / 2, SPECQ_ENOTSUP, "%s: block table too large", who);
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
  p.bits = reinterpret_cast<uint64_t*>(at + 16);
  p.rows = at + 16 + 2 * (int64_t)p.B * ceil_div(p.C, 64);
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
                      const int32_t* dst, int n, const int32_t* n_dev, int P, const PagesParams* remap,
                      hipStream_t stream) {
  for (int t0 = 0; t0 < n_tensors || (t0 == 0 && remap != nullptr); t0 += kPagesTensors) {
    PagesCopyParams c = {};
    const int t1 = n_tensors - t0 < kPagesTensors ? n_tensors : t0 + kPagesTensors;
    uint64_t bits = 0;
    for (int small = 0; small < 2; ++small) {  // the large tensors first
      for (int t = t0; t < t1; ++t) {
        if ((bytes[t] <= kPagesChunk / 4) != (small == 1)) continue;
        const int i = c.tensors++;
        c.base[i] = static_cast<uint8_t*>(base[t]);
        c.stride[i] = stride[t];
        c.bytes[i] = bytes[t];
        c.first[i + 1] = c.first[i] + (small ? 0 : (int)ceil_div64(bytes[t], kPagesChunk));
        bits |= (uintptr_t)base[t] | (uint64_t)stride[t] | (uint64_t)bytes[t];
      }
      if (small == 0) c.large = c.tensors;
    }
    c.vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
    c.src = src; c.dst = dst; c.n_dev = n_dev; c.n = n; c.P = P;
    if (remap != nullptr && t0 == 0) {
      const int64_t wgs = ceil_div64((int64_t)remap->B * remap->C, 1024);
      c.remap = (int)(wgs < 256 ? wgs : 256);
      c.tbl = remap->tbl; c.s_bt = remap->s_bt; c.B = remap->B; c.C = remap->C; c.map = remap->map;
    }
    // Eight workgroups of 256 threads to a CU, each walking its units.
    const int per = c.first[c.large] > 1 ? c.first[c.large] : 1;
    const int64_t units = c.tensors == 0 ? 0 : (int64_t)n * per, most = 8ll * device_cus();
    const int rc = launch(reinterpret_cast<const void*>(&pages_copy_kernel), c.remap + (int)(units < most ? units : most),
                          256, 0, stream, &c);
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
  // Every entry may want a page, and a want's place among them is an int.
  SPECQ_REQUIRE((int64_t)B * max_pages <= INT32_MAX, SPECQ_ENOTSUP, "kv_pages_reserve: block table of %lld entries is too large",
                (long long)B * max_pages);
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
  return pages_copy(n_tensors, base, page_stride, page_bytes, p.src, p.dst, B, nullptr, n_pages, nullptr, st);
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
  return pages_copy(n_tensors, base, page_stride, page_bytes, p.src, p.dst, n_pages, p.n_moves, n_pages, &p, st);
}

extern "C" int specq_kv_pages_copy(const int32_t* src, const int32_t* dst, int n, int n_pages, int n_tensors,
                                   void* const* base, const int64_t* page_stride, const int64_t* page_bytes,
                                   void* stream) {
  clear_error();
  SPECQ_REQUIRE(n >= 0 && n_pages > 0 && (n == 0 || (src && dst)), SPECQ_EINVAL, "kv_pages_copy: bad sizes or pointers");
  if (int rc = pages_tensors("kv_pages_copy", n_tensors, base, page_stride, page_bytes)) return rc;
  if (n == 0) return SPECQ_OK;
  return pages_copy(n_tensors, base, page_stride, page_bytes, src, dst, n, nullptr, n_pages, nullptr, (hipStream_t)stream);
}
