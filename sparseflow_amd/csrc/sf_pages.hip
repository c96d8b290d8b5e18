// The pages of a cache: sequences that grow, shrink, fork and end, and pools that are
// compacted.  Everything is on the device, so that a serving step can be captured.
//
// A call is two or three small kernels in turn: one workgroup to a request looks what it needs
// (and gives back what it frees), one workgroup deals the free pages out, lowest first, to the
// requests in turn, and workgroups write the tables and copy the pages.  Bound by launches (256
// forks and ends: six kernels of 3 to 9 us, 48 us a pass) and copies (4100 pages of 68 KB to
// other places: 207 us, the copying 184 of them at 4.6 TB/s).
#include "sf_seq.h"

namespace sf {
namespace {

constexpr int kPageThreads = 256;
constexpr int kDealThreads = 1024;

__device__ __forceinline__ int64_t pages_of(int64_t length, int page) { return (length + page - 1) / page; }

__device__ __forceinline__ bool page_ok(const PagesArgs& a, int64_t p) { return p >= 0 && p < a.pages; }

// Whether an earlier request names the same row (all threads of the workgroup ask).
__device__ __forceinline__ bool named_before(const int32_t* rows, int64_t request) {
  __shared__ int found;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  const int32_t mine = rows[request];
  for (int64_t i = threadIdx.x; i < request; i += kPageThreads)
    if (rows[i] == mine) found = 1;
  __syncthreads();
  return found != 0;
}

// Request blockIdx.x of a resize: shrinks at once, or says what growing needs.
__global__ __launch_bounds__(kPageThreads) void k_pages_release(PagesArgs a) {
  const int64_t q = blockIdx.x;
  const int64_t row = a.rows[q], size = a.other[q];
  const bool again = named_before(a.rows, q);
  const bool ok = !again && row >= 0 && row < a.states && size >= 0 && pages_of(size, a.page_size) <= a.width;
  int64_t old = ok ? a.lengths[row] : 0;
  old = old < 0 ? 0 : old;
  __syncthreads();
  if (ok && size <= old) {
    int64_t end = pages_of(old, a.page_size);
    end = end > a.width ? a.width : end;
    int32_t* table = a.tables + row * a.width;
    for (int64_t i = pages_of(size, a.page_size) + threadIdx.x; i < end; i += kPageThreads) {
      const int64_t p = table[i];
      if (page_ok(a, p)) atomicSub(a.refs + p, 1);
      table[i] = -1;
    }
  }
  if (threadIdx.x != 0) return;
  a.need[q] = !ok ? -1 : size <= old ? 0 : (int32_t)(pages_of(size, a.page_size) - pages_of(old, a.page_size));
  a.old[q] = (int32_t)old;
  if (ok && size <= old) a.lengths[row] = (int32_t)size;
}

// Requests of a fork: a page for the parent's last, partial one.
__global__ __launch_bounds__(kPageThreads) void k_pages_fork_need(PagesArgs a) {
  const int64_t q = blockIdx.x;
  const int64_t child = a.rows[q], parent = a.other[q];
  const bool again = named_before(a.rows, q);
  if (threadIdx.x != 0) return;
  const bool ok = !again && child >= 0 && child < a.states && parent >= 0 && parent < a.states && a.lengths[child] == 0;
  int64_t n = ok ? a.lengths[parent] : 0;
  const bool fits = n >= 0 && pages_of(n, a.page_size) <= a.width;
  a.need[q] = !ok || !fits ? -1 : n % a.page_size != 0;
  a.old[q] = (int32_t)n;
}

// The sum of v over the workgroup's threads before this one, and over all.
__device__ __forceinline__ int64_t block_before(int64_t v, int64_t& total) {
  __shared__ int64_t part[kDealThreads / kWave];
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  int64_t in = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t o = __shfl_up(in, d, kWave);
    if (lane >= d) in += o;
  }
  __syncthreads();
  if (lane == kWave - 1) part[wave] = in;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kDealThreads / kWave; ++w) {
    before += w < wave ? part[w] : 0;
    total += part[w];
  }
  return before + in - v;
}

// One workgroup: request q's pages are list[first[q]] on.  GROW: a last, partial page that
// others use too has to be replaced.
template <bool GROW>
__global__ __launch_bounds__(kDealThreads) void k_pages_deal(PagesArgs a) {
  int64_t all = 0;
  for (int64_t at = 0; at < a.requests; at += kDealThreads) {
    const int64_t q = at + threadIdx.x;
    int64_t need = 0;
    if (q < a.requests) {
      need = a.need[q];
      if (GROW && need >= 0) {
        const int64_t old = a.old[q], row = a.rows[q], last = old / a.page_size;
        if (a.other[q] > old && old % a.page_size != 0 && last < a.width) {
          const int64_t p = a.tables[row * a.width + last];
          if (page_ok(a, p) && a.refs[p] > 1) {
            need += 1 << 30;  // (widths are below 2^30)
            a.shared[q] = (int32_t)p;
          }
        }
        a.need[q] = (int32_t)need;
        need = (need & ((1 << 30) - 1)) + (need >> 30);
      }
      need = need < 0 ? 0 : need;
    }
    int64_t total;
    const int64_t before = all + block_before(need, total);
    if (q < a.requests) a.first[q] = before > 0x7fffffff ? 0x7fffffff : (int32_t)before;
    all += total;
  }
  int64_t found = 0;
  for (int64_t at = 0; at < a.pages && found < all; at += 4 * kDealThreads) {
    const int64_t p0 = at + 4 * threadIdx.x;
    int free[4], n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      free[i] = p0 + i < a.pages && a.refs[p0 + i] <= 0;
      n += free[i];
    }
    int64_t total, rank = found + block_before(n, total);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (free[i]) a.list[rank++] = (int32_t)(p0 + i);
    found += total;
  }
  if (threadIdx.x == 0) a.counts[0] = (int32_t)found;
}

// Copies page `from` of every pool to page `to`, the workgroup's share of it: the pools' 16-byte
// units one pool after another, four of a thread under way at a time.  (A page of 68 KB in four
// pools by one workgroup, pool by pool: 221 us for a compaction that moves 4100 of them.)
__device__ __forceinline__ void copy_page(const PagePools& pools, int64_t from, int64_t to, int part, int parts) {
  typedef uint32_t V __attribute__((ext_vector_type(4)));
  const int64_t all = pools.count > 0 ? pools.units[pools.count - 1] : 0, per = (all + parts - 1) / parts;
  const int64_t begin = part * per, end = begin + per < all ? begin + per : all;
  for (int64_t k = begin + threadIdx.x; k < end; k += 4 * kPageThreads) {
    V v[4];
    V* d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = k + u * kPageThreads < end ? k + u * kPageThreads : end - 1;
      int i = 0;
      while (at >= pools.units[i]) ++i;
      const int64_t off = 16 * (at - (i > 0 ? pools.units[i - 1] : 0));
      v[u] = *reinterpret_cast<const V*>(pools.at[i] + from * pools.bytes[i] + off);
      d[u] = reinterpret_cast<V*>(pools.at[i] + to * pools.bytes[i] + off);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (k + u * kPageThreads < end) *d[u] = v[u];
  }
  if (!pools.odd) return;
  for (int i = 0; i < pools.count; ++i) {
    if (pools.units[i] > (i > 0 ? pools.units[i - 1] : 0)) continue;
    const int64_t bytes = pools.bytes[i];
    for (int64_t k = part * kPageThreads + threadIdx.x; k < bytes; k += parts * kPageThreads)
      pools.at[i][to * bytes + k] = pools.at[i][from * bytes + k];
  }
}

// Request `id / parts` after the deal: the table, the users' counts and the copy of a
// page that is no longer shared.
__global__ __launch_bounds__(kPageThreads) void k_pages_grown(PagesArgs a, int parts) {
  const int64_t id = a.block0 + blockIdx.x, q = id / parts;
  const int part = (int)(id - q * parts);
  const int32_t raw = a.need[q];
  const int64_t old = a.old[q], size = a.other[q], row = a.rows[q];
  const int64_t need = raw < 0 ? -1 : (raw & ((1 << 30) - 1)) + (raw >> 30);
  const bool ok = need >= 0 && (need == 0 || a.first[q] + need <= a.counts[0]);
  if (part == 0 && threadIdx.x == 0) a.granted[q] = ok;
  if (!ok || size <= old) return;
  const int64_t first = a.first[q], shared = raw >> 30;
  if (shared) copy_page(a.pools, a.shared[q], a.list[first], part, parts);
  if (part != 0) return;
  const int64_t from = pages_of(old, a.page_size) - shared, end = pages_of(size, a.page_size);
  for (int64_t i = from + threadIdx.x; i < end; i += kPageThreads) {
    const int32_t p = a.list[first + i - from];
    a.tables[row * a.width + i] = p;
    a.refs[p] = 1;
  }
  if (threadIdx.x == 0) {
    if (shared) atomicSub(a.refs + a.shared[q], 1);
    a.lengths[row] = (int32_t)size;
  }
}

// A fork's child: shares the parent's full pages and has the last, partial one copied.
__global__ __launch_bounds__(kPageThreads) void k_pages_forked(PagesArgs a, int parts) {
  const int64_t id = a.block0 + blockIdx.x, q = id / parts;
  const int part = (int)(id - q * parts);
  const int64_t need = a.need[q], n = a.old[q], child = a.rows[q], parent = a.other[q];
  const bool ok = need >= 0 && (need == 0 || a.first[q] + need <= a.counts[0]);
  if (part == 0 && threadIdx.x == 0) a.granted[q] = ok;
  if (!ok || n == 0) return;
  const int32_t* from = a.tables + parent * a.width;
  const int64_t whole = n / a.page_size;
  if (part == 0) {
    int32_t* table = a.tables + child * a.width;
    for (int64_t i = threadIdx.x; i < whole; i += kPageThreads) {
      const int32_t p = from[i];
      table[i] = p;
      if (page_ok(a, p)) atomicAdd(a.refs + p, 1);
    }
    if (threadIdx.x == 0) {
      a.lengths[child] = (int32_t)n;
      if (need) {
        const int32_t p = a.list[a.first[q]];
        table[whole] = p;
        a.refs[p] = 1;
      }
    }
  }
  if (need && page_ok(a, from[whole])) copy_page(a.pools, from[whole], a.list[a.first[q]], part, parts);
}

// One workgroup: the live pages from `live` on go to the free ones below it, in order.
__global__ __launch_bounds__(kDealThreads) void k_pages_moves(PagesArgs a) {
  int64_t live = 0;
  for (int64_t at = 0; at < a.pages; at += 4 * kDealThreads) {
    const int64_t p0 = at + 4 * threadIdx.x;
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += p0 + i < a.pages && a.refs[p0 + i] > 0;
    live += n;
  }
  int64_t total;
  block_before(live, total);
  live = total;
  int64_t holes = 0, strays = 0;
  for (int64_t at = 0; at < a.pages; at += 4 * kDealThreads) {
    const int64_t p0 = at + 4 * threadIdx.x;
    int hole[4], stray[4], nh = 0, ns = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = p0 + i < a.pages, used = in && a.refs[p0 + i] > 0;
      hole[i] = in && !used && p0 + i < live;
      stray[i] = used && p0 + i >= live;
      nh += hole[i], ns += stray[i];
    }
    int64_t both;
    const int64_t before = block_before(nh + ((int64_t)ns << 32), both);
    int64_t h = holes + (before & 0xffffffff), s = strays + (before >> 32);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (hole[i]) a.to[h++] = (int32_t)(p0 + i);
      if (stray[i]) a.list[s++] = (int32_t)(p0 + i);
    }
    holes += both & 0xffffffff, strays += both >> 32;
  }
  if (threadIdx.x == 0) {
    a.counts[0] = (int32_t)strays;
    a.granted[0] = (int32_t)live;
  }
}

// The first kMoveBlocks workgroups make the moves' copies and move their pages' users, the others
// rename the moved pages in the tables: they look for them among the sources, which are in order.
constexpr int kMoveBlocks = 2048, kRenameBlocks = 512;
__global__ __launch_bounds__(kPageThreads) void k_pages_move(PagesArgs a, int parts) {
  const int64_t moves = a.counts[0];
  if (blockIdx.x < kMoveBlocks) {
    for (int64_t w = blockIdx.x; w < moves * parts; w += kMoveBlocks) {
      const int64_t i = w / parts;
      const int32_t from = a.list[i], to = a.to[i];
      copy_page(a.pools, from, to, (int)(w - i * parts), parts);
      if (w == i * parts && threadIdx.x == 0) {
        a.refs[to] = a.refs[from];
        a.refs[from] = 0;
      }
    }
    return;
  }
  if (moves == 0) return;
  const int64_t low = a.list[0], n = a.states * a.width;
  for (int64_t i = (int64_t)(blockIdx.x - kMoveBlocks) * kPageThreads + threadIdx.x; i < n; i += kRenameBlocks * kPageThreads) {
    const int32_t p = a.tables[i];
    if (p < low || p >= a.pages) continue;
    int64_t lo = 0, hi = moves;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) >> 1;
      if (a.list[mid] <= p) lo = mid;
      else hi = mid;
    }
    if (a.list[lo] == p) a.tables[i] = a.to[lo];
  }
}

// Pages rows[i] of the pools to pages other[i].
__global__ __launch_bounds__(kPageThreads) void k_pages_copy(PagesArgs a, int parts) {
  const int64_t id = a.block0 + blockIdx.x, q = id / parts;
  const int64_t from = a.rows[q], to = a.other[q];
  if (!page_ok(a, from) || !page_ok(a, to) || from == to) return;
  copy_page(a.pools, from, to, (int)(id - q * parts), parts);
}

// Workgroups to a page: 16 KB each.
int page_parts(const PagesArgs& a) {
  int64_t bytes = 0;
  for (int i = 0; i < a.pools.count; ++i) bytes += a.pools.bytes[i];
  const int64_t parts = (bytes + 16383) / 16384;
  return (int)(parts < 1 ? 1 : parts > 64 ? 64 : parts);
}

int last_error() { return (int)hipGetLastError(); }

// Calls kernel(args, parts) with `parts` workgroups to a request, in as many launches as that takes.
template <typename Kernel>
int launch_parts(const PagesArgs& a, Kernel kernel, hipStream_t stream) {
  const int parts = page_parts(a);
  return launch_blocks(a, &PagesArgs::block0, a.requests * parts, [&](const PagesArgs& part, unsigned grid) {
    kernel<<<grid, kPageThreads, 0, stream>>>(part, parts);
  });
}

}  // namespace

// (requests: at most 2^20, see sparseflow.h)
int launch_pages_resize(const PagesArgs& a, hipStream_t stream) {
  timing_begin(K_PAGES, stream);
  k_pages_release<<<(unsigned)a.requests, kPageThreads, 0, stream>>>(a);
  k_pages_deal<true><<<1, kDealThreads, 0, stream>>>(a);
  int rc = last_error();
  if (rc == (int)hipSuccess) rc = launch_parts(a, k_pages_grown, stream);
  timing_end(K_PAGES, stream);
  return rc;
}

int launch_pages_fork(const PagesArgs& a, hipStream_t stream) {
  timing_begin(K_PAGES, stream);
  k_pages_fork_need<<<(unsigned)a.requests, kPageThreads, 0, stream>>>(a);
  k_pages_deal<false><<<1, kDealThreads, 0, stream>>>(a);
  int rc = last_error();
  if (rc == (int)hipSuccess) rc = launch_parts(a, k_pages_forked, stream);
  timing_end(K_PAGES, stream);
  return rc;
}

int launch_pages_compact(const PagesArgs& a, hipStream_t stream) {
  timing_begin(K_PAGES, stream);
  k_pages_moves<<<1, kDealThreads, 0, stream>>>(a);
  k_pages_move<<<kMoveBlocks + kRenameBlocks, kPageThreads, 0, stream>>>(a, page_parts(a));
  timing_end(K_PAGES, stream);
  return last_error();
}

int launch_pages_copy(const PagesArgs& a, hipStream_t stream) {
  timing_begin(K_PAGES, stream);
  const int rc = launch_parts(a, k_pages_copy, stream);
  timing_end(K_PAGES, stream);
  return rc;
}

}  // namespace sf
