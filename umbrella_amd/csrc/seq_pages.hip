// Pages of a paged cache copied from place to place, in every pool of the cache by one launch: what a fork's children and a compaction ask for.
//
// A pool is an array [n][groups][rows][row] -- keys, values or pooled blocks of a layer, latent rows, a recurrent layer's states -- whose pages share
// their numbers with the other pools'.  A move (src, dst, tokens) copies the first ceil(tokens / per) rows of each group (per 0: the whole page) and
// leaves the rest of dst as it is.  A table of page numbers may be rewritten beside it.
//
// Bytes in, bytes out: bound by memory.  A workgroup takes a piece of 256 x LOADS x 16 bytes of what one move copies in one pool, groups one behind the other as if
// they were neighbours, a thread's loads all in flight before its first store.  Stores go past the caches: nobody reads a new page before a step does, and a fork's
// siblings read the same begun page again (us: 48 begun pages of 16, 24 pools of 8 x 16 KB, 24 of 8 x 2 KB and 48 states of 512 KB, 148 MB, 47.7 -> 33.2;
// 75 pages of 48 pools of 128 KB, 944 MB, 192 either way, 4.9 TB/s where a plain copy of a store reaches 5.2).
#include "seq_common.h"
#include <algorithm>

struct PagePool {
  char* base;
  long page_bytes;
  int group_bytes, row_bytes, groups, rows, per;
  int width;                                 // bytes a load moves: what the pool's addresses and sizes are whole numbers of
  int first;                                 // the pool's first piece among all pools'
};
constexpr int POOLS_MAX = 48, LOADS = 8;
struct PagePools { PagePool p[POOLS_MAX]; int n, pieces; };

// items of sizeof(V) bytes: the first `take` of every `group`
template <typename V> __device__ __forceinline__ void copy_piece(char* __restrict__ dst, const char* __restrict__ src, unsigned i0, unsigned items, unsigned take, unsigned group) {
  V v[LOADS];
  unsigned at[LOADS];
  const unsigned skip = group - take;
  if (skip) {
    // i / take by a reciprocal, at most one off where i is below 2^22: both factors are within 2^-24 of what they are
    const float inv = 1.f / (float)take;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const unsigned i = i0 + 256 * u;
      unsigned g = (unsigned)((float)i * inv);
      if (items > (1u << 22)) g = i / take;
      g -= g * take > i;
      g += (g + 1) * take <= i;
      at[u] = i + g * skip;
    }
  } else {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) at[u] = i0 + 256 * u;
  }
#pragma unroll
  for (int u = 0; u < LOADS; ++u)
    if (i0 + 256 * u < items) v[u] = reinterpret_cast<const V*>(src)[at[u]];
#pragma unroll
  for (int u = 0; u < LOADS; ++u)
    if (i0 + 256 * u < items) __builtin_nontemporal_store(v[u], reinterpret_cast<V*>(dst) + at[u]);
}

// grid (the pools' pieces and, behind them, the table's; moves)
__global__ __launch_bounds__(256) void pages_copy_kernel(PagePools pools, const int* __restrict__ moves, int n_moves, int n_pages, int* __restrict__ table, long n_table,
                                                         const int* __restrict__ where) {
  const int piece = blockIdx.x;
  if (piece >= pools.pieces) {
    const long blocks = gridDim.x - pools.pieces;
    for (long i = ((long)blockIdx.y * blocks + piece - pools.pieces) * 256 + threadIdx.x; i < n_table; i += blocks * gridDim.y * 256) {
      const int p = table[i];
      if (p >= 0 && p < n_pages) table[i] = where[p];
    }
    return;
  }
  const int src = moves[3 * blockIdx.y], dst = moves[3 * blockIdx.y + 1], tokens = moves[3 * blockIdx.y + 2];
  if (src < 0 || src >= n_pages || dst < 0 || dst >= n_pages || src == dst || tokens < 1) return;
  int lo = 0, hi = pools.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pools.p[mid].first <= piece) lo = mid;
    else hi = mid - 1;
  }
  const PagePool q = pools.p[__builtin_amdgcn_readfirstlane(lo)];
  const int n = q.per ? min(q.rows, (tokens - 1) / q.per + 1) : q.rows;
  const unsigned take = (unsigned)n * q.row_bytes / q.width, group = q.group_bytes / q.width, items = take * q.groups, per_piece = 256 * LOADS;
  const unsigned i0 = (unsigned)(piece - q.first) * per_piece;
  if (i0 >= items) return;
  const char* s = q.base + src * q.page_bytes;
  char* d = q.base + dst * q.page_bytes;
  if (q.width == 16) copy_piece<u32x4>(d, s, i0 + threadIdx.x, items, take, group);
  else if (q.width == 4) copy_piece<unsigned>(d, s, i0 + threadIdx.x, items, take, group);
  else if (q.width == 2) copy_piece<u16>(d, s, i0 + threadIdx.x, items, take, group);
  else copy_piece<unsigned char>(d, s, i0 + threadIdx.x, items, take, group);
}

extern "C" int umb_pages_copy(const UmbPagePool* pools, int n_pools, const int* moves, int n_moves, int n_pages, int* table, long n_table,
                              const int* where, hipStream_t st) {
  if (n_pools < 0 || n_moves < 0 || n_pages < 1 || n_table < 0 || (n_pools > 0 && !pools) || (n_moves > 0 && !moves) || (n_table > 0 && (!table || !where)))
    return UMB_EINVAL;
  for (int i = 0; i < n_pools; ++i) {
    const UmbPagePool& q = pools[i];
    if (!q.base || q.page_bytes < 1 || q.groups < 1 || q.rows < 1 || q.row_bytes < 1 || q.per < 0 || q.per > (1 << 28) || q.groups > (1 << 30) ||
        q.rows > (1 << 30) / q.groups || q.row_bytes > (1 << 30) / (q.groups * q.rows) || q.groups * q.rows * q.row_bytes > q.page_bytes)
      return UMB_EINVAL;
  }
  for (int z0 = 0; z0 < n_pools || z0 == 0; z0 += POOLS_MAX) {
    PagePools pp;
    pp.n = n_pools - z0 < POOLS_MAX ? n_pools - z0 : POOLS_MAX;
    long pieces = 0;
    for (int i = 0; i < pp.n; ++i) {
      const UmbPagePool& q = pools[z0 + i];
      PagePool& p = pp.p[i];
      p.base = reinterpret_cast<char*>(q.base);
      p.page_bytes = q.page_bytes;
      p.row_bytes = (int)q.row_bytes;
      p.group_bytes = (int)(q.rows * q.row_bytes);
      p.groups = (int)q.groups;
      p.rows = (int)q.rows;
      p.per = (int)q.per;
      const unsigned long any = (unsigned long)q.base | (unsigned long)q.page_bytes | (unsigned long)q.row_bytes;
      p.width = any % 16 == 0 ? 16 : any % 4 == 0 ? 4 : any % 2 == 0 ? 2 : 1;
      p.first = (int)pieces;
      pieces += ((long)p.group_bytes * p.groups / p.width + 256 * LOADS - 1) / (256 * LOADS);
    }
    if (pieces > 0x7ffffff) return UMB_EINVAL;
    pp.pieces = (int)pieces;
    const bool tab = n_table > 0 && z0 == 0;
    for (int y0 = 0; y0 < n_moves || y0 == 0; y0 += 65535) {
      const int m = n_moves - y0 < 65535 ? n_moves - y0 : 65535;
      const long rows = tab && y0 == 0 ? std::min(256L, n_table / (m > 0 ? m : 1) / 256 + 1) : 0;      // workgroups of the table in each row of the grid
      if (m < 1) pp.pieces = 0;                // (the table alone)
      if (pp.pieces + rows < 1) break;
      hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)(pp.pieces + rows), m > 0 ? m : 1), dim3(256), 0, st, pp, moves + 3L * y0, m, n_pages, table, n_table, where);
      UMB_LAUNCH_CHECK();
    }
  }
  return UMB_OK;
}
