// Pages of a paged cache copied from place to place, in every pool of the cache by one launch: what a fork's children and a compaction ask for.
//
// A pool is an array [n][groups][rows][row] -- keys, values or pooled blocks of a layer, latent rows, a recurrent layer's states -- whose pages share
// their numbers with the other pools'.  A move (src, dst, tokens) copies the first ceil(tokens / per) rows of each group (per 0: the whole page) and
// leaves the rest of dst as it is.  A table of page numbers may be rewritten beside it.
//
// Bytes in, bytes out: bound by memory.  A workgroup takes one piece of PIECE bytes of one page of one pool, a thread's loads all in flight before its
// first store.
#include "seq_common.h"
#include <algorithm>

struct PagePool {
  char* base;
  long page_bytes, group_bytes;
  int groups, rows, row_bytes, per;
  int width, pad;                            // bytes a load moves: what the pool's addresses and sizes are whole numbers of
};
constexpr int POOLS_MAX = 48, PIECE = 16384, LOADS = PIECE / (256 * 16);
struct PagePools { PagePool p[POOLS_MAX]; };

template <typename V> __device__ __forceinline__ void copy_piece(char* __restrict__ dst, const char* __restrict__ src, int n) {
  const V* s = reinterpret_cast<const V*>(src);
  V* d = reinterpret_cast<V*>(dst);
  const int items = n / (int)sizeof(V);
  for (int i0 = threadIdx.x; i0 < items; i0 += 256 * LOADS) {
    V v[LOADS];
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      if (i0 + 256 * u < items) v[u] = s[i0 + 256 * u];
#pragma unroll
    for (int u = 0; u < LOADS; ++u)
      if (i0 + 256 * u < items) d[i0 + 256 * u] = v[u];
  }
}

// grid (pieces, moves, pools and, behind them, the table)
__global__ __launch_bounds__(256) void pages_copy_kernel(PagePools pools, int n_pools, const int* __restrict__ moves, int n_moves, int n_pages,
                                                         int* __restrict__ table, long n_table, const int* __restrict__ where) {
  if ((int)blockIdx.z == n_pools) {
    const long step = (long)gridDim.x * gridDim.y * 256;
    for (long i = ((long)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < n_table; i += step) {
      const int p = table[i];
      if (p >= 0 && p < n_pages) table[i] = where[p];
    }
    return;
  }
  if ((int)blockIdx.y >= n_moves) return;
  const PagePool& q = pools.p[blockIdx.z];
  const int src = moves[3 * blockIdx.y], dst = moves[3 * blockIdx.y + 1], tokens = moves[3 * blockIdx.y + 2];
  if (src < 0 || src >= n_pages || dst < 0 || dst >= n_pages || src == dst || tokens < 1) return;
  const int n = q.per ? min(q.rows, (tokens - 1) / q.per + 1) : q.rows;
  // rows that are all wanted stand together; otherwise each group's first ones do
  const bool whole = n == q.rows;
  const long bytes = whole ? (long)q.groups * q.group_bytes : (long)n * q.row_bytes;
  const int pieces = (int)((bytes + PIECE - 1) / PIECE);
  const int piece = whole ? (int)blockIdx.x : (int)(blockIdx.x % pieces), group = whole ? 0 : (int)(blockIdx.x / pieces);
  if (piece >= pieces || group >= q.groups) return;
  const long off = group * q.group_bytes + (long)piece * PIECE;
  const int len = (int)min((long)PIECE, bytes - (long)piece * PIECE);
  const char* s = q.base + src * q.page_bytes + off;
  char* d = q.base + dst * q.page_bytes + off;
  if (q.width == 16) copy_piece<u32x4>(d, s, len);
  else if (q.width == 4) copy_piece<unsigned>(d, s, len);
  else if (q.width == 2) copy_piece<u16>(d, s, len);
  else copy_piece<unsigned char>(d, s, len);
}

extern "C" int umb_pages_copy(const UmbPagePool* pools, int n_pools, const int* moves, int n_moves, int n_pages, int* table, long n_table,
                              const int* where, hipStream_t st) {
  if (n_pools < 0 || n_moves < 0 || n_pages < 1 || n_table < 0 || (n_pools > 0 && !pools) || (n_moves > 0 && !moves) || (n_table > 0 && (!table || !where)))
    return UMB_EINVAL;
  for (int i = 0; i < n_pools; ++i) {
    const UmbPagePool& q = pools[i];
    if (!q.base || q.page_bytes < 1 || q.groups < 1 || q.rows < 1 || q.row_bytes < 1 || q.per < 0 || q.groups > (1 << 20) || q.rows > (1 << 28) ||
        q.row_bytes > (1 << 30) || q.per > (1 << 28) || q.rows * q.row_bytes > q.page_bytes / q.groups)
      return UMB_EINVAL;
  }
  for (int z0 = 0; z0 < n_pools || z0 == 0; z0 += POOLS_MAX) {
    PagePools pp;
    const int n = n_pools - z0 < POOLS_MAX ? n_pools - z0 : POOLS_MAX;
    long pieces = 1;
    for (int i = 0; i < n; ++i) {
      const UmbPagePool& q = pools[z0 + i];
      PagePool& p = pp.p[i];
      p.base = reinterpret_cast<char*>(q.base);
      p.page_bytes = q.page_bytes;
      p.group_bytes = q.rows * q.row_bytes;
      p.groups = (int)q.groups;
      p.rows = (int)q.rows;
      p.row_bytes = (int)q.row_bytes;
      p.per = (int)q.per;
      const unsigned long any = (unsigned long)q.base | (unsigned long)q.page_bytes | (unsigned long)q.row_bytes;
      p.width = any % 16 == 0 ? 16 : any % 4 == 0 ? 4 : any % 2 == 0 ? 2 : 1;
      const long w = ((long)q.groups * p.group_bytes + PIECE - 1) / PIECE, g = q.groups * ((p.group_bytes + PIECE - 1) / PIECE);
      pieces = std::max(pieces, std::max(w, q.per ? g : 1L));
    }
    const bool tab = n_table > 0 && z0 == 0;
    if (n < 1 && !tab) break;
    if (pieces > 0x7fffffff) return UMB_EINVAL;
    for (int y0 = 0; y0 < n_moves || y0 == 0; y0 += 65535) {
      const int m = n_moves - y0 < 65535 ? n_moves - y0 : 65535;
      const int planes = n + (tab && y0 == 0 ? 1 : 0);
      if (planes < 1 || (m < 1 && !(tab && y0 == 0))) break;
      hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)pieces, m > 0 ? m : 1, planes), dim3(256), 0, st, pp, n, moves + 3L * y0, m, n_pages, table,
                         tab && y0 == 0 ? n_table : 0, where);
      UMB_LAUNCH_CHECK();
    }
  }
  return UMB_OK;
}
