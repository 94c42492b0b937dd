// Low-rank adapters of many requests beside a projection that all of them share:
//     out[t] = base[t] + scale[a] B_a (A_a x[t]),  a = adapter[t]
// x [T][K], A [S][R][K], B [S][N][R] in `dtype`; base and out fp32 [T][N]; of adapter a the first rank[a] of R count.  A row whose number is none of
// 0 .. S - 1 is its base.
//
// Two launches: u = A x, fp32, summed over K in `parts` pieces; then out.  Rows of one adapter are taken together, up to 64, so that A and B are read once
// for them: in a window of 256 rows the row whose place among its adapter's rows is a multiple of 64 stands for the 64 from it on, and every other row's
// turn is empty.  Nothing has to be sorted or counted beforehand, and the order of a row's sums does not depend on which rows come with it.
//
// u enters the second product with 22 bits or more: three bf16 terms (each the rest that the one before left), two fp16 ones behind a power of two per row
// (whatever u's size), or itself in fp32.
#include "seq_common.h"
#include <algorithm>

constexpr int WINDOW = 256, TILE = 64, R_MAX = 128;

template <typename P> struct Frag { u32x4 v; };
template <> struct Frag<F32> { f32x4 lo, hi; };
template <typename P> __device__ __forceinline__ f32x4 mma(const Frag<P>& a, const Frag<P>& b, f32x4 c) { return P::mfma(a.v, b.v, c); }
template <> __device__ __forceinline__ f32x4 mma<F32>(const Frag<F32>& a, const Frag<F32>& b, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], c, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[i], b.hi[i], c, 0, 0, 0);
  return c;
}
// eight elements p[0 .. n), nothing behind them
template <typename P, bool WHOLE> __device__ __forceinline__ Frag<P> load8(const typename El<P>::type* p, int n) {
  if constexpr (WHOLE) {
    Frag<P> f{};
    if (n > 0) {
      if constexpr (std::is_same_v<P, F32>) { f.lo = *reinterpret_cast<const f32x4*>(p); f.hi = *reinterpret_cast<const f32x4*>(p + 4); }
      else f.v = *reinterpret_cast<const u32x4*>(p);
    }
    return f;
  } else {
    typename El<P>::type e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : (typename El<P>::type)0;
    return __builtin_bit_cast(Frag<P>, e);
  }
}

// The rows that block `i` of a window stands for: those of its own row's adapter from that row on, TILE at most, if the row's place among them is a multiple of
// TILE; none otherwise.  rows: LDS [TILE]; all threads of 256 call it.
struct Tile { int adapter, n; };
__device__ __forceinline__ Tile rows_of(int t, int T, int S, const int* __restrict__ adapter, int* rows, int* waves) {
  const int w0 = t / WINDOW * WINDOW, i = w0 + threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int mine = adapter[t], other = i < T ? adapter[i] : mine;
  if (mine < 0 || mine >= S) mine = -1;
  if (other < 0 || other >= S) other = -1;
  const bool same = i < T && other == mine;
  const unsigned long long bal = __ballot(same);
  if (lane == 0) waves[wave] = __popcll(bal);
  __syncthreads();
  int at = __popcll(bal & ((1ull << lane) - 1ull)), all = 0;
#pragma unroll
  for (int w = 0; w < WINDOW / 64; ++w) { if (w < wave) at += waves[w]; all += waves[w]; }
  if (i == t) waves[4] = at;
  __syncthreads();
  const int first = waves[4];
  if (first % TILE) return Tile{mine, 0};
  if (same && at >= first && at < first + TILE) rows[at - first] = i;
  __syncthreads();
  return Tile{mine, min(TILE, all - first)};
}

// ---- u[part][t][r] = sum over the part's K of A x.  grid (rows, parts); a wave a quarter of the part's K where there are at most 16 rows, otherwise a quarter of
// the rows
template <typename P, bool WHOLE, int RF>
__global__ __launch_bounds__(256) void adapter_down_kernel(float* __restrict__ u, const typename El<P>::type* __restrict__ x, const typename El<P>::type* __restrict__ a,
                                                           const int* __restrict__ adapter, const int* __restrict__ rank, int T, int K, int S, int R, int per) {
  __shared__ int rows[TILE], waves[5];
  __shared__ f32x4 part[3][RF][64];
  const Tile tile = rows_of(blockIdx.x, T, S, adapter, rows, waves);
  if (tile.n < 1 || tile.adapter < 0) return;
  const int ra = rank ? min(max(rank[tile.adapter], 0), R) : R;
  if (ra < 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const bool few = tile.n <= 16;
  const int k0 = blockIdx.y * per, k1 = min(K, k0 + per);
  // (steps of 32)
  const int steps = (k1 - k0 + 31) / 32, s0 = few ? steps * wave / 4 : 0, s1 = few ? steps * (wave + 1) / 4 : steps;
  const int own = few ? j : wave * 16 + j;
  if (!few && wave * 16 >= tile.n) return;
  const typename El<P>::type* xr = x + (long)rows[min(own, tile.n - 1)] * K;
  const typename El<P>::type* ar[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) ar[f] = a + ((long)tile.adapter * R + min(16 * f + j, ra - 1)) * K;
  f32x4 acc[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = s0; s < s1; ++s) {
    const int k = k0 + 32 * s + 8 * g, n = k1 - k;
    const Frag<P> b = load8<P, WHOLE>(xr + k, n);
#pragma unroll
    for (int f = 0; f < RF; ++f)
      if (16 * f < ra) acc[f] = mma<P>(load8<P, WHOLE>(ar[f] + k, n), b, acc[f]);
  }
  if (few) {
    if (wave > 0)
#pragma unroll
      for (int f = 0; f < RF; ++f) part[wave - 1][f][lane] = acc[f];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int f = 0; f < RF; ++f) acc[f] = (acc[f] + part[0][f][lane]) + (part[1][f][lane] + part[2][f][lane]);
  }
  if (own >= tile.n) return;
  float* to = u + ((long)blockIdx.y * T + rows[own]) * R;
#pragma unroll
  for (int f = 0; f < RF; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (16 * f + 4 * g + e < ra) to[16 * f + 4 * g + e] = acc[f][e];
}

// ---- out = base + B (scale u).  grid (rows, pieces of N); a wave takes 16 columns at a time, all the tile's rows for them
template <typename P> struct Terms { static constexpr int N = 1; };
template <> struct Terms<BF16> { static constexpr int N = 3; };
template <> struct Terms<F16> { static constexpr int N = 2; };

template <typename P, bool WHOLE, bool QUADS, int RC>
__global__ __launch_bounds__(256) void adapter_up_kernel(float* out, const float* base, const float* __restrict__ u, const typename El<P>::type* __restrict__ b,
                                                         const int* __restrict__ adapter, const float* __restrict__ scale, const int* __restrict__ rank, int T, int N,
                                                         int S, int R, int parts, int columns) {
  typedef typename El<P>::type E;
  constexpr int NT = Terms<P>::N;
  __shared__ int rows[TILE], waves[5];
  __shared__ __attribute__((aligned(16))) E terms[NT][RC][TILE / 16][64][8];
  __shared__ float power[TILE];
  const Tile tile = rows_of(blockIdx.x, T, S, adapter, rows, waves);
  if (tile.n < 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.y * columns, n1 = min(N, n0 + columns);
  const int ra = tile.adapter < 0 ? 0 : rank ? min(max(rank[tile.adapter], 0), R) : R;
  if (ra < 1) {
    if (out != base)
      for (int i = wave; i < tile.n; i += 4)
        for (int n = n0 + lane; n < n1; n += 64) out[(long)rows[i] * N + n] = base[(long)rows[i] * N + n];
    return;
  }
  const float sc = scale ? scale[tile.adapter] : 1.f;
  // a row's terms by four lanes: lane j, g of the fragments is row j, elements 32 c + 8 g ..
  const int i = threadIdx.x >> 2, q = threadIdx.x & 3;
  float v[RC][8], most = 0.f;
#pragma unroll
  for (int c = 0; c < RC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int r = 32 * c + 8 * q + e;
      float s = 0.f;
      if (i < tile.n && r < ra) {
        for (int p = 0; p < parts; ++p) s += u[((long)p * T + rows[i]) * R + r];
        s *= sc;
      }
      v[c][e] = s;
      most = fmaxf(most, fabsf(s));
    }
  if constexpr (NT == 2) {                   // fp16: the row's largest between 1 and 2
    most = fmaxf(most, __shfl_xor(most, 1, 64));
    most = fmaxf(most, __shfl_xor(most, 2, 64));
    const int e = most > 0.f && most < INFINITY ? ilogbf(most) : 0;
    if (q == 0) power[i] = ldexpf(1.f, max(e, -126));
#pragma unroll
    for (int c = 0; c < RC; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = ldexpf(v[c][k], -max(e, -126));
  }
#pragma unroll
  for (int c = 0; c < RC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      E* to = &terms[0][c][i >> 4][q * 16 + (i & 15)][e];
      constexpr long next = (long)RC * (TILE / 16) * 64 * 8;
      if constexpr (NT == 1) *to = v[c][e];
      else {
        float x = v[c][e];
        const E hi = P::from_f(x);
        to[0] = hi;
        float rest = x - P::to_f(hi);
        if (!(fabsf(rest) < INFINITY)) rest = 0.f;
        if constexpr (NT == 2) to[next] = P::from_f(rest * 2048.f);
        else {
          const E mid = P::from_f(rest);
          to[next] = mid;
          to[2 * next] = P::from_f(rest - P::to_f(mid));
        }
      }
    }
  __syncthreads();
  const int frags = (tile.n + 15) >> 4;
  for (int n = n0 + 16 * wave; n < n1; n += 64) {
    Frag<P> w[RC];
    const E* br = b + ((long)tile.adapter * N + min(n + j, N - 1)) * R;
#pragma unroll
    for (int c = 0; c < RC; ++c) w[c] = load8<P, WHOLE>(br + 32 * c + 8 * g, (WHOLE ? (ra + 7) & ~7 : ra) - 32 * c - 8 * g);
    if (WHOLE && (ra & 7)) {                 // what stands behind the rank is nobody's
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        E e[8];
        __builtin_memcpy(e, &w[c], sizeof e);
#pragma unroll
        for (int k = 0; k < 8; ++k) if (32 * c + 8 * g + k >= ra) e[k] = (E)0;
        __builtin_memcpy(&w[c], e, sizeof e);
      }
    }
#pragma unroll
    for (int f = 0; f < TILE / 16; ++f) {
      if (f >= frags) break;
      const int at = f * 16 + j, col = n + 4 * g;
      const bool in = at < tile.n;
      const long o = (long)rows[in ? at : 0] * N + col;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (in) {
        if (QUADS) { if (col < n1) x = *reinterpret_cast<const f32x4*>(base + o); }
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (col + e < n1) x[e] = base[o + e];
      }
      f32x4 acc = {0.f, 0.f, 0.f, 0.f}, low = acc;
#pragma unroll
      for (int c = 0; c < RC; ++c) {
        const Frag<P>* t = reinterpret_cast<const Frag<P>*>(&terms[0][c][f][lane][0]);
        constexpr long next = (long)RC * (TILE / 16) * 64;
        if constexpr (NT == 3) {
          low = mma<P>(w[c], t[2 * next], low);
          low = mma<P>(w[c], t[next], low);
          acc = mma<P>(w[c], t[0], acc);
        } else {
          if constexpr (NT == 2) low = mma<P>(w[c], t[next], low);
          acc = mma<P>(w[c], t[0], acc);
        }
      }
      if constexpr (NT == 3) acc += low;
      if constexpr (NT == 2) acc = (acc + low * (1.f / 2048.f)) * power[at];
      if (!in) continue;
      x += acc;
      if (QUADS) { if (col < n1) *reinterpret_cast<f32x4*>(out + o) = x; }
      else
#pragma unroll
        for (int e = 0; e < 4; ++e) if (col + e < n1) out[o + e] = x[e];
    }
  }
}

extern "C" int umb_seq_adapters_parts(int T, int K) {
  if (T < 1 || K < 1) return 0;
  const int steps = (K + 31) / 32, want = std::max(1, 512 / std::min(T, 512));
  return std::max(1, std::min({want, (steps + 3) / 4, 16}));
}

template <typename P, bool WHOLE>
static int adapters_launch(float* out, const float* base, const void* x, const void* a, const void* b, const int* adapter, const float* scale, const int* rank, int T,
                           int N, int K, int S, int R, bool quads, float* u, hipStream_t st) {
  typedef typename El<P>::type E;
  const int parts = umb_seq_adapters_parts(T, K), per = (((K + 31) / 32 + parts - 1) / parts) * 32;
#define DOWN(RF) hipLaunchKernelGGL((adapter_down_kernel<P, WHOLE, RF>), dim3(T, parts), dim3(256), 0, st, u, (const E*)x, (const E*)a, adapter, rank, T, K, S, R, per)
  if (R <= 16) DOWN(1);
  else if (R <= 32) DOWN(2);
  else if (R <= 64) DOWN(4);
  else DOWN(8);
#undef DOWN
  UMB_LAUNCH_CHECK();
  const int columns = 256 * (1 + (N - 1) / (256 * 65535)), pieces = (N + columns - 1) / columns;
#define UP(RC)                                                                                                                                        \
  if (quads) hipLaunchKernelGGL((adapter_up_kernel<P, WHOLE, true, RC>), dim3(T, pieces), dim3(256), 0, st, out, base, u, (const E*)b, adapter, scale, rank, \
                                T, N, S, R, parts, columns);                                                                                          \
  else hipLaunchKernelGGL((adapter_up_kernel<P, WHOLE, false, RC>), dim3(T, pieces), dim3(256), 0, st, out, base, u, (const E*)b, adapter, scale, rank, T, N, \
                          S, R, parts, columns)
  if (R <= 32) { UP(1); }
  else if (R <= 64) { UP(2); }
  else { UP(4); }
#undef UP
  UMB_LAUNCH_CHECK();
  return UMB_OK;
}

extern "C" int umb_seq_adapters(float* out, const float* base, const void* x, const void* a, const void* b, const int* adapter, const float* scale, const int* rank,
                                int T, int N, int K, int S, int R, float* scratch, long scratch_floats, int dtype, hipStream_t st) {
  if (!out || !base || !x || !a || !b || !adapter || !scratch || T < 1 || N < 1 || K < 1 || S < 1 || R < 1 || R > R_MAX || N > (1 << 24) || K > (1 << 24) ||
      scratch_floats < (long)umb_seq_adapters_parts(T, K) * T * R)
    return UMB_EINVAL;
  const bool quads = N % 4 == 0 && ((uintptr_t)out | (uintptr_t)base) % 16 == 0;
  const bool whole = K % 8 == 0 && R % 8 == 0 && ((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) % 16 == 0;
  DISPATCH_SEQ_DTYPE(dtype, {
    return whole ? adapters_launch<P, true>(out, base, x, a, b, adapter, scale, rank, T, N, K, S, R, quads, scratch, st)
                 : adapters_launch<P, false>(out, base, x, a, b, adapter, scale, rank, T, N, K, S, R, quads, scratch, st);
  })
}
