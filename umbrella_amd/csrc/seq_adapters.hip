// Low-rank adapters of many requests beside a projection that all of them share:
//     out[t] = base[t] + scale[a] B_a (A_a x[t]),  a = adapter[t]
// x [T][K], A [S][R][K], B [S][N][R] in `dtype`; base and out fp32 [T][N]; of adapter a the first rank[a] of R count.  A row whose number is none of
// 0 .. S - 1 is its base.
//
// Two launches (one where the factors are small): u = A x, fp32, summed over K in `parts` pieces; then out.  Rows of one adapter are taken together, so that A and B are read once for them.
// Up to 256 rows: tiles of 16; the row whose place among its adapter's rows is a multiple of 16 stands for those from it on, and every other row's block is
// empty: nothing is sorted or counted beforehand.  More rows: tiles of 64, worked out for each window of 256.
//
// Bound by memory: x, A, B and the base are read once and out is written once, in pieces of 256 contiguous bytes and more, which fragments read from
// memory directly (16 rows x 64 bytes) are not: they took 46 + 71 us where
// staging takes 11.7 + 14.8 (1999 tokens, fp16, 4096 x 4096, rank 32; 8192 tokens, bf16, 4096 x 6144, rank 64: 83 + 222, 34 + 93).  Of those 34 the plan is 3,
// loads are 11, the products 5; the rest is LDS and its barriers, which more or deeper stages (28 - 33 for 31) did not change.
//
// u enters the second product with 22 bits or more: three bf16 terms (each the rest that the one before left), two fp16 ones behind a power of two per row
// (whatever u's size), or itself in fp32.
#include "seq_common.h"
#include <algorithm>

constexpr int WINDOW = 256, R_MAX = 128;

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
// COUNT elements p[0 .. n), zeros behind them (WHOLE: all of them or none, 16-byte aligned; otherwise whole pieces by loads of 16 bytes at any address,
// the last one's elements alone: element by element a rank of 100 took 55 us where this takes 32, 29 rows of K 1465 31 against 14)
template <typename P, bool WHOLE, typename F, int COUNT> __device__ __forceinline__ F load_some(const typename El<P>::type* p, int n) {
  typedef typename El<P>::type E;
  static_assert(sizeof(F) == COUNT * sizeof(E));
  u32x4 w[sizeof(F) / 16];
  if constexpr (WHOLE) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(F) / 16); ++i) w[i] = n > 0 ? reinterpret_cast<const u32x4*>(p)[i] : u32x4{0u, 0u, 0u, 0u};
    return __builtin_bit_cast(F, w);
  } else {
    E e[COUNT];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) e[i] = (E)0;
    if (n >= COUNT) __builtin_memcpy(e, p, sizeof e);
    else if (n > 0)
#pragma unroll
      for (int i = 0; i < COUNT - 1; ++i) if (i < n) e[i] = p[i];
    return __builtin_bit_cast(F, e);
  }
}

// Rows of one adapter, TILE at most, in LDS `rows` [TILE]; n 0: none.  All threads of 256 call what makes one.
struct Tile { int adapter, n; };

// up to WINDOW rows: block t stands for the rows of row t's adapter from t on, if t's place among them is a multiple of TILE
template <int TILE> __device__ __forceinline__ Tile tile_of_row(int t, int T, int S, const int* __restrict__ adapter, int* rows, int* waves) {
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
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

// More rows: plan, of each window: how many tiles; their adapters; their first places and sizes (first + 1024 n); the window's rows, those of a tile side by
// side.  An adapter is known by its first row, which a table of 512 places finds whatever the adapters' numbers are; a row's place among its adapter's is counted
// in its wave and over the waves in front, so that every workgroup that makes a window's plan makes the same.  Every one of the first product does, and one leaves it
// for the second (in a launch in front, adapter by adapter: 26.8 us where this takes 24.8 for 1999 rows of 4 adapters; 300 rows of 64 in any order 40 against 20).
constexpr int PLAN_TILE = 64, PLAN_INTS = 1 + 3 * WINDOW, PLACES = 2 * WINDOW;
struct PlanRoom { int key[PLACES], first[PLACES], count[WINDOW / 64][WINDOW], front[WINDOW], sums[WINDOW / 64]; };
__device__ __forceinline__ void plan_window(int* p, PlanRoom& room, int window, const int* __restrict__ adapter, int T, int S) {
  constexpr int WAVES = WINDOW / 64;
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6, t = window * WINDOW + i;
  const bool is = t < T;
  int id = is ? adapter[t] : -1;
  if (id < 0 || id >= S) id = -1;
  for (int k = i; k < PLACES; k += WINDOW) { room.key[k] = -2; room.first[k] = WINDOW; }
#pragma unroll
  for (int w = 0; w < WAVES; ++w) room.count[w][i] = 0;
  __syncthreads();
  int at = (int)(((unsigned)id * 2654435761u) >> 23);        // 0 .. 511
  if (is) {
    // (256 keys at most in 512 places: each finds its own or a free one)
    for (;;) {
      const int was = atomicCAS(&room.key[at], -2, id);
      if (was == -2 || was == id) break;
      at = (at + 1) % PLACES;
    }
    atomicMin(&room.first[at], i);
  }
  __syncthreads();
  const int own = is ? room.first[at] : WINDOW;
  unsigned long long same = __ballot(own == __builtin_amdgcn_readfirstlane(own));
  if (same != ~0ull) {
    unsigned lo = 0u, hi = 0u;
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      lo |= own == __builtin_amdgcn_readlane(own, k) ? 1u << k : 0u;
      hi |= own == __builtin_amdgcn_readlane(own, 32 + k) ? 1u << k : 0u;
    }
    same = lo | (unsigned long long)hi << 32;
  }
  int place = __popcll(same & ((1ull << lane) - 1ull));
  if (is && place == 0) room.count[wave][own] = __popcll(same);
  __syncthreads();
  if (is)
    for (int w = 0; w < wave; ++w) place += room.count[w][own];
  // of the adapter whose first row is row i
  int n = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) n += room.count[w][i];
  const int k = (n + PLAN_TILE - 1) / PLAN_TILE;
  int upto = n | k << 16;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(upto, o, 64); if (lane >= o) upto += v; }
  if (lane == 63) room.sums[wave] = upto;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) { if (w < wave) upto += room.sums[w]; all += room.sums[w]; }
  const int front = (upto & 0xffff) - n, tile = (upto >> 16) - k;
  room.front[i] = front;
  for (int e = 0; e < k; ++e) {
    p[1 + tile + e] = id;
    p[1 + WINDOW + tile + e] = front + e * PLAN_TILE + 1024 * min(PLAN_TILE, n - e * PLAN_TILE);
  }
  if (i == 0) p[0] = all >> 16;
  __syncthreads();
  if (is) p[1 + 2 * WINDOW + room.front[own] + place] = t;
}
__device__ __forceinline__ Tile tile_of_plan(const int* __restrict__ p, int k, int* rows) {
  const int said = p[1 + WINDOW + k], n = said / 1024, first = said % 1024;
  __syncthreads();                           // (the tile before this one may still be read)
  if ((int)threadIdx.x < n) rows[threadIdx.x] = p[1 + 2 * WINDOW + first + threadIdx.x];
  __syncthreads();
  return Tile{p[1 + k], n};
}

// Which block of the grid this one is.  Blocks go round the eight dies; with a plan each die takes neighbours, whose adapters its cache then holds
// (the second product of 8192 rows, 4096 x 6144, rank 64: 99 -> 92 us).
struct Place { int x, y; };
template <int TF> __device__ __forceinline__ Place place_of() {
  if constexpr (TF == 1) return Place{(int)blockIdx.x, (int)blockIdx.y};
  const unsigned all = gridDim.x * gridDim.y, l = blockIdx.y * gridDim.x + blockIdx.x, die = l % 8, at = die * (all / 8) + min(die, all % 8) + l / 8;
  return Place{(int)(at % gridDim.x), (int)(at / gridDim.x)};
}

// each tile that is this block's: block = row, or, with a plan (TF 4), every slots-th tile of a window
template <int TF, typename F>
__device__ __forceinline__ void each_tile(int block, const int* p, int slots, int T, int S, const int* adapter, int* rows, int* waves, F f) {
  if constexpr (TF == 1) {
    const Tile t = tile_of_row<16>(block, T, S, adapter, rows, waves);
    if (t.n > 0) f(t);
  } else {
    const int n = p[0];                      // p: its window's plan
    for (int k = block % slots; k < n; k += slots) f(tile_of_plan(p, k, rows));
  }
}

// ---- A x of a tile over K's k0 .. k1.  Stages of KB bytes of K, of 16 TF tokens and 16 RF ranks, go through registers to LDS, the next AHEAD stages' loads in flight
// behind this one's products.  TF 4: a wave 16 of the tokens; 1: a quarter of the stage's K, and wave 0 is left with the sums.
template <typename P, int RF, int TF, int KB> struct Down {
  typedef typename El<P>::type E;
  static constexpr int ES = sizeof(E), KC = KB / ES, VE = 16 / ES, LD = KB + 16, STEPS = KC / 32, PER_ROW = KB / 16, ROWS = 256 / PER_ROW;
  static constexpr int NX = 16 * TF / ROWS > 0 ? 16 * TF / ROWS : 1, NA = 16 * RF / ROWS > 0 ? 16 * RF / ROWS : 1, ROOM = (16 * TF + 16 * RF) * LD;
  static_assert(16 % ROWS == 0 && (TF == 4 || STEPS % 4 == 0) && (TF == 4 || 3 * RF * 64 * 16 <= ROOM));
};
template <typename P, bool WHOLE, int RF, int TF, int KB, int AHEAD>
__device__ __forceinline__ void down_sums(f32x4 (&acc)[RF], char* stage, const int* rows, Tile tile, int ra, const typename El<P>::type* __restrict__ x,
                                          const typename El<P>::type* __restrict__ ap, int K, int k0, int k1) {
  typedef Down<P, RF, TF, KB> D;
  constexpr int NX = D::NX, NA = D::NA, LD = D::LD, KC = D::KC, ROWS = D::ROWS, VE = D::VE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4, row = threadIdx.x / D::PER_ROW, piece = threadIdx.x % D::PER_ROW;
  u32x4 xs[AHEAD][NX], as[AHEAD][NA];
  // rows that are not there are zeros
  auto load = [&](u32x4 (&xv)[NX], u32x4 (&av)[NA], int k) __attribute__((always_inline)) {
    const int at = k + piece * VE, left = k1 - at;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int r = row + i * ROWS;
      const bool in = r < tile.n;
      xv[i] = load_some<P, WHOLE, u32x4, VE>(x + (long)rows[in ? r : 0] * K + at, in ? left : 0);
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int r = row + i * ROWS;
      av[i] = load_some<P, WHOLE, u32x4, VE>(ap + (long)(r < ra ? r : 0) * K + at, r < ra ? left : 0);
    }
  };
#pragma unroll
  for (int f = 0; f < RF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](u32x4 (&xv)[NX], u32x4 (&av)[NA], int k) __attribute__((always_inline)) {
    if (k > k0) __syncthreads();             // (the stage before this one has been read)
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<u32x4*>(stage + (row + i * ROWS) * LD + piece * 16) = xv[i];
#pragma unroll
    for (int i = 0; i < NA; ++i) *reinterpret_cast<u32x4*>(stage + (16 * TF + row + i * ROWS) * LD + piece * 16) = av[i];
    __syncthreads();
    if (k + AHEAD * KC < k1) load(xv, av, k + AHEAD * KC);
    // (All ranks and rows, zeros among them.  With `if (16 * f < ra)` in front of a product the compiler, in the kernels of 8 tiles of ranks, moves the last of its four sums
    // to another register one to three instructions behind it, where eight are wanted: 28 such moves, and none without it.)
    constexpr int MINE = TF == 4 ? D::STEPS : D::STEPS / 4;
#pragma unroll
    for (int s0 = 0; s0 < MINE; ++s0) {
      const int s = TF == 4 ? s0 : wave * MINE + s0;
      const char* at = stage + j * LD + (32 * s + 8 * g) * D::ES;
      const Frag<P> b = *reinterpret_cast<const Frag<P>*>(at + (TF == 4 ? wave * 16 * LD : 0));
#pragma unroll
      for (int f = 0; f < RF; ++f) acc[f] = mma<P>(*reinterpret_cast<const Frag<P>*>(at + (16 * TF + 16 * f) * LD), b, acc[f]);
    }
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) if (k0 + i * KC < k1 || i == 0) load(xs[i], as[i], k0 + i * KC);
  for (int k = k0; k < k1; k += AHEAD * KC)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) if (k + i * KC < k1) step(xs[i], as[i], k + i * KC);
  if constexpr (TF == 1) {
    __syncthreads();
    f32x4(*part)[RF][64] = reinterpret_cast<f32x4(*)[RF][64]>(stage);
    if (wave > 0)
#pragma unroll
      for (int f = 0; f < RF; ++f) part[wave - 1][f][lane] = acc[f];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int f = 0; f < RF; ++f) acc[f] = (acc[f] + part[0][f][lane]) + (part[1][f][lane] + part[2][f][lane]);
  }
}

// u[part][t][r].  grid (parts, rows or slots: the parts fastest, since blocks go round the eight dies and of a window's slots the first few alone have tiles)
template <typename P, bool WHOLE, int RF, int TF, int KB, int AHEAD>
__global__ __launch_bounds__(256) void adapter_down_kernel(float* __restrict__ u, const typename El<P>::type* __restrict__ x, const typename El<P>::type* __restrict__ a,
                                                           const int* __restrict__ adapter, const int* __restrict__ rank, int* __restrict__ plan, int slots,
                                                           int T, int K, int S, int R, int per) {
  __shared__ int rows[16 * TF], waves[5];
  __shared__ __attribute__((aligned(16))) char stage[Down<P, RF, TF, KB>::ROOM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  __shared__ int own_plan[TF == 1 ? 1 : PLAN_INTS];
  static_assert(TF == 1 || sizeof(PlanRoom) <= sizeof stage);
  const Place at = place_of<TF>();
  const int k0 = at.x * per, k1 = min(K, k0 + per);
  if constexpr (TF > 1) {
    plan_window(own_plan, *reinterpret_cast<PlanRoom*>(stage), at.y / slots, adapter, T, S);
    __syncthreads();
    if (at.x == 0 && at.y % slots == 0)
      for (int i = threadIdx.x; i < PLAN_INTS; i += 256) plan[(long)(at.y / slots) * PLAN_INTS + i] = own_plan[i];
  }
  each_tile<TF>(at.y, own_plan, slots, T, S, adapter, rows, waves, [&](const Tile tile) {
    if (tile.adapter < 0) return;
    const int ra = rank ? min(max(rank[tile.adapter], 0), R) : R;
    if (ra < 1) return;
    f32x4 acc[RF];
    down_sums<P, WHOLE, RF, TF, KB, AHEAD>(acc, stage, rows, tile, ra, x, a + (long)tile.adapter * R * K, K, k0, k1);
    const int own = TF == 4 ? wave * 16 + j : j;
    if ((TF == 1 && wave > 0) || own >= tile.n) return;
    float* to = u + ((long)at.x * T + rows[own]) * R;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
      const int r = 16 * f + 4 * g;
      if (r + 4 <= ra && R % 4 == 0) *reinterpret_cast<f32x4*>(to + r) = acc[f];
      else
#pragma unroll
        for (int e = 0; e < 4; ++e) if (r + e < ra) to[r + e] = acc[f][e];
    }
  });
}

// ---- out = base + B (scale u).  grid (pieces of N, rows or slots).  RF > 0: u is worked out here too, once for each piece of N, from an A that is small enough for that.
//  Stages of CS columns: a wave's share of them for all the tile's rows goes to LDS, from where whole rows
// leave, joined by the base (asked for in front of everything else).
template <typename P> struct Terms { static constexpr int N = 1; };
template <> struct Terms<BF16> { static constexpr int N = 3; };
template <> struct Terms<F16> { static constexpr int N = 2; };

template <typename P, bool WHOLE, bool QUADS, int RC, int TF, int RF, int KB>
__global__ __launch_bounds__(256) void adapter_up_kernel(float* out, const float* base, const float* __restrict__ u, const typename El<P>::type* __restrict__ b,
                                                         const int* __restrict__ adapter, const float* __restrict__ scale, const int* __restrict__ rank,
                                                         const int* __restrict__ plan, int slots, int T, int N, int S, int R, int parts, int columns,
                                                         const typename El<P>::type* __restrict__ x0, const typename El<P>::type* __restrict__ a, int K) {
  typedef typename El<P>::type E;
  constexpr bool BOTH = RF > 0;
  constexpr int UR = 16 * RF + 4;
  __shared__ __attribute__((aligned(16))) char stage[BOTH ? Down<P, BOTH ? RF : 1, 1, BOTH ? KB : 512>::ROOM : 16];
  __shared__ __attribute__((aligned(16))) float own_u[BOTH ? 16 : 1][UR];
  constexpr int NT = Terms<P>::N, CS = TF == 1 ? 256 : RC == 4 ? 64 : 128, LD = CS + 4, HF = CS / 64, NB = 16 * TF * CS / 1024, PER_ROW = CS / 4, ROWS = 256 / PER_ROW;
  __shared__ int rows[16 * TF], waves[5];
  __shared__ __attribute__((aligned(16))) E terms[NT][RC][TF][64][8];
  __shared__ __attribute__((aligned(16))) float sums[16 * TF][LD];
  __shared__ float power[16 * TF];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const int row = threadIdx.x / PER_ROW, quad = threadIdx.x % PER_ROW;
  const Place at = place_of<TF>();
  const int n0 = at.x * columns, n1 = min(N, n0 + columns);
  each_tile<TF>(at.y, TF == 1 ? plan : plan + (long)(at.y / slots) * PLAN_INTS, slots, T, S, adapter, rows, waves, [&](const Tile tile) {
    const int ra = tile.adapter < 0 ? 0 : rank ? min(max(rank[tile.adapter], 0), R) : R;
    if (ra < 1 && out == base) return;
    f32x4 x[NB];
    Frag<P> w[HF][RC];
    auto ask = [&](int n) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = row + i * ROWS, col = n + 4 * quad;
        const float* o = base + (long)rows[r < tile.n ? r : 0] * N + col;
        x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (r < tile.n) {
          if (QUADS) { if (col < n1) x[i] = *reinterpret_cast<const f32x4*>(o); }
          else if (col + 3 < n1) __builtin_memcpy(&x[i], o, sizeof x[i]);
          else
#pragma unroll
            for (int e = 0; e < 3; ++e) if (col + e < n1) x[i][e] = o[e];
        }
      }
      if (ra < 1) return;
#pragma unroll
      for (int h = 0; h < HF; ++h) {
        const E* br = b + ((long)tile.adapter * N + min(n + 16 * (wave * HF + h) + j, N - 1)) * R;
#pragma unroll
        for (int c = 0; c < RC; ++c) w[h][c] = load_some<P, WHOLE, Frag<P>, 8>(br + 32 * c + 8 * g, (WHOLE ? (ra + 7) & ~7 : ra) - 32 * c - 8 * g);
      }
    };
    ask(n0);
    if constexpr (BOTH)
      if (ra > 0) {
        f32x4 acc[BOTH ? RF : 1];
        down_sums<P, WHOLE, BOTH ? RF : 1, 1, BOTH ? KB : 512, 1>(acc, stage, rows, tile, ra, x0, a + (long)tile.adapter * R * K, K, 0, K);
        if (wave == 0)
#pragma unroll
          for (int f = 0; f < RF; ++f) *reinterpret_cast<f32x4*>(&own_u[j][16 * f + 4 * g]) = acc[f];
        __syncthreads();
      }
    if (ra > 0) {
      const float sc = scale ? scale[tile.adapter] : 1.f;
      // a row's terms by four lanes (64 rows), or one of 16 rows by sixteen: lane j, g of the fragments is row j, elements 32 c + 8 g ..
      const int i = threadIdx.x >> 2, q = threadIdx.x & 3;
      if (i < 16 * TF) {
        float v[RC][8], most = 0.f;
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
        if (BOTH) {
#pragma unroll
          for (int c = 0; c < RC; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int r = 32 * c + 8 * q + e;
              if (r < ra && r < 16 * RF) v[c][e] = own_u[i][r];
            }
        } else if (i < tile.n) {
          const float* ur = u + (long)rows[i] * R;
#pragma unroll 4
          for (int p = 0; p < parts; ++p, ur += (long)T * R)
#pragma unroll
            for (int c = 0; c < RC; ++c) {
              const int r = 32 * c + 8 * q;
              if (r + 8 <= ra && R % 4 == 0) {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(ur + r), hi = *reinterpret_cast<const f32x4*>(ur + r + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { v[c][e] += lo[e]; v[c][4 + e] += hi[e]; }
              } else if (r + 8 <= ra) {
                float w[8];
                __builtin_memcpy(w, ur + r, sizeof w);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] += w[e];
              } else
#pragma unroll
                for (int e = 0; e < 7; ++e) if (r + e < ra) v[c][e] += ur[r + e];
            }
        }
#pragma unroll
        for (int c = 0; c < RC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[c][e] *= sc;
            most = fmaxf(most, fabsf(v[c][e]));
          }
        if constexpr (NT == 2) {             // fp16: the row's largest between 1 and 2
          most = fmaxf(most, __shfl_xor(most, 1, 64));
          most = fmaxf(most, __shfl_xor(most, 2, 64));
          const int e = most > 0.f && most < INFINITY ? max(ilogbf(most), -126) : 0;
          if (q == 0) power[i] = ldexpf(1.f, e);
#pragma unroll
          for (int c = 0; c < RC; ++c)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[c][k] = ldexpf(v[c][k], -e);
        }
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          E t[NT][8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (NT == 1) t[0][e] = v[c][e];
            else {
              t[0][e] = P::from_f(v[c][e]);
              float rest = v[c][e] - P::to_f(t[0][e]);
              if (!(fabsf(rest) < INFINITY)) rest = 0.f;
              if constexpr (NT == 2) t[1][e] = P::from_f(rest * 2048.f);
              else {
                t[1][e] = P::from_f(rest);
                t[2][e] = P::from_f(rest - P::to_f(t[1][e]));
              }
            }
          }
#pragma unroll
          for (int k = 0; k < NT; ++k) __builtin_memcpy(&terms[k][c][i >> 4][q * 16 + (i & 15)][0], t[k], sizeof t[k]);
        }
      }
      __syncthreads();
    }
    const int frags = TF == 1 ? 1 : (tile.n + 15) >> 4;
    for (int n = n0; n < n1; n += CS) {
      if (ra > 0) {
        if (WHOLE && (ra & 7)) {             // what stands behind the rank is nobody's
#pragma unroll
          for (int h = 0; h < HF; ++h)
#pragma unroll
            for (int c = 0; c < RC; ++c) {
              E e[8];
              __builtin_memcpy(e, &w[h][c], sizeof e);
#pragma unroll
              for (int k = 0; k < 8; ++k) if (32 * c + 8 * g + k >= ra) e[k] = (E)0;
              __builtin_memcpy(&w[h][c], e, sizeof e);
            }
        }
#pragma unroll
        for (int f = 0; f < TF; ++f) {
          if (f >= frags) break;
          f32x4 acc[HF], low[HF];
#pragma unroll
          for (int h = 0; h < HF; ++h) acc[h] = low[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < RC; ++c) {
            const Frag<P>* t = reinterpret_cast<const Frag<P>*>(&terms[0][c][f][lane][0]);
            constexpr long next = (long)RC * TF * 64;
            const Frag<P> t0 = t[0];
#pragma unroll
            for (int h = 0; h < HF; ++h) acc[h] = mma<P>(w[h][c], t0, acc[h]);
#pragma unroll
            for (int k = NT - 1; k > 0; --k) {
              const Frag<P> tk = t[k * next];
#pragma unroll
              for (int h = 0; h < HF; ++h) low[h] = mma<P>(w[h][c], tk, low[h]);
            }
          }
#pragma unroll
          for (int h = 0; h < HF; ++h) {
            if constexpr (NT == 3) acc[h] += low[h];
            if constexpr (NT == 2) acc[h] = (acc[h] + low[h] * (1.f / 2048.f)) * power[f * 16 + j];
            *reinterpret_cast<f32x4*>(&sums[f * 16 + j][16 * (wave * HF + h) + 4 * g]) = acc[h];
          }
        }
        __syncthreads();
      }
      f32x4 y[NB];
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = row + i * ROWS;
        y[i] = x[i];
        if (ra > 0 && r < tile.n) y[i] += *reinterpret_cast<const f32x4*>(&sums[r][4 * quad]);
      }
      if (n + CS < n1) ask(n + CS);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int r = row + i * ROWS, col = n + 4 * quad;
        if (r >= tile.n) continue;
        float* o = out + (long)rows[r] * N + col;
        if (QUADS) { if (col < n1) __builtin_nontemporal_store(y[i], reinterpret_cast<f32x4*>(o)); }
        else if (col + 3 < n1) __builtin_memcpy(o, &y[i], sizeof y[i]);
        else
#pragma unroll
          for (int e = 0; e < 3; ++e) if (col + e < n1) o[e] = y[i][e];
      }
      __syncthreads();                       // (the next stage's sums, the next tile's terms)
    }
  });
}

// Both products in one launch: A is read again for each piece of N, 64 KB of it (128 in fp32) by a workgroup at most, in 1 to 2 us, which is what a launch costs.
// One token, bf16, 2048 x 2560, rank 8: 3.1 + 4.9 us by two launches, 6.8 by one; the whole call
// 16.6 and 12.6.
static bool adapter_fused(int T, int K, int R) { return T <= 64 && R <= 64 && (long)R * K <= 32768; }
// pieces of K: more workgroups, and as many sums that the second product reads (1999 rows, 4096 x 4096, rank 32: 8 pieces 25.9 us, 4 24.9)
static int adapter_parts(int T, int K) { return std::max(1, std::min(T > 4096 ? 2 : T > 1024 ? 4 : 8, (K + 511) / 512)); }
static long plan_ints(int T) { return T > WINDOW ? (long)((T + WINDOW - 1) / WINDOW) * PLAN_INTS : 0; }

extern "C" long umb_seq_adapters_floats(int T, int K, int R) {
  return T < 1 || T > (1 << 20) || K < 1 || R < 1 || R > R_MAX || adapter_fused(T, K, R) ? 0 : (((long)adapter_parts(T, K) * T * R + 3) & ~3L) + plan_ints(T);
}

template <typename P, bool WHOLE, int TF>
static int adapters_launch(float* out, const float* base, const void* x, const void* a, const void* b, const int* adapter, const float* scale, const int* rank, int T,
                           int N, int K, int S, int R, bool quads, float* u, hipStream_t st) {
  typedef typename El<P>::type E;
  const int parts = adapter_parts(T, K), per = (((K + 31) / 32 + parts - 1) / parts) * 32;
  int* plan = nullptr;
  int slots = 1, blocks = T, tiles = T;
  if (TF > 1) {
    plan = reinterpret_cast<int*>(u + (((long)parts * T * R + 3) & ~3L));
    const int windows = (T + WINDOW - 1) / WINDOW;
    // A window of few adapters has some five tiles; of many one each and more.  Blocks without a tile cost the making of a plan, blocks of several take them in turn (us:
    // 1000 rows of 8 adapters in any order 8 slots 20, 16 29; of 64 8 slots 77, 16 68, 32 61; 300 rows of 64 58, 33, 20; beyond 2048 rows all blocks are busy).
    slots = T > 2048 || S <= 8 ? 8 : 32;
    blocks = windows * slots;
    tiles = (T + PLAN_TILE - 1) / PLAN_TILE;
  }
  int columns = 256;
  while (columns < 1024 && (long)tiles * (N / (2 * columns)) >= 1024) columns *= 2;
  const int pieces = (N + columns - 1) / columns;
#define UP(RC, RF, KB)                                                                                                                                         \
  if (quads) hipLaunchKernelGGL((adapter_up_kernel<P, WHOLE, true, RC, TF, RF, KB>), dim3(pieces, blocks), dim3(256), 0, st, out, base, u, (const E*)b, adapter, scale, \
                                rank, plan, slots, T, N, S, R, parts, columns, (const E*)x, (const E*)a, K);                                                   \
  else hipLaunchKernelGGL((adapter_up_kernel<P, WHOLE, false, RC, TF, RF, KB>), dim3(pieces, blocks), dim3(256), 0, st, out, base, u, (const E*)b, adapter, scale, \
                          rank, plan, slots, T, N, S, R, parts, columns, (const E*)x, (const E*)a, K)
  if constexpr (TF == 1)
    if (adapter_fused(T, K, R)) {
      if (R <= 16) { UP(1, 1, 1024); }
      else if (R <= 32) { UP(1, 2, 512); }
      else { UP(2, 4, 512); }
      UMB_LAUNCH_CHECK();
      return UMB_OK;
    }
#define DOWN(RF, KB, AHEAD)                                                                                                                                       \
  hipLaunchKernelGGL((adapter_down_kernel<P, WHOLE, RF, TF, KB, AHEAD>), dim3(parts, blocks), dim3(256), 0, st, u, (const E*)x, (const E*)a, adapter, rank, plan, slots, \
                     T, K, S, R, per)
  // bytes of K a stage, and stages in flight
  if (R <= 16) DOWN(1, (TF == 1 ? 1024 : 512), (TF == 1 ? 1 : 2));
  else if (R <= 32) DOWN(2, 512, (TF == 1 ? 1 : 2));
  else if (R <= 64) DOWN(4, (TF == 1 ? 512 : 256), (TF == 1 ? 1 : 2));
  else DOWN(8, (TF == 1 && !std::is_same_v<P, F32> ? 256 : TF == 1 ? 512 : 256), 1);
#undef DOWN
  UMB_LAUNCH_CHECK();
  if (R <= 32) { UP(1, 0, 0); }
  else if (R <= 64) { UP(2, 0, 0); }
  else { UP(4, 0, 0); }
#undef UP
  UMB_LAUNCH_CHECK();
  return UMB_OK;
}

static bool overlap(const void* p, long n, const void* q, long m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return a < b + m && b < a + n;
}

extern "C" int umb_seq_adapters(float* out, const float* base, const void* x, const void* a, const void* b, const int* adapter, const float* scale, const int* rank,
                                int T, int N, int K, int S, int R, float* scratch, long scratch_floats, int dtype, hipStream_t st) {
  if (!out || !base || !x || !a || !b || !adapter || T < 1 || T > (1 << 20) || N < 1 || K < 1 || S < 1 || R < 1 || R > R_MAX || N > (1 << 24) || K > (1 << 24) ||
      (umb_seq_adapters_floats(T, K, R) > 0 && (!scratch || (uintptr_t)scratch % 16 || scratch_floats < umb_seq_adapters_floats(T, K, R))))
    return UMB_EINVAL;
  // (workgroups read x, a and b while others write; a base that is out itself is read by who writes there)
  const long bytes = 4L * T * N, es = (long)seq_elem_bytes(dtype);
  if (overlap(out, bytes, x, es * T * K) || overlap(out, bytes, a, es * S * R * K) || overlap(out, bytes, b, es * S * R * N) || (out != base && overlap(out, bytes, base, bytes)))
    return UMB_EINVAL;
  const bool quads = N % 4 == 0 && ((uintptr_t)out | (uintptr_t)base) % 16 == 0;
  const bool whole = K % 8 == 0 && R % 8 == 0 && ((uintptr_t)x | (uintptr_t)a | (uintptr_t)b) % 16 == 0;
  DISPATCH_SEQ_DTYPE(dtype, {
    auto launch = T <= WINDOW ? (whole ? adapters_launch<P, true, 1> : adapters_launch<P, false, 1>) : (whole ? adapters_launch<P, true, 4> : adapters_launch<P, false, 4>);
    return launch(out, base, x, a, b, adapter, scale, rank, T, N, K, S, R, quads, scratch, st);
  })
}
