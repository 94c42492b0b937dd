// The next token of every row of logits, each row with its own temperature, top-k, top-p and min-p, from a given random number.
//
// Order: value descending, index ascending.  w = exp((x - max) / T).  Each of the three filters keeps a prefix of that order: the first k; those
// in front of which less than p of the first k's mass stands; those with w >= m.  The shortest prefix is kept, and of it the first token whose mass,
// with all in front of it, exceeds u times the kept mass is drawn.
//
// Weights are 64-bit floats, and a border between two tokens falls where 64-bit sums put it.  (In 32 bits a flat row of 128256 values has thousands of borders that
// the sum's order moves.)  What is summed in no fixed order is summed as whole numbers.  Sums that are no better than some 1e-12 of the row (bins) or lack its
// faintest tokens say where a border may be, never where it is: where the token drawn is not the same for all that they may stand for, the row is searched whole.
//
// Nothing is sorted but what stands next to a border.  Three launches (two for rows of one slice):
//   slices   a row in slices, each read once into registers: its largest, and counts and masses of bins T / 32 wide, 1024 below the largest (a token
//            further down weighs less than 2^-46, all of them together up to 7e-9).  Bins lie on one lattice, floor(32 x / T), and masses are relative to their bin's
//            middle, so that slices' add up as whole numbers, count and mass in one 64-bit atomic
//   collect  the row's bins, summed up from the top, say which bins hold the k-th value, the ends of top-p and min-p and the token drawn (intervals, since
//            the mass behind p and u is known to a bin only, and the bins' masses to BIN_OFF); their tokens are collected.  A row of a small k has counts alone, and
//            all tokens down to the k-th value's bin are collected
//   resolve  a row's collected tokens by one workgroup: where they are many, bins again, up to 256 in each bin; then in order: the exact ends, then the draw, each by
//            the least and the most that the sums in front may be
// us (slices, collect, resolve): a row of 32000 3.8, 8, 10.4; 8 of 128256 5.2, 11.2, 10.4; 48 of 151936 12.6, 19.8, 17; 256 of 128256 37.7, 29.5, 14.6.
// Bound by the logits where rows are many: the first launch reads them from memory, the second once more, from the cache behind it; by launches and barriers where
// they are few.
// Rows of up to SMALL_V values are taken whole by the last launch alone (1000 values 15 - 17 us, 1500 20 against 16 - 18 by two).
// Searched eight bits of the key at a time, by one workgroup, four passes a border: a row with more than CAP tokens next to a border, or a quarter of a slice (equal
// logits by the thousand), or whose border the bins' masses leave open (by their bounds one of 500 000 nearly flat rows of 151936 with a p; two equal logits that p
// halves).  ms: 128256 equal values 1.1, 2.0 with a p, 2.9 with a k too; 48 rows of as many rounded to whole numbers, with a p, 1.25.
#include "seq_common.h"
#include <algorithm>

constexpr int SAMPLE_VMAX = 1 << 19;         // a Mass holds so many
constexpr double MAGIC = 4503599627370496.0; // 2^52: added to a number below 2^51, it leaves the nearest whole number in the low bits

// NaN counts as -inf; larger values have larger keys
__device__ __forceinline__ unsigned key_of(float x) {
  unsigned u = __float_as_uint(x == x ? x : -INFINITY);
  if (u == 0x80000000u) u = 0u;              // -0 is 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float of_key(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
constexpr unsigned KEY_NONE = 0x007fffffu;   // of -inf

// a token's weight, and its mass in whole numbers
__device__ __forceinline__ double weight_of(unsigned key, float top, double t) {
  const float x = of_key(key);
  return key <= KEY_NONE ? 0.0 : x == top ? 1.0 : top < INFINITY ? exp(((double)x - (double)top) / t) : 0.0;
}
// A sum of weights of at most 1 in whole numbers, the same in any order: of 2^-40, and of what each weight's rounding to those leaves, of 2^-84.  2^19 of them
// are good to 2^-66.  (In 2^-44 alone, 128255 tokens of 2e-9 beside one of 1 were 1e-9 off together, and every third draw among them the token beside the right one.)
struct Mass {
  unsigned long long hi;
  long long lo;
  __device__ __forceinline__ double value() const { return (double)hi * (1.0 / 1099511627776.0) + (double)lo * (1.0 / 19342813113834066795298816.0); }
  __device__ __forceinline__ Mass operator+(const Mass& o) const { return Mass{hi + o.hi, lo + o.lo}; }
  __device__ __forceinline__ Mass operator-(const Mass& o) const { return Mass{hi - o.hi, lo - o.lo}; }
  __device__ __forceinline__ Mass operator*(int n) const { return Mass{hi * (unsigned long long)n, lo * n}; }
};
__device__ __forceinline__ Mass mass_of(double w) {
  const double ONE = 1099511627776.0, REST = 17592186044416.0, HALF = 1.5 * MAGIC;
  const double h = fma(w, ONE, MAGIC), l = fma(fma(w, ONE, MAGIC - h), REST, HALF);            // (both differences are exact)
  return Mass{(unsigned long long)__double_as_longlong(h) & 0xfffffffffffffull, __double_as_longlong(l) - __double_as_longlong(HALF)};
}

struct RowSettings { double t, p, m, u; int k; bool greedy; };
__device__ __forceinline__ RowSettings row_settings(int row, int V, const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                                                    const float* uniforms) {
  RowSettings s;
  const float t = temperature ? temperature[row] : 1.f, p = top_p ? top_p[row] : 1.f, m = min_p ? min_p[row] : 0.f, u = uniforms[row];
  const int k = top_k ? top_k[row] : 0;
  s.greedy = !(t > 0.f);
  s.t = t;
  s.k = k > 0 && k < V ? k : V;
  s.p = p;
  s.m = m == m ? m : 0.f;
  s.u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
  return s;
}

constexpr int ST = 1024;
struct Pick {                                // the element that a search ended at: its key, its place among its equals, what stands in front of those
  unsigned key;
  int tie, count;
  Mass mass;
};
// LDS of the searches; sums of a digit's masses, and of everything (0) and of what min-p keeps (1)
struct SlowRoom {
  unsigned cnt[256];
  unsigned long long hi[256], lo[256], wide[6];
  Mass front;
  int digit, count, tie;
};

// The first element, in order, at which what has come up to and with it reaches a goal: BY_COUNT the goal-th element; otherwise the first whose
// mass up to and with it is at least (OVER: more than) `goal`.  There is one by the caller's choice of the goal, or the last element is taken.
// Four passes over the row, eight bits of the key each.
enum { BY_COUNT, AT_LEAST, OVER };
template <int HOW>
__device__ Pick find_in_row(const float* __restrict__ row, int V, float top, double t, double goal, SlowRoom& room) {
  Pick got{0u, 0, 0, Mass{0ull, 0ll}};
  unsigned mask = 0u;
  auto reached = [&](double n, double q) { return HOW == BY_COUNT ? n >= goal : HOW == AT_LEAST ? q >= goal : q > goal; };
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) { room.cnt[threadIdx.x] = 0u; room.hi[threadIdx.x] = room.lo[threadIdx.x] = 0ull; }
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += ST) {
      const unsigned k = key_of(row[i]);
      if ((k & mask) == got.key && k > KEY_NONE) {
        const int d = (k >> shift) & 255;
        atomicAdd(&room.cnt[d], 1u);
        const Mass q = mass_of(weight_of(k, top, t));
        if (q.hi) atomicAdd(&room.hi[d], q.hi);
        if (q.lo) atomicAdd(&room.lo[d], (unsigned long long)q.lo);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int n = got.count, d = 255, last = -1;
      Mass q = got.mass;
      auto of = [&](int i) { return Mass{room.hi[i], (long long)room.lo[i]}; };
      for (; d >= 0; --d) {
        if (!room.cnt[d]) continue;
        if (reached((double)(n + room.cnt[d]), (q + of(d)).value())) break;
        last = d;
        n += room.cnt[d];
        q = q + of(d);
      }
      if (d < 0) { d = last < 0 ? 0 : last; n -= room.cnt[d]; q = q - of(d); }
      room.digit = d;
      room.count = n;
      room.front = q;
    }
    __syncthreads();
    got.key |= (unsigned)room.digit << shift;
    got.count = room.count;
    got.mass = room.front;
    mask |= 255u << shift;
    if (shift == 0) {                        // equals, in the order of their indices
      const int n = room.cnt[room.digit];
      const Mass q = mass_of(weight_of(got.key, top, t));
      if (threadIdx.x == 0) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (reached((double)(got.count + mid + 1), (got.mass + q * (mid + 1)).value())) hi = mid;
          else lo = mid + 1;
        }
        room.tie = lo;
      }
      __syncthreads();
      got.tie = room.tie;
    }
  }
  __syncthreads();
  return got;
}

// the whole of a row by one workgroup, some eleven passes over it
__device__ __attribute__((noinline)) void sample_slow(int r, int* __restrict__ tokens, float* __restrict__ probs, const float* __restrict__ row, int V, RowSettings s,
                                                      float top, SlowRoom& room) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned long long* wide = room.wide;
  // everything's and min-p's counts and masses
  __syncthreads();
  if (tid < 6) wide[tid] = 0ull;
  __syncthreads();
  unsigned long long n_all = 0, n_min = 0;
  Mass q_all{0ull, 0ll}, q_min{0ull, 0ll};
  for (int i = tid; i < V; i += ST) {
    const unsigned k = key_of(row[i]);
    const double w = weight_of(k, top, s.t);
    const Mass q = mass_of(w);
    if (k > KEY_NONE) { ++n_all; q_all = q_all + q; if (w >= s.m) { ++n_min; q_min = q_min + q; } }
  }
  atomicAdd(&wide[0], n_all);
  atomicAdd(&wide[1], q_all.hi);
  atomicAdd(&wide[2], (unsigned long long)q_all.lo);
  atomicAdd(&wide[3], n_min);
  atomicAdd(&wide[4], q_min.hi);
  atomicAdd(&wide[5], (unsigned long long)q_min.lo);
  __syncthreads();
  n_all = wide[0];
  q_all = Mass{wide[1], (long long)wide[2]};
  long n = (long)wide[3];
  Mass q{wide[4], (long long)wide[5]};
  if (n < 1) { n = 1; q = mass_of(1.0); }
  Mass q_k = q_all;
  if ((unsigned long long)s.k < n_all) {
    const Pick e = find_in_row<BY_COUNT>(row, V, top, s.t, (double)s.k, room);
    q_k = e.mass + mass_of(weight_of(e.key, top, s.t)) * (e.tie + 1);
    if (s.k < n) { n = s.k; q = q_k; }
  }
  if (s.p < 1.0) {
    const Pick e = find_in_row<AT_LEAST>(row, V, top, s.t, fmax(s.p, 0.0) * q_k.value(), room);
    if (e.count + e.tie + 1 < n) { n = e.count + e.tie + 1; q = e.mass + mass_of(weight_of(e.key, top, s.t)) * (e.tie + 1); }
  }
  const double mass = q.value();
  const Pick e = find_in_row<OVER>(row, V, top, s.t, s.u * mass, room);
  // the tie-th of the values equal to e's, by index
  int seen = 0;
  for (int i0 = 0; i0 < V; i0 += ST) {
    const int i = i0 + tid;
    const bool is = i < V && key_of(row[i]) == e.key;
    const unsigned long long bal = __ballot(is);
    __syncthreads();
    if (lane == 0) room.cnt[wave] = __popcll(bal);
    __syncthreads();
    int before = seen, all = seen;
    for (int w = 0; w < ST / 64; ++w) { if (w < wave) before += room.cnt[w]; all += room.cnt[w]; }
    if (is && before + __popcll(bal & ((1ull << lane) - 1ull)) == e.tie) {
      tokens[r] = i;
      if (probs) probs[r] = (float)(weight_of(e.key, top, s.t) / mass);
    }
    seen = all;
    if (seen > e.tie) break;
  }
}

// ------------------------------------------------------------------ bins
constexpr int BINS = 1024, SMALL_V = 1024, CAP = 2048, K_COUNT = 1024, P_MAX = 64, FEW = 128;
constexpr double PER_T = 32.0, LATTICE = 1099511627776.0;         // bins a T; beyond 2^40 neighbouring floats are 2^16 bins apart and more
// A bin's masses: 48 bits for 2^15 of them, 16 above for their number.  What each has above a bin's least weight, at most 0.0313 of its middle's, in 2^-37 of that:
// half a step, 3.7e-12 of the least weight, and the polynomial's 5e-13 are BIN_OFF.  (The weights themselves would be held in 2^-32: 1.2e-10.)
constexpr double BIN_ONE = 137438953472.0, BIN_LEAST = 0.9844964370058922, BIN_OFF = 4.5e-12;
constexpr double FAINT = 1.4e-14;                                // more than a token below the bins weighs: e^(-1023 / 32)
// resolve's bins: in 2^-46 of a power of two that a bin's weights reach to half of at least, so that 2^17 of them are good to 2^-46 of what they weigh, however far down
constexpr int FINE_BITS = 46;
__device__ __forceinline__ int fine_shift(int bin) { return (max(bin - 1, 0) * 47273) >> 20; }            // log2 of e^((bin - 1) / 32), rounded down
__device__ __forceinline__ double power_of_two(int e) { return __longlong_as_double((long long)(1023 + e) << 52); }

// e^((f - 1/2) / 32) - BIN_LEAST of 0 <= f < 1 in whole numbers of 1 / BIN_ONE: the polynomial of degree 4 that meets the first in the five Chebyshev points, good to 5e-13 of it,
// without its constant, rounded by the addition of 2^52.  The coefficients are held in registers: as literals each costs two moves an element.
struct BinExp {
  double c[5];
  __device__ __forceinline__ BinExp() {
    const double k[5] = {0.0, 0.03076551363223118, 0.0004807113442785956, 5.006866963355461e-06, 3.97368340715931e-08};
#pragma unroll
    for (int i = 0; i < 5; ++i) c[i] = k[i] * BIN_ONE + (i == 0 ? MAGIC : 0.0);
#pragma unroll
    for (int i = 0; i < 5; ++i) asm volatile("" : "+v"(c[i]));
  }
  __device__ __forceinline__ unsigned long long operator()(double f) const {
    double p = c[4];
#pragma unroll
    for (int i = 3; i >= 0; --i) p = fma(p, f, c[i]);
    return (unsigned long long)__double_as_longlong(p) & 0x7ffffffffffffull;
  }
};
// e^d of -40 < d <= 0.1 to some 2e-15 of it (a power of two times Taylor's sum to the 12th power of a rest of at most 0.347), 0 below
__device__ __forceinline__ double exp_down(double d) {
  if (!(d > -40.0)) return 0.0;
  const double n = rint(d * 1.4426950408889634074);
  const double r = fma(-n, 2.3190468138462996e-17, fma(-n, 0.69314718055994530942, d));
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return p * __longlong_as_double((long long)(1023 + (int)n) << 52);
}
// a value's weight beside the row's largest; values of an infinite one's row weigh nothing but for the infinite ones
__device__ __forceinline__ double weight_at(float x, float top, double inv_t) {
  return x == top ? 1.0 : top < INFINITY ? exp_down(((double)x - (double)top) * inv_t) : 0.0;
}
__device__ __forceinline__ unsigned long long fine_of(double w, int shift) {
  return (unsigned long long)__double_as_longlong(fma(w, power_of_two(FINE_BITS + shift), MAGIC)) & 0xfffffffffffffull;
}
// whether a value weighs anything beside `top`, as far as infinities and the lattice's end tell
__device__ __forceinline__ bool counts(float x, float top, double per) {
  return x > -INFINITY && (x == top || (top < INFINITY && fabs((double)x * per) < LATTICE));
}
// where a value lies on the lattice; monotone in x, whatever T is
__device__ __forceinline__ double line_of(float x, double per) { return x < INFINITY ? fmin(fmax((double)x * per, -LATTICE), LATTICE) : LATTICE; }

// the least float x of which x per >= goal, a whole number
__device__ __forceinline__ float least_at(double goal, double per) {
  const double v = goal / per;
  if (v >= 3.4028235e38) return INFINITY;
  unsigned k = key_of(v > -3.4028235e38 ? (float)v : -3.402823466e38f);
  for (int i = 0; i < 4 && (double)of_key(k) * per < goal; ++i) ++k;
  for (int i = 0; i < 4 && k > KEY_NONE + 1 && (double)of_key(k - 1) * per >= goal; ++i) --k;
  return of_key(k);
}

struct SliceHead { float top; int at, pad[2]; };
// how far off a bin's mass may be, of itself: and where a value lies on the lattice, of some |line| / T, is known to 2^-53 of that
__device__ __forceinline__ double off_of(double line) { return BIN_OFF + 1e-17 * (fabs(line) + BINS); }
// beside an infinite value, or one beyond the lattice, only its equals count
__device__ __forceinline__ bool is_flat(float top, double per) { return top == INFINITY || !(fabs((double)top * per) < LATTICE); }
// what collect leaves for resolve; `mass` and `count`: in front of each bin
struct RowSaid {
  double all;
  int count_all, slots, k_binds, k0, m0, m1; // k_binds 2: the k-th is the last of bin k0
  int p_binds, m_binds, whole, pad;          // whole: everything down to the last collected token is collected
};
struct RowSums {
  double mass[BINS];
  int count[BINS];
  short slot[BINS];                          // its place among the bins that are collected, -1: it is not
  RowSaid said;
};
static_assert(sizeof(RowSums) % 16 == 0 && sizeof(RowSaid) % 16 == 0);
// How a row is cut: slices of `slice` values (P), which the first launch counts; chunks of `chunk` values, every Q-th of which the second launch's block q looks
// through, with room for a quarter of them.  Few rows: as many workgroups as there are pieces of 8192; many: larger pieces, and as many workgroups as stay
// resident, since each adds up its row's bins first.  Rows of one slice take the second launch alone, which makes their bins (us: 8192 values 19.5 -> 16, 256 rows
// of 12000 32 -> 22; up to 32768 where the rows keep the chip busy: 32000 values 64 rows 27.6 either way, 256 rows 39 -> 29.5, one 20.4 -> 20.7).
struct Cut { int slice, P, chunk, Q, cap; };
static Cut cut_of(int rows, int V) {
  const bool few = (long)rows * ((V + 8191) / 8192) <= 512;
  Cut c;
  c.slice = c.chunk = V <= 8192 ? 8192 : V <= 16384 ? 16384 : V <= 32768 && rows > 64 ? 32768 : few ? 8192 : 16384;
  c.P = (V + c.slice - 1) / c.slice;
  c.Q = few ? c.P : std::max(1, std::min(c.P, 512 / rows));
  c.cap = (c.P + c.Q - 1) / c.Q * (c.chunk / 4);
  return c;
}
struct Scratch { SliceHead* heads; unsigned long long *bins, *found; int* taken; RowSums* sums; };
__host__ __device__ __forceinline__ long row_bytes(const Cut& c) { return (long)c.P * (16 + BINS * 8) + (long)c.Q * c.cap * 8 + P_MAX * 4 + (long)sizeof(RowSums); }
__device__ __forceinline__ Scratch scratch_of(char* base, int row, const Cut& c) {
  char* p = base + row * row_bytes(c);
  Scratch s;
  s.bins = reinterpret_cast<unsigned long long*>(p);
  s.found = s.bins + (long)c.P * BINS;
  s.sums = reinterpret_cast<RowSums*>(s.found + (long)c.Q * c.cap);
  s.heads = reinterpret_cast<SliceHead*>(s.sums + 1);
  s.taken = reinterpret_cast<int*>(s.heads + c.P);
  return s;
}

// a slice's values in registers: element e of thread t is value index_of(e); -inf behind the row's end and for NaN
template <int NT, int NE, bool VEC> __device__ __forceinline__ int index_of(int base, int e) {
  return VEC ? base + ((e >> 2) * NT + (int)threadIdx.x) * 4 + (e & 3) : base + e * NT + (int)threadIdx.x;
}
template <int NT, int NE, bool VEC> __device__ __forceinline__ void load_slice(float (&x)[NE], const float* __restrict__ row, int base, int V) {
  if constexpr (VEC) {
#pragma unroll
    for (int e = 0; e < NE; e += 4) {
      const int i = index_of<NT, NE, VEC>(base, e);
      f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (i + 3 < V) v = *reinterpret_cast<const f32x4*>(row + i);
      else
#pragma unroll
        for (int k = 0; k < 3; ++k) if (i + k < V) v[k] = row[i + k];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[e + k] = v[k];
    }
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int i = index_of<NT, NE, VEC>(base, e);
      x[e] = i < V ? row[i] : -INFINITY;
    }
  }
#pragma unroll
  for (int e = 0; e < NE; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
}

// counts and masses of a slice's values, whose largest is `top`
template <int NE> __device__ __forceinline__ void bin_slice(const float (&x)[NE], unsigned long long* bins, float top, double per, int k) {
  const double first = floor(line_of(top, per));
  if (top == INFINITY || !(fabs((double)top * per) < LATTICE)) {   // its equals alone count
#pragma unroll
    for (int e = 0; e < NE; ++e) if (x[e] == top) atomicAdd(bins, 1ull << 48);
  } else if (k >= 1 && k <= K_COUNT) {
    // (-inf, and what the lattice does not reach, are far below)
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const double j = first - floor((double)x[e] * per);
      const int at = (int)j;
      if (j < BINS) atomicAdd(reinterpret_cast<unsigned*>(bins + at) + 1, 1u << 16);
    }
  } else {
    const BinExp weight;
#pragma unroll
    for (int e = 0; e < NE; ++e) {           // (worked out for all, so that elements run side by side)
      const double l = (double)x[e] * per, f = floor(l), j = first - f;
      const int at = (int)j;
      const unsigned long long v = (1ull << 48) + weight(l - f);
      if (j < BINS) atomicAdd(bins + at, v);
    }
  }
}

// grid (slices, rows)
template <int NT, int NE, bool VEC>
__global__ __launch_bounds__(NT) void sample_slices_kernel(char* __restrict__ scratch, Cut cut, const float* __restrict__ logits, long ld, int V,
                                                           const float* __restrict__ temperature, const int* __restrict__ top_k) {
  __shared__ unsigned long long bins[BINS];
  __shared__ float tops[NT / 64];
  __shared__ int at;
  const int r = blockIdx.y, p = blockIdx.x, base = p * NT * NE, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float x[NE];
  load_slice<NT, NE, VEC>(x, logits + (long)r * ld, base, V);
  for (int i = threadIdx.x; i < BINS; i += NT) bins[i] = 0ull;
  if (threadIdx.x == 0) at = 0x7fffffff;
  float top = -INFINITY;
#pragma unroll
  for (int e = 0; e < NE; ++e) top = fmaxf(top, x[e]);
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) top = fmaxf(top, tops[w]);
  const Scratch s = scratch_of(scratch, r, cut);
  const float t = temperature ? temperature[r] : 1.f;
  if (!(t > 0.f)) {                          // the first of the largest
#pragma unroll
    for (int e = 0; e < NE; ++e) if (x[e] == top) atomicMin(&at, index_of<NT, NE, VEC>(base, e));
    __syncthreads();
  }
  if (threadIdx.x == 0) s.heads[p] = SliceHead{top, at, {0, 0}};
  if (!(top > -INFINITY) || !(t > 0.f)) return;
  bin_slice<NE>(x, bins, top, PER_T / (double)t, top_k ? top_k[r] : 0);
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) s.bins[p * BINS + i] = bins[i];
}

// another lane's value by the vector unit alone; lanes that have none get 0
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T lanes(T v) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8);
  int w[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof v);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], CTRL, ROWS, 0xf, false);
  T r;
  __builtin_memcpy(&r, w, sizeof r);
  return r;
}
// sums over a wave's lanes in front of each, and with it: within rows of 16, then the rows in front
template <typename T> __device__ __forceinline__ T wave_upto(T v) {
  v += lanes<0x111, 0xf>(v);
  v += lanes<0x112, 0xf>(v);
  v += lanes<0x114, 0xf>(v);
  v += lanes<0x118, 0xf>(v);
  v += lanes<0x142, 0xa>(v);
  v += lanes<0x143, 0xc>(v);
  return v;
}
// the same over a workgroup of NT
template <int NT, typename T> __device__ __forceinline__ T sum_upto(T v, T* room /* NT / 64 */) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  static_assert(NT <= 1024);
  v = wave_upto(v);
  __syncthreads();
  if (lane == 63) room[wave] = v;
  __syncthreads();
  T w = lane < NT / 64 ? room[lane] : T(0);
  w += lanes<0x111, 0xf>(w);
  w += lanes<0x112, 0xf>(w);
  w += lanes<0x114, 0xf>(w);
  w += lanes<0x118, 0xf>(w);
  const T before = __shfl(w, wave > 0 ? wave - 1 : 0, 64);
  return wave > 0 ? v + before : v;
}
// two sums at once, in rooms that nobody holds yet
template <int NT, typename T, typename U> __device__ __forceinline__ void sums_upto(T& v, U& w, T* room_v, U* room_w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_upto(v);
  w = wave_upto(w);
  if (lane == 63) { room_v[wave] = v; room_w[wave] = w; }
  __syncthreads();
  T a = lane < wave ? room_v[lane] : T(0);   // (of the waves in front, of which there are 15 at most)
  U b = lane < wave ? room_w[lane] : U(0);
  auto row = [](auto& x) {
    x += lanes<0x111, 0xf>(x);
    x += lanes<0x112, 0xf>(x);
    x += lanes<0x114, 0xf>(x);
    x += lanes<0x118, 0xf>(x);
  };
  row(a);
  row(b);
  v += __shfl(a, 15, 64);
  w += __shfl(b, 15, 64);
}
// how many threads hold a, and how many b; `cell`, 0, is this call's alone (one addition a wave: sixteen waves that read sixteen words each took 1 us and more)
struct Two { int a, b; };
__device__ __forceinline__ Two how_many(bool a, bool b, int* cell, bool also_a = false, bool also_b = false) {
  const int n = (__popcll(__ballot(a)) + __popcll(__ballot(also_a))) | ((__popcll(__ballot(b)) + __popcll(__ballot(also_b))) << 16);
  if ((threadIdx.x & 63) == 0 && n) atomicAdd(cell, n);
  __syncthreads();
  const int w = *cell;
  return Two{w & 0xffff, w >> 16};
}

// grid (Q, rows); a thread a bin.  ONE: rows of one slice, whose bins are made here too
template <int NE, bool VEC, bool ONE>
__global__ __launch_bounds__(BINS, NE > 16 ? 4 : 8) void sample_collect_kernel(char* __restrict__ scratch, Cut cut, const float* __restrict__ logits, long ld, int V,
                                                              const float* __restrict__ uniforms, const float* __restrict__ temperature, const int* __restrict__ top_k,
                                                              const float* __restrict__ top_p, const float* __restrict__ min_p) {
  constexpr int NT = BINS;
  __shared__ double m_in[BINS], wave_m[NT / 64];
  __shared__ int shift[P_MAX], c_in[BINS], wave_c[NT / 64], cells[3], found;
  __shared__ float bounds[4][2], tops[NT / 64];
  __shared__ unsigned long long bins[ONE ? BINS : 1];
  __shared__ int at_top;
  const int r = blockIdx.y, P = cut.P, b = threadIdx.x, lane = b & 63;
  int p = blockIdx.x;                        // chunk
  const RowSettings set = row_settings(r, V, temperature, top_k, top_p, min_p, uniforms);
  if (!ONE && set.greedy) return;
  const Scratch s = scratch_of(scratch, r, cut);
  float x[NE];                               // (asked for early: what comes in between is latency)
  load_slice<NT, NE, VEC>(x, logits + (long)r * ld, p * NT * NE, V);
  float head = -INFINITY, top;
  if constexpr (ONE) {
#pragma unroll
    for (int e = 0; e < NE; ++e) head = fmaxf(head, x[e]);
    head = wave_max(head);
    if (lane == 0) tops[b >> 6] = head;
    bins[b] = 0ull;
    if (b == 0) at_top = 0x7fffffff;
    __syncthreads();
    top = wave_max(tops[lane & (NT / 64 - 1)]);
    if (set.greedy) {                        // the first of the largest
#pragma unroll
      for (int e = 0; e < NE; ++e) if (x[e] == top) atomicMin(&at_top, index_of<NT, NE, VEC>(0, e));
      __syncthreads();
    }
    if (b == 0) s.heads[0] = SliceHead{top, at_top, {0, 0}};
    if (set.greedy) return;
  } else {
    head = lane < P ? s.heads[lane].top : -INFINITY;
    top = wave_max(head);
  }
  if (!(top > -INFINITY)) return;
  const double per = PER_T / set.t, line = line_of(top, per), first = floor(line);
  if (!ONE && b < P) {
    const double d = first - floor(line_of(head, per));
    shift[b] = d < BINS && counts(head, top, per) ? (int)d : BINS;
  }
  if (b == 0) found = 0;
  if (b < 3) cells[b] = 0;
  if constexpr (ONE) bin_slice<NE>(x, bins, top, per, top_k ? top_k[r] : 0);
  __syncthreads();
  unsigned long long q = 0ull;
  int c = 0;
  constexpr int BATCH = NE <= 8 ? 16 : 8;    // slices asked for together
  if constexpr (ONE) {
    c = (int)(bins[b] >> 48);
    q = bins[b] & 0xffffffffffffull;
  } else
    for (int i0 = 0; i0 < P; i0 += BATCH) {
      unsigned long long v[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int k = i0 + i < P ? b - shift[i0 + i] : -1;
        v[i] = k >= 0 ? s.bins[(i0 + i) * BINS + k] : 0ull;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        c += (int)(v[i] >> 48);
        q += v[i] & 0xffffffffffffull;
      }
    }
  // (a bin's middle beside the largest)
  const bool flat = is_flat(top, per);
  double m = flat ? (b == 0 ? (double)c : 0.0) : fma((double)c, BIN_LEAST, (double)q * (1.0 / BIN_ONE)) * exp_down((first - b + 0.5 - line) * (1.0 / PER_T));
  const int c_own = c;
  sums_upto<NT>(c, m, wave_c, wave_m);
  c_in[b] = c;
  m_in[b] = m;
  __syncthreads();
  const int c_all = c_in[BINS - 1];
  // slack: both sides of a comparison may be off, here and where resolve makes it again; faint: what the tokens in no bin may weigh
  const double all = m_in[BINS - 1], slack = (flat ? 1e-13 : 6.0 * off_of(line)) * all, faint = flat ? 0.0 : FAINT * (V - c_all), m_ex = b > 0 ? m_in[b - 1] : 0.0;
  // the bins that each end may lie in: k0, [p0, p1], [m0, m1], [d0, d1]; BINS: nowhere
  const int k = set.m > 1.0 ? 1 : set.k;
  const bool whole = top_k && top_k[r] >= 1 && top_k[r] <= K_COUNT, k_binds = k < c_all;
  const int k0 = k_binds ? how_many(c < k, false, &cells[0]).a : BINS;
  const bool k_exact = k_binds && c_in[k0] == k;
  bool p_binds = false, m_binds = false;
  int m0 = BINS, m1 = BINS, from[4] = {0, BINS, BINS, BINS}, to[4] = {min(k0, BINS - 1), -1, -1, -1};       // runs of bins that are wanted
  if (!whole) {
    const double mk_hi = k_binds ? m_in[k0] : all + faint, mk_lo = !k_binds ? all : k_exact ? mk_hi : k0 > 0 ? m_in[k0 - 1] : 0.0;
    int p0 = BINS, p1 = BINS;
    if (set.p < 1.0) {
      const Two n = how_many(m < set.p * mk_lo - slack, m_ex < set.p * mk_hi + slack, &cells[1]);
      p0 = n.a;
      p1 = max(0, n.b - 1);
    }
    if (set.m > 0.0 && set.m <= 1.0) {
      const double off = fabs(line) * 1e-15 + 1e-6, at = first - line - PER_T * log(set.m);
      m0 = (int)fmin(fmax(ceil(at - off), 0.0), (double)BINS);
      m1 = (int)fmin(fmax(floor(at + 1.0 + off), 0.0), (double)BINS);
      if (m1 >= BINS) m1 = m0 = BINS;        // (what weighs less is in no bin)
    }
    const int end = min(min(k0, p1), m1);
    p_binds = p0 <= end && p0 < BINS;
    m_binds = m0 <= end && m0 < BINS;
    double lo = mk_lo, hi = mk_hi;
    if (p_binds) { lo = fmin(lo, set.p * mk_lo - slack); hi = fmin(hi, m_in[min(p1, BINS - 1)]); }
    if (m_binds) { lo = fmin(lo, m0 > 0 ? m_in[m0 - 1] : 0.0); hi = fmin(hi, m_in[m1]); }
    lo = fmax(lo, 0.0);
    const Two d = how_many(m <= set.u * lo - slack, m_ex <= set.u * hi + slack, &cells[2]);
    const int d0 = d.a, d1 = d.b - 1;
    from[0] = d0;
    to[0] = min(d1, end);
    if (p_binds) { from[1] = p0; to[1] = min(p1, end); }
    if (m_binds) { from[2] = m0; to[2] = m1; }
    if (k_binds && !k_exact && (k0 <= end || p_binds)) from[3] = to[3] = k0;
  }
  auto wanted = [&](int j) { return (j >= from[0] && j <= to[0]) || (j >= from[1] && j <= to[1]) || (j >= from[2] && j <= to[2]) || (j >= from[3] && j <= to[3]); };
  const bool flag = wanted(b);
  // the wanted runs as values: the least float of a run's last bin the least above its first
  if (b >= NT - 8) {
    const int i = (b & 7) >> 1, above = b & 1, f = i == 0 ? from[0] : i == 1 ? from[1] : i == 2 ? from[2] : from[3], t = i == 0 ? to[0] : i == 1 ? to[1] : i == 2 ? to[2] : to[3];
    float v;
    if (flat || !(per > 0.0)) v = above ? NAN : f <= 0 && t >= 0 ? (flat ? top : -3.402823466e38f) : NAN;
    else v = least_at(above ? first - f + 1.0 : first - t, per);
    bounds[i][above] = v;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    // (a bin's place among the wanted ones: the runs may touch, so they are counted)
    const int g = sum_upto<NT>((int)flag, wave_c);
    RowSums& o = *s.sums;
    o.mass[b] = m_ex;
    o.count[b] = c - c_own;
    o.slot[b] = flag ? (short)(g - 1) : (short)-1;
    if (b == BINS - 1) o.said = RowSaid{all, c_all, g, k_binds ? (k_exact ? 2 : 1) : 0, k0, m0, m1, p_binds, m_binds, whole, 0};
  }
  unsigned long long* const to_found = s.found + (long)blockIdx.x * cut.cap;
  for (;;) {
    unsigned mask = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (from[i] <= to[i]) {
        const float lo = bounds[i][0], hi = bounds[i][1];
#pragma unroll
        for (int e = 0; e < NE; ++e) mask |= x[e] >= lo && !(x[e] >= hi) ? 1u << e : 0u;
      }
    if (__ballot(mask != 0u)) {              // (one atomic a wave)
      const int n = __popc(mask);
      int at = n, start = 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) { const int v = __shfl_up(at, o, 64); if (lane >= o) at += v; }
      if (lane == 63) start = atomicAdd(&found, at);
      at += __shfl(start, 63, 64) - n;
#pragma unroll
      for (int e = 0; e < NE; ++e)
        if (mask >> e & 1) {
          if (at < cut.cap) to_found[at] = ((unsigned long long)key_of(x[e]) << 32) | (unsigned)(0x7fffffff - index_of<NT, NE, VEC>(p * NT * NE, e));
          ++at;
        }
    }
    p += gridDim.x;
    if (p >= P) break;
    load_slice<NT, NE, VEC>(x, logits + (long)r * ld, p * NT * NE, V);
  }
  __syncthreads();
  if (b == 0) s.taken[blockIdx.x] = found;
}

// lane ^ X's value by the vector unit alone
template <int X> __device__ __forceinline__ unsigned lane_xor(unsigned v) {
  static_assert(X == 1 || X == 2 || X == 3 || X == 4 || X == 7 || X == 8 || X == 15 || X == 16 || X == 31 || X == 63);
  if constexpr (X == 4) return lane_xor<3>(lane_xor<7>(v));
  else if constexpr (X == 31) return lane_xor<16>(lane_xor<15>(v));
  else if constexpr (X == 63) {
    const unsigned w = lane_xor<31>(v);
    const auto a = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return threadIdx.x & 32 ? a[0] : a[1];
  } else if constexpr (X == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? a[0] : a[1];
  } else {
    constexpr int ctrl = X == 1 ? 0xb1 : X == 2 ? 0x4e : X == 3 ? 0x1b : X == 7 ? 0x141 : X == 15 ? 0x140 : 0x128;
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, false);
  }
}
// of lanes whose numbers differ by X the one in front takes the larger value
template <int X> __device__ __forceinline__ void order(unsigned long long& v) {
  constexpr int top = X >= 32 ? 32 : X >= 16 ? 16 : X >= 8 ? 8 : X >= 4 ? 4 : X >= 2 ? 2 : 1;
  const unsigned long long o = lane_xor<X>((unsigned)v) | ((unsigned long long)lane_xor<X>((unsigned)(v >> 32)) << 32);
  v = (v < o) == ((threadIdx.x & top) == 0) ? o : v;
}
__device__ __forceinline__ void sort_wave(unsigned long long& v) {
  order<1>(v);
  order<3>(v), order<1>(v);
  order<7>(v), order<2>(v), order<1>(v);
  order<15>(v), order<4>(v), order<2>(v), order<1>(v);
  order<31>(v), order<8>(v), order<4>(v), order<2>(v), order<1>(v);
  order<63>(v), order<16>(v), order<8>(v), order<4>(v), order<2>(v), order<1>(v);
}
// Largest first, `n` a power of two of 64 to 2 ST, values that differ (or are 0).  Runs of 64 by the lanes of a wave, then pairs of runs: a value's place is its own plus
// how many of the other run are larger.  w: room for as many.
__device__ __forceinline__ void sort_down(unsigned long long* v, unsigned long long* w, int n) {
  typedef unsigned long long u64;
  const int lane = threadIdx.x & 63, i0 = (threadIdx.x >> 6) * 128 + lane;
  const bool on[2] = {i0 < n, i0 + 64 < n};
  __syncthreads();
  u64 a[2] = {on[0] ? v[i0] : 0ull, on[1] ? v[i0 + 64] : 0ull};
  int at[2] = {i0, i0 + 64};
  if (on[0]) {                               // (a wave's are there or not together)
    sort_wave(a[0]);
    sort_wave(a[1]);
  }
  int turns = 0;
  while (64 << turns < n) ++turns;
  u64 *to = turns & 1 ? w : v, *other = turns & 1 ? v : w;
  for (int run = 64;; run <<= 1) {
    __syncthreads();                         // (the first: all have been read; then: the buffer before last has)
#pragma unroll
    for (int e = 0; e < 2; ++e) if (on[e]) to[at[e]] = a[e];
    __syncthreads();
    if (run >= n) break;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (on[e]) {
        const int base = (at[e] & ~(run - 1)) ^ run;         // the other run
        const bool second = (at[e] & run) != 0;              // of equals (zeros) the first run's stand in front
        int lo = 0;
        for (int step = run; step > 0; step >>= 1) {
          const int m = lo + step;
          if (m <= run) {
            const u64 x = to[base + m - 1];
            if (x > a[e] || (second && x == a[e])) lo = m;
          }
        }
        at[e] = (at[e] & ~(2 * run - 1)) + (at[e] & (run - 1)) + lo;
      }
    u64* const t = to;
    to = other;
    other = t;
  }
}

// a workgroup a row
template <bool SMALL>
__global__ __launch_bounds__(ST) void sample_resolve_kernel(int* __restrict__ tokens, float* __restrict__ probs, char* __restrict__ scratch, Cut row_cut,
                                                            const float* __restrict__ logits, long ld, int V, const float* __restrict__ uniforms,
                                                            const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                            const float* __restrict__ min_p) {
  typedef unsigned long long u64;
  __shared__ __attribute__((aligned(16))) u64 v[CAP], raw[CAP];    // tokens; whole masses of bins, then masses (as 64-bit floats) in front of each bin, up to and with each token
  __shared__ double front_m[CAP];                                  // mass and count in front of each bin
  __shared__ int front_c[CAP], start[CAP];                         // where a bin's tokens start in v
  __shared__ u64 wide[ST / 64];
  __shared__ double wide_m[ST / 64];
  __shared__ int narrow[ST / 64], cells[3];
  __shared__ short slot[BINS];
  __shared__ unsigned char want[CAP];
  __shared__ SlowRoom room;
  __shared__ int from[P_MAX + 1], got[4], ranks, taken, sum_c;
  __shared__ Mass sum_m;
  __shared__ double masses, masses_off;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* row = logits + (long)r * ld;
  const RowSettings set = row_settings(r, V, temperature, top_k, top_p, min_p, uniforms);
  const Scratch s = SMALL ? Scratch{} : scratch_of(scratch, r, row_cut);
  float top = -INFINITY;
  int first_at = 0, had = 0;
  RowSaid said{};
  double bin_m = 0.0;                        // of bin tid
  int bin_c = 0, bin_slot = -1;
  if constexpr (!SMALL) {                    // (asked for with the heads; of a greedy row it is whatever stands there)
    said = s.sums->said;
    bin_m = s.sums->mass[tid];
    bin_c = s.sums->count[tid];
    bin_slot = s.sums->slot[tid];
  }
  if constexpr (SMALL) {
    u64 best = 0ull;
    for (int i = tid; i < V; i += ST) {
      const u64 k = ((u64)key_of(row[i]) << 32) | (unsigned)(0x7fffffff - i);
      v[i] = k;
      best = k > best ? k : best;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { const u64 k = __shfl_xor(best, o, 64); best = k > best ? k : best; }
    if (lane == 0) wide[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < ST / 64; ++w) best = wide[w] > best ? wide[w] : best;
    __syncthreads();
    top = of_key((unsigned)(best >> 32));
    first_at = 0x7fffffff - (int)(best & 0xffffffffu);
  } else {
    const SliceHead h = lane < row_cut.P ? s.heads[lane] : SliceHead{-INFINITY, 0, {0, 0}};
    top = wave_max(h.top);
    const unsigned long long bal = __ballot(h.top == top);
    first_at = __shfl(h.at, __ffsll(bal) - 1, 64);
    had = lane < row_cut.Q ? s.taken[lane] : 0;
  }
  if (!(top > -INFINITY) || set.greedy) {
    if (tid == 0) {
      tokens[r] = top > -INFINITY ? first_at : -1;
      if (probs) probs[r] = top > -INFINITY ? 1.f : 0.f;
    }
    return;
  }
  const double inv_t = 1.0 / set.t, per = PER_T / set.t, line = line_of(top, per), first = floor(line);
  auto value = [](u64 t) { return of_key((unsigned)(t >> 32)); };
  auto token_weight = [&](u64 t) { return (unsigned)(t >> 32) > KEY_NONE ? weight_at(value(t), top, inv_t) : 0.0; };
  int n = V, slots = 1;
  bool whole = true, p_binds = set.p < 1.0, m_binds = set.m > 0.0 && set.m <= 1.0;
  const int k = set.m > 1.0 ? 1 : set.k;
  int m0 = 0, m1 = BINS - 1, found = 0;
  static_assert(CAP * 8 >= BINS * 14 && BINS == ST);
  auto mass_at = [&](int i) { return __longlong_as_double((long long)raw[i]); };
  auto leave = [&](int i, double m) { raw[i] = (u64)__double_as_longlong(m); };
  double* const slot_m = reinterpret_cast<double*>(v);               // mass and count in front of each collected bin, while v holds no tokens
  int* const slot_c = reinterpret_cast<int*>(v + BINS);
  short* const slot_bin = reinterpret_cast<short*>(slot_c + BINS);
  if constexpr (!SMALL) {
    if (__ballot(had > row_cut.cap)) {
      sample_slow(r, tokens, probs, row, V, set, top, room);
      return;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int x = __shfl_up(had, o, 64); if (lane >= o) had += x; }
    if (wave == 0) {
      if (lane < row_cut.Q) from[lane + 1] = had;
      if (lane == 0) from[0] = 0;
    }
    __syncthreads();
    n = found = from[row_cut.Q];
    whole = said.whole;
    if (!whole) {
      p_binds = said.p_binds;
      m_binds = said.m_binds;
      m0 = said.m0;
      m1 = said.m1;
    }
    slots = said.slots;
    slot[tid] = (short)bin_slot;
    if (found > FEW && bin_slot >= 0) {
      slot_m[bin_slot] = bin_m;
      slot_c[bin_slot] = bin_c;
      slot_bin[bin_slot] = (short)tid;
    }
  }
  // (putting in order takes 13 us for 1024 tokens and more, 6 for 300, 1.6 for 64 and fewer; the bins and looking again 5, and a dozen tokens are left)
  const bool many = !SMALL && found > FEW;
  // bins of the collected tokens: all in one (front of it nothing); those of collect; or `cut` in each of those
  int cut = 1;
  if (many) while (2 * cut * slots <= CAP && cut < 256) cut *= 2;
  auto place = [&](u64 t, int* shift = nullptr) -> int {
    if (SMALL || (whole && !many)) return 0;
    const double l = floor(line_of(value(t), per) * cut), c = floor(l * (1.0 / cut));
    const int j = max(0, min(BINS - 1, (int)(first - c)));
    if (shift) *shift = fine_shift(j);
    return many ? max(0, (int)slot[j]) * cut + (cut - 1 - (int)(l - c * cut)) : j;
  };
  // f of each collected token, slice behind slice in memory; four loads of a thread in flight
  auto each = [&](auto f) {
    int at = 0;
    for (int i0 = tid; i0 < found; i0 += 4 * ST) {
      u64 t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e * ST;
        if (i < found) {
          while (from[at + 1] <= i) ++at;
          t[e] = s.found[(long)at * row_cut.cap + i - from[at]];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) if (i0 + e * ST < found) f(i0 + e * ST, t[e]);
    }
  };
  if (tid < 4) got[tid] = 2 * CAP;
  if (tid < 3) cells[tid] = 0;
  if (tid == 0) { taken = 0; sum_c = 0; sum_m = Mass{0ull, 0ll}; }
  if (many) for (int i = tid; i < CAP; i += ST) { raw[i] = 0ull; start[i] = 0; }
  __syncthreads();
  // min-p's end: as many as weigh enough
  int count_m = 0;
  Mass mass_m{0ull, 0ll};
  auto enough = [&](u64 t, double w) {
    if (!m_binds || !(w >= set.m) || (unsigned)(t >> 32) <= KEY_NONE) return;
    if (!SMALL && !whole) {
      const int j = (int)(first - floor(line_of(value(t), per)));
      if (j < m0 || j > m1) return;
    }
    ++count_m;
    mass_m = mass_m + mass_of(w);
  };
  if (many)
    each([&](int, u64 t) {
      const double w = token_weight(t);
      enough(t, w);
      int shift;
      const int b = place(t, &shift);
      atomicAdd(&raw[b], fine_of(w, shift));
      atomicAdd(&start[b], 1);
    });
  else {
    if constexpr (!SMALL) {
      each([&](int i, u64 t) { v[i] = t; });
      __syncthreads();
    }
    for (int i = tid; i < n; i += ST) enough(v[i], token_weight(v[i]));
  }
  double end_m = 0.0, front_of_m = 0.0;
  if (m_binds) {
    if (__ballot(count_m > 0)) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        mass_m = mass_m + Mass{__shfl_xor(mass_m.hi, o, 64), __shfl_xor(mass_m.lo, o, 64)};
        count_m += __shfl_xor(count_m, o, 64);
      }
      if (lane == 0) { atomicAdd(&sum_m.hi, mass_m.hi); atomicAdd(reinterpret_cast<u64*>(&sum_m.lo), (u64)mass_m.lo); atomicAdd(&sum_c, count_m); }
    }
    __syncthreads();
    count_m = sum_c;
    end_m = sum_m.value();
    if (!SMALL && !whole) { count_m += s.sums->count[m0]; front_of_m = s.sums->mass[m0]; end_m += front_of_m; }
  }
  __syncthreads();
  int how_k = SMALL || whole ? (k < n ? 1 : 0) : said.k_binds, count = SMALL || whole ? n : said.count_all;
  double mass = 0.0;                         // of everything, then of the first k
  if (!SMALL && !whole) {
    mass = said.all;
    if (how_k == 2) {
      count = k;
      mass = said.k0 + 1 < BINS ? s.sums->mass[said.k0 + 1] : said.all;
    }
  }
  // Sums from the bins: in front of a collected token, and of everything, off by `off` of them.  The collected tokens' own sums are good to 64 bits (bins of them to
  // 2^-46 of each weight: 1e-14).  Of the first k, those that are in no bin may weigh `faint`.
  const bool rough = !SMALL && !whole, flat = is_flat(top, per);
  const double off = rough ? (flat ? 0.0 : off_of(line)) + 2e-14 : 0.0, faint = !SMALL && how_k == 0 && !flat ? FAINT * max(0, k - said.count_all) : 0.0;
  if (many) {
    // each bin's sums, from those in front of it; then which bins the ends may lie in, as collect does
    const int b0 = 2 * tid;
    const int used = slots * cut;
    auto mass_of_bin = [&](int b) { return b < used ? (double)raw[b] * power_of_two(-FINE_BITS - fine_shift(slot_bin[b / cut])) : 0.0; };
    const double q0 = mass_of_bin(b0), q1 = mass_of_bin(b0 + 1);
    const int c0 = start[b0], c1 = start[b0 + 1];
    double qs = q0 + q1;
    int cs = c0 + c1;
    __syncthreads();
    sums_upto<ST>(qs, cs, wide_m, narrow);
    __syncthreads();
    leave(b0, qs - (q0 + q1));
    leave(b0 + 1, qs - q1);
    start[b0] = cs - c0 - c1;
    start[b0 + 1] = cs - c1;
    __syncthreads();
    double ex[2], in[2];
    int c_in[2], c_ex[2];
    bool is[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = b0 + e;
      is[e] = b < used;
      ex[e] = in[e] = 0.0;
      c_ex[e] = c_in[e] = 0;
      if (is[e]) {
        const int z = b / cut * cut, j = b / cut;
        ex[e] = whole ? mass_at(b) : slot_m[j] + (mass_at(b) - mass_at(z));
        in[e] = ex[e] + (e ? q1 : q0);
        c_ex[e] = whole ? start[b] : slot_c[j] + start[b] - start[z];
        c_in[e] = c_ex[e] + (e ? c1 : c0);
      }
      front_m[b] = ex[e];
      front_c[b] = c_ex[e];
    }
    if (whole) {
      if (tid == ST - 1) masses = qs;
      __syncthreads();
      mass = masses;
    }
    const double slack = (6.0 * off + 1e-12) * mass;
    auto before = [&](bool a0, bool a1, bool b0, bool b1, int call) -> Two {       // bins, of both a thread's
      return how_many(is[0] && a0, is[0] && b0, &cells[call], is[1] && a1, is[1] && b1);
    };
    const int k0 = how_k == 1 ? before(c_in[0] < k, c_in[1] < k, false, false, 0).a : used;
    double lo = mass, hi = mass + faint;
    if (k0 < used) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) if (b0 + e == k0) { masses = in[e]; got[0] = c_in[e] == k ? 1 : 0; }
      __syncthreads();
      hi = masses;
      if (got[0] == 1) {
        how_k = 2;
        count = k;
        lo = mass = hi;
      } else lo = front_m[k0];
      __syncthreads();
      if (tid == 0) got[0] = 2 * CAP;
    }
    int p0 = used, p1 = -1;
    if (p_binds) {
      const double l = set.p * lo - slack, h = set.p * hi + slack;
      const Two n = before(in[0] < l, in[1] < l, ex[0] < h, ex[1] < h, 1);
      p0 = n.a;
      p1 = max(n.b - 1, 0);
      if (p0 < used) {
        lo = fmin(lo, set.p * lo - slack);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e) if (b0 + e == p1) masses = in[e];
        __syncthreads();
        hi = fmin(hi, masses);
      }
    }
    if (m_binds) { lo = fmin(lo, end_m - slack); hi = fmin(hi, end_m + slack); }
    lo = fmax(lo, 0.0);
    const double ulo = set.u * lo - slack, uhi = set.u * hi + slack;
    const Two d = before(in[0] <= ulo, in[1] <= ulo, ex[0] <= uhi, ex[1] <= uhi, 2);
    const int d0 = d.a, d1 = d.b - 1;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int b = b0 + e;
      want[b] = is[e] && ((b >= p0 && b <= p1) || (b >= d0 && b <= d1) || (how_k == 1 && b == k0));
    }
    __syncthreads();
    each([&](int, u64 t) {
      if (want[place(t)]) {
        const int at = atomicAdd(&taken, 1);
        if (at < CAP) v[at] = t;
      }
    });
    __syncthreads();
    n = taken;
    if (n > CAP) {
      sample_slow(r, tokens, probs, row, V, set, top, room);
      return;
    }
  } else if (!SMALL && !whole) {
    front_m[tid] = bin_m;
    front_c[tid] = bin_c;
  } else if (tid == 0) { front_m[0] = 0.0; front_c[0] = 0; }
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += ST) v[i] = 0ull;
  sort_down(v, raw, size);
  // mass up to and with each token, and its rank
  const int e0 = 2 * tid;
  double w[2] = {0.0, 0.0}, in[2] = {0.0, 0.0};
  int rank[2] = {1 << 30, 1 << 30}, bin[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (e0 + e < n) {
      w[e] = token_weight(v[e0 + e]);
      bin[e] = place(v[e0 + e]);
      if (e0 + e == 0 || place(v[e0 + e - 1]) != bin[e]) start[bin[e]] = e0 + e;
    }
  const double sum = sum_upto<ST>(w[0] + w[1], wide_m);
  leave(e0, sum - w[1]);
  leave(e0 + 1, sum);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (e0 + e < n) {
      const int at = start[bin[e]];
      in[e] = front_m[bin[e]] + (mass_at(e0 + e) - (at > 0 ? mass_at(at - 1) : 0.0));
      rank[e] = front_c[bin[e]] + e0 + e - at;
    }
  // the ends: what is kept is the first `count`, whose mass is from mass - less to mass + more
  if ((SMALL || whole) && !many) {
    if (e0 <= n - 1 && n - 1 <= e0 + 1) masses = in[n - 1 - e0];
    __syncthreads();
    mass = masses;
  }
  double in_off[2] = {0.0, 0.0}, less = off * mass, more = less + faint;
  if (rough)
#pragma unroll
    for (int e = 0; e < 2; ++e) if (e0 + e < n) in_off[e] = off * front_m[bin[e]] + 2e-14 * in[e];
  __syncthreads();
  if (how_k == 1) {
#pragma unroll
    for (int e = 0; e < 2; ++e) if (rank[e] == k - 1) { got[0] = 0; masses = in[e]; masses_off = in_off[e]; }
  }
  __syncthreads();
  if (how_k == 1 && got[0] == 0) { count = k; mass = masses; less = more = masses_off; }
  // twice the first element for which it may be so, and 1 if it need not be (in any case it is so for no earlier one); one atomic a wave
  auto first_of = [&](bool x, bool y, bool sure_x, bool sure_y, int* to) {
    const unsigned long long one = __ballot(x || y);
    if (one && lane == __ffsll(one) - 1) atomicMin(to, x ? 2 * e0 + !sure_x : 2 * e0 + 2 + !sure_y);
  };
  // top-p's end: the first token that reaches p of the mass
  const double p = fmax(set.p, 0.0), limit = p * (mass - less), at_most = p * (mass + more);
  first_of(e0 < n && p_binds && in[0] + in_off[0] >= limit, e0 + 1 < n && p_binds && in[1] + in_off[1] >= limit, in[0] - in_off[0] >= at_most, in[1] - in_off[1] >= at_most,
           &got[1]);
  __syncthreads();
  const int kp = got[1] >> 1;
  bool open = false;
#pragma unroll
  for (int e = 0; e < 2; ++e) if (e0 + e == kp) { ranks = rank[e] + 1; masses = in[e]; masses_off = in_off[e]; }
  __syncthreads();
  if (m_binds && count_m < count) { count = count_m; mass = end_m; less = more = rough ? off * front_of_m + 2e-14 * end_m : 0.0; }
  if (p_binds && kp < CAP && ranks < count) {
    count = ranks;
    mass = masses;
    less = more = masses_off;
    open = !SMALL && (got[1] & 1);
  }
  if (count < 1) { count = 1; mass = 1.0; less = more = 0.0; }
  // the draw: the first over the goal, the last kept one where the sums' rounding leaves none
  const double goal = set.u * (mass - less), goal_most = set.u * (mass + more);
  const bool kept[2] = {e0 < n && w[0] > 0.0 && rank[0] < count, e0 + 1 < n && w[1] > 0.0 && rank[1] < count};
  first_of(kept[0] && in[0] + in_off[0] > goal, kept[1] && in[1] + in_off[1] > goal, in[0] - in_off[0] > goal_most, in[1] - in_off[1] > goal_most, &got[2]);
  __syncthreads();
  int at = got[2] >> 1;
  if (!SMALL && (open || (got[2] & 1))) {
    sample_slow(r, tokens, probs, row, V, set, top, room);
    return;
  }
  if (at >= CAP) {
    if (tid == 0) got[3] = -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (kept[e]) atomicMax(&got[3], e0 + e);
    __syncthreads();
    at = max(got[3], 0);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (e0 + e == at) {
      tokens[r] = 0x7fffffff - (int)(v[at] & 0xffffffffu);
      if (probs) probs[r] = (float)(w[e] / mass);
    }
}

extern "C" long umb_sample_requests_bytes(int rows, int V) {
  if (rows < 1 || V < 1 || V > SAMPLE_VMAX) return 0;
  return V <= SMALL_V ? 16 : rows * row_bytes(cut_of(rows, V));
}

extern "C" int umb_sample_requests(int* tokens, float* probs, const float* logits, long ld, int rows, int V, const float* uniforms,
                                   const float* temperature, const int* top_k, const float* top_p, const float* min_p, void* scratch, long scratch_bytes,
                                   hipStream_t st) {
  if (!tokens || !logits || !uniforms || !scratch || rows < 1 || V < 1 || V > SAMPLE_VMAX || ld < V || (uintptr_t)scratch % 16 ||
      scratch_bytes < umb_sample_requests_bytes(rows, V))
    return UMB_EINVAL;
  if (V <= SMALL_V) {
    hipLaunchKernelGGL((sample_resolve_kernel<true>), dim3(rows), dim3(ST), 0, st, tokens, probs, (char*)nullptr, Cut{}, logits, ld, V, uniforms, temperature, top_k,
                       top_p, min_p);
    UMB_LAUNCH_CHECK();
    return UMB_OK;
  }
  const Cut cut = cut_of(rows, V);
  const bool vec = (uintptr_t)logits % 16 == 0 && ld % 4 == 0;
  for (int r0 = 0; r0 < rows; r0 += 65535) {                 // (a grid's rows)
    const int n = rows - r0 < 65535 ? rows - r0 : 65535;
    char* const sc = static_cast<char*>(scratch) + r0 * row_bytes(cut);
    const float* const x = logits + r0 * ld;
    auto at = [&](auto* p) { return p ? p + r0 : p; };
#define ONE_SLICE(NE, VEC)                                                                                                                       \
  hipLaunchKernelGGL((sample_collect_kernel<NE, VEC, true>), dim3(1, n), dim3(BINS), 0, st, sc, cut, x, ld, V, at(uniforms), at(temperature), at(top_k), \
                     at(top_p), at(min_p))
#define SLICES(NT, NE, VEC)                                                                                                                         \
  hipLaunchKernelGGL((sample_slices_kernel<NT, NE, VEC>), dim3(cut.P, n), dim3(NT), 0, st, sc, cut, x, ld, V, at(temperature), at(top_k));           \
  hipLaunchKernelGGL((sample_collect_kernel<NT * NE / BINS, VEC, false>), dim3(cut.Q, n), dim3(BINS), 0, st, sc, cut, x, ld, V, at(uniforms),        \
                     at(temperature), at(top_k), at(top_p), at(min_p))
    if (cut.P == 1) {
      if (cut.slice == 8192) { if (vec) ONE_SLICE(8, true); else ONE_SLICE(8, false); }
      else if (cut.slice == 16384) { if (vec) ONE_SLICE(16, true); else ONE_SLICE(16, false); }
      else { if (vec) ONE_SLICE(32, true); else ONE_SLICE(32, false); }
    }
    else if (cut.slice == 8192 && vec) { SLICES(512, 16, true); }
    else if (cut.slice == 8192) { SLICES(512, 16, false); }
    else if (vec) { SLICES(512, 32, true); }
    else { SLICES(512, 32, false); }
#undef ONE_SLICE
#undef SLICES
    hipLaunchKernelGGL((sample_resolve_kernel<false>), dim3(n), dim3(ST), 0, st, at(tokens), at(probs), sc, cut, x, ld, V, at(uniforms), at(temperature), at(top_k),
                       at(top_p), at(min_p));
    UMB_LAUNCH_CHECK();
  }
  return UMB_OK;
}
