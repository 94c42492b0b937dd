// The next token of every row of logits, each row with its own temperature, top-k, top-p and min-p, from a given random number.
//
// Order: value descending, index ascending.  w = exp((x - max) / T).  Each of the three filters keeps a prefix of that order: the first k; those
// in front of which less than p of the first k's mass stands; those with w >= m.  The shortest prefix is kept, and of it the first token whose mass,
// with all in front of it, exceeds u times the kept mass is drawn.
//
// Weights are 64-bit floats, summed as whole numbers of 2^-44 of the largest: such sums are the same in any order, and a border between two tokens
// falls where a 64-bit sum of any order puts it but for some 1e-12 of the mass.  (In 32 bits a flat row of 128256 values has thousands of borders that
// the sum's order moves.)
#include "seq_common.h"
#include <algorithm>

constexpr int SAMPLE_VMAX = 1 << 19;         // 2^19 weights of at most 2^44 are a number of 63 bits
constexpr double MASS_ONE = 17592186044416.0;

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
__device__ __forceinline__ unsigned long long mass_of(double w) { return (unsigned long long)(w * MASS_ONE + 0.5); }

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
  unsigned long long mass;
};

// The first element, in order, at which what has come up to and with it reaches a goal: BY_COUNT the goal-th element; otherwise the first whose
// mass up to and with it is at least (OVER: more than) `goal`.  There is one by the caller's choice of the goal, or the last element is taken.
// Four passes over the row, eight bits of the key each.
enum { BY_COUNT, AT_LEAST, OVER };
template <int HOW>
__device__ Pick find_in_row(const float* __restrict__ row, int V, float top, double t, double goal, unsigned* cnt, unsigned long long* sum, int* shared) {
  Pick got{0u, 0, 0, 0ull};
  unsigned mask = 0u;
  auto reached = [&](double n, double q) { return HOW == BY_COUNT ? n >= goal : HOW == AT_LEAST ? q >= goal : q > goal; };
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) { cnt[threadIdx.x] = 0u; sum[threadIdx.x] = 0ull; }
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += ST) {
      const unsigned k = key_of(row[i]);
      if ((k & mask) == got.key && k > KEY_NONE) {
        const int d = (k >> shift) & 255;
        atomicAdd(&cnt[d], 1u);
        const unsigned long long q = mass_of(weight_of(k, top, t));
        if (q) atomicAdd(&sum[d], q);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int n = got.count, d = 255, last = -1;
      unsigned long long q = got.mass;
      for (; d >= 0; --d) {
        if (!cnt[d]) continue;
        if (reached((double)(n + cnt[d]), (double)(q + sum[d]))) break;
        last = d;
        n += cnt[d];
        q += sum[d];
      }
      if (d < 0) { d = last < 0 ? 0 : last; n -= cnt[d]; q -= sum[d]; }
      shared[0] = d;
      shared[1] = n;
      reinterpret_cast<unsigned long long*>(shared)[1] = q;
    }
    __syncthreads();
    got.key |= (unsigned)shared[0] << shift;
    got.count = shared[1];
    got.mass = reinterpret_cast<unsigned long long*>(shared)[1];
    mask |= 255u << shift;
    if (shift == 0) {                        // equals, in the order of their indices
      const int n = cnt[shared[0]];
      const unsigned long long q = mass_of(weight_of(got.key, top, t));
      if (threadIdx.x == 0) {
        int lo = 0, hi = n - 1;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (reached((double)(got.count + mid + 1), (double)(got.mass + q * (mid + 1)))) hi = mid;
          else lo = mid + 1;
        }
        shared[4] = lo;
      }
      __syncthreads();
      got.tie = shared[4];
    }
  }
  __syncthreads();
  return got;
}

// one workgroup a row
__global__ __launch_bounds__(ST) void sample_requests_kernel(int* __restrict__ tokens, float* __restrict__ probs, const float* __restrict__ logits, long ld, int V,
                                                             const float* __restrict__ uniforms, const float* __restrict__ temperature,
                                                             const int* __restrict__ top_k, const float* __restrict__ top_p, const float* __restrict__ min_p) {
  __shared__ unsigned cnt[256];
  __shared__ unsigned long long sum[256];
  __shared__ __attribute__((aligned(16))) int shared[8];
  __shared__ unsigned long long wide[16];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* row = logits + (long)r * ld;
  const RowSettings s = row_settings(r, V, temperature, top_k, top_p, min_p, uniforms);
  unsigned best = 0u;
  int at = V;
  for (int i = tid; i < V; i += ST) {
    const unsigned k = key_of(row[i]);
    if (k > best) { best = k; at = i; }
  }
  unsigned long long b = ((unsigned long long)best << 32) | (unsigned)(0x7fffffff - at);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const unsigned long long x = __shfl_xor(b, o, 64); b = x > b ? x : b; }
  if (lane == 0) wide[wave] = b;
  __syncthreads();
  for (int i = 0; i < 16; ++i) b = wide[i] > b ? wide[i] : b;
  const unsigned top_key = (unsigned)(b >> 32);
  const float top = of_key(top_key);
  if (top_key <= KEY_NONE || s.greedy) {
    if (tid == 0) {
      tokens[r] = top_key <= KEY_NONE ? -1 : 0x7fffffff - (int)(b & 0xffffffffu);
      if (probs) probs[r] = top_key <= KEY_NONE ? 0.f : 1.f;
    }
    return;
  }
  // everything's and min-p's counts and masses
  __syncthreads();
  if (tid < 4) wide[tid] = 0ull;
  __syncthreads();
  unsigned long long n_all = 0, q_all = 0, n_min = 0, q_min = 0;
  for (int i = tid; i < V; i += ST) {
    const unsigned k = key_of(row[i]);
    const double w = weight_of(k, top, s.t);
    const unsigned long long q = mass_of(w);
    if (k > KEY_NONE) { ++n_all; q_all += q; if (w >= s.m) { ++n_min; q_min += q; } }
  }
  atomicAdd(&wide[0], n_all);
  atomicAdd(&wide[1], q_all);
  atomicAdd(&wide[2], n_min);
  atomicAdd(&wide[3], q_min);
  __syncthreads();
  n_all = wide[0];
  q_all = wide[1];
  long n = (long)wide[2];
  unsigned long long q = wide[3];
  if (n < 1) { n = 1; q = mass_of(1.0); }
  unsigned long long q_k = q_all;
  if ((unsigned long long)s.k < n_all) {
    const Pick e = find_in_row<BY_COUNT>(row, V, top, s.t, (double)s.k, cnt, sum, shared);
    q_k = e.mass + mass_of(weight_of(e.key, top, s.t)) * (e.tie + 1);
    if (s.k < n) { n = s.k; q = q_k; }
  }
  if (s.p < 1.0) {
    const Pick e = find_in_row<AT_LEAST>(row, V, top, s.t, fmax(s.p, 0.0) * (double)q_k, cnt, sum, shared);
    if (e.count + e.tie + 1 < n) { n = e.count + e.tie + 1; q = e.mass + mass_of(weight_of(e.key, top, s.t)) * (e.tie + 1); }
  }
  const Pick e = find_in_row<OVER>(row, V, top, s.t, s.u * (double)q, cnt, sum, shared);
  // the tie-th of the values equal to e's, by index
  int seen = 0;
  for (int i0 = 0; i0 < V; i0 += ST) {
    const int i = i0 + tid;
    const bool is = i < V && key_of(row[i]) == e.key;
    const unsigned long long bal = __ballot(is);
    __syncthreads();
    if (lane == 0) cnt[wave] = __popcll(bal);
    __syncthreads();
    int before = seen, all = seen;
    for (int w = 0; w < ST / 64; ++w) { if (w < wave) before += cnt[w]; all += cnt[w]; }
    if (is && before + __popcll(bal & ((1ull << lane) - 1ull)) == e.tie) {
      tokens[r] = i;
      if (probs) probs[r] = (float)(weight_of(e.key, top, s.t) * MASS_ONE / (double)q);
    }
    seen = all;
    if (seen > e.tie) break;
  }
}

extern "C" long umb_sample_requests_bytes(int rows, int V) { return rows < 1 || V < 1 || V > SAMPLE_VMAX ? 0 : 16; }

extern "C" int umb_sample_requests(int* tokens, float* probs, const float* logits, long ld, int rows, int V, const float* uniforms,
                                   const float* temperature, const int* top_k, const float* top_p, const float* min_p, void* scratch, long scratch_bytes,
                                   hipStream_t st) {
  if (!tokens || !logits || !uniforms || !scratch || rows < 1 || V < 1 || V > SAMPLE_VMAX || ld < V || (uintptr_t)scratch % 16 ||
      scratch_bytes < umb_sample_requests_bytes(rows, V))
    return UMB_EINVAL;
  hipLaunchKernelGGL(sample_requests_kernel, dim3(rows), dim3(ST), 0, st, tokens, probs, logits, ld, V, uniforms, temperature, top_k, top_p, min_p);
  UMB_LAUNCH_CHECK();
  return UMB_OK;
}
