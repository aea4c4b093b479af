// What the kernels that choose tokens and those that write distributions out share: an order-preserving image of floats, masses in
// fixed point, first maxima, and the search for the digit at which a running count or mass reaches its mark.
#pragma once
#include "common.h"

// (for all that is behind this)  A scaled logit is rounded to a float before anything else is done with it: its key, its mass and its
// probability are those of one number, wherever they are worked out (a product joined with the subtraction of the maximum is another
// one), so that the kernels that choose and those that write distributions out keep the same tokens.
#pragma clang fp contract(off)

namespace {

constexpr int THREADS = 1024;
constexpr int RADIX_BINS = 2048;
constexpr int FIX_PLACES = 44;

__device__ __forceinline__ unsigned order_key(float f) {  // a < b  <=>  key(a) < key(b)
  const unsigned u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct MaxIdx { float v; int i; };

__device__ __forceinline__ MaxIdx better(MaxIdx a, MaxIdx b) {  // larger value, then smaller index; NaN never wins
  if (b.v > a.v || (b.v == a.v && b.i < a.i)) return b;
  return a;
}

// f(i, row[i]) for this thread's share of row[begin..end), in no particular order; eight loads under way at a time (64 rows of
// 151,936 with top-k and top-p, 19 logits a thread: 143 -> 124 us; up to 16 rows, at most 10 logits a thread, no difference).
template <typename F>
__device__ __forceinline__ void for_share(const float* __restrict__ row, int begin, int end, F f) {
  constexpr int AT_ONCE = 8;
  for (int base = begin + threadIdx.x; base < end; base += AT_ONCE * THREADS) {
    float v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) v[j] = row[min(base + j * THREADS, end - 1)];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (base + j * THREADS < end) f(base + j * THREADS, v[j]);
  }
}

// The first maximum of row[begin..end); index 0x7fffffff: there is none but NaN.
__device__ MaxIdx block_argmax(const float* __restrict__ row, int begin, int end, MaxIdx* red) {
  MaxIdx best = {-INFINITY, 0x7fffffff};
  for_share(row, begin, end, [&](int i, float v) { best = better(best, MaxIdx{v, i}); });
  for (int o = MS_WAVE / 2; o > 0; o >>= 1) {
    MaxIdx other = {__shfl_xor(best.v, o, MS_WAVE), __shfl_xor(best.i, o, MS_WAVE)};
    best = better(best, other);
  }
  const int lane = threadIdx.x & (MS_WAVE - 1), wave = threadIdx.x / MS_WAVE;
  __syncthreads();
  if (lane == 0) red[wave] = best;
  __syncthreads();
  MaxIdx r = red[0];
  for (int w = 1; w < (int)(blockDim.x / MS_WAVE); ++w) r = better(r, red[w]);
  return r;
}

__device__ __forceinline__ unsigned long long fixed_mass(float s, float zmax) {
  return (unsigned long long)(expf(s - zmax) * (float)(1ull << FIX_PLACES));   // at most 2^44: exact for a float
}

__device__ __forceinline__ float key_value(unsigned key) {   // the float whose key this is
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ int level_shift(int level) { return level == 1 ? 21 : (level == 2 ? 10 : 0); }
__device__ __forceinline__ int level_bins(int level) { return level == 3 ? 1024 : RADIX_BINS; }

struct Found { int bin; unsigned long long count_above, mass_above, count_in, mass_in; };

// The first bin, from the top, at which the running count (by_mass = false) or mass of the bins so far reaches
// `need`; with it the count and mass of the bins above it and of the bin itself.  If none does, the lowest
// bin that holds anything (or bin 0).  Every thread of the block calls this and gets the same answer.
__device__ Found first_bin_reaching(const unsigned* __restrict__ count, const unsigned long long* __restrict__ mass,
                                    int bins, bool by_mass, unsigned long long need) {
  __shared__ unsigned long long wave_c[THREADS / MS_WAVE], wave_m[THREADS / MS_WAVE];
  __shared__ Found found;
  __shared__ int lowest;
  const int t = threadIdx.x, lane = t & (MS_WAVE - 1), wave = t / MS_WAVE;
  // thread t owns bins hi and hi - 1, hi = bins - 1 - 2 t: thread 0 the two topmost
  const int hi = bins - 1 - 2 * t;
  unsigned long long c[2] = {0, 0}, m[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (hi - j >= 0) { c[j] = count[hi - j]; m[j] = mass[hi - j]; }
  unsigned long long sc = c[0] + c[1], sm = m[0] + m[1];     // inclusive scan over threads, from the top
  for (int o = 1; o < MS_WAVE; o <<= 1) {
    const unsigned long long oc = __shfl_up(sc, o, MS_WAVE), om = __shfl_up(sm, o, MS_WAVE);
    if (lane >= o) { sc += oc; sm += om; }
  }
  if (t == 0) { found.bin = -1; lowest = bins; }
  __syncthreads();
  if (lane == MS_WAVE - 1) { wave_c[wave] = sc; wave_m[wave] = sm; }
  __syncthreads();
  unsigned long long before_c = 0, before_m = 0;
  for (int w = 0; w < wave; ++w) { before_c += wave_c[w]; before_m += wave_m[w]; }
  unsigned long long run_c = before_c + sc - (c[0] + c[1]), run_m = before_m + sm - (m[0] + m[1]);   // above bin hi
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (hi - j < 0) break;
    const unsigned long long upto = (by_mass ? run_m + m[j] : run_c + c[j]), above = by_mass ? run_m : run_c;
    if (above < need && upto >= need) found = Found{hi - j, run_c, run_m, c[j], m[j]};   // one thread at most
    if (c[j]) atomicMin(&lowest, hi - j);
    run_c += c[j]; run_m += m[j];
  }
  __syncthreads();
  if (found.bin < 0 && t == 0) {   // fewer tokens (or less mass) than asked for: everything is kept
    const int b = lowest < bins ? lowest : 0;
    unsigned long long tc = 0, tm = 0;
    for (int w = 0; w < THREADS / MS_WAVE; ++w) { tc += wave_c[w]; tm += wave_m[w]; }
    found = Found{b, tc - count[b], tm - mass[b], count[b], mass[b]};
  }
  __syncthreads();
  const Found f = found;
  __syncthreads();
  return f;
}

}  // namespace
