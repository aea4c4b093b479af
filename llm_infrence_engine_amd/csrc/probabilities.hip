// The distributions that tokens are drawn from, whole: out[r, i] = e^(s_i - max) / sum over the kept e^(s_j - max) for the kept
// i of row r and 0 for the others, s = logits / temperature.  What is kept is what csrc/sampling.hip keeps, token by token: the masses
// e^(s - max) that decide are its own (fixed_mass) and their sums exact, whoever adds them up in which order; a row without
// temperature is a one at its first maximum.
//
// The work is two readings of the logits and one writing; the rest is to find the floor, the smallest value kept, in few
// launches and without a sort.  A row is spread over n_chunks blocks; with `target` = top_p times the mass that top-k keeps:
//   1 every chunk's maximum; with a top-k also the maxima of groups of a wave's lanes (as many groups as four times k or so); with
//     neither top-k nor top-p the chunk's mass against its maximum too, and 4 is next (33 rows of 100,003: 18 us, in three launches 26)
//   2 top-k: the k-th largest group maximum is no larger than the k-th largest value, and only a few more than k values are above
//     it (50 of 384 groups: 54 expected): these are collected as candidates, those equal to it counted
//     top-p alone: every chunk's mass, and a histogram of masses by the distance from the maximum (1/128 wide, 2,048 of them), joined
//     in float: its sums depend on the order, so it only says where to look
//   3 top-p alone: the values of the histogram's bin in which the target falls, with a neighbour's where it falls that near its
//     edge, are the candidates; the mass above them is summed up anew
//   4 a thread to a candidate: count and mass of the larger ones say whether it is kept, the least kept one is the floor (from many
//     candidates a radix descent over their keys finds it); then every block writes its chunk
// What the candidates cannot decide (more than MAX_CANDIDATES of them, a k beyond half the groups, a target outside the
// candidates' masses) every block of the row finds by itself with a radix descent over the whole row: right for any input, and
// slow (a row of 151,936: 105 us for a k of half of them, 190 for top-p 0.5 of normal logits at a temperature of 3, 360 where all are
// alike; 25 to 38 otherwise).  Half the groups are 32 to a block at most, and a row has 512 / rows blocks, rounded up: k up to 64 with
// 256 rows, 32 with 512 (151,936, top-k 50, top-p 0.9: 140 us with 256 rows, 580 with 512).
#include "sampling.h"
#include "api.h"
#include <algorithm>
#include <type_traits>

namespace {

constexpr int MAX_CHUNKS = 32, WAVES = THREADS / MS_WAVE;
constexpr int MAX_CANDIDATES = THREADS;
constexpr int BINS = 2048;
constexpr float BINS_A_UNIT = 128.f;
constexpr float SUM_ERROR = 1.0f / 131072.f;     // of the histogram's sums, of the whole mass: some 60 additions of floats behind one another

struct RowWork {                       // one per row, in the workspace the caller brings
  unsigned chunk_max[MAX_CHUNKS];      // key of the largest scaled logit of every chunk (no temperature: the largest itself)
  unsigned n_candidates, n_ties;       // ties: values equal to the bound
  unsigned bound;                      // top-k: every value above it is a candidate
  int bin;                             // top-p alone: the middle bin of the candidates, < 0: none
  double chunk_sum[MAX_CHUNKS];        // neither top-k nor top-p: of the exponentials, against the chunk's own maximum
  unsigned long long chunk_mass[MAX_CHUNKS];
  unsigned long long chunk_above[MAX_CHUNKS];      // mass of the values above the candidates'
  int chunk_first[MAX_CHUNKS];         // no temperature: where the largest stands
  unsigned candidates[MAX_CANDIDATES];          // keys
  float hist[BINS];
  unsigned groups[MAX_CHUNKS * WAVES * 4];
};

// What a row asks for, and how its candidates are found.
struct RowPlan {
  float inv_t, p;
  int k;                 // 0: no top-k
  bool greedy, use_p;
  bool all;              // few enough values: all are candidates
  int groups;            // of a wave (0: none, or too few for k)
};

__device__ __forceinline__ RowPlan plan_of(const float* temperature, const int* top_k, const float* top_p, int r, int V, int n_chunks) {
  RowPlan a;
  const float T = temperature[r];
  a.greedy = !(T > 0.f);
  a.inv_t = 1.0f / T;
  const int k = top_k ? top_k[r] : 0;
  a.k = k > 0 && k < V ? k : 0;
  a.p = top_p ? top_p[r] : 1.f;
  a.use_p = a.p < 1.f;
  a.all = V <= MAX_CANDIDATES;
  const int waves = n_chunks * WAVES;
  a.groups = !a.k || a.all ? 0 : 4LL * a.k <= waves ? 1 : 4LL * a.k <= 2 * waves ? 2 : 2LL * a.k <= 4 * waves ? 4 : 0;
  return a;
}

// A row in quads of four values on 16 bytes: quad q of a row that begins `lead` values behind such a place holds its values
// 4 q - lead .. + 3.
__device__ __forceinline__ int lead_of(const float* row) { return (int)(((uintptr_t)row >> 2) & 3); }

__device__ __forceinline__ int quads_of_chunk(const float* row, int V, int n_chunks) {
  return ((lead_of(row) + V + 3) / 4 + n_chunks - 1) / n_chunks;
}
// Binary places of a mass in a chunk's histogram: as many as a bin of all of the chunk's values has room for.
__device__ __forceinline__ int places_of(int quads) { return min(20, __builtin_clz(4 * max(1, quads)) - 1); }

__device__ __forceinline__ void quad_range(const float* row, int V, int n_chunks, int c, int* begin, int* end) {
  const int quads = (lead_of(row) + V + 3) / 4, len = quads_of_chunk(row, V, n_chunks);
  *begin = min(quads, c * len);
  *end = min(quads, *begin + len);
}

// f(i, v): the values i .. i + 3 of this thread's quads begin .. end - 1 (places outside the row: NaN).  Four quads are under way at
// a time, none behind a condition; the quads at a row's ends, which may lie in part outside of it, come last, value by value.
template <typename F>
__device__ __forceinline__ void for_quads(const float* __restrict__ row, int V, int begin, int end, F f) {
  constexpr int AT_ONCE = 4;
  const int lead = lead_of(row), first = max(begin, lead ? 1 : 0), until = min(end, (lead + V) / 4);      // the whole quads
  const float* base = row - lead;
  for (int q0 = first + threadIdx.x; q0 < until; q0 += AT_ONCE * THREADS) {
    float4 v[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) v[j] = *reinterpret_cast<const float4*>(base + 4 * (size_t)min(q0 + j * THREADS, until - 1));
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (q0 + j * THREADS < until) f(4 * (q0 + j * THREADS) - lead, v[j]);
  }
  // the first quad of a row that begins inside it, and the last of one that ends inside it
  const int q = threadIdx.x == 0 ? begin : end - 1;
  if (threadIdx.x < 2 && begin < end && (q < first || q >= until) && (threadIdx.x == 0 || end - 1 != begin)) {
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * q - lead + i;
      e[i] = at >= 0 && at < V ? row[at] : __builtin_nanf("");
    }
    f(4 * q - lead, make_float4(e[0], e[1], e[2], e[3]));
  }
}
template <typename F>
__device__ __forceinline__ void for_values(const float* __restrict__ row, int V, int begin, int end, F f) {
  for_quads(row, V, begin, end, [&](int, const float4& v) { f(v.x); f(v.y); f(v.z); f(v.w); });
}

// e^x for x <= 0 by the hardware's exp2, the product with log2(e) in two parts (2 units in the last place); NaN: 0, and below
// e^-200, which no float holds, 0 too.
__device__ __forceinline__ float exp_of(float x) {
  x = fmaxf(x, -200.f);
  const float t = x * 1.44269502f;
  const float r = fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269502f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e * 0.693147181f, r, e);
}

// fixed_mass as a double (NaN: none): a thread adds up to 512 of them without rounding, 2^53, in a third of the instructions.
__device__ __forceinline__ double whole_mass(float s, float zmax) {
  return (double)truncf(expf(fmaxf(s - zmax, -200.f)) * (float)(1ull << FIX_PLACES));
}
constexpr int EXACT_SUMS = 504 * THREADS;      // values a chunk: a thread has four more of an uneven share, and four of a row's end
constexpr double MASS_UNIT = 1.0 / (double)(1ull << FIX_PLACES);

__device__ double block_sum_double(double v, double* red) {
  for (int o = MS_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  __syncthreads();
  if ((threadIdx.x & (MS_WAVE - 1)) == 0) red[threadIdx.x / MS_WAVE] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < WAVES; ++w) s += red[w];
  return s;
}

__device__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* red) {
  for (int o = MS_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  __syncthreads();
  if ((threadIdx.x & (MS_WAVE - 1)) == 0) red[threadIdx.x / MS_WAVE] = v;
  __syncthreads();
  unsigned long long s = 0;
  for (int w = 0; w < WAVES; ++w) s += red[w];
  return s;
}

// Over a row's chunks, a chunk to a lane (a loop over them waits for one after another: 32 of them 10 us).
__device__ __forceinline__ unsigned largest_key(const RowWork& w, int n_chunks) {
  const int lane = threadIdx.x & (MS_WAVE - 1);
  unsigned best = lane < n_chunks ? w.chunk_max[lane] : 0u;
  for (int o = MAX_CHUNKS / 2; o > 0; o >>= 1) best = max(best, (unsigned)__shfl_xor((int)best, o, MS_WAVE));
  return __builtin_amdgcn_readfirstlane(best);
}
__device__ __forceinline__ unsigned long long sum_of(const unsigned long long* chunks, int n_chunks) {
  const int lane = threadIdx.x & (MS_WAVE - 1);
  unsigned long long v = lane < n_chunks ? chunks[lane] : 0ull;
  for (int o = MAX_CHUNKS / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  return __shfl(v, 0, MS_WAVE);
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// ---- 1
__global__ void __launch_bounds__(THREADS)
probabilities_max_kernel(const float* __restrict__ logits, size_t ld, int V, const float* __restrict__ temperature,
                         const int* __restrict__ top_k, const float* __restrict__ top_p, RowWork* __restrict__ work, int n_chunks) {
  __shared__ unsigned red[WAVES];
  __shared__ MaxIdx red_mi[WAVES];
  const int r = blockIdx.y, c = blockIdx.x, lane = threadIdx.x & (MS_WAVE - 1), wave = threadIdx.x / MS_WAVE;
  RowWork& w = work[r];
  const RowPlan a = plan_of(temperature, top_k, top_p, r, V, n_chunks);
  const float* row = logits + (size_t)r * ld;
  int begin, end;
  quad_range(row, V, n_chunks, c, &begin, &end);
  if (a.greedy) {
    MaxIdx best = {-INFINITY, 0x7fffffff};
    for_quads(row, V, begin, end, [&](int i, const float4& v) {
      best = better(best, MaxIdx{v.x, i});
      best = better(best, MaxIdx{v.y, i + 1});
      best = better(best, MaxIdx{v.z, i + 2});
      best = better(best, MaxIdx{v.w, i + 3});
    });
    for (int o = MS_WAVE / 2; o > 0; o >>= 1) best = better(best, MaxIdx{__shfl_xor(best.v, o, MS_WAVE), __shfl_xor(best.i, o, MS_WAVE)});
    if (lane == 0) red_mi[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < WAVES; ++k) best = better(best, red_mi[k]);
      w.chunk_max[c] = __float_as_uint(best.v);
      w.chunk_first[c] = best.i;
    }
    return;
  }
  if (!a.k && !a.use_p) {
    // nothing to look for: the mass with the maximum, every thread's against its own so far, joined against the chunk's
    __shared__ float red_f[WAVES];
    __shared__ double red_d[WAVES];
    float most = -INFINITY;
    double sum = 0.0;
    for_quads(row, V, begin, end, [&](int, const float4& v) {
      const float s[4] = {v.x * a.inv_t, v.y * a.inv_t, v.z * a.inv_t, v.w * a.inv_t};
      const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));      // (NaN never wins)
      if (top > most) {
        sum *= (double)exp_of(most - top);
        most = top;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += (double)exp_of(s[i] - most);
    });
    float best = most;
    for (int o = MS_WAVE / 2; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor(best, o, MS_WAVE));
    if (lane == 0) red_f[wave] = best;
    __syncthreads();
    best = red_f[0];
    for (int k = 1; k < WAVES; ++k) best = fmaxf(best, red_f[k]);
    sum = block_sum_double(sum * (double)exp_of(most - best), red_d);
    if (threadIdx.x == 0) { w.chunk_max[c] = order_key(best); w.chunk_sum[c] = sum; }
    return;
  }
  if (c == 0 && threadIdx.x == 0) { w.n_candidates = 0u; w.n_ties = 0u; w.bin = -1; w.bound = 0u; }
  if (threadIdx.x == 0) { w.chunk_mass[c] = 0ull; w.chunk_above[c] = 0ull; }
  if (a.use_p && !a.k && !a.all)
    for (int i = c * THREADS + threadIdx.x; i < BINS; i += n_chunks * THREADS) w.hist[i] = 0.f;
  unsigned best = 0;
  for_values(row, V, begin, end, [&](float v) {
    const float s = v * a.inv_t;
    best = s == s ? max(best, order_key(s)) : best;     // NaN never wins
  });
  for (int o = 1; o < MS_WAVE; o <<= 1) {
    if (a.groups && o * a.groups == MS_WAVE && (lane & (o - 1)) == 0) w.groups[(c * WAVES + wave) * a.groups + lane / o] = best;
    best = max(best, (unsigned)__shfl_xor((int)best, o, MS_WAVE));
  }
  if (lane == 0) {
    red[wave] = best;
    if (a.groups == 1) w.groups[c * WAVES + wave] = best;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < WAVES; ++k) best = max(best, red[k]);
    w.chunk_max[c] = best;
  }
}

// A block's candidates, gathered here and handed over at once (an addition in memory for each was waited for by its wave).
struct Candidates {
  unsigned n, base, keys[MAX_CANDIDATES];
  __device__ __forceinline__ void add(unsigned key) {
    const unsigned at = atomicAdd(&n, 1u);
    if (at < MAX_CANDIDATES) keys[at] = key;
  }
  __device__ void begin() {      // (the block does these two together)
    if (threadIdx.x == 0) n = 0u;
    __syncthreads();
  }
  __device__ void hand_over(RowWork& w) {
    __syncthreads();
    if (n == 0u) return;
    if (threadIdx.x == 0) base = atomicAdd(&w.n_candidates, n);
    __syncthreads();
    const unsigned at = base + threadIdx.x;
    if (threadIdx.x < n && at < MAX_CANDIDATES) w.candidates[at] = keys[threadIdx.x];
  }
};

// ---- 2
__global__ void __launch_bounds__(THREADS)
probabilities_collect_kernel(const float* __restrict__ logits, size_t ld, int V, const float* __restrict__ temperature,
                             const int* __restrict__ top_k, const float* __restrict__ top_p, RowWork* __restrict__ work, int n_chunks) {
  __shared__ unsigned long long red[WAVES];
  __shared__ unsigned hist[BINS];
  __shared__ Candidates here;
  const int r = blockIdx.y, c = blockIdx.x;
  RowWork& w = work[r];
  const RowPlan a = plan_of(temperature, top_k, top_p, r, V, n_chunks);
  if (a.greedy || (!a.k && !a.use_p)) return;
  const float* row = logits + (size_t)r * ld;
  int begin, end;
  quad_range(row, V, n_chunks, c, &begin, &end);
  const float zmax = key_value(largest_key(w, n_chunks));
  if (!finite(zmax)) return;      // no mass: the last kernel puts a one where the greedy choice stands
  if (a.all) {
    here.begin();
    for_values(row, V, begin, end, [&](float v) {
      const float s = v * a.inv_t;
      if (s == s) here.add(order_key(s));
    });
    here.hand_over(w);
    return;
  }
  if (a.k) {
    if (!a.groups) return;
    // the k-th largest of the group maxima, bit by bit; every wave does it for itself, N keys to a lane
    const int n = n_chunks * WAVES * a.groups, lane = threadIdx.x & (MS_WAVE - 1);
    auto kth = [&](auto size) __attribute__((always_inline)) {
      constexpr int N = decltype(size)::value;
      unsigned key[N], most = 0u, least = 0xffffffffu;
#pragma unroll
      for (int i = 0; i < N; ++i) key[i] = w.groups[min(lane + i * MS_WAVE, n - 1)];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (lane + i * MS_WAVE >= n) key[i] = 0u;         // (the bound of k <= n keys is no smaller for them)
        most = max(most, key[i]);
        least = min(least, key[i]);
      }
      for (int o = MS_WAVE / 2; o > 0; o >>= 1) {
        most = max(most, (unsigned)__shfl_xor((int)most, o, MS_WAVE));
        least = min(least, (unsigned)__shfl_xor((int)least, o, MS_WAVE));
      }
      most = __builtin_amdgcn_readfirstlane(most);
      least = __builtin_amdgcn_readfirstlane(least);
      if (most == least) return most;
      int bit = 31 - __builtin_clz(most ^ least);         // above it all keys are alike
      unsigned prefix = most & ~(0xffffffffu >> (31 - bit));
      for (; bit >= 0; --bit) {
        const unsigned with = prefix | (1u << bit);
        int count = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) count += __builtin_popcountll(__ballot(key[i] >= with));
        if (count >= a.k) prefix = with;
      }
      return prefix;
    };
    const unsigned bound = n <= 4 * MS_WAVE ? kth(std::integral_constant<int, 4>{}) : n <= 8 * MS_WAVE ? kth(std::integral_constant<int, 8>{})
                                                                                    : kth(std::integral_constant<int, MAX_CHUNKS * WAVES * 4 / MS_WAVE>{});
    unsigned ties = 0;
    here.begin();
    for_values(row, V, begin, end, [&](float v) {
      const float s = v * a.inv_t;
      if (!(s == s)) return;
      const unsigned key = order_key(s);
      if (key > bound) here.add(key);
      ties += key == bound;
    });
    here.hand_over(w);
    const unsigned long long all = block_sum_u64(ties, red);
    if (threadIdx.x == 0) {
      if (all) atomicAdd(&w.n_ties, (unsigned)all);
      if (c == 0) w.bound = bound;
    }
    return;
  }
  double mine = 0.0;
  // In LDS a value adds to its bin, as a whole number, what its mass is of the mass at the bin's beginning, e^-f at f behind it (f <
  // 1/128: 1 - f + f^2/2 is off by 2^-23), rounded to the chunk's places.  Float additions in LDS took 5 times as long as whole ones
  // (20 M values into 2,048 bins: 107 us, 23, the reading alone 23).
  const int places = places_of(quads_of_chunk(row, V, n_chunks));
  const float whole = (float)(1 << places);
  for (int i = threadIdx.x; i < BINS; i += THREADS) hist[i] = 0u;
  __syncthreads();
  for_values(row, V, begin, end, [&](float v) {
    const float s = v * a.inv_t, x = (zmax - s) * BINS_A_UNIT;
    mine += whole_mass(s, zmax);
    if (x < (float)BINS) {
      const int bin = (int)x;
      const float f = (x - (float)bin) * (1.0f / BINS_A_UNIT);
      atomicAdd(&hist[bin], (unsigned)(fmaf(fmaf(0.5f, f, -1.0f), f, 1.0f) * whole + 0.5f));
    }
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS)
    if (hist[i]) unsafeAtomicAdd(&w.hist[i], (float)hist[i] / whole * exp_of((float)i * (-1.0f / BINS_A_UNIT)));
  const unsigned long long mass = block_sum_u64((unsigned long long)mine, red);
  if (threadIdx.x == 0) w.chunk_mass[c] = mass;
}

// What the mass of the larger values must not have reached: top_p times the whole, and a unit of mass at least, so that the largest
// value is always kept.
__device__ __forceinline__ unsigned long long target_of(float p, unsigned long long total) {
  const double target = (double)p * (double)total;
  return target >= 1.0 ? (unsigned long long)target : 1ull;
}

// ---- 3
__global__ void __launch_bounds__(THREADS)
probabilities_near_kernel(const float* __restrict__ logits, size_t ld, int V, const float* __restrict__ temperature,
                          const int* __restrict__ top_k, const float* __restrict__ top_p, RowWork* __restrict__ work, int n_chunks) {
  __shared__ unsigned long long red[WAVES];
  __shared__ float wave_sum_sm[WAVES];
  __shared__ int found, up, down;      // the target's bin; the first and the last that count
  __shared__ Candidates here;
  const int r = blockIdx.y, c = blockIdx.x, lane = threadIdx.x & (MS_WAVE - 1), wave = threadIdx.x / MS_WAVE;
  RowWork& w = work[r];
  const RowPlan a = plan_of(temperature, top_k, top_p, r, V, n_chunks);
  if (a.greedy || a.k || !a.use_p || a.all) return;
  const float zmax = key_value(largest_key(w, n_chunks));
  if (!finite(zmax)) return;
  const double whole = (double)sum_of(w.chunk_mass, n_chunks) * MASS_UNIT;
  const float* row = logits + (size_t)r * ld;
  // what the histogram may be off by: a mass by half a place of that at its bin's beginning, e^(1/128) times its own at most (2^-14
  // where one chunk has 152,064 values), and the sums
  const float half = 0.5f / (float)(1 << places_of(quads_of_chunk(row, V, n_chunks)));
  const float target = (float)((double)a.p * whole), near = (float)whole * (half * (1.0f + 1.0f / 64.f) + SUM_ERROR);
  // the first bin at which the running mass reaches the target; a thread owns two bins
  const float h0 = w.hist[2 * threadIdx.x], h1 = w.hist[2 * threadIdx.x + 1];
  float run = h0 + h1;
  for (int o = 1; o < MS_WAVE; o <<= 1) {
    const float v = __shfl_up(run, o, MS_WAVE);
    if (lane >= o) run += v;
  }
  if (lane == MS_WAVE - 1) wave_sum_sm[wave] = run;
  if (threadIdx.x == 0) found = BINS;
  __syncthreads();
  for (int k = 0; k < wave; ++k) run += wave_sum_sm[k];
  if (run >= target) atomicMin(&found, run - h1 >= target ? 2 * (int)threadIdx.x : 2 * (int)threadIdx.x + 1);
  __syncthreads();
  // (sums of floats may fall short of a target that is nearly everything: the last bin that has any would be no surer)
  if (found >= BINS) return;
  if (found >> 1 == (int)threadIdx.x) {
    const float upto = found & 1 ? run : run - h1, from = upto - (found & 1 ? h1 : h0);
    up = target - from < near ? -1 : found;
    down = upto - target < near ? BINS : found;
  }
  __syncthreads();
  if (up < 0 || down == BINS) {
    // a neighbour is the next bin that holds anything: where few tokens have most of the mass, many between them are empty
    const bool before = up < 0, behind = down == BINS;
    __syncthreads();
    if (before && h0 + h1 > 0.f) {
      if (h1 > 0.f && 2 * (int)threadIdx.x + 1 < found) atomicMax(&up, 2 * (int)threadIdx.x + 1);
      else if (h0 > 0.f && 2 * (int)threadIdx.x < found) atomicMax(&up, 2 * (int)threadIdx.x);
    }
    if (behind && h0 + h1 > 0.f) {
      if (h0 > 0.f && 2 * (int)threadIdx.x > found) atomicMin(&down, 2 * (int)threadIdx.x);
      else if (h1 > 0.f && 2 * (int)threadIdx.x + 1 > found) atomicMin(&down, 2 * (int)threadIdx.x + 1);
    }
    __syncthreads();
  }
  const float high = zmax - (float)up * (1.0f / BINS_A_UNIT), low = zmax - (float)(min(down, BINS - 1) + 1) * (1.0f / BINS_A_UNIT);
  if (c == 0 && threadIdx.x == 0) w.bin = found;
  int begin, end;
  quad_range(row, V, n_chunks, c, &begin, &end);
  double above = 0.0;
  here.begin();
  for_values(row, V, begin, end, [&](float v) {
    const float s = v * a.inv_t;
    if (s > high) above += whole_mass(s, zmax);
    else if (s >= low) here.add(order_key(s));
  });
  here.hand_over(w);
  const unsigned long long mass = block_sum_u64((unsigned long long)above, red);
  if (threadIdx.x == 0) w.chunk_above[c] = mass;
}

struct Kept { unsigned floor; unsigned long long mass; };

// The floor among what `each` hands to its function, scaled logits in any order (NaN: nobody), and the mass of what is kept: a radix
// descent of the block over their keys.  `need`, from the mass that top-k keeps, is what the larger values' must not have reached.
template <typename Each, typename Need>
__device__ __forceinline__ Kept descend(const Each& each, int k, bool use_p, const Need& need_of, float zmax, unsigned* lc,
                                        unsigned long long* lm, unsigned long long* red) {
  const int lane = threadIdx.x & (MS_WAVE - 1);
  unsigned long long total = 0;
  // the key at which the running count (or mass) from the top reaches `need`, among keys of at least `least`; total: the mass upto it
  auto search = [&](bool by_mass, unsigned long long need, unsigned least) {
    unsigned digits = 0;
    unsigned long long above = 0, mass = 0;
    for (int level = 1; level <= 3; ++level) {
      const int shift = level_shift(level), bins = level_bins(level);
      __syncthreads();
      for (int i = threadIdx.x; i < bins; i += THREADS) { lc[i] = 0u; lm[i] = 0ull; }
      __syncthreads();
      each([&](float s) {
        const unsigned key = order_key(s);
        const bool in = s == s && key >= least && (level == 1 || (key >> (shift + (level == 2 ? 11 : 10))) == digits);
        const int bin = (int)((key >> shift) & (unsigned)(bins - 1));
        unsigned long long m = in ? fixed_mass(s, zmax) : 0ull;
        const unsigned long long who = __ballot(in);
        if (!who) return;
        const int leader = __builtin_ctzll(who);
        if (__ballot(in && bin != __shfl(bin, leader, MS_WAVE)) == 0 && __builtin_popcountll(__ballot(true)) == MS_WAVE) {
          // one bin for all of them, as in rows of few different values: one addition for the wave
          for (int o = MS_WAVE / 2; o > 0; o >>= 1) m += __shfl_xor(m, o, MS_WAVE);
          if (lane == leader) { atomicAdd(&lc[bin], (unsigned)__builtin_popcountll(who)); atomicAdd(&lm[bin], m); }
        } else if (in) {
          atomicAdd(&lc[bin], 1u);
          atomicAdd(&lm[bin], m);
        }
      });
      __syncthreads();
      const Found f = first_bin_reaching(lc, lm, bins, by_mass, need - above);
      digits = level == 1 ? (unsigned)f.bin : (digits << (level == 2 ? 11 : 10)) | (unsigned)f.bin;
      above += by_mass ? f.mass_above : f.count_above;
      mass += f.mass_above + (level == 3 ? f.mass_in : 0ull);
    }
    total = mass;
    return digits;
  };
  unsigned floor = 0u;
  if (k) {
    floor = search(false, (unsigned long long)k, 0u);
  } else {
    unsigned long long mine = 0ull;
    each([&](float s) { mine += s == s ? fixed_mass(s, zmax) : 0ull; });
    total = block_sum_u64(mine, red);
  }
  if (use_p) {
    const unsigned long long need = need_of(total);
    if (need == 0ull || need > total) return Kept{0u, 0ull};      // (it does not fall among them)
    floor = search(true, need, floor);
  }
  return Kept{floor, total};
}

// ---- 4
__global__ void __launch_bounds__(THREADS)
probabilities_write_kernel(const float* __restrict__ logits, size_t ld, int V, const float* __restrict__ temperature,
                           const int* __restrict__ top_k, const float* __restrict__ top_p, const RowWork* __restrict__ work,
                           int n_chunks, float* __restrict__ out, size_t out_ld) {
  __shared__ MaxIdx red_mi[WAVES];
  __shared__ unsigned long long red[WAVES];
  __shared__ unsigned keys[RADIX_BINS];
  __shared__ unsigned long long masses[RADIX_BINS];
  __shared__ unsigned floor_sm;
  const int r = blockIdx.y, c = blockIdx.x;
  const RowWork& w = work[r];
  const RowPlan a = plan_of(temperature, top_k, top_p, r, V, n_chunks);
  const float* row = logits + (size_t)r * ld;
  float* to = out + (size_t)r * out_ld;
  int begin, end;
  quad_range(row, V, n_chunks, c, &begin, &end);
  // four values of the row's quads at a time where out's rows lie as the logits' do
  const bool alike = lead_of(row) == lead_of(to);
  auto store = [&](int i, const float4& v) {
    if (alike && i >= 0 && i + 3 < V) {
      *reinterpret_cast<float4*>(to + i) = v;
    } else {
      const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j >= 0 && i + j < V) to[i + j] = e[j];
    }
  };
  const unsigned top = a.greedy ? 0u : largest_key(w, n_chunks);
  const float zmax = a.greedy ? 0.f : key_value(top);
  int one = -1;
  if (a.greedy) {
    const int lane = threadIdx.x & (MS_WAVE - 1);
    MaxIdx best = {-INFINITY, 0x7fffffff};
    if (lane < n_chunks) best = MaxIdx{__uint_as_float(w.chunk_max[lane]), w.chunk_first[lane]};
    for (int o = MAX_CHUNKS / 2; o > 0; o >>= 1) best = better(best, MaxIdx{__shfl_xor(best.v, o, MS_WAVE), __shfl_xor(best.i, o, MS_WAVE)});
    best.i = __shfl(best.i, 0, MS_WAVE);
    one = best.i == 0x7fffffff ? 0 : best.i;
  } else if (!finite(zmax)) {
    const MaxIdx best = block_argmax(row, 0, V, red_mi);
    one = best.i == 0x7fffffff ? 0 : best.i;
  }
  if (one >= 0) {
    const int lead = lead_of(row);
    for (int q = begin + threadIdx.x; q < end; q += THREADS) {
      const int i = 4 * q - lead;
      store(i, make_float4(i == one ? 1.f : 0.f, i + 1 == one ? 1.f : 0.f, i + 2 == one ? 1.f : 0.f, i + 3 == one ? 1.f : 0.f));
    }
    return;
  }

  Kept kept = {0u, 0ull};
  double kept_sum;
  if (!a.k && !a.use_p) {
    const int lane = threadIdx.x & (MS_WAVE - 1);
    double v = lane < n_chunks ? w.chunk_sum[lane] * (double)exp_of(key_value(w.chunk_max[lane]) - zmax) : 0.0;
    for (int o = MAX_CHUNKS / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
    kept_sum = __shfl(v, 0, MS_WAVE);
  } else {
    // A candidate knows how many are larger, and their mass.  Top-k keeps it if these are fewer than k; top-p if what is larger has
    // not reached the target.  Values equal to the bound are one candidate more, as often as they were counted.
    const int n = (int)w.n_candidates;
    bool known = n <= MAX_CANDIDATES && (a.all || (a.k ? a.groups > 0 : w.bin >= 0));
    const bool tied = a.k && !a.all, above_them = !a.k && !a.all;
    const unsigned ties = tied ? w.n_ties : 0u, bound = w.bound;
    const unsigned long long tie_mass = tied ? ties * fixed_mass(key_value(bound), zmax) : 0ull;
    const bool ties_in_k = ties > 0 && n < a.k;
    const unsigned long long above = above_them ? sum_of(w.chunk_above, n_chunks) : 0ull, whole = above_them ? sum_of(w.chunk_mass, n_chunks) : 0ull;
    unsigned mine = 0u;
    unsigned long long mass = 0ull, larger = 0ull;
    unsigned count = 0;
    if (known && n <= MS_WAVE) {
      // few enough for a wave: every wave of the block does it for itself
      const int lane = threadIdx.x & (MS_WAVE - 1);
      if (lane < n) {
        mine = w.candidates[lane];
        mass = fixed_mass(key_value(mine), zmax);
      }
      for (int j = 0; j < n; ++j) {
        const unsigned key = __builtin_amdgcn_readlane(mine, j);
        const unsigned hi = __builtin_amdgcn_readlane((unsigned)(mass >> 32), j), lo = __builtin_amdgcn_readlane((unsigned)mass, j);
        const unsigned long long theirs = ((unsigned long long)hi << 32) | lo;
        count += key > mine;
        larger += key > mine ? theirs : 0ull;
      }
      const auto sum = [&](unsigned long long v) {
        for (int o = MS_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
        return v;
      };
      bool in = lane < n && (!a.k || count < (unsigned)a.k), ties_in = ties_in_k;
      unsigned long long kept_mass = sum(in ? mass : 0ull) + (ties_in ? tie_mass : 0ull);
      if (a.use_p) {
        const unsigned long long target = target_of(a.p, above_them ? whole : kept_mass);
        known = above < target && above + kept_mass >= target;      // (it falls among the candidates)
        ties_in = ties_in && kept_mass - tie_mass < target;
        in = in && above + larger < target;
        kept_mass = sum(in ? mass : 0ull) + (ties_in ? tie_mass : 0ull);
      }
      unsigned floor = in ? mine : 0xffffffffu;
      for (int o = MS_WAVE / 2; o > 0; o >>= 1) floor = min(floor, (unsigned)__shfl_xor((int)floor, o, MS_WAVE));
      kept = Kept{ties_in ? min(floor, bound) : floor, above + kept_mass};
    } else if (known && !tied) {
      // many, and each of them itself: the descent over them (one row of 151,936 normal logits, top-p 0.9 at temperatures 0.7 and 3:
      // 36 and 38 us; when they took 41 and 45, compared with each other 58 and 100)
      const float s = (int)threadIdx.x < n ? key_value(w.candidates[threadIdx.x]) : NAN;
      kept = descend([&](auto f) { f(s); }, a.k, a.use_p, [&](unsigned long long total) -> unsigned long long {
        if (!above_them) return target_of(a.p, total);
        const unsigned long long target = target_of(a.p, whole);
        return target > above && target - above <= total ? target - above : 0ull;
      }, zmax, keys, masses, red);
      known = kept.mass > 0ull;
      kept.mass += above;
    } else if (known) {
      if ((int)threadIdx.x < n) {
        mine = w.candidates[threadIdx.x];
        mass = fixed_mass(key_value(mine), zmax);
        keys[threadIdx.x] = mine;
        masses[threadIdx.x] = mass;
      }
      if (threadIdx.x == 0) floor_sm = 0xffffffffu;
      __syncthreads();
      if ((int)threadIdx.x < n)
        for (int j = 0; j < n; ++j)
          if (keys[j] > mine) { ++count; larger += masses[j]; }
      bool in = (int)threadIdx.x < n && (!a.k || count < (unsigned)a.k), ties_in = ties_in_k;
      unsigned long long kept_mass = block_sum_u64(in ? mass : 0ull, red) + (ties_in ? tie_mass : 0ull);
      if (a.use_p) {
        const unsigned long long target = target_of(a.p, kept_mass);
        ties_in = ties_in && kept_mass - tie_mass < target;
        in = in && larger < target;
        kept_mass = block_sum_u64(in ? mass : 0ull, red) + (ties_in ? tie_mass : 0ull);
      }
      if (in) atomicMin(&floor_sm, mine);
      __syncthreads();
      kept = Kept{ties_in ? min(floor_sm, bound) : floor_sm, kept_mass};
    }
    if (!known) {
      const int quads = (lead_of(row) + V + 3) / 4;
      kept = descend([&](auto f) { for_values(row, V, 0, quads, [&](float v) { f(v * a.inv_t); }); }, a.k, a.use_p,
                     [&](unsigned long long total) { return target_of(a.p, total); }, zmax, keys, masses, red);
    }
    kept_sum = (double)kept.mass * MASS_UNIT;
  }
  const float inv = (float)(1.0 / kept_sum), floor = kept.floor ? key_value(kept.floor) : -INFINITY;
  for_quads(row, V, begin, end, [&](int i, const float4& v) {
    auto value = [&](float x) {
      const float s = x * a.inv_t;
      return s >= floor ? exp_of(s - zmax) * inv : 0.f;
    };
    store(i, make_float4(value(v.x), value(v.y), value(v.z), value(v.w)));
  });
}

}  // namespace

// Bytes of workspace ms_probabilities needs for n_rows rows (any contents: the first kernel makes it ready).
extern "C" long long ms_probabilities_workspace_bytes(int n_rows) { return (long long)sizeof(RowWork) * (n_rows > 0 ? n_rows : 0); }

// out[r, :] = the distribution ms_sample would draw row r's token from; arguments as there.
extern "C" int ms_probabilities(const float* logits, long long ld, int n_rows, int vocab, const float* temperature,
                                const int* top_k, const float* top_p, float* out, long long out_ld, void* workspace,
                                int use_top_k, int use_top_p, hipStream_t stream) {
  if (n_rows <= 0) return MS_OK;
  if (vocab <= 0 || ld < vocab || out_ld < vocab || n_rows > 65535 || temperature == nullptr) return MS_BAD_ARG;
  if (workspace == nullptr || ((uintptr_t)workspace % 8)) return MS_BAD_ARG;
  RowWork* work = (RowWork*)workspace;
  if (!use_top_k) top_k = nullptr;
  if (!use_top_p) top_p = nullptr;
  // about two blocks a CU
  int n_chunks = (2 * ms_compute_units() + n_rows - 1) / n_rows;
  n_chunks = std::max(1, std::min(std::min(n_chunks, MAX_CHUNKS), (vocab + 2047) / 2048));
  n_chunks = std::max(n_chunks, std::min((vocab - 1) / EXACT_SUMS + 1, MAX_CHUNKS));
  const dim3 grid(n_chunks, n_rows), block(THREADS);
  probabilities_max_kernel<<<grid, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_k, top_p, work, n_chunks);
  if (top_k || top_p) probabilities_collect_kernel<<<grid, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_k, top_p, work, n_chunks);
  if (top_p) probabilities_near_kernel<<<grid, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_k, top_p, work, n_chunks);
  probabilities_write_kernel<<<grid, block, 0, stream>>>(logits, (size_t)ld, vocab, temperature, top_k, top_p, work, n_chunks, out, (size_t)out_ld);
  return ms_launch_status();
}
