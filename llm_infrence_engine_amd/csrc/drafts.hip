// What decides about a step's drafted tokens, and what moves the entries of those that stay.
//
// Verification.  The tokens of a request's tree are numbered so that a parent comes before its children; token 0 is the
// root, the request's last token.  Row n of p is the distribution the target model gives behind token n, row n of q the one
// the children of n were drawn from, independently of each other.  From the root down, the children of the last accepted
// token are tried in the order of their numbers.  Behind j refusals what is left of the target is max(0, p - t q) / S, with
//
//   t = 0, S = 1 at first;    on a refusal  t += S,  S = sum_x max(0, p(x) - t q(x))
//
// (max(0, max(0, p - t q) / S - q) is max(0, p - (t + S) q) / S), so a child x with the number u is accepted if
// u q(x) S < p(x) - t q(x), and the accepted or finally drawn token is distributed as p whatever q is.  Where the last child
// is refused, or there is none, the request's next token is drawn from max(0, p - t q) by the root's number: the first whose
// sum in index order exceeds that number times the whole.  Without q a child stands for itself (q is one there): it is
// accepted if u S < p(x), and a refusal takes p(x) out of p and S.  Products and sums are double: u q is then exact, and
// where a token is drawn hangs on a sum over the vocabulary.
//
// What costs is the sums over the vocabulary, one after another along a path (a refusal, a sum, the next child) where each needs a
// row of p and of q; everything between them hangs on a few numbers.  A block that does them alone draws 1.2 MB a sum at the rate
// of one CU (verification of a tree of 8 behind a vocabulary of 151,936: 130 us).  So a request has up to 32 blocks: its first,
// the leader, walks the tree and says which sum is needed next (the row, t); every block sums its chunk of the vocabulary; the
// leader adds the chunks up in order.  Orders and sums travel as 64-bit words of a value and the order's number, stored and polled
// past the L2s, so there is no fence, and a word of an earlier order is never taken for one of this (a kernel in front clears
// them).  Waits are bounded: a leader that has not heard from a chunk sums it up itself, then and from then on, so it never
// depends on a block that may not be running; helpers wait for a block launched before them, and not for ever.
#include "common.h"
#include "api.h"
#include <algorithm>

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 1024, WAVES = THREADS / MS_WAVE;
constexpr int MAX_TENSORS = 16;
constexpr int MAX_CHUNKS = 32;
constexpr int MAX_KNOWN = 1024;              // tokens of a tree (children of a token) that LDS has room for
constexpr int ORDER_WORDS = 4;               // of a request's words the order's, then two of every chunk
constexpr int REQUEST_WORDS = ORDER_WORDS + 2 * MAX_CHUNKS;
constexpr unsigned WHOLE = 0x80000000u, NONE = 0xffffffffu;      // of an order's row: p itself; no further order

__device__ __forceinline__ void put(u64* word, unsigned value, unsigned tag) {
  __hip_atomic_store((__attribute__((address_space(1))) u64*)word, ((u64)tag << 32) | value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 look(const u64* word) {
  return __hip_atomic_load((const __attribute__((address_space(1))) u64*)word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ void __launch_bounds__(256) clear_words_kernel(u64* __restrict__ words, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) words[i] = 0ull;
}

__device__ __forceinline__ double block_sum_double(double v, double* red) {
  for (int o = MS_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  __syncthreads();
  if ((threadIdx.x & (MS_WAVE - 1)) == 0) red[threadIdx.x / MS_WAVE] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < WAVES; ++w) s += red[w];
  return s;
}

// The chunks' sums added up in a fixed order, a chunk to a lane.
__device__ __forceinline__ double sum_of(const double* part, int n) {
  const int lane = threadIdx.x & (MS_WAVE - 1);
  double v = lane < n ? part[lane] : 0.0;
  for (int o = MAX_CHUNKS / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  return __shfl(v, 0, MS_WAVE);
}

// What is left of a row of the target: max(0, p - t q); without q p without the tokens of `gone` (of which, with `parents`, those
// of `parent` count).
struct Rest {
  const float *p, *q;
  double t;
  const int *gone, *parents;
  int n_gone, parent;
  __device__ __forceinline__ double weight(float pe, float qe, int e) const {
    const double v = pe;
    if (q) return fmax(0.0, v - t * (double)qe);
    for (int j = 0; j < n_gone; ++j)
      if (gone[j] == e && (!parents || parents[j] == parent)) return 0.0;
    return v;
  }
};

// A thread's share of the sum over lo .. hi - 1, four entries under way at a time.
__device__ __forceinline__ double share_of(const Rest& rest, int lo, int hi) {
  constexpr int AT_ONCE = 4;
  double sum = 0.0;
  for (int e0 = lo + (int)threadIdx.x; e0 < hi; e0 += AT_ONCE * THREADS) {
    float pe[AT_ONCE], qe[AT_ONCE] = {};
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) pe[j] = rest.p[min(e0 + j * THREADS, hi - 1)];
    if (rest.q) {
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) qe[j] = rest.q[min(e0 + j * THREADS, hi - 1)];
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (e0 + j * THREADS < hi) sum += rest.weight(pe[j], qe[j], e0 + j * THREADS);
  }
  return sum;
}

__global__ void __launch_bounds__(THREADS)
verify_drafts_kernel(const float* __restrict__ p, const float* __restrict__ q, int V, const int* __restrict__ tokens,
                     const int* __restrict__ parents, const int* __restrict__ q_start, const float* __restrict__ uniforms,
                     int* __restrict__ nodes, int depth, int* __restrict__ counts, int* __restrict__ out, u64* __restrict__ words,
                     int n_chunks, int patience) {
  __shared__ double red[WAVES], part[MAX_CHUNKS], order_t;
  __shared__ int known_parent[MAX_KNOWN], known_token[MAX_KNOWN], gone[MAX_KNOWN];
  __shared__ float known_u[MAX_KNOWN], known_p[MAX_KNOWN], known_q[MAX_KNOWN];
  __shared__ int n_gone, first_e, last_e;
  __shared__ unsigned order_row, missing;
  const int r = blockIdx.x / n_chunks, c = blockIdx.x - r * n_chunks, lane = threadIdx.x & (MS_WAVE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MS_WAVE);
  const int t0 = q_start[r], length = q_start[r + 1] - t0;
  u64* mine = words + (size_t)r * REQUEST_WORDS;
  const int len = (V + n_chunks - 1) / n_chunks;
  const auto lo_of = [&](int k) { return (int)min((long long)V, (long long)k * len); };

  // what an order's sum is over (the whole block calls this)
  const auto rest_of = [&](unsigned row, double t) {
    const int node = (int)(row & ~WHOLE);
    Rest rest = {p + (size_t)(t0 + node) * V, nullptr, t, gone, nullptr, 0, node};
    if (row & WHOLE) return rest;
    if (q) { rest.q = q + (size_t)(t0 + node) * V; return rest; }
    __syncthreads();
    if (threadIdx.x == 0) n_gone = 0;
    __syncthreads();
    for (int i = node + 1 + (int)threadIdx.x; i < length; i += THREADS)
      if (parents[t0 + i] == node) {
        const int at = atomicAdd(&n_gone, 1);
        if (at < MAX_KNOWN) gone[at] = tokens[t0 + i];
      }
    __syncthreads();
    rest.n_gone = n_gone;
    if (rest.n_gone > MAX_KNOWN) {
      rest.gone = tokens + t0 + node + 1;
      rest.parents = parents + t0 + node + 1;
      rest.n_gone = length - node - 1;
    }
    return rest;
  };

  if (c > 0) {
    // ---- a helper: its chunk of every order's sum, until there is no further order
    unsigned tag = 0;
    for (;;) {
      if (wave == 0) {
        unsigned row = NONE, hi = 0, lo = 0;
        for (int looks = 0;; ++looks) {
          const u64 word = look(mine + min(lane, 2));
          const unsigned theirs = (unsigned)(word >> 32), first = __builtin_amdgcn_readfirstlane(theirs);
          if (first > tag && __ballot(theirs != first) == 0) {      // an order, all of its words
            tag = first;
            row = __builtin_amdgcn_readlane((unsigned)word, 0);
            hi = __builtin_amdgcn_readlane((unsigned)word, 1);
            lo = __builtin_amdgcn_readlane((unsigned)word, 2);
            break;
          }
          if (looks >= (1 << 21)) break;                            // (seconds; the leader does without)
          __builtin_amdgcn_s_sleep(1);
        }
        if (lane == 0) { order_row = row; order_t = __longlong_as_double((long long)(((u64)hi << 32) | lo)); }
      }
      __syncthreads();
      const unsigned row = order_row;
      const double t = order_t;
      if (row == NONE) return;
      const Rest rest = rest_of(row, t);
      const u64 sum = (u64)__double_as_longlong(block_sum_double(share_of(rest, lo_of(c), lo_of(c + 1)), red));
      if (threadIdx.x < 2) put(mine + ORDER_WORDS + 2 * c + threadIdx.x, (unsigned)(threadIdx.x ? sum : sum >> 32), tag);
    }
  }

  // ---- the leader
  int* path = nodes + (size_t)r * depth;
  unsigned tag = 0;
  const auto say = [&](unsigned row, double t) {      // (lanes 0 to 2 of wave 0)
    const u64 bits = (u64)__double_as_longlong(t);
    if (lane < 3) put(mine + lane, lane == 0 ? row : (unsigned)(lane == 1 ? bits >> 32 : bits), tag);
  };
  if (length <= 0) {      // a request that pads a captured batch
    tag = 1;
    if (wave == 0) say(NONE, 0.0);
    for (int i = threadIdx.x; i < depth; i += THREADS) path[i] = -1;
    if (threadIdx.x == 0) { counts[r] = 0; out[r] = -1; }
    return;
  }
  const bool in_lds = length <= MAX_KNOWN;
  if (in_lds)
    for (int i = threadIdx.x; i < length; i += THREADS) {
      const int up = parents[t0 + i], x = tokens[t0 + i];
      const bool fits = i > 0 && up >= 0 && up < i && x >= 0 && x < V;
      const size_t at = (size_t)(t0 + (fits ? up : 0)) * V + (fits ? x : 0);
      known_parent[i] = fits ? up : -1;      // (a guess that is no token is nobody's)
      known_token[i] = x;
      known_u[i] = uniforms[t0 + i];
      known_p[i] = p[at];
      known_q[i] = q ? q[at] : 1.f;
    }
  if (threadIdx.x == 0) missing = 0u;
  for (int i = 1 + (int)threadIdx.x; i < depth; i += THREADS) path[i] = -1;
  __syncthreads();

  // (wave 0's)
  const auto is_child = [&](int i, int node) {
    if (i >= length) return false;
    if (in_lds) return known_parent[i] == node;
    const int x = tokens[t0 + i];
    return parents[t0 + i] == node && x >= 0 && x < V;
  };
  const auto token_of = [&](int i) { return in_lds ? known_token[i] : tokens[t0 + i]; };
  int node = 0, next = 1, count = 1;
  bool tried = false, summed = false, whole = false;      // a child was refused here; the sum over what is left is known; it is of p
  unsigned row = NONE;                                    // the last order
  double t = 0.0, S = 1.0;
  for (;;) {
    if (wave == 0) {
      unsigned row = NONE;
      while (row == NONE) {
        int child = length;
        if (count < depth)
          for (int base = next; base < length; base += MS_WAVE) {
            const u64 hit = __ballot(is_child(base + lane, node));
            if (hit) { child = base + __builtin_ctzll(hit); break; }
          }
        if (child >= length) {             // the path ends here
          if (!summed) whole = !tried;
          else if (S > 0.0 || whole) break;
          else whole = true;               // nothing is left: the target's own distribution
          row = (unsigned)node | (whole ? WHOLE : 0u);
          break;
        }
        next = child + 1;
        const int x = token_of(child);
        const double u = in_lds ? known_u[child] : uniforms[t0 + child];
        const size_t at = (size_t)(t0 + node) * V + x;
        double px = in_lds ? known_p[child] : p[at];
        bool taken;
        if (q) {
          const double qx = in_lds ? known_q[child] : q[at];
          taken = u * qx * S < px - t * qx;
        } else {
          u64 twin = 0;                    // a guess that was refused already has nothing left
          for (int base = node + 1; base < child && !twin; base += MS_WAVE)
            twin = __ballot(base + lane < child && is_child(base + lane, node) && token_of(base + lane) == x);
          if (twin) px = 0.0;
          taken = u * S < px;
        }
        if (taken) {
          node = child;
          if (lane == 0) path[count] = node;
          ++count;
          t = 0.0; S = 1.0; tried = summed = whole = false;
        } else {
          tried = true;
          if (q) {
            t += S;
            row = (unsigned)node;
          } else {
            S -= px;
          }
        }
      }
      ++tag;
      if (lane == 0) { order_row = row; order_t = t; }
      if (row != NONE) say(row, t);
    }
    __syncthreads();
    if (order_row == NONE) break;
    row = order_row;
    const Rest rest = rest_of(row, order_t);
    const double own = block_sum_double(share_of(rest, 0, lo_of(1)), red);
    if (wave == 0) {
      // the other chunks, a lane each
      const bool absent = lane < n_chunks && ((missing >> lane) & 1u);
      double sum = own;
      bool have = lane >= n_chunks || lane == 0;
      for (int looks = 0; looks < patience; ++looks) {
        if (!have && !absent) {
          const u64 hi = look(mine + ORDER_WORDS + 2 * lane), lo = look(mine + ORDER_WORDS + 2 * lane + 1);
          if ((unsigned)(hi >> 32) == tag && (unsigned)(lo >> 32) == tag) {
            sum = __longlong_as_double((long long)((hi << 32) | (lo & 0xffffffffu)));
            have = true;
          }
        }
        if (__ballot(!have && !absent) == 0) break;
        __builtin_amdgcn_s_sleep(1);
      }
      if (lane < n_chunks) part[lane] = sum;
      const u64 gap = __ballot(!have);
      if (lane == 0) missing = (unsigned)gap;
    }
    __syncthreads();
    for (unsigned todo = missing; todo; todo &= todo - 1) {
      const int k = __builtin_ctz(todo);
      const double sum = block_sum_double(share_of(rest, lo_of(k), lo_of(k + 1)), red);
      if (threadIdx.x == 0) part[k] = sum;
    }
    __syncthreads();
    S = sum_of(part, n_chunks);
    summed = true;
    __syncthreads();
  }
  if (wave == 0) say(NONE, 0.0);           // (the tag was counted up for it)

  // ---- the token behind the path: the chunk in which the mark falls, then the first entry that passes it, 4,096 at a time
  const Rest rest = rest_of(row, order_t);
  const double target = (double)uniforms[t0] * S;
  double upto = lane < n_chunks ? part[lane] : 0.0;      // sums over the chunks, one to a lane
  const double mass = upto;
  for (int o = 1; o < MAX_CHUNKS; o <<= 1) {
    const double v = __shfl_up(upto, o, MS_WAVE);
    if (lane >= o) upto += v;
  }
  const u64 passing_chunks = __ballot(lane < n_chunks && mass > 0.0 && upto > target), some_chunks = __ballot(lane < n_chunks && mass > 0.0);
  // (a sum in this order may stay below the mark: then the last chunk that has any)
  const int chunk = passing_chunks ? __builtin_ctzll(passing_chunks) : some_chunks ? 63 - __builtin_clzll(some_chunks) : 0;
  double run = __shfl(upto - mass, chunk, MS_WAVE);
  if (threadIdx.x == 0) { first_e = V; last_e = -1; }
  __syncthreads();
  const int hi = lo_of(chunk + 1);
  for (int base = lo_of(chunk); base < hi; base += 4 * THREADS) {
    const int e0 = base + 4 * (int)threadIdx.x;
    double w[4], here = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = min(e0 + j, hi - 1);
      w[j] = rest.weight(rest.p[e], rest.q ? rest.q[e] : 0.f, e);
      if (e0 + j >= hi) w[j] = 0.0;
      here += w[j];
    }
    double here_upto = here;               // sums over the threads before, in index order
    for (int o = 1; o < MS_WAVE; o <<= 1) {
      const double v = __shfl_up(here_upto, o, MS_WAVE);
      if (lane >= o) here_upto += v;
    }
    __syncthreads();
    if (lane == MS_WAVE - 1) red[wave] = here_upto;
    __syncthreads();
    double before = run, all = 0.0;
    for (int k = 0; k < WAVES; ++k) {
      if (k < wave) before += red[k];
      all += red[k];
    }
    double sum = before + here_upto - here;
    int passes = V, some = -1;             // the thread's first entry that passes the mark, its last that has any weight
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sum += w[j];
      if (w[j] > 0.0) {
        if (sum > target) passes = min(passes, e0 + j);
        some = e0 + j;
      }
    }
    const u64 passing = __ballot(passes < V), weighty = __ballot(some >= 0);
    if (passing && lane == __builtin_ctzll(passing)) atomicMin(&first_e, passes);
    if (weighty && lane == 63 - __builtin_clzll(weighty)) atomicMax(&last_e, some);
    __syncthreads();
    if (first_e < V) break;                // (the same for all)
    run += all;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    path[0] = 0;
    out[r] = first_e < V ? first_e : max(last_e, 0);
    counts[r] = count;
  }
}

// Entry first[r] + nodes[r][i] of request r's cache to first[r] + i, for i < counts[r], in every layer and head.  A path is
// increasing, so an entry moves to an earlier place, and a place that has been written is the source of no later entry: a wave may
// take entries in order as long as it has read a group of them before it writes that group.
// A block works a request's moves out once (where they lie: table and pages) and its waves then walk (layer, head) pairs of one
// tensor; where each thread did it for itself it waited for path, table and entry one after another (32 requests, 64 layers of 8
// heads of 128 in bfloat16: 98 us).  In transposed pages an entry is one value of every row, so what has to be read and written
// is all lines of its page's part of a head: 184 MB read and 102 written for those 75, 61 us as a copy takes them.  There a wave reads a row's 32 bytes
// around the moves' places, puts the values in and writes the 32 bytes back, whole lines for memory (68 us; value by value 74).
struct KeepTensor {
  void* pages;
  int heads, width, transposed, none;
};
struct KeepTensors { KeepTensor t[MAX_TENSORS]; };

constexpr int KEEP_WAVES = 4;

template <typename T>
__global__ void __launch_bounds__(KEEP_WAVES * MS_WAVE)
keep_tokens_kernel(KeepTensors tensors, int layers, int num_pages, int page_size, const int* __restrict__ block_table,
                   int table_stride, const int* __restrict__ table_rows, const int* __restrict__ first,
                   const int* __restrict__ nodes, int depth, const int* __restrict__ counts) {
  __shared__ int from_page[MS_WAVE], from_slot[MS_WAVE], to_page[MS_WAVE], to_slot[MS_WAVE], n_moves;
  const KeepTensor kt = tensors.t[blockIdx.z];
  const int r = blockIdx.y, lane = threadIdx.x & (MS_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MS_WAVE);
  const int count = min(counts[r], depth), base = first[r];
  const int* table = block_table + (size_t)(table_rows ? table_rows[r] : r) * table_stride;
  const int* path = nodes + (size_t)r * depth;
  const int pairs = layers * kt.heads, width = kt.width;
  const size_t page_values = (size_t)kt.heads * page_size * width, layer_values = page_values * num_pages;
  const bool pieces = !kt.transposed && width * sizeof(T) % 16 == 0 && (uintptr_t)kt.pages % 16 == 0;
  const bool segments = kt.transposed && page_size * sizeof(T) % 32 == 0 && (uintptr_t)kt.pages % 16 == 0;
  for (int i0 = 0; i0 < count; i0 += MS_WAVE) {
    if (wave == 0) {
      const int i = i0 + lane;
      int fp = 0, fs = 0, tp = 0, ts = 0;
      bool moves = false;
      if (i < count) {
        const long long from = (long long)base + path[i], to = (long long)base + i;
        moves = path[i] > i && to >= 0 && from / page_size < table_stride;
        if (moves) {
          fp = table[from / page_size]; fs = (int)(from % page_size);
          tp = table[to / page_size]; ts = (int)(to % page_size);
          moves = fp > 0 && fp < num_pages && tp > 0 && tp < num_pages;      // (the null page, pages of no pool: left alone)
        }
      }
      const unsigned long long who = __ballot(moves);
      if (moves) {
        const int at = __builtin_popcountll(who & ((1ull << lane) - 1));
        from_page[at] = fp; from_slot[at] = fs; to_page[at] = tp; to_slot[at] = ts;
      }
      if (lane == 0) n_moves = __builtin_popcountll(who);
    }
    __syncthreads();
    const int n = n_moves;
    for (int lh = blockIdx.x * KEEP_WAVES + wave; lh < pairs; lh += gridDim.x * KEEP_WAVES) {
      const int layer = lh / kt.heads, head = lh - layer * kt.heads;
      T* const at = (T*)kt.pages + layer * layer_values + (size_t)head * page_size * width;
      if (pieces) {
        constexpr int GROUP = 4;
        const int per = width * (int)sizeof(T) / 16, total = n * per;
        for (int x0 = lane; x0 - lane < total; x0 += GROUP * MS_WAVE) {
          uint4 v[GROUP];
          size_t to[GROUP];
#pragma unroll
          for (int g = 0; g < GROUP; ++g) {
            const int x = min(x0 + g * MS_WAVE, total - 1), m = x / per, e = (x - m * per) * (16 / (int)sizeof(T));
            to[g] = to_page[m] * page_values + (size_t)to_slot[m] * width + e;
            v[g] = *reinterpret_cast<const uint4*>(at + from_page[m] * page_values + (size_t)from_slot[m] * width + e);
          }
#pragma unroll
          for (int g = 0; g < GROUP; ++g)
            if (x0 + g * MS_WAVE < total) *reinterpret_cast<uint4*>(at + to[g]) = v[g];
        }
      } else if (segments) {
        constexpr int SEG = 32 / sizeof(T), GROUP = 4;      // slots of a segment, moves at a time
        for (int m0 = 0; m0 < n;) {
          const int page = to_page[m0], seg = to_slot[m0] / SEG;
          int m1 = m0 + 1;
          while (m1 < n && to_page[m1] == page && to_slot[m1] / SEG == seg) ++m1;
          for (int e = lane; e < width; e += MS_WAVE) {
            T* const place = at + page * page_values + (size_t)e * page_size + seg * SEG;
            union { uint4 q[2]; T v[SEG]; } row;
            row.q[0] = reinterpret_cast<const uint4*>(place)[0];
            row.q[1] = reinterpret_cast<const uint4*>(place)[1];
            for (int m = m0; m < m1; m += GROUP) {
              T v[GROUP];
#pragma unroll
              for (int i = 0; i < GROUP; ++i) {
                const int k = min(m + i, m1 - 1);
                v[i] = at[from_page[k] * page_values + (size_t)e * page_size + from_slot[k]];
              }
#pragma unroll
              for (int i = 0; i < GROUP; ++i) {
                const int slot = __builtin_amdgcn_readfirstlane(m + i < m1 ? to_slot[m + i] % SEG : SEG);      // the same for the wave
#pragma unroll
                for (int k = 0; k < SEG; ++k)
                  if (k == slot) row.v[k] = v[i];
              }
            }
            reinterpret_cast<uint4*>(place)[0] = row.q[0];
            reinterpret_cast<uint4*>(place)[1] = row.q[1];
          }
          m0 = m1;
        }
      } else {
        constexpr int GROUP = 8;
        const int total = n * width;
        const size_t along = kt.transposed ? page_size : 1, slot = kt.transposed ? 1 : width;
        for (int x0 = lane; x0 - lane < total; x0 += GROUP * MS_WAVE) {
          T v[GROUP];
          size_t to[GROUP];
#pragma unroll
          for (int g = 0; g < GROUP; ++g) {
            const int x = min(x0 + g * MS_WAVE, total - 1), m = x / width, e = x - m * width;
            to[g] = to_page[m] * page_values + to_slot[m] * slot + e * along;
            v[g] = at[from_page[m] * page_values + from_slot[m] * slot + e * along];
          }
#pragma unroll
          for (int g = 0; g < GROUP; ++g)
            if (x0 + g * MS_WAVE < total) at[to[g]] = v[g];
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace

// Blocks to a request: about one a CU, and a thousand entries of the vocabulary to each.
static int verify_chunks(int n_requests, int vocab) {
  const int n = std::min(ms_compute_units() / std::max(1, n_requests), (vocab + THREADS - 1) / THREADS);
  return std::max(1, std::min(n, MAX_CHUNKS));
}

static int g_patience = 64;      // looks at what has not come (about 50 us)

// Tests: how often a leader looks for the other blocks' sums before it works them out itself (0 restores the choice; < 0: never).
extern "C" void ms_verify_drafts_patience(int looks) { g_patience = looks < 0 ? 0 : looks ? looks : 64; }

// Bytes of workspace ms_verify_drafts needs for n_requests (any contents).
extern "C" long long ms_verify_drafts_workspace_bytes(int n_requests) { return (long long)sizeof(u64) * REQUEST_WORDS * (n_requests > 0 ? n_requests : 0); }

extern "C" int ms_verify_drafts(const float* p, const float* q, int n_tokens, int vocab, const int* tokens, const int* parents,
                                const int* q_start, const float* uniforms, int n_requests, int* nodes, int depth, int* counts,
                                int* out, void* workspace, hipStream_t stream) {
  if (n_requests <= 0) return MS_OK;
  if (n_tokens < 0 || vocab <= 0 || depth <= 0 || n_requests > 65535) return MS_BAD_ARG;
  if (workspace == nullptr || ((uintptr_t)workspace % 8)) return MS_BAD_ARG;
  const int n_chunks = verify_chunks(n_requests, vocab), n_words = n_requests * REQUEST_WORDS;
  if (n_chunks > 1) clear_words_kernel<<<dim3((n_words + 255) / 256), dim3(256), 0, stream>>>((u64*)workspace, n_words);
  verify_drafts_kernel<<<dim3(n_requests * n_chunks), dim3(THREADS), 0, stream>>>(p, q, vocab, tokens, parents, q_start, uniforms, nodes, depth, counts, out, (u64*)workspace, n_chunks, g_patience);
  return ms_launch_status();
}

extern "C" int ms_keep_tokens_max() { return MAX_TENSORS; }

// tensors: host memory, n_tensors of KeepTensor's 24 bytes
extern "C" int ms_keep_tokens(const void* tensors, int n_tensors, int layers, int num_pages, int page_size, const int* block_table,
                              int table_stride, const int* table_rows, const int* first, const int* nodes, int depth,
                              const int* counts, int n_requests, int dtype, hipStream_t stream) {
  if (n_tensors <= 0 || n_requests <= 0 || layers <= 0) return MS_OK;
  if (n_tensors > MAX_TENSORS || num_pages <= 0 || page_size <= 0 || table_stride <= 0 || depth <= 0 || n_requests > 65535)
    return MS_BAD_ARG;
  KeepTensors ts = {};
  int most = 1;
  for (int i = 0; i < n_tensors; ++i) {
    ts.t[i] = ((const KeepTensor*)tensors)[i];
    if (ts.t[i].pages == nullptr || ts.t[i].heads <= 0 || ts.t[i].width <= 0) return MS_BAD_ARG;
    most = std::max(most, ts.t[i].heads);
  }
  const long long pairs = (long long)layers * most;
  if (pairs > 0x3fffffffLL) return MS_UNSUPPORTED;
  // a pair to a wave while there are at most 128 waves a CU, four times what it holds at once: 93 us with 16, 68 with 128 (32
  // requests, 64 layers of 8 heads of 128 in bfloat16)
  const long long room = std::max(1LL, 128LL * ms_compute_units() / KEEP_WAVES / ((long long)n_requests * n_tensors));
  dim3 grid((unsigned)std::min((pairs + KEEP_WAVES - 1) / KEEP_WAVES, room), n_requests, n_tensors), block(KEEP_WAVES * MS_WAVE);
#define LAUNCH(T) keep_tokens_kernel<T><<<grid, block, 0, stream>>>(ts, layers, num_pages, page_size, block_table, table_stride, table_rows, first, nodes, depth, counts)
  if (dtype == MS_F32) LAUNCH(unsigned);
  else if (dtype == MS_BF16) LAUNCH(unsigned short);
  else return MS_BAD_ARG;
#undef LAUNCH
  return ms_launch_status();
}
