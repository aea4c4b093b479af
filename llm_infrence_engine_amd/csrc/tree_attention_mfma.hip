// The attention of csrc/tree_attention.hip on the matrix cores (v_mfma_f32_16x16x32_bf16), bfloat16 in, float softmax.
//
// A column is a (token, query head of the group) pair; a block owns COLS columns of one (request, key/value head) and a share
// of the request's keys, so a key that is brought in serves all of them.  Its waves are KG groups of WC: the waves of a group
// own neighbouring columns, NT tiles of 16 each, and walk the same keys, a tile of KEYS at a time, which go from the pages
// straight to LDS (global_load_lds) one tile ahead; the groups take the tiles in turn and merge at the end.  Products and the
// layout of LDS are those of csrc/attention_prompt.hip:
//
//   S^T[key, col] = K[key, :] . Q^T[:, col],   O^T[dim, col] += V^T[dim, key] . P^T[key, col]
//
// where row r of the u-th score product of a unit of 32 keys is its key 8 (r / 4) + 4 u + r % 4, so that a lane (quarter kq)
// holds the scores of the keys 8 kq .. + 7 and needs one 16-byte read of a value's row.  Keys from before the step are visible
// to every column; only units that reach into the step's own entries (the last ones) look at the mask.
// Rounding: the product takes bfloat16, so a weight e^(s - ref) meets the values in two parts, its upper half and what that leaves
// out, together off by 2^-15 of it at most; the sum that divides is of the same parts.  Scores, exponentials, sums and results up to
// the last rounding are float: against 64 bits the result is off by 0.0017 of its norm, as one that is rounded at the end alone (with
// weights of one bfloat16 0.0019 to 0.0023).  The second product of the values costs what it takes: 4 trees of up to 63 behind
// 16,011 keys 101 -> 127 us, 8 of up to 16 behind 2,000 18.6 -> 19.1, smaller ones nothing.
// The keys of a request are shared out over n_splits blocks, which leave unnormalised float results that a second kernel
// adds up: with few columns there is one (request, head) tile for a handful of CUs, and a step waits for the longest chain.
#include "attention_tiles.h"
#include "api.h"
#include <algorithm>
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) unsigned short u16x8;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

constexpr int MAX_SPLITS = 128;

template <int D> __device__ __forceinline__ int permute(int key) {     // where a key's 16-byte pieces lie, by its number in its unit
  return D == 128 ? (key & 3) | ((key >> 1) & 12) : D == 64 ? ((key >> 1) & 1) | ((key >> 2) & 6) : (key >> 3) & 3;
}

// The maximum over the four lanes, 16 apart, that share a column.
__device__ __forceinline__ float column_max(float x) {
  const unsigned u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned w = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What the upper half of a weight's bits, a bfloat16 too small by less than 2^-7, leaves out.  2^-21 of the weight comes on top, which
// all weights have alike, so that it falls out of the result: no rest of a weight above zero is zero, and an infinite value
// stays infinite.
__device__ __forceinline__ float rest_of(float weight) {
  return fmaf(weight, 1.0f + 1.0f / 2097152.0f, -__uint_as_float(__float_as_uint(weight) & 0xffff0000u));
}

template <int D, int WC, int KG, int NT>
struct Shape {
  static constexpr int COLS = WC * NT * 16, KEYS = WC == 4 ? 64 : 32, CHUNKS = KEYS / 16;
  static constexpr int CHUNK = 16 * D;                 // values of a chunk of 16 keys, of keys as of values
  static constexpr int STAGE = 2 * CHUNKS * CHUNK;     // a tile: its chunks of keys, then those of values
  static constexpr size_t LDS = (size_t)KG * 2 * STAGE * 2;
};

template <int D, int WC, int KG, int NT>
__global__ void __launch_bounds__(KG * WC * MS_WAVE, D == 128 || NT == 2 ? 2 : 4)
tree_attention_mfma_kernel(const bf16* __restrict__ q, size_t q_stride, const bf16* __restrict__ k_pages,
                           const bf16* __restrict__ vt_pages, const int* __restrict__ block_table, int table_stride,
                           const int* __restrict__ table_rows, const int* __restrict__ q_start,
                           const int* __restrict__ context_lens, const unsigned* __restrict__ tree, int words,
                           bf16* __restrict__ out, size_t out_stride, float* __restrict__ part_o, float* __restrict__ part_ml,
                           int nh, int nkv, int page_size, int page_shift, float scale_log2e, int n_requests, int n_splits, int per) {      // n_requests 0: a tile to a request
  typedef Shape<D, WC, KG, NT> S;
  constexpr int COLS = S::COLS, KEYS = S::KEYS, CHUNKS = S::CHUNKS, CHUNK = S::CHUNK, STAGE = S::STAGE;
  constexpr int CT = D / 16, PIECES = D / 8, LOADS = CHUNK * 2 / 1024, MINE = CHUNKS / WC;      // chunks a wave brings
  constexpr int UNITS = NT == 1 ? KEYS / 32 : 1;      // of 32 keys that go through the stages of a tile together
  extern __shared__ __align__(16) unsigned char lds_raw[];
  bf16* lds = reinterpret_cast<bf16*>(lds_raw);       // [KG][2 tiles][STAGE]
  const int lane = threadIdx.x & (MS_WAVE - 1);
  const int kg = __builtin_amdgcn_readfirstlane(threadIdx.x / (WC * MS_WAVE));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MS_WAVE) - kg * WC;   // in its group
  const int col16 = lane & 15, kq = lane >> 4;
  const int g = blockIdx.x, rep = nh / nkv, split = blockIdx.z;

  int r, tile, n_tiles;
  if (n_requests == 0) {
    r = blockIdx.y; tile = 0;
  } else {
    find_tile(q_start, n_requests, rep, COLS, blockIdx.y, lane, r, tile, n_tiles);
    if (r < 0) return;
  }
  const int* table = block_table + (size_t)(table_rows ? table_rows[r] : r) * table_stride;
  const int q0 = q_start[r], qlen = q_start[r + 1] - q0, context = context_lens[r], before = context - qlen, ncols = qlen * rep;
  const int t_begin = split * per, t_end = min((context + KEYS - 1) / KEYS, t_begin + per);
  if (t_begin >= t_end || qlen <= 0) return;
  const int c0 = (tile * WC + wave) * NT * 16;
  const bool works = c0 < ncols;       // without columns a wave still brings its chunks

  // ---- bringing a tile: the wave's chunks of keys and of values
  unsigned k_src[MINE][LOADS], v_src[LOADS];                   // what a lane asks for, in bytes from the chunk's first value
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int at = j * 512 + lane * 8, key = at / D, piece = (at % D) / 8;
#pragma unroll
    for (int b = 0; b < MINE; ++b) k_src[b][j] = (key * D + (piece ^ permute<D>(((wave * MINE + b) & 1) * 16 + key)) * 8) * 2;
    const int dim = at / 16, half = (at >> 3) & 1;
    v_src[j] = (dim * page_size + (half ^ ((dim >> 3) & 1)) * 8) * 2;
  }
  const size_t page_bytes = (size_t)nkv * page_size * D * 2, head_bytes = (size_t)g * page_size * D * 2;
  const char *k_head = (const char*)k_pages + head_bytes, *v_head = (const char*)vt_pages + head_bytes;
  auto page_of = [&](int t, int b) {        // the page of one of the wave's chunks of tile t; past the context: the null page
    const int key = t * KEYS + (wave * MINE + b) * 16;
    return key < context ? __builtin_amdgcn_readfirstlane(table[page_shift >= 0 ? key >> page_shift : key / page_size]) : 0;
  };
  auto bring = [&](int t, const int* pages, int stage) {
#pragma unroll
    for (int b = 0; b < MINE; ++b) {
      const int key = t * KEYS + (wave * MINE + b) * 16, off = page_shift >= 0 ? key & (page_size - 1) : key % page_size;
      const size_t page = pages[b] * page_bytes;
      const char *kp = k_head + page + off * (D * 2), *vp = v_head + page + off * 2;
      bf16* to = lds + (kg * 2 + stage) * STAGE + (wave * MINE + b) * CHUNK;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) __builtin_amdgcn_global_load_lds((global_void*)(kp + k_src[b][j]), (lds_void*)(to + j * 512), 16, 0, 0);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) __builtin_amdgcn_global_load_lds((global_void*)(vp + v_src[j]), (lds_void*)(to + CHUNKS * CHUNK + j * 512), 16, 0, 0);
    }
  };
  // Values behind the context may be anything a reused page still holds, and of the step's own entries those that are not
  // finite would reach columns that do not see them (a NaN times a weight of zero): the wave that brought them makes them
  // zeros, and says of the latter that they have to be added for the columns that do (`spoiled`: the tile, counted from 1).
  __shared__ int spoiled[KG][2];
  const bool some_masked = t_end * KEYS > before;
  if (some_masked) {
    if (threadIdx.x < 2 * KG) spoiled[threadIdx.x >> 1][threadIdx.x & 1] = 0;
    __syncthreads();
  }
  auto tidy = [&](int t, int stage) {
    bool wild = false;
#pragma unroll
    for (int b = 0; b < MINE; ++b)
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int at = j * 512 + lane * 8, dim = at / 16, half = ((at >> 3) ^ (dim >> 3)) & 1;
        u16x8* place = reinterpret_cast<u16x8*>(lds + (kg * 2 + stage) * STAGE + CHUNKS * CHUNK + (wave * MINE + b) * CHUNK + at);
        u16x8 raw = *place;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = t * KEYS + (wave * MINE + b) * 16 + half * 8 + i;
          const bool gone = key >= context, bad = (key >= before) & ((raw[i] & 0x7f80) == 0x7f80) & !gone;
          wild |= bad;
          raw[i] = gone | bad ? (unsigned short)0 : raw[i];
        }
        *place = raw;
      }
    if (__builtin_amdgcn_ballot_w64(wild) != 0 && lane == 0) spoiled[kg][stage] = t + 1;
  };
  int pages[MINE];
  if (t_begin + kg < t_end) {
#pragma unroll
    for (int b = 0; b < MINE; ++b) pages[b] = page_of(t_begin + kg, b);
    bring(t_begin + kg, pages, 0);
  }
  if (t_begin + kg + KG < t_end) {
#pragma unroll
    for (int b = 0; b < MINE; ++b) pages[b] = page_of(t_begin + kg + KG, b);
  }

  // ---- this lane's columns
  bool idle[NT];
  unsigned first_words[NT][2];         // (most trees have no more)
  bf16x8 qv[NT][D / 32];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = c0 + t * 16 + col16, cc = min(c, ncols - 1), tok = q0 + cc / rep;
    idle[t] = c >= ncols;
    const unsigned* mask = tree + (size_t)tok * words;
    first_words[t][0] = mask[0];
    first_words[t][1] = words > 1 ? mask[1] : 0u;
    const bf16* qp = q + (size_t)tok * q_stride + (size_t)(g * rep + cc % rep) * D + kq * 8;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) qv[t][s] = *reinterpret_cast<const bf16x8*>(qp + s * 32);
  }
  // which of the keys base + kq * 8 + (0..7) column tile t sees, a bit each
  auto visible = [&](int t, int base) -> unsigned {
    const int rel = base + kq * 8 - before;            // the first one's number in the step; below 0: from before
    if (idle[t]) return 0u;
    if (rel <= -8) return 0xffu;
    const int at = max(rel, 0), w = at >> 5;
    auto word = [&](int i) -> unsigned { return i == 0 ? first_words[t][0] : i == 1 ? first_words[t][1] : i < words ? tree[(size_t)(q0 + (c0 + t * 16 + col16) / rep) * words + i] : 0u; };
    unsigned bits = (unsigned)((((unsigned long long)word(w + 1) << 32) | word(w)) >> (at & 31)) & 0xffu;
    if (rel < 0) bits = ((bits << -rel) | ((1u << -rel) - 1u)) & 0xffu;
    const int left = qlen - rel;
    return left >= 8 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1u);
  };

  // The sums of the exponentials are those of the parts that meet the values: a product of P^T with ones more for each.
  float m[NT];
  f32x4 o[CT][NT] = {}, lsum[NT] = {};
#pragma unroll
  for (int t = 0; t < NT; ++t) m[t] = -INFINITY;
  bf16x8 ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.0f;

  int k_row[2], k_perm[2];             // where a lane's fragments lie: key rows of the u-th product of a unit ..
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int key = (col16 >> 2) * 8 + u * 4 + (col16 & 3);
    k_row[u] = (key >> 4) * CHUNK + (key & 15) * D;
    k_perm[u] = permute<D>(key);
  }
  const int v_row = CHUNKS * CHUNK + (kq >> 1) * CHUNK + col16 * 16 + (((kq & 1) ^ (col16 >> 3)) * 8);     // .. and of 16 dims' values

  // The queries and masks have arrived: said here, by a use that nothing moves past the loop.  Otherwise the compiler may wait for
  // them, and with them for the tile that has just been asked for, before the first product of every turn.
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) asm volatile("" : "+v"(qv[t][s]));
    asm volatile("" : "+v"(first_words[t][0]), "+v"(first_words[t][1]));
  }
  const int turns = (t_end - t_begin + KG - 1) / KG;
  for (int turn = 0; turn < turns; ++turn) {
    const int t = t_begin + turn * KG + kg, stage = turn & 1;
    if (t < t_end && (t + 1) * KEYS > before) {      // reaches into the step's own entries, or behind them
      __builtin_amdgcn_s_waitcnt(0x0F70);              // (vmcnt(0))
      __builtin_amdgcn_sched_barrier(0);
      tidy(t, stage);
    }
    // This tile has landed (vmcnt), and the wave's reads of the one before it have ended (lgkmcnt), so that its place may
    // be filled again.
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + KG < t_end) {
      bring(t + KG, pages, stage ^ 1);
      if (t + 2 * KG < t_end) {
#pragma unroll
        for (int b = 0; b < MINE; ++b) pages[b] = page_of(t + 2 * KG, b);
      }
    }
    if (!works || t >= t_end) continue;      // the same for the whole wave
#pragma unroll
    for (int unit = 0; unit < KEYS / 32; unit += UNITS) {
    const int base = t * KEYS + unit * 32;
    const bf16* st = lds + (kg * 2 + stage) * STAGE + unit * 2 * CHUNK;

    // scores: s[n][u][t] holds keys base + n*32 + kq*8 + u*4 + (0..3) of column t*16 + col16.  With one tile of columns the units
    // go through every stage together, so that products of one run while the other waits for its own; with two there are no
    // registers for it.
    f32x4 s[UNITS][2][NT];
#pragma unroll
    for (int n = 0; n < UNITS; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t2 = 0; t2 < NT; ++t2) s[n][u][t2] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
#pragma unroll
      for (int n = 0; n < UNITS; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(st + n * 2 * CHUNK + k_row[u] + (((ks * 4 + kq) ^ k_perm[u]) & (PIECES - 1)) * 8);
#pragma unroll
          for (int t2 = 0; t2 < NT; ++t2) s[n][u][t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qv[t2][ks], s[n][u][t2], 0, 0, 0);
        }
    const bool masked = base + UNITS * 32 > before;     // reaches into the step's own entries, or behind them
    unsigned sees[UNITS][NT];
    if (masked) {
#pragma unroll
      for (int n = 0; n < UNITS; ++n)
#pragma unroll
        for (int t2 = 0; t2 < NT; ++t2) {
          sees[n][t2] = visible(t2, base + n * 32);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!((sees[n][t2] >> (u * 4 + i)) & 1u)) s[n][u][t2][i] = -INFINITY;
        }
    }
    // m is the reference of the exponents: it follows the maximum when that has run ahead by REF_SLACK
    float bmax[NT];
    bool ahead = false;
#pragma unroll
    for (int t2 = 0; t2 < NT; ++t2) {
      float bm = -INFINITY;
#pragma unroll
      for (int n = 0; n < UNITS; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) bm = fmaxf(bm, s[n][u][t2][i]);
      bmax[t2] = bm;
      ahead |= bm * scale_log2e > m[t2] + REF_SLACK;
    }
    if (__builtin_amdgcn_ballot_w64(ahead) != 0) {
#pragma unroll
      for (int t2 = 0; t2 < NT; ++t2) {
        const float bm = column_max(bmax[t2]) * scale_log2e;
        const bool step = bm > m[t2] + REF_SLACK;
        const float corr = step ? fast_exp2(m[t2] - bm) : 1.0f;      // m = -inf: 0
        if (step) m[t2] = bm;
        lsum[t2] *= corr;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][t2] *= corr;
      }
    }
    // Values are read two fragments ahead of their products, the first ones before the exponentials (4 of up to 63 behind 16,011
    // keys 131 -> 127 us; the same for the keys made no difference).
    const auto values = [&](int f) { return *reinterpret_cast<const bf16x8*>(st + f / CT * 2 * CHUNK + v_row + f % CT * 256); };
    bf16x8 now[2] = {values(0), values(1)}, next[2];
    __builtin_amdgcn_sched_barrier(0);
    bf16x8 p[UNITS][NT], rest[UNITS][NT];
#pragma unroll
    for (int n = 0; n < UNITS; ++n)
#pragma unroll
      for (int t2 = 0; t2 < NT; ++t2) {
        const float ref = m[t2] == -INFINITY ? 0.f : m[t2];
        u32x4 high;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float a = fast_exp2(fmaf(s[n][i / 4][t2][i % 4], scale_log2e, -ref));
          const float b = fast_exp2(fmaf(s[n][i / 4][t2][i % 4 + 1], scale_log2e, -ref));
          high[i / 2] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
          rest[n][t2][i] = (__bf16)rest_of(a);
          rest[n][t2][i + 1] = (__bf16)rest_of(b);
        }
        p[n][t2] = __builtin_bit_cast(bf16x8, high);
        lsum[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[n][t2], lsum[t2], 0, 0, 0);
        lsum[t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, rest[n][t2], lsum[t2], 0, 0, 0);
      }
#pragma unroll
    for (int f = 0; f < UNITS * CT; f += 2) {
      if (f + 2 < UNITS * CT) { next[0] = values(f + 2); next[1] = values(f + 3); }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int t2 = 0; t2 < NT; ++t2) {
            const int n = (f + i) / CT, c = (f + i) % CT;
            o[c][t2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(now[i], part ? rest[n][t2] : p[n][t2], o[c][t2], 0, 0, 0);
          }
      __builtin_amdgcn_sched_barrier(0);
      now[0] = next[0]; now[1] = next[1];
    }
    if (masked && spoiled[kg][stage] == t + 1) {       // (rare: the values are read again from where they are)
      int rows = page_size;
      asm volatile("" : "+s"(rows));                   // (nothing of this is worked out ahead of the loop and kept in registers)
#pragma unroll
      for (int n = 0; n < UNITS; ++n)
        for (int k = 0; k < 32; ++k) {
          const int key = base + n * 32 + k;
          if (key < before || key >= context) continue;
          const int owner = (k >> 3) * 16 + col16;
          const bf16* from = vt_pages + ((size_t)table[key / rows] * nkv + g) * rows * D + key % rows;
#pragma unroll
          for (int t2 = 0; t2 < NT; ++t2) {
            float mine = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine = (k & 7) == i ? (float)p[n][t2][i] + (float)rest[n][t2][i] : mine;
            const float w = __shfl(mine, owner, MS_WAVE);
            const bool see = (__shfl(sees[n][t2], owner, MS_WAVE) >> (k & 7)) & 1u;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              asm volatile("" : "+s"(rows) : : "memory");      // (.. nor the places of all dims at once)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const unsigned raw = __builtin_bit_cast(unsigned short, from[(size_t)(c * 16 + kq * 4 + i) * rows]);
                if (see && (raw & 0x7f80u) == 0x7f80u) o[c][t2][i] += w * __uint_as_float(raw << 16);
              }
            }
          }
        }
    }
    }
  }

  float l[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) l[t] = lsum[t][0];      // every row of the product of ones is the column's sum
  constexpr int OWN = CT >= KG ? CT / KG : 1;          // tiles of dims a group ends up with
  if constexpr (KG > 1) {
    __shared__ float sm_m[KG][COLS], sm_l[KG][COLS];
    f32x4* sm_o = reinterpret_cast<f32x4*>(lds);       // [group of the sums][wave][tile of dims][NT][64]
    static_assert((size_t)KG * WC * CT * NT * MS_WAVE * 16 <= S::LDS, "all sums fit");
    __syncthreads();                                   // nobody reads keys or values any more
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c = (wave * NT + t) * 16 + col16;
      if (kq == 0) { sm_m[kg][c] = m[t]; sm_l[kg][c] = l[t]; }
#pragma unroll
      for (int d = 0; d < CT; ++d)
        if (d / OWN != kg) sm_o[(((kg * WC + wave) * CT + d) * NT + t) * MS_WAVE + lane] = o[d][t];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int c = (wave * NT + t) * 16 + col16;
      float big = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; ++k) big = fmaxf(big, sm_m[k][c]);
      const float safe = big == -INFINITY ? 0.f : big;
      l[t] = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) l[t] = fmaf(sm_l[k][c], fast_exp2(sm_m[k][c] - safe), l[t]);
#pragma unroll
      for (int d = 0; d < CT; ++d) {
        if (d / OWN != kg) continue;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KG; ++k) {
          const float f = fast_exp2(sm_m[k][c] - safe);
          sum += (k == kg ? o[d][t] : sm_o[(((k * WC + wave) * CT + d) * NT + t) * MS_WAVE + lane]) * f;
        }
        o[d][t] = sum;
      }
      m[t] = big;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (idle[t]) continue;
    const int c = c0 + t * 16 + col16, tok = q0 + c / rep, head = g * rep + c % rep;
    if (n_splits > 1) {
      const size_t slot = ((size_t)tok * nh + head) * n_splits + split;
#pragma unroll
      for (int d = 0; d < CT; ++d)
        if (KG == 1 || d / OWN == kg) *reinterpret_cast<f32x4*>(part_o + slot * D + d * 16 + kq * 4) = o[d][t];
      if (kq == 0 && kg == 0) { part_ml[slot * 2] = m[t]; part_ml[slot * 2 + 1] = l[t]; }
    } else {
      const float inv = l[t] != 0.f ? 1.0f / l[t] : 0.f;      // nothing visible: zeros (a NaN stays one)
      bf16* op = out + (size_t)tok * out_stride + (size_t)head * D + kq * 4;
#pragma unroll
      for (int d = 0; d < CT; ++d) {
        if (KG > 1 && d / OWN != kg) continue;
        bf16x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (__bf16)(o[d][t][i] * inv);
        *reinterpret_cast<bf16x4*>(op + d * 16) = w;
      }
    }
  }
}

// out[n, h, :] = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the splits that n's request used, a wave to a (token,
// head): a split's reference and sum to a lane, then every lane its dims of one split after another.
constexpr int COMBINE_WAVES = 4, AT_ONCE = 8;      // (parts a lane asks for at a time)

template <typename T, int D>
__global__ void __launch_bounds__(COMBINE_WAVES * MS_WAVE)
tree_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int* __restrict__ token_req,
                    const int* __restrict__ q_start, const int* __restrict__ context_lens, int n_requests, T* __restrict__ out,
                    size_t out_stride, int n_tokens, int nh, int share, int n_splits) {
  constexpr int DL = (D + MS_WAVE - 1) / MS_WAVE;
  const int lane = threadIdx.x & (MS_WAVE - 1);
  const long long item = (long long)blockIdx.x * COMBINE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / MS_WAVE);
  const int n = (int)(item / nh), h = (int)(item - (long long)n * nh);
  if (n >= n_tokens || n >= q_start[n_requests]) return;      // (a token that pads a captured batch)
  const int context = context_lens[token_req[n]];
  const int used = min((context + share - 1) / share, n_splits);
  const size_t slot0 = (size_t)item * n_splits;
  float m[MAX_SPLITS / MS_WAVE], l[MAX_SPLITS / MS_WAVE], top = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < MAX_SPLITS / MS_WAVE; ++i) {
    const int s = lane + i * MS_WAVE;
    m[i] = s < used ? part_ml[(slot0 + s) * 2] : -INFINITY;
    l[i] = s < used ? part_ml[(slot0 + s) * 2 + 1] : 0.f;
    top = fmaxf(top, m[i]);
  }
  top = wave_max(top);
  if (top == -INFINITY) top = 0.f;
#pragma unroll
  for (int i = 0; i < MAX_SPLITS / MS_WAVE; ++i) {
    m[i] = fast_exp2(m[i] - top);
    den = fmaf(m[i], l[i], den);
  }
  den = wave_sum(den);
  float acc[DL] = {};
  for (int s0 = 0; s0 < used; s0 += AT_ONCE) {
    float part[AT_ONCE][DL];
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s)
#pragma unroll
      for (int e = 0; e < DL; ++e) part[s][e] = part_o[(slot0 + min(s0 + s, used - 1)) * D + min(lane + e * MS_WAVE, D - 1)];
#pragma unroll
    for (int s = 0; s < AT_ONCE; ++s) {
      const int at = s0 + s;
      const float w = at < used ? __shfl(at < MS_WAVE ? m[0] : m[1], at & (MS_WAVE - 1), MS_WAVE) : 0.f;
#pragma unroll
      for (int e = 0; e < DL; ++e) acc[e] = fmaf(w, at < used ? part[s][e] : 0.f, acc[e]);      // (behind the last: it again, which may be infinite)
    }
  }
  const float inv = den != 0.f ? 1.0f / den : 0.f;
#pragma unroll
  for (int e = 0; e < DL; ++e)
    if (lane + e * MS_WAVE < D) out[(size_t)n * out_stride + (size_t)h * D + lane + e * MS_WAVE] = from_float<T>(acc[e] * inv);
}

// ---- the 32-bit path (v_mfma_f32_16x16x4_f32): scores, exponentials, weights and values are floats.  A wave owns NT tiles of 16
// columns and takes every F32_WAVES-th tile of 16 keys of the block's share, with the next one's keys and values on their way in
// registers; the waves merge through LDS, each its part of the dims.  A step of the score product takes one entry of each of four
// quarters of 16 dims, and one of the value product one key of each of four quarters of 16, so that a lane reads 16 bytes of its
// key's row and has its own keys' weights where they are: O^T[dim, col] += V^T[dim, key] . P^T[key, col].  Pages may have any size.
// 157 TFLOP/s are more than it can be fed: it waits for its loads (6 trees of up to 13 tokens behind 700 keys, 14 heads of 64 on 2:
// 9 us, 60 on the vector ALUs, which read every key for every column).
constexpr int F32_WAVES = 8;

template <int D, int NT>
__global__ void __launch_bounds__(F32_WAVES * MS_WAVE, 2)
tree_attention_f32_kernel(const float* __restrict__ q, size_t q_stride, const float* __restrict__ k_pages,
                          const float* __restrict__ v_pages, const int* __restrict__ block_table, int table_stride,
                          const int* __restrict__ table_rows, const int* __restrict__ q_start, const int* __restrict__ context_lens,
                          const unsigned* __restrict__ tree, int words, float* __restrict__ out, size_t out_stride,
                          float* __restrict__ part_o, float* __restrict__ part_ml, int nh, int nkv, int page_size, int page_shift,
                          float scale_log2e, int n_requests, int n_splits, int share) {
  constexpr int CT = D / 16, COLS = NT * 16;
  extern __shared__ __align__(16) unsigned char lds_raw[];
  f32x4* sm_o = reinterpret_cast<f32x4*>(lds_raw);       // [wave][tile of dims][NT][64]
  __shared__ float sm_m[F32_WAVES][COLS], sm_l[F32_WAVES][COLS];
  const int lane = threadIdx.x & (MS_WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / MS_WAVE);
  const int col16 = lane & 15, kq = lane >> 4;
  const int g = blockIdx.x, rep = nh / nkv, split = blockIdx.z;
  int r, tile, n_tiles;
  if (n_requests == 0) {
    r = blockIdx.y; tile = 0;
  } else {
    find_tile(q_start, n_requests, rep, COLS, blockIdx.y, lane, r, tile, n_tiles);
    if (r < 0) return;
  }
  const int* table = block_table + (size_t)(table_rows ? table_rows[r] : r) * table_stride;
  const int q0 = q_start[r], qlen = q_start[r + 1] - q0, context = context_lens[r], before = context - qlen, ncols = qlen * rep;
  const int t_begin = split * (share / 16), t_end = min((context + 15) / 16, t_begin + share / 16);
  if (t_begin >= t_end || qlen <= 0) return;

  // the row of the lane's key of a tile among all rows of keys (of values the same); past the context: the last one's
  auto row_of = [&](int t) {
    const int key = min(t * 16 + col16, context - 1), page = page_shift >= 0 ? key >> page_shift : key / page_size;
    return (table[page] * nkv + g) * page_size + (key - page * page_size);
  };
  // at 128 dims there are no registers for the next tile's values beside its keys: they are asked for where a tile's turn begins
  constexpr bool VALUES_EARLY = D < 128;
  float4 k[2][CT];
  float v[VALUES_EARLY ? 2 : 1][CT][4];
  auto load_keys = [&](int row, float4 (&kf)[CT]) __attribute__((always_inline)) {
    const float* kp = k_pages + (size_t)row * D + kq * 4;
#pragma unroll
    for (int c = 0; c < CT; ++c) kf[c] = *reinterpret_cast<const float4*>(kp + c * 16);
  };
  auto load_values = [&](int row, float (&vf)[CT][4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* vp = v_pages + (size_t)__shfl(row, kq * 4 + i, MS_WAVE) * D + col16;
#pragma unroll
      for (int c = 0; c < CT; ++c) vf[c][i] = vp[c * 16];
    }
  };
  int row_now = 0, row_next = 0;
  if (t_begin + wave < t_end) {
    row_now = row_of(t_begin + wave);
    load_keys(row_now, k[0]);
    if (VALUES_EARLY) load_values(row_now, v[0]);
  }
  if (t_begin + wave + F32_WAVES < t_end) row_next = row_of(t_begin + wave + F32_WAVES);

  bool idle[NT];
  float4 qv[NT][CT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int c = tile * COLS + t * 16 + col16, cc = min(c, ncols - 1);
    idle[t] = c >= ncols;
    const float* qp = q + (size_t)(q0 + cc / rep) * q_stride + (size_t)(g * rep + cc % rep) * D + kq * 4;
#pragma unroll
    for (int j = 0; j < CT; ++j) qv[t][j] = *reinterpret_cast<const float4*>(qp + j * 16);
  }
  // which of the keys base + kq * 4 + (0..3) column tile t sees
  auto visible = [&](int t, int base) -> unsigned {
    const int rel = base + kq * 4 - before;
    if (idle[t]) return 0u;
    if (rel <= -4) return 0xfu;
    const unsigned* mask = tree + (size_t)(q0 + min(tile * COLS + t * 16 + col16, ncols - 1) / rep) * words;
    const int at = max(rel, 0), w = at >> 5;
    const unsigned lo = w < words ? mask[w] : 0u, hi = w + 1 < words ? mask[w + 1] : 0u;
    unsigned bits = (unsigned)((((unsigned long long)hi << 32) | lo) >> (at & 31)) & 0xfu;
    if (rel < 0) bits = ((bits << -rel) | ((1u << -rel) - 1u)) & 0xfu;
    const int left = qlen - rel;
    return left >= 4 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1u);
  };
  float m[NT], l[NT];
  f32x4 o[CT][NT] = {};
#pragma unroll
  for (int t = 0; t < NT; ++t) { m[t] = -INFINITY; l[t] = 0.f; }

  auto step = [&](int t, float4 (&kf)[CT], float (&vf)[CT][4], float4 (&kn)[CT], float (&vn)[CT][4]) __attribute__((always_inline)) {
    if (!VALUES_EARLY) load_values(row_now, vf);
    if (t + F32_WAVES < t_end) {
      load_keys(row_next, kn);
      if (VALUES_EARLY) load_values(row_next, vn);
      row_now = row_next;
      if (t + 2 * F32_WAVES < t_end) row_next = row_of(t + 2 * F32_WAVES);
    }
    const int base = t * 16;
    // a score is summed in four parts: the rounding of the longer chain of one made results off by up to 2.2 times what a plain
    // product in float is (now 1.1; 120 steps of up to 16 tokens behind up to 600 keys)
    f32x4 s[NT], quarter[NT][4] = {};
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        quarter[n][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j].x, qv[n][j].x, quarter[n][0], 0, 0, 0);
        quarter[n][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j].y, qv[n][j].y, quarter[n][1], 0, 0, 0);
        quarter[n][2] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j].z, qv[n][j].z, quarter[n][2], 0, 0, 0);
        quarter[n][3] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j].w, qv[n][j].w, quarter[n][3], 0, 0, 0);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = (quarter[n][0] + quarter[n][1]) + (quarter[n][2] + quarter[n][3]);
    const bool masked = base + 16 > before;
    unsigned sees[NT];
    bool spoiled = false;
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        sees[n] = visible(n, base);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = (sees[n] >> i) & 1u ? s[n][i] : -INFINITY;
      }
      // (as in the kernel above: what no column may meet, and what not every column may)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = base + kq * 4 + i;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const bool gone = key >= context, wild = (key >= before) & !(fabsf(vf[c][i]) < INFINITY) & !gone;
          spoiled |= wild;
          vf[c][i] = gone | wild ? 0.f : vf[c][i];
        }
      }
    }
    f32x4 p[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float top = fmaxf(m[n], column_max(fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3]))) * scale_log2e);
      const float ref = top == -INFINITY ? 0.f : top, corr = fast_exp2(m[n] - ref);      // 0 while nothing has been seen
      m[n] = top;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[n][i] = fast_exp2(fmaf(s[n][i], scale_log2e, -ref));
        sum += p[n][i];
      }
      l[n] = fmaf(l[n], corr, sum);
#pragma unroll
      for (int c = 0; c < CT; ++c) o[c][n] *= corr;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[c][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[c][i], p[n][i], o[c][n], 0, 0, 0);
    if (masked && __builtin_amdgcn_ballot_w64(spoiled) != 0) {
      int dims = D;
      for (int x = 0; x < 16; ++x) {
        const int key = base + x;
        if (key < before || key >= context) continue;
        const int page = key / page_size, owner = (x >> 2) * 16 + col16;
        const float* from = v_pages + ((size_t)table[page] * nkv + g) * page_size * D + (size_t)(key - page * page_size) * D;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float w = __shfl((x & 3) == 0 ? p[n][0] : (x & 3) == 1 ? p[n][1] : (x & 3) == 2 ? p[n][2] : p[n][3], owner, MS_WAVE);
          const bool see = (__shfl(sees[n], owner, MS_WAVE) >> (x & 3)) & 1u;
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            asm volatile("" : "+s"(dims) : : "memory");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float value = from[min(c * 16 + kq * 4 + i, dims - 1)];
              if (see && !(fabsf(value) < INFINITY)) o[c][n][i] += w * value;
            }
          }
        }
      }
    }
  };
  for (int t = t_begin + wave; t < t_end; t += 2 * F32_WAVES) {
    step(t, k[0], v[0], k[1], v[VALUES_EARLY]);
    if (t + F32_WAVES < t_end) step(t + F32_WAVES, k[1], v[VALUES_EARLY], k[0], v[0]);
  }

  // every wave merges every F32_WAVES-th (tile of dims, tile of columns)
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] += __shfl_xor(l[t], 16, MS_WAVE);
    l[t] += __shfl_xor(l[t], 32, MS_WAVE);
    if (kq == 0) { sm_m[wave][t * 16 + col16] = m[t]; sm_l[wave][t * 16 + col16] = l[t]; }
#pragma unroll
    for (int c = 0; c < CT; ++c) sm_o[((wave * CT + c) * NT + t) * MS_WAVE + lane] = o[c][t];
  }
  __syncthreads();
  for (int part = wave; part < CT * NT; part += F32_WAVES) {
    const int c = part / NT, t = part - c * NT;
    float big = -INFINITY, den = 0.f;
#pragma unroll
    for (int w = 0; w < F32_WAVES; ++w) big = fmaxf(big, sm_m[w][t * 16 + col16]);
    const float safe = big == -INFINITY ? 0.f : big;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < F32_WAVES; ++w) {
      const float f = fast_exp2(sm_m[w][t * 16 + col16] - safe);
      den = fmaf(sm_l[w][t * 16 + col16], f, den);
      sum += sm_o[((w * CT + c) * NT + t) * MS_WAVE + lane] * f;
    }
    const int col = tile * COLS + t * 16 + col16;
    if (col >= ncols) continue;
    const int tok = q0 + col / rep, head = g * rep + col % rep;
    if (n_splits > 1) {
      const size_t slot = ((size_t)tok * nh + head) * n_splits + split;
      *reinterpret_cast<f32x4*>(part_o + slot * D + c * 16 + kq * 4) = sum;
      if (c == 0 && kq == 0) { part_ml[slot * 2] = big; part_ml[slot * 2 + 1] = den; }
    } else {
      *reinterpret_cast<f32x4*>(out + (size_t)tok * out_stride + (size_t)head * D + c * 16 + kq * 4) = sum * (den != 0.f ? 1.0f / den : 0.f);
    }
  }
}

struct Call {
  const bf16 *q, *k, *vt;
  const int *table, *rows, *token_req, *q_start, *ctx;
  const unsigned* tree;
  bf16* out;
  float *part_o, *part_ml;
  size_t q_stride, out_stride;
  int table_stride, words, n_requests, n_tokens, max_q_len, nh, nkv, page_size, n_splits, share;
  float scale_log2e;
  hipStream_t stream;
};

inline long long column_tiles(int n_requests, int n_tokens, int max_q_len, int rep, int cols) {
  return std::min((long long)n_tokens * rep / cols + n_requests, ((long long)max_q_len * rep + cols - 1) / cols * n_requests);
}

// Allows a kernel more LDS than the default 64 KB, once on every device it runs on (`raised`: the kernel's own flags).
constexpr int MAX_DEVICES = 64;
inline bool raise_lds(const void* kernel, size_t bytes, bool* raised) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAX_DEVICES) return false;
  if (!raised[dev]) raised[dev] = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == hipSuccess;
  return raised[dev];
}

inline int page_shift_of(int page_size) {   // log2 of a power of two, else -1
  return page_size & (page_size - 1) ? -1 : __builtin_ctz(page_size);
}

template <int D, int WC, int KG, int NT>
int launch(const Call& a) {
  typedef Shape<D, WC, KG, NT> S;
  static bool raised[MAX_DEVICES] = {};
  if (!raise_lds(reinterpret_cast<const void*>(&tree_attention_mfma_kernel<D, WC, KG, NT>), S::LDS, raised)) return MS_LAUNCH_FAILED;
  const int rep = a.nh / a.nkv;
  const bool one = (long long)a.max_q_len * rep <= S::COLS;
  const long long tiles = one ? a.n_requests : column_tiles(a.n_requests, a.n_tokens, a.max_q_len, rep, S::COLS);
  if (tiles > 65535) return MS_UNSUPPORTED;
  tree_attention_mfma_kernel<D, WC, KG, NT><<<dim3(a.nkv, (unsigned)tiles, a.n_splits), dim3(KG * WC * MS_WAVE), S::LDS, a.stream>>>(
      a.q, a.q_stride, a.k, a.vt, a.table, a.table_stride, a.rows, a.q_start, a.ctx, a.tree, a.words, a.out, a.out_stride, a.part_o,
      a.part_ml, a.nh, a.nkv, a.page_size, page_shift_of(a.page_size), a.scale_log2e, one ? 0 : a.n_requests, a.n_splits, a.share / S::KEYS);
  if (a.n_splits > 1) {
    const long long items = (long long)a.n_tokens * a.nh;
    tree_combine_kernel<bf16, D><<<dim3((unsigned)((items + COMBINE_WAVES - 1) / COMBINE_WAVES)), dim3(COMBINE_WAVES * MS_WAVE), 0, a.stream>>>(
        a.part_o, a.part_ml, a.token_req, a.q_start, a.ctx, a.n_requests, a.out, a.out_stride, a.n_tokens, a.nh, a.share, a.n_splits);
  }
  return ms_launch_status();
}

// Kinds of block: WC waves over columns, KG groups over keys (at 32 and 64 dims F times as many), NT tiles of 16 columns a wave.
// A block's time is a chain of turns (KG tiles of keys): 2.1 us around them, `alone` us a turn with one block on a CU, `pair`
// where there are two (0: its LDS leaves room for one).
struct Kind { int wc, kg, nt; double alone, pair; };
constexpr Kind KINDS[2][4] = {{{1, 8, 1, 0.75, 0.0}, {2, 4, 1, 0.37, 1.02}, {4, 2, 1, 0.73, 1.37}, {4, 1, 2, 0.93, 1.19}},     // 32, 64 dims
                              {{1, 4, 1, 1.22, 0.0}, {2, 2, 1, 0.64, 0.89}, {4, 1, 1, 1.13, 1.12}, {4, 1, 2, 1.62, 1.83}}};  // 128 dims

}  // namespace

// kind * 65536 + how many times 64 keys a block takes, for a step of these sizes (all bounds); -1: sizes this kernel does not
// take.  Narrow kinds share a small step out over the chip, and every block's chain is short; wide ones read the keys less
// often.  The choice is the least of a model: a launch (4.3 us), then the chains, as often as all blocks take the chip's room, or
// the keys at 13.5 TB/s (what all tiles of columns drew together, from L2s and memory), whichever is longer, and the second kernel
// (3.1 us, the parts written and read at 4.4 TB/s).  Its numbers were fitted, with weights of one part, to the times of all kinds and
// shares at 44 steps of 64 and 128 dims (1 to 64 requests of 1 to 63 tokens behind 64 to 16,011 keys), and 32 dims take those of 64;
// at these steps its choice takes 1.9% longer than the fastest on average, 16% at most.  us measured, the choice against the
// fastest and the slowest kind with its best share: 8 tokens of 14 heads of 64 on 2 behind 192 keys 7.1, 6.9 (128 columns a
// block: 9.5); 28 heads of 128 on 4: 8 x 16 behind 2,000 19.8, 19.8 (16 columns: 26.6), 32 x 8 behind 1,000 23.0, 21.1 (16 columns:
// 32.4); 40 on 8: 2 x 16 behind 4,000 19.6, 19.5 (128 columns: 22.5), 4 x 63 behind 16,011 126, 126 (16 columns: 293).
extern "C" int ms_tree_attention_mfma_plan(int n_requests, int n_tokens, int max_q_len, int max_context_len, int num_heads,
                                           int num_kv_heads, int head_dim, int page_size) {
  if ((head_dim != 32 && head_dim != 64 && head_dim != 128) || page_size <= 0 || page_size % 16) return -1;
  if (n_requests <= 0 || n_tokens <= 0 || max_q_len <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads) return -1;
  const int rep = num_heads / num_kv_heads;
  if ((long long)max_q_len * rep > 0x3fffffffLL) return -1;
  const long long context = std::max(1, max_context_len);
  if (context > 64LL * 65535) return -1;
  const double cus = ms_compute_units(), cols = (double)n_tokens * rep;
  double best = 0.0;
  int choice = -1;
  for (int kind = 0; kind < 4; ++kind) {
    const Kind k = KINDS[head_dim == 128][kind];
    const int width = k.wc * k.nt * 16, turn = (k.wc == 4 ? 64 : 32) * k.kg;
    // a request ends in half a tile on average, unless one tile is all it has
    const double tiles = ((long long)max_q_len * rep <= width ? (double)n_requests : cols / width + 0.5 * n_requests) * num_kv_heads;
    const double draws = tiles * context * head_dim * 4 / 13.5e6;
    for (const int n : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 16, 20, 24, 32, 48, 64, 96, 128}) {
      const long long share = ((context + n - 1) / n + turn - 1) / turn * turn, turns = share / turn, splits = (context + share - 1) / share;
      if (splits > MAX_SPLITS || share / 64 > 0xffff) continue;
      const double blocks = tiles * splits;
      const bool pairs = k.pair > 0.0 && blocks > cus;
      const double rounds = std::max(1.0, blocks / (pairs ? 2.0 * cus : cus));
      double us = 4.3 + std::max((turns * (pairs ? k.pair : k.alone) + 2.1) * rounds, draws);
      if (splits > 1) us += 3.1 + (double)n_tokens * num_heads * splits * (head_dim + 2) * 8 / 4.4e6;
      if (choice < 0 || us < best) { best = us; choice = kind * 65536 + (int)(share / 64); }
      if (n > 1 && turns == 1) break;
    }
  }
  return choice;
}

// part_o: float [n_tokens, num_heads, n_splits, head_dim], part_ml: float [n_tokens, num_heads, n_splits, 2] (null with one).
extern "C" int ms_tree_attention_mfma(const void* q, long long q_stride, const void* k_pages, const void* vt_pages,
                                      const int* block_table, int table_stride, const int* table_rows, const int* token_req,
                                      const int* q_start, const int* context_lens, const int* tree, int words, void* out,
                                      long long out_stride, void* part_o, void* part_ml, int n_requests, int n_tokens,
                                      int max_q_len, int num_heads, int num_kv_heads, int head_dim, int page_size, float scale,
                                      int kind, int share, int n_splits, hipStream_t stream) {
  if (n_requests <= 0 || n_tokens <= 0 || max_q_len <= 0) return MS_OK;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || table_stride <= 0 || words <= 0) return MS_BAD_ARG;
  if (!(scale > 0.f)) return MS_UNSUPPORTED;   // maxima are taken of the raw scores
  if (share <= 0 || share % 64) return MS_BAD_ARG;
  if (n_splits < 1 || n_splits > MAX_SPLITS || (n_splits > 1 && (part_o == nullptr || part_ml == nullptr))) return MS_BAD_ARG;
  if (page_size <= 0 || page_size % 16 || num_kv_heads > 65535) return MS_UNSUPPORTED;
  if (q_stride % 8 || out_stride % 4 || ((uintptr_t)q % 16) || ((uintptr_t)out % 8) || ((uintptr_t)part_o % 16)) return MS_UNSUPPORTED;
  if (((uintptr_t)k_pages | (uintptr_t)vt_pages) % 16) return MS_UNSUPPORTED;
  const int rep = num_heads / num_kv_heads;
  if ((long long)max_q_len * rep > 0x3fffffffLL || (long long)n_tokens * num_heads > 0x3fffffffLL) return MS_UNSUPPORTED;
  const Call a = {(const bf16*)q, (const bf16*)k_pages, (const bf16*)vt_pages, block_table, table_rows, token_req, q_start, context_lens,
                  (const unsigned*)tree, (bf16*)out, (float*)part_o, (float*)part_ml, (size_t)q_stride, (size_t)out_stride, table_stride,
                  words, n_requests, n_tokens, max_q_len, num_heads, num_kv_heads, page_size, n_splits, share, scale * 1.4426950408889634f, stream};
#define GO(D, F) switch (kind) { case 0: return launch<D, 1, 4 * F, 1>(a); case 1: return launch<D, 2, 2 * F, 1>(a); \
                                 case 2: return launch<D, 4, F, 1>(a); case 3: return launch<D, 4, 1, 2>(a); }
  if (head_dim == 32) GO(32, 2);
  if (head_dim == 64) GO(64, 2);
  if (head_dim == 128) GO(128, 1);
#undef GO
  return MS_UNSUPPORTED;
}

// Keys that a block of the 32-bit kernel takes, for a step of these sizes (all bounds); 0: sizes it does not take.  About a block a
// CU, but never less than a tile for every wave: a block's turns of F32_WAVES tiles come one after another, 1 us each.
extern "C" int ms_tree_attention_f32_share(int n_requests, int n_tokens, int max_q_len, int max_context_len, int num_heads,
                                           int num_kv_heads, int head_dim) {
  if ((head_dim != 32 && head_dim != 64 && head_dim != 128) || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads) return 0;
  if (n_requests <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
  const int rep = num_heads / num_kv_heads, turn = 16 * F32_WAVES;
  if ((long long)max_q_len * rep > 0x3fffffffLL) return 0;
  const long long blocks = column_tiles(n_requests, n_tokens, max_q_len, rep, head_dim == 128 ? 16 : 32) * num_kv_heads;
  const long long context = std::max(1, max_context_len), turns = (context + turn - 1) / turn;
  const long long splits = std::max(1LL, std::min({turns, (long long)MAX_SPLITS, ms_compute_units() / blocks}));
  return (int)((turns + splits - 1) / splits * turn);
}

// As ms_tree_attention_mfma, for float: values [P, nkv, page_size, head_dim], pages of any size; num_pages: rows are counted in an int.
extern "C" int ms_tree_attention_f32(const float* q, long long q_stride, const float* k_pages, const float* v_pages,
                                     const int* block_table, int table_stride, const int* table_rows, const int* token_req,
                                     const int* q_start, const int* context_lens, const int* tree, int words, float* out,
                                     long long out_stride, float* part_o, float* part_ml, int n_requests, int n_tokens, int max_q_len,
                                     int num_heads, int num_kv_heads, int head_dim, int page_size, long long num_pages, float scale,
                                     int share, int n_splits, hipStream_t stream) {
  if (n_requests <= 0 || n_tokens <= 0 || max_q_len <= 0) return MS_OK;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || table_stride <= 0 || words <= 0 || page_size <= 0) return MS_BAD_ARG;
  if (!(scale > 0.f)) return MS_UNSUPPORTED;   // maxima are taken of the raw scores
  if (share <= 0 || share % 16 || n_splits < 1 || n_splits > MAX_SPLITS || (n_splits > 1 && (part_o == nullptr || part_ml == nullptr))) return MS_BAD_ARG;
  if (num_kv_heads > 65535 || num_pages * num_kv_heads * page_size >= (1ll << 31)) return MS_UNSUPPORTED;
  if (q_stride % 4 || out_stride % 4 || ((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pages | (uintptr_t)part_o) % 16) return MS_UNSUPPORTED;
  const int rep = num_heads / num_kv_heads;
  if ((long long)max_q_len * rep > 0x3fffffffLL || (long long)n_tokens * num_heads > 0x3fffffffLL) return MS_UNSUPPORTED;
  auto go = [&](auto dims, auto nt) {
    constexpr int D = decltype(dims)::value, NT = decltype(nt)::value;
    constexpr int lds = F32_WAVES * (D / 16) * NT * MS_WAVE * (int)sizeof(f32x4);
    static bool raised[MAX_DEVICES] = {};
    if (!raise_lds(reinterpret_cast<const void*>(&tree_attention_f32_kernel<D, NT>), lds, raised)) return (int)MS_LAUNCH_FAILED;
    const bool one = (long long)max_q_len * rep <= NT * 16;
    const long long tiles = one ? n_requests : column_tiles(n_requests, n_tokens, max_q_len, rep, NT * 16);
    if (tiles > 65535) return (int)MS_UNSUPPORTED;
    tree_attention_f32_kernel<D, NT><<<dim3(num_kv_heads, (unsigned)tiles, n_splits), dim3(F32_WAVES * MS_WAVE), lds, stream>>>(
        q, (size_t)q_stride, k_pages, v_pages, block_table, table_stride, table_rows, q_start, context_lens, (const unsigned*)tree, words, out,
        (size_t)out_stride, part_o, part_ml, num_heads, num_kv_heads, page_size, page_shift_of(page_size), scale * 1.4426950408889634f,
        one ? 0 : n_requests, n_splits, share);
    if (n_splits > 1) {
      const long long items = (long long)n_tokens * num_heads;
      tree_combine_kernel<float, D><<<dim3((unsigned)((items + COMBINE_WAVES - 1) / COMBINE_WAVES)), dim3(COMBINE_WAVES * MS_WAVE), 0, stream>>>(
          part_o, part_ml, token_req, q_start, context_lens, n_requests, out, (size_t)out_stride, n_tokens, num_heads, share, n_splits);
    }
    return ms_launch_status();
  };
  if (head_dim == 32) return go(std::integral_constant<int, 32>{}, std::integral_constant<int, 2>{});
  if (head_dim == 64) return go(std::integral_constant<int, 64>{}, std::integral_constant<int, 2>{});
  if (head_dim == 128) return go(std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
  return MS_UNSUPPORTED;
}
