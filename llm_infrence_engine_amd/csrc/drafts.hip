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
#include "common.h"
#include "api.h"

namespace {

constexpr int THREADS = 1024;
constexpr int MAX_TENSORS = 16;

__device__ __forceinline__ double block_sum_double(double v, double* red) {
  for (int o = MS_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, MS_WAVE);
  __syncthreads();
  if ((threadIdx.x & (MS_WAVE - 1)) == 0) red[threadIdx.x / MS_WAVE] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < THREADS / MS_WAVE; ++w) s += red[w];
  return s;
}

__global__ void __launch_bounds__(THREADS)
verify_drafts_kernel(const float* __restrict__ p, const float* __restrict__ q, int V, const int* __restrict__ tokens,
                     const int* __restrict__ parents, const int* __restrict__ q_start, const float* __restrict__ uniforms,
                     int* __restrict__ nodes, int depth, int* __restrict__ counts, int* __restrict__ out) {
  __shared__ double red[THREADS / MS_WAVE];
  __shared__ int chosen;
  const int r = blockIdx.x, t0 = q_start[r], length = q_start[r + 1] - t0;
  int* path = nodes + (size_t)r * depth;
  if (length <= 0) {      // a row that pads a captured batch
    for (int i = threadIdx.x; i < depth; i += THREADS) path[i] = -1;
    if (threadIdx.x == 0) { counts[r] = 0; out[r] = -1; }
    return;
  }
  int node = 0, count = 1;
  double t, S;
  int tried;
  if (threadIdx.x == 0) path[0] = 0;
  for (;;) {
    const float* pr = p + (size_t)(t0 + node) * V;
    const float* qr = q ? q + (size_t)(t0 + node) * V : nullptr;
    t = 0.0; S = 1.0; tried = 0;
    int taken = -1;
    if (count < depth)
      for (int i = node + 1; i < length && taken < 0; ++i) {
        if (parents[t0 + i] != node) continue;
        const int x = tokens[t0 + i];
        const double u = uniforms[t0 + i];
        if (x < 0 || x >= V) continue;      // no token: nobody's guess
        ++tried;
        if (qr) {
          const double px = pr[x], qx = qr[x];
          if (u * qx * S < px - t * qx) { taken = i; break; }
          t += S;
          double mine = 0.0;
          for (int e = threadIdx.x; e < V; e += THREADS) mine += fmax(0.0, (double)pr[e] - t * (double)qr[e]);
          S = block_sum_double(mine, red);
        } else {
          bool gone = false;
          for (int j = node + 1; j < i; ++j) gone |= parents[t0 + j] == node && tokens[t0 + j] == x;
          const double px = gone ? 0.0 : (double)pr[x];
          if (u * S < px) { taken = i; break; }
          S -= px;
        }
      }
    if (taken < 0) break;
    node = taken;
    if (threadIdx.x == 0) path[count] = node;
    ++count;
  }
  for (int i = count + threadIdx.x; i < depth; i += THREADS) path[i] = -1;

  const float* pr = p + (size_t)(t0 + node) * V;
  const float* qr = q && t > 0.0 ? q + (size_t)(t0 + node) * V : nullptr;
  auto left = [&](int e, bool whole) -> double {
    const double v = pr[e];
    if (whole) return v;
    if (qr) return fmax(0.0, v - t * (double)qr[e]);
    if (!q && tried)
      for (int j = node + 1; j < length; ++j)
        if (parents[t0 + j] == node && tokens[t0 + j] == e) return 0.0;
    return v;
  };
  const int per = (V + THREADS - 1) / THREADS, lo = min(V, (int)threadIdx.x * per), hi = min(V, lo + per);
  bool whole = false;
  double mine, total;
  for (;;) {
    mine = 0.0;
    for (int e = lo; e < hi; ++e) mine += left(e, whole);
    total = block_sum_double(mine, red);
    if (total > 0.0 || whole) break;
    whole = true;
  }
  __shared__ double upto[THREADS];
  upto[threadIdx.x] = mine;
  if (threadIdx.x == 0) chosen = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    const double target = (double)uniforms[t0] * total;
    double run = 0.0;
    int pick = -1, last = 0;
    for (int k = 0; k < THREADS; ++k) {
      if (upto[k] > 0.0) last = k;
      if (run + upto[k] > target) { pick = k; break; }
      run += upto[k];
    }
    if (pick < 0) {      // (the sum in this order stayed below the mark: the last that has any)
      pick = last;
      run -= upto[last];
    }
    int found = 0;
    for (int e = min(V, pick * per); e < min(V, pick * per + per); ++e) {
      const double v = left(e, whole);
      if (v > 0.0) found = e;
      run += v;
      if (run > target) break;
    }
    out[r] = found;
    counts[r] = count;
  }
}

// Entry first[r] + nodes[r][i] of request r's cache to first[r] + i, for i < counts[r], in every layer and head.  A path is
// increasing, so an entry moves to its own place or an earlier one and no later entry of the path is written over; a block
// reads CHUNK entries before it writes them.
struct KeepTensor {
  void* pages;
  int heads, width, transposed;
};
struct KeepTensors { KeepTensor t[MAX_TENSORS]; };

constexpr int KEEP_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(KEEP_THREADS)
keep_tokens_kernel(KeepTensors tensors, int layers, int num_pages, int page_size, const int* __restrict__ block_table,
                   int table_stride, const int* __restrict__ table_rows, const int* __restrict__ first,
                   const int* __restrict__ nodes, int depth, const int* __restrict__ counts) {
  const KeepTensor kt = tensors.t[blockIdx.z];
  const int r = blockIdx.y, count = min(counts[r], depth), base = first[r];
  const int* table = block_table + (size_t)(table_rows ? table_rows[r] : r) * table_stride;
  const int* path = nodes + (size_t)r * depth;
  auto place = [&](int at, size_t& page, int& slot) {      // false: no page of this cache
    if (at < 0 || at / page_size >= table_stride) return false;
    const int id = table[at / page_size];
    slot = at % page_size;
    page = (size_t)id;
    return id > 0 && id < num_pages;
  };
  for (int lh = blockIdx.x; lh < layers * kt.heads; lh += gridDim.x) {
    const int layer = lh / kt.heads, head = lh - layer * kt.heads;
    T* pages = (T*)kt.pages + (size_t)layer * num_pages * kt.heads * page_size * kt.width;
    for (int e = threadIdx.x; e < kt.width; e += KEEP_THREADS) {
      // a thread moves its entries of every token in order
      for (int i = 0; i < count; ++i) {
        if (path[i] <= i) continue;
        size_t from, to;
        int from_slot, to_slot;
        if (!place(base + path[i], from, from_slot) || !place(base + i, to, to_slot)) continue;
        const size_t hf = (from * kt.heads + head) * page_size * kt.width, ht = (to * kt.heads + head) * page_size * kt.width;
        if (kt.transposed) pages[ht + (size_t)e * page_size + to_slot] = pages[hf + (size_t)e * page_size + from_slot];
        else pages[ht + (size_t)to_slot * kt.width + e] = pages[hf + (size_t)from_slot * kt.width + e];
      }
    }
  }
}

}  // namespace

extern "C" int ms_verify_drafts(const float* p, const float* q, int n_tokens, int vocab, const int* tokens, const int* parents,
                                const int* q_start, const float* uniforms, int n_requests, int* nodes, int depth, int* counts,
                                int* out, hipStream_t stream) {
  if (n_requests <= 0) return MS_OK;
  if (n_tokens < 0 || vocab <= 0 || depth <= 0 || n_requests > 65535) return MS_BAD_ARG;
  verify_drafts_kernel<<<dim3(n_requests), dim3(THREADS), 0, stream>>>(p, q, vocab, tokens, parents, q_start, uniforms, nodes, depth, counts, out);
  return ms_launch_status();
}

extern "C" int ms_keep_tokens_max() { return MAX_TENSORS; }

extern "C" int ms_keep_tokens(void* const* pages, const int* heads, const int* widths, const int* transposed, int n_tensors,
                              int layers, int num_pages, int page_size, const int* block_table, int table_stride,
                              const int* table_rows, const int* first, const int* nodes, int depth, const int* counts,
                              int n_requests, int dtype, hipStream_t stream) {
  if (n_tensors <= 0 || n_requests <= 0 || layers <= 0) return MS_OK;
  if (n_tensors > MAX_TENSORS || num_pages <= 0 || page_size <= 0 || table_stride <= 0 || depth <= 0 || n_requests > 65535)
    return MS_BAD_ARG;
  KeepTensors ts = {};
  int most = 1;
  for (int i = 0; i < n_tensors; ++i) {
    if (heads[i] <= 0 || widths[i] <= 0) return MS_BAD_ARG;
    ts.t[i] = {pages[i], heads[i], widths[i], transposed[i]};
    most = heads[i] > most ? heads[i] : most;
  }
  const long long items = (long long)layers * most;
  if (items > 0x7fffffffLL) return MS_UNSUPPORTED;
  dim3 grid((unsigned)(items < 65535 ? items : 65535), n_requests, n_tensors), block(KEEP_THREADS);
#define LAUNCH(T) keep_tokens_kernel<T><<<grid, block, 0, stream>>>(ts, layers, num_pages, page_size, block_table, table_stride, table_rows, first, nodes, depth, counts)
  if (dtype == MS_F32) LAUNCH(unsigned);
  else if (dtype == MS_BF16) LAUNCH(unsigned short);
  else return MS_BAD_ARG;
#undef LAUNCH
  return ms_launch_status();
}
