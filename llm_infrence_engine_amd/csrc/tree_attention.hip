// Attention of a step that checks trees of drafted tokens, keys read in place from pages.  Request r owns tokens
// q_start[r] .. q_start[r + 1] - 1 of the step, whose keys and values are stored as the last of its context_lens[r] entries.
// Token n, the request's i-th of the step, sees every entry before the step's and of the step's entries those whose bit is
// set in its row of `tree` (bit j % 32 of word j / 32: the request's j-th token):
//
//   out[n, h] = sum_j e^(s_j - max s) v_j / sum_j e^(s_j - max s) over the visible j,  s_j = scale q[n, h] . k_j
//
// A token that sees nothing gets zeros.  What is not visible cannot reach a result: such a score is replaced, never
// added to, and such a value is not multiplied (a NaN times a weight of zero would be one).
// Scores, maximum, exponentials, their sum and the weighted sum of values are float.
// This is the kernel of the sizes and layouts that csrc/tree_attention_mfma.hip does not take: a block owns one
// (token, query head), its waves take blocks of 64 keys in turn (a lane reads its own key's row, then every lane its own
// entries of one row of values after another) and are merged through LDS in order.  Every key is read for every token and head:
// 8 trees of up to 16 behind up to 2,000 keys, 28 heads of 48 on 4 in bfloat16, 465 us.
#include "common.h"
#include "api.h"

namespace {

constexpr int WAVES = 4, MAX_D = 256, MAX_C = MAX_D / MS_WAVE;

template <typename T>
__global__ void __launch_bounds__(WAVES * MS_WAVE)
tree_attention_kernel(const T* __restrict__ q, size_t q_stride, const T* __restrict__ k_pages, const T* __restrict__ v_pages,
                      const int* __restrict__ block_table, int table_stride, const int* __restrict__ table_rows,
                      const int* __restrict__ token_req, const int* __restrict__ q_start, const int* __restrict__ context_lens,
                      const int* __restrict__ n_live_tokens, const unsigned* __restrict__ tree, int words, T* __restrict__ out,
                      size_t out_stride, int nh, int nkv, int d, int dv, int page_size, float scale, int v_transposed) {
  __shared__ float qs[MAX_D], ms[WAVES], ls[WAVES], accs[WAVES][MAX_D];
  const int n = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & (MS_WAVE - 1), wave = threadIdx.x / MS_WAVE;
  if (n_live_tokens && n >= *n_live_tokens) return;      // a token that pads a captured batch
  const int r = token_req[n], kvh = h / (nh / nkv);
  const int q0 = q_start[r], qlen = q_start[r + 1] - q0, context = context_lens[r], before = context - qlen;
  if (n < q0 || n >= q0 + qlen) return;                  // (nor is one without a count of live ones)
  const int* table = block_table + (size_t)(table_rows ? table_rows[r] : r) * table_stride;
  const unsigned* bits = tree + (size_t)n * words;
  for (int i = threadIdx.x; i < d; i += WAVES * MS_WAVE) qs[i] = to_float(q[(size_t)n * q_stride + (size_t)h * d + i]) * scale;
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[MAX_C] = {};
  for (int base = wave * MS_WAVE; base < context; base += WAVES * MS_WAVE) {
    const int j = base + lane, i = j - before;
    const bool sees = j < context && (i < 0 || (i < 32 * words && (bits[i >> 5] >> (i & 31)) & 1u));
    float score = -INFINITY;
    size_t vrow = 0;
    if (sees) {
      const int page = j / page_size, off = j - page * page_size;
      const size_t head = (size_t)table[page] * nkv + kvh;
      const T* kp = k_pages + (head * page_size + off) * d;
      vrow = v_transposed ? head * dv * page_size + off : (head * page_size + off) * dv;
      float dot = 0.f;
      for (int e = 0; e < d; ++e) dot = fmaf(qs[e], to_float(kp[e]), dot);
      score = dot;
    }
    const float top = fmaxf(m, wave_max(score)), ref = top == -INFINITY ? 0.f : top;
    const float p = sees ? expf(score - ref) : 0.f, corr = expf(m - ref);      // 0 while nothing has been seen
    l = l * corr + wave_sum(p);
    m = top;
#pragma unroll
    for (int c = 0; c < MAX_C; ++c) acc[c] *= corr;
    for (unsigned long long left = __ballot(sees); left; left &= left - 1) {
      const int u = __builtin_ctzll(left);
      const float pu = __shfl(p, u, MS_WAVE);
      const unsigned lo = __shfl((unsigned)vrow, u, MS_WAVE), hi = __shfl((unsigned)(vrow >> 32), u, MS_WAVE);
      const T* vp = v_pages + (((size_t)hi << 32) | lo);
#pragma unroll
      for (int c = 0; c < MAX_C; ++c) {
        const int e = lane + c * MS_WAVE;
        if (e < dv) acc[c] = fmaf(pu, to_float(vp[v_transposed ? (size_t)e * page_size : (size_t)e]), acc[c]);
      }
    }
  }
  if (lane == 0) { ms[wave] = m; ls[wave] = l; }
#pragma unroll
  for (int c = 0; c < MAX_C; ++c) accs[wave][lane + c * MS_WAVE] = acc[c];
  __syncthreads();
  float top = ms[0];
  for (int w = 1; w < WAVES; ++w) top = fmaxf(top, ms[w]);
  if (top == -INFINITY) top = 0.f;
  float total = 0.f, factor[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) { factor[w] = expf(ms[w] - top); total = fmaf(ls[w], factor[w], total); }
  const float inv = total != 0.f ? 1.0f / total : 0.f;      // (a NaN stays one)
  T* op = out + (size_t)n * out_stride + (size_t)h * dv;
  for (int e = threadIdx.x; e < dv; e += WAVES * MS_WAVE) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) o = fmaf(accs[w][e], factor[w], o);
    op[e] = from_float<T>(o * inv);
  }
}

}  // namespace

extern "C" int ms_tree_attention_generic(const void* q, long long q_stride, const void* k_pages, const void* v_pages,
                                         const int* block_table, int table_stride, const int* table_rows, const int* token_req,
                                         const int* q_start, const int* context_lens, const int* n_live_tokens, const int* tree,
                                         int words, void* out, long long out_stride, int n_tokens, int num_heads,
                                         int num_kv_heads, int head_dim, int value_dim, int page_size, float scale,
                                         int v_transposed, int dtype, hipStream_t stream) {
  if (n_tokens <= 0) return MS_OK;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || page_size <= 0 || table_stride <= 0 || words <= 0)
    return MS_BAD_ARG;
  if (head_dim <= 0 || head_dim > MAX_D || value_dim <= 0 || value_dim > MAX_D || num_heads > 65535) return MS_UNSUPPORTED;
  dim3 grid(n_tokens, num_heads), block(WAVES * MS_WAVE);
#define LAUNCH(T) tree_attention_kernel<T><<<grid, block, 0, stream>>>((const T*)q, (size_t)q_stride, (const T*)k_pages, (const T*)v_pages, block_table, table_stride, table_rows, token_req, q_start, context_lens, n_live_tokens, (const unsigned*)tree, words, (T*)out, (size_t)out_stride, num_heads, num_kv_heads, head_dim, value_dim, page_size, scale, v_transposed)
  if (dtype == MS_F32) LAUNCH(float);
  else if (dtype == MS_BF16) LAUNCH(bf16);
  else return MS_BAD_ARG;
#undef LAUNCH
  return ms_launch_status();
}
