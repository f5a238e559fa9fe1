// Paged causal attention over a cache held in 8 bits (see cache_8bit.cu for codes, blocks and scales).
//
// Per query head h at position p, kv head h / group, over the positions j <= p (with a window: j > p - window):
//   s_j = scale (k_scale_j / 127) sum_d q_d c_jd,   out = sum_j softmax(s)_j (v_scale_j / 127) c'_j
// the block's scale goes on the score and on the probability, so only whole numbers of up to 7 bits and a sign are multiplied with
// the queries and the probabilities.  A sink (float32 [heads]) joins the softmax's denominator once, with no key and no value.
// A row that sees no key (its pages are outside the pool) is zero.
#include "common.cuh"

namespace {

struct Attn8 {
  const void* q;
  void* out;
  long long q_stride, out_stride;
  const int8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  const int *block_table, *positions, *seq_of_token;
  const float* sink;
  int max_pages, num_pages, page_size, block, num_seqs, heads, kv_heads, group, head_dim, window;
  float scale;
  int* status;
};

// Any head size up to 256, any page size, any mix of portions, both run types: one warp per (token, query head), keys in position
// order, float32 on the CUDA cores.
template <typename T>
__global__ void __launch_bounds__(128) attention_8bit_simple_kernel(const Attn8 p) {
  constexpr int PER_LANE = 8;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= p.heads) return;
  const int kvh = h / p.group;
  const int pos = p.positions[t], seq = p.seq_of_token[t];
  T* out = static_cast<T*>(p.out) + (size_t)t * p.out_stride + (size_t)h * p.head_dim;
  const T* q = static_cast<const T*>(p.q) + (size_t)t * p.q_stride + (size_t)h * p.head_dim;
  float qv[PER_LANE], acc[PER_LANE];
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < p.head_dim ? to_float<T>(q[d]) : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  if (pos < 0 || seq < 0 || seq >= p.num_seqs) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
  } else {
    const int first = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
    const int* table = p.block_table + (size_t)seq * p.max_pages;
    for (int j = first; j <= pos; ++j) {
      const int page_index = j / p.page_size;
      const int page = page_index < p.max_pages ? table[page_index] : -1;
      if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
        break;
      }
      const size_t entry = ((size_t)page * p.kv_heads + kvh) * p.page_size + j % p.page_size;
      const int8_t *k = p.k_pages + entry * p.head_dim, *v = p.v_pages + entry * p.head_dim;
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int d = lane + 32 * i;
        if (d < p.head_dim) dot = fmaf(qv[i], (float)k[d], dot);
      }
      const float s = warp_sum(dot) * (p.k_scale[entry / p.block] * (1.0f / 127.0f)) * p.scale;
      const float m_new = fmaxf(m, s);
      const float corr = m == m_new ? 1.0f : expf(m - m_new), e = expf(s - m_new);
      const float w = e * (p.v_scale[entry / p.block] * (1.0f / 127.0f));
      l = l * corr + e;
#pragma unroll
      for (int i = 0; i < PER_LANE; ++i) {
        const int d = lane + 32 * i;
        if (d < p.head_dim) acc[i] = fmaf(w, (float)v[d], acc[i] * corr);
      }
      m = m_new;
    }
  }
  if (p.sink != nullptr) {
    const float m_new = fmaxf(m, p.sink[h]), corr = m == -INFINITY ? 0.0f : expf(m - m_new);
    l = l * corr + expf(p.sink[h] - m_new);
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) acc[i] *= corr;
  }
  const float over = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const int d = lane + 32 * i;
    if (d < p.head_dim) out[d] = from_float<T>(acc[i] * over);
  }
}

}  // namespace

TGE_API int tge_attention_8bit_simple(const void* q, int is_bf16, long long q_stride, const void* k_pages, const void* v_pages,
                                      const float* k_scale, const float* v_scale, int num_pages, int page_size, int block,
                                      const int* block_table, int max_pages, const int* positions, const int* seq_of_token, int num_seqs,
                                      int tokens, void* out, long long out_stride, int heads, int kv_heads, int head_dim, float scale,
                                      int window, const float* sink, int* status, cudaStream_t stream) {
  TGE_REQUIRE(tokens >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256 && window >= 0,
              "attention_8bit: bad sizes heads=%d kv_heads=%d head_dim=%d", heads, kv_heads, head_dim);
  TGE_REQUIRE(num_pages > 0 && page_size > 0 && block > 0 && page_size % block == 0 && max_pages > 0, "attention_8bit: bad page geometry");
  if (tokens == 0) return 0;
  const Attn8 p{q, out, q_stride, out_stride, (const int8_t*)k_pages, (const int8_t*)v_pages, k_scale, v_scale, block_table, positions,
                seq_of_token, sink, max_pages, num_pages, page_size, block, num_seqs, heads, kv_heads, heads / kv_heads, head_dim, window,
                scale, status};
  const dim3 grid(tokens, (heads + 3) / 4);
  if (is_bf16)
    tge_launch(attention_8bit_simple_kernel<__nv_bfloat16>, grid, 128, 0, stream, p);
  else
    tge_launch(attention_8bit_simple_kernel<float>, grid, 128, 0, stream, p);
  return tge_launched("attention_8bit", 1);
}
