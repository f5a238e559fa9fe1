// Log probabilities of given tokens, with the entropy of their rows, their ranks and the best alternatives.
//
// Per row x of `vocab` logits, m = max x, Z = sum exp(x - m):
//   logprob = x_t - m - ln Z,  entropy = ln Z - sum exp(x - m) (x - m) / Z,  rank = how many tokens come before t,
//   and the `top` first tokens with their log probabilities, in the order of falling logits, the lower index first among equals.
// -inf is a token that cannot come: it adds nothing to either sum.  A row with NaN, with +inf or without a finite logit has no
// distribution: its log probabilities and its entropy are NaN (ranks and the order of the tokens still follow the logits, NaN last).
#include "common.cuh"

namespace {

constexpr int THREADS = 512;
constexpr int MOST_TOP = 32;

// An unsigned number that orders like the logit (-0 as 0, NaN below everything), and with the index below it, so that keys of a row
// are all different: a larger key comes first.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t bits = __float_as_uint(x + 0.0f);
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0u;
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int index) {
  return ((unsigned long long)ordered(x) << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float logit_of(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0u ? __int_as_float(0x7fc00000) : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

__device__ __forceinline__ unsigned long long block_largest(unsigned long long v, unsigned long long* scratch) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, offset);
    v = o > v ? o : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < THREADS / 32 ? scratch[threadIdx.x & 31] : 0ull;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, offset);
    v = o > v ? o : v;
  }
  return v;
}

// One block per row, which passes over it once for the largest key, once for the sums and once per alternative.
template <typename T>
__global__ void __launch_bounds__(THREADS) token_logprobs_simple_kernel(const T* logits, long long stride, const int* tokens, int vocab,
                                                                        int top, float* logprob, float* entropy, int* rank, int* top_ids,
                                                                        float* top_logprobs, int* status) {
  __shared__ unsigned long long keys[32];
  __shared__ float sums[32];
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x;
  const T* x = logits + (size_t)r * stride;
  const int token = tokens[r];
  const bool known = token >= 0 && token < vocab;
  if (!known && threadIdx.x == 0) atomicOr(status, TGE_STATUS_BAD_TOKEN);
  unsigned long long best = 0;
  bool broken = false;
  for (int i = threadIdx.x; i < vocab; i += THREADS) {
    const float v = to_float<T>(x[i]);
    broken |= !(v < INFINITY);
    best = max(best, key_of(v, i));
  }
  broken = __syncthreads_or(broken);
  best = block_largest(best, keys);
  const float m = logit_of(best);
  broken |= !(m > -INFINITY);
  const unsigned long long mine = known ? key_of(to_float<T>(x[token]), token) : ~0ull;
  float z = 0.0f, weighed = 0.0f, before = 0.0f;
  for (int i = threadIdx.x; i < vocab; i += THREADS) {
    const float v = to_float<T>(x[i]), d = v - m, e = expf(d);
    z += e;
    weighed = e > 0.0f ? fmaf(e, d, weighed) : weighed;
    before += key_of(v, i) > mine ? 1.0f : 0.0f;
  }
  z = block_sum(z, sums);
  weighed = block_sum(weighed, sums);
  before = block_sum(before, sums);
  const float nan = __int_as_float(0x7fc00000), log_z = logf(z);
  if (threadIdx.x == 0) {
    logprob[r] = broken || !known ? nan : logit_of(mine) - m - log_z;
    entropy[r] = broken ? nan : log_z - weighed / z;
    rank[r] = known ? (int)before : -1;
  }
  for (int k = 0; k < top; ++k) {
    if (threadIdx.x == 0) {
      top_ids[(size_t)r * top + k] = (int)~(uint32_t)best;
      top_logprobs[(size_t)r * top + k] = broken ? nan : logit_of(best) - m - log_z;
    }
    unsigned long long next = 0;
    for (int i = threadIdx.x; i < vocab && k + 1 < top; i += THREADS) {
      const unsigned long long key = key_of(to_float<T>(x[i]), i);
      if (key < best) next = max(next, key);
    }
    best = block_largest(next, keys);
  }
}

}  // namespace

TGE_API int tge_token_logprobs(const void* logits, int is_bf16, long long stride, const int* tokens, int rows, int vocab, int top,
                               float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs, int* status,
                               cudaStream_t stream) {
  TGE_REQUIRE(rows >= 0 && vocab > 0 && stride >= vocab, "token_logprobs: bad sizes rows=%d vocab=%d stride=%lld", rows, vocab, stride);
  TGE_REQUIRE(top >= 0 && top <= MOST_TOP && top <= vocab, "token_logprobs: %d alternatives of %d tokens, at most %d", top, vocab, MOST_TOP);
  if (rows == 0) return 0;
  if (is_bf16)
    tge_launch(token_logprobs_simple_kernel<__nv_bfloat16>, rows, THREADS, 0, stream, (const __nv_bfloat16*)logits, stride, tokens, vocab, top,
               logprob, entropy, rank, top_ids, top_logprobs, status);
  else
    tge_launch(token_logprobs_simple_kernel<float>, rows, THREADS, 0, stream, (const float*)logits, stride, tokens, vocab, top, logprob,
               entropy, rank, top_ids, top_logprobs, status);
  return tge_launched("token_logprobs", 1);
}
