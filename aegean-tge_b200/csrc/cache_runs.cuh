// Entries of a paged cache of codes read back: the positions that a step's queries may see, request after request, in runs of 64 positions
// [runs, kv_heads, 64, head_dim] (zeros behind a request's last), a block table over those runs and (starts, if wanted) the requests'
// first tokens counted from the first one's.  For cache_8bit.cu and cache_4bit.cu, which read the codes.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

namespace {

struct RunPlan {
  const int *block_table, *q_start, *start_pos;
  int max_pages, num_pages, page_size, first_seq, num_seqs, window;
  int *table, *starts;
  int runs, width;
  int* status;
};

// The first position that a step's queries see, from `start` on.  Pages in front of it are given back, also where they lie in its run of 64:
// those positions are zeros and nobody's fault.
__device__ __forceinline__ int first_seen(const RunPlan& p, int start) { return p.window > 0 ? max(start - p.window + 1, 0) : 0; }

struct Span { int first, count; };             // a request's runs: from position 64 first on
__device__ __forceinline__ Span span_of(const RunPlan& p, int seq) {
  const int start = p.start_pos[seq], held = start + p.q_start[seq + 1] - p.q_start[seq];
  Span s;
  s.first = first_seen(p, start) >> 6;
  s.count = max((held + 63) / 64 - s.first, 0);
  return s;
}

// The block table over the runs, and the first tokens if wanted.  A kernel of its own: attention kernels look block tables and first tokens up while
// the kernel in front of them still runs, so these have to be there before that one lets them start.  One block, a request to a thread at a time:
// one request after the other took 64 of them 9 us longer.
// The attention kernels size their memory by the host's numbers: where these leave out what the requests hold, the step is reported, and with first
// tokens of zero no request brings any.
constexpr int PLAN_THREADS = 256;
__global__ void __launch_bounds__(PLAN_THREADS) read_plan_kernel(const RunPlan p) {
  __shared__ int first_run[PLAN_THREADS], count[PLAN_THREADS], runs_upto[PLAN_THREADS], of_warp[PLAN_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int total = 0;
  bool beyond = false;
  for (int base = p.first_seq; base < p.num_seqs; base += PLAN_THREADS) {
    const int here = min(PLAN_THREADS, p.num_seqs - base);
    Span s{0, 0};
    if ((int)threadIdx.x < here) s = span_of(p, base + threadIdx.x);
    beyond |= s.first + s.count > p.width;
    int upto = s.count;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += v;
    }
    first_run[threadIdx.x] = s.first;
    count[threadIdx.x] = s.count;
    runs_upto[threadIdx.x] = upto - s.count;
    if (lane == 31) of_warp[warp] = upto;
    __syncthreads();
    for (int r = warp; r < here; r += PLAN_THREADS / 32) {
      int before = total + runs_upto[r];
      for (int w = 0; w < r >> 5; ++w) before += of_warp[w];
      for (int i = lane; i < p.width; i += 32) {
        const int at = i - first_run[r];
        p.table[(size_t)(base - p.first_seq + r) * p.width + i] = at >= 0 && at < count[r] ? before + at : -1;
      }
    }
    for (int w = 0; w < PLAN_THREADS / 32; ++w) total += of_warp[w];
    __syncthreads();
  }
  beyond = __syncthreads_or(beyond || total > p.runs);
  if (beyond && threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
  for (int i = threadIdx.x; i <= p.num_seqs - p.first_seq && p.starts != nullptr; i += PLAN_THREADS)
    p.starts[i] = beyond ? 0 : p.q_start[p.first_seq + i] - p.q_start[p.first_seq];
}

// Whose run is this?  The request (-1: the caller counted more runs than there are) and the run's place in it, by a whole block.
__device__ __forceinline__ void find_owner(const RunPlan& p, int run, int (&found)[2]) {
  if (threadIdx.x < 32) {                      // 32 requests at a time
    int before = 0, seq_found = -1, first_run = 0, index = 0;
    for (int base = p.first_seq; base < p.num_seqs && seq_found < 0; base += 32) {
      const int seq = base + threadIdx.x;
      Span s{0, 0};
      if (seq < p.num_seqs) s = span_of(p, seq);
      int upto = s.count;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, offset);
        if ((int)threadIdx.x >= offset) upto += v;
      }
      const unsigned mine = __ballot_sync(0xffffffffu, run < before + upto);
      if (mine != 0) {
        const int who = __ffs(mine) - 1;
        seq_found = base + who;
        index = run - before - (__shfl_sync(0xffffffffu, upto, who) - __shfl_sync(0xffffffffu, s.count, who));
        first_run = __shfl_sync(0xffffffffu, s.first, who);
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (threadIdx.x == 0) { found[0] = seq_found; found[1] = first_run + index; }
  }
  __syncthreads();
}

// float16 pages are over powers of two, multiples of 8: few runs differ.
__device__ __forceinline__ int exponent_above(float s) {      // of such a power that is no smaller than s > 0
  return min(max(((int)(__float_as_uint(s) >> 23) - 126 + 7) & ~7, -120), 120);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// max that keeps NaN, and turns an infinity into one
__device__ __forceinline__ float magnitude(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : __int_as_float(0x7fc00000);
}
__device__ __forceinline__ float larger(float a, float b) { return a > b || !(a == a) ? a : b; }

struct Eight { float x[8]; };
// Eight numbers as they lie in memory.
template <typename T> struct Raw;
template <> struct Raw<__nv_bfloat16> { uint4 w; };
template <> struct Raw<float> { float4 a, b; };
__device__ __forceinline__ Raw<__nv_bfloat16> raw_eight(const __nv_bfloat16* src) { return {*reinterpret_cast<const uint4*>(src)}; }
__device__ __forceinline__ Raw<float> raw_eight(const float* src) { return {reinterpret_cast<const float4*>(src)[0], reinterpret_cast<const float4*>(src)[1]}; }
__device__ __forceinline__ Eight eight(const Raw<__nv_bfloat16>& r) {
  const uint32_t w[4] = {r.w.x, r.w.y, r.w.z, r.w.w};
  Eight e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e.x[2 * i] = __uint_as_float(w[i] << 16);
    e.x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  return e;
}
__device__ __forceinline__ Eight eight(const Raw<float>& r) { return Eight{{r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w}}; }
template <typename T>
__device__ __forceinline__ Eight eight(const T* src) { return eight(raw_eight(src)); }

__device__ __forceinline__ void put_eight(__nv_bfloat16* dst, const Eight& e) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(e.x[2 * i], e.x[2 * i + 1]);
  *reinterpret_cast<uint4*>(dst) = raw;
}
__device__ __forceinline__ void put_eight(__half* dst, const Eight& e) {
  uint4 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(e.x[2 * i], e.x[2 * i + 1]);
  *reinterpret_cast<uint4*>(dst) = raw;
}
__device__ __forceinline__ void put_eight(float* dst, const Eight& e) {
  reinterpret_cast<float4*>(dst)[0] = make_float4(e.x[0], e.x[1], e.x[2], e.x[3]);
  reinterpret_cast<float4*>(dst)[1] = make_float4(e.x[4], e.x[5], e.x[6], e.x[7]);
}

}  // namespace
