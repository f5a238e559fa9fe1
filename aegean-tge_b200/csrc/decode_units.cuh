// Single tokens over a paged cache of codes: how their work is cut among blocks, and how the parts are joined.  For attention_8bit.cu and
// attention_4bit.cu, whose kernels multiply (m16n8k16 and the like, positions or numbers of a head along the 16, heads along the 8).
//
// Work: the slices of 16 positions of all (request, kv head, tile of heads) units in one row, cut into equal runs, one per block, whatever the
// requests' lengths; the blocks work that out from the lengths on the device, so a captured graph stays right as they grow.  A unit
// counts as BEGIN slices more than it has: what a block spends on its queries, its first copies and the joining of its warps.  A run
// that holds a whole unit writes its output; parts of units are left as (maximum, sum, unnormalised output) in scratch memory, at
// most two per block, and a second kernel joins them in the order of the positions.  Few units over short contexts go without: a
// cluster of blocks has a unit, its slices in equal shares, and joins them through its shared memory.
#pragma once

#include "common.cuh"

namespace {

constexpr int DWARPS = 4;
// Measured with the 8-bit kernel as it was, and not with the 4-bit one: 64 requests of 2,048 to 4,096 at 40 heads over 8 at 0 / 12 / 24: 80.9 / 80.2 /
// 82.5 us (77.4 now), four of 32,768 47.8 / 45.6 / 45.9 (41.7), eight of 2,048 16.5 / 14.4 / 14.4 (10.9)
constexpr int BEGIN = 12;
constexpr float NONE = -3.0e38f;                // a running maximum before the first score (finite: -inf less this is still -inf)
constexpr float LOG2E = 1.4426950408889634f;

struct DecodeUnits {
  void* out;
  long long out_stride;
  const float* sink;
  const int *block_table, *q_start, *start_pos;
  int max_pages, num_pages, num_seqs, group, window;
  int units;                                    // per request: kv heads x tiles of heads
  int head_tiles, least;                        // least: slices of a run
  int page_shift;                               // pages are powers of two here: no division in the loop
  float *parts, *states;                        // [2 x blocks][heads of a tile][head_dim], [2 x blocks][heads of a tile][2]
};

// The row of a request's token; -1: it brings none.
__device__ __forceinline__ int row_of(const DecodeUnits& p, int seq) {
  const int row = p.q_start[seq], behind = p.q_start[seq + 1];
  return behind > row ? row : -1;
}

// The slices of 16 positions that request `seq` sees: [first, first + count), one at least.  `wrong`: what is to be reported of a token whose
// position is none, or one that the block table has no room for; the others are served as far as they go.
struct Slices { int lo, hi, first, count, wrong; };
__device__ __forceinline__ Slices slices_of(const DecodeUnits& p, int seq) {
  Slices s;
  const int start = p.start_pos[seq], here = p.q_start[seq], behind = p.q_start[seq + 1];      // one trip to memory
  const int pos = behind > here ? start : -1, room = p.max_pages << p.page_shift;
  s.hi = min(max(pos, -1), room - 1) + 1;
  s.wrong = behind <= here ? 0 : start < 0 ? TGE_STATUS_BAD_ROW : start >= room ? TGE_STATUS_BAD_PAGE : 0;
  s.lo = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
  s.first = s.lo >> 4;
  s.count = max((s.hi + 15) / 16 - s.first, 1);
  return s;
}

// What requests [0, upto) count for in the row, by the whole warp.
__device__ __forceinline__ int slices_before(const DecodeUnits& p, int upto, int lane) {
  int n = 0;
  for (int seq = lane; seq < upto; seq += 32) n += (slices_of(p, seq).count + BEGIN) * p.units;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) n += __shfl_xor_sync(0xffffffffu, n, offset);
  return n;
}
__device__ __forceinline__ int run_length(const DecodeUnits& p, int total, int blocks) { return max((total + blocks - 1) / blocks, p.least); }

// A head's sink in base-2 units (a finite one however large: it leaves zeros, not NaN).
__device__ __forceinline__ float sink_of(const DecodeUnits& p, int head) {
  const float sink = p.sink[head] * LOG2E;
  return sink > 3.4e38f ? 3.4e38f : sink;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {      // an 8x8 tile of 16-bit numbers across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ int cluster_rank() {
  int r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// What lies at `mine`'s place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ float2 of_rank(const float2* mine, int rank) {
  uint32_t at;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

// Where a block's run begins, by a whole warp: the request, where its units begin in the row, where the run begins and ends, the request's token.
__device__ __forceinline__ void find_run(const DecodeUnits& p, int lane, int (&start_of)[5]) {
  // 32 requests at a time; the first of them stay where they are
  const int first_count = lane < p.num_seqs ? (slices_of(p, lane).count + BEGIN) * p.units : 0;
  const int first_token = lane < p.num_seqs ? row_of(p, lane) : 0;
  int total = __reduce_add_sync(0xffffffffu, first_count);
  for (int seq = 32 + lane; seq - lane < p.num_seqs; seq += 32)
    total += __reduce_add_sync(0xffffffffu, seq < p.num_seqs ? (slices_of(p, seq).count + BEGIN) * p.units : 0);
  const int run = run_length(p, total, gridDim.x);
  const int from = (int)min((long long)run * blockIdx.x, (long long)total);
  int seq = 0, base = 0, token = first_token;
  while (seq < p.num_seqs) {
    int n = first_count;
    if (seq > 0) {
      n = seq + lane < p.num_seqs ? (slices_of(p, seq + lane).count + BEGIN) * p.units : 0;
      token = seq + lane < p.num_seqs ? row_of(p, seq + lane) : 0;
    }
    int upto = n;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += o;
    }
    const unsigned here = __ballot_sync(0xffffffffu, from < base + upto);
    const int who = here ? __ffs(here) - 1 : 31;
    const int behind = __shfl_sync(0xffffffffu, upto, who), mine = __shfl_sync(0xffffffffu, n, who);
    token = __shfl_sync(0xffffffffu, token, who);
    if (here) {
      base += behind - mine;
      seq += who;
      break;
    }
    base += behind;
    seq += 32;
  }
  if (lane == 0) {
    start_of[0] = seq;
    start_of[1] = base;
    start_of[2] = from;
    start_of[3] = min(from + run, total);
    start_of[4] = token;
  }
}

// The end of a block's part of a unit: its warps' states meet in shared memory, and become the output where that is all of the unit (or of a cluster's
// blocks all have come so far), else a part.  o: what the accumulators hold, a head's numbers times 1 / worth.
template <int HD, int NT>
struct Meeting {
  static constexpr int PITCH = HD + 4;
  float m[DWARPS][8 * NT], l[DWARPS][8 * NT], v[DWARPS][8 * NT];
};
template <typename T, int HD, int NT, bool CLUSTER, class Order>
__device__ __forceinline__ void leave_part(const DecodeUnits& p, Meeting<HD, NT>& meet, float* merge_o, float2* part_state, const float (&o)[NT][HD / 16][4],
                                           const float (&m)[NT][2], const float (&l)[NT][2], const float (&worth)[NT][2], int warp, int lane, int count,
                                           int skip, int length, int token, int head0, int heads_here, int rank, int ranks) {
  constexpr int HEADS = 8 * NT, MTILES = HD / 16, PITCH = HD + 4;   // merge_o: [warps][HEADS][PITCH], a head's numbers in the order of the accumulators
  const int g = lane >> 2, t = lane & 3;
  // the warps' states meet in shared memory: the two numbers of a lane and a tile side by side, then the lanes g, then the tiles
  __syncthreads();                                              // whoever still reads the unit before
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[nt][e];
#pragma unroll
      for (int offset = 4; offset < 32; offset <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
      const int head = 8 * nt + 2 * t + e;
      if (g == 0) {
        meet.m[warp][head] = m[nt][e];
        meet.l[warp][head] = sum;
        meet.v[warp][head] = worth[nt][e];
      }
      float* dst = merge_o + (warp * HEADS + head) * PITCH + 2 * g;
#pragma unroll
      for (int i = 0; i < MTILES; ++i) *reinterpret_cast<float2*>(dst + 16 * i) = make_float2(o[nt][i][e], o[nt][i][2 + e]);
    }
  }
  __syncthreads();
  const bool whole = !CLUSTER && length == count;
  const size_t place = (size_t)(2 * blockIdx.x + (skip == 0 ? 1 : 0)) * HEADS;
  for (int i = threadIdx.x; i < heads_here * (HD / 2); i += DWARPS * 32) {
    const int head = i / (HD / 2), pair = i - head * (HD / 2);
    float most = NONE;
#pragma unroll
    for (int w = 0; w < DWARPS; ++w) most = fmaxf(most, meet.m[w][head]);
    float sum = 0.0f;
    float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < DWARPS; ++w) {
      const float f = exp2_fast(meet.m[w][head] - most), fv = f * meet.v[w][head];
      const float2 x = *reinterpret_cast<const float2*>(merge_o + (w * HEADS + head) * PITCH + 2 * pair);
      sum = fmaf(f, meet.l[w][head], sum);
      acc.x = fmaf(fv, x.x, acc.x);
      acc.y = fmaf(fv, x.y, acc.y);
    }
    if (whole) {
      if (token < 0) continue;
      if (p.sink != nullptr) {
        const float sink = sink_of(p, head0 + head), top = fmaxf(most, sink), down = exp2_fast(most - top);
        sum = fmaf(sum, down, exp2_fast(sink - top));
        acc.x *= down;
        acc.y *= down;
      }
      const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
      T* dst = static_cast<T*>(p.out) + (size_t)token * p.out_stride + (size_t)(head0 + head) * HD + Order::number_of(pair);
      dst[0] = from_float<T>(acc.x * over);
      dst[1] = from_float<T>(acc.y * over);
    } else if (!CLUSTER) {
      *reinterpret_cast<float2*>(p.parts + (place + head) * HD + 2 * pair) = acc;
      if (pair == 0) *reinterpret_cast<float2*>(p.states + (place + head) * 2) = make_float2(most, sum);
    } else {
      *reinterpret_cast<float2*>(merge_o + head * PITCH + 2 * pair) = acc;             // in the first warp's place: read by this thread alone
      if (pair == 0) part_state[head] = make_float2(most, sum);
    }
  }
  if constexpr (CLUSTER) {
    cluster_sync();
    for (int i = rank * DWARPS * 32 + threadIdx.x; token >= 0 && i < heads_here * (HD / 2); i += ranks * DWARPS * 32) {
      const int head = i / (HD / 2), pair = i - head * (HD / 2);
      const float sink = p.sink != nullptr ? sink_of(p, head0 + head) : NONE;
      float top = sink, all = 0.0f;
      for (int r = 0; r < ranks; ++r) top = fmaxf(top, of_rank(&part_state[head], r).x);
      float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int r = 0; r < ranks; ++r) {
        const float2 state = of_rank(&part_state[head], r), x = of_rank(reinterpret_cast<const float2*>(merge_o + head * PITCH + 2 * pair), r);
        const float f = exp2_fast(state.x - top);
        all = fmaf(state.y, f, all);
        acc.x = fmaf(x.x, f, acc.x);
        acc.y = fmaf(x.y, f, acc.y);
      }
      if (p.sink != nullptr) all += exp2_fast(sink - top);
      const float over = all == 0.0f ? 0.0f : 1.0f / all;
      T* dst = static_cast<T*>(p.out) + (size_t)token * p.out_stride + (size_t)(head0 + head) * HD + Order::number_of(pair);
      dst[0] = from_float<T>(acc.x * over);
      dst[1] = from_float<T>(acc.y * over);
    }
    cluster_sync();                                             // nobody leaves while another reads its memory
  }
}

// Joins the parts of the units that more than one block worked on: one block per unit, two warps per head, which take the first and the
// second half of its parts.
constexpr int JOIN_WARPS = 16, JOIN_AHEAD = 8;

template <typename T, int HD, int NT, class Order>
__global__ void __launch_bounds__(JOIN_WARPS * 32) decode_join_kernel(const DecodeUnits p, int blocks) {
  constexpr int HEADS = 8 * NT, PAIRS = HD / 64;                   // pairs of numbers of a lane
  __shared__ int where[2];
  __shared__ float half_m[8], half_l[8], half_o[8][HD];
  pdl_trigger();
  const int seq = blockIdx.x, unit = blockIdx.y, lane = threadIdx.x & 31, warp = uniform_warp_index();
  if (warp == 0) {
    const int total = slices_before(p, p.num_seqs, lane), run = run_length(p, total, blocks);
    const int count = slices_of(p, seq).count, from = slices_before(p, seq, lane) + unit * (count + BEGIN) + BEGIN;
    if (lane == 0) {
      where[0] = from / run;
      where[1] = (from + count - 1) / run;
    }
  }
  __syncthreads();
  const int first = where[0], last = where[1];
  pdl_wait();                                                     // by every block: who waits for this kernel waits for the one before too
  if (first == last) return;
  const int kvh = unit / p.head_tiles, tile = unit - kvh * p.head_tiles;
  const int heads_here = min(HEADS, p.group - tile * HEADS), head0 = kvh * p.group + tile * HEADS;
  const int token = row_of(p, seq);
  if (token < 0) return;
  const int middle = first + (last - first + 2) / 2;
  const bool second = warp >= 8;
  for (int head = warp & 7; head < (heads_here + 7) / 8 * 8; head += 8) {
    const bool valid = head < heads_here;
    const int from = second ? middle : first, to = valid ? (second ? last + 1 : middle) : 0;
    // the block in which the unit begins left its part in its second place, the others in their first
    auto place = [&](int b) { return (size_t)(2 * b + (b == first ? 1 : 0)) * HEADS + head; };
    float most = NONE, sum = 0.0f;
    float2 acc[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) acc[i] = make_float2(0.0f, 0.0f);
    for (int b0 = from; b0 < to; b0 += 32) {
      // 32 parts' states, a lane each, then their numbers, the whole warp each
      const int count = min(32, to - b0);
      float2 state = make_float2(NONE, 0.0f);
      if (lane < count) state = *reinterpret_cast<const float2*>(p.states + place(b0 + lane) * 2);
      float2 x[JOIN_AHEAD][PAIRS];
      auto load = [&](int b) {
#pragma unroll
        for (int k = 0; k < JOIN_AHEAD; ++k)
#pragma unroll
          for (int i = 0; i < PAIRS; ++i)
            x[k][i] = b + k < count ? *reinterpret_cast<const float2*>(p.parts + place(b0 + b + k) * HD + 2 * (lane + 32 * i)) : make_float2(0.0f, 0.0f);
      };
      load(0);                                                     // on their way while the states' maximum is found
      const float top = fmaxf(most, warp_max(state.x));
      const float weight = exp2_fast(state.x - top), down = exp2_fast(most - top);
      sum = fmaf(sum, down, warp_sum(weight * state.y));
      most = top;
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) { acc[i].x *= down; acc[i].y *= down; }
      for (int b = 0; b < count; b += JOIN_AHEAD) {
        if (b > 0) load(b);
#pragma unroll
        for (int k = 0; k < JOIN_AHEAD; ++k) {
          const float f = __shfl_sync(0xffffffffu, weight, (b + k) & 31);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            acc[i].x = b + k < count ? fmaf(f, x[k][i].x, acc[i].x) : acc[i].x;
            acc[i].y = b + k < count ? fmaf(f, x[k][i].y, acc[i].y) : acc[i].y;
          }
        }
      }
    }
    __syncthreads();
    if (second) {
      if (lane == 0) {
        half_m[head & 7] = most;
        half_l[head & 7] = sum;
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) *reinterpret_cast<float2*>(&half_o[head & 7][2 * (lane + 32 * i)]) = acc[i];
    }
    __syncthreads();
    if (!second && valid) {
      const float sink = p.sink != nullptr ? sink_of(p, head0 + head) : NONE;
      const float top = fmaxf(fmaxf(most, half_m[head & 7]), sink);
      const float f0 = exp2_fast(most - top), f1 = exp2_fast(half_m[head & 7] - top);
      const float all = fmaf(sum, f0, f1 * half_l[head & 7]) + (p.sink != nullptr ? exp2_fast(sink - top) : 0.0f);
      const float over = all == 0.0f ? 0.0f : 1.0f / all;
      T* dst = static_cast<T*>(p.out) + (size_t)token * p.out_stride + (size_t)(head0 + head) * HD;
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(&half_o[head & 7][2 * (lane + 32 * i)]);
        const int d = Order::number_of(lane + 32 * i);
        dst[d] = from_float<T>(fmaf(acc[i].x, f0, f1 * x.x) * over);
        dst[d + 1] = from_float<T>(fmaf(acc[i].y, f0, f1 * x.y) * over);
      }
    }
  }
}

}  // namespace
