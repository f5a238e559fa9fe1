// A paged key/value cache held in 4 bits: norm, rotation, quantisation and store of a step's keys and values; reading entries back.
//
// An entry (a position's key or value of one kv head) is cut into groups of 32 numbers.  A group has a base and a step, both bfloat16, and a
// code c of 0..15 stands for base + (c - 8) step, so that the sixteen values cover the group from its smallest number to its largest:
//   base = bf16(lo + (hi - lo) 8/15)                                  rounded to nearest
//   step = bf16(max((hi - base) / 7, (base - lo) / 8))                rounded up: no number lies outside
//   c    = rint((x - base) / step) + 8                                ties to even; 8 where the step is zero
// That is 5 bits a number, 4 of the code and 32 for every 32 numbers.  An entry is a function of its own row alone.
// An entry with a number that is not finite, or that is 2^96 or more, reads as NaN (so that no sum or product over a cache overflows).
//
// Pages: codes uint8 [pages, kv_heads, page, 16 groups]; (step, base) bfloat16 [pages, kv_heads, page, 2 groups].  Four neighbours' codes make a
// unit of 16 bits, the first of them lowest; unit (g, j), numbers 32 j + 4 g .. + 3, is the (g groups + j)-th of its entry.  That is the order in
// which attention_4bit.cu wants them: a lane's numbers of all groups side by side.  A last group that is not full has codes of zero behind.
//
// Norm of a head's queries and keys, before the rotation: x / sqrt(mean(x^2) + eps) times a weight per number.  Rotation over the first `rotary`
// numbers of a head: numbers d and d + rotary / 2 (or, for pairs, 2 d and 2 d + 1) become (lo cos - hi sin, lo sin + hi cos).  Both in float32, every
// product and sum rounded for itself and the mean taken in 64 bits, so that entries are the same wherever they are computed: what lies near
// the border between two codes would go either way otherwise.
#include <algorithm>
#include <type_traits>

#include "cache_runs.cuh"

namespace {

constexpr int GROUP = 32;                      // numbers of a group
constexpr int MOST_GROUPS = 8;                 // head_dim <= 256
constexpr float LIMIT = 0x1p96f;

struct Group { float step, base; };

__device__ __forceinline__ float bf16_nearest(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
__device__ __forceinline__ float bf16_above(float x) {            // x >= 0
  return __uint_as_float((__float_as_uint(x) + 0xffffu) & 0xffff0000u);
}
__device__ __forceinline__ Group group_of(float lo, float hi) {
  Group g;
  g.base = bf16_nearest(__fadd_rn(lo, __fmul_rn(__fsub_rn(hi, lo), (float)(8.0 / 15.0))));
  g.step = bf16_above(fmaxf(__fdiv_rn(__fsub_rn(hi, g.base), 7.0f), __fmul_rn(__fsub_rn(g.base, lo), 0.125f)));
  return g;
}
__device__ __forceinline__ uint32_t code_of(const Group& g, float x) {
  if (!(g.step > 0.0f)) return 8u;
  return (uint32_t)min(max(__float2int_rn(__fdiv_rn(__fsub_rn(x, g.base), g.step)) + 8, 0), 15);
}
// The same where a group's numbers go through one after the other.  The quotient is rounded as the division rounds it: q = fl(y r), r the step's rounded
// reciprocal, and then fl(q + fl(y - q step) r), which is the nearest number of y / step (P. Markstein, Computation of elementary functions on
// the IBM RISC System/6000 processor, 1990) while nothing underflows; smaller steps are divided by.  With 1.5 2^23 + 8 added the sum's last four
// bits are the code (ties to even: 8 is), which lies within 0..15 without a clamp: the step has been rounded up.
struct Coder4 {
  float base, step, over;
  bool by_parts;
  __device__ __forceinline__ explicit Coder4(const Group& g) {
    base = g.base;
    step = g.step;
    over = __frcp_rn(g.step);
    by_parts = g.step > 1e-25f;
  }
  __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) const {
    if (!by_parts) {
      const Group g{step, base};
      return code_of(g, a) | code_of(g, b) << 4 | code_of(g, c) << 8 | code_of(g, d) << 12;
    }
    auto sum = [&](float x) {
      const float y = __fsub_rn(x, base), q = __fmul_rn(y, over);
      return __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-q, step, y), over, q), 12582920.0f));
    };
    return (sum(a) & 15u) | (sum(b) & 15u) << 4 | (sum(c) & 15u) << 8 | (sum(d) & 15u) << 12;
  }
};
__device__ __forceinline__ uint32_t packed(const Group& g) { return (__float_as_uint(g.step) >> 16) | (__float_as_uint(g.base) & 0xffff0000u); }
__device__ __forceinline__ Group unpacked(uint32_t w) { return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)}; }
__device__ __forceinline__ float value_of(const Group& g, uint32_t code) { return fmaf((float)((int)code - 8), g.step, g.base); }
constexpr uint32_t NO_GROUP = 0x7fc07fc0u;      // step and base NaN

struct StoreParams4 {
  const void* qkv;
  void* q_out;
  long long row_stride, q_stride;
  const float *cos_table, *sin_table, *q_norm, *k_norm;
  double eps;
  int table_rows;
  const int *positions, *seq_of_token, *block_table;
  int max_pages;
  uint8_t *k_pages, *v_pages;
  uint32_t *k_groups, *v_groups;
  int num_pages, page_size, tokens, num_seqs, heads, kv_heads, head_dim, rotary, pairs;
  int* status;
};

__device__ __forceinline__ float turned_first(float lo, float hi, float c, float s) { return __fsub_rn(__fmul_rn(lo, c), __fmul_rn(hi, s)); }
__device__ __forceinline__ float turned_second(float lo, float hi, float c, float s) { return __fadd_rn(__fmul_rn(lo, s), __fmul_rn(hi, c)); }
// (A mean that float32 has no room for goes over an even power of two first: the same bits times its root.)
__device__ __forceinline__ float over_root(double sum, int count, double eps) {
  const double mean = sum / count + eps;
  if (mean > 1e38) return __fmul_rn(__fdiv_rn(1.0f, __fsqrt_rn((float)(mean * 0x1p-140))), 0x1p-70f);
  return __fdiv_rn(1.0f, __fsqrt_rn((float)mean));
}
__device__ __forceinline__ double lanes_sum(double v, int lanes) {
  for (int offset = lanes / 2; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
  return v;
}

// A positive normal float32 as a double by its bits: the conversion does 16 numbers a clock and SM, this and the sum some 60 (a store of 8,192 tokens at 40 heads
// over 8 with norms 99 us with the one, 87 with the other, before the codes' quotients were found by parts).  0 becomes 2^-127, which no sum with an eps shows.
__device__ __forceinline__ double widened(float x) {
  const uint32_t bits = __float_as_uint(x);
  return __hiloint2double((int)((bits >> 3) + 0x38000000u), (int)(bits << 29));
}

// Queries alone have no kv heads and no pages.

// Any head size up to 256, any strides: one warp per (token, head), a lane per number of a group.
constexpr int WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) store_4bit_kernel(const StoreParams4 p) {
  pdl_trigger();
  const int lane = threadIdx.x & 31, t = blockIdx.x, h = blockIdx.y * WARPS + (threadIdx.x >> 5);
  const int pos = p.positions[t], seq = p.seq_of_token[t];
  pdl_wait();
  if (h >= p.heads + 2 * p.kv_heads) return;
  const bool is_query = h < p.heads, is_key = !is_query && h < p.heads + p.kv_heads, turn = p.rotary > 0 && (is_query || is_key);
  if (pos < 0 || (p.rotary > 0 && pos >= p.table_rows) || seq < 0 || seq >= p.num_seqs) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
    return;
  }
  const T* row = static_cast<const T*>(p.qkv) + (size_t)t * p.row_stride + (size_t)h * p.head_dim;
  const float* weight = is_query ? p.q_norm : is_key ? p.k_norm : nullptr;
  float over = 1.0f;
  if (weight != nullptr) {
    double sum = 0.0;
    for (int d = lane; d < p.head_dim; d += 32) {
      const double x = to_float<T>(row[d]);
      sum += x * x;
    }
    over = over_root(lanes_sum(sum, 32), p.head_dim, p.eps);
  }
  auto plain = [&](int d) {
    const float x = to_float<T>(row[d]);
    return weight != nullptr ? __fmul_rn(__fmul_rn(x, over), weight[d]) : x;
  };
  const int half = p.rotary >> 1;
  auto number = [&](int d) {
    const float own = plain(d);
    if (!turn || d >= p.rotary) return own;
    const bool first = p.pairs ? (d & 1) == 0 : d < half;
    const float other = plain(p.pairs ? d ^ 1 : first ? d + half : d - half);
    const size_t at = (size_t)pos * half + (p.pairs ? d >> 1 : first ? d : d - half);
    const float c = p.cos_table[at], s = p.sin_table[at];
    return first ? turned_first(own, other, c, s) : turned_second(other, own, c, s);
  };
  if (is_query) {
    T* dst = static_cast<T*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * p.head_dim;
    for (int d = lane; d < p.head_dim; d += 32) dst[d] = from_float<T>(number(d));
    return;
  }
  const int page_index = pos / p.page_size;
  const int page = page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
    return;
  }
  const int groups = (p.head_dim + GROUP - 1) / GROUP;
  const size_t entry = ((size_t)page * p.kv_heads + (h - p.heads - (is_key ? 0 : p.kv_heads))) * p.page_size + pos % p.page_size;
  uint16_t* codes = reinterpret_cast<uint16_t*>(is_key ? p.k_pages : p.v_pages) + entry * 8 * groups;
  uint32_t* to = (is_key ? p.k_groups : p.v_groups) + entry * groups;
  float x[MOST_GROUPS];
  bool fine = true;
#pragma unroll
  for (int j = 0; j < MOST_GROUPS; ++j) {
    const int d = GROUP * j + lane;
    x[j] = d < p.head_dim ? number(d) : 0.0f;
    fine &= fabsf(x[j]) < LIMIT;
  }
  fine = __all_sync(0xffffffffu, fine);
#pragma unroll
  for (int j = 0; j < MOST_GROUPS; ++j) {
    if (j >= groups) break;
    const bool inside = GROUP * j + lane < p.head_dim;
    const Group g = group_of(-warp_max(inside ? -x[j] : -INFINITY), warp_max(inside ? x[j] : -INFINITY));
    uint32_t unit = fine && inside ? code_of(g, x[j]) << (4 * (lane & 3)) : 0u;
    unit |= __shfl_xor_sync(0xffffffffu, unit, 1);
    unit |= __shfl_xor_sync(0xffffffffu, unit, 2);
    if ((lane & 3) == 0) codes[(lane >> 2) * groups + j] = (uint16_t)unit;
    if (lane == 0) to[j] = fine ? packed(g) : NO_GROUP;
  }
}

// ---------------------------------------------------------------------------
// The same by units of eight numbers, for head sizes 32, 64, 128 and 256 that are rotated whole or not at all and rows on 16 bytes.  A block has a token; HEAD / 16
// lanes have a head's row, eight numbers of its first half and eight of its second, and take the token's heads in turn, three rows on their way at
// a time, the angles loaded once.  Bound by the trips to memory one behind the other where there are few tokens; what bounds it where
// there are many was not profiled.  us: one token 2.5; 2,048 at 28 heads over 4 9.8, with norms 14.9 (34 MB, 5.5 at a copy's rate); 8,192 at 40 over 8
// 51 and 75 (33).  With a division for every code 3.4, 11.8, 18, 62 and 99; two rows or four blocks to an SM 12 and 11
// where this takes 9.7; rows asked into L2 ahead no faster.
// ---------------------------------------------------------------------------
constexpr int UNIT_THREADS = 256, UNIT_AHEAD = 3;         // at most; as many as it takes for a token's heads in UNIT_AHEAD turns

template <typename T, int HEAD, bool NORM>
__global__ void __launch_bounds__(UNIT_THREADS, sizeof(T) == 2 ? 3 : 2) store_4bit_units_kernel(const StoreParams4 p) {
  constexpr int LANES = HEAD / 16, HALF = HEAD / 2, GROUPS = HEAD / GROUP;
  pdl_trigger();
  const int rows_at_once = blockDim.x / LANES, mine = threadIdx.x / LANES, j = threadIdx.x % LANES;
  const bool rotate = p.rotary > 0;
  const int t = blockIdx.x, pos = p.positions[t], seq = p.seq_of_token[t];
  pdl_wait();
  // the first rows are on their way before anything has to be looked up
  const T* row = static_cast<const T*>(p.qkv) + (size_t)t * p.row_stride + 8 * j;
  const int heads = p.heads + 2 * p.kv_heads;
  Raw<T> lo_raw[UNIT_AHEAD], hi_raw[UNIT_AHEAD];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < UNIT_AHEAD; ++i) {
      const int h = min(h0 + i * rows_at_once, heads - 1);
      lo_raw[i] = raw_eight(row + (size_t)h * HEAD);
      hi_raw[i] = raw_eight(row + (size_t)h * HEAD + HALF);
    }
  };
  load(mine);
  if (pos < 0 || (rotate && pos >= p.table_rows) || seq < 0 || seq >= p.num_seqs) {
    if (threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
    return;
  }
  // halves: the angles of numbers 8 j .. of the first half; pairs: four angles for the eight of the first half, four for those of the second
  Eight c, s;
  if (rotate) {
    const size_t at = (size_t)pos * HALF;
    if (p.pairs) {
      auto four_and_four = [&](const float* table) {
        const float4 a = *reinterpret_cast<const float4*>(table + at + 4 * j), b = *reinterpret_cast<const float4*>(table + at + HALF / 2 + 4 * j);
        return Eight{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
      };
      c = four_and_four(p.cos_table);
      s = four_and_four(p.sin_table);
    } else {
      c = eight(p.cos_table + at + 8 * j);
      s = eight(p.sin_table + at + 8 * j);
    }
  }
  const int page_index = pos / p.page_size, slot = pos - page_index * p.page_size;
  const int page = page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
  const bool here = page >= 0 && page < p.num_pages;
  if (!here && p.kv_heads > 0 && threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
  for (int h0 = mine; h0 < heads + mine; h0 += UNIT_AHEAD * rows_at_once) {       // the same number of rounds for every lane of a warp
    if (h0 != mine) load(h0);
#pragma unroll
    for (int i = 0; i < UNIT_AHEAD; ++i) {
      const int h = h0 + i * rows_at_once;
      Eight lo = eight(lo_raw[i]), hi = eight(hi_raw[i]);
      const bool valid = h < heads, to_cache = h >= p.heads, turns = h < p.heads + p.kv_heads;
      if constexpr (NORM) {
        const float* weight = to_cache ? p.k_norm : p.q_norm;
        const bool normed = turns && weight != nullptr;
        if (__any_sync(0xffffffffu, normed)) {
          double sum = 0.0;
          float rough = 0.0f;
          auto add = [&](float x) {
            const float square = x * x;                             // (of a bfloat16 exactly)
            rough += square;
            if constexpr (sizeof(T) == 2) sum += widened(square);
            else {
              const double wide = widened(fabsf(x));
              sum = fma(wide, wide, sum);
            }
          };
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            add(lo.x[k]);
            add(hi.x[k]);
          }
          if (!(rough <= 1e38f) || p.eps < 1e-30) {                 // squares that float32 has no room for, numbers that are not finite
            sum = 0.0;
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += (double)lo.x[k] * (double)lo.x[k] + (double)hi.x[k] * (double)hi.x[k];
          }
          const float over = over_root(lanes_sum(sum, LANES), HEAD, p.eps);
          if (normed) {
            const Eight a = eight(weight + 8 * j), b = eight(weight + HALF + 8 * j);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              lo.x[k] = __fmul_rn(__fmul_rn(lo.x[k], over), a.x[k]);
              hi.x[k] = __fmul_rn(__fmul_rn(hi.x[k], over), b.x[k]);
            }
          }
        }
      }
      if (rotate && turns) {
        auto turn = [](float& u, float& v, float cos, float sin) {
          const float a = u, b = v;
          u = turned_first(a, b, cos, sin);
          v = turned_second(a, b, cos, sin);
        };
        if (p.pairs) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            turn(lo.x[2 * k], lo.x[2 * k + 1], c.x[k], s.x[k]);
            turn(hi.x[2 * k], hi.x[2 * k + 1], c.x[4 + k], s.x[4 + k]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) turn(lo.x[k], hi.x[k], c.x[k], s.x[k]);
        }
      }
      if (valid && !to_cache) {
        T* dst = static_cast<T*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * HEAD + 8 * j;
        put_eight(dst, lo);
        put_eight(dst + HALF, hi);
      }
      if (!__any_sync(0xffffffffu, valid && to_cache)) continue;
      float low[2] = {lo.x[0], hi.x[0]}, high[2] = {lo.x[0], hi.x[0]}, nothing = 0.0f;       // NaN where a number is not finite
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        nothing = __fmaf_rn(lo.x[k], 0.0f, __fmaf_rn(hi.x[k], 0.0f, nothing));
        low[0] = fminf(low[0], lo.x[k]);
        low[1] = fminf(low[1], hi.x[k]);
        high[0] = fmaxf(high[0], lo.x[k]);
        high[1] = fmaxf(high[1], hi.x[k]);
      }
      if (HEAD == 32) {
        low[0] = low[1] = fminf(low[0], low[1]);
        high[0] = high[1] = fmaxf(high[0], high[1]);
      }
#pragma unroll
      for (int offset = 1; offset < (LANES < 4 ? LANES : 4); offset <<= 1)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          low[half] = fminf(low[half], __shfl_xor_sync(0xffffffffu, low[half], offset));
          high[half] = fmaxf(high[half], __shfl_xor_sync(0xffffffffu, high[half], offset));
        }
      const bool mine_fine = nothing == 0.0f && fmaxf(fmaxf(-low[0], high[0]), fmaxf(-low[1], high[1])) < LIMIT;
      constexpr uint32_t OF_HEAD = LANES == 32 ? 0xffffffffu : (1u << (LANES & 31)) - 1u;
      const bool fine = (__ballot_sync(0xffffffffu, !mine_fine) >> (threadIdx.x & 31 & ~(LANES - 1)) & OF_HEAD) == 0u;
      const Group of[2] = {group_of(low[0], high[0]), group_of(low[1], high[1])};
      uint32_t unit[2][2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Coder4 coder(of[half]);
        const Eight& x = half ? hi : lo;
#pragma unroll
        for (int u = 0; u < 2; ++u) unit[half][u] = fine ? coder.four(x.x[4 * u], x.x[4 * u + 1], x.x[4 * u + 2], x.x[4 * u + 3]) : 0u;
      }
      // what the lane four away has of the groups beside this one's (a head of 128 numbers)
      [[maybe_unused]] const bool odd = (j & 4) != 0;
      [[maybe_unused]] uint32_t other = 0;
      if constexpr (HEAD == 128) other = __shfl_xor_sync(0xffffffffu, odd ? unit[0][0] | unit[1][0] << 16 : unit[0][1] | unit[1][1] << 16, 4);
      if (valid && to_cache && here) {
        const bool is_key = turns;
        const size_t entry = ((size_t)page * p.kv_heads + (h - p.heads - (is_key ? 0 : p.kv_heads))) * p.page_size + slot;
        uint8_t* codes = (is_key ? p.k_pages : p.v_pages) + entry * (HEAD / 2);
        uint32_t* to = (is_key ? p.k_groups : p.v_groups) + entry * GROUPS;
        if constexpr (HEAD == 32) {
          *reinterpret_cast<uint32_t*>(codes + 4 * j) = unit[0][0] | unit[0][1] << 16;
          *reinterpret_cast<uint32_t*>(codes + 8 + 4 * j) = unit[1][0] | unit[1][1] << 16;
        } else if constexpr (HEAD == 64) {
          *reinterpret_cast<uint2*>(codes + 8 * j) = make_uint2(unit[0][0] | unit[1][0] << 16, unit[0][1] | unit[1][1] << 16);
        } else if constexpr (HEAD == 128) {
          const uint32_t a = odd ? __byte_perm(other, unit[0][1], 0x5410) : __byte_perm(unit[0][0], other, 0x5410);
          const uint32_t b = odd ? __byte_perm(other, unit[1][1], 0x5432) : __byte_perm(unit[1][0], other, 0x7610);
          *reinterpret_cast<uint2*>(codes + 8 * (2 * (j & 3) + (odd ? 1 : 0))) = make_uint2(a, b);
        } else {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int u = 0; u < 2; ++u)
              reinterpret_cast<uint16_t*>(codes)[(2 * (j & 3) + u) * GROUPS + half * (GROUPS / 2) + (j >> 2)] = (uint16_t)unit[half][u];
        }
        if ((j & 3) == 0) {
          to[HEAD == 32 ? 0 : j >> 2] = fine ? packed(of[0]) : NO_GROUP;
          if (HEAD != 32) to[GROUPS / 2 + (j >> 2)] = fine ? packed(of[1]) : NO_GROUP;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Entries read back (see cache_runs.cuh for the runs of 64 positions).  In float32, bfloat16, or for the attention kernel that takes float16 pages
// (attention_tc2.cuh) in float16 over powers of two of a run and head.  For attention (starts are wanted): it multiplies every value of a tile with a
// probability, unseen ones with zero, so values are finite there: a position whose value's groups are not gets a key that is not, which whoever sees it
// turns into the same and nobody else looks at.
// Bound by the bytes written, 3.2 (6.4) to a byte read.  A thread has the units of one g: a position's four neighbours of every group.
// ---------------------------------------------------------------------------
struct ReadParams4 : RunPlan {
  const uint8_t *k_pages, *v_pages;
  const uint32_t *k_groups, *v_groups;
  int kv_heads, head_dim;
  void *k_out, *v_out;
  float2* factors;                             // [runs, kv_heads, 64], for float16 output: of runs whose entries lie far apart, see below
  int* exponents;                              // [runs, kv_heads], for float16 output: f below, e above; 1: the run has factors
};

__device__ __forceinline__ void put_four(float* dst, const float (&x)[4]) { *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void put_four(__nv_bfloat16* dst, const float (&x)[4]) {
  uint2 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
  h[0] = __floats2bfloat162_rn(x[0], x[1]);
  h[1] = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(dst) = raw;
}
__device__ __forceinline__ void put_four(__half* dst, const float (&x)[4]) {
  uint2 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
  h[0] = __floats2half2_rn(x[0], x[1]);
  h[1] = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(dst) = raw;
}

// BYTES on their own boundary as words (two bytes: the lower half of one).
template <int BYTES>
struct Words { uint32_t w[(BYTES + 3) / 4]; };
template <int BYTES>
__device__ __forceinline__ Words<BYTES> words_at(const void* src) {
  Words<BYTES> r;
  if constexpr (BYTES == 2) r.w[0] = *static_cast<const uint16_t*>(src);
  else if constexpr (BYTES == 4) r.w[0] = *static_cast<const uint32_t*>(src);
  else if constexpr (BYTES == 8) {
    const uint2 v = *static_cast<const uint2*>(src);
    r.w[0] = v.x; r.w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = static_cast<const uint4*>(src)[i];
      r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
    }
  }
  return r;
}

// What a group's values are at most, in magnitude (NaN, infinite: it has none).
__device__ __forceinline__ float group_most(uint32_t w) {
  const Group g = unpacked(w);
  return larger(fabsf(fmaf(7.0f, g.step, g.base)), fabsf(fmaf(-8.0f, g.step, g.base)));
}
template <int GROUPS>
__device__ __forceinline__ float entry_most(const Words<4 * GROUPS>& of) {
  float most = 0.0f;
#pragma unroll
  for (int j = 0; j < GROUPS; ++j) most = larger(most, group_most(of.w[j]));
  return most;
}

// float16's numbers are 2^-24 apart below 2^-14, so a group whose largest number is at least 2^-13 of the run's power keeps 2^-12 of it, which is what
// float16 keeps of any.  A run with a smaller group holds every entry over a power of two of its own, and these go to the attention as factors: what
// multiplies a key's scores, and the logarithm to the base 2 of what multiplies a value's probability; so does a run with values of zero beside
// others, because a row that sees those alone adds nothing, whatever the others' power says.  What then is below 2^-24 of its own entry's largest
// number is zero in a portion, as it would be beside that number in a float32 sum.
__device__ __forceinline__ int exponent_just_above(float s) {     // of the smallest power of two above s
  return s > 0.0f ? min(max((int)(__float_as_uint(s) >> 23) - 126, -120), 120) : 0;
}

template <typename T, int GROUPS>
__global__ void __launch_bounds__(256) read_4bit_kernel(const ReadParams4 p) {
  constexpr bool HALVES = std::is_same<T, __half>::value;
  constexpr int HEAD = GROUPS * GROUP, AHEAD = GROUPS <= 4 && !HALVES ? 2 : 1;
  __shared__ int found[2];
  __shared__ float most[2][2], least[2][2];    // float16: the largest numbers of the run's first and second 32 positions, keys' and values', and its smallest groups'
  const int run = blockIdx.x, page_shift = __ffs(p.page_size) - 1;
  pdl_wait();
  pdl_trigger();                               // behind the wait: see read_plan_kernel
  find_owner(p, run, found);
  const int seq = found[0], tile = found[1];
  for (int kvh = blockIdx.y; kvh < p.kv_heads; kvh += gridDim.y) {
    T* k_dst = static_cast<T*>(p.k_out) + ((size_t)run * p.kv_heads + kvh) * 64 * HEAD;
    T* v_dst = static_cast<T*>(p.v_out) + ((size_t)run * p.kv_heads + kvh) * 64 * HEAD;
    if (seq < 0) {
      for (int i = threadIdx.x; i < 64 * HEAD; i += 256) k_dst[i] = v_dst[i] = from_float<T>(0.0f);
      if (HALVES && threadIdx.x == 0) p.exponents[(size_t)run * p.kv_heads + kvh] = 0;
      continue;
    }
    const int start = p.start_pos[seq], held = start + p.q_start[seq + 1] - p.q_start[seq], seen_from = first_seen(p, start);
    auto entry_of = [&](int pos, bool& here) {
      const int page_index = pos >> page_shift;
      const int page = pos < held && page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
      here = page >= 0 && page < p.num_pages;
      return here ? ((size_t)(page * p.kv_heads + kvh) << page_shift) + (pos & (p.page_size - 1)) : (size_t)0;
    };
    [[maybe_unused]] float over[2] = {1.0f, 1.0f};
    [[maybe_unused]] bool apart = false;
    if constexpr (HALVES) {
      __syncthreads();                         // whoever still reads those of the head before
      float of[2] = {0.0f, 0.0f};
      if (threadIdx.x < 64) {
        bool here;
        const size_t entry = entry_of(tile * 64 + threadIdx.x, here);
        float small[2] = {INFINITY, INFINITY};
        if (here) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const Words<4 * GROUPS> w = words_at<4 * GROUPS>((kv ? p.v_groups : p.k_groups) + entry * GROUPS);
            of[kv] = entry_most<GROUPS>(w);
#pragma unroll
            for (int j = 0; j < GROUPS; ++j) {
              const float g = group_most(w.w[j]);
              if (g > 0.0f) small[kv] = fminf(small[kv], g);
            }
          }
          if (of[1] == 0.0f) small[1] = 0.0f;
        }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const float a = warp_max(of[kv] < INFINITY ? of[kv] : 0.0f), b = -warp_max(-small[kv]);
          if ((threadIdx.x & 31) == 0) {
            most[threadIdx.x >> 5][kv] = a;
            least[threadIdx.x >> 5][kv] = b;
          }
        }
      }
      __syncthreads();
      int e[2];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float m = fmaxf(most[0][kv], most[1][kv]);
        e[kv] = m > 0.0f ? exponent_above(m) : 0;
        over[kv] = power_of_two(-e[kv]);
        apart |= m > 0.0f && fminf(least[0][kv], least[1][kv]) < power_of_two(e[kv]) * 0x1p-13f;
      }
      if (threadIdx.x == 0) p.exponents[(size_t)run * p.kv_heads + kvh] = (int)((uint32_t)e[0] << 16 | ((uint32_t)e[1] & 0xffffu)) | (apart ? 1 : 0);
      // (no factor is infinite or NaN, whatever the entry: a masked position has one too)
      if (apart && threadIdx.x < 64)
        p.factors[((size_t)run * p.kv_heads + kvh) * 64 + threadIdx.x] =
            make_float2(of[0] < INFINITY ? power_of_two(exponent_just_above(of[0])) : 1.0f, of[1] > 0.0f && of[1] < INFINITY ? (float)exponent_just_above(of[1]) : -200.0f);
    }
    const int g = threadIdx.x & 7;
    for (int j0 = threadIdx.x >> 3; j0 < 64; j0 += 32 * AHEAD) {
      Words<2 * GROUPS> codes[AHEAD][2];
      Words<4 * GROUPS> groups[AHEAD][2];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int pos = tile * 64 + j0 + 32 * i;
        bool here;
        const size_t entry = entry_of(pos, here);
        if (!here && pos >= seen_from && pos < held) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          codes[i][kv] = {};
          groups[i][kv] = {};
          if (here) {
            codes[i][kv] = words_at<2 * GROUPS>((kv ? p.v_pages : p.k_pages) + entry * (HEAD / 2) + 2 * GROUPS * g);
            groups[i][kv] = words_at<4 * GROUPS>((kv ? p.v_groups : p.k_groups) + entry * GROUPS);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const bool no_value = p.starts != nullptr && !(entry_most<GROUPS>(groups[i][1]) < INFINITY);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          [[maybe_unused]] float by = 1.0f;
          if constexpr (HALVES) {
            by = over[kv];
            if (apart) {
              const float m = entry_most<GROUPS>(groups[i][kv]);
              by = m < INFINITY ? power_of_two(-exponent_just_above(m)) : 1.0f;
            }
          }
          T* dst = (kv ? v_dst : k_dst) + (j0 + 32 * i) * HEAD + 4 * g;
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) {
            const Group of = unpacked(groups[i][kv].w[j]);
            const uint32_t unit = codes[i][kv].w[j >> 1] >> (16 * (j & 1));
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              // 2^23 + code, less 2^23 + 8: the code less 8, exactly
              x[k] = fmaf(__uint_as_float(0x4b000000u | ((unit >> (4 * k)) & 15u)) - 8388616.0f, of.step, of.base);
              if constexpr (HALVES) x[k] *= by;
              if (no_value) x[k] = kv ? 0.0f : NAN;
            }
            put_four(dst + GROUP * j, x);
          }
        }
      }
    }
  }
}

// Any head size and page: a warp to a position.
template <typename T>
__global__ void __launch_bounds__(256) read_4bit_simple_kernel(const ReadParams4 p) {
  __shared__ int found[2];
  const int run = blockIdx.x, groups = (p.head_dim + GROUP - 1) / GROUP;
  pdl_wait();
  pdl_trigger();                               // behind the wait: see read_plan_kernel
  find_owner(p, run, found);
  const int seq = found[0], tile = found[1], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int start = seq >= 0 ? p.start_pos[seq] : 0, held = seq >= 0 ? start + p.q_start[seq + 1] - p.q_start[seq] : 0, seen_from = first_seen(p, start);
  for (int kvh = blockIdx.y; kvh < p.kv_heads; kvh += gridDim.y) {
    T* k_dst = static_cast<T*>(p.k_out) + ((size_t)run * p.kv_heads + kvh) * 64 * p.head_dim;
    T* v_dst = static_cast<T*>(p.v_out) + ((size_t)run * p.kv_heads + kvh) * 64 * p.head_dim;
    for (int j = warp; j < 64; j += 8) {
      const int pos = tile * 64 + j, page_index = pos / p.page_size;
      const int page = pos < held && page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
      const bool here = page >= 0 && page < p.num_pages;
      if (!here && pos >= seen_from && pos < held && lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
      const size_t entry = here ? ((size_t)page * p.kv_heads + kvh) * p.page_size + pos % p.page_size : 0;
      bool no_value = false;
      if (here && p.starts != nullptr) no_value = __any_sync(0xffffffffu, lane < groups && !(group_most(p.v_groups[entry * groups + min(lane, groups - 1)]) < INFINITY));
      for (int d = lane; d < p.head_dim; d += 32) {
        const int jj = d / GROUP, unit = (d % GROUP / 4) * groups + jj, up = 4 * (d & 3);
        float x[2] = {0.0f, 0.0f};
        if (here) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv)
            x[kv] = value_of(unpacked((kv ? p.v_groups : p.k_groups)[entry * groups + jj]),
                             (reinterpret_cast<const uint16_t*>(kv ? p.v_pages : p.k_pages)[entry * 8 * groups + unit] >> up) & 15u);
          if (no_value) { x[0] = NAN; x[1] = 0.0f; }
        }
        k_dst[j * p.head_dim + d] = from_float<T>(x[0]);
        v_dst[j * p.head_dim + d] = from_float<T>(x[1]);
      }
    }
  }
}

int cache_shape(const char* what, int num_pages, int page_size, int kv_heads, int head_dim, int max_pages) {
  TGE_REQUIRE(num_pages > 0 && page_size > 0 && kv_heads > 0 && max_pages > 0, "%s: bad page geometry", what);
  TGE_REQUIRE(head_dim > 0 && head_dim <= GROUP * MOST_GROUPS, "%s: head size %d, at most %d", what, head_dim, GROUP * MOST_GROUPS);
  return 0;
}

bool whole_groups(int head_dim) { return head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256; }

}  // namespace

// Without a block table and pages (null): the queries alone, of rows that hold nothing else.
TGE_API int tge_store_4bit(const void* qkv, int is_bf16, long long row_stride, void* q_out, long long q_stride, const float* cos_table,
                           const float* sin_table, int table_rows, int rotary, int pairs, const float* q_norm, const float* k_norm, double eps,
                           const int* positions, const int* seq_of_token, int num_seqs, const int* block_table, int max_pages, void* k_pages,
                           void* v_pages, void* k_groups, void* v_groups, int num_pages, int page_size, int tokens, int heads, int kv_heads, int head_dim,
                           int* status, cudaStream_t stream) {
  const bool alone = k_pages == nullptr && block_table == nullptr;
  TGE_REQUIRE(!alone || (v_pages == nullptr && k_groups == nullptr && v_groups == nullptr), "store_4bit: pages of keys or of values only");
  if (alone) {
    kv_heads = num_pages = max_pages = 0;
    page_size = 1;
  }
  const int rc = alone ? cache_shape("store_4bit", 1, 1, 1, head_dim, 1) : cache_shape("store_4bit", num_pages, page_size, kv_heads, head_dim, max_pages);
  if (rc != 0) return rc;
  TGE_REQUIRE(tokens >= 0 && heads > 0 && num_seqs >= 0, "store_4bit: bad sizes");
  TGE_REQUIRE(rotary >= 0 && rotary <= head_dim && rotary % 2 == 0, "store_4bit: rotary width %d must be even and at most head_dim %d", rotary, head_dim);
  TGE_REQUIRE(row_stride >= (long long)(heads + 2 * kv_heads) * head_dim && q_stride >= (long long)heads * head_dim, "store_4bit: rows too short");
  TGE_REQUIRE(((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_groups | (uintptr_t)v_groups) % 4 == 0, "store_4bit: pages on less than 4 bytes");
  if (tokens == 0) return 0;
  const StoreParams4 p{qkv, q_out, row_stride, q_stride, cos_table, sin_table, q_norm, k_norm, eps, table_rows, positions, seq_of_token, block_table, max_pages,
                       (uint8_t*)k_pages, (uint8_t*)v_pages, (uint32_t*)k_groups, (uint32_t*)v_groups, num_pages, page_size, tokens, num_seqs, heads,
                       kv_heads, head_dim, rotary, pairs, status};
  const int size = is_bf16 ? 2 : 4;
  const uintptr_t all = (uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)k_pages | (uintptr_t)v_pages;
  if (whole_groups(head_dim) && (rotary == 0 || rotary == head_dim) && row_stride * size % 16 == 0 && q_stride * size % 16 == 0 && all % 16 == 0) {
    auto run = [&](auto type, auto normed) {
      using T = decltype(type);
      constexpr bool NORM = decltype(normed)::value;
      const int lanes = (heads + 2 * kv_heads + UNIT_AHEAD - 1) / UNIT_AHEAD * (head_dim / 16);
      const int threads = std::min(UNIT_THREADS, std::max(64, (lanes + 31) / 32 * 32));
      auto launch = [&](void (*kernel)(StoreParams4)) { tge_launch(kernel, dim3(tokens), threads, 0, stream, p); };
      switch (head_dim) {
        case 32: launch(store_4bit_units_kernel<T, 32, NORM>); break;
        case 64: launch(store_4bit_units_kernel<T, 64, NORM>); break;
        case 128: launch(store_4bit_units_kernel<T, 128, NORM>); break;
        default: launch(store_4bit_units_kernel<T, 256, NORM>); break;
      }
    };
    auto typed = [&](auto type) {
      if (q_norm != nullptr || k_norm != nullptr) run(type, std::true_type());
      else run(type, std::false_type());
    };
    if (is_bf16) typed(__nv_bfloat16());
    else typed(float());
    return tge_launched("store_4bit", 1);
  }
  const dim3 grid(tokens, (heads + 2 * kv_heads + WARPS - 1) / WARPS);
  if (is_bf16)
    tge_launch(store_4bit_kernel<__nv_bfloat16>, grid, WARPS * 32, 0, stream, p);
  else
    tge_launch(store_4bit_kernel<float>, grid, WARPS * 32, 0, stream, p);
  return tge_launched("store_4bit", 1);
}

// `type`: 0 float32, 1 bfloat16, 2 float16 over powers of two with `factors` (see attention_tc2.cuh; TGE_UNSUPPORTED for sizes that this is not built for).
TGE_API int tge_read_4bit(const void* k_pages, const void* v_pages, const void* k_groups, const void* v_groups, int num_pages, int page_size,
                          const int* block_table, int max_pages, const int* q_start, const int* start_pos, int first_seq, int num_seqs, int kv_heads,
                          int head_dim, int window, void* k_out, void* v_out, int type, void* factors, int* table, int* starts, int runs, int width,
                          int* status, cudaStream_t stream) {
  const int rc = cache_shape("read_4bit", num_pages, page_size, kv_heads, head_dim, max_pages);
  if (rc != 0) return rc;
  TGE_REQUIRE(first_seq >= 0 && num_seqs >= first_seq && runs >= 0 && width >= 0 && window >= 0 && kv_heads <= 65535, "read_4bit: bad sizes");
  TGE_REQUIRE(((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_groups | (uintptr_t)v_groups) % 4 == 0, "read_4bit: pages on less than 4 bytes");
  if (num_seqs == first_seq) return 0;
  const ReadParams4 p{{block_table, q_start, start_pos, max_pages, num_pages, page_size, first_seq, num_seqs, window, table, starts, runs, width, status},
                      (const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint32_t*)k_groups, (const uint32_t*)v_groups, kv_heads, head_dim, k_out, v_out,
                      static_cast<float2*>(factors), factors == nullptr ? nullptr : static_cast<int*>(factors) + (size_t)runs * kv_heads * 128};
  const bool units = whole_groups(head_dim) && (page_size & (page_size - 1)) == 0 && (long long)num_pages * kv_heads <= 0x7fffffffll &&
                     ((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_groups | (uintptr_t)v_groups | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0;
  if (type == 2 && (!units || factors == nullptr || (uintptr_t)factors % 16 != 0)) return TGE_UNSUPPORTED;
  tge_launch(read_plan_kernel, 1, PLAN_THREADS, 0, stream, p);
  if (runs == 0) return tge_launched("read_4bit", 1);
  // a block takes several heads of its run where there are many runs: finding whose it is costs as much as a head
  const int at_once = 10 * tge_sm_count();
  const dim3 grid(runs, std::max(1, std::min(kv_heads, (at_once + runs) / (runs + 1))));
  auto run = [&](auto out) {
    using T = decltype(out);
    if (!units) {
      if constexpr (!std::is_same<T, __half>::value) tge_launch(read_4bit_simple_kernel<T>, grid, 256, 0, stream, p);
    } else if (head_dim == 32) tge_launch(read_4bit_kernel<T, 1>, grid, 256, 0, stream, p);
    else if (head_dim == 64) tge_launch(read_4bit_kernel<T, 2>, grid, 256, 0, stream, p);
    else if (head_dim == 128) tge_launch(read_4bit_kernel<T, 4>, grid, 256, 0, stream, p);
    else tge_launch(read_4bit_kernel<T, 8>, grid, 256, 0, stream, p);
  };
  if (type == 2) run(__half());
  else if (type == 1) run(__nv_bfloat16());
  else run(float());
  return tge_launched("read_4bit", 2);
}
