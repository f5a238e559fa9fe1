// Paged causal attention over a cache held in 4 bits (see cache_4bit.cu for codes, groups and the order they lie in).
//
// Per query head h at position p, kv head h / group, over the positions i <= p (with a window: i > p - window):
//   s_i = scale sum_j [ step_ij sum_d q_d (c_id - 8) + base_ij sum_d q_d ],   out = sum_i softmax(s)_i [ (c'_i - 8) step'_i + base'_i ]
// j over the groups of 32 numbers, d over a group's.  A sink (float32 [heads]) joins the softmax's denominator once, with no key and no value.
// A row that sees no key (its pages are outside the pool) is zero.
#include "common.cuh"
#include "decode_units.cuh"

namespace {

struct Attn4 {
  const void* q;
  void* out;
  long long q_stride, out_stride;
  const uint8_t *k_pages, *v_pages;
  const uint32_t *k_groups, *v_groups;          // (step, base), a bfloat16 each
  const int *block_table, *positions, *seq_of_token;
  const float* sink;
  int max_pages, num_pages, page_size, num_seqs, heads, kv_heads, group, head_dim, window;
  float scale;
  int* status;
};

__device__ __forceinline__ float step_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float base_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Any head size up to 256, any page size, any mix of portions, both run types: one warp per (token, query head), keys in position
// order, float32 on the CUDA cores, a lane per number of a group.
template <typename T>
__global__ void __launch_bounds__(128) attention_4bit_simple_kernel(const Attn4 p) {
  constexpr int MOST_GROUPS = 8;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= p.heads) return;
  const int kvh = h / p.group, groups = (p.head_dim + 31) / 32;
  const int pos = p.positions[t], seq = p.seq_of_token[t];
  T* out = static_cast<T*>(p.out) + (size_t)t * p.out_stride + (size_t)h * p.head_dim;
  const T* q = static_cast<const T*>(p.q) + (size_t)t * p.q_stride + (size_t)h * p.head_dim;
  float qv[MOST_GROUPS], acc[MOST_GROUPS];
#pragma unroll
  for (int j = 0; j < MOST_GROUPS; ++j) {
    const int d = lane + 32 * j;
    qv[j] = d < p.head_dim ? to_float<T>(q[d]) : 0.0f;
    acc[j] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  if (pos < 0 || seq < 0 || seq >= p.num_seqs) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
  } else {
    const int first = p.window > 0 ? max(pos - p.window + 1, 0) : 0;
    const int* table = p.block_table + (size_t)seq * p.max_pages;
    for (int i = first; i <= pos; ++i) {
      const int page_index = i / p.page_size;
      const int page = page_index < p.max_pages ? table[page_index] : -1;
      if (page < 0 || page >= p.num_pages) {
        if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
        break;
      }
      const size_t entry = ((size_t)page * p.kv_heads + kvh) * p.page_size + i % p.page_size;
      auto value = [&](const uint8_t* pages, const uint32_t* pairs, int j) {
        const uint32_t unit = reinterpret_cast<const uint16_t*>(pages)[entry * 8 * groups + (lane >> 2) * groups + j], w = pairs[entry * groups + j];
        return fmaf((float)((int)((unit >> (4 * (lane & 3))) & 15u) - 8), step_of(w), base_of(w));
      };
      float dot = 0.0f;
#pragma unroll
      for (int j = 0; j < MOST_GROUPS; ++j)
        if (lane + 32 * j < p.head_dim) dot = fmaf(qv[j], value(p.k_pages, p.k_groups, j), dot);
      const float s = warp_sum(dot) * p.scale;
      const float m_new = fmaxf(m, s);
      const float corr = m == m_new ? 1.0f : expf(m - m_new), e = expf(s - m_new);
      l = l * corr + e;
#pragma unroll
      for (int j = 0; j < MOST_GROUPS; ++j)
        if (lane + 32 * j < p.head_dim) acc[j] = fmaf(e, value(p.v_pages, p.v_groups, j), acc[j] * corr);
      m = m_new;
    }
  }
  if (p.sink != nullptr) {                     // minus infinity is none, however large a one leaves zeros
    const float sink = p.sink[h] > 3.4e38f ? 3.4e38f : p.sink[h], m_new = fmaxf(m, sink), corr = m == -INFINITY ? 0.0f : expf(m - m_new);
    l = l * corr + (sink == -INFINITY ? 0.0f : expf(sink - m_new));
#pragma unroll
    for (int j = 0; j < MOST_GROUPS; ++j) acc[j] *= corr;
  }
  const float over = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < MOST_GROUPS; ++j) {
    const int d = lane + 32 * j;
    if (d < p.head_dim) out[d] = from_float<T>(acc[j] * over);
  }
}

// ---------------------------------------------------------------------------
// Single tokens on the tensor cores: head sizes 64, 128 and 256, pages of 16, 32, 64, ... positions.
//
// What bounds it: instructions (some 390 a slice of 16 positions and warp, over everything that a launch does: no counter splits them by part) and waits for
// loads; DRAM would take 39 of the 75 us below.
// A warp takes slices of 16 positions, nothing of them passes through shared memory.
//   scores   S^T [16 positions x 8 heads] = sum_j step_j (C_j [16 x 32] Q_j^T [32 x 8]) (m16n8k16 of float16, two to a group): a lane needs, of positions
//            g and g + 8 (g = lane / 4), its quarter (t = lane % 4) of every group, which is how they lie.  Four bits under a mask are a float16 already,
//            one of its smallest numbers, c 2^-24 or c 2^-20, which the tensor core multiplies exactly.  What they are too large by, and the bases, are one
//            more product (bfloat16, as they are held): [step_j, base_j] [16 x 2 groups] times [-8 sum q, sum q], the sums of a group's queries in three parts of eight bits.
//   values   O_j^T [32 x 8 heads] += (C'_j - 8)^T [32 x 16 positions] (P step_j)^T [16 x 8] in bfloat16, and for the bases one more product,
//            B^T [2 groups x 16 positions] P^T: a lane needs, of positions 2t, 2t + 1, 2t + 8, 2t + 9, four neighbours of every group (g).
//            bfloat16 has float32's range, so that no value's size, however far from the others', has to be held over a power of two; a code becomes one
//            by its bits below the exponent of 128, and 136 is taken off: a sum over a long context must not be the difference of two large ones.
// Queries are over a power of two above their row's largest number, so that a product with the largest step stays finite.  p is at most 2^8 and is
// rounded with its step to bfloat16, as a bfloat16 cache's probabilities are; float32 runs take queries and probabilities in three such parts.
// Probabilities turn from S^T's accumulators into P^T's operand by two 8x8 transposes a group.  The running maximum is raised only when a score
// passes it by 2^8; the sums of probabilities stay in their lanes until the end.
//
// Measured, with the joining: 64 requests of 2,048 to 4,096 positions at 40 heads over 8 (258 MB with their pairs) 75.2 us; four of 32,768 to 65,536 69.4; eight of
// 2,048 at 28 heads over 4 (a cluster each unit) 10.3, one 7.3.  Without raising the scores of rows beyond 2^110, which float32 would have no room for,
// 74.6 and 68.8.  Keys in bfloat16, their codes raised by 128 and the sums lowered after: 76.8, the base of what follows.  Not taken: entries through rings in shared memory, bulk copies asked for by each warp or by each block, 77 and 79 (fewer waits, more instructions); pages
// asked into L2 ahead 90; one slice at a time with four blocks on an SM 79, three 90; values with 136 taken off by a product with a constant 82, queries in shared memory 78.
// Without any conversion or scaling at all that kernel of 76.8 would have taken 56, without products too 50.
//
// Work: see decode_units.cuh; few units over short contexts go to a cluster each (decode_cluster).
// ---------------------------------------------------------------------------
struct Decode4 : DecodeUnits {
  const void* q;
  long long q_stride;
  const uint8_t *k_pages, *v_pages;
  const uint32_t *k_groups, *v_groups;
  int kv_heads, page_size;
  int q_whole;                                  // queries may be read 16 bytes at a time
  float scale;
  int* status;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t two_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Codes n of the units in both halves of x as c - 8 in bfloat16: 128 + c, less 136.
__device__ __forceinline__ uint32_t centred_codes(uint32_t x, int n) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(r) : "r"(x >> (4 * n)));      // (x & mask) | pattern
  asm("add.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(r), "r"(0xc308c308u));
  return r;
}
// Codes n and n + 1 (n even) in float16, as they lie: c 2^-24 and c 2^-20.
__device__ __forceinline__ void tiny_codes(uint32_t x, int n, uint32_t& even, uint32_t& odd) {
  even = (x >> (4 * n)) & 0x000f000fu;
  odd = (x >> (4 * n)) & 0x00f000f0u;
}
// Halves `which` (0: lower) of two words, the first one's below.
__device__ __forceinline__ uint32_t halves_of(uint32_t a, uint32_t b, int which) { return __byte_perm(a, b, which ? 0x7632 : 0x5410); }

// PARTS pairs of bfloat16 that add up to a pair of numbers (three: to all of their 24 bits).
template <int PARTS>
__device__ __forceinline__ void in_parts(float lo, float hi, uint32_t (&to)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    to[i] = two_bf16(lo, hi);
    lo -= step_of(to[i]);
    hi -= base_of(to[i]);
  }
}

template <int WORDS>
__device__ __forceinline__ void load_words(const void* src, uint32_t (&x)[WORDS]) {
  static_assert(WORDS == 1 || WORDS == 2 || WORDS % 4 == 0, "");
  if constexpr (WORDS == 1) asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];\n" : "=r"(x[0]) : "l"(src));
  else if constexpr (WORDS == 2) asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];\n" : "=r"(x[0]), "=r"(x[1]) : "l"(src));
  else
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                   : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]) : "l"(static_cast<const uint4*>(src) + i / 4));
}

// A slice's entries as a lane has them.
template <int HD>
struct Entries {
  static constexpr int G = HD / 32;
  uint32_t k[2][G], v[4][G / 2], k_of[2][G], v_of[2][G];

  __device__ __forceinline__ void load_keys(const Decode4& p, size_t row, int g, int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load_words(p.k_pages + (row + g + 8 * i) * (HD / 2) + 4 * G * t, k[i]);
      load_words(p.k_groups + (row + g + 8 * i) * G, k_of[i]);
    }
  }
  __device__ __forceinline__ void load_values(const Decode4& p, size_t row, int g, int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) load_words(p.v_pages + (row + 2 * t + (i & 1) + 8 * (i >> 1)) * (HD / 2) + 2 * G * g, v[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) load_words(p.v_groups + (row + g + 8 * i) * G, v_of[i]);
  }
};

// Words t and t + 4 of a position's pairs (zero where there are none): an operand's row.
template <int G>
__device__ __forceinline__ uint32_t word_of(const uint32_t (&w)[G], int t, int from) {
  if (from >= G) return 0u;
  if constexpr (G == 2) return t == 0 ? w[0] : t == 1 ? w[1] : 0u;
  else {
    const uint32_t even = t & 2 ? w[from + 2] : w[from], odd = t & 2 ? w[from + 3] : w[from + 1];
    return t & 1 ? odd : even;
  }
}

// A tile's queries as operands: numbers (2b, 4 + 2b) and (2b + 1, 5 + 2b) of the lane's eight of group j (bfloat16 runs: in float16, times 2^15 and 2^11, so
// that their products with codes are all over 2^9; else in PARTS parts), and what multiplies the pairs of groups t and t + 4, in three parts.
template <int HD, int PARTS>
struct Queries {
  static constexpr int G = HD / 32, SUMS = G > 4 ? 2 : 1;
  static constexpr float OVER = PARTS == 1 ? 0x1p-9f : 1.0f;               // what scores come out times
  uint32_t x[G][2][2][PARTS], sums[SUMS][3];

  // `head`: the head's row, of which the lane takes numbers 32 j + 8 t ..; returns the power of two that they are over (NaN if a number is not finite).
  template <typename T>
  __device__ __forceinline__ float take(const T* head, bool valid, bool whole, int t) {
    float v[G][8], most = 0.0f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      const T* src = head + 32 * j + 8 * t;
      if (!valid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
      } else if (whole) {
        uint32_t w[2 * sizeof(T)];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
          const uint4 raw = reinterpret_cast<const uint4*>(src)[i];
          w[4 * i] = raw.x; w[4 * i + 1] = raw.y; w[4 * i + 2] = raw.z; w[4 * i + 3] = raw.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = sizeof(T) == 4 ? __uint_as_float(w[i % (2 * sizeof(T))]) : i & 1 ? base_of(w[i / 2]) : step_of(w[i / 2]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = to_float<T>(src[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        most = fmaxf(most, fabsf(v[j][i]));
        fine &= fabsf(v[j][i]) < INFINITY;
      }
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // most < 2^up; a bfloat16 of 2^127 and more is at most 2 - 2^-7 over 2^127, and that times 2^15 is a float16 still
    const int up = most > 0.0f ? min(max((int)(__float_as_uint(most) >> 23) - 126, -120), PARTS == 1 ? 127 : 120) : 0;
    const float down = up < 127 ? __uint_as_float((uint32_t)(127 - up) << 23) : 0x1p-127f;
    float sum[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      sum[j] = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[j] += v[j][i] *= down;
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float lo = v[j][2 * b + n], hi = v[j][4 + 2 * b + n], by = n ? 0x1p11f : 0x1p15f;
          if constexpr (PARTS == 1) x[j][b][n][0] = two_f16(lo * by, hi * by);
          else in_parts<PARTS>(lo, hi, x[j][b][n]);
        }
    }
#pragma unroll
    for (int half = 0; half < SUMS; ++half) {
      float mine = 0.0f;
#pragma unroll
      for (int j = 4 * half; j < (G < 4 * half + 4 ? G : 4 * half + 4); ++j) mine = t == (j & 3) ? sum[j] : mine;
      mine *= OVER;
      in_parts<3>(PARTS == 1 ? -8.0f * mine : 0.0f, mine, sums[half]);               // (codes of bfloat16 runs are 8 too large)
    }
    const unsigned rest = __ballot_sync(0xffffffffu, !fine) >> (threadIdx.x & 28);
    return (rest & 15u) == 0u ? __uint_as_float((uint32_t)(127 + up) << 23) : __int_as_float(0x7fc00000);
  }
};

// The first of the two numbers of a head that a pair in the accumulators' order is (tile pair / 8, lanes g = pair % 8).
struct Order4 {
  static __device__ __forceinline__ int number_of(int pair) { return 32 * (pair >> 4) + 4 * (pair & 7) + 2 * ((pair >> 3) & 1); }
};

// Slices that a warp has on their way at a time, blocks on an SM.
__host__ __device__ constexpr int decode_ahead(int head_dim, int tiles, int parts) { return parts == 1 && head_dim * tiles <= 128 ? 2 : 1; }
__host__ __device__ constexpr int decode_blocks_per_sm(int head_dim, int tiles, int parts) { return parts == 1 && head_dim * tiles <= 64 ? 4 : parts == 1 && head_dim * tiles <= 128 ? 3 : 2; }

template <typename T, int HD, int NT, bool CLUSTER>
__global__ void __launch_bounds__(DWARPS * 32, decode_blocks_per_sm(HD, NT, sizeof(T) == 2 ? 1 : 3)) decode_4bit_kernel(const Decode4 p) {
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 3, HEADS = 8 * NT, MTILES = HD / 16, G = HD / 32, AHEAD = decode_ahead(HD, NT, PARTS);
  extern __shared__ float merge_o[];                              // see leave_part
  __shared__ Meeting<HD, NT> meet;
  __shared__ int start_of[5];
  __shared__ float2 part_state[CLUSTER ? HEADS : 1];              // what merge_o's first place is over: (maximum, sum)
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = uniform_warp_index();
  const int g = lane >> 2, t = lane & 3;
  if (!CLUSTER && warp == 0) find_run(p, lane, start_of);         // where this block's run begins
  int seq, base = 0, at = 0, end = 1, token, unit = 0, rank = 0, ranks = 1;
  if constexpr (CLUSTER) {
    rank = cluster_rank();
    ranks = cluster_size();
    const int which = blockIdx.x / ranks;
    seq = which / p.units;
    unit = which - seq * p.units;
    token = row_of(p, seq);
  } else {
    __syncthreads();
    seq = start_of[0];
    base = start_of[1];
    at = start_of[2];
    end = start_of[3];
    token = start_of[4];
  }
  bool waited = false;

  while (at < end) {
    const Slices s = slices_of(p, seq);
    int skip, length;
    bool next_seq = false;
    if constexpr (CLUSTER) {
      skip = s.count * rank / ranks;
      length = s.count * (rank + 1) / ranks - skip;                // (none is fine)
      at = end;
    } else {
      unit = (at - base) / (s.count + BEGIN);
      const int begin = base + unit * (s.count + BEGIN);
      const int upto = min(begin + s.count + BEGIN, end);          // where this unit's part of the run ends
      skip = max(at - begin - BEGIN, 0);
      length = upto - begin - BEGIN - skip;
      at = upto;
      next_seq = unit == p.units - 1 && upto == begin + s.count + BEGIN;
      if (length <= 0) continue;                                   // no more than the begin of a unit
    }
    const int kvh = unit / p.head_tiles, tile = unit - kvh * p.head_tiles;
    const int heads_here = min(HEADS, p.group - tile * HEADS), head0 = kvh * p.group + tile * HEADS;
    const int* table = p.block_table + (size_t)seq * p.max_pages;
    // the warps' shares of the run's slices, one behind the other
    const int first = s.first + skip + length * warp / DWARPS, last = s.first + skip + length * (warp + 1) / DWARPS;
    bool bad = false;
    auto page_at = [&](int index) { return index < p.max_pages ? table[index] : -1; };
    // where a page's entries start; one outside the pool reads page 0, unseen
    auto start_at = [&](int page) { return (size_t)((page >= 0 && page < p.num_pages ? page : 0) * p.kv_heads + kvh) << p.page_shift; };
    // the slice to ask for next, its page and the one behind it
    int asked = first, page = page_at((first << 4) >> p.page_shift), page_behind = page_at(((first << 4) >> p.page_shift) + 1);
    size_t row = start_at(page) + ((first << 4) & (p.page_size - 1));
    // the slices asked for last: where they lie, and which of them are this warp's and on a page of the pool
    size_t rows[AHEAD];
    bool there[AHEAD];
    auto ask = [&] {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        rows[i] = row;
        there[i] = asked < last && page >= 0 && page < p.num_pages;
        bad |= asked < last && !there[i];
        ++asked;
        row += 16;
        if (((asked << 4) & (p.page_size - 1)) == 0) {
          page = page_behind;
          page_behind = page_at(((asked << 4) >> p.page_shift) + 1);
          row = start_at(page);
        }
      }
    };
    if (!waited) pdl_wait();                                       // all above is what the step was given
    waited = true;
    Entries<HD> c[AHEAD];
    if (first < last) {
      ask();
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) c[i].load_keys(p, rows[i], g, t);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) c[i].load_values(p, rows[i], g, t);
    }
    Queries<HD, PARTS> q[NT];
    float factor[NT][2];                                          // of the scores of heads 2t, 2t + 1
    float o[NT][MTILES][4], o_base[NT][4], m[NT][2], l[NT][2];
    bool far = false;                                             // a power that has no room for OVER beside it: scores are raised by that first
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool valid = token >= 0 && 8 * nt + g < heads_here;
      const T* src = static_cast<const T*>(p.q) + (size_t)max(token, 0) * p.q_stride + (size_t)(head0 + (valid ? 8 * nt + g : 0)) * HD;
      const float power = q[nt].template take<T>(src, valid, p.q_whole != 0, t);
      far |= PARTS == 1 && power > 0x1p110f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        factor[nt][e] = __shfl_sync(0xffffffffu, power, 4 * (2 * t + e));
        m[nt][e] = NONE;
        l[nt][e] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o_base[nt][e] = 0.0f;
    }
    far = __any_sync(0xffffffffu, far);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) factor[nt][e] *= p.scale * (far ? LOG2E : LOG2E / Queries<HD, PARTS>::OVER);

    for (int slice = first; slice < last; slice += AHEAD) {
      bool here[AHEAD];
      float sc[AHEAD][NT][4];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        here[i] = there[i];
        Entries<HD>& x = c[i];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][nt][e] = 0.0f;
          const uint32_t a0 = word_of<G>(x.k_of[0], t, 0), a1 = word_of<G>(x.k_of[1], t, 0);
          if constexpr (G <= 4) {                                  // the pairs once beside the first part of the sums, once beside the second
            mma_bf16(sc[i][nt], a0, a1, a0, a1, q[nt].sums[0][0], q[nt].sums[0][1]);
            mma_bf16(sc[i][nt], a0, a1, 0u, 0u, q[nt].sums[0][2], 0u);
          } else {
            const uint32_t a2 = word_of<G>(x.k_of[0], t, 4), a3 = word_of<G>(x.k_of[1], t, 4);
#pragma unroll
            for (int part = 0; part < 3; ++part) mma_bf16(sc[i][nt], a0, a1, a2, a3, q[nt].sums[0][part], q[nt].sums[Queries<HD, PARTS>::SUMS - 1][part]);
          }
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const uint32_t x0 = halves_of(x.k[0][j / 2], x.k[0][(G + j) / 2], j & 1), x1 = halves_of(x.k[1][j / 2], x.k[1][(G + j) / 2], j & 1);
          const float step0 = step_of(x.k_of[0][j]), step1 = step_of(x.k_of[1][j]);
          float acc[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][e] = 0.0f;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            uint32_t a0, a1, a2, a3;
            if constexpr (PARTS == 1) {
              tiny_codes(x0, 2 * b, a0, a2);
              tiny_codes(x1, 2 * b, a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt], a0, a1, a2, a3, q[nt].x[j][b][0][0], q[nt].x[j][b][1][0]);
            } else {
              a0 = centred_codes(x0, 2 * b); a1 = centred_codes(x1, 2 * b); a2 = centred_codes(x0, 2 * b + 1); a3 = centred_codes(x1, 2 * b + 1);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int part = 0; part < PARTS; ++part) mma_bf16(acc[nt], a0, a1, a2, a3, q[nt].x[j][b][0][part], q[nt].x[j][b][1][part]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[i][nt][e] = fmaf(acc[nt][e], e < 2 ? step0 : step1, sc[i][nt][e]);
        }
      }
      const bool more = slice + AHEAD < last;
      if (more) {
        ask();
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) c[i].load_keys(p, rows[i], g, t);
      }

      if (far)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sc[i][nt][e] *= 1.0f / Queries<HD, PARTS>::OVER;
              sc[i][nt][e] = fmaf(sc[i][nt][e] * factor[nt][e & 1], 0.0f, sc[i][nt][e]);       // NaN where float32 has no room for the score
            }
      bool raise = false;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][nt][e] *= factor[nt][e & 1];
        const int k0 = (slice + i) * 16;
        if (!here[i] || k0 < s.lo || k0 + 16 > s.hi) {              // some of the slice's positions are not seen
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int k = k0 + g + 8 * half;
            const bool see = here[i] && k >= s.lo && k < s.hi;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) sc[i][nt][2 * half + e] = see ? sc[i][nt][2 * half + e] : -INFINITY;
#pragma unroll
            for (int j = 0; j < G; ++j) c[i].v_of[half][j] = see ? c[i].v_of[half][j] : 0u;      // they may be anything, NaN too
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) raise |= fmaxf(sc[i][nt][e], sc[i][nt][2 + e]) > m[nt][e] + 8.0f;
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float down[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float most = m[nt][e];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) most = fmaxf(most, fmaxf(sc[i][nt][e], sc[i][nt][2 + e]));
#pragma unroll
            for (int offset = 4; offset < 32; offset <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
            down[e] = exp2_fast(m[nt][e] - most);
            m[nt][e] = most;
            l[nt][e] *= down[e];
          }
#pragma unroll
          for (int i = 0; i < MTILES; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][i][e] *= down[e & 1];
#pragma unroll
          for (int e = 0; e < 4; ++e) o_base[nt][e] *= down[e & 1];
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        Entries<HD>& x = c[i];
        const uint32_t b0 = transposed(word_of<G>(x.v_of[0], t, 0)), b2 = transposed(word_of<G>(x.v_of[1], t, 0));
        uint32_t b1 = 0u, b3 = 0u;
        if constexpr (G > 4) {
          b1 = transposed(word_of<G>(x.v_of[0], t, 4));
          b3 = transposed(word_of<G>(x.v_of[1], t, 4));
        }
        float (&e)[NT][4] = sc[i];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int k = 0; k < 4; ++k) e[nt][k] = exp2_fast(e[nt][k] - m[nt][k & 1]);
          l[nt][0] += e[nt][0] + e[nt][2];
          l[nt][1] += e[nt][1] + e[nt][3];
          uint32_t low[PARTS], high[PARTS];
          in_parts<PARTS>(e[nt][0], e[nt][1], low);
          in_parts<PARTS>(e[nt][2], e[nt][3], high);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) mma_bf16(o_base[nt], b0, b1, b2, b3, transposed(low[part]), transposed(high[part]));
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float step0 = step_of(x.v_of[0][j]), step1 = step_of(x.v_of[1][j]);
          uint32_t pr[NT][PARTS][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t low[PARTS], high[PARTS];
            in_parts<PARTS>(e[nt][0] * step0, e[nt][1] * step0, low);
            in_parts<PARTS>(e[nt][2] * step1, e[nt][3] * step1, high);
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              pr[nt][part][0] = transposed(low[part]);
              pr[nt][part][1] = transposed(high[part]);
            }
          }
          const uint32_t x0 = halves_of(x.v[0][j / 2], x.v[1][j / 2], j & 1), x1 = halves_of(x.v[2][j / 2], x.v[3][j / 2], j & 1);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t a0 = centred_codes(x0, 2 * b), a1 = centred_codes(x0, 2 * b + 1), a2 = centred_codes(x1, 2 * b), a3 = centred_codes(x1, 2 * b + 1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) mma_bf16(o[nt][2 * j + b], a0, a1, a2, a3, pr[nt][part][0], pr[nt][part][1]);
          }
        }
      }
      if (more)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) c[i].load_values(p, rows[i], g, t);
    }
    if (token >= 0 && lane == 0 && (bad || s.wrong != 0)) atomicOr(p.status, s.wrong != 0 ? s.wrong : TGE_STATUS_BAD_PAGE);

    // the bases' sums: row 2 j + 1 of their product, lanes g = 2 j + 1 (from the fifth group on the rows behind)
    float worth[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < G; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float sum = __shfl_sync(0xffffffffu, o_base[nt][(j < 4 ? 0 : 2) + e], 4 * (2 * (j & 3) + 1) + t);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            o[nt][2 * j + b][e] += sum;
            o[nt][2 * j + b][2 + e] += sum;
          }
        }
      worth[nt][0] = worth[nt][1] = 1.0f;
    }
    leave_part<T, HD, NT, CLUSTER, Order4>(p, meet, merge_o, part_state, o, m, l, worth, warp, lane, s.count, skip, length, token, head0, heads_here, rank, ranks);
    if (next_seq && at < end) {
      base = at;
      ++seq;
      token = row_of(p, seq);
    }
  }
  if (!waited) pdl_wait();
}

template <typename T, int HD, int NT>
int launch_decode(Decode4 p, int blocks, int cluster, cudaStream_t stream) {
  constexpr int smem = DWARPS * 8 * NT * (HD + 4) * 4;
  static bool ready[64] = {};                                     // shared memory beyond 48 KB, clusters of 16: asked for once per device
  int device = 0;
  cudaGetDevice(&device);
  if (device >= 64 || !ready[device]) {
    cudaError_t rc = cudaFuncSetAttribute(decode_4bit_kernel<T, HD, NT, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (rc == cudaSuccess && smem > 48 * 1024) rc = cudaFuncSetAttribute(decode_4bit_kernel<T, HD, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc == cudaSuccess && smem > 48 * 1024) rc = cudaFuncSetAttribute(decode_4bit_kernel<T, HD, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    TGE_REQUIRE(rc == cudaSuccess, "attention_4bit: %d bytes of shared memory, clusters of 16: %s", smem, cudaGetErrorString(rc));
    if (device < 64) ready[device] = true;
  }
  if (cluster > 0) {
    tge_launch_clusters(decode_4bit_kernel<T, HD, NT, true>, dim3(p.num_seqs * p.units * cluster), DWARPS * 32, smem, cluster, stream, p);
    return tge_launched("attention_4bit", 1);
  }
  p.states = p.parts + (size_t)2 * blocks * 8 * NT * HD;
  tge_launch(decode_4bit_kernel<T, HD, NT, false>, blocks, DWARPS * 32, smem, stream, p);
  tge_launch(decode_join_kernel<T, HD, NT, Order4>, dim3(p.num_seqs, p.units), JOIN_WARPS * 32, 0, stream, p, blocks);
  return tge_launched("attention_4bit", 2);
}

// Blocks of a launch: all that are on the device at a time, so that all runs advance together.
int decode_blocks(int head_dim, int tile_heads, int is_bf16) { return tge_sm_count() * decode_blocks_per_sm(head_dim, tile_heads / 8, is_bf16 ? 1 : 3); }

}  // namespace

// Heads of a tile: a group of up to 8 heads makes one tile of 8, more go by 16 (one pass over the codes for twice the accumulators, which
// heads of 256 numbers have no registers for).
static int decode_tile(int group, int head_dim) { return group <= 8 || head_dim > 128 ? 8 : 16; }

// Blocks of a cluster per unit, which joins its parts itself; 0: runs of slices and a second kernel.  A rule on what the host knows, the units and the
// bound of their lengths (the block table's, also under a window), while all clusters are on the device at a time.  Measured with bfloat16 and heads of 128
// alone; it decides for the other sizes and for float32 too.  us at 28 heads over 4 (four units a request) with 4 / 8 / 16 / none: 1 request of 512
// 5.9 / 6.3 / 6.9 / 6.8, 16 of them 7.9 / 14.3 / 27.6 / 9.5; 1 of 2,048 10.0 / 7.8 / 7.2 / 7.7, 8 of them 13.0 / 10.3 / 16.6 / 11.0; 4 of 4,096 17.1 /
// 12.2 / 11.0 / 11.2, 8 of them 21.0 / 14.9 / 21.3 / 13.9; 1 of 8,192 26 / 16 / 11.5 / 12.0, of 16,384 53 / 30 / 18.6 / 15.8.
static int decode_cluster(long long units, int head_dim, int tile, int is_bf16, long long positions) {
  const int blocks = decode_blocks(head_dim, tile, is_bf16);
  if (positions <= 512 && 4 * units <= blocks) return 4;
  if (positions > 1024 && positions <= 8192 && units <= 16) return 16;
  return positions <= 2048 && 8 * units <= blocks ? 8 : 0;
}

// float32 scratch numbers of tge_attention_4bit_decode; -1: sizes that it does not take.
TGE_API long long tge_attention_4bit_decode_floats(int is_bf16, int num_seqs, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_size < 16 || (page_size & (page_size - 1)) != 0 || kv_heads <= 0 || heads % kv_heads != 0) return -1;
  const int tile = decode_tile(heads / kv_heads, head_dim);
  const long long units = (long long)kv_heads * ((heads / kv_heads + tile - 1) / tile);
  // places in the row of all slices are counted in 32 bits, units along a grid's second axis
  if (units > 65535 || (long long)max_pages * page_size > (1ll << 30) ||
      units * num_seqs * ((long long)max_pages * page_size / 16 + 1 + BEGIN) > (1ll << 30)) return -1;
  if (decode_cluster(units * num_seqs, head_dim, tile, is_bf16, (long long)max_pages * page_size) > 0) return 0;
  return 2ll * decode_blocks(head_dim, tile, is_bf16) * tile * (head_dim + 2);
}

TGE_API int tge_attention_4bit_decode(const void* q, int is_bf16, long long q_stride, const void* k_pages, const void* v_pages, const void* k_groups,
                                      const void* v_groups, int num_pages, int page_size, const int* block_table, int max_pages, const int* q_start,
                                      const int* start_pos, int num_seqs, void* out, long long out_stride, int heads, int kv_heads, int head_dim,
                                      float scale, int window, const float* sink, float* parts, long long part_floats, int* status, cudaStream_t stream) {
  const long long need = tge_attention_4bit_decode_floats(is_bf16, num_seqs, heads, kv_heads, head_dim, page_size, max_pages);
  if (need < 0 || ((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_groups | (uintptr_t)v_groups) % 16 != 0) return TGE_UNSUPPORTED;
  TGE_REQUIRE(part_floats >= need, "attention_4bit: %lld floats of scratch memory, %lld wanted", part_floats, need);
  TGE_REQUIRE(num_pages > 0 && max_pages > 0 && window >= 0, "attention_4bit: bad page geometry");
  if ((long long)num_pages * kv_heads > 0x7fffffffll) return TGE_UNSUPPORTED;
  if (num_seqs == 0) return 0;
  const int group = heads / kv_heads, tile = decode_tile(group, head_dim);
  Decode4 p;
  p.out = out;
  p.out_stride = out_stride;
  p.sink = sink;
  p.block_table = block_table;
  p.q_start = q_start;
  p.start_pos = start_pos;
  p.max_pages = max_pages;
  p.num_pages = num_pages;
  p.num_seqs = num_seqs;
  p.group = group;
  p.window = window;
  p.head_tiles = (group + tile - 1) / tile;
  p.units = kv_heads * p.head_tiles;
  p.least = 2 * DWARPS;
  p.page_shift = __builtin_ctz(page_size);
  p.parts = parts;
  p.states = nullptr;
  p.q = q;
  p.q_stride = q_stride;
  p.k_pages = (const uint8_t*)k_pages;
  p.v_pages = (const uint8_t*)v_pages;
  p.k_groups = (const uint32_t*)k_groups;
  p.v_groups = (const uint32_t*)v_groups;
  p.kv_heads = kv_heads;
  p.page_size = page_size;
  p.q_whole = (uintptr_t)q % 16 == 0 && q_stride * (is_bf16 ? 2 : 4) % 16 == 0;
  p.scale = scale;
  p.status = status;
  const int blocks = decode_blocks(head_dim, tile, is_bf16);
  const int cluster = decode_cluster((long long)p.units * num_seqs, head_dim, tile, is_bf16, (long long)max_pages * page_size);
  auto run = [&](auto type) {
    using T = decltype(type);
    if (head_dim == 256) return launch_decode<T, 256, 1>(p, blocks, cluster, stream);
    if (head_dim == 128) return tile == 8 ? launch_decode<T, 128, 1>(p, blocks, cluster, stream) : launch_decode<T, 128, 2>(p, blocks, cluster, stream);
    return tile == 8 ? launch_decode<T, 64, 1>(p, blocks, cluster, stream) : launch_decode<T, 64, 2>(p, blocks, cluster, stream);
  };
  return is_bf16 ? run(__nv_bfloat16()) : run(float());
}

TGE_API int tge_attention_4bit_simple(const void* q, int is_bf16, long long q_stride, const void* k_pages, const void* v_pages, const void* k_groups,
                                      const void* v_groups, int num_pages, int page_size, const int* block_table, int max_pages,
                                      const int* positions, const int* seq_of_token, int num_seqs, int tokens, void* out, long long out_stride,
                                      int heads, int kv_heads, int head_dim, float scale, int window, const float* sink, int* status, cudaStream_t stream) {
  TGE_REQUIRE(tokens >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && head_dim > 0 && head_dim <= 256 && window >= 0,
              "attention_4bit: bad sizes heads=%d kv_heads=%d head_dim=%d", heads, kv_heads, head_dim);
  TGE_REQUIRE(num_pages > 0 && page_size > 0 && max_pages > 0, "attention_4bit: bad page geometry");
  TGE_REQUIRE(((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_groups | (uintptr_t)v_groups) % 4 == 0, "attention_4bit: pages on less than 4 bytes");
  if (tokens == 0) return 0;
  const Attn4 p{q, out, q_stride, out_stride, (const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint32_t*)k_groups, (const uint32_t*)v_groups, block_table,
                positions, seq_of_token, sink, max_pages, num_pages, page_size, num_seqs, heads, kv_heads, heads / kv_heads, head_dim, window, scale, status};
  const dim3 grid(tokens, (heads + 3) / 4);
  if (is_bf16)
    tge_launch(attention_4bit_simple_kernel<__nv_bfloat16>, grid, 128, 0, stream, p);
  else
    tge_launch(attention_4bit_simple_kernel<float>, grid, 128, 0, stream, p);
  return tge_launched("attention_4bit", 1);
}
