// A paged key/value cache held in 8 bits: rotation, quantisation and store of a step's keys and values; reading entries back.
//
// A block is `block` consecutive positions of one request and kv head (a power of two that divides the page; keys and values have
// blocks of their own).  Its scale s is the largest magnitude in it, a code c = rint(127 x / s), ties to even, and c stands for
// c s / 127.  Pages: codes int8 [pages, kv_heads, page, head_dim], scales float32 [pages, kv_heads, page / block].  Appending to a
// block that is partly filled makes its scale the larger of its own and the new rows' one; codes of a scale s that grows to s'
// become rint(c s / s').  A block that begins in this step forgets what the page held.  A value that is not finite makes its block's
// scale NaN: the block reads as NaN until it is begun anew.  With blocks of one position an entry is a function of its own row alone,
// whatever step brought it; larger blocks cost less memory (4 / block bytes beside head_dim) and depend on what shares the block.
//
// Rotation (rotate-half over the first `rotary` numbers of a head, float32), as in elementwise.cu:
//   lo' = lo cos - hi sin ; hi' = lo sin + hi cos
// keys are quantised from these float32 numbers, with no rounding to the run's type in between.  127 x is exact for a bfloat16 x and
// the division is rounded once, so x = s (k + 1/2) / 127 meets its tie exactly and goes to even wherever it is computed.
#include <algorithm>
#include <type_traits>

#include "cache_runs.cuh"

namespace {

constexpr int WARPS = 8;
constexpr int MAX_PER_LANE = 8;                // head_dim <= 256

// Codes of a block of scale s: rint(127 x / s).  Scales beyond 1e30 (where 127 x may pass float32's largest number) are divided
// out in two steps that are exact powers of two apart.
struct Coder {
  float over, shrink;
  bool any;
  __device__ __forceinline__ explicit Coder(float scale) {
    shrink = scale > 1e30f ? 9.5367431640625e-7f : 1.0f;
    over = scale * shrink;
    any = scale > 0.0f;                        // false for a block of zeros and for NaN
  }
  __device__ __forceinline__ int code(float x) const {
    return any ? min(max(__float2int_rn(__fdiv_rn(127.0f * (x * shrink), over)), -127), 127) : 0;
  }
};

__device__ __forceinline__ float warp_larger(float v) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, offset));
  return v;
}

struct StoreParams {
  const void* qkv;
  void* q_out;
  long long row_stride, q_stride;
  const float *cos_table, *sin_table;
  int table_rows;
  const int *positions, *seq_of_token, *q_start, *block_table;
  int max_pages;
  int8_t *k_pages, *v_pages;
  float *k_scale, *v_scale;
  int num_pages, page_size, block, tokens, num_seqs, heads, kv_heads, head_dim, rotary;
  int* status;
};

// One product rounded, the other inside the sum: spelled out, so that every kernel here rounds alike.
__device__ __forceinline__ float turned_lo(float lo, float hi, float c, float s) { return __fmaf_rn(lo, c, -__fmul_rn(hi, s)); }
__device__ __forceinline__ float turned_hi(float lo, float hi, float c, float s) { return __fmaf_rn(lo, s, __fmul_rn(hi, c)); }

// Number d of a head's row at `src`, rotated for position `pos`.
template <typename T>
__device__ __forceinline__ float rotated(const StoreParams& p, const T* src, int d, int pos, bool rotate) {
  const float own = to_float<T>(src[d]);
  if (!rotate || d >= p.rotary) return own;
  const int half = p.rotary >> 1, j = d < half ? d : d - half;
  const float other = to_float<T>(src[d < half ? d + half : d - half]);
  const float c = p.cos_table[(size_t)pos * half + j], s = p.sin_table[(size_t)pos * half + j];
  return d < half ? turned_lo(own, other, c, s) : turned_hi(other, own, c, s);
}

// One warp per (token, head): a query head is rotated into q_out; a key or value head is quantised by the warp of the block's first
// token in this step, which walks the tokens of its block.
template <typename T>
__global__ void __launch_bounds__(WARPS * 32) store_8bit_kernel(const StoreParams p) {
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  const int h = blockIdx.y * WARPS + (threadIdx.x >> 5);
  const int pos = p.positions[t], seq = p.seq_of_token[t];
  pdl_wait();
  if (h >= p.heads + 2 * p.kv_heads) return;
  const bool rotate = p.rotary > 0;
  if (pos < 0 || (rotate && pos >= p.table_rows) || seq < 0 || seq >= p.num_seqs) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
    return;
  }
  const T* rows = static_cast<const T*>(p.qkv) + (size_t)h * p.head_dim;
  if (h < p.heads) {
    const T* src = rows + (size_t)t * p.row_stride;
    T* dst = static_cast<T*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * p.head_dim;
    for (int d = lane; d < p.head_dim; d += 32) dst[d] = from_float<T>(rotated<T>(p, src, d, pos, rotate));
    return;
  }
  const bool is_key = h < p.heads + p.kv_heads;
  const int kvh = h - p.heads - (is_key ? 0 : p.kv_heads);
  const int first = p.q_start[seq], last = p.q_start[seq + 1];
  const int inside = pos & (p.block - 1);
  if (t != first && inside != 0) return;                         // an earlier token of the step leads this block
  const int count = min(p.block - inside, last - t);
  const int page_index = pos / p.page_size;
  const int page = page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
  if (page < 0 || page >= p.num_pages || count <= 0 || t + count > p.tokens) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
    return;
  }
  if (rotate && is_key && pos + count > p.table_rows) {
    if (lane == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
    return;
  }
  const int slot = pos % p.page_size;
  const size_t entry = ((size_t)page * p.kv_heads + kvh) * p.page_size;
  int8_t* codes = (is_key ? p.k_pages : p.v_pages) + (entry + slot) * p.head_dim;
  float* scale_at = (is_key ? p.k_scale : p.v_scale) + (entry + slot) / p.block;
  const bool turn = rotate && is_key;

  float most = 0.0f;
  for (int j = 0; j < count; ++j) {
    const T* src = rows + (size_t)(t + j) * p.row_stride;
    for (int d = lane; d < p.head_dim; d += 32) most = larger(most, magnitude(rotated<T>(p, src, d, pos + j, turn)));
  }
  most = warp_larger(most);
  const float before = inside != 0 ? *scale_at : 0.0f;
  const float scale = larger(before, most);
  if (inside != 0 && !(before >= scale)) {                       // the scale grew: what the block held is rounded again
    const Coder again(scale);
    int8_t* old = codes - (size_t)inside * p.head_dim;
    for (int i = lane; i < inside * p.head_dim; i += 32) {
      const float stands = (float)old[i] * (before * again.shrink);
      old[i] = (int8_t)(again.any ? __float2int_rn(__fdiv_rn(stands, again.over)) : 0);
    }
  }
  const Coder coder(scale);
  for (int j = 0; j < count; ++j) {
    const T* src = rows + (size_t)(t + j) * p.row_stride;
    for (int d = lane; d < p.head_dim; d += 32) codes[(size_t)j * p.head_dim + d] = (int8_t)coder.code(rotated<T>(p, src, d, pos + j, turn));
  }
  __syncwarp();
  if (lane == 0) *scale_at = scale;
}

// ---------------------------------------------------------------------------
// The same by units of eight numbers, for head sizes 16, 32, ..., 256 that are rotated whole or not at all and rows on 16 bytes.  Bound by
// the rows' bytes.  HEAD / 16 lanes (a group) have a head's row, eight numbers of its first half and the eight that they are rotated
// with.  The first blocks have a token each: its groups take its query heads (and, with blocks of one position, its key and value heads) in
// turn, three rows on their way at a time, the angles loaded once.  With larger blocks the others have a (block of positions, key or value
// head) each: its groups take the block's rows in turn, once for the scale and, from cache, once for the codes.
// With the read-back below: one token 7.2 us; a prompt of 2,048 tokens at 28 heads over 4 13.5 us (43 MB; 6.6 at a copy's rate); 64 tokens
// of requests that hold up to 512 (25,109 together) at 40 heads over 8, blocks of 16, 46 us (165 MB, 25 at that rate).  With a warp to a head, as above: 25, 57 and 92 us.
// ---------------------------------------------------------------------------
constexpr int UNIT_THREADS = 256, UNIT_AHEAD = 3;         // at most; as many as it takes for a token's heads in UNIT_AHEAD turns

__device__ __forceinline__ void turn(Eight& lo, Eight& hi, const Eight& c, const Eight& s) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float l = lo.x[i], h = hi.x[i];
    lo.x[i] = turned_lo(l, h, c.x[i], s.x[i]);
    hi.x[i] = turned_hi(l, h, c.x[i], s.x[i]);
  }
}
__device__ __forceinline__ float largest_of(const Eight& lo, const Eight& hi) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = larger(larger(most, magnitude(lo.x[i])), magnitude(hi.x[i]));
  return most;
}
__device__ __forceinline__ void put_codes(int8_t* dst, const Coder& coder, const Eight& e) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(coder.code(e.x[4 * i]), coder.code(e.x[4 * i + 1]), 0x0040),
                       __byte_perm(coder.code(e.x[4 * i + 2]), coder.code(e.x[4 * i + 3]), 0x0040), 0x5410);
  *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
}

template <typename T, int HEAD>
__global__ void __launch_bounds__(UNIT_THREADS, sizeof(T) == 2 ? 3 : 2) store_8bit_units_kernel(const StoreParams p) {
  constexpr int LANES = HEAD / 16, HALF = HEAD / 2;
  const int GROUPS = blockDim.x / LANES;
  __shared__ float scales[UNIT_THREADS / LANES];
  __shared__ int found[2];
  pdl_trigger();
  const int group = threadIdx.x / LANES, j = threadIdx.x % LANES;
  const bool rotate = p.rotary > 0;
  const T* rows = static_cast<const T*>(p.qkv) + 8 * j;
  auto angles = [&](int pos, Eight& c, Eight& s) {
    if (rotate) {
      c = eight(p.cos_table + (size_t)pos * HALF + 8 * j);
      s = eight(p.sin_table + (size_t)pos * HALF + 8 * j);
    }
  };
  auto all_lanes = [&](float most) {                              // over the lanes of a head
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, offset));
    return most;
  };
  if ((int)blockIdx.x < p.tokens) {
    const int t = blockIdx.x, pos = p.positions[t], seq = p.seq_of_token[t];
    pdl_wait();
    // the first rows are on their way before anything has to be looked up
    const T* row = rows + (size_t)t * p.row_stride;
    const int heads = p.heads + (p.block == 1 ? 2 * p.kv_heads : 0);
    Raw<T> lo_raw[UNIT_AHEAD], hi_raw[UNIT_AHEAD];
    auto load = [&](int h0) {
#pragma unroll
      for (int i = 0; i < UNIT_AHEAD; ++i) {
        const int h = min(h0 + i * GROUPS, heads - 1);
        lo_raw[i] = raw_eight(row + (size_t)h * HEAD);
        hi_raw[i] = raw_eight(row + (size_t)h * HEAD + HALF);
      }
    };
    load(group);
    if (pos < 0 || (rotate && pos >= p.table_rows) || seq < 0 || seq >= p.num_seqs) {
      if (threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
      return;
    }
    Eight c, s;
    angles(pos, c, s);
    const int page_index = pos / p.page_size, slot = pos - page_index * p.page_size;
    const int page = page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
    const bool here = page >= 0 && page < p.num_pages;
    if (!here && p.block == 1 && threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
    for (int h0 = group; h0 < heads + group; h0 += UNIT_AHEAD * GROUPS) {       // the same number of rounds for every lane of a warp
      if (h0 != group) load(h0);
#pragma unroll
      for (int i = 0; i < UNIT_AHEAD; ++i) {
        const int h = h0 + i * GROUPS;
        Eight lo = eight(lo_raw[i]), hi = eight(hi_raw[i]);
        const bool valid = h < heads, to_cache = h >= p.heads;
        if (rotate && h < p.heads + p.kv_heads) turn(lo, hi, c, s);
        if (valid && !to_cache) {
          T* dst = static_cast<T*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * HEAD + 8 * j;
          put_eight(dst, lo);
          put_eight(dst + HALF, hi);
        }
        if (__any_sync(0xffffffffu, valid && to_cache)) {
          const float scale = all_lanes(largest_of(lo, hi));
          if (valid && to_cache && here) {
            const bool is_key = h < p.heads + p.kv_heads;
            const size_t entry = ((size_t)page * p.kv_heads + (h - p.heads - (is_key ? 0 : p.kv_heads))) * p.page_size + slot;
            const Coder coder(scale);
            int8_t* codes = (is_key ? p.k_pages : p.v_pages) + entry * HEAD + 8 * j;
            put_codes(codes, coder, lo);
            put_codes(codes + HALF, coder, hi);
            if (j == 0) (is_key ? p.k_scale : p.v_scale)[entry] = scale;
          }
        }
      }
    }
    return;
  }
  // a block of positions of one request: the requests' blocks one after the other
  const int shift = __ffs(p.block) - 1, number = blockIdx.x - p.tokens;
  const int item = number / (2 * p.kv_heads), head = number - item * 2 * p.kv_heads;
  if (threadIdx.x < 32) {
    int before = 0, seq_found = -1, index = 0;
    for (int base = 0; base < p.num_seqs && seq_found < 0; base += 32) {
      const int seq = base + threadIdx.x;
      int n = 0, first = 0;
      if (seq < p.num_seqs) {
        const int start = p.q_start[seq], count = p.q_start[seq + 1] - start;
        if (count > 0 && start >= 0 && start < p.tokens) {
          const int pos = p.positions[start];
          first = pos >> shift;
          n = pos >= 0 ? ((pos + count - 1) >> shift) - first + 1 : 0;
        }
      }
      int upto = n;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, offset);
        if ((int)threadIdx.x >= offset) upto += v;
      }
      const unsigned mine = __ballot_sync(0xffffffffu, item < before + upto);
      if (mine != 0) {
        const int who = __ffs(mine) - 1;
        seq_found = base + who;
        index = item - before - (__shfl_sync(0xffffffffu, upto, who) - __shfl_sync(0xffffffffu, n, who)) + __shfl_sync(0xffffffffu, first, who);
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (threadIdx.x == 0) { found[0] = seq_found; found[1] = index; }
  }
  __syncthreads();
  const int seq = found[0];
  pdl_wait();
  if (seq < 0) return;
  const int start = p.q_start[seq], count = p.q_start[seq + 1] - start, first_pos = p.positions[start];
  const int lo_pos = found[1] << shift, from = max(lo_pos, first_pos), to = min(lo_pos + p.block, first_pos + count);
  const bool is_key = head < p.kv_heads, rotated_here = rotate && is_key;
  const int page_index = lo_pos / p.page_size;
  const int page = page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
  if (page < 0 || page >= p.num_pages || start + (to - first_pos) > p.tokens) {
    if (threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
    return;
  }
  if (rotated_here && to > p.table_rows) {
    if (threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_ROW);
    return;
  }
  const size_t entry = ((size_t)page * p.kv_heads + (is_key ? head : head - p.kv_heads)) * p.page_size + (lo_pos - page_index * p.page_size);
  int8_t* codes = (is_key ? p.k_pages : p.v_pages) + entry * HEAD + 8 * j;     // of the block's first position
  float* scale_at = (is_key ? p.k_scale : p.v_scale) + (entry >> shift);
  const float before = from > lo_pos ? *scale_at : 0.0f;
  const T* row0 = rows + (size_t)(p.heads + head) * HEAD + (size_t)(start - first_pos) * p.row_stride;    // position pos at pos rows from here
  auto row_of = [&](int pos, Eight& lo, Eight& hi) {
    const T* row = row0 + (long long)pos * p.row_stride;
    lo = eight(row);
    hi = eight(row + HALF);
    if (rotated_here) {
      Eight c, s;
      angles(pos, c, s);
      turn(lo, hi, c, s);
    }
  };
  float most = 0.0f;
  for (int pos = from + group; pos < to; pos += GROUPS) {
    Eight lo, hi;
    row_of(pos, lo, hi);
    most = larger(most, largest_of(lo, hi));
  }
  most = all_lanes(most);
  if (j == 0) scales[group] = most;
  __syncthreads();
  most = before;
  for (int i = 0; i < GROUPS; ++i) most = larger(most, scales[i]);
  const Coder coder(most);
  if (from > lo_pos && !(before >= most))                          // the scale grew: what the block held is rounded again
    for (int i = group; i < from - lo_pos; i += GROUPS)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        int8_t* at = codes + (size_t)i * HEAD + half * HALF;
        const uint2 raw = *reinterpret_cast<const uint2*>(at);
        uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          int again[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float stands = (float)(int8_t)(w[k] >> (8 * b)) * (before * coder.shrink);
            again[b] = coder.any ? __float2int_rn(__fdiv_rn(stands, coder.over)) : 0;
          }
          w[k] = __byte_perm(__byte_perm(again[0], again[1], 0x0040), __byte_perm(again[2], again[3], 0x0040), 0x5410);
        }
        *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
      }
  for (int pos = from + group; pos < to; pos += GROUPS) {
    Eight lo, hi;
    row_of(pos, lo, hi);
    put_codes(codes + (size_t)(pos - lo_pos) * HEAD, coder, lo);
    put_codes(codes + (size_t)(pos - lo_pos) * HEAD + HALF, coder, hi);
  }
  __syncthreads();                                                 // every thread has read the scale
  if (threadIdx.x == 0) *scale_at = most;
}

// ---------------------------------------------------------------------------
// Entries read back: the positions that a step's queries may see, request after request, in runs of 64 positions
// [runs, kv_heads, 64, head_dim] (zeros behind a request's last), a block table over those runs and (starts, if wanted) the requests'
// first tokens counted from the first one's.  In float16 with a power of two for each run and head, for the attention kernel that takes these.
// For attention (starts are wanted): it multiplies every value of a tile with a probability, unseen ones with zero, so values are finite there:
// a position whose values' scale is not gets a key that is not, which whoever sees it turns into the same and nobody else looks at.
// Bound by the bytes written, two (four) to a code read: 8,128 positions of 8 heads in float16 50 MB, 12.7 us with the plan.
// ---------------------------------------------------------------------------
struct ReadParams : RunPlan {
  const int8_t *k_pages, *v_pages;
  const float *k_scale, *v_scale;
  int block, kv_heads, head_dim;
  void *k_out, *v_out;
  float2* factors;                             // [runs, kv_heads, 64], for float16 output: of runs whose scales lie far apart, see below
  int* exponents;                              // [runs, kv_heads], for float16 output: f below, e above; 1: the run has factors
};

// float16 pages: keys and values over powers of two of their run and head, so that all of them are at most 1.  Multiples of 8: few runs differ.
// float16's numbers are 2^-24 apart below 2^-14, so a position whose scale is at least 2^-13 of the power keeps 2^-12 of its own largest
// number, which is what float16 keeps of any.  A run with a smaller scale (its largest one is above 2^-8 of the power: they lie 2^5 apart at
// least) holds whole codes over 128, which float16 has exactly, and the scales go to the attention as factors: what multiplies a key's scores,
// and the logarithm to the base 2 of what multiplies a value's probability.  So does a run with values of zero beside others: a row that sees those
// alone adds nothing, whatever the others' power says.
template <typename T, bool UNITS>
__global__ void __launch_bounds__(256) read_8bit_kernel(const ReadParams p) {
  constexpr bool HALVES = std::is_same<T, __half>::value;
  __shared__ int found[2];
  __shared__ float most[2][2], least[2][2];    // float16: the largest and smallest scales of the run's first and second 32 positions, keys' and values'
  const int run = blockIdx.x;
  pdl_wait();
  pdl_trigger();                               // behind the wait: see read_plan_kernel
  find_owner(p, run, found);
  const int seq = found[0], tile = found[1];
  for (int kvh = blockIdx.y; kvh < p.kv_heads; kvh += gridDim.y) {
  T* k_dst = static_cast<T*>(p.k_out) + ((size_t)run * p.kv_heads + kvh) * 64 * p.head_dim;
  T* v_dst = static_cast<T*>(p.v_out) + ((size_t)run * p.kv_heads + kvh) * 64 * p.head_dim;
  if (seq < 0) {                               // the caller counted more runs than there are
    for (int i = threadIdx.x; i < 64 * p.head_dim; i += blockDim.x) k_dst[i] = v_dst[i] = from_float<T>(0.0f);
    if (HALVES && threadIdx.x == 0) p.exponents[(size_t)run * p.kv_heads + kvh] = 0;
    continue;
  }
  const int start = p.start_pos[seq], held = start + p.q_start[seq + 1] - p.q_start[seq], seen_from = first_seen(p, start);
  if constexpr (UNITS) {
    // 16 bytes of the output to a thread and turn, side by side across a warp, four turns' codes of keys and values on their way together
    // (head sizes and pages are powers of two here: a division per eight numbers would cost more than they do)
    constexpr int EACH = 16 / sizeof(T), AHEAD = 4;
    const int unit_shift = __ffs(p.head_dim / EACH) - 1, page_shift = __ffs(p.page_size) - 1, shift = __ffs(p.block) - 1;
    [[maybe_unused]] float k_over = 1.0f, v_over = 1.0f;
    [[maybe_unused]] bool whole_codes = false;
    if constexpr (HALVES) {
      __syncthreads();                         // whoever still reads those of the head before
      float ks = 0.0f, vs = 0.0f;
      if (threadIdx.x < 64) {
        const int pos = tile * 64 + threadIdx.x, page_index = pos >> page_shift;
        const int page = pos < held && page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
        const bool here = page >= 0 && page < p.num_pages;
        const size_t block = ((((size_t)(page * p.kv_heads + kvh) << page_shift) + (pos & (p.page_size - 1))) >> shift);
        ks = here ? fabsf(p.k_scale[block]) : 0.0f;
        vs = here ? fabsf(p.v_scale[block]) : 0.0f;
        const float k = warp_max(ks < INFINITY ? ks : 0.0f), v = warp_max(vs < INFINITY ? vs : 0.0f);
        const float k_least = -warp_max(ks > 0.0f ? -ks : -INFINITY), v_least = -warp_max(here && vs >= 0.0f ? -vs : -INFINITY);
        if ((threadIdx.x & 31) == 0) {
          most[threadIdx.x >> 5][0] = k;
          most[threadIdx.x >> 5][1] = v;
          least[threadIdx.x >> 5][0] = k_least;
          least[threadIdx.x >> 5][1] = v_least;
        }
      }
      __syncthreads();
      const float k = fmaxf(most[0][0], most[1][0]), v = fmaxf(most[0][1], most[1][1]);
      const int e = k > 0.0f ? exponent_above(k) : 0, f = v > 0.0f ? exponent_above(v) : 0;
      k_over = power_of_two(-e);
      v_over = power_of_two(-f);
      whole_codes = fminf(least[0][0], least[1][0]) < power_of_two(e) * 0x1p-13f || (v > 0.0f && fminf(least[0][1], least[1][1]) < power_of_two(f) * 0x1p-13f);
      if (threadIdx.x == 0) p.exponents[(size_t)run * p.kv_heads + kvh] = (int)((uint32_t)e << 16 | ((uint32_t)f & 0xffffu)) | (whole_codes ? 1 : 0);
      // (no factor is infinite or NaN, whatever the scale: a masked position has one too)
      if (whole_codes && threadIdx.x < 64)
        p.factors[((size_t)run * p.kv_heads + kvh) * 64 + threadIdx.x] =
            make_float2(ks < INFINITY ? fminf(ks * (128.0f / 127.0f), 3.402823466e38f) : 1.0f, vs > 0.0f && vs < INFINITY ? log2f(vs) + 0.0113153133f : -200.0f);
    }
    const int part = threadIdx.x & ((1 << unit_shift) - 1), apart = blockDim.x >> unit_shift;      // positions between two of a thread's turns
    for (int j0 = threadIdx.x >> unit_shift; j0 < 64; j0 += AHEAD * apart) {
      uint32_t raw[AHEAD][2][EACH / 4];
      float scale[AHEAD][2];
      int at[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int j = j0 + i * apart, pos = tile * 64 + j;
        at[i] = j < 64 ? j * p.head_dim + EACH * part : -1;
        const int page_index = pos >> page_shift, slot = pos & (p.page_size - 1);
        const bool held_here = j < 64 && pos < held;
        const int page = held_here && page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
        const bool here = page >= 0 && page < p.num_pages;
        if (held_here && !here && pos >= seen_from) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          scale[i][kv] = 0.0f;
#pragma unroll
          for (int k = 0; k < EACH / 4; ++k) raw[i][kv][k] = 0u;
        }
        if (here) {
          const size_t entry = ((size_t)(page * p.kv_heads + kvh) << page_shift) + slot, from = entry * p.head_dim + EACH * part;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int8_t* src = (kv ? p.v_pages : p.k_pages) + from;
            if constexpr (EACH == 8) {
              const uint2 x = *reinterpret_cast<const uint2*>(src);
              raw[i][kv][0] = x.x;
              raw[i][kv][1] = x.y;
            } else {
              raw[i][kv][0] = *reinterpret_cast<const uint32_t*>(src);
            }
            scale[i][kv] = (kv ? p.v_scale : p.k_scale)[entry >> shift];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (at[i] >= 0) {
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            float s = scale[i][kv] * (1.0f / 127.0f);
            if constexpr (HALVES) s = whole_codes ? (s == 0.0f || !(fabsf(s) < INFINITY) ? s : copysignf(1.0f / 128.0f, s)) : s * (kv == 0 ? k_over : v_over);
            if (!(fabsf(scale[i][1]) < INFINITY) && p.starts != nullptr) s = kv == 0 ? NAN : 0.0f;
            float x[EACH];
#pragma unroll
            for (int k = 0; k < EACH; ++k)     // 2^23 + (byte ^ 128), less 2^23 + 128: the code, exactly
              x[k] = (__uint_as_float(__byte_perm(raw[i][kv][k >> 2] ^ 0x80808080u, 0x4b000000u, 0x7440 + (k & 3))) - 8388736.0f) * s;
            T* dst = (kv ? v_dst : k_dst) + at[i];
            if constexpr (EACH == 8) put_eight(dst, Eight{{x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]}});
            else *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
          }
        }
    }
    continue;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int j = warp; j < 64; j += 8) {
    const int pos = tile * 64 + j;
    const int page_index = pos / p.page_size;
    const int page = pos < held && page_index < p.max_pages ? p.block_table[(size_t)seq * p.max_pages + page_index] : -1;
    const bool here = page >= 0 && page < p.num_pages;
    if (!here && pos >= seen_from && pos < held && lane == 0) atomicOr(p.status, TGE_STATUS_BAD_PAGE);
    const size_t entry = here ? ((size_t)page * p.kv_heads + kvh) * p.page_size + pos % p.page_size : 0;
    float ks = here ? p.k_scale[entry / p.block] * (1.0f / 127.0f) : 0.0f;
    float vs = here ? p.v_scale[entry / p.block] * (1.0f / 127.0f) : 0.0f;
    if (!(fabsf(vs) < INFINITY) && p.starts != nullptr) {
      ks = NAN;
      vs = 0.0f;
    }
    for (int d = lane; d < p.head_dim; d += 32) {
      k_dst[j * p.head_dim + d] = from_float<T>(here ? (float)p.k_pages[entry * p.head_dim + d] * ks : 0.0f);
      v_dst[j * p.head_dim + d] = from_float<T>(here ? (float)p.v_pages[entry * p.head_dim + d] * vs : 0.0f);
    }
  }
  }
}

int cache_shape(const char* what, int num_pages, int page_size, int block, int kv_heads, int head_dim, int max_pages) {
  TGE_REQUIRE(num_pages > 0 && page_size > 0 && kv_heads > 0 && max_pages > 0, "%s: bad page geometry", what);
  TGE_REQUIRE(head_dim > 0 && head_dim <= 32 * MAX_PER_LANE, "%s: head size %d, at most %d", what, head_dim, 32 * MAX_PER_LANE);
  TGE_REQUIRE(block > 0 && (block & (block - 1)) == 0 && page_size % block == 0, "%s: blocks of %d positions in pages of %d", what, block, page_size);
  return 0;
}

}  // namespace

TGE_API int tge_store_8bit(const void* qkv, int is_bf16, long long row_stride, void* q_out, long long q_stride, const float* cos_table,
                           const float* sin_table, int table_rows, int rotary, const int* positions, const int* seq_of_token,
                           const int* q_start, int num_seqs, const int* block_table, int max_pages, void* k_pages, void* v_pages,
                           float* k_scale, float* v_scale, int num_pages, int page_size, int block, int tokens, int heads, int kv_heads,
                           int head_dim, int* status, cudaStream_t stream) {
  const int rc = cache_shape("store_8bit", num_pages, page_size, block, kv_heads, head_dim, max_pages);
  if (rc != 0) return rc;
  TGE_REQUIRE(tokens >= 0 && heads > 0 && num_seqs >= 0, "store_8bit: bad sizes");
  TGE_REQUIRE(rotary >= 0 && rotary <= head_dim && rotary % 2 == 0, "store_8bit: rotary width %d must be even and at most head_dim %d", rotary, head_dim);
  TGE_REQUIRE(row_stride >= (long long)(heads + 2 * kv_heads) * head_dim && q_stride >= (long long)heads * head_dim, "store_8bit: rows too short");
  if (tokens == 0) return 0;
  const StoreParams p{qkv, q_out, row_stride, q_stride, cos_table, sin_table, table_rows, positions, seq_of_token, q_start, block_table,
                      max_pages, (int8_t*)k_pages, (int8_t*)v_pages, k_scale, v_scale, num_pages, page_size, block, tokens, num_seqs,
                      heads, kv_heads, head_dim, rotary, status};
  const size_t bytes = is_bf16 ? 16 : 32;                          // of eight numbers
  const bool power = head_dim >= 16 && (head_dim & (head_dim - 1)) == 0;
  const long long blocks = tokens + (block > 1 ? ((long long)tokens / block + 2ll * num_seqs) * 2 * kv_heads : 0);
  if (power && (rotary == 0 || rotary == head_dim) && blocks < 0x7fffffffll && row_stride * bytes / 8 % 16 == 0 && q_stride * bytes / 8 % 16 == 0 &&
      ((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos_table | (uintptr_t)sin_table | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0) {
    auto run = [&](auto type) {
      using T = decltype(type);
      const int lanes = (heads + (block == 1 ? 2 * kv_heads : 0) + UNIT_AHEAD - 1) / UNIT_AHEAD * (head_dim / 16);
      const int threads = std::min(UNIT_THREADS, std::max(64, (lanes + 31) / 32 * 32));
      auto launch = [&](void (*kernel)(StoreParams)) { tge_launch(kernel, dim3((unsigned)blocks), threads, 0, stream, p); };
      switch (head_dim) {
        case 16: launch(store_8bit_units_kernel<T, 16>); break;
        case 32: launch(store_8bit_units_kernel<T, 32>); break;
        case 64: launch(store_8bit_units_kernel<T, 64>); break;
        case 128: launch(store_8bit_units_kernel<T, 128>); break;
        default: launch(store_8bit_units_kernel<T, 256>); break;
      }
    };
    if (is_bf16) run(__nv_bfloat16());
    else run(float());
    return tge_launched("store_8bit", 1);
  }
  const dim3 grid(tokens, (heads + 2 * kv_heads + WARPS - 1) / WARPS);
  if (is_bf16)
    tge_launch(store_8bit_kernel<__nv_bfloat16>, grid, WARPS * 32, 0, stream, p);
  else
    tge_launch(store_8bit_kernel<float>, grid, WARPS * 32, 0, stream, p);
  return tge_launched("store_8bit", 1);
}

TGE_API int tge_read_8bit(const void* k_pages, const void* v_pages, const float* k_scale, const float* v_scale, int num_pages, int page_size,
                          int block, const int* block_table, int max_pages, const int* q_start, const int* start_pos, int first_seq,
                          int num_seqs, int kv_heads, int head_dim, int window, void* k_out, void* v_out, int type, void* factors, int* table,
                          int* starts, int runs, int width, int* status, cudaStream_t stream) {
  const int rc = cache_shape("read_8bit", num_pages, page_size, block, kv_heads, head_dim, max_pages);
  if (rc != 0) return rc;
  TGE_REQUIRE(first_seq >= 0 && num_seqs >= first_seq && runs >= 0 && width >= 0 && window >= 0 && kv_heads <= 65535, "read_8bit: bad sizes");
  if (num_seqs == first_seq) return 0;
  const ReadParams p{{block_table, q_start, start_pos, max_pages, num_pages, page_size, first_seq, num_seqs, window, table, starts, runs, width, status},
                     (const int8_t*)k_pages, (const int8_t*)v_pages, k_scale, v_scale, block, kv_heads, head_dim, k_out, v_out, static_cast<float2*>(factors),
                     factors == nullptr ? nullptr : static_cast<int*>(factors) + (size_t)runs * kv_heads * 128};
  const bool units = head_dim >= 16 && (head_dim & (head_dim - 1)) == 0 && (page_size & (page_size - 1)) == 0 &&
                     (long long)num_pages * kv_heads <= 0x7fffffffll && ((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0;
  if (type == 2 && (!units || factors == nullptr || (uintptr_t)factors % 16 != 0)) return TGE_UNSUPPORTED;
  tge_launch(read_plan_kernel, 1, PLAN_THREADS, 0, stream, p);
  if (runs == 0) return tge_launched("read_8bit", 1);
  // a block takes several heads of its run where there are many runs: finding whose it is costs as much as a head
  const int at_once = 10 * tge_sm_count();
  const dim3 grid(runs, std::max(1, std::min(kv_heads, (at_once + runs) / (runs + 1))));
  if (type == 2)
    tge_launch(read_8bit_kernel<__half, true>, grid, 256, 0, stream, p);
  else if (type == 1)
    tge_launch(units ? read_8bit_kernel<__nv_bfloat16, true> : read_8bit_kernel<__nv_bfloat16, false>, grid, 256, 0, stream, p);
  else
    tge_launch(units ? read_8bit_kernel<float, true> : read_8bit_kernel<float, false>, grid, 256, 0, stream, p);
  return tge_launched("read_8bit", 2);
}
