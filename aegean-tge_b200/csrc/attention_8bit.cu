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

// ---------------------------------------------------------------------------
// Single tokens on the tensor cores: head sizes 64, 128 and 256, pages of 16, 32, 64, ... positions.
//
// What bounds it: the cache's bytes, 2 head_dim + 8 / block of them a position and kv head.  A warp takes slices of 16 positions and
// nothing of them passes through shared memory: codes go from global memory into the registers that hold them as operands.
//   scores   S^T [16 positions x 8 heads] = C [16 x d] Q^T [d x 8]   (m16n8k32 of 8-bit whole numbers, a position per row): a lane
//            needs, of positions g and g + 8 (g = lane / 4), a quarter of the row, whole 16-byte chunks, because the order of d is
//            free as long as the queries come in the same one.  The codes are operands as they are.  A row of queries is rounded to
//            whole numbers of 15 bits (float32: 22) of its largest and taken as two (three) digits to the base 128, whose products are
//            added exactly in 32 bits.  2^-15 of the row's largest number is a 64th of what bfloat16 has rounded that number by; numbers
//            below 2^-6 of it lose more than bfloat16 had (a third digit: the 64 requests below 87 us where this takes 83);
//   values   O^T [d x 8 heads] += C'^T [d x 16 positions] P^T [16 x 8]   (m16n8k16 of float16): a lane needs, of positions 2t, 2t + 1,
//            2t + 8, 2t + 9 (t = lane % 4), the numbers that are rows g and g + 8 of every 16-row tile; which 16 numbers of d make a
//            tile is free too, so they are those of one 16-byte chunk.  A code becomes a float16 exactly: its byte, the sign bit turned over,
//            below the exponent of 1,024, less 1,152.  (Whole numbers would need no conversion here either, but a probability's small
//            numbers matter: a long tail of 2^-16 each must not become zeros.)  p is at most 2^8; its product with its position's scale
//            goes over the largest such product that the head had when it was last looked for, times 2^6, is at most 2^15, and keeps
//            11 bits down to 2^-20 of that product and some down to 2^-30: a large value that the head hardly weighs takes nothing from
//            the others.  float32 runs add what float16 leaves of it as a second part.
// Every load of the codes is 16 bytes a lane and whole 128-byte lines a warp.  Probabilities turn from S^T's accumulators into P^T's
// operand by two 8x8 transposes.  With heads as the narrow side of 8, a group of up to 8 heads wastes no more than its rest.
// The running maximum is raised only when a score passes it by 2^8, the products' one looked for again when a scale is twice it (one vote a
// slice); the sums of probabilities stay in their lanes until the end.
//
// Work: the slices of all (request, kv head, tile of heads) units in one row, cut into equal runs, one per block, whatever the
// requests' lengths; the blocks work that out from the lengths on the device, so a captured graph stays right as they grow.  A unit
// counts as BEGIN slices more than it has: what a block spends on its queries, its first copies and the joining of its warps.  A run
// that holds a whole unit writes its output; parts of units are left as (maximum, sum, unnormalised output) in scratch memory, at
// most two per block, and a second kernel joins them in the order of the positions.  Few units over short contexts (decode_cluster) go without: a
// cluster of blocks has a unit, its slices in equal shares, and joins them through its shared memory.
//
// Measured, with the joining: 64 requests of 2,048 to 4,096 positions at 40 heads over 8 (425 MB with their scales) 76.8 us, 5.5 TB/s or 0.85 of a
// copy's rate; a kernel that only reads the same pages takes 71.7.  Four of 32,768 41.6 us, eight of 2,048 at 28 heads over 4 (a cluster each unit)
// 9.9, of 512 7.1: the trips to memory one behind the other.  Not taken: the codes through rings in shared memory (117 us where this took 83), two slices of
// each warp on their way (94), slices dealt to the warps in turn instead of in runs (91 beside 81), pages asked into L2 a slice ahead (86).
// ---------------------------------------------------------------------------
constexpr int DWARPS = 4;
// The 64 requests at 0 / 12 / 24: 80.9 / 80.2 / 82.5 us, four of 32,768 47.8 / 45.6 / 45.9, eight of 2,048 16.5 / 14.4 / 14.4
constexpr int BEGIN = 12;
constexpr float NONE = -3.0e38f;                // a running maximum before the first score (finite: -inf less this is still -inf)
constexpr float LOG2E = 1.4426950408889634f;
// Probabilities times their values' scales are held over the largest such product of their head when it was last looked for, times HELD; it is
// looked for again where a value's scale alone is twice that.  LEAST, MOST: that product is taken as this where it is smaller or larger, so that
// it, the factor and their reciprocals are ordinary numbers for the fast division.
constexpr float HELD = 64.0f, LEAST = 1e-36f, MOST = 8e37f;

struct Decode8 {
  Attn8 a;
  const int *q_start, *start_pos;
  int units;                                    // per request: kv heads x tiles of heads
  int head_tiles, least;                        // least: slices of a run
  int page_shift, block_shift;                  // pages and blocks are powers of two here: no division in the loop
  int q_by_eight;                               // queries may be read eight bytes (two words) at a time
  float *parts, *states;                        // [2 x blocks][heads of a tile][head_dim], [2 x blocks][heads of a tile][2]
};

// The row of a request's token; -1: it brings none.
__device__ __forceinline__ int row_of(const Decode8& p, int seq) {
  const int row = p.q_start[seq], behind = p.q_start[seq + 1];
  return behind > row ? row : -1;
}

// The slices of 16 positions that request `seq` sees: [first, first + count), one at least.  `wrong`: what is to be reported of a token whose
// position is none, or one that the block table has no room for; the others are served as far as they go.
struct Slices { int lo, hi, first, count, wrong; };
__device__ __forceinline__ Slices slices_of(const Decode8& p, int seq) {
  Slices s;
  const int start = p.start_pos[seq], here = p.q_start[seq], behind = p.q_start[seq + 1];      // one trip to memory
  const int pos = behind > here ? start : -1, room = p.a.max_pages << p.page_shift;
  s.hi = min(max(pos, -1), room - 1) + 1;
  s.wrong = behind <= here ? 0 : start < 0 ? TGE_STATUS_BAD_ROW : start >= room ? TGE_STATUS_BAD_PAGE : 0;
  s.lo = p.a.window > 0 ? max(pos - p.a.window + 1, 0) : 0;
  s.first = s.lo >> 4;
  s.count = max((s.hi + 15) / 16 - s.first, 1);
  return s;
}

// What requests [0, upto) count for in the row, by the whole warp.
__device__ __forceinline__ int slices_before(const Decode8& p, int upto, int lane) {
  int n = 0;
  for (int seq = lane; seq < upto; seq += 32) n += (slices_of(p, seq).count + BEGIN) * p.units;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) n += __shfl_xor_sync(0xffffffffu, n, offset);
  return n;
}
__device__ __forceinline__ int run_length(const Decode8& p, int total, int blocks) { return max((total + blocks - 1) / blocks, p.least); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Codes of bytes `which` of two words as two float16.
__device__ __forceinline__ uint32_t two_codes(uint32_t a, uint32_t b, uint32_t which) {
  uint32_t r = __byte_perm(a, b, which), v;
  asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;\n" : "=r"(v) : "r"(r));       // (r & mask) ^ pattern: 1,024 + (byte ^ 128)
  asm("add.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(v), "r"(0xe480e480u));            // - 1,152
  return r;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {      // an 8x8 tile of 16-bit numbers across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// What float16 leaves of a pair.
__device__ __forceinline__ void leave(uint32_t taken, float& lo, float& hi) {
  float a, b;
  asm("{\n.reg .b16 x, y;\nmov.b32 {x, y}, %2;\ncvt.f32.f16 %0, x;\ncvt.f32.f16 %1, y;\n}\n" : "=f"(a), "=f"(b) : "r"(taken));
  lo -= a;
  hi -= b;
}

template <int HD>
struct Codes {
  static constexpr int KC = HD / 64;            // 16-byte chunks of a key that a lane holds
  static constexpr int VB = HD >= 128 ? 16 : HD / 8, VC = HD / 8 / VB;   // bytes of a chunk of a value, chunks
  uint32_t k[2][KC][4];
  uint32_t v[4][VC][VB / 4];
  float ks[2], vs[2];
};

__device__ __forceinline__ void load16(const void* src, uint32_t (&x)[4]) {
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "l"(src));
}
__device__ __forceinline__ void load16(const void* src, uint32_t (&x)[2]) {     // the half of it that heads of 64 numbers have
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];\n" : "=r"(x[0]), "=r"(x[1]) : "l"(src));
}

template <int HD>
__device__ __forceinline__ void load_keys(const Decode8& p, Codes<HD>& c, size_t row, int g, int t) {
  const int8_t* src = p.a.k_pages + (row + g) * HD + 16 * t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int j = 0; j < Codes<HD>::KC; ++j) load16(src + 8 * i * HD + 64 * j, c.k[i][j]);
    c.ks[i] = p.a.k_scale[(row + g + 8 * i) >> p.block_shift];
  }
}
template <int HD>
__device__ __forceinline__ void load_values(const Decode8& p, Codes<HD>& c, size_t row, int g, int t) {
  const int8_t* src = p.a.v_pages + (row + 2 * t) * HD + Codes<HD>::VB * g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < Codes<HD>::VC; ++j) load16(src + ((i & 1) + 8 * (i >> 1)) * HD + 128 * j, c.v[i][j]);
#pragma unroll
  for (int i = 0; i < 2; ++i) c.vs[i] = p.a.v_scale[(row + g + 8 * i) >> p.block_shift];
}

// Four numbers of a row of queries.
template <typename T>
__device__ __forceinline__ void four(const T* q, bool vector, float (&x)[4]) {
  if (vector) {
    if constexpr (sizeof(T) == 2) {
      const uint2 raw = *reinterpret_cast<const uint2*>(q);
      x[0] = __uint_as_float(raw.x << 16); x[1] = __uint_as_float(raw.x & 0xffff0000u);
      x[2] = __uint_as_float(raw.y << 16); x[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
      const float2 lo = *reinterpret_cast<const float2*>(q), hi = *reinterpret_cast<const float2*>(q + 2);
      x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = to_float<T>(q[i]);
  }
}

// A row of queries as DIGITS whole numbers to the base 128 per number, four numbers to a word, in the order of the codes' words; the lane has
// a quarter of the row, the four lanes of a row agree on its largest number.  Words w of chunk j go to to[j][digit][lane], four side by
// side.  Returns what the whole numbers are to be multiplied with (NaN if a number is not finite).
template <typename T, int HD, int DIGITS>
__device__ __forceinline__ float query_digits(const T* q, bool valid, bool vector, int t, uint32_t (*to)[DIGITS][32][4]) {
  constexpr float TOP = DIGITS == 2 ? 16256.0f : 2080768.0f;          // 127 x 128^(DIGITS - 1)
  float most = 0.0f;
  bool fine = true;
  auto each = [&](auto use) {
#pragma unroll
    for (int j = 0; j < HD / 64; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (valid) four<T>(q + 16 * (t + 4 * j) + 4 * w, vector, x);
        use(j, w, x);
      }
  };
  each([&](int, int, const float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      most = fmaxf(most, fabsf(x[i]));
      fine &= fabsf(x[i]) < INFINITY;
    }
  });
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
  const float over = most > TOP * 3e-39f ? TOP / most : 0.0f;         // (float32 has no larger factor: rows below that are zeros)
  each([&](int j, int w, const float (&x)[4]) {
    int whole[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) whole[i] = __float2int_rn(x[i] * over);
#pragma unroll
    for (int digit = DIGITS - 1; digit >= 0; --digit) {
      int here[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rest = (whole[i] + 64) >> 7;
        here[i] = digit > 0 ? whole[i] - 128 * rest : whole[i];
        whole[i] = rest;
      }
      to[j][digit][threadIdx.x & 31][w] = __byte_perm(__byte_perm(here[0], here[1], 0x0040), __byte_perm(here[2], here[3], 0x0040), 0x5410);
    }
  });
  // a number that is not finite in any quarter
  const unsigned rest = __ballot_sync(0xffffffffu, !fine) >> (threadIdx.x & 28);
  return (rest & 15u) == 0u ? most * (1.0f / TOP) : __int_as_float(0x7fc00000);
}

// The first of the two numbers of d that a pair in the accumulators' order is (tile pair / 8, lanes g = pair % 8).
template <int HD>
__device__ __forceinline__ int number_of(int pair) {
  constexpr int VB = Codes<HD>::VB;
  const int i = pair >> 3, g = pair & 7, j = i / (VB / 2);
  return VB * (g + 8 * j) + 2 * (i - j * (VB / 2));
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

// Blocks on an SM.  Codes on their way are what hides the memory's latency, and they are in registers: five blocks of heads of 128 numbers have
// room too, but bring more parts to join (eight requests of 2,048 14.4 us, with four 13.7; the 64 of up to 4,096 80 both; with three 87).
__host__ __device__ constexpr int decode_blocks_per_sm(int head_dim, int tiles) { return head_dim * tiles <= 64 ? 6 : head_dim * tiles <= 128 ? 4 : 3; }

template <typename T, int HD, int NT, bool CLUSTER>
__global__ void __launch_bounds__(DWARPS * 32, decode_blocks_per_sm(HD, NT)) decode_8bit_kernel(const Decode8 p) {
  constexpr int DIGITS = sizeof(T) == 2 ? 2 : 3, PARTS = sizeof(T) == 2 ? 1 : 2;
  constexpr int HEADS = 8 * NT, MTILES = HD / 16, PITCH = HD + 4;
  using C = Codes<HD>;
  extern __shared__ float merge_o[];                              // [warps][HEADS][PITCH], a head's numbers in the order of the accumulators
  __shared__ float merge_m[DWARPS][HEADS], merge_l[DWARPS][HEADS], merge_v[DWARPS][HEADS], factors[HEADS];
  __shared__ __align__(16) uint32_t queries[NT][C::KC][DIGITS][32][4];
  __shared__ int start_of[5];
  __shared__ float2 part_state[CLUSTER ? HEADS : 1];              // what merge_o's first place is over: (maximum, sum)
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = uniform_warp_index();
  const int g = lane >> 2, t = lane & 3;
  if (!CLUSTER && warp == 0) {                                    // where this block's run begins
    // 32 requests at a time; the first of them stay where they are
    const int first_count = lane < p.a.num_seqs ? (slices_of(p, lane).count + BEGIN) * p.units : 0;
    const int first_token = lane < p.a.num_seqs ? row_of(p, lane) : 0;
    int total = __reduce_add_sync(0xffffffffu, first_count);
    for (int seq = 32 + lane; seq - lane < p.a.num_seqs; seq += 32)
      total += __reduce_add_sync(0xffffffffu, seq < p.a.num_seqs ? (slices_of(p, seq).count + BEGIN) * p.units : 0);
    const int run = run_length(p, total, gridDim.x);
    const int from = (int)min((long long)run * blockIdx.x, (long long)total);
    int seq = 0, base = 0, token = first_token;
    while (seq < p.a.num_seqs) {
      int n = first_count;
      if (seq > 0) {
        n = seq + lane < p.a.num_seqs ? (slices_of(p, seq + lane).count + BEGIN) * p.units : 0;
        token = seq + lane < p.a.num_seqs ? row_of(p, seq + lane) : 0;
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
    const int heads_here = min(HEADS, p.a.group - tile * HEADS), head0 = kvh * p.a.group + tile * HEADS;
    const int* table = p.a.block_table + (size_t)seq * p.a.max_pages;
    // the warps' shares of the run's slices, one behind the other
    const int first = s.first + skip + length * warp / DWARPS, last = s.first + skip + length * (warp + 1) / DWARPS;
    bool bad = false;
    auto page_at = [&](int index) { return index < p.a.max_pages ? table[index] : -1; };
    // where a page's entries start; one outside the pool reads page 0, unseen
    auto start_at = [&](int page) { return (size_t)((page >= 0 && page < p.a.num_pages ? page : 0) * p.a.kv_heads + kvh) << p.page_shift; };
    // the slice to ask for next, its page and the one behind it
    int asked = first, page = page_at((first << 4) >> p.page_shift), page_behind = page_at(((first << 4) >> p.page_shift) + 1);
    size_t row = start_at(page) + ((first << 4) & (p.a.page_size - 1));
    auto advance = [&] {
      ++asked;
      row += 16;
      if (((asked << 4) & (p.a.page_size - 1)) == 0) {
        page = page_behind;
        page_behind = page_at(((asked << 4) >> p.page_shift) + 1);
        row = start_at(page);
      }
    };
    if (!waited) pdl_wait();                                       // all above is what the step was given
    waited = true;
    C c;
    if (first < last) {
      load_keys<HD>(p, c, row, g, t);
      load_values<HD>(p, c, row, g, t);
    }
    if (warp < NT) {
      const bool valid = token >= 0 && 8 * warp + g < heads_here;
      const T* src = static_cast<const T*>(p.a.q) + (size_t)max(token, 0) * p.a.q_stride + (size_t)(head0 + (valid ? 8 * warp + g : 0)) * HD;
      const float unit_of = query_digits<T, HD, DIGITS>(src, valid, p.q_by_eight != 0, t, queries[warp]) * (p.a.scale * (LOG2E / 127.0f));
      if (t == 0) factors[8 * warp + g] = unit_of;
    }
    __syncthreads();
    float factor[NT][2];                                          // of the scores of heads 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      factor[nt][0] = factors[8 * nt + 2 * t];
      factor[nt][1] = factors[8 * nt + 2 * t + 1];
    }
    // a head's running maximum, its sum of probabilities, and what products of a probability and a value's scale are multiplied with
    float o[NT][MTILES][4], m[NT][2], l[NT][2], over[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
      m[nt][0] = m[nt][1] = NONE;
      l[nt][0] = l[nt][1] = 0.0f;
      over[nt][0] = over[nt][1] = HELD / LEAST;
    }

    for (int slice = first; slice < last; ++slice) {
      const bool here = page >= 0 && page < p.a.num_pages;         // `asked` is this slice still
      bad |= !here;
      advance();

      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        int acc[DIGITS][4];
#pragma unroll
        for (int digit = 0; digit < DIGITS; ++digit)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[digit][e] = 0;
#pragma unroll
        for (int j = 0; j < C::KC; ++j)
#pragma unroll
          for (int digit = 0; digit < DIGITS; ++digit) {
            const uint4 q = *reinterpret_cast<const uint4*>(queries[nt][j][digit][lane]);
            mma_s8(acc[digit], c.k[0][j][0], c.k[1][j][0], c.k[0][j][1], c.k[1][j][1], q.x, q.y);
            mma_s8(acc[digit], c.k[0][j][2], c.k[1][j][2], c.k[0][j][3], c.k[1][j][3], q.z, q.w);
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // at most 256 x 127 x 127 in a digit's sum: two of them fit 32 bits, the third is added in float32
          float sum = (float)(128 * acc[DIGITS - 2][e] + acc[DIGITS - 1][e]);
          if constexpr (DIGITS == 3) sum = fmaf((float)acc[0][e], 16384.0f, sum);
          sc[nt][e] = sum;
        }
      }
      const float f0 = c.ks[0], f1 = c.ks[1];
      float v0 = c.vs[0], v1 = c.vs[1];
      float e[NT][4], held[NT][4];                                   // probabilities; with their values' scales, as the tensor core gets them
      bool raise = false;                                            // (an unseen position's scale costs a look, no more)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          held[nt][i] = v0 * over[nt][i];
          held[nt][2 + i] = v1 * over[nt][i];
          raise |= fmaxf(fabsf(held[nt][i]), fabsf(held[nt][2 + i])) > 2.0f * HELD;
        }
      if (slice + 1 < last) load_keys<HD>(p, c, row, g, t);

#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[nt][e] *= f0 * factor[nt][e];
          sc[nt][2 + e] *= f1 * factor[nt][e];
        }
      if (!here || slice * 16 < s.lo || slice * 16 + 16 > s.hi) {    // some of the slice's positions are not seen
        const int k0 = slice * 16 + g;
        const bool see0 = here && k0 >= s.lo && k0 < s.hi, see1 = here && k0 + 8 >= s.lo && k0 + 8 < s.hi;
        v0 = see0 ? v0 : 0.0f;                                       // their scales may be anything, NaN too
        v1 = see1 ? v1 : 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sc[nt][e] = see0 ? sc[nt][e] : -INFINITY;
            sc[nt][2 + e] = see1 ? sc[nt][2 + e] : -INFINITY;
            held[nt][e] = see0 ? held[nt][e] : 0.0f;
            held[nt][2 + e] = see1 ? held[nt][2 + e] : 0.0f;
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) raise |= fmaxf(sc[nt][i], sc[nt][2 + i]) > m[nt][i] + 8.0f;
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float down[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float most = fmaxf(sc[nt][i], sc[nt][2 + i]);
#pragma unroll
            for (int offset = 4; offset < 32; offset <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
            most = fmaxf(most, m[nt][i]);
            const float fall = exp2_fast(m[nt][i] - most);
            m[nt][i] = most;
            l[nt][i] *= fall;
            // the largest product here; what the largest so far comes to under the new maximum
            float seen = fmaxf(fabsf(exp2_fast(sc[nt][i] - most) * v0), fabsf(exp2_fast(sc[nt][2 + i] - most) * v1));
#pragma unroll
            for (int offset = 4; offset < 32; offset <<= 1) seen = fmaxf(seen, __shfl_xor_sync(0xffffffffu, seen, offset));
            const float so_far = __fdividef(HELD, over[nt][i]) * fall, now = fminf(fmaxf(fmaxf(so_far, seen), LEAST), MOST);
            over[nt][i] = __fdividef(HELD, now);
            down[i] = __fdividef(so_far, now);
          }
#pragma unroll
          for (int i = 0; i < MTILES; ++i) {
            o[nt][i][0] *= down[0]; o[nt][i][1] *= down[1];
            o[nt][i][2] *= down[0]; o[nt][i][3] *= down[1];
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[nt][i] = exp2_fast(sc[nt][i] - m[nt][i & 1]);
            held[nt][i] = e[nt][i] * (i < 2 ? v0 : v1) * over[nt][i & 1];        // (in this order: a large value may have no probability)
          }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[nt][i] = exp2_fast(sc[nt][i] - m[nt][i & 1]);
            held[nt][i] *= e[nt][i];
          }
      }
      uint32_t pr[NT][PARTS][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        l[nt][0] += e[nt][0] + e[nt][2];
        l[nt][1] += e[nt][1] + e[nt][3];
        float (&h)[4] = held[nt];
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t x = two_halves(h[0], h[1]), y = two_halves(h[2], h[3]);
          pr[nt][part][0] = transposed(x);
          pr[nt][part][1] = transposed(y);
          if (part + 1 < PARTS) {
            leave(x, h[0], h[1]);
            leave(y, h[2], h[3]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C::VC; ++j)
#pragma unroll
        for (int w = 0; w < C::VB / 4; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // bytes 2 half and 2 half + 1 of a word of positions 2t and 2t + 1, and of 2t + 8 and 2t + 9: rows g and g + 8 of a tile
            const uint32_t low = half ? 0x6622 : 0x4400, high = half ? 0x7733 : 0x5511;
            const uint32_t a0 = two_codes(c.v[0][j][w], c.v[1][j][w], low), a1 = two_codes(c.v[0][j][w], c.v[1][j][w], high);
            const uint32_t a2 = two_codes(c.v[2][j][w], c.v[3][j][w], low), a3 = two_codes(c.v[2][j][w], c.v[3][j][w], high);
            const int i = (j * (C::VB / 4) + w) * 2 + half;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) mma_f16(o[nt][i], a0, a1, a2, a3, pr[nt][part][0], pr[nt][part][1]);
          }
      if (slice + 1 < last) load_values<HD>(p, c, row, g, t);
    }
    if (token >= 0 && lane == 0 && (bad || s.wrong != 0)) atomicOr(p.a.status, s.wrong != 0 ? s.wrong : TGE_STATUS_BAD_PAGE);

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
          merge_m[warp][head] = m[nt][e];
          merge_l[warp][head] = sum;
          merge_v[warp][head] = __fdividef(1.0f / 127.0f, over[nt][e]);
        }
        float* dst = merge_o + (warp * HEADS + head) * PITCH + 2 * g;
#pragma unroll
        for (int i = 0; i < MTILES; ++i) *reinterpret_cast<float2*>(dst + 16 * i) = make_float2(o[nt][i][e], o[nt][i][2 + e]);
      }
    }
    __syncthreads();
    const bool whole = !CLUSTER && length == s.count;
    const size_t place = (size_t)(2 * blockIdx.x + (skip == 0 ? 1 : 0)) * HEADS;
    for (int i = threadIdx.x; i < heads_here * (HD / 2); i += DWARPS * 32) {
      const int head = i / (HD / 2), pair = i - head * (HD / 2);
      float most = NONE;
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) most = fmaxf(most, merge_m[w][head]);
      float sum = 0.0f;
      float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) {
        const float f = exp2_fast(merge_m[w][head] - most), fv = f * merge_v[w][head];
        const float2 x = *reinterpret_cast<const float2*>(merge_o + (w * HEADS + head) * PITCH + 2 * pair);
        sum = fmaf(f, merge_l[w][head], sum);
        acc.x = fmaf(fv, x.x, acc.x);
        acc.y = fmaf(fv, x.y, acc.y);
      }
      if (whole) {
        if (token < 0) continue;
        if (p.a.sink != nullptr) {
          const float sink = p.a.sink[head0 + head] * LOG2E, top = fmaxf(most, sink), down = exp2_fast(most - top);
          sum = fmaf(sum, down, exp2_fast(sink - top));
          acc.x *= down;
          acc.y *= down;
        }
        const float over = sum == 0.0f ? 0.0f : 1.0f / sum;
        T* dst = static_cast<T*>(p.a.out) + (size_t)token * p.a.out_stride + (size_t)(head0 + head) * HD + number_of<HD>(pair);
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
        const float sink = p.a.sink != nullptr ? p.a.sink[head0 + head] * LOG2E : NONE;
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
        if (p.a.sink != nullptr) all += exp2_fast(sink - top);
        const float over = all == 0.0f ? 0.0f : 1.0f / all;
        T* dst = static_cast<T*>(p.a.out) + (size_t)token * p.a.out_stride + (size_t)(head0 + head) * HD + number_of<HD>(pair);
        dst[0] = from_float<T>(acc.x * over);
        dst[1] = from_float<T>(acc.y * over);
      }
      cluster_sync();                                             // nobody leaves while another reads its memory
    }
    if (next_seq && at < end) {
      base = at;
      ++seq;
      token = row_of(p, seq);
    }
  }
  if (!waited) pdl_wait();
}

// Joins the parts of the units that more than one block worked on: one block per unit, two warps per head, which take the first and the
// second half of its parts.
constexpr int JOIN_WARPS = 16, JOIN_AHEAD = 8;

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) decode_8bit_join_kernel(const Decode8 p, int blocks) {
  constexpr int HEADS = 8 * NT, PAIRS = HD / 64;                   // pairs of numbers of a lane
  __shared__ int where[2];
  __shared__ float half_m[8], half_l[8], half_o[8][HD];
  pdl_trigger();
  const int seq = blockIdx.x, unit = blockIdx.y, lane = threadIdx.x & 31, warp = uniform_warp_index();
  if (warp == 0) {
    const int total = slices_before(p, p.a.num_seqs, lane), run = run_length(p, total, blocks);
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
  const int heads_here = min(HEADS, p.a.group - tile * HEADS), head0 = kvh * p.a.group + tile * HEADS;
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
      const float sink = p.a.sink != nullptr ? p.a.sink[head0 + head] * LOG2E : NONE;
      const float top = fmaxf(fmaxf(most, half_m[head & 7]), sink);
      const float f0 = exp2_fast(most - top), f1 = exp2_fast(half_m[head & 7] - top);
      const float all = fmaf(sum, f0, f1 * half_l[head & 7]) + (p.a.sink != nullptr ? exp2_fast(sink - top) : 0.0f);
      const float over = all == 0.0f ? 0.0f : 1.0f / all;
      T* dst = static_cast<T*>(p.a.out) + (size_t)token * p.a.out_stride + (size_t)(head0 + head) * HD;
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(&half_o[head & 7][2 * (lane + 32 * i)]);
        const int d = number_of<HD>(lane + 32 * i);
        dst[d] = from_float<T>(fmaf(acc[i].x, f0, f1 * x.x) * over);
        dst[d + 1] = from_float<T>(fmaf(acc[i].y, f0, f1 * x.y) * over);
      }
    }
  }
}

template <typename T, int HD, int NT>
int launch_decode(Decode8 p, int blocks, int cluster, cudaStream_t stream) {
  constexpr int smem = DWARPS * 8 * NT * (HD + 4) * 4;
  static bool ready[64] = {};                                     // shared memory beyond 48 KB, clusters of 16: asked for once per device
  int device = 0;
  cudaGetDevice(&device);
  if (device >= 64 || !ready[device]) {
    cudaError_t rc = cudaFuncSetAttribute(decode_8bit_kernel<T, HD, NT, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (rc == cudaSuccess && smem > 48 * 1024) rc = cudaFuncSetAttribute(decode_8bit_kernel<T, HD, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc == cudaSuccess && smem > 48 * 1024) rc = cudaFuncSetAttribute(decode_8bit_kernel<T, HD, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    TGE_REQUIRE(rc == cudaSuccess, "attention_8bit: %d bytes of shared memory, clusters of 16: %s", smem, cudaGetErrorString(rc));
    if (device < 64) ready[device] = true;
  }
  if (cluster > 0) {
    tge_launch_clusters(decode_8bit_kernel<T, HD, NT, true>, dim3(p.a.num_seqs * p.units * cluster), DWARPS * 32, smem, cluster, stream, p);
    return tge_launched("attention_8bit", 1);
  }
  p.states = p.parts + (size_t)2 * blocks * 8 * NT * HD;
  tge_launch(decode_8bit_kernel<T, HD, NT, false>, blocks, DWARPS * 32, smem, stream, p);
  tge_launch(decode_8bit_join_kernel<T, HD, NT>, dim3(p.a.num_seqs, p.units), JOIN_WARPS * 32, 0, stream, p, blocks);
  return tge_launched("attention_8bit", 2);
}

// Blocks of a launch: all that are on the device at a time, so that all runs advance together.
int decode_blocks(int head_dim, int tile_heads) { return tge_sm_count() * decode_blocks_per_sm(head_dim, tile_heads / 8); }

}  // namespace

// Heads of a tile: a group of up to 8 heads makes one tile of 8, more go by 16 (one pass over the codes for twice the accumulators, which
// heads of 256 numbers have no registers for).
static int decode_tile(int group, int head_dim) { return group <= 8 || head_dim > 128 ? 8 : 16; }

// Blocks of a cluster per unit, which joins its parts itself; 0: runs of slices and a second kernel.  A rule on what the host knows, the units and the
// bound of their lengths.  Clusters of 8 while all of them are on the device at a time, us with them / with runs: one to 16 requests of 512
// at 28 heads over 4 8.2 to 10.3 / 10.3 to 11.8, of 2,048 10.3 to 13.3 / 10.3 to 14.7, of 4,096 12.3 to 18.5 / 12.3 to 18.5 (8 of them 14.4 / 16.2); of
// 8,192 18 / 16.  Clusters of 16 for few units and longer bounds: one to four requests of 4,096 10.3 to 12.3, of 8,192 14 to 15, of 16,384 18.5
// to 22 / 18.6 to 18.9; 32 units of them are not on the device at a time (18.5 us where 8 take 10.3).
static int decode_cluster(long long units, int head_dim, int tile, long long positions) {
  if (units <= 16 && positions > 2048 && positions <= 8192) return 16;
  return 8 * units <= decode_blocks(head_dim, tile) && positions <= 4096 ? 8 : 0;
}

// float32 scratch numbers of tge_attention_8bit_decode; -1: sizes that it does not take.
TGE_API long long tge_attention_8bit_decode_floats(int is_bf16, int num_seqs, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_size < 16 || (page_size & (page_size - 1)) != 0 || kv_heads <= 0 || heads % kv_heads != 0) return -1;
  const int tile = decode_tile(heads / kv_heads, head_dim);
  const long long units = (long long)kv_heads * ((heads / kv_heads + tile - 1) / tile);
  // places in the row of all slices are counted in 32 bits, units along a grid's second axis
  if (units > 65535 || (long long)max_pages * page_size > (1ll << 30) ||
      units * num_seqs * ((long long)max_pages * page_size / 16 + 1 + BEGIN) > (1ll << 30)) return -1;
  if (decode_cluster(units * num_seqs, head_dim, tile, (long long)max_pages * page_size) > 0) return 0;
  return 2ll * decode_blocks(head_dim, tile) * tile * (head_dim + 2);
}

TGE_API int tge_attention_8bit_decode(const void* q, int is_bf16, long long q_stride, const void* k_pages, const void* v_pages, const float* k_scale,
                                      const float* v_scale, int num_pages, int page_size, int block, const int* block_table, int max_pages,
                                      const int* q_start, const int* start_pos, int num_seqs, void* out, long long out_stride, int heads, int kv_heads,
                                      int head_dim, float scale, int window, const float* sink, float* parts, long long part_floats, int* status,
                                      cudaStream_t stream) {
  const long long need = tge_attention_8bit_decode_floats(is_bf16, num_seqs, heads, kv_heads, head_dim, page_size, max_pages);
  if (need < 0 || ((uintptr_t)k_pages | (uintptr_t)v_pages) % 16 != 0) return TGE_UNSUPPORTED;
  TGE_REQUIRE(part_floats >= need, "attention_8bit: %lld floats of scratch memory, %lld wanted", part_floats, need);
  TGE_REQUIRE(num_pages > 0 && block > 0 && page_size % block == 0 && max_pages > 0 && window >= 0, "attention_8bit: bad page geometry");
  if ((long long)num_pages * kv_heads > 0x7fffffffll) return TGE_UNSUPPORTED;
  if (num_seqs == 0) return 0;
  const int group = heads / kv_heads, tile = decode_tile(group, head_dim);
  Decode8 p;
  p.a = Attn8{q, out, q_stride, out_stride, (const int8_t*)k_pages, (const int8_t*)v_pages, k_scale, v_scale, block_table, nullptr, nullptr, sink,
              max_pages, num_pages, page_size, block, num_seqs, heads, kv_heads, group, head_dim, window, scale, status};
  p.q_start = q_start;
  p.start_pos = start_pos;
  p.head_tiles = (group + tile - 1) / tile;
  p.units = kv_heads * p.head_tiles;
  p.least = 2 * DWARPS;
  const int element = is_bf16 ? 2 : 4;
  p.q_by_eight = (uintptr_t)q % 8 == 0 && q_stride * element % 8 == 0;
  p.page_shift = __builtin_ctz(page_size);
  p.block_shift = __builtin_ctz(block);
  p.parts = parts;
  const int blocks = decode_blocks(head_dim, tile);
  const int cluster = decode_cluster((long long)p.units * num_seqs, head_dim, tile, (long long)max_pages * page_size);
  auto run = [&](auto type) {
    using T = decltype(type);
    if (head_dim == 256) return launch_decode<T, 256, 1>(p, blocks, cluster, stream);
    if (head_dim == 128) return tile == 8 ? launch_decode<T, 128, 1>(p, blocks, cluster, stream) : launch_decode<T, 128, 2>(p, blocks, cluster, stream);
    return tile == 8 ? launch_decode<T, 64, 1>(p, blocks, cluster, stream) : launch_decode<T, 64, 2>(p, blocks, cluster, stream);
  };
  return is_bf16 ? run(__nv_bfloat16()) : run(float());
}

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
