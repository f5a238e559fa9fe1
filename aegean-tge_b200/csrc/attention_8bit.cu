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
// Single tokens on the tensor cores: head sizes 64, 128 and 256, pages that are multiples of 16 positions.
//
// What bounds it: the cache's bytes, 2 head_dim + 8 / block of them a position and kv head.  A warp takes slices of 16 positions and
// nothing of them passes through shared memory: codes go from global memory into the registers that hold them as operands.
//   scores   S^T [16 positions x 8 heads] = C [16 x d] Q^T [d x 8]   (mma m16n8k16, a position per row): a lane needs, of positions
//            g and g + 8 (g = lane / 4), a quarter of the row, whole 16-byte chunks, because the order of d is free as long as the
//            queries come in the same one;
//   values   O^T [d x 8 heads] += C'^T [d x 16 positions] P^T [16 x 8]: a lane needs, of positions 2t, 2t + 1, 2t + 8, 2t + 9
//            (t = lane % 4), the numbers that are rows g and g + 8 of every 16-row tile; which 16 numbers of d make a tile is free
//            too, so they are those of one 16-byte chunk.
// Every load of the codes is 16 bytes a lane and whole 128-byte lines a warp.  Probabilities turn from S^T's accumulators into P^T's
// operand by two 8x8 transposes.  With heads as the narrow side of 8, a group of up to 8 heads wastes no more than its rest.
// A code becomes a bfloat16 exactly: (0x4300 | low seven bits) - (0x4300 | sign bit), that is 128 + low - (128 or 256), two numbers at a
// time.  Scales go on scores and probabilities in float32.  The running maximum is raised only when a score passes it by 2^8 (one
// vote a slice); the sums of probabilities stay in their lanes until the end.
// float32 queries and probabilities are the sum of three bfloat16 numbers each, products of parts are added in float32.
//
// Work: the slices of all (request, kv head, tile of heads) units in one row, cut into equal runs, one per block, whatever the
// requests' lengths; the blocks work that out from the lengths on the device, so a captured graph stays right as they grow.  A run
// that holds a whole unit writes its output; parts of units are left as (maximum, sum, unnormalised output) in scratch memory, at
// most two per block, and a second kernel joins them in the order of the positions.
// ---------------------------------------------------------------------------
constexpr int DWARPS = 8;
constexpr float NONE = -3.0e38f;                // a running maximum before the first score (finite: -inf less this is still -inf)

struct Decode8 {
  Attn8 a;
  const int *q_start, *start_pos;
  int units;                                    // per request: kv heads x tiles of heads
  int head_tiles, least;                        // least: slices of a run
  float* parts;                                 // [2 x blocks][heads of a tile][head_dim + 2]
};

// The slices of 16 positions that request `seq` sees: [first, first + count).
struct Slices { int pos, lo, hi, first, count; };
__device__ __forceinline__ Slices slices_of(const Decode8& p, int seq) {
  Slices s;
  s.pos = p.start_pos[seq];
  s.hi = min(max(s.pos + 1, 0), p.a.max_pages * p.a.page_size);
  s.lo = p.a.window > 0 ? max(s.pos - p.a.window + 1, 0) : 0;
  s.first = s.lo >> 4;
  s.count = max((s.hi + 15) / 16 - s.first, 1);
  return s;
}

// Sum of the slice counts of requests [0, upto), by the whole warp.
__device__ __forceinline__ int slices_before(const Decode8& p, int upto, int lane) {
  int n = 0;
  for (int seq = lane; seq < upto; seq += 32) n += slices_of(p, seq).count;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) n += __shfl_xor_sync(0xffffffffu, n, offset);
  return n;
}
__device__ __forceinline__ int run_length(const Decode8& p, int total, int blocks) { return max((total + blocks - 1) / blocks, p.least); }

__device__ __forceinline__ uint32_t even_codes(uint32_t x) {      // bytes 0 and 2 as two bfloat16
  uint32_t low, high, r;
  asm("lop3.b32 %0, %1, 0x007f007f, 0x43004300, 0xea;\n" : "=r"(low) : "r"(x));
  asm("lop3.b32 %0, %1, 0x00800080, 0x43004300, 0xea;\n" : "=r"(high) : "r"(x));
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(low), "r"(high));
  return r;
}
__device__ __forceinline__ uint32_t odd_codes(uint32_t x) { return even_codes(x >> 8); }

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {      // an 8x8 tile of 16-bit numbers across the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// What bfloat16 leaves of a pair, as the next pair of parts.
__device__ __forceinline__ void leave(uint32_t taken, float& lo, float& hi) {
  const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&taken));
  lo -= v.x;
  hi -= v.y;
}

template <int HD>
struct Codes {
  static constexpr int KC = HD / 64;            // 16-byte chunks of a key that a lane holds
  static constexpr int VB = HD >= 128 ? 16 : HD / 8, VC = HD / 8 / VB;   // bytes of a chunk of a value, chunks
  uint4 k[2][KC];
  uint32_t v[4][VC][VB / 4];
  float ks[2], vs[2];
};

template <int HD>
__device__ __forceinline__ void load_keys(const Decode8& p, Codes<HD>& c, size_t row, int g, int t) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const size_t entry = row + g + 8 * i;
#pragma unroll
    for (int j = 0; j < Codes<HD>::KC; ++j)
      c.k[i][j] = __ldcs(reinterpret_cast<const uint4*>(p.a.k_pages + entry * HD) + t + 4 * j);
    c.ks[i] = p.a.k_scale[entry / p.a.block];
  }
}
template <int HD>
__device__ __forceinline__ void load_values(const Decode8& p, Codes<HD>& c, size_t row, int g, int t) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int8_t* src = p.a.v_pages + (row + 2 * t + (i & 1) + 8 * (i >> 1)) * HD;
#pragma unroll
    for (int j = 0; j < Codes<HD>::VC; ++j) {
      if constexpr (Codes<HD>::VB == 16) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4*>(src) + g + 8 * j);
        c.v[i][j][0] = x.x; c.v[i][j][1] = x.y; c.v[i][j][2] = x.z; c.v[i][j][3] = x.w;
      } else {
        const uint2 x = __ldcs(reinterpret_cast<const uint2*>(src) + g);
        c.v[i][j][0] = x.x; c.v[i][j][1] = x.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) c.vs[i] = p.a.v_scale[(row + g + 8 * i) / p.a.block];
}

// The queries' parts as operands: for head `h` the four numbers from d on, in the order (d, d + 2), (d + 1, d + 3).
template <typename T, int PARTS>
__device__ __forceinline__ void query_operands(const T* q, bool valid, int d, uint32_t (&b)[PARTS][2]) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = valid ? to_float<T>(q[d + i]) : 0.0f;
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    b[part][0] = two_bf16(x[0], x[2]);
    b[part][1] = two_bf16(x[1], x[3]);
    leave(b[part][0], x[0], x[2]);
    leave(b[part][1], x[1], x[3]);
  }
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(DWARPS * 32, HD * NT * (sizeof(T) / 2) <= 128 ? 2 : 1) decode_8bit_kernel(const Decode8 p) {
  constexpr int PARTS = sizeof(T) == 2 ? 1 : 3;
  constexpr int HEADS = 8 * NT, KSTEPS = HD / 16, MTILES = HD / 16, PITCH = HD + 4;
  using C = Codes<HD>;
  extern __shared__ float merge_o[];                              // [warps][HEADS][PITCH]
  __shared__ float merge_m[DWARPS][HEADS], merge_l[DWARPS][HEADS];
  __shared__ int start_of[4];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = uniform_warp_index();
  const int g = lane >> 2, t = lane & 3;
  if (warp == 0) {                                                // where this block's run begins
    const int total = slices_before(p, p.a.num_seqs, lane) * p.units, run = run_length(p, total, gridDim.x);
    const int from = (int)min((long long)run * blockIdx.x, (long long)total);
    int seq = 0, base = 0;
    while (seq < p.a.num_seqs) {                                  // 32 requests at a time
      const int n = seq + lane < p.a.num_seqs ? slices_of(p, seq + lane).count * p.units : 0;
      int upto = n;
#pragma unroll
      for (int offset = 1; offset < 32; offset <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, offset);
        if (lane >= offset) upto += o;
      }
      const unsigned here = __ballot_sync(0xffffffffu, from < base + upto);
      const int who = here ? __ffs(here) - 1 : 31;
      const int behind = __shfl_sync(0xffffffffu, upto, who), mine = __shfl_sync(0xffffffffu, n, who);
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
    }
  }
  __syncthreads();
  int seq = start_of[0], base = start_of[1], at = start_of[2];
  const int end = start_of[3];
  pdl_wait();

  while (at < end) {
    const Slices s = slices_of(p, seq);
    const int unit = (at - base) / s.count, skip = (at - base) - unit * s.count;
    const int length = min(s.count - skip, end - at);
    const int kvh = unit / p.head_tiles, tile = unit - kvh * p.head_tiles;
    const int heads_here = min(HEADS, p.a.group - tile * HEADS), head0 = kvh * p.a.group + tile * HEADS;
    const int token = p.q_start[seq];
    const int* table = p.a.block_table + (size_t)seq * p.a.max_pages;

    uint32_t q[NT][KSTEPS][PARTS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool valid = 8 * nt + g < heads_here;
      const T* src = static_cast<const T*>(p.a.q) + (size_t)token * p.a.q_stride + (size_t)(head0 + (valid ? 8 * nt + g : 0)) * HD;
#pragma unroll
      for (int kc = 0; kc < KSTEPS; ++kc) query_operands<T, PARTS>(src, valid, 16 * (t + 4 * (kc >> 2)) + 4 * (kc & 3), q[nt][kc]);
    }
    float o[NT][MTILES][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MTILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.0f;
      m[nt][0] = m[nt][1] = NONE;
      l[nt][0] = l[nt][1] = 0.0f;
    }
    const float factor = p.a.scale * (1.4426950408889634f / 127.0f);

    const int first = s.first + skip, last = first + length;
    bool bad = false;
    // the entry at which a slice starts; a page outside the pool reads page 0, unseen
    auto page_of = [&](int slice) {
      const int index = slice * 16 / p.a.page_size;
      return slice < last && index < p.a.max_pages ? table[index] : -1;
    };
    auto row_of = [&](int slice, int page) {
      const bool here = page >= 0 && page < p.a.num_pages;
      return ((size_t)(here ? page : 0) * p.a.kv_heads + kvh) * p.a.page_size + (slice * 16) % p.a.page_size;
    };
    C c;
    int slice = first + warp;
    int page = page_of(slice), page_next = page_of(slice + DWARPS);
    if (slice < last) {
      const size_t row = row_of(slice, page);
      load_keys<HD>(p, c, row, g, t);
      load_values<HD>(p, c, row, g, t);
    }
    for (; slice < last; slice += DWARPS) {
      const int next = slice + DWARPS;
      const size_t row_next = row_of(next, page_next);
      const bool here = page >= 0 && page < p.a.num_pages;
      bad |= !here;
      page = page_next;
      page_next = page_of(next + DWARPS);

      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nt][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < C::KC; ++j) {
        const uint32_t *w0 = reinterpret_cast<const uint32_t*>(&c.k[0][j]), *w1 = reinterpret_cast<const uint32_t*>(&c.k[1][j]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = even_codes(w0[w]), a1 = even_codes(w1[w]), a2 = odd_codes(w0[w]), a3 = odd_codes(w1[w]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
              mma_16x8x16(sc[nt], a0, a1, a2, a3, q[nt][4 * j + w][part][0], q[nt][4 * j + w][part][1]);
        }
      }
      const float f0 = c.ks[0] * factor, f1 = c.ks[1] * factor;
      const float v0 = c.vs[0] * (1.0f / 127.0f), v1 = c.vs[1] * (1.0f / 127.0f);
      if (next < last) load_keys<HD>(p, c, row_next, g, t);

      const int k0 = slice * 16 + g;
      const bool see0 = here && k0 >= s.lo && k0 < s.hi, see1 = here && k0 + 8 >= s.lo && k0 + 8 < s.hi;
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[nt][e] = see0 ? sc[nt][e] * f0 : -INFINITY;
          sc[nt][2 + e] = see1 ? sc[nt][2 + e] * f1 : -INFINITY;
          raise |= fmaxf(sc[nt][e], sc[nt][2 + e]) > m[nt][e] + 8.0f;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float down[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float most = fmaxf(sc[nt][e], sc[nt][2 + e]);
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
            most = fmaxf(most, m[nt][e]);
            down[e] = exp2f(m[nt][e] - most);
            m[nt][e] = most;
            l[nt][e] *= down[e];
          }
#pragma unroll
          for (int i = 0; i < MTILES; ++i) {
            o[nt][i][0] *= down[0]; o[nt][i][1] *= down[1];
            o[nt][i][2] *= down[0]; o[nt][i][3] *= down[1];
          }
        }
      }
      uint32_t pr[NT][PARTS][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float e0 = exp2f(sc[nt][0] - m[nt][0]), e1 = exp2f(sc[nt][1] - m[nt][1]);
        float e2 = exp2f(sc[nt][2] - m[nt][0]), e3 = exp2f(sc[nt][3] - m[nt][1]);
        l[nt][0] += e0 + e2;
        l[nt][1] += e1 + e3;
        // an unseen position's scale may be anything, NaN too
        e0 = see0 ? e0 * v0 : 0.0f; e1 = see0 ? e1 * v0 : 0.0f;
        e2 = see1 ? e2 * v1 : 0.0f; e3 = see1 ? e3 * v1 : 0.0f;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint32_t x = two_bf16(e0, e1), y = two_bf16(e2, e3);
          pr[nt][part][0] = transposed(x);
          pr[nt][part][1] = transposed(y);
          if (part + 1 < PARTS) {
            leave(x, e0, e1);
            leave(y, e2, e3);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < C::VC; ++j)
#pragma unroll
        for (int w = 0; w < C::VB / 4; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // two bytes of a word of positions 2t and 2t + 1, and of 2t + 8 and 2t + 9: rows g and g + 8 of a tile
            const uint32_t x = __byte_perm(c.v[0][j][w], c.v[1][j][w], half ? 0x7632 : 0x5410);
            const uint32_t y = __byte_perm(c.v[2][j][w], c.v[3][j][w], half ? 0x7632 : 0x5410);
            const uint32_t a0 = even_codes(x), a1 = odd_codes(x), a2 = even_codes(y), a3 = odd_codes(y);
            const int i = (j * (C::VB / 4) + w) * 2 + half;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) mma_16x8x16(o[nt][i], a0, a1, a2, a3, pr[nt][part][0], pr[nt][part][1]);
          }
      if (next < last) load_values<HD>(p, c, row_next, g, t);
    }
    if (bad && lane == 0) atomicOr(p.a.status, TGE_STATUS_BAD_PAGE);

    // the warps' states meet in shared memory
    __syncthreads();                                              // whoever still reads the unit before
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int head = 8 * nt + 2 * t + e;
        if (g == 0) {
          merge_m[warp][head] = m[nt][e];
          merge_l[warp][head] = sum;
        }
        float* dst = merge_o + (warp * HEADS + head) * PITCH;
#pragma unroll
        for (int i = 0; i < MTILES; ++i) {
          const int j = i / (C::VB / 2), inner = i - j * (C::VB / 2);
          *reinterpret_cast<float2*>(dst + C::VB * (g + 8 * j) + 2 * inner) = make_float2(o[nt][i][e], o[nt][i][2 + e]);
        }
      }
    }
    __syncthreads();
    const bool whole = length == s.count;
    float* part = p.parts + (size_t)(2 * blockIdx.x + (skip == 0 ? 1 : 0)) * HEADS * (HD + 2);
    for (int i = threadIdx.x; i < heads_here * HD; i += DWARPS * 32) {
      const int head = i / HD, d = i - head * HD;
      float most = NONE;
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) most = fmaxf(most, merge_m[w][head]);
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < DWARPS; ++w) {
        const float f = exp2f(merge_m[w][head] - most);
        sum = fmaf(f, merge_l[w][head], sum);
        acc = fmaf(f, merge_o[(w * HEADS + head) * PITCH + d], acc);
      }
      if (whole) {
        if (p.a.sink != nullptr) {
          const float sink = p.a.sink[head0 + head] * 1.4426950408889634f, top = fmaxf(most, sink), down = exp2f(most - top);
          sum = fmaf(sum, down, exp2f(sink - top));
          acc *= down;
        }
        static_cast<T*>(p.a.out)[(size_t)token * p.a.out_stride + (size_t)(head0 + head) * HD + d] = from_float<T>(sum == 0.0f ? 0.0f : acc / sum);
      } else {
        part[head * (HD + 2) + d] = acc;
        if (d == 0) {
          part[head * (HD + 2) + HD] = most;
          part[head * (HD + 2) + HD + 1] = sum;
        }
      }
    }
    at += length;
    if (at == base + s.count * p.units) {
      base = at;
      ++seq;
    }
  }
}

// Joins the parts of the units that more than one block worked on: one block per unit.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(256) decode_8bit_join_kernel(const Decode8 p, int blocks) {
  constexpr int HEADS = 8 * NT;
  __shared__ int where[3];
  pdl_trigger();
  const int seq = blockIdx.x, unit = blockIdx.y, lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    const int total = slices_before(p, p.a.num_seqs, lane) * p.units, run = run_length(p, total, blocks);
    const int count = slices_of(p, seq).count, from = slices_before(p, seq, lane) * p.units + unit * count;
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
  const int token = p.q_start[seq];
  for (int i = threadIdx.x; i < heads_here * HD; i += blockDim.x) {
    const int head = i / HD, d = i - head * HD;
    // the block in which the unit begins left its part in its second place, the others in their first
    auto state = [&](int b) { return p.parts + ((size_t)(2 * b + (b == first ? 1 : 0)) * HEADS + head) * (HD + 2); };
    float most = p.a.sink != nullptr ? p.a.sink[head0 + head] * 1.4426950408889634f : NONE;
    float sum = p.a.sink != nullptr ? 1.0f : 0.0f, acc = 0.0f;
    for (int b = first; b <= last; ++b) {
      const float* part = state(b);
      const float m = part[HD], top = fmaxf(most, m), down = exp2f(most - top), f = exp2f(m - top);
      sum = fmaf(sum, down, f * part[HD + 1]);
      acc = fmaf(acc, down, f * part[d]);
      most = top;
    }
    static_cast<T*>(p.a.out)[(size_t)token * p.a.out_stride + (size_t)(head0 + head) * HD + d] = from_float<T>(sum == 0.0f ? 0.0f : acc / sum);
  }
}

template <typename T, int HD, int NT>
int launch_decode(Decode8 p, int blocks, cudaStream_t stream) {
  constexpr int smem = DWARPS * 8 * NT * (HD + 4) * 4;
  static bool ready[64] = {};                                     // shared memory beyond 48 KB is asked for once per device
  int device = 0;
  cudaGetDevice(&device);
  if (smem > 48 * 1024 && (device >= 64 || !ready[device])) {
    const cudaError_t rc = cudaFuncSetAttribute(decode_8bit_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    TGE_REQUIRE(rc == cudaSuccess, "attention_8bit: %d bytes of shared memory: %s", smem, cudaGetErrorString(rc));
    if (device < 64) ready[device] = true;
  }
  tge_launch(decode_8bit_kernel<T, HD, NT>, blocks, DWARPS * 32, smem, stream, p);
  tge_launch(decode_8bit_join_kernel<T, HD, NT>, dim3(p.a.num_seqs, p.units), 256, 0, stream, p, blocks);
  return tge_launched("attention_8bit", 2);
}

// Blocks of a launch: all that are on the device at a time, so that all runs advance together.
int decode_blocks(int head_dim, int tile_heads, bool is_bf16) { return tge_sm_count() * (head_dim * (tile_heads / 8) * (is_bf16 ? 1 : 2) <= 128 ? 2 : 1); }

}  // namespace

// Heads of a tile: a group of up to 8 heads makes one tile of 8, more go by 16 (one pass over the codes for twice the accumulators, which
// heads of 256 numbers have no registers for).
static int decode_tile(int group, int head_dim) { return group <= 8 || head_dim > 128 ? 8 : 16; }

// float32 scratch numbers of tge_attention_8bit_decode; -1: sizes that it does not take.
TGE_API long long tge_attention_8bit_decode_floats(int is_bf16, int num_seqs, int heads, int kv_heads, int head_dim, int page_size, int max_pages) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || page_size % 16 != 0 || kv_heads <= 0 || heads % kv_heads != 0) return -1;
  const int tile = decode_tile(heads / kv_heads, head_dim);
  const long long units = (long long)kv_heads * ((heads / kv_heads + tile - 1) / tile);
  // places in the row of all slices are counted in 32 bits, units along a grid's second axis
  if (units > 65535 || (long long)max_pages * page_size > (1ll << 30) ||
      units * num_seqs * ((long long)max_pages * page_size / 16 + 1) > (1ll << 30)) return -1;
  return 2ll * decode_blocks(head_dim, tile, is_bf16 != 0) * tile * (head_dim + 2);
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
  if (num_seqs == 0) return 0;
  const int group = heads / kv_heads, tile = decode_tile(group, head_dim);
  Decode8 p;
  p.a = Attn8{q, out, q_stride, out_stride, (const int8_t*)k_pages, (const int8_t*)v_pages, k_scale, v_scale, block_table, nullptr, nullptr, sink,
              max_pages, num_pages, page_size, block, num_seqs, heads, kv_heads, group, head_dim, window, scale, status};
  p.q_start = q_start;
  p.start_pos = start_pos;
  p.head_tiles = (group + tile - 1) / tile;
  p.units = kv_heads * p.head_tiles;
  p.least = DWARPS;
  p.parts = parts;
  const int blocks = decode_blocks(head_dim, tile, is_bf16 != 0);
  auto run = [&](auto type) {
    using T = decltype(type);
    if (head_dim == 256) return launch_decode<T, 256, 1>(p, blocks, stream);
    if (head_dim == 128) return tile == 8 ? launch_decode<T, 128, 1>(p, blocks, stream) : launch_decode<T, 128, 2>(p, blocks, stream);
    return tile == 8 ? launch_decode<T, 64, 1>(p, blocks, stream) : launch_decode<T, 64, 2>(p, blocks, stream);
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
