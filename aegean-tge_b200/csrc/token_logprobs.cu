// Log probabilities of given tokens, with the entropy of their rows, their ranks and the best alternatives.
//
// Per row x of `vocab` logits, m = max x, Z = sum exp(x - m):
//   logprob = x_t - m - ln Z,  entropy = ln Z - sum exp(x - m) (x - m) / Z,  rank = how many tokens come before t,
//   and the `top` first tokens with their log probabilities, in the order of falling logits, the lower index first among equals.
// -inf is a token that cannot come: it adds nothing to either sum.  A row with NaN, with +inf or without a finite logit has no
// distribution: its log probabilities and its entropy are NaN (ranks and the order of the tokens still follow the logits, NaN last).
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MOST_TOP = 32;
constexpr int MINE = 16;                        // logits of a thread and round
constexpr int ROUND = THREADS * MINE;
constexpr int ROOM = 8 * THREADS + MOST_TOP;    // keys in the list of candidates: what one load of all threads may add to a full choice
constexpr int MOST_SPLITS = 128, MOST_CLUSTER = 16;
constexpr float LEAST = -3.402823466e38f;       // where a thread's reference starts: finite, so that -inf less it is -inf
constexpr float LOG2E = 1.4426950408889634f;

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

__device__ __forceinline__ unsigned long long warp_largest(unsigned long long v, int width = 32) {
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, offset);
    if (offset < width) v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ unsigned long long block_largest(unsigned long long v, unsigned long long* scratch) {
  v = warp_largest(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_largest((threadIdx.x & 31) < THREADS / 32 ? scratch[threadIdx.x & 31] : 0ull);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Sums over some of a row's logits: z = sum exp(x - m), w = sum exp(x - m) (x - m), relative to a reference m that no logit passes by more
// than 16; how many of them come before the given token.
struct Sums {
  float m, z, w;
  int before;
  // the same relative to `to`
  __device__ __forceinline__ void move(float to) {
    const float f = exp2_fast((m - to) * LOG2E);
    w = z > 0.0f && f > 0.0f ? f * fmaf(z, m - to, w) : 0.0f;      // (0 times a distance that may be infinite)
    z = z > 0.0f ? f * z : z;                          // NaN stays
    if (!(z == z)) w = z;
    m = to;
  }
};

// The sums of a block's threads, in every thread.
__device__ __forceinline__ Sums block_sums(Sums mine, float* scratch, int* counts) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = warp_max(mine.m);
  __syncthreads();
  if (lane == 0) scratch[warp] = top;
  __syncthreads();
  top = warp_max(lane < THREADS / 32 ? scratch[lane] : LEAST);
  mine.move(top);
  mine.before = __reduce_add_sync(0xffffffffu, mine.before);
  if (lane == 0) counts[warp] = mine.before;
  mine.z = block_sum(mine.z, scratch);
  mine.w = block_sum(mine.w, scratch);
  mine.before = __reduce_add_sync(0xffffffffu, lane < THREADS / 32 ? counts[lane] : 0);
  return mine;
}

constexpr int GROUPS = THREADS / 4;             // groups of four lanes
static_assert(GROUPS == 64, "two groups to a lane");

// A bar that at least `top` keys pass (are above) and not many more: just below the top-th largest of the groups' largest keys, if so many
// groups have one, else 0.  `key`: the thread's largest (0: none).  scratch: 64 keys and one for the result.
__device__ __forceinline__ unsigned long long bar_of(unsigned long long key, int top, unsigned long long* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  key = warp_largest(key, 4);
  __syncthreads();
  if ((lane & 3) == 0) scratch[threadIdx.x >> 2] = key;
  if (threadIdx.x == 0) scratch[64] = 0ull;
  __syncthreads();
  const unsigned long long a = scratch[lane], b = scratch[lane + 32];
#pragma unroll
  for (int i = 0; i < GROUPS * 32 / THREADS; ++i) {
    const unsigned long long mine = scratch[warp * (GROUPS * 32 / THREADS) + i];
    const int in_front = __popc(__ballot_sync(0xffffffffu, a > mine)) + __popc(__ballot_sync(0xffffffffu, b > mine));
    if (lane == 0 && mine != 0ull && in_front == top - 1) scratch[64] = mine - 1;
  }
  __syncthreads();
  return scratch[64];
}

// The `top` largest of the `count` keys at `list`, sorted, to its start; the smallest of them (0 if there are fewer).  Few keys find their
// places by counting those in front of them; of many, those above a bar come to the start first.  MOST: a bound of `count`.
template <int MOST>
__device__ __forceinline__ unsigned long long choose(unsigned long long* list, int count, int top, unsigned long long* scratch, int* counter) {
  constexpr int EACH = (MOST + THREADS - 1) / THREADS;
  __syncthreads();
  if (count > 64) {
    unsigned long long mine[EACH], largest = 0ull;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = threadIdx.x + i * THREADS;
      mine[i] = at < count ? list[at] : 0ull;
      largest = max(largest, mine[i]);
    }
    const unsigned long long bar = bar_of(largest, top, scratch);
    if (threadIdx.x == 0) *counter = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (mine[i] > bar) list[atomicAdd(counter, 1)] = mine[i];
    __syncthreads();
    count = *counter;
  }
  if (count <= THREADS) {
    const unsigned long long mine = (int)threadIdx.x < count ? list[threadIdx.x] : 0ull;
    int ahead = 0;
    if ((int)(threadIdx.x & ~31) < count)
      for (int i = 0; i < count; ++i) ahead += list[i] > mine ? 1 : 0;
    __syncthreads();
    if ((int)threadIdx.x < count && ahead < top) list[ahead] = mine;
  } else {                                       // keys that rise with their place, say: one after the other
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
      unsigned long long next = 0;
      for (int i = threadIdx.x; i < count; i += THREADS) next = list[i] < last ? max(next, list[i]) : next;
      last = block_largest(next, scratch);
      if (threadIdx.x == 0) scratch[32 + k] = last;
    }
    __syncthreads();
    if ((int)threadIdx.x < top) list[threadIdx.x] = scratch[32 + threadIdx.x];
  }
  __syncthreads();
  return count >= top ? list[top - 1] : 0ull;
}

struct LogprobParams {
  const void* logits;
  const int* tokens;
  long long stride;
  int rows, vocab, top, splits, chunk;          // a row goes in `splits` chunks of `chunk` logits, one block each
  float *logprob, *entropy, *top_logprobs;
  int *rank, *top_ids;
  float* sums;                                  // [rows, splits, 4]
  unsigned long long* keys;                     // [rows, splits, top]
  int* status;
};

// What a row's answers are, once its sums and its first keys are known.
__device__ __forceinline__ void answer(const LogprobParams& p, int r, const Sums& all, float own, bool known, const unsigned long long* keys) {
  const float nan = __int_as_float(0x7fc00000);
  const bool broken = !(all.z > 0.0f);                                // NaN, or nothing but -inf
  const float log_z = logf(all.z);
  if (threadIdx.x == 0) {
    p.logprob[r] = broken || !known ? nan : own - all.m - log_z;
    p.entropy[r] = broken ? nan : log_z - all.w / all.z;
    p.rank[r] = known ? all.before : -1;
  }
  if ((int)threadIdx.x < p.top) {
    const unsigned long long key = keys[threadIdx.x];
    p.top_ids[(size_t)r * p.top + threadIdx.x] = (int)~(uint32_t)key;
    p.top_logprobs[(size_t)r * p.top + threadIdx.x] = broken ? nan : logit_of(key) - all.m - log_z;
  }
}

// The chunks of a row, SPLITS of them at most, joined by a block: their sums in order, and the best of their best (`list`: room for all of them).
template <int SPLITS>
__device__ void join_chunks(const LogprobParams& p, int r, float own, bool known, unsigned long long* list, unsigned long long* scratch, int* listed,
                            int* counter) {
  constexpr int PER_LANE = (SPLITS + 31) / 32;
  const int lane = threadIdx.x & 31;
  __syncthreads();                               // whoever still reads the block's own list
  if (threadIdx.x == 0) *listed = 0;
  // every warp for itself, splits lane by lane
  Sums part[PER_LANE], all{LEAST, 0.0f, 0.0f, 0};
  unsigned long long least = 0;
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    const int split = lane + 32 * i;
    part[i] = Sums{LEAST, 0.0f, 0.0f, 0};
    if (split < p.splits) {
      const float4 s = *reinterpret_cast<const float4*>(p.sums + 4 * ((size_t)r * p.splits + split));
      part[i] = Sums{s.x, s.y, s.z, __float_as_int(s.w)};
      // no key below the last of a chunk's best is among the row's
      if (p.top > 0) least = max(least, p.keys[((size_t)r * p.splits + split) * p.top + p.top - 1]);
    }
    all.m = fmaxf(all.m, part[i].m);
  }
  all.m = warp_max(all.m);
  least = warp_largest(least);
#pragma unroll
  for (int i = 0; i < PER_LANE; ++i) {
    part[i].move(all.m);
    all.z += part[i].z;
    all.w += part[i].w;
    all.before += part[i].before;
  }
  all.z = warp_sum(all.z);
  all.w = warp_sum(all.w);
  all.before = __reduce_add_sync(0xffffffffu, all.before);
  __syncthreads();
  for (int i = threadIdx.x; i < p.splits * p.top; i += THREADS) {
    const unsigned long long key = p.keys[(size_t)r * p.splits * p.top + i];
    if (key != 0 && key >= least) list[atomicAdd(listed, 1)] = key;
  }
  __syncthreads();
  if (p.top > 0) choose<SPLITS * MOST_TOP>(list, *listed, p.top, scratch, counter);
  answer(p, r, all, own, known, list);
}

// Sixteen logits of a thread in loads of 16 bytes, `per` of them each: load k holds those from first + (k THREADS + thread) per on.
// What lies behind the chunk is -inf (and told apart by its index where that matters).
template <typename T, bool VECTOR>
__device__ __forceinline__ void take(const T* x, int first, int end, float (&v)[MINE]) {
  constexpr int per = 16 / sizeof(T);
#pragma unroll
  for (int k = 0; k < MINE / per; ++k) {
    const int at = first + (k * THREADS + threadIdx.x) * per;
    if (VECTOR && at + per <= end) {
      uint32_t raw[4];
      asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(raw[0]), "=r"(raw[1]), "=r"(raw[2]), "=r"(raw[3]) : "l"(x + at));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (per == 4) {
          v[4 * k + i] = __uint_as_float(raw[i]);
        } else {
          v[8 * k + 2 * i] = __uint_as_float(raw[i] << 16);
          v[8 * k + 2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < per; ++i) v[per * k + i] = at + i < end ? to_float<T>(x[at + i]) : -INFINITY;
    }
  }
}

// One pass over a chunk of a row: a thread holds its next sixteen logits on their way while it works on these, keeps sums of its own, and looks
// at single logits only where its largest reaches the smallest of the best so far.  Those that do are listed with the block's others; the list
// is cut to the best now and then.  After the first round the best are a choice among the largest of 64 groups of four lanes and whatever
// passes the n-th of those, then whatever passes the n-th of the chunk's first 1, 2, 4, 8, ... rounds: of random rows some hundred logits are
// ever listed.  A row that lists more than there is room for (rising logits) is looked through again.
//
// 1,024 rows of 152,064 float32 logits with the 20 best: 118 us, 5.3 TB/s or 0.81 of a copy's rate (without alternatives 105); 70 % of the issue
// slots are taken, some 20 instructions a logit.  In bfloat16 152 us, for the same number of instructions and the conversions.  One row
// with 5 alternatives 9.0 us: the trips of three rounds and of the joining.  Not taken: cuts after rounds 1, 4, 16, ... only (127 us); a bar that
// stays where the first round put it, with a barrier every round (365).
template <typename T, bool VECTOR, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, 4) token_logprobs_kernel(const LogprobParams p) {
  constexpr int per = 16 / sizeof(T);
  __shared__ unsigned long long list[ROOM], scratch[65];
  __shared__ float floats[32];
  __shared__ int counts[32], listed, counter;
  pdl_trigger();
  const int r = blockIdx.x / p.splits, split = blockIdx.x - r * p.splits, lane = threadIdx.x & 31;
  const int begin = split * p.chunk, end = min(begin + p.chunk, p.vocab);
  if (threadIdx.x == 0) listed = 0;
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + (size_t)r * p.stride;
  float v[MINE], ahead[MINE];
  take<T, VECTOR>(x, begin, end, v);
  const int token = p.tokens[r];
  const bool known = token >= 0 && token < p.vocab;
  if (!known && split == 0 && threadIdx.x == 0) atomicOr(p.status, TGE_STATUS_BAD_TOKEN);
  const float own = known ? to_float<T>(x[token]) : 0.0f;
  // before the token come logits that are larger and, with a lower index, equal ones: those of at least `own` in front of it and
  // of at least the next float behind it
  const uint32_t bits = __float_as_uint(own + 0.0f);
  const float above = own != own ? own : __uint_as_float(bits & 0x80000000u ? bits - 1 : bits + 1);
  const bool token_is_nan = own != own;
  // the round that looks at indices: the token's; in a cluster, whose chunks end inside a round, the chunk's last one if the token lies behind
  // it (what take() puts behind a chunk is -inf, and so may the token be)
  const int near = CLUSTER ? min(token, end - 1) : token;
  Sums mine{LEAST, 0.0f, 0.0f, 0};
  unsigned long long least = 0;                  // the smallest of the best so far (0: not as many yet)
  __syncthreads();

  auto index_of = [&](int first, int i) { return first + ((i / per) * THREADS + (int)threadIdx.x) * per + i % per; };
  // Cuts the list to the best of the chunk up to `upto`.
  auto settle = [&](int upto) {
    __syncthreads();
    const int count = listed;
    if (count <= ROOM) {
      least = max(least, choose<ROOM>(list, count, p.top, scratch, &counter));
      if (threadIdx.x == 0) listed = min(count, p.top);
      __syncthreads();
      return;
    }
    // More than there is room for: all of the chunk up to here again, a load of every thread at a time.
    __syncthreads();
    if (threadIdx.x == 0) listed = 0;
    least = 0;
    __syncthreads();
    for (int from = begin; from < upto; from += THREADS * per) {
      for (int i = 0; i < per; ++i) {
        const int index = from + (int)threadIdx.x * per + i;
        const unsigned long long key = index < upto ? key_of(to_float<T>(x[index]), index) : 0ull;
        if (key > least) list[atomicAdd(&listed, 1)] = key;
      }
      __syncthreads();
      const int so_far = listed;
      least = max(least, choose<ROOM>(list, so_far, p.top, scratch, &counter));
      if (threadIdx.x == 0) listed = min(so_far, p.top);
      __syncthreads();
    }
  };

  float bar = __int_as_float(0x7fc00000);        // the logit of `least`; NaN where anything may enter
  for (int first = begin, round = 1; first < end; first += ROUND, ++round) {
    if (first + ROUND < end) take<T, VECTOR>(x, first + ROUND, end, ahead);
    float quad[MINE / 4];                        // the largest of four
#pragma unroll
    for (int k = 0; k < MINE / 4; ++k) quad[k] = fmaxf(fmaxf(v[4 * k], v[4 * k + 1]), fmaxf(v[4 * k + 2], v[4 * k + 3]));
    const float largest = fmaxf(fmaxf(quad[0], quad[1]), fmaxf(quad[2], quad[3]));
    if (largest > mine.m + 16.0f) mine.move(largest);
    float z = 0.0f, w = 0.0f;
    if (fabsf(mine.m) < 64.0f) {                // m log2 e rounded once, 4e-6 off at most; w in units of ln 2
      const float less = -mine.m * LOG2E;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const float d = fmaf(v[i], LOG2E, less), e = exp2_fast(d);
        z += e;
        w = fmaf(e, fmaxf(d, -200.0f), w);      // -inf has no weight (and NaN shows in z)
      }
      mine.w = fmaf(w, 0.6931471805599453f, mine.w);
    } else {
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const float d = v[i] - mine.m, e = exp2_fast(d * LOG2E);
        z += e;
        w = fmaf(e, fmaxf(d, -200.0f), w);
      }
      mine.w += w;
    }
    mine.z += z;
    if (!token_is_nan && (near < first || near >= first + ROUND)) {
      const float from = first < token ? own : above;
#pragma unroll
      for (int i = 0; i < MINE; ++i) mine.before += v[i] >= from ? 1 : 0;
    } else {
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int index = index_of(first, i);
        const bool ahead_of = token_is_nan ? v[i] == v[i] || index < token : v[i] >= (index < token ? own : above);
        mine.before += index < end && ahead_of ? 1 : 0;
      }
    }

    if (p.top > 0) {
      if (round == 1) {                          // the first of a thread's largest logits, of all that it has
        int at = -1;
#pragma unroll
        for (int i = MINE - 1; i >= 0; --i) at = v[i] == largest ? i : at;
        const int index = index_of(first, max(at, 0));
        least = bar_of(at >= 0 && index < end ? key_of(largest, index) : 0ull, p.top, scratch);
        bar = logit_of(least);
      }
      if (__any_sync(0xffffffffu, !(largest < bar))) {
#pragma unroll
        for (int k = 0; k < MINE / 4; ++k)
          if (__any_sync(0xffffffffu, !(quad[k] < bar))) {
#pragma unroll
            for (int i = 4 * k; i < 4 * k + 4; ++i)
              if (!(v[i] < bar)) {
                const int index = index_of(first, i);
                const unsigned long long key = key_of(v[i], index);
                if (index < end && key > least) {
                  const int at = atomicAdd(&listed, 1);
                  if (at < ROOM) list[at] = key;
                }
              }
          }
      }
      if ((round & (round - 1)) == 0) {          // after rounds 1, 2, 4, 8, ...: the bar rises as the best get rarer
        settle(min(first + ROUND, end));
        bar = logit_of(least);
      }
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i) v[i] = ahead[i];
  }
  if (p.top > 0) settle(end);
  const int found = p.top > 0 ? min(listed, p.top) : 0;
  mine = block_sums(mine, floats, counts);
  if (!CLUSTER && p.splits == 1) {
    answer(p, r, mine, own, known, list);
    return;
  }
  const size_t place = (size_t)r * p.splits + split;
  if (threadIdx.x == 0) *reinterpret_cast<float4*>(p.sums + 4 * place) = make_float4(mine.m, mine.z, mine.w, __int_as_float(mine.before));
  if ((int)threadIdx.x < p.top) p.keys[place * p.top + threadIdx.x] = (int)threadIdx.x < found ? list[threadIdx.x] : 0ull;
  if constexpr (CLUSTER) {                       // a row's blocks are a cluster: its first one joins them
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
    if (split == 0) join_chunks<MOST_CLUSTER>(p, r, own, known, list, scratch, &listed, &counter);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) token_logprobs_join_kernel(const LogprobParams p) {
  __shared__ unsigned long long list[MOST_SPLITS * MOST_TOP], scratch[65];
  __shared__ int listed, counter;
  pdl_trigger();
  pdl_wait();
  const int token = p.tokens[blockIdx.x];
  const bool known = token >= 0 && token < p.vocab;
  const float own = known ? to_float<T>(static_cast<const T*>(p.logits)[(size_t)blockIdx.x * p.stride + token]) : 0.0f;
  join_chunks<MOST_SPLITS>(p, blockIdx.x, own, known, list, scratch, &listed, &counter);
}

// How rows are cut into chunks of one block each.  A block costs its rounds and about two more (the first choice, the joining), and as many run at a
// time as the device holds; a second kernel costs about three.  Few rows go in clusters of 8 or 16 blocks (16 of these clusters are on the
// device at a time), which need none.  Of all cuts the one that is done first, the fewest chunks among equals.  Rows of 152,064 with 20
// alternatives, us with clusters / a second kernel: one 12.5 / 12.5 (from the host, with 5, 22 / 24), 8 14.5 / 16.6, 64 24.8 / 26.8; with 32 one
// 16.5 / 12.6 and 64 31 / 33.
struct Cut { int splits, chunk, cluster; };
Cut cut_of(int rows, int vocab) {
  const int rounds = (vocab + ROUND - 1) / ROUND;
  const long long at_once = 4ll * tge_sm_count();
  long long best = (rows + at_once - 1) / at_once * (rounds + 2);
  Cut cut{1, vocab, 0};
  for (int splits = 2; splits <= rounds && splits <= MOST_SPLITS; ++splits) {
    const int mine = (rounds + splits - 1) / splits;
    const long long cost = ((long long)rows * splits + at_once - 1) / at_once * (mine + 2) + 3;
    if (cost < best) {
      best = cost;
      cut = Cut{(vocab + mine * ROUND - 1) / (mine * ROUND), mine * ROUND, 0};
    }
  }
  for (int blocks = 8; blocks <= MOST_CLUSTER; blocks += 8) {
    const int chunk = ((vocab + blocks - 1) / blocks + 63) / 64 * 64;
    const long long cost = (chunk + ROUND - 1) / ROUND + 2;
    if ((long long)chunk * (blocks - 1) < vocab && rows <= (blocks == 8 ? at_once / 8 : 16) && cost < best) {
      best = cost;
      cut = Cut{blocks, chunk, blocks};
    }
  }
  return cut;
}

template <typename T, bool VECTOR>
int in_clusters(const LogprobParams& p, int blocks, cudaStream_t stream) {
  static bool ready[64] = {};                    // clusters of 16: asked for once per device
  int device = 0;
  cudaGetDevice(&device);
  if (device >= 64 || !ready[device]) {
    const cudaError_t rc = cudaFuncSetAttribute(token_logprobs_kernel<T, VECTOR, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    TGE_REQUIRE(rc == cudaSuccess, "token_logprobs: clusters of 16: %s", cudaGetErrorString(rc));
    if (device < 64) ready[device] = true;
  }
  tge_launch_clusters(token_logprobs_kernel<T, VECTOR, true>, dim3(p.rows * p.splits), THREADS, 0, blocks, stream, p);
  return tge_launched("token_logprobs", 1);
}

}  // namespace

// float32 scratch numbers of tge_token_logprobs (16-byte aligned).
TGE_API long long tge_token_logprobs_floats(int rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0) return 0;
  const int splits = cut_of(rows, vocab).splits;
  return splits == 1 ? 0 : (long long)rows * splits * (4 + 2 * top);
}

TGE_API int tge_token_logprobs(const void* logits, int is_bf16, long long stride, const int* tokens, int rows, int vocab, int top,
                               float* logprob, float* entropy, int* rank, int* top_ids, float* top_logprobs, float* scratch,
                               long long scratch_floats, int* status, cudaStream_t stream) {
  TGE_REQUIRE(rows >= 0 && vocab > 0 && vocab < 0x7fff0000 && stride >= vocab, "token_logprobs: bad sizes rows=%d vocab=%d stride=%lld", rows, vocab, stride);
  TGE_REQUIRE(top >= 0 && top <= MOST_TOP && top <= vocab, "token_logprobs: %d alternatives of %d tokens, at most %d", top, vocab, MOST_TOP);
  if (rows == 0) return 0;
  const Cut cut = cut_of(rows, vocab);
  LogprobParams p{logits, tokens, stride, rows, vocab, top, cut.splits, cut.chunk, logprob, entropy, top_logprobs,
                  rank, top_ids, scratch, nullptr, status};
  TGE_REQUIRE((long long)rows * p.splits < 0x7fffffffll, "token_logprobs: %d rows of %d logits", rows, vocab);
  TGE_REQUIRE(scratch_floats >= tge_token_logprobs_floats(rows, vocab, top), "token_logprobs: %lld floats of scratch memory", scratch_floats);
  p.keys = reinterpret_cast<unsigned long long*>(scratch + 4 * (size_t)rows * p.splits);
  const int element = is_bf16 ? 2 : 4;
  const bool vector = (uintptr_t)logits % 16 == 0 && stride * element % 16 == 0;
  auto run = [&](auto type) {
    using T = decltype(type);
    if (cut.cluster > 0) return vector ? in_clusters<T, true>(p, cut.cluster, stream) : in_clusters<T, false>(p, cut.cluster, stream);
    if (vector) tge_launch(token_logprobs_kernel<T, true, false>, rows * p.splits, THREADS, 0, stream, p);
    else tge_launch(token_logprobs_kernel<T, false, false>, rows * p.splits, THREADS, 0, stream, p);
    if (p.splits == 1) return tge_launched("token_logprobs", 1);
    tge_launch(token_logprobs_join_kernel<T>, rows, THREADS, 0, stream, p);
    return tge_launched("token_logprobs", 2);
  };
  return is_bf16 ? run(__nv_bfloat16()) : run(float());
}
