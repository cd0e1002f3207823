// Losses over the log probabilities of packed sequences, and their gradients: the clipped policy loss and the loss of pairs.
//
// Sequence s has the tokens [offsets[s], offsets[s + 1]); an id below zero marks a token that does not count.  Both are HBM-bound: a token
// reads its log probabilities, its id and what else is given once and writes a gradient, 20 to 36 bytes in all.  What stands against one pass
// is that a gradient hangs on how many tokens count, or on its sequence's sum: the first pass over the ids leaves a bit for each token, so
// that the second one reads an eighth of a byte in their place.
//   few tokens (kFew): everything by one CTA in one launch;
//   else a pass over the ids (policy) or over all (pairs), one over the sequences, one over the tokens.
// 600 tokens take 3.0 us (a launch), 131072 of 256 sequences 10.7, 8.4 M with 64-bit ids 48.9 (their 235 MB at a copy's rate 35.7): 12 for the ids, 33 for the
// tokens, with half of the warps that an SM could hold (64 registers, most of them loads on their way) and neither memory nor the issue slots full.  Pairs: 1500 tokens 3.9 us, 400001 10.7, 4.2 M of 128 sequences 21.7 (7.7): 9 to 10 each for sums and gradient.
// Every sum is taken in a fixed order, over a CTA's tokens in fp32 and beyond that, as of the sums over a sequence, in 64 bits.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr uint32_t kTile = 2048;                           // tokens of a CTA in the passes that count and sum
constexpr uint32_t kWords = kTile / 32;
constexpr int kThreads = 256, kEach = kTile / kThreads;   // (with 16 tokens to a thread the loads in flight took the registers of all but two CTAs)
constexpr uint32_t kPass = 2048;                           // tokens of a CTA in the pass that writes gradients
// What one CTA does alone: the policy loss of up to 4096 tokens (20 sequences: 7.7 us for 8.7 of three kernels; 6000 tokens 10.2 for 8.7), pairs up to 6144 (6.6 for
// 7.5; 8000 tokens 7.9 for 7.7), of up to 2048 sequences.
constexpr uint32_t kFewPolicy = 4096, kFew = 6144, kFewSequences = 2048;
constexpr int kFewThreads = 1024, kFewEach = kFew / kFewThreads;
constexpr uint32_t kShort = 24;                            // tokens of a sequence that a lane sums by itself

// ---- sequences

// An id, loaded where the call stands: left to itself the compiler moves loads down to the votes that need them, one round trip after another.
__device__ __forceinline__ float ld_id(const float* p) { return ld_stream(p); }
__device__ __forceinline__ int32_t ld_id(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.cs.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int64_t ld_id(const int64_t* p) {
  int64_t v;
  asm volatile("ld.global.cs.s64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}

template <class Id>
struct Packed {
  const Id *ids, *offsets;
  uint64_t tokens;
  uint32_t sequences;
  // An offset as it is used: none leads outside the tokens, whatever the memory holds.
  __device__ __forceinline__ uint64_t offset(uint32_t s) const {
    const Id v = offsets[s];
    if (!(v > Id(0))) return 0;
    if constexpr (std::is_floating_point<Id>::value) return v >= (float)tokens ? tokens : (uint64_t)v;   // (exact: tokens up to 2^24)
    else return min((uint64_t)v, tokens);
  }
};

// The last sequence that begins at or before token t, found by a whole warp: 32 of what is left are looked at together.
template <class Id>
__device__ __forceinline__ uint32_t sequence_of(const Packed<Id>& p, uint64_t t) {
  uint32_t lo = 0, end = p.sequences;
  while (end - lo > 1) {
    const uint32_t step = (end - lo + 32) / 33, at = lo + ((threadIdx.x & 31) + 1) * step;
    const uint32_t before = __popc(__ballot_sync(0xffffffffu, at < end && p.offset(at) <= t));
    lo += before * step;
    end = min(end, lo + step);
  }
  return lo;
}

// A sequence, and where it ends, that the warp has found before.
struct Found {
  uint32_t s;
  uint64_t end = 0;
};
// The sequences of the warp's 128 tokens from `base` on, four neighbours to each lane.  `before`: of tokens before them; long sequences are looked for once.
// `owner`: the first one where it is known (see note_owner), else kNone.
constexpr uint32_t kNone = 0xffffffffu, kBlock = 128;
template <class Id>
__device__ __forceinline__ void sequences_of(const Packed<Id>& p, uint64_t base, uint32_t owner, uint32_t (&of)[4], Found& before) {
  if (base + 128 <= before.end) {
#pragma unroll
    for (int k = 0; k < 4; ++k) of[k] = before.s;
    return;
  }
  const uint32_t lane = threadIdx.x & 31, first = owner == kNone ? sequence_of(p, base) : owner;
  const uint64_t none = ~0ull, next = first + 1 + lane < p.sequences ? p.offset(first + 1 + lane) : none;
  const uint32_t begins = __popc(__ballot_sync(0xffffffffu, next < base + 128));
  const uint64_t mine = base + 4 * lane;
  before.s = first;
  before.end = __shfl_sync(0xffffffffu, next, 0);
#pragma unroll
  for (int k = 0; k < 4; ++k) of[k] = first;
  if (begins < 32) {                                       // the 32 next beginnings reach over the 128 tokens
    for (uint32_t i = 0; i < begins; ++i) {
      const uint64_t b = __shfl_sync(0xffffffffu, next, i);
#pragma unroll
      for (int k = 0; k < 4; ++k) of[k] += b <= mine + k;
    }
    return;
  }
  uint32_t lo = first;
#pragma unroll
  for (int k = 0; k < 4; ++k) {                            // sequences of a few tokens, or many empty ones: each lane for itself, in growing steps from where it is
    uint32_t step = 1;
    while (step < p.sequences - lo && p.offset(lo + step) <= mine + k) lo += step, step *= 2;
    uint32_t end = min(step, p.sequences - lo) + lo;
    while (end - lo > 1) {
      const uint32_t middle = lo + (end - lo) / 2;
      if (p.offset(middle) <= mine + k) lo = middle;
      else end = middle;
    }
    of[k] = lo;
  }
}

// What the passes leave for one another.
struct Shared {
  uint32_t ticket;                                         // CTAs that have finished
  uint32_t live;                                           // sequences with a token that counts
  float share;                                             // 1 / the tokens that count
};
struct Workspace {
  Shared* shared;
  uint32_t* counts;                                        // of each tile
  uint32_t* bits;                                          // which tokens count
  uint32_t* owner;                                         // of each kBlock tokens: the sequence of the first one
  float* share;                                            // of each sequence: 1 / its tokens that count (0: there is none); or its gradient
  float4* partial;                                         // of each CTA of the pass over the tokens
  double *whole, *head, *tail;                             // sums: of sequences inside a tile; of a tile's part of one that began before, or goes on
};
uint64_t up(uint64_t n) { return (n + 255) & ~255ull; }
uint64_t tiles_of(uint64_t tokens) { return tokens ? (tokens + kTile - 1) / kTile : 1; }   // (the first one clears the ticket)
Workspace lay_out(void* base, uint64_t tokens, uint64_t sequences, bool pairs, uint64_t* bytes) {
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    char* p = static_cast<char*>(base) + at;
    at += up(n);
    return p;
  };
  const uint64_t tiles = tiles_of(tokens);
  Workspace w = {};
  w.shared = reinterpret_cast<Shared*>(take(sizeof(Shared)));
  w.counts = reinterpret_cast<uint32_t*>(take(tiles * 4));
  w.bits = reinterpret_cast<uint32_t*>(take(tiles * kWords * 4));
  w.owner = reinterpret_cast<uint32_t*>(take(tiles * (kTile / kBlock) * 4));
  w.share = reinterpret_cast<float*>(take(sequences * 4));
  if (pairs) {
    w.partial = reinterpret_cast<float4*>(take((sequences + kThreads / 32 - 1) / (kThreads / 32) * sizeof(float4)));
    w.whole = reinterpret_cast<double*>(take(sequences * 8));
    w.head = reinterpret_cast<double*>(take(tiles * 8));
    w.tail = reinterpret_cast<double*>(take(tiles * 8));
  } else {
    w.partial = reinterpret_cast<float4*>(take((tokens + kThreads * 4 - 1) / (kThreads * 4) * sizeof(float4)));
  }
  *bytes = at;
  return w;
}

// A warp that looks at sequence s = [from, to) leaves it at the blocks that begin in it, which then need no search (two round trips to memory: 131072 tokens
// of 256 sequences 10.5 -> 10.3 us, 400001 in pairs 10.9 -> 10.7).
__device__ __forceinline__ void note_owner(const Workspace& w, uint32_t s, uint64_t from, uint64_t to) {
  for (uint64_t b = (from + kBlock - 1) / kBlock + (threadIdx.x & 31); b * kBlock < to; b += 32) w.owner[b] = s;
}
// The block's, as it is used: whatever the memory holds, one of the sequences.
template <class Id>
__device__ __forceinline__ uint32_t owner_of(const Packed<Id>& p, const Workspace& w, uint64_t base, uint64_t begin) {
  const uint32_t s = w.owner[base / kBlock];
  return base < begin ? 0 : min(s, p.sequences - 1);
}

using polar_b200::warp_sum;
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
// The sums of four values over the CTA, in its first warp.
template <int THREADS, class T>
__device__ __forceinline__ void sums4(T (&v)[4], T* slots) {
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = warp_sum(v[i]);
    if (lane == 0) slots[warp * 4 + i] = v[i];
  }
  __syncthreads();
  if (warp == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = warp_sum(lane < kWarps ? slots[lane * 4 + i] : T(0));
}

// Up to this many CTAs the last one of a pass adds up what all have left.  It costs each of them an atomic at its end, some 1 us in which nothing else takes its place: with
// several CTAs one after another on an SM a kernel for the sums is cheaper (8.4 M tokens, 4096 CTAs: 59.9 -> 52.7 us; 131072 tokens, 128 CTAs: 10.4 -> 11.3).
constexpr uint32_t kFewCtas = 1024;
constexpr int kFinishThreads = 1024;

__device__ __forceinline__ float4 ld_l2(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
// What this thread has written is seen by who takes a later ticket, and by those it meets at a barrier then.
__device__ __forceinline__ uint32_t take_ticket(uint32_t* ticket) {
  uint32_t before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
  return before;
}
template <int THREADS>
__device__ void all_sums(const float4* partial, uint32_t ctas, double (&total)[4], double* slots) {
#pragma unroll
  for (int i = 0; i < 4; ++i) total[i] = 0;
#pragma unroll 8
  for (uint32_t c = threadIdx.x; c < ctas; c += THREADS) {
    const float4 p = ld_l2(partial + c);
    total[0] += p.x, total[1] += p.y, total[2] += p.z, total[3] += p.w;
  }
  sums4<THREADS>(total, slots);
}
// Leaves a CTA's sums and tells whether it was the last one to; then the sums of all CTAs are in `total` of its first thread, added in an
// order that does not hang on which CTA was last.
template <int THREADS>
__device__ bool last_sums(float4 mine, float4* partial, uint32_t ctas, uint32_t* ticket, double (&total)[4], double* slots) {
  __shared__ bool last;
  if (threadIdx.x == 0) {
    partial[blockIdx.x] = mine;
    last = take_ticket(ticket) == ctas - 1;
  }
  __syncthreads();
  if (!last) return false;
  all_sums<THREADS>(partial, ctas, total, slots);
  return true;
}

// A bit for each token of a tile that counts, and how many there are; nothing outside the sequences counts.
template <class Id>
__global__ void __launch_bounds__(kThreads) mark_kernel(Packed<Id> p, Workspace w) {
  __shared__ uint32_t sums[kThreads / 32];
  pdl_enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) w.shared->ticket = w.shared->live = 0;
  const uint64_t begin = p.offset(0), end = p.offset(p.sequences);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t base = (uint64_t)blockIdx.x * kTile + warp * (32 * kEach);
  uint32_t mine = 0;
  Id ids[kEach];                                           // (all loads on their way before the first vote, and none behind a branch)
  if (base + 32 * kEach <= p.tokens) {                     // (the same for the whole warp)
#pragma unroll
    for (int j = 0; j < kEach; ++j) ids[j] = ld_id(p.ids + base + lane + 32 * j);
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j) ids[j] = ld_id(p.ids + min(base + 32 * j + lane, p.tokens - 1));
  }
  if (base >= begin && base + 32 * kEach <= end) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint32_t b = __ballot_sync(0xffffffffu, !(ids[j] < Id(0)));
      if (lane == j) mine = b;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint64_t t = base + 32 * j + lane;
      const uint32_t b = __ballot_sync(0xffffffffu, !(ids[j] < Id(0)) && t >= begin && t < end);
      if (lane == j) mine = b;
    }
  }
  if (lane < kEach) w.bits[base / 32 + lane] = mine;
  const uint32_t n = __reduce_add_sync(0xffffffffu, __popc(mine));
  if (lane == 0) sums[warp] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t total = 0;
    for (uint32_t s : sums) total += s;
    w.counts[blockIdx.x] = total;
  }
}

// How many tokens of [from, to) count, by a whole warp; from < to.
__device__ __forceinline__ uint64_t counted(const Workspace& w, uint64_t from, uint64_t to) {
  const uint32_t lane = threadIdx.x & 31;
  auto words = [&](uint64_t a, uint64_t b) {               // bits [a, b) of one tile
    uint32_t n = 0;
    for (uint64_t i = a / 32 + lane; i * 32 < b; i += 32) {
      uint32_t bits = w.bits[i];
      if (i * 32 < a) bits &= ~0u << (a & 31);
      if (i * 32 + 32 > b) bits &= ~0u >> (32 - (b & 31));
      n += __popc(bits);
    }
    return n;
  };
  const uint64_t first = from / kTile, last = (to - 1) / kTile;
  uint32_t n;
  uint64_t total = 0;
  if (first == last) {
    n = words(from, to);
  } else {
    n = words(from, (first + 1) * kTile) + words(last * kTile, to);
#pragma unroll 4
    for (uint64_t i = first + 1 + lane; i < last; i += 32) total += w.counts[i];
  }
  total += n;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  return total;
}

// What a token's term is multiplied by: the tokens that count altogether by one CTA, or of each sequence by a warp.
constexpr int kTotalThreads = 1024;
// (Up to kFewTiles tiles every CTA of the next kernel adds the counts up by itself while its loads are on their way: a launch less.  77777 tokens 6.2 us for 8.2 with
// this kernel, 1 M 10.2 for 11.0, 2 M 14.4 both; beyond, what the CTAs read through L2 costs more than the launch: 4 M 21.3 for 19.6, 8.4 M without a reference and with
// ids of 32 bits, where the bound is, 40.0 for 36.9.)
constexpr uint32_t kFewTiles = 4096;
__global__ void __launch_bounds__(kTotalThreads) total_kernel(Workspace w, uint32_t tiles) {
  __shared__ unsigned long long sums[kTotalThreads / 32];
  pdl_enter();
  unsigned long long n = 0;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < tiles; i += kTotalThreads) n += w.counts[i];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (unsigned long long s : sums) n += s;
    w.shared->share = n ? 1.f / (float)n : 0.f;
  }
}
// Where sequences are short a lane looks at each, and its warp at the others in turn; else a warp at each.
constexpr uint64_t kLane = 64;                             // tokens of a sequence that a lane looks at by itself
template <class Id>
bool short_ones(const Packed<Id>& p) {
  return p.sequences >= 1024 && p.tokens <= kLane * p.sequences;
}
// How many tokens of [from, to) count, by a lane: at most kLane of them, in three words.
__device__ __forceinline__ uint32_t counted_alone(const Workspace& w, uint64_t from, uint64_t to) {
  const uint64_t first = from / 32, last = (to - 1) / 32;
  uint32_t bits[3], n = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) bits[k] = w.bits[min(first + k, last)];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (first + k > last) break;
    if (k == 0) bits[k] &= ~0u << (from & 31);
    if (first + k == last) bits[k] &= ~0u >> (31 - ((to - 1) & 31));
    n += __popc(bits[k]);
  }
  return n;
}
// note_owner by a lane, of a sequence of fewer tokens than a block has.
__device__ __forceinline__ void note_owner_alone(const Workspace& w, uint32_t s, uint64_t from, uint64_t to) {
  const uint64_t b = (from + kBlock - 1) / kBlock;
  if (b * kBlock < to) w.owner[b] = s;
}
static_assert(kLane < kBlock && kLane <= 64, "three words, one block");

template <class Id, bool SHORT>
__global__ void __launch_bounds__(kThreads) shares_kernel(Packed<Id> p, Workspace w) {
  __shared__ uint32_t live;
  if (threadIdx.x == 0) live = 0;
  __syncthreads();
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31;
  uint32_t mine = 0;
  for (uint32_t i = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); SHORT ? i <= (p.sequences - 1) / 32 : i < p.sequences; i += gridDim.x * (kThreads / 32)) {
    if (SHORT) {
      const uint32_t s = i * 32 + lane;
      const bool there = s < p.sequences;
      const uint64_t from = there ? p.offset(s) : 0, to = there ? p.offset(s + 1) : 0;
      const bool some = from < to, alone = some && to - from <= kLane;
      uint64_t n = 0;
      if (alone) n = counted_alone(w, from, to), note_owner_alone(w, s, from, to);
      for (uint32_t todo = __ballot_sync(0xffffffffu, some && !alone); todo; todo &= todo - 1) {
        const int who = __ffs(todo) - 1;
        const uint64_t a = __shfl_sync(0xffffffffu, from, who), b = __shfl_sync(0xffffffffu, to, who), all = counted(w, a, b);
        note_owner(w, i * 32 + who, a, b);
        if (lane == who) n = all;
      }
      if (there) w.share[s] = n ? 1.f / (float)n : 0.f;
      mine += __popc(__ballot_sync(0xffffffffu, n != 0));
    } else {
      const uint64_t from = p.offset(i), to = p.offset(i + 1);
      const uint64_t n = from < to ? counted(w, from, to) : 0;
      note_owner(w, i, from, to);
      if (lane == 0) w.share[i] = n ? 1.f / (float)n : 0.f;
      mine += n != 0;
    }
  }
  if (lane == 0 && mine) atomicAdd(&live, mine);
  __syncthreads();
  if (threadIdx.x == 0 && live) atomicAdd(&w.shared->live, live);
}

// ---- the policy loss

struct Policy {
  const float *logprob, *old, *reference, *entropy, *advantage;
  float *loss, *g_logprob, *g_entropy;
  float high, low;                                         // what the ratio is clipped to
  double log_high, log_low;
  float fp32_high, fp32_low, near;                         // the same in fp32, and how far from them it decides
  float kl, bonus, count;
  int by_sequence, per_token;
};

// The terms of N tokens, whatever they hold; of those that do not count nothing is used.
template <int N>
struct Terms {
  float surrogate[N], kl[N], slope[N];
  bool clipped[N];
};
// On which side of the clipping border a token lies is decided by the difference of the logarithms in 64 bits, where it is exact: in fp32 rounding would decide
// for tokens on the border.  Away from it both agree, and fp32 is asked.
// exp(q) - 1 - q is taken near zero by the series from its second term on (the ninth is below 2^-24 of the first up to 1/2): as a difference all
// its digits would go.  Both take the slow way for all N where one needs it; two tokens at a time share an instruction of the series.
// (The exponential's argument has d's rounding, so that the approximate one, good to 2 ulp and the argument's rounding, gives nothing away.)
template <int N>
__device__ __forceinline__ Terms<N> terms(const Policy& o, const float* logprob, const float* old, const float* reference, const float* advantage) {
  Terms<N> t;
  float d[N], beyond[N], nearest = 1.f;                    // beyond: above zero where the ratio is past the border that its advantage drives it to
#pragma unroll
  for (int k = 0; k < N; ++k) {
    d[k] = logprob[k] - old[k];
    beyond[k] = advantage[k] < 0.f ? o.fp32_low - d[k] : d[k] - o.fp32_high;
    nearest = fminf(nearest, fabsf(beyond[k]));
  }
  if (nearest <= o.near) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const double exact = (double)logprob[k] - (double)old[k];
      if (d[k] == d[k]) beyond[k] = (advantage[k] < 0.f ? exact < o.log_low : exact > o.log_high) ? 1.f : -1.f;
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const bool cut = beyond[k] > 0.f;
    t.clipped[k] = cut && fabsf(advantage[k]) > 0.f;       // (of two zeros neither is above the other; nor is a NaN, which then shows in the gradient)
    float ratio;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ratio) : "f"(d[k] * 1.4426950408889634f));
    t.surrogate[k] = (cut ? (advantage[k] < 0.f ? o.low : o.high) : ratio) * advantage[k];
    t.slope[k] = t.clipped[k] ? 0.f : -t.surrogate[k];
    t.kl[k] = 0.f;
  }
  if (!o.reference) return t;
  float q[N], grown[N], farthest = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    q[k] = reference[k] - logprob[k];
    farthest = fmaxf(farthest, fabsf(q[k]));               // (a NaN stays one by the series too)
  }
  auto both = [](float v) { return pair(v, v); };
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const Pair x = pair(q[k], q[N > 1 ? k + 1 : k]);
    Pair y = fma2(both(1.f / 40320), x, both(1.f / 5040));
    y = fma2(y, x, both(1.f / 720)), y = fma2(y, x, both(1.f / 120)), y = fma2(y, x, both(1.f / 24)), y = fma2(y, x, both(1.f / 6));
    y = mul2(mul2(fma2(y, x, both(0.5f)), x), x);
    const float2 kl = halves(y), more = halves(add2(x, y));
    t.kl[k] = kl.x, grown[k] = more.x;
    if (N > 1) t.kl[k + 1] = kl.y, grown[k + 1] = more.y;
  }
  if (farthest >= 0.5f) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (fabsf(q[k]) >= 0.5f) {
        grown[k] = expm1f(q[k]);
        t.kl[k] = grown[k] - q[k];
      }
  }
  if (o.kl != 0.f) {                                       // (a term of weight zero is none: exp(q) may have left fp32)
#pragma unroll
    for (int k = 0; k < N; ++k) t.slope[k] = fmaf(-o.kl, grown[k], t.slope[k]);
  }
  return t;
}
__device__ __forceinline__ void write_loss(const Policy& o, const double* total) {
  double loss = -total[0];
  if (o.kl != 0.f) loss += (double)o.kl * total[1];
  if (o.bonus != 0.f) loss -= (double)o.bonus * total[2];
  o.loss[0] = (float)loss;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.loss[i + 1] = (float)total[i];
}

// Four neighbours; `whole`: for all threads of the CTA a vector inside the array.  (Else no load stands behind a branch of its own either.)
__device__ __forceinline__ float4 load4(const float* p, uint64_t t, uint64_t end, bool whole) {
  if (!p) return make_float4(0.f, 0.f, 0.f, 0.f);
  if (whole) return ld_stream(reinterpret_cast<const float4*>(p + t));
  float4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) (&v.x)[k] = ld_stream(p + min(t + k, end - 1));
  return v;
}
// Of four neighbours those of [begin, end).
__device__ __forceinline__ void store4(float* p, float4 v, uint64_t t, uint64_t begin, uint64_t end, bool vectors) {
  if (vectors && t >= begin && t + 4 <= end) {
    st_stream(reinterpret_cast<float4*>(p + t), v);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t + k >= begin && t + k < end) p[t + k] = (&v.x)[k];
}

// few_tiles: the tiles whose counts each CTA adds up by itself.  LOOK: a token's sequence is needed.  PARTS: of kPart tokens that a CTA has, with all their loads on their way.
constexpr uint32_t kPart = kThreads * 4;
template <class Id, bool LOOK, int PARTS>
__global__ void __launch_bounds__(kThreads) policy_kernel(Packed<Id> p, Workspace w, Policy o, bool vectors, uint32_t few_tiles) {
  __shared__ float slots[kThreads / 8];
  __shared__ uint32_t tokens[kThreads / 32];
  __shared__ double wide[kThreads / 8];
  pdl_enter();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t begin = p.offset(0), end = p.offset(p.sequences);
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  float4 lp[PARTS], old[PARTS], ref[PARTS], ent[PARTS], adv[PARTS];
  uint32_t bits[PARTS], owner[PARTS];
  const bool whole = vectors && (uint64_t)(blockIdx.x + 1) * PARTS * kPart <= p.tokens;
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    const uint64_t t = ((uint64_t)blockIdx.x * PARTS + h) * kPart + threadIdx.x * 4;
    lp[h] = load4(o.logprob, t, p.tokens, whole), old[h] = load4(o.old, t, p.tokens, whole);
    ref[h] = load4(o.reference, t, p.tokens, whole), ent[h] = load4(o.entropy, t, p.tokens, whole);
    adv[h] = load4(o.per_token ? o.advantage : nullptr, t, p.tokens, whole);
    bits[h] = w.bits[t / 32] >> (t & 31) & 15;             // (the last tile's words are all there)
    owner[h] = LOOK && o.by_sequence ? owner_of(p, w, t - 4 * lane, begin) : kNone;
  }
  Found found;
  float even;
  if (o.count > 0.f) {
    even = 1.f / o.count;
  } else if (o.by_sequence) {
    even = 1.f / (float)w.shared->live;
  } else if (few_tiles) {
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x; i < few_tiles; i += kThreads) n += w.counts[i];
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) tokens[warp] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) n += tokens[i];
    even = n ? 1.f / (float)n : 0.f;
  } else {
    even = w.shared->share;
  }
#pragma unroll
  for (int h = 0; h < PARTS; ++h) {
    const uint64_t base = ((uint64_t)blockIdx.x * PARTS + h) * kPart + warp * 128, t = base + 4 * lane;
    uint32_t of[4] = {0, 0, 0, 0};
    if (LOOK && base < end) sequences_of(p, base, owner[h], of, found);
    float4 g, ge;
    if (LOOK && !o.per_token)
#pragma unroll
      for (int k = 0; k < 4; ++k) (&adv[h].x)[k] = bits[h] >> k & 1 ? o.advantage[of[k]] : 0.f;
    const Terms<4> e = terms<4>(o, &lp[h].x, &old[h].x, &ref[h].x, &adv[h].x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool counts = bits[h] >> k & 1;
      const float weight = LOOK && o.by_sequence && counts ? even * w.share[of[k]] : even;
      if (counts) {
        sum[0] += e.surrogate[k] * weight, sum[1] += e.kl[k] * weight, sum[2] += (&ent[h].x)[k] * weight;
        if (e.clipped[k]) sum[3] += weight;
      }
      (&g.x)[k] = counts ? e.slope[k] * weight : 0.f;
      (&ge.x)[k] = counts ? -o.bonus * weight : 0.f;
    }
    if (o.g_logprob) store4(o.g_logprob, g, t, begin, end, vectors);
    if (o.g_entropy) store4(o.g_entropy, ge, t, begin, end, vectors);
  }
  sums4<kThreads>(sum, slots);
  if (gridDim.x > kFewCtas) {
    if (threadIdx.x == 0) w.partial[blockIdx.x] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    return;
  }
  double total[4];
  if (last_sums<kThreads>(make_float4(sum[0], sum[1], sum[2], sum[3]), w.partial, gridDim.x, &w.shared->ticket, total, wide) && threadIdx.x == 0)
    write_loss(o, total);
}
__global__ void __launch_bounds__(kFinishThreads) policy_finish_kernel(Workspace w, Policy o, uint32_t ctas) {
  __shared__ double slots[kFinishThreads / 8];
  pdl_enter();
  double total[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t c = threadIdx.x; c < ctas; c += kFinishThreads) {
    const float4 p = w.partial[c];
    total[0] += p.x, total[1] += p.y, total[2] += p.z, total[3] += p.w;
  }
  sums4<kFinishThreads>(total, slots);
  if (threadIdx.x == 0) write_loss(o, total);
}

// ---- one CTA for few tokens: which of them count, and how many before each word of 32

struct FewTokens {
  uint32_t bits[kFew / 32], before[kFew / 32 + 1];
  uint32_t offsets[kFewSequences + 1];
  uint32_t warps[kFewThreads / 32];
  __device__ __forceinline__ uint32_t until(uint32_t t) const {   // how many of the tokens before t count
    return before[t / 32] + (t & 31 ? __popc(bits[t / 32] & ~(~0u << (t & 31))) : 0);
  }
  __device__ __forceinline__ uint32_t sequence(uint32_t t, uint32_t sequences) const {
    uint32_t lo = 0, end = sequences;
    while (end - lo > 1) {
      const uint32_t middle = lo + (end - lo) / 2;
      if (offsets[middle] <= t) lo = middle;
      else end = middle;
    }
    return lo;
  }
  __device__ __forceinline__ bool counts(uint32_t t) const { return bits[t / 32] >> (t & 31) & 1; }
};
// Which tokens count, and the offsets, to be read behind a barrier.  Thread i's tokens are i, i + kFewThreads, ..., EACH at most; the result: which of its own count.
// (One, two, four or six: instructions that come from memory are much of such a launch.  600 tokens 3.0 us where eight took 3.4, 1500 in pairs 3.8 for 4.2.)
template <int EACH, class Id>
__device__ __forceinline__ uint32_t few_tokens(const Packed<Id>& p, FewTokens& f) {
  const uint32_t begin = (uint32_t)p.offset(0), end = (uint32_t)p.offset(p.sequences);
  for (uint32_t s = threadIdx.x; s <= p.sequences; s += kFewThreads) f.offsets[s] = (uint32_t)p.offset(s);
  Id ids[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (j * kFewThreads >= p.tokens) break;
    ids[j] = ld_id(p.ids + min((uint64_t)(j * kFewThreads + threadIdx.x), p.tokens - 1));
  }
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const uint32_t t = j * kFewThreads + threadIdx.x;
    uint32_t b = 0;
    if (j * kFewThreads < p.tokens) {
      const bool counts = t >= begin && t < end && !(ids[j] < Id(0));
      b = __ballot_sync(0xffffffffu, counts);
      mine |= (uint32_t)counts << j;
    }
    if ((threadIdx.x & 31) == 0) f.bits[t / 32] = b;
  }
  return mine;
}
// How many count before each word, between two barriers.
template <int EACH>
__device__ __forceinline__ void few_counts(FewTokens& f) {
  constexpr uint32_t kHeld = EACH * kFewThreads / 32;
  const uint32_t lane = threadIdx.x & 31;
  if (threadIdx.x < kHeld) {                               // the words' counts, summed up over the warps of those threads
    const uint32_t n = __popc(f.bits[threadIdx.x]);
    uint32_t upto = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    f.before[threadIdx.x] = upto - n;
    if (lane == 31) f.warps[threadIdx.x >> 5] = upto;
  }
  __syncthreads();
  if (threadIdx.x < kHeld) {
    uint32_t more = 0;
    for (uint32_t i = 0; i < threadIdx.x >> 5; ++i) more += f.warps[i];
    f.before[threadIdx.x] += more;
    if (threadIdx.x == kHeld - 1) f.before[kHeld] = f.before[threadIdx.x] + __popc(f.bits[threadIdx.x]);
  }
  __syncthreads();
}

template <class Id, int EACH>
__global__ void __launch_bounds__(kFewThreads) policy_few_kernel(Packed<Id> p, Policy o) {
  __shared__ FewTokens f;
  __shared__ float share[kFewSequences], advantage[kFewSequences];
  __shared__ double slots[kFewThreads / 8];
  __shared__ uint32_t live;
  if (threadIdx.x == 0) live = 0;
  pdl_enter();
  // the first tokens' values and the sequences' are on their way while the ids are counted
  const uint32_t early = min(threadIdx.x, (uint32_t)p.tokens - 1);
  const float first_lp = ld_stream(o.logprob + early), first_old = ld_stream(o.old + early);
  const float first_ref = o.reference ? ld_stream(o.reference + early) : 0.f, first_entropy = o.entropy ? ld_stream(o.entropy + early) : 0.f;
  const uint32_t advantages = o.per_token ? (uint32_t)p.tokens : p.sequences;
  static_assert(kFewSequences == 2 * kFewThreads, "two sequences to a thread");
  const float first_adv = ld_stream(o.advantage + min(threadIdx.x, advantages - 1));
  const float next_adv = ld_stream(o.advantage + min(threadIdx.x + kFewThreads, advantages - 1));
  const uint32_t mine = few_tokens<EACH>(p, f);
  advantage[threadIdx.x] = first_adv, advantage[threadIdx.x + kFewThreads] = next_adv;
  __syncthreads();
  const bool look = o.by_sequence || !o.per_token;
  float even;
  if (o.by_sequence) {
    few_counts<EACH>(f);
    uint32_t full = 0;
    for (uint32_t s = threadIdx.x; s < p.sequences; s += kFewThreads) {
      const uint32_t from = f.offsets[s], to = f.offsets[s + 1], n = from < to ? f.until(to) - f.until(from) : 0;
      share[s] = n ? 1.f / (float)n : 0.f;
      full += n != 0;
    }
    if (full) atomicAdd(&live, full);
    __syncthreads();
    even = o.count > 0.f ? 1.f / o.count : 1.f / (float)live;
  } else {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < EACH * kFewThreads / 32; i += 32) n += __popc(f.bits[i + (threadIdx.x & 31)]);
    n = __reduce_add_sync(0xffffffffu, n);
    even = o.count > 0.f ? 1.f / o.count : n ? 1.f / (float)n : 0.f;
  }
  const uint32_t begin = f.offsets[0], end = f.offsets[p.sequences];
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < EACH && j * kFewThreads < (int)p.tokens; ++j) {
    const uint32_t t = j * kFewThreads + threadIdx.x;
    if (t < begin || t >= end) continue;
    const bool counts = mine >> j & 1;
    float g = 0.f, weight = 0.f;
    if (counts) {
      const uint32_t s = look ? f.sequence(t, p.sequences) : 0;
      weight = o.by_sequence ? even * share[s] : even;
      const float lp = j ? o.logprob[t] : first_lp, old = j ? o.old[t] : first_old, ref = j ? (o.reference ? o.reference[t] : 0.f) : first_ref;
      const float a = !o.per_token ? advantage[s] : j ? o.advantage[t] : first_adv;
      const Terms<1> e = terms<1>(o, &lp, &old, &ref, &a);
      sum[0] += e.surrogate[0] * weight, sum[1] += e.kl[0] * weight;
      if (e.clipped[0]) sum[3] += weight;
      if (o.entropy) sum[2] += (j ? o.entropy[t] : first_entropy) * weight;
      g = e.slope[0] * weight;
    }
    if (o.g_logprob) o.g_logprob[t] = g;
    if (o.g_entropy) o.g_entropy[t] = -o.bonus * weight;
  }
  // (shuffles are what this costs: warps without tokens take none, and the others 32 bits)
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (warp * 32 < p.tokens) sum[i] = warp_sum(sum[i]);
    if (lane == 0) slots[warp * 4 + i] = sum[i];
  }
  __syncthreads();
  if (warp != 0) return;
  static_assert(kFewThreads == 32 * 32, "a lane for each warp's sums");
  double total[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) total[i] = warp_sum(slots[lane * 4 + i]);
  if (threadIdx.x == 0) write_loss(o, total);
}

// ---- the loss of pairs

struct Pairs {
  const float *logprob, *reference;
  float *loss, *rewards, *g_logprob;
  float beta, smoothing, margin, count;
  int average;
};

// A pair's loss by z, its rewards' difference without the margin, and the loss's derivative.  log(1 + e^-|z|) and e^-|z| / (1 + e^-|z|):
// nothing overflows.  Each side of the loss is a sum of what is not below zero, and a side of weight zero is none: z may be infinite (a token
// whose logit was masked), and where smoothing leaves the small side alone nothing cancels.
__device__ __forceinline__ float pair_loss(float z, float smoothing, float* slope) {
  const float e = expf(-fabsf(z)), more = log1pf(e);
  const float against = e / (1.f + e), with = 1.f / (1.f + e);   // sigmoid(-|z|), sigmoid(|z|)
  *slope = z >= 0.f ? smoothing * with - (1.f - smoothing) * against : smoothing * against - (1.f - smoothing) * with;
  const float right = smoothing == 1.f ? 0.f : (1.f - smoothing) * (more + fmaxf(-z, 0.f));
  const float wrong = smoothing == 0.f ? 0.f : smoothing * (more + fmaxf(z, 0.f));
  return right + wrong;
}
struct Pair2 {
  float loss, right, gap;
};
// Rewards, the loss, and in `chosen` and `rejected` the gradients at each token that counts.  Sums in 64 bits; n: tokens that count.
__device__ __forceinline__ Pair2 pair_terms(const Pairs& o, uint32_t pair, double chosen, double rejected, uint64_t n_chosen, uint64_t n_rejected,
                                            float inv_count, float* g_chosen, float* g_rejected) {
  const double beta = o.beta;
  if (o.average) chosen /= (double)(n_chosen ? n_chosen : 1), rejected /= (double)(n_rejected ? n_rejected : 1);
  const double gap = beta * (chosen - rejected);
  if (o.rewards) o.rewards[2 * pair] = (float)(beta * chosen), o.rewards[2 * pair + 1] = (float)(beta * rejected);
  float slope;
  Pair2 r;
  r.loss = pair_loss((float)(gap - (double)o.margin), o.smoothing, &slope);
  r.right = gap > 0 ? 1.f : 0.f;
  r.gap = (float)gap;
  slope *= o.beta * inv_count;
  *g_chosen = o.average ? (n_chosen ? slope / (float)n_chosen : 0.f) : slope;
  *g_rejected = o.average ? (n_rejected ? -slope / (float)n_rejected : 0.f) : -slope;
  return r;
}

// The sums of a tile's sequences, or of its parts of them, and which of its tokens count.
template <class Id>
__global__ void __launch_bounds__(kThreads) sums_kernel(Packed<Id> p, Workspace w, Pairs o) {
  __shared__ double values[kTile];
  __shared__ double slots[kThreads / 32];
  __shared__ uint32_t sums[kThreads / 32], span[2];
  pdl_enter();
  if (blockIdx.x == 0 && threadIdx.x == 0) w.shared->ticket = 0;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t begin = p.offset(0), end = p.offset(p.sequences);
  const uint64_t tile = (uint64_t)blockIdx.x * kTile, tile_end = min(tile + kTile, p.tokens);
  const uint64_t from = max(tile, begin), to = min(tile_end, end);
  float lp[kEach], ref[kEach];
  Id ids[kEach];                                           // (all loads on their way before the first vote, and none behind a branch)
  uint32_t mine = 0, bits = 0;
  // places within the tile: the thread's first one, and what lies in a sequence
  const uint32_t at = warp * (32 * kEach) + lane, low = from < to ? (uint32_t)(from - tile) : 0, high = from < to ? (uint32_t)(to - tile) : 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) lp[j] = ref[j] = 0.f;
  if (tile + kTile <= p.tokens) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) ids[j] = ld_id(p.ids + tile + at + 32 * j), lp[j] = ld_stream(o.logprob + tile + at + 32 * j);
    if (o.reference)
#pragma unroll
      for (int j = 0; j < kEach; ++j) ref[j] = ld_stream(o.reference + tile + at + 32 * j);
  } else if (p.tokens) {
    const uint32_t last = (uint32_t)(p.tokens - 1 - tile);
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint64_t t = tile + min(at + 32 * j, last);
      ids[j] = ld_id(p.ids + t), lp[j] = ld_stream(o.logprob + t);
      if (o.reference) ref[j] = ld_stream(o.reference + t);
    }
  }
  // (the tile's first and last sequence are looked for while these are on their way)
  if (warp < 2 && from < to) {
    const uint32_t s = sequence_of(p, warp == 0 ? from : to - 1);
    if (lane == 0) span[warp] = s;
  }
  if (from < to) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const uint32_t i = at + 32 * j;
      const bool counts = !(ids[j] < Id(0)) && i >= low && i < high;
      const uint32_t b = __ballot_sync(0xffffffffu, counts);
      if (lane == j) mine = b;
      bits |= (uint32_t)counts << j;
    }
  }
  if (lane < kEach) w.bits[tile / 32 + warp * kEach + lane] = mine;
  const uint32_t n = __reduce_add_sync(0xffffffffu, __popc(mine));
  if (lane == 0) sums[warp] = n;
  double sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const double d = bits >> j & 1 ? (double)lp[j] - (double)ref[j] : 0.0;
    values[warp * (32 * kEach) + 32 * j + lane] = d;
    sum += d;
  }
  sum = warp_sum(sum);
  if (lane == 0) slots[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t total = 0;
    for (uint32_t s : sums) total += s;
    w.counts[blockIdx.x] = total;
  }
  if (from >= to) return;
  const uint32_t first = span[0], last = span[1];
  auto keep = [&](uint32_t s, uint64_t a, uint64_t b, double v) {
    if (a < tile) w.head[blockIdx.x] = v;
    else if (b > tile + kTile) w.tail[blockIdx.x] = v;
    else w.whole[s] = v;
  };
  if (first == last) {
    if (threadIdx.x == 0) {
      double v = 0;
      for (double s : slots) v += s;
      keep(first, p.offset(first), p.offset(first + 1), v);
    }
    return;
  }
  // each lane looks at one sequence and, where there are many, sums a short one by itself; the warp sums the others in turn
  const uint32_t alone = last - first >= 64 ? kShort : 0;
  for (uint32_t chunk = first; chunk <= last; chunk += kThreads) {
    const uint32_t s = chunk + lane * (kThreads / 32) + warp;
    const uint64_t a = s <= last ? p.offset(s) : 0, b = s <= last ? p.offset(s + 1) : 0;
    const uint32_t lo = (uint32_t)(max(a, from) - tile), hi = max(a, from) < min(b, to) ? (uint32_t)(min(b, to) - tile) : lo;
    if (hi > lo && hi - lo <= alone) {
      double v = 0;
      for (uint32_t i = lo; i < hi; ++i) v += values[i];
      keep(s, a, b, v);
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, hi - lo > alone); todo; todo &= todo - 1) {
      const int who = __ffs(todo) - 1;
      const uint64_t sa = __shfl_sync(0xffffffffu, a, who), sb = __shfl_sync(0xffffffffu, b, who);
      double v = 0;
      for (uint32_t i = (uint32_t)(max(sa, from) - tile) + lane; i < (uint32_t)(min(sb, to) - tile); i += 32) v += values[i];
      v = warp_sum(v);
      if (lane == who) keep(s, sa, sb, v);
    }
  }
}

// A sequence's sum from what its tiles have left, by a whole warp.
__device__ __forceinline__ double sum_of(const Workspace& w, uint32_t s, uint64_t from, uint64_t to) {
  const uint64_t first = from / kTile, last = (to - 1) / kTile;
  if (first == last) {
    // (one that ends where the tile does may have begun before it: then first < last)
    return w.whole[s];
  }
  double v = 0;
#pragma unroll 4
  for (uint64_t i = first + 1 + (threadIdx.x & 31); i <= last; i += 32) v += w.head[i];
  return warp_sum(v) + w.tail[first];
}

// A warp per sequence, or a lane for each short one.  The loss is written by the last CTA or, where the gradient's kernel comes next, by one more CTA of that, while nothing waits for it.
__device__ __forceinline__ void write_loss(const Pairs& o, const double* total) {
  o.loss[0] = (float)total[0], o.loss[1] = (float)total[1], o.loss[2] = (float)total[2];
}
template <class Id, bool SHORT>
__global__ void __launch_bounds__(kThreads) pairs_kernel(Packed<Id> p, Workspace w, Pairs o, float inv_count, bool gradient_next) {
  __shared__ float slots[kThreads / 8];
  __shared__ double wide[kThreads / 8], sums[kThreads / 32];
  __shared__ uint64_t counts[kThreads / 32];
  pdl_enter();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  if (SHORT) {
    const uint32_t s = blockIdx.x * kThreads + threadIdx.x;
    const bool there = s < p.sequences;
    const uint64_t from = there ? p.offset(s) : 0, to = there ? p.offset(s + 1) : 0;
    const bool some = from < to, alone = some && to - from <= kLane;
    double d = 0;
    uint64_t n = 0;
    if (alone) {
      const uint64_t first = from / kTile, last = (to - 1) / kTile;
      d = first == last ? w.whole[s] : w.head[last] + w.tail[first];
      if (o.average) n = counted_alone(w, from, to);
      note_owner_alone(w, s, from, to);
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, some && !alone); todo; todo &= todo - 1) {
      const int who = __ffs(todo) - 1;
      const uint32_t its = s - lane + who;
      const uint64_t a = __shfl_sync(0xffffffffu, from, who), b = __shfl_sync(0xffffffffu, to, who), all = o.average ? counted(w, a, b) : 0;
      const double v = sum_of(w, its, a, b);
      note_owner(w, its, a, b);
      if (lane == who) d = v, n = all;
    }
    const double rejected = __shfl_down_sync(0xffffffffu, d, 1);
    const uint64_t n_rejected = __shfl_down_sync(0xffffffffu, n, 1);
    if (there && (lane & 1) == 0) {
      const Pair2 r = pair_terms(o, s / 2, d, rejected, n, n_rejected, inv_count, w.share + s, w.share + s + 1);
      sum[0] = r.loss * inv_count, sum[1] = r.right * inv_count, sum[2] = r.gap * inv_count;
    }
  } else {
    const uint32_t s = blockIdx.x * (kThreads / 32) + warp;
    if (s < p.sequences) {
      const uint64_t from = p.offset(s), to = p.offset(s + 1);
      note_owner(w, s, from, to);
      const double d = from < to ? sum_of(w, s, from, to) : 0;
      const uint64_t n = o.average && from < to ? counted(w, from, to) : 0;
      if (lane == 0) sums[warp] = d, counts[warp] = n;
    }
    __syncthreads();
    if (lane == 0 && (warp & 1) == 0 && s < p.sequences) {
      const Pair2 r = pair_terms(o, s / 2, sums[warp], sums[warp + 1], counts[warp], counts[warp + 1], inv_count, w.share + s, w.share + s + 1);
      sum[0] = r.loss * inv_count, sum[1] = r.right * inv_count, sum[2] = r.gap * inv_count;
    }
  }
  sums4<kThreads>(sum, slots);
  if (gradient_next) {
    if (threadIdx.x == 0) w.partial[blockIdx.x] = make_float4(sum[0], sum[1], sum[2], 0.f);
    return;
  }
  double total[4];
  if (last_sums<kThreads>(make_float4(sum[0], sum[1], sum[2], 0.f), w.partial, gridDim.x, &w.shared->ticket, total, wide) && threadIdx.x == 0) write_loss(o, total);
}

template <class Id>
__global__ void __launch_bounds__(kThreads) pairs_grad_kernel(Packed<Id> p, Workspace w, Pairs o, uint32_t partials, bool vectors) {
  __shared__ double wide[kThreads / 8];
  pdl_enter();
  if (blockIdx.x == 0) {
    double total[4];
    all_sums<kThreads>(w.partial, partials, total, wide);
    if (threadIdx.x == 0) write_loss(o, total);
    return;
  }
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t begin = p.offset(0), end = p.offset(p.sequences);
  Found found;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint64_t base = (uint64_t)(blockIdx.x - 1) * kPass + h * (kPass / 2) + warp * 128, t = base + 4 * lane;
    if (base >= end) return;
    uint32_t of[4];
    const uint32_t bits = w.bits[t / 32] >> (t & 31) & 15; // (the last tile's words are all there)
    sequences_of(p, base, owner_of(p, w, base, begin), of, found);
    float4 g, share;
    share.x = w.share[of[0]];
    // (mostly the whole warp's tokens are of one sequence)
    if (base + 128 <= found.end) share.y = share.z = share.w = share.x;
    else share.y = w.share[of[1]], share.z = w.share[of[2]], share.w = w.share[of[3]];
#pragma unroll
    for (int k = 0; k < 4; ++k) (&g.x)[k] = bits >> k & 1 ? (&share.x)[k] : 0.f;
    store4(o.g_logprob, g, t, begin, end, vectors);
  }
}

template <class Id, int EACH>
__global__ void __launch_bounds__(kFewThreads) pairs_few_kernel(Packed<Id> p, Pairs o, float inv_count) {
  extern __shared__ double values[];
  double* const sums = values + p.tokens;                  // of each sequence
  __shared__ FewTokens f;
  __shared__ float share[kFewSequences];
  __shared__ double slots[kFewThreads / 8];
  pdl_enter();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float lp[EACH], ref[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (j * kFewThreads >= p.tokens) break;
    const uint32_t t = min(j * kFewThreads + threadIdx.x, (uint32_t)p.tokens - 1);
    lp[j] = ld_stream(o.logprob + t);
    ref[j] = o.reference ? ld_stream(o.reference + t) : 0.f;
  }
  const uint32_t mine = few_tokens<EACH>(p, f);
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const uint32_t t = j * kFewThreads + threadIdx.x;
    if (t < p.tokens) values[t] = mine >> j & 1 ? (double)lp[j] - (double)ref[j] : 0.0;
  }
  __syncthreads();
  if (o.average) few_counts<EACH>(f);
  double total[4] = {0, 0, 0, 0};
  auto terms_of = [&](uint32_t pair, double chosen, double rejected) {
    auto counted = [&](uint32_t s) { return o.average && f.offsets[s] < f.offsets[s + 1] ? f.until(f.offsets[s + 1]) - f.until(f.offsets[s]) : 0; };
    const Pair2 r = pair_terms(o, pair, chosen, rejected, counted(2 * pair), counted(2 * pair + 1), inv_count, share + 2 * pair, share + 2 * pair + 1);
    total[0] += (double)(r.loss * inv_count), total[1] += (double)(r.right * inv_count), total[2] += (double)(r.gap * inv_count);
  };
  const uint32_t pairs = p.sequences / 2;
  if (pairs <= kFewThreads / 32) {                         // a warp for each pair, half of it for each of its sequences
    if (warp < pairs) {
      const uint32_t s = 2 * warp + lane / 16, to = f.offsets[s + 1];
      double v = 0;
#pragma unroll 4
      for (uint32_t t = f.offsets[s] + lane % 16; t < to; t += 16) v += values[t];
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      const double rejected = __shfl_sync(0xffffffffu, v, 16);
      if (lane == 0) terms_of(warp, v, rejected);
    }
  } else {                                                 // a lane for each short sequence, the warp for the others in turn; then a thread for each pair
    for (uint32_t first = warp; first < p.sequences; first += kFewThreads) {
      const uint32_t s = first + lane * (kFewThreads / 32), from = s < p.sequences ? f.offsets[s] : 0, to = s < p.sequences ? max(f.offsets[s + 1], from) : 0;
      double mine_sum = 0;
      if (to - from <= kShort)
        for (uint32_t t = from; t < to; ++t) mine_sum += values[t];
      for (uint32_t todo = __ballot_sync(0xffffffffu, to - from > kShort); todo; todo &= todo - 1) {
        const int who = __ffs(todo) - 1;
        const uint32_t a = __shfl_sync(0xffffffffu, from, who), b = __shfl_sync(0xffffffffu, to, who);
        double v = 0;
#pragma unroll 4
        for (uint32_t t = a + lane; t < b; t += 32) v += values[t];
        v = warp_sum(v);
        if (lane == who) mine_sum = v;
      }
      if (s < p.sequences) sums[s] = mine_sum;
    }
    __syncthreads();
    if (threadIdx.x < pairs) terms_of(threadIdx.x, sums[2 * threadIdx.x], sums[2 * threadIdx.x + 1]);
    static_assert(kFewSequences == 2 * kFewThreads, "a pair to a thread");
#pragma unroll
    for (int i = 0; i < 3; ++i) total[i] = warp_sum(total[i]);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (lane == 0) slots[warp * 4 + i] = total[i];
  __syncthreads();                                         // (behind which the shares are read, too)
  if (warp == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) total[i] = warp_sum(slots[lane * 4 + i]);
  if (threadIdx.x == 0) write_loss(o, total);
  if (!o.g_logprob) return;
  const uint32_t begin = f.offsets[0], end = f.offsets[p.sequences];
  for (uint32_t t = begin + threadIdx.x; t < end; t += kFewThreads)
    o.g_logprob[t] = f.counts(t) ? share[f.sequence(t, p.sequences)] : 0.f;
}

// ---- host side

template <class F>
int with_ids(int id_type, F f) {
  switch (id_type) {
    case POLAR_B200_IDS_F32: return f(float());
    case POLAR_B200_IDS_I32: return f(int32_t());
    default: return f(int64_t());
  }
}
bool few(uint64_t tokens, uint64_t sequences, uint64_t most) { return tokens <= most && sequences <= kFewSequences; }
int check_sequences(const void* ids, const void* offsets, int id_type, uint64_t tokens, uint64_t sequences) {
  if (id_type < POLAR_B200_IDS_F32 || id_type > POLAR_B200_IDS_I64) return fail(POLAR_B200_ERR_INVALID, "unknown type of ids");
  if (tokens > 1ull << 36 || sequences > 0x7fffffffull) return fail(POLAR_B200_ERR_INVALID, "too many tokens or sequences");
  if (id_type == POLAR_B200_IDS_F32 && tokens > 1ull << 24)
    return fail(POLAR_B200_ERR_INVALID, "offsets in fp32 are exact up to 2^24 tokens");
  if (id_type == POLAR_B200_IDS_I32 && tokens > 0x7fffffffull) return fail(POLAR_B200_ERR_INVALID, "offsets in 32 bits reach up to 2^31 - 1 tokens");
  if (sequences && !offsets) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  if (sequences && tokens && !ids) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  return POLAR_B200_OK;
}
// Whether a written array of a value per token overlaps one that is read or written, unless it is read by the same thread (`same`: an array
// of a value per token, at the same place).
bool overlaps(const void* w, uint64_t w_bytes, const void* o, uint64_t o_bytes, bool same) {
  if (!w || !o || !w_bytes || !o_bytes || (same && w == o)) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(w), b = reinterpret_cast<uintptr_t>(o);
  return a < b + o_bytes && b < a + w_bytes;
}
uint64_t id_bytes(int id_type) { return id_type == POLAR_B200_IDS_I64 ? 8 : 4; }

// The caller's workspace, or one from the pool for as long as `f` takes.
template <class F>
int with_workspace(void* workspace, uint64_t workspace_bytes, uint64_t need, cudaStream_t st, F f) {
  if (workspace) {
    if (workspace_bytes < need || !aligned16(workspace)) return fail(POLAR_B200_ERR_WORKSPACE, "workspace too small or not 16-byte aligned");
    return f(workspace);
  }
  void* own = nullptr;
  cudaError_t e = scratch_alloc(&own, need, st);
  if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "scratch (workspace)", e);
  const int rc = f(own);
  e = scratch_free(own, st);
  if (rc == POLAR_B200_OK && e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "returning scratch", e);
  return rc;
}

template <class Id>
int run_policy(const Packed<Id>& p, const Policy& o, void* workspace, uint64_t workspace_bytes, cudaStream_t st) {
  if (few(p.tokens, p.sequences, kFewPolicy)) {
    const uint64_t each = (p.tokens + kFewThreads - 1) / kFewThreads;
    auto kernel = each <= 1 ? policy_few_kernel<Id, 1> : each <= 2 ? policy_few_kernel<Id, 2> : policy_few_kernel<Id, kFewPolicy / kFewThreads>;
    return launch("fpolicy_loss", kernel, dim3(1), kFewThreads, 0, st, p, o);
  }
  uint64_t need;
  lay_out(nullptr, p.tokens, p.sequences, false, &need);
  return with_workspace(workspace, workspace_bytes, need, st, [&](void* base) {
    const Workspace w = lay_out(base, p.tokens, p.sequences, false, &need);
    const uint32_t tiles = (uint32_t)tiles_of(p.tokens);
    int rc = launch("fpolicy_loss: ids", mark_kernel<Id>, dim3(tiles), kThreads, 0, st, p, w);
    if (rc) return rc;
    if (o.by_sequence) {
      const uint64_t each = short_ones(p) ? kThreads : kThreads / 32, ctas = (p.sequences + each - 1) / each, most = 8ull * sm_count();
      rc = launch("fpolicy_loss: shares", short_ones(p) ? shares_kernel<Id, true> : shares_kernel<Id, false>, dim3((unsigned)(ctas < most ? ctas : most)), kThreads, 0, st, p, w);
    } else if (o.count == 0.f && tiles > kFewTiles) {
      rc = launch("fpolicy_loss: total", total_kernel, dim3(1), kTotalThreads, 0, st, w, tiles);
    }
    if (rc) return rc;
    const bool vectors = aligned16(o.logprob) && aligned16(o.old) && aligned16(o.reference) && aligned16(o.entropy) && aligned16(o.g_logprob) &&
                         aligned16(o.g_entropy) && (!o.per_token || aligned16(o.advantage));
    // (half as many tokens to a CTA where there would not be one for each SM)
    const bool look = o.by_sequence || !o.per_token, short_ = p.tokens <= 2ull * kPart * sm_count();
    auto kernel = short_ ? (look ? policy_kernel<Id, true, 1> : policy_kernel<Id, false, 1>) : look ? policy_kernel<Id, true, 2> : policy_kernel<Id, false, 2>;
    const uint64_t each = short_ ? kPart : 2 * kPart;
    const uint32_t ctas = (uint32_t)((p.tokens + each - 1) / each);
    rc = launch("fpolicy_loss", kernel, dim3(ctas), kThreads, 0, st, p, w, o, vectors, tiles <= kFewTiles ? tiles : 0u);
    if (rc || ctas <= kFewCtas) return rc;
    return launch("fpolicy_loss: sums", policy_finish_kernel, dim3(1), kFinishThreads, 0, st, w, o, ctas);
  });
}

template <class Id>
int run_pairs(const Packed<Id>& p, const Pairs& o, void* workspace, uint64_t workspace_bytes, cudaStream_t st) {
  const float inv_count = o.count > 0.f ? 1.f / o.count : 2.f / (float)p.sequences;
  if (few(p.tokens, p.sequences, kFew)) {
    constexpr size_t kBytes = (kFew + kFewSequences) * sizeof(double);
    const uint64_t each = (p.tokens + kFewThreads - 1) / kFewThreads;
    auto kernel = each <= 1 ? pairs_few_kernel<Id, 1> : each <= 2 ? pairs_few_kernel<Id, 2> : each <= 4 ? pairs_few_kernel<Id, 4> : pairs_few_kernel<Id, kFewEach>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes);
    if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "fpreference_loss", e);
    return launch("fpreference_loss", kernel, dim3(1), kFewThreads, (p.tokens + p.sequences) * sizeof(double), st, p, o, inv_count);
  }
  uint64_t need;
  lay_out(nullptr, p.tokens, p.sequences, true, &need);
  return with_workspace(workspace, workspace_bytes, need, st, [&](void* base) {
    const Workspace w = lay_out(base, p.tokens, p.sequences, true, &need);
    const uint32_t tiles = (uint32_t)tiles_of(p.tokens);
    int rc = launch("fpreference_loss: sums", sums_kernel<Id>, dim3(tiles), kThreads, 0, st, p, w, o);
    if (rc) return rc;
    const uint32_t each = short_ones(p) ? kThreads : kThreads / 32, ctas = (uint32_t)(((uint64_t)p.sequences + each - 1) / each);
    const bool gradient = o.g_logprob && p.tokens;
    rc = launch("fpreference_loss", short_ones(p) ? pairs_kernel<Id, true> : pairs_kernel<Id, false>, dim3(ctas), kThreads, 0, st, p, w, o, inv_count, gradient);
    if (rc || !gradient) return rc;
    return launch("fpreference_loss: gradient", pairs_grad_kernel<Id>, dim3((unsigned)((p.tokens + kPass - 1) / kPass) + 1), kThreads, 0, st, p, w, o, ctas,
                  aligned16(o.g_logprob));
  });
}

}  // namespace
}  // namespace polar_b200

using namespace polar_b200;

extern "C" {

uint64_t polar_b200_fpolicy_loss_workspace_bytes(uint64_t tokens, uint64_t sequences) {
  if (tokens > 1ull << 36 || sequences > 0x7fffffffull || few(tokens, sequences, kFewPolicy)) return 0;
  uint64_t bytes;
  lay_out(nullptr, tokens, sequences, false, &bytes);
  return bytes;
}
uint64_t polar_b200_fpreference_loss_workspace_bytes(uint64_t tokens, uint64_t pairs) {
  if (tokens > 1ull << 36 || pairs > 0x3fffffffull || few(tokens, 2 * pairs, kFew)) return 0;
  uint64_t bytes;
  lay_out(nullptr, tokens, 2 * pairs, true, &bytes);
  return bytes;
}

int polar_b200_fpolicy_loss(const polar_b200_policy_batch* b, const polar_b200_policy_options* o, float* loss, float* gLogProb, float* gEntropy,
                            void* workspace, uint64_t workspace_bytes, void* stream) {
  clear_error();
  if (!b || !o || !loss) return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: no batch, options or loss");
  int rc = check_sequences(b->ids, b->offsets, b->id_type, b->tokens, b->sequences);
  if (rc) return rc;
  if (!(o->clip_low >= 0.f && o->clip_low <= 1.f && o->clip_high >= 0.f)) return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: 0 <= clip_low <= 1 and clip_high >= 0 are needed");
  if (!(std::isfinite(o->kl_weight) && std::isfinite(o->entropy_weight) && std::isfinite(o->count) && o->count >= 0.f))
    return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: finite weights and a count of zero or more are needed");
  if (gEntropy && !b->entropy) return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: the entropy's gradient needs the entropy");
  const uint64_t n = b->sequences ? b->tokens : 0;
  if (n && (!b->logProb || !b->oldLogProb || !b->advantage)) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  const uint64_t advantages = b->advantage_per_token ? b->tokens : b->sequences;
  const struct { const void* p; uint64_t bytes; bool by_token; } read[] = {
      {b->logProb, 4 * b->tokens, true}, {b->oldLogProb, 4 * b->tokens, true}, {b->refLogProb, 4 * b->tokens, true}, {b->entropy, 4 * b->tokens, true},
      {b->advantage, 4 * advantages, b->advantage_per_token != 0}, {b->ids, id_bytes(b->id_type) * b->tokens, false},
      {b->offsets, id_bytes(b->id_type) * (b->sequences + 1), false}};
  for (const auto& r : read)
    if (overlaps(gLogProb, 4 * b->tokens, r.p, r.bytes, r.by_token) || overlaps(gEntropy, 4 * b->tokens, r.p, r.bytes, r.by_token) ||
        overlaps(loss, 20, r.p, r.bytes, false))
      return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: what is written overlaps something else");
  if (overlaps(gLogProb, 4 * b->tokens, gEntropy, 4 * b->tokens, false) || overlaps(loss, 20, gLogProb, 4 * b->tokens, false) ||
      overlaps(loss, 20, gEntropy, 4 * b->tokens, false))
    return fail(POLAR_B200_ERR_INVALID, "fpolicy_loss: what is written overlaps something else");
  if (n == 0) return polar_b200_ffill(0.f, loss, 5, stream);
  LaunchDeviceScope on(stream, loss);
  Policy k = {};
  k.logprob = b->logProb, k.old = b->oldLogProb, k.reference = b->refLogProb, k.entropy = b->entropy, k.advantage = b->advantage;
  k.loss = loss, k.g_logprob = gLogProb, k.g_entropy = gEntropy;
  k.high = 1.f + o->clip_high, k.low = 1.f - o->clip_low;
  k.log_high = std::log1p((double)o->clip_high), k.log_low = o->clip_low == 1.f ? -std::numeric_limits<double>::infinity() : std::log1p(-(double)o->clip_low);
  // d and the border are each rounded by 2^-24 of themselves
  k.fp32_high = (float)k.log_high, k.fp32_low = (float)k.log_low;
  k.near = (float)(2.4e-7 * std::max(std::isinf(k.log_high) ? 0.0 : k.log_high, std::isinf(k.log_low) ? 0.0 : -k.log_low));
  k.kl = b->refLogProb ? o->kl_weight : 0.f, k.bonus = b->entropy ? o->entropy_weight : 0.f, k.count = o->count;
  k.by_sequence = o->by_sequence, k.per_token = b->advantage_per_token;
  return with_ids(b->id_type, [&](auto id) {
    using Id = decltype(id);
    const Packed<Id> p = {static_cast<const Id*>(b->ids), static_cast<const Id*>(b->offsets), b->tokens, (uint32_t)b->sequences};
    return run_policy(p, k, workspace, workspace_bytes, as_stream(stream));
  });
}

int polar_b200_fpreference_loss(const float* logProb, const float* refLogProb, const void* ids, const void* offsets, int id_type, uint64_t tokens,
                                uint64_t pairs, const polar_b200_preference_options* o, float* loss, float* rewards, float* gLogProb,
                                void* workspace, uint64_t workspace_bytes, void* stream) {
  clear_error();
  if (!o || !loss) return fail(POLAR_B200_ERR_INVALID, "fpreference_loss: no options or loss");
  if (pairs > 0x3fffffffull) return fail(POLAR_B200_ERR_INVALID, "too many tokens or sequences");
  int rc = check_sequences(ids, offsets, id_type, tokens, 2 * pairs);
  if (rc) return rc;
  if (!(std::isfinite(o->beta) && std::isfinite(o->margin) && o->smoothing >= 0.f && o->smoothing <= 1.f && std::isfinite(o->count) && o->count >= 0.f))
    return fail(POLAR_B200_ERR_INVALID, "fpreference_loss: finite beta and margin, 0 <= smoothing <= 1 and a count of zero or more are needed");
  if (pairs && tokens && !logProb) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  const uint64_t reward_bytes = 8 * pairs;
  const struct { const void* p; uint64_t bytes; } read[] = {{logProb, 4 * tokens}, {refLogProb, 4 * tokens}, {ids, id_bytes(id_type) * tokens},
                                                            {offsets, id_bytes(id_type) * (2 * pairs + 1)}};
  for (const auto& r : read)
    if (overlaps(gLogProb, 4 * tokens, r.p, r.bytes, &r < read + 2) || overlaps(rewards, reward_bytes, r.p, r.bytes, false) ||
        overlaps(loss, 12, r.p, r.bytes, false))
      return fail(POLAR_B200_ERR_INVALID, "fpreference_loss: what is written overlaps something else");
  if (overlaps(rewards, reward_bytes, gLogProb, 4 * tokens, false) || overlaps(loss, 12, gLogProb, 4 * tokens, false) || overlaps(loss, 12, rewards, reward_bytes, false))
    return fail(POLAR_B200_ERR_INVALID, "fpreference_loss: what is written overlaps something else");
  if (pairs == 0) return polar_b200_ffill(0.f, loss, 3, stream);
  LaunchDeviceScope on(stream, loss);
  const Pairs k = {logProb, refLogProb, loss, rewards, gLogProb, o->beta, o->smoothing, o->margin, o->count, o->average};
  return with_ids(id_type, [&](auto id) {
    using Id = decltype(id);
    const Packed<Id> p = {static_cast<const Id*>(ids), static_cast<const Id*>(offsets), tokens, (uint32_t)(2 * pairs)};
    return run_pairs(p, k, workspace, workspace_bytes, as_stream(stream));
  });
}

}  // extern "C"
