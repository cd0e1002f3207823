// Log probabilities of given classes or tokens, the rows' entropies and likeliest alternatives, and the gradient.
//
// With m the row's maximum, d = x - m, S = sum(exp d) and T = sum(exp(d) * d):
//   logSumExp = m + log S,   logProb = d[id] - log S,   entropy = log S - T / S,
// where no term cancels another: d <= 0, so T <= 0 and log S >= 0.  A -inf logit has exp d = 0 and no part in T.
// Of a row that is nearly certain S is 1 and a little, and log S that little: the one largest element is left out of the sum, so that nothing is
// rounded beside its 1, and log S = log1p(the rest).
#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxTop = 32;

// The id of a row: whole in 0 .. classes - 1, kPadding below zero, kWrong for anything else.
constexpr int64_t kPadding = -1, kWrong = -2;
__device__ __forceinline__ int64_t read_id(const void* ids, int type, uint64_t row, uint64_t classes) {
  int64_t id;
  if (type == POLAR_B200_IDS_F32) {
    const float f = static_cast<const float*>(ids)[row];
    if (f < 0.f) return kPadding;
    if (!(f < (float)classes) || f != truncf(f)) return kWrong;
    id = (int64_t)f;
  } else {
    id = type == POLAR_B200_IDS_I32 ? static_cast<const int32_t*>(ids)[row] : static_cast<const int64_t*>(ids)[row];
  }
  return id < 0 ? kPadding : (uint64_t)id < classes ? id : kWrong;
}
__device__ __forceinline__ void write_id(void* ids, int type, uint64_t at, uint32_t id) {
  if (type == POLAR_B200_IDS_F32) static_cast<float*>(ids)[at] = (float)id;
  else if (type == POLAR_B200_IDS_I32) static_cast<int32_t*>(ids)[at] = (int32_t)id;
  else static_cast<int64_t*>(ids)[at] = (int64_t)id;
}

// An order over (value, index): larger values first, of equal ones the lower index; NaN above everything, -0 as +0.
// Never 0, which stands for "none".
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_of(float v, uint32_t index) { return (uint64_t)ordered(v) << 32 | (uint32_t)~index; }

// What the id, the sums and the alternatives of a row become.
struct Results {
  const void* ids;
  int id_type;
  float *logprob, *entropy, *logsumexp;
  void* top_ids;
  float* top_logprob;
  uint32_t top;
};

// ---- the running sums ---------------------------------------------------------------------------------
// A thread's (or a row's) largest element so far (-inf: none), S without the 1 of that element, and T; both relative to m, the largest clamped to finite
// values, so that no difference from it is a NaN where an element is -inf.
constexpr float kLowest = -3.402823466e38f;
struct Running {
  float top = -INFINITY, m = kLowest, s = 0.f, t = 0.f;
  __device__ __forceinline__ bool any() const { return top > -INFINITY; }
  __device__ __forceinline__ float log_sum() const { return log1pf(s); }
};
// d = x - m never enters below this: the exponential is zero there, and zero times d is zero and no NaN.  NaN stays NaN.
__device__ __forceinline__ float at_least(float d) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(d) : "f"(-1000.f));
  return d;
}
__device__ __forceinline__ float exp_fast(float d) {       // 2^(d log2 e): off by |d| 2^-24 from the product and 2 ulp
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.4426950408889634f));
  return e;
}
// To a larger top; `before`: whether the largest so far, which is of the sum now, was this thread's.
__device__ __forceinline__ void raise_to(Running& r, float top, bool before) {
  const float m = fmaxf(top, kLowest), d = at_least(r.m - m), f = exp_fast(d), sum = r.s + (before ? 1.f : 0.f);
  r.t = f * (r.t + d * sum);
  r.s = f * sum;
  r.m = m;
  r.top = top;
}
// The same sums two elements at a time.
struct RunningPair {
  float top = -INFINITY, m = kLowest;
  Pair s = 0, t = 0;
  __device__ __forceinline__ Running joined() const {
    Running r;
    r.top = top, r.m = m, r.s = halves(s).x + halves(s).y, r.t = halves(t).x + halves(t).y;
    return r;
  }
};
__device__ __forceinline__ void raise_to(RunningPair& r, float top, bool before) {
  Running one = r.joined();
  raise_to(one, top, before);
  r.top = one.top, r.m = one.m, r.s = pair(one.s, 0.f), r.t = pair(one.t, 0.f);
}
__device__ __forceinline__ void add(RunningPair& r, float a, float b) {
  const float2 x = halves(add2(pair(a, b), pair(-r.m, -r.m)));
  const Pair d = pair(at_least(x.x), at_least(x.y));
  const float2 w = halves(mul2(d, pair(1.4426950408889634f, 1.4426950408889634f)));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(w.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(w.y));
  const Pair p = pair(e.x, e.y);
  r.s = add2(r.s, p);
  r.t = fma2(p, d, r.t);
}
__device__ __forceinline__ void add(RunningPair& r, float4 v) { add(r, v.x, v.y), add(r, v.z, v.w); }
__device__ __forceinline__ float max4(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
// The largest of the lanes' values (NaN only where all are).
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  if (LANES == 32) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
  }
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
// The larger and the smaller of two; NaN for both where one is.
__device__ __forceinline__ void order(float& high, float& low) {
  const float a = high, b = low;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(high) : "f"(a), "f"(b));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(low) : "f"(a), "f"(b));
}
// Whether the lane is the first of `LANES` neighbouring ones for which something holds.
template <int LANES>
__device__ __forceinline__ bool first_of(bool holds) {
  const uint32_t lane = threadIdx.x & 31, group = LANES == 32 ? 0xffffffffu : ((1u << LANES % 32) - 1) << (lane & ~(LANES - 1));
  return lane + 1 == (uint32_t)__ffs(__ballot_sync(0xffffffffu, holds) & group);
}
// The lanes' sums, which are around the same maximum.  A row with +inf is NaN.
template <int LANES>
__device__ __forceinline__ void sum_over(Running& r) {
#pragma unroll
  for (int off = LANES / 2; off > 0; off >>= 1) {
    r.s += __shfl_xor_sync(0xffffffffu, r.s, off);
    r.t += __shfl_xor_sync(0xffffffffu, r.t, off);
  }
  if (r.top == INFINITY) r.s = NAN;
}
// The sums of `LANES` neighbouring lanes, in each of them: of the lanes that have met the largest element, the first keeps its 1 out.
template <int LANES>
__device__ __forceinline__ Running join(const Running& r) {
  Running all;
  all.top = lanes_max<LANES>(r.top);
  all.m = fmaxf(all.top, kLowest);
  const bool keeps_out = first_of<LANES>(r.any() && r.top == all.top);
  const float d = at_least(r.m - all.m), f = exp_fast(d), sum = r.s + (r.any() && !keeps_out ? 1.f : 0.f);
  all.s = f * sum;
  all.t = f * (r.t + d * sum);
  sum_over<LANES>(all);
  return all;
}

// ---- a row as vectors -----------------------------------------------------------------------------------
// Rows begin where they begin (an odd number of classes, a pitch): vector i holds the elements 4 i - shift ... + 3, so that all but the
// first and the last one are whole and on a 16-byte boundary.
struct Row {
  const float* aligned;
  uint32_t shift, classes, vectors, whole_from, whole_to;
  __device__ __forceinline__ Row(const float* x, uint32_t n) {
    shift = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 15) >> 2;
    aligned = x - shift;
    classes = n;
    vectors = (uint32_t)(((uint64_t)n + shift + 3) >> 2);
    whole_from = shift ? 1 : 0;
    whole_to = (uint32_t)(((uint64_t)n + shift) >> 2);
  }
  __device__ __forceinline__ float4 whole(uint32_t i) const { return reinterpret_cast<const float4*>(aligned)[i]; }
  __device__ __forceinline__ bool is_whole(uint32_t i) const { return i >= whole_from && i < whole_to; }
  // whether component c of vector i is an element
  __device__ __forceinline__ bool has(uint32_t i, uint32_t c) const {
    const uint64_t e = 4ull * i + c;
    return e >= shift && e < (uint64_t)classes + shift;
  }
  __device__ __forceinline__ uint32_t element(uint32_t i, uint32_t c) const { return 4 * i + c - shift; }
  // a vector at the edge, -inf where there is no element
  __device__ __forceinline__ float4 edge(uint32_t i) const {
    const float* p = aligned + 4ull * i;
    return make_float4(has(i, 0) ? p[0] : -INFINITY, has(i, 1) ? p[1] : -INFINITY, has(i, 2) ? p[2] : -INFINITY, has(i, 3) ? p[3] : -INFINITY);
  }
  __device__ __forceinline__ float4 vector(uint32_t i) const { return is_whole(i) ? whole(i) : edge(i); }
};

// ---- the alternatives -----------------------------------------------------------------------------------
// One pass finds them too.  If `top` threads or more have met a maximum of at least some bound, the `top` largest elements are all of at
// least that bound.  So after the first few vectors, and again whenever the part of the row that has been seen has grown fourfold, the
// threads' maxima give a bound (a search by counting them), and from then on an element that reaches it is kept: about 4 `top` for each
// fourfold, whatever the row's length.  Where a chunk holds all of a row, the bound is one of its elements.  At the end what is kept is thinned
// out by a bound of its own, and what that leaves (little more than `top`) is placed by counting what is above it.  -inf is never kept: where fewer than `top` elements are above it, the first of it follow.  A row where more is kept
// than there is room for (equal logits by the hundred), or with a NaN, which no maximum shows, is looked through a second time by
// warps that sort as they go.
constexpr int kInFlight = 4;                               // vectors of a thread in flight
constexpr uint32_t kFewTop = 8;
constexpr uint32_t kPlaced = 48;                           // as many a part of a warp places right away, by counting
__device__ __forceinline__ float float_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// The largest bound, nearly, that `top` of the LANES N keys of neighbouring lanes of a warp reach (all lanes take part; each group finds its
// own).  Keys of kLowest count for vectors not met; with fewer keys than `top` that is the bound, and everything reaches it.  Found by halving, the first
// BY_VALUE steps by value, where numbers of a short row are told apart sooner (60000 x 400 with 20 alternatives: 73 us, without 77, since the steps
// by order go through all the powers of two down to zero); by order it takes 32 steps at most, whatever the numbers are.
template <int BY_VALUE, int LANES, int N>
__device__ __forceinline__ float bound_of(const uint32_t (&key)[N], uint32_t top) {
  const uint32_t lowest = ordered(kLowest);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) most = max(most, key[i]);
  if (top <= kFewTop && top <= LANES) {                    // few: the largest key of the lanes, the next, ...
    uint32_t mine = most, largest = 0;
    for (uint32_t k = 0; k < top; ++k) {
      largest = mine;
      if (LANES == 32) {
        largest = __reduce_max_sync(0xffffffffu, largest);
      } else {
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, off));
      }
      if (mine == largest) mine = 0;                       // (more than one lane at a time where maxima are equal: 0 in the end, at most)
    }
    return float_of(max(largest, ordered(kLowest)));
  }
  // the numbers met, the largest and the least of them
  uint32_t least = ~0u, met = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) least = min(least, key[i] > lowest ? key[i] : ~0u), met += key[i] > lowest;
  if (LANES == 32) {
    most = __reduce_max_sync(0xffffffffu, most);
    least = __reduce_min_sync(0xffffffffu, least);
    met = __reduce_add_sync(0xffffffffu, met);
  } else {
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) {
      most = max(most, __shfl_xor_sync(0xffffffffu, most, off));
      least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
      met += __shfl_xor_sync(0xffffffffu, met, off);
    }
  }
  // `top` or more reach lo, fewer reach hi + 1
  uint32_t lo = met < top ? lowest : least, hi = met < top ? lowest : most;
  for (int step = 0; LANES == 32 ? lo < hi : __any_sync(0xffffffffu, lo < hi); ++step) {
    uint32_t mid = hi - (hi - lo) / 2;
    if (step < BY_VALUE) mid = min(max(ordered(0.5f * float_of(lo) + 0.5f * float_of(hi)), lo + 1), hi);
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += key[i] >= mid;
    if (LANES == 32) {
      n = __reduce_add_sync(0xffffffffu, n);
    } else {
#pragma unroll
      for (int off = LANES / 2; off > 0; off >>= 1) n += __shfl_xor_sync(0xffffffffu, n, off);
    }
    if (n >= top) lo = mid;
    else hi = mid - 1;
    if (n >= top && n <= top + top / 4 + 1) hi = lo;
  }
  return float_of(lo);
}

// What a team (a CTA, a warp or a part of one) keeps.
struct Kept {
  unsigned long long* rank;
  uint32_t* count;                                         // goes on beyond the room
  uint32_t room;
};

// A chunk: kInFlight vectors of a thread, `stride` apart, all of them on their way at once.
struct Chunk {
  float4 v[kInFlight];
  float high[kInFlight], rest[kInFlight][3];               // of each vector the largest element and the others (order_all)

  // `inner`: all of them are whole.  -inf where there is no element.
  __device__ __forceinline__ void load(const Row& row, uint32_t i, uint32_t stride, bool inner, bool edges) {
    if (inner) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) v[u] = row.whole(i + u * stride);
      return;
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      v[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (row.is_whole(i + u * stride)) v[u] = row.whole(i + u * stride);
    }
    if (edges) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (i + u * stride < row.vectors && !row.is_whole(i + u * stride)) v[u] = row.edge(i + u * stride);
    }
  }
  // The largest element (a NaN is none), and of each vector the largest met so far.
  template <bool TOP>
  __device__ __forceinline__ float largest(float (&maxima)[kInFlight]) const {
    float m[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      m[u] = max4(v[u]);
      if (TOP) maxima[u] = fmaxf(maxima[u], m[u]);
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  }
  // The elements with the largest of all in high[0], the other vectors' in high[1] and so on; all are NaN that one of these is ordered with.
  __device__ __forceinline__ void order_all() {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      float a = v[u].x, b = v[u].y, c = v[u].z, d = v[u].w;
      order(a, b), order(c, d), order(a, c);
      high[u] = a, rest[u][0] = b, rest[u][1] = c, rest[u][2] = d;
    }
    order(high[0], high[1]), order(high[2], high[3]), order(high[0], high[2]);
  }
  // The elements that reach the bound.
  __device__ __forceinline__ void keep(const Kept& kept, float most, float bound, const Row& row, uint32_t i, uint32_t stride) const {
    if (!(most >= bound && *(volatile uint32_t*)kept.count <= kept.room)) return;
    uint32_t which = 0;                                    // of the 16 elements
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      which |= (v[u].x >= bound ? 1u << 4 * u : 0) | (v[u].y >= bound ? 2u << 4 * u : 0) | (v[u].z >= bound ? 4u << 4 * u : 0) |
               (v[u].w >= bound ? 8u << 4 * u : 0);
    uint32_t at = atomicAdd(kept.count, (uint32_t)__popc(which));
    while (which) {
      const uint32_t e = __ffs(which) - 1, u = e >> 2;
      which &= which - 1;
      const float4 x = u & 2 ? (u & 1 ? v[3] : v[2]) : (u & 1 ? v[1] : v[0]);
      const float value = e & 2 ? (e & 1 ? x.w : x.z) : (e & 1 ? x.y : x.x);
      if (at < kept.room) kept.rank[at] = rank_of(value, row.element(i + u * stride, e & 3));
      ++at;
    }
  }
  // The elements enter the sums.  `left`: the number of vectors from the first of the warp's to the row's end, where not `all` are there.
  __device__ __forceinline__ void add_to(RunningPair& r, bool all, uint32_t left, uint32_t stride) const {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      if (all || u * stride < left) add(r, v[u]);
  }
  // The same with `instead` in the place of the largest one (order_all).
  __device__ __forceinline__ void add_to(RunningPair& r, float instead, bool all, uint32_t left, uint32_t stride) const {
    add(r, instead, high[1]);
    add(r, high[2], high[3]);
#pragma unroll
    for (int u = 0; u < kInFlight; u += 2)                 // (two vectors at a time)
      if (all || u * stride < left) {
        add(r, rest[u][0], rest[u][1]);
        add(r, rest[u][2], rest[u + 1][0]);
        add(r, rest[u + 1][1], rest[u + 1][2]);
      }
  }
};

// The sums of a warp over the vectors first, first + stride, ... of a row, joined; `base` is the first of the warp's
// `first`s, `chunks` the same for a warp (or, where bounds are a matter for the CTA, for all of it).  All lanes go by the largest element that one of
// them has met: a chunk that has a larger one is rare, and only such a chunk is ordered, so that its largest can stay out of the sum (all chunks
// ordered, by each lane's own largest: 200 x 60000 10.9 us, so 9.8).  find_bound(maxima, chunk) takes the whole team.
template <bool TOP, class FindBound>
__device__ __forceinline__ Running scan(const Row& row, uint32_t base, uint32_t first, uint32_t stride, uint32_t chunks, float (&maxima)[kInFlight],
                                        const Kept& kept, FindBound find_bound) {
  RunningPair r;
  float bound = INFINITY;
  const uint32_t chunk = kInFlight * stride, lane = threadIdx.x & 31;
  uint32_t next_bound = 0, holder = 32;                    // the lane that has met the largest element
  const bool edges = row.whole_from != 0 || row.whole_to != row.vectors;
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) maxima[u] = kLowest;
  for (uint32_t n = 0; n < chunks; ++n) {
    const uint32_t i = first + n * chunk, left = row.vectors > base + n * chunk ? row.vectors - (base + n * chunk) : 0;
    const bool inner = n > 0 && (n + 1) * chunk <= row.whole_to;   // all vectors of the chunk are whole
    Chunk c;
    c.load(row, i, stride, inner, edges);
    const float most = c.template largest<TOP>(maxima);
    if (TOP) {
      if (n == next_bound) {
        bound = find_bound(maxima, c.v);
        next_bound = 4 * n + 3;
      }
      c.keep(kept, most, bound, row, i, stride);
    }
    if (__any_sync(0xffffffffu, most > r.top)) {
      const float top = lanes_max<32>(most);
      raise_to(r, top, lane == holder);
      holder = __ffs(__ballot_sync(0xffffffffu, most == top)) - 1;
      c.order_all();
      c.add_to(r, lane == holder ? -INFINITY : c.high[0], inner, left, stride);
    } else {
      c.add_to(r, inner, left, stride);
    }
  }
  Running all = r.joined();
  sum_over<32>(all);
  return all;
}
// The same of rows that are one chunk of `LANES` lanes.
template <int LANES, bool TOP, class FindBound>
__device__ __forceinline__ Running scan_once(const Row& row, uint32_t member, const Kept& kept, FindBound find_bound) {
  Chunk c;
  float maxima[kInFlight];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u) maxima[u] = kLowest;
  c.load(row, member, LANES, false, row.whole_from != 0 || row.whole_to != row.vectors);
  const float most = c.template largest<TOP>(maxima);
  if (TOP) c.keep(kept, most, find_bound(maxima, c.v), row, member, LANES);
  RunningPair r;
  r.top = lanes_max<LANES>(most);
  if (r.top != r.top) r.top = -INFINITY;                   // (nothing but NaN)
  r.m = fmaxf(r.top, kLowest);
  c.order_all();
  c.add_to(r, first_of<LANES>(r.top > -INFINITY && most == r.top) ? -INFINITY : c.high[0], false, row.vectors, LANES);
  Running all = r.joined();
  sum_over<LANES>(all);
  return all;
}

// Of `n` ranks in shared memory, up to ROOM, those stay that may be among the `top` largest, in front: a warp looks for a bound that `top` of them
// reach and few more, by counting them, as above.  Returns how many stay.
template <uint32_t ROOM>
__device__ __forceinline__ uint32_t thin_out(unsigned long long* ranks, uint32_t n, uint32_t top, uint32_t lane) {
  const uint32_t enough = top + top / 4 + 1;
  if (n <= enough || n <= 32) return n;                    // (not worth it)
  constexpr uint32_t kEach = ROOM / 32;
  unsigned long long rank[kEach];
  uint32_t key[kEach], most = 0, least = ~0u;
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    rank[i] = 32 * i + lane < n ? ranks[32 * i + lane] : 0;
    key[i] = (uint32_t)(rank[i] >> 32);
    most = max(most, key[i]);
    if (key[i]) least = min(least, key[i]);
  }
  uint32_t lo = __reduce_min_sync(0xffffffffu, least), hi = __reduce_max_sync(0xffffffffu, most);   // all reach lo; of hi + 1 none
  while (lo < hi) {
    const uint32_t mid = hi - (hi - lo) / 2;
    uint32_t reach = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) reach += key[i] >= mid;
    reach = __reduce_add_sync(0xffffffffu, reach);
    if (reach >= top) lo = mid;
    else hi = mid - 1;
    if (reach >= top && reach <= enough) hi = lo;
  }
  uint32_t total = 0;
  __syncwarp();
#pragma unroll
  for (uint32_t i = 0; i < kEach; ++i) {
    const uint32_t up = __ballot_sync(0xffffffffu, key[i] >= lo && key[i] != 0);
    if (up >> lane & 1) ranks[total + __popc(up & ((1u << lane) - 1))] = rank[i];
    total += __popc(up);
  }
  __syncwarp();
  return total;
}

// A warp's sorted list of ranks, the largest in lane 0; takes the elements of one vector per lane.
__device__ __forceinline__ void take(unsigned long long& list, const Row& row, uint32_t i, uint32_t top, uint32_t lane) {
  const float4 v = i < row.vectors ? row.vector(i) : make_float4(0.f, 0.f, 0.f, 0.f);
  const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (uint32_t c = 0; c < 4; ++c) {
    const unsigned long long rank = i < row.vectors && row.has(i, c) ? rank_of(x[c], row.element(i, c)) : 0;
    uint32_t left = __ballot_sync(0xffffffffu, rank > __shfl_sync(0xffffffffu, list, top - 1));
    while (left) {
      const unsigned long long r = __shfl_sync(0xffffffffu, rank, __ffs(left) - 1), above = __shfl_up_sync(0xffffffffu, list, 1);
      const uint32_t at = __popc(__ballot_sync(0xffffffffu, list > r));
      if (lane == at) list = r;
      else if (lane > at) list = above;
      left &= left - 1;
      left &= __ballot_sync(0xffffffffu, rank > __shfl_sync(0xffffffffu, list, top - 1));
    }
  }
}
// The first `wanted` elements of -inf among the vectors that a team has, in their order, one after the other into `to`; by one warp.
__device__ __forceinline__ void take_shut_out(unsigned long long* to, uint32_t wanted, const Row& row, uint32_t begin, uint32_t width, uint32_t stride,
                                              uint32_t lane) {
  uint32_t found = 0;
  for (uint32_t j = lane;; j += 32) {
    const uint32_t i = j / width * stride + begin + j % width;
    if (!__any_sync(0xffffffffu, i < row.vectors) || found >= wanted) return;
    const float4 v = i < row.vectors ? row.vector(i) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c) mine += x[c] == -INFINITY && i < row.vectors && row.has(i, c);
    uint32_t at = mine;                                    // lanes lie in the order of their elements
#pragma unroll
    for (int off = 1; off < 32; off *= 2) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, at, off);
      if ((int)lane >= off) at += o;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, at, 31);
    at += found - mine;
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c)
      if (x[c] == -INFINITY && i < row.vectors && row.has(i, c)) {
        if (at < wanted) to[at] = rank_of(x[c], row.element(i, c));
        ++at;
      }
    found += all;
  }
}
__device__ __forceinline__ void write_row(const Results& o, uint64_t row, int64_t id, float given, const Running& r) {
  const float log_sum = r.log_sum();
  const bool dead = !r.any() && r.s == 0.f;                // (NaN is none)
  if (o.logprob) o.logprob[row] = id == kPadding ? 0.f : id == kWrong ? NAN : dead ? -INFINITY : given - r.m - log_sum;
  if (o.entropy) o.entropy[row] = dead ? 0.f : log_sum - r.t / (1.f + r.s);
  if (o.logsumexp) o.logsumexp[row] = dead ? -INFINITY : r.m + log_sum;
}
__device__ __forceinline__ void write_top(const Results& o, uint64_t row, uint32_t at, uint32_t id, float x, const Running& r, float log_sum) {
  if (o.top_ids) write_id(o.top_ids, o.id_type, row * o.top + at, id);
  if (o.top_logprob) o.top_logprob[row * o.top + at] = !r.any() && r.s == 0.f ? -INFINITY : x - r.m - log_sum;
}
__device__ __forceinline__ void write_top(const Results& o, uint64_t row, uint32_t at, unsigned long long rank, const Running& r, float log_sum) {
  write_top(o, row, at, ~(uint32_t)rank, float_of((uint32_t)(rank >> 32)), r, log_sum);
}

// Many classes: a CTA per row, or a cluster of CTAs where there are few rows.
template <int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprob_wide_kernel(const float* logits, uint32_t classes, uint64_t pitch, Results o) {
  constexpr uint32_t kWarps = THREADS / 32, kRoom = TOP ? 512 : 1, kTop = TOP ? kMaxTop : 1;
  __shared__ float part[3][kWarps], joined[3];
  __shared__ unsigned long long kept_ranks[kRoom], left[kRoom], sorted[kTop], theirs[8 * kTop];
  __shared__ uint32_t n_kept, n_left, keys[2][TOP ? THREADS : 1];
  pdl_enter();
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ctas = gridDim.y, rank = blockIdx.y;
  const uint64_t r = blockIdx.x;
  const Row row(logits + r * pitch, classes);
  const uint32_t first = rank * THREADS + tid, stride = ctas * THREADS;
  int64_t id = kPadding;
  float given = 0.f;
  if (rank == 0 && tid == 0 && o.logprob) {
    id = read_id(o.ids, o.id_type, r, classes);
    if (id >= 0) given = logits[r * pitch + id];
  }
  if (TOP) {
    if (tid == 0) n_kept = n_left = 0;
    if (tid < kMaxTop) sorted[tid] = 0;
  }
  int turn = 0;
  // (two arrays in turn: a barrier is between a round's reads and the writes of the next but one)
  auto find_bound = [&](const float (&maxima)[kInFlight], const float4 (&)[kInFlight]) {
    uint32_t k[4];                                         // of 128 groups of threads: enough for 32 alternatives
    keys[turn][tid] = ordered(fmaxf(fmaxf(maxima[0], maxima[1]), fmaxf(maxima[2], maxima[3])));
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      k[i] = keys[turn][32 * i + lane];
#pragma unroll
      for (uint32_t j = 128; j < THREADS; j += 128) k[i] = max(k[i], keys[turn][j + 32 * i + lane]);
    }
    turn ^= 1;
    return bound_of<0, 32>(k, o.top);
  };
  float maxima[kInFlight];
  const uint32_t chunks = (row.vectors + kInFlight * stride - 1) / (kInFlight * stride);
  Running all = scan<TOP>(row, first - lane, first, stride, chunks, maxima, Kept{kept_ranks, &n_kept, kRoom}, find_bound);
  if (lane == 0) part[0][warp] = all.top, part[1][warp] = all.s, part[2][warp] = all.t;
  __syncthreads();
  all = Running();
  if (lane < kWarps) all.top = part[0][lane], all.m = fmaxf(all.top, kLowest), all.s = part[1][lane], all.t = part[2][lane];
  all = join<32>(all);
  if (TOP) {
    const uint32_t n = n_kept;                             // the same for all threads, as what hangs on it
    if (n <= kRoom && all.s == all.s) {
      const float4 none[kInFlight] = {};
      const float bound = n > 64 ? find_bound(maxima, none) : kLowest;
      for (uint32_t i = tid; i < n; i += THREADS)
        if (kept_ranks[i] >= (uint64_t)ordered(bound) << 32) left[atomicAdd(&n_left, 1u)] = kept_ranks[i];
    } else {
      unsigned long long list = 0;
      for (uint32_t j = warp * 32 + lane;; j += THREADS) {
        const uint32_t i = j / THREADS * stride + rank * THREADS + j % THREADS;
        if (!__any_sync(0xffffffffu, i < row.vectors)) break;
        take(list, row, i, o.top, lane);
      }
      if (lane < o.top && list) left[atomicAdd(&n_left, 1u)] = list;
    }
    __syncthreads();
    const uint32_t total = n_left;
    for (uint32_t i = tid; i < total; i += THREADS) {      // no two ranks are alike: a place for each
      uint32_t above = 0;
      const unsigned long long mine = left[i];
      for (uint32_t j = 0; j < total; ++j) above += left[j] > mine;
      if (above < o.top) sorted[above] = mine;
    }
    if (total < o.top && warp == 0) take_shut_out(sorted + total, o.top - total, row, rank * THREADS, THREADS, stride, lane);
    __syncthreads();
  }
  if (ctas == 1) {
    if (tid == 0) write_row(o, r, id, given, all);
    if (TOP && tid < o.top) write_top(o, r, tid, sorted[tid], all, all.log_sum());
    return;
  }
  if (tid == 0) joined[0] = all.top, joined[1] = all.s, joined[2] = all.t;
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  if (rank == 0) {
    all = Running();
    if (lane < ctas) {
      all.top = ld_cluster(&joined[0], lane), all.s = ld_cluster(&joined[1], lane), all.t = ld_cluster(&joined[2], lane);
      all.m = fmaxf(all.top, kLowest);
    }
    all = join<32>(all);
    if (tid == 0) write_row(o, r, id, given, all);
    if (TOP) {
      const uint32_t total = ctas * o.top;
      for (uint32_t i = tid; i < total; i += THREADS)
        theirs[i] = __double_as_longlong(ld_cluster(reinterpret_cast<const double*>(&sorted[i % o.top]), i / o.top));
      __syncthreads();
      for (uint32_t i = tid; i < total; i += THREADS) {
        uint32_t above = 0;
        const unsigned long long mine = theirs[i];
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) {                 // each list is sorted: how many of it are above, a halving at a time
          uint32_t n = 0;
#pragma unroll
          for (uint32_t step = 32; step > 0; step /= 2)
            if (c < ctas && n + step <= o.top && theirs[c * o.top + n + step - 1] > mine) n += step;
          above += n;
        }
        if (above < o.top && mine) write_top(o, r, above, mine, all, all.log_sum());
      }
    }
  }
  cluster_arrive();                                        // nobody leaves while its shared memory may still be read
  cluster_wait();
}

// The vectors of a row, at most: rows that begin elsewhere on a boundary may have one more or less.
__host__ __device__ constexpr uint32_t chunk_vectors(uint32_t classes) { return (classes + 6) / 4; }

// A warp per row or, for short rows, LANES lanes.  ONCE: a row is one chunk, whose largest element is known before the sums (60000 x 400 with five
// alternatives 51 us, by the loop 58).  As many CTAs on an SM as do without spills.
template <int LANES, bool TOP, bool ONCE>
__global__ void __launch_bounds__(kThreads, TOP ? 4 : ONCE ? 6 : 5) logprob_warp_kernel(const float* logits, uint32_t rows, uint32_t classes, uint64_t pitch, Results o) {
  constexpr uint32_t kRoom = !TOP ? 1 : LANES == 32 ? 512 : 128, kTeams = kThreads / LANES, kRows = 32 / LANES;
  __shared__ unsigned long long kept_ranks[kTeams][kRoom];
  __shared__ uint32_t n_kept[kTeams];
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, team = threadIdx.x / LANES, member = threadIdx.x % LANES;
  const uint64_t first = ((uint64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kRows;   // the warp's first row
  if (first >= rows) return;
  const uint64_t r = first + lane / LANES;
  const bool live = r < rows;
  const Row row(logits + (live ? r : first) * pitch, classes);   // (lanes without a row of their own look at the warp's first)
  int64_t id = kPadding;
  float given = 0.f;
  if (member == 0 && o.logprob && live) {
    id = read_id(o.ids, o.id_type, r, classes);
    if (id >= 0) given = logits[r * pitch + id];
  }
  unsigned long long* kept = kept_ranks[team];
  if (TOP && member == 0) n_kept[team] = 0;
  __syncwarp();
  auto find_bound = [&](const float (&maxima)[kInFlight], const float4 (&v)[kInFlight]) {
    if (o.top > kFewTop && classes <= kPlaced) return kLowest;
    // Where the row is here and has few vectors beside `top`, a bound of its elements, which few more than `top` reach (60000 x 200 with 32: 71 us, of
    // the vectors' maxima 81; x 400 with 20, from where on it is these, 73 either way)
    if (o.top > kFewTop && ONCE && classes < 8 * o.top) {
      uint32_t k[4 * kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        k[4 * u] = ordered(fmaxf(v[u].x, kLowest)), k[4 * u + 1] = ordered(fmaxf(v[u].y, kLowest));
        k[4 * u + 2] = ordered(fmaxf(v[u].z, kLowest)), k[4 * u + 3] = ordered(fmaxf(v[u].w, kLowest));
      }
      return bound_of<6, LANES>(k, o.top);
    }
    uint32_t k[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) k[u] = ordered(maxima[u]);
    return bound_of<6, LANES>(k, o.top);
  };
  const Kept to{kept, &n_kept[team], kRoom};
  Running all;
  if constexpr (ONCE) {
    all = scan_once<LANES, TOP>(row, member, to, find_bound);
  } else {
    float maxima[kInFlight];
    const uint32_t chunks = (chunk_vectors(classes) + kInFlight * LANES - 1) / (kInFlight * LANES);
    all = scan<TOP>(row, 0, member, LANES, chunks, maxima, to, find_bound);
  }
  if (member == 0 && live) write_row(o, r, id, given, all);
  if (!TOP) return;
  __syncwarp();
  const uint32_t n = live ? n_kept[team] : o.top;
  const bool sorts = live && (n > kRoom || all.s != all.s);
  const bool simple = !sorts && n >= o.top && n <= (LANES == 32 ? 64 : kPlaced);
  const float log_sum = all.log_sum();
  if (simple && live) {                                    // few: each team places its own, by counting what is above
    for (uint32_t i = member; i < n; i += LANES) {
      uint32_t above = 0;
      const unsigned long long mine = kept[i];
      for (uint32_t j = 0; j < n; ++j) above += kept[j] > mine;
      if (above < o.top) write_top(o, r, above, mine, all, log_sum);
    }
  }
  uint32_t others = __ballot_sync(0xffffffffu, live && !simple && member == 0);
  if (others == 0) return;
  // the other rows one after the other, by the whole warp
  for (; others; others &= others - 1) {
    const int who = __ffs(others) - 1;
    const uint64_t q = first + who / LANES;
    Running sums;
    sums.top = __shfl_sync(0xffffffffu, all.top, who), sums.m = __shfl_sync(0xffffffffu, all.m, who), sums.s = __shfl_sync(0xffffffffu, all.s, who);
    const float its_log_sum = __shfl_sync(0xffffffffu, log_sum, who);
    if (__shfl_sync(0xffffffffu, (int)sorts, who)) {
      const Row its(logits + q * pitch, classes);
      unsigned long long list = 0;
      for (uint32_t i = lane; i - lane < its.vectors; i += 32) take(list, its, i, o.top, lane);
      if (lane < o.top) write_top(o, q, lane, list, sums, its_log_sum);
      continue;
    }
    unsigned long long* its_kept = kept_ranks[(threadIdx.x - lane + who) / LANES];
    const uint32_t its_n = __shfl_sync(0xffffffffu, n, who);
    const uint32_t total = LANES < 32 || its_n <= 128 ? thin_out<128>(its_kept, its_n, o.top, lane) : thin_out<512>(its_kept, its_n, o.top, lane);
    for (uint32_t i = lane; i < total; i += 64) {          // two of them against all, for each lane
      uint32_t above_a = 0, above_b = 0;
      const unsigned long long a = its_kept[i], b = i + 32 < total ? its_kept[i + 32] : 0;
#pragma unroll 4
      for (uint32_t j = 0; j < total; ++j) {
        const unsigned long long other = its_kept[j];
        above_a += other > a;
        above_b += other > b;
      }
      if (above_a < o.top) write_top(o, q, above_a, a, sums, its_log_sum);
      if (above_b < o.top && b) write_top(o, q, above_b, b, sums, its_log_sum);
    }
    if (total < o.top) {
      const Row its(logits + q * pitch, classes);
      __syncwarp();
      take_shut_out(its_kept, o.top - total, its, 0, 32, 32, lane);
      __syncwarp();
      if (lane + total < o.top) write_top(o, q, lane + total, its_kept[lane], sums, its_log_sum);
    }
    __syncwarp();
  }
}

// Up to kThreadClasses classes: a thread per row, its logits in registers (65536 x 10: 2.8 us; x 32, where 32 threads that each read a float of
// their row touch as many cache lines at a time, 12.7, with eight lanes per row 7.5).
constexpr uint32_t kThreadClasses = 16, kThreadRows = 128;
template <int MOST>
__global__ void __launch_bounds__(kThreadRows) logprob_thread_kernel(const float* logits, uint32_t rows, uint32_t classes, uint64_t pitch, Results o) {
  pdl_enter();
  const uint64_t r = (uint64_t)blockIdx.x * kThreadRows + threadIdx.x;
  if (r >= rows) return;
  const float* x = logits + r * pitch;
  float v[MOST];
#pragma unroll
  for (int c = 0; c < MOST; ++c) v[c] = c < classes ? x[c] : -INFINITY;
  int64_t id = kPadding;
  float given = 0.f;
  if (o.logprob) {
    id = read_id(o.ids, o.id_type, r, classes);
    if (id >= 0) given = x[id];
  }
  RunningPair sums;                                        // of each element and the largest before it the smaller one: all but the largest
  float low[MOST];
#pragma unroll
  for (int c = 0; c < MOST; ++c) low[c] = v[c], order(sums.top, low[c]);
  sums.m = fmaxf(sums.top, kLowest);
#pragma unroll
  for (int c = 0; c < MOST; c += 2) add(sums, low[c], low[c + 1]);
  Running all = sums.joined();
  if (all.top == INFINITY) all.s = NAN;
  write_row(o, r, id, given, all);
  const float log_sum = all.log_sum();
  unsigned long long last = ~0ull;
  for (uint32_t k = 0; k < o.top; ++k) {                   // the largest below the one before
    unsigned long long best = 0;
#pragma unroll
    for (int c = 0; c < MOST; ++c) {
      const unsigned long long q = c < classes ? rank_of(v[c], c) : 0;
      if (q < last && q > best) best = q;
    }
    write_top(o, r, k, ~(uint32_t)best, float_of((uint32_t)(best >> 32)), all, log_sum);
    last = best;
  }
}

// ---- the gradient ---------------------------------------------------------------------------------------
// A stream, bound by HBM: a logit is read, its gradient written, some ten instructions in between.  What a row has in common:
struct RowGradient {
  float lse, constant, g_entropy, g;                       // constant: -(gLogProb + gEntropy * entropy); g: what the id's class gets besides
  int64_t id;
  bool nothing;                                            // zeros, whatever the logits hold
};
struct GradientArgs {
  const void* ids;
  int id_type;
  const float *logsumexp, *entropy, *g_logprob, *g_entropy;
};
__device__ __forceinline__ RowGradient row_gradient(const GradientArgs& a, uint64_t row, uint64_t classes) {
  RowGradient r;
  r.id = read_id(a.ids, a.id_type, row, classes);
  r.lse = a.logsumexp[row];
  r.g = a.g_logprob[row];
  r.g_entropy = a.g_entropy ? a.g_entropy[row] : 0.f;
  const float h = a.g_entropy ? a.entropy[row] : 0.f;
  if (r.id == kPadding) r.g = 0.f;
  r.nothing = r.lse == -INFINITY || (r.g == 0.f && r.g_entropy == 0.f);
  if (r.id == kWrong && r.g != 0.f) r.g = NAN;
  r.constant = r.g_entropy != 0.f ? -r.g - r.g_entropy * h : -r.g;
  return r;
}
__device__ __forceinline__ float gradient_at(const RowGradient& r, float x, int64_t column) {
  const float l = at_least(x - r.lse);                     // (a logit of -inf has p = 0, and 0 times the rest is to be 0)
  const float v = exp_fast(l) * (r.constant - r.g_entropy * l);
  return r.nothing ? 0.f : column == r.id ? v + r.g : v;
}

// Longer rows: `parts` teams (CTAs or warps) per row, UNROLL vectors of a thread in flight.  ALIKE: the rows of both matrices lie alike on their
// 16-byte boundaries.
template <int TEAM, int UNROLL, bool ALIKE>
__global__ void __launch_bounds__(kThreads) logprob_grad_kernel(const float* logits, uint32_t rows, uint32_t classes, uint64_t pitch, GradientArgs a,
                                                                float* dlogits, uint64_t dpitch, uint32_t parts) {
  pdl_enter();
  const uint64_t team = (uint64_t)blockIdx.x * (kThreads / TEAM) + threadIdx.x / TEAM;
  const uint64_t r = TEAM == kThreads ? blockIdx.x / parts : team / parts;
  if (r >= rows) return;
  const uint32_t begin = (uint32_t)(team - r * parts) * (TEAM * UNROLL) + threadIdx.x % TEAM;
  const float* x = logits + r * pitch;
  float* dx = dlogits + r * dpitch;
  const Row row(x, classes);
  float4 v[UNROLL];
  if (ALIKE) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const uint32_t i = begin + u * TEAM;
      if (row.is_whole(i)) v[u] = ld_stream(reinterpret_cast<const float4*>(row.aligned) + i);
      else if (i < row.vectors) v[u] = row.edge(i);
    }
  }
  const RowGradient g = row_gradient(a, r, classes);
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const uint32_t i = begin + u * TEAM;
    if (i >= row.vectors) break;
    const int64_t c = (int64_t)4 * i - row.shift;
    if (!ALIKE) v[u] = row.vector(i);
    const float4 d = make_float4(gradient_at(g, v[u].x, c), gradient_at(g, v[u].y, c + 1), gradient_at(g, v[u].z, c + 2), gradient_at(g, v[u].w, c + 3));
    if (ALIKE && row.is_whole(i)) {
      st_stream(reinterpret_cast<float4*>(dx - row.shift) + i, d);
    } else {
      if (row.has(i, 0)) dx[c] = d.x;
      if (row.has(i, 1)) dx[c + 1] = d.y;
      if (row.has(i, 2)) dx[c + 2] = d.z;
      if (row.has(i, 3)) dx[c + 3] = d.w;
    }
  }
}

// Short rows: four elements per thread of the matrix as one line, across the rows' ends.  DENSE: nothing lies between the rows, and both
// matrices begin on 16-byte boundaries.
template <bool DENSE>
__global__ void __launch_bounds__(kThreads) logprob_grad_short_kernel(const float* logits, uint64_t total, uint32_t classes, uint64_t pitch,
                                                                      GradientArgs a, float* dlogits, uint64_t dpitch) {
  pdl_enter();
  const uint64_t block = (uint64_t)blockIdx.x * (kThreads * 4), first = block / classes;
  const uint32_t into = (uint32_t)(block - first * classes) + 4 * threadIdx.x;   // classes and elements from the start of the block's first row
  const uint64_t e = block + 4 * threadIdx.x;
  if (e >= total) return;
  const uint32_t q = into / classes;
  uint64_t r = first + q;
  uint32_t c = into - q * classes;
  const uint32_t n = total - e < 4 ? (uint32_t)(total - e) : 4;
  float x[4], d[4];
  if (DENSE && n == 4) {
    *reinterpret_cast<float4*>(x) = ld_stream(reinterpret_cast<const float4*>(logits + e));
  } else {
    uint64_t rr = r;
    uint32_t cc = c;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (k < n) {
        x[k] = logits[rr * pitch + cc];
        if (++cc == classes) cc = 0, ++rr;
      }
  }
  RowGradient g = row_gradient(a, r, classes);
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k)
    if (k < n) {
      d[k] = gradient_at(g, x[k], c);
      if (!DENSE || n < 4) dlogits[r * dpitch + c] = d[k];
      if (++c == classes && k + 1 < n) {
        c = 0;
        g = row_gradient(a, ++r, classes);
      }
    }
  if (DENSE && n == 4) st_stream(reinterpret_cast<float4*>(dlogits + e), make_float4(d[0], d[1], d[2], d[3]));
}

constexpr uint64_t kMaxClasses = 1ull << 31, kMaxRows = 0x7fffffffull;

int check_ids(const char* what, uint64_t rows, uint64_t classes, uint64_t pitch, int id_type) {
  if (id_type != POLAR_B200_IDS_F32 && id_type != POLAR_B200_IDS_I32 && id_type != POLAR_B200_IDS_I64)
    return fail(POLAR_B200_ERR_INVALID, "ids are held in fp32, in 32 or in 64 bits");
  if (rows > kMaxRows || classes > kMaxClasses || pitch < classes || pitch > 1ull << 40) return fail(POLAR_B200_ERR_INVALID, what);
  if (id_type == POLAR_B200_IDS_F32 && classes > 1ull << 24)
    return fail(POLAR_B200_ERR_INVALID, "ids in fp32 reach to 2^24 classes");
  return POLAR_B200_OK;
}

}  // namespace
}  // namespace polar_b200

using namespace polar_b200;

extern "C" {

int polar_b200_flogprob(const float* logits, uint64_t rows, uint64_t classes, uint64_t pitch, const void* ids, int id_type,
                        float* logprob, float* entropy, float* logsumexp, uint64_t top, void* top_ids, float* top_logprob,
                        void* stream) {
  clear_error();
  int rc = check_ids("flogprob: too many rows or classes, or rows closer than their length", rows, classes, pitch, id_type);
  if (rc) return rc;
  if (top > kMaxTop || top > classes) return fail(POLAR_B200_ERR_INVALID, "flogprob: at most 32 alternatives, and no more than classes");
  if (rows == 0) return POLAR_B200_OK;
  if (classes == 0) return fail(POLAR_B200_ERR_INVALID, "flogprob: rows without classes");
  if (!logits || (logprob && !ids)) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  if (!top_ids && !top_logprob) top = 0;
  const void* some = logprob ? logprob : entropy ? entropy : logsumexp ? logsumexp : top_logprob ? (const void*)top_logprob : top_ids;
  if (!some) return POLAR_B200_OK;                         // nothing is asked for
  LaunchDeviceScope on(stream, some);
  cudaStream_t st = as_stream(stream);
  const Results o{ids, id_type, logprob, entropy, logsumexp, top_ids, top_logprob, (uint32_t)top};
  const uint32_t n = (uint32_t)classes;
  if (classes <= kThreadClasses) {
    const dim3 grid((unsigned)((rows + kThreadRows - 1) / kThreadRows));
    auto go = [&](auto kernel) { return launch("flogprob", kernel, grid, kThreadRows, 0, st, logits, (uint32_t)rows, n, pitch, o); };
    return classes <= 8 ? go(logprob_thread_kernel<8>) : go(logprob_thread_kernel<16>);
  }
  // A warp per row as long as there are rows enough for every SM (20000 x 8192: 100 us against 111 with a CTA of 128 threads per row, with five
  // alternatives 132 and 155; 300 x 8000 with five 16.6 and 7.1; up to 1024 classes always).  Where there are more rows than six to an SM, as many
  // lanes to a short row as hold it in one chunk: 60000 x 100 7.3 us with 8 lanes, with a warp 21; x 200 13.0 with 16, with a warp 21, with twenty
  // alternatives 54 and, a warp then, 73; but 300 x 100 with twenty 7.1 us with 8 lanes, 4.5 with a warp.
  const uint64_t sms = (uint64_t)sm_count();
  if (classes <= 1024 || (classes <= 8192 && rows >= 16 * sms)) {
    const uint32_t lanes = rows <= 6 * sms ? 32 : classes <= 4 * kInFlight * 8 - 3 ? 8 : classes <= 4 * kInFlight * 16 - 3 ? 16 : 32;
    const uint64_t warps = (rows * lanes + 31) / 32;
    const dim3 grid((unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)));
    auto go = [&](auto kernel) { return launch("flogprob", kernel, grid, kThreads, 0, st, logits, (uint32_t)rows, n, pitch, o); };
    if (lanes == 8) return top ? go(logprob_warp_kernel<8, true, true>) : go(logprob_warp_kernel<8, false, true>);
    if (lanes == 16) return top ? go(logprob_warp_kernel<16, true, true>) : go(logprob_warp_kernel<16, false, true>);
    if (chunk_vectors(n) <= kInFlight * 32) return top ? go(logprob_warp_kernel<32, true, true>) : go(logprob_warp_kernel<32, false, true>);
    return top ? go(logprob_warp_kernel<32, true, false>) : go(logprob_warp_kernel<32, false, false>);
  }
  // Few rows: CTAs of 512 threads, in clusters of up to eight per row while the SMs hold them at two per SM and each has some 7000 classes
  // (1 x 131072: 4.7 us, with twenty alternatives 9.2; of 128 threads 6.5 and 14.0; 20 x 9000 with five 4.7 us in one CTA, 7.5 in two).  Many rows:
  // CTAs of 128 threads, since barriers then hold up fewer loads (2048 x 50001: 69 us, with five alternatives 79; of 512 threads 76 and 97).  In
  // between, threads for all of an SM: 200 x 60000 9.9 us with 512, 14.8 with 256; 592 x 29572 11.3 with 256, 13.8 with 128.
  unsigned ctas = 1;
  while (ctas < 8 && rows * ctas * 2 <= 2 * sms && classes / (2 * ctas) >= 7000) ctas *= 2;
  const dim3 grid((unsigned)rows, ctas);
  auto go = [&](auto with, auto without, unsigned threads) {
    return launch_clusters("flogprob", top ? with : without, grid, threads, 0, st, ctas, logits, n, pitch, o);
  };
  if (rows <= 2 * sms) return go(logprob_wide_kernel<512, true>, logprob_wide_kernel<512, false>, 512);
  return rows <= 4 * sms ? go(logprob_wide_kernel<256, true>, logprob_wide_kernel<256, false>, 256)
                         : go(logprob_wide_kernel<128, true>, logprob_wide_kernel<128, false>, 128);
}

int polar_b200_flogprob_grad(const float* logits, uint64_t rows, uint64_t classes, uint64_t pitch, const void* ids, int id_type,
                             const float* logsumexp, const float* entropy, const float* g_logprob, const float* g_entropy,
                             float* dlogits, uint64_t dpitch, void* stream) {
  clear_error();
  int rc = check_ids("flogprob_grad: too many rows or classes, or rows closer than their length", rows, classes, pitch, id_type);
  if (rc) return rc;
  if (dpitch < classes || dpitch > 1ull << 40) return fail(POLAR_B200_ERR_INVALID, "flogprob_grad: rows of the result closer than their length");
  if (rows == 0 || classes == 0) return POLAR_B200_OK;
  if (!logits || !ids || !logsumexp || !g_logprob || !dlogits || (g_entropy && !entropy))
    return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  if (logits == dlogits && pitch != dpitch) return fail(POLAR_B200_ERR_INVALID, "flogprob_grad: in place the rows lie alike");
  LaunchDeviceScope on(stream, dlogits);
  cudaStream_t st = as_stream(stream);
  const GradientArgs args{ids, id_type, logsumexp, entropy, g_logprob, g_entropy};
  if (classes <= 40) {                                     // (65536 x 10: 3.6 us; x 50 9.0, a team of eight lanes per row 8.6)
    const uint64_t total = rows * classes, blocks = (total + kThreads * 4 - 1) / (kThreads * 4);
    if (blocks > 0x7fffffffull) return fail(POLAR_B200_ERR_INVALID, "matrix too large");
    const bool dense = pitch == classes && dpitch == classes && aligned16(logits) && aligned16(dlogits);
    return launch("flogprob_grad", dense ? logprob_grad_short_kernel<true> : logprob_grad_short_kernel<false>, dim3((unsigned)blocks), kThreads, 0, st,
                  logits, total, (uint32_t)classes, pitch, args, dlogits, dpitch);
  }
  const bool alike = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) == 0 && (rows == 1 || ((pitch ^ dpitch) & 3) == 0);
  auto go = [&](auto kernel, unsigned team, unsigned unroll) {
    const uint64_t parts = (classes + 6) / 4 / (team * unroll) + 1, blocks = (rows * parts + kThreads / team - 1) / (kThreads / team);
    if (blocks > 0x7fffffffull) return fail(POLAR_B200_ERR_INVALID, "matrix too large");
    return launch("flogprob_grad", kernel, dim3((unsigned)blocks), kThreads, 0, st, logits, (uint32_t)rows, (uint32_t)classes, pitch, args, dlogits,
                  dpitch, (uint32_t)parts);
  };
  // A team per row, four vectors of a thread in flight: 65536 x 100 10.7 us with eight lanes, 18.9 with a warp; 20000 x 1000 29.9 with a warp, 41
  // with a CTA; 20000 x 4000 103 and 99; 8192 x 32000 329 us with CTAs (6.4 TB/s), as with two vectors; 999 x 10007 10.9, with two 12.4;
  // 20000 x 4000 with two 103.
  if (classes <= 400) return alike ? go(logprob_grad_kernel<8, 4, true>, 8, 4) : go(logprob_grad_kernel<8, 4, false>, 8, 4);
  if (classes <= 3000) return alike ? go(logprob_grad_kernel<32, 4, true>, 32, 4) : go(logprob_grad_kernel<32, 4, false>, 32, 4);
  return alike ? go(logprob_grad_kernel<kThreads, 4, true>, kThreads, 4) : go(logprob_grad_kernel<kThreads, 4, false>, kThreads, 4);
}

}  // extern "C"
