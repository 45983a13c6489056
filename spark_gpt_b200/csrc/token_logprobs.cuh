// Log probabilities of given tokens, the entropy and the largest alternatives of each row of
// logits, and the gradient.
//
//   z = x / temperature, p = softmax(z), logprob = log p[token], H = -sum p log p
//   d x = (g (1[j = token] - p_j) - g_H p_j (log p_j + H)) / temperature
//
// With c = log2(e) / temperature and the row's largest logit m: u = x c - m c <= 0, s = sum 2^u,
// q = sum 2^u u, so log p = ln2 (u - log2 s) and H = ln2 (log2 s - q / s), without
// cancellation of large terms.  A row keeps (m, log2 s) for the backward pass.  The product m c is
// rounded once and the same in every term, so its rounding is a common shift that cancels.
//
// Forward: one pass over the row with a running maximum per thread; when it rises by d in the
// exponent, s <- s 2^-d and q <- 2^-d (q - d s).
//
// The alternatives cost the pass next to nothing.  Each thread's maximum is of elements of its own,
// so the n-th largest maximum (of groups of threads) is a lower bound of the row's n-th
// largest logit.  A thread also keeps the maxima of up to eight segments of its elements; only the
// segments whose maximum reaches the bound, about n of them in all threads, are read
// again, and the few elements that reach it are ranked.
//
// Bounds: DRAM, and close behind it the exponential unit (one a logit, 16 a cycle and SM) and the
// issue slots: 16384 rows of 50257 bf16 are read in 267 us, 6.2 TB/s, and with five alternatives
// in 312.  4096 such rows, 2.3 times what is resident, take 78 us by their last wave; a quarter of
// them left out and with five alternatives 86 us forward, while L2 writes back the
// gradients of the step before (74 on their own), and 117 us backward (48 and 111 us at
// the copy bandwidth), 130 with none left out; 65536 rows of 259 bf16 14 and 14 us (5.2 and 10.5); 8 rows of 131072 fp32
// with twenty alternatives 12 us.
//
// Values in masks: a -inf logit has probability 0 and adds nothing to H; a row of -inf alone has
// log probabilities -inf, H = 0 and no gradient; the token's own -inf logit in another row has the
// gradient g / temperature.  A NaN logit makes its row NaN.  A row whose token
// is `ignore` is left out: logprob 0, H 0, alternatives (0, -1), gradient 0.  Any other token
// outside [0, V) gives logprob NaN and a NaN gradient row.  In the pass logits below a floor of
// about -1e8 / c count as the floor, so that x c - m c, whose product is exact and whose
// shift is rounded, stays finite and small; rows with |m c| of 5e7 and more (the type's lowest
// value or -inf everywhere, very small temperatures) are computed again from (x - m) c.
#pragma once

#include "common.cuh"
#include "layer_norm.cuh"     // from_f32, F2
#include "route_experts.cuh"  // order_key

namespace b200moe {

constexpr int kMaxAlternatives = 32;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kUnderflow = -200.f;     // 2^-200 is 0 in fp32
constexpr float kFloorShift = 1e8f;
constexpr float kLargestShift = 5e7f;    // far enough above the floor that 2^(floor c - m c) is 0

// In this range of temperatures c, 1 / temperature and the floor (-7e-23 to -7e27) are normal numbers.
constexpr float kLeastTemperature = 1e-30f, kMostTemperature = 1e20f;

// The floor for a scale c: a number of 8 significant bits, so that it is the same in bf16.
inline float logit_floor(float c) {
  const float f = kFloorShift / c;
  uint32_t b;
  memcpy(&b, &f, 4);
  b &= 0xffff0000u;
  float r;
  memcpy(&r, &b, 4);
  return -r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_approx(float u) {  // 2 ulp; results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(u));
  return r;
}

// (x - m) c, kept finite: -inf and values far below m give kUnderflow, NaN stays.
__device__ __forceinline__ float rel_log2(float x, float m, float c) {
  return max_nan((x - m) * c, kUnderflow);
}
__device__ __forceinline__ bool needs_care(float m, float c) {
  return !(fabsf(m) * c < kLargestShift);
}

// Value and index in one key: larger value first, then lower index (index < 2^32).
__device__ __forceinline__ unsigned long long pick_key(float v, unsigned i) {
  return (static_cast<unsigned long long>(order_key(v)) << 32) | (0xffffffffu - i);
}

// Sixteen elements as pairs, and the largest of them.
template <typename T>
struct Sixteen;
template <>
struct Sixteen<__nv_bfloat16> {
  static constexpr int kVecs = 2, kWidth = 8;
  uint4 v[kVecs];
  __device__ __forceinline__ void clear(float floor) {
    const uint32_t f = pack_bf16x2(floor, floor);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(f, f, f, f);
  }
  __device__ __forceinline__ void load(int i, const __nv_bfloat16* p) {
    v[i] = *reinterpret_cast<const uint4*>(p);
  }
  __device__ __forceinline__ float floor_and_max(float floor) {
    const __nv_bfloat162 f = __float2bfloat162_rn(floor);
    __nv_bfloat162 m = f;
    __nv_bfloat162* a = reinterpret_cast<__nv_bfloat162*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = __hmax2_nan(a[i], f);
      m = __hmax2(m, a[i]);
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ F2 pair(int i) const {
    const uint32_t w = reinterpret_cast<const uint32_t*>(v)[i];
    return f2(bf16_lo(w), bf16_hi(w));
  }
};
template <>
struct Sixteen<float> {
  static constexpr int kVecs = 4, kWidth = 4;
  float4 v[kVecs];
  __device__ __forceinline__ void clear(float floor) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = make_float4(floor, floor, floor, floor);
  }
  __device__ __forceinline__ void load(int i, const float* p) {
    v[i] = *reinterpret_cast<const float4*>(p);
  }
  __device__ __forceinline__ float floor_and_max(float floor) {
    float m = floor;
    float* a = reinterpret_cast<float*>(v);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      a[i] = max_nan(a[i], floor);
      m = fmaxf(m, a[i]);
    }
    return m;
  }
  __device__ __forceinline__ F2 pair(int i) const {
    const float* a = reinterpret_cast<const float*>(v);
    return f2(a[2 * i], a[2 * i + 1]);
  }
};

// A part [lo, hi) of a row as 16-byte vectors with single elements before and after:
// `head` elements, then `vecs` vectors from element `lo + head`, then `tail` elements.
struct Span {
  int lo, head, vecs, tail;
  template <typename T>
  __device__ __forceinline__ static Span make(const T* row, int lo, int hi) {
    constexpr int W = 16 / sizeof(T);
    Span s;
    s.lo = lo;
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row + lo) / sizeof(T)) % W);
    s.head = min((W - off) % W, hi - lo);
    s.vecs = (hi - lo - s.head) / W;
    s.tail = hi - lo - s.head - s.vecs * W;
    return s;
  }
  template <typename T>
  __device__ __forceinline__ int vec_at(int i) const {  // element of vector i
    return lo + head + i * static_cast<int>(16 / sizeof(T));
  }
  template <typename T>
  __device__ __forceinline__ int edge_at(int i) const {  // element of edge i < head + tail
    return i < head ? lo + i : vec_at<T>(vecs) + i - head;
  }
};

// The shift m c, rounded on its own: contracted into a fused difference of two shifts it would
// leave its rounding error there.
__device__ __forceinline__ float shift_of(float m, float c) { return __fmul_rn(m, c); }

// Running sums of a thread or a group, relative to the shift m c.
struct Sums {
  float m, s, q;
};
// The same sums relative to a larger maximum.
__device__ __forceinline__ Sums raise_to(Sums a, float m, float c) {
  const float d = shift_of(a.m, c) - shift_of(m, c), f = exp2_approx(d);
  return Sums{m, a.s * f, f * fmaf(d, a.s, a.q)};
}

// Sixteen more elements into the running sums.
template <typename T>
__device__ __forceinline__ float take_sixteen(Sixteen<T>& x, float c, float floor, float& m, F2& s2,
                                              F2& q2) {
  const float vm = x.floor_and_max(floor), mn = fmaxf(m, vm);
  const float sh = shift_of(mn, c), d = shift_of(m, c) - sh, f = exp2_approx(d);
  m = mn;
  const F2 c2 = f2(c, c), nsh = f2(-sh, -sh), f22 = f2(f, f), d2 = f2(d, d);
  q2 = mul2(fma2(d2, s2, q2), f22);
  s2 = mul2(s2, f22);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const F2 u2 = fma2(x.pair(k), c2, nsh);
    const float2 u = unpack(u2);
    const F2 e2 = f2(exp2_approx(u.x), exp2_approx(u.y));
    s2 = add2(s2, e2);
    q2 = fma2(e2, u2, q2);
  }
  return vm;
}

// How a row's turns (of Sixteen's vectors of all threads) are cut into segments.
constexpr int kSegments = 8;
struct Segments {
  int turns, per, n;  // turns of the row, turns of a segment, segments
  template <int G, typename T>
  __device__ __forceinline__ static Segments make(const Span& sp) {
    constexpr int K = Sixteen<T>::kVecs;
    Segments g;
    g.turns = (sp.vecs + K * G - 1) / (K * G);
    g.per = max(1, (g.turns + kSegments - 1) / kSegments);
    g.n = (g.turns + g.per - 1) / g.per;
    return g;
  }
};

// The vectors of the next turn are loaded before this one's are used.  PICK: seg[i G + t] gets the
// thread's largest logit of segment i.
template <int G, bool PICK, typename T>
__device__ __forceinline__ Sums stream_row(const T* __restrict__ row, const Span& sp, int t,
                                           float c, float floor, float* seg) {
  using S16 = Sixteen<T>;
  constexpr int K = S16::kVecs, W = S16::kWidth;
  float m = floor;
  F2 s2 = f2(0.f, 0.f), q2 = s2;
  const T* p = row + sp.lo + sp.head;
  const Segments sg = PICK ? Segments::make<G, T>(sp) : Segments{0, 1, 0};
  float seg_max = floor;
  int at = 0, turn = 0;
  auto note = [&](float vm) {
    if constexpr (PICK) {
      seg_max = fmaxf(seg_max, vm);
      if (++turn == sg.per) {
        seg[at * G + t] = seg_max;
        ++at;
        turn = 0;
        seg_max = floor;
      }
    }
  };
  int i = t;
  S16 next;
  bool full = i + (K - 1) * G < sp.vecs;
  if (full) {
#pragma unroll
    for (int k = 0; k < K; ++k) next.load(k, p + static_cast<long long>(i + k * G) * W);
  }
  while (full) {
    S16 x = next;
    i += K * G;
    full = i + (K - 1) * G < sp.vecs;
    if (full) {
#pragma unroll
      for (int k = 0; k < K; ++k) next.load(k, p + static_cast<long long>(i + k * G) * W);
    }
    note(take_sixteen(x, c, floor, m, s2, q2));
  }
  if (i < sp.vecs) {
    S16 x;
    x.clear(floor);
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
      if (i + k * G < sp.vecs) x.load(k, p + static_cast<long long>(i + k * G) * W);
    note(take_sixteen(x, c, floor, m, s2, q2));
  }
  if constexpr (PICK) {
    if (turn) {
      seg[at * G + t] = seg_max;
      ++at;
    }
    for (; at < sg.n; ++at) seg[at * G + t] = floor;
  }
  Sums a{m, sum2(s2), sum2(q2)};
  for (int e = t; e < sp.head + sp.tail; e += G) {
    const float x = max_nan(to_f32(row[sp.edge_at<T>(e)]), floor);
    a = raise_to(a, fmaxf(a.m, x), c);
    const float u = fmaf(x, c, -shift_of(a.m, c)), v = exp2_approx(u);
    a.s += v;
    a.q = fmaf(v, u, a.q);
  }
  return a;
}

// ---------------------------------------------------------------------------
// groups of G threads: part of a warp, a warp, or a whole block
// ---------------------------------------------------------------------------
template <int G>
constexpr int logprob_block() { return G <= 32 ? 256 : G; }
// The lanes of this thread's group in its warp.
template <int G>
__device__ __forceinline__ unsigned group_mask() {
  if constexpr (G >= 32) return 0xffffffffu;
  else return ((1u << G) - 1u) << (threadIdx.x & (32 - G));
}
template <int G>
__device__ __forceinline__ void group_sync() {
  if constexpr (G <= 32) __syncwarp(group_mask<G>());
  else __syncthreads();
}
// Over the lanes of a group (of its part in this warp).
template <int G, typename Op>
__device__ __forceinline__ float lanes_reduce(float v, Op op) {
  constexpr int L = G < 32 ? G : 32;
  const unsigned mask = group_mask<G>();
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(mask, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_reduce<G>(v, [](float a, float b) { return a + b; });
}

template <int G>
constexpr int pick_capacity() { return G <= 32 ? 256 : G <= 128 ? 512 : 1024; }

constexpr int kMaxPairs = 256;
template <int G, bool PICK>
struct GroupShared;
template <int G>
struct GroupShared<G, false> {
  float m[G > 32 ? G / 32 : 1], s[G > 32 ? G / 32 : 1], q[G > 32 ? G / 32 : 1];
  Sums part;  // this block's, as the first block of a cluster reads it
};
template <int G>
struct GroupShared<G, true> {
  float m[G > 32 ? G / 32 : 1], s[G > 32 ? G / 32 : 1], q[G > 32 ? G / 32 : 1];
  alignas(16) unsigned group_key[64];
  unsigned bound;
  int count;
  int n_pairs;
  int pairs[kMaxPairs];  // a segment to read again: segment G + thread
  float seg[kSegments * G];
  unsigned long long best;
  unsigned long long keys[pick_capacity<G>()];
  Sums part;
  int listed;  // the list below holds the part's alternatives
  unsigned long long list[kMaxAlternatives];
};

// Sums relative to one m over the group, every thread's being relative to it already.
template <int G, typename Sh>
__device__ __forceinline__ Sums group_add(Sums a, int t, Sh& sh) {
  a.s = lanes_sum<G>(a.s);
  a.q = lanes_sum<G>(a.q);
  if constexpr (G > 32) {
    if ((t & 31) == 0) {
      sh.s[t / 32] = a.s;
      sh.q[t / 32] = a.q;
    }
    __syncthreads();
    a.s = warp_sum((t & 31) < G / 32 ? sh.s[t & 31] : 0.f);
    a.q = warp_sum((t & 31) < G / 32 ? sh.q[t & 31] : 0.f);
  }
  return a;
}
template <int G, typename Sh, typename Op>
__device__ __forceinline__ float group_max(float m, float least, int t, Sh& sh, Op op) {
  m = lanes_reduce<G>(m, op);
  if constexpr (G > 32) {
    if ((t & 31) == 0) sh.m[t / 32] = m;
    __syncthreads();
    m = lanes_reduce<32>((t & 31) < G / 32 ? sh.m[t & 31] : least, op);
  }
  return m;
}
template <int G, typename Sh>
__device__ __forceinline__ Sums group_join(Sums a, float c, float floor, int t, Sh& sh) {
  const float m = group_max<G>(a.m, floor, t, sh, [](float x, float y) { return fmaxf(x, y); });
  return group_add<G>(raise_to(a, m, c), t, sh);
}

// The `top` largest elements of the span to sh.list, in order; false (for all threads) where
// too many segments or elements tie with the bound, or too few numbers reach the floor.
template <int G, typename T>
__device__ __forceinline__ bool pick_top(const T* __restrict__ row, const Span& sp, float my_max,
                                         int top, int t,
                                         GroupShared<G, true>& sh) {
  const int lane = t & 31;
  const unsigned mine = order_key(my_max);
  unsigned bound;
  if constexpr (G == 32) {
    int rank = 0;
#pragma unroll
    for (int j = 1; j < 32; ++j) {
      const unsigned o = __shfl_xor_sync(0xffffffffu, mine, j);
      rank += (o > mine || (o == mine && (lane ^ j) < lane)) ? 1 : 0;
    }
    const unsigned who = __ballot_sync(0xffffffffu, rank == top - 1);
    bound = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
    if (top > 20) {
      // A higher one from two groups a lane, its first and its last segments: of 32 maxima the
      // smallest is reached by some 130 elements, the 32nd of 64 by 44 (16384 x 8192 bf16
      // with 32 alternatives: 115 us, 538 from the lanes' maxima alone; with 20 the same).
      const Segments sg = Segments::make<G, T>(sp);
      unsigned a = 0, b = 0;
      for (int i = 0; i < sg.n; ++i) {
        const unsigned k = order_key(sh.seg[i * 32 + t]);
        if (2 * i < sg.n) a = max(a, k);
        else b = max(b, k);
      }
      int above_a = 0, above_b = 0;
#pragma unroll 8
      for (int j = 0; j < 32; ++j) {
        const unsigned oa = __shfl_sync(0xffffffffu, a, j), ob = __shfl_sync(0xffffffffu, b, j);
        above_a += (oa > a) + (ob > a);
        above_b += (oa > b) + (ob > b);
      }
      // the smallest maximum with fewer than `top` above it: at least `top` reach it
      bound = max(bound, __reduce_min_sync(0xffffffffu, min(above_a < top ? a : 0xffffffffu,
                                                            above_b < top ? b : 0xffffffffu)));
    }
    if (lane == 0) sh.count = sh.n_pairs = 0;
    __syncwarp();
  } else {
    constexpr int L = G / 64;  // threads whose maxima are joined: 64 groups
    unsigned g = mine;
#pragma unroll
    for (int o = 1; o < L; o <<= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (t % L == 0) sh.group_key[t / L] = g;
    if (t == 0) sh.count = sh.n_pairs = 0;
    __syncthreads();
    if (t < 128) {  // threads 2 i and 2 i + 1 rank group i, each against half of the groups
      const int i = t / 2, half = t % 2 * 32;
      const unsigned a = sh.group_key[i];
      int rank = 0;
#pragma unroll
      for (int j = half; j < half + 32; j += 4) {
        const uint4 k = *reinterpret_cast<const uint4*>(&sh.group_key[j]);
        rank += (k.x > a || (k.x == a && j < i)) + (k.y > a || (k.y == a && j + 1 < i)) +
                (k.z > a || (k.z == a && j + 2 < i)) + (k.w > a || (k.w == a && j + 3 < i));
      }
      rank += __shfl_xor_sync(0xffffffffu, rank, 1);
      if (rank == top - 1) sh.bound = a;
    }
    __syncthreads();
    bound = sh.bound;
  }
  auto push = [&](float v, int at) {
    if (order_key(v) < bound) return;
    const int n = atomicAdd(&sh.count, 1);
    if (n < pick_capacity<G>()) sh.keys[n] = pick_key(v, static_cast<unsigned>(at));
  };
  const Segments sg = Segments::make<G, T>(sp);
  if (mine >= bound) {
    for (int i = 0; i < sg.n; ++i) {
      if (order_key(sh.seg[i * G + t]) < bound) continue;
      const int n = atomicAdd(&sh.n_pairs, 1);
      if (n < kMaxPairs) sh.pairs[n] = i * G + t;
    }
  }
  group_sync<G>();
  const int n_pairs = sh.n_pairs, len = sg.per * Sixteen<T>::kVecs;  // vectors of a segment
  if (n_pairs <= kMaxPairs) {
    for (int j = t; j < n_pairs * len; j += G) {
      const int pair = sh.pairs[j / len];
      const int i = pair % G + (pair / G * len + j % len) * G;
      if (i >= sp.vecs) continue;
      constexpr int W = 16 / sizeof(T);
      const int at = sp.vec_at<T>(i);
      const uint4 v = *reinterpret_cast<const uint4*>(row + at);
      const T* x = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int k = 0; k < W; ++k) push(to_f32(x[k]), at + k);
    }
  }
  for (int i = t; i < sp.head + sp.tail; i += G) {
    const int at = sp.edge_at<T>(i);
    push(to_f32(row[at]), at);
  }
  group_sync<G>();
  const int n = sh.count;
  const bool ok = n_pairs <= kMaxPairs && n >= top && n <= pick_capacity<G>();
  if (ok) {
    for (int i = t; i < n; i += G) {
      const unsigned long long key = sh.keys[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += sh.keys[j] > key ? 1 : 0;
      if (rank < top) sh.list[rank] = key;
    }
  }
  group_sync<G>();
  return ok;
}

// The same by one search of the row for each alternative, for any values (4096 x 50257 bf16 with
// three logits allowed and five alternatives: 850 us, 92 the other way).
template <int G, typename T>
__device__ __forceinline__ void pick_top_any(const T* __restrict__ row, int V, int top, int t,
                                             GroupShared<G, true>& sh) {
  unsigned long long last = ~0ull;
  for (int r = 0; r < top; ++r) {
    if (t == 0) sh.best = 0ull;
    group_sync<G>();
    unsigned long long best = 0ull;
    for (int i = t; i < V; i += G) {
      const unsigned long long key = pick_key(to_f32(row[i]), i);
      if (key < last && key > best) best = key;
    }
    if (best) atomicMax(&sh.best, best);
    group_sync<G>();
    last = sh.best;
    if (t == 0) sh.list[r] = last;
    group_sync<G>();
  }
}

// The sums of a row from (x - m) c, for any values.
template <int G, typename Sh, typename T>
__device__ __forceinline__ Sums careful_sums(const T* __restrict__ row, int V, float c, int t,
                                             Sh& sh) {
  float m = -INFINITY;
  for (int i = t; i < V; i += G) m = max_nan(m, to_f32(row[i]));
  group_sync<G>();
  m = group_max<G>(m, -INFINITY, t, sh, [](float x, float y) { return max_nan(x, y); });
  Sums a{m, 0.f, 0.f};
  for (int i = t; i < V; i += G) {
    const float u = rel_log2(to_f32(row[i]), m, c), e = exp2_approx(u);
    a.s += e;
    a.q = fmaf(e, u, a.q);
  }
  a = group_add<G>(a, t, sh);
  group_sync<G>();
  return a;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
// This block's shared-memory address `p` in block `rank` of the cluster.
template <typename U>
__device__ __forceinline__ const U* of_block(const U* p, unsigned rank) {
  uint64_t a;
  asm("mapa.u64 %0, %1, %2;" : "=l"(a) : "l"(p), "r"(rank));
  return reinterpret_cast<const U*>(a);
}

// G threads a row, 256 / G rows a block up to a warp a row; with G > 32 a row may be split over
// the S blocks of a cluster, whose parts the first block reads out of their shared memory.
// Alternatives (PICK) need G >= 32.
template <int G, bool PICK, typename T>
constexpr int logprob_blocks() {  // of an SM, as many as the registers of the pass allow
  return G <= 32 ? (PICK ? 3 : 4) : (sizeof(T) == 2 ? 1536 : 1024) / G;
}
template <int G, bool PICK, typename T>
__global__ void __launch_bounds__(logprob_block<G>(), logprob_blocks<G, PICK, T>())
token_logprobs_fwd_kernel(const T* __restrict__ logits, long long ld,
                          const long long* __restrict__ tokens, long long rows, int V, int S,
                          float c, float inv_t, float floor, long long ignore, int top,
                          float* __restrict__ logprob, float* __restrict__ entropy,
                          float* __restrict__ top_logprobs, long long* __restrict__ top_ids,
                          float2* __restrict__ stats) {
  constexpr int RPB = logprob_block<G>() / G;
  using Sh = GroupShared<G, PICK>;
  __shared__ Sh shared[RPB];
  const int t = threadIdx.x % G;
  Sh& sh = shared[threadIdx.x / G];
  const int part = G > 32 ? blockIdx.x % S : 0;
  // parts start on multiples of 64 elements
  const int per = G > 32 && S > 1 ? ((V + S - 1) / S + 63) / 64 * 64 : V;
  const int lo = min(part * per, V), hi = min(lo + per, V);
  const long long step = static_cast<long long>(gridDim.x / S) * RPB;
  long long r = static_cast<long long>(blockIdx.x / S) * RPB + threadIdx.x / G;
  long long next_tok = r < rows ? tokens[r] : 0;
  for (; r < rows; r += step) {
    const T* row = logits + r * ld;
    const long long tok = next_tok;
    if (r + step < rows) next_tok = tokens[r + step];
    if (tok == ignore) {
      if (part == 0) {
        if (t == 0) {
          logprob[r] = 0.f;
          entropy[r] = 0.f;
          if (stats) stats[r] = make_float2(0.f, 0.f);
        }
        for (int i = t; PICK && i < top; i += G) {
          top_logprobs[r * top + i] = 0.f;
          top_ids[r * top + i] = -1;
        }
      }
      continue;
    }
    // read early: it is needed when the sums are there
    const bool bad = tok < 0 || tok >= V;
    const float x_tok = bad ? __int_as_float(0x7fc00000) : to_f32(row[tok]);
    const Span sp = Span::make(row, lo, hi);
    float* seg = nullptr;
    if constexpr (PICK) seg = sh.seg;
    const Sums mine = stream_row<G, PICK>(row, sp, t, c, floor, seg);
    Sums a = group_join<G>(mine, c, floor, t, sh);
    bool listed = true;
    if constexpr (PICK) listed = pick_top<G>(row, sp, mine.m, top, t, sh);
    if constexpr (G > 32) {
      if (S > 1) {
        if (t == 0) {
          sh.part = a;
          if constexpr (PICK) sh.listed = listed;
        }
        cluster_barrier();
        if (part == 0) {
          float m = a.m;
          for (int i = 1; i < S; ++i) m = fmaxf(m, of_block(&sh, i)->part.m);
          a = raise_to(a, m, c);
          for (int i = 1; i < S; ++i) {
            const Sh* o = of_block(&sh, i);
            const Sums b = raise_to(o->part, m, c);
            a.s += b.s;
            a.q += b.q;
            if constexpr (PICK) listed = listed && o->listed;
          }
        }
        if constexpr (PICK) {
          if (part == 0 && listed) {
            // all S lists to keys; a key's rank is its place in its list and, in each other list,
            // the number of larger keys (the lists fall)
            for (int i = t; i < S * top; i += G) sh.keys[i] = of_block(&sh, i / top)->list[i % top];
            __syncthreads();
            for (int i = t; i < S * top; i += G) {
              const unsigned long long key = sh.keys[i];
              int rank = i % top;
              for (int l = 0; l < S; ++l) {
                if (l == i / top) continue;
                int a0 = 0, b0 = top;
                while (a0 < b0) {
                  const int mid = (a0 + b0) / 2;
                  if (sh.keys[l * top + mid] > key) a0 = mid + 1;
                  else b0 = mid;
                }
                rank += a0;
              }
              if (rank < top) sh.list[rank] = key;
            }
            __syncthreads();
          }
        }
      }
    }
    if (part == 0) {
      const bool care = needs_care(a.m, c);
      if (care) a = careful_sums<G>(row, V, c, t, sh);
      const float l2s = log2f(a.s), shift = shift_of(a.m, c);
      const bool none = a.m == -INFINITY;
      auto logp = [&](float x) {
        if (none || (x == -INFINITY && a.s == a.s)) return -INFINITY;
        const float u = care ? -INFINITY : fmaf(x, c, -shift);
        return u > -INFINITY ? kLn2 * (u - l2s) : (x - a.m) * inv_t - kLn2 * l2s;
      };
      if (t == 0) {
        logprob[r] = bad ? x_tok : logp(x_tok);
        entropy[r] = none ? 0.f : kLn2 * (l2s - a.q / a.s);
        if (stats) stats[r] = make_float2(a.m, l2s);
      }
      if constexpr (PICK) {
        if (care || !listed) pick_top_any<G>(row, V, top, t, sh);
        for (int i = t; i < top; i += G) {
          const unsigned long long key = sh.list[i];
          top_ids[r * top + i] = 0xffffffffu - static_cast<unsigned>(key);
          top_logprobs[r * top + i] = logp(order_value(static_cast<unsigned>(key >> 32)));
        }
      }
    }
    if constexpr (G > 32) {
      if (S > 1) cluster_barrier();
      else __syncthreads();
    } else if constexpr (G == 32) {
      __syncwarp();
    }
  }
}

// The gradient of the elements [lo, hi) of a row: block (or warp) `part` of `parts`.  VEC: the
// gradient's rows lie on 16-byte boundaries where the logits' do.  A subnormal p times g /
// temperature may be a normal number, so p is the square of 2^(u / 2), which the flushing form
// keeps, at 4 ulp (16384 x 8192 bf16: 78 us, 94 with exp2f).
template <int G, bool VEC, typename T>
__global__ void __launch_bounds__(logprob_block<G>())
token_logprobs_bwd_kernel(const T* __restrict__ logits, long long ld,
                          const long long* __restrict__ tokens, long long rows, int V, int S,
                          float c, float inv_t, long long ignore,
                          const float2* __restrict__ stats, const float* __restrict__ entropy,
                          const float* __restrict__ d_logprob,
                          const float* __restrict__ d_entropy, T* __restrict__ d_logits,
                          long long ld_out) {
  constexpr int RPB = logprob_block<G>() / G, W = 16 / sizeof(T);
  const int t = threadIdx.x % G;
  const int part = G > 32 ? blockIdx.x % S : 0;
  const int per = S > 1 ? ((V + S - 1) / S + 63) / 64 * 64 : V;
  const int lo = min(part * per, V), hi = min(lo + per, V);
  const long long step = static_cast<long long>(gridDim.x / S) * RPB;
  for (long long r = static_cast<long long>(blockIdx.x / S) * RPB + threadIdx.x / G; r < rows;
       r += step) {
    const T* row = logits + r * ld;
    T* out = d_logits + r * ld_out;
    const long long tok = tokens[r];
    const float2 st = stats[r];
    const bool zero = tok == ignore || st.x == -INFINITY;
    float g = d_logprob ? d_logprob[r] * inv_t : 0.f;
    const float ge = d_entropy ? d_entropy[r] * inv_t : 0.f;
    if (tok < 0 || tok >= V) g = __int_as_float(0x7fc00000);
    // d = p (ka + kb u) + g [j = token], u = log2 p
    const float ka = -(g + ge * entropy[r]), kb = -ge * kLn2;
    const bool care = needs_care(st.x, c);
    const float sh = shift_of(st.x, c);
    auto one = [&](int i) {
      if (zero) return 0.f;
      const float x = to_f32(row[i]);
      const float u = care ? rel_log2(x, st.x, c) - st.y
                           : max_nan(fmaf(x, c, -sh), kUnderflow) - st.y;
      return fmaf(exp2f(u), fmaf(kb, u, ka), i == tok ? g : 0.f);
    };
    // Two elements that are not the token, from u / 2 (every halving is exact).
    const float ch = 0.5f * c, shh = 0.5f * sh, lh = 0.5f * st.y;
    const F2 c2 = f2(ch, ch), nsh = f2(-shh, -shh), nl = f2(-lh, -lh), ka2 = f2(ka, ka),
             kb2 = f2(2.f * kb, 2.f * kb);
    auto two = [&](F2 x) {
      const float2 u = unpack(fma2(x, c2, nsh));
      const F2 u2 = add2(f2(max_nan(u.x, 0.5f * kUnderflow), max_nan(u.y, 0.5f * kUnderflow)), nl);
      const float2 h = unpack(u2);
      const F2 e2 = f2(exp2_approx(h.x), exp2_approx(h.y));
      return unpack(mul2(mul2(e2, e2), fma2(kb2, u2, ka2)));
    };
    if (!VEC || care) {
      // single elements, coalesced over the threads, eight in flight
      int i = lo + t;
      if (!care && !zero) {
        for (; i + 7 * G < hi; i += 8 * G) {
          T v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = row[i + k * G];
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
            const float2 d = two(f2(to_f32(v[k]), to_f32(v[k + 1])));
            out[i + k * G] = from_f32<T>(i + k * G == tok ? d.x + g : d.x);
            out[i + (k + 1) * G] = from_f32<T>(i + (k + 1) * G == tok ? d.y + g : d.y);
          }
        }
      }
      for (; i < hi; i += G) out[i] = from_f32<T>(one(i));
      continue;
    }
    const Span sp = Span::make(row, lo, hi);
    for (int i = t; i < sp.head + sp.tail; i += G) {
      const int at = sp.edge_at<T>(i);
      out[at] = from_f32<T>(one(at));
    }
    auto vec = [&](const uint4& v, int at) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      float o[W];
#pragma unroll
      for (int k = 0; k < W / 2; ++k) {
        const F2 x = sizeof(T) == 2 ? f2(bf16_lo(w[k]), bf16_hi(w[k]))
                                    : f2(__uint_as_float(w[2 * k % 4]), __uint_as_float(w[(2 * k + 1) % 4]));
        const float2 d = two(x);
        o[2 * k] = d.x;
        o[2 * k + 1] = d.y;
      }
      const long long hot = tok - at;
      if (hot >= 0 && hot < W) {
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k == hot) o[k] += g;
      }
      store_chunk<T, true>(out + at, o);
    };
    if (zero) {
      for (int i = t; i < sp.vecs; i += G)
        *reinterpret_cast<uint4*>(out + sp.vec_at<T>(i)) = make_uint4(0u, 0u, 0u, 0u);
      continue;
    }
    constexpr int K = 2;  // vectors a turn
    int i = t;
    for (; i + (K - 1) * G < sp.vecs; i += K * G) {
      uint4 v[K];
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = *reinterpret_cast<const uint4*>(row + sp.vec_at<T>(i + k * G));
#pragma unroll
      for (int k = 0; k < K; ++k) vec(v[k], sp.vec_at<T>(i + k * G));
    }
    for (; i < sp.vecs; i += G) {
      const int at = sp.vec_at<T>(i);
      vec(*reinterpret_cast<const uint4*>(row + at), at);
    }
  }
}

}  // namespace b200moe
