// Expert routing with sigmoid or softmax scores, a selection bias and expert groups, its
// gradient, and the counts and bias update of loss-free balancing.
//
//   s = sigmoid(x) or softmax(x);  c = s + bias
//   groups: keep the `kept` groups of the largest max(c) or largest two-score sum
//   selected: the k largest c of the kept groups, by falling c, equal values by rising index
//   w_r = scale s_r / (sum s + 1e-20), or scale s_r
// A bias selects only: it has no part in w and no gradient.
//
// A NaN score ranks below every number, so the ids are in range and distinct whatever
// the logits hold.
//
// L lanes take a token (4 to 32), eight consecutive experts a lane, so that a lane's logits are
// one or two 16-byte loads and 64 experts put four tokens in a warp: what bounds these kernels is
// instructions (the forward's issue slots are 67-74% busy, the softmax gradient's 64, the sigmoid
// gradient's 44; DRAM below 15%), and a reduction serves several tokens at once.  Up to 64 experts a lane sorts its keys and k rounds take the largest first
// key; from 65 on the few keys that reach a bound are listed and ranked (256 experts, top-8:
// 25 us for 32768 tokens, 34 with the rounds; with 8 lanes a token the bound lets through a third
// of the keys and the rounds are as fast).  65536 tokens, 64 experts, top-8, softmax, bf16:
// 21 us forward, 9.7 us backward; 16381 tokens, 256 experts in 8 groups, top-8, sigmoid, fp32: 19 and
// 7.4 us (25 and 36 MB in all, 3.9 and 5.5 us at the copy bandwidth).
#pragma once

#include <climits>

#include "common.cuh"
#include "layer_norm.cuh"  // from_f32, store_chunk
#include "router.cuh"      // load_chunk, group_max, group_sum, GroupTokens

namespace b200moe {

constexpr int kRouteMaxExperts = 256;
constexpr int kRouteMaxGroups = 32;
constexpr int kRouteThreads = 128;
constexpr int kRouteList = 32;  // keys that reach the bound, at most (else: k rounds)
constexpr float kRouteNormEps = 1e-20f;

// Order-preserving map of floats to unsigned (0 is free for "taken"; NaN becomes 1; the
// two zeros are equal).
__device__ __forceinline__ unsigned order_key(float v) {
  const unsigned b = __float_as_uint(v + 0.f);
  if (v != v) return 1u;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned key) {
  if (key <= 1u) return key ? __int_as_float(0x7fc00000) : -INFINITY;
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// The same as signed values, two instructions where the score is a number: kTaken below NaN below
// the numbers.
constexpr int kTaken = INT_MIN;
__device__ __forceinline__ int select_key(float v) {  // v is not -0: scores are not
  const int b = __float_as_int(v);
  const int k = b ^ ((b >> 31) & 0x7fffffff);
  return v == v ? k : kTaken + 1;
}
__device__ __forceinline__ float select_value(int k) {
  const float v = __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
  return k <= kTaken + 1 ? __int_as_float(0x7fc00000) : v;
}

template <int L>
__device__ __forceinline__ int group_max_key(int v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}

__device__ __forceinline__ float rcp_approx(float v) {  // 1 ulp; 0 below 2^-126
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// 1 / (1 + e^-x) below kSmallLogit is e^x (to one part in 10^37), which keeps the scores below 2^-126
// that the reciprocal makes 0.
constexpr float kSmallLogit = -87.f;
__device__ __forceinline__ float sigmoid_score(float x) {
  return x < kSmallLogit ? expf(x) : rcp_approx(1.0f + expf(-x));
}

// Scores of a lane's experts (z: its logits, -inf beyond E).  expf, since the selection hangs on
// them; the reciprocals are within 1 ulp.  `small`: with the sigmoid scores below 2^-126.  A row of
// -inf alone has softmax scores 0.
template <int L>
__device__ __forceinline__ void route_scores(float (&z)[kVpt], bool sigmoid, bool small) {
  if (sigmoid) {
    if (small) {
#pragma unroll
      for (int j = 0; j < kVpt; ++j) z[j] = sigmoid_score(z[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kVpt; ++j) z[j] = rcp_approx(1.0f + expf(-z[j]));
    }
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kVpt; ++j) m = fmaxf(m, z[j]);
  m = group_max<L>(m);
  const bool none = m == -INFINITY;
  float t = 0.f;
#pragma unroll
  for (int j = 0; j < kVpt; ++j) {
    z[j] = expf(z[j] - (none ? 0.f : m));
    t += z[j];
  }
  t = group_sum<L>(t);  // by every lane of the warp, whatever its token holds
  const float inv = none ? 0.f : rcp_approx(t);
#pragma unroll
  for (int j = 0; j < kVpt; ++j) z[j] *= inv;
}

// The two largest of two falling pairs.
__device__ __forceinline__ void merge_two(int& a, int& b, int c, int d) {
  const int lo = min(a, c);
  a = max(a, c);
  b = max(lo, max(b, d));
}

// Sorts a lane's keys, falling; `order` gets the places they had, four bits each.  Only
// neighbours that are out of order change places, so equal keys keep theirs.
__device__ __forceinline__ void sort_keys(int (&key)[kVpt], unsigned& order) {
  int id[kVpt];
#pragma unroll
  for (int j = 0; j < kVpt; ++j) id[j] = j;
#pragma unroll
  for (int pass = 0; pass < kVpt; ++pass) {
#pragma unroll
    for (int j = pass & 1; j + 1 < kVpt; j += 2) {
      const bool swap = key[j + 1] > key[j];
      const int hi = max(key[j], key[j + 1]), lo = min(key[j], key[j + 1]);
      const int first = swap ? id[j + 1] : id[j], second = swap ? id[j] : id[j + 1];
      key[j] = hi;
      key[j + 1] = lo;
      id[j] = first;
      id[j + 1] = second;
    }
  }
  order = 0u;
#pragma unroll
  for (int j = 0; j < kVpt; ++j) order |= static_cast<unsigned>(id[j]) << (4 * j);
}

// `lanes_per_group`: the lanes of an expert group where each lane's eight experts lie in one group
// and the groups are a power of two of lanes; else 0 (the groups are scanned in shared memory).
template <int L, typename T>
__global__ void __launch_bounds__(kRouteThreads)
route_experts_fwd_kernel(const T* __restrict__ logits, long long ld, long long rows, int E, int k,
                         int vec, const float* __restrict__ bias, int sigmoid, int groups,
                         int lanes_per_group, int kept, int top2, int normalize, float scale,
                         long long* __restrict__ selected, float* __restrict__ weights) {
  constexpr int TPB = kRouteThreads / L;
  constexpr int SLOTS = L < 16 ? (kMaxTopK + L - 1) / L : kRouteList / L;
  __shared__ __align__(16) float sh_s[TPB][L * kVpt];
  __shared__ unsigned long long sh_list[TPB][L < 16 ? 1 : kRouteList];
  __shared__ __align__(16) int sh_key[TPB][L * kVpt];
  __shared__ int sh_group[TPB][kRouteMaxGroups];
  __shared__ unsigned sh_stay[TPB];
  const int sub = threadIdx.x & (L - 1), tok = threadIdx.x / L, e0 = sub * kVpt;
  const int per = E / groups;
  float bs[kVpt];
#pragma unroll
  for (int j = 0; j < kVpt; ++j) bs[j] = bias && e0 + j < E ? bias[e0 + j] : 0.f;
  const GroupTokens gt = GroupTokens::make<L>(rows);
  bool small = false;  // the round is done again, with the scores below 2^-126
  for (long long rnd = 0; rnd < gt.rounds;) {
    const long long t = gt.first + rnd * gt.stride;
    const bool valid = t < rows;
    float s[kVpt];
    int key[kVpt];
    load_chunk(logits + (valid ? t : 0) * ld, e0, E, valid, vec != 0, s);
    route_scores<L>(s, sigmoid != 0, small);
#pragma unroll
    for (int j = 0; j < kVpt; ++j) key[j] = e0 + j < E ? select_key(s[j] + bs[j]) : kTaken;
    if (bias) {  // the winners' scores without the bias are read from here
      *reinterpret_cast<float4*>(&sh_s[tok][e0]) = make_float4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<float4*>(&sh_s[tok][e0 + 4]) = make_float4(s[4], s[5], s[6], s[7]);
    }
    if (groups > 1 && lanes_per_group == 0) {
#pragma unroll
      for (int j = 0; j < kVpt; ++j) sh_key[tok][e0 + j] = key[j];
      if (sub == 0) sh_stay[tok] = 0u;
      __syncwarp();
      for (int g = sub; g < groups; g += L) {
        int a = kTaken, b = kTaken;
        for (int i = 0; i < per; ++i) merge_two(a, b, sh_key[tok][g * per + i], kTaken);
        sh_group[tok][g] = top2 ? select_key(select_value(a) + select_value(b)) : a;
      }
      __syncwarp();
      for (int g = sub; g < groups; g += L) {
        const int a = sh_group[tok][g];
        int rank = 0;
        for (int i = 0; i < groups; ++i) {
          const int o = sh_group[tok][i];
          rank += (o > a || (o == a && i < g)) ? 1 : 0;
        }
        if (rank < kept) atomicOr(&sh_stay[tok], 1u << g);
      }
      __syncwarp();
      const unsigned stay = sh_stay[tok];
#pragma unroll
      for (int j = 0; j < kVpt; ++j)
        if (e0 + j < E && !((stay >> ((e0 + j) / per)) & 1u)) key[j] = kTaken;
    }
    unsigned order = 0u;
    if constexpr (L < 16) sort_keys(key, order);
    if (lanes_per_group > 0) {
      int a = key[0], b = key[1];
      if constexpr (L >= 16) {
        a = max(key[0], key[1]);
        b = min(key[0], key[1]);
#pragma unroll
        for (int j = 2; j < kVpt; ++j) merge_two(a, b, key[j], kTaken);
      }
      for (int o = 1; o < lanes_per_group; o <<= 1)
        merge_two(a, b, __shfl_xor_sync(0xffffffffu, a, o), __shfl_xor_sync(0xffffffffu, b, o));
      if (top2) a = select_key(select_value(a) + select_value(b));
      const int mine = sub / lanes_per_group;
      int rank = 0;
      for (int g = 0; g < groups; ++g) {
        const int o = __shfl_sync(0xffffffffu, a, g * lanes_per_group, L);
        rank += (o > a || (o == a && g < mine)) ? 1 : 0;
      }
#pragma unroll
      for (int j = 0; j < kVpt; ++j) key[j] = rank < kept ? key[j] : kTaken;
    }
    __syncwarp();
    // the k largest: a lane's winners, their ranks (k and more: none) and scores
    float won_s[SLOTS];
    int won_e[SLOTS], won_r[SLOTS];
    bool ranked = false;
    if constexpr (L >= 16) {
      // The k-th largest of the lanes' maxima bounds the k-th largest key from below, and few keys
      // reach it (about 10 of 256 for k = 8): they are listed and ranked against one another.
      // Equal maxima are taken out together, which only lowers the bound.
      int head = key[0], bound = kTaken;
#pragma unroll
      for (int j = 1; j < kVpt; ++j) head = max(head, key[j]);
      for (int r = 0; r < k; ++r) {
        bound = group_max_key<L>(head);
        head = head == bound ? kTaken : head;
      }
      bound = max(bound, kTaken + 1);
      const int shift = threadIdx.x & 31 & ~(L - 1);
      const unsigned lower = (1u << sub) - 1u, all = L == 32 ? 0xffffffffu : (1u << (L & 31)) - 1u;
      int n = 0;
#pragma unroll
      for (int j = 0; j < kVpt; ++j) {
        const bool here = key[j] >= bound;
        const unsigned who = __ballot_sync(0xffffffffu, here) >> shift & all;
        const int at = n + __popc(who & lower);
        if (here && at < kRouteList)
          sh_list[tok][at] = static_cast<unsigned long long>(static_cast<unsigned>(key[j]) ^ 0x80000000u) << 32 |
                             (kRouteMaxExperts - 1 - (e0 + j));
        n += __popc(who);
      }
      __syncwarp();
      if (!__any_sync(0xffffffffu, n > kRouteList)) {
        ranked = true;
#pragma unroll
        for (int q = 0; q < SLOTS; ++q) {
          const int c = q * L + sub;
          const unsigned long long mine = c < n ? sh_list[tok][c] : 0ull;
          int rank = 0;
          for (int i = 0; i < n; ++i) rank += sh_list[tok][i] > mine ? 1 : 0;
          won_r[q] = c < n ? rank : k;
          won_e[q] = c < n ? kRouteMaxExperts - 1 - static_cast<int>(mine & 0xffffffffu) : 0;
          won_s[q] = 0.f;
          if (won_r[q] < k)
            won_s[q] = bias ? sh_s[tok][won_e[q]]
                            : select_value(static_cast<int>(static_cast<unsigned>(mine >> 32) ^ 0x80000000u));
        }
        if constexpr (L == 16) {
          // By rank, as the rounds have them: a token's scores are then added in one order, whether
          // or not the token beside it in the warp took the rounds.
          __syncwarp();
#pragma unroll
          for (int q = 0; q < SLOTS; ++q)
            if (won_r[q] < k)
              sh_list[tok][won_r[q]] = static_cast<unsigned long long>(won_e[q]) << 32 | __float_as_uint(won_s[q]);
          __syncwarp();
          const unsigned long long mine = sub < k ? sh_list[tok][sub] : 0ull;
#pragma unroll
          for (int q = 0; q < SLOTS; ++q) {
            won_r[q] = q * L + sub;
            won_e[q] = q ? 0 : static_cast<int>(mine >> 32);
            won_s[q] = q ? 0.f : __uint_as_float(static_cast<unsigned>(mine));
          }
        }
      }
    }
    if (!ranked) {
      // k rounds: the largest of the lanes' first keys, its lowest lane, whose keys move up
      if constexpr (L >= 16) sort_keys(key, order);
      int won_k[SLOTS];
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        won_k[q] = 0;
        won_e[q] = 0;
        won_r[q] = q * L + sub;
        for (int i = 0; i < L && q * L + i < k; ++i) {
          const int best = group_max_key<L>(key[0]);
          unsigned owners = __ballot_sync(0xffffffffu, key[0] == best);
          if constexpr (L < 32) owners = owners >> (threadIdx.x & 31 & ~(L - 1)) & ((1u << L) - 1u);
          const int owner = __ffs(owners) - 1;
          const int e = owner * kVpt + (__shfl_sync(0xffffffffu, order, owner, L) & 7u);
          const bool here = sub == owner;
#pragma unroll
          for (int j = 0; j + 1 < kVpt; ++j) key[j] = here ? key[j + 1] : key[j];
          key[kVpt - 1] = here ? kTaken : key[kVpt - 1];
          order = here ? order >> 4 : order;
          won_e[q] = sub == i ? e : won_e[q];
          won_k[q] = sub == i ? best : won_k[q];
        }
        won_s[q] = 0.f;
        if (won_r[q] < k) won_s[q] = bias ? sh_s[tok][won_e[q]] : select_value(won_k[q]);
      }
    }
    // A score that the reciprocal makes 0 changes the outcome only where it is chosen.
    if (sigmoid && !small) {
      bool zero = false;
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) zero |= valid && won_r[q] < k && won_s[q] == 0.f;
      small = __any_sync(0xffffffffu, zero);
      if (small) {
        __syncwarp();
        continue;
      }
    }
    small = false;
    ++rnd;
    float f = scale;
    if (normalize) {
      float total = 0.f;
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) total += won_s[q];
      f = scale / (group_sum<L>(total) + kRouteNormEps);
    }
    if (valid) {
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) {
        if (won_r[q] < k) {
          selected[t * k + won_r[q]] = won_e[q];
          weights[t * k + won_r[q]] = won_s[q] * f;
        }
      }
    }
    __syncwarp();  // the staging areas are free for the next token
  }
}

// dx of the weights' gradient; ids outside [0, E) take no part and raise a fault.  Sigmoid scores
// need the selected logits alone; softmax needs the row.
template <int L, typename T>
__global__ void __launch_bounds__(kRouteThreads)
route_experts_bwd_kernel(const T* __restrict__ logits, long long ld,
                         const long long* __restrict__ selected,
                         const float* __restrict__ d_weights, long long rows, int E, int k,
                         int vec, int vec_out, int sigmoid, int normalize, float scale,
                         T* __restrict__ d_logits) {
  constexpr int TPB = kRouteThreads / L, SLOTS = (kMaxTopK + L - 1) / L;
  __shared__ __align__(16) float sh_s[TPB][L * kVpt];
  __shared__ __align__(16) float sh_d[TPB][L * kVpt];
  const int sub = threadIdx.x & (L - 1), tok = threadIdx.x / L, e0 = sub * kVpt;
  const GroupTokens gt = GroupTokens::make<L>(rows);
  for (long long rnd = 0; rnd < gt.rounds; ++rnd) {
    const long long t = gt.first + rnd * gt.stride;
    const bool valid = t < rows;
    const T* row = logits + (valid ? t : 0) * ld;
    float s[kVpt];
    if (!sigmoid) {
      load_chunk(row, e0, E, valid, vec != 0, s);
      route_scores<L>(s, false, false);
      *reinterpret_cast<float4*>(&sh_s[tok][e0]) = make_float4(s[0], s[1], s[2], s[3]);
      *reinterpret_cast<float4*>(&sh_s[tok][e0 + 4]) = make_float4(s[4], s[5], s[6], s[7]);
    }
    *reinterpret_cast<float4*>(&sh_d[tok][e0]) = make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<float4*>(&sh_d[tok][e0 + 4]) = make_float4(0.f, 0.f, 0.f, 0.f);
    int e[SLOTS];
    float p[SLOTS], dw[SLOTS];
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      const int r = q * L + sub;
      e[q] = -1;
      p[q] = dw[q] = 0.f;
      if (valid && r < k) {
        const long long id = selected[t * k + r];
        dw[q] = d_weights[t * k + r];
        if (id < 0 || id >= E) raise_fault(kFaultBadExpert);
        else e[q] = static_cast<int>(id);
      }
    }
    __syncwarp();
    float total = 0.f, dot = 0.f;
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      if (e[q] >= 0)
        p[q] = sigmoid ? sigmoid_score(to_f32(row[e[q]])) : sh_s[tok][e[q]];
      total += p[q];
      dot = fmaf(dw[q], p[q], dot);
    }
    float f = scale, sub_dw = 0.f;
    if (normalize) {
      f = 1.0f / (group_sum<L>(total) + kRouteNormEps);
      sub_dw = group_sum<L>(dot) * f;
      f *= scale;
    }
    float through = 0.f;  // softmax: sum of ds p
#pragma unroll
    for (int q = 0; q < SLOTS; ++q) {
      const float d = f * (dw[q] - sub_dw);
      through = fmaf(e[q] >= 0 ? d : 0.f, p[q], through);
      if (e[q] >= 0) sh_d[tok][e[q]] = sigmoid ? d * p[q] * (1.0f - p[q]) : d;
    }
    if (!sigmoid) through = group_sum<L>(through);
    __syncwarp();
    float o[kVpt];
    *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(&sh_d[tok][e0]);
    *reinterpret_cast<float4*>(o + 4) = *reinterpret_cast<const float4*>(&sh_d[tok][e0 + 4]);
    if (!sigmoid) {
#pragma unroll
      for (int j = 0; j < kVpt; ++j) o[j] = s[j] * (o[j] - through);
    }
    if (valid) {
      T* out = d_logits + t * E + e0;
      if (vec_out && e0 + kVpt <= E) {
        store_chunk<T, true>(out, o);
        if constexpr (sizeof(T) == 4) store_chunk<T, true>(out + 4, o + 4);
      } else {
#pragma unroll
        for (int j = 0; j < kVpt; ++j)
          if (e0 + j < E) out[j] = from_f32<T>(o[j]);
      }
    }
    __syncwarp();
  }
}

// counts[e] += occurrences of e in ids[0..n); counts start at zero.  Integer sums: the
// order of the additions does not matter.  Ids outside [0, E) are not counted.
__device__ __forceinline__ void count_block(const long long* __restrict__ ids, long long n, int E,
                                            int* sh) {
  for (int e = threadIdx.x; e < E; e += blockDim.x) sh[e] = 0;
  __syncthreads();
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
  auto add = [&](long long e) {
    if (e >= 0 && e < E) atomicAdd(&sh[e], 1);
  };
  for (; i + 3 * step < n; i += 4 * step) {
    const long long a = ids[i], b = ids[i + step], c = ids[i + 2 * step], d = ids[i + 3 * step];
    add(a);
    add(b);
    add(c);
    add(d);
  }
  for (; i < n; i += step) add(ids[i]);
  __syncthreads();
}

__global__ void expert_counts_kernel(const long long* __restrict__ ids, long long n, int E,
                                     int* __restrict__ counts) {
  __shared__ int sh[kRouteMaxExperts];
  count_block(ids, n, E, sh);
  for (int e = threadIdx.x; e < E; e += blockDim.x)
    if (sh[e]) atomicAdd(&counts[e], sh[e]);
}

// out = bias + rate sign(sum(counts) - E counts[e]): exact in integers.  Called by a block of
// kRouteMaxExperts threads or more.
__device__ __forceinline__ void move_bias(const float* __restrict__ bias, long long n, int E,
                                          float rate, float* __restrict__ out) {
  __shared__ long long part[32];
  long long total = n;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = total;
  __syncthreads();
  total = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) total += part[i];
  const int e = threadIdx.x;
  if (e < E) {
    const long long d = total - n * E;
    out[e] = bias[e] + (d > 0 ? rate : (d < 0 ? -rate : 0.f));
  }
}

__global__ void balance_bias_kernel(const float* __restrict__ bias, const int* __restrict__ counts,
                                    int E, float rate, float* __restrict__ out) {
  const int e = threadIdx.x;
  move_bias(bias, e < E ? counts[e] : 0, E, rate, out);
}

// Counts and moves the bias in one launch.  counts: E + 1 zeros, the last of them the number of
// blocks that have added theirs; the last block to do so (none waits) moves the bias.  One block
// alone needs no counts.
__global__ void balance_step_kernel(const long long* __restrict__ ids, long long n, int E,
                                    const float* __restrict__ bias, float rate,
                                    int* __restrict__ counts, float* __restrict__ out) {
  __shared__ int sh[kRouteMaxExperts];
  __shared__ int last;
  count_block(ids, n, E, sh);
  const int e = threadIdx.x;
  long long mine = e < E ? sh[e] : 0;
  if (gridDim.x > 1) {
    for (int i = e; i < E; i += blockDim.x)
      if (sh[i]) atomicAdd(&counts[i], sh[i]);
    __threadfence();
    __syncthreads();
    if (e == 0) last = atomicAdd(&counts[E], 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    mine = e < E ? __ldcg(&counts[e]) : 0;
  }
  move_bias(bias, mine, E, rate, out);
}

}  // namespace b200moe
