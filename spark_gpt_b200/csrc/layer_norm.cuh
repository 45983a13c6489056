// Layer norm, forward and backward.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) r, y = h w + b
//   g = dy w;  dx = r (g - mean(g) - h mean(g h));  dw = sum_t dy h;  db = sum_t dy
//
// All sums are fp32; y and dx are rounded once, to the rows' type.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "router.cuh"  // to_f32

namespace b200moe {

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Sum over the block (every thread gets it); `sh` holds 32 floats.
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x % 32 < (blockDim.x >> 5) ? sh[threadIdx.x % 32] : 0.f;
  return warp_sum(v);
}

constexpr int kNormThreads = 256;

// ---------------------------------------------------------------------------
// pairs of fp32 values in one 64-bit register: one instruction for both
// ---------------------------------------------------------------------------
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  const float2 v = unpack(a);
  return v.x + v.y;
}

// ---------------------------------------------------------------------------
// rows of up to 16384 columns: the row stays on the SM
// ---------------------------------------------------------------------------
// G threads take a row, NE columns each, in chunks of W consecutive columns: chunk i of
// thread t starts at column (i G + t) W.  W is a 16-byte vector where the rows start on 16
// bytes and H is a multiple of it (VEC), else 1, whose loads are coalesced over the threads
// whatever the rows' alignment.  A thread's columns are the same in every row.
template <typename T, bool VEC>
constexpr int norm_width() { return VEC ? 16 / static_cast<int>(sizeof(T)) : 1; }

// NE values of a row as loaded (bf16 vectors stay packed: half the registers), read in pairs.
template <typename T, bool VEC, int NE>
struct RowVals {
  float v[NE];
  __device__ __forceinline__ F2 pair(int p) const { return f2(v[2 * p], v[2 * p + 1]); }
  __device__ __forceinline__ void load(const T* p, int i) {
    if constexpr (VEC) {
      const float4 a = *reinterpret_cast<const float4*>(p);
      v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
    } else {
      v[i] = to_f32(*p);
    }
  }
  __device__ __forceinline__ void zero(int i) {
    constexpr int W = norm_width<T, VEC>();
#pragma unroll
    for (int k = 0; k < W; ++k) v[W * i + k] = 0.f;
  }
};
template <int NE>
struct RowVals<__nv_bfloat16, true, NE> {
  uint32_t v[NE / 2];
  __device__ __forceinline__ F2 pair(int p) const { return f2(bf16_lo(v[p]), bf16_hi(v[p])); }
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int i) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
  }
  __device__ __forceinline__ void zero(int i) {
    v[4 * i] = v[4 * i + 1] = v[4 * i + 2] = v[4 * i + 3] = 0u;
  }
};

// body(i, guard) for the chunks i = 0, STEP, ... < NC of a thread's row, guard being whether the
// chunk may lie past the row's end.  Single-element chunks go in blocks of eight that are
// either whole for every thread, without a test or a branch between their loads, or tested one
// by one.  (Vectors are tested each: the branch keeps the compiler from loading all of a row
// at once, for which there are no registers.)
template <int NC, int STEP, int W, int G, typename Body>
__device__ __forceinline__ void each_chunk(int H, Body&& body) {
  constexpr int B = W > 1 ? NC : (NC < 8 ? NC : 8);
#pragma unroll
  for (int i0 = 0; i0 < NC; i0 += B) {
    if (W == 1 && (i0 + B) * G <= H) {
#pragma unroll
      for (int i = i0; i < i0 + B && i < NC; i += STEP) body(i, std::false_type());
    } else {
#pragma unroll
      for (int i = i0; i < i0 + B && i < NC; i += STEP) body(i, std::true_type());
    }
  }
}

// The W values of a chunk (for W = 1 a single one) to p, rounded to T.
template <typename T, bool VEC>
__device__ __forceinline__ void store_chunk(T* p, const float* o) {
  if constexpr (!VEC) {
    *p = from_f32<T>(o[0]);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]),
                                              pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
  }
}

// fp32 parameters in shared memory: a chunk of eight columns is kept as two halves of four in
// two planes, so that the 16-byte reads of a warp's lanes are consecutive (in column
// order they are 32 bytes apart and take twice the shared-memory cycles); other chunks
// are in column order.
template <int W>
__device__ __forceinline__ int param_at(int c, int plane) {
  return W == 8 ? ((c >> 2) & 1) * plane + (c >> 3) * 4 + (c & 3) : c;
}
template <int W>
__device__ __forceinline__ void stage_params(float* sh, int plane, const float* __restrict__ p,
                                             float missing, int H) {
  for (int c = threadIdx.x; c < H; c += blockDim.x) sh[param_at<W>(c, plane)] = p ? p[c] : missing;
}
// Pairs of the chunk that starts at column c (W > 1).
template <int W>
__device__ __forceinline__ void read_params(const float* sh, int plane, int c, F2 (&o)[W / 2]) {
  if constexpr (W == 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 a = *reinterpret_cast<const float4*>(sh + h * plane + c / 2);
      o[2 * h] = f2(a.x, a.y);
      o[2 * h + 1] = f2(a.z, a.w);
    }
  } else {
    const float4 a = *reinterpret_cast<const float4*>(sh + c);
    o[0] = f2(a.x, a.y);
    o[1] = f2(a.z, a.w);
  }
}

// Sums over the G threads of a row (G a power of two; every thread gets them).  Groups of
// more than a warp meet at a named barrier; `sh` (two halves of G / 32 entries, used in
// turn) needs no second barrier, because a half is written again only after the barrier of the
// sum in between, which every reader of it has passed.
template <int G>
struct GroupSum {
  float2* sh;
  int bar, half;
  template <bool BOTH>
  __device__ __forceinline__ float2 add(float a, float b) {
    constexpr int L = G < 32 ? G : 32;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      if (BOTH) b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if constexpr (G > 32) {
      float2* p = sh + half * (G / 32);
      half ^= 1;
      if ((threadIdx.x & 31) == 0) p[(threadIdx.x % G) / 32] = make_float2(a, b);
      asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(G) : "memory");
      a = 0.f;
      b = 0.f;
#pragma unroll
      for (int i = 0; i < G / 32; ++i) {
        const float2 v = p[i];
        a += v.x;
        if (BOTH) b += v.y;
      }
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float one(float a) { return add<false>(a, 0.f).x; }
  __device__ __forceinline__ float2 two(float a, float b) { return add<true>(a, b); }
};

// cp.async of one chunk (16 bytes, or one fp32 value).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Planes of eight-column chunks hold half of the columns, at most the shape's G NE / 2.
constexpr int norm_plane(int cols) { return cols / 2; }
constexpr int kNormSmem = 224 * 1024;  // shared memory that a block alone on its SM takes at most

// Forward: vector rows go through a ring in shared memory, up to three rows of each group on their
// way while one is computed (one block of 512 threads an SM: 65536 x 1024 bf16 in 44 us, 6.1 TB/s;
// 48 us with the rows loaded to registers and three blocks of 256 threads, 51-53 with two or
// four or with the next row loaded ahead; 41.5 us at the copy bandwidth; 33 M elements in rows
// of 64 bf16 29 us, 40 from registers, of 1024 24, 27; fp32 of 64 40, 50, of 128 the same).
// Rows that are not vectors are loaded to registers.  They are bound by the number of loads and
// stores, four an element, two of them of w and b: in fp32 these stay in registers (33 M
// elements in rows of 1001: 41 us, 44 from shared memory); bf16, with twice the elements to
// the byte, needs the third block more (55 us, 78 with two).
template <typename T, bool VEC, int G, int NE>
struct NormFwdShape {
  static constexpr int W = norm_width<T, VEC>(), CB = W * static_cast<int>(sizeof(T));
  static constexpr bool kRing = VEC;
  static constexpr bool kHold = !VEC && sizeof(T) == 4;  // w and b in registers
  static constexpr int kThreads = kRing || G > kNormThreads ? 512 : kNormThreads;
  static constexpr int kBlocks = kThreads > kNormThreads ? 1 : kHold ? 2 : 3;  // of an SM
  static constexpr int kRows = kThreads / G;
  static constexpr int kRow = G * NE * static_cast<int>(sizeof(T));  // bytes of a row's places
  static constexpr int kParams = kHold ? 0 : 8 * G * NE;
  static constexpr int kFit = (kNormSmem - kParams) / (kRows * kRow);
  static constexpr int kStages = !kRing ? 0 : kFit < 3 ? kFit : 3;
  static constexpr int kSmem = kParams + kStages * kRows * kRow;
};

// Groups of less than a warp share its shuffles, so every group of a block makes the same
// number of rounds; a row past the end is computed on zeros and not stored.
template <typename T, bool VEC, int G, int NE>
__global__ void __launch_bounds__(NormFwdShape<T, VEC, G, NE>::kThreads, NormFwdShape<T, VEC, G, NE>::kBlocks)
layer_norm_rows_fwd_kernel(const T* __restrict__ x, long long ld, const float* __restrict__ w,
                           const float* __restrict__ b, long long rows, int H, float eps,
                           T* __restrict__ y, float* __restrict__ mean,
                           float* __restrict__ rstd) {
  using Shape = NormFwdShape<T, VEC, G, NE>;
  constexpr int W = Shape::W, NC = NE / W, RPB = Shape::kRows, D = Shape::kStages, CB = Shape::CB;
  constexpr int PL = norm_plane(G * NE);
  extern __shared__ __align__(16) float params[];  // w, then b: G NE columns each, then the ring
  __shared__ float2 sh[RPB * 2 * (G > 32 ? G / 32 : 1)];
  const int grp = threadIdx.x / G, t = threadIdx.x % G;
  GroupSum<G> sum{sh + grp * 2 * (G / 32), 1 + grp, 0};
  const float inv = 1.0f / H;
  float* pw = params;
  float* pb = params + G * NE;
  char* ring = reinterpret_cast<char*>(params + 2 * G * NE) + grp * (D * Shape::kRow) + t * CB;
  const long long step = gridDim.x * static_cast<long long>(RPB);
  const long long first = blockIdx.x * static_cast<long long>(RPB);
  auto fetch = [&](long long r, int slot) {
    if (r < rows) {
      const T* xr = x + r * ld;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (i * G + t) * W;
        if (c < H) copy_async<CB>(smem_u32(ring + slot * Shape::kRow + i * G * CB), xr + c);
      }
    }
    copy_async_commit();  // a group for every row keeps the count
  };
  if constexpr (D > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(first + grp + d * step, d);
  }
  float hw[Shape::kHold ? NE : 1], hb[Shape::kHold ? NE : 1];
  if constexpr (Shape::kHold) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int c = i * G + t;
      hw[i] = w && c < H ? w[c] : 1.f;
      hb[i] = b && c < H ? b[c] : 0.f;
    }
  } else {
    stage_params<W>(pw, PL, w, 1.f, H);
    stage_params<W>(pb, PL, b, 0.f, H);
    __syncthreads();
  }
  int slot = 0;
  for (long long r0 = first; r0 < rows; r0 += step) {
    const long long r = r0 + grp;
    const bool in = r < rows;
    const T* xr = x + (in ? r : 0) * ld;
    RowVals<T, VEC, NE> v;
    if constexpr (D > 0) copy_async_wait<D - 1>();
    each_chunk<NC, 1, W, G>(H, [&](int i, auto guard) {
      const int c = (i * G + t) * W;
      if (!in || (guard.value && c >= H)) v.zero(i);
      else if constexpr (D > 0) v.load(reinterpret_cast<const T*>(ring + slot * Shape::kRow + i * G * CB), i);
      else v.load(xr + c, i);
    });
    F2 s0 = f2(0.f, 0.f), s1 = s0;
#pragma unroll
    for (int p = 0; p < NE / 2; p += 2) {
      s0 = add2(s0, v.pair(p));
      s1 = add2(s1, v.pair(p + 1));
    }
    const float mu = sum.one(sum2(add2(s0, s1))) * inv;
    if constexpr (D > 0) {  // the row is in registers: its place is free
      fetch(r + D * step, slot);
      slot = slot + 1 == D ? 0 : slot + 1;
    }
    const F2 nm = f2(-mu, -mu);
    float q = 0.f;
    if constexpr (W > 1) {
      F2 q2 = f2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        if ((i * G + t) * W >= H) continue;
#pragma unroll
        for (int k = 0; k < W / 2; ++k) {
          const F2 d = add2(v.pair(i * (W / 2) + k), nm);
          q2 = fma2(d, d, q2);
        }
      }
      q = sum2(q2);
    } else {
      each_chunk<NC, 1, W, G>(H, [&](int i, auto guard) {
        const float d = !guard.value || i * G + t < H ? v.v[i] - mu : 0.f;
        q = fmaf(d, d, q);
      });
    }
    const float rs = 1.0f / sqrtf(sum.one(q) * inv + eps);
    if (!in) continue;
    const F2 r2 = f2(rs, rs);
    each_chunk<NC, 1, W, G>(H, [&](int i, auto guard) {
      const int c = (i * G + t) * W;
      if (guard.value && c >= H) return;
      float o[W];
      if constexpr (W > 1) {
        F2 ww[W / 2], bb[W / 2];
        read_params<W>(pw, PL, c, ww);
        read_params<W>(pb, PL, c, bb);
#pragma unroll
        for (int k = 0; k < W / 2; ++k) {
          const float2 f = unpack(fma2(mul2(add2(v.pair(i * (W / 2) + k), nm), r2), ww[k], bb[k]));
          o[2 * k] = f.x;
          o[2 * k + 1] = f.y;
        }
      } else {
        if constexpr (Shape::kHold) o[0] = fmaf((v.v[i] - mu) * rs, hw[i], hb[i]);
        else o[0] = fmaf((v.v[i] - mu) * rs, pw[c], pb[c]);
      }
      store_chunk<T, VEC>(y + r * H + c, o);
    });
    if (mean && t == 0) {
      mean[r] = mu;
      rstd[r] = rs;
    }
  }
}

// dx of each row, and the sums over this block's rows of dy h and dy per column, which a thread
// keeps for its columns over all its rows: the rows are read once for both.
//
// The accumulators (2 NE fp32) leave no registers to hold rows in flight, so the rows go
// through shared memory: each thread copies its own chunks of the next rows (two ahead, one
// for the longest) with cp.async and reads back what it copied, so no barrier is needed,
// and the two passes over a row read it from there.  bf16 rows that are not vectors (2-byte
// chunks, which cp.async does not have) are loaded to registers one row ahead and stored to
// their place when the row before is done.
//
// 65536 x 1024 bf16: 66 us (402 MB, 62 us at the copy bandwidth), against 82 us with the rows
// in registers at 16 warps an SM and 75 us with four blocks of 128 threads.

// One block an SM: 384 threads may hold 168 registers each; rows of 256 threads and more
// take 512 threads (128 registers).
template <int G>
constexpr int norm_bwd_block() { return G > 128 ? 512 : 384; }
template <typename T, int NE>
constexpr int norm_stage_bytes() { return 2 * NE * static_cast<int>(sizeof(T)); }  // of a thread
// Shared memory: the weights, then the ring, which the final join of the block's sums reuses
// (2 NE fp32 of each thread).
template <typename T, bool VEC, int G, int NE>
constexpr int norm_bwd_stages() {
  return norm_width<T, VEC>() * static_cast<int>(sizeof(T)) >= 4 &&
                 4 * G * NE + norm_bwd_block<G>() * 2 * norm_stage_bytes<T, NE>() <= kNormSmem
             ? 2 : 1;
}
template <typename T, bool VEC, int G, int NE>
constexpr int norm_bwd_smem() {
  constexpr int ring = norm_bwd_stages<T, VEC, G, NE>() * norm_stage_bytes<T, NE>();
  return 4 * G * NE + norm_bwd_block<G>() * (ring > 8 * NE ? ring : 8 * NE);
}

template <typename T, bool VEC, int G, int NE>
__global__ void __launch_bounds__(norm_bwd_block<G>(), 1)
layer_norm_rows_bwd_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ x,
                           long long ld, const float* __restrict__ w,
                           const float* __restrict__ mean, const float* __restrict__ rstd,
                           long long rows, int H, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int W = norm_width<T, VEC>(), NC = NE / W, NT = norm_bwd_block<G>(), RPB = NT / G;
  constexpr int PL = norm_plane(G * NE), CB = W * static_cast<int>(sizeof(T));
  constexpr int STEP = W > 1 ? 1 : 2, PW = W > 1 ? W / 2 : 1;  // chunks and pairs a turn
  constexpr bool ASYNC = CB >= 4;
  constexpr int D = norm_bwd_stages<T, VEC, G, NE>();
  extern __shared__ __align__(16) float params[];
  __shared__ float2 sh[RPB * 2 * (G > 32 ? G / 32 : 1)];
  const int grp = threadIdx.x / G, t = threadIdx.x % G;
  GroupSum<G> sum{sh + grp * 2 * (G / 32), 1 + grp, 0};
  const float inv = 1.0f / H;
  // the weights of single-element chunks in registers, where there are enough
  constexpr bool HOLD = W == 1 && (sizeof(T) == 4 || G < 256);
  F2 hw[HOLD ? NE / 2 : 1];
  if constexpr (!HOLD) {
    stage_params<W>(params, PL, w, 1.f, H);
    __syncthreads();
  } else {
#pragma unroll
    for (int p = 0; p < NE / 2; ++p) {
      const int c = 2 * p * G + t;
      hw[p] = f2(w && c < H ? w[c] : 1.f, w && c + G < H ? w[c + G] : 1.f);
    }
  }
  // ring of the group: [stage][x, dy][chunk][thread]
  constexpr int ROW = G * NE * static_cast<int>(sizeof(T));
  char* ring = reinterpret_cast<char*>(params + G * NE) + grp * (D * 2 * ROW) + t * CB;
  F2 aw[NE / 2], ab[NE / 2];
#pragma unroll
  for (int p = 0; p < NE / 2; ++p) aw[p] = ab[p] = f2(0.f, 0.f);
  const long long step = gridDim.x * static_cast<long long>(RPB);
  const long long first = blockIdx.x * static_cast<long long>(RPB);

  auto fetch = [&](long long r, int slot) {
    if (r < rows) {
      const T* xr = x + r * ld;
      const T* gr = dy + r * ld_dy;
      char* at = ring + slot * (2 * ROW);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = (i * G + t) * W;
        if (c >= H) continue;
        copy_async<CB>(smem_u32(at + i * G * CB), xr + c);
        copy_async<CB>(smem_u32(at + ROW + i * G * CB), gr + c);
      }
    }
    copy_async_commit();  // a group for every row keeps the count
  };
  // the same in two halves for 2-byte chunks: to registers, and from there to the place
  T hx[ASYNC ? 1 : NE], hg[ASYNC ? 1 : NE];
  auto hold = [&](long long r) {
    const T* xr = x + r * ld;
    const T* gr = dy + r * ld_dy;
    if (r >= rows) return;
    each_chunk<(ASYNC ? 1 : NE), 1, 1, G>(H, [&](int i, auto guard) {
      if (guard.value && i * G + t >= H) return;
      hx[i] = xr[i * G + t];
      hg[i] = gr[i * G + t];
    });
  };
  auto put = [&]() {
#pragma unroll
    for (int i = 0; i < (ASYNC ? 1 : NE); ++i) {
      *reinterpret_cast<T*>(ring + i * G * CB) = hx[i];
      *reinterpret_cast<T*>(ring + ROW + i * G * CB) = hg[i];
    }
  };
  if constexpr (ASYNC) {
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(first + grp + d * step, d);
  } else {
    hold(first + grp);
    put();
  }
  float next_rs = 0.f, next_mu = 0.f;
  if (first + grp < rows) {
    next_rs = rstd[first + grp];
    next_mu = mean[first + grp];
  }
  int slot = 0;
  for (long long r0 = first; r0 < rows; r0 += step) {
    const long long r = r0 + grp;
    const bool in = r < rows;
    const float rs = next_rs, nm = -next_mu * next_rs;
    if (r + step < rows) {
      next_rs = rstd[r + step];
      next_mu = mean[r + step];
    }
    if constexpr (ASYNC) copy_async_wait<D - 1>();
    else hold(r + step);
    const char* at = ring + slot * (2 * ROW);
    const F2 r2 = f2(rs, rs), n2 = f2(nm, nm);
    F2 s1 = f2(0.f, 0.f), s2 = s1;
    // the chunk's pairs of x and dy; for W = 1 a "pair" is two chunks, the second 0 past H
    auto pairs = [&](int i, F2* v, F2* g, bool guard) {
      if constexpr (W == 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(at + i * G * CB);
        const uint4 b = *reinterpret_cast<const uint4*>(at + ROW + i * G * CB);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w}, e[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = f2(bf16_lo(u[k]), bf16_hi(u[k]));
          g[k] = f2(bf16_lo(e[k]), bf16_hi(e[k]));
        }
      } else if constexpr (W == 4) {
        const float4 a = *reinterpret_cast<const float4*>(at + i * G * CB);
        const float4 b = *reinterpret_cast<const float4*>(at + ROW + i * G * CB);
        v[0] = f2(a.x, a.y);
        v[1] = f2(a.z, a.w);
        g[0] = f2(b.x, b.y);
        g[1] = f2(b.z, b.w);
      } else {
        const bool two = !guard || (i + 1) * G + t < H;
        v[0] = f2(to_f32(*reinterpret_cast<const T*>(at + i * G * CB)),
                  two ? to_f32(*reinterpret_cast<const T*>(at + (i + 1) * G * CB)) : 0.f);
        g[0] = f2(to_f32(*reinterpret_cast<const T*>(at + ROW + i * G * CB)),
                  two ? to_f32(*reinterpret_cast<const T*>(at + ROW + (i + 1) * G * CB)) : 0.f);
      }
    };
    auto weights = [&](int i, F2 (&o)[PW]) {
      const int c = (i * G + t) * W;
      if constexpr (W > 1) read_params<W>(params, PL, c, o);
      else if constexpr (HOLD) o[0] = hw[i / 2];
      else o[0] = f2(params[c], c + G < H ? params[c + G] : 0.f);
    };
    if (in) {
      each_chunk<NC, STEP, W, G>(H, [&](int i, auto guard) {
        if (guard.value && (i * G + t) * W >= H) return;
        F2 v[PW], g[PW], ww[PW];
        pairs(i, v, g, guard.value);
        weights(i, ww);
#pragma unroll
        for (int k = 0; k < PW; ++k) {
          const int p = i * W / 2 + k;
          const F2 h = fma2(v[k], r2, n2), gw = mul2(g[k], ww[k]);
          s1 = add2(s1, gw);
          s2 = fma2(gw, h, s2);
          aw[p] = fma2(g[k], h, aw[p]);
          ab[p] = add2(ab[p], g[k]);
        }
      });
    }
    const float2 m = sum.two(sum2(s1), sum2(s2));
    if (in && dx) {
      // dx = r g w + (h (-r c2) + (-r c1)), c1 and c2 the two means
      const float k1 = -rs * m.x * inv, k2 = -rs * m.y * inv;
      const F2 k12 = f2(k1, k1), k22 = f2(k2, k2);
      each_chunk<NC, STEP, W, G>(H, [&](int i, auto guard) {
        const int c = (i * G + t) * W;
        if (guard.value && c >= H) return;
        F2 v[PW], g[PW], ww[PW];
        float o[2 * PW];
        pairs(i, v, g, guard.value);
        weights(i, ww);
#pragma unroll
        for (int k = 0; k < PW; ++k) {
          const F2 h = fma2(v[k], r2, n2);
          const float2 f = unpack(fma2(mul2(g[k], ww[k]), r2, fma2(h, k22, k12)));
          o[2 * k] = f.x;
          o[2 * k + 1] = f.y;
        }
        store_chunk<T, VEC>(dx + r * H + c, o);
        if (W == 1 && (!guard.value || c + G < H)) store_chunk<T, VEC>(dx + r * H + c + G, o + 1);
      });
    }
    if constexpr (ASYNC) {
      fetch(r + D * step, slot);
      slot = slot + 1 == D ? 0 : slot + 1;
    } else {
      put();
    }
  }
  if (!part) return;
  // the block's sums: every group writes its own, then they are added in the groups' order
  if constexpr (ASYNC) copy_async_wait<0>();
  __syncthreads();
  float* cols = params + G * NE;  // [group][dw, db][pair][thread][2]
#pragma unroll
  for (int p = 0; p < NE / 2; ++p) {
    float* at = cols + grp * (2 * G * NE) + (p * G + t) * 2;
    *reinterpret_cast<float2*>(at) = unpack(aw[p]);
    *reinterpret_cast<float2*>(at + G * NE) = unpack(ab[p]);
  }
  __syncthreads();
  float* out = part + static_cast<long long>(blockIdx.x) * 2 * H;
  for (int i = threadIdx.x; i < G * NE; i += NT) {
    const int p = i / (2 * G), th = i / 2 % G, z = i % 2;
    const int c = W > 1 ? (p / PW * G + th) * W + p % PW * 2 + z : (2 * p + z) * G + th;
    if (c >= H) continue;
    float a = 0.f, d = 0.f;
    for (int q = 0; q < RPB; ++q) {
      a += cols[q * (2 * G * NE) + i];
      d += cols[q * (2 * G * NE) + G * NE + i];
    }
    out[c] = a;
    out[H + c] = d;
  }
}

// ---------------------------------------------------------------------------
// longer rows: a block goes over its row once for each sum, by single elements (2048 x 32768 bf16:
// 128 us forward, 306 backward; 42 and 62 at the copy bandwidth)
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_fwd_kernel(const T* __restrict__ x, long long ld, const float* __restrict__ w,
                      const float* __restrict__ b, long long rows, int H, float eps,
                      T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float sh[32];
  for (long long t = blockIdx.x; t < rows; t += gridDim.x) {
    const T* xr = x + t * ld;
    T* yr = y + t * H;
    float s = 0.f;
    for (int c = threadIdx.x; c < H; c += kNormThreads) s += to_f32(xr[c]);
    const float mu = block_sum(s, sh) / H;
    float q = 0.f;
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
      const float d = to_f32(xr[c]) - mu;
      q = fmaf(d, d, q);
    }
    const float r = 1.0f / sqrtf(block_sum(q, sh) / H + eps);
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
      float v = (to_f32(xr[c]) - mu) * r;
      if (w) v *= w[c];
      if (b) v += b[c];
      yr[c] = from_f32<T>(v);
    }
    if (mean && threadIdx.x == 0) {
      mean[t] = mu;
      rstd[t] = r;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_dx_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ x,
                     long long ld, const float* __restrict__ w, const float* __restrict__ mean,
                     const float* __restrict__ rstd, long long rows, int H, T* __restrict__ dx) {
  __shared__ float sh[32];
  for (long long t = blockIdx.x; t < rows; t += gridDim.x) {
    const T* xr = x + t * ld;
    const T* gr = dy + t * ld_dy;
    const float mu = mean[t], r = rstd[t];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
      const float g = to_f32(gr[c]) * (w ? w[c] : 1.f);
      s1 += g;
      s2 = fmaf(g, (to_f32(xr[c]) - mu) * r, s2);
    }
    const float c1 = block_sum(s1, sh) / H;
    const float c2 = block_sum(s2, sh) / H;
    for (int c = threadIdx.x; c < H; c += kNormThreads) {
      const float g = to_f32(gr[c]) * (w ? w[c] : 1.f);
      const float h = (to_f32(xr[c]) - mu) * r;
      dx[t * H + c] = from_f32<T>(r * (g - c1 - h * c2));
    }
  }
}

// Partial column sums over the rows of blockIdx.y (of `parts`): part[y][0..H) of
// dy h and part[y][H..2H) of dy.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
layer_norm_dw_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ x,
                     long long ld, const float* __restrict__ mean, const float* __restrict__ rstd,
                     long long rows, int H, float* __restrict__ part) {
  const int c = blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= H) return;
  const long long per = (rows + gridDim.y - 1) / gridDim.y;
  const long long lo = blockIdx.y * per, hi = min(rows, lo + per);
  float sw = 0.f, sb = 0.f;
  for (long long t = lo; t < hi; ++t) {
    const float g = to_f32(dy[t * ld_dy + c]);
    sw = fmaf(g, (to_f32(x[t * ld + c]) - mean[t]) * rstd[t], sw);
    sb += g;
  }
  float* p = part + 2LL * blockIdx.y * H + c;  // 2 H may pass 32 bits
  p[0] = sw;
  p[static_cast<long long>(H)] = sb;
}

// dw, db: the partials summed in a fixed order, 32 columns a block, eight threads a column.
__global__ void __launch_bounds__(kNormThreads)
layer_norm_dw_sum_kernel(const float* __restrict__ part, int parts, int H, float* __restrict__ dw,
                         float* __restrict__ db) {
  __shared__ float sh[8][32];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const long long c = blockIdx.x * 32LL + lane;
  float s = 0.f;
  if (c < 2LL * H) {
#pragma unroll 4
    for (int p = q; p < parts; p += 8) s += part[2LL * p * H + c];
  }
  sh[q][lane] = s;
  __syncthreads();
  if (q || c >= 2LL * H) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sh[i][lane];
  if (c < H) dw[c] = s;
  else db[c - H] = s;
}

}  // namespace b200moe
