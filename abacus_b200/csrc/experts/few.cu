// The ragged products for a handful of rows an expert: single tokens, short batches.
//
// Such a product reads each used expert's matrix once and does 2 operations an element and row with it, so the matrices'
// bytes bound it: at 4 bytes an element fp32 FMAs keep up with memory to some 20 rows an expert, at 2 bytes to some 10.
// The tensor-core path pads every expert to 128 rows and, in fp32, first writes its matrices out as bf16 parts (16 bytes
// moved an element in place of 4). Here a matrix is read where it lies, in any alignment, and sums are fp32 FMAs in a
// fixed order. A block takes up to 4 rows of one expert at a time, and of an expert with more reads its part of the matrix
// again from L2. 32 experts of 2048 x 2048 in fp32 take 93 us with a row each (5.8 TB/s) and 131 us with four.
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>
#include "few.h"
#include "offsets.cuh"
#include "sigmoid.cuh"

namespace abacus {
namespace ragged {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Elements of a 16-byte unit, and loading one: `left` elements are inside the row. WIDE: units are aligned and whole.
template <class T>
constexpr int kUnit = 16 / static_cast<int>(sizeof(T));

// Rows of an expert that a block takes at a time. (Eight, with fp32 matrices, took the registers of a third block an SM:
// 242 us for 8 rows of each of 32 experts of 2048 x 2048.)
constexpr int kRows = 4;

template <class T, bool WIDE>
__device__ __forceinline__ void load_unit(const T* p, int left, float (&v)[kUnit<T>]) {
  if constexpr (WIDE) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (left > 0) raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kUnit<T>; ++i) v[i] = i < left ? to_f(p[i]) : 0.f;
  }
}

__device__ __forceinline__ int offset_at(const FewParams& p, int e) { return e == 0 ? 0 : min(max(p.offsets[e], 0), p.rows); }

template <class TO>
__device__ __forceinline__ void zero_columns(const FewParams& p, int col0, int cols) {
  const int width = min(cols, p.n - col0);
  if (width <= 0) return;
  for (long long r = offset_at(p, p.experts) + threadIdx.x / 32; r < p.rows; r += kWarps)
    for (int c = threadIdx.x % 32; c < width; c += 32) put(static_cast<TO*>(p.out) + r * p.ld_out + col0 + c, 0.f);
}

// ------------------------------------------------------------------ out[r] = a[r] B[e]
// A block makes 8 units of columns (128 bytes of every row of B); 32 groups of 8 threads take the contraction in turn.
constexpr int kChunk = 512;  // contraction elements of the rows kept in shared memory

template <int R, class TA, class TB, class TO, bool WIDE>
__device__ void few_block(const FewParams& p, int e, int r0, int rows, int col0, float* smem) {
  constexpr int V = kUnit<TB>, C = 8 * V;
  const TA* a = static_cast<const TA*>(p.a);
  const TB* b = static_cast<const TB*>(p.b) + e * p.stride_b + col0;
  const int group = threadIdx.x / 8, place = threadIdx.x % 8;
  const int left = p.n - col0 - place * V;
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[r][v] = 0.f;
  for (int k0 = 0; k0 < p.k; k0 += kChunk) {
    const int count = min(kChunk, p.k - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < R * kChunk; i += kThreads) {
      const int r = i / kChunk, kk = i % kChunk;
      smem[kk * R + r] = r < rows && kk < count ? to_f(a[(r0 + r) * p.ld_a + k0 + kk]) : 0.f;
    }
    __syncthreads();
#pragma unroll 4
    for (int kk = group; kk < count; kk += kThreads / 8) {
      float w[V];
      load_unit<TB, WIDE>(b + (k0 + kk) * p.ld_b + place * V, left, w);
      float x[R];
      if constexpr (R >= 4) {
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          const float4 q = *reinterpret_cast<const float4*>(smem + kk * R + r);
          x[r] = q.x; x[r + 1] = q.y; x[r + 2] = q.z; x[r + 3] = q.w;
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = smem[kk * R + r];
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[r][v] = fmaf(x[r], w[v], acc[r][v]);
    }
  }
  // The four groups of a warp, then the warps.
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      acc[r][v] += __shfl_xor_sync(0xffffffffu, acc[r][v], 8);
      acc[r][v] += __shfl_xor_sync(0xffffffffu, acc[r][v], 16);
    }
  __syncthreads();
  if (threadIdx.x % 32 < 8) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) smem[(threadIdx.x / 32 * R + r) * C + place * V + v] = acc[r][v];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * C; i += kThreads) {
    const int r = i / C, c = i % C;
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += smem[(w * R + r) * C + c];
    if (r < rows && col0 + c < p.n) put(static_cast<TO*>(p.out) + (r0 + r) * p.ld_out + col0 + c, sum);
  }
}

template <class TA, class TB, class TO, bool WIDE>
__global__ void __launch_bounds__(kThreads) few_kernel(const FewParams p) {
  constexpr int C = 8 * kUnit<TB>;
  constexpr int kFloats = kRows * (kChunk > kWarps * C ? kChunk : kWarps * C);
  __shared__ __align__(16) float smem[kFloats];
  const int e = blockIdx.y, col0 = blockIdx.x * C;
  if (e == p.experts) {
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x < 32)
      check_offsets(p.offsets, p.experts, p.rows, threadIdx.x, p.status);
    if (blockIdx.z == 0) zero_columns<TO>(p, col0, C);
    return;
  }
  const int end = offset_at(p, e + 1);
  for (int r0 = offset_at(p, e) + blockIdx.z * kRows; r0 < end; r0 += gridDim.z * kRows) {
    const int rows = min(kRows, end - r0);
    if (rows == 1) few_block<1, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
    else if (rows == 2) few_block<2, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
    else few_block<4, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
  }
}

// ------------------------------------------------------------------ out[r] = a[r] B[e]^T + add[r]
// A warp takes 4 rows of B at a time, its lanes along them; the rows of a wait in shared memory.
constexpr int kSpan = 1024;  // contraction elements kept
constexpr int kDots = 4;

template <int R, class TA, class TB, class TO, bool WIDE>
__device__ void dot_block(const FewParams& p, int e, int r0, int rows, int col0, float* smem) {
  constexpr int V = kUnit<TB>;
  const TA* a = static_cast<const TA*>(p.a);
  const int lane = threadIdx.x % 32, c0 = col0 + threadIdx.x / 32 * kDots;
  const TB* b = static_cast<const TB*>(p.b) + e * p.stride_b;
  float acc[R][kDots];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kDots; ++j) acc[r][j] = 0.f;
  for (int k0 = 0; k0 < p.k; k0 += kSpan) {
    const int count = min(kSpan, p.k - k0);
    __syncthreads();
    for (int i = threadIdx.x; i < R * kSpan; i += kThreads) {
      const int r = i / kSpan, kk = i % kSpan;
      smem[i] = r < rows && kk < count ? to_f(a[(r0 + r) * p.ld_a + k0 + kk]) : 0.f;
    }
    __syncthreads();
    if (c0 < p.n) {
#pragma unroll 2
      for (int kk = lane * V; kk < count; kk += 32 * V) {
        float w[kDots][V];
#pragma unroll
        for (int j = 0; j < kDots; ++j)
          load_unit<TB, WIDE>(b + min(c0 + j, p.n - 1) * p.ld_b + k0 + kk, count - kk, w[j]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float x[V];
#pragma unroll
          for (int v = 0; v < V; v += 4) {
            const float4 q = *reinterpret_cast<const float4*>(smem + r * kSpan + kk + v);
            x[v] = q.x; x[v + 1] = q.y; x[v + 2] = q.z; x[v + 3] = q.w;
          }
#pragma unroll
          for (int j = 0; j < kDots; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[r][j] = fmaf(x[v], w[j][v], acc[r][j]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < kDots; ++j) {
#pragma unroll
      for (int d = 16; d > 0; d /= 2) acc[r][j] += __shfl_xor_sync(0xffffffffu, acc[r][j], d);
      if (lane == 0 && r < rows && c0 + j < p.n) {
        const float more = p.add ? p.add[(r0 + r) * p.ld_add + c0 + j] : 0.f;
        put(static_cast<TO*>(p.out) + (r0 + r) * p.ld_out + c0 + j, acc[r][j] + more);
      }
    }
}

template <class TA, class TB, class TO, bool WIDE>
__global__ void __launch_bounds__(kThreads) dot_kernel(const FewParams p) {
  __shared__ __align__(16) float smem[kRows * kSpan];
  constexpr int C = kWarps * kDots;
  const int e = blockIdx.y, col0 = blockIdx.x * C;
  if (e == p.experts) {
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x < 32)
      check_offsets(p.offsets, p.experts, p.rows, threadIdx.x, p.status);
    if (blockIdx.z == 0) zero_columns<TO>(p, col0, C);
    return;
  }
  const int end = offset_at(p, e + 1);
  for (int r0 = offset_at(p, e) + blockIdx.z * kRows; r0 < end; r0 += gridDim.z * kRows) {
    const int rows = min(kRows, end - r0);
    if (rows == 1) dot_block<1, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
    else if (rows == 2) dot_block<2, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
    else dot_block<4, TA, TB, TO, WIDE>(p, e, r0, rows, col0, smem);
  }
}

// ------------------------------------------------------------------ out[e] = sum_r a[r]^T b[r]
// Bound by writing the result. A lane makes 4 columns of 8 rows of it, going once over the expert's rows.
constexpr int kOutRows = 8;

template <class TA, class TB, class TO, bool WIDE>
__global__ void __launch_bounds__(kThreads) outer_kernel(const FewParams p) {
  const int e = blockIdx.z, lane = threadIdx.x % 32;
  if (blockIdx.x == 0 && blockIdx.y == 0 && e == 0 && threadIdx.x < 32)
    check_offsets(p.offsets, p.experts, p.rows, lane, p.status);
  // Four columns side by side where they can be stored at once, else 32 apart.
  const int n0 = blockIdx.x * 128 + lane * (WIDE ? 4 : 1), m0 = (blockIdx.y * kWarps + threadIdx.x / 32) * kOutRows;
  constexpr int kApart = WIDE ? 1 : 32;
  if (m0 >= p.m || n0 >= p.n) return;
  const TA* a = static_cast<const TA*>(p.a);
  const TB* b = static_cast<const TB*>(p.b);
  float acc[kOutRows][4];
#pragma unroll
  for (int i = 0; i < kOutRows; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  const int end = offset_at(p, e + 1);
#pragma unroll 2
  for (long long r = offset_at(p, e); r < end; ++r) {
    float x[kOutRows], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = n0 + j * kApart < p.n ? to_f(b[r * p.ld_b + n0 + j * kApart]) : 0.f;
#pragma unroll
    for (int i = 0; i < kOutRows; ++i) x[i] = m0 + i < p.m ? to_f(a[r * p.ld_a + m0 + i]) : 0.f;
#pragma unroll
    for (int i = 0; i < kOutRows; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
  TO* out = static_cast<TO*>(p.out) + (static_cast<long long>(e) * p.m + m0) * p.n + n0;
#pragma unroll
  for (int i = 0; i < kOutRows; ++i) {
    if (m0 + i >= p.m) break;
    TO* row = out + static_cast<long long>(i) * p.n;
    if constexpr (WIDE && sizeof(TO) == 4) {  // WIDE: rows of the result hold whole aligned groups of 4
      *reinterpret_cast<float4*>(row) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    } else if constexpr (WIDE) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(acc[i][0], acc[i][1]), hi = __floats2bfloat162_rn(acc[i][2], acc[i][3]);
      *reinterpret_cast<uint2*>(row) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + j * kApart < p.n) put(row + j * kApart, acc[i][j]);
    }
  }
}

__global__ void __launch_bounds__(kThreads) few_swiglu_kernel(const float* g, const float* u, float* h, long long n) {
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * kThreads)
    h[i] = g[i] * sigmoid<24>(g[i]) * u[i];
}

__global__ void __launch_bounds__(kThreads) few_swiglu_bwd_kernel(const float* dh, const float* g, const float* u, float* dg,
                                                                  float* du, long long n) {
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * kThreads) {
    const float x = g[i], sig = sigmoid<24>(x), through = dh[i] * sig;
    dg[i] = through * u[i] * (1.f + x * (1.f - sig));
    du[i] = through * x;
  }
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// The matrices' rows are made of whole aligned 16-byte units.
bool wide_b(const FewParams& p, int row_length) {
  const int unit = p.b_bf16 ? 8 : 4;
  return aligned(p.b, 16) && row_length % unit == 0 && p.ld_b % unit == 0 && p.stride_b % unit == 0;
}

// f(zero of a's type, of b's, of the result's) for the combinations that a product is called with: bits 4, 2 and 1 of a
// combination say which of the three are bf16.
template <int... USED, class F>
cudaError_t with_types(const FewParams& p, F&& f) {
  const int which = (p.a_bf16 ? 4 : 0) | (p.b_bf16 ? 2 : 0) | (p.out_bf16 ? 1 : 0);
  auto call = [&](auto used) {
    constexpr int kUsed = decltype(used)::value;
    if (which != kUsed) return false;
    f(std::conditional_t<(kUsed & 4) != 0, __nv_bfloat16, float>{}, std::conditional_t<(kUsed & 2) != 0, __nv_bfloat16, float>{},
      std::conditional_t<(kUsed & 1) != 0, __nv_bfloat16, float>{});
    return true;
  };
  return (call(std::integral_constant<int, USED>{}) || ...) ? cudaGetLastError() : cudaErrorInvalidValue;
}

// Blocks that share an expert's rows, so that an expert which has most of them is not left to one block a strip (256 rows,
// all of one of 32 experts of 2048 x 2816 in fp32: 243 us against 787); those without rows leave at once (evenly spread
// rows: 234 us against 250 for 8 rows of each of 32 experts of 2048 x 2048).
unsigned shares_of(const FewParams& p) { return (p.rows + 31) / 32; }

unsigned blocks_of(long long n) {
  const long long b = (n + kThreads - 1) / kThreads;
  return static_cast<unsigned>(b < 1 ? 1 : b > 2048 ? 2048 : b);
}

}  // namespace

cudaError_t launch_few(const FewParams& p, cudaStream_t stream) {
  const bool wide = wide_b(p, p.n);
  const int cols = 8 * (p.b_bf16 ? 8 : 4);
  const dim3 grid((p.n + cols - 1) / cols, p.experts + 1, shares_of(p));
  return with_types<0, 3, 6, 7>(p, [&](auto a, auto b, auto o) {
    using A = decltype(a);
    using B = decltype(b);
    using O = decltype(o);
    if (wide) few_kernel<A, B, O, true><<<grid, kThreads, 0, stream>>>(p);
    else few_kernel<A, B, O, false><<<grid, kThreads, 0, stream>>>(p);
  });
}

cudaError_t launch_few_transposed(const FewParams& p, cudaStream_t stream) {
  const bool wide = wide_b(p, p.k);
  const dim3 grid((p.n + kWarps * kDots - 1) / (kWarps * kDots), p.experts + 1, shares_of(p));
  return with_types<0, 2, 3, 6, 7>(p, [&](auto a, auto b, auto o) {
    using A = decltype(a);
    using B = decltype(b);
    using O = decltype(o);
    if (wide) dot_kernel<A, B, O, true><<<grid, kThreads, 0, stream>>>(p);
    else dot_kernel<A, B, O, false><<<grid, kThreads, 0, stream>>>(p);
  });
}

cudaError_t launch_few_weights(const FewParams& p, cudaStream_t stream) {
  const bool wide = p.n % 4 == 0 && aligned(p.out, 16);
  const dim3 grid((p.n + 127) / 128, (p.m + kWarps * kOutRows - 1) / (kWarps * kOutRows), p.experts);
  return with_types<0, 3, 5, 7>(p, [&](auto a, auto b, auto o) {
    using A = decltype(a);
    using B = decltype(b);
    using O = decltype(o);
    if (wide) outer_kernel<A, B, O, true><<<grid, kThreads, 0, stream>>>(p);
    else outer_kernel<A, B, O, false><<<grid, kThreads, 0, stream>>>(p);
  });
}

cudaError_t launch_few_swiglu(const float* g, const float* u, float* h, long long n, cudaStream_t stream) {
  few_swiglu_kernel<<<blocks_of(n), kThreads, 0, stream>>>(g, u, h, n);
  return cudaGetLastError();
}

cudaError_t launch_few_swiglu_bwd(const float* dh, const float* g, const float* u, float* dg, float* du, long long n,
                                  cudaStream_t stream) {
  few_swiglu_bwd_kernel<<<blocks_of(n), kThreads, 0, stream>>>(dh, g, u, dg, du, n);
  return cudaGetLastError();
}

}  // namespace ragged
}  // namespace abacus
