// Rows of a mixture of experts: sorting (token, choice) assignments by expert,
// gathering token rows into that order, and summing the experts' rows back.
//
// With assignment i = t K + k of token t to expert e(i) (an id outside [0, E)
// drops it), `order` is the stable sort of the assignments by e, dropped ones
// last; `slot` its inverse, -1 for a dropped one; offsets[e] the first sorted
// row of expert e. Then
//
//   dispatch:  xs[slot(t, k)] = x[t]           d x[t] = sum_k d xs[slot(t, k)]
//   combine:   out[t] = sum_k w(t, k) ys[slot(t, k)]
//              d ys[slot(t, k)] = w(t, k) d out[t]
//              d w(t, k) = <ys[slot(t, k)], d out[t]>
//
// and sorted rows at or after offsets[E] are zeros (xs, d ys).
//
// The sort is a counting sort, stable because every warp takes a contiguous
// run of assignments and ranks equal experts by lane: one launch up to 1024
// assignments, above that one more that counts per part. No atomic decides a
// place, so results repeat bit for bit. Every block of the second launch adds up
// all parts' counts of all bins, so its work grows as their square: 524,288
// assignments take 40 us over 128 experts, 66 over 256 and 222 over 1024.
//
// The row kernels are bound by memory; each row is read once and written once:
// 65536 tokens, 2 choices, 768 bf16 take 46 us to dispatch (6.5 TB/s), 55 us to
// combine (5.5) and 77 us for the gradients of that (6.5; 86 with the launch, one
// call after another); the plan takes 7 us.
// One warp takes a token: it reads x[t] once for its K copies, and sums its K
// rows in the order of k, in fp32. Rows move in the widest unit (16 bytes down
// to one element) that the row length and the pointers' alignment allow.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <algorithm>
#include "../common/host.h"
#include "expert_rows.h"

namespace abacus {
namespace ops {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kSortWarps = 8;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kPart = 1024;        // assignments of one CTA, or a multiple of it with more than ...
constexpr long long kParts = 1024;  // ... so many CTAs, each of which adds up all of their counts

// Assignments of a CTA of the sort of n.
long long part_of(long long n) { return kPart * ((n + kPart * kParts - 1) / (kPart * kParts)); }

__device__ __forceinline__ int bin_of(const int64_t* indices, long long i, int experts) {
  const int64_t e = indices[i];
  return e >= 0 && e < experts ? static_cast<int>(e) : experts;
}

__global__ void __launch_bounds__(kSortThreads) count_kernel(const int64_t* __restrict__ indices, long long n,
                                                             long long part, int experts, int* __restrict__ counts) {
  __shared__ int hist[kMaxExperts + 1];
  for (int e = threadIdx.x; e <= experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const long long begin = blockIdx.x * part;
  const long long end = min(begin + part, n);
  for (long long i = begin + threadIdx.x; i < end; i += kSortThreads) atomicAdd(&hist[bin_of(indices, i, experts)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kSortThreads)
    counts[static_cast<long long>(e) * gridDim.x + blockIdx.x] = hist[e];
}

// counts: (experts + 1, parts) from count_kernel; unused with one part.
__global__ void __launch_bounds__(kSortThreads) place_kernel(const int64_t* __restrict__ indices, long long n,
                                                             long long part, int experts,
                                                             const int* __restrict__ counts, int* __restrict__ offsets,
                                                             int* __restrict__ order, int* __restrict__ slot) {
  extern __shared__ int smem[];
  const int bins = experts + 1, parts = gridDim.x;
  int* start = smem;           // [bins] rows of all bins before this one
  int* cursor = smem + bins;   // [warps][bins] next place of a warp's assignments
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) cursor[i] = 0;
  __syncthreads();
  // A warp's run of this part, in whole groups of 32.
  const long long run = part / kSortWarps;
  const long long begin = blockIdx.x * part + warp * run;
  const long long end = min(begin + run, n);
  for (long long i = begin + lane; i < end; i += 32) atomicAdd(&cursor[warp * bins + bin_of(indices, i, experts)], 1);
  __syncthreads();
  for (int e = warp; e < bins; e += kSortWarps) {
    int before = 0, all = 0;
    if (parts > 1) {
      for (int p = lane; p < parts; p += 32) {
        const int c = counts[static_cast<long long>(e) * parts + p];
        all += c;
        before += p < static_cast<int>(blockIdx.x) ? c : 0;
      }
      all = __reduce_add_sync(0xffffffffu, all);
      before = __reduce_add_sync(0xffffffffu, before);
    }
    // Lane w: where warp w's assignments to this bin start.
    const int mine = lane < kSortWarps ? cursor[lane * bins + e] : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < kSortWarps; d *= 2) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (lane < kSortWarps) cursor[lane * bins + e] = before + sum - mine;
    if (lane == kSortWarps - 1) start[e] = parts > 1 ? all : sum;
  }
  __syncthreads();
  if (warp == 0) {  // exclusive sum over the bins
    int carry = 0;
    for (int e0 = 0; e0 < bins; e0 += 32) {
      const int e = e0 + lane;
      const int v = e < bins ? start[e] : 0;
      int sum = v;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
      }
      if (e < bins) {
        start[e] = carry + sum - v;
        if (blockIdx.x == 0) offsets[e] = carry + sum - v;  // bin E starts where the last expert ends
      }
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __syncthreads();
  for (long long i0 = begin; i0 < end; i0 += 32) {
    const long long i = i0 + lane;
    const bool in = i < end;
    const int e = in ? bin_of(indices, i, experts) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    int place = 0;
    if (in) place = cursor[warp * bins + e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (in) {
      if (lane == 31 - __clz(same)) cursor[warp * bins + e] = place + 1;
      place += start[e];
      order[place] = static_cast<int>(i);
      slot[i] = e < experts ? place : -1;
    }
    __syncwarp();
  }
}

template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <class T, int N>
__device__ __forceinline__ void zero_tail(T* rows, long long count, const int* end, long long packs, long long warp,
                                          long long warps, int lane) {
  Pack<T, N> zero;
#pragma unroll
  for (int e = 0; e < N; ++e) zero.v[e] = from_float<T>(0.f);
  for (long long r = max(*end, 0) + warp; r < count; r += warps) {
    Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(rows) + r * packs;
    for (long long c = lane; c < packs; c += 32) dst[c] = zero;
  }
}

template <class T, int N>
__global__ void __launch_bounds__(256) dispatch_kernel(const T* __restrict__ x, long long ld, const int* __restrict__ slot,
                                                       const int* __restrict__ end, T* __restrict__ xs, long long tokens,
                                                       int choices, long long packs) {
  const int lane = threadIdx.x % 32;
  const long long warp = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const long long warps = static_cast<long long>(gridDim.x) * blockDim.x / 32;
  const long long count = tokens * choices;
  for (long long t = warp; t < tokens; t += warps) {
    const Pack<T, N>* src = reinterpret_cast<const Pack<T, N>*>(x + t * ld);
    for (long long c = lane; c < packs; c += 128) {
      Pack<T, N> v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + 32 * j < packs) v[j] = src[c + 32 * j];
      for (int k = 0; k < choices; ++k) {
        const long long s = slot[t * choices + k];
        if (s < 0 || s >= count) continue;
        Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(xs) + s * packs;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + 32 * j < packs) dst[c + 32 * j] = v[j];
      }
    }
  }
  zero_tail<T, N>(xs, count, end, packs, warp, warps, lane);
}

constexpr int units_at_once(int n) { return n >= 8 ? 1 : n == 4 ? 2 : 4; }

// out[t] = sum_k w(t, k) ys[slot(t, k)], or without weights the plain sum. A lane sums several units at once where they
// are narrow, so that about as many bytes are in flight (at 8-byte units one at a time left half of the bandwidth unused;
// two 16-byte bf16 units at a time cost registers and were slower, 63 us against 55 for 65536 tokens of 768).
template <class T, int N>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ ys, const float* __restrict__ weights,
                                                      const int* __restrict__ slot, T* __restrict__ out, long long tokens,
                                                      int choices, long long packs) {
  constexpr int kUnits = units_at_once(N);
  const int lane = threadIdx.x % 32;
  const long long warp = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const long long warps = static_cast<long long>(gridDim.x) * blockDim.x / 32;
  const long long count = tokens * choices;
  for (long long t = warp; t < tokens; t += warps) {
    Pack<T, N>* dst = reinterpret_cast<Pack<T, N>*>(out) + t * packs;
    for (long long c = lane; c < packs; c += 32 * kUnits) {
      float acc[kUnits][N];
#pragma unroll
      for (int j = 0; j < kUnits; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) acc[j][e] = 0.f;
#pragma unroll 2
      for (int k = 0; k < choices; ++k) {
        const long long s = slot[t * choices + k];
        if (s < 0 || s >= count) continue;
        const float w = weights ? weights[t * choices + k] : 1.f;
        const Pack<T, N>* src = reinterpret_cast<const Pack<T, N>*>(ys) + s * packs + c;
        Pack<T, N> y[kUnits];
#pragma unroll
        for (int j = 0; j < kUnits; ++j)
          if (c + 32 * j < packs) y[j] = src[32 * j];
#pragma unroll
        for (int j = 0; j < kUnits; ++j)
          if (c + 32 * j < packs)
#pragma unroll
            for (int e = 0; e < N; ++e) acc[j][e] = fmaf(w, to_float(y[j].v[e]), acc[j][e]);
      }
#pragma unroll
      for (int j = 0; j < kUnits; ++j) {
        Pack<T, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = from_float<T>(acc[j][e]);
        if (c + 32 * j < packs) dst[c + 32 * j] = o;
      }
    }
  }
}

// GROUP choices of a token at a time, so that d out[t] is read once for them: two where the number of choices is even, one
// where it is odd. Two at a time against one, 65536 tokens with 2 choices: bf16 rows of 768 86 against 101 us, of 770 (4-byte
// units) 125 against 147, fp32 rows of 768 159 against 169; 8-byte units lose by it (bf16 772 120 against 116, fp32 770 191
// against 183). An odd number taken by two with a last one alone would make three choices of 768 bf16 116 us in place of
// 141, and 9001 tokens' three of 770 fp32 52 in place of 43.
template <class T, int N, int GROUP>
__global__ void __launch_bounds__(256) combine_bwd_kernel(const T* __restrict__ dout, const T* __restrict__ ys,
                                                          const float* __restrict__ weights, const int* __restrict__ slot,
                                                          const int* __restrict__ end, T* __restrict__ dys,
                                                          float* __restrict__ dweights, long long tokens, int choices,
                                                          long long packs) {
  constexpr int kUnits = units_at_once(N);
  const int lane = threadIdx.x % 32;
  const long long warp = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  const long long warps = static_cast<long long>(gridDim.x) * blockDim.x / 32;
  const long long count = tokens * choices;
  for (long long t = warp; t < tokens; t += warps) {
    const Pack<T, N>* d = reinterpret_cast<const Pack<T, N>*>(dout) + t * packs;
    for (int k = 0; k < choices; k += GROUP) {
      // A dropped choice reads row 0 (loads without conditions overlap better) and stores nothing.
      long long row[GROUP];
      bool kept[GROUP], any = false;
      float w[GROUP], dot[GROUP];
#pragma unroll
      for (int i = 0; i < GROUP; ++i) {
        const long long r = slot[t * choices + k + i];
        kept[i] = r >= 0 && r < count;
        any = any || kept[i];
        row[i] = (kept[i] ? r : 0) * packs;
        w[i] = weights[t * choices + k + i];
        dot[i] = 0.f;
      }
      if (any) {
#pragma unroll 2
        for (long long c = lane; c < packs; c += 32 * kUnits) {
          Pack<T, N> a[kUnits], y[GROUP][kUnits];
#pragma unroll
          for (int j = 0; j < kUnits; ++j) {
            if (c + 32 * j >= packs) continue;
            a[j] = d[c + 32 * j];
#pragma unroll
            for (int i = 0; i < GROUP; ++i) y[i][j] = reinterpret_cast<const Pack<T, N>*>(ys)[row[i] + c + 32 * j];
          }
#pragma unroll
          for (int j = 0; j < kUnits; ++j) {
            if (c + 32 * j >= packs) continue;
#pragma unroll
            for (int i = 0; i < GROUP; ++i) {
              Pack<T, N> o;
#pragma unroll
              for (int e = 0; e < N; ++e) {
                const float g = to_float(a[j].v[e]);
                dot[i] = fmaf(g, to_float(y[i][j].v[e]), dot[i]);
                o.v[e] = from_float<T>(w[i] * g);
              }
              if (kept[i]) reinterpret_cast<Pack<T, N>*>(dys)[row[i] + c + 32 * j] = o;
            }
          }
        }
      }
#pragma unroll
      for (int m = 16; m > 0; m /= 2) {
#pragma unroll
        for (int i = 0; i < GROUP; ++i) dot[i] += __shfl_xor_sync(0xffffffffu, dot[i], m);
      }
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < GROUP; ++i) dweights[t * choices + k + i] = kept[i] ? dot[i] : 0.f;
      }
    }
  }
  zero_tail<T, N>(dys, count, end, packs, warp, warps, lane);
}

int row_blocks(long long tokens, const torch::Tensor& t) {
  const long long sms = at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount;
  return static_cast<int>(std::max<long long>(1, std::min<long long>((tokens + 7) / 8, sms * 8)));
}

// Elements of the widest unit that divides the row length (and every row's address).
int pack_of(int64_t dim, int64_t ld, int element, std::initializer_list<const void*> ptrs) {
  int n = 16 / element;
  while (n > 1) {
    bool ok = dim % n == 0 && ld % n == 0;
    for (const void* p : ptrs) ok = ok && reinterpret_cast<uintptr_t>(p) % (n * element) == 0;
    if (ok) return n;
    n /= 2;
  }
  return 1;
}

template <class F>
void with_pack(const torch::Tensor& t, int n, F&& f) {
  if (t.scalar_type() == torch::kFloat32) {
    if (n == 4) f(float{}, std::integral_constant<int, 4>{});
    else if (n == 2) f(float{}, std::integral_constant<int, 2>{});
    else f(float{}, std::integral_constant<int, 1>{});
  } else {
    if (n == 8) f(__nv_bfloat16{}, std::integral_constant<int, 8>{});
    else if (n == 4) f(__nv_bfloat16{}, std::integral_constant<int, 4>{});
    else if (n == 2) f(__nv_bfloat16{}, std::integral_constant<int, 2>{});
    else f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
  }
}

void check_rows(const torch::Tensor& t, const char* name) {
  // (The stride of a single column says nothing: a transposed row has a stride of its length there.)
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&
                  (t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16),
              name, " must be a 2-D fp32 or bf16 CUDA tensor with unit inner stride");
}

void check_slot(const torch::Tensor& slot) {
  TORCH_CHECK(slot.is_cuda() && slot.dim() == 2 && slot.scalar_type() == torch::kInt32 && slot.is_contiguous(),
              "slot must be a contiguous 2-D int32 CUDA tensor");
}

const int* end_of(const torch::Tensor& offsets) {
  TORCH_CHECK(offsets.is_cuda() && offsets.dim() == 1 && offsets.scalar_type() == torch::kInt32 &&
                  offsets.is_contiguous() && offsets.numel() >= 2,
              "offsets must be a contiguous int32 CUDA tensor of experts + 1 values");
  return offsets.data_ptr<int>() + offsets.numel() - 1;
}

}  // namespace

int64_t expert_plan_parts(int64_t n) { return n == 0 ? 0 : (n + part_of(n) - 1) / part_of(n); }

void expert_plan(torch::Tensor indices, int64_t n_experts, torch::Tensor offsets, torch::Tensor order,
                 torch::Tensor slot, torch::Tensor counts) {
  const c10::cuda::CUDAGuard guard(indices.device());
  const long long n = indices.numel();
  const long long parts = expert_plan_parts(n);
  TORCH_CHECK(indices.is_cuda() && indices.scalar_type() == torch::kInt64 && indices.is_contiguous(),
              "indices must be a contiguous int64 CUDA tensor");
  TORCH_CHECK(n_experts >= 1 && n_experts <= kMaxExperts, "expert_plan takes 1 to ", kMaxExperts, " experts, got ", n_experts);
  TORCH_CHECK(n < (1ll << 31) - kPart, "too many assignments");
  for (const auto* t : {&offsets, &order, &slot, &counts})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == torch::kInt32 && t->is_contiguous(), "expert_plan outputs are int32");
  TORCH_CHECK(offsets.numel() == n_experts + 1 && order.numel() == n && slot.numel() == n &&
                  (parts <= 1 || counts.numel() >= parts * (n_experts + 1)),
              "expert_plan output sizes");
  const int bins = static_cast<int>(n_experts) + 1;
  const auto stream = at::cuda::getCurrentCUDAStream();
  if (parts > 1) {
    count_kernel<<<static_cast<unsigned>(parts), kSortThreads, 0, stream>>>(
        indices.data_ptr<int64_t>(), n, part_of(n), static_cast<int>(n_experts), counts.data_ptr<int>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    host::note_launch();
  }
  const unsigned grid = static_cast<unsigned>(std::max<long long>(parts, 1));  // no assignments: the offsets are still written
  place_kernel<<<grid, kSortThreads, sizeof(int) * bins * (1 + kSortWarps), stream>>>(
      indices.data_ptr<int64_t>(), n, part_of(n), static_cast<int>(n_experts), parts > 1 ? counts.data_ptr<int>() : nullptr,
      offsets.data_ptr<int>(), order.data_ptr<int>(), slot.data_ptr<int>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  host::note_launch();
}

void expert_dispatch(torch::Tensor x, torch::Tensor slot, torch::Tensor offsets, torch::Tensor xs) {
  const c10::cuda::CUDAGuard guard(x.device());
  check_rows(x, "x");
  check_rows(xs, "xs");
  check_slot(slot);
  const int* end = end_of(offsets);
  const long long tokens = slot.size(0), choices = slot.size(1), dim = x.size(1);
  TORCH_CHECK(x.size(0) == tokens && xs.size(0) == tokens * choices && xs.size(1) == dim && xs.is_contiguous() &&
                  xs.scalar_type() == x.scalar_type(),
              "expert_dispatch shapes");
  if (tokens == 0 || choices == 0 || dim == 0) return;
  const int element = static_cast<int>(x.element_size());
  with_pack(x, pack_of(dim, x.stride(0), element, {x.data_ptr(), xs.data_ptr()}), [&](auto zero, auto n) {
    using T = decltype(zero);
    constexpr int N = decltype(n)::value;
    dispatch_kernel<T, N><<<row_blocks(tokens, x), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
        static_cast<const T*>(x.data_ptr()), x.stride(0), slot.data_ptr<int>(), end, static_cast<T*>(xs.data_ptr()),
        tokens, static_cast<int>(choices), dim / N);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  host::note_launch();
}

void expert_combine(torch::Tensor ys, c10::optional<torch::Tensor> weights, torch::Tensor slot, torch::Tensor out) {
  const c10::cuda::CUDAGuard guard(ys.device());
  check_rows(ys, "ys");
  check_rows(out, "out");
  check_slot(slot);
  const long long tokens = slot.size(0), choices = slot.size(1), dim = ys.size(1);
  TORCH_CHECK(ys.size(0) == tokens * choices && ys.is_contiguous() && out.size(0) == tokens && out.size(1) == dim &&
                  out.is_contiguous() && out.scalar_type() == ys.scalar_type(),
              "expert_combine shapes");
  if (weights)
    TORCH_CHECK(weights->is_cuda() && weights->scalar_type() == torch::kFloat32 && weights->is_contiguous() &&
                    weights->numel() == tokens * choices,
                "weights must be a contiguous fp32 CUDA tensor of the slots' shape");
  if (tokens == 0 || dim == 0) return;
  if (choices == 0) {
    out.zero_();
    return;
  }
  const int element = static_cast<int>(ys.element_size());
  with_pack(ys, pack_of(dim, dim, element, {ys.data_ptr(), out.data_ptr()}), [&](auto zero, auto n) {
    using T = decltype(zero);
    constexpr int N = decltype(n)::value;
    combine_kernel<T, N><<<row_blocks(tokens, ys), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
        static_cast<const T*>(ys.data_ptr()), weights ? weights->data_ptr<float>() : nullptr, slot.data_ptr<int>(),
        static_cast<T*>(out.data_ptr()), tokens, static_cast<int>(choices), dim / N);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  host::note_launch();
}

void expert_combine_bwd(torch::Tensor dout, torch::Tensor ys, torch::Tensor weights, torch::Tensor slot,
                        torch::Tensor offsets, torch::Tensor dys, torch::Tensor dweights) {
  const c10::cuda::CUDAGuard guard(ys.device());
  check_rows(dout, "dout");
  check_rows(ys, "ys");
  check_rows(dys, "dys");
  check_slot(slot);
  const int* end = end_of(offsets);
  const long long tokens = slot.size(0), choices = slot.size(1), dim = ys.size(1);
  TORCH_CHECK(ys.size(0) == tokens * choices && ys.is_contiguous() && dys.sizes() == ys.sizes() && dys.is_contiguous() &&
                  dout.size(0) == tokens && dout.size(1) == dim && dout.is_contiguous() &&
                  dout.scalar_type() == ys.scalar_type() && dys.scalar_type() == ys.scalar_type(),
              "expert_combine_bwd shapes");
  for (const auto* t : {&weights, &dweights})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == torch::kFloat32 && t->is_contiguous() && t->numel() == tokens * choices,
                "weights must be a contiguous fp32 CUDA tensor of the slots' shape");
  if (tokens == 0 || choices == 0) return;
  const int element = static_cast<int>(ys.element_size());
  with_pack(ys, pack_of(dim, dim, element, {ys.data_ptr(), dout.data_ptr(), dys.data_ptr()}), [&](auto zero, auto n) {
    using T = decltype(zero);
    constexpr int N = decltype(n)::value;
    const auto kernel = choices % 2 == 0 ? combine_bwd_kernel<T, N, 2> : combine_bwd_kernel<T, N, 1>;
    kernel<<<row_blocks(tokens, ys), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
        static_cast<const T*>(dout.data_ptr()), static_cast<const T*>(ys.data_ptr()), weights.data_ptr<float>(),
        slot.data_ptr<int>(), end, static_cast<T*>(dys.data_ptr()), dweights.data_ptr<float>(), tokens,
        static_cast<int>(choices), dim / N);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  host::note_launch();
}

}  // namespace ops
}  // namespace abacus
