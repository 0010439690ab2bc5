// The ragged products for few rows (see few.cu).
#pragma once
#include <cuda_runtime.h>

namespace abacus {
namespace ragged {

// Row counts for which these kernels are the faster path, both sides measured (us forward / with gradients, matrices of 1023 x 1021 to
// 2048 x 2048): fp32, 8 experts of 8 rows 67 / 192 against the tensor-core path's 120 / 290, of 16 rows 119 / 290
// against 120 / 299; bf16 odd, 32 experts of 4 rows 50 / 134 against 60 / 159, of 8 rows 83 / 215 against 60 / 159. The
// bound on all rows is for experts with most of them, whose matrix is read again for every four: with all of 256 rows in
// one of 32 experts these kernels take 243 / 775 against 127 / 452.
constexpr bool few_rows(long long rows, long long experts, bool bf16) {
  return rows <= (bf16 ? 4 : 8) * experts && rows <= 256;
}

struct FewParams {
  const void* a;      // sorted rows (rows, k); for the weights product (rows, m)
  const void* b;      // the experts' matrices; for the weights product sorted rows (rows, n)
  const float* add;   // transposed product: added to the sum (may be null)
  void* out;
  bool a_bf16, b_bf16, out_bf16;
  long long ld_a, ld_b, stride_b, ld_out, ld_add;
  const int* offsets;
  int experts, rows;
  int k, n, m;
  int* status;
};
// out[r] = a[r] B[e], B (k, n).      out[r] = a[r] B[e]^T + add[r], B (n, k).      out[e] = sum_r a[r]^T b[r], (m, n).
cudaError_t launch_few(const FewParams& p, cudaStream_t stream);
cudaError_t launch_few_transposed(const FewParams& p, cudaStream_t stream);
cudaError_t launch_few_weights(const FewParams& p, cudaStream_t stream);

// h = silu(g) u, and (dg, du) from dh, n fp32 numbers each; dg may be dh.
cudaError_t launch_few_swiglu(const float* g, const float* u, float* h, long long n, cudaStream_t stream);
cudaError_t launch_few_swiglu_bwd(const float* dh, const float* g, const float* u, float* dg, float* du, long long n,
                                  cudaStream_t stream);

}  // namespace ragged
}  // namespace abacus
