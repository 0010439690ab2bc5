// Matrix products grouped by expert over rows of ragged counts: parameters and
// launchers shared by the kernel's translation units and the torch bindings.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

namespace abacus {
namespace ragged {

constexpr int kMaxExperts = 256;

// Rows whose products a weight gradient with one plane sums in one accumulator; with more rows in an expert it needs the
// workspace of Params::partial.
constexpr int kRunRows = 1 << 14;

enum Epilogue : int { kStore = 0, kSwiGLU = 1, kSwiGLUBwd = 2 };

// What a launch computes, over sorted rows r of expert e = [offsets[e], offsets[e + 1]):
//  rows, store:      out0[r] = sum over segments s of a[s][r] B[s][e]
//  rows, SwiGLU:     out0 = a B[0], out1 = a B[1], out2 = silu(out0) * out1
//  rows, SwiGLU bwd: dh = a B[0]; out0 = dh u sig (1 + g (1 - sig)), out1 = dh g sig  (g = in0, u = in1; one plane)
//  weights:          out_o[e] = sum over r of a[r]^T b[o][r]
// Rows at or after offsets[experts] get zeros. What the SwiGLU forms hand to the next product (its out2, its
// backward's out0 and out1) is written as that product's operand, in bf16 planes; their rows and those of g and u are
// padded to whole 16-byte units, which the other results (the caller's contiguous tensors) may not be.
struct alignas(64) Params {
  CUtensorMap a[2];
  CUtensorMap b[2];
  const int* offsets;
  int experts;
  int rows;      // all sorted rows, owned or not
  int k;         // rows: length of a contraction segment
  int segments;  // rows: 1 or 2
  int m;         // weights: rows of an output matrix
  int n;         // columns of an output (hidden units for SwiGLU)
  int n_tiles;   // column tiles of one output
  int outputs;   // weights: 1 or 2
  void* out[3];
  const void* in[2];
  long long ld[3];     // row stride of out, in elements
  long long ld_in;     // of in
  long long plane;     // distance of the planes of an operand that is written
  int wide;            // rows of a plain result can move in 16-byte units
  float* partial;      // weights with one plane and more than kRunRows rows: partial_floats() of each CTA
  int* status;
};

struct Shape {
  int planes;   // bf16 parts of an operand: 1 (bf16), 2 or 3 (fp32)
  bool pair;    // two CTAs on one 256 x 256 tile, or one CTA on a 128 x 128 tile
  bool weights; // which of the two kinds of product
  bool b_mn;    // rows: B is stored (k, n) rather than (n, k)
  Epilogue epilogue;
};

// Tile of a shape.
constexpr int tile_rows(bool pair) { return pair ? 256 : 128; }
constexpr int tile_cols(bool pair) { return pair ? 256 : 128; }

// Sums of one CTA's part of a tile, 128 rows by a tile's columns.
constexpr long long partial_floats(bool pair) { return 128ll * tile_cols(pair); }

// Launches with at most `units` output tiles to do; cudaErrorInvalidValue for a combination that is not built.
cudaError_t launch(const Params& p, const Shape& s, long long units, int sms, cudaStream_t stream);
template <int PLANES, bool PAIR>
cudaError_t launch_shape(const Params& p, const Shape& s, long long units, int sms, cudaStream_t stream);

// bf16 parts of a (batch, rows, cols) tensor of any strides, in `planes` consecutive (batch, rows, ld) arrays; columns
// cols .. ld - 1 are zeros. planes == 1 takes bf16 (a copy), else fp32.
struct StageParams {
  const void* src;
  bool src_bf16;
  long long stride_batch, stride_row, stride_col;
  long long batch, rows, cols, ld;
  int planes;
  void* dst;
  const int* offsets;  // batch + 1 row offsets (may be null): matrices whose expert has no rows are left out
};
cudaError_t launch_stage(const StageParams& p, int sms, cudaStream_t stream);

// The SwiGLU derivative of the fp32 forms, whose product writes dh: (rows, ld) fp32 dh, g and u to (planes, rows, ld_out)
// bf16 parts of the gradients of gate and up. ld is a multiple of 4, ld_out the next multiple of 8 of cols.
struct SwiGLUBwdParams {
  const float* dh;
  const float* g;
  const float* u;
  long long ld;
  long long rows, cols, ld_out;
  int planes;
  __nv_bfloat16* dg;
  __nv_bfloat16* du;
};
cudaError_t launch_swiglu_bwd(const SwiGLUBwdParams& p, int sms, cudaStream_t stream);

}  // namespace ragged
}  // namespace abacus
