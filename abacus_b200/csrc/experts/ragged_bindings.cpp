// Torch side of the ragged expert products: checks, tensor maps, launch shapes.
//
// Operands are bf16 with their planes as the leading dimension: (P, rows, cols)
// for sorted rows, (P, E, rows, cols) for the experts' matrices, with 16-byte
// aligned rows (`stage` makes them). P = 1 works on bf16 results, P = 2 and 3
// on fp32 ones.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include "../common/host.h"
#include "bindings.h"
#include "ragged.h"

namespace abacus {
namespace ragged {
namespace {

// Map over `outer` matrices of (rows, cols) bf16 elements; a box is 64 columns by box_rows rows.
CUtensorMap map_of(const torch::Tensor& t, int64_t cols, int64_t rows, int64_t row_stride, int64_t outer,
                   int64_t outer_stride, int box_rows) {
  CUtensorMap m;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_stride * 2), static_cast<cuuint64_t>(outer_stride * 2)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = host::encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, t.data_ptr(), dims, strides, box, step,
                                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(r), " (cols=", cols,
              " rows=", rows, " stride=", row_stride, ")");
  return m;
}

void check_operand(const torch::Tensor& t, int64_t dims, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kBFloat16 && t.dim() == dims, name, " must be a ", dims,
              "-D bf16 CUDA tensor (planes first)");
  TORCH_CHECK(t.size(0) >= 1 && t.size(0) <= 3, name, " must have 1 to 3 planes");
  TORCH_CHECK(t.stride(dims - 1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
              " must have unit inner stride and a 16-byte aligned start");
  for (int64_t d = 0; d < dims - 1; ++d)
    TORCH_CHECK(t.size(d) <= 1 || (t.stride(d) % 8 == 0 && t.stride(d) > 0), name, " rows must be 16-byte aligned");
  TORCH_CHECK(t.size(dims - 2) <= 1 || t.stride(dims - 2) >= t.size(dims - 1), name, " rows must not overlap");
}

// A dimension of length 1 may have any stride; the map wants an aligned one.
int64_t stride_or(const torch::Tensor& t, int64_t d, int64_t otherwise) {
  return t.size(d) > 1 ? t.stride(d) : (otherwise + 7) / 8 * 8;
}

// Sorted rows (P, S, C).
CUtensorMap rows_map(const torch::Tensor& t, int box_rows) {
  const int64_t ld = stride_or(t, 1, t.size(2));
  return map_of(t, t.size(2), t.size(1), ld, t.size(0), stride_or(t, 0, t.size(1) * ld), box_rows);
}

// The experts' matrices (P, E, R, C) as P E matrices.
CUtensorMap experts_map(const torch::Tensor& t, int box_rows) {
  const int64_t ld = stride_or(t, 2, t.size(3));
  const int64_t matrix = t.size(1) > 1 ? t.stride(1) : t.size(0) > 1 ? t.stride(0) : t.size(2) * ld;
  TORCH_CHECK(t.size(0) == 1 || t.size(1) == 1 || t.stride(0) == t.size(1) * t.stride(1),
              "planes of the experts' matrices must follow each other");
  return map_of(t, t.size(3), t.size(2), ld, t.size(0) * t.size(1), (matrix + 7) / 8 * 8, box_rows);
}

void check_result(const torch::Tensor& t, const torch::Tensor& like, int64_t planes, at::IntArrayRef shape, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.is_contiguous() && t.sizes() == shape &&
                  t.scalar_type() == (planes == 1 ? torch::kBFloat16 : torch::kFloat32),
              name, " must be a contiguous ", planes == 1 ? "bf16" : "fp32", " tensor of shape ", shape);
}

// Rows that a SwiGLU form keeps for itself: fp32 (rows, cols) with rows padded to 16 bytes.
void check_kept(const torch::Tensor& t, const torch::Tensor& like, int64_t rows, int64_t cols, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols &&
                  t.scalar_type() == torch::kFloat32 && t.stride(1) == 1 && t.stride(0) % 4 == 0 &&
                  t.stride(0) >= (cols + 3) / 4 * 4 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
              name, " must be fp32 with 16-byte aligned rows");
}

// An operand that a SwiGLU form writes: (planes, rows, cols) with padded rows.
void check_written(const torch::Tensor& t, const torch::Tensor& like, int64_t planes, int64_t rows, int64_t cols, const char* name) {
  check_operand(t, 3, name);
  TORCH_CHECK(t.device() == like.device() && t.size(0) == planes && t.size(1) == rows && t.size(2) == cols &&
                  t.stride(1) % 8 == 0 && t.stride(1) >= (cols + 7) / 8 * 8 &&
                  (rows == 0 || t.stride(0) == rows * t.stride(1)),
              name, " must be (planes, rows, columns) with padded rows");
}

bool wide(std::initializer_list<torch::Tensor> ts, int64_t n) {
  bool ok = true;
  for (const auto& t : ts)
    ok = ok && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && n * t.element_size() % 16 == 0;
  return ok;
}

Params params_of(const torch::Tensor& offsets, const torch::Tensor& like, int64_t sorted_rows) {
  TORCH_CHECK(offsets.is_cuda() && offsets.device() == like.device() && offsets.scalar_type() == torch::kInt32 &&
                  offsets.dim() == 1 && offsets.is_contiguous() && offsets.numel() >= 2,
              "offsets must be a contiguous int32 CUDA tensor of experts + 1 values");
  TORCH_CHECK(offsets.numel() - 1 <= kMaxExperts, "ragged products take at most ", kMaxExperts, " experts, got ",
              offsets.numel() - 1);
  TORCH_CHECK(sorted_rows < (1ll << 31) - 512, "too many rows");
  Params p = {};
  p.offsets = offsets.data_ptr<int>();
  p.experts = static_cast<int>(offsets.numel() - 1);
  p.rows = static_cast<int>(sorted_rows);
  p.segments = p.outputs = 1;
  p.status = host::status_ptr(static_cast<int>(like.get_device()));
  return p;
}

int sms_of(const torch::Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

void run(const Params& p, const Shape& s, const torch::Tensor& like) {
  const long long m_tiles = s.weights ? static_cast<long long>(p.experts) * ((p.m + tile_rows(s.pair) - 1) / tile_rows(s.pair))
                                      : static_cast<long long>(p.rows) / tile_rows(s.pair) + p.experts + 1;
  C10_CUDA_CHECK(launch(p, s, m_tiles * p.n_tiles * p.outputs, sms_of(like), at::cuda::getCurrentCUDAStream()));
  host::note_launch();
}

// Column tiles of an output with n columns, a tile making `cols` of them.
int tiles_of(int64_t n, int cols) { return static_cast<int>((n + cols - 1) / cols); }

// Pairs for experts with rows enough to fill their 256-row tiles, single CTAs for short ones. With uneven loads (the
// largest of 32 experts has four times the average) the two cross near 192 rows on average: y / dx / SwiGLU of 2048 x 1408
// in bf16, on pairs against singles, 128 rows 61 / 58 / 112 against 58 / 59 / 95 us, 192 rows 71 / 65 / 107 against
// 70 / 68 / 131, 256 rows 75 / 70 / 132 against 82 / 85 / 157; in fp32 with 192 rows 351 / 304 / 537 against 296 / 268 / 586,
// with 256 rows 359 / 319 / 696 against 361 / 347 / 714. With equal loads they cross where a second 128-row tile begins
// (y in bf16: 128 rows 58 against 47, 160 rows 58 against 68). The average does not see one long expert among short ones:
// with 8000 of 10,000 rows in one of 64 experts of 768 x 1536 (an average of 157), which run on singles, y takes 68 us and would take
// 60 on pairs, SwiGLU 122 and 146.
bool use_pair_rows(const Params& p) { return p.rows >= 192ll * p.experts; }

void check_rows_and_matrices(const torch::Tensor& a, const torch::Tensor& b, int64_t experts, int64_t k, const char* name) {
  check_operand(a, 3, "the rows");
  check_operand(b, 4, name);
  TORCH_CHECK(a.device() == b.device() && a.size(0) == b.size(0) && b.size(1) == experts && a.size(2) == k, name,
              " do not match the rows");
}

}  // namespace

torch::Tensor stage(torch::Tensor t, int64_t planes, c10::optional<torch::Tensor> offsets) {
  const c10::cuda::CUDAGuard guard(t.device());
  TORCH_CHECK(t.is_cuda() && (t.dim() == 2 || t.dim() == 3), "stage takes 2-D or 3-D CUDA tensors");
  const bool bf16 = t.scalar_type() == torch::kBFloat16;
  TORCH_CHECK(bf16 ? planes == 1 : t.scalar_type() == torch::kFloat32 && (planes == 2 || planes == 3),
              "stage makes 1 plane of bf16 or 2 or 3 of fp32");
  const bool batched = t.dim() == 3;
  const int64_t batch = batched ? t.size(0) : 1, rows = t.size(-2), cols = t.size(-1), ld = (cols + 7) / 8 * 8;
  auto out = torch::empty(batched ? std::vector<int64_t>{planes, batch, rows, ld} : std::vector<int64_t>{planes, rows, ld},
                          t.options().dtype(torch::kBFloat16));
  StageParams p;
  p.src = t.data_ptr();
  p.src_bf16 = bf16;
  p.stride_batch = batched ? t.stride(0) : 0;
  p.stride_row = t.stride(-2);
  p.stride_col = t.stride(-1);
  p.batch = batch;
  p.rows = rows;
  p.cols = cols;
  p.ld = ld;
  p.planes = static_cast<int>(planes);
  p.dst = out.data_ptr();
  p.offsets = nullptr;
  if (offsets) {
    TORCH_CHECK(batched && offsets->is_cuda() && offsets->scalar_type() == torch::kInt32 && offsets->is_contiguous() &&
                    offsets->numel() == batch + 1,
                "offsets of the experts' matrices");
    p.offsets = offsets->data_ptr<int>();
  }
  C10_CUDA_CHECK(launch_stage(p, sms_of(t), at::cuda::getCurrentCUDAStream()));
  host::note_launch();
  return out.narrow(-1, 0, cols);
}

void rows(std::vector<torch::Tensor> a, std::vector<torch::Tensor> b, torch::Tensor offsets, torch::Tensor out,
          bool transposed) {
  TORCH_CHECK(a.size() == b.size() && (a.size() == 1 || a.size() == 2), "one or two segments");
  const c10::cuda::CUDAGuard guard(out.device());
  const int64_t s = out.size(0), n = out.size(1);
  Params p = params_of(offsets, out, s);
  const int64_t k = a[0].size(2), planes = a[0].size(0);
  for (size_t i = 0; i < a.size(); ++i) {
    check_rows_and_matrices(a[i], b[i], p.experts, k, "the experts' matrices");
    TORCH_CHECK(a[i].size(0) == planes && a[i].size(1) == s && b[i].size(transposed ? 3 : 2) == k &&
                    b[i].size(transposed ? 2 : 3) == n,
                "ragged product shapes");
  }
  check_result(out, a[0], planes, {s, n}, "the result");
  if (s == 0 || n == 0) return;
  TORCH_CHECK(k > 0, "empty contraction");
  Shape shape = {static_cast<int>(planes), use_pair_rows(p), false, !transposed, kStore};
  const int local = shape.pair ? tile_cols(true) / 2 : tile_cols(false);
  for (size_t i = 0; i < a.size(); ++i) {
    p.a[i] = rows_map(a[i], 128);
    p.b[i] = experts_map(b[i], transposed ? local : 64);
  }
  p.segments = static_cast<int>(a.size());
  p.k = static_cast<int>(k);
  p.n = static_cast<int>(n);
  p.n_tiles = tiles_of(n, tile_cols(shape.pair));
  p.out[0] = out.data_ptr();
  p.ld[0] = n;
  p.wide = wide({out}, n);
  run(p, shape, out);
}

void swiglu(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor offsets, torch::Tensor g,
            torch::Tensor u, torch::Tensor h) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t s = x.size(1), k = x.size(2), n = g.size(1), planes = x.size(0);
  Params p = params_of(offsets, x, s);
  for (const auto& w : {w_gate, w_up}) {
    check_rows_and_matrices(x, w, p.experts, k, "the experts' matrices");
    TORCH_CHECK(w.size(2) == k && w.size(3) == n, "ragged SwiGLU shapes");
  }
  for (const auto& t : {g, u}) check_kept(t, x, s, n, "gate and up");
  check_written(h, x, planes, s, n, "their product");
  if (s == 0 || n == 0) return;
  TORCH_CHECK(k > 0, "empty contraction");
  Shape shape = {static_cast<int>(planes), use_pair_rows(p), false, true, kSwiGLU};
  p.a[0] = rows_map(x, 128);
  p.b[0] = experts_map(w_gate, 64);
  p.b[1] = experts_map(w_up, 64);
  p.k = static_cast<int>(k);
  p.n = static_cast<int>(n);
  p.n_tiles = tiles_of(n, tile_cols(shape.pair) / 2);
  p.out[0] = g.data_ptr();
  p.out[1] = u.data_ptr();
  p.out[2] = h.data_ptr();
  p.ld[0] = g.stride(0);
  p.ld[1] = u.stride(0);
  p.ld[2] = h.stride(1);
  p.plane = h.stride(0);
  run(p, shape, x);
}

void swiglu_bwd(torch::Tensor dy, torch::Tensor w_down, torch::Tensor offsets, torch::Tensor g, torch::Tensor u,
                torch::Tensor dg, torch::Tensor du) {
  const c10::cuda::CUDAGuard guard(dy.device());
  const int64_t s = dy.size(1), k = dy.size(2), n = g.size(1), planes = dy.size(0);
  Params p = params_of(offsets, dy, s);
  check_rows_and_matrices(dy, w_down, p.experts, k, "the down matrices");
  TORCH_CHECK(w_down.size(2) == n && w_down.size(3) == k, "ragged SwiGLU backward shapes");
  for (const auto& t : {g, u}) check_kept(t, dy, s, n, "gate and up");
  for (const auto& t : {dg, du}) check_written(t, dy, planes, s, n, "the gradients of gate and up");
  TORCH_CHECK(g.stride(0) == u.stride(0), "gate and up must have one row stride");
  if (s == 0 || n == 0) return;
  TORCH_CHECK(k > 0, "empty contraction");
  TORCH_CHECK(du.stride(0) == dg.stride(0) && du.stride(1) == dg.stride(1),
              "the gradients of gate and up must be laid out alike");
  // With one plane the derivative is the product's epilogue. With several the epilogue already holds half a tile of fp32
  // sums a thread, and the product and a pass over dh are faster: 165 + 100 us against 334 us in one kernel (16384 rows of
  // 768 -> 1536, three planes).
  const bool fused = planes == 1;
  Shape shape = {static_cast<int>(planes), use_pair_rows(p), false, false, fused ? kSwiGLUBwd : kStore};
  p.a[0] = rows_map(dy, 128);
  p.b[0] = experts_map(w_down, shape.pair ? tile_cols(true) / 2 : tile_cols(false));
  p.k = static_cast<int>(k);
  p.n = static_cast<int>(n);
  p.n_tiles = tiles_of(n, tile_cols(shape.pair));
  p.ld_in = g.stride(0);
  p.plane = dg.stride(0);
  if (fused) {
    p.in[0] = g.data_ptr();
    p.in[1] = u.data_ptr();
    p.out[0] = dg.data_ptr();
    p.out[1] = du.data_ptr();
    p.ld[0] = p.ld[1] = dg.stride(1);
    run(p, shape, dy);
    return;
  }
  const auto dh = torch::empty({s, g.stride(0)}, g.options());
  p.out[0] = dh.data_ptr();
  p.ld[0] = g.stride(0);
  p.wide = 1;
  run(p, shape, dy);
  const SwiGLUBwdParams q = {dh.data_ptr<float>(), g.data_ptr<float>(), u.data_ptr<float>(), g.stride(0), s, n, dg.stride(1),
                             static_cast<int>(planes), static_cast<__nv_bfloat16*>(dg.data_ptr()),
                             static_cast<__nv_bfloat16*>(du.data_ptr())};
  C10_CUDA_CHECK(launch_swiglu_bwd(q, sms_of(dy), at::cuda::getCurrentCUDAStream()));
  host::note_launch();
}

void weights(torch::Tensor x, std::vector<torch::Tensor> dy, torch::Tensor offsets, std::vector<torch::Tensor> dw) {
  TORCH_CHECK(dy.size() == dw.size() && (dy.size() == 1 || dy.size() == 2), "one or two outputs");
  const c10::cuda::CUDAGuard guard(x.device());
  check_operand(x, 3, "the rows");
  const int64_t s = x.size(1), m = x.size(2), n = dy[0].size(2), planes = x.size(0);
  Params p = params_of(offsets, x, s);
  for (size_t i = 0; i < dy.size(); ++i) {
    check_operand(dy[i], 3, "the rows' gradients");
    TORCH_CHECK(dy[i].device() == x.device() && dy[i].size(0) == planes && dy[i].size(1) == s && dy[i].size(2) == n,
                "ragged weight gradient shapes");
    check_result(dw[i], x, planes, {p.experts, m, n}, "the weight gradients");
  }
  if (m == 0 || n == 0) return;
  if (s == 0) {
    for (auto& t : dw) t.zero_();
    return;
  }
  // A tile is 256 x 256 in a pair, so outputs that fill half of one or less take single CTAs.
  Shape shape = {static_cast<int>(planes), m > 128 && n > 128, true, true, kStore};
  p.a[0] = rows_map(x, 64);
  for (size_t i = 0; i < dy.size(); ++i) {
    p.b[i] = rows_map(dy[i], 64);
    p.out[i] = dw[i].data_ptr();
  }
  p.outputs = static_cast<int>(dy.size());
  p.m = static_cast<int>(m);
  p.n = static_cast<int>(n);
  p.n_tiles = tiles_of(n, tile_cols(shape.pair));
  p.ld[0] = n;
  p.wide = wide({dw[0], dw.back()}, n);
  torch::Tensor partial;
  if (planes == 1 && s > kRunRows) {
    partial = torch::empty({sms_of(x), partial_floats(shape.pair)}, x.options().dtype(torch::kFloat32));
    p.partial = partial.data_ptr<float>();
  }
  run(p, shape, x);
}

}  // namespace ragged
}  // namespace abacus
