// extern "C" entry points of MXFP4 and of the products of rows grouped by
// expert: argument validation and kernel sequencing. No function allocates
// device memory or synchronises.
#include "abi_common.hpp"
#include "experts.hpp"

namespace inferno {
namespace {

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_bytes(const char* what, const char* part, size_t got, size_t want) {
  if (got == want) return INFERNO_OK;
  set_error(std::string(what) + " matrix: its " + part + " must take " + std::to_string(want) +
            " bytes, got " + std::to_string(got));
  return INFERNO_ERR_SIZE;
}

ExpertMat mat(const inferno_experts* w) {
  return ExpertMat{w->experts, w->rows, w->cols, w->format == INFERNO_MXFP4, w->data};
}

int check_shape(const char* what, const inferno_experts* w) {
  INF_CHECK_ARG(w != nullptr, "null expert matrices");
  INF_CHECK_ARG(w->format == INFERNO_BF16 || w->format == INFERNO_MXFP4,
                "the format of expert matrices must be BF16 or MXFP4");
  if (w->experts == 0 || w->rows == 0 || w->cols == 0 || w->rows > (size_t(1) << 24) ||
      w->cols > (size_t(1) << 24) || w->experts > size_t(kMaxExperts) ||
      w->rows * w->cols > (size_t(1) << 33)) {
    set_error(std::string(what) + " matrix: sizes out of range, experts=" +
              std::to_string(w->experts) + ", rows=" + std::to_string(w->rows) + ", cols=" +
              std::to_string(w->cols));
    return INFERNO_ERR_INVALID;
  }
  if (w->format == INFERNO_MXFP4)
    INF_CHECK_ARG(w->cols % kMxBlock == 0, "the columns of an MXFP4 matrix must be a multiple of 32");
  else
    INF_CHECK_ARG(w->cols % 8 == 0, "the columns of a bf16 matrix must be a multiple of 8");
  return INFERNO_OK;
}

int check_mat(const char* what, const inferno_experts* w) {
  int st;
  if ((st = check_shape(what, w))) return st;
  if ((st = check_bytes(what, "packed form", w->data_bytes, expert_layout(mat(w)).bytes))) return st;
  INF_CHECK_ARG(w->data != nullptr, "null pointer in an expert matrix");
  INF_CHECK_ARG(aligned(w->data, 16), "an expert matrix must lie at a multiple of 16 bytes");
  return INFERNO_OK;
}

constexpr size_t kMostRows = size_t(1) << 22;

ExpertProduct product(const inferno_experts* w0, const inferno_experts* w1, const uint8_t* x_scales,
                      size_t rows, size_t k, const uint32_t* offsets) {
  ExpertProduct p{};
  p.m[0] = mat(w0);
  p.mats = w1 ? 2 : 1;
  if (w1) p.m[1] = mat(w1);
  p.x_scales = x_scales;
  p.A = rows;
  p.k = k;
  p.offsets = offsets;
  return p;
}

int check_x_dtype(const inferno_experts* w, int x_dtype) {
  INF_CHECK_ARG(x_dtype == INFERNO_BF16 || (x_dtype == INFERNO_MXFP4 && w->format == INFERNO_MXFP4),
                "x dtype must be BF16, or MXFP4 with weights in MXFP4");
  return INFERNO_OK;
}

int check_kind(const inferno_experts* w, int matrices, int x_dtype) {
  INF_CHECK_ARG(matrices == 1 || matrices == 2, "matrices must be 1 or 2");
  return check_x_dtype(w, x_dtype);
}

int check_rows(size_t x_rows, size_t k) {
  INF_CHECK_ARG(x_rows <= kMostRows && k <= kMostRows && x_rows * k <= kMostRows, "too many rows");
  return INFERNO_OK;
}

int check_form(const ExpertPlan& plan) {
  INF_CHECK_ARG(plan.width > 0, "INFERNO_EXPERTS_FORM names no form of this product");
  return INFERNO_OK;
}

int run_product(void* stream, const inferno_experts* w0, const inferno_experts* w1, const void* x,
                int x_dtype, const uint8_t* x_scales, size_t x_rows, const uint32_t* offsets,
                const uint32_t* sorted, size_t k, int out_dtype, void* out, void* workspace,
                size_t workspace_bytes) {
  INF_CHECK_ARG(out_dtype == INFERNO_F32 || out_dtype == INFERNO_BF16,
                "out dtype must be F32 or BF16");
  if (int st = check_x_dtype(w0, x_dtype)) return st;
  INF_CHECK_ARG(k > 0, "k must be positive");
  INF_CHECK_ARG(k == 1 || sorted, "several result rows per input row need sorted");
  INF_CHECK_ARG(!sorted || offsets, "sorted rows need the experts' offsets");
  INF_CHECK_ARG(offsets || w0->experts == 1, "several experts need offsets");
  if (x_rows == 0) return INFERNO_OK;
  if (int st = check_rows(x_rows, k)) return st;
  INF_CHECK_ARG(x && out, "null pointer");
  INF_CHECK_ARG((x_dtype == INFERNO_MXFP4) == (x_scales != nullptr),
                "x_scales belong to MXFP4 rows, which need them");
  INF_CHECK_ARG(aligned(x, 16) && aligned(out, 16), "x and out must lie at multiples of 16 bytes");
  INF_CHECK_ARG(aligned(offsets, 4) && aligned(sorted, 4),
                "offsets and sorted must lie at multiples of 4 bytes");
  ExpertProduct p = product(w0, w1, x_scales, x_rows * k, k, offsets);
  const ExpertPlan plan = plan_product(p);
  if (int st = check_form(plan)) return st;
  if (int st = need_ws(workspace, workspace_bytes, product_workspace(p, plan))) return st;
  INF_CHECK_ARG(aligned(workspace, 16), "the workspace must lie at a multiple of 16 bytes");
  if (int st_ = require_device()) return st_;
  p.x = x;
  p.sorted = sorted;
  p.out_dtype = out_dtype;
  p.out = out;
  p.workspace = workspace;
  return launch_expert_product(as_stream(stream), p, plan);
}

}  // namespace
}  // namespace inferno

using namespace inferno;

extern "C" {

int inferno_mxfp4_quantize(void* stream, const void* x, int x_dtype, size_t rows, size_t cols,
                           void* codes, uint8_t* scales, void* values) {
  clear_error();
  INF_CHECK_ARG(x_dtype == INFERNO_F32 || x_dtype == INFERNO_BF16, "x dtype must be F32 or BF16");
  INF_CHECK_ARG(cols > 0 && cols % kMxBlock == 0, "the columns must be a multiple of 32");
  if (rows == 0) return INFERNO_OK;
  INF_CHECK_ARG(cols < (size_t(1) << 32) && rows < (size_t(1) << 32) &&
                    rows * cols <= (size_t(1) << 34),
                "too many values");
  INF_CHECK_ARG(x && codes && scales, "null pointer");
  INF_CHECK_ARG(aligned(x, 16) && aligned(codes, 16) && aligned(values, 16),
                "x, codes and values must lie at multiples of 16 bytes");
  if (int st_ = require_device()) return st_;
  return launch_mxfp4_quantize(as_stream(stream), x, x_dtype, rows * cols, codes, scales, values);
}

size_t inferno_experts_packed_bytes(const inferno_experts* w) {
  clear_error();
  return check_shape("given", w) ? 0 : expert_layout(mat(w)).bytes;
}

int inferno_experts_pack(void* stream, const inferno_experts* w, const void* weights,
                         size_t weights_bytes, const uint8_t* scales, size_t scales_bytes,
                         void* packed) {
  clear_error();
  int st;
  if ((st = check_shape("given", w))) return st;
  const bool fp4 = w->format == INFERNO_MXFP4;
  const size_t values = w->experts * w->rows * w->cols;
  if ((st = check_bytes("given", fp4 ? "codes" : "weights", weights_bytes,
                        fp4 ? values / 2 : values * 2)))
    return st;
  if ((st = check_bytes("given", "scales", scales_bytes, fp4 ? values / kMxBlock : 0))) return st;
  if ((st = check_bytes("given", "packed form", w->data_bytes, expert_layout(mat(w)).bytes)))
    return st;
  INF_CHECK_ARG(weights && packed && fp4 == (scales != nullptr),
                "null pointer, or scales of matrices in bf16");
  INF_CHECK_ARG(aligned(weights, 16) && aligned(packed, 16),
                "the weights and their packed form must lie at multiples of 16 bytes");
  if (int st_ = require_device()) return st_;
  return launch_experts_pack(as_stream(stream), mat(w), weights, scales, packed);
}

size_t inferno_grouped_workspace_bytes(const inferno_experts* w, int matrices, int x_dtype,
                                       size_t x_rows, size_t k, int grouped) {
  clear_error();
  if (check_shape("given", w) || check_kind(w, matrices, x_dtype)) return 0;
  if (check_rows(x_rows, k) || x_rows * k == 0) return 0;
  static const uint8_t scale = 127;  // (only whether there are scales and offsets counts)
  static const uint32_t offset = 0;
  const ExpertProduct p = product(w, matrices == 2 ? w : nullptr,
                                  x_dtype == INFERNO_MXFP4 ? &scale : nullptr, x_rows * k, k,
                                  grouped ? &offset : nullptr);
  const ExpertPlan plan = plan_product(p);
  return check_form(plan) ? 0 : product_workspace(p, plan);
}

int inferno_grouped_matmul(void* stream, const inferno_experts* w, const void* x, int x_dtype,
                           const uint8_t* x_scales, size_t x_rows, const uint32_t* offsets,
                           const uint32_t* sorted, size_t k, int out_dtype, void* out, void* workspace,
                           size_t workspace_bytes) {
  clear_error();
  if (int st = check_mat("weight", w)) return st;
  return run_product(stream, w, nullptr, x, x_dtype, x_scales, x_rows, offsets, sorted, k,
                     out_dtype, out, workspace, workspace_bytes);
}

int inferno_grouped_gate_up_swiglu(void* stream, const inferno_experts* gate,
                                   const inferno_experts* up, const void* x, int x_dtype,
                                   const uint8_t* x_scales, size_t x_rows, const uint32_t* offsets,
                                   const uint32_t* sorted, size_t k, int out_dtype, void* out, void* workspace,
                           size_t workspace_bytes) {
  clear_error();
  int st;
  if ((st = check_mat("gate", gate))) return st;
  if ((st = check_mat("up", up))) return st;
  INF_CHECK_ARG(gate->experts == up->experts && gate->rows == up->rows && gate->cols == up->cols &&
                    gate->format == up->format,
                "the gate and up matrices must have the same sizes and format");
  return run_product(stream, gate, up, x, x_dtype, x_scales, x_rows, offsets, sorted, k, out_dtype,
                     out, workspace, workspace_bytes);
}

}  // extern "C"
