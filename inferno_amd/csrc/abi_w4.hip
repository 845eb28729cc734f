// extern "C" entry points of the products with 4-bit weights: argument
// validation, workspace carving and kernel sequencing. No function allocates
// device memory or synchronises.
#include <cmath>

#include "abi_common.hpp"
#include "w4.hpp"

namespace inferno {
namespace {

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_bytes(const char* what, const char* part, size_t got, size_t want) {
  if (got == want) return INFERNO_OK;
  set_error(std::string("4-bit ") + what + " matrix: its " + part + " must take " +
            std::to_string(want) + " bytes, got " + std::to_string(got));
  return INFERNO_ERR_SIZE;
}

W4Mat mat(const inferno_w4* w) {
  return W4Mat{w->experts, w->rows,           w->cols,  w->group,
               w->scale_dtype, w->has_zeros != 0, w->packed};
}

int check_shape(const char* what, const inferno_w4* w) {
  INF_CHECK_ARG(w != nullptr, "null 4-bit matrix");
  const size_t most = size_t(1) << 31;
  if (w->experts == 0 || w->rows == 0 || w->cols == 0 || w->cols >= most ||
      w->rows > (size_t(1) << 25) ||  // a launch has less than 2^32 threads
      w->experts > size_t(kMaxExperts) || w->rows * w->cols >= 4 * most) {
    set_error(std::string("4-bit ") + what + " matrix: sizes out of range, experts=" +
              std::to_string(w->experts) + ", rows=" + std::to_string(w->rows) + ", cols=" +
              std::to_string(w->cols));
    return INFERNO_ERR_INVALID;
  }
  const size_t g = w->group;
  INF_CHECK_ARG(g == 32 || g == 64 || (g > 0 && g % kW4Chunk == 0),
                "the group of a 4-bit matrix must be 32, 64 or a multiple of 128");
  INF_CHECK_ARG(w->cols % 32 == 0 && w->cols % g == 0,
                "the columns of a 4-bit matrix must be a multiple of 32 and of its group");
  INF_CHECK_ARG(w->scale_dtype == INFERNO_F32 || w->scale_dtype == INFERNO_BF16,
                "scales must be F32 or BF16");
  return INFERNO_OK;
}

int check_w4(const char* what, const inferno_w4* w) {
  int st;
  if ((st = check_shape(what, w))) return st;
  if ((st = check_bytes(what, "packed form", w->packed_bytes, w4_layout(mat(w)).bytes))) return st;
  INF_CHECK_ARG(w->packed != nullptr, "null pointer in a 4-bit matrix");
  INF_CHECK_ARG(aligned(w->packed, 16), "a packed matrix must lie at a multiple of 16 bytes");
  return INFERNO_OK;
}

// gate and up go through one kernel.
int check_pair(const inferno_w4* gate, const inferno_w4* up) {
  int st;
  if ((st = check_w4("gate", gate))) return st;
  if ((st = check_w4("up", up))) return st;
  INF_CHECK_ARG(gate->experts == up->experts && gate->rows == up->rows && gate->cols == up->cols,
                "the gate and up matrices must have the same sizes");
  INF_CHECK_ARG(gate->group == up->group && gate->scale_dtype == up->scale_dtype &&
                    (gate->has_zeros != 0) == (up->has_zeros != 0),
                "the gate and up matrices must have the same group, scale type and zero points");
  return INFERNO_OK;
}

int check_x(const void* x, int x_dtype, const float* x_scales, size_t x_group, size_t cols) {
  INF_CHECK_ARG(x_dtype == INFERNO_F32 || x_dtype == INFERNO_BF16 || x_dtype == INFERNO_I8,
                "x dtype must be F32, BF16 or I8");
  INF_CHECK_ARG(x != nullptr, "null pointer");
  INF_CHECK_ARG(aligned(x, 16), "x must lie at a multiple of 16 bytes");
  if (x_dtype != INFERNO_I8) return INFERNO_OK;
  INF_CHECK_ARG(x_scales != nullptr, "8-bit activations need their scales");
  INF_CHECK_ARG(x_group == 0 || x_group == cols || (x_group % kW4Chunk == 0 && cols % x_group == 0),
                "x_group must be 0 (the row) or a multiple of 128 that divides the columns");
  return INFERNO_OK;
}

// Launches count their threads in 32 bits.
int check_tokens(size_t rows, size_t cols) {
  INF_CHECK_ARG(rows < (size_t(1) << 31) && rows * cols < (size_t(1) << 36), "too many tokens");
  return INFERNO_OK;
}

// Room for two planes of fp16, which any call fits.
W4Acts carve_acts(Carver& c, size_t rows, size_t cols) {
  const size_t n = rows * w4_chunks(cols);
  W4Acts a{};
  a.planes = c.take<int8_t>(n * 4 * kW4Chunk);
  a.xs = c.take<float>(rows * w4_xs_stride(cols));
  return a;
}

// The same region for the matrices and activations of one call.
W4Acts acts_for(W4Acts a, const inferno_w4* w, int x_dtype, size_t T, size_t k) {
  a.P = x_dtype == INFERNO_I8 ? 1 : 3;
  a.fine = mat(w).fine();
  // Two planes of fp16 are more to move than three of digits, but need no joins,
  // of which fine groups have four in a chunk. fp32 tokens, two planes of fp16 and
  // three digits: 128 experts' down, 512 tokens 335 and 250 us (groups of 128); 64
  // experts, 256 tokens 178 and 222 us (groups of 32, whole pass).
  if (w4_by_tiles(T, k, w->experts)) {
    if (x_dtype == INFERNO_BF16) a.halves = 1;
    else if (x_dtype == INFERNO_F32 && a.fine) a.halves = 2;
  }
  return a;
}

W4Product product(const inferno_w4* w, const W4Acts& x, size_t T, float* out) {
  W4Product p{};
  p.m[0] = mat(w);
  p.mats = 1;
  p.x = x;
  p.T = T;
  p.out = out;
  return p;
}

W4Token tokens(const inferno_w4* w, const void* x, int x_dtype, size_t T, float* out) {
  W4Token q{};
  q.m[0] = mat(w);
  q.mats = 1;
  q.x = x;
  q.x_dtype = x_dtype;
  q.T = T;
  q.slots = q.segments = 1;
  q.out = out;
  return q;
}

struct W4MoeScratch {
  uint32_t* offsets;
  uint32_t* sorted;
  uint32_t* active;
  W4Acts x, h_acts;
  float* h;
  float* y;
};

W4MoeScratch carve_w4_moe(Carver& c, size_t T, size_t k, size_t E, size_t H, size_t I) {
  W4MoeScratch m;
  m.offsets = c.take<uint32_t>(E + 1);
  m.sorted = c.take<uint32_t>(T * k);
  m.active = c.take<uint32_t>(E + 1);
  m.x = carve_acts(c, T, H);
  m.h = c.take<float>(T * k * I);
  m.h_acts = carve_acts(c, T * k, I);
  m.y = c.take<float>(T * k * H);
  return m;
}

int check_ws(void* workspace, size_t have, size_t need) {
  if (int st = need_ws(workspace, have, need)) return st;
  INF_CHECK_ARG(aligned(workspace, 16), "the workspace must lie at a multiple of 16 bytes");
  return INFERNO_OK;
}

}  // namespace
}  // namespace inferno

using namespace inferno;

extern "C" {

size_t inferno_w4_packed_bytes(const inferno_w4* w) {
  clear_error();
  return check_shape("given", w) ? 0 : w4_layout(mat(w)).bytes;
}

int inferno_w4_pack(void* stream, const inferno_w4* w, const void* codes, size_t codes_bytes,
                    const void* scales, size_t scales_bytes, const void* zeros, size_t zeros_bytes,
                    void* packed) {
  clear_error();
  int st;
  if ((st = check_shape("given", w))) return st;
  const size_t rows = w->experts * w->rows, groups = rows * (w->cols / w->group);
  const size_t each = w->scale_dtype == INFERNO_BF16 ? 2 : 4;
  if ((st = check_bytes("given", "codes", codes_bytes, rows * (w->cols / 2)))) return st;
  if ((st = check_bytes("given", "scales", scales_bytes, groups * each))) return st;
  if (w->has_zeros && (st = check_bytes("given", "zero points", zeros_bytes, groups))) return st;
  if ((st = check_bytes("given", "packed form", w->packed_bytes, w4_layout(mat(w)).bytes))) return st;
  INF_CHECK_ARG(codes && scales && packed && (zeros || !w->has_zeros), "null pointer");
  INF_CHECK_ARG(aligned(codes, 4) && aligned(scales, each),
                "codes must lie at a multiple of 4 bytes, scales at one of their size");
  INF_CHECK_ARG(aligned(packed, 16), "a packed matrix must lie at a multiple of 16 bytes");
  INF_CHECK_ARG(rows * w->cols < (size_t(1) << 42), "too many codes");
  if (int st_ = require_device()) return st_;
  return launch_w4_pack(as_stream(stream), mat(w), codes, scales, w->has_zeros ? zeros : nullptr,
                        packed);
}

size_t inferno_w4_workspace_bytes(size_t T, size_t cols) {
  Carver c{nullptr};
  carve_acts(c, T, cols);
  return c.used;
}

int inferno_w4_matvec_add2(void* stream, const inferno_w4* w, const void* x, int x_dtype,
                           const float* x_scales, size_t x_group, const float* residual_a,
                           const float* residual_b, size_t T, float* out, void* workspace,
                           size_t workspace_bytes) {
  clear_error();
  int st;
  if ((st = check_w4("weight", w))) return st;
  INF_CHECK_ARG(w->experts == 1, "a plain product takes one matrix");
  if (T == 0) return INFERNO_OK;
  if ((st = check_x(x, x_dtype, x_scales, x_group, w->cols))) return st;
  if ((st = check_tokens(T, std::max(w->cols, w->rows)))) return st;
  INF_CHECK_ARG(out, "null pointer");
  if ((st = check_ws(workspace, workspace_bytes, inferno_w4_workspace_bytes(T, w->cols)))) return st;
  if (int st_ = require_device()) return st_;
  hipStream_t s = as_stream(stream);
  if (x_dtype != INFERNO_I8) {
    W4Token q = tokens(w, x, x_dtype, T, out);
    q.res_a = residual_a;
    q.res_b = residual_b;
    if (w4_token_fits(q)) return launch_w4_token(s, q);
  }
  Carver c{static_cast<char*>(workspace)};
  const W4Acts a = acts_for(carve_acts(c, T, w->cols), w, x_dtype, T, 0);
  if ((st = launch_w4_stage(s, x, x_dtype, x_scales, x_group, T, w->cols, a))) return st;
  W4Product p = product(w, a, T, out);
  p.res_a = residual_a;
  p.res_b = residual_b;
  return launch_w4_product(s, p);
}

int inferno_w4_gate_up_swiglu(void* stream, const inferno_w4* gate, const inferno_w4* up,
                              const void* x, int x_dtype, const float* x_scales, size_t x_group,
                              size_t T, float* out, void* workspace, size_t workspace_bytes) {
  clear_error();
  int st;
  if ((st = check_pair(gate, up))) return st;
  INF_CHECK_ARG(gate->experts == 1, "a plain product takes one matrix");
  if (T == 0) return INFERNO_OK;
  if ((st = check_x(x, x_dtype, x_scales, x_group, gate->cols))) return st;
  if ((st = check_tokens(T, std::max(gate->cols, gate->rows)))) return st;
  INF_CHECK_ARG(out, "null pointer");
  if ((st = check_ws(workspace, workspace_bytes, inferno_w4_workspace_bytes(T, gate->cols))))
    return st;
  if (int st_ = require_device()) return st_;
  hipStream_t s = as_stream(stream);
  if (x_dtype != INFERNO_I8) {
    W4Token q = tokens(gate, x, x_dtype, T, out);
    q.m[1] = mat(up);
    q.mats = 2;
    if (w4_token_fits(q)) return launch_w4_token(s, q);
  }
  Carver c{static_cast<char*>(workspace)};
  const W4Acts a = acts_for(carve_acts(c, T, gate->cols), gate, x_dtype, T, 0);
  if ((st = launch_w4_stage(s, x, x_dtype, x_scales, x_group, T, gate->cols, a))) return st;
  W4Product p = product(gate, a, T, out);
  p.m[1] = mat(up);
  p.mats = 2;
  return launch_w4_product(s, p);
}

size_t inferno_w4_moe_workspace_bytes(size_t T, size_t k, size_t E, size_t H, size_t I) {
  Carver c{nullptr};
  carve_w4_moe(c, T, k, E, H, I);
  return c.used;
}

int inferno_w4_moe(void* stream, const inferno_w4* gate, const inferno_w4* up,
                   const inferno_w4* down, const void* x, int x_dtype, const float* x_scales,
                   size_t x_group, const uint32_t* expert_ids, const float* expert_weights,
                   size_t T, size_t k, float* out, void* workspace, size_t workspace_bytes) {
  clear_error();
  int st;
  if ((st = check_pair(gate, up))) return st;
  if ((st = check_w4("down", down))) return st;
  const size_t E = gate->experts, H = gate->cols, I = gate->rows;
  INF_CHECK_ARG(down->experts == E && down->rows == H && down->cols == I,
                "the down matrices must have the gate's sizes, rows and columns changed over");
  INF_CHECK_ARG(k > 0 && k <= size_t(kMaxTopK), "top_k must be in 1..=16");
  if (T == 0) return INFERNO_OK;
  if ((st = check_x(x, x_dtype, x_scales, x_group, H))) return st;
  INF_CHECK_ARG(T < (size_t(1) << 27), "too many tokens");
  if ((st = check_tokens(T * k, std::max(H, I)))) return st;
  INF_CHECK_ARG(expert_ids && expert_weights && out, "null pointer");
  if ((st = check_ws(workspace, workspace_bytes, inferno_w4_moe_workspace_bytes(T, k, E, H, I))))
    return st;
  if (int st_ = require_device()) return st_;
  hipStream_t s = as_stream(stream);
  Carver c{static_cast<char*>(workspace)};
  const W4MoeScratch m = carve_w4_moe(c, T, k, E, H, I);
  if (T == 1 && x_dtype != INFERNO_I8) {
    // gate and up of every rank, then the sum over the ranks (h rows of ids of
    // no expert are not written, and count nothing)
    W4Token g = tokens(gate, x, x_dtype, 1, m.h), d = tokens(down, m.h, INFERNO_F32, 1, out);
    g.m[1] = mat(up);
    g.mats = 2;
    g.slots = k;
    d.segments = k;
    d.sum = true;
    g.ids = d.ids = expert_ids;
    g.route_w = expert_weights;
    if (w4_token_fits(g) && w4_token_fits(d)) {
      if ((st = launch_w4_token(s, g))) return st;
      return launch_w4_token(s, d);
    }
  }
  if ((st = launch_dispatch(s, expert_ids, T, k, E, m.offsets, m.sorted, m.active))) return st;
  const W4Acts xa = acts_for(m.x, gate, x_dtype, T, k),
               ha = acts_for(m.h_acts, down, INFERNO_F32, T, k);
  if ((st = launch_w4_stage(s, x, x_dtype, x_scales, x_group, T, H, xa))) return st;
  W4Product g = product(gate, xa, T, m.h);
  g.m[1] = mat(up);
  g.mats = 2;
  g.offsets = m.offsets;
  g.sorted = m.sorted;
  g.active = m.active;
  g.k = k;
  g.route_w = expert_weights;
  if ((st = launch_w4_product(s, g))) return st;
  if ((st = launch_w4_stage(s, m.h, INFERNO_F32, nullptr, 0, T * k, I, ha))) return st;
  W4Product d = product(down, ha, T, m.y);
  d.offsets = m.offsets;
  d.sorted = m.sorted;
  d.active = m.active;
  d.k = k;
  d.x_by_assignment = true;
  if ((st = launch_w4_product(s, d))) return st;
  return launch_w4_combine(s, m.y, expert_ids, T, H, k, E, out);
}

}  // extern "C"
