// Products with 4-bit weights: operands and launchers (w4.hip).
#pragma once
#include "kernels.hpp"

namespace inferno {

constexpr int kW4Chunk = 128;  // columns of one step: 64 bytes of codes per row

// One matrix, or one per expert, as the caller stores it.
struct W4Mat {
  const uint8_t* codes;  // [rows, K/2], the even column in the low nibble
  const void* scales;    // [rows, K/group] fp32 or bf16
  const uint8_t* zeros;  // [rows, K/group], or null: 8
};

// Activations as int8 digits, the operands of the integer matrix cores.
// A value of a 128-column chunk is (65536 d0 + 256 d1 + d2) xs (3 planes; d in
// [-128, 127]), or d0 xs (1 plane, int8 activations).
//   planes [rows][chunks][planes][128]: the digits of one chunk in the order
//     in which the lanes of the weights' tile hold its columns;
//   xs [rows][chunks].
struct W4Acts {
  int8_t* planes;
  float* xs;
  int P;      // planes: 3 or 1
  bool fine;  // groups of 32 or 64 columns
};

inline size_t w4_chunks(size_t K) { return (K + kW4Chunk - 1) / kW4Chunk; }

// Writes the activations' digits. x: fp32, bf16, or int8 with x_scales
// [R, K / x_group] (x_group 0: one per row).
int launch_w4_stage(hipStream_t s, const void* x, int x_dtype, const float* x_scales,
                    size_t x_group, size_t R, size_t K, const W4Acts& a);

// One product launch. Dense: every token; routed: the assignments of each
// expert (dispatch outputs), activation rows by token or by assignment.
struct W4Product {
  W4Mat m[2];
  int mats;         // 2: silu(m0 x) * (m1 x) [* weight]
  int scale_dtype;
  size_t K, N, group;
  W4Acts x;
  size_t T;         // tokens
  // routed (offsets not null): assignments sorted by expert
  const uint32_t* offsets;
  const uint32_t* sorted;
  const uint32_t* active;
  size_t k, E;
  bool x_by_assignment;
  const float* route_w;  // [T*k], multiplied into the result, or null
  const float* res_a;    // added (dense), or null
  const float* res_b;
  float* out;            // [T, N], or [T*k, N]
};
int launch_w4_product(hipStream_t s, const W4Product& p);

// out[t] = sum over the ranks of token t, in rank order, of y[t*k + r]; ids of
// no expert count nothing.
int launch_w4_combine(hipStream_t s, const float* y, const uint32_t* ids, size_t T, size_t H,
                      size_t k, size_t E, float* out);

}  // namespace inferno
