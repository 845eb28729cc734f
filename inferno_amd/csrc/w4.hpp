// Products with 4-bit weights: operands and launchers (w4.hip).
#pragma once
#include "kernels.hpp"

namespace inferno {

constexpr int kW4Chunk = 128;  // columns of one step: 64 bytes of codes per row

// One matrix, or one per expert, packed: for every tile of 16 rows and chunk of
// 128 columns the 1024 bytes of codes that a wavefront's lanes take in one load
// (16 each), then for all of them the scales of the 16 rows (one each, or four
// for groups of 32 and 64: one per 32 columns), then likewise the zero points.
// Rows behind the last and columns behind cols count nothing.
struct W4Mat {
  size_t experts, rows, cols, group;
  int scale_dtype;
  bool zeros;
  const void* packed;
  bool fine() const { return group < size_t(kW4Chunk); }
};
struct W4Layout {
  size_t scales, zeros, bytes;  // byte offsets, and the size
};
W4Layout w4_layout(const W4Mat& m);
inline size_t w4_chunks(size_t K) { return (K + kW4Chunk - 1) / kW4Chunk; }

// Packs codes [rows, cols/2] (the even column in the low nibble), scales [rows,
// cols/group] and zeros [rows, cols/group] or null (8).
int launch_w4_pack(hipStream_t s, const W4Mat& m, const void* codes, const void* scales,
                   const void* zeros, void* packed);

// Activations as operands of the matrix cores: int8 digits, or fp16 (halves).
// A value of a 128-column chunk is (65536 d0 + 256 d1 + d2) xs (3 planes; d in
// [-128, 127]), or d0 xs (1 plane, int8 activations); with halves the sum of its
// planes' fp16 values times xs.
//   planes [rows][chunks][planes][128 or 256 bytes]: one chunk in the order
//     in which the lanes of the weights' tile hold its columns;
//   xs [rows][chunks, to a multiple of 2 with 0].
inline size_t w4_xs_stride(size_t K) { return (w4_chunks(K) + 1) / 2 * 2; }
struct W4Acts {
  int8_t* planes;
  float* xs;
  int P;       // planes of digits: 3 or 1
  int halves;  // or planes of fp16 (two for fp32, one for bf16), 256 bytes of a chunk each
  bool fine;   // groups of 32 or 64 columns
};
// Whether products of T tokens (of k experts each; 0: one matrix) take the
// kernel that has fp16 for activations other than int8.
bool w4_by_tiles(size_t T, size_t k, size_t experts);

// Writes the activations' digits. x: fp32, bf16, or int8 with x_scales
// [R, K / x_group] (x_group 0: one per row).
int launch_w4_stage(hipStream_t s, const void* x, int x_dtype, const float* x_scales,
                    size_t x_group, size_t R, size_t K, const W4Acts& a);

// One product launch. Dense: every token; routed: the assignments of each
// expert (dispatch outputs), activation rows by token or by assignment.
struct W4Product {
  W4Mat m[2];
  int mats;         // 2: silu(m0 x) * (m1 x) [* weight], both of one format
  W4Acts x;
  size_t T;         // tokens
  // routed (offsets not null): assignments sorted by expert
  const uint32_t* offsets;
  const uint32_t* sorted;
  const uint32_t* active;
  size_t k;
  bool x_by_assignment;
  const float* route_w;  // [T*k], multiplied into the result, or null
  const float* res_a;    // added (dense), or null
  const float* res_b;
  float* out;            // [T, N], or [T*k, N]
};
int launch_w4_product(hipStream_t s, const W4Product& p);

// One to four fp32 or bf16 tokens of a matrix, or one token of its experts, in
// one launch, as far as the tokens' digits fit a workgroup's LDS (4 tokens of 4096
// columns, 1 of 17536). ids: expert ids[y] of each slot y, result row y (none for an
// id of no expert), or with `sum` the sum over the segments r of row r of x times
// expert ids[r].
struct W4Token {
  W4Mat m[2];
  int mats;
  const void* x;
  int x_dtype;
  size_t T, slots, segments;
  bool sum;
  const uint32_t* ids;   // or null
  const float* route_w;  // by slot, or null
  const float* res_a;
  const float* res_b;
  float* out;
};
bool w4_token_fits(const W4Token& q);
int launch_w4_token(hipStream_t s, const W4Token& q);

// out[t] = sum over the ranks of token t, in rank order, of y[t*k + r]; ids of
// no expert count nothing.
int launch_w4_combine(hipStream_t s, const float* y, const uint32_t* ids, size_t T, size_t H,
                      size_t k, size_t E, float* out);

}  // namespace inferno
