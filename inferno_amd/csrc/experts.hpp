// Products of rows grouped by expert, weights in bf16 or MXFP4: operands and
// launchers (experts_rows.hip), and the 4-bit format itself (mxfp4.hip).
#pragma once
#include "kernels.hpp"

namespace inferno {

constexpr int kMxBlock = 32;    // columns of one MXFP4 scale

// One matrix, or one per expert, packed: for every tile of 16 rows and step of 64
// bytes of a row (32 columns in bf16, 128 in MXFP4) the 1024 bytes that a wavefront
// takes in one load, lane l 16 bytes of row l % 16, number l / 16. (As rows lie,
// four neighbouring lanes ask for four rows, and the address unit, which joins
// neighbours, takes 16 bytes a cycle instead of 64: with them it was busy for nine
// cycles of ten.) After all of them, for MXFP4, one word per lane for every tile and
// four steps: the scales of its row's 32 columns in the four. Rows behind the last
// and columns behind cols are zeros, of scale 1.
struct ExpertMat {
  size_t experts, rows, cols;
  bool fp4;
  const void* data;
};
struct ExpertLayout {
  size_t tiles, steps, quads;  // of one expert
  size_t scales, bytes;        // byte offset of the scales, and the size
};
inline ExpertLayout expert_layout(const ExpertMat& m) {
  const size_t step = m.fp4 ? 128 : 32;
  ExpertLayout l{};
  l.tiles = (m.rows + 15) / 16;
  l.steps = (m.cols + step - 1) / step;
  l.quads = m.fp4 ? (l.steps + 3) / 4 : 0;
  l.scales = m.experts * l.tiles * l.steps * 1024;
  l.bytes = l.scales + m.experts * l.tiles * l.quads * 256;
  return l;
}

int launch_mxfp4_quantize(hipStream_t s, const void* x, int x_dtype, size_t n, void* codes,
                          void* scales, void* values);
// weights: bf16 [experts, rows, cols], or codes [experts, rows, cols / 2] with
// scales [experts, rows, cols / 32].
int launch_experts_pack(hipStream_t s, const ExpertMat& m, const void* weights, const void* scales,
                        void* packed);

// One product launch. Row c of expert e's range [offsets[e], offsets[e+1]) is
// result row a = sorted[c] (c itself without sorted), of input row a / k.
struct ExpertProduct {
  ExpertMat m[2];
  int mats;                // 2: silu(m0 x) * (m1 x)
  const void* x;           // bf16 [A / k, cols], or codes [A / k, cols / 2]
  const uint8_t* x_scales; // of codes [A / k, cols / 32]; null: bf16
  size_t A, k;             // result rows, result rows per input row
  const uint32_t* offsets; // [experts + 1], or null: one range of all rows
  const uint32_t* sorted;  // [A], or null
  int out_dtype;
  void* out;               // [A, rows]
  void* workspace;         // product_workspace bytes
};

// Which kernel takes a product: tiles (experts_tiles.hip) of `rows` grouped rows by
// 64 * width weight rows, the columns shared by `splits` workgroups; or
// (experts_rows.hip) 16 * width grouped rows, the columns shared by `shares`
// wavefronts.
struct ExpertPlan {
  bool tiles;
  int width, rows, shares;  // width 0: the environment names a form that there is not
  size_t splits;
};
ExpertPlan plan_product(const ExpertProduct& p);
size_t product_workspace(const ExpertProduct& p, const ExpertPlan& plan);
int launch_expert_product(hipStream_t s, const ExpertProduct& p, const ExpertPlan& plan);

}  // namespace inferno
