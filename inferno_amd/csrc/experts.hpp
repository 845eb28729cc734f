// Products of rows grouped by expert, weights in bf16 or MXFP4: operands and
// launchers (experts_rows.hip), and the 4-bit format itself (mxfp4.hip).
#pragma once
#include "kernels.hpp"

namespace inferno {

constexpr int kMxBlock = 32;    // columns of one scale
constexpr int kMxChunk = 128;   // columns of one packed chunk: 64 bytes of codes per row

// One matrix, or one per expert. bf16: [experts][rows][cols] as they are. MXFP4,
// packed: for every tile of 16 rows and chunk of 128 columns the 1024 bytes of
// codes that a wavefront takes in one load, lane l the 32 columns l / 16 of row
// l % 16; after all of them, for every tile and four chunks, one word per lane:
// the scales of its row's 32 columns in the four chunks. Rows behind the last
// and columns behind cols are zeros of scale 1.
struct ExpertMat {
  size_t experts, rows, cols;
  bool fp4;
  const void* data;
};
struct MxLayout {
  size_t tiles, chunks, quads;  // of one expert
  size_t scales, bytes;         // byte offset of the scales, and the size
};
inline MxLayout mx_layout(const ExpertMat& m) {
  MxLayout l{};
  l.tiles = (m.rows + 15) / 16;
  l.chunks = (m.cols + kMxChunk - 1) / kMxChunk;
  l.quads = (l.chunks + 3) / 4;
  l.scales = m.experts * l.tiles * l.chunks * 1024;
  l.bytes = l.scales + m.experts * l.tiles * l.quads * 256;
  return l;
}

int launch_mxfp4_quantize(hipStream_t s, const void* x, int x_dtype, size_t n, void* codes,
                          void* scales, void* values);
int launch_mxfp4_pack(hipStream_t s, const ExpertMat& m, const void* codes, const void* scales,
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
  int width, rows, shares;
  size_t splits;
};
ExpertPlan plan_product(const ExpertProduct& p);
size_t product_workspace(const ExpertProduct& p);
int launch_expert_product(hipStream_t s, const ExpertProduct& p);

}  // namespace inferno
