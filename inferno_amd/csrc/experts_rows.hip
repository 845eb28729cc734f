// Products of rows grouped by expert: 16 weight rows by 16 grouped rows, the
// operands straight from memory in the order of the matrix instructions.
//
// The weights are the first operand (lane l: row l % 16, quarter l / 16 of the
// columns of a step), the grouped rows the second, so that a lane's four sums
// are four neighbouring values of one result row. A workgroup's wavefronts share
// the columns, 128 at a time, and add their sums in order through LDS.
#include "experts_dev.hpp"

namespace inferno {
namespace {

using namespace experts;

constexpr int kWaves = 4;

template <bool WFP4, bool XFP4, int MATS>
__global__ void __launch_bounds__(kWaves* kWave) experts_rows_kernel(Product p) {
  __shared__ floatx4 part[kWaves][MATS][kWave];
  uint32_t e, c0, c1;
  const uint32_t slot = blockIdx.x / p.tiles;
  if (slot >= find_tile<16>(p, slot, e, c0, c1)) return;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile = blockIdx.x - slot * p.tiles;  // of weight rows
  const uint32_t c = c0 + n;
  const uint32_t a = c < c1 ? result_row(p, c) : p.A;
  const bool on = a < p.A;
  const size_t xrow = on ? a / p.k : 0;
  const uint32_t wrow = min(tile * 16 + n, p.N - 1);
  floatx4 acc[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) acc[m] = floatx4{0.f, 0.f, 0.f, 0.f};
  const uint4 none = make_uint4(0, 0, 0, 0);
  for (uint32_t ch = wave; ch < p.chunks; ch += kWaves) {
    if constexpr (WFP4) {
      const uint32_t col = ch * kMxChunk + 32 * g;
      const bool in = on && col < p.K;  // whole blocks of 32
      const size_t wt = (size_t(e) * p.tiles + tile);
      uint4 w[MATS];
      uint32_t ws[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        w[m] = reinterpret_cast<const uint4*>(p.w[m])[(wt * p.chunks + ch) * 64 + lane];
        ws[m] = p.ws[m][(wt * p.quads + ch / 4) * 64 + lane] >> (8 * (ch % 4)) & 255u;
      }
      if constexpr (XFP4) {
        const size_t at = xrow * (p.K / 32) + col / 32;
        const uint4 xv = in ? reinterpret_cast<const uint4*>(p.x)[at] : none;
        const uint32_t xs = in ? p.xs[at] : 127u;
#pragma unroll
        for (int m = 0; m < MATS; ++m) acc[m] = mfma_fp4(w[m], xv, acc[m], ws[m], xs);
      } else {
        const uint4* at = reinterpret_cast<const uint4*>(p.x + (xrow * p.K + (in ? col : 0)) * 2);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 xv = in ? at[j] : none;
#pragma unroll
          for (int m = 0; m < MATS; ++m) {
            const uint32_t cw = j == 0 ? w[m].x : j == 1 ? w[m].y : j == 2 ? w[m].z : w[m].w;
            acc[m] = mfma_bf16(widen(cw, scale_of(ws[m])), __builtin_bit_cast(bf16x8, xv), acc[m]);
          }
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t col = ch * kMxChunk + 32 * j + 8 * g;
        const bool in = col < p.K;
        const uint4 xv =
            on && in ? *reinterpret_cast<const uint4*>(p.x + (xrow * p.K + col) * 2) : none;
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const size_t at = ((size_t(e) * p.N + wrow) * p.K + col) * 2;
          const uint4 w = in ? *reinterpret_cast<const uint4*>(p.w[m] + at) : none;
          acc[m] = mfma_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, xv), acc[m]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MATS; ++m) part[wave][m][lane] = acc[m];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int m = 0; m < MATS; ++m)
    for (int v = 1; v < kWaves; ++v) acc[m] += part[v][m][lane];
  if (!on) return;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = MATS == 2 ? silu_mul(acc[0][i], acc[MATS - 1][i]) : acc[0][i];
  store4(p, a, tile * 16 + 4 * g, y);
}

}  // namespace

int launch_expert_product(hipStream_t s, const ExpertProduct& q) {
  Product p{};
  const ExpertMat& m = q.m[0];
  const MxLayout l = mx_layout(m);
  for (int i = 0; i < q.mats; ++i) {
    p.w[i] = static_cast<const uint8_t*>(q.m[i].data);
    p.ws[i] = reinterpret_cast<const uint32_t*>(p.w[i] + l.scales);
  }
  p.x = static_cast<const uint8_t*>(q.x);
  p.xs = q.x_scales;
  p.offsets = q.offsets;
  p.sorted = q.sorted;
  p.E = uint32_t(m.experts);
  p.A = uint32_t(q.A);
  p.k = uint32_t(q.k);
  p.N = uint32_t(m.rows);
  p.K = uint32_t(m.cols);
  p.tiles = uint32_t(l.tiles);
  p.chunks = uint32_t(l.chunks);
  p.quads = uint32_t(l.quads);
  p.out = q.out;
  p.out_f32 = q.out_dtype == INFERNO_F32;
  const size_t most = q.offsets ? q.A / 16 + std::min(m.experts, q.A) : (q.A + 15) / 16;
  if (most * l.tiles * (kWaves * kWave) >= size_t(1) << 32) {
    set_error("too many rows for one launch");
    return INFERNO_ERR_INVALID;
  }
  const unsigned grid = unsigned(l.tiles * most);
  auto go = [&](auto wf, auto xf) {
    constexpr bool W = decltype(wf)::value, X = decltype(xf)::value;
    if (q.mats == 2) experts_rows_kernel<W, X, 2><<<grid, kWaves * kWave, 0, s>>>(p);
    else experts_rows_kernel<W, X, 1><<<grid, kWaves * kWave, 0, s>>>(p);
  };
  if (!m.fp4) go(std::false_type{}, std::false_type{});
  else if (q.x_scales) go(std::true_type{}, std::true_type{});
  else go(std::true_type{}, std::false_type{});
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
