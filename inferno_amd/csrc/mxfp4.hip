// MXFP4: rows to 4-bit floating point with one power-of-two scale per 32
// columns, and the packing of experts' weights, in bf16 too.
//
// A block's scale is 2^(floor(log2 m) - 2), m its largest magnitude: 4 <= m /
// scale < 8, and the largest code stands for 6, so that quotients above 6
// saturate. Codes are the nearest ones, halfway values to the code whose last
// bit is 0 (v_cvt_scalef32_pk_fp4_*).
//
// Bound by bytes: 8192 rows of 6144 in bf16 take 22 us, 5.8 TB/s, with one load of 16
// bytes a thread, two lane exchanges and one store of four. One row of 2048 takes 8 us
// of which a launch of nothing is 6.
#include "experts.hpp"

namespace inferno {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;

// Eight values per thread, four neighbouring threads per block. Rows are whole
// blocks, so that all of them are one long row.
template <typename XT, bool VALUES>
__global__ void __launch_bounds__(kThreads)
    mxfp4_quantize_kernel(const XT* __restrict__ x, size_t n8, uint32_t* __restrict__ codes,
                          uint8_t* __restrict__ scales, XT* __restrict__ values) {
  const size_t i = size_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= n8) return;  // blocks of four threads leave together
  constexpr bool kF32 = sizeof(XT) == 4;
  uint32_t raw[kF32 ? 8 : 4];
  const uint4* src = reinterpret_cast<const uint4*>(x) + i * (kF32 ? 2 : 1);
#pragma unroll
  for (int j = 0; j < (kF32 ? 2 : 1); ++j) {
    const uint4 u = src[j];
    raw[4 * j] = u.x; raw[4 * j + 1] = u.y; raw[4 * j + 2] = u.z; raw[4 * j + 3] = u.w;
  }
  float v[8];
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (kF32) v[j] = bits_to_f32(raw[j]);
    else v[j] = bits_to_f32(j & 1 ? raw[j / 2] & 0xffff0000u : raw[j / 2] << 16);
    most = max(most, f32_to_bits(v[j]) & 0x7fffffffu);
  }
  most = max(most, uint32_t(__shfl_xor(int(most), 1, kWave)));
  most = max(most, uint32_t(__shfl_xor(int(most), 2, kWave)));
  const uint32_t e = most >> 23;
  const bool finite = e < 255;
  // the biased exponent of the scale; blocks below 2^-125, zeros too, have 2^-127
  const uint32_t s = finite ? (e > 2 ? e - 2 : 0) : 255u;
  uint32_t q = 0;
  if (finite) {
    const float scale = bits_to_f32(s << 23);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
  }
  codes[i] = q;
  if (i % 4 == 0) scales[i / 4] = uint8_t(s);
  if constexpr (VALUES) {
    // powers of two by ldexp: the scale of the smallest blocks is subnormal
    uint32_t out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t c = q >> (4 * j), m = c & 1, ex = (c >> 1) & 3;
      const uint32_t halves = ex ? ((2 + m) << ex) >> 1 : m;
      float f = ldexpf(0.5f * float(halves), int(s) - 127);
      f = c & 8 ? -f : f;
      out[j] = finite ? f32_to_bits(f) : 0x7fc00000u;
    }
    uint4* to = reinterpret_cast<uint4*>(values) + i * (kF32 ? 2 : 1);
    if constexpr (kF32) {
      to[0] = make_uint4(out[0], out[1], out[2], out[3]);
      to[1] = make_uint4(out[4], out[5], out[6], out[7]);
    } else {  // two significant bits: exact
      to[0] = make_uint4(out[0] >> 16 | (out[1] & 0xffff0000u), out[2] >> 16 | (out[3] & 0xffff0000u),
                         out[4] >> 16 | (out[5] & 0xffff0000u), out[6] >> 16 | (out[7] & 0xffff0000u));
    }
  }
}

// Once per matrix: 128 experts of 1536 x 4096 in bf16 take 0.57 ms, 5.7 TB/s.
// One thread per 16 bytes, of `pieces` a row; those of a tile's first step of four
// bring the scales.
__global__ void __launch_bounds__(kThreads)
    experts_pack_kernel(const uint4* __restrict__ weights, const uint8_t* __restrict__ scales,
                        size_t N, size_t pieces, size_t tiles, size_t steps, size_t quads, size_t n,
                        uint4* __restrict__ to, uint32_t* __restrict__ to_scales) {
  for (size_t i = size_t(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += size_t(gridDim.x) * kThreads) {
    const uint32_t lane = uint32_t(i % 64);
    const size_t at = i / 64, c = at % steps, tile = at / steps;  // of all experts
    const size_t e = tile / tiles, row = (tile - e * tiles) * 16 + lane % 16;
    const size_t piece = c * 4 + lane / 16, src = (e * N + row) * pieces;
    const bool there = row < N;
    to[i] = there && piece < pieces ? weights[src + piece] : make_uint4(0, 0, 0, 0);
    if (scales && c % 4 == 0) {
      uint32_t w = 0;
      for (uint32_t j = 0; j < 4; ++j) {
        const size_t b = piece + 4 * j;
        w |= (there && b < pieces ? uint32_t(scales[src + b]) : 127u) << (8 * j);
      }
      to_scales[(tile * quads + c / 4) * 64 + lane] = w;
    }
  }
}

}  // namespace

int launch_mxfp4_quantize(hipStream_t s, const void* x, int x_dtype, size_t n, void* codes,
                          void* scales, void* values) {
  const size_t n8 = n / 8;
  const unsigned grid = unsigned((n8 + kThreads - 1) / kThreads);
  uint32_t* c = static_cast<uint32_t*>(codes);
  uint8_t* sc = static_cast<uint8_t*>(scales);
  auto go = [&](auto type, auto with) {
    using XT = decltype(type);
    mxfp4_quantize_kernel<XT, decltype(with)::value><<<grid, kThreads, 0, s>>>(
        static_cast<const XT*>(x), n8, c, sc, static_cast<XT*>(values));
  };
  if (x_dtype == INFERNO_F32) {
    if (values) go(0u, std::true_type{});
    else go(0u, std::false_type{});
  } else {
    if (values) go(uint16_t(0), std::true_type{});
    else go(uint16_t(0), std::false_type{});
  }
  INF_LAUNCHED();
  return INFERNO_OK;
}

int launch_experts_pack(hipStream_t s, const ExpertMat& m, const void* weights, const void* scales,
                        void* packed) {
  const ExpertLayout l = expert_layout(m);
  const size_t n = m.experts * l.tiles * l.steps * 64;
  const size_t most = size_t(1) << 20;  // workgroups
  const unsigned grid = unsigned(std::min((n + kThreads - 1) / kThreads, most));
  experts_pack_kernel<<<grid, kThreads, 0, s>>>(
      static_cast<const uint4*>(weights), static_cast<const uint8_t*>(scales), m.rows,
      m.cols / (m.fp4 ? 32 : 8), l.tiles, l.steps, l.quads, n, static_cast<uint4*>(packed),
      reinterpret_cast<uint32_t*>(static_cast<char*>(packed) + l.scales));
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
