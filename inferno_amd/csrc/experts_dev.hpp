// Device side of the products of rows grouped by expert: which rows a workgroup
// has, and fragments of the matrix instructions.
#pragma once
#include "experts.hpp"

namespace inferno {
namespace experts {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

struct Product {
  const uint8_t* w[2];      // codes, or bf16
  const uint32_t* ws[2];    // packed scales
  const uint8_t* x;
  const uint8_t* xs;        // scales of codes
  uint32_t x_bytes;         // of x; below 2^32 where rows go through LDS
  const uint32_t* offsets;  // or null
  const uint32_t* sorted;   // or null
  uint32_t E, A, k;
  uint32_t N, K;
  uint32_t tiles, chunks, quads;  // packed weights of an expert: 16-row tiles, chunks, four chunks
  void* out;
  bool out_f32;
  uint32_t splits;          // shares of the columns in launches of their own workgroups
  float* partial;           // [splits][matrices][A][N, to a multiple of 4]: their sums
};

// Tile `t` of at most TM rows of one expert, tiles counted expert by expert:
// rows [c0, c1) of the grouped order. Returns the number of all tiles; t is one
// of them if it is below. Every wavefront finds its own (257 words at most, which
// L2 holds, and one scan over the lanes): a launch before the product would
// cost more. Ranges that are not ascending, or end behind the last row, are cut,
// so that whatever lies in offsets no row index is A or more.
template <uint32_t TM>
__device__ __forceinline__ uint32_t find_tile(const Product& p, uint32_t t, uint32_t& e,
                                              uint32_t& c0, uint32_t& c1) {
  if (!p.offsets) {
    e = 0;
    c0 = min(t * TM, p.A);
    c1 = min(c0 + TM, p.A);
    return (p.A + TM - 1) / TM;
  }
  const uint32_t lane = threadIdx.x & 63;
  uint32_t o[5], sum = 0, n[4];
#pragma unroll
  for (uint32_t j = 0; j < 5; ++j) o[j] = min(p.offsets[min(4 * lane + j, p.E)], p.A);
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    n[j] = o[j + 1] > o[j] ? (o[j + 1] - o[j] + TM - 1) / TM : 0;
    sum += n[j];
  }
  uint32_t upto = sum;  // tiles of this lane's experts and those before
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t v = uint32_t(__shfl_up(int(upto), d, kWave));
    if (int(lane) >= d) upto += v;
  }
  const uint32_t all = __builtin_amdgcn_readlane(upto, 63);
  const uint64_t behind = __ballot(upto > t);
  if (behind == 0) return all;
  const int at = __ffsll((unsigned long long)behind) - 1;
  uint32_t rest = t - (upto - sum), j = 0;  // of the lane `at` alone
#pragma unroll
  for (uint32_t i = 0; i < 3; ++i)
    if (j == i && rest >= n[i]) {
      rest -= n[i];
      j = i + 1;
    }
  const uint32_t first = j == 0 ? o[0] : j == 1 ? o[1] : j == 2 ? o[2] : o[3];
  const uint32_t last = j == 0 ? o[1] : j == 1 ? o[2] : j == 2 ? o[3] : o[4];
  e = __builtin_amdgcn_readlane(4 * lane + j, at);
  c0 = __builtin_amdgcn_readlane(first + rest * TM, at);
  c1 = min(c0 + TM, __builtin_amdgcn_readlane(last, at));
  return all;
}

// Result row of grouped row c < A; A or more: none (an index out of range).
__device__ __forceinline__ uint32_t result_row(const Product& p, uint32_t c) {
  return p.sorted ? p.sorted[c] : c;
}

// Where the sums of a share, matrix and grouped row begin in `partial`.
__device__ __forceinline__ size_t partial_row(const Product& p, uint32_t mats, uint32_t split,
                                              uint32_t m, uint32_t c) {
  return ((size_t(split) * mats + m) * p.A + c) * ((p.N + 3) & ~3u);
}

// 2^(byte - 127) where only the exponent is read (v_cvt_scalef32_*: 255 is NaN).
__device__ __forceinline__ float scale_of(uint32_t byte) { return bits_to_f32(byte << 23); }

// Eight codes to bf16, exactly: two significant bits.
__device__ __forceinline__ bf16x8 widen(uint32_t codes, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ floatx4 mfma_bf16(bf16x8 a, bf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 32 codes per lane of either operand, each with the scale in the lowest byte of
// its lane's word.
__device__ __forceinline__ floatx4 mfma_fp4(uint4 a, uint4 b, floatx4 c, uint32_t as, uint32_t bs) {
  const intx8 av = {int(a.x), int(a.y), int(a.z), int(a.w), 0, 0, 0, 0};
  const intx8 bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, int(as), 0, int(bs));
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// Four neighbouring values of one result row.
__device__ __forceinline__ void store4(const Product& p, uint32_t row, uint32_t n, const float (&y)[4]) {
  if (n >= p.N) return;
  const size_t at = size_t(row) * p.N + n;
  if (p.out_f32) {
    float* to = static_cast<float*>(p.out) + at;
    if (p.N % 4 == 0) {
      *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (n + i < p.N) to[i] = y[i];
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(p.out) + at;
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __builtin_bit_cast(uint16_t, (__bf16)y[i]);
  if (p.N % 4 == 0) {
    *reinterpret_cast<uint2*>(to) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (n + i < p.N) to[i] = uint16_t(h[i]);
  }
}

}  // namespace experts

// Tiles of up to 128 rows by 16 * 4 * width weight rows of both matrices; `tiles`:
// at least as many as there are.
int launch_experts_tiles(hipStream_t s, const experts::Product& p, int mats, bool wfp4, bool xfp4,
                         size_t tiles, int width);

}  // namespace inferno
