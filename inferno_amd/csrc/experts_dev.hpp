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
  const uint8_t* w[2];      // packed weights
  const uint32_t* ws[2];    // and their scales
  const uint8_t* x;
  const uint8_t* xs;        // scales of codes
  uint32_t x_bytes;         // of x; below 2^32 where rows go through LDS
  const uint32_t* offsets;  // or null
  const uint32_t* sorted;   // or null
  uint32_t E, A, k;
  uint32_t per_k;           // 2^32 / k + 1, of k above 1
  uint32_t N, K;
  uint32_t tiles, steps, quads;  // of an expert's packed weights
  void* out;
  bool out_f32;
  uint32_t splits;          // shares of the columns in launches of their own workgroups
  float* partial;           // [splits][matrices][A][N, to a multiple of 4]: their sums
};

// The work of workgroup b of a launch of tiles of at most TM rows by `units`
// workgroups each (blocks of weight rows, shares of the columns).
struct Work {
  uint32_t e, c0, c1;  // expert, rows [c0, c1) of the grouped order
  uint32_t unit;
};

// Finds it, or says that there is none (launches have as many workgroups as the
// rows can need at most). Every wavefront finds its own (257 words, which L2 holds,
// and one scan over the lanes): a launch before the product would cost more. Ranges
// that are not ascending, or end behind the last row, are cut, so that whatever lies
// in offsets no row index is A or more.
// With XCD, each of the eight XCDs, to which workgroups go in turn, has one run of
// the work, in which an expert's tiles of one unit follow each other: what they
// share comes to the XCD's L2 once.
template <uint32_t TM, bool XCD>
__device__ __forceinline__ bool find_work(const Product& p, uint32_t b, uint32_t units, Work& w) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t o[5], n[4], sum = 0;
  if (p.offsets) {
#pragma unroll
    for (uint32_t j = 0; j < 5; ++j) o[j] = p.offsets[min(4 * lane + j, p.E)];
#pragma unroll
    for (uint32_t j = 0; j < 5; ++j) o[j] = min(o[j], p.A);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 5; ++j) o[j] = 4 * lane + j ? p.A : 0;
  }
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
  const uint32_t all = __builtin_amdgcn_readlane(upto, 63) * units;
  if constexpr (XCD) {
    const uint32_t run = (all + 7) / 8;
    if (b / 8 >= run) return false;
    b = b % 8 * run + b / 8;
  }
  if (b >= all) return false;
  const uint32_t t = b / units;
  const int at = __ffsll((unsigned long long)__ballot(upto > t)) - 1;
  // of the lane `at` alone: its expert j, which has tiles before .. before + n[j]
  uint32_t before = upto - sum, j = 0;
#pragma unroll
  for (uint32_t i = 0; i < 3; ++i)
    if (j == i && t >= before + n[i]) {
      before += n[i];
      j = i + 1;
    }
  const uint32_t begin = __builtin_amdgcn_readlane(j == 0 ? o[0] : j == 1 ? o[1] : j == 2 ? o[2] : o[3], at);
  const uint32_t end = __builtin_amdgcn_readlane(j == 0 ? o[1] : j == 1 ? o[2] : j == 2 ? o[3] : o[4], at);
  const uint32_t tiles = __builtin_amdgcn_readlane(j == 0 ? n[0] : j == 1 ? n[1] : j == 2 ? n[2] : n[3], at);
  const uint32_t inside = b - __builtin_amdgcn_readlane(before, at) * units;
  w.e = __builtin_amdgcn_readlane(4 * lane + j, at);
  w.unit = XCD ? inside / tiles : inside % units;
  const uint32_t tile = XCD ? inside - w.unit * tiles : inside / units;
  w.c0 = begin + tile * TM;
  w.c1 = min(w.c0 + TM, end);
  return true;
}

// Result rows of grouped rows c < A, in place; A or more: none (an index out of
// range). All loads at once, since each takes as long as all.
template <int N>
__device__ __forceinline__ void result_rows(const Product& p, uint32_t (&c)[N]) {
  if (!p.sorted) return;
  uint32_t a[N];
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = p.sorted[c[i]];
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = a[i];
}

// Input row of a result row (0 where there is none). With a < 2^22 and k <= 1024, a
// (2^32 / k + 1) / 2^32 is a / k but for less than 1 / k.
__device__ __forceinline__ uint32_t input_row(const Product& p, uint32_t a) {
  if (a >= p.A) return 0;
  if (p.k == 1) return a;
  return p.k <= 1024 ? __umulhi(a, p.per_k) : a / p.k;
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

// Four neighbouring values of one result row. Rows of a length that is no multiple
// of four lie at any multiple of a value's size.
__device__ __forceinline__ void store4(const Product& p, uint32_t row, uint32_t n, const float (&y)[4]) {
  if (n >= p.N) return;
  const size_t at = size_t(row) * p.N + n;
  const bool whole = p.N % 4 == 0;
  if (p.out_f32) {
    float* to = static_cast<float*>(p.out) + at;
    if (whole) {
      *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
    } else if (n + 4 <= p.N) {
      __builtin_memcpy(to, y, 16);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 3; ++i)
        if (n + i < p.N) to[i] = y[i];
    }
    return;
  }
  uint16_t* to = static_cast<uint16_t*>(p.out) + at;
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __builtin_bit_cast(uint16_t, (__bf16)y[i]);
  const uint2 two = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  if (whole) {
    *reinterpret_cast<uint2*>(to) = two;
  } else if (n + 4 <= p.N) {
    __builtin_memcpy(to, &two, 8);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
      if (n + i < p.N) to[i] = uint16_t(h[i]);
  }
}

}  // namespace experts

// Tiles of up to `rows` (32, 64 or 128) by 64 * width weight rows of all matrices;
// `tiles`: at least as many as there are.
int launch_experts_tiles(hipStream_t s, const experts::Product& p, int mats, bool wfp4, bool xfp4,
                         size_t tiles, int width, int rows);

}  // namespace inferno
