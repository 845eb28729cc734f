// Products with 4-bit weights and group scales on the integer matrix cores.
//
//   y[t, n] = sum_g s[n, g] sum_{c in g} (q[n, c] - z[n, g]) x[t, c]
//
// The inner sum is formed exactly. A code is widened to 16 (q - 8), an int8, by
// one mask (its nibble stays in the high half of the byte), and an activation
// is one int8 digit (8-bit activations) or three, a 24-bit fixed-point value
// relative to the largest of its 128-column chunk: exact for every bf16 value
// down to 2^-14 of the largest, and off by at most 2^-23 of it for fp32. The
// int32 sums of a group are exact, the groups are added in fp32. Zero points
// start a group's sum at -16 (z - 8) times the digits' sum.
//
// Tile: 16 weight rows (the 16 columns of a 16x16 MFMA result) by 16 digit
// rows. A lane holds 32 codes of its row per chunk (16 bytes: low nibbles are
// the even columns, high nibbles the odd ones). Any order of the columns
// inside a group gives the same sum, so the codes are used as they lie and the
// digits are laid out to match.
#include "w4.hpp"

namespace inferno {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kMaxDigits = 127 * 65536 + 127 * 256 + 127;  // largest three-digit value

// ------------------------------------------------------------------ digits

struct Stage {
  const void* x;
  const float* x_scales;
  size_t x_group;  // > 0
  size_t R, K, C;
  W4Acts a;
};

__device__ __forceinline__ void load32(const float* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
  }
}
__device__ __forceinline__ void load32(const uint16_t* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[8 * i + 2 * j] = bits_to_f32(w[j] << 16);
      v[8 * i + 2 * j + 1] = bits_to_f32(w[j] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load32(const int8_t* p, float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) v[16 * i + j] = float(int8_t(w[j / 4] >> (8 * (j % 4))));
  }
}

// Byte offset in a chunk of column c of the chunk's block b (32 columns).
// Coarse groups: the block's lanes hold its even columns, then its odd ones.
// Fine groups: eight columns per lane of each block, even ones then odd ones.
__device__ __forceinline__ int place(bool fine, int b, int c) {
  return fine ? (c / 8) * 32 + b * 8 + (c & 1) * 4 + (c % 8) / 2
              : b * 32 + (c & 1) * 16 + c / 2;
}

// One thread per 32 columns; the four threads of a chunk share its largest
// value. Columns behind K are digits of 0.
template <typename XT, int P>
__global__ void __launch_bounds__(256) w4_stage_kernel(Stage p) {
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.R * p.C * 4) return;  // four threads of one chunk go together
  const size_t rc = i / 4, r = rc / p.C, c = rc % p.C;
  const int b = int(i % 4);
  const size_t col = c * kW4Chunk + b * 32;
  float v[32];
  if (col < p.K) {
    load32(static_cast<const XT*>(p.x) + r * p.K + col, v);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = 0.f;
  }
  int X[32];
  float xs;
  if (P == 1) {
#pragma unroll
    for (int j = 0; j < 32; ++j) X[j] = int(v[j]);
    // the chunk's first column lies in [0, K)
    xs = p.x_scales[r * (p.K / p.x_group) + c * kW4Chunk / p.x_group] * 0.0625f;
  } else {
    uint32_t most = 0;  // as integers: NaN lies above infinity
#pragma unroll
    for (int j = 0; j < 32; ++j) most = max(most, f32_to_bits(v[j]) & 0x7fffffffu);
    most = max(most, uint32_t(__shfl_xor(int(most), 1, kWave)));
    most = max(most, uint32_t(__shfl_xor(int(most), 2, kWave)));
    const bool finite = most < 0x7f800000u;
    // the largest power of two that keeps the value in three digits; chunks
    // below 2^-96 share its step, 2^-118
    int e = max(int(most >> 23) - 127, -96);
    int up = 22 - e;
    if (ldexpf(bits_to_f32(most), up) > float(kMaxDigits)) --up;
#pragma unroll
    for (int j = 0; j < 32; ++j) X[j] = finite ? int(rintf(ldexpf(v[j], up))) : 0;
    xs = finite ? ldexpf(1.f, -up - 4) : bits_to_f32(0x7fc00000u);
  }
  int8_t* out = p.a.planes + rc * (P * kW4Chunk);
  int sum[3] = {0, 0, 0};
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    int d[3] = {X[j], 0, 0};
    if (P == 3) {
      const uint32_t u = uint32_t(X[j] + 0x808080);
      d[0] = int(u >> 16) - 128;
      d[1] = int((u >> 8) & 255u) - 128;
      d[2] = int(u & 255u) - 128;
    }
#pragma unroll
    for (int q = 0; q < P; ++q) {
      out[q * kW4Chunk + place(p.a.fine, b, j)] = int8_t(d[q]);
      sum[q] += d[q];
    }
  }
  if (b == 0) p.a.xs[rc] = xs;
  if (p.a.sums == nullptr) return;
  constexpr int S = P == 3 ? 4 : 1;
  if (p.a.fine) {
    for (int q = 0; q < S; ++q) p.a.sums[(rc * 4 + b) * S + q] = q < P ? sum[q] : 0;
  } else {
    for (int q = 0; q < S; ++q) {
      int t = q < P ? sum[q] : 0;
      t += __shfl_xor(t, 1, kWave);
      t += __shfl_xor(t, 2, kWave);
      if (b == 0) p.a.sums[rc * S + q] = t;
    }
  }
}

// ----------------------------------------------------------------- product

struct Product {
  W4Mat m[2];
  int scale_bf16;
  uint32_t K, N, C, groups;  // columns, rows, chunks, groups per row
  uint32_t log2_group;       // fine groups
  uint32_t chunks_per_group; // coarse groups
  const int8_t* planes;
  const float* xs;
  const int* sums;
  uint32_t T;
  const uint32_t* offsets;
  const uint32_t* sorted;
  const uint32_t* active;
  uint32_t k;
  int x_by_assignment;
  const float* route_w;
  const float* res_a;
  const float* res_b;
  float* out;
};

__device__ __forceinline__ float load_scale(const void* p, int bf16, size_t i) {
  return bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i])
              : static_cast<const float*>(p)[i];
}

// 4x4 transpose of the dwords that the four 16-lane rows of a wavefront hold:
// dword j of row q becomes dword q of row j.
__device__ __forceinline__ void transpose4(uint32_t (&d)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const auto r = __builtin_amdgcn_permlane32_swap(d[j], d[j + 2], false, false);
    d[j] = r[0];
    d[j + 2] = r[1];
  }
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(d[j], d[j + 1], false, false);
    d[j] = r[0];
    d[j + 1] = r[1];
  }
}

enum Kind { kPack3, kOne, kWide3 };

// Tokens of one tile: kPack3 holds a token's three digits in rows 4 t, 4 t + 1,
// 4 t + 2 of one 16x16 result (one lane then has all three sums of a token);
// kOne and kWide3 hold 16 tokens, kWide3 in three results, one per digit.
template <int KIND>
struct KindOf {
  static constexpr int P = KIND == kOne ? 1 : 3;
  static constexpr int tokens = KIND == kPack3 ? 4 : 16;
  static constexpr int tiles = KIND == kWide3 ? 3 : 1;
  static constexpr int values = KIND == kPack3 ? 1 : 4;  // tokens per lane
};

// Sum of a token's digits' sums as a float. Without zero points a sum is at
// most 2^21 and the upper two join as integers; any byte as a zero point makes
// it 2^26.
template <bool ZEROS>
__device__ __forceinline__ float join(int hi, int mid, int lo) {
  if (ZEROS) return fmaf(float(hi), 65536.f, fmaf(float(mid), 256.f, float(lo)));
  return fmaf(float((hi << 8) + mid), 256.f, float(lo));
}

// One workgroup: 16 rows of the matrices (the same rows of both), all tokens
// of one expert (or of the batch) in tiles; the four wavefronts share the
// chunks and add their sums in order.
template <bool FINE, int MATS, int KIND, bool ZEROS>
__global__ void __launch_bounds__(256) w4_rows_kernel(Product p) {
  using KO = KindOf<KIND>;
  constexpr int P = KO::P, TT = KO::tokens, NT = KO::tiles, NV = KO::values;
  constexpr int S = P == 3 ? 4 : 1;
  __shared__ float part[4][MATS * NV][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = lane & 15, quad = lane >> 4;
  size_t expert = 0;
  uint32_t first = 0, end = p.T;
  if (p.offsets) {
    if (blockIdx.y >= p.active[0]) return;
    expert = p.active[1 + blockIdx.y];
    first = p.offsets[expert];
    end = p.offsets[expert + 1];
  }
  const uint32_t row = blockIdx.x * 16 + n;
  const size_t mrow = expert * p.N + min(row, p.N - 1);
  const uint32_t c0 = p.C * wave / 4, c1 = p.C * (wave + 1) / 4;
  // activation row of assignment (or token) i
  auto x_row = [&](uint32_t i) -> size_t {
    const uint32_t j = min(i, end - 1);
    if (!p.offsets) return j;
    const uint32_t a = p.sorted[j];
    return p.x_by_assignment ? a : a / p.k;
  };
  for (uint32_t t0 = first; t0 < end; t0 += TT) {
    // this lane's operand row, and the tokens whose sums it gets
    const size_t xr = x_row(t0 + (KIND == kPack3 ? n / 4 : n));
    const int plane = KIND == kPack3 ? min(n & 3, 2) : 0;
    size_t vr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) vr[i] = x_row(t0 + (KIND == kPack3 ? quad : 4 * quad + i));
    float acc[MATS][NV];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[m][i] = 0.f;
    for (uint32_t c = c0; c < c1; ++c) {
      v4u xe[NT], xo[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const v4u* x = reinterpret_cast<const v4u*>(
            p.planes + ((xr * p.C + c) * P + plane + t) * kW4Chunk + quad * 32);
        xe[t] = x[0];
        xo[t] = x[1];
      }
      float xs[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) xs[i] = p.xs[vr[i] * p.C + c];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        uint32_t d[4] = {0, 0, 0, 0};
        if (c * kW4Chunk + quad * 32 < p.K) {
          const v4u v = *reinterpret_cast<const v4u*>(p.m[m].codes + mrow * (p.K / 2) +
                                                      c * (kW4Chunk / 2) + quad * 16);
          d[0] = v[0]; d[1] = v[1]; d[2] = v[2]; d[3] = v[3];
        }
        if (FINE) transpose4(d);
        v4i lo, hi;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u = d[j] ^ 0x88888888u;  // q - 8 in four bits
          lo[j] = int((u << 4) & 0xf0f0f0f0u);
          hi[j] = int(u & 0xf0f0f0f0u);
        }
        // digit sums of the tokens of this lane, for zero points
        auto start = [&](int t, int block, float z) {
          v4i s = {0, 0, 0, 0};
          if (!ZEROS) return s;
          const int by = -16 * (int(z) - 8);
          if (KIND == kPack3) {
            const int* at = p.sums + ((vr[0] * p.C + c) * (FINE ? 4 : 1) + block) * S;
#pragma unroll
            for (int i = 0; i < 3; ++i) s[i] = by * at[i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[i] = by * p.sums[((vr[i] * p.C + c) * (FINE ? 4 : 1) + block) * S + t];
          }
          return s;
        };
        float value[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) value[i] = 0.f;
#pragma unroll
        for (int b = 0; b < (FINE ? 4 : 1); ++b) {
          const uint32_t g = FINE ? min((c * kW4Chunk + 32 * b) >> p.log2_group, p.groups - 1)
                                  : c / p.chunks_per_group;
          const float ws = load_scale(p.m[m].scales, p.scale_bf16, mrow * p.groups + g);
          const float z = ZEROS ? float(p.m[m].zeros[mrow * p.groups + g]) : 0.f;
          v4i sum[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sum[t] = start(t, b, z);
            if (FINE) {
              auto two = [](int a, int b) { return (long(uint32_t(b)) << 32) | uint32_t(a); };
              const long xb = b < 2 ? two(xe[t][2 * b], xe[t][2 * b + 1])
                                    : two(xo[t][2 * b - 4], xo[t][2 * b - 3]);
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(xb, two(lo[b], hi[b]), sum[t], 0, 0, 0);
            } else {
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, xe[t]), lo,
                                                             sum[t], 0, 0, 0);
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, xo[t]), hi,
                                                             sum[t], 0, 0, 0);
            }
          }
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            float f;
            if (KIND == kPack3) f = join<ZEROS>(sum[0][0], sum[0][1], sum[0][2]);
            else if (KIND == kOne) f = float(sum[0][i]);
            else f = join<ZEROS>(sum[0][i], sum[NT > 1 ? 1 : 0][i], sum[NT > 2 ? 2 : 0][i]);
            value[i] = fmaf(ws, f, value[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[m][i] = fmaf(value[i], xs[i], acc[m][i]);
      }
    }
    __syncthreads();  // the last tile's sums are read
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int i = 0; i < NV; ++i) part[wave][m * NV + i][lane] = acc[m][i];
    __syncthreads();
    // wavefront i writes token value i of every lane
    if (wave < NV && row < p.N) {
      const int i = wave;
      const uint32_t t = t0 + (KIND == kPack3 ? quad : 4 * quad + i);
      if (t < end) {
        float v[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          v[m] = part[0][m * NV + i][lane];
          for (int w = 1; w < 4; ++w) v[m] += part[w][m * NV + i][lane];
        }
        const size_t a = p.offsets ? p.sorted[t] : t;
        float y = v[0];
        if (MATS == 2) y = v[0] / (1.f + expf(-v[0])) * v[MATS - 1];
        if (p.route_w) y *= p.route_w[a];
        const size_t at = a * p.N + row;
        if (p.res_a) y += p.res_a[at];
        if (p.res_b) y += p.res_b[at];
        p.out[at] = y;
      }
    }
  }
}

template <bool FINE, int MATS, bool ZEROS>
void run_rows(hipStream_t s, const Product& p, dim3 grid, int kind) {
  if (kind == kPack3) w4_rows_kernel<FINE, MATS, kPack3, ZEROS><<<grid, 256, 0, s>>>(p);
  else if (kind == kOne) w4_rows_kernel<FINE, MATS, kOne, ZEROS><<<grid, 256, 0, s>>>(p);
  else w4_rows_kernel<FINE, MATS, kWide3, ZEROS><<<grid, 256, 0, s>>>(p);
}

// ----------------------------------------------------------------- combine

__global__ void __launch_bounds__(256)
    w4_combine_kernel(const float* __restrict__ y, const uint32_t* __restrict__ ids, size_t n,
                      uint32_t H, uint32_t k, uint32_t E, float* __restrict__ out) {
  const size_t i = size_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const size_t t = i / H, h = i % H;
  float v = 0.f;
  for (uint32_t r = 0; r < k; ++r) {
    const size_t a = t * k + r;
    if (ids[a] < E) v += y[a * H + h];
  }
  out[i] = v;
}

}  // namespace

int launch_w4_stage(hipStream_t s, const void* x, int x_dtype, const float* x_scales,
                    size_t x_group, size_t R, size_t K, const W4Acts& a) {
  const Stage p{x, x_scales, x_group ? x_group : K, R, K, w4_chunks(K), a};
  const unsigned grid = unsigned((R * p.C * 4 + 255) / 256);
  if (x_dtype == INFERNO_F32) w4_stage_kernel<float, 3><<<grid, 256, 0, s>>>(p);
  else if (x_dtype == INFERNO_BF16) w4_stage_kernel<uint16_t, 3><<<grid, 256, 0, s>>>(p);
  else w4_stage_kernel<int8_t, 1><<<grid, 256, 0, s>>>(p);
  INF_LAUNCHED();
  return INFERNO_OK;
}

int launch_w4_product(hipStream_t s, const W4Product& q) {
  Product p{};
  p.m[0] = q.m[0];
  p.m[1] = q.m[1];
  p.scale_bf16 = q.scale_dtype == INFERNO_BF16;
  p.K = uint32_t(q.K);
  p.N = uint32_t(q.N);
  p.C = uint32_t(w4_chunks(q.K));
  p.groups = uint32_t(q.K / q.group);
  p.log2_group = q.group == 32 ? 5 : 6;
  p.chunks_per_group = uint32_t(q.group / kW4Chunk);
  p.planes = q.x.planes;
  p.xs = q.x.xs;
  p.sums = q.x.sums;
  p.T = uint32_t(q.T);
  p.offsets = q.offsets;
  p.sorted = q.sorted;
  p.active = q.active;
  p.k = uint32_t(q.k);
  p.x_by_assignment = q.x_by_assignment;
  p.route_w = q.route_w;
  p.res_a = q.res_a;
  p.res_b = q.res_b;
  p.out = q.out;
  const unsigned slots = q.offsets ? unsigned(std::min(q.E, q.T * q.k)) : 1u;
  const dim3 grid(unsigned((q.N + 15) / 16), slots);
  const int kind = q.x.P == 1 ? kOne : q.T <= 4 ? kPack3 : kWide3;
  const bool zeros = q.m[0].zeros != nullptr;
  if (q.x.fine) {
    if (q.mats == 2) zeros ? run_rows<true, 2, true>(s, p, grid, kind)
                           : run_rows<true, 2, false>(s, p, grid, kind);
    else zeros ? run_rows<true, 1, true>(s, p, grid, kind)
               : run_rows<true, 1, false>(s, p, grid, kind);
  } else {
    if (q.mats == 2) zeros ? run_rows<false, 2, true>(s, p, grid, kind)
                           : run_rows<false, 2, false>(s, p, grid, kind);
    else zeros ? run_rows<false, 1, true>(s, p, grid, kind)
               : run_rows<false, 1, false>(s, p, grid, kind);
  }
  INF_LAUNCHED();
  return INFERNO_OK;
}

int launch_w4_combine(hipStream_t s, const float* y, const uint32_t* ids, size_t T, size_t H,
                      size_t k, size_t E, float* out) {
  const size_t n = T * H;
  w4_combine_kernel<<<unsigned((n + 255) / 256), 256, 0, s>>>(y, ids, n, uint32_t(H), uint32_t(k),
                                                              uint32_t(E), out);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
