// Products with 4-bit weights and group scales on the integer matrix cores.
//
//   y[t, n] = sum_g s[n, g] sum_{c in g} (q[n, c] - z[n, g]) x[t, c]
//
// The inner sum is formed exactly. A code is widened to 16 (q - 8), an int8, by
// one mask (its nibble stays in the high half of the byte), or to q - z with
// four codes in one subtraction; an activation is one int8 digit (8-bit
// activations) or three, a 24-bit fixed-point value relative to the largest of
// its 128-column chunk: exact for every bf16 value down to 2^-14 of the
// largest, and off by at most 2^-23 of it for fp32. The int32 sums of a group
// are exact, the groups are added in fp32.
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

// Four bytes, byte i of them byte `at` of d[i].
__device__ __forceinline__ uint32_t gather4(uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                            int at) {
  const uint32_t sel = uint32_t(at) | uint32_t(at + 4) << 8;  // byte `at` of each of a pair
  const uint32_t lo = __builtin_amdgcn_perm(b, a, sel), hi = __builtin_amdgcn_perm(d, c, sel);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// One thread per 32 columns; the four threads of a chunk share its largest
// value. Columns behind K are digits of 0. A plane's 128 bytes of a chunk are
// two halves of four 16-byte pieces, a piece for each 16-lane row of the
// weights' tile. Coarse groups: lane row b holds block b's codes, its piece of
// the first half the block's even columns, of the second half the odd ones.
// Fine groups: lane row r holds columns 8 r .. 8 r + 7 of every block; half h
// has those of blocks 2 h and 2 h + 1, four even ones, four odd ones each.
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
  uint32_t X[32];  // digit 0 in the highest of P bytes, offset by 128
  float xs;
  if (P == 1) {
#pragma unroll
    for (int j = 0; j < 32; ++j) X[j] = uint32_t(int(v[j]) + 128);
    // the chunk's first column lies in [0, K)
    xs = p.x_scales[r * (p.K / p.x_group) + c * kW4Chunk / p.x_group];
  } else {
    uint32_t most = 0;  // as integers: NaN lies above infinity
#pragma unroll
    for (int j = 0; j < 32; ++j) most = max(most, f32_to_bits(v[j]) & 0x7fffffffu);
    most = max(most, uint32_t(__shfl_xor(int(most), 1, kWave)));
    most = max(most, uint32_t(__shfl_xor(int(most), 2, kWave)));
    const bool finite = most < 0x7f800000u;
    // the largest power of two that keeps the value in three digits; chunks
    // below 2^-96 share its step, 2^-118
    const int e = max(int(most >> 23) - 127, -96);
    int up = 22 - e;
    if (ldexpf(bits_to_f32(most), up) > float(kMaxDigits)) --up;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      X[j] = uint32_t((finite ? int(rintf(ldexpf(v[j], up))) : 0) + 0x808080);
    xs = finite ? ldexpf(1.f, -up) : bits_to_f32(0x7fc00000u);
  }
  int8_t* out = p.a.planes + rc * (P * kW4Chunk);
#pragma unroll
  for (int q = 0; q < P; ++q) {
    uint32_t w[2][4];  // [even, odd][four columns]: columns 8 m + 2 i (+ 1)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        w[o][m] = gather4(X[8 * m + o], X[8 * m + o + 2], X[8 * m + o + 4], X[8 * m + o + 6],
                          P - 1 - q) ^ 0x80808080u;
    int8_t* plane = out + q * kW4Chunk;
    if (p.a.fine) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
        *reinterpret_cast<uint2*>(plane + (b / 2) * 64 + m * 16 + (b % 2) * 8) =
            make_uint2(w[0][m], w[1][m]);
    } else {
#pragma unroll
      for (int o = 0; o < 2; ++o)
        *reinterpret_cast<uint4*>(plane + o * 64 + b * 16) =
            make_uint4(w[o][0], w[o][1], w[o][2], w[o][3]);
    }
  }
  if (b == 0) p.a.xs[rc] = xs;
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

// Sum of a token's digits' sums as a float; a sum is at most 2^21.
__device__ __forceinline__ float join(int hi, int mid, int lo) {
  return fmaf(float((hi << 8) + mid), 256.f, float(lo));
}

// Four even and four odd columns of a dword of codes as int8: 16 (q - 8), or
// q - z with zero points (zz: z in every byte, at most 127, so that no byte
// borrows from the next).
template <bool ZEROS>
__device__ __forceinline__ void widen(uint32_t d, uint32_t zz, int& even, int& odd) {
  if (ZEROS) {
    even = int((((d & 0x0f0f0f0fu) | 0x80808080u) - zz) ^ 0x80808080u);
    odd = int(((((d >> 4) & 0x0f0f0f0fu) | 0x80808080u) - zz) ^ 0x80808080u);
  } else {
    const uint32_t u = d ^ 0x88888888u;
    even = int((u << 4) & 0xf0f0f0f0u);
    odd = int(u & 0xf0f0f0f0u);
  }
}

__device__ __forceinline__ uint32_t spread(uint32_t z) { return min(z, 127u) * 0x01010101u; }

// The scale of one group, for widen's codes.
template <bool ZEROS>
__device__ __forceinline__ float code_scale(const Product& p, int m, size_t i) {
  return load_scale(p.m[m].scales, p.scale_bf16, i) * (ZEROS ? 1.f : 0.0625f);
}

__device__ __forceinline__ long two(uint32_t a, uint32_t b) {
  return long((uint64_t(b) << 32) | a);
}

// One workgroup: 16 rows of the matrices (the same rows of both), all tokens
// of one expert (or of the batch) in tiles; the four wavefronts share the
// chunks and add their sums in order.
template <bool FINE, int MATS, int KIND, bool ZEROS>
__global__ void __launch_bounds__(256) w4_rows_kernel(Product p) {
  using KO = KindOf<KIND>;
  constexpr int P = KO::P, TT = KO::tokens, NT = KO::tiles, NV = KO::values;
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
            p.planes + ((xr * p.C + c) * P + plane + t) * kW4Chunk + quad * 16);
        xe[t] = x[0];
        xo[t] = x[4];
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
        float ws[FINE ? 4 : 1];
#pragma unroll
        for (int b = 0; b < (FINE ? 4 : 1); ++b) {
          const uint32_t g = FINE ? min((c * kW4Chunk + 32 * b) >> p.log2_group, p.groups - 1)
                                  : c / p.chunks_per_group;
          ws[b] = code_scale<ZEROS>(p, m, mrow * p.groups + g);
          const uint32_t zz = ZEROS ? spread(p.m[m].zeros[mrow * p.groups + g]) : 0u;
          if (FINE) {
            int l, h;
            widen<ZEROS>(d[b], zz, l, h);
            lo[b] = l;
            hi[b] = h;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              int l, h;
              widen<ZEROS>(d[j], zz, l, h);
              lo[j] = l;
              hi[j] = h;
            }
          }
        }
        float value[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) value[i] = 0.f;
#pragma unroll
        for (int b = 0; b < (FINE ? 4 : 1); ++b) {
          v4i sum[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sum[t] = v4i{0, 0, 0, 0};
            if (FINE) {
              const long xb = b < 2 ? two(xe[t][2 * b], xe[t][2 * b + 1])
                                    : two(xo[t][2 * b - 4], xo[t][2 * b - 3]);
              sum[t] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                  xb, two(uint32_t(lo[b]), uint32_t(hi[b])), sum[t], 0, 0, 0);
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
            if (KIND == kPack3) f = join(sum[0][0], sum[0][1], sum[0][2]);
            else if (KIND == kOne) f = float(sum[0][i]);
            else f = join(sum[0][i], sum[NT > 1 ? 1 : 0][i], sum[NT > 2 ? 2 : 0][i]);
            value[i] = fmaf(ws[b], f, value[i]);
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

// Many tokens. One workgroup: 64 tokens by 64 RT rows of the matrices; a
// wavefront takes RT tiles of 16 rows of each matrix against all tokens. The
// weights go from memory to the wavefront that owns them, one chunk ahead; the
// tokens' digits go through LDS (two buffers, filled by the LDS DMA one chunk
// ahead) in the order in which the matrix instructions' lanes read them, so
// that a read is 1 KB without bank conflicts. Tiles of 16 tokens that an
// expert does not have are left out.
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;

constexpr int kTileTokens = 64;

template <bool FINE, int MATS, int P, bool ZEROS, int RT>
__global__ void __launch_bounds__(256, 2) w4_tile_kernel(Product p) {
  constexpr int F = MATS * RT, TT = kTileTokens / 16, B = FINE ? 4 : 1;
  __shared__ __align__(16) int8_t xt[2][TT][2 * P][kWave * 16];
  __shared__ __align__(16) float xst[2][kTileTokens];
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
  const uint32_t row0 = (blockIdx.x * 4 + wave) * (16 * RT) + n;
  const uint8_t* codes[F];
  size_t group0[RT];  // of the row's first group
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const size_t mrow = expert * p.N + min(row0 + 16 * r, p.N - 1);
    group0[r] = mrow * p.groups;
#pragma unroll
    for (int m = 0; m < MATS; ++m) codes[m * RT + r] = p.m[m].codes + mrow * (p.K / 2);
  }
  auto x_row = [&](uint32_t i) -> size_t {
    const uint32_t j = min(i, end - 1);
    if (!p.offsets) return j;
    const uint32_t a = p.sorted[j];
    return p.x_by_assignment ? a : a / p.k;
  };
  for (uint32_t t0 = first + blockIdx.z * kTileTokens; t0 < end; t0 += gridDim.z * kTileTokens) {
    const uint32_t tokens = min(end - t0, uint32_t(kTileTokens));
    // wavefront w copies the digits of token tile w, the first one the scales
    const int8_t* xp = p.planes + x_row(t0 + 16 * wave + n) * p.C * (P * kW4Chunk) + quad * 16;
    const float* sp = p.xs + x_row(t0 + lane) * p.C;
    float acc[F][TT][4];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][t][i] = 0.f;
    auto copy = [&](uint32_t c) {
      if (16u * wave < tokens) {
#pragma unroll
        for (int i = 0; i < 2 * P; ++i)
          __builtin_amdgcn_global_load_lds((gptr_t)(xp + size_t(c) * (P * kW4Chunk) + i * 64),
                                           (lptr_t)&xt[c & 1][wave][i][0], 16, 0, 0);
      }
      if (wave == 0)
        __builtin_amdgcn_global_load_lds((gptr_t)(sp + c), (lptr_t)&xst[c & 1][0], 4, 0, 0);
    };
    v4u next[F];
    float next_s[F][B];
    uint32_t next_z[F][B];
    auto fetch = [&](uint32_t c) {
      // columns behind K meet digits of 0: any codes do
      const uint32_t at = min(c * (kW4Chunk / 2) + quad * 16, p.K / 2 - 16);
#pragma unroll
      for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int f = m * RT + r;
          next[f] = *reinterpret_cast<const v4u*>(codes[f] + at);
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const uint32_t g = FINE ? min((c * kW4Chunk + 32 * b) >> p.log2_group, p.groups - 1)
                                    : c / p.chunks_per_group;
            next_s[f][b] = code_scale<ZEROS>(p, m, group0[r] + g);
            next_z[f][b] = ZEROS ? p.m[m].zeros[group0[r] + g] : 0u;
          }
        }
    };
    copy(0);
    fetch(0);
    for (uint32_t c = 0; c < p.C; ++c) {
      v4i lo[F], hi[F];
      float ws[F][B];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        uint32_t d[4] = {next[f][0], next[f][1], next[f][2], next[f][3]};
        if (FINE) transpose4(d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          int l, h;
          widen<ZEROS>(d[j], ZEROS ? spread(next_z[f][FINE ? j : 0]) : 0u, l, h);
          lo[f][j] = l;
          hi[f][j] = h;
        }
#pragma unroll
        for (int b = 0; b < B; ++b) ws[f][b] = next_s[f][b];
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's copies are in LDS
      __builtin_amdgcn_s_barrier();  // everybody's are, and chunk c - 1 is read
      if (c + 1 < p.C) {
        copy(c + 1);
        fetch(c + 1);
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if (16u * t < tokens) {  // uniform
          v4u x[2 * P];
#pragma unroll
          for (int i = 0; i < 2 * P; ++i)
            x[i] = *reinterpret_cast<const v4u*>(&xt[c & 1][t][i][lane * 16]);
          const float4 s4 = *reinterpret_cast<const float4*>(&xst[c & 1][16 * t + 4 * quad]);
          const float xs[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int f = 0; f < F; ++f) {
            float value[4];
#pragma unroll
            for (int b = 0; b < B; ++b) {
              v4i sum[P];
#pragma unroll
              for (int q = 0; q < P; ++q) {
                sum[q] = v4i{0, 0, 0, 0};
                if (FINE) {
                  const v4u u = x[2 * q + b / 2];
                  sum[q] = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                      two(u[2 * (b % 2)], u[2 * (b % 2) + 1]),
                      two(uint32_t(lo[f][b]), uint32_t(hi[f][b])), sum[q], 0, 0, 0);
                } else {
                  sum[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                      __builtin_bit_cast(v4i, x[2 * q]), lo[f], sum[q], 0, 0, 0);
                  sum[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                      __builtin_bit_cast(v4i, x[2 * q + 1]), hi[f], sum[q], 0, 0, 0);
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = P == 3 ? join(sum[0][i], sum[P / 2][i], sum[P - 1][i])
                                       : float(sum[0][i]);
                value[i] = b == 0 ? ws[f][b] * v : fmaf(ws[f][b], v, value[i]);
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[f][t][i] = fmaf(value[i], xs[i], acc[f][t][i]);
          }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t j = t0 + 16 * t + 4 * quad + i;
        if (j >= end) continue;
        const size_t a = p.offsets ? p.sorted[j] : j;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t row = row0 + 16 * r;
          if (row >= p.N) continue;
          float y = acc[r][t][i];
          if (MATS == 2) y = y / (1.f + expf(-y)) * acc[(MATS - 1) * RT + r][t][i];
          if (p.route_w) y *= p.route_w[a];
          const size_t at = a * p.N + row;
          if (p.res_a) y += p.res_a[at];
          if (p.res_b) y += p.res_b[at];
          p.out[at] = y;
        }
      }
    }
    __syncthreads();  // the last chunk is read: the next tokens' first may come
  }
}

template <bool FINE, int MATS, int P, bool ZEROS>
void run_tiles(hipStream_t s, const Product& p, unsigned slots, unsigned blocks) {
  constexpr int RT = MATS == 2 ? 2 : 4;
  const dim3 grid((p.N + 64 * RT - 1) / (64 * RT), slots, blocks);
  w4_tile_kernel<FINE, MATS, P, ZEROS, RT><<<grid, 256, 0, s>>>(p);
}

template <bool FINE, bool ZEROS>
void run_tiles(hipStream_t s, const Product& p, int mats, int P, unsigned slots, unsigned blocks) {
  if (mats == 2 && P == 3) run_tiles<FINE, 2, 3, ZEROS>(s, p, slots, blocks);
  else if (mats == 2) run_tiles<FINE, 2, 1, ZEROS>(s, p, slots, blocks);
  else if (P == 3) run_tiles<FINE, 1, 3, ZEROS>(s, p, slots, blocks);
  else run_tiles<FINE, 1, 1, ZEROS>(s, p, slots, blocks);
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
  const bool zeros = q.m[0].zeros != nullptr;
  const size_t per_slot = q.T * (q.offsets ? q.k : 1) / slots;
  if (per_slot > 16) {
    // workgroups of a slot beyond its tokens end at once; a slot with more
    // tokens than they take goes round again
    const size_t blocks = q.offsets ? std::min<size_t>(2 * per_slot / kTileTokens + 1, 8)
                                    : (q.T + kTileTokens - 1) / kTileTokens;
    const unsigned z = unsigned(std::min<size_t>(blocks, 65535));
    if (q.x.fine) zeros ? run_tiles<true, true>(s, p, q.mats, q.x.P, slots, z)
                        : run_tiles<true, false>(s, p, q.mats, q.x.P, slots, z);
    else zeros ? run_tiles<false, true>(s, p, q.mats, q.x.P, slots, z)
               : run_tiles<false, false>(s, p, q.mats, q.x.P, slots, z);
    INF_LAUNCHED();
    return INFERNO_OK;
  }
  const dim3 grid(unsigned((q.N + 15) / 16), slots);
  const int kind = q.x.P == 1 ? kOne : q.T <= 4 ? kPack3 : kWide3;
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
