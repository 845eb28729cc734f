// Products with 4-bit weights and group scales on the matrix cores.
//
//   y[t, n] = sum_g s[n, g] sum_{c in g} (q[n, c] - z[n, g]) x[t, c]
//
// int8 activations and few tokens: the inner sum is formed exactly. A code is
// widened to 16 (q - 8), an int8, by one mask (its nibble stays in the high half of
// the byte), or to q - z with four codes in one subtraction; an activation is one
// int8 digit (8-bit activations) or three, a 24-bit fixed-point value relative to
// the largest of its 128-column chunk: exact for every bf16 value down to 2^-14 of
// the largest, and off by at most 2^-23 of it for fp32. The int32 sums of a group
// are exact, the groups are added in fp32. Joining three sums is six vector
// instructions a result and chunk, more than their matrix instructions take, so
// many bf16 tokens (and fp32 ones with groups of 32 or 64) go as fp16 instead,
// one plane (two) of values scaled by a power of two for each chunk, against
// codes widened to fp16, q - z whole; a chunk's sums are formed in fp32.
//
// Why fp32 has three digits: with four (off by 2^-31 of the largest) one to four
// tokens take as long, but 16 tokens of 8 of 64 experts with groups of 32 97
// instead of 78 us, 128 and 512 of 10 of 128 experts 454 and 701 instead of 318 and
// 605 (h is fp32), 256 of one matrix 2048 x 6144 115 instead of 94; with two chunks
// ahead as three digits have, the registers do not suffice and it is more.
//
// Tile: 16 weight rows (the 16 columns of a 16x16 MFMA result) by 16 digit
// rows. A lane holds 32 codes of its row per chunk (16 bytes: low nibbles are
// the even columns, high nibbles the odd ones); the packed matrix has the 1 KB
// of a tile's chunk together in the lanes' order. Any order of the columns
// inside a group gives the same sum, so no code moves inside its bytes, and the
// digits are laid out to match.
#include <atomic>
#include <type_traits>

#include "w4.hpp"

namespace inferno {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kMaxDigits = 127 * 65536 + 127 * 256 + 127;  // largest three-digit value

// ------------------------------------------------------------------ digits

struct Stage {
  const void* x;
  const float* x_scales;
  size_t x_group;  // > 0
  size_t R, K, C, xs_stride;
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

// The power of two (its exponent) that takes a chunk whose largest magnitude has
// the bits `most` to three digits: the largest one that fits; chunks below 2^-126,
// fp32's smallest normal value, share their step, 2^-148.
__device__ __forceinline__ int digits_up(uint32_t most) {
  const int up = 22 - max(int(most >> 23) - 127, -126);
  return ldexpf(bits_to_f32(most), up) > float(kMaxDigits) ? up - 1 : up;
}
// A value's three digits in bytes 2, 1, 0, each offset by 128.
__device__ __forceinline__ uint32_t digits_of(float v, int up, bool finite) {
  return uint32_t((finite ? int(rintf(ldexpf(v, up))) : 0) + 0x808080);
}
__device__ __forceinline__ float digits_scale(int up, bool finite) {
  return finite ? ldexpf(1.f, -up) : bits_to_f32(0x7fc00000u);
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
    const int up = digits_up(most);
#pragma unroll
    for (int j = 0; j < 32; ++j) X[j] = digits_of(v[j], up, finite);
    xs = digits_scale(up, finite);
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
  if (b == 0) p.a.xs[r * p.xs_stride + c] = xs;
  if (b == 1 && c + 1 == p.C && p.C < p.xs_stride) p.a.xs[r * p.xs_stride + p.C] = 0.f;
}

// The same as fp16 in PLANES planes: one holds a bf16 value whole (to 2^-31 of its
// chunk's largest), two an fp32 value but for 2^-23 of itself. The chunk's largest
// is taken to [2^14, 2^15). A plane's 256 bytes of a chunk are four pieces of 64,
// one for each dword of a lane's codes; in a piece every 16-lane row of the
// weights' tile has the 8 columns of its dword in the order in which
// Halves::widen gives them.
template <typename XT, int PLANES>
__global__ void __launch_bounds__(256) w4_stage_halves_kernel(Stage p) {
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
  uint32_t most = 0;  // as integers: NaN lies above infinity
#pragma unroll
  for (int j = 0; j < 32; ++j) most = max(most, f32_to_bits(v[j]) & 0x7fffffffu);
  most = max(most, uint32_t(__shfl_xor(int(most), 1, kWave)));
  most = max(most, uint32_t(__shfl_xor(int(most), 2, kWave)));
  const bool finite = most < 0x7f800000u;
  const int up = 14 - max(int(most >> 23) - 127, -126);
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = finite ? ldexpf(v[j], up) : 0.f;
  int8_t* out = p.a.planes + rc * (PLANES * 2 * kW4Chunk);
#pragma unroll
  for (int q = 0; q < PLANES; ++q) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      v8h h;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float& value = v[8 * m + (j % 2) * 4 + j / 2];
        h[j] = _Float16(value);
        value -= float(h[j]);
      }
      // coarse groups: lane row b, dword m; fine ones: lane row m, dword b
      const int piece = p.a.fine ? b : m, row = p.a.fine ? m : b;
      *reinterpret_cast<v8h*>(out + q * 2 * kW4Chunk + piece * 64 + row * 16) = h;
    }
  }
  if (b == 0) p.a.xs[r * p.xs_stride + c] = digits_scale(up, finite);
  if (b == 1 && c + 1 == p.C && p.C < p.xs_stride) p.a.xs[r * p.xs_stride + p.C] = 0.f;
}

// -------------------------------------------------------------------- pack

struct Pack {
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  uint8_t* to;
  size_t scales_at, zeros_at;  // byte offsets in `to`
  uint32_t tiles;              // all experts'
  uint32_t row_tiles, N, K, C, group, groups;
  bool fine;
};

// One tile's chunk, by one wavefront. Rows behind N and columns behind K get the
// code, the scale and the zero point that count nothing.
template <typename ST>
__device__ __forceinline__ void pack_chunk(const Pack& p, size_t tc) {
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const uint32_t tile = uint32_t(tc / p.C), c = uint32_t(tc % p.C);
  const uint32_t row = tile % p.row_tiles * 16 + n;
  const size_t mrow = size_t(tile / p.row_tiles) * p.N + min(row, p.N - 1);
  const uint32_t* src = reinterpret_cast<const uint32_t*>(p.codes + mrow * (p.K / 2));
  v4u v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // coarse groups: block `quad`; fine ones: dword `quad` of every block
    const int block = p.fine ? j : quad, word = p.fine ? quad : j;
    const uint32_t col = c * kW4Chunk + 32 * block;
    const bool in = row < p.N && col < p.K;
    const uint32_t u = src[in ? col / 8 + word : 0];
    v[j] = p.zeros ? (in ? u : 0u) : (in ? u ^ 0x88888888u : 0u);  // q, or q - 8
  }
  *reinterpret_cast<v4u*>(p.to + tc * 1024 + lane * 16) = v;
  // lane (n, quad): the scale of block `quad`, or for coarse groups of all
  if (!p.fine && quad) return;
  const uint32_t col = c * kW4Chunk + 32 * quad;
  const bool in = row < p.N && col < p.K;
  const size_t from = mrow * p.groups + (in ? col / p.group : 0);
  const size_t at = p.fine ? (tc * 16 + n) * 4 + quad : tc * 16 + n;
  const ST s = static_cast<const ST*>(p.scales)[from];
  reinterpret_cast<ST*>(p.to + p.scales_at)[at] = in ? s : ST(0);
  if (p.zeros) p.to[p.zeros_at + at] = in ? uint8_t(min(uint32_t(p.zeros[from]), 127u)) : 0;
}

template <typename ST>
__global__ void __launch_bounds__(256) w4_pack_kernel(Pack p) {
  for (size_t tc = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6); tc < size_t(p.tiles) * p.C;
       tc += size_t(gridDim.x) * 4)
    pack_chunk<ST>(p, tc);
}

// ----------------------------------------------------------------- product

struct Mat {
  const uint8_t* codes;   // [tiles][chunks][64][16]
  const uint8_t* scales;  // [tiles][chunks][16][1 or 4] of the scale type
  const uint8_t* zeros;   // likewise, bytes
};

struct Product {
  Mat m[2];
  uint32_t N, C, row_tiles;  // rows, chunks and row tiles of one expert's matrix
  const int8_t* planes;
  const float* xs;
  uint32_t xs_stride;
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

// The expert of slot y and its assignments, or all tokens; false: none. Uniform
// values.
struct Slot {
  uint32_t expert, first, end;
};
__device__ __forceinline__ bool slot_of(const Product& p, uint32_t y, Slot& s) {
  s = Slot{0, 0, p.T};
  if (!p.offsets) return true;
  if (y >= p.active[0]) return false;
  s.expert = __builtin_amdgcn_readfirstlane(p.active[1 + y]);
  s.first = __builtin_amdgcn_readfirstlane(p.offsets[s.expert]);
  s.end = __builtin_amdgcn_readfirstlane(p.offsets[s.expert + 1]);
  return true;
}

// Activation row of assignment (or token) i of a slot; the last one's behind it.
__device__ __forceinline__ size_t x_row(const Product& p, const Slot& s, uint32_t i) {
  const uint32_t j = min(i, s.end - 1);
  if (!p.offsets) return j;
  const uint32_t a = p.sorted[j];
  return p.x_by_assignment ? a : a / p.k;
}

__device__ __forceinline__ void store_result(const Product& p, uint32_t j, uint32_t row, float g,
                                             const float* u) {
  const size_t a = p.offsets ? p.sorted[j] : j;
  float y = u ? g / (1.f + expf(-g)) * *u : g;
  if (p.route_w) y *= p.route_w[a];
  const size_t at = a * p.N + row;
  if (p.res_a) y += p.res_a[at];
  if (p.res_b) y += p.res_b[at];
  p.out[at] = y;
}

// A lane's codes of a chunk as operands of the matrix instructions: for coarse
// groups the even columns, then the odd ones; for fine groups both of each block
// in one pair of registers.
template <bool FINE>
struct Wide {
  v4i half[2];
  __device__ __forceinline__ void put(int j, uint32_t even, uint32_t odd) {
    half[0][j] = int(even);
    half[1][j] = int(odd);
  }
};
template <>
struct Wide<true> {
  long block[4];
  __device__ __forceinline__ void put(int j, uint32_t even, uint32_t odd) {
    block[j] = long(uint64_t(odd) << 32 | even);
  }
};

// The same as fp16: q - 8 or q - z, one register quadruple for each dword of
// codes, whose columns come in the order 0 4 1 5 2 6 3 7. The widening is the
// well-known one by the exponent: 0x6400 with a code in its low bits is 1024 + q,
// with a code four bits up 1024 + 16 q.
struct Halves {
  v4u dword[4];

  template <bool FINE, bool ZEROS>
  __device__ __forceinline__ void widen(const v4u& q, uint32_t z) {
    const v2h sixteenth = {_Float16(0.0625f), _Float16(0.0625f)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v2h low = {_Float16(-1032.f), _Float16(-1032.f)}, high = {_Float16(-72.f), _Float16(-72.f)};
      if (ZEROS) {  // (1024 + z) with the sign bit, and 960 less
        const uint32_t zz = FINE ? (z >> (8 * j)) & 255u : z;
        low = __builtin_bit_cast(v2h, zz * 0x00010001u | 0xe400e400u);
        high = low + v2h{_Float16(960.f), _Float16(960.f)};
      }
      uint32_t u = ZEROS ? q[j] : q[j] ^ 0x88888888u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const v2h a = __builtin_bit_cast(v2h, (u & 0x000f000fu) | 0x64006400u);
        const v2h b = __builtin_bit_cast(v2h, (u & 0x00f000f0u) | 0x64006400u);
        dword[j][2 * i] = __builtin_bit_cast(uint32_t, a + low);
        dword[j][2 * i + 1] =
            __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, sixteenth, high));
        u >>= 8;
      }
    }
  }
};

// One chunk of one weight tile on its way: codes, and the scales and zero
// points of this lane's row (of its four blocks for fine groups).
template <bool FINE, bool ZEROS, typename ST>
struct Codes {
  static constexpr int B = FINE ? 4 : 1;
  typedef ST SV __attribute__((ext_vector_type(B)));
  v4u q;
  SV s;
  uint32_t z;

  // tc: the tile's chunk
  __device__ __forceinline__ void load(const Mat& m, size_t tc, int lane) {
    q = reinterpret_cast<const v4u*>(m.codes)[tc * 64 + lane];
    s = reinterpret_cast<const SV*>(m.scales)[tc * 16 + (lane & 15)];
    if (ZEROS) {
      if (FINE) z = reinterpret_cast<const uint32_t*>(m.zeros)[tc * 16 + (lane & 15)];
      else z = m.zeros[tc * 16 + (lane & 15)];
    }
  }
  // Even and odd columns as int8: 16 (q - 8), or q - z with zero points (z is at
  // most 127: no byte borrows from the next).
  __device__ __forceinline__ void widen(Wide<FINE>& w) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t even, odd;
      if (ZEROS) {
        const uint32_t zz = (FINE ? (z >> (8 * j)) & 255u : z) * 0x01010101u;
        even = (((q[j] & 0x0f0f0f0fu) | 0x80808080u) - zz) ^ 0x80808080u;
        odd = ((((q[j] >> 4) & 0x0f0f0f0fu) | 0x80808080u) - zz) ^ 0x80808080u;
      } else {
        even = (q[j] << 4) & 0xf0f0f0f0u;
        odd = q[j] & 0xf0f0f0f0u;
      }
      w.put(j, even, odd);
    }
  }
  __device__ __forceinline__ void widen(Halves& w) const { w.template widen<FINE, ZEROS>(q, z); }
  // Scale of block b; 0 for a chunk that is not `there`.
  __device__ __forceinline__ float plain_scale(int b, bool there) const {
    float v;
    if constexpr (sizeof(ST) == 2) v = bf16_bits_to_f32(s[b]);
    else v = s[b];
    return there ? v : 0.f;
  }
  // The same for the int8 values of widen.
  __device__ __forceinline__ float scale(int b, bool there) const {
    return plain_scale(b, there) * (ZEROS ? 1.f : 0.0625f);
  }
};

// Sums of one chunk's block b: 16 digit rows (the two halves x0, x1 of a plane)
// by 16 weight rows.
template <bool FINE>
__device__ __forceinline__ v4i dot(const v4u& x0, const v4u& x1, const Wide<FINE>& w, int b) {
  v4i s = {0, 0, 0, 0};
  if constexpr (FINE) {
    const v4u& u = b < 2 ? x0 : x1;
    const long x = long(uint64_t(u[2 * (b % 2) + 1]) << 32 | u[2 * (b % 2)]);
    return __builtin_amdgcn_mfma_i32_16x16x32_i8(x, w.block[b], s, 0, 0, 0);
  } else {
    s = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, x0), w.half[0], s, 0, 0, 0);
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(v4i, x1), w.half[1], s, 0, 0,
                                                 0);
  }
}

// Sum of a token's digits' sums as a float; a sum is at most 2^21.
__device__ __forceinline__ float join(int hi, int mid, int lo) {
  return fmaf(float((hi << 8) + mid), 256.f, float(lo));
}

// Token tiles of the rows kernel. kPack3 holds a token's three digits in rows
// 4 t, 4 t + 1, 4 t + 2 of one 16x16 result (one lane then has all three sums of
// a token); kOne and kWide3 hold 16 tokens, kWide3 in three results, one per
// digit.
enum Kind { kPack3, kOne, kWide3 };

// Few tokens. A wavefront takes RT tiles of 16 rows of the matrices (the same
// rows of both) and all tokens of one expert (or of the batch) in tiles. `split`
// wavefronts share the chunks of these rows and add their sums in order; a
// workgroup's four cover 4 RT / split tiles.
template <bool FINE, int MATS, int P, bool ZEROS, typename ST, int RT>
__global__ void __launch_bounds__(256) w4_rows_kernel(Product p, int split) {
  constexpr int B = FINE ? 4 : 1, F = MATS * RT;
  __shared__ float part[4][F * 4][kWave];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  Slot slot;
  if (!slot_of(p, blockIdx.y, slot)) return;
  const uint32_t end = slot.end;
  const uint32_t tile0 = (blockIdx.x * (4 / split) + wave / split) * RT;
  size_t tile[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    tile[i] = (size_t(slot.expert) * p.row_tiles + min(tile0 + i, p.row_tiles - 1)) * p.C;
  // chunks in pairs
  const uint32_t pairs = (p.C + 1) / 2, share = wave % split;
  const uint32_t c0 = pairs * share / split * 2, c1 = pairs * (share + 1) / split * 2;
  uint32_t t0 = slot.first;
  auto run = [&](auto kind) __attribute__((always_inline)) {
    constexpr int KIND = decltype(kind)::value;
    constexpr int NT = KIND == kWide3 ? 3 : 1;   // results
    constexpr int NV = KIND == kPack3 ? 1 : 4;   // tokens per lane
    // this lane's operand row, and the tokens whose sums it gets
    const int8_t* xp = p.planes + x_row(p, slot, t0 + (KIND == kPack3 ? n / 4 : n)) * p.C *
                                      (P * kW4Chunk) +
                       (KIND == kPack3 ? min(n & 3, 2) * kW4Chunk : 0) + quad * 16;
    const float* sp[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
      sp[i] = p.xs + x_row(p, slot, t0 + (KIND == kPack3 ? quad : 4 * quad + i)) * p.xs_stride;
    float acc[F][NV];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[f][i] = 0.f;
    // loads on their way, of two chunks
    Codes<FINE, ZEROS, ST> w[2][F];
    v4u x[2][NT][2];
    float2 xs[NV], next_xs[NV];
    auto load = [&](uint32_t chunk, int to) {
      const uint32_t c = min(chunk, p.C - 1);
#pragma unroll
      for (int f = 0; f < F; ++f) w[to][f].load(p.m[f / RT], tile[f % RT] + c, lane);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const v4u* at =
            reinterpret_cast<const v4u*>(xp + size_t(c) * (P * kW4Chunk) + t * kW4Chunk);
        x[to][t][0] = at[0];
        x[to][t][1] = at[4];
      }
    };
    auto load_xs = [&](uint32_t pair_at) {
      const uint32_t c = min(pair_at, 2 * pairs - 2);
#pragma unroll
      for (int i = 0; i < NV; ++i) next_xs[i] = *reinterpret_cast<const float2*>(sp[i] + c);
    };
    auto step = [&](uint32_t c, int cur) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        Wide<FINE> wide;
        w[cur][f].widen(wide);
        float value[NV];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          v4i sum[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            sum[t] = dot<FINE>(x[cur][t][0], x[cur][t][1], wide, b);
          const float ws = w[cur][f].scale(b, c < p.C);
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            float v;
            if (KIND == kPack3) v = join(sum[0][0], sum[0][1], sum[0][2]);
            else if (KIND == kOne) v = float(sum[0][i]);
            else v = join(sum[0][i], sum[NT / 2][i], sum[NT - 1][i]);
            value[i] = b == 0 ? ws * v : fmaf(ws, v, value[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
          acc[f][i] = fmaf(value[i], cur ? xs[i].y : xs[i].x, acc[f][i]);
      }
      load(c + 2, cur);
    };
    if (c0 < c1) {
      load_xs(c0);
      load(c0, 0);
      load(c0 + 1, 1);
      // two at a time without a way past the second (a chunk behind the end has
      // scales of 0): the wait counts of a loop hold for its shortest path
      for (uint32_t c = c0; c < c1; c += 2) {
#pragma unroll
        for (int i = 0; i < NV; ++i) xs[i] = next_xs[i];
        load_xs(c + 2);
        step(c, 0);
        step(c + 1, 1);
      }
    }
    const uint32_t j0 = t0 + (KIND == kPack3 ? quad : 4 * quad);
    t0 += KIND == kPack3 ? 4 : 16;
    if (split == 1) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const uint32_t row = (tile0 + r) * 16 + n;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (row < p.N && j0 + i < end)
            store_result(p, j0 + i, row, acc[r][i],
                         MATS == 2 ? &acc[(MATS - 1) * RT + r][i] : nullptr);
      }
      return;
    }
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int i = 0; i < NV; ++i) part[wave][f * NV + i][lane] = acc[f][i];
    __syncthreads();
    // the wavefronts of a tile write the token values in turn
    for (int v = int(share); v < RT * NV; v += split) {
      const int r = v / NV, i = v % NV;
      const uint32_t row = (tile0 + r) * 16 + n;
      if (row >= p.N || j0 + i >= end) continue;
      float y[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        const int f = m * RT + r;
        y[m] = part[wave - share][f * NV + i][lane];
        for (int k = 1; k < split; ++k) y[m] += part[wave - share + k][f * NV + i][lane];
      }
      store_result(p, j0 + i, row, y[0], MATS == 2 ? &y[MATS - 1] : nullptr);
    }
    __syncthreads();  // before the next tokens' sums
  };
  while (t0 < end) {
    if constexpr (P == 1) {
      run(std::integral_constant<int, kOne>{});
    } else {
      if (end - t0 <= 4) run(std::integral_constant<int, kPack3>{});
      else run(std::integral_constant<int, kWide3>{});
    }
  }
}

// One to four tokens, without other launches: a workgroup forms the digits of the
// tokens by itself, in LDS, while its first weights are on their way, and takes
// 16 rows of the matrices (the same rows of both). `segments` matrices follow
// each other along the chunks (one token's experts for the sum over its ranks;
// else one), which the workgroup's wavefronts share. Their sums are added in
// order.
struct Tokens {
  Product p;
  const void* x;      // [T or segments, K]
  uint32_t K, segments;
  bool sum;             // over the segments
  const uint32_t* ids;  // experts: of blockIdx.y, or of the segments; null: one matrix
  uint32_t E;
};

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 f = reinterpret_cast<const float4*>(p)[i];
    v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
  }
}
__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = bits_to_f32(w[j] << 16);
    v[2 * j + 1] = bits_to_f32(w[j] & 0xffff0000u);
  }
}

// Bytes of LDS: digits and scales of all chunks, and the wavefronts' sums.
inline size_t token_lds(size_t rows, size_t chunks, int mats, int waves) {
  return rows * chunks * (3 * kW4Chunk + 4) + size_t(waves) * mats * kWave * 4 + 16;
}

template <bool FINE, int MATS, bool ZEROS, typename ST, typename XT, int WAVES>
__global__ void __launch_bounds__(WAVES* kWave) w4_token_kernel(Tokens a) {
  constexpr int B = FINE ? 4 : 1;
  extern __shared__ __align__(16) int8_t token_shared[];
  const Product& p = a.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const bool sum = a.sum;
  const uint32_t T = sum ? 1 : p.T, rows = sum ? a.segments : T;
  const uint32_t total = a.segments * p.C;             // chunks
  int8_t* digits = token_shared;                       // [total][T][3][128]
  float* xs = reinterpret_cast<float*>(digits + size_t(total) * T * (3 * kW4Chunk));  // [total][T]
  float* part = xs + size_t(total) * T;                // [WAVES][MATS][64]
  uint32_t expert = 0;
  if (a.ids && !sum) {
    expert = __builtin_amdgcn_readfirstlane(a.ids[blockIdx.y]);
    if (expert >= a.E) return;  // the same for the workgroup
  }
  const uint32_t pairs = (total + 1) / 2;
  const uint32_t c0 = pairs * wave / WAVES * 2, c1 = pairs * (wave + 1) / WAVES * 2;
  const uint32_t my_id = sum && uint32_t(lane) < a.segments ? a.ids[lane] : 0u;
  Codes<FINE, ZEROS, ST> w[2][MATS];
  bool there[2];
  auto load = [&](uint32_t chunk, int to) {
    const uint32_t cc = min(chunk, total - 1);
    uint32_t e = expert, c = cc;
    there[to] = chunk < total;
    if (sum) {
      const uint32_t r = cc / p.C;
      c = cc - r * p.C;
      e = __builtin_amdgcn_readlane(my_id, r);
      there[to] = there[to] && e < a.E;
      e = e < a.E ? e : 0;  // an id of no expert: any weights, with scales of 0
    }
    const size_t at = (size_t(e) * p.row_tiles + blockIdx.x) * p.C + c;
#pragma unroll
    for (int m = 0; m < MATS; ++m) w[to][m].load(p.m[m], at, lane);
  };
  if (c0 < c1) {
    load(c0, 0);
    load(c0 + 1, 1);
  }
  // eight columns per thread; 16 neighbouring threads share a chunk's largest
  // value. Columns behind K are digits of 0.
  for (uint32_t i = threadIdx.x; i < rows * p.C * 16; i += WAVES * kWave) {
    const uint32_t row = i / (p.C * 16), in_row = i - row * (p.C * 16), c = in_row / 16;
    const uint32_t col = in_row * 8, b = in_row / 4 % 4, e = in_row % 4;  // block, eighth
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // (no row was written for an id of no expert)
    if (col < a.K && !(sum && a.ids[row] >= a.E))
      load8(static_cast<const XT*>(a.x) + size_t(row) * a.K + col, v);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, f32_to_bits(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) most = max(most, uint32_t(__shfl_xor(int(most), m, kWave)));
    const bool finite = most < 0x7f800000u;
    const int up = digits_up(most);
    uint32_t X[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) X[j] = digits_of(v[j], up, finite);
    const uint32_t at = sum ? row * p.C + c : c * T + row;
    int8_t* out = digits + size_t(at) * (3 * kW4Chunk);
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const uint32_t even = gather4(X[0], X[2], X[4], X[6], 2 - q) ^ 0x80808080u;
      const uint32_t odd = gather4(X[1], X[3], X[5], X[7], 2 - q) ^ 0x80808080u;
      int8_t* plane = out + q * kW4Chunk;
      if (FINE) {
        *reinterpret_cast<uint2*>(plane + (b / 2) * 64 + e * 16 + (b % 2) * 8) =
            make_uint2(even, odd);
      } else {
        *reinterpret_cast<uint32_t*>(plane + b * 16 + e * 4) = even;
        *reinterpret_cast<uint32_t*>(plane + 64 + b * 16 + e * 4) = odd;
      }
    }
    if (in_row % 16 == 0) xs[at] = digits_scale(up, finite);
  }
  __syncthreads();
  float acc[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) acc[m] = 0.f;
  const uint32_t mine = min(uint32_t(n / 4), T - 1), his = min(uint32_t(quad), T - 1);
  const int8_t* xp = digits + (mine * 3 + min(n & 3, 2)) * kW4Chunk + quad * 16;
  auto step = [&](uint32_t chunk, int cur) {
    const uint32_t cc = min(chunk, total - 1);
    const v4u* at = reinterpret_cast<const v4u*>(xp + size_t(cc) * T * (3 * kW4Chunk));
    const v4u x0 = at[0], x1 = at[4];
    const float scale = xs[cc * T + his];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
      Wide<FINE> wide;
      w[cur][m].widen(wide);
      float value = 0.f;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const v4i u = dot<FINE>(x0, x1, wide, b);
        value = fmaf(w[cur][m].scale(b, there[cur]), join(u[0], u[1], u[2]), value);
      }
      acc[m] = fmaf(value, scale, acc[m]);
    }
    load(chunk + 2, cur);
  };
  for (uint32_t c = c0; c < c1; c += 2) {
    step(c, 0);
    step(c + 1, 1);
  }
#pragma unroll
  for (int m = 0; m < MATS; ++m) part[(wave * MATS + m) * kWave + lane] = acc[m];
  __syncthreads();
  const uint32_t row = blockIdx.x * 16 + n;
  if (wave || uint32_t(quad) >= T || row >= p.N) return;
  float y[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    y[m] = part[m * kWave + lane];
    for (int k = 1; k < WAVES; ++k) y[m] += part[(k * MATS + m) * kWave + lane];
  }
  const uint32_t j = a.ids && !sum ? blockIdx.y : uint32_t(quad);
  store_result(p, j, row, y[0], MATS == 2 ? &y[MATS - 1] : nullptr);
}

// Many tokens. One workgroup: 64 tokens by 128 RT / KS rows of the matrices; a
// wavefront takes RT tiles of 16 rows of each matrix against all tokens, and one
// of KS shares of the chunks (a step of one chunk costs a workgroup 0.5 us or more
// whatever it holds; one of four shares at once, 256 int8 tokens of a pair 2048 x
// 6144, 2.7 us). The weights go from memory to the wavefront that owns them; the
// tokens' values go through LDS (two buffers of one chunk) in the order in which the matrix
// instructions' lanes read them, so that a read is 1 KB without bank conflicts.
// Both are two chunks ahead in registers, since a chunk's loads take longer
// than its arithmetic (copies to LDS that bypass registers would have to be
// complete before any LDS read). Tiles of 16 tokens that an expert does not
// have are left out; a tile's pieces are read while the one before is in use,
// where they fit the registers.
// What bounds it: one workgroup per CU (170 to 256 registers), whose loads,
// reads from LDS and arithmetic overlap only in part. 512 bf16 tokens of 10 of
// 128 experts, gate and up 1536 x 4096: 344 to 352 us (by card) for 0.82 GB of
// weights (2.3 TB/s), three digits 418; down, three digits: 246 to 261 us. 64 int8
// tokens, gate and up: 147 to 150 us (5.6 TB/s with the caches' help). One matrix
// pair 2048 x 6144, 256 tokens: int8 36, bf16 56 us, three digits 84.
constexpr int kTileTokens = 64;
constexpr int kTileWaves = 8;

template <bool FINE, int MATS, bool HALF, int P, bool ZEROS, typename ST, int RT, int KS>
__global__ void __launch_bounds__(kTileWaves* kWave, 2) w4_tile_kernel(Product p) {
  constexpr int F = MATS * RT, TT = kTileTokens / 16, B = FINE ? 4 : 1;
  constexpr int RW = kTileWaves / KS;  // wavefronts of a share
  constexpr int PC = HALF ? 4 * P : 2 * P;  // pieces of 64 bytes of a token's chunk
  // chunks that loads are ahead; with two, fine groups of fp16 go through scratch
  // memory (64 tokens, groups of 32: 95 us, with one 74)
  constexpr int LOOK = FINE && HALF ? 1 : 2;
  constexpr int XB = PC <= 4 ? 2 : 1;  // token tiles whose pieces are in registers
  struct Chunks {
    int8_t x[2][TT][PC][kWave * 16];
    float s[2][kTileTokens];
  };
  __shared__ __align__(16) union {
    Chunks chunks[KS];
    float part[kTileWaves][F * 4][kWave];  // sums of one token tile
  } lds;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  Slot slot;
  // A routed product has eight slots in a row of workgroups, so that those of one
  // expert (neighbours but seven) share the L2 of one XCD, which then takes the
  // expert's tokens from memory once (gate and up of 512 tokens 380 -> 362 us
  // with the next tile's reads ahead).
  const uint32_t block = p.offsets ? blockIdx.x / 8 : blockIdx.x;
  if (!slot_of(p, blockIdx.y * 8 + blockIdx.x % 8, slot)) return;
  const uint32_t end = slot.end;
  // this wavefront's row tiles; those behind the last are the last one again
  const int share = wave / RW;
  const uint32_t tile0 = (block * RW + wave % RW) * RT;
  size_t tile[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
    tile[r] = (size_t(slot.expert) * p.row_tiles + min(tile0 + r, p.row_tiles - 1)) * p.C;
  auto& xt = lds.chunks[share].x;
  auto& xst = lds.chunks[share].s;
  // this share's chunks, in pairs; every share takes as many steps
  const uint32_t pairs = (p.C + 1) / 2, steps = (pairs + KS - 1) / KS * 2;
  const uint32_t c0 = pairs * share / KS * 2, c1 = min(pairs * (share + 1) / KS * 2, p.C);
  for (uint32_t t0 = slot.first + blockIdx.z * kTileTokens; t0 < end;
       t0 += gridDim.z * kTileTokens) {
    const uint32_t tokens = min(end - t0, uint32_t(kTileTokens));
    auto run = [&](auto token_tiles) __attribute__((always_inline)) {
      constexpr int NT = decltype(token_tiles)::value;
      // a share's wavefronts bring the digits of its chunks: RW / 4 of them those
      // of a token tile (or one those of 4 / RW tiles), the first its scales
      constexpr int kPieces = RW >= 4 ? 4 * PC / RW : PC, kBring = RW >= 4 ? 1 : 4 / RW;
      const int cw = wave % RW, ct0 = RW >= 4 ? cw * 4 / RW : cw * kBring;
      const int cp = RW >= 4 ? cw * kPieces % PC : 0;
      const int8_t* xp[kBring];
      const float* sp[kBring];
      bool brings[kBring];
#pragma unroll
      for (int i = 0; i < kBring; ++i) {
        const size_t xr = x_row(p, slot, t0 + 16 * (ct0 + i) + n);
        xp[i] = p.planes + xr * p.C * (PC * 64) + cp * 64 + quad * 16;
        sp[i] = p.xs + xr * p.xs_stride;
        brings[i] = 16u * (ct0 + i) < tokens;
      }
      float acc[F][NT][4];
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[f][t][i] = 0.f;
      // Loads on their way, of even and odd chunks. A chunk behind the end is the
      // last one again.
      Codes<FINE, ZEROS, ST> w[LOOK][F];
      v4u digits[LOOK][kBring][kPieces];
      float digit_s[LOOK][kBring];
      auto load_digits = [&](uint32_t chunk, int to) {
        const uint32_t c = min(chunk, p.C - 1);
#pragma unroll
        for (int k = 0; k < kBring; ++k)
          if (brings[k]) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
              digits[to][k][i] =
                  *reinterpret_cast<const v4u*>(xp[k] + size_t(c) * (PC * 64) + i * 64);
            digit_s[to][k] = sp[k][c];
          }
      };
      auto store_digits = [&](uint32_t c, int from) {
#pragma unroll
        for (int k = 0; k < kBring; ++k)
          if (brings[k]) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
              *reinterpret_cast<v4u*>(&xt[c & 1][ct0 + k][cp + i][lane * 16]) = digits[from][k][i];
            if (cp == 0 && lane < 16) xst[c & 1][16 * (ct0 + k) + n] = digit_s[from][k];
          }
      };
      auto load_codes = [&](uint32_t chunk, int to) {
        const uint32_t c = min(chunk, p.C - 1);
#pragma unroll
        for (int f = 0; f < F; ++f) w[to][f].load(p.m[f / RT], tile[f % RT] + c, lane);
      };
      auto step = [&](uint32_t c, int cur) {
        // everybody has stored chunk c, and has read chunk c - 1
        __syncthreads();
        const int next = LOOK == 2 ? cur ^ 1 : 0;
        store_digits(c + 1, next);
        load_digits(c + 1 + LOOK, next);
        std::conditional_t<HALF, Halves, Wide<FINE>> wide[F];
        float ws[F][B];
#pragma unroll
        for (int f = 0; f < F; ++f) {
          w[cur][f].widen(wide[f]);
#pragma unroll
          for (int b = 0; b < B; ++b) ws[f][b] = HALF ? w[cur][f].plain_scale(b, c < c1) : w[cur][f].scale(b, c < c1);
        }
        load_codes(c + LOOK, cur);
        v4u x[XB][PC];
        auto read = [&](int t) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < PC; ++i)
            x[t % XB][i] = *reinterpret_cast<const v4u*>(&xt[c & 1][t][i][lane * 16]);
        };
        if (XB == 2) read(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (XB == 1) read(t);
          else if (t + 1 < NT) read(t + 1);
          const float4 s4 = *reinterpret_cast<const float4*>(&xst[c & 1][16 * t + 4 * quad]);
          const float xs[4] = {s4.x, s4.y, s4.z, s4.w};
          const v4u(&held)[PC] = x[t % XB];
#pragma unroll
          for (int f = 0; f < F; ++f) {
            float value[4];
#pragma unroll
            for (int b = 0; b < B; ++b) {
              float sum[4];
              if constexpr (HALF) {
                v4f u = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int d = FINE ? b : 0; d < (FINE ? b + 1 : 4); ++d)
#pragma unroll
                  for (int q = 0; q < P; ++q)
                    u = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(v8h, held[4 * q + d]),
                        __builtin_bit_cast(v8h, wide[f].dword[d]), u, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = u[i];
              } else {
                v4i u[P];
#pragma unroll
                for (int q = 0; q < P; ++q)
                  u[q] = dot<FINE>(held[2 * q], held[2 * q + 1], wide[f], b);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  sum[i] = P == 3 ? join(u[0][i], u[P / 2][i], u[P - 1][i]) : float(u[0][i]);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                value[i] = b == 0 ? ws[f][b] * sum[i] : fmaf(ws[f][b], sum[i], value[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[f][t][i] = fmaf(value[i], xs[i], acc[f][t][i]);
            if (FINE) __builtin_amdgcn_sched_barrier(0);  // (registers)
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      // (c0 is even)
      load_digits(c0, 0);
      if (LOOK == 2) load_digits(c0 + 1, LOOK - 1);
      load_codes(c0, 0);
      if (LOOK == 2) load_codes(c0 + 1, LOOK - 1);
      store_digits(c0, 0);
      load_digits(c0 + LOOK, 0);
      // two at a time without a way past the second (a chunk behind the end has
      // scales of 0): the wait counts of a loop hold for its shortest path
#pragma unroll 1
      for (uint32_t c = c0; c < c0 + steps; c += LOOK) {
        step(c, 0);
        if (LOOK == 2) step(c + 1, LOOK - 1);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (KS > 1) {
          // the shares write the sums of the token tiles in turn
          __syncthreads();
#pragma unroll
          for (int f = 0; f < F; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) lds.part[wave][f * 4 + i][lane] = acc[f][t][i];
          __syncthreads();
          if (share != t % KS) continue;
#pragma unroll
          for (int f = 0; f < F; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = lds.part[wave % RW][f * 4 + i][lane];
#pragma unroll
              for (int k = 1; k < KS; ++k) v += lds.part[k * RW + wave % RW][f * 4 + i][lane];
              acc[f][t][i] = v;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t j = t0 + 16 * t + 4 * quad + i;
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint32_t row = (tile0 + r) * 16 + n;
            if (j < end && row < p.N)
              store_result(p, j, row, acc[r][t][i],
                           MATS == 2 ? &acc[(MATS - 1) * RT + r][t][i] : nullptr);
          }
        }
      }
    };
    // a loop for each number of token tiles: a branch for each tile inside one
    // loop takes twice the registers
    if (tokens > 48) run(std::integral_constant<int, 4>{});
    else if (tokens > 32) run(std::integral_constant<int, 3>{});
    else if (tokens > 16) run(std::integral_constant<int, 2>{});
    else run(std::integral_constant<int, 1>{});
    __syncthreads();  // the last chunk is read: the next tokens' first may come
  }
}

// Calls f with the instance's constants: (fine groups, matrices, zero points,
// scale type) as values of integral_constant and a scale.
template <typename Fn>
void by_format(const W4Product& q, Fn f) {
  auto scale = [&](auto fine, auto mats, auto zeros) {
    q.m[0].scale_dtype == INFERNO_BF16 ? f(fine, mats, zeros, uint16_t{})
                                       : f(fine, mats, zeros, 0.f);
  };
  auto zero = [&](auto fine, auto mats) {
    q.m[0].zeros ? scale(fine, mats, std::true_type{}) : scale(fine, mats, std::false_type{});
  };
  auto mat = [&](auto fine) {
    q.mats == 2 ? zero(fine, std::integral_constant<int, 2>{})
                : zero(fine, std::integral_constant<int, 1>{});
  };
  q.m[0].fine() ? mat(std::true_type{}) : mat(std::false_type{});
}

// ----------------------------------------------------------------- combine

// Rows of a token's assignments, added in the order of its ranks; those of no
// expert are left out (they were never written). Each thread takes VEC columns
// and has the rows of four ranks on their way: 512 tokens of 4096 columns and 10
// ranks 16 us, one column and one row at a time 41 us (the 84 MB are still in the
// last-level cache).
template <int VEC>
__global__ void __launch_bounds__(256)
    w4_combine_kernel(const float* __restrict__ y, const uint32_t* __restrict__ ids, size_t T,
                      uint32_t H, uint32_t k, uint32_t E, float* __restrict__ out) {
  typedef float Vec __attribute__((ext_vector_type(VEC)));
  const uint32_t h = (blockIdx.x * 256 + threadIdx.x) * VEC;
  if (h >= H) return;
  for (size_t t = blockIdx.y; t < T; t += gridDim.y) {
    Vec sum = 0.f;
    for (uint32_t r = 0; r < k; r += 4) {
      Vec v[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const size_t a = t * k + r + i;
        v[i] = 0.f;
        if (r + i < k && ids[a] < E) v[i] = *reinterpret_cast<const Vec*>(y + a * H + h);
      }
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sum += v[i];
    }
    *reinterpret_cast<Vec*>(out + t * H + h) = sum;
  }
}

}  // namespace

int launch_w4_stage(hipStream_t s, const void* x, int x_dtype, const float* x_scales,
                    size_t x_group, size_t R, size_t K, const W4Acts& a) {
  const Stage p{x, x_scales, x_group ? x_group : K, R, K, w4_chunks(K), w4_xs_stride(K), a};
  const unsigned grid = unsigned((R * p.C * 4 + 255) / 256);
  if (a.halves == 2) w4_stage_halves_kernel<float, 2><<<grid, 256, 0, s>>>(p);
  else if (a.halves == 1) w4_stage_halves_kernel<uint16_t, 1><<<grid, 256, 0, s>>>(p);
  else if (x_dtype == INFERNO_F32) w4_stage_kernel<float, 3><<<grid, 256, 0, s>>>(p);
  else if (x_dtype == INFERNO_BF16) w4_stage_kernel<uint16_t, 3><<<grid, 256, 0, s>>>(p);
  else w4_stage_kernel<int8_t, 1><<<grid, 256, 0, s>>>(p);
  INF_LAUNCHED();
  return INFERNO_OK;
}

W4Layout w4_layout(const W4Mat& m) {
  const size_t per = m.fine() ? 4 : 1;
  const size_t tc = m.experts * ((m.rows + 15) / 16) * w4_chunks(m.cols);
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  W4Layout l;
  l.scales = up(tc * 1024);
  l.zeros = l.scales + up(tc * 16 * per * (m.scale_dtype == INFERNO_BF16 ? 2 : 4));
  l.bytes = l.zeros + (m.zeros ? up(tc * 16 * per) : 0);
  return l;
}

int launch_w4_pack(hipStream_t s, const W4Mat& m, const void* codes, const void* scales,
                   const void* zeros, void* packed) {
  const W4Layout l = w4_layout(m);
  Pack p{};
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = scales;
  p.zeros = static_cast<const uint8_t*>(zeros);
  p.to = static_cast<uint8_t*>(packed);
  p.scales_at = l.scales;
  p.zeros_at = l.zeros;
  p.row_tiles = uint32_t((m.rows + 15) / 16);
  p.tiles = uint32_t(m.experts * p.row_tiles);
  p.N = uint32_t(m.rows);
  p.K = uint32_t(m.cols);
  p.C = uint32_t(w4_chunks(m.cols));
  p.group = uint32_t(m.group);
  p.groups = uint32_t(m.cols / m.group);
  p.fine = m.fine();
  const unsigned grid = unsigned(std::min((size_t(p.tiles) * p.C + 3) / 4, size_t(1) << 22));
  if (m.scale_dtype == INFERNO_BF16) w4_pack_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
  else w4_pack_kernel<float><<<grid, 256, 0, s>>>(p);
  INF_LAUNCHED();
  return INFERNO_OK;
}

bool w4_by_tiles(size_t T, size_t k, size_t experts) {
  // Measured: the tile kernel's step costs the same for 1 to 16 tokens. One expert
  // of 16 tokens: rows 12.3 and 21.5 (one and three planes), tiles 14.3 and 32.5
  // us. Routed, where the tile kernel reads an expert's weights once for all its
  // tokens: 64 experts of 3 tokens each rows 92, tiles 96 us, of 4 rows 104, tiles
  // 96; 128 of 3 rows 268, tiles 277, of 5 rows 294, tiles 282, of 15 rows 509,
  // tiles 380.
  return k ? T * k / std::min(experts, T * k) > 3 : T > 16;
}

int launch_w4_product(hipStream_t s, const W4Product& q) {
  Product p{};
  for (int m = 0; m < q.mats; ++m) {
    const W4Layout l = w4_layout(q.m[m]);
    const uint8_t* at = static_cast<const uint8_t*>(q.m[m].packed);
    p.m[m] = Mat{at, at + l.scales, at + l.zeros};
  }
  p.N = uint32_t(q.m[0].rows);
  p.C = uint32_t(w4_chunks(q.m[0].cols));
  p.row_tiles = (p.N + 15) / 16;
  p.planes = q.x.planes;
  p.xs = q.x.xs;
  p.xs_stride = uint32_t(w4_xs_stride(q.m[0].cols));
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
  const unsigned slots = q.offsets ? unsigned(std::min(q.m[0].experts, q.T * q.k)) : 1u;
  const size_t per_slot = q.T * (q.offsets ? q.k : 1) / slots;
  const bool one = q.x.P == 1;
  const bool tile = w4_by_tiles(q.T, q.offsets ? q.k : 0, q.m[0].experts);
  if (tile) {
    // workgroups of a slot beyond its tokens end at once; a slot with more
    // tokens than they take goes round again
    const size_t blocks = q.offsets ? std::min<size_t>(2 * per_slot / kTileTokens + 1, 8)
                                    : (q.T + kTileTokens - 1) / kTileTokens;
    by_format(q, [&](auto fine, auto mats, auto zeros, auto st) {
      constexpr int M = decltype(mats)::value, RT = M == 2 ? 1 : 2;
      using ST = decltype(st);
      auto go = [&](auto half, auto planes, auto shares) {
        constexpr int P = decltype(planes)::value, KS = decltype(shares)::value;
        constexpr unsigned tiles = RT * kTileWaves / KS;
        const unsigned row_blocks = (p.row_tiles + tiles - 1) / tiles;
        const dim3 grid(q.offsets ? row_blocks * 8 : row_blocks, (slots + 7) / 8,
                        unsigned(std::min<size_t>(blocks, 65535)));
        w4_tile_kernel<fine.value, M, half.value, P, zeros.value, ST, RT, KS>
            <<<grid, kTileWaves * kWave, 0, s>>>(p);
      };
      // shares of the chunks until there is a workgroup for every CU
      const size_t groups =
          (p.row_tiles + RT * kTileWaves - 1) / (RT * kTileWaves) * slots * blocks;
      const std::false_type digits;
      const std::true_type halves;
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, 2> two;
      const std::integral_constant<int, 4> four;
      if (q.x.halves == 1) {
        groups < 256 ? go(halves, one, two) : go(halves, one, one);
      } else if (q.x.P == 3 || q.x.halves) {
        if constexpr (fine.value) {
          groups < 256 ? go(halves, two, two) : go(halves, two, one);
        } else {
          const std::integral_constant<int, 3> three;
          groups < 256 ? go(digits, three, two) : go(digits, three, one);
        }
      } else if (groups < 128) {
        go(digits, one, four);
      } else {
        groups < 256 ? go(digits, one, two) : go(digits, one, one);
      }
    });
  } else {
    // Measured over 81 to 32768 row tiles (whole passes, rt / split): enough
    // tiles take two or four together, which share the loads of the digits (16
    // assignments of 128 experts, down: 1/1 209, 2/2 193, 4/2 190 us; 64 tokens:
    // 1/1 360, 2/2 325, 4/2 298; 81 tiles of one matrix: 1/4 12.6, 2/4 15.5);
    // int8 tokens have fewer digits to share (gate and up 1/1 345, 2/2 380). A
    // tile's chunks are split so that neighbouring wavefronts read neighbouring
    // memory, but short matrices less (one token, down: 2/2 42.5, 2/4 43.8).
    const size_t tiles = size_t(p.row_tiles) * slots;
    const int rt = tiles < 384 || (one && q.mats == 2) ? 1 : q.mats == 1 && tiles >= 16384 ? 4 : 2;
    const int split = q.mats == 1 ? (tiles >= 2048 ? 2 : 4) : one && tiles >= 8192 ? 1 : 4;
    by_format(q, [&](auto fine, auto mats, auto zeros, auto st) {
      constexpr int M = decltype(mats)::value;
      const unsigned units = (p.row_tiles + rt - 1) / rt;
      const dim3 grid((units * split + 3) / 4, slots);
      using ST = decltype(st);
      auto go = [&](auto tiles) {
        constexpr int RT = decltype(tiles)::value;
        if (one)
          w4_rows_kernel<fine.value, M, 1, zeros.value, ST, RT><<<grid, 256, 0, s>>>(p, split);
        else
          w4_rows_kernel<fine.value, M, 3, zeros.value, ST, RT><<<grid, 256, 0, s>>>(p, split);
      };
      if (rt == 4 && M == 1) go(std::integral_constant<int, M == 1 ? 4 : 1>{});
      else if (rt == 2) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 1>{});
    });
  }
  INF_LAUNCHED();
  return INFERNO_OK;
}

// LDS of a launch of the token kernel: three workgroups of four wavefronts per CU,
// or two of sixteen (sums). At the border (4 tokens of 4096 columns, gate and up of
// 1536 rows) this launch takes 9.6 us a call, staging and product 11 to 13.
constexpr size_t kTokenLds = 53 * 1024, kTokenSumLds = 80 * 1024;

bool w4_token_fits(const W4Token& q) {
  const size_t rows = q.sum ? q.segments : q.T;
  return q.T <= 4 && q.segments <= kWave && rows * w4_chunks(q.m[0].cols) < 4096 &&
         token_lds(rows, w4_chunks(q.m[0].cols), q.mats, q.sum ? 16 : 4) <=
             (q.sum ? kTokenSumLds : kTokenLds);
}

namespace {

// Raises a kernel's dynamic LDS limit (64 KB by default), once per device.
template <typename K>
int allow_lds(K kern, size_t bytes, std::atomic<uint64_t>& devices) {
  int dev = 0;
  INF_HIP(hipGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (devices.load() & bit) return INFERNO_OK;
  INF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                              hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
  devices.fetch_or(bit);
  return INFERNO_OK;
}

}  // namespace

int launch_w4_token(hipStream_t s, const W4Token& q) {
  Tokens a{};
  for (int m = 0; m < q.mats; ++m) {
    const W4Layout l = w4_layout(q.m[m]);
    const uint8_t* at = static_cast<const uint8_t*>(q.m[m].packed);
    a.p.m[m] = Mat{at, at + l.scales, at + l.zeros};
  }
  a.p.N = uint32_t(q.m[0].rows);
  a.p.C = uint32_t(w4_chunks(q.m[0].cols));
  a.p.row_tiles = (a.p.N + 15) / 16;
  a.p.T = uint32_t(q.T);
  a.p.route_w = q.route_w;
  a.p.res_a = q.res_a;
  a.p.res_b = q.res_b;
  a.p.out = q.out;
  a.x = q.x;
  a.K = uint32_t(q.m[0].cols);
  a.segments = uint32_t(q.segments);
  a.ids = q.ids;
  a.E = uint32_t(q.m[0].experts);
  a.sum = q.sum;
  const bool bf16 = q.x_dtype == INFERNO_BF16;
  const dim3 grid(a.p.row_tiles, unsigned(q.slots));
  W4Product f{};
  f.m[0] = q.m[0];
  f.mats = q.mats;
  int status = INFERNO_OK;
  by_format(f, [&](auto fine, auto mats, auto zeros, auto st) {
    using ST = decltype(st);
    constexpr int M = decltype(mats)::value;
    auto go = [&](auto x, auto waves) {
      constexpr int W = decltype(waves)::value;
      const size_t rows = q.sum ? q.segments : q.T;
      const size_t lds = token_lds(rows, a.p.C, M, W);
      auto kern = w4_token_kernel<fine.value, M, zeros.value, ST, decltype(x), W>;
      if constexpr (W == 16) {
        static std::atomic<uint64_t> raised{0};
        if (lds > 64 * 1024 && (status = allow_lds(kern, kTokenSumLds, raised))) return;
      }
      kern<<<grid, W * kWave, lds, s>>>(a);
    };
    if constexpr (M == 1) {
      if (q.sum) return go(0.f, std::integral_constant<int, 16>{});
    }
    if (bf16) go(uint16_t{}, std::integral_constant<int, 4>{});
    else go(0.f, std::integral_constant<int, 4>{});
  });
  if (status) return status;
  INF_LAUNCHED();
  return INFERNO_OK;
}

int launch_w4_combine(hipStream_t s, const float* y, const uint32_t* ids, size_t T, size_t H,
                      size_t k, size_t E, float* out) {
  const bool wide = H % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const size_t threads = wide ? H / 4 : H;
  const dim3 grid(unsigned((threads + 255) / 256), unsigned(std::min<size_t>(T, 65535)));
  if (wide)
    w4_combine_kernel<4>
        <<<grid, 256, 0, s>>>(y, ids, T, uint32_t(H), uint32_t(k), uint32_t(E), out);
  else
    w4_combine_kernel<1>
        <<<grid, 256, 0, s>>>(y, ids, T, uint32_t(H), uint32_t(k), uint32_t(E), out);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
