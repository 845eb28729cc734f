// Residual addition, RMSNorm and 8-bit activations with scales, per row:
//   s = x + residual                       (fp32)
//   y = s / sqrt(mean(s^2) + eps) * w
//   q = rint(127 s w / A), A = max |s w| over the value's group
//   scale = A / sqrt(mean(s^2) + eps) / 127
// The root cancels in q, so q is the quotient of two products of two fp32
// values each, exact in 64 bits: q does not depend on how the squares are
// summed, and is the same in every kernel. The squares are summed in 64 bits:
// those of fp32 values pass fp32's range from 2^64 on. A row of zeros has y = 0
// and scale = 0 also with eps = 0, where the root is 0.
#include <type_traits>

#include "kernels.hpp"

namespace inferno {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(uint16_t v) { return bf16_bits_to_f32(v); }
__device__ __forceinline__ void store_act(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_act(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }

// |product| as an order-preserving integer: NaN lies above infinity, so that a
// group that holds one has a NaN as its largest value.
__device__ __forceinline__ uint64_t magnitude(float s, float w) {
  return __builtin_bit_cast(uint64_t, double(s) * double(w)) & 0x7fffffffffffffffull;
}

// A group without a finite, positive largest value has q = 0.
__device__ __forceinline__ int8_t quantised(float s, float w, double largest) {
  if (!(largest > 0.0) || isinf(largest)) return 0;
  return int8_t(rint(127.0 * (double(s) * double(w)) / largest));
}

// A product of fp32 values as fp32 bits: at most 2^100 and at least 2^-100.
__device__ __forceinline__ bool sound(uint32_t a) { return a - (27u << 23) <= (200u << 23); }

// A group's scale, from the exact largest product or from its fp32 rounding.
__device__ __forceinline__ float group_scale(double largest, double inv) {
  const float f = float(largest);
  return float((sound(f32_to_bits(f)) ? double(f) : largest) * inv / 127.0);
}

// 1 / sqrt(mean(s^2) + eps) from the sum of squares; 0 for a row of zeros.
__device__ __forceinline__ double inverse_root(double sq, double H, float eps) {
  const double mean = sq / H + double(eps);
  return mean == 0.0 ? 0.0 : 1.0 / sqrt(mean);
}

// s / sqrt(..) in 32 bits; in 64 for a row whose factor is no normal fp32 value: with
// eps = 0 rows below 2^-127 have one that passes fp32's range, rows from 2^126 on one
// that fp32 holds in fewer bits.
__device__ __forceinline__ bool factor_fits(double inv) { return inv < 0x1p127 && inv > 0x1p-126; }
__device__ __forceinline__ float scaled(float s, double inv, bool fits) {
  return fits ? s * float(inv) : float(double(s) * inv);
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(v, m, kWave);
    v = o > v ? o : v;
  }
  return v;
}

// Any width and alignment: one workgroup per row, the row read again from
// memory (or the cache) for each of the three steps. sum may be x or residual,
// which are therefore not __restrict__ (in either kernel).
template <typename XT, typename OT>
__global__ void __launch_bounds__(kThreads)
    add_norm_q8_row_kernel(const XT* x, const float* residual,
                           const float* __restrict__ w, float eps, size_t H, size_t group,
                           float* sum, OT* __restrict__ normed, int8_t* __restrict__ q,
                           float* __restrict__ scales) {
  __shared__ double part[kThreads / kWave];
  __shared__ uint64_t part64[kThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x, at = row * H;
  // sum may be the residual itself (or x): read once, afterwards sum is read
  auto total = [&](size_t i) {
    return sum ? sum[at + i] : value_of(x[at + i]) + (residual ? residual[at + i] : 0.f);
  };
  double sq = 0.0;
  for (size_t i = tid; i < H; i += kThreads) {
    const float s = value_of(x[at + i]) + (residual ? residual[at + i] : 0.f);
    if (sum) sum[at + i] = s;
    sq = fma(double(s), double(s), sq);
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) sq += __shfl_xor(sq, m, kWave);
  if (lane == 0) part[wave] = sq;
  __syncthreads();
  sq = 0.0;
  for (int i = 0; i < kThreads / kWave; ++i) sq += part[i];
  const double inv = inverse_root(sq, double(H), eps);
  const bool fits = factor_fits(inv);
  if (normed)
    for (size_t i = tid; i < H; i += kThreads)
      store_act(normed + at + i, scaled(total(i), inv, fits) * w[i]);
  if (!q) return;
  if (group == 0) {
    uint64_t a = 0;
    for (size_t i = tid; i < H; i += kThreads) a = max(a, magnitude(total(i), w[i]));
    a = wave_max64(a);
    if (lane == 0) part64[wave] = a;
    __syncthreads();
    for (int i = 0; i < kThreads / kWave; ++i) a = max(a, part64[i]);
    const double largest = __builtin_bit_cast(double, a);
    for (size_t i = tid; i < H; i += kThreads) q[at + i] = quantised(total(i), w[i], largest);
    if (tid == 0) scales[row] = group_scale(largest, inv);
    return;
  }
  const size_t groups = H / group;
  for (size_t g = wave; g < groups; g += kThreads / kWave) {
    uint64_t a = 0;
    for (size_t i = g * group + lane; i < (g + 1) * group; i += kWave)
      a = max(a, magnitude(total(i), w[i]));
    const double largest = __builtin_bit_cast(double, wave_max64(a));
    for (size_t i = g * group + lane; i < (g + 1) * group; i += kWave)
      q[at + i] = quantised(total(i), w[i], largest);
    if (lane == 0) scales[row * groups + g] = group_scale(largest, inv);
  }
}

// Largest of a value over 2^STEPS neighbouring lanes, in each of them.
template <int STEPS>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if (STEPS >= 1) v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0xB1, 0xF, 0xF, false)));
  if (STEPS >= 2) v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x4E, 0xF, 0xF, false)));
  if (STEPS >= 3) v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x141, 0xF, 0xF, false)));
  if (STEPS >= 4) v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), 0x140, 0xF, 0xF, false)));
  if (STEPS >= 5) {
    const auto o = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(o[0], o[1]);
  }
  if (STEPS >= 6) {
    const auto o = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max(o[0], o[1]);
  }
  return v;
}
template <int STEPS>
__device__ __forceinline__ uint64_t lanes_max64(uint64_t v) {
#pragma unroll
  for (int m = 1; m < (1 << STEPS); m <<= 1) {
    const uint64_t o = __shfl_xor(v, m, kWave);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
}
__device__ __forceinline__ void load4(const uint16_t* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  v[0] = bits_to_f32(u.x << 16); v[1] = bits_to_f32(u.x & 0xffff0000u);
  v[2] = bits_to_f32(u.y << 16); v[3] = bits_to_f32(u.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(uint16_t* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) =
      make_uint2(uint32_t(f32_to_bf16_bits(v[0])) | uint32_t(f32_to_bf16_bits(v[1])) << 16,
                 uint32_t(f32_to_bf16_bits(v[2])) | uint32_t(f32_to_bf16_bits(v[3])) << 16);
}

// Widths of a multiple of 4 up to 1024 NV, rows on 16 bytes: one workgroup per
// row, the row in registers (four neighbouring values per thread, NV times), so
// that memory is read once. Quotients are formed in 32 bits, with an error below
// 127 * 4 * 2^-24; one that lies nearer than 2^-14 to the border between two
// values is formed again in 64 bits, as are those of groups whose largest value
// is far from 1 (a product could leave fp32's range). STEPS: log2 of a group's
// lanes, 0: the row is one group.
template <typename XT, typename OT, int NV, int STEPS>
__global__ void __launch_bounds__(kThreads)
    add_norm_q8_kernel(const XT* x, const float* residual,
                       const float* __restrict__ w, float eps, uint32_t H, float* sum,
                       OT* __restrict__ normed, int8_t* __restrict__ q,
                       float* __restrict__ scales) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ double part[kWaves];
  __shared__ uint32_t top[kWaves];
  __shared__ uint64_t top64[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t at = size_t(blockIdx.x) * H;
  float v[NV][4], g[NV][4];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint32_t i = min(uint32_t(j * kThreads + tid) * 4, H - 4);  // clamped: loads together
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    load4(x + at + i, v[j]);
    if (residual) load4(residual + at + i, r);
    load4(w + i, g[j]);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[j][e] += r[e];
  }
  double sq = 0.0;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint32_t i = uint32_t(j * kThreads + tid) * 4;
    if (i < H) {
      if (sum) store4(sum + at + i, v[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sq = fma(double(v[j][e]), double(v[j][e]), sq);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j][e] = g[j][e] = 0.f;
    }
  }
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) sq += __shfl_xor(sq, m, kWave);
  if (lane == 0) part[wave] = sq;
  uint32_t most = 0;
  if (STEPS == 0 && q) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        most = max(most, f32_to_bits(v[j][e] * g[j][e]) & 0x7fffffffu);
    most = lanes_max<6>(most);
    if (lane == 0) top[wave] = most;
  }
  __syncthreads();
  sq = part[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) sq += part[i];
  const double inv = inverse_root(sq, double(H), eps);
  if (normed) {
    const bool fits = factor_fits(inv);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = uint32_t(j * kThreads + tid) * 4;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = scaled(v[j][e], inv, fits) * g[j][e];
      if (i < H) store4(normed + at + i, y);
    }
  }
  if (!q) return;
  if (STEPS == 0) {
    most = top[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) most = max(most, top[i]);
  }
  // four quotients in 32 bits; true where one has to be formed again
  auto quotients = [&](int j, uint32_t a, uint32_t& packed) {
    const float by = 127.f / bits_to_f32(a);
    bool again = !sound(a);
    packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = v[j][e] * g[j][e] * by, r = rintf(t);
      again |= fabsf(fabsf(t - r) - 0.5f) < 6.1035e-5f;
      packed |= (uint32_t(int(r)) & 255u) << (8 * e);
    }
    return again;
  };
  auto exactly = [&](int j, double a) {
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      packed |= (uint32_t(quantised(v[j][e], g[j][e], a)) & 255u) << (8 * e);
    return packed;
  };
  auto magnitude4 = [&](int j) {
    uint64_t a = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) a = max(a, magnitude(v[j][e], g[j][e]));
    return a;
  };
  if (STEPS == 0) {
    uint32_t out[NV];
    bool again = false;
#pragma unroll
    for (int j = 0; j < NV; ++j) again |= quotients(j, most, out[j]);
    double largest = double(bits_to_f32(most));
    if (__syncthreads_or(again)) {
      uint64_t a = 0;
#pragma unroll
      for (int j = 0; j < NV; ++j) a = max(a, magnitude4(j));
      a = lanes_max64<6>(a);
      if (lane == 0) top64[wave] = a;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) a = max(a, top64[i]);
      largest = __builtin_bit_cast(double, a);
#pragma unroll
      for (int j = 0; j < NV; ++j) out[j] = exactly(j, largest);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = uint32_t(j * kThreads + tid) * 4;
      if (i < H) *reinterpret_cast<uint32_t*>(q + at + i) = out[j];
    }
    if (tid == 0) scales[blockIdx.x] = group_scale(largest, inv);
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint32_t i = uint32_t(j * kThreads + tid) * 4;
    uint32_t a = 0, out;
#pragma unroll
    for (int e = 0; e < 4; ++e) a = max(a, f32_to_bits(v[j][e] * g[j][e]) & 0x7fffffffu);
    a = lanes_max<STEPS>(a);
    double largest = double(bits_to_f32(a));
    if (__any(quotients(j, a, out))) {
      largest = __builtin_bit_cast(double, lanes_max64<STEPS>(magnitude4(j)));
      out = exactly(j, largest);
    }
    if (i < H) {
      *reinterpret_cast<uint32_t*>(q + at + i) = out;
      if (tid % (1u << STEPS) == 0)
        scales[(at + i) >> (STEPS + 2)] = group_scale(largest, inv);
    }
  }
}

template <typename XT, typename OT>
void run_rows(hipStream_t s, const AddNormQ8& p) {
  add_norm_q8_row_kernel<XT, OT><<<unsigned(p.rows), kThreads, 0, s>>>(
      static_cast<const XT*>(p.x), p.residual, p.w, p.eps, p.H, p.group, p.sum,
      static_cast<OT*>(p.normed), p.q, p.scales);
}

template <typename XT, typename OT, int NV>
void run_registers(hipStream_t s, const AddNormQ8& p) {
  auto go = [&](auto steps) {
    add_norm_q8_kernel<XT, OT, NV, decltype(steps)::value><<<unsigned(p.rows), kThreads, 0, s>>>(
        static_cast<const XT*>(p.x), p.residual, p.w, p.eps, uint32_t(p.H), p.sum,
        static_cast<OT*>(p.normed), p.q, p.scales);
  };
  if (p.group == 32) go(std::integral_constant<int, 3>{});
  else if (p.group == 64) go(std::integral_constant<int, 4>{});
  else if (p.group == 128) go(std::integral_constant<int, 5>{});
  else go(std::integral_constant<int, 0>{});
}

template <typename XT, typename OT>
void run(hipStream_t s, const AddNormQ8& p) {
  auto on = [](const void* q, size_t to) { return reinterpret_cast<uintptr_t>(q) % to == 0; };
  const size_t n = (p.H + 4 * kThreads - 1) / (4 * kThreads);
  if (p.H % 4 || n > 8 || !on(p.x, 4 * sizeof(XT)) || !on(p.residual, 16) || !on(p.w, 16) ||
      !on(p.sum, 16) || !on(p.normed, 4 * sizeof(OT)) || !on(p.q, 4))
    run_rows<XT, OT>(s, p);
  else if (n <= 1) run_registers<XT, OT, 1>(s, p);
  else if (n <= 2) run_registers<XT, OT, 2>(s, p);
  else if (n <= 4) run_registers<XT, OT, 4>(s, p);
  else if (n <= 6) run_registers<XT, OT, 6>(s, p);
  else run_registers<XT, OT, 8>(s, p);
}

}  // namespace

int launch_add_norm_q8(hipStream_t s, const AddNormQ8& p) {
  if (p.rows == 0) return INFERNO_OK;
  const bool xb = p.x_dtype == INFERNO_BF16, ob = p.act_dtype == INFERNO_BF16;
  if (xb && ob) run<uint16_t, uint16_t>(s, p);
  else if (xb) run<uint16_t, float>(s, p);
  else if (ob) run<float, uint16_t>(s, p);
  else run<float, float>(s, p);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
