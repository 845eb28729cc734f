// Residual addition, RMSNorm and 8-bit activations with scales, per row:
//   s = x + residual                       (fp32)
//   y = s / sqrt(mean(s^2) + eps) * w
//   q = rint(127 s w / A), A = max |s w| over the value's group
//   scale = A / sqrt(mean(s^2) + eps) / 127
// The root cancels in q, so q is the quotient of two products of two fp32
// values each, exact in 64 bits: q does not depend on how the squares are
// summed, and is the same in every kernel. The squares are summed in 64 bits:
// those of fp32 values pass fp32's range from 2^64 on.
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

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(v, m, kWave);
    v = o > v ? o : v;
  }
  return v;
}

// Any width and alignment: one workgroup per row, the row read again from
// memory (or the cache) for each of the three steps.
template <typename XT, typename OT>
__global__ void __launch_bounds__(kThreads)
    add_norm_q8_row_kernel(const XT* __restrict__ x, const float* residual,
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
  const float root = float(sqrt(sq / double(H) + double(eps)));
  if (normed)
    for (size_t i = tid; i < H; i += kThreads) store_act(normed + at + i, total(i) / root * w[i]);
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
    if (tid == 0) scales[row] = float(largest / double(root) / 127.0);
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
    if (lane == 0) scales[row * groups + g] = float(largest / double(root) / 127.0);
  }
}

template <typename XT, typename OT>
void run(hipStream_t s, const AddNormQ8& p) {
  add_norm_q8_row_kernel<XT, OT><<<unsigned(p.rows), kThreads, 0, s>>>(
      static_cast<const XT*>(p.x), p.residual, p.w, p.eps, p.H, p.group, p.sum,
      static_cast<OT*>(p.normed), p.q, p.scales);
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
