// Top-k over the best groups of experts, one wavefront per token.
//
// Selection value v_e = sigmoid(l_e) + b_e, or l_e + b_e with softmax scores
// (as the router's top-k). A group's value is its largest v, or the sum of its
// two largest; the topk_group best groups stay open (value descending, then
// the lower group), and of their experts the k best win (v descending, then
// the lower id). Values are formed in 64 bits: in 32 bits, values next to each
// other round to one or change places.
#include "kernels.hpp"
#include "routing_dev.hpp"

namespace inferno {
namespace {

constexpr int kPer = kMaxExperts / kWave;  // candidates per lane
constexpr int kTokens = 4;                 // per workgroup, one wavefront each

// Order-preserving map of a double onto u64; every NaN above +infinity.
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  if (v != v) return ~0ull;
  if (v == 0.0) return 1ull << 63;  // -0 and +0 are one value
  return (b >> 63) ? ~b : (b | (1ull << 63));
}

__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmax(v, __shfl_xor(v, m, kWave));
  return v;
}

__global__ void __launch_bounds__(kTokens* kWave)
    group_topk_kernel(const float* __restrict__ logits, const float* __restrict__ bias, size_t T,
                      int E, int k, int score_fn, int norm, float scale, int groups,
                      int topk_group, int rule, uint32_t* __restrict__ ids,
                      float* __restrict__ weights, uint32_t* __restrict__ token_idx) {
  __shared__ double value_s[kTokens][kMaxExperts];
  __shared__ uint64_t group_s[kTokens][kMaxExperts];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t t = size_t(blockIdx.x) * kTokens + wave;
  if (t >= T) return;  // no barrier of the workgroup below
  double* value = value_s[wave];
  uint64_t* gkey = group_s[wave];
  const float* row = logits + t * size_t(E);
  float lg[kPer], score[kPer];
  float lmax = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    lg[j] = e < E ? row[e] : -INFINITY;
    lmax = fmaxf(lmax, lg[j]);
  }
  lmax = wave_max(lmax);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    double v;
    if (score_fn == INFERNO_SCORE_SIGMOID) {
      v = 1.0 / (1.0 + exp(-double(lg[j])));
      score[j] = float(v);
    } else {
      v = lg[j];
      score[j] = e < E && lmax != -INFINITY ? expf(lg[j] - lmax) : 0.f;
    }
    if (e < E) value[e] = v + (bias ? double(bias[e]) : 0.0);
  }
  float all = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) all += lane + j * kWave < E ? score[j] : 0.f;
  all = wave_sum(all);
  __builtin_amdgcn_wave_barrier();  // LDS is in order within a wavefront
  const int size = E / groups;
  for (int g = lane; g < groups; g += kWave) {
    double a = -INFINITY, b = -INFINITY;
    bool nan = false;
    for (int i = 0; i < size; ++i) {
      const double v = value[g * size + i];
      nan |= v != v;
      b = fmax(b, fmin(a, v));
      a = fmax(a, v);
    }
    const double two = size > 1 ? a + b : a;
    gkey[g] = nan ? ~0ull : order_key(rule == INFERNO_GROUP_TOP2 ? two : a);
  }
  __builtin_amdgcn_wave_barrier();
  uint64_t key[kPer];
  bool live[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    live[j] = e < E;
    key[j] = 0;
    if (!live[j]) continue;
    const int g = e / size;
    const uint64_t mine = gkey[g];
    int before = 0;
    for (int o = 0; o < groups; ++o) before += gkey[o] > mine || (gkey[o] == mine && o < g);
    live[j] = before < topk_group;
    key[j] = order_key(value[e]);
  }
  float sum = 0.f, mine_w = 0.f;
  uint32_t mine_id = 0;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    int id = INT32_MAX;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (live[j] && (id == INT32_MAX || key[j] > best)) {
        best = key[j];
        id = lane + j * kWave;
      }
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const uint64_t ob = __shfl_xor(best, m, kWave);
      const int oi = __shfl_xor(id, m, kWave);
      const bool take = oi != INT32_MAX && (id == INT32_MAX || ob > best || (ob == best && oi < id));
      best = take ? ob : best;
      id = take ? oi : id;
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (id == lane + j * kWave) {
        s = score[j];
        live[j] = false;
      }
    }
    s = __shfl(s, id & 63, kWave);
    sum += s;  // rank order
    if (lane == r) {
      mine_w = s;
      mine_id = uint32_t(id);
    }
  }
  if (!norm) sum = all;
  const bool divide = (norm || score_fn == INFERNO_SCORE_SOFTMAX) && sum > 0.f && isfinite(sum);
  if (lane < k) {
    const size_t a = t * size_t(k) + lane;
    ids[a] = mine_id;
    weights[a] = (divide ? mine_w / sum : mine_w) * scale;
    if (token_idx) token_idx[a] = uint32_t(t);
  }
}

}  // namespace

int launch_group_topk(hipStream_t s, const float* logits, const float* bias, size_t T, size_t E,
                      size_t k, int score_fn, int norm, float scale, size_t groups,
                      size_t topk_group, int rule, uint32_t* ids, float* weights,
                      uint32_t* token_idx) {
  group_topk_kernel<<<unsigned((T + kTokens - 1) / kTokens), kTokens * kWave, 0, s>>>(
      logits, bias, T, int(E), int(k), score_fn, norm, scale, int(groups), int(topk_group), rule,
      ids, weights, token_idx);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
