// Top-k over the best groups of experts, one wavefront per token.
//
// Selection value v_e = sigmoid(l_e) + b_e, or l_e + b_e with softmax scores
// (as the router's top-k). A group's value is its largest v, or the sum of its
// two largest; the topk_group best groups stay open (value descending, then
// the lower group), and of their experts the k best win (v descending, then
// the lower id), by the values in 64 bits: in 32 bits, values next to each
// other round to one or change places.
//
// Values are first formed in 32 bits. They decide wherever the values that they
// order are further apart than their roundings, which is checked for every open
// group against every closed one (a sum of two rounds by their magnitudes, which
// it may be far below), for the last winner against the best loser and for
// neighbouring winners. Where winners fail, the experts that may be among the k
// best (one per lane) are formed and ranked in 64 bits; a token whose groups fail,
// with more of them than lanes, or with a NaN is done again in 64 bits as a whole.
// 8192 tokens of 256 experts in 8 groups: 15.6 us (15.3 with the last open and the
// first closed group alone compared); whole rows in 64 bits for every failure 20.3,
// for every token 28 us. All 8192 wavefronts are resident at once: what bounds it is
// their instructions and, for few tokens, one chain of cross-lane steps (29 tokens:
// 6.4 us).
#include "kernels.hpp"
#include "routing_dev.hpp"

namespace inferno {
namespace {

constexpr int kTokens = 4;  // per workgroup, one wavefront each

struct GroupTopk {
  const float* logits;
  const float* bias;
  size_t T;
  int E, k, score_fn, norm;
  float scale;
  int groups, size, topk_group, rule;
  int lanes;  // of one group: a power of two, groups * lanes <= 64 (0: more groups)
  uint32_t* ids;
  float* weights;
  uint32_t* token_idx;
};

// One wavefront's scratch.
union Scratch {
  struct {
    double value[kMaxExperts];
    uint64_t group[kMaxExperts];
  } exact;
  struct {
    float value[2 * kMaxExperts];  // a group's values one place apart from the next's
    uint32_t key[kWave];
    uint32_t id[kWave];
    float by_rank[kMaxTopK];
  } fast;
};

// Order-preserving map of a double onto u64; every NaN above +infinity.
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  if (v != v) return ~0ull;
  if (v == 0.0) return 1ull << 63;  // -0 and +0 are one value
  return (b >> 63) ? ~b : (b | (1ull << 63));
}

// Weight of a winner: `sum` of the winners' scores, or of all.
__device__ __forceinline__ float weight_of(const GroupTopk& p, float score, float sum) {
  const bool divide =
      (p.norm || p.score_fn == INFERNO_SCORE_SOFTMAX) && sum > 0.f && isfinite(sum);
  return (divide ? score / sum : score) * p.scale;
}

// What the winners' logits are taken relative to: normalised weights are ratios of
// their scores alone, which vanish together if the row's largest logit is in a
// closed group and more than 87 above them. top: the winners' largest logit.
__device__ __forceinline__ float weights_from(const GroupTopk& p, float lmax, float top) {
  return p.norm && fabsf(lmax) < INFINITY && top > -INFINITY ? top : lmax;
}

// The same for sigmoids, which are exp(l) in 32 bits from -17 down: whether the
// winners' are so small that they vanish. sum: of their scores.
__device__ __forceinline__ bool vanishing(const GroupTopk& p, float sum, float top) {
  return p.norm && sum < 0x1p-80f && top > -INFINITY;
}

__device__ __forceinline__ void exact_row(const GroupTopk& p, size_t t, Scratch& scratch) {
  constexpr int kPer = kMaxExperts / kWave;
  const int lane = threadIdx.x & 63;
  double* value = scratch.exact.value;
  uint64_t* gkey = scratch.exact.group;
  const float* row = p.logits + t * size_t(p.E);
  float lg[kPer], score[kPer];
  float lmax = -INFINITY;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    lg[j] = e < p.E ? row[e] : -INFINITY;
    lmax = fmaxf(lmax, lg[j]);
  }
  lmax = wave_max(lmax);
  float all = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    double v;
    if (p.score_fn == INFERNO_SCORE_SIGMOID) {
      v = 1.0 / (1.0 + exp(-double(lg[j])));
      score[j] = float(v);
    } else {
      v = lg[j];
      score[j] = e < p.E && lmax != -INFINITY ? expf(lg[j] - lmax) : 0.f;
    }
    if (e < p.E) {
      value[e] = v + (p.bias ? double(p.bias[e]) : 0.0);
      all += score[j];
    }
  }
  all = wave_sum(all);
  __builtin_amdgcn_wave_barrier();  // LDS is in order within a wavefront
  for (int g = lane; g < p.groups; g += kWave) {
    double a = -INFINITY, b = -INFINITY;
    bool nan = false;
    for (int i = 0; i < p.size; ++i) {
      const double v = value[g * p.size + i];
      nan |= v != v;
      b = fmax(b, fmin(a, v));
      a = fmax(a, v);
    }
    const double two = p.size > 1 ? a + b : a;
    gkey[g] = nan ? ~0ull : order_key(p.rule == INFERNO_GROUP_TOP2 ? two : a);
  }
  __builtin_amdgcn_wave_barrier();
  uint64_t key[kPer];
  bool live[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + j * kWave;
    live[j] = e < p.E;
    key[j] = 0;
    if (!live[j]) continue;
    const int g = e / p.size;
    const uint64_t mine = gkey[g];
    int before = 0;
    for (int o = 0; o < p.groups; ++o) before += gkey[o] > mine || (gkey[o] == mine && o < g);
    live[j] = before < p.topk_group;
    key[j] = order_key(value[e]);
  }
  float sum = 0.f, mine_w = 0.f, mine_l = -INFINITY;
  uint32_t mine_id = 0;
  for (int r = 0; r < p.k; ++r) {
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
    float s = 0.f, l = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (id == lane + j * kWave) {
        s = score[j];
        l = lg[j];
        live[j] = false;
      }
    }
    s = __shfl(s, id & 63, kWave);
    l = __shfl(l, id & 63, kWave);
    sum += s;  // rank order
    if (lane == r) {
      mine_w = s;
      mine_l = l;
      mine_id = uint32_t(id);
    }
  }
  if (!__any(mine_l != mine_l)) {
    const float top = wave_max(mine_l);
    const bool softmax = p.score_fn == INFERNO_SCORE_SOFTMAX;
    const float from = softmax ? weights_from(p, lmax, top) : top;
    if (softmax ? from != lmax : vanishing(p, sum, top)) {  // uniform
      mine_w = expf(mine_l - from);
      sum = 0.f;
      for (int r = 0; r < p.k; ++r) sum += __shfl(mine_w, r, kWave);  // rank order
    }
  }
  if (lane < p.k) {
    const size_t a = t * size_t(p.k) + lane;
    p.ids[a] = mine_id;
    p.weights[a] = weight_of(p, mine_w, p.norm ? sum : all);
    if (p.token_idx) p.token_idx[a] = uint32_t(t);
  }
}

// The sigmoid but for 2^-22: the rounding of l log2(e) moves it by at most
// max(|l| s (1 - s)) 2^-24 = 0.23 2^-24, that of the product with the constant's
// as much; exponential, sum and reciprocal are off by a few 2^-24 of themselves.
__device__ __forceinline__ float near_sigmoid(float l) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * l));
}

__device__ __forceinline__ float lane_of(float v, int lane) {  // lane: uniform
  return bits_to_f32(__builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, v), lane));
}

// Whether a > b holds for the 64-bit values of two 32-bit ones. A sigmoid is
// off by at most 2^-22, the addition of the bias by 2^-24 of the value; `times`
// values were added. Infinities and NaN: no.
__device__ __forceinline__ bool above(float a, float b, bool sigmoid, float times) {
  const float off = (sigmoid ? 0x1p-20f : 0.f) + 0x1p-22f * fmaxf(fabsf(a), fabsf(b));
  return a - b > times * off;
}

// The same in 32 bits; false if a value lies too near another one. PER: experts
// per lane.
template <int PER>
__device__ __forceinline__ bool fast_row(const GroupTopk& p, size_t t, Scratch& scratch) {
  auto& s = scratch.fast;
  const int lane = threadIdx.x & 63;
  const bool sigmoid = p.score_fn == INFERNO_SCORE_SIGMOID;
  const float* row = p.logits + t * size_t(p.E);
  float lg[PER], bs[PER], score[PER], v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = min(lane + j * kWave, p.E - 1);
    lg[j] = row[e];
    bs[j] = p.bias ? p.bias[e] : 0.f;
  }
  float lmax = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float both = lg[j] + bs[j];
    nan |= both != both;  // +-infinity with the other as bias too
    // a sum behind fp32's range, so that infinite values below are infinite ones
    nan |= fabsf(both) == INFINITY && fmaxf(fabsf(lg[j]), fabsf(bs[j])) < INFINITY;
    lmax = fmaxf(lmax, lg[j]);
  }
  if (__any(nan)) return false;
  if (!sigmoid) {
    lmax = bits_to_f32([](uint32_t k) { return (k >> 31) ? k ^ 0x80000000u : ~k; }(
        wave_umax(total_order_key(lmax))));
    if (lmax == -INFINITY) return false;
  }
  float all = 0.f;
  const float magic = 1.f / float(p.size);
  int group[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + j * kWave;
    score[j] = sigmoid ? near_sigmoid(lg[j]) : expf(lg[j] - lmax);
    v[j] = (sigmoid ? score[j] : lg[j]) + bs[j];
    // e / size for e < 256: the quotient's error is far below 1 / (2 size)
    group[j] = int((float(e) + 0.5f) * magic);
    if (e < p.E) {
      all += score[j];
      s.value[e + group[j]] = v[j];  // group g begins at g * (size + 1)
    }
  }
  __builtin_amdgcn_wave_barrier();  // LDS is in order within a wavefront
  uint64_t open = ~0ull;            // bit g * lanes: group g is
  if (p.topk_group < p.groups) {
    const int L = p.lanes, g = lane / L, sub = lane % L;
    float a = -INFINITY, b = -INFINITY;  // the two largest of this lane's share
    if (g < p.groups)
      for (int i = sub; i < p.size; i += L) {
        const float x = s.value[g * (p.size + 1) + i];
        b = fmaxf(b, fminf(a, x));
        a = fmaxf(a, x);
      }
    for (int m = 1; m < L; m <<= 1) {
      const float oa = __shfl_xor(a, m, kWave), ob = __shfl_xor(b, m, kWave);
      b = fmaxf(fminf(a, oa), fmaxf(b, ob));
      a = fmaxf(a, oa);
    }
    const bool two = p.rule == INFERNO_GROUP_TOP2 && p.size > 1;
    const float gv = two ? a + b : a;
    // +infinity and -infinity: a NaN, which counts as the best group but compares as
    // none
    if (__any(gv != gv)) return false;
    int before = 0;
    for (int o = 0; o < p.groups; ++o) {
      const float x = lane_of(gv, o * L);
      before += x > gv || (x == gv && o < g);
    }
    const bool mine = g < p.groups && sub == 0, in = before < p.topk_group;
    open = __ballot(mine && in);
    // How far gv may be off: each summand by 2^-24 of itself (and a sigmoid by
    // 2^-22), their sum by 2^-24 of it, which is less than of both magnitudes; twice
    // that, so that the roundings of these two borders are in it. An infinite value
    // is one in 64 bits too.
    const float size = two ? fabsf(a) + fabsf(b) : fabsf(a);
    const bool infinite = fabsf(a) == INFINITY || (two && fabsf(b) == INFINITY);
    const float off =
        infinite ? 0.f : size * 0x1p-22f + (sigmoid ? (two ? 0x1p-20f : 0x1p-21f) : 0.f);
    if (__any(mine && off == INFINITY)) return false;  // a sum behind fp32's range
    const uint32_t lowest = ~wave_umax(mine && in ? ~total_order_key(gv - off) : 0u);
    if (lowest <= wave_umax(mine && !in ? total_order_key(gv + off) : 0u)) return false;
  }
  uint32_t key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = lane + j * kWave;
    const bool is = e < p.E &&
                    (p.topk_group == p.groups || (open >> (min(group[j], 63 / p.lanes) * p.lanes) & 1));
    key[j] = is ? max(total_order_key(v[j]), 1u) : 0u;
  }
  // the k-th largest key, bit by bit from the top; done as soon as exactly k
  // keys are at or above the prefix
  uint32_t kth = 0, n = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = kth | (1u << b);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) m += uint32_t(__popcll(__ballot(key[j] >= c)));
    if (m >= uint32_t(p.k)) {
      kth = c;
      n = m;
      if (m == uint32_t(p.k)) break;  // uniform
    }
  }
  auto value_of = [](uint32_t k) {
    return bits_to_f32((k >> 31) ? k ^ 0x80000000u : ~k);
  };
  // puts the experts that `is` holds for next to each other, and returns how many
  auto gather = [&](auto is) {
    uint32_t base = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const bool win = is(key[j]);
      const uint64_t m = __ballot(win);
      const uint32_t at = base + __builtin_amdgcn_mbcnt_hi(
                                     uint32_t(m >> 32),
                                     __builtin_amdgcn_mbcnt_lo(uint32_t(m), 0u));
      if (win && at < uint32_t(kWave)) {
        s.key[at] = key[j];
        s.id[at] = uint32_t(lane + j * kWave);
      }
      base += uint32_t(__popcll(m));
    }
    __builtin_amdgcn_wave_barrier();
    return base;
  };
  bool clear = false;
  uint32_t rank = 0, id = 0;  // of this lane's winner, if it has one
  if (n == uint32_t(p.k)) {   // else keys are equal
    gather([&](uint32_t k) { return k >= kth; });
    uint32_t loser = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) loser = max(loser, key[j] < kth ? key[j] : 0u);
    const uint32_t mine = s.key[min(lane, p.k - 1)];
    id = s.id[min(lane, p.k - 1)];
    uint32_t same = 0, below = wave_umax(loser);  // the best key below this winner's, 0: none
    for (int i = 0; i < p.k; ++i) {
      const uint32_t o = __builtin_amdgcn_readlane(mine, i);
      rank += o > mine ? 1u : 0u;
      same += o == mine ? 1u : 0u;
      if (o < mine) below = max(below, o);
    }
    clear = same == 1 && (below == 0 || above(value_of(mine), value_of(below), sigmoid, 1.f));
    if (lane >= p.k) rank = uint32_t(p.k);
  }
  if (__any(rank < uint32_t(p.k) && !clear)) {
    // In 64 bits, but only the experts that may be among the k best: those not
    // clearly below the k-th largest key.
    kth = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t c = kth | (1u << b);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) m += uint32_t(__popcll(__ballot(key[j] >= c)));
      if (m >= uint32_t(p.k)) kth = c;
    }
    const uint32_t many = gather([&](uint32_t k) {
      return k >= kth || (k && !above(value_of(kth), value_of(k), sigmoid, 1.f));
    });
    if (many > uint32_t(kWave)) return false;
    id = s.id[min(uint32_t(lane), many - 1)];
    double exact = row[id];
    if (sigmoid) exact = 1.0 / (1.0 + exp(-exact));
    exact += p.bias ? double(p.bias[id]) : 0.0;
    const uint64_t mine = order_key(exact);
    rank = 0;
    for (uint32_t i = 0; i < many; ++i) {
      const uint32_t high = __builtin_amdgcn_readlane(uint32_t(mine >> 32), i);
      const uint32_t low = __builtin_amdgcn_readlane(uint32_t(mine), i);
      const uint64_t o = uint64_t(high) << 32 | low;
      const uint32_t other = __builtin_amdgcn_readlane(id, i);
      rank += o > mine || (o == mine && other < id) ? 1u : 0u;
    }
    if (uint32_t(lane) >= many) rank = uint32_t(p.k);
  }
  const bool won = rank < uint32_t(p.k);
  const float l = row[id];
  if (!sigmoid && p.norm) {
    const uint32_t top = wave_umax(won ? total_order_key(l) : 0u);
    lmax = weights_from(p, lmax, value_of(top));
  }
  float my_score = sigmoid ? 1.f / (1.f + expf(-l)) : expf(l - lmax);
  float sum = 0.f;
  auto add_up = [&] {
    if (won) s.by_rank[rank] = my_score;
    __builtin_amdgcn_wave_barrier();
    const float ranked = s.by_rank[min(lane, p.k - 1)];
    sum = 0.f;
    for (int r = 0; r < p.k; ++r) sum += lane_of(ranked, r);  // rank order
  };
  if (p.norm) {
    add_up();
    if (sigmoid && sum < 0x1p-80f) {  // uniform
      const uint32_t key = wave_umax(won ? total_order_key(l) : 0u);
      const float top = value_of(key);
      if (vanishing(p, sum, top)) {
        my_score = expf(l - top);
        __builtin_amdgcn_wave_barrier();
        add_up();
      }
    }
  } else {
    sum = wave_sum(all);
  }
  if (won) {
    const size_t a = t * size_t(p.k) + rank;
    p.ids[a] = id;
    p.weights[a] = weight_of(p, my_score, sum);
    if (p.token_idx) p.token_idx[a] = uint32_t(t);
  }
  return true;
}

template <int PER>
__global__ void __launch_bounds__(kTokens* kWave) group_topk_kernel(GroupTopk p) {
  __shared__ Scratch scratch[kTokens];
  const int wave = threadIdx.x >> 6;
  const size_t t = size_t(blockIdx.x) * kTokens + wave;
  if (t >= p.T) return;  // no barrier of the workgroup below
  if (p.lanes == 0 || !fast_row<PER>(p, t, scratch[wave])) {
    __builtin_amdgcn_wave_barrier();
    exact_row(p, t, scratch[wave]);
  }
}

}  // namespace

int launch_group_topk(hipStream_t s, const float* logits, const float* bias, size_t T, size_t E,
                      size_t k, int score_fn, int norm, float scale, size_t groups,
                      size_t topk_group, int rule, uint32_t* ids, float* weights,
                      uint32_t* token_idx) {
  int lanes = groups > 64 ? 0 : 1;
  while (lanes && groups * lanes * 2 <= 64) lanes *= 2;
  const GroupTopk p{logits, bias, T, int(E), int(k), score_fn, norm, scale, int(groups),
                    int(E / groups), int(topk_group), rule, lanes, ids, weights, token_idx};
  const unsigned grid = unsigned((T + kTokens - 1) / kTokens);
  if (E <= 64) group_topk_kernel<1><<<grid, kTokens * kWave, 0, s>>>(p);
  else if (E <= 128) group_topk_kernel<2><<<grid, kTokens * kWave, 0, s>>>(p);
  else group_topk_kernel<4><<<grid, kTokens * kWave, 0, s>>>(p);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
