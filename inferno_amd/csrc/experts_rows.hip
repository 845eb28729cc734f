// Products of rows grouped by expert, few rows: two tiles of 16 weight rows (one of
// each matrix, if there are two) by 16 or 32 grouped rows, the operands straight from
// memory to registers in the order of the matrix instructions. And which kernel takes
// a product.
//
// The weights are the first operand (lane l: row l % 16, quarter l / 16 of the
// columns of a step), the grouped rows the second, so that a lane's four sums
// are four neighbouring values of one result row. Of a workgroup's four wavefronts
// SHARES take the same weight rows and share the columns; they add their sums in
// order through LDS. What bounds it is how many bytes are on their way: every
// wavefront loads kAhead chunks of 128 columns before it uses the first.
//
// One token, microseconds of a call among others: down of 8 of 256 experts, 6144 x
// 2048 in MXFP4, 12.0 (4.5 TB/s); gate and up of 8 of 64 experts, 768 x 2048 in bf16,
// 11.3 (4.5 TB/s); gate and up of a shared expert, 1536 x 4096 in MXFP4, 8.5, where a
// launch of nothing takes 6.2. With twice as many chunks ahead the three launches take,
// from one to the next of a graph, 16.2, 15.2 and 6.4 in place of 14.1, 13.3 and 6.6;
// with four times as many in MXFP4 the first takes 21 and the last 7.2.
#include <cmath>
#include <cstdio>

#include "experts_dev.hpp"

namespace inferno {
namespace {

using namespace experts;

constexpr int kWaves = 4;
constexpr int kTiles = 2;         // of 16 weight rows, of a wavefront
constexpr uint32_t kChunk = 128;  // columns
constexpr double kCUs = 256;

// One chunk's operands of a wavefront, 128 columns.
template <bool WFP4, bool XFP4, int RT, int NB>
struct Chunk {
  uint4 w[RT][WFP4 ? 1 : 4], x[NB][XFP4 ? 1 : 4];
  uint32_t ws[RT], xs[NB];
};

template <bool WFP4, bool XFP4, int MATS, int NB, int SHARES>
__global__ void __launch_bounds__(kWaves* kWave) experts_rows_kernel(Product p, uint32_t blocks) {
  constexpr int RT = kTiles;
  using C = Chunk<WFP4, XFP4, RT, NB>;
  constexpr int kAhead = WFP4 && XFP4 ? 4 : 2;
  constexpr int kPerMat = RT / MATS;
  __shared__ floatx4 part[SHARES > 1 ? kWaves : 1][RT][NB][kWave];
  Work work;
  if (!find_work<16 * NB, false>(p, blockIdx.x, blocks, work)) return;
  const uint32_t e = work.e, c0 = work.c0, c1 = work.c1;
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t share = wave % SHARES;
  // the wavefront's first weight tile of each matrix
  const uint32_t first_tile = (work.unit * (kWaves / SHARES) + wave / SHARES) * kPerMat;
  const uint32_t pitch = XFP4 ? p.K / 2 : p.K * 2;
  // rows behind the tile's last are computed as it is, and not stored
  uint32_t a[NB];
  const uint8_t* x[NB];
  const uint8_t* xs[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) a[b] = min(c0 + 16 * b + n, c1 - 1);
  result_rows(p, a);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const size_t row = input_row(p, a[b]);
    x[b] = p.x + row * pitch;
    xs[b] = p.xs + row * (p.K / kMxBlock);
  }
  const uint8_t* w[RT];
  const uint32_t* ws[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const uint32_t tile = min(first_tile + r % kPerMat, p.tiles - 1);
    const size_t at = size_t(e) * p.tiles + tile;
    w[r] = p.w[r / kPerMat] + at * p.steps * 1024 + lane * 16;
    if constexpr (WFP4) ws[r] = p.ws[r / kPerMat] + at * p.quads * 64 + lane;
  }
  // column of the lane's 16 bytes number j of a chunk
  auto column = [&](uint32_t ch, int j) {
    return ch * kChunk + (WFP4 ? 32 * g + 8 * j : 32 * j + 8 * g);
  };
  auto load = [&](uint32_t ch, C& v) {
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      if constexpr (WFP4) {
        v.w[m][0] = *reinterpret_cast<const uint4*>(w[m] + size_t(ch) * 1024);
        v.ws[m] = ws[m][size_t(ch / 4) * 64] >> (8 * (ch % 4));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v.w[m][j] =
              *reinterpret_cast<const uint4*>(w[m] + size_t(min(4 * ch + j, p.steps - 1)) * 1024);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (XFP4) {
        const uint32_t col = column(ch, 0);
        v.x[b][0] = *reinterpret_cast<const uint4*>(x[b] + (col < p.K ? col / 2 : 0));
        v.xs[b] = xs[b][col < p.K ? col / kMxBlock : 0];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t col = column(ch, j);
          v.x[b][j] = *reinterpret_cast<const uint4*>(x[b] + (col < p.K ? col * 2 : 0));
        }
      }
    }
  };
  floatx4 acc[RT][NB];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[m][b] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto use = [&](uint32_t ch, C& v) {
    if ((ch + 1) * kChunk > p.K) {  // the last chunk: nothing behind the last column
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t keep = column(ch, j) < p.K ? ~0u : 0u;
        auto cut = [&](uint4& u) { u = make_uint4(u.x & keep, u.y & keep, u.z & keep, u.w & keep); };
#pragma unroll
        for (int b = 0; b < NB; ++b)
          if (j == 0 || !XFP4) cut(v.x[b][XFP4 ? 0 : j]);
        if constexpr (!WFP4) {
#pragma unroll
          for (int m = 0; m < RT; ++m) cut(v.w[m][j]);
        }
      }
    }
    if constexpr (WFP4 && XFP4) {
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          acc[m][b] = mfma_fp4(v.w[m][0], v.x[b][0], acc[m][b], v.ws[m], v.xs[b]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          bf16x8 f;
          if constexpr (WFP4) {
            const uint4 c = v.w[m][0];
            f = widen(j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w, scale_of(v.ws[m] & 255u));
          } else {
            f = __builtin_bit_cast(bf16x8, v.w[m][j]);
          }
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[m][b] = mfma_bf16(f, __builtin_bit_cast(bf16x8, v.x[b][j]), acc[m][b]);
        }
    }
  };
  // this wavefront's chunks
  const uint32_t chunks = (p.K + kChunk - 1) / kChunk;
  const uint32_t first = chunks * share / SHARES, last = chunks * (share + 1) / SHARES;
  if (first < last) {
    C v[kAhead];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) load(min(first + d, last - 1), v[d]);
    for (uint32_t ch = first; ch < last; ch += kAhead) {
#pragma unroll
      for (int d = 0; d < kAhead; ++d) {
        if (ch + d < last) use(ch + d, v[d]);
        load(min(ch + d + kAhead, last - 1), v[d]);
      }
    }
  }
  if constexpr (SHARES > 1) {
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int b = 0; b < NB; ++b) part[wave][m][b][lane] = acc[m][b];
    __syncthreads();
  }
  // the wavefronts of a share write the 16 rows number b in turn
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (share != uint32_t(b % SHARES)) continue;
    if constexpr (SHARES > 1) {
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        acc[m][b] = part[wave - share][m][b][lane];
        for (int v = 1; v < SHARES; ++v) acc[m][b] += part[wave - share + v][m][b][lane];
      }
    }
    if (c0 + 16 * b + n >= c1 || a[b] >= p.A) continue;
#pragma unroll
    for (int r = 0; r < kPerMat; ++r) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        y[i] = MATS == 2 ? silu_mul(acc[r][b][i], acc[r + RT - kPerMat][b][i]) : acc[r][b][i];
      store4(p, a[b], (first_tile + r) * 16 + 4 * g, y);
    }
  }
}

template <int NB, int SHARES>
int launch(hipStream_t s, const Product& p, int mats, bool wfp4, bool xfp4, size_t tiles) {
  const size_t per = kWaves / SHARES * kTiles / mats;  // weight tiles of a workgroup
  const size_t blocks = (p.tiles + per - 1) / per;
  if (tiles * blocks * (kWaves * kWave) >= size_t(1) << 32) {
    set_error("too many rows for one launch");
    return INFERNO_ERR_INVALID;
  }
  auto go = [&](auto wf, auto xf) {
    constexpr bool W = decltype(wf)::value, X = decltype(xf)::value;
    const unsigned grid = unsigned(tiles * blocks), threads = kWaves * kWave;
    if (mats == 1)
      experts_rows_kernel<W, X, 1, NB, SHARES><<<grid, threads, 0, s>>>(p, unsigned(blocks));
    else
      experts_rows_kernel<W, X, 2, NB, SHARES><<<grid, threads, 0, s>>>(p, unsigned(blocks));
  };
  if (!wfp4) go(std::false_type{}, std::false_type{});
  else if (xfp4) go(std::true_type{}, std::true_type{});
  else go(std::true_type{}, std::false_type{});
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace

// What a form of tiles costs a CU: every workgroup `tile` and for each 256 bytes of a
// row `stage`, and the first one `first` a stage that nothing overlaps with. The unit
// is a tenth of the stage of a tile of 64 rows by 128 weight rows. Only the ratios
// count: of products of 30 us and more a unit was 0.08 us at the median (MXFP4 by bf16
// 0.05), half of them within a third of that.
struct TileCost {
  int width, rows;
  double first, stage, tile;
};
constexpr TileCost kTileCosts[3][4] = {
    {{4, 128, 7, 25, 44}, {2, 128, 6.7, 14, 47}, {2, 64, 2.7, 10, 7}, {2, 32, 0.9, 10.4, 10}},
    {{4, 64, 12.7, 10.4, 49}, {2, 64, 3.3, 10, 12}, {2, 32, 2.9, 5.1, 6.6}, {}},
    {{4, 128, 9.6, 29.6, 62}, {2, 128, 7.1, 16.6, 34}, {2, 64, 4.2, 10, 13}, {2, 32, 3.4, 10.2, 16}}};
// What this kernel costs with 16 or 32 rows a workgroup: `chunk` for each chunk of a
// wavefront, and for each turn of workgroups over the CUs `turn` and for each chunk
// `turn_chunk`; of all that `start`.
struct RowsCost {
  double chunk, turn_chunk, turn;
};
constexpr RowsCost kRowsCosts[3][2] = {
    {{4.6, 9.4, 57}, {4.2, 27, 16}}, {{4.7, 6.5, 26}, {9.9, 12, 12}}, {{1.3, 2.6, 36}, {2.2, 6.6, 16}}};
constexpr double kRowsStart[3] = {-13, -24, -27};
// The launch that joins shares of the columns, and a value of them.
constexpr double kJoin[2] = {135, 92}, kJoinValue[2] = {5e-5, 2e-5};

// "t4-128/1": tiles of 128 rows by 64 * 4 weight rows, the columns in one share;
// "r2/4": this kernel with 16 * 2 rows, the columns shared by four wavefronts.
ExpertPlan named_form(const char* name) {
  ExpertPlan r{};
  r.tiles = std::sscanf(name, "t%d-%d/%zu", &r.width, &r.rows, &r.splits) == 3;
  if (r.tiles) return r;
  if (std::sscanf(name, "r%d/%d", &r.width, &r.shares) != 2) return ExpertPlan{};
  r.rows = 16 * r.width;
  r.splits = 1;
  return r;
}

// The costs were fitted to 1600 products (1 to 256 experts or one matrix, 1 to 8192
// tokens) timed in every form that the kernels have, by such a search as
// perf/experts_forms.py makes. Of 1600 others, drawn anew, the form that is taken was
// 4% slower than the fastest of all on the mean, 14% at the 95th percentile and 46% at
// most: groups of 15 rows by 729 x 6304 in bf16, tiles of 32 rows where 128 rows with
// the columns in two shares take 31 us in place of 46. (17 rows of one matrix, 4751 x
// 5872, take 16 rows a workgroup and two wavefronts, 22 us; 32 and four take 16.) Some of
// both sides, microseconds, tokens x columns x weight rows of one matrix in bf16: 4096 x
// 2048 x 2048 by tiles of 128 x 256 41, by 64 x 128 49; 1536 x 2048 x 2048 33 and 23;
// 384 x 4096 x 512 by 32 x 128 17, with the columns in two shares 14; 100 x 6144 x 1024
// by 32 x 128 23, in four shares 13, by this kernel 12. Down of 640 tokens of 8 of 64
// experts, 2048 x 768, MXFP4 by MXFP4, by 128 x 256 33, by 64 x 128 27; gate and up of
// 1024 tokens of 10 of 128 experts, 1536 x 4096, MXFP4 by bf16, by 32 x 128 327, by 64 x
// 256 293.
ExpertPlan plan_product(const ExpertProduct& q) {
  const ExpertMat& m = q.m[0];
  const bool xfp4 = q.x_scales != nullptr;
  const int form = !m.fp4 ? 0 : !xfp4 ? 1 : 2;
  ExpertPlan r{};
  r.splits = 1;
  // experts that the rows reach if each picks one by chance, and rows of one
  const double E = double(m.experts), A = double(q.A), N = double(m.rows) * q.mats;
  const double K = double(m.cols);
  const double used = q.offsets ? E * (1.0 - std::pow(1.0 - 1.0 / E, A)) : 1.0;
  const double rows = A / used;
  // workgroups of tiles of so many rows by 64 * width weight rows, the last tile of an
  // expert counted as `part` of one
  auto tiles = [&](int width, double height, double part) {
    const double n = q.offsets ? used * std::max(1.0, rows / height + (rows > height / 2 ? part : 0.0))
                               : std::ceil(A / height);
    return n * std::ceil(N / (64.0 * width));
  };
  const size_t pitch = xfp4 ? m.cols / 2 : m.cols * 2, stages = (pitch + 255) / 256;
  // (tiles copy rows by offsets of 32 bits)
  const bool only_rows = switch_off("INFERNO_EXPERTS_TILES") || q.A / q.k * pitch >= size_t(1) << 32;
  const bool only_tiles = !only_rows && switch_on("INFERNO_EXPERTS_TILES");
  const char* name = std::getenv("INFERNO_EXPERTS_FORM");
  const ExpertPlan named = name ? named_form(name) : ExpertPlan{};
  double least = 0;
  auto offer = [&](double time, bool by_tiles, int width, int height, int shares, size_t splits) {
    if (name && (named.tiles != by_tiles || named.width != width || named.rows != height ||
                 named.shares != shares || named.splits != splits))
      return;
    if (r.width && time >= least) return;
    least = time;
    r = ExpertPlan{by_tiles, width, height, shares, splits};
  };

  if (q.offsets && rows <= 8 && !only_tiles && !name) {
    // The weights' bytes bound it, the kernels differ by what each CU has on its way.
    // With enough workgroups of the lowest tiles these win (64 tokens of 8 of 64 experts,
    // gate and up 768 x 2048 in MXFP4 by bf16: 22 against 32 us; 8 tokens: both 18),
    // with fewer this kernel, which needs no barrier between stages (4 tokens in bf16:
    // 30 against 33).
    if (only_rows || tiles(2, 32, 0.5) < 384) {
      // wavefronts on the same weights where that makes workgroups enough, or shortens
      // long rows (one token of 8 of 64 experts, gate and up 768 x 2048 in bf16: 15.5
      // with one, 12 with two, 12.5 with four; 4 tokens 34.5, 30 and 27)
      const double mine = used * std::ceil(N / 32);
      r.width = 1;
      r.shares = mine < 256 || (mine < 1024 && K >= 2048) ? 4 : K >= 1536 ? 2 : 1;
      return r;
    }
  } else if (!only_tiles) {
    for (int width = 1; width <= 2; ++width)
      for (int shares = 1; shares <= 4; shares *= 2) {
        const RowsCost& c = kRowsCosts[form][width - 1];
        const double chunks = std::ceil(K / (128.0 * shares));
        const double turns =
            std::ceil(used * std::ceil(rows / (16.0 * width)) * std::ceil(N * shares / 128) / kCUs);
        offer(kRowsStart[form] + c.chunk * chunks + turns * (c.turn_chunk * chunks + c.turn), false, width,
              16 * width, shares, 1);
      }
    if (only_rows) return r;
  }
  // Shares of the columns, of twelve stages or more, where the workgroups are few. (Rows
  // in MXFP4 have four times the columns in a stage: 12288 for two shares.)
  for (const TileCost& c : kTileCosts[form]) {
    for (size_t splits = 1; c.width && splits <= 8; splits *= 2) {
      if (splits > 1 && (xfp4 || c.width > 2 || splits * 12 > stages)) break;
      const double n = tiles(c.width, c.rows, xfp4 ? 0.3 : 0.7) * double(splits) / kCUs;
      const double turns = q.offsets ? std::max(1.0, n) : std::ceil(n);
      const double mine = std::ceil(double(stages) / double(splits));
      const double join = splits > 1 ? kJoin[m.fp4] + kJoinValue[m.fp4] * double(splits) * A * N : 0;
      offer(c.first * mine + turns * (c.stage * mine + c.tile) + join, true, c.width, c.rows, 0, splits);
    }
  }
  return r;
}

size_t product_workspace(const ExpertProduct& q, const ExpertPlan& r) {
  return r.splits > 1 ? r.splits * q.mats * q.A * ((q.m[0].rows + 3) / 4 * 16) : 0;
}

int launch_expert_product(hipStream_t s, const ExpertProduct& q, const ExpertPlan& plan) {
  Product p{};
  const ExpertMat& m = q.m[0];
  const ExpertLayout l = expert_layout(m);
  for (int i = 0; i < q.mats; ++i) {
    p.w[i] = static_cast<const uint8_t*>(q.m[i].data);
    p.ws[i] = reinterpret_cast<const uint32_t*>(p.w[i] + l.scales);
  }
  p.x = static_cast<const uint8_t*>(q.x);
  p.xs = q.x_scales;
  p.offsets = q.offsets;
  p.sorted = q.sorted;
  p.E = uint32_t(m.experts);
  p.A = uint32_t(q.A);
  p.k = uint32_t(q.k);
  p.per_k = q.k > 1 ? uint32_t((size_t(1) << 32) / q.k + 1) : 0;
  p.N = uint32_t(m.rows);
  p.K = uint32_t(m.cols);
  p.tiles = uint32_t(l.tiles);
  p.steps = uint32_t(l.steps);
  p.quads = uint32_t(l.quads);
  p.out = q.out;
  p.out_f32 = q.out_dtype == INFERNO_F32;
  auto tiles_of = [&](size_t rows) {
    return q.offsets ? q.A / rows + std::min(m.experts, q.A) : (q.A + rows - 1) / rows;
  };
  const bool xfp4 = q.x_scales != nullptr;
  const size_t x_bytes = q.A / q.k * (xfp4 ? m.cols / 2 : m.cols * 2);
  p.x_bytes = uint32_t(x_bytes);
  p.splits = uint32_t(plan.splits);
  p.partial = static_cast<float*>(q.workspace);
  if (plan.tiles) return launch_experts_tiles(s, p, q.mats, m.fp4, xfp4, tiles_of(plan.rows), plan.width, plan.rows);
  const size_t tiles = tiles_of(16 * plan.width);
  auto pick = [&](auto width) -> int {
    constexpr int NB = decltype(width)::value;
    if (plan.shares == 1) return launch<NB, 1>(s, p, q.mats, m.fp4, xfp4, tiles);
    if (plan.shares == 2) return launch<NB, 2>(s, p, q.mats, m.fp4, xfp4, tiles);
    return launch<NB, 4>(s, p, q.mats, m.fp4, xfp4, tiles);
  };
  if (plan.width == 1) return pick(std::integral_constant<int, 1>{});
  return pick(std::integral_constant<int, 2>{});
}

}  // namespace inferno
