// Products of rows grouped by expert, few rows: one or two tiles of 16 weight rows
// (of both matrices) by 16 or 32 grouped rows, the operands straight from memory to registers in the
// order of the matrix instructions.
//
// The weights are the first operand (lane l: row l % 16, quarter l / 16 of the
// columns of a step), the grouped rows the second, so that a lane's four sums
// are four neighbouring values of one result row. Of a workgroup's four wavefronts
// SHARES take the same weight rows and share the columns; they add their sums in
// order through LDS. What bounds it is how many bytes are on their way: every
// wavefront loads kAhead chunks of 128 columns before it uses the first.
#include <cmath>

#include "experts_dev.hpp"

namespace inferno {
namespace {

using namespace experts;

constexpr int kWaves = 4;
constexpr uint32_t kChunk = 128;  // columns

// One chunk's operands of a wavefront, 128 columns.
template <bool WFP4, bool XFP4, int RT, int NB>
struct Chunk {
  uint4 w[RT][WFP4 ? 1 : 4], x[NB][XFP4 ? 1 : 4];
  uint32_t ws[RT], xs[NB];
};

template <bool WFP4, bool XFP4, int MATS, int RT, int NB, int SHARES>
__global__ void __launch_bounds__(kWaves* kWave) experts_rows_kernel(Product p, uint32_t blocks) {
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

template <int RT, int NB, int SHARES>
int launch(hipStream_t s, const Product& p, int mats, bool wfp4, bool xfp4, size_t tiles) {
  const size_t per = kWaves / SHARES * RT / mats;  // weight tiles of a workgroup
  const size_t blocks = (p.tiles + per - 1) / per;
  if (tiles * blocks * (kWaves * kWave) >= size_t(1) << 32) {
    set_error("too many rows for one launch");
    return INFERNO_ERR_INVALID;
  }
  auto go = [&](auto wf, auto xf) {
    constexpr bool W = decltype(wf)::value, X = decltype(xf)::value;
    const unsigned grid = unsigned(tiles * blocks), threads = kWaves * kWave;
    if (mats == 1)
      experts_rows_kernel<W, X, 1, RT, NB, SHARES><<<grid, threads, 0, s>>>(p, unsigned(blocks));
    else if constexpr (RT > 1)
      experts_rows_kernel<W, X, 2, RT, NB, SHARES><<<grid, threads, 0, s>>>(p, unsigned(blocks));
  };
  if (!wfp4) go(std::false_type{}, std::false_type{});
  else if (xfp4) go(std::true_type{}, std::true_type{});
  else go(std::true_type{}, std::false_type{});
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace

// The rules compare sizes that decide: how many rows an expert has, how many
// workgroups a form makes, and how much each of them has to do. Times are
// microseconds of one call, this kernel against the other or one form of tiles
// against another.
ExpertPlan plan_product(const ExpertProduct& q) {
  const ExpertMat& m = q.m[0];
  const bool xfp4 = q.x_scales != nullptr, widened = m.fp4 && !xfp4;
  ExpertPlan r{};
  r.splits = 1;
  // experts that the rows reach if each picks one by chance, and rows of one
  const double E = double(m.experts), A = double(q.A), N = double(m.rows) * q.mats;
  const double K = double(m.cols);
  const double used = q.offsets ? E * (1.0 - std::pow(1.0 - 1.0 / E, A)) : 1.0;
  const double rows = A / used;
  // workgroups of tiles of so many rows by 64 * width weight rows, and of this
  // kernel's narrow form with all wavefronts on one pair of weight tiles
  auto tiles = [&](int width, double height) {
    const double n = q.offsets ? used * std::max(1.0, rows / height + (rows > height / 2 ? 0.5 : 0.0))
                               : std::ceil(A / height);
    return n * std::ceil(N / (64.0 * width));
  };
  const double groups = std::ceil(rows / 16) * used * std::ceil(N / 32);
  const size_t pitch = xfp4 ? m.cols / 2 : m.cols * 2, stages = (pitch + 255) / 256;

  // This kernel reads every row again for 32 weight rows, tiles have four wavefronts
  // wait for each other. With enough workgroups of the lowest tiles these win (8 tokens
  // of 8 of 64 experts, gate and up 768 x 2048 in bf16: 44 against 53 us); with fewer
  // as soon as this kernel's have much to do (64 tokens by 6144 x 2048 in bf16: 15
  // against 13 us, two such matrices 19 against 21).
  const bool many = tiles(2, 32) >= 384;
  r.tiles = many || (rows > 8 && groups * K > (q.offsets || rows > 32 ? 1.5e6 : 2e6));
  if (switch_on("INFERNO_EXPERTS_TILES")) r.tiles = true;
  if (switch_off("INFERNO_EXPERTS_TILES") || q.A / q.k * pitch >= size_t(1) << 32) r.tiles = false;
  if (!r.tiles) {
    r.width = rows > 64 ? 2 : 1;
    const double mine = groups / r.width;
    r.shares = mine < 256 || (mine < 1024 && K >= 2048) ? 4 : K >= 1536 ? 2 : 1;
    return r;
  }
  // The largest tiles of which there are enough; then, where a workgroup's columns are
  // long, shares of them. Experts have uneven numbers of rows, so that a tile holds
  // twice their mean, or fills the CUs with workgroups.
  double most = 0;  // workgroups up to which shares are doubled
  if (!m.fp4) {
    most = 192;
    if (q.offsets) {
      r.width = rows > 64 && tiles(4, 128) >= 384 ? 4 : 2;
      r.rows = r.width == 4                                                  ? 128
               : rows <= 12                                                  ? 32
               : rows <= 28 || (rows > 80 && tiles(2, 128) < 384)            ? 64
                                                                             : 128;
    } else {
      // (short columns: more workgroups, which start and end while others run)
      const bool brief = m.cols <= 2048;
      r.width = tiles(4, 128) >= (brief ? 512 : 192) ? 4 : 2;
      r.rows = r.width == 4 || (!brief && tiles(2, 128) >= 192) ? 128 : tiles(2, 64) >= 192 ? 64 : 32;
    }
  } else if (widened) {
    most = 256;
    r.width = rows >= 16 && tiles(4, 64) >= 512 ? 4 : 2;
    r.rows = r.width == 4 || (rows >= 32 && tiles(2, 64) >= 512) ? 64 : 32;
  } else {
    r.width = rows >= 64 && tiles(4, 128) >= 500 ? 4 : 2;
    r.rows = r.width == 4 || (K >= 4096 && rows >= 64 && tiles(2, 128) >= 512) ? 128
             : tiles(2, 64) >= 192                                             ? 64
                                                                               : 32;
  }
  if (r.width == 2)
    while (r.splits < 8 && r.splits * 24 <= stages && double(r.splits) * tiles(2, r.rows) <= most)
      r.splits *= 2;
  return r;
}

size_t product_workspace(const ExpertProduct& q) {
  const ExpertPlan r = plan_product(q);
  return r.splits > 1 ? r.splits * q.mats * q.A * ((q.m[0].rows + 3) / 4 * 16) : 0;
}

int launch_expert_product(hipStream_t s, const ExpertProduct& q) {
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
  const ExpertPlan plan = plan_product(q);
  p.splits = uint32_t(plan.splits);
  p.partial = static_cast<float*>(q.workspace);
  if (plan.tiles) return launch_experts_tiles(s, p, q.mats, m.fp4, xfp4, tiles_of(plan.rows), plan.width, plan.rows);
  const size_t tiles = tiles_of(16 * plan.width);
  auto pick = [&](auto width) -> int {
    constexpr int NB = decltype(width)::value;
    if (plan.shares == 1) return launch<2, NB, 1>(s, p, q.mats, m.fp4, xfp4, tiles);
    if (plan.shares == 2) return launch<2, NB, 2>(s, p, q.mats, m.fp4, xfp4, tiles);
    return launch<2, NB, 4>(s, p, q.mats, m.fp4, xfp4, tiles);
  };
  if (plan.width == 1) return pick(std::integral_constant<int, 1>{});
  return pick(std::integral_constant<int, 2>{});
}

}  // namespace inferno
