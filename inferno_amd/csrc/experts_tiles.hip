// Products of rows grouped by expert, many rows: tiles of up to 128 grouped rows
// by 256 weight rows (128 gate and 128 up) on 16x16 matrix instructions.
//
// A wavefront owns four tiles of 16 weight rows against all rows of the tile, so
// that the weights go from memory to registers once per workgroup, four steps
// ahead, and only the grouped rows, which all four wavefronts read, go through
// LDS (copied there directly, two buffers of 256 bytes a row). Of every 32
// matrix instructions of a step (512 cycles) a wavefront reads 8 KB from LDS: half
// of what LDS delivers. A step is 64 bytes of a row for either operand in bf16 (32
// columns) and in 4 bits (128 columns); 4-bit weights against bf16 rows are
// widened in registers, four steps from one load.
// Tiles are cut at 128 rows, what is left takes the narrowest form of 16, 32, 64
// or 128 rows that holds it.
#include "experts_dev.hpp"

namespace inferno {
namespace {

using namespace experts;

constexpr int kWaves = 4;
constexpr uint32_t kRows = 128;      // grouped rows of a tile
constexpr uint32_t kStageBytes = 256;  // of a row in LDS: four steps

typedef __attribute__((address_space(3))) void* lptr_t;

// 16 bytes per lane from off + soff of a buffer to l and the bytes behind it. (As
// a buffer load: behind a global_load_lds the compiler waits for all loads before
// the next use of any.)
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t from, uint32_t off, uint32_t soff,
                                       uint8_t* l) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lptr_t)l, 16, int(off), int(soff), 0, 0);
}

struct Tile {
  uint32_t e, c0, c1;  // expert, grouped rows
  uint32_t first;      // of the workgroup's 16-row weight tiles
  uint32_t split;      // which share of the columns
};

template <bool WFP4, bool XFP4, int MATS, int RT, int NB>
struct Run {
  static constexpr uint32_t kBuf = NB * 16 * kStageBytes;
  static constexpr int kPerMat = RT / MATS;
  // steps that weights are ahead: what the registers beside 128 rows' sums hold
  static constexpr int kAhead = WFP4 && !XFP4 ? 1 : NB * RT == 32 ? 2 : 4;
  // loads of weights that a stage issues behind its copies
  static constexpr int kBehind = WFP4 && !XFP4 ? 2 * RT : 4 * RT;

  const Product& p;
  const Tile& t;
  uint32_t lane, wave, n, g;
  uint32_t steps;            // of 64 bytes of a weight row (or a chunk)
  uint32_t pitch;            // bytes of a grouped row
  const uint8_t* wbase[RT];   // of the wavefront's weight tiles
  const uint8_t* sbase[RT];   // of their scales
  uint32_t woff[RT];          // bf16: of the lane's row
  uint32_t glast;            // bf16: of its columns in the last step, the first ones if it has none
  uint32_t xrow[NB];         // byte offsets of the rows that this wavefront copies
  __amdgpu_buffer_rsrc_t xbuf;
  uint32_t piece;            // of the lane's 16 bytes of a row's stage (in the first copy)
  floatx4 acc[RT][NB];

  __device__ __forceinline__ Run(const Product& p_, const Tile& t_) : p(p_), t(t_) {}

  // weights of step s (from 0; the last again behind it)
  __device__ __forceinline__ uint4 weight(int r, uint32_t s) const {
    const uint32_t at = min(s, steps - 1);
    if constexpr (WFP4) {
      return *reinterpret_cast<const uint4*>(wbase[r] + size_t(at) * 1024 + lane * 16);
    } else {
      const uint32_t off = woff[r] + (at == steps - 1 ? glast : 16 * g);
      return *reinterpret_cast<const uint4*>(wbase[r] + size_t(at) * 64 + off);
    }
  }
  __device__ __forceinline__ uint32_t weight_scale(int r, uint32_t quad) const {
    return reinterpret_cast<const uint32_t*>(sbase[r] + size_t(min(quad, p.quads - 1)) * 256)[lane];
  }

  // The rows' bytes of stage s to LDS. Without a branch, so that the loads around
  // it can be counted; behind the last column come other bytes of the row, which
  // the last stage masks.
  __device__ __forceinline__ void copy_rows(uint32_t s, uint8_t* __restrict__ to) const {
    const uint32_t most = min(pitch - s * kStageBytes, kStageBytes) - 16;
#pragma unroll
    for (int u = 0; u < NB; ++u)
      copy16(xbuf, xrow[u] + min(piece ^ (64 * ((wave * NB + u) & 3)), most), s * kStageBytes,
             to + (wave * NB + u) * 1024);
  }

  // Scales of MXFP4 rows: the thread's row's sixteen of stage s (0 behind the
  // last, where the codes are zeros). Rows of scales lie at any byte.
  __device__ __forceinline__ void load_scales(uint32_t s, const uint8_t* row, uint32_t (&v)[4]) const {
    const uint32_t blocks = p.K / kMxBlock;
    if (blocks < 4) {
      v[0] = row[0];
      if (blocks > 1) v[0] |= uint32_t(row[1]) << 8;
      if (blocks > 2) v[0] |= uint32_t(row[2]) << 16;
      v[1] = v[2] = v[3] = 0;
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = s * 16 + 4 * j, at = min(b, blocks - 4), shift = 8 * (b - at);
      uint32_t u;
      __builtin_memcpy(&u, row + at, 4);
      v[j] = shift < 32 ? u >> shift : 0;
    }
  }
  // From four words of four blocks, one a step, to one word per block of a step.
  __device__ __forceinline__ static uint4 transpose(const uint32_t (&v)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u);  // 0.0 1.0 0.1 1.1
    const uint32_t b = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u);
    const uint32_t d = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
    return make_uint4(__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u),
                      __builtin_amdgcn_perm(d, b, 0x05040100u), __builtin_amdgcn_perm(d, b, 0x07060302u));
  }

  // One stage: the copies of the next one, then four steps over this one.
  template <bool LAST>
  __device__ __forceinline__ void stage(uint32_t s, uint8_t* __restrict__ next,
                                        const uint8_t* __restrict__ cur,
                                        const uint8_t* __restrict__ cur_scales, uint4 (&w)[kAhead][RT],
                                        uint32_t (&ws)[RT]) {
    uint4 w_next[RT];
    uint32_t ws_next[RT];
    if constexpr (!LAST) {
      copy_rows(s + 1, next);
      asm volatile("" ::: "memory");  // the loads below are younger
      if constexpr (WFP4 && !XFP4) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          w_next[r] = weight(r, s + 1);
          ws_next[r] = weight_scale(r, (s + 1) / 4);
        }
      }
    }
    uint32_t xs[NB];
    if constexpr (XFP4) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
        xs[b] = *reinterpret_cast<const uint32_t*>(cur_scales + (b * 16 + n) * 16 + g * 4);
    }
    const uint32_t x0 = n * kStageBytes + 16 * ((WFP4 && !XFP4 ? 4 * g : g) ^ n);
    auto step = [&](auto jc) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      __builtin_amdgcn_sched_barrier(0);  // (registers)
      const uint32_t at = x0 ^ (WFP4 && !XFP4 ? 16 * j : 64 * j);
      uint4 xv[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
        xv[b] = *reinterpret_cast<const uint4*>(cur + b * 4096 + at);
      if constexpr (LAST) {  // nothing behind the last column
        const uint32_t col = s * kStageBytes + 16 * (WFP4 && !XFP4 ? 4 * g + j : 4 * j + g);
        const uint32_t keep = col < pitch ? ~0u : 0u;
#pragma unroll
        for (int b = 0; b < NB; ++b)
          xv[b] = make_uint4(xv[b].x & keep, xv[b].y & keep, xv[b].z & keep, xv[b].w & keep);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if constexpr (WFP4 && XFP4) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const intx8 av = {int(w[j % kAhead][r].x), int(w[j % kAhead][r].y), int(w[j % kAhead][r].z), int(w[j % kAhead][r].w), 0, 0, 0, 0};
            const intx8 bv = {int(xv[b].x), int(xv[b].y), int(xv[b].z), int(xv[b].w), 0, 0, 0, 0};
            acc[r][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                av, bv, acc[r][b], 4, 4, j, int(ws[r]), j, int(xs[b]));
          }
        } else {
          bf16x8 a;
          if constexpr (WFP4) {
            const uint4 c = w[0][r];
            a = widen(j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w,
                      scale_of((ws[r] >> (8 * (s & 3))) & 255u));
          } else {
            uint4 v = w[j % kAhead][r];
            if constexpr (LAST) {  // nothing behind the last column
              const uint32_t keep = (4 * s + j) * 32 + 8 * g < p.K ? ~0u : 0u;
              v = make_uint4(v.x & keep, v.y & keep, v.z & keep, v.w & keep);
            }
            a = __builtin_bit_cast(bf16x8, v);
          }
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[r][b] = mfma_bf16(a, __builtin_bit_cast(bf16x8, xv[b]), acc[r][b]);
        }
      }
      if constexpr (!(WFP4 && !XFP4) && (!LAST || j + kAhead < 4)) {
#pragma unroll
        for (int r = 0; r < RT; ++r) w[j % kAhead][r] = weight(r, 4 * s + j + kAhead);
      }
    };
    step(std::integral_constant<int, 0>{});
    if (LAST && !(WFP4 && !XFP4) && 4 * s + 1 >= steps) return;
    step(std::integral_constant<int, 1>{});
    if (LAST && !(WFP4 && !XFP4) && 4 * s + 2 >= steps) return;
    step(std::integral_constant<int, 2>{});
    if (LAST && !(WFP4 && !XFP4) && 4 * s + 3 >= steps) return;
    step(std::integral_constant<int, 3>{});
    if constexpr (!LAST && WFP4 && !XFP4) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        w[0][r] = w_next[r];
        ws[r] = ws_next[r];
      }
    }
  }

  __device__ __forceinline__ void operator()(uint8_t* smem) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    n = lane & 15;
    g = lane >> 4;
    pitch = XFP4 ? p.K / 2 : p.K * 2;
    steps = WFP4 ? p.chunks : (p.K + 31) / 32;
    const uint32_t stages = (pitch + kStageBytes - 1) / kStageBytes;
    const uint32_t first = stages * t.split / p.splits, last = stages * (t.split + 1) / p.splits;
    const uint32_t all_tiles = (p.N + 15) / 16;
    glast = (steps - 1) * 32 + 8 * g < p.K ? 16 * g : 0;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int m = r / kPerMat;
      const uint32_t tile = min(t.first + wave * kPerMat + r % kPerMat, all_tiles - 1);
      if constexpr (WFP4) {
        const size_t at = size_t(t.e) * p.tiles + tile;
        wbase[r] = p.w[m] + at * p.chunks * 1024;
        sbase[r] = reinterpret_cast<const uint8_t*>(p.ws[m]) + at * p.quads * 256;
      } else {
        wbase[r] = p.w[m] + (size_t(t.e) * p.N + tile * 16) * p.K * 2;
        woff[r] = min(n, p.N - 1 - tile * 16) * p.K * 2;
      }
    }
    auto input_row = [&](uint32_t row) {
      const uint32_t a = result_row(p, min(t.c0 + row, t.c1 - 1));
      return a < p.A ? a / p.k : 0;  // (of an index out of range no result is written)
    };
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      // four rows a copy; the pieces of a row exclusive-or'ed with it, so that 16
      // rows' reads of one column touch all banks
      xrow[u] = input_row(4 * (wave * NB + u) + g) * pitch;
    }
    piece = 16 * (n ^ g);
    xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.x), 0, int(p.x_bytes), 0x00020000);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[r][b] = floatx4{0.f, 0.f, 0.f, 0.f};

    uint8_t* const scales = smem + 2 * kBuf;
    // every thread brings a row's scales, the same row several times if there are
    // fewer rows than threads
    const uint32_t srow = threadIdx.x % (NB * 16);
    const uint8_t* scale_row = nullptr;
    uint32_t sv[4];
    if constexpr (XFP4) {
      scale_row = p.xs + size_t(input_row(srow)) * (p.K / kMxBlock);
      load_scales(first, scale_row, sv);
    }
    uint4 w[kAhead][RT];
    uint32_t ws[RT], ws_next[RT];
    copy_rows(first, smem + (first & 1) * kBuf);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int r = 0; r < RT; ++r) w[j][r] = weight(r, (WFP4 && !XFP4 ? 1 : 4) * first + j);
    if constexpr (WFP4) {
#pragma unroll
      for (int r = 0; r < RT; ++r) ws[r] = weight_scale(r, XFP4 ? first : first / 4);
    }
    if constexpr (XFP4) {
      *reinterpret_cast<uint4*>(scales + (first & 1) * (NB * 256) + srow * 16) = transpose(sv);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (uint32_t s = first; s + 1 < last; ++s) {
      uint8_t* const cur = smem + (s & 1) * kBuf;
      uint8_t* const next = smem + ((s & 1) ^ 1) * kBuf;
      if constexpr (XFP4) {
        load_scales(s + 1, scale_row, sv);
#pragma unroll
        for (int r = 0; r < RT; ++r) ws_next[r] = weight_scale(r, s + 1);
        stage<false>(s, next, cur, scales + (s & 1) * (NB * 256), w, ws);
        *reinterpret_cast<uint4*>(scales + ((s & 1) ^ 1) * (NB * 256) + srow * 16) = transpose(sv);
#pragma unroll
        for (int r = 0; r < RT; ++r) ws[r] = ws_next[r];
      } else {
        stage<false>(s, next, cur, nullptr, w, ws);
      }
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kBehind) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    {
      const uint32_t s = last - 1;
      stage<true>(s, nullptr, smem + (s & 1) * kBuf, scales + (s & 1) * (NB * 256), w, ws);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t c = t.c0 + 16 * b + n;
      if (c >= t.c1) continue;
      if (p.splits > 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t at = (t.first + wave * kPerMat + r % kPerMat) * 16 + 4 * g;
          if (at < p.N)
            *reinterpret_cast<floatx4*>(
                p.partial + partial_row(p, MATS, t.split, r / kPerMat, c) + at) = acc[r][b];
        }
        continue;
      }
      const uint32_t a = result_row(p, c);
      if (a >= p.A) continue;
#pragma unroll
      for (int r = 0; r < kPerMat; ++r) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = MATS == 2 ? silu_mul(acc[r][b][i], acc[r + RT - kPerMat][b][i]) : acc[r][b][i];
        store4(p, a, (t.first + wave * kPerMat + r) * 16 + 4 * g, y);
      }
    }
  }
};

template <bool WFP4, bool XFP4, int MATS, int RT>
__global__ void __launch_bounds__(kWaves* kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
    experts_tiles_kernel(Product p, uint32_t blocks) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tile_shared[];
  Tile t;
  const uint32_t block = blockIdx.x / p.splits, slot = block / blocks;
  if (slot >= find_tile<kRows>(p, slot, t.e, t.c0, t.c1)) return;
  t.first = (block - slot * blocks) * (kWaves * RT / MATS);
  t.split = blockIdx.x - block * p.splits;
  const uint32_t rows = t.c1 - t.c0;
  if (rows <= 16) Run<WFP4, XFP4, MATS, RT, 1>(p, t)(tile_shared);
  else if (rows <= 32) Run<WFP4, XFP4, MATS, RT, 2>(p, t)(tile_shared);
  else if (rows <= 64) Run<WFP4, XFP4, MATS, RT, 4>(p, t)(tile_shared);
  else Run<WFP4, XFP4, MATS, RT, 8>(p, t)(tile_shared);
}

// The sums of the shares in order, and what follows a product: one thread per four
// values of a grouped row.
template <int MATS>
__global__ void __launch_bounds__(256) experts_join_kernel(Product p, uint32_t quarter) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, c = i / quarter, n = (i - c * quarter) * 4;
  if (c >= p.A) return;
  if (p.offsets && (c < p.offsets[0] || c >= p.offsets[p.E])) return;
  const uint32_t a = result_row(p, c);
  if (a >= p.A) return;
  floatx4 sum[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    const float* at = p.partial + partial_row(p, MATS, 0, m, c) + n;
    const size_t step = partial_row(p, MATS, 1, 0, 0);
    sum[m] = *reinterpret_cast<const floatx4*>(at);
    for (uint32_t v = 1; v < p.splits; ++v) sum[m] += *reinterpret_cast<const floatx4*>(at + v * step);
  }
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = MATS == 2 ? silu_mul(sum[0][i], sum[MATS - 1][i]) : sum[0][i];
  store4(p, a, n, y);
}

template <int RT>
int launch(hipStream_t s, const Product& p, int mats, bool wfp4, bool xfp4, size_t tiles) {
  const size_t per = kWaves * RT / mats;  // weight tiles of a workgroup
  const size_t blocks = ((p.N + 15) / 16 + per - 1) / per;
  const size_t lds = 2 * kRows * kStageBytes + (xfp4 ? 2 * kRows * 16 : 0);
  const size_t grid = tiles * blocks * p.splits;
  if (grid * (kWaves * kWave) >= size_t(1) << 32) {
    set_error("too many rows for one launch");
    return INFERNO_ERR_INVALID;
  }
  auto go = [&](auto kernel) -> int {
    if (lds > 65536)
      INF_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    kernel<<<unsigned(grid), kWaves * kWave, lds, s>>>(p, uint32_t(blocks));
    INF_LAUNCHED();
    if (p.splits > 1) {
      const uint32_t quarter = (p.N + 3) / 4;
      const unsigned n = unsigned((size_t(p.A) * quarter + 255) / 256);
      if (mats == 2) experts_join_kernel<2><<<n, 256, 0, s>>>(p, quarter);
      else experts_join_kernel<1><<<n, 256, 0, s>>>(p, quarter);
      INF_LAUNCHED();
    }
    return INFERNO_OK;
  };
  auto with = [&](auto wf, auto xf) -> int {
    constexpr bool W = decltype(wf)::value, X = decltype(xf)::value;
    return mats == 2 ? go(experts_tiles_kernel<W, X, 2, RT>) : go(experts_tiles_kernel<W, X, 1, RT>);
  };
  if (!wfp4) return with(std::false_type{}, std::false_type{});
  return xfp4 ? with(std::true_type{}, std::true_type{}) : with(std::true_type{}, std::false_type{});
}

}  // namespace

int launch_experts_tiles(hipStream_t s, const Product& p, int mats, bool wfp4, bool xfp4,
                         size_t tiles, int width) {
  return width == 4 ? launch<4>(s, p, mats, wfp4, xfp4, tiles)
                    : launch<2>(s, p, mats, wfp4, xfp4, tiles);
}

}  // namespace inferno
