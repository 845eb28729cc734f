// Products of rows grouped by expert, many rows: tiles of up to 32, 64 or 128 grouped
// rows by 128 or 256 weight rows (of two matrices half each) on 16x16 matrix
// instructions.
//
// Each of four wavefronts owns two or four tiles of 16 weight rows against all rows of
// the tile, so that the weights, packed in the order of the lanes, go from memory to
// registers once per workgroup, four steps ahead, and only the grouped rows, which all
// wavefronts read, go through LDS (copied there directly, two buffers of 256 bytes a
// row). Of the 32 matrix instructions of a step of the largest tile (512 cycles) a
// wavefront reads 8 KB from LDS: half of what LDS delivers. A step is 64 bytes of a row
// for either operand in bf16 (32 columns) and in 4 bits (128 columns); 4-bit weights
// against bf16 rows are widened in registers, four steps from one load. What is left of
// an expert's rows takes the narrowest code of 16, 32, 64 or 128 rows that holds it.
// Where the columns are long and the workgroups few, several share a tile's columns;
// a second launch adds their sums in order.
//
// Measured (a large copy moves 4.94 TB/s here, a large bf16 library product reaches 1.35
// PFLOP/s): gate and up, 1536 x 4096, of 4096 tokens of 10 of 128 experts, MXFP4 by
// bf16, 868 us: 1.19 PFLOP/s, the matrix cores; in bf16 1181 us, 0.87 PFLOP/s. Down, 4096
// x 1536, of 2048 such tokens in bf16 447 us: 1.6 GB of weights and 336 MB of fp32
// results, 4.5 TB/s. Down of 4096 tokens of 8 of 256 experts, 6144 x 2048, MXFP4 by
// MXFP4, 568 us: 1.7 GB and 805 MB, 4.5 TB/s. Where rows are few it is the weights'
// bytes: 512 tokens of those experts' gate and up 579 us, 5.9 TB/s; 64 tokens of 10 of
// 128 in bf16 507 us, 6.1 TB/s. Short columns pay for each tile's start and end: down of
// 5620 tokens of 8 of 64 experts, 2048 x 768 in bf16, 204 us, 0.69 PFLOP/s; of 6863 in
// MXFP4 153 us, 2.0 TB/s.
// Tiles of 256 rows by eight wavefronts were slower, as were results stored past the
// caches.
#include "experts_dev.hpp"

namespace inferno {
namespace {

using namespace experts;

constexpr int kWaves = 4;
constexpr uint32_t kStageBytes = 256;  // of a row in LDS: four steps

typedef __attribute__((address_space(3))) void* lptr_t;

// 16 bytes per lane from off + soff of a buffer to l and the bytes behind it. (As
// a buffer load: behind a global_load_lds the compiler waits for all loads before
// the next use of any.)
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t from, uint32_t off, uint32_t soff,
                                       uint8_t* l) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lptr_t)l, 16, int(off), int(soff), 0, 0);
}

template <bool WFP4, bool XFP4, int MATS, int RT, int NB>
struct Run {
  // 4-bit weights against bf16 rows: a lane's 16 bytes of step j are number 4 g + j of
  // a row's stage, else 4 j + g
  static constexpr bool kWiden = WFP4 && !XFP4;
  static constexpr uint32_t kBuf = NB * 16 * kStageBytes;
  static constexpr int kPerMat = RT / MATS;
  static constexpr int kAhead = kWiden ? 1 : 4;   // steps of weights in registers
  static constexpr int kHalf = NB == 8 ? 4 : NB;  // 16-row groups read from LDS at once
  // loads of weights that a stage issues behind its copies
  static constexpr int kBehind = kWiden ? 2 * RT : 4 * RT;

  const Product& p;
  const Work& t;
  uint32_t first_tile, split;  // weight tiles of a matrix from here; share of the columns
  uint32_t lane, wave, n, g;
  uint32_t pitch;            // bytes of a grouped row
  const uint8_t* wbase[RT];   // of the wavefront's weight tiles
  const uint8_t* sbase[RT];   // of their scales
  uint32_t xrow[NB];         // byte offsets of the rows that this wavefront copies
  __amdgpu_buffer_rsrc_t xbuf;
  uint32_t piece;            // of the lane's 16 bytes of a row's stage (in the first copy)
  floatx4 acc[RT][NB];

  __device__ __forceinline__ Run(const Product& p_, const Work& t_) : p(p_), t(t_) {}

  // weights of step s (from 0; the last again behind it)
  __device__ __forceinline__ uint4 weight(int r, uint32_t s) const {
    return *reinterpret_cast<const uint4*>(wbase[r] + size_t(min(s, p.steps - 1)) * 1024 + lane * 16);
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
      copy16(xbuf, xrow[u] + min(piece ^ ((kWiden ? 16 : 64) * ((wave * NB + u) & 3)), most),
             s * kStageBytes,
             to + (wave * NB + u) * 1024);
  }

  // Scales of MXFP4 rows: the thread's row's sixteen of stage s (0 behind the
  // last, where the codes are zeros). Rows of scales lie at any byte; the last
  // stage takes the last sixteen and moves them.
  __device__ __forceinline__ void load_scales(uint32_t s, const uint8_t* row, uint32_t (&v)[4]) const {
    const uint32_t blocks = p.K / kMxBlock, at = min(s * 16, blocks - 16), by = s * 16 - at;
    __builtin_memcpy(v, row + at, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = __builtin_amdgcn_alignbyte(j < 3 ? v[j + 1] : 0u, v[j], by & 3);
    if (by & 4) v[0] = v[1], v[1] = v[2], v[2] = v[3], v[3] = 0;
    if (by & 8) v[0] = v[2], v[1] = v[3], v[2] = v[3] = 0;
  }
  // The same of the only stage of a row of fewer.
  __device__ __forceinline__ void load_few_scales(const uint8_t* row, uint32_t (&v)[4]) const {
    const uint32_t blocks = p.K / kMxBlock;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = 0;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (4 * j + i < blocks) v[j] |= uint32_t(row[4 * j + i]) << (8 * i);
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
      if constexpr (kWiden) {
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
    const uint32_t x0 =
        n * kStageBytes + 16 * (kWiden ? (4 * g) ^ (n >> 2 | (n & 3) << 2) : g ^ n);
    auto step = [&](auto jc) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      __builtin_amdgcn_sched_barrier(0);  // (registers)
      const uint32_t at = x0 ^ (kWiden ? 16 * j : 64 * j);
      bf16x8 wide[kWiden ? RT : 1];
      if constexpr (kWiden) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint4 c = w[0][r];
          wide[r] = widen(j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w,
                          scale_of((ws[r] >> (8 * (s & 3))) & 255u));
        }
      }
      const uint32_t col = s * kStageBytes + 16 * (kWiden ? 4 * g + j : 4 * j + g);
      const uint32_t keep_x = col < pitch ? ~0u : 0u;  // nothing behind the last column
#pragma unroll
      for (int h = 0; h < NB; h += kHalf) {
        if (h) __builtin_amdgcn_sched_barrier(0);  // (registers)
        uint4 xv[kHalf];
#pragma unroll
        for (int b = 0; b < kHalf; ++b) {
          xv[b] = *reinterpret_cast<const uint4*>(cur + (h + b) * 4096 + at);
          if constexpr (LAST)
            xv[b] = make_uint4(xv[b].x & keep_x, xv[b].y & keep_x, xv[b].z & keep_x, xv[b].w & keep_x);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if constexpr (WFP4 && XFP4) {
            const uint4 v = w[j][r];
            const intx8 av = {int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
#pragma unroll
            for (int b = 0; b < kHalf; ++b) {
              const intx8 bv = {int(xv[b].x), int(xv[b].y), int(xv[b].z), int(xv[b].w), 0, 0, 0, 0};
              acc[r][h + b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                  av, bv, acc[r][h + b], 4, 4, j, int(ws[r]), j, int(xs[h + b]));
            }
          } else {
            bf16x8 a;
            if constexpr (kWiden) {
              a = wide[r];
            } else {
              a = __builtin_bit_cast(bf16x8, w[j][r]);
            }
#pragma unroll
            for (int b = 0; b < kHalf; ++b)
              acc[r][h + b] = mfma_bf16(a, __builtin_bit_cast(bf16x8, xv[b]), acc[r][h + b]);
          }
        }
      }
      if constexpr (!kWiden && !LAST) {
#pragma unroll
        for (int r = 0; r < RT; ++r) w[j][r] = weight(r, 4 * s + 4 + j);
      }
    };
    step(std::integral_constant<int, 0>{});
    if (LAST && !kWiden && 4 * s + 1 >= p.steps) return;
    step(std::integral_constant<int, 1>{});
    if (LAST && !kWiden && 4 * s + 2 >= p.steps) return;
    step(std::integral_constant<int, 2>{});
    if (LAST && !kWiden && 4 * s + 3 >= p.steps) return;
    step(std::integral_constant<int, 3>{});
    if constexpr (!LAST && kWiden) {
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
    first_tile = t.unit / p.splits * (kWaves * kPerMat);
    split = t.unit % p.splits;
    pitch = XFP4 ? p.K / 2 : p.K * 2;
    const uint32_t stages = (pitch + kStageBytes - 1) / kStageBytes;
    const uint32_t first = stages * split / p.splits, last = stages * (split + 1) / p.splits;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int m = r / kPerMat;
      const uint32_t tile = min(first_tile + wave * kPerMat + r % kPerMat, p.tiles - 1);
      const size_t at = size_t(t.e) * p.tiles + tile;
      wbase[r] = p.w[m] + at * p.steps * 1024;
      sbase[r] = reinterpret_cast<const uint8_t*>(p.ws[m]) + at * p.quads * 256;
    }
    // rows behind the tile's last are copied as it is, and not stored
    uint32_t a[NB + 1];
#pragma unroll
    for (int u = 0; u < NB; ++u) a[u] = min(t.c0 + 4 * (wave * NB + u) + g, t.c1 - 1);
    const uint32_t srow = threadIdx.x % (NB * 16);
    a[NB] = min(t.c0 + srow, t.c1 - 1);
    result_rows(p, a);
#pragma unroll
    for (int u = 0; u < NB; ++u) xrow[u] = input_row(p, a[u]) * pitch;  // four rows a copy
    // the 16 pieces of a row lie exclusive-or'ed with its number (kWiden: with the
    // number's halves exchanged), so that the 16 lanes that LDS serves at once,
    // eight of quarter g and eight of the next, touch all banks
    piece = 16 * (n ^ (kWiden ? 4 * g : g));
    xbuf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.x), 0, int(p.x_bytes), 0x00020000);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[r][b] = floatx4{0.f, 0.f, 0.f, 0.f};

    uint8_t* const scales = smem + 2 * kBuf;
    // every thread brings a row's scales, the same row several times if there are
    // fewer rows than threads
    const uint8_t* scale_row = nullptr;
    uint32_t sv[4];
    if constexpr (XFP4) {
      scale_row = p.xs + size_t(input_row(p, a[NB])) * (p.K / kMxBlock);
      if (p.K >= 16 * kMxBlock) load_scales(first, scale_row, sv);
      else load_few_scales(scale_row, sv);
    }
    uint4 w[kAhead][RT];
    uint32_t ws[RT], ws_next[RT];
    copy_rows(first, smem + (first & 1) * kBuf);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int r = 0; r < RT; ++r) w[j][r] = weight(r, (kWiden ? 1 : 4) * first + j);
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
    uint32_t to[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) to[b] = min(t.c0 + 16 * b + n, t.c1 - 1);
    if (p.splits == 1) result_rows(p, to);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t c = t.c0 + 16 * b + n;
      if (c >= t.c1) continue;
      if (p.splits > 1) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t at = (first_tile + wave * kPerMat + r % kPerMat) * 16 + 4 * g;
          if (at < p.N)
            *reinterpret_cast<floatx4*>(
                p.partial + partial_row(p, MATS, split, r / kPerMat, c) + at) = acc[r][b];
        }
        continue;
      }
      if (to[b] >= p.A) continue;
#pragma unroll
      for (int r = 0; r < kPerMat; ++r) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[i] = MATS == 2 ? silu_mul(acc[r][b][i], acc[r + RT - kPerMat][b][i]) : acc[r][b][i];
        store4(p, to[b], (first_tile + wave * kPerMat + r) * 16 + 4 * g, y);
      }
    }
  }
};

template <bool WFP4, bool XFP4, int MATS, int RT, int NB>
__global__ void __launch_bounds__(kWaves* kWave) __attribute__((amdgpu_waves_per_eu(NB == 8 ? 2 : NB == 4 ? 3 : 4)))
    experts_tiles_kernel(Product p, uint32_t blocks) {
  extern __shared__ __attribute__((aligned(16))) uint8_t tile_shared[];
  Work t;
  if (!find_work<NB * 16, true>(p, blockIdx.x, blocks * p.splits, t)) return;
  const uint32_t rows = t.c1 - t.c0;
  if (rows <= 16) return Run<WFP4, XFP4, MATS, RT, 1>(p, t)(tile_shared);
  if (rows <= 32) return Run<WFP4, XFP4, MATS, RT, 2>(p, t)(tile_shared);
  if constexpr (NB > 2)
    if (rows <= 64) return Run<WFP4, XFP4, MATS, RT, 4>(p, t)(tile_shared);
  if constexpr (NB > 4) Run<WFP4, XFP4, MATS, RT, 8>(p, t)(tile_shared);
}

// The sums of the shares in order, and what follows a product: one thread per four
// values of a grouped row. Latency bounds it: 100 rows of 512 in eight shares take 2.8
// us with all loads at once, 4.4 with one after the other.
template <int MATS, int SPLITS>
__global__ void __launch_bounds__(256) experts_join_kernel(Product p, uint32_t quarter) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, c = i / quarter, n = (i - c * quarter) * 4;
  if (c >= p.A) return;
  floatx4 part[MATS][SPLITS];
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int v = 0; v < SPLITS; ++v)
      part[m][v] = *reinterpret_cast<const floatx4*>(p.partial + partial_row(p, MATS, v, m, c) + n);
  const uint32_t a = p.sorted ? p.sorted[c] : c;
  if (p.offsets && (c < p.offsets[0] || c >= p.offsets[p.E])) return;
  if (a >= p.A) return;
  floatx4 sum[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    sum[m] = part[m][0];
#pragma unroll
    for (int v = 1; v < SPLITS; ++v) sum[m] += part[m][v];
  }
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = MATS == 2 ? silu_mul(sum[0][i], sum[MATS - 1][i]) : sum[0][i];
  store4(p, a, n, y);
}

template <int SPLITS>
void join(hipStream_t s, const Product& p, int mats) {
  const uint32_t quarter = (p.N + 3) / 4;
  const unsigned n = unsigned((size_t(p.A) * quarter + 255) / 256);
  if (mats == 2) experts_join_kernel<2, SPLITS><<<n, 256, 0, s>>>(p, quarter);
  else experts_join_kernel<1, SPLITS><<<n, 256, 0, s>>>(p, quarter);
}

template <bool WFP4, bool XFP4, int RT, int NB>
int launch(hipStream_t s, const Product& p, int mats, size_t tiles) {
  const size_t per = kWaves * RT / mats;  // weight tiles of a workgroup
  const size_t blocks = ((p.N + 15) / 16 + per - 1) / per;
  const size_t lds = 2 * NB * 16 * (kStageBytes + (XFP4 ? 16 : 0));
  const size_t grid = (tiles * blocks * p.splits + 7) / 8 * 8;  // each XCD the same number
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
    return INFERNO_OK;
  };
  return mats == 2 ? go(experts_tiles_kernel<WFP4, XFP4, 2, RT, NB>)
                   : go(experts_tiles_kernel<WFP4, XFP4, 1, RT, NB>);
}

}  // namespace

int launch_experts_tiles(hipStream_t s, const Product& p, int mats, bool wfp4, bool xfp4,
                         size_t tiles, int width, int rows) {
  int st;
  if (!wfp4) {
    st = width == 4    ? launch<false, false, 4, 8>(s, p, mats, tiles)
         : rows == 128 ? launch<false, false, 2, 8>(s, p, mats, tiles)
         : rows == 64  ? launch<false, false, 2, 4>(s, p, mats, tiles)
                       : launch<false, false, 2, 2>(s, p, mats, tiles);
  } else if (!xfp4) {
    st = width == 4   ? launch<true, false, 4, 4>(s, p, mats, tiles)
         : rows == 64 ? launch<true, false, 2, 4>(s, p, mats, tiles)
                      : launch<true, false, 2, 2>(s, p, mats, tiles);
  } else {
    st = width == 4    ? launch<true, true, 4, 8>(s, p, mats, tiles)
         : rows == 128 ? launch<true, true, 2, 8>(s, p, mats, tiles)
         : rows == 64  ? launch<true, true, 2, 4>(s, p, mats, tiles)
                       : launch<true, true, 2, 2>(s, p, mats, tiles);
  }
  if (st || p.splits == 1) return st;
  if (p.splits == 2) join<2>(s, p, mats);
  else if (p.splits == 4) join<4>(s, p, mats);
  else join<8>(s, p, mats);
  INF_LAUNCHED();
  return INFERNO_OK;
}

}  // namespace inferno
