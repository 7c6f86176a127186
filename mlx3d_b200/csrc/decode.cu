// Gated feature decoder on the 5th-generation tensor cores:
//   g = x Wg^T, u = x Wu^T, h = act(g) * u, y = h Wd^T
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// The hidden values never reach global memory.  A CTA works on tiles of 128
// rows (pixels) and chunks of 64 hidden units; forward and dx walk the chunks
// of a tile, the weight gradients walk the tiles of one chunk and keep their
// sums in TMEM.  All operands are 128-byte-swizzled panels (tc_common.cuh): the
// same panel serves as a K-major and as an MN-major operand, so x, dy and each
// weight are laid out once and never transposed.
//
// Warps have roles: one fetches inputs, one weights, one issues the matrix
// instructions, warpgroups apply the activation, drain and store finished tiles.
#include <cuda.h>

#include "feature_common.cuh"
#include "tc_common.cuh"

namespace gs {

constexpr int kTile = 128;              // rows of a tile (M of the matrix instructions)
constexpr int kChunk = 64;              // hidden units of a chunk
constexpr int kPanel = kTile * 128;     // bytes of a 128-row panel
// Warps of the forward and dx kernel: 0 issues matrix instructions, 1 fetches
// weights, 2 stores tiles, 3 fetches inputs, 4-11 (two warpgroups) activate,
// 12-15 drain finished tiles.  Of the weight-gradient kernel: 0 issues, 1
// fetches, 4-19 (four warpgroups) activate.
constexpr int kDecodeThreads = 512, kEpilogue = 256, kDrain = 128;
constexpr int kDwThreads = 640, kDwEpilogue = 512;
// Tiles of one sum in TMEM, 8 instructions each.  A matrix instruction cuts its products to
// the last bit of a float32 accumulator, always towards zero: a sum of like-signed terms
// loses 2^-22.2 of itself an instruction (measured: 1.4 % of the result after 16384 tiles).
// Longer walks move their sums to 64-bit partial sums every 256 tiles, which leaves 2.1e-4,
// less than half of float16's half step, and costs 1 % of the weight gradients' time for
// 1600x1060 rows, 64-256-152; every 128 tiles 1.1e-4 and 3 %.
constexpr int kSumTiles = 256;
constexpr int kMaxXStages = 4, kMaxWStages = 16;
constexpr uint32_t kTmemCols = 512;
constexpr size_t kMaxSmem = 232448;     // 227 KB

enum { kFwd = 0, kDx = 1, kDw = 2 };

__device__ unsigned long long g_decode_wait_failures;

int decode_wait_failures(unsigned long long* out, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_decode_wait_failures, sizeof(*out));
  if (e == cudaSuccess && reset) {
    const unsigned long long z = 0;
    e = cudaMemcpyToSymbol(g_decode_wait_failures, &z, sizeof(z));
  }
  return (int)e;
}

struct DecodeArgs {
  CUtensorMap map_x, map_dy;  // x and dy in boxes of 128 rows of one panel
  const uint8_t* image;
  void* out;        // y or dx
  void* partials;   // weight gradients: [split][chunk][column of the sums in TMEM][row], float or (wide) double
  int wide;         // some CTA sums over more than kSumTiles tiles
  int64_t n;
  int d, f, c;
  int dp, cp;    // d, c rounded up to 16
  int nxp, nyp;  // 64-element panels of x and dy
  int chunks;
  int chunk_bytes;
  int act;
  int x_stages, w_stages;  // shared-memory stages of inputs and weight chunks
  int out_pitch;           // bytes of a row of the output stage, 0: rows stored from registers
  int out_vec;             // bytes of a store to the output stage
  int out_bulk;            // the output stage is stored by one bulk copy
  int bars_at;             // the barriers' place, behind the stages
};

__host__ __device__ __forceinline__ int round_up(int v, int m) { return (v + m - 1) / m * m; }

// A chunk of the weight image: the gate's and up's 64 hidden units as 128 rows
// (gate first) of ceil(d / 64) panels, then Wd's columns of these hidden units
// as one panel of cp rows.
static int chunk_bytes_of(int d, int c) { return (d + 63) / 64 * kPanel + round_up(c, 16) * tc::kPanelRow; }

// Columns of the weight gradients' sums: 128 rows of [dWg ; dWu] (64 or 128 columns), then
// dWd in blocks of 128 rows and 64 columns.
__host__ __device__ __forceinline__ int dw_columns(int d, int c) { return (d > 64 ? 128 : 64) + (c + 127) / 128 * 64; }

template <typename T>
__global__ void k_decode_prepare(const T* __restrict__ wg, const T* __restrict__ wu, const T* __restrict__ wd, int d,
                                 int f, int c, int chunk_bytes, uint8_t* image) {
  const int nxp = (d + 63) / 64;
  const int j = blockIdx.y;
  uint8_t* out = image + (size_t)j * chunk_bytes;
  const int units = chunk_bytes >> 4;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < units; i += gridDim.x * blockDim.x) {
    int row = i >> 3;
    const int unit = i & 7;
    __align__(16) T v[8];
    const T zero = from_f32<T>(0.0f);
    uint32_t off;
    if (row < nxp * kTile) {
      const int p = row / kTile;
      row -= p * kTile;
      const int h = j * kChunk + (row & 63), d0 = p * 64 + unit * 8;
      const T* w = row < 64 ? wg : wu;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = h < f && d0 + e < d ? w[(size_t)h * d + d0 + e] : zero;
      off = p * kPanel + tc::panel_offset(row, unit);
    } else {
      row -= nxp * kTile;
      const int h0 = j * kChunk + unit * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = row < c && h0 + e < f ? wd[(size_t)row * f + h0 + e] : zero;
      off = nxp * kPanel + tc::panel_offset(row, unit);
    }
    *reinterpret_cast<uint4*>(out + off) = *reinterpret_cast<const uint4*>(v);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fma_sat(float a, float b, float c) {
  float y;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// act(g) of two values and, where wanted, act'(g).  The exponential and the
// reciprocal are the hardware approximations (2 ulp; the results are rounded to
// 16 bits).  The special-function unit (16 a clock and SM) is the other bound,
// so two values share one reciprocal: 1 / a = b * (1 / ab).
//   silu: l = 1 / (1 + 2^t), t = -g log2 e up to 63 so that the product stays
//         finite; 2^-62 is taken off and the result clamped to [0, 1], which
//         makes l zero where t was cut.
//   gelu: Phi(-|g|) = e^(-g^2 / 2) P(t) / 2, t = 1 / (1 + p |g| / sqrt 2), the
//         five-term form of Abramowitz and Stegun, Handbook of Mathematical
//         Functions, 7.1.26 (|error| of erf <= 1.5e-7); its exponential is the
//         density's too.
template <int ACT, bool SLOPE>
__device__ __forceinline__ void gate2(F2 g, F2& a, F2& slope) {
  float g0, g1;
  split(g, g0, g1);
  if (ACT == GS_ACT_SILU) {
    float t0, t1, p0, p1;
    split(mul(g, f2(-1.4426950408889634f)), t0, t1);
    t0 = fminf(t0, 63.0f);
    t1 = fminf(t1, 63.0f);
    const F2 e = f2(ex2(t0), ex2(t1));
    split(add(e, f2(1.0f)), p0, p1);
    const float inv = rcp(p0 * p1);
    const F2 l = f2(fma_sat(inv, p1, -0x1p-62f), fma_sat(inv, p0, -0x1p-62f));
    a = mul(g, l);
    if (SLOPE) slope = fma(a, fma(l, f2(-1.0f), f2(1.0f)), l);
  } else {
    float d0, d1, e0, e1, q0, q1;
    // |g| stops at 1e9 (Phi is 0 or 1 long before): the denominators' product stays finite
    const F2 d = fma(f2(fminf(fabsf(g0), 1e9f), fminf(fabsf(g1), 1e9f)), f2(0.3275911f * 0.70710678118654752f), f2(1.0f));
    split(d, d0, d1);
    const float inv = rcp(d0 * d1);
    const F2 t = f2(inv * d1, inv * d0);
    split(mul(mul(g, g), f2(-0.72134752044448170f)), e0, e1);
    const F2 e = f2(ex2(e0), ex2(e1));  // e^(-g^2 / 2)
    F2 q = fma(t, f2(0.5f * 1.061405429f), f2(0.5f * -1.453152027f));
    q = fma(t, q, f2(0.5f * 1.421413741f));
    q = fma(t, q, f2(0.5f * -0.284496736f));
    q = fma(t, q, f2(0.5f * 0.254829592f));
    split(mul(mul(t, q), e), q0, q1);  // Phi(-|g|)
    const F2 phi = f2(g0 < 0.0f ? q0 : 1.0f - q0, g1 < 0.0f ? q1 : 1.0f - q1);
    a = mul(g, phi);
    if (SLOPE) slope = fma(mul(g, e), f2(0.39894228040143268f), phi);
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(F2 v) {
  float lo, hi;
  split(v, lo, hi);
  return pack2<T>(lo, hi);
}

// ------------------------------------------------------------ shared pieces
// Barriers of a CTA.  A wait that gives up raises `abort`, which makes every
// other wait give up too; the roles then leave their loops, the CTA frees its
// TMEM and returns, and the launch is counted in gs_wait_failures.
struct Bars {
  unsigned long long xfull[kMaxXStages], xempty[kMaxXStages];
  unsigned long long wfull[kMaxWStages], wempty[kMaxWStages];
  unsigned long long gfull[2], hfull[2], dhfull, dhread, sfree;  // sfree: dW's operand stage
  unsigned long long yfull[2], yempty[2];
  unsigned long long ofull, oempty;  // output stage
  uint32_t tmem;
  volatile int abort;
};

__device__ __forceinline__ bool wait_for(Bars* b, unsigned long long* bar, unsigned parity) {
  for (int i = 0; i < (1 << 22); ++i) {
    unsigned done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 15) == 15 && b->abort) return false;
  }
  b->abort = 1;
  return false;
}
// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool passed(unsigned long long* bar, unsigned parity) {
  unsigned done;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(done)
               : "r"(smem_addr(bar)), "r"(parity)
               : "memory");
  return done;
}

// Position in a ring of stages: the stage, and the parity of the phase that
// fills it (a consumer waits for `parity`, a producer for its complement, which
// the first round passes at once).
struct Ring {
  int at = 0;
  unsigned parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++at == stages) {
      at = 0;
      parity ^= 1;
    }
  }
};
__device__ __forceinline__ void arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Panels start on 1024-byte boundaries of shared memory, which the kernels declare
// for their base; a launch where it is not so is counted as failed.
__device__ __forceinline__ bool panels_aligned(const uint8_t* smem) {
  const bool ok = (smem_addr(smem) & 1023) == 0;
  if (!ok && threadIdx.x == 0) atomicAdd(&g_decode_wait_failures, 1ull);
  return ok;
}

__device__ __forceinline__ void init_bars(Bars* b) {
  for (int i = 0; i < kMaxXStages; ++i) {
    mbar_init(&b->xfull[i], 1);
    mbar_init(&b->xempty[i], 1);
  }
  for (int i = 0; i < kMaxWStages; ++i) {
    mbar_init(&b->wfull[i], 1);
    mbar_init(&b->wempty[i], 1);
  }
  for (int i = 0; i < 2; ++i) {
    mbar_init(&b->gfull[i], 1);
    mbar_init(&b->yfull[i], 1);
    mbar_init(&b->yempty[i], kDrain);
  }
  mbar_init(&b->sfree, 1);
  b->abort = 0;
}

// Inputs are fetched by the copy engine, one box of 128 rows x 64 columns per
// panel, with zeros past the last row and column.  It needs rows of a multiple of
// 16 bytes from a 16-byte boundary; other inputs are copied to padded rows first
// (k_pad_rows).  Cutting panel units out of misaligned rows inside this kernel
// cost more than that copy: gathered by loader warps from 4-byte words, from
// shifted 16-byte chunks of a row per thread or exchanged between lanes, 128 rows
// of 150 took 5600 to 10000 cycles, against 1900 for the weight gradients' matrix
// instructions.
__device__ __forceinline__ void fetch_panel(uint8_t* dst, const CUtensorMap* map, int col, int row,
                                            unsigned long long* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(smem_addr(dst)), "l"(map), "r"(col), "r"(row), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void fetch_panels(uint8_t* panels, const CUtensorMap* map, int count, int row,
                                             unsigned long long* bar) {
  for (int p = 0; p < count; ++p) fetch_panel(panels + p * kPanel, map, p * 64, row, bar);
}

// One lane's loop over this CTA's tiles.
template <bool DY>
__device__ __forceinline__ void fetch_inputs(const DecodeArgs& a, Bars* b, uint8_t* stages, int stage_bytes,
                                             int64_t first, int64_t step, int64_t tiles) {
  Ring fill;
  for (int64_t t = first; t < tiles; t += step) {
    if (!wait_for(b, &b->xempty[fill.at], fill.parity ^ 1)) break;
    unsigned long long* full = &b->xfull[fill.at];
    uint8_t* xs = stages + fill.at * stage_bytes;
    mbar_arrive_expect_tx(full, stage_bytes);
    fetch_panels(xs, &a.map_x, a.nxp, (int)(t * kTile), full);
    if (DY) fetch_panels(xs + a.nxp * kPanel, &a.map_dy, a.nyp, (int)(t * kTile), full);
    fill.next(a.x_stages);
  }
}

// COLS hidden units of a thread's row: g, u and (backward) dh from TMEM, then
// h = act(g) u, dg = dh u act'(g), du = dh act(g) as pairs of 16-bit operands.
template <int MODE, int COLS>
struct GateIn {
  uint32_t g[COLS], u[COLS], dh[MODE == kFwd ? 1 : COLS];
  __device__ __forceinline__ void load(uint32_t at_g, uint32_t at_u, uint32_t at_dh) {
    tc::tmem_ld(at_g, g);
    tc::tmem_ld(at_u, u);
    if constexpr (MODE != kFwd) tc::tmem_ld(at_dh, dh);
  }
  __device__ __forceinline__ void settle() {
    tc::tmem_wait_ld();
    tc::after_wait(g);
    tc::after_wait(u);
    if constexpr (MODE != kFwd) tc::after_wait(dh);
  }
  template <typename T, int ACT>
  __device__ __forceinline__ void compute(uint32_t* h, uint32_t* dg, uint32_t* du) const {
#pragma unroll
    for (int e = 0; e < COLS / 2; ++e) {
      F2 act, slope;
      gate2<ACT, MODE != kFwd>(f2(g[2 * e], g[2 * e + 1]), act, slope);
      const F2 uu = f2(u[2 * e], u[2 * e + 1]);
      if constexpr (MODE != kDx) h[e] = pack2<T>(mul(act, uu));
      if constexpr (MODE != kFwd) {
        const F2 d = f2(dh[2 * e], dh[2 * e + 1]);
        dg[e] = pack2<T>(mul(mul(d, uu), slope));
        du[e] = pack2<T>(mul(d, act));
      }
    }
  }
};

// 32 columns of an output row (or `left`, if fewer), in stores of `vec` bytes.  Rows
// of 2-byte alignment are written in words all the same: a row that starts inside one
// (`odd`) stores its columns (2e - 1, 2e) together, `before` being the word of the two
// columns before these (first: there are none), and single columns at its ends: column
// by column, the drain warps held up everything else (forward of 1600x1060 rows,
// 32-128-151: 373 us instead of 262).
__device__ __forceinline__ void store_row32(uint8_t* p, const uint32_t (&w)[16], int left, int vec, bool odd,
                                            uint32_t before, bool first) {
  if (vec == 4 && left >= 32) {  // (the tests below cost as much as the stores)
#pragma unroll
    for (int e = 0; e < 16; ++e) *reinterpret_cast<uint32_t*>(p + 4 * e) = w[e];
  } else if (vec == 16) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (8 * e < left)
        *reinterpret_cast<uint4*>(p + 16 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
  } else if (vec == 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (4 * e < left) *reinterpret_cast<uint2*>(p + 8 * e) = make_uint2(w[2 * e], w[2 * e + 1]);
  } else if (vec == 4) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (2 * e < left) *reinterpret_cast<uint32_t*>(p + 4 * e) = w[e];
  } else {
    // (no branches: lanes of both kinds sit side by side)
    uint8_t* q = odd ? p - 2 : p;
    const uint32_t bytes = odd ? 0x5432 : 0x7654;
    if (odd ? !first : left > 1) *reinterpret_cast<uint32_t*>(q) = __byte_perm(before, w[0], bytes);
    if (odd && first) *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    if (left > 32) {
#pragma unroll
      for (int e = 1; e < 16; ++e) *reinterpret_cast<uint32_t*>(q + 4 * e) = __byte_perm(w[e - 1], w[e], bytes);
    } else {
      const int words = odd ? left : left - 1;
      uint32_t last = w[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) {
        if (2 * e < words) *reinterpret_cast<uint32_t*>(q + 4 * e) = __byte_perm(w[e - 1], w[e], bytes);
        if (2 * e < left) last = w[e];
      }
      if ((left & 1) != (odd ? 1 : 0))
        *reinterpret_cast<uint16_t*>(p + 2 * left - 2) = (uint16_t)(left & 1 ? last : last >> 16);
    }
  }
}

// --------------------------------------------------------- forward and dx
// Per chunk q of the CTA's sequence of (tile, chunk):
//   first products   [g | u] = x [Wg | Wu]^T  (and dh = dy Wd)  -> TMEM buffer q & 1
//   activation       two warpgroups, 32 hidden units each: TMEM -> registers ->
//                    16-bit operands, written over the buffer's own columns
//   second products  y += h Wd^T, or dx += [dg | du] [Wg ; Wu], A from TMEM
// The first products of chunk q + 1 are issued before the second ones of q, so
// the tensor core works while the warpgroups do.  Finished tiles are taken by
// four drain warps, through shared memory to a bulk store: rows straight from
// the registers would write one sector per thread and instruction.
template <typename T, int MODE, int ACT>
__global__ void __launch_bounds__(kDecodeThreads, 1) k_decode(const __grid_constant__ DecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
  constexpr uint32_t kBuf = MODE == kFwd ? 128 : 192;  // TMEM columns of a chunk: g, u (, dh)
  // TMEM: two chunk buffers, then the accumulators of finished tiles
  const int width = MODE == kFwd ? a.c : a.d, wp = MODE == kFwd ? a.cp : a.dp;
  constexpr uint32_t kOut = 2 * kBuf;
  const int nout = wp <= (512 - (int)kOut) / 2 ? 2 : 1;
  const uint32_t out_cols = (512 - kOut) / nout;
  const int stage_bytes = (a.nxp + (MODE == kFwd ? 0 : a.nyp)) * kPanel;
  uint8_t* ws = smem + a.x_stages * stage_bytes;
  uint8_t* os = ws + a.w_stages * a.chunk_bytes;
  Bars* b = reinterpret_cast<Bars*>(smem + a.bars_at);
  if (!panels_aligned(smem)) return;

  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
  if (warp == 0) tc::tmem_alloc(&b->tmem, kTmemCols);
  if (threadIdx.x == 0) {
    init_bars(b);
    for (int i = 0; i < 2; ++i) mbar_init(&b->hfull[i], kEpilogue);
    mbar_init(&b->ofull, kDrain);
    mbar_init(&b->oempty, a.out_bulk ? 1 : kDrain);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = b->tmem;
  const int64_t tiles = (a.n + kTile - 1) / kTile;
  const int64_t mine = (tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;  // tiles of this CTA
  const int64_t total = mine * a.chunks;
  const bool resident = a.w_stages >= a.chunks;

  if (warp == 3) {
    if (lane == 0 && resident) fetch_inputs<MODE != kFwd>(a, b, smem, stage_bytes, blockIdx.x, gridDim.x, tiles);
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && resident) {
      for (int j = 0; j < a.chunks; ++j) {
        mbar_arrive_expect_tx(&b->wfull[j], a.chunk_bytes);
        bulk_g2s(ws + j * a.chunk_bytes, a.image + (size_t)j * a.chunk_bytes, a.chunk_bytes, &b->wfull[j]);
      }
    } else if (lane == 0) {
      // Weights stream through the stages.  The copy engine serves one SM's
      // requests in order, so the next tile's panels are spread over this
      // tile's chunks: fetched at once they would hold up the weights.
      constexpr bool kDy = MODE != kFwd;
      const int panels = a.nxp + (kDy ? a.nyp : 0);
      Ring w, x;
      auto fetch_some = [&](int64_t i, int from, int to) {  // panels [from, to) of this CTA's tile i
        unsigned long long* full = &b->xfull[x.at];
        const int row = (int)((blockIdx.x + i * gridDim.x) * kTile);
        for (int p = from; p < to; ++p) {
          uint8_t* dst = smem + x.at * stage_bytes + p * kPanel;
          const bool dy = p >= a.nxp;
          fetch_panel(dst, dy ? &a.map_dy : &a.map_x, (dy ? p - a.nxp : p) * 64, row, full);
        }
      };
      mbar_arrive_expect_tx(&b->xfull[0], stage_bytes);
      fetch_some(0, 0, panels);
      x.next(a.x_stages);
      bool ok = true;
      for (int64_t i = 0; i < mine && ok; ++i) {
        bool open = false;  // the next tile's stage is free
        int done = 0;
        for (int j = 0; j < a.chunks; ++j) {
          ok = wait_for(b, &b->wempty[w.at], w.parity ^ 1);
          if (!ok) break;
          mbar_arrive_expect_tx(&b->wfull[w.at], a.chunk_bytes);
          bulk_g2s(ws + w.at * a.chunk_bytes, a.image + (size_t)j * a.chunk_bytes, a.chunk_bytes, &b->wfull[w.at]);
          w.next(a.w_stages);
          // with one stage, this tile's first products must all be done first
          if (i + 1 == mine || (a.x_stages == 1 && j + 1 < a.chunks)) continue;
          if (!open) {
            ok = wait_for(b, &b->xempty[x.at], x.parity ^ 1);
            if (!ok) break;
            mbar_arrive_expect_tx(&b->xfull[x.at], stage_bytes);
            open = true;
          }
          const int upto = panels * (j + 1) / a.chunks;
          fetch_some(i + 1, done, upto);
          done = upto;
        }
        x.next(a.x_stages);
      }
    }
    __syncwarp();
  } else if (warp == 0) {
    // This warp's instructions bound short tiles: counters instead of
    // divisions, and all operands of the matrix instructions made uniform
    // before the elected lane issues them.
    Ring x, w1, w2, y;
    int j1 = 0, j2 = 0;
    bool ok = true, wait_w = true;
    const uint32_t id1 = tc::instr_desc(kBf16, 128, false, false), idh = tc::instr_desc(kBf16, 64, false, true);
    const uint32_t id2 = tc::instr_desc(kBf16, wp, false, MODE == kDx);
    const uint32_t x0 = tc::desc_k(smem_addr(smem)), wk0 = tc::desc_k(smem_addr(ws));
    const uint32_t wn0 = tc::desc_mn(smem_addr(ws), kPanel);
    const uint32_t xstep = stage_bytes >> 4, wstep = a.chunk_bytes >> 4, wdn = a.nxp * (kPanel >> 4);
    const int k1 = a.dp / 16, kh = a.cp / 16;
    auto first_products = [&](uint32_t buf_, unsigned long long* done) {
      if (j1 == 0) ok &= wait_for(b, &b->xfull[x.at], x.parity);
      if (wait_w) ok &= wait_for(b, &b->wfull[w1.at], w1.parity);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      tc::fence_after();
      const uint32_t buf = tc::uniform(buf_), xd = tc::uniform(x0 + x.at * xstep);
      const uint32_t wk = tc::uniform(wk0 + w1.at * wstep), wn = tc::uniform(wn0 + w1.at * wstep + wdn);
      const bool last = j1 + 1 == a.chunks;
      if (tc::elect_one()) {
        tc::mma_ss(buf, xd, wk, id1, false);
#pragma unroll
        for (int k = 1; k < GS_DECODE_MAX_D / 16; ++k)
          if (k < k1)
            tc::mma_ss(buf, xd + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, wk + (k >> 2) * (kPanel >> 4) + (k & 3) * 2,
                       id1, true);
        if (MODE == kDx) {
          const uint32_t yd = xd + wdn;
          tc::mma_ss(buf + 128, yd, wn, idh, false);
#pragma unroll
          for (int k = 1; k < GS_DECODE_MAX_C / 16; ++k)
            if (k < kh)
              tc::mma_ss(buf + 128, yd + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, wn + k * 128, idh, true);
        }
        tc::commit(done);
        if (last) tc::commit(&b->xempty[x.at]);
      }
      __syncwarp();
      w1.next(a.w_stages);
      ++j1;
      if (last) {
        x.next(a.x_stages);
        j1 = 0;
        if (resident) wait_w = false;
      }
    };
    first_products(tmem, &b->gfull[0]);
    unsigned qb = 0, qphase = 0;  // chunk's buffer and its phase
    for (int64_t q = 0; q < total && ok; ++q) {
      if (q + 1 < total) first_products(tmem + (qb ^ 1) * kBuf, &b->gfull[qb ^ 1]);
      if (j2 == 0) ok &= wait_for(b, &b->yempty[y.at], y.parity ^ 1);
      ok &= wait_for(b, &b->hfull[qb], qphase);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      tc::fence_after();
      const uint32_t buf = tc::uniform(tmem + qb * kBuf), out = tc::uniform(tmem + kOut + y.at * out_cols);
      const uint32_t wk = tc::uniform(wk0 + w2.at * wstep + wdn), wn = tc::uniform(wn0 + w2.at * wstep);
      const bool last = j2 + 1 == a.chunks, more = __all_sync(~0u, j2 > 0);
      if (tc::elect_one()) {
        if (MODE == kFwd) {
          tc::mma_ts(out, buf, wk, id2, more);
#pragma unroll
          for (int k = 1; k < 4; ++k)  // h in the columns of g, 16 of each 32
            tc::mma_ts(out, buf + (k >> 1) * 32 + (k & 1) * 8, wk + k * 2, id2, true);
        } else {
          tc::mma_ts(out, buf, wn, id2, more);
#pragma unroll
          for (int k = 1; k < 8; ++k)  // dg in the columns of g, du in those of u
            tc::mma_ts(out, buf + (k >> 1) * 32 + (k & 1) * 8, wn + k * 128, id2, true);
        }
        if (!resident) tc::commit(&b->wempty[w2.at]);
        if (last) tc::commit(&b->yfull[y.at]);
      }
      __syncwarp();
      w2.next(a.w_stages);
      ++j2;
      if (last) {
        y.next(nout);
        j2 = 0;
      }
      qb ^= 1;
      if (qb == 0) qphase ^= 1;
    }
    // Every issued instruction has finished when this phase completes.
    if (!ok && tc::elect_one()) tc::commit(&b->sfree);
    __syncwarp();
  } else if (warp == 2) {
    if (a.out_bulk) {  // finished tiles: output stage -> global memory
      uint8_t* out = static_cast<uint8_t*>(a.out);
      const int row_bytes = width * 2;
      for (int64_t i = 0; i < mine; ++i) {
        const int64_t t = blockIdx.x + i * gridDim.x;
        if (!__all_sync(~0u, wait_for(b, &b->ofull, (unsigned)i & 1))) break;
        const int rows = (int)min((int64_t)kTile, a.n - t * kTile);
        uint8_t* dst = out + t * kTile * row_bytes;
        const int bytes = rows * row_bytes & ~15;
        if (lane == 0 && bytes > 0)
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_addr(os)),
                       "r"(bytes)
                       : "memory");
        for (int e = bytes + 2 * lane; e < rows * row_bytes; e += 64)
          *reinterpret_cast<uint16_t*>(dst + e) = *reinterpret_cast<const uint16_t*>(os + e);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive(&b->oempty);
      }
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  } else if (warp >= 12) {  // finished tiles: TMEM -> output stage (or global memory)
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool staged = a.out_pitch > 0;
    Ring y;
    for (int64_t i = 0; i < mine; ++i) {
      bool ok = wait_for(b, &b->yfull[y.at], y.parity);
      if (ok && a.out_bulk) ok = wait_for(b, &b->oempty, (unsigned)(i & 1) ^ 1);
      if (!__all_sync(~0u, ok)) break;
      tc::fence_after();
      const int64_t t = blockIdx.x + i * gridDim.x;
      const uint32_t src = lanes + kOut + y.at * out_cols;
      const bool here = staged || t * kTile + row < a.n;
      uint8_t* p = staged ? os + row * a.out_pitch : static_cast<uint8_t*>(a.out) + (t * kTile + row) * width * 2;
      // Up to 160 columns are read and rounded before any is stored: the next
      // tile's second products wait for the accumulator.
      const bool odd = reinterpret_cast<uintptr_t>(p) & 2;
      uint32_t before = 0;
      for (int c0 = 0; c0 < width; c0 += 160, p += 320) {
        uint32_t w[5][16];
#pragma unroll
        for (int g = 0; g < 5; ++g) {
          if (c0 + 32 * g < width) {
            uint32_t v[32];
            __syncwarp();
            tc::tmem_ld(src + c0 + 32 * g, v);
            tc::tmem_wait_ld();
            tc::after_wait(v);
#pragma unroll
            for (int e = 0; e < 16; ++e) w[g][e] = pack2<T>(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1]));
          }
        }
        if (c0 + 160 >= width) {
          tc::fence_before();
          arrive(&b->yempty[y.at]);
        }
#pragma unroll
        for (int g = 0; g < 5; ++g)
          if (here && c0 + 32 * g < width)
            store_row32(p + 64 * g, w[g], width - c0 - 32 * g, a.out_vec, odd, g > 0 ? w[g > 0 ? g - 1 : 0][15] : before,
                        c0 + g == 0);
        before = w[4][15];
      }
      __syncwarp();
      if (a.out_bulk) {
        tc::fence_async_smem();
        arrive(&b->ofull);
      } else if (staged) {  // padded rows, written by the drain warps themselves in 16-byte units
        arrive(&b->ofull);
        if (!__all_sync(~0u, wait_for(b, &b->ofull, (unsigned)i & 1))) break;
        const int per_row = width >> 3, l = threadIdx.x - 384;
        const int rows = (int)min((int64_t)kTile, a.n - t * kTile);
        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + t * kTile * width * 2);
        int r = l / per_row, u = l - r * per_row;
        const int dr = kDrain / per_row, du = kDrain - dr * per_row;
#pragma unroll 4
        for (int e = l; e < rows * per_row; e += kDrain) {
          dst[e] = *reinterpret_cast<const uint4*>(os + r * a.out_pitch + u * 16);
          r += dr;
          u += du;
          if (u >= per_row) {
            u -= per_row;
            ++r;
          }
        }
        arrive(&b->oempty);
        if (!__all_sync(~0u, wait_for(b, &b->oempty, (unsigned)i & 1))) break;
      }
      y.next(nout);
    }
  } else if (warp >= 4) {  // activation: each warpgroup half of a chunk's hidden units
    const int wg = (warp >> 2) - 1;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    // TMEM loads take about 300 cycles: the next columns, of the next chunk
    // too if it is ready, are on their way while the current ones are computed.
    constexpr int kCols = MODE == kFwd ? 16 : 8, kPasses = 32 / kCols;
    GateIn<MODE, kCols> v[2];
    Ring q;
    bool have = false;
    for (int64_t i = 0; i < total; ++i) {
      const uint32_t buf = lanes + (uint32_t)q.at * kBuf + wg * 32;
      if (!have) {
        if (!__all_sync(~0u, wait_for(b, &b->gfull[q.at], q.parity))) break;
        tc::fence_after();
        v[0].load(buf, buf + 64, buf + 128);
      }
      unsigned long long* full = &b->hfull[q.at];
      q.next(2);
      have = false;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        v[p & 1].settle();
        if (p + 1 < kPasses) {
          v[(p + 1) & 1].load(buf + (p + 1) * kCols, buf + 64 + (p + 1) * kCols, buf + 128 + (p + 1) * kCols);
        } else if (i + 1 < total && __all_sync(~0u, passed(&b->gfull[q.at], q.parity))) {
          tc::fence_after();
          const uint32_t next = lanes + (uint32_t)q.at * kBuf + wg * 32;
          v[0].load(next, next + 64, next + 128);
          have = true;
        }
        uint32_t h[kCols / 2], dg[kCols / 2], du[kCols / 2];
        v[p & 1].template compute<T, ACT>(h, dg, du);
        // over columns of g and u that this warp has read
        if constexpr (MODE == kFwd) {
          tc::tmem_st(buf + p * (kCols / 2), h);
        } else {
          tc::tmem_st(buf + p * (kCols / 2), dg);
          tc::tmem_st(buf + 64 + p * (kCols / 2), du);
        }
      }
      tc::tmem_wait_st();
      tc::fence_before();
      arrive(full);
    }
  }
  __syncthreads();
  if (b->abort) {  // what is in flight must end before the CTA does (bounded)
    if (threadIdx.x == 0) {
      atomicAdd(&g_decode_wait_failures, 1ull);
      mbar_wait(&b->sfree, 0);
      for (unsigned par = 0; par < 2; ++par) {
        for (int i = 0; i < a.w_stages; ++i) mbar_wait(&b->wfull[i], par);
        for (int i = 0; i < a.x_stages; ++i) mbar_wait(&b->xfull[i], par);
      }
    }
    __syncthreads();
  }
  if (warp == 0) tc::tmem_free(tmem, kTmemCols);
}

// --------------------------------------------------------- weight gradients
// A CTA keeps one chunk's weights and walks tiles; per tile
//   [g | u] = x [Wg | Wu]^T, dh = dy Wd         -> TMEM
//   activation (four warpgroups, 16 hidden units each) -> dg, du, h panels in
//                shared memory, rows = pixels
//   [dWg ; dWu] += [dg | du]^T x,  dWd += dy^T h -> TMEM, summed over all tiles
// The panels are K-major for nobody: both operands of the sums over pixels are
// MN-major, x and dy from the same panels the first products read.  The next
// tile's [g | u] is issued before this tile's sums.
template <typename T, int ACT>
__global__ void __launch_bounds__(kDwThreads, 1) k_decode_dw(const __grid_constant__ DecodeArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);
  const int stage_bytes = (a.nxp + a.nyp) * kPanel;
  uint8_t* ws = smem + a.x_stages * stage_bytes;
  uint8_t* st = ws + a.chunk_bytes;  // dg, du, h panels
  Bars* b = reinterpret_cast<Bars*>(smem + a.bars_at);
  if (!panels_aligned(smem)) return;
  const int mblocks = (a.c + 127) / 128;
  const int acc_cols = dw_columns(a.d, a.c);
  const int nbuf = acc_cols <= 192 ? 2 : 1;  // [g | u] buffers
  // TMEM: [g | u] at 0 (and 128), dh, the sums
  const uint32_t col_dh = nbuf * 128, col_gu = col_dh + 64, col_dd = col_gu + (a.dp > 64 ? 128 : 64);

  const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: uniform
  if (warp == 0) tc::tmem_alloc(&b->tmem, kTmemCols);
  if (threadIdx.x == 0) {
    init_bars(b);
    for (int i = 0; i < 2; ++i) mbar_init(&b->hfull[i], kDwEpilogue);
    mbar_init(&b->dhfull, 1);
    mbar_init(&b->dhread, kDwEpilogue);
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = b->tmem;
  const int64_t tiles = (a.n + kTile - 1) / kTile;
  const int64_t mine = (tiles - blockIdx.x + gridDim.x - 1) / gridDim.x;

  if (warp == 1) {
    if (lane == 0) fetch_inputs<true>(a, b, smem, stage_bytes, blockIdx.x, gridDim.x, tiles);
    __syncwarp();
  } else if (warp == 0) {
    bool ok = true;
    if (lane == 0) {
      mbar_arrive_expect_tx(&b->wfull[0], a.chunk_bytes);
      bulk_g2s(ws, a.image + (size_t)blockIdx.y * a.chunk_bytes, a.chunk_bytes, &b->wfull[0]);
    }
    __syncwarp();
    ok = wait_for(b, &b->wfull[0], 0);
    const uint32_t id1 = tc::instr_desc(kBf16, 128, false, false), idh = tc::instr_desc(kBf16, 64, false, true);
    const uint32_t idg = tc::instr_desc(kBf16, a.dp, true, true), idd = tc::instr_desc(kBf16, 64, true, true);
    const uint32_t xstep = stage_bytes >> 4, ypart = a.nxp * (kPanel >> 4);
    const uint32_t xk0 = tc::desc_k(smem_addr(smem)), xn0 = tc::desc_mn(smem_addr(smem), kPanel);
    const uint32_t wk = tc::uniform(tc::desc_k(smem_addr(ws))), sn = tc::uniform(tc::desc_mn(smem_addr(st), kPanel));
    const uint32_t wn = tc::uniform(tc::desc_mn(smem_addr(ws), kPanel) + ypart);
    const int k1 = a.dp / 16, kh = a.cp / 16;
    Ring xg, xh, xs;  // stages of the next [g | u], dh and sums
    unsigned gb = 0;
    auto gu_products = [&]() {
      ok &= wait_for(b, &b->xfull[xg.at], xg.parity);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      tc::fence_after();
      const uint32_t xd = tc::uniform(xk0 + xg.at * xstep), buf = tc::uniform(tmem + gb * 128);
      if (tc::elect_one()) {
        tc::mma_ss(buf, xd, wk, id1, false);
#pragma unroll
        for (int k = 1; k < GS_DECODE_MAX_D / 16; ++k)
          if (k < k1)
            tc::mma_ss(buf, xd + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, wk + (k >> 2) * (kPanel >> 4) + (k & 3) * 2,
                       id1, true);
      }
      __syncwarp();
      xg.next(a.x_stages);
      if (nbuf == 2) gb ^= 1;
    };
    auto dh_products = [&]() {
      const uint32_t yd = tc::uniform(xk0 + xh.at * xstep + ypart), buf = tc::uniform(tmem + col_dh);
      if (tc::elect_one()) {
        tc::mma_ss(buf, yd, wn, idh, false);
#pragma unroll
        for (int k = 1; k < GS_DECODE_MAX_C / 16; ++k)
          if (k < kh) tc::mma_ss(buf, yd + (k >> 2) * (kPanel >> 4) + (k & 3) * 2, wn + k * 128, idh, true);
        tc::commit(&b->dhfull);
      }
      __syncwarp();
      xh.next(a.x_stages);
    };
    gu_products();
    if (ok) dh_products();
    const uint32_t tgu = tc::uniform(tmem + col_gu), tdd = tc::uniform(tmem + col_dd);
    for (int64_t i = 0; i < mine && ok; ++i) {
      // The next tile's first products go before this one's sums as soon as its
      // inputs are there: [g | u] at once with two buffers, else, like dh, when
      // this tile's have been read.
      const bool more_tiles = i + 1 < mine;
      auto ready = [&]() { return more_tiles && __all_sync(~0u, passed(&b->xfull[xg.at], xg.parity)); };
      bool ahead = false;
      if (nbuf == 2 && ready()) {
        gu_products();
        ahead = true;
      }
      ok &= wait_for(b, &b->dhread, (unsigned)i & 1);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      tc::fence_after();
      if (!ahead && ready()) {
        gu_products();
        ahead = true;
      }
      if (ahead) dh_products();
      // its panels are written
      ok &= wait_for(b, &b->hfull[0], (unsigned)i & 1);
      ok = __all_sync(~0u, ok);
      if (!ok) break;
      tc::fence_after();
      if (!ahead && ready()) {
        gu_products();
        dh_products();
        ahead = true;
      }
      const uint32_t xd = tc::uniform(xn0 + xs.at * xstep), yd = xd + ypart;
      const bool more = __all_sync(~0u, i % kSumTiles != 0);
      if (tc::elect_one()) {
        tc::mma_ss(tgu, sn, xd, idg, more);
#pragma unroll
        for (int k = 1; k < 8; ++k) tc::mma_ss(tgu, sn + k * 128, xd + k * 128, idg, true);
        // A dy panel past nyp is other shared memory: it only reaches rows >= c of the sums, which are not read.
        const uint32_t hn = sn + 2 * (kPanel >> 4);
#pragma unroll
        for (int m = 0; m < GS_DECODE_MAX_C / 128; ++m) {
          if (m >= mblocks) break;
          const uint32_t ym = yd + m * 2 * (kPanel >> 4);
          tc::mma_ss(tdd + m * 64, ym, hn, idd, more);
#pragma unroll
          for (int k = 1; k < 8; ++k) tc::mma_ss(tdd + m * 64, ym + k * 128, hn + k * 128, idd, true);
        }
        tc::commit(&b->sfree);
        tc::commit(&b->xempty[xs.at]);
      }
      __syncwarp();
      xs.next(a.x_stages);
      if (!ahead && more_tiles) {
        gu_products();
        if (ok) dh_products();
      }
    }
    if (!ok) {
      mbar_wait(&b->wfull[0], 0);
      if (tc::elect_one()) tc::commit(&b->yfull[0]);
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int wg = (warp >> 2) - 1, row = (warp & 3) * 32 + lane;  // 16 hidden units a thread
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    // The sums in TMEM to this CTA's partial sums (more: added to them), as they lie, so that
    // a warp's 32 rows are neighbours in memory.
    auto put_sums = [&](auto* partials, bool more) {
      tc::fence_after();
      auto* part = partials + ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * dw_columns(a.d, a.c) * kTile + row;
      auto put = [&](int col) {
        uint32_t v[16];
        __syncwarp();
        tc::tmem_ld(lanes + col_gu + col, v);
        tc::tmem_wait_ld();
        tc::after_wait(v);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          auto* to = part + (col + e) * kTile;
          *to = more ? *to + __uint_as_float(v[e]) : __uint_as_float(v[e]);
        }
      };
      for (int c0 = wg * 16; c0 < a.dp; c0 += 64) put(c0);
      for (int m = 0; m < mblocks; ++m) put((int)(col_dd - col_gu) + m * 64 + wg * 16);
      tc::fence_before();
    };
    bool ok = true;
    for (int64_t i = 0; i < mine; ++i) {
      const uint32_t buf = lanes + (nbuf == 2 ? (uint32_t)(i & 1) * 128 : 0) + wg * 16, dhc = lanes + col_dh + wg * 16;
      ok = __all_sync(~0u, wait_for(b, &b->dhfull, (unsigned)i & 1));
      if (!ok) break;
      tc::fence_after();
      uint32_t pg[8], pu[8], ph[8];
      GateIn<kDw, 8> v[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) v[p].load(buf + 8 * p, buf + 64 + 8 * p, dhc + 8 * p);
#pragma unroll
      for (int p = 0; p < 2; ++p) v[p].settle();
      tc::fence_before();
      arrive(&b->dhread);
#pragma unroll
      for (int p = 0; p < 2; ++p) v[p].template compute<T, ACT>(ph + 4 * p, pg + 4 * p, pu + 4 * p);
      // the previous tile's sums have read the panels
      if (i > 0) ok = __all_sync(~0u, wait_for(b, &b->sfree, (unsigned)(i - 1) & 1));
      if (!ok) break;
      // (this tile's sums, which start anew, wait for its panels, hence for these reads)
      if (i > 0 && i % kSumTiles == 0) put_sums(static_cast<double*>(a.partials), i > kSumTiles);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t off = tc::panel_offset(row, wg * 2 + q);
        *reinterpret_cast<uint4*>(st + off) = make_uint4(pg[4 * q], pg[4 * q + 1], pg[4 * q + 2], pg[4 * q + 3]);
        *reinterpret_cast<uint4*>(st + kPanel + off) = make_uint4(pu[4 * q], pu[4 * q + 1], pu[4 * q + 2], pu[4 * q + 3]);
        *reinterpret_cast<uint4*>(st + 2 * kPanel + off) =
            make_uint4(ph[4 * q], ph[4 * q + 1], ph[4 * q + 2], ph[4 * q + 3]);
      }
      tc::fence_async_smem();
      arrive(&b->hfull[0]);
    }
    if (ok && mine > 0) ok = __all_sync(~0u, wait_for(b, &b->sfree, (unsigned)(mine - 1) & 1));
    if (ok && mine > 0) {
      if (a.wide) put_sums(static_cast<double*>(a.partials), mine > kSumTiles);
      else put_sums(static_cast<float*>(a.partials), false);
    }
  }
  __syncthreads();
  if (b->abort) {  // what is in flight must end before the CTA does (bounded)
    if (threadIdx.x == 0) {
      atomicAdd(&g_decode_wait_failures, 1ull);
      mbar_wait(&b->yfull[0], 0);
      for (unsigned par = 0; par < 2; ++par)
        for (int i = 0; i < a.x_stages; ++i) mbar_wait(&b->xfull[i], par);
    }
    __syncthreads();
  }
  if (warp == 0) tc::tmem_free(tmem, kTmemCols);
}

// A few rows of a small block (a picked point, a handful of samples): one launch
// that reads the weights where they are, one block per row, a warp per hidden
// unit and then per output.  h stays in 32 bits.  The matrix path's weight layout
// and pipeline start cost more than this whole call: one row, 32-64-20, 15 us
// from Python instead of 45.
constexpr int kFewThreads = 256;
template <typename T, int ACT>
__global__ void __launch_bounds__(kFewThreads) k_decode_few(const T* __restrict__ x, const T* __restrict__ wg,
                                                            const T* __restrict__ wu, const T* __restrict__ wd, int d,
                                                            int f, int c, T* __restrict__ y) {
  extern __shared__ float few[];
  float *xs = few, *hs = few + d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  x += (size_t)blockIdx.x * d;
  y += (size_t)blockIdx.x * c;
  for (int i = threadIdx.x; i < d; i += kFewThreads) xs[i] = to_f32(x[i]);
  __syncthreads();
#pragma unroll 4
  for (int h = warp; h < f; h += kFewThreads / 32) {
    float g = 0.0f, u = 0.0f;
    for (int i = lane; i < d; i += 32) {
      g = fmaf(xs[i], to_f32(wg[(size_t)h * d + i]), g);
      u = fmaf(xs[i], to_f32(wu[(size_t)h * d + i]), u);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      g += __shfl_xor_sync(~0u, g, o);
      u += __shfl_xor_sync(~0u, u, o);
    }
    if (lane == 0) {
      F2 a, slope;
      float a0, a1;
      gate2<ACT, false>(f2(g), a, slope);
      split(a, a0, a1);
      hs[h] = a0 * u;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int o = warp; o < c; o += kFewThreads / 32) {
    float s = 0.0f;
    for (int i = lane; i < f; i += 32) s = fmaf(hs[i], to_f32(wd[(size_t)o * f + i]), s);
#pragma unroll
    for (int k = 16; k; k >>= 1) s += __shfl_xor_sync(~0u, s, k);
    if (lane == 0) y[o] = from_f32<T>(s);
  }
}

// Sums the splits' partial weight gradients (P) in order, in 64 bits, and rounds.  Threads
// follow the partial sums' layout, of which each is read once.
template <typename T, typename P>
__global__ void k_decode_reduce(const P* __restrict__ partials, int splits, int chunks, int d, int f, int c, T* dg, T* du,
                                T* dd) {
  const int columns = dw_columns(d, c), first_dd = d > 64 ? 128 : 64;
  const int64_t total = (int64_t)chunks * columns * kTile;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int row = (int)(i % kTile), col = (int)(i / kTile % columns);
    const int h0 = (int)(i / kTile / columns) * kChunk;
    T* out;
    if (col < first_dd) {
      const int h = h0 + (row & 63);
      if (col >= d || h >= f) continue;
      out = (row < 64 ? dg : du) + (size_t)h * d + col;
    } else {
      const int o = (col - first_dd) / 64 * 128 + row, h = h0 + (col & 63);
      if (o >= c || h >= f) continue;
      out = dd + (size_t)o * f + h;
    }
    double s = 0.0;
#pragma unroll 8
    for (int p = 0; p < splits; ++p) s += partials[p * total + i];
    *out = from_f32<T>((float)s);
  }
}

static int decode_splits(int64_t n, int f) {
  const int chunks = (f + kChunk - 1) / kChunk;
  const int64_t tiles = ceil_div(n, kTile);
  return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, std::max(1, 148 / chunks)));
}

static bool decode_wide(int64_t n, int f) { return ceil_div(ceil_div(n, kTile), decode_splits(n, f)) > kSumTiles; }

static int check_dims(const char* who, int64_t n, int dtype, int d, int f, int c) {
  if (dtype != GS_F16 && dtype != GS_BF16)
    return set_error(GS_ERR_INVALID_ARG, "%s: dtype must be GS_F16 or GS_BF16 (got %d)", who, dtype);
  if (n < 0 || n > GS_DECODE_MAX_N)
    return set_error(GS_ERR_INVALID_ARG, "%s: n must be in [0, %d]", who, GS_DECODE_MAX_N);
  if (d < 1 || d > GS_DECODE_MAX_D)
    return set_error(GS_ERR_INVALID_ARG, "%s: d must be in [1, %d] (got %d)", who, GS_DECODE_MAX_D, d);
  if (c < 1 || c > GS_DECODE_MAX_C)
    return set_error(GS_ERR_INVALID_ARG, "%s: c must be in [1, %d] (got %d)", who, GS_DECODE_MAX_C, c);
  if (f < 1 || f > GS_DECODE_MAX_F)
    return set_error(GS_ERR_INVALID_ARG, "%s: f must be in [1, %d] (got %d)", who, GS_DECODE_MAX_F, f);
  return GS_OK;
}

static int check_workspace(const char* who, const void* ws, size_t have, size_t need) {
  if (need > 0 && (!ws || have < need)) return set_error(GS_ERR_CAPACITY, "%s: workspace too small", who);
  if (!aligned(ws, 16)) return set_error(GS_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", who);
  return GS_OK;
}

static int check_image(const char* who, const void* image, size_t image_bytes, int d, int f, int c) {
  if (!image || image_bytes < gs_decode_image_bytes(d, f, c))
    return set_error(GS_ERR_CAPACITY, "%s: weight image too small", who);
  if (!aligned(image, 16)) return set_error(GS_ERR_INVALID_ARG, "%s: image must be 16-byte aligned", who);
  return GS_OK;
}

// Rows of `width` elements to rows of `padded` (a multiple of 8), zeros behind:
// one thread per 16 bytes written, reading `Part`s, the largest of 2, 4 and 8 bytes
// that divides a row and the address.
template <typename Part>
__global__ void k_pad_rows(const Part* __restrict__ src, int64_t n, int width, int per_row, uint4* __restrict__ dst) {
  constexpr int kParts = 16 / sizeof(Part), kElems = sizeof(Part) / 2;
  const int parts = width / kElems;  // of a row
  const int64_t total = n * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row;
    const int p0 = (int)(i - row * per_row) * kParts;
    union {
      Part part[kParts];
      uint4 all;
    } v;
    v.all = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < kParts; ++e)
      if (p0 + e < parts) v.part[e] = __ldg(src + row * parts + p0 + e);
    dst[i] = v.all;
  }
}

static bool fetchable(const void* p, int width) { return width % 8 == 0 && aligned(p, 16); }

static size_t padded_bytes(int64_t n, int width) { return ((size_t)n * round_up(width, 8) * 2 + 255) & ~(size_t)255; }

// Returns rows the copy engine can fetch: p itself, or its padded copy at *ws
// (which is moved past it).
static const void* fetchable_rows(const void* p, int64_t n, int width, uint8_t** ws, cudaStream_t s) {
  if (fetchable(p, width)) return p;
  uint4* out = reinterpret_cast<uint4*>(*ws);
  *ws += padded_bytes(n, width);
  const int per_row = round_up(width, 8) / 8;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n * per_row, 256), 148 * 64);
  const uintptr_t m = reinterpret_cast<uintptr_t>(p) | (uintptr_t)(width * 2);
  if (m % 8 == 0) k_pad_rows<uint2><<<grid, 256, 0, s>>>(static_cast<const uint2*>(p), n, width, per_row, out);
  else if (m % 4 == 0) k_pad_rows<uint32_t><<<grid, 256, 0, s>>>(static_cast<const uint32_t*>(p), n, width, per_row, out);
  else k_pad_rows<uint16_t><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(p), n, width, per_row, out);
  return out;
}

// A map of (n, width) 16-bit elements, rows round_up(width, 8) apart, in boxes of
// 128 rows x 64 columns with the panels' swizzle.
static bool panel_map(CUtensorMap* map, const void* base, int dtype, int64_t n, int width) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (!encode) return false;
  // Encoding needs a current context, which a thread that has made no runtime
  // call yet (autograd's) does not have.
  int device;
  if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)n}, strides[1] = {(cuuint64_t)round_up(width, 8) * 2};
  const cuuint32_t box[2] = {64, kTile}, step[2] = {1, 1};
  return encode(map, dtype == GS_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static DecodeArgs decode_args(int64_t n, int d, int f, int c, int act, const void* image) {
  DecodeArgs a{};
  a.image = static_cast<const uint8_t*>(image);
  a.n = n; a.d = d; a.f = f; a.c = c;
  a.dp = round_up(d, 16); a.cp = round_up(c, 16);
  a.nxp = (d + 63) / 64; a.nyp = (c + 63) / 64;
  a.chunks = (f + kChunk - 1) / kChunk;
  a.chunk_bytes = chunk_bytes_of(d, c);
  a.act = act;
  return a;
}

// Shared memory of a launch: input stages, weight stages, output stage, barriers.
// Weight chunks are kept resident if they all fit beside two input stages.  Else three
// stages stream them; where only two would fit, resident weights beside a single input
// stage are better (dx of 1600x1060 rows, 64-256-152: 505 us, streamed 531; with three
// stages, 64-256-128: 432 us, streamed 401).  The largest blocks stream them through two
// stages.  What is left goes to further input stages.
template <int MODE>
static size_t plan_smem(DecodeArgs& a) {
  constexpr size_t kMost = kMaxSmem - sizeof(Bars);
  const size_t in = (size_t)(a.nxp + (MODE == kFwd ? 0 : a.nyp)) * kPanel;
  if (MODE == kDw) {
    const size_t own = a.chunk_bytes + 3 * (size_t)kPanel;
    a.w_stages = 1;
    a.x_stages = (int)std::min<size_t>(kMaxXStages, (kMost - own) / in);
    a.bars_at = (int)(own + a.x_stages * in);
    return a.bars_at + sizeof(Bars);
  }
  const int width = MODE == kFwd ? a.c : a.d, row = width * 2;
  // The stage has the output's own layout where its rows are an odd number of
  // out_vec bytes apart, so that a column's stores hit all banks: one bulk copy
  // a tile.  An even number of 16-byte units is padded by one, and the drain
  // warps copy the rows themselves (one bulk copy a row took 5000 cycles a tile:
  // forward, 1600x1060 rows of 64 classes, 498 us instead of 283).
  a.out_vec = width % 8 == 0 ? 16 : width % 4 == 0 ? 8 : width % 2 == 0 ? 4 : 2;
  a.out_pitch = width % 8 == 0 ? (row / 16 | 1) * 16 : row;
  bool staged = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  a.out_bulk = staged && a.out_pitch == row;
  size_t out = staged ? ((size_t)kTile * a.out_pitch + 127) & ~(size_t)127 : 0;
  const size_t all = (size_t)a.chunks * a.chunk_bytes, two = (size_t)std::min(a.chunks, 2) * a.chunk_bytes;
  const bool fit = a.chunks <= kMaxWStages;  // the barriers
  if (fit && out + 2 * in + all <= kMost) {
    a.x_stages = 2;
  } else if (out + 2 * in + two + a.chunk_bytes <= kMost) {
    a.x_stages = 2;
  } else if (fit && out + in + all <= kMost) {
    a.x_stages = 1;
  } else {
    if (out + in + two > kMost) {
      out = 0;
      staged = false;
    }
    a.x_stages = out + 2 * in + two <= kMost ? 2 : 1;
  }
  if (!staged) {
    a.out_pitch = 0;
    a.out_bulk = 0;
    // rows of the caller's own output: its alignment bounds the store size
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.out);
    while (a.out_vec > 2 && at % a.out_vec) a.out_vec /= 2;
  }
  a.w_stages = (int)std::min<size_t>(std::min(a.chunks, kMaxWStages), (kMost - out - a.x_stages * in) / a.chunk_bytes);
  while (a.x_stages >= 2 && a.x_stages < kMaxXStages &&
         out + (a.x_stages + 1) * in + (size_t)a.w_stages * a.chunk_bytes <= kMost)
    ++a.x_stages;
  a.bars_at = (int)(a.x_stages * in + (size_t)a.w_stages * a.chunk_bytes + out);
  return a.bars_at + sizeof(Bars);
}

template <typename T, int MODE, int ACT>
static int launch_decode_as(DecodeArgs a, dim3 grid, cudaStream_t s) {
  // one CTA per SM: each takes all of TMEM
  const size_t smem = std::max<size_t>(plan_smem<MODE>(a), 120 * 1024);
  auto* kernel = MODE == kDw ? k_decode_dw<T, ACT> : k_decode<T, MODE == kDx ? kDx : kFwd, ACT>;
  // (always the same limit: threads may launch different sizes at once)
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
  if (e != cudaSuccess) return set_error(GS_ERR_CUDA, "k_decode: %s", cudaGetErrorString(e));
  kernel<<<grid, MODE == kDw ? kDwThreads : kDecodeThreads, smem, s>>>(a);
  return check_launch("k_decode");
}

template <int MODE>
static int launch_decode(const DecodeArgs& a, int dtype, dim3 grid, cudaStream_t s) {
  if (dtype == GS_F16)
    return a.act == GS_ACT_SILU ? launch_decode_as<__half, MODE, GS_ACT_SILU>(a, grid, s)
                                : launch_decode_as<__half, MODE, GS_ACT_GELU>(a, grid, s);
  return a.act == GS_ACT_SILU ? launch_decode_as<__nv_bfloat16, MODE, GS_ACT_SILU>(a, grid, s)
                              : launch_decode_as<__nv_bfloat16, MODE, GS_ACT_GELU>(a, grid, s);
}

}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_decode_image_bytes(int d, int f, int c) {
  if (d < 1 || d > GS_DECODE_MAX_D || c < 1 || c > GS_DECODE_MAX_C || f < 1 || f > GS_DECODE_MAX_F) return 0;
  return (size_t)((f + kChunk - 1) / kChunk) * chunk_bytes_of(d, c);
}

int gs_decode_prepare(const void* w_gate, const void* w_up, const void* w_down, int dtype, int d, int f, int c,
                      void* image, size_t image_bytes, void* stream) {
  clear_error();
  if (int e = check_dims("gs_decode_prepare", 0, dtype, d, f, c)) return e;
  if (int e = check_image("gs_decode_prepare", image, image_bytes, d, f, c)) return e;
  if (!w_gate || !w_up || !w_down) return set_error(GS_ERR_INVALID_ARG, "gs_decode_prepare: NULL pointer");
  const int cb = chunk_bytes_of(d, c), chunks = (f + kChunk - 1) / kChunk;
  const dim3 grid((unsigned)ceil_div(cb / 16, 256), (unsigned)chunks);
  cudaStream_t s = as_stream(stream);
  if (dtype == GS_F16)
    k_decode_prepare<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(w_gate),
                                                  static_cast<const __half*>(w_up),
                                                  static_cast<const __half*>(w_down), d, f, c, cb,
                                                  static_cast<uint8_t*>(image));
  else
    k_decode_prepare<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(w_gate),
                                                         static_cast<const __nv_bfloat16*>(w_up),
                                                         static_cast<const __nv_bfloat16*>(w_down), d, f, c, cb,
                                                         static_cast<uint8_t*>(image));
  return check_launch("k_decode_prepare");
}

size_t gs_decode_workspace_bytes(const void* x, const void* dy, int64_t n, int d, int f, int c, int weights) {
  if (n < 0 || gs_decode_image_bytes(d, f, c) == 0) return 0;
  size_t bytes = fetchable(x, d) ? 0 : padded_bytes(n, d);
  if (dy && !fetchable(dy, c)) bytes += padded_bytes(n, c);
  if (weights)
    bytes += (size_t)decode_splits(n, f) * ((f + kChunk - 1) / kChunk) * dw_columns(d, c) * kTile *
             (decode_wide(n, f) ? sizeof(double) : sizeof(float));
  return bytes;
}

int gs_decode_is_few(int64_t n, int d, int f, int c) {
  return n >= 0 && n <= GS_DECODE_FEW_N && d >= 1 && c >= 1 && f >= 1 &&
         (int64_t)f * (2 * (int64_t)d + c) <= GS_DECODE_FEW_WEIGHTS;
}

int gs_decode_forward_few(const void* x, const void* w_gate, const void* w_up, const void* w_down, int dtype, int64_t n,
                          int d, int f, int c, int activation, void* y, void* stream) {
  clear_error();
  if (int e = check_dims("gs_decode_forward_few", n, dtype, d, f, c)) return e;
  if (!gs_decode_is_few(n, d, f, c))
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward_few: more than %d rows or %d weights", GS_DECODE_FEW_N,
                     GS_DECODE_FEW_WEIGHTS);
  if (activation != GS_ACT_SILU && activation != GS_ACT_GELU)
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward_few: unknown activation %d", activation);
  if (n == 0) return GS_OK;
  if (!x || !w_gate || !w_up || !w_down || !y)
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward_few: NULL pointer");
  const size_t smem = sizeof(float) * ((size_t)d + f);
  auto launch = [&](auto zero) {
    using T = decltype(zero);
    auto* kernel = activation == GS_ACT_SILU ? k_decode_few<T, GS_ACT_SILU> : k_decode_few<T, GS_ACT_GELU>;
    if (smem > 48 * 1024) {
      const int most = 4 * (GS_DECODE_MAX_D + GS_DECODE_FEW_WEIGHTS / 3);  // of any call
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e != cudaSuccess) return set_error(GS_ERR_CUDA, "k_decode_few: %s", cudaGetErrorString(e));
    }
    kernel<<<(unsigned)n, kFewThreads, smem, as_stream(stream)>>>(
        static_cast<const T*>(x), static_cast<const T*>(w_gate), static_cast<const T*>(w_up),
        static_cast<const T*>(w_down), d, f, c, static_cast<T*>(y));
    return check_launch("k_decode_few");
  };
  return dtype == GS_F16 ? launch(__half{}) : launch(__nv_bfloat16{});
}

int gs_decode_forward(const void* x, int dtype, int64_t n, int d, int f, int c, int activation, const void* image,
                      size_t image_bytes, void* y, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int e = check_dims("gs_decode_forward", n, dtype, d, f, c)) return e;
  if (activation != GS_ACT_SILU && activation != GS_ACT_GELU)
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward: unknown activation %d", activation);
  if (n == 0) return GS_OK;
  if (!x || !y) return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward: NULL pointer");
  if (int e = check_image("gs_decode_forward", image, image_bytes, d, f, c)) return e;
  if (int e = check_workspace("gs_decode_forward", workspace, workspace_bytes,
                              gs_decode_workspace_bytes(x, nullptr, n, d, f, c, 0)))
    return e;
  cudaStream_t s = as_stream(stream);
  DecodeArgs a = decode_args(n, d, f, c, activation, image);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const void* rows = fetchable_rows(x, n, d, &ws, s);
  if (rows != x)
    if (int e = check_launch("k_pad_rows")) return e;
  if (!panel_map(&a.map_x, rows, dtype, n, d)) return set_error(GS_ERR_CUDA, "gs_decode_forward: tensor map refused");
  a.out = y;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, kTile), 148);
  return launch_decode<kFwd>(a, dtype, dim3(grid), s);
}

int gs_decode_backward(const void* x, const void* dy, int dtype, int64_t n, int d, int f, int c, int activation,
                       const void* image, size_t image_bytes, void* dx, void* d_gate, void* d_up, void* d_down,
                       void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (int e = check_dims("gs_decode_backward", n, dtype, d, f, c)) return e;
  if (activation != GS_ACT_SILU && activation != GS_ACT_GELU)
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_backward: unknown activation %d", activation);
  const bool weights = d_gate || d_up || d_down;
  if (weights && (!d_gate || !d_up || !d_down))
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_backward: give all weight gradients or none");
  if (!weights && !dx) return GS_OK;
  cudaStream_t s = as_stream(stream);
  const int chunks = (f + kChunk - 1) / kChunk;
  int splits = 0;
  bool wide = false;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (n > 0) {
    if (!x || !dy) return set_error(GS_ERR_INVALID_ARG, "gs_decode_backward: NULL pointer");
    if (int e = check_image("gs_decode_backward", image, image_bytes, d, f, c)) return e;
    if (int e = check_workspace("gs_decode_backward", workspace, workspace_bytes,
                                gs_decode_workspace_bytes(x, dy, n, d, f, c, weights)))
      return e;
    DecodeArgs a = decode_args(n, d, f, c, activation, image);
    const void* xr = fetchable_rows(x, n, d, &ws, s);
    const void* yr = fetchable_rows(dy, n, c, &ws, s);
    if (int e = check_launch("k_pad_rows", (xr != x) + (yr != dy))) return e;
    if (!panel_map(&a.map_x, xr, dtype, n, d) || !panel_map(&a.map_dy, yr, dtype, n, c))
      return set_error(GS_ERR_CUDA, "gs_decode_backward: tensor map refused");
    if (dx) {
      a.out = dx;
      const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, kTile), 148);
      if (int e = launch_decode<kDx>(a, dtype, dim3(grid), s)) return e;
    }
    if (!weights) return GS_OK;
    splits = decode_splits(n, f);
    a.partials = ws;
    a.wide = wide = decode_wide(n, f);
    if (int e = launch_decode<kDw>(a, dtype, dim3((unsigned)splits, (unsigned)a.chunks), s)) return e;
  }
  if (!weights) return GS_OK;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div((int64_t)chunks * dw_columns(d, c) * kTile, 256), 148 * 8);
  auto reduce = [&](auto zero, const auto* part) {
    using T = decltype(zero);
    k_decode_reduce<<<grid, 256, 0, s>>>(part, splits, chunks, d, f, c, static_cast<T*>(d_gate), static_cast<T*>(d_up),
                                         static_cast<T*>(d_down));
  };
  auto reduce_as = [&](auto zero) {
    if (wide) reduce(zero, reinterpret_cast<const double*>(ws));
    else reduce(zero, reinterpret_cast<const float*>(ws));
  };
  if (dtype == GS_F16) reduce_as(__half{});
  else reduce_as(__nv_bfloat16{});
  return check_launch("k_decode_reduce");
}

}  // extern "C"
