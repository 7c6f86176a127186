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
// This form is sequential: load, first products, activation, second products.
#include "feature_common.cuh"
#include "tc_common.cuh"

namespace gs {

constexpr int kTile = 128;              // rows of a tile (M of the matrix instructions)
constexpr int kChunk = 64;              // hidden units of a chunk
constexpr int kPanel = kTile * 128;     // bytes of a 128-row panel
constexpr int kDecodeThreads = 256;
constexpr uint32_t kTmemCols = 512;
// TMEM columns
constexpr uint32_t kColG = 0, kColU = 64, kColDh = 128, kColH = 192, kColOut = 256;

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
  const void* x;
  const void* dy;
  const uint8_t* image;
  void* out;        // y or dx
  float* partials;  // weight gradients: [split][gate f*d | up f*d | down c*f]
  int64_t n;
  int d, f, c;
  int dp, cp;    // d, c rounded up to 16
  int nxp, nyp;  // 64-element panels of x and dy
  int chunks;
  int chunk_bytes;
  int act;
};

__host__ __device__ __forceinline__ int round_up(int v, int m) { return (v + m - 1) / m * m; }

// A chunk of the weight image: the gate's and up's 64 hidden units as 128 rows
// (gate first) of ceil(d / 64) panels, then Wd's columns of these hidden units
// as one panel of cp rows.
static int chunk_bytes_of(int d, int c) { return (d + 63) / 64 * kPanel + round_up(c, 16) * tc::kPanelRow; }

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

// act(g), and act'(g) where wanted.  exp and the reciprocal are the hardware
// approximations (2 ulp): the results are rounded to 16 bits.
template <int ACT, bool SLOPE>
__device__ __forceinline__ void gate(float g, float& a, float& slope) {
  if (ACT == GS_ACT_SILU) {
    const float s = __frcp_rn(1.0f + __expf(-g));
    a = g * s;
    if (SLOPE) slope = s + a * (1.0f - s);
  } else {
    const float phi = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    a = g * phi;
    if (SLOPE) slope = phi + g * 0.39894228040143268f * __expf(-0.5f * g * g);
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

// `rows` x `width` elements into panels; rows past the end of the input become
// zero.  Columns past `width` were zeroed once and are never written.
template <typename T>
__device__ __forceinline__ void load_tile(uint8_t* panels, const T* __restrict__ src, int width, int rows) {
  if (width % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int per_row = width >> 3;
    for (int i = threadIdx.x; i < kTile * per_row; i += kDecodeThreads) {
      const int row = i / per_row, unit = i - row * per_row;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < rows) v = __ldg(reinterpret_cast<const uint4*>(src) + i);
      *reinterpret_cast<uint4*>(panels + (unit >> 3) * kPanel + tc::panel_offset(row, unit & 7)) = v;
    }
    return;
  }
  for (int i = threadIdx.x; i < kTile * width; i += kDecodeThreads) {
    const int row = i / width, col = i - row * width;
    *reinterpret_cast<T*>(panels + (col >> 6) * kPanel + tc::panel_elem(row, col & 63)) =
        row < rows ? src[i] : from_f32<T>(0.0f);
  }
}

template <typename T, int MODE, int ACT>
__global__ void __launch_bounds__(kDecodeThreads, 1) k_decode(DecodeArgs a) {
  extern __shared__ uint8_t raw[];
  __shared__ unsigned long long bars[2];
  __shared__ uint32_t tmem_slot;
  uint8_t* smem = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  uint8_t* xs = smem;
  uint8_t* ys = xs + a.nxp * kPanel;
  uint8_t* ws = ys + (MODE == kFwd ? 0 : a.nyp * kPanel);
  uint8_t* st = ws + a.chunk_bytes;  // dg, du, h panels (weight gradients)
  unsigned long long* wbar = &bars[0];
  unsigned long long* mbar = &bars[1];
  constexpr bool kBf16 = sizeof(T) == 2 && !__is_same(T, __half);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quarter = warp & 3, half = warp >> 2;
  const int row = quarter * 32 + lane;
  if (warp == 0) tc::tmem_alloc(&tmem_slot, kTmemCols);
  if (threadIdx.x == 0) {
    mbar_init(wbar, 1);
    mbar_init(mbar, 1);
  }
  for (uint32_t i = threadIdx.x * 16; i < (uint32_t)(ws - xs); i += kDecodeThreads * 16)
    *reinterpret_cast<uint4*>(xs + i) = make_uint4(0, 0, 0, 0);
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);

  const int64_t tiles = (a.n + kTile - 1) / kTile;
  unsigned wphase = 0, mphase = 0;
  bool ok = true, loaded = false;
  const T* x = static_cast<const T*>(a.x);
  const T* dy = static_cast<const T*>(a.dy);

  for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
    const int rows = (int)min((int64_t)kTile, a.n - t * kTile);
    load_tile<T>(xs, x + t * kTile * a.d, a.d, rows);
    if (MODE != kFwd) load_tile<T>(ys, dy + t * kTile * a.c, a.c, rows);
    tc::fence_async_smem();
    __syncthreads();
    const int j0 = MODE == kDw ? blockIdx.y : 0, j1 = MODE == kDw ? j0 + 1 : a.chunks;
    for (int j = j0; j < j1; ++j) {
      if (threadIdx.x == 0) {
        if (!loaded || (MODE != kDw && a.chunks > 1)) {
          mbar_arrive_expect_tx(wbar, a.chunk_bytes);
          bulk_g2s(ws, a.image + (size_t)j * a.chunk_bytes, a.chunk_bytes, wbar);
          ok = mbar_wait(wbar, wphase);
          wphase ^= 1;
        }
        // first products: [g | u] = x [Wg | Wu]^T
        const uint32_t wgu = smem_addr(ws), wdn = wgu + a.nxp * kPanel;
        for (int k = 0; k < a.dp / 16; ++k) {
          const uint32_t at = (k >> 2) * kPanel + (k & 3) * 32;
          tc::mma_ss(tmem + kColG, tc::desc_k(smem_addr(xs) + at), tc::desc_k(wgu + at),
                     tc::instr_desc(kBf16, 128, false, false), k > 0);
        }
        if (MODE != kFwd) {  // dh = dy Wd
          for (int k = 0; k < a.cp / 16; ++k)
            tc::mma_ss(tmem + kColDh, tc::desc_k(smem_addr(ys) + (k >> 2) * kPanel + (k & 3) * 32),
                       tc::desc_mn(wdn + k * 2048, kPanel), tc::instr_desc(kBf16, 64, false, true), k > 0);
        }
        tc::commit(mbar);
      }
      loaded = true;
      ok &= mbar_wait(mbar, mphase);
      mphase ^= 1;
      tc::fence_after();
      uint32_t g[32], u[32], dh[32];
      tc::tmem_ld32(lanes + kColG + half * 32, g);
      tc::tmem_ld32(lanes + kColU + half * 32, u);
      if (MODE != kFwd) tc::tmem_ld32(lanes + kColDh + half * 32, dh);
      tc::tmem_wait_ld();
      tc::after_wait(g);
      tc::after_wait(u);
      if (MODE != kFwd) tc::after_wait(dh);
      uint32_t ph[16], pg[16], pu[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float a0, a1, s0, s1;
        gate<ACT, MODE != kFwd>(__uint_as_float(g[2 * i]), a0, s0);
        gate<ACT, MODE != kFwd>(__uint_as_float(g[2 * i + 1]), a1, s1);
        const float u0 = __uint_as_float(u[2 * i]), u1 = __uint_as_float(u[2 * i + 1]);
        if (MODE != kDx) ph[i] = pack2<T>(a0 * u0, a1 * u1);
        if (MODE != kFwd) {
          const float d0 = __uint_as_float(dh[2 * i]), d1 = __uint_as_float(dh[2 * i + 1]);
          pg[i] = pack2<T>(d0 * u0 * s0, d1 * u1 * s1);
          pu[i] = pack2<T>(d0 * a0, d1 * a1);
        }
      }
      if (MODE == kFwd) {
        tc::tmem_st16(lanes + kColH + half * 16, ph);
        tc::tmem_wait_st();
      } else if (MODE == kDx) {
        tc::tmem_st16(lanes + kColH + half * 16, pg);
        tc::tmem_st16(lanes + kColH + 32 + half * 16, pu);
        tc::tmem_wait_st();
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t off = tc::panel_offset(row, half * 4 + q);
          *reinterpret_cast<uint4*>(st + off) = make_uint4(pg[4 * q], pg[4 * q + 1], pg[4 * q + 2], pg[4 * q + 3]);
          *reinterpret_cast<uint4*>(st + kPanel + off) =
              make_uint4(pu[4 * q], pu[4 * q + 1], pu[4 * q + 2], pu[4 * q + 3]);
          *reinterpret_cast<uint4*>(st + 2 * kPanel + off) =
              make_uint4(ph[4 * q], ph[4 * q + 1], ph[4 * q + 2], ph[4 * q + 3]);
        }
        tc::fence_async_smem();
      }
      tc::fence_before();
      ok = __syncthreads_and(ok);
      if (!ok) break;
      if (threadIdx.x == 0) {
        tc::fence_after();
        const uint32_t wgu = smem_addr(ws), wdn = wgu + a.nxp * kPanel;
        if (MODE == kFwd) {  // y += h Wd^T
          for (int k = 0; k < 4; ++k)
            tc::mma_ts(tmem + kColOut, tmem + kColH + k * 8, tc::desc_k(wdn + k * 32),
                       tc::instr_desc(kBf16, a.cp, false, false), j > 0 || k > 0);
        } else if (MODE == kDx) {  // dx += [dg | du] [Wg ; Wu]
          for (int k = 0; k < 8; ++k)
            tc::mma_ts(tmem + kColOut, tmem + kColH + k * 8, tc::desc_mn(wgu + k * 2048, kPanel),
                       tc::instr_desc(kBf16, a.dp, false, true), j > 0 || k > 0);
        } else {
          const uint32_t sa = smem_addr(st);
          const bool first = t == blockIdx.x;
          for (int k = 0; k < 8; ++k)  // [dWg ; dWu] += [dg | du]^T x
            tc::mma_ss(tmem + kColOut, tc::desc_mn(sa + k * 2048, kPanel), tc::desc_mn(smem_addr(xs) + k * 2048, kPanel),
                       tc::instr_desc(kBf16, a.dp, true, true), !first || k > 0);
          for (int m = 0; m < (a.c + 127) / 128; ++m)  // dWd += dy^T h
            for (int k = 0; k < 8; ++k)
              tc::mma_ss(tmem + kColOut + 128 + m * 64, tc::desc_mn(smem_addr(ys) + m * 2 * kPanel + k * 2048, kPanel),
                         tc::desc_mn(sa + 2 * kPanel + k * 2048, kPanel), tc::instr_desc(kBf16, 64, true, true),
                         !first || k > 0);
        }
        tc::commit(mbar);
      }
      ok &= mbar_wait(mbar, mphase);
      mphase ^= 1;
      tc::fence_after();
    }
    if (MODE != kDw && ok) {
      const int width = MODE == kFwd ? a.c : a.d;
      T* out = static_cast<T*>(a.out) + (t * kTile + row) * width;
      for (int c0 = half * 32; c0 < width; c0 += 64) {
        uint32_t v[32];
        tc::tmem_ld32(lanes + kColOut + c0, v);
        tc::tmem_wait_ld();
        tc::after_wait(v);
        if (row < rows)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c0 + i < width) out[c0 + i] = from_f32<T>(__uint_as_float(v[i]));
      }
    }
    tc::fence_before();
    ok = __syncthreads_and(ok);
    tc::fence_after();
  }
  if (MODE == kDw && ok) {
    const size_t fd = (size_t)a.f * a.d;
    float* part = a.partials + (size_t)blockIdx.x * (2 * fd + (size_t)a.c * a.f);
    const int j = blockIdx.y;
    const int h = j * kChunk + (row & 63);
    float* gu = part + (row < 64 ? 0 : fd) + (size_t)h * a.d;
    for (int c0 = half * 32; c0 < a.d; c0 += 64) {
      uint32_t v[32];
      tc::tmem_ld32(lanes + kColOut + c0, v);
      tc::tmem_wait_ld();
      tc::after_wait(v);
      if (h < a.f)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (c0 + i < a.d) gu[c0 + i] = __uint_as_float(v[i]);
    }
    for (int m = 0; m < (a.c + 127) / 128; ++m) {
      uint32_t v[32];
      tc::tmem_ld32(lanes + kColOut + 128 + m * 64 + half * 32, v);
      tc::tmem_wait_ld();
      tc::after_wait(v);
      const int c = m * 128 + row, h0 = j * kChunk + half * 32;
      if (c < a.c)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (h0 + i < a.f) part[2 * fd + (size_t)c * a.f + h0 + i] = __uint_as_float(v[i]);
    }
    tc::fence_before();
  }
  if (!ok && threadIdx.x == 0) atomicAdd(&g_decode_wait_failures, 1ull);
  __syncthreads();
  if (warp == 0) tc::tmem_free(tmem, kTmemCols);
}

// Sums the splits' partial weight gradients in order and rounds once.
template <typename T>
__global__ void k_decode_reduce(const float* __restrict__ partials, int splits, int64_t fd, int64_t cf, T* dg, T* du,
                                T* dd) {
  const int64_t total = 2 * fd + cf;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    float s = 0.0f;
    for (int p = 0; p < splits; ++p) s += partials[p * total + i];
    T* out = i < fd ? dg + i : i < 2 * fd ? du + (i - fd) : dd + (i - 2 * fd);
    *out = from_f32<T>(s);
  }
}

static int decode_splits(int64_t n, int f) {
  const int chunks = (f + kChunk - 1) / kChunk;
  const int64_t tiles = ceil_div(n, kTile);
  return (int)std::max<int64_t>(1, std::min<int64_t>(tiles, std::max(1, 148 / chunks)));
}

static int check_dims(const char* who, int64_t n, int dtype, int d, int f, int c) {
  if (dtype != GS_F16 && dtype != GS_BF16)
    return set_error(GS_ERR_INVALID_ARG, "%s: dtype must be GS_F16 or GS_BF16 (got %d)", who, dtype);
  if (n < 0) return set_error(GS_ERR_INVALID_ARG, "%s: n is negative", who);
  if (d < 1 || d > GS_DECODE_MAX_D)
    return set_error(GS_ERR_INVALID_ARG, "%s: d must be in [1, %d] (got %d)", who, GS_DECODE_MAX_D, d);
  if (c < 1 || c > GS_DECODE_MAX_C)
    return set_error(GS_ERR_INVALID_ARG, "%s: c must be in [1, %d] (got %d)", who, GS_DECODE_MAX_C, c);
  if (f < 1 || f > GS_DECODE_MAX_F)
    return set_error(GS_ERR_INVALID_ARG, "%s: f must be in [1, %d] (got %d)", who, GS_DECODE_MAX_F, f);
  return GS_OK;
}

static int check_image(const char* who, const void* image, size_t image_bytes, int d, int f, int c) {
  if (!image || image_bytes < gs_decode_image_bytes(d, f, c))
    return set_error(GS_ERR_CAPACITY, "%s: weight image too small", who);
  if (!aligned(image, 16)) return set_error(GS_ERR_INVALID_ARG, "%s: image must be 16-byte aligned", who);
  return GS_OK;
}

static DecodeArgs decode_args(const void* x, const void* dy, int64_t n, int d, int f, int c, int act,
                              const void* image) {
  DecodeArgs a{};
  a.x = x; a.dy = dy; a.image = static_cast<const uint8_t*>(image);
  a.n = n; a.d = d; a.f = f; a.c = c;
  a.dp = round_up(d, 16); a.cp = round_up(c, 16);
  a.nxp = (d + 63) / 64; a.nyp = (c + 63) / 64;
  a.chunks = (f + kChunk - 1) / kChunk;
  a.chunk_bytes = chunk_bytes_of(d, c);
  a.act = act;
  return a;
}

template <typename T, int MODE, int ACT>
static int launch_decode_as(const DecodeArgs& a, dim3 grid, cudaStream_t s) {
  size_t smem = 1024 + (size_t)a.nxp * kPanel + a.chunk_bytes;
  if (MODE != kFwd) smem += (size_t)a.nyp * kPanel;
  if (MODE == kDw) smem += 3 * (size_t)kPanel;
  smem = std::max<size_t>(smem, 120 * 1024);  // one CTA per SM: each takes all of TMEM
  cudaError_t e = cudaFuncSetAttribute(k_decode<T, MODE, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return set_error(GS_ERR_CUDA, "k_decode: %s", cudaGetErrorString(e));
  k_decode<T, MODE, ACT><<<grid, kDecodeThreads, smem, s>>>(a);
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

int gs_decode_forward(const void* x, int dtype, int64_t n, int d, int f, int c, int activation, const void* image,
                      size_t image_bytes, void* y, void* stream) {
  clear_error();
  if (int e = check_dims("gs_decode_forward", n, dtype, d, f, c)) return e;
  if (activation != GS_ACT_SILU && activation != GS_ACT_GELU)
    return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward: unknown activation %d", activation);
  if (n == 0) return GS_OK;
  if (!x || !y) return set_error(GS_ERR_INVALID_ARG, "gs_decode_forward: NULL pointer");
  if (int e = check_image("gs_decode_forward", image, image_bytes, d, f, c)) return e;
  DecodeArgs a = decode_args(x, nullptr, n, d, f, c, activation, image);
  a.out = y;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, kTile), 148);
  return launch_decode<kFwd>(a, dtype, dim3(grid), as_stream(stream));
}

size_t gs_decode_workspace_bytes(int64_t n, int d, int f, int c) {
  if (n < 0 || gs_decode_image_bytes(d, f, c) == 0) return 0;
  return (size_t)decode_splits(n, f) * (2 * (size_t)f * d + (size_t)c * f) * sizeof(float);
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
  cudaStream_t s = as_stream(stream);
  const int64_t fd = (int64_t)f * d, cf = (int64_t)c * f;
  if (n > 0) {
    if (!x || !dy) return set_error(GS_ERR_INVALID_ARG, "gs_decode_backward: NULL pointer");
    if (int e = check_image("gs_decode_backward", image, image_bytes, d, f, c)) return e;
  }
  if (weights && n > 0 && (!workspace || workspace_bytes < gs_decode_workspace_bytes(n, d, f, c)))
    return set_error(GS_ERR_CAPACITY, "gs_decode_backward: workspace too small");
  DecodeArgs a = decode_args(x, dy, n, d, f, c, activation, image);
  if (dx && n > 0) {
    a.out = dx;
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, kTile), 148);
    if (int e = launch_decode<kDx>(a, dtype, dim3(grid), s)) return e;
  }
  if (!weights) return GS_OK;
  int splits = 0;
  if (n > 0) {
    splits = decode_splits(n, f);
    a.partials = static_cast<float*>(workspace);
    if (int e = launch_decode<kDw>(a, dtype, dim3((unsigned)splits, (unsigned)a.chunks), s)) return e;
  }
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(2 * fd + cf, 256), 148 * 8);
  const float* part = static_cast<const float*>(workspace);
  if (dtype == GS_F16)
    k_decode_reduce<__half><<<grid, 256, 0, s>>>(part, splits, fd, cf, static_cast<__half*>(d_gate),
                                                 static_cast<__half*>(d_up), static_cast<__half*>(d_down));
  else
    k_decode_reduce<__nv_bfloat16><<<grid, 256, 0, s>>>(part, splits, fd, cf, static_cast<__nv_bfloat16*>(d_gate),
                                                        static_cast<__nv_bfloat16*>(d_up),
                                                        static_cast<__nv_bfloat16*>(d_down));
  return check_launch("k_decode_reduce");
}

}  // extern "C"
