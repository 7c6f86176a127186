// Teacher cache: a row's k largest logits, kept in 8 or 4 bits.
//
// Writing is a selection; the order is (value descending, index ascending), held
// in one sortable key per class.
//   k_teacher_write_rows  few entries, short rows: one thread per row keeps its K
//                         best keys sorted in registers and takes K classes at a
//                         time (sorting network, then a bitonic merge), which
//                         needs no exchange between lanes.  A block stages its
//                         rows in shared memory with one bulk copy.
//   k_teacher_write_warp  anything else: one warp per row.  A first pass finds
//                         each lane's largest value; the K-th largest of these is
//                         a bound that at least K classes reach and few others do.
//                         A second pass collects those, 32 at a time, sorts them
//                         across the warp and merges them into the best 32.
// Reading is a gather of whole records, a group of lanes per record.
#include "feature_common.cuh"

namespace gs {

constexpr int kWriteWarps = 8;
// rows (threads) of a staging block: 64 take 299 us for 1920x1080x150 with the read, 32 or 128 305
constexpr int kStagedRows = 64;
constexpr size_t kStagedSmem = 48 * 1024;  // its shared memory at most

__device__ unsigned long long g_teacher_wait_failures;

int teacher_wait_failures(unsigned long long* out, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_teacher_wait_failures, sizeof(*out));
  if (e == cudaSuccess && reset) {
    const unsigned long long z = 0;
    e = cudaMemcpyToSymbol(g_teacher_wait_failures, &z, sizeof(z));
  }
  return (int)e;
}

struct TeacherWriteArgs {
  const void* logits;
  int64_t n, classes;
  uint8_t* records;  // of first_row
  int k, bits, rec_bytes;
};

// Sortable keys: a larger key comes first.  16-bit types: the value's bits made
// monotonic in the upper half, the inverted class below, one 32-bit word.  float:
// the same with 32 bits each.  0 is no class.
template <typename T>
struct Key {
  using Word = uint32_t;
  static constexpr uint32_t kLow = sizeof(T) == 2 && __is_same(T, __half) ? 0x0400u : 0x0080u;   // lowest finite
  static constexpr uint32_t kHigh = sizeof(T) == 2 && __is_same(T, __half) ? 0xfc00u : 0xff80u;  // +inf
  static __device__ __forceinline__ Word make(T v, int c) {
    uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
    if (b == 0x8000u) b = 0;  // -0 equals 0
    b ^= b & 0x8000u ? 0xffffu : 0x8000u;
    return b > kLow && b < kHigh ? (b << 16) | (0xffffu - (uint32_t)c) : 0u;
  }
  // Keys of neighbouring classes c and c + 1 from one word, without the test for
  // infinities, NaN and the lowest value: in the order, -inf and the lowest value
  // come last anyway (absent() tells them in the result), +inf and NaN first
  // (spoilt() tells that they are there).
  static __device__ __forceinline__ void quick(uint32_t w, uint32_t inverted, Word& k0, Word& k1) {
    T z[2];
    z[0] = z[1] = from_f32<T>(0.0f);
    if constexpr (__is_same(T, __half)) {
      const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(z));
      w = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __nv_bfloat162 v =
          __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(z));
      w = *reinterpret_cast<const uint32_t*>(&v);
    }
    const uint32_t sign = (w >> 15) & 0x00010001u;
    w ^= sign * 0x7fffu | 0x80008000u;
    k0 = (w << 16) | inverted;
    k1 = (w & 0xffff0000u) | (inverted - 1);
  }
  static __device__ __forceinline__ bool absent(Word w) { return w >> 16 <= kLow; }
  static __device__ __forceinline__ bool spoilt(Word w) { return w >> 16 >= kHigh; }
  static __device__ __forceinline__ float value(Word w) {
    uint32_t b = w >> 16;
    b ^= b & 0x8000u ? 0x8000u : 0xffffu;
    const unsigned short h = (unsigned short)b;
    return to_f32(*reinterpret_cast<const T*>(&h));
  }
  static __device__ __forceinline__ int index(Word w) { return (int)(0xffffu - (w & 0xffffu)); }
  static __device__ __forceinline__ Word shuffle(Word w, int from) { return __shfl_sync(~0u, w, from); }
  static __device__ __forceinline__ Word exchange(Word w, int mask) { return __shfl_xor_sync(~0u, w, mask); }
};
template <>
struct Key<float> {
  using Word = unsigned long long;
  static __device__ __forceinline__ Word make(float v, int c) {
    uint32_t b = __float_as_uint(v + 0.0f);  // -0 equals 0
    if (!(v > -FLT_MAX && v < INFINITY)) return 0ull;
    b ^= b & 0x80000000u ? 0xffffffffu : 0x80000000u;
    return ((Word)b << 32) | (0xffffffffu - (uint32_t)c);
  }
  static __device__ __forceinline__ float value(Word w) {
    uint32_t b = (uint32_t)(w >> 32);
    b ^= b & 0x80000000u ? 0x80000000u : 0xffffffffu;
    return __uint_as_float(b);
  }
  static __device__ __forceinline__ int index(Word w) { return (int)(0xffffffffu - (uint32_t)w); }
  static __device__ __forceinline__ Word shuffle(Word w, int from) { return __shfl_sync(~0u, w, from); }
  static __device__ __forceinline__ Word exchange(Word w, int mask) { return __shfl_xor_sync(~0u, w, mask); }
};

// code = levels (first - v) / (first - last) to nearest, ties to even, levels =
// 2^bits - 1.  The 32-bit quotient decides except next to a border, where the exact
// differences do (with few mantissa bits in the logits many quotients lie exactly
// between two codes): levels (first - v) against code and a half times the span, all of
// whose terms count (64-bit differences lose the smallest, and a write of 1920x1080x150 bf16
// takes 297 us with them, 305 so).  Spans that overflow, or whose reciprocal does, are
// scaled by a power of two first, v only for the quotient: it may be small enough to lose bits.
struct Quantiser {
  float scale, first, last, inv;
  __device__ __forceinline__ Quantiser(float f, float l, float levels) {
    const float span = f - l;
    scale = span > FLT_MAX ? 0.25f : span < 0x1p-60f ? 0x1p80f : 1.0f;
    first = f * scale;
    last = l * scale;
    inv = levels / (first - last);
  }
  __device__ __forceinline__ int operator()(float v, float levels) const {
    const float q = (first - v * scale) * inv, near = rintf(q);
    if (fabsf(q - near) < 0.499f) return (int)near;  // |error of q| < 255 * 4 * 2^-24 < 1e-4
    // 2 levels (first - v) - m (first - last): each product is exact in 64 bits
    const float low = floorf(q);
    const double l2 = 2.0f * levels, m = 2.0f * low + 1.0f;
    const double over = sum_of((l2 - m) * first, -l2 * ((double)v * scale), m * last);
    return (int)low + (over > 0.0 || (over == 0.0 && ((int)low & 1)) ? 1 : 0);
  }
  // a + b + c with the exact sum's sign (zero only where that is).  What rounding takes
  // from a + b is a value of 64 bits again, the last term here; where rounding takes
  // something from s + c too, c does not cancel s, and the sum outweighs both.
  static __device__ __forceinline__ double sum_of(double a, double b, double c) {
    const double s = a + b, part = s - a;
    return (s + c) + ((a - (s - part)) + (b - part));
  }
};
// (first - last) / levels, rounded once: the 64-bit product with 1 / levels, corrected
// by its remainder.  Where rounding up would take the last code's value out of float32's
// range, which stands for an absent entry, the step below.
__device__ __forceinline__ float step_of(float first, float last, int bits) {
  const double span = (double)first - (double)last, levels = (double)((1 << bits) - 1);
  const double inv = bits == 8 ? 1.0 / 255.0 : 1.0 / 15.0, q = span * inv;
  const float step = (float)__fma_rn(__fma_rn(-q, levels, span), inv, q);
  const bool lost = record_value(first, step, (1 << bits) - 1) == -INFINITY;
  return __uint_as_float(__float_as_uint(step) - (lost ? 1u : 0u));
}

template <typename W>
__device__ __forceinline__ void order(W& hi, W& lo) {  // hi >= lo afterwards
  const W a = hi, b = lo;
  hi = max(a, b);
  lo = min(a, b);
}
// Descending sort of N registers (Batcher's odd-even merge sort).
template <int N, typename W>
__device__ __forceinline__ void sort_desc(W (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order(v[i + j], v[i + j + k]);
}
// The N largest of two descending runs, descending, in `best`.
template <int N, typename W>
__device__ __forceinline__ void merge_desc(W (&best)[N], const W (&other)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) best[i] = max(best[i], other[N - 1 - i]);
#pragma unroll
  for (int k = N / 2; k >= 1; k /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & k) == 0) order(best[i], best[i + k]);
}

// One thread per row, MAX >= k a power of two; the block's rows are contiguous in
// memory and in shared memory.
template <typename T, int MAX>
__global__ void __launch_bounds__(kStagedRows) k_teacher_write_rows(TeacherWriteArgs a, int block_rows, int bulk) {
  using K = Key<T>;
  using W = typename K::Word;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ unsigned long long bar;
  const int C = (int)a.classes, l = threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.x * block_rows;
  const int rows = (int)min((int64_t)block_rows, a.n - r0);
  T* tile = reinterpret_cast<T*>(smem);
  const T* src = static_cast<const T*>(a.logits) + r0 * C;
  const bool whole = bulk && rows == block_rows;
  if (l == 0) {
    mbar_init(&bar, 1);
    if (whole) {
      const uint32_t bytes = (uint32_t)(rows * C * sizeof(T));
      mbar_arrive_expect_tx(&bar, bytes);
      bulk_g2s(tile, src, bytes, &bar);
    }
  }
  if (!whole)
#pragma unroll 4
    for (int i = l; i < rows * C; i += blockDim.x) tile[i] = src[i];
  __syncthreads();
  if (whole && !mbar_wait(&bar, 0)) {
    if (l == 0) atomicAdd(&g_teacher_wait_failures, 1ull);
    mbar_wait(&bar, 0);  // the copy in flight must end before the block does (bounded)
    return;
  }
  // Rows an even number of words apart: lane l starts at word l, so that the lanes
  // read different banks.
  const T* row = tile + (l < rows ? l : 0) * C;
  constexpr int kWord = 4 / sizeof(T);
  const bool skew = C % (2 * kWord) == 0;
  W best[MAX];
  auto scan = [&]() {  // any row, every test
#pragma unroll
    for (int i = 0; i < MAX; ++i) best[i] = 0;
    const int turn = skew ? (l * kWord) % C : 0;
    for (int c0 = 0; c0 < C; c0 += MAX) {
      W next[MAX];
#pragma unroll
      for (int i = 0; i < MAX; ++i) {
        int c = c0 + i + turn;
        if (c >= C) c -= C;
        next[i] = c0 + i < C ? K::make(row[c], c) : 0;
      }
      sort_desc(next);
      merge_desc(best, next);
    }
  };
  if constexpr (sizeof(T) == 2) {
    // Rows of whole words, two classes a word, few instructions a class.
    if (C % 2 == 0 && !skew) {
#pragma unroll
      for (int i = 0; i < MAX; ++i) best[i] = 0;
      const uint32_t* words = reinterpret_cast<const uint32_t*>(row);
      for (int c0 = 0; c0 < C; c0 += MAX) {
        W next[MAX];
        const uint32_t inverted = 0xffffu - (uint32_t)c0;
#pragma unroll
        for (int i = 0; i < MAX; i += 2) {
          next[i] = next[i + 1] = 0;
          if (c0 + i < C) K::quick(words[(c0 + i) >> 1], inverted - i, next[i], next[i + 1]);
        }
        sort_desc(next);
        merge_desc(best, next);
      }
      bool again = K::spoilt(best[0]);
#pragma unroll
      for (int i = 0; i < MAX; ++i)
        if (K::absent(best[i])) best[i] = 0;
      if (again) scan();
    } else {
      scan();
    }
  } else {
    scan();
  }
  __syncthreads();  // the tile is not needed any more: records are put together in its place
  const float first = best[0] ? K::value(best[0]) : 0.0f, levels = (float)((1 << a.bits) - 1);
  float last = first;
#pragma unroll
  for (int i = 0; i < MAX; ++i)
    if (i < a.k && best[i]) last = K::value(best[i]);
  // records an odd number of words apart
  const int pitch = a.rec_bytes + 4;
  if (l < rows) {
    uint8_t* rec = smem + l * pitch;
    *reinterpret_cast<float*>(rec) = first;
    *reinterpret_cast<float*>(rec + 4) = step_of(first, last, a.bits);
    const Quantiser quantise(first, last, levels);
    uint8_t* codes = rec + 8 + 2 * a.k;
    int low = 0;
#pragma unroll
    for (int i = 0; i < MAX; ++i) {
      if (i >= a.k) break;
      const int code = best[i] && first > last ? quantise(K::value(best[i]), levels) : 0;
      reinterpret_cast<int16_t*>(rec + 8)[i] = best[i] ? (int16_t)K::index(best[i]) : (int16_t)-1;
      if (a.bits == 8) codes[i] = (uint8_t)code;
      else if (i & 1) codes[i >> 1] = (uint8_t)(low | code << 4);
      else if (i + 1 == a.k) codes[i >> 1] = (uint8_t)code;
      low = code;
    }
    for (int b = 8 + 2 * a.k + (a.k * a.bits + 7) / 8; b < a.rec_bytes; ++b) rec[b] = 0;
  }
  __syncthreads();
  const int words = a.rec_bytes / 4;
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.records + r0 * a.rec_bytes);
  for (int i = l; i < rows * words; i += blockDim.x) {
    const int r = i / words;
    dst[i] = *reinterpret_cast<const uint32_t*>(smem + r * pitch + 4 * (i - r * words));
  }
}

// Across a warp: lane i's key of a descending sort of 32.
template <typename K>
__device__ __forceinline__ typename K::Word warp_sort(typename K::Word v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j >= 1; j /= 2) {
      const auto o = K::exchange(v, j);
      const bool larger = ((lane & k) == 0) == ((lane & j) == 0);
      v = (o > v) == larger ? o : v;
    }
  return v;
}
// The 32 largest of two descending runs, descending.
template <typename K>
__device__ __forceinline__ typename K::Word warp_merge(typename K::Word best, typename K::Word other, int lane) {
  const auto turned = K::shuffle(other, 31 - lane);
  best = best > turned ? best : turned;
#pragma unroll
  for (int j = 16; j >= 1; j /= 2) {
    const auto o = K::exchange(best, j);
    const bool larger = (lane & j) == 0;
    best = (o > best) == larger ? o : best;
  }
  return best;
}

template <typename T>
__global__ void __launch_bounds__(kWriteWarps * 32) k_teacher_write_warp(TeacherWriteArgs a) {
  using K = Key<T>;
  using W = typename K::Word;
  __shared__ W pending[kWriteWarps][64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWriteWarps + warp;
  if (r >= a.n) return;
  const int C = (int)a.classes, k = a.k;
  const T* s = static_cast<const T*>(a.logits) + r * C;
  const float low = lowest_of<T>();
  // Values decide until a class is taken: its key is made then.
  auto value_at = [&](int c) {
    const float v = to_f32(s[c]);
    return v > low && v < INFINITY ? v : -INFINITY;
  };
  float top = -INFINITY;  // largest of this lane
#pragma unroll 8
  for (int c = lane; c < C; c += 32) top = fmaxf(top, value_at(c));
  // At least k classes reach the k-th largest of the lanes' largest.
#pragma unroll
  for (int j = 2; j <= 32; j *= 2)
#pragma unroll
    for (int d = j / 2; d >= 1; d /= 2) {
      const float o = __shfl_xor_sync(~0u, top, d);
      top = ((lane & j) == 0) == ((lane & d) == 0) ? fmaxf(top, o) : fminf(top, o);
    }
  float bound = __shfl_sync(~0u, top, k - 1);  // -inf: fewer than k lanes have a class at all
  W best = 0;
  int held = 0;
  W* queue = pending[warp];
  for (int c0 = 0; c0 < C; c0 += 32 * 4) {
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = c0 + 32 * q + lane;
      v[q] = c < C ? value_at(c) : -INFINITY;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool mine = v[q] >= bound && v[q] != -INFINITY;
      const unsigned take = __ballot_sync(~0u, mine);
      if (take == 0) continue;
      const int c = c0 + 32 * q + lane;
      if (mine) queue[held + __popc(take & ((1u << lane) - 1))] = K::make(s[c], c);
      held += __popc(take);
      __syncwarp();
      if (held >= 32) {  // held is the same in every lane
        best = warp_merge<K>(best, warp_sort<K>(queue[lane], lane), lane);
        const W kth = K::shuffle(best, k - 1);
        if (kth != 0) bound = fmaxf(bound, K::value(kth));  // (equal values are sorted out by their keys)
        const W rest = lane < held - 32 ? queue[32 + lane] : 0;
        __syncwarp();
        queue[lane] = rest;
        held -= 32;
        __syncwarp();
      }
    }
  }
  if (held > 0) best = warp_merge<K>(best, warp_sort<K>(lane < held ? queue[lane] : 0, lane), lane);
  const bool mine = lane < k && best != 0;
  const int count = __popc(__ballot_sync(~0u, mine));
  const float value = mine ? K::value(best) : 0.0f;
  const float first = __shfl_sync(~0u, value, 0), last = __shfl_sync(~0u, value, count > 0 ? count - 1 : 0);
  const float levels = (float)((1 << a.bits) - 1);
  const int code = mine && first > last ? Quantiser(first, last, levels)(value, levels) : 0;
  uint8_t* rec = a.records + r * a.rec_bytes;
  if (lane == 0)
    *reinterpret_cast<float2*>(rec) = make_float2(first, step_of(first, last, a.bits));
  if (lane < k) reinterpret_cast<int16_t*>(rec + 8)[lane] = mine ? (int16_t)K::index(best) : (int16_t)-1;
  uint8_t* codes = rec + 8 + 2 * k;
  int used = 8 + 2 * k;
  if (a.bits == 8) {
    if (lane < k) codes[lane] = (uint8_t)code;
    used += k;
  } else {
    const int hi = __shfl_down_sync(~0u, code, 1);
    if (!(lane & 1) && lane < k) codes[lane >> 1] = (uint8_t)(code | (lane + 1 < k ? hi << 4 : 0));
    used += (k + 1) / 2;
  }
  for (int b = used + lane; b < a.rec_bytes; b += 32) rec[b] = 0;
}

// LANES (a power of two >= k) lanes per record, several records in flight.
template <int LANES>
__global__ void __launch_bounds__(256) k_teacher_read(const uint8_t* __restrict__ records, int64_t n_records,
                                                      const int64_t* __restrict__ rows, int64_t first_row, int64_t n,
                                                      int k, int bits, int rec_bytes, float* __restrict__ values,
                                                      int32_t* __restrict__ index) {
  constexpr int kFlight = 4, kGroups = 256 / LANES;
  const int e = threadIdx.x % LANES, group = threadIdx.x / LANES;
  for (int64_t r0 = (int64_t)blockIdx.x * kGroups * kFlight; r0 < n; r0 += (int64_t)gridDim.x * kGroups * kFlight) {
    int64_t rec[kFlight];
    float v[kFlight];
    int idx[kFlight];
#pragma unroll
    for (int q = 0; q < kFlight; ++q) {
      const int64_t r = r0 + q * kGroups + group;
      rec[q] = r < n ? (rows ? __ldg(rows + r) : first_row + r) : -1;
    }
#pragma unroll
    for (int q = 0; q < kFlight; ++q) {
      v[q] = -INFINITY;
      idx[q] = -1;
      if (rec[q] >= 0 && rec[q] < n_records && e < k) {
        const uint8_t* p = records + rec[q] * rec_bytes;
        const float2 head = __ldg(reinterpret_cast<const float2*>(p));
        const int i = __ldg(reinterpret_cast<const int16_t*>(p + 8) + e);
        const int byte = __ldg(p + 8 + 2 * k + (bits == 8 ? e : e >> 1));
        if (i >= 0) {
          idx[q] = i;
          v[q] = record_value(head.x, head.y, bits == 8 ? byte : (byte >> ((e & 1) * 4)) & 15);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < kFlight; ++q) {
      const int64_t r = r0 + q * kGroups + group;
      if (r < n && e < k) {
        values[r * k + e] = v[q];
        index[r * k + e] = idx[q];
      }
    }
  }
}

// The same for K = 8, 16 or 32 entries: K / 4 lanes per record, four entries each, so
// that a warp's results are whole contiguous lines; two records in flight per lane.
template <int K, int BITS>
__global__ void __launch_bounds__(256) k_teacher_read_whole(const uint8_t* __restrict__ records, int64_t n_records,
                                                            const int64_t* __restrict__ rows, int64_t first_row,
                                                            int64_t n, float* __restrict__ values,
                                                            int32_t* __restrict__ index) {
  constexpr int kBytes = (8 + 2 * K + K * BITS / 8 + 15) / 16 * 16, kLanes = K / 4, kFlight = 2;
  constexpr int kGroups = 256 / kLanes;
  const int q = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  for (int64_t r0 = (int64_t)blockIdx.x * kGroups * kFlight; r0 < n; r0 += (int64_t)gridDim.x * kGroups * kFlight) {
    int64_t rec[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int64_t r = r0 + i * kGroups + group;
      rec[i] = r < n ? (rows ? __ldg(rows + r) : first_row + r) : -1;
    }
    float2 head[kFlight];
    uint2 idx[kFlight];
    uint32_t codes[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      head[i] = make_float2(0.0f, 0.0f);
      idx[i] = make_uint2(0xffffffffu, 0xffffffffu);
      codes[i] = 0;
      if (rec[i] >= 0 && rec[i] < n_records) {
        const uint8_t* p = records + rec[i] * kBytes;
        head[i] = __ldg(reinterpret_cast<const float2*>(p));
        idx[i] = __ldg(reinterpret_cast<const uint2*>(p + 8) + q);
        if (BITS == 8) codes[i] = __ldg(reinterpret_cast<const uint32_t*>(p + 8 + 2 * K) + q);
        else codes[i] = __ldg(reinterpret_cast<const uint16_t*>(p + 8 + 2 * K) + q);
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int64_t r = r0 + i * kGroups + group;
      float v[4];
      int c[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[j] = max((int)(int16_t)((j < 2 ? idx[i].x : idx[i].y) >> (16 * (j & 1))), -1);
        v[j] = c[j] >= 0 ? record_value(head[i].x, head[i].y, (int)(codes[i] >> (BITS * j)) & ((1 << BITS) - 1)) : -INFINITY;
      }
      if (r < n) {
        *(reinterpret_cast<float4*>(values + r * K) + q) = make_float4(v[0], v[1], v[2], v[3]);
        *(reinterpret_cast<int4*>(index + r * K) + q) = make_int4(c[0], c[1], c[2], c[3]);
      }
    }
  }
}

template <int K>
static int launch_read_whole(const void* records, int64_t n_records, const int64_t* rows, int64_t first_row, int64_t n,
                             int bits, float* values, int32_t* index, cudaStream_t st) {
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, 256 / (K / 4) * 2), 148 * 32);
  auto* kernel = bits == 8 ? k_teacher_read_whole<K, 8> : k_teacher_read_whole<K, 4>;
  kernel<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(records), n_records, rows, first_row, n, values, index);
  return check_launch("k_teacher_read_whole");
}

template <typename T, int MAX>
static int launch_rows(const TeacherWriteArgs& a, cudaStream_t st) {
  const size_t row = a.classes * sizeof(T);
  // 64 rows or 32 (whole warps, and a multiple of 16 bytes)
  int rows = kStagedRows;
  while (rows > 32 && rows * row > kStagedSmem) rows /= 2;
  const size_t smem = std::max((size_t)rows * row, (size_t)rows * (a.rec_bytes + 4));
  auto* kernel = k_teacher_write_rows<T, MAX>;
  if (smem > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kStagedSmem);
    if (e != cudaSuccess) return set_error(GS_ERR_CUDA, "k_teacher_write_rows: %s", cudaGetErrorString(e));
  }
  kernel<<<(unsigned)ceil_div(a.n, rows), rows, smem, st>>>(a, rows, aligned(a.logits, 16));
  return check_launch("k_teacher_write_rows");
}

template <typename T>
static int launch_write(const TeacherWriteArgs& a, cudaStream_t st) {
  // A thread per row needs many rows, short ones and few entries (its network grows
  // with k log^2 k).
  if (a.n >= 148 * 32 && a.classes * sizeof(T) <= kStagedSmem / 32 && a.k <= 16)
    return a.k <= 4 ? launch_rows<T, 4>(a, st) : a.k <= 8 ? launch_rows<T, 8>(a, st) : launch_rows<T, 16>(a, st);
  k_teacher_write_warp<T><<<(unsigned)ceil_div(a.n, kWriteWarps), kWriteWarps * 32, 0, st>>>(a);
  return check_launch("k_teacher_write_warp");
}

template <int LANES>
static int launch_read(const void* records, int64_t n_records, const int64_t* rows, int64_t first_row, int64_t n, int k,
                       int bits, float* values, int32_t* index, cudaStream_t st) {
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, 256 / LANES * 4), 148 * 32);
  k_teacher_read<LANES><<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(records), n_records, rows, first_row, n, k,
                                              bits, record_bytes(k, bits), values, index);
  return check_launch("k_teacher_read");
}

static int check_cache(const char* who, int64_t n, const void* records, int64_t n_records, int k, int bits) {
  if (k < 1 || k > GS_CACHE_MAX_K)
    return set_error(GS_ERR_INVALID_ARG, "%s: k must be in [1, %d] (got %d)", who, GS_CACHE_MAX_K, k);
  if (bits != 8 && bits != 4) return set_error(GS_ERR_INVALID_ARG, "%s: bits must be 8 or 4 (got %d)", who, bits);
  if (n < 0 || n_records < 0) return set_error(GS_ERR_INVALID_ARG, "%s: negative size", who);
  if (n > 0 && n_records > 0 && !records) return set_error(GS_ERR_INVALID_ARG, "%s: NULL pointer", who);
  if (!aligned(records, 16)) return set_error(GS_ERR_INVALID_ARG, "%s: records must be 16-byte aligned", who);
  return GS_OK;
}

}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_teacher_record_bytes(int k, int bits) {
  if (k < 1 || k > GS_CACHE_MAX_K || (bits != 8 && bits != 4)) return 0;
  return (size_t)record_bytes(k, bits);
}

int gs_teacher_write(const void* logits, int dtype, int64_t n, int64_t classes, void* records,
                     int64_t n_records, int64_t first_row, int k, int bits, void* stream) {
  clear_error();
  if (int e = check_cache("gs_teacher_write", n, records, n_records, k, bits)) return e;
  if (!dtype_ok(dtype)) return set_error(GS_ERR_INVALID_ARG, "gs_teacher_write: unknown dtype %d", dtype);
  if (classes < 1 || classes > GS_CACHE_MAX_CLASSES)
    return set_error(GS_ERR_INVALID_ARG, "gs_teacher_write: classes must be in [1, %d]", GS_CACHE_MAX_CLASSES);
  if (first_row < 0 || first_row > n_records || n > n_records - first_row)
    return set_error(GS_ERR_INVALID_ARG, "gs_teacher_write: rows [%lld, %lld) are outside the cache of %lld rows",
                     (long long)first_row, (long long)(first_row + n), (long long)n_records);
  if (n == 0) return GS_OK;
  if (!logits) return set_error(GS_ERR_INVALID_ARG, "gs_teacher_write: NULL pointer");
  if (ceil_div(n, kWriteWarps) > INT32_MAX)
    return set_error(GS_ERR_CAPACITY, "gs_teacher_write: too many rows for one call");
  TeacherWriteArgs a{};
  a.logits = logits; a.n = n; a.classes = classes; a.k = k; a.bits = bits;
  a.rec_bytes = record_bytes(k, bits);
  a.records = static_cast<uint8_t*>(records) + first_row * a.rec_bytes;
  cudaStream_t st = as_stream(stream);
  if (dtype == GS_F32) return launch_write<float>(a, st);
  if (dtype == GS_F16) return launch_write<__half>(a, st);
  return launch_write<__nv_bfloat16>(a, st);
}

int gs_teacher_read(const void* records, int64_t n_records, const int64_t* rows, int64_t first_row, int64_t n,
                    int k, int bits, float* values, int32_t* index, void* stream) {
  clear_error();
  if (int e = check_cache("gs_teacher_read", n, records, n_records, k, bits)) return e;
  if (n == 0) return GS_OK;
  if (!values || !index) return set_error(GS_ERR_INVALID_ARG, "gs_teacher_read: NULL pointer");
  cudaStream_t st = as_stream(stream);
  if (aligned(values, 16) && aligned(index, 16)) {
    if (k == 8) return launch_read_whole<8>(records, n_records, rows, first_row, n, bits, values, index, st);
    if (k == 16) return launch_read_whole<16>(records, n_records, rows, first_row, n, bits, values, index, st);
    if (k == 32) return launch_read_whole<32>(records, n_records, rows, first_row, n, bits, values, index, st);
  }
  if (k <= 4) return launch_read<4>(records, n_records, rows, first_row, n, k, bits, values, index, st);
  if (k <= 8) return launch_read<8>(records, n_records, rows, first_row, n, k, bits, values, index, st);
  if (k <= 16) return launch_read<16>(records, n_records, rows, first_row, n, k, bits, values, index, st);
  return launch_read<32>(records, n_records, rows, first_row, n, k, bits, values, index, st);
}

}  // extern "C"
