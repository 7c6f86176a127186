// Teacher cache: a row's k largest logits, kept in 8 or 4 bits.
//
// Writing: one warp per row.  The order is (value descending, index
// ascending); entry j + 1 is the best one that comes after entry j in that
// order, found by a scan of the row (from cache after the first) and a warp
// reduction.
// Reading: one thread per entry.
#include "feature_common.cuh"

namespace gs {

constexpr int kWriteWarps = 8;

struct TeacherWriteArgs {
  const void* logits;
  int64_t n, classes;
  uint8_t* records;  // of first_row
  int k, bits, rec_bytes;
};

// code = (2^bits - 1) (first - v) / (first - last) to nearest, ties to even.
// The 32-bit quotient decides except next to a border, where the exact
// differences do: with few mantissa bits in the logits many quotients lie
// exactly between two codes.
__device__ __forceinline__ int quantise(float first, float last, float v, float levels) {
  const float q = (first - v) * levels / (first - last);
  const float near = rintf(q);
  if (fabsf(q - near) < 0.499f) return (int)near;  // |error of q| < 255 * 3 * 2^-24 < 1e-4
  return (int)rint(((double)first - (double)v) * (double)levels / ((double)first - (double)last));
}

template <typename T>
__global__ void __launch_bounds__(kWriteWarps * 32) k_teacher_write_rows(TeacherWriteArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * kWriteWarps + warp;
  if (r >= a.n) return;
  const T* s = static_cast<const T*>(a.logits) + r * a.classes;
  const float low = lowest_of<T>();
  float mine = -INFINITY;  // lane e holds entry e
  int mine_idx = -1;
  float prev = INFINITY;
  int prev_idx = -1;
  float first = 0.0f, last = 0.0f;
  int count = 0;
  for (int e = 0; e < a.k; ++e) {
    float best = -INFINITY;
    int best_idx = INT32_MAX;
    for (int c = lane; c < a.classes; c += 32) {
      const float v = to_f32(s[c]);
      if (!(v > low) || v == INFINITY) continue;
      const bool after = v < prev || (v == prev && c > prev_idx);
      if (after && v > best) {  // ascending c: the lowest index stays
        best = v;
        best_idx = c;
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float ov = __shfl_xor_sync(~0u, best, o);
      const int oi = __shfl_xor_sync(~0u, best_idx, o);
      if (ov > best || (ov == best && oi < best_idx)) {
        best = ov;
        best_idx = oi;
      }
    }
    if (best == -INFINITY) break;
    if (e == 0) first = best;
    last = best;
    prev = best;
    prev_idx = best_idx;
    ++count;
    if (lane == e) {
      mine = best;
      mine_idx = best_idx;
    }
  }
  const float levels = (float)((1 << a.bits) - 1);
  int code = 0;
  if (lane < count && first > last) code = quantise(first, last, mine, levels);
  uint8_t* rec = a.records + r * a.rec_bytes;
  if (lane == 0) {
    const float scale = (float)(((double)first - (double)last) / (double)levels);
    *reinterpret_cast<float2*>(rec) = make_float2(first, scale);
  }
  if (lane < a.k) reinterpret_cast<int16_t*>(rec + 8)[lane] = (int16_t)mine_idx;
  uint8_t* codes = rec + 8 + 2 * a.k;
  int used = 8 + 2 * a.k;
  if (a.bits == 8) {
    if (lane < a.k) codes[lane] = (uint8_t)code;
    used += a.k;
  } else {
    const int hi = __shfl_down_sync(~0u, code, 1);
    if (!(lane & 1) && lane < a.k) codes[lane >> 1] = (uint8_t)(code | (lane + 1 < a.k ? hi << 4 : 0));
    used += (a.k + 1) / 2;
  }
  for (int b = used + lane; b < a.rec_bytes; b += 32) rec[b] = 0;
}

__global__ void k_teacher_read(const uint8_t* __restrict__ records, int64_t n_records, const int64_t* rows,
                               int64_t first_row, int64_t n, int k, int bits, int rec_bytes, float* values,
                               int32_t* index) {
  const int64_t total = n * k;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / k;
    const int e = (int)(i - r * k);
    const int64_t rec = rows ? rows[r] : first_row + r;
    float v = -INFINITY;
    int idx = -1;
    if (rec >= 0 && rec < n_records) {
      const uint8_t* p = records + rec * rec_bytes;
      const float2 head = *reinterpret_cast<const float2*>(p);
      idx = reinterpret_cast<const int16_t*>(p + 8)[e];
      if (idx >= 0) v = record_value(head.x, head.y, record_code(p + 8 + 2 * k, e, bits));
      else idx = -1;
    }
    values[i] = v;
    index[i] = idx;
  }
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
  const unsigned grid = (unsigned)ceil_div(n, kWriteWarps);
  cudaStream_t st = as_stream(stream);
  if (dtype == GS_F32) k_teacher_write_rows<float><<<grid, kWriteWarps * 32, 0, st>>>(a);
  else if (dtype == GS_F16) k_teacher_write_rows<__half><<<grid, kWriteWarps * 32, 0, st>>>(a);
  else k_teacher_write_rows<__nv_bfloat16><<<grid, kWriteWarps * 32, 0, st>>>(a);
  return check_launch("k_teacher_write_rows");
}

int gs_teacher_read(const void* records, int64_t n_records, const int64_t* rows, int64_t first_row, int64_t n,
                    int k, int bits, float* values, int32_t* index, void* stream) {
  clear_error();
  if (int e = check_cache("gs_teacher_read", n, records, n_records, k, bits)) return e;
  if (n == 0) return GS_OK;
  if (!values || !index) return set_error(GS_ERR_INVALID_ARG, "gs_teacher_read: NULL pointer");
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n * k, 256), 148 * 32);
  k_teacher_read<<<grid, 256, 0, as_stream(stream)>>>(static_cast<const uint8_t*>(records), n_records, rows,
                                                      first_row, n, k, bits, record_bytes(k, bits), values, index);
  return check_launch("k_teacher_read");
}

}  // extern "C"
