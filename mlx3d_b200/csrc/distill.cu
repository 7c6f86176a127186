// Distillation from a teacher's largest logits: loss and gradient.
//
//   p = softmax over the row's present teacher entries z_k / T
//   q = softmax over all classes s_c / T
//   L = w T^2 sum_k p_k (log p_k - log q_{i_k}),  dL/ds_c = w T (q_c - sum_{i_k = c} p_k)
//
// One warp per row; the running maximum and sum of the student's softmax are
// kept per lane in one pass and merged over the warp, the gradient rereads the
// row from cache.
#include "feature_common.cuh"

namespace gs {

constexpr int kDistillWarps = 8;
constexpr int kDistillMaxBlocks = 148 * 8;

struct DistillArgs {
  const void* logits;
  int64_t n, classes;
  gs_teacher t;
  int rec_bytes;
  float temp, inv_temp;
  const float* weight;
  float grad_scale;  // scale * T
  const float* cot;
  int cot_per_row;
  float* row_loss;
  double* partials;  // one per block, or NULL
  void* grad;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Entry e of row r: index -1 where absent.
__device__ __forceinline__ void teacher_entry(const DistillArgs& a, int64_t r, int64_t rec, int e, float* z, int* idx) {
  const gs_teacher& t = a.t;
  int i;
  float v;
  if (a.rec_bytes) {
    if (rec < 0) {
      *z = -INFINITY;
      *idx = -1;
      return;
    }
    const uint8_t* p = static_cast<const uint8_t*>(t.records) + rec * a.rec_bytes;
    const float2 head = *reinterpret_cast<const float2*>(p);
    i = reinterpret_cast<const int16_t*>(p + 8)[e];
    v = record_value(head.x, head.y, record_code(p + 8 + 2 * t.k, e, t.bits));
  } else {
    const int64_t at = r * t.k + e;
    i = t.index[at];
    v = t.values_dtype == GS_F32   ? static_cast<const float*>(t.values)[at]
        : t.values_dtype == GS_F16 ? to_f32(static_cast<const __half*>(t.values)[at])
                                   : to_f32(static_cast<const __nv_bfloat16*>(t.values)[at]);
  }
  const bool here = i >= 0 && i < a.classes && v != -INFINITY;
  *z = here ? v : -INFINITY;
  *idx = here ? i : -1;
}

template <typename T>
__global__ void __launch_bounds__(kDistillWarps * 32) k_distill_rows(DistillArgs a) {
  extern __shared__ float2 smem[];  // k (index, p) pairs per warp
  __shared__ double block_sum[kDistillWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = a.t.k;
  float2* ent = smem + warp * k;
  const T* logits = static_cast<const T*>(a.logits);
  double acc = 0.0;
  for (int64_t r = (int64_t)blockIdx.x * kDistillWarps + warp; r < a.n; r += (int64_t)gridDim.x * kDistillWarps) {
    const T* s = logits + r * a.classes;
    // teacher
    int64_t rec = 0;
    if (a.rec_bytes) {
      rec = a.t.rows ? a.t.rows[r] : a.t.first_row + r;
      if (rec < 0 || rec >= a.t.n_records) rec = -1;
    }
    float zmax = -INFINITY;
    bool any = false;
    for (int e = lane; e < k; e += 32) {
      float z;
      int idx;
      teacher_entry(a, r, rec, e, &z, &idx);
      ent[e] = make_float2(__int_as_float(idx), z);
      any |= idx >= 0;
      zmax = fmaxf(zmax, z);
    }
    any = __any_sync(~0u, any);
    T* g = static_cast<T*>(a.grad);
    if (g) g += r * a.classes;
    const float w = a.weight ? a.weight[r] : 1.0f;
    if (!any) {  // nothing to learn from: no loss, no gradient
      if (g)
        for (int64_t c = lane; c < a.classes; c += 32) g[c] = from_f32<T>(0.0f);
      if (a.row_loss && lane == 0) a.row_loss[r] = 0.0f;
      __syncwarp();
      continue;
    }
    zmax = warp_max(zmax);
    float tot = 0.0f;
    for (int e = lane; e < k; e += 32)
      if (__float_as_int(ent[e].x) >= 0) tot += expf((ent[e].y - zmax) * a.inv_temp);
    tot = warp_sum(tot);
    const float log_tot = logf(tot);
    // student: running maximum and sum
    float m = -INFINITY, sum = 0.0f;
    for (int64_t c = lane; c < a.classes; c += 32) {
      const float v = to_f32(s[c]);
      if (v > m) {
        sum = sum * expf((m - v) * a.inv_temp) + 1.0f;
        m = v;
      } else {
        sum += expf((v - (m == -INFINITY ? 0.0f : m)) * a.inv_temp);
      }
    }
    const float mw = warp_max(m);
    sum = warp_sum(m == mw ? sum : sum * expf((m - mw) * a.inv_temp));
    m = mw;
    const float lse = logf(sum);
    float loss = 0.0f;
    for (int e = lane; e < k; e += 32) {
      const int idx = __float_as_int(ent[e].x);
      float p = 0.0f;
      if (idx >= 0) {
        const float zz = (ent[e].y - zmax) * a.inv_temp;
        p = expf(zz) / tot;
        const float logq = (to_f32(s[idx]) - m) * a.inv_temp - lse;
        if (p != 0.0f) loss += p * (zz - log_tot - logq);
      }
      ent[e].y = p;
    }
    loss = warp_sum(loss) * (a.temp * a.temp) * w;
    if (lane == 0) {
      if (a.row_loss) a.row_loss[r] = loss;
      acc += (double)loss;
    }
    if (g) {
      const float f = w * a.grad_scale * (a.cot ? a.cot[a.cot_per_row ? r : 0] : 1.0f);
      for (int64_t c = lane; c < a.classes; c += 32)
        g[c] = from_f32<T>(expf((to_f32(s[c]) - m) * a.inv_temp - lse) * f);
      __syncwarp();
      // The teacher's classes: the first entry of a class writes q - (sum of the class's p).
      for (int e = lane; e < k; e += 32) {
        const int idx = __float_as_int(ent[e].x);
        if (idx < 0) continue;
        bool first = true;
        float p = 0.0f;
        for (int j = 0; j < k; ++j)
          if (__float_as_int(ent[j].x) == idx) {
            first &= j >= e;
            p += ent[j].y;
          }
        if (first) g[idx] = from_f32<T>((expf((to_f32(s[idx]) - m) * a.inv_temp - lse) - p) * f);
      }
    }
    __syncwarp();
  }
  if (a.partials) {
    if (lane == 0) block_sum[warp] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0.0;
      for (int i = 0; i < kDistillWarps; ++i) t += block_sum[i];
      a.partials[blockIdx.x] = t;
    }
  }
}

__global__ void k_distill_finish(const double* partials, int n, double scale, float* loss) {
  __shared__ double part[256];
  double t = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) t += partials[i];
  part[threadIdx.x] = t;
  for (int o = 128; o; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
  }
  if (threadIdx.x == 0) *loss = (float)(part[0] * scale);
}

}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_distill_workspace_bytes(void) { return sizeof(double) * kDistillMaxBlocks; }

int gs_distill(const void* logits, int dtype, int64_t n, int64_t classes, const gs_teacher* teacher,
               float temperature, const float* weight, double scale, const float* cotangent,
               int cotangent_per_row, float* row_loss, float* loss, void* grad, void* workspace,
               size_t workspace_bytes, void* stream) {
  clear_error();
  if (!dtype_ok(dtype)) return set_error(GS_ERR_INVALID_ARG, "gs_distill: unknown dtype %d", dtype);
  if (n < 0 || classes < 1 || classes > INT32_MAX)
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: logits must be (n >= 0, 1 <= classes < 2^31)");
  if (!teacher) return set_error(GS_ERR_INVALID_ARG, "gs_distill: teacher is NULL");
  const bool cached = teacher->bits != 0;
  const int max_k = cached ? GS_CACHE_MAX_K : GS_TEACHER_MAX_K;
  if (teacher->k < 1 || teacher->k > max_k)
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: k must be in [1, %d] (got %d)", max_k, teacher->k);
  if (!(temperature > 0.0f) || temperature > FLT_MAX || 1.0f / temperature > FLT_MAX)
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: temperature must be positive and finite");
  if (cached) {
    if (teacher->bits != 8 && teacher->bits != 4)
      return set_error(GS_ERR_INVALID_ARG, "gs_distill: bits must be 8 or 4 (got %d)", teacher->bits);
    if (teacher->n_records < 0) return set_error(GS_ERR_INVALID_ARG, "gs_distill: n_records is negative");
    if (!aligned(teacher->records, 16))
      return set_error(GS_ERR_INVALID_ARG, "gs_distill: records must be 16-byte aligned");
  } else if (!dtype_ok(teacher->values_dtype)) {
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: unknown values_dtype %d", teacher->values_dtype);
  }
  if (n > 0 && (!logits || (cached ? (!teacher->records && teacher->n_records > 0) : (!teacher->index || !teacher->values))))
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: NULL pointer");
  if (loss && (!workspace || workspace_bytes < gs_distill_workspace_bytes()))
    return set_error(GS_ERR_CAPACITY, "gs_distill: workspace too small");
  DistillArgs a{};
  a.logits = logits; a.n = n; a.classes = classes;
  a.t = *teacher;
  a.rec_bytes = cached ? record_bytes(teacher->k, teacher->bits) : 0;
  a.temp = temperature; a.inv_temp = 1.0f / temperature;
  a.weight = weight;
  a.grad_scale = (float)(scale * (double)temperature);
  a.cot = cotangent; a.cot_per_row = cotangent_per_row;
  a.row_loss = row_loss; a.grad = grad;
  a.partials = loss ? static_cast<double*>(workspace) : nullptr;
  cudaStream_t st = as_stream(stream);
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, kDistillWarps), kDistillMaxBlocks);
  if (grid > 0) {
    const size_t smem = sizeof(float2) * kDistillWarps * teacher->k;
    if (dtype == GS_F32) k_distill_rows<float><<<grid, kDistillWarps * 32, smem, st>>>(a);
    else if (dtype == GS_F16) k_distill_rows<__half><<<grid, kDistillWarps * 32, smem, st>>>(a);
    else k_distill_rows<__nv_bfloat16><<<grid, kDistillWarps * 32, smem, st>>>(a);
    if (int e = check_launch("k_distill_rows")) return e;
  }
  if (loss) {
    k_distill_finish<<<1, 256, 0, st>>>(a.partials, (int)grid, scale, loss);
    return check_launch("k_distill_finish");
  }
  return GS_OK;
}

}  // extern "C"
