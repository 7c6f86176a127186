// Distillation from a teacher's largest logits: loss and gradient.
//
//   p = softmax over the row's present teacher entries z_k / T
//   q = softmax over all classes s_c / T
//   L = w T^2 sum_k p_k (log p_k - log q_{i_k}),  dL/ds_c = w T (q_c - sum_{i_k = c} p_k)
//
// Bound by memory: the logits are read once and the gradient written once.
//   k_distill_warp  short rows: every warp walks tiles of its own, loaded
//                   and stored by bulk copies, with no block barrier; dozens of
//                   warps per SM overlap their copies with each other's
//                   arithmetic.  The classes of a row are shared by 4 to 32 lanes;
//                   the teacher's few entries by as many as make the tile's rows a
//                   whole warp.  Instructions bound it: 1920x1080x150 in float32
//                   takes 492 us (its bytes at a copy's rate: 396) with 8 entries,
//                   with one lane per row for the entries (8 of 32 busy) 15 % more.
//                   More than 8 entries a row are compared pair by pair: 16 take 1251.
//   k_distill_long  rows that fit in a warp's registers: one warp per row.
//   k_distill_row   longer rows: one block per row.
#include "feature_common.cuh"

namespace gs {

constexpr int kDistillMaxBlocks = 148 * 16;
constexpr int kWarpBlock = 128, kRowThreads = 256;

__device__ unsigned long long g_distill_wait_failures;

int distill_wait_failures(unsigned long long* out, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_distill_wait_failures, sizeof(*out));
  if (e == cudaSuccess && reset) {
    const unsigned long long z = 0;
    e = cudaMemcpyToSymbol(g_distill_wait_failures, &z, sizeof(z));
  }
  return (int)e;
}

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

// Over G consecutive lanes.
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
// 2^x to 2 ulp.  Arguments are (difference) * (log2 e / T): three roundings,
// each relative to the exponent.
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// ln x and 1 / x to 2 ulp
__device__ __forceinline__ float ln_of(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y * 0.69314718055994531f;
}
__device__ __forceinline__ float rcp_of(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float2 checked_entry(int idx, float z, int64_t classes) {
  const bool here = idx >= 0 && idx < classes && z != -INFINITY;
  return make_float2(__int_as_float(here ? idx : -1), here ? z : -INFINITY);
}
template <int STRIDE, typename V>
__device__ __forceinline__ void stage_arrays(const DistillArgs& a, float2* ents, int64_t at, int count, int first) {
  const V* z = static_cast<const V*>(a.t.values) + at;
  const int32_t* idx = a.t.index + at;
#pragma unroll 4
  for (int i = first; i < count; i += STRIDE) ents[i] = checked_entry(__ldg(idx + i), to_f32(z[i]), a.classes);
}

// Teacher entries of `rows` rows from r0 as (index, z), index -1 where absent,
// by STRIDE threads of which this is number `first`.
template <int STRIDE>
__device__ __forceinline__ void stage_entries(const DistillArgs& a, float2* ents, int64_t r0, int rows, int first) {
  const int k = a.t.k;
  if (!a.rec_bytes) {
    if (a.t.values_dtype == GS_F32) stage_arrays<STRIDE, float>(a, ents, r0 * k, rows * k, first);
    else if (a.t.values_dtype == GS_F16) stage_arrays<STRIDE, __half>(a, ents, r0 * k, rows * k, first);
    else stage_arrays<STRIDE, __nv_bfloat16>(a, ents, r0 * k, rows * k, first);
    return;
  }
  const uint32_t per_k = 0xffffffffu / k + 1;  // i / k for i < 2^16
#pragma unroll 4
  for (int i = first; i < rows * k; i += STRIDE) {
    const int r = k == 1 ? i : (int)__umulhi((uint32_t)i, per_k), e = i - r * k;
    const int64_t rec = a.t.rows ? __ldg(a.t.rows + r0 + r) : a.t.first_row + r0 + r;
    float2 v = make_float2(__int_as_float(-1), -INFINITY);
    if (rec >= 0 && rec < a.t.n_records) {
      const uint8_t* p = static_cast<const uint8_t*>(a.t.records) + rec * a.rec_bytes;
      const float2 head = *reinterpret_cast<const float2*>(p);
      v = checked_entry(reinterpret_cast<const int16_t*>(p + 8)[e],
                        record_value(head.x, head.y, record_code(p + 8 + 2 * k, e, a.t.bits)), a.classes);
    }
    ents[i] = v;
  }
}

// The sum of a double per thread over the block, in a fixed order.
__device__ __forceinline__ void block_partial(double v, double* out) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) t += part[i];
    *out = t;
  }
}

// The teacher's side of a row by a warp: entries (index, z) become
// (index, p); returns whether any is present (in every lane).
//   term = sum_k p_k ((z_k - max z) - (s_k - m)) / T - log sum_k exp((z_k - max z) / T)
// so that the loss is T^2 (term + log sum_c exp((s_c - m) / T)), as sum_k p_k = 1.
template <typename Logit>
__device__ __forceinline__ bool teacher_terms(float2* ent, int k, int lane, float m, float inv_temp, Logit logit,
                                              float& term) {
  const float c2 = inv_temp * kLog2e;
  float zmax = -INFINITY;
  bool mine = false;
  for (int e = lane; e < k; e += 32) {
    mine |= __float_as_int(ent[e].x) >= 0;
    zmax = fmaxf(zmax, ent[e].y);
  }
  const unsigned present = __ballot_sync(~0u, mine);
  zmax = group_max<32>(zmax);
  float tot = 0.0f;
  for (int e = lane; e < k; e += 32)
    if (__float_as_int(ent[e].x) >= 0) tot += exp2_of((ent[e].y - zmax) * c2);
  tot = group_sum<32>(tot);
  const float inv_tot = rcp_of(tot);
  float sum = 0.0f;
  for (int e = lane; e < k; e += 32) {
    const int idx = __float_as_int(ent[e].x);
    float p = 0.0f;
    if (idx >= 0) {
      const float z = ent[e].y - zmax;
      p = exp2_of(z * c2) * inv_tot;
      if (p != 0.0f) sum += p * ((z - (logit(idx) - m)) * inv_temp);
    }
    ent[e].y = p;
  }
  term = group_sum<32>(sum) - ln_of(tot);
  return present != 0;
}

// Gradients of the teacher's classes, scaled: the first entry of a class holds
// (class, f (q - sum of the class's p)), every other one (-1, -).
template <typename Logit>
__device__ __forceinline__ void class_gradients(const float2* ent, float2* out, int k, bool repeats, int lane, float m,
                                                float c2, float inv_sum, float f, Logit logit) {
  for (int e = lane; e < k; e += 32) {
    const int idx = __float_as_int(ent[e].x);
    int to = -1;
    float g = 0.0f;
    if (idx >= 0) {
      bool first = true;
      float p = ent[e].y;
      if (repeats) {
        p = 0.0f;
        for (int j = 0; j < k; ++j) {
          const float2 o = ent[j];
          if (__float_as_int(o.x) == idx) {
            first &= j >= e;
            p += o.y;
          }
        }
      }
      if (first) {
        to = idx;
        g = (exp2_of((logit(idx) - m) * c2) * inv_sum - p) * f;
      }
    }
    out[e] = make_float2(__int_as_float(to), g);
  }
}

// What a warp keeps of a row besides its logits and entries.
struct RowState {
  float weight, factor;  // of the loss, of the gradient
  float term;            // the teacher's part of the loss; NaN-free "none": any == 0
  float m, inv;          // maximum and 1 / sum of the student's exponentials
  int any, repeats;      // entries present; a class twice among them
  float lse;
};

// Over the L neighbouring lanes that share a row's entries; lane `sub` of them has
// entries sub, sub + L, ...: with MAX > 0 up to MAX of them, in registers, otherwise
// any number, through memory.
//
// The teacher's softmax of one row: entries (index, z) -> (index, p).
template <int L, int MAX>
__device__ __forceinline__ void teacher_row(float2* ent, int k, int sub, float inv_temp, RowState& st) {
  const float c2 = inv_temp * kLog2e;
  float zmax = -INFINITY, tot = 0.0f, sum = 0.0f;
  bool any = false, twice = false;
  if constexpr (MAX > 0) {
    int idx[MAX];
    float z[MAX];
#pragma unroll
    for (int i = 0; i < MAX; ++i) {
      const int e = sub + L * i;
      const float2 v = e < k ? ent[e] : make_float2(__int_as_float(-1), -INFINITY);
      idx[i] = __float_as_int(v.x);
      z[i] = v.y;
      zmax = fmaxf(zmax, v.y);
      any |= idx[i] >= 0;
      idx[i] = idx[i] >= 0 ? idx[i] : -1 - e;  // absent entries differ from each other
#pragma unroll
      for (int j = 0; j < i; ++j) twice |= idx[i] == idx[j];
    }
#pragma unroll
    for (int d = 1; d < L; ++d)
#pragma unroll
      for (int i = 0; i < MAX; ++i) {
        const int other = __shfl_xor_sync(~0u, idx[i], d);
#pragma unroll
        for (int j = 0; j < MAX; ++j) twice |= other == idx[j];
      }
    zmax = group_max<L>(zmax);
#pragma unroll
    for (int i = 0; i < MAX; ++i) {
      const float d = z[i] - zmax;
      z[i] = idx[i] >= 0 ? exp2_of(d * c2) : 0.0f;
      if (z[i] != 0.0f) sum += z[i] * (d * inv_temp);
      tot += z[i];
    }
    tot = group_sum<L>(tot);
    const float inv = rcp_of(tot);
#pragma unroll
    for (int i = 0; i < MAX; ++i)
      if (sub + L * i < k) ent[sub + L * i].y = z[i] * inv;
    sum = group_sum<L>(sum) * inv;
  } else {
    for (int e = sub; e < k; e += L) {
      const float2 v = ent[e];
      const int idx = __float_as_int(v.x);
      zmax = fmaxf(zmax, v.y);
      any |= idx >= 0;
      if (idx >= 0)
        for (int j = 0; j < e; ++j) twice |= __float_as_int(ent[j].x) == idx;
    }
    zmax = group_max<L>(zmax);
    for (int e = sub; e < k; e += L) {
      const float2 v = ent[e];
      float x = 0.0f;
      if (__float_as_int(v.x) >= 0) {
        const float d = v.y - zmax;
        x = exp2_of(d * c2);
        if (x != 0.0f) sum += x * (d * inv_temp);
      }
      tot += x;
      ent[e].y = x;
    }
    tot = group_sum<L>(tot);
    const float inv = rcp_of(tot);
    for (int e = sub; e < k; e += L) ent[e].y *= inv;
    sum = group_sum<L>(sum) * inv;
  }
  int found = (any ? 1 : 0) | (twice ? 2 : 0);
#pragma unroll
  for (int o = L / 2; o; o >>= 1) found |= __shfl_xor_sync(~0u, found, o);
  st.any = found & 1;
  st.repeats = found & 2;
  st.term = sum - ln_of(tot);  // sum_k p_k log p_k
}

// sum_k p_k (s_k - m) / T of a row, this lane's part, and the gradients of the
// teacher's classes (unless fix is NULL): the first entry of a class holds (class,
// factor * (q - sum of the class's p)), every other one (-1, -).
template <int L, int MAX, typename T>
__device__ __forceinline__ float class_row(const T* s, const float2* ent, float2* fix, int k, int sub, float inv_temp,
                                           const RowState& st) {
  const float c2 = inv_temp * kLog2e;
  float cross = 0.0f;
#pragma unroll MAX > 0 ? MAX : 1
  for (int i = 0; i < (MAX > 0 ? MAX : k); ++i) {
    const int e = sub + L * i;
    if (e >= k) break;
    const float2 v = ent[e];
    const int idx = __float_as_int(v.x);
    int to = -1;
    float g = 0.0f;
    if (idx >= 0) {
      const float d = to_f32(s[idx]) - st.m;
      if (v.y != 0.0f) cross += v.y * (d * inv_temp);
      if (fix) {
        bool first = true;
        float p = v.y;
        if (st.repeats) {
          p = 0.0f;
#pragma unroll 1
          for (int j = 0; j < k; ++j) {
            const float2 o = ent[j];
            if (__float_as_int(o.x) == idx) {
              first &= j >= e;
              p += o.y;
            }
          }
        }
        if (first) {
          to = idx;
          g = (exp2_of(d * c2) * st.inv - p) * st.factor;
        }
      }
    }
    if (fix) fix[e] = make_float2(__int_as_float(to), g);
  }
  return cross;
}

// Shared memory of a warp: two tiles, then entries, fixes, row states.
constexpr int kWarpBuffers = 2;
constexpr int kTileRows = 8;
__host__ __device__ inline size_t warp_tile_bytes(int rows, int64_t classes, int elem) {
  return ((size_t)rows * classes * elem + 127) & ~(size_t)127;
}
__host__ __device__ inline size_t warp_smem(int rows, int64_t classes, int elem, int k) {
  return kWarpBuffers * warp_tile_bytes(rows, classes, elem) + (((size_t)rows * (16 * k + sizeof(RowState)) + 127) & ~(size_t)127);
}

// G lanes share a row, each holding EACH of its logits in registers, as pairs of
// neighbours; the first FULL of them exist for sure.  Pairs are aligned: with an ODD
// number of classes every second row starts inside one, and shares its first and last
// pair with the rows beside it.  The exponentials of all rows of the tile (ROUNDS
// times 32 / G, a multiple of 8, which is one of 16 bytes) stay in registers for the
// gradient; with ROUNDS = 0 a tile has kTileRows rows and they are computed again.
template <typename T, int G, int EACH, int FULL, int ROUNDS, bool ODD>
__global__ void __launch_bounds__(kWarpBlock, EACH * ROUNDS >= 40 ? 5 : 6) k_distill_warp(DistillArgs a, int bulk_in, int bulk_out) {
  constexpr int tile_rows = ROUNDS > 0 ? ROUNDS * (32 / G) : kTileRows;
  // lanes per row for the teacher's entries, and entries of a lane where k <= 8
  constexpr int L = tile_rows >= 32 ? 1 : 32 / tile_rows, kFew = 8 / L;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ unsigned long long bars[kWarpBlock / 32][kWarpBuffers];
  const int C = (int)a.classes, k = a.t.k, warp = threadIdx.x >> 5, wl = threadIdx.x & 31;
  const int group = wl / G, lane = wl % G;
  const float c2 = a.inv_temp * kLog2e;
  uint8_t* own = smem + warp * warp_smem(tile_rows, C, sizeof(T), k);
  const size_t tile_bytes = warp_tile_bytes(tile_rows, C, sizeof(T));
  float2* ents = reinterpret_cast<float2*>(own + kWarpBuffers * tile_bytes);
  float2* fixes = ents + tile_rows * k;
  RowState* state = reinterpret_cast<RowState*>(fixes + tile_rows * k);
  if (wl == 0)
    for (int i = 0; i < kWarpBuffers; ++i) mbar_init(&bars[warp][i], 1);
  __syncwarp();
  const int64_t tiles = (a.n + tile_rows - 1) / tile_rows, step = (int64_t)gridDim.x * (blockDim.x >> 5);
  const T* logits = static_cast<const T*>(a.logits);
  const uint32_t whole_bytes = (uint32_t)(tile_rows * C * sizeof(T));
  auto fetch = [&](int64_t t, int buf) {  // whole tiles only
    if (wl == 0 && bulk_in && (t + 1) * tile_rows <= a.n) {
      mbar_arrive_expect_tx(&bars[warp][buf], whole_bytes);
      bulk_g2s(own + buf * tile_bytes, logits + t * tile_rows * C, whole_bytes, &bars[warp][buf]);
    }
  };
  double acc = 0.0;
  int buf = 0;
  unsigned phase = 0;
  int64_t t = blockIdx.x + (int64_t)gridDim.x * warp;
  if (t < tiles) fetch(t, 0);
  for (; t < tiles; t += step) {
    const int64_t r0 = t * tile_rows;
    const int rows = (int)min((int64_t)tile_rows, a.n - r0);
    const bool whole = rows == tile_rows;
    T* tile = reinterpret_cast<T*>(own + buf * tile_bytes);
    stage_entries<32>(a, ents, r0, rows, wl);
    __syncwarp();
    const int sub = wl % L;
    for (int rr = 0; rr < rows; rr += 32 / L) {
      const int r = rr + wl / L;
      if (L == 1 && r >= rows) break;
      const int held = L == 1 || r < rows ? k : 0;  // (every lane takes part in the exchanges)
      RowState st;
      st.weight = a.weight && r < rows ? a.weight[r0 + r] : 1.0f;
      st.factor = st.weight * a.grad_scale * (a.cot && r < rows ? a.cot[a.cot_per_row ? r0 + r : 0] : 1.0f);
      if (k <= 8) teacher_row<L, kFew>(ents + r * k, held, sub, a.inv_temp, st);
      else teacher_row<L, 0>(ents + r * k, held, sub, a.inv_temp, st);
      if (sub == 0 && r < rows) state[r] = st;
    }
    if (wl == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last tile has left
    __syncwarp();
    if (t + step < tiles) fetch(t + step, buf ^ 1);
    if (bulk_in && whole) {
      if (!__all_sync(~0u, mbar_wait(&bars[warp][buf], phase))) {
        // copies in flight must end before the block does (bounded)
        if (wl == 0) {
          atomicAdd(&g_distill_wait_failures, 1ull);
          mbar_wait(&bars[warp][buf], phase);
        }
        if (wl == 0 && t + step < tiles) mbar_wait(&bars[warp][buf ^ 1], buf ? phase ^ 1 : phase);
        break;
      }
    } else {
#pragma unroll 4
      for (int i = wl; i < rows * C; i += 32) tile[i] = logits[r0 * C + i];
    }
    __syncwarp();
    // the student's maximum and sum, by the rows' lanes
    F2 kept[ROUNDS > 0 ? ROUNDS : 1][EACH / 2];
    // the first class of a lane's pair i; -1 for the first pair of a row that starts inside it
    auto first_of = [&](int i, int lead) { return 2 * (lane + G * i) - lead; };
    auto lead_of = [&](int r) { return ODD ? r & 1 : 0; };
    auto read = [&](const T* s, int i, int lead, float none) {
      const int c = first_of(i, lead);
      if constexpr (ODD) {
        if (i > 0 && 2 * i + 1 < FULL) return load_pair(s + c);
        if (c >= C) return f2(none);
        float x, y;
        split(load_pair(s + c), x, y);
        return f2(i > 0 || c >= 0 ? x : none, 2 * i + 1 < FULL || c + 1 < C ? y : none);
      } else {
        return 2 * i + 1 < FULL || c < C ? load_pair(s + c) : f2(none);
      }
    };
    auto scaled = [&](F2 v, float m) {  // exp((v - m) / T)
      float x, y;
      split(mul(add(v, f2(-m)), f2(c2)), x, y);
      return f2(exp2_of(x), exp2_of(y));
    };
    auto exponentials = [&](int rr, F2(&v)[EACH / 2]) {
      const bool live = rr + group < rows;
      const int r = live ? rr + group : rows - 1;
      const T* s = tile + r * C;
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < EACH / 2; ++i) {
        v[i] = read(s, i, lead_of(r), -INFINITY);
        float x, y;
        split(v[i], x, y);
        m = fmaxf(m, fmaxf(x, y));
      }
      m = group_max<G>(m);
      F2 sums = f2(0.0f);
#pragma unroll
      for (int i = 0; i < EACH / 2; ++i) {
        v[i] = scaled(v[i], m);  // (0 where there is no class: m is finite, or the row is NaN)
        sums = add(sums, v[i]);
      }
      float x, y;
      split(sums, x, y);
      const float sum = group_sum<G>(x + y);
      if (lane == 0 && live) {
        state[r].m = m;
        state[r].inv = rcp_of(sum);
        state[r].lse = ln_of(sum);
      }
    };
    if constexpr (ROUNDS > 0) {
#pragma unroll
      for (int q = 0; q < ROUNDS; ++q) exponentials(q * (32 / G), kept[q]);
    } else {
      for (int rr = 0; rr < rows; rr += 32 / G) exponentials(rr, kept[0]);
    }
    __syncwarp();
    // the loss and the gradients of the teacher's classes
    for (int rr = 0; rr < rows; rr += 32 / L) {
      const int r = rr + wl / L;
      if (L == 1 && r >= rows) break;
      const int held = L == 1 || r < rows ? k : 0;
      const RowState st = state[L == 1 ? r : min(r, rows - 1)];
      float2* fix = a.grad ? fixes + r * k : nullptr;
      float cross = k <= 8 ? class_row<L, kFew>(tile + r * C, ents + r * k, fix, held, sub, a.inv_temp, st)
                           : class_row<L, 0>(tile + r * C, ents + r * k, fix, held, sub, a.inv_temp, st);
      cross = group_sum<L>(cross);
      if (sub == 0 && r < rows) {
        const float loss = st.any ? (st.term - cross + st.lse) * (a.temp * a.temp) * st.weight : 0.0f;
        if (a.row_loss) a.row_loss[r0 + r] = loss;
        acc += (double)loss;
      }
    }
    if (a.grad) {
      __syncwarp();
      auto gradients = [&](int rr, const F2(&v)[EACH / 2]) {
        const int r = rr + group;
        if (r >= rows) return;
        const RowState st = state[r];
        T* s = tile + r * C;
        const F2 f = f2(st.inv * st.factor);
        const int lead = lead_of(r);
#pragma unroll
        for (int i = 0; i < EACH / 2; ++i) {
          const int c = first_of(i, lead);
          const F2 g = st.any ? mul(ROUNDS > 0 ? v[i] : scaled(read(s, i, lead, 0.0f), st.m), f) : f2(0.0f);
          if constexpr (ODD) {
            const bool low = i > 0 || c >= 0, high = 2 * i + 1 < FULL || c + 1 < C;
            if (low && high) {
              store_pair(s + c, g);
            } else if (c < C) {  // the other half is a neighbouring row's
              float x, y;
              split(g, x, y);
              s[low ? c : c + 1] = from_f32<T>(low ? x : y);
            }
          } else {
            if (2 * i + 1 < FULL || c < C) store_pair(s + c, g);
          }
        }
      };
      if constexpr (ROUNDS > 0) {
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) gradients(q * (32 / G), kept[q]);
      } else {
        for (int rr = 0; rr < rows; rr += 32 / G) gradients(rr, kept[0]);
      }
      __syncwarp();
      const uint32_t per_k = 0xffffffffu / k + 1;
      for (int i = wl; i < rows * k; i += 32) {
        const float2 g = fixes[i];
        const int r = k == 1 ? i : (int)__umulhi((uint32_t)i, per_k);
        if (__float_as_int(g.x) >= 0) tile[r * C + __float_as_int(g.x)] = from_f32<T>(g.y);
      }
      T* dst = static_cast<T*>(a.grad) + r0 * C;
      if (bulk_out && whole) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (wl == 0) {
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_addr(tile)),
                       "r"(whole_bytes)
                       : "memory");
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      } else {
        __syncwarp();
#pragma unroll 4
        for (int i = wl; i < rows * C; i += 32) dst[i] = tile[i];
        // the buffer's next bulk copy comes after these ordinary writes and reads of it
        if (bulk_in) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
    }
    __syncwarp();
    buf ^= 1;
    if (buf == 0) phase ^= 1;
  }
  if (wl == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (a.partials) block_partial(acc, a.partials + blockIdx.x);
}

// A row in 16-byte units of memory, the first and last of which may reach outside it.
template <typename T>
struct RowUnits {
  static constexpr int kUnit = 16 / sizeof(T);
  union Unit {
    uint4 all;
    T e[kUnit];
  };
  const T* src;
  int classes, lead, units;  // lead: elements before the row in its first unit
  __device__ __forceinline__ RowUnits(const T* s, int c) : src(s), classes(c) {
    lead = (int)((reinterpret_cast<uintptr_t>(s) & 15) / sizeof(T));
    units = (lead + c + kUnit - 1) / kUnit;
  }
  __device__ __forceinline__ bool whole(int u) const {
    return u * kUnit >= lead && (u + 1) * kUnit <= lead + classes;
  }
  __device__ __forceinline__ Unit read(int u) const {  // elements outside the row are -inf
    Unit v;
    if (whole(u)) {
      v.all = __ldg(reinterpret_cast<const uint4*>(src - lead) + u);
    } else {
#pragma unroll
      for (int i = 0; i < kUnit; ++i) {
        const int c = u * kUnit + i - lead;
        v.e[i] = c >= 0 && c < classes ? src[c] : from_f32<T>(-INFINITY);
      }
    }
    return v;
  }
  // vector: g starts in a unit where the row does
  __device__ __forceinline__ void write(T* g, int u, const Unit& v, bool vector) const {
    if (vector && whole(u)) {
      reinterpret_cast<uint4*>(g - lead)[u] = v.all;
    } else {
#pragma unroll
      for (int i = 0; i < kUnit; ++i) {
        const int c = u * kUnit + i - lead;
        if (c >= 0 && c < classes) g[c] = v.e[i];
      }
    }
  }
};

// One warp per row, the row in its registers: UNITS 16-byte units a lane, straight
// from global memory, which is read once.  Tiles of 8 such rows in shared memory left
// four warps per SM: 200000 rows of 1000 in float16, 32 entries, loss and gradient
// 1008 us instead of 342; 153846 of 1300 in float32 2037 instead of 364.
constexpr int kLongBlock = 128;
template <typename T, int UNITS>
__global__ void __launch_bounds__(kLongBlock, UNITS == 4 ? 8 : UNITS == 8 && sizeof(T) == 4 ? 6 : 4) k_distill_long(DistillArgs a, int vector_out) {
  extern __shared__ float2 entries[];
  using Units = RowUnits<T>;
  const int C = (int)a.classes, k = a.t.k, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2 *ent = entries + warp * 2 * k, *fix = ent + k;
  const float c2 = a.inv_temp * kLog2e;
  double acc = 0.0;
  for (int64_t r = (int64_t)blockIdx.x * (kLongBlock / 32) + warp; r < a.n; r += (int64_t)gridDim.x * (kLongBlock / 32)) {
    const Units row(static_cast<const T*>(a.logits) + r * C, C);
    typename Units::Unit v[UNITS];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) v[i] = row.read(lane + 32 * i);
    stage_entries<32>(a, ent, r, 1, lane);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
#pragma unroll
      for (int e = 0; e < Units::kUnit; ++e) m = fmaxf(m, to_f32(v[i].e[e]));
    m = group_max<32>(m);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < UNITS; ++i)
#pragma unroll
      for (int e = 0; e < Units::kUnit; ++e) sum += exp2_of((to_f32(v[i].e[e]) - m) * c2);
    sum = group_sum<32>(sum);
    __syncwarp();
    const float w = a.weight ? a.weight[r] : 1.0f;
    const float f = w * a.grad_scale * (a.cot ? a.cot[a.cot_per_row ? r : 0] : 1.0f);
    auto logit = [&](int i) { return to_f32(row.src[i]); };
    float term;
    const bool any = teacher_terms(ent, k, lane, m, a.inv_temp, logit, term);
    const float inv = rcp_of(sum);
    if (lane == 0) {
      const float loss = any ? (term + ln_of(sum)) * (a.temp * a.temp) * w : 0.0f;
      if (a.row_loss) a.row_loss[r] = loss;
      acc += (double)loss;
    }
    __syncwarp();
    if (a.grad) {
      T* g = static_cast<T*>(a.grad) + r * C;
      bool repeats = k > 32;  // (looked for entry by entry there)
      if (!repeats) {
        const int idx = lane < k ? __float_as_int(ent[lane].x) : -1;
        const unsigned same = __match_any_sync(~0u, idx >= 0 ? idx : -1 - lane);
        repeats = __any_sync(~0u, (same & (same - 1)) != 0);
      }
      class_gradients(ent, fix, any ? k : 0, repeats, lane, m, c2, inv, f, logit);
      const float qf = inv * f;
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        const int u = lane + 32 * i;
#pragma unroll
        for (int e = 0; e < Units::kUnit; ++e)
          v[i].e[e] = from_f32<T>(any ? exp2_of((to_f32(v[i].e[e]) - m) * c2) * qf : 0.0f);
        if (u < row.units) row.write(g, u, v[i], vector_out);
      }
      __syncwarp();
      if (any)
        for (int e = lane; e < k; e += 32)
          if (__float_as_int(fix[e].x) >= 0) g[__float_as_int(fix[e].x)] = from_f32<T>(fix[e].y);
    }
    __syncwarp();
  }
  if (a.partials) block_partial(acc, a.partials + blockIdx.x);
}

// One block per row.  A row starts anywhere; it is moved in 16-byte units of
// memory, the first and last of which may reach outside it and are taken element
// by element.  Each of the three passes reads the row, the later ones from L2:
// four blocks of 256 threads per SM that read again took 61 us for 1031 rows of
// 32001, three of 512 that kept their row in shared memory 69 us.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) k_distill_row(DistillArgs a, int vector_out) {
  __shared__ float red[kRowThreads / 32], stats[2];
  __shared__ float2 ent[GS_TEACHER_MAX_K], fix[GS_TEACHER_MAX_K];
  using Units = RowUnits<T>;
  constexpr int kUnit = Units::kUnit;
  const int C = (int)a.classes, k = a.t.k, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float c2 = a.inv_temp * kLog2e;
  double acc = 0.0;
  for (int64_t r = blockIdx.x; r < a.n; r += gridDim.x) {
    const Units row(static_cast<const T*>(a.logits) + r * C, C);
    const int units = row.units;
    stage_entries<kRowThreads>(a, ent, r, 1, threadIdx.x);
    float m = -INFINITY;
#pragma unroll 4
    for (int u = threadIdx.x; u < units; u += kRowThreads) {
      const typename Units::Unit v = row.read(u);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) m = fmaxf(m, to_f32(v.e[i]));
    }
    m = group_max<32>(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = group_max<32>(lane < kRowThreads / 32 ? red[lane] : -INFINITY);
    __syncthreads();
    float sum = 0.0f;
#pragma unroll 2
    for (int u = threadIdx.x; u < units; u += kRowThreads) {
      const typename Units::Unit v = row.read(u);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) sum += exp2_of((to_f32(v.e[i]) - m) * c2);
    }
    sum = group_sum<32>(sum);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    const float w = a.weight ? a.weight[r] : 1.0f;
    const float f = w * a.grad_scale * (a.cot ? a.cot[a.cot_per_row ? r : 0] : 1.0f);
    if (warp == 0) {
      sum = group_sum<32>(lane < kRowThreads / 32 ? red[lane] : 0.0f);
      auto logit = [&](int i) { return to_f32(row.src[i]); };
      float term;
      const bool any = teacher_terms(ent, k, lane, m, a.inv_temp, logit, term);
      __syncwarp();
      const float inv = rcp_of(sum);
      if (a.grad) class_gradients(ent, fix, any ? k : 0, true, lane, m, c2, inv, f, logit);
      if (lane == 0) {
        const float loss = any ? (term + ln_of(sum)) * (a.temp * a.temp) * w : 0.0f;
        if (a.row_loss) a.row_loss[r] = loss;
        acc += (double)loss;
        stats[0] = inv;
        stats[1] = any ? 1.0f : 0.0f;
      }
    }
    __syncthreads();
    if (a.grad) {
      T* g = static_cast<T*>(a.grad) + r * C;
      const bool any = stats[1] > 0.0f;
      const float qf = stats[0] * f;
#pragma unroll 2
      for (int u = threadIdx.x; u < units; u += kRowThreads) {
        typename Units::Unit v;
        if (any) v = row.read(u);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v.e[i] = from_f32<T>(any ? exp2_of((to_f32(v.e[i]) - m) * c2) * qf : 0.0f);
        row.write(g, u, v, vector_out);
      }
      __syncthreads();
      if (any)
        for (int e = threadIdx.x; e < k; e += kRowThreads)
          if (__float_as_int(fix[e].x) >= 0) g[__float_as_int(fix[e].x)] = from_f32<T>(fix[e].y);
    }
    __syncthreads();
  }
  if (a.partials) block_partial(acc, a.partials + blockIdx.x);
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

template <typename T, int G, int EACH, int FULL, int ROUNDS>
static int launch_warps(const DistillArgs& a, cudaStream_t st, unsigned* blocks) {
  const int64_t rows = ROUNDS > 0 ? ROUNDS * (32 / G) : kTileRows;
  const size_t own = warp_smem((int)rows, a.classes, sizeof(T), a.t.k);
  int warps = kWarpBlock / 32;
  while (warps > 1 && own * warps > 100 * 1024) warps /= 2;
  const size_t smem = own * warps;
  auto* kernel = a.classes % 2 ? k_distill_warp<T, G, EACH, FULL, ROUNDS, true>
                               : k_distill_warp<T, G, EACH, FULL, ROUNDS, false>;
  // (always the same limit, what the static part leaves: threads may launch different sizes at once)
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024);
  if (e != cudaSuccess) return set_error(GS_ERR_CUDA, "k_distill_warp: %s", cudaGetErrorString(e));
  const int64_t resident = 148 * std::max<int64_t>(1, std::min<int64_t>(16, (227 * 1024) / (int64_t)(smem + 1024)));
  *blocks = (unsigned)std::min<int64_t>(ceil_div(ceil_div(a.n, rows), warps), resident);
  kernel<<<*blocks, warps * 32, smem, st>>>(a, aligned(a.logits, 16), aligned(a.grad, 16));
  return check_launch("k_distill_warp");
}

template <typename T>
static int launch_distill(const DistillArgs& a, cudaStream_t st, unsigned* blocks) {
  // Lanes of a row: enough that a lane's share fits in registers, few enough that
  // the reductions do not outweigh it.
  const int64_t c = a.classes;
  if (c <= 16) return launch_warps<T, 4, 4, 0, 6>(a, st, blocks);
  if (c <= 32) return launch_warps<T, 4, 8, 4, 4>(a, st, blocks);
  if (c <= 64) return launch_warps<T, 8, 8, 4, 4>(a, st, blocks);
  if (c <= 96) return launch_warps<T, 8, 12, 8, 2>(a, st, blocks);
  if (c <= 128) return launch_warps<T, 8, 16, 12, 2>(a, st, blocks);
  if (c <= 160) return launch_warps<T, 8, 20, 16, 2>(a, st, blocks);
  if (c <= 256) return launch_warps<T, 16, 16, 10, 4>(a, st, blocks);
  const bool alike = ((reinterpret_cast<uintptr_t>(a.logits) ^ reinterpret_cast<uintptr_t>(a.grad)) & 15) == 0;
  // Rows of little more than a kilobyte keep too few of a warp's loads in flight below: loss
  // and gradient of 666667 rows of 300 with 8 entries take 378 us here in float16, 990 there,
  // in float32 607 and 609; 400000 rows of 500 in float32 486 here, 382 there.  (With 32
  // entries, compared pair by pair here, 300 in float16 take 1336 and 1271, in float32 2038
  // and 804.)
  if (c <= 512 && c * sizeof(T) <= 1280) return launch_warps<T, 16, 32, 16, 0>(a, st, blocks);
  // Longer rows that fit in a warp's registers from wherever they start.
  constexpr int kUnit = 16 / sizeof(T), kPerUnit = 32 * kUnit;
  if (c <= 12 * kPerUnit - (kUnit - 1)) {
    *blocks = (unsigned)std::min<int64_t>(ceil_div(a.n, kLongBlock / 32), kDistillMaxBlocks);
    auto* kernel = c <= 4 * kPerUnit - (kUnit - 1)   ? k_distill_long<T, 4>
                   : c <= 8 * kPerUnit - (kUnit - 1) ? k_distill_long<T, 8>
                                                     : k_distill_long<T, 12>;
    kernel<<<*blocks, kLongBlock, kLongBlock / 32 * 2 * sizeof(float2) * a.t.k, st>>>(a, alike);
    return check_launch("k_distill_long");
  }
  *blocks = (unsigned)std::min<int64_t>(a.n, kDistillMaxBlocks);
  k_distill_row<T><<<*blocks, kRowThreads, 0, st>>>(a, alike);
  return check_launch("k_distill_row");
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
  if (n < 0 || classes < 1 || classes > GS_DISTILL_MAX_CLASSES)
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: logits must be (n >= 0, 1 <= classes <= %d)",
                     GS_DISTILL_MAX_CLASSES);
  if (!teacher) return set_error(GS_ERR_INVALID_ARG, "gs_distill: teacher is NULL");
  const bool cached = teacher->bits != 0;
  const int max_k = cached ? GS_CACHE_MAX_K : GS_TEACHER_MAX_K;
  if (teacher->k < 1 || teacher->k > max_k)
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: k must be in [1, %d] (got %d)", max_k, teacher->k);
  // The loss has the factor T^2, the exponents 1 / T: both must be normal float32 numbers.
  if (!(temperature >= GS_DISTILL_MIN_TEMPERATURE && temperature <= GS_DISTILL_MAX_TEMPERATURE))
    return set_error(GS_ERR_INVALID_ARG, "gs_distill: temperature must be in [%g, %g]", GS_DISTILL_MIN_TEMPERATURE,
                     GS_DISTILL_MAX_TEMPERATURE);
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
  unsigned grid = 0;
  if (n > 0) {
    const int e = dtype == GS_F32   ? launch_distill<float>(a, st, &grid)
                  : dtype == GS_F16 ? launch_distill<__half>(a, st, &grid)
                                    : launch_distill<__nv_bfloat16>(a, st, &grid);
    if (e) return e;
  }
  if (loss) {
    k_distill_finish<<<1, 256, 0, st>>>(a.partials, (int)grid, scale, loss);
    return check_launch("k_distill_finish");
  }
  return GS_OK;
}

}  // extern "C"
