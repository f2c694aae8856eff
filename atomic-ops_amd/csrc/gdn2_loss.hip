// Cross-entropy of rows of logits and its gradient, on gfx950:
//   loss = lse - (1 - e) x[t] - e mean(x) + z lse^2,  lse = m + log sum exp(x - m), m = max x
//   dx_j = s (p_j (1 + 2 z lse) - (1 - e) [j = t] - e / V),  p_j = exp(x_j - m) / sum
// A row's maximum and sum come from one pass (each thread rescales its sum where its maximum grows); the gradient's p
// is formed from them, not from lse, whose rounding (2^-24 |lse|) would be an error of every p.  Statistics are
// float32, the sum over the rows 64 bits, in a fixed order.  Bound by memory, two exponentials an element close behind: 8192 x
// 131072 bfloat16 971 us, 4.4 TB/s of reads and writes (a copy 5.2); 16384 x 256 float32 11 us, 2.9 TB/s.
#include "gdn2_kernels.hpp"

namespace gdn2 {

constexpr float LOG2E = 1.44269504088896341f;
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

template <int DT>
struct LossVec {                       // 16 bytes of logits
  static constexpr int E = DT == LIN_F32 ? 4 : 8;
  using T = std::conditional_t<DT == LIN_F32, float, std::conditional_t<DT == LIN_BF16, uint16_t, _Float16>>;
  static __device__ __forceinline__ float one(const T* p) {
    if constexpr (DT == LIN_BF16) return bf16_val(*p);
    else return (float)*p;
  }
  static __device__ __forceinline__ void put(T* p, float v) {
    if constexpr (DT == LIN_BF16) *p = (uint16_t)bf16_bits(v);
    else *p = (T)v;
  }
  static __device__ __forceinline__ void load(const T* p, float* x) { widen(*reinterpret_cast<const uint4*>(p), x); }
  static __device__ __forceinline__ void widen(const uint4& u, float* x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == LIN_F32) x[i] = __uint_as_float(w[i]);
      else if constexpr (DT == LIN_BF16) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const h2v h = __builtin_bit_cast(h2v, w[i]);
        x[2 * i] = (float)h[0];
        x[2 * i + 1] = (float)h[1];
      }
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == LIN_F32) w[i] = __float_as_uint(x[i]);
      else if constexpr (DT == LIN_BF16) w[i] = bf16_pack(x[2 * i], x[2 * i + 1]);
      else {
        const h2v h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
        w[i] = __builtin_bit_cast(uint32_t, h);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// max, sum of exp(x - max), sum of x / V (a sum of x could overflow) of a part of a row
struct LossStat {
  float m, s, x;
};
__device__ __forceinline__ float loss_base(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ LossStat loss_join(const LossStat& a, const LossStat& b) {
  const float m = fmaxf(a.m, b.m), at = loss_base(m);
  return {m, a.s * __builtin_amdgcn_exp2f((a.m - at) * LOG2E) + b.s * __builtin_amdgcn_exp2f((b.m - at) * LOG2E), a.x + b.x};
}
template <int E>
__device__ __forceinline__ void loss_take(LossStat& t, const float* x, float per) {
  float m = x[0];
#pragma unroll
  for (int e = 1; e < E; ++e) m = fmaxf(m, x[e]);
  if (m > t.m) {
    t.s *= __builtin_amdgcn_exp2f((t.m - loss_base(m)) * LOG2E);
    t.m = m;
  }
  const float at = loss_base(t.m);
#pragma unroll
  for (int e = 0; e < E; ++e) t.s += __builtin_amdgcn_exp2f((x[e] - at) * LOG2E);
  if (per != 0.f)
#pragma unroll
    for (int e = 0; e < E; ++e) t.x = fmaf(x[e], per, t.x);
}

__device__ __forceinline__ int64_t loss_target(const LossArgs& a, int row) {
  return a.target_bytes == 8 ? static_cast<const int64_t*>(a.targets)[row] : static_cast<const int32_t*>(a.targets)[row];
}

// What a row's gradient is formed with
struct LossGrad {
  float base, up, off, hit;
  __device__ __forceinline__ float operator()(float v) const { return fmaf(up, __builtin_amdgcn_exp2f((v - base) * LOG2E), -off); }
};
// Its loss (one thread's), and what its gradient takes
template <int DT>
__device__ __forceinline__ LossGrad loss_finish(const LossArgs& a, int row, const typename LossVec<DT>::T* x, int t, const LossStat& st, bool first) {
  const float log_s = logf(st.s), lse = st.m + log_s;
  if (first && a.row_loss) {
    // (differences with the maximum first: lse itself loses log sum beside a row of the type's lowest values)
    float loss = log_s + (1.f - a.smoothing) * (st.m - LossVec<DT>::one(x + t));
    if (a.smoothing != 0.f) loss += a.smoothing * (st.m - st.x);
    if (a.z_loss != 0.f) loss += a.z_loss * lse * lse;
    a.row_loss[row] = loss;
  }
  float s = a.reduction == 2 && a.dlogits ? *a.scale : 1.f;
  if (a.upstream) s *= a.upstream[a.upstream_ld ? row : 0];
  return {loss_base(st.m), s * (1.f + 2.f * a.z_loss * lse) / st.s, s * a.smoothing / (float)a.V, s * (1.f - a.smoothing)};
}
// A row without statistics: ignored, or with a target outside; false: neither
template <int DT>
__device__ __forceinline__ bool loss_skipped(const LossArgs& a, int row, int64_t t, typename LossVec<DT>::T* d, int thread, int threads) {
  const bool ignored = t == a.ignore;
  if (!ignored && t >= 0 && t < a.V) return false;
  const float v = ignored ? 0.f : NAN;
  if (thread == 0 && a.row_loss) a.row_loss[row] = v;
  if (d) {
    using V = LossVec<DT>;
    const int head = min(a.V, (int)((16 - (reinterpret_cast<uintptr_t>(d) & 15)) % 16 / sizeof(typename V::T))), body = (a.V - head) / V::E * V::E;
    float x[V::E];
#pragma unroll
    for (int e = 0; e < V::E; ++e) x[e] = v;
    for (int j = head + V::E * thread; j < head + body; j += V::E * threads) V::store(d + j, x);
    for (int j = thread; j < a.V - body; j += threads) V::put(d + (j < head ? j : body + j), v);
  }
  return true;
}

// A workgroup of T threads a row.  NV vectors of 16 bytes a thread hold the row in registers between its statistics and its
// gradient, so that it is read once; NV 0: longer rows, read twice (the second time mostly from the last cache level).  The exponentials cost as much as the memory, so that several workgroups a CU, one loading while
// another computes, are worth more than a longer row in registers: 8192 rows of 32000 in bfloat16, 1024 threads with 4 vectors
// 294 us, 512 with 8 218 (4.8 TB/s); of 65536, 1024 with 8 577, 512 with 16 455; read twice 526 and 487.
template <int DT, int T, int NV>
__global__ __launch_bounds__(T) void loss_rows_kernel(LossArgs a) {
  using V = LossVec<DT>;
  using E_ = typename V::T;
  constexpr int E = V::E, W = T / WAVE;
  __shared__ LossStat part[W];
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const E_* x = static_cast<const E_*>(a.logits) + (size_t)row * a.ld;
    E_* d = a.dlogits ? static_cast<E_*>(a.dlogits) + (size_t)row * a.V : nullptr;
    const int64_t t = loss_target(a, row);
    if (loss_skipped<DT>(a, row, t, d, threadIdx.x, T)) continue;
    const float per = a.smoothing != 0.f ? 1.f / (float)a.V : 0.f;
    LossStat st{-INFINITY, 0.f, 0.f};
    // elements before the first whole 16 bytes, whole ones, the rest
    const int head = min(a.V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(E_))), body = (a.V - head) / E * E;
    const int odd = a.V - body, own = head + E * threadIdx.x, at = (int)threadIdx.x < head ? threadIdx.x : body + threadIdx.x;
    uint4 raw[NV ? NV : 1];
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (own + i * (E * T) < head + body) raw[i] = *reinterpret_cast<const uint4*>(x + own + i * (E * T));
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (own + i * (E * T) < head + body) {
          float v[E];
          V::widen(raw[i], v);
          loss_take<E>(st, v, per);
        }
    } else {
#pragma unroll 2
      for (int j = own; j < head + body; j += E * T) {
        float v[E];
        V::load(x + j, v);
        loss_take<E>(st, v, per);
      }
    }
    if ((int)threadIdx.x < odd) {
      const float v = V::one(x + at);
      loss_take<1>(st, &v, per);
    }
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) st = loss_join(st, {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.x, o)});
    __syncthreads();                     // (the row before is done with part)
    if (lane_id() == 0) part[wave_id()] = st;
    __syncthreads();
    st = part[lane_id() % W];            // (every wave joins them in the same order)
#pragma unroll
    for (int o = 1; o < W; o *= 2) st = loss_join(st, {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.x, o)});
    const LossGrad grad = loss_finish<DT>(a, row, x, (int)t, st, threadIdx.x == 0);
    if (!d) continue;
    const bool same = (reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(d) & 15);
    auto put = [&](int j, float* v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = grad(v[e]);
      if (same) V::store(d + j, v);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) V::put(d + j + e, v[e]);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (own + i * (E * T) < head + body) {
          float v[E];
          V::widen(raw[i], v);
          put(own + i * (E * T), v);
        }
    } else {
#pragma unroll 2
      for (int j = own; j < head + body; j += E * T) {
        float v[E];
        V::load(x + j, v);
        put(j, v);
      }
    }
    if ((int)threadIdx.x < odd) V::put(d + at, grad(V::one(x + at)));
    // the target's own: over what the same thread has written there
    const int tj = (int)t, holder = tj < head ? tj : tj >= head + body ? tj - body : (tj - head) / E % T;
    if ((int)threadIdx.x == holder) V::put(d + tj, grad(V::one(x + tj)) - grad.hit);
  }
}

// A wave a row, for rows of up to 64 NV vectors whose starts (and their gradients') are whole 16 bytes
template <int DT, int NV>
__global__ __launch_bounds__(256) void loss_waves_kernel(LossArgs a) {
  using V = LossVec<DT>;
  using E_ = typename V::T;
  constexpr int E = V::E;
  const int row = blockIdx.x * 4 + wave_id(), l = lane_id();
  if (row >= a.rows) return;
  const E_* x = static_cast<const E_*>(a.logits) + (size_t)row * a.ld;
  E_* d = a.dlogits ? static_cast<E_*>(a.dlogits) + (size_t)row * a.V : nullptr;
  const int64_t t = loss_target(a, row);
  float v[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (E * (l + WAVE * i) < a.V) V::load(x + E * (l + WAVE * i), v[i]);
  if (loss_skipped<DT>(a, row, t, d, l, WAVE)) return;
  LossStat st{-INFINITY, 0.f, 0.f};
  const float per = a.smoothing != 0.f ? 1.f / (float)a.V : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (E * (l + WAVE * i) < a.V) loss_take<E>(st, v[i], per);
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) st = loss_join(st, {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.x, o)});
  const LossGrad grad = loss_finish<DT>(a, row, x, (int)t, st, l == 0);
  if (!d) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = E * (l + WAVE * i);
    if (j >= a.V) continue;
#pragma unroll
    for (int e = 0; e < E; ++e) v[i][e] = grad(v[i][e]);
    V::store(d + j, v[i]);
  }
  // the target's own: over what the same lane has written there
  if (l == (int)t / E % WAVE) V::put(d + t, grad(V::one(x + t)) - grad.hit);
}

// One workgroup: 1 / the rows that count (at least one)
__global__ __launch_bounds__(1024) void loss_count_kernel(LossArgs a) {
  __shared__ int part[16];
  int n = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.rows; i += 1024) n += loss_target(a, i) != a.ignore;      // (the loads go together)
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) n += __shfl_xor(n, o);
  if (lane_id() == 0) part[wave_id()] = n;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) n += part[w];
  *a.scale = 1.f / (float)max(n, 1);
}

// One workgroup: the rows' sum or mean
__global__ __launch_bounds__(1024) void loss_sum_kernel(LossArgs a) {
  __shared__ double part[16];
  __shared__ int count[16];
  double s = 0.0;
  int n = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.rows; i += 1024) {
    s += (double)a.row_loss[i];
    n += loss_target(a, i) != a.ignore;
  }
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) {
    s += __shfl_xor(s, o);
    n += __shfl_xor(n, o);
  }
  if (lane_id() == 0) {
    part[wave_id()] = s;
    count[wave_id()] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) {
    s += part[w];
    n += count[w];
  }
  *a.loss = (float)(a.reduction == 2 ? s / (double)max(n, 1) : s);
}

// (zeros stay zeros: a row without a gradient has none, whatever its factor, an infinity or NaN of a padded row among them)
template <int DT>
__global__ __launch_bounds__(256) void scale_rows_kernel(typename LossVec<DT>::T* x, int rows, int V, const float* factor, int ld) {
  using L = LossVec<DT>;
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const float f = factor[ld ? row : 0];
    if (f == 1.f) {
      if (!ld) return;
      continue;
    }
    auto* p = x + (size_t)row * V;
    for (int j = threadIdx.x; j < V; j += 256) {
      const float v = L::one(p + j);
      L::put(p + j, v == 0.f ? v : v * f);
    }
  }
}

size_t loss_workspace_bytes(int rows) { return 256 + (size_t)rows * 4; }

// Which kernel takes the rows: a wave each up to 256 vectors of 16 bytes where they are aligned; else a workgroup each, as
// small as holds the row, or of 1024 threads where there are fewer rows than CUs; beyond 8192 vectors rows are read twice.
template <int DT>
static void loss_go(const LossArgs& a, hipStream_t s) {
  constexpr int E = LossVec<DT>::E;
  const int vecs = (a.V + E - 1) / E;
  auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const bool aligned = (low(a.logits) | low(a.dlogits)) % 16 == 0 && a.ld % E == 0 && a.V % E == 0;
  // (a grid has fewer than 2^32 threads, 64 of them a row: what goes beyond would be left out without an error)
  auto wave = [&](auto k) {
    constexpr int MOST = 1 << 25;
    for (int r = 0; r < a.rows; r += MOST) {
      LossArgs b = a;
      b.rows = a.rows - r < MOST ? a.rows - r : MOST;
      b.logits = static_cast<const typename LossVec<DT>::T*>(a.logits) + (size_t)r * a.ld;
      b.targets = static_cast<const char*>(a.targets) + (size_t)r * a.target_bytes;
      if (a.upstream && a.upstream_ld) b.upstream = a.upstream + r;
      if (a.row_loss) b.row_loss = a.row_loss + r;
      if (a.dlogits) b.dlogits = static_cast<typename LossVec<DT>::T*>(a.dlogits) + (size_t)r * a.V;
      hipLaunchKernelGGL(k, dim3((b.rows + 3) / 4), dim3(256), 0, s, b);
    }
  };
  auto rows = [&](auto k, int threads) { hipLaunchKernelGGL(k, dim3(a.rows < 65536 ? a.rows : 65536), dim3(threads), 0, s, a); };
  if (aligned && vecs <= 256) {
    if (vecs <= 64) wave(loss_waves_kernel<DT, 1>);
    else if (vecs <= 128) wave(loss_waves_kernel<DT, 2>);
    else wave(loss_waves_kernel<DT, 4>);
  } else if (vecs > 8192) {
    rows(loss_rows_kernel<DT, 1024, 0>, 1024);
  } else if (a.rows < cu_count()) {
    if (vecs <= 1024) rows(loss_rows_kernel<DT, 1024, 1>, 1024);
    else if (vecs <= 2048) rows(loss_rows_kernel<DT, 1024, 2>, 1024);
    else if (vecs <= 4096) rows(loss_rows_kernel<DT, 1024, 4>, 1024);
    else rows(loss_rows_kernel<DT, 1024, 8>, 1024);
  } else if (vecs <= 256) {
    rows(loss_rows_kernel<DT, 256, 1>, 256);
  } else if (vecs <= 512) {
    rows(loss_rows_kernel<DT, 256, 2>, 256);
  } else if (vecs <= 1024) {
    rows(loss_rows_kernel<DT, 256, 4>, 256);
  } else if (vecs <= 2048) {
    rows(loss_rows_kernel<DT, 512, 4>, 512);
  } else if (vecs <= 4096) {
    rows(loss_rows_kernel<DT, 512, 8>, 512);
  } else {
    rows(loss_rows_kernel<DT, 512, 16>, 512);
  }
}

hipError_t launch_cross_entropy(const LossArgs& a, hipStream_t s) {
  if (a.reduction == 2 && a.dlogits) hipLaunchKernelGGL(loss_count_kernel, dim3(1), dim3(1024), 0, s, a);
  if (a.dtype == LIN_F32) loss_go<LIN_F32>(a, s);
  else if (a.dtype == LIN_BF16) loss_go<LIN_BF16>(a, s);
  else loss_go<LIN_F16>(a, s);
  if (a.reduction && a.loss) hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_scale_rows(void* x, int dtype, int rows, int V, const float* factor, int factor_ld, hipStream_t s) {
  const dim3 grid(rows < 2048 ? rows : 2048);
  if (dtype == LIN_F32) hipLaunchKernelGGL(scale_rows_kernel<LIN_F32>, grid, dim3(256), 0, s, static_cast<float*>(x), rows, V, factor, factor_ld);
  else if (dtype == LIN_BF16)
    hipLaunchKernelGGL(scale_rows_kernel<LIN_BF16>, grid, dim3(256), 0, s, static_cast<uint16_t*>(x), rows, V, factor, factor_ld);
  else hipLaunchKernelGGL(scale_rows_kernel<LIN_F16>, grid, dim3(256), 0, s, static_cast<_Float16*>(x), rows, V, factor, factor_ld);
  return hipGetLastError();
}

}  // namespace gdn2
