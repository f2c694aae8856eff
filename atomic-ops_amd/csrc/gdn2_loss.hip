// Cross-entropy of rows of logits and its gradient, on gfx950:
//   loss = lse - (1 - e) x[t] - e mean(x) + z lse^2,  lse = m + log sum exp(x - m), m = max x
//   dx_j = s (p_j (1 + 2 z lse) - (1 - e) [j = t] - e / V),  p_j = exp(x_j - m) / sum
// A row's maximum and sum come from one pass (each thread rescales its sum where its maximum grows); the gradient's p
// is formed from them, not from lse, whose rounding (2^-24 |lse|) would be an error of every p.  Statistics are
// float32, the sum over the rows 64 bits, in a fixed order.  Bound by memory.
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
  static __device__ __forceinline__ void load(const T* p, float* x) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
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
  for (int e = 0; e < E; ++e) {
    t.s += __builtin_amdgcn_exp2f((x[e] - at) * LOG2E);
    t.x = fmaf(x[e], per, t.x);
  }
}

__device__ __forceinline__ int64_t loss_target(const LossArgs& a, int row) {
  return a.target_bytes == 8 ? static_cast<const int64_t*>(a.targets)[row] : static_cast<const int32_t*>(a.targets)[row];
}

// A workgroup a row: its statistics, its loss, its gradient.
constexpr int LOSS_THREADS = 256;
template <int DT>
__global__ __launch_bounds__(LOSS_THREADS) void loss_rows_kernel(LossArgs a) {
  using V = LossVec<DT>;
  using T = typename V::T;
  constexpr int E = V::E, W = LOSS_THREADS / WAVE;
  __shared__ LossStat part[W];
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.logits) + (size_t)row * a.ld;
    T* d = a.dlogits ? static_cast<T*>(a.dlogits) + (size_t)row * a.V : nullptr;
    const int64_t t = loss_target(a, row);
    const bool ignored = t == a.ignore, outside = !ignored && (t < 0 || t >= a.V);
    if (ignored || outside) {
      const float v = ignored ? 0.f : NAN;
      if (threadIdx.x == 0 && a.row_loss) a.row_loss[row] = v;
      if (d)
        for (int j = threadIdx.x; j < a.V; j += LOSS_THREADS) V::put(d + j, v);
      continue;
    }
    LossStat st{-INFINITY, 0.f, 0.f};
    const float per = 1.f / (float)a.V;
    // elements before the first whole 16 bytes, whole ones, the rest
    const int head = min(a.V, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T))), body = (a.V - head) / E * E;
    for (int j = head + E * threadIdx.x; j < head + body; j += E * LOSS_THREADS) {
      float v[E];
      V::load(x + j, v);
      loss_take<E>(st, v, per);
    }
    const int odd = a.V - body;
    if ((int)threadIdx.x < odd) {
      const float v = V::one(x + ((int)threadIdx.x < head ? threadIdx.x : body + threadIdx.x));
      loss_take<1>(st, &v, per);
    }
#pragma unroll
    for (int o = 1; o < WAVE; o *= 2) st = loss_join(st, {__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.x, o)});
    __syncthreads();                     // (the row before is done with part)
    if (lane_id() == 0) part[wave_id()] = st;
    __syncthreads();
    st = part[0];
#pragma unroll
    for (int w = 1; w < W; ++w) st = loss_join(st, part[w]);
    const float base = loss_base(st.m), log_s = logf(st.s), lse = st.m + log_s;
    if (threadIdx.x == 0 && a.row_loss) {
      // (differences with the maximum first: lse itself loses log sum beside a row of the type's lowest values)
      float loss = log_s + (1.f - a.smoothing) * (st.m - V::one(x + t));
      if (a.smoothing != 0.f) loss += a.smoothing * (st.m - st.x);
      if (a.z_loss != 0.f) loss += a.z_loss * lse * lse;
      a.row_loss[row] = loss;
    }
    if (!d) continue;
    float s = a.reduction == 2 ? *a.scale : 1.f;
    if (a.upstream) s *= a.upstream[a.upstream_ld ? row : 0];
    const float up = s * (1.f + 2.f * a.z_loss * lse) / st.s, off = s * a.smoothing / (float)a.V, hit = s * (1.f - a.smoothing);
    auto grad = [&](float v, int j) __attribute__((always_inline)) {
      const float p = up * __builtin_amdgcn_exp2f((v - base) * LOG2E) - off;
      return j == (int)t ? p - hit : p;
    };
    const bool same = (reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(d) & 15);
    for (int j = head + E * threadIdx.x; j < head + body; j += E * LOSS_THREADS) {
      float v[E];
      V::load(x + j, v);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = grad(v[e], j + e);
      if (same) V::store(d + j, v);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) V::put(d + j + e, v[e]);
    }
    if ((int)threadIdx.x < odd) {
      const int j = (int)threadIdx.x < head ? threadIdx.x : body + threadIdx.x;
      V::put(d + j, grad(V::one(x + j), j));
    }
  }
}

// One workgroup: 1 / the rows that count (at least one)
__global__ __launch_bounds__(1024) void loss_count_kernel(LossArgs a) {
  __shared__ int part[16];
  int n = 0;
  for (int i = threadIdx.x; i < a.rows; i += 1024) n += loss_target(a, i) != a.ignore;
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
    for (int j = threadIdx.x; j < V; j += 256) L::put(p + j, L::one(p + j) * f);
  }
}

size_t loss_workspace_bytes(int rows) { return 256 + (size_t)rows * 4; }

hipError_t launch_cross_entropy(const LossArgs& a, hipStream_t s) {
  if (a.reduction == 2 && a.dlogits) hipLaunchKernelGGL(loss_count_kernel, dim3(1), dim3(1024), 0, s, a);
  const dim3 grid(a.rows < 65536 ? a.rows : 65536);
  if (a.dtype == LIN_F32) hipLaunchKernelGGL(loss_rows_kernel<LIN_F32>, grid, dim3(LOSS_THREADS), 0, s, a);
  else if (a.dtype == LIN_BF16) hipLaunchKernelGGL(loss_rows_kernel<LIN_BF16>, grid, dim3(LOSS_THREADS), 0, s, a);
  else hipLaunchKernelGGL(loss_rows_kernel<LIN_F16>, grid, dim3(LOSS_THREADS), 0, s, a);
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
