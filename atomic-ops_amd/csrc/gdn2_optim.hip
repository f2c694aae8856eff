// AdamW over many tensors, on gfx950: with c = max_norm / max(norm, max_norm) of all gradients,
//   g' = c g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - m / (sqrt(v) r + eps) s,   r = 1 / sqrt(1 - b2^t), s = lr / (1 - b1^t).
// One pass over the gradients for the norm, one workgroup that forms c and every tensor's r, s and step, one pass that
// updates: bound by memory (186 tensors of 35 M float32 elements: the update 172 us, 5.7 TB/s, the norm 44; 200 M bfloat16 with
// masters 1132, 5.3 TB/s, and 116).  The tensors come in the kernels' argument blocks (so a captured graph holds them), up
// to 200 to a launch.
//
// The norm is summed in 64 bits, so that c does not turn on the order of the sum (but for one rounding in 10^8).
// Products and sums of the update are rounded one by one (no fma): what an 8-bit state becomes turns on a value's last
// bit, and an update is the same numbers however a compiler would fuse it.
//
// A 16-bit parameter is kept as a float32 master as well; where the parameter is no longer the master's rounding (a checkpoint
// was loaded into it), the parameter counts.
//
// States of 8 bits: blocks of 256 elements share a float32 scale.  m = c |c| s with c in -127 .. 127; v = (c^2 s)^2 with c
// in 0 .. 255: squares put the codes closer together towards 0, so that elements a hundred times below their block's
// largest keep codes of their own (m 12.7, sqrt(v) 25.5).  A value between two codes takes the upper one with the
// probability that keeps its mean: rounded to the nearest, v would never decay, since a step takes 0.1 % of it, less than
// half of any code's distance.  (v above 0 takes code 1 at least: with 0 the update would be m / eps.)  The step itself
// uses m and v as formed, in 32 bits.  Bound by what it computes: 4.2 M elements 27 us, 2.5 TB/s (25 with codes off by one beside
// a border, from the hardware's quotient and root alone; 30 with correctly rounded ones formed where they are near).
#include "gdn2_optim.hpp"

namespace gdn2 {

constexpr int OPT_CHUNK = 8192;            // elements of a workgroup of the update
constexpr int OPT_CHUNK8 = 2048;           // ... with states of 8 bits (bound by what it computes: many small ones)
constexpr int OPT_NORM_CHUNK = 16384;      // ... of the norm
constexpr int OPT_BLOCK = 256;             // elements of a scale
constexpr int64_t OPT_GRID = (1 << 24) - 1;            // workgroups of 256 threads in a grid, which has fewer than 2^32
constexpr int OPT_TENSORS = 200, OPT_GRADS = 200, OPT_STEPS = 200;

// What a tensor's update needs beside it; written by opt_begin_kernel
struct OptHyper {
  float b1, nb1, b2, nb2, eps, keep, size, root;
  uint32_t hash, pad[3];
};
struct OptGrads {
  const void* g[OPT_GRADS];
  int64_t n[OPT_GRADS];
  int start[OPT_GRADS + 1];                // first workgroup
  int tensors;
};
struct OptSteps {
  struct {
    float* step;
    double lr, b1, b2, eps, wd;
    uint32_t ordinal, pad;
  } t[OPT_STEPS];
  int tensors;
};
struct OptTensors {
  struct {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs, *master;
    int64_t n;
    int start;                             // first workgroup
    int16_t vec, hyper;                    // whether every pointer takes whole vectors; the tensor's place in hyper
  } t[OPT_TENSORS];
  int tensors;
};
static_assert(sizeof(OptGrads) < 16000 && sizeof(OptSteps) < 16000 && sizeof(OptTensors) < 16000, "argument blocks");

template <int DT>
struct OptType {
  using T = std::conditional_t<DT == LIN_F32, float, std::conditional_t<DT == LIN_BF16, uint16_t, _Float16>>;
  static __device__ __forceinline__ float get(const T* p) {
    if constexpr (DT == LIN_BF16) return bf16_val(*p);
    else return (float)*p;
  }
  static __device__ __forceinline__ void put(T* p, float v) {
    if constexpr (DT == LIN_BF16) *p = (uint16_t)bf16_bits(v);
    else *p = (T)v;
  }
  // The master of a 16-bit parameter: w, unless something else than an update has been written into p since
  static __device__ __forceinline__ float master(float w, T p) {
    T r;
    put(&r, w);
    return __builtin_bit_cast(uint16_t, r) == __builtin_bit_cast(uint16_t, p) ? w : get(&p);
  }
  static __device__ __forceinline__ void master4(const float* w, const T* p, float* x) {
    const float4 v = *reinterpret_cast<const float4*>(w);
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
    x[0] = master(v.x, e[0]); x[1] = master(v.y, e[1]); x[2] = master(v.z, e[2]); x[3] = master(v.w, e[3]);
  }
  static __device__ __forceinline__ void get4(const T* p, float* x) {
    if constexpr (DT == LIN_F32) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = get(e + i);
    }
  }
  static __device__ __forceinline__ void put4(T* p, const float* x) {
    if constexpr (DT == LIN_F32) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else {
      uint2 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) put(e + i, x[i]);
      *reinterpret_cast<uint2*>(p) = u;
    }
  }
};

// The tensor of a workgroup: the last whose first one is not above it
template <class F>
__device__ __forceinline__ int opt_find(int tensors, int b, F start) {
  int lo = 0, hi = tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (start(mid) <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A workgroup's part of the sum of squares (squares of 32-bit numbers are exact in 64)
template <int DT>
__global__ __launch_bounds__(256) void opt_norm_kernel(OptGrads a, double* part) {
  using O = OptType<DT>;
  using T = typename O::T;
  __shared__ double sums[4];
  const int b = blockIdx.x, i = opt_find(a.tensors, b, [&](int k) { return a.start[k]; });
  const int64_t at = (int64_t)(b - a.start[i]) * OPT_NORM_CHUNK, n = min((int64_t)OPT_NORM_CHUNK, a.n[i] - at);
  const T* g = static_cast<const T*>(a.g[i]) + at;
  double s = 0.0;
  constexpr int E = 16 / sizeof(T);
  const int whole = (reinterpret_cast<uintptr_t>(g) & 15) ? 0 : (int)(n / E);
#pragma unroll 8
  for (int j = threadIdx.x; j < whole; j += 256) {
    const uint4 u = *reinterpret_cast<const uint4*>(g + E * j);
    const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double v = O::get(x + e);
      s = fma(v, v, s);
    }
  }
  for (int j = E * whole + threadIdx.x; j < n; j += 256) {
    const double x = O::get(g + j);
    s = fma(x, x, s);
  }
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) s += __shfl_xor(s, o);
  if (lane_id() == 0) sums[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[b] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// One workgroup: c (where parts > 0), and the tensors' steps and factors
__global__ __launch_bounds__(1024) void opt_begin_kernel(OptSteps a, const double* part, int parts, double max_norm, float* coef,
                                                         float* norm, OptHyper* hyper) {
  if ((int)threadIdx.x < a.tensors) {
    const auto& t = a.t[threadIdx.x];
    const float step = *t.step + 1.f;
    *t.step = step;
    OptHyper h{};
    h.b1 = (float)t.b1;
    h.nb1 = (float)(1.0 - t.b1);
    h.b2 = (float)t.b2;
    h.nb2 = (float)(1.0 - t.b2);
    h.eps = (float)t.eps;
    h.keep = (float)(1.0 - t.lr * t.wd);
    h.size = (float)(t.lr / (1.0 - pow(t.b1, (double)step)));
    h.root = (float)(1.0 / sqrt(1.0 - pow(t.b2, (double)step)));
    h.hash = t.ordinal * 0x7F4A7C15u + (uint32_t)step * 0x6C62272Fu;
    hyper[threadIdx.x] = h;
  }
  if (parts == 0) return;
  __shared__ double sums[16];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 1024) s += part[i];
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) s += __shfl_xor(s, o);
  if (lane_id() == 0) sums[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) s += sums[w];
  s = sqrt(s);
  if (norm) *norm = (float)s;
  // (a norm that is not a number is not below max_norm; an infinite max_norm scales nothing, whatever the norm)
  *coef = max_norm > 0.0 && max_norm < INFINITY && !(s < max_norm) ? (float)(max_norm / s) : 1.f;
}

struct OptState {
  float m, v;
};
__device__ __forceinline__ float opt_one(const OptHyper& h, float c, float g, float p, OptState& x, float* root = nullptr) {
#pragma clang fp contract(off)
  g = g * c;
  x.m = x.m * h.b1 + g * h.nb1;
  x.v = x.v * h.b2 + (g * g) * h.nb2;
  const float u = sqrtf(x.v);
  if (root) *root = u;
  return p * h.keep - (x.m / (u * h.root + h.eps)) * h.size;
}

template <int DT>
__global__ __launch_bounds__(256) void opt_update_kernel(OptTensors a, const float* coef, const OptHyper* hyper) {
  using O = OptType<DT>;
  using T = typename O::T;
  const int b = blockIdx.x, i = opt_find(a.tensors, b, [&](int k) { return a.t[k].start; });
  const auto& t = a.t[i];
  const OptHyper h = hyper[t.hyper];
  const float c = coef ? *coef : 1.f;
  const int64_t at = (int64_t)(b - t.start) * OPT_CHUNK;
  const int n = (int)min((int64_t)OPT_CHUNK, t.n - at), whole = t.vec ? n / 4 : 0;
  T* p = static_cast<T*>(t.p) + at;
  const T* g = static_cast<const T*>(t.g) + at;
  float *m = static_cast<float*>(t.m) + at, *v = static_cast<float*>(t.v) + at, *w = DT == LIN_F32 ? nullptr : t.master + at;
#pragma unroll 2
  for (int j = 4 * threadIdx.x; j < 4 * whole; j += 1024) {
    float gx[4], px[4], mx[4], vx[4];
    O::get4(g + j, gx);
    if constexpr (DT == LIN_F32) O::get4(p + j, px);
    else O::master4(w + j, p + j, px);
    OptType<LIN_F32>::get4(m + j, mx);
    OptType<LIN_F32>::get4(v + j, vx);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      OptState x{mx[e], vx[e]};
      px[e] = opt_one(h, c, gx[e], px[e], x);
      mx[e] = x.m;
      vx[e] = x.v;
    }
    if constexpr (DT != LIN_F32) OptType<LIN_F32>::put4(w + j, px);
    O::put4(p + j, px);
    OptType<LIN_F32>::put4(m + j, mx);
    OptType<LIN_F32>::put4(v + j, vx);
  }
  for (int j = 4 * whole + threadIdx.x; j < n; j += 256) {
    OptState x{m[j], v[j]};
    float start;
    if constexpr (DT == LIN_F32) start = p[j];
    else start = O::master(w[j], p[j]);
    const float q = opt_one(h, c, O::get(g + j), start, x);
    if constexpr (DT != LIN_F32) w[j] = q;
    O::put(p + j, q);
    m[j] = x.m;
    v[j] = x.v;
  }
}

// ---- states of 8 bits ---------------------------------------------------------------------------------------------

__device__ __forceinline__ float opt_m_value(int c, float s) {
#pragma clang fp contract(off)
  return (float)(c * (c < 0 ? -c : c)) * s;
}
__device__ __forceinline__ float opt_v_value(int c, float s) {
#pragma clang fp contract(off)
  const float u = (float)(c * c) * s;
  return u * u;
}
__device__ __forceinline__ uint32_t opt_hash(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x5D8AF3B5u;
  x = (x ^ (x >> 15)) * 0x2F6B4E1Du;
  return x ^ (x >> 16);
}
__device__ __forceinline__ float opt_dither(uint32_t bits) { return ((float)bits + 0.5f) * (1.f / 65536.f); }
// floor(sqrt(x / s)) as correctly rounded division and root give it: a code turns on it where a value lies at a code's own, and
// most do, since a step moves v by a thousandth and its scale with it.  The quotient by the inverse is within two units of the
// last place; its remainder (exact) corrects it, twice, and it is the rounded one.  Its root rounds to the whole number n or beyond
// where it is above n^2 - n u, u the distance of the number below n ((n - u / 2)^2 is between the two, and no quotient).
__device__ __forceinline__ float opt_floor_root(float x, float s, float inv) {
#pragma clang fp contract(off)
  float q = x * inv;
  q = fmaf(fmaf(-q, s, x), inv, q);
  q = fmaf(fmaf(-q, s, x), inv, q);
  const float n = fmaxf(rintf(__builtin_amdgcn_sqrtf(q)), 1.f), u = __uint_as_float((__float_as_uint(n) - 1) & 0x7f800000u) * 0x1p-23f;
  return fmaf(n, u, fmaf(-n, n, q)) > 0.f ? n : n - 1.f;
}
// ... of four values; inv: 1 / s, or 0 where there is no code
__device__ __forceinline__ void opt_roots(const float* x, float s, float inv, float* root) {
#pragma clang fp contract(off)
  const float all = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(s)));      // (the wave's)
  if (all < 0x1p-100f) {                   // (remainders would be cut)
#pragma unroll 1
    for (int e = 0; e < 4; ++e) root[e] = floorf(sqrtf(x[e] / s));
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) root[e] = opt_floor_root(x[e], s, inv);
}
// root: floor(sqrt(|m| / s)), floor(sqrt(u / s))
__device__ __forceinline__ int opt_m_code(float m, float s, float inv, float root, float r) {
#pragma clang fp contract(off)
  const float a = fabsf(m), c = fminf(root, 126.f), low = c * c * s, high = (c + 1.f) * (c + 1.f) * s;
  const int k = inv > 0.f ? (int)c + (a - low > r * (high - low)) : 0;
  return m < 0.f ? -k : k;
}
__device__ __forceinline__ int opt_v_code(float v, float s, float inv, float root, float r) {
#pragma clang fp contract(off)
  const float c = fminf(root, 254.f);
  float low = c * c * s, high = (c + 1.f) * (c + 1.f) * s;
  low = low * low;
  high = high * high;
  const int k = inv > 0.f ? (int)c + (v - low > r * (high - low)) : 0;
  return inv > 0.f && v > 0.f && k < 1 ? 1 : k;
}
// largest of a wave; NaN where one of it is not finite
__device__ __forceinline__ float opt_wave_max(float x) {
  const bool bad = __any(!(x < INFINITY));
#pragma unroll
  for (int o = 1; o < WAVE; o *= 2) x = fmaxf(x, __shfl_xor(x, o));
  return bad ? NAN : x;
}

// A wave takes a block of 256 elements at a time, a lane four of them.
template <int DT>
__global__ __launch_bounds__(256) void opt_update8_kernel(OptTensors a, const float* coef, const OptHyper* hyper) {
#pragma clang fp contract(off)
  using O = OptType<DT>;
  using T = typename O::T;
  const int b = blockIdx.x, i = opt_find(a.tensors, b, [&](int k) { return a.t[k].start; });
  const auto& t = a.t[i];
  const OptHyper h = hyper[t.hyper];
  const float c = coef ? *coef : 1.f;
  const int64_t first = (int64_t)(b - t.start) * OPT_CHUNK8;
  for (int k = wave_id(); k < OPT_CHUNK8 / OPT_BLOCK; k += 4) {
    const int64_t at = first + k * OPT_BLOCK;
    if (at >= t.n) break;
    const int64_t block = at / OPT_BLOCK, j = at + 4 * lane_id();
    const int n = (int)max((int64_t)0, min((int64_t)4, t.n - j));
    T* p = static_cast<T*>(t.p) + j;
    const T* g = static_cast<const T*>(t.g) + j;
    float* w = DT == LIN_F32 ? nullptr : t.master + j;
    int8_t* mc = static_cast<int8_t*>(t.m) + j;
    uint8_t* vc = static_cast<uint8_t*>(t.v) + j;
    float gx[4] = {}, px[4] = {};
    int cm[4] = {}, cv[4] = {};
    const bool vec = t.vec && n == 4;
    if (vec) {
      O::get4(g, gx);
      if constexpr (DT == LIN_F32) O::get4(p, px);
      else O::master4(w, p, px);
      const uint32_t um = *reinterpret_cast<const uint32_t*>(mc), uv = *reinterpret_cast<const uint32_t*>(vc);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cm[e] = (int8_t)(um >> (8 * e));
        cv[e] = (uint8_t)(uv >> (8 * e));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) {
          gx[e] = O::get(g + e);
          if constexpr (DT == LIN_F32) px[e] = p[e];
          else px[e] = O::master(w[e], p[e]);
          cm[e] = mc[e];
          cv[e] = vc[e];
        }
    }
    const float s_m = t.ms[block], s_v = t.vs[block];
    float mx[4], vx[4], ux[4], m_top = 0.f, v_top = 0.f;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= n) {
        mx[e] = vx[e] = ux[e] = 0.f;
        continue;
      }
      OptState x{opt_m_value(cm[e], s_m), opt_v_value(cv[e], s_v)};
      px[e] = opt_one(h, c, gx[e], px[e], x, &ux[e]);
      mx[e] = x.m;
      vx[e] = x.v;
      bad |= !(fabsf(x.m) < INFINITY);
      m_top = fmaxf(m_top, fabsf(x.m));
      v_top = fmaxf(v_top, x.v);
      if (!(x.v < INFINITY)) v_top = INFINITY;
    }
    m_top = opt_wave_max(bad ? INFINITY : m_top);
    v_top = opt_wave_max(v_top);
    const float new_m = m_top * (1.f / 16129.f), new_v = sqrtf(v_top) * (1.f / 65025.f);
    const float inv_m = new_m > 0.f ? 1.f / new_m : 0.f, inv_v = new_v > 0.f ? 1.f / new_v : 0.f;
    float am[4], rm[4], rv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) am[e] = fabsf(mx[e]);
    opt_roots(am, new_m, inv_m, rm);
    opt_roots(ux, new_v, inv_v, rv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t r = opt_hash((uint32_t)(j + e) * 0x9E3779B1u + h.hash);
      cm[e] = opt_m_code(mx[e], new_m, inv_m, rm[e], opt_dither(r & 0xffffu));
      cv[e] = opt_v_code(vx[e], new_v, inv_v, rv[e], opt_dither(r >> 16));
    }
    if (vec) {
      if constexpr (DT != LIN_F32) OptType<LIN_F32>::put4(w, px);
      O::put4(p, px);
      uint32_t um = 0, uv = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        um |= (uint32_t)(cm[e] & 255) << (8 * e);
        uv |= (uint32_t)cv[e] << (8 * e);
      }
      *reinterpret_cast<uint32_t*>(mc) = um;
      *reinterpret_cast<uint32_t*>(vc) = uv;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) {
          if constexpr (DT != LIN_F32) w[e] = px[e];
          O::put(p + e, px[e]);
          mc[e] = (int8_t)cm[e];
          vc[e] = (uint8_t)cv[e];
        }
    }
    if (lane_id() == 0) {                  // (read by the whole wave above)
      t.ms[block] = new_m;
      t.vs[block] = new_v;
    }
  }
}

// p and master: where m and v go
__global__ __launch_bounds__(256) void opt_unpack_kernel(OptTensors a) {
  const int b = blockIdx.x, i = opt_find(a.tensors, b, [&](int k) { return a.t[k].start; });
  const auto& t = a.t[i];
  const int64_t first = (int64_t)(b - t.start) * OPT_CHUNK8;
  const int n = (int)min((int64_t)OPT_CHUNK8, t.n - first);
  const int8_t* mc = static_cast<const int8_t*>(t.m) + first;
  const uint8_t* vc = static_cast<const uint8_t*>(t.v) + first;
  float *m = static_cast<float*>(t.p) + first, *v = t.master + first;
  const int whole = t.vec ? n / 4 : 0;
#pragma unroll 2
  for (int j = 4 * threadIdx.x; j < 4 * whole; j += 1024) {
    const uint32_t um = *reinterpret_cast<const uint32_t*>(mc + j), uv = *reinterpret_cast<const uint32_t*>(vc + j);
    const float s_m = t.ms[(first + j) / OPT_BLOCK], s_v = t.vs[(first + j) / OPT_BLOCK];
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = opt_m_value((int8_t)(um >> (8 * e)), s_m);
      y[e] = opt_v_value((uint8_t)(uv >> (8 * e)), s_v);
    }
    OptType<LIN_F32>::put4(m + j, x);
    OptType<LIN_F32>::put4(v + j, y);
  }
  for (int j = 4 * whole + threadIdx.x; j < n; j += 256) {
    m[j] = opt_m_value(mc[j], t.ms[(first + j) / OPT_BLOCK]);
    v[j] = opt_v_value(vc[j], t.vs[(first + j) / OPT_BLOCK]);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------

static int64_t opt_parts(const gdn2_adamw_tensor* t, int n) {
  int64_t parts = 0;
  for (int i = 0; i < n; ++i) parts += (t[i].numel + OPT_NORM_CHUNK - 1) / OPT_NORM_CHUNK;
  return parts;
}
// coefficient, factors, the norm's parts
static size_t opt_hyper_bytes(int n) { return 256 + ((size_t)n * sizeof(OptHyper) + 255) / 256 * 256; }
size_t adamw_workspace_bytes(const gdn2_adamw_tensor* t, int n) { return opt_hyper_bytes(n) + 8 * (size_t)opt_parts(t, n); }

// The tensors of a type, at(i), as many to a launch as an argument block holds: go(block, the first's place, workgroups)
template <class A, class F>
static void opt_each(int n, int dtype, int bits, A at, F go) {
  const int size = dtype == LIN_F32 ? 4 : 2, chunk = bits == 8 ? OPT_CHUNK8 : OPT_CHUNK;
  OptTensors a{};
  int64_t blocks = 0;
  int first = 0;
  auto flush = [&] {
    if (a.tensors) go(a, first, (int)blocks);
    a.tensors = 0;
    blocks = 0;
  };
  for (int i = 0; i < n; ++i) {
    const gdn2_adamw_tensor x = at(i);
    if (x.dtype != dtype) continue;
    const int64_t b = (x.numel + chunk - 1) / chunk;
    if (a.tensors == OPT_TENSORS || blocks + b > OPT_GRID || (a.tensors && i - first > 0x7fff)) flush();
    if (a.tensors == 0) first = i;
    auto& o = a.t[a.tensors++];
    o.p = x.p; o.g = x.g; o.m = x.m; o.v = x.v; o.ms = x.m_scale; o.vs = x.v_scale; o.master = x.master;
    o.n = x.numel;
    o.start = (int)blocks;
    o.hyper = (int16_t)(i - first);
    auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
    o.vec = (low(x.p) | low(x.g)) % (4 * size) == 0 && (low(x.m) | low(x.v)) % (bits == 8 ? 4 : 16) == 0 && low(x.master) % 16 == 0;
    blocks += b;
  }
  flush();
}

hipError_t launch_adamw(const gdn2_adamw_tensor* t, int n, int bits, double max_norm, float* norm, void* workspace, hipStream_t s) {
  float* coef = static_cast<float*>(workspace);
  OptHyper* hyper = reinterpret_cast<OptHyper*>(static_cast<char*>(workspace) + 256);
  double* part = reinterpret_cast<double*>(static_cast<char*>(workspace) + opt_hyper_bytes(n));
  const bool clip = max_norm > 0.0 || norm;
  int64_t parts = 0;
  for (int dtype = LIN_F32; clip && dtype <= LIN_F16; ++dtype) {
    OptGrads a{};
    int64_t blocks = 0;
    auto flush = [&] {
      if (a.tensors) {
        auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, s, a, part + parts); };
        dtype == LIN_F32 ? go(opt_norm_kernel<LIN_F32>) : dtype == LIN_BF16 ? go(opt_norm_kernel<LIN_BF16>) : go(opt_norm_kernel<LIN_F16>);
      }
      parts += blocks;
      blocks = a.tensors = 0;
    };
    for (int i = 0; i < n; ++i) {
      if (t[i].dtype != dtype) continue;
      const int64_t b = (t[i].numel + OPT_NORM_CHUNK - 1) / OPT_NORM_CHUNK;
      if (a.tensors == OPT_GRADS || blocks + b > OPT_GRID) flush();
      a.g[a.tensors] = t[i].g;
      a.n[a.tensors] = t[i].numel;
      a.start[a.tensors++] = (int)blocks;
      blocks += b;
    }
    flush();
  }
  for (int i = 0; i < n; i += OPT_STEPS) {
    OptSteps a{};
    for (; a.tensors < OPT_STEPS && i + a.tensors < n; ++a.tensors) {
      const gdn2_adamw_tensor& x = t[i + a.tensors];
      auto& o = a.t[a.tensors];
      o.step = x.step; o.lr = x.lr; o.b1 = x.beta1; o.b2 = x.beta2; o.eps = x.eps; o.wd = x.weight_decay;
      o.ordinal = (uint32_t)x.ordinal;
    }
    hipLaunchKernelGGL(opt_begin_kernel, dim3(1), dim3(1024), 0, s, a, part, i ? 0 : (int)parts, max_norm, coef, norm, hyper + i);
  }
  for (int dtype = LIN_F32; dtype <= LIN_F16; ++dtype)
    opt_each(n, dtype, bits, [&](int i) { return t[i]; }, [&](const OptTensors& a, int from, int blocks) {
      auto go = [&](auto k) { hipLaunchKernelGGL(k, dim3(blocks), dim3(256), 0, s, a, clip ? coef : nullptr, hyper + from); };
      if (bits == 8) dtype == LIN_F32 ? go(opt_update8_kernel<LIN_F32>) : dtype == LIN_BF16 ? go(opt_update8_kernel<LIN_BF16>) : go(opt_update8_kernel<LIN_F16>);
      else dtype == LIN_F32 ? go(opt_update_kernel<LIN_F32>) : dtype == LIN_BF16 ? go(opt_update_kernel<LIN_BF16>) : go(opt_update_kernel<LIN_F16>);
    });
  return hipGetLastError();
}

hipError_t launch_adamw_unpack(const gdn2_adamw_tensor* t, int n, float* const* m_out, float* const* v_out, hipStream_t s) {
  auto at = [&](int i) {                   // (as a float32 parameter whose place m takes, with v for a master)
    gdn2_adamw_tensor x = t[i];
    x.dtype = LIN_F32;
    x.p = m_out[i];
    x.g = nullptr;
    x.master = v_out[i];
    return x;
  };
  opt_each(n, LIN_F32, 8, at, [&](const OptTensors& a, int, int blocks) { hipLaunchKernelGGL(opt_unpack_kernel, dim3(blocks), dim3(256), 0, s, a); });
  return hipGetLastError();
}

}  // namespace gdn2
