// Rows of activations times a matrix of 4-bit weights with group scales, on gfx950:
//   y[m][n] = sum_g s[g][n] (sum_{k in g} x[m][k] q[k][n] - z[g][n] sum_{k in g} x[m][k])  (+ bias, + residual)
// with whole q in 0 .. 15 and one scale s and zero z (bfloat16) for each column and group of 32, 64 or
// 128 rows of the matrix.
//
// The products run on the matrix cores with q itself as an operand, which 16 bits hold exactly: a byte
// 0 .. 15 read as an fp8 e4m3 number is q 2^-9 (its subnormals and first binade are one even grid), so
// two masks and four conversions with the scale 2^9 make eight operands of a word of eight nibbles.
// Activations of 16 bits are the other operand as they are, of float32 as three bfloat16 pieces of
// eight bits each, whose sum is x.  So no product is rounded; sums, group sums of x and the scaling
// are float32, and y is rounded once.
#include "gdn2_kernels.hpp"

namespace gdn2 {

// Operands of lane l in a 32-deep product: eight k values (group c = l / 16) of row or column l % 16.
template <bool F16>
__device__ __forceinline__ void w4_mfma(f4& acc, const s8& a, const s8& b) {
  if constexpr (F16) asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
  else asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(acc) : "v"(a), "v"(b));
}
template <bool F16>
__device__ __forceinline__ void w4_mfma_first(f4& acc, const s8& a, const s8& b) {      // acc = a b
  if constexpr (F16) asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=&v"(acc) : "v"(a), "v"(b));
  else asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(acc) : "v"(a), "v"(b));
}

// Eight nibbles as operands: element e of 0 .. 3 is nibble 2 e, of 4 .. 7 nibble 2 (e - 4) + 1.
template <bool F16, bool HI>
__device__ __forceinline__ uint32_t w4_pair(uint32_t bytes) {            // bytes 0, 1 or (HI) 2, 3
  if constexpr (F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(bytes, 512.f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(bytes, 512.f, HI));
}
template <bool F16>
__device__ __forceinline__ s8 w4_operand(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  return __builtin_bit_cast(s8, make_uint4(w4_pair<F16, false>(lo), w4_pair<F16, true>(lo), w4_pair<F16, false>(hi),
                                           w4_pair<F16, true>(hi)));
}

// Eight activations as operands: one piece of 16 bits, or float32's three, the smallest first.
template <int XT>
struct W4Frag {
  static constexpr int NP = XT == W4_F32 ? 3 : 1;
  s8 p[NP];
};
__device__ __forceinline__ uint32_t w4_high_halves(float a, float b) {     // upper 16 bits of a | of b << 16
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float w4_top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// Cut, not rounded: each piece is the next eight bits, and both differences are exact.
__device__ __forceinline__ void w4_split(const float* x, W4Frag<W4_F32>& f) {
  uint32_t h[4], m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[2 * i], b = x[2 * i + 1];
    const float ra = a - w4_top(a), rb = b - w4_top(b);
    h[i] = w4_high_halves(a, b);
    m[i] = w4_high_halves(ra, rb);
    l[i] = w4_high_halves(ra - w4_top(ra), rb - w4_top(rb));
  }
  f.p[0] = __builtin_bit_cast(s8, make_uint4(l[0], l[1], l[2], l[3]));
  f.p[1] = __builtin_bit_cast(s8, make_uint4(m[0], m[1], m[2], m[3]));
  f.p[2] = __builtin_bit_cast(s8, make_uint4(h[0], h[1], h[2], h[3]));
}

// x[m][k .. k+7], zero outside M and K
template <int XT>
__device__ __forceinline__ W4Frag<XT> w4_load_x(const W4Args& a, int m, int k) {
  W4Frag<XT> f;
  if constexpr (XT == W4_F32) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (m < a.M) {
      const float* p = static_cast<const float*>(a.x) + (size_t)m * a.ldx + k;
      if (a.vec) {
        if (k < a.K) {
          const float4 u = *reinterpret_cast<const float4*>(p), w = *reinterpret_cast<const float4*>(p + 4);
          v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
          v[4] = w.x; v[5] = w.y; v[6] = w.z; v[7] = w.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < a.K) v[e] = p[e];
      }
    }
    w4_split(v, f);
  } else {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (m < a.M) {
      const uint16_t* p = static_cast<const uint16_t*>(a.x) + (size_t)m * a.ldx + k;
      if (a.vec) {
        if (k < a.K) u = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < a.K ? p[e] : 0u;
        u = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
      }
    }
    f.p[0] = __builtin_bit_cast(s8, u);
  }
  return f;
}

template <int XT>
__device__ __forceinline__ float w4_ld(const void* p, size_t i) {
  if constexpr (XT == W4_F32) return static_cast<const float*>(p)[i];
  else if constexpr (XT == W4_BF16) return bf16_val(static_cast<const uint16_t*>(p)[i]);
  else return (float)static_cast<const _Float16*>(p)[i];
}
template <int XT>
__device__ __forceinline__ void w4_st(void* p, size_t i, float v) {
  if constexpr (XT == W4_F32) static_cast<float*>(p)[i] = v;
  else if constexpr (XT == W4_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)bf16_bits(v);
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

__device__ __forceinline__ void w4_hold(f4& a) { asm volatile("" : "+v"(a)); }

// A workgroup takes 16 NB columns and 16 MT rows; its waves take the 128-deep blocks of the sum in
// turn and add their parts through LDS in wave order.
template <int XT, int GROUP, int MT, int NB>
__global__ __launch_bounds__(512) void w4_rows_kernel(W4Args a) {
  constexpr bool F16 = XT == W4_F16;
  constexpr int NP = W4Frag<XT>::NP, NG = W4_KB / GROUP, SG = GROUP / 32;
  extern __shared__ f4 red[];                        // [wave][nb][mt][lane]
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), W = blockDim.x / WAVE;
  const int nb0 = blockIdx.x * NB, m0 = blockIdx.y * 16 * MT;
  const s8 ones = __builtin_bit_cast(s8, F16 ? make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u)
                                             : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
  f4 tot[NB][MT];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) tot[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  for (int kb = w; kb < a.nkb; kb += W) {
    uint4 q[NB], mt[NB][NG];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const size_t nb = min(nb0 + i, a.nnb - 1);
      q[i] = reinterpret_cast<const uint4*>(a.q)[(nb * a.nkb + kb) * WAVE + l];
#pragma unroll
      for (int g = 0; g < NG; ++g)
        mt[i][g] = reinterpret_cast<const uint4*>(a.meta)[((nb * a.nkb + kb) * NG + g) * 4 + c];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f4 acc[NB][MT], xs[MT];
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        const int j = g * SG + s;
        W4Frag<XT> x[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) x[t] = w4_load_x<XT>(a, m0 + 16 * t + r, kb * W4_KB + 32 * j + 8 * c);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const s8 op = w4_operand<F16>(j == 0 ? q[i].x : j == 1 ? q[i].y : j == 2 ? q[i].z : q[i].w);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int p = 0; p < NP; ++p) {
              if (s == 0 && p == 0) w4_mfma_first<F16>(acc[i][t], op, x[t].p[p]);
              else w4_mfma<F16>(acc[i][t], op, x[t].p[p]);
            }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            if (s == 0 && p == 0) w4_mfma_first<F16>(xs[t], ones, x[t].p[p]);
            else w4_mfma<F16>(xs[t], ones, x[t].p[p]);
          }
      }
      drain(xs[0]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        w4_hold(xs[t]);
#pragma unroll
        for (int i = 0; i < NB; ++i) w4_hold(acc[i][t]);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint32_t sz[4] = {mt[i][g].x, mt[i][g].y, mt[i][g].z, mt[i][g].w};
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = bf16_val(sz[e] & 0xffffu), z = __uint_as_float(sz[e] & 0xffff0000u);
            tot[i][t][e] = fmaf(s, fmaf(-z, xs[t][e], acc[i][t][e]), tot[i][t][e]);
          }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[((w * NB + i) * MT + t) * WAVE + l] = tot[i][t];
  __syncthreads();
  for (int x = threadIdx.x; x < NB * MT * WAVE; x += blockDim.x) {
    f4 s = red[x];
    for (int v = 1; v < W; ++v) {
      const f4 u = red[v * NB * MT * WAVE + x];
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += u[e];
    }
    const int lane = x & 63, t = (x / WAVE) % MT, i = x / (WAVE * MT);
    const int m = m0 + 16 * t + (lane & 15), n = (nb0 + i) * 16 + 4 * (lane >> 4);
    if (m >= a.M) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (n + e >= a.N) break;
      float v = s[e];
      if (a.bias) v += w4_ld<XT>(a.bias, n + e);
      if (a.res) v += w4_ld<XT>(a.res, (size_t)m * a.ldr + n + e);
      w4_st<XT>(a.y, (size_t)m * a.N + n + e, v);
    }
  }
}

template <int XT, int GROUP>
static void w4_go(const W4Args& a, hipStream_t s) {
  auto go = [&](auto mt, auto nb) {
    constexpr int MT = decltype(mt)::value, NB = decltype(nb)::value;
    const int W = a.nkb < 8 ? a.nkb : 8;
    const dim3 grid((a.nnb + NB - 1) / NB, (a.M + 16 * MT - 1) / (16 * MT));
    hipLaunchKernelGGL((w4_rows_kernel<XT, GROUP, MT, NB>), grid, dim3(W * WAVE), (size_t)W * NB * MT * WAVE * 16, s, a);
  };
  using std::integral_constant;
  if (a.M <= 16) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
}

template <int XT>
static void w4_go_group(int group, const W4Args& a, hipStream_t s) {
  if (group == 32) w4_go<XT, 32>(a, s);
  else if (group == 64) w4_go<XT, 64>(a, s);
  else w4_go<XT, 128>(a, s);
}

hipError_t launch_w4(int dtype, int group, const W4Args& a, hipStream_t s) {
  if (dtype == W4_F32) w4_go_group<W4_F32>(group, a, s);
  else if (dtype == W4_BF16) w4_go_group<W4_BF16>(group, a, s);
  else w4_go_group<W4_F16>(group, a, s);
  return hipGetLastError();
}

}  // namespace gdn2
