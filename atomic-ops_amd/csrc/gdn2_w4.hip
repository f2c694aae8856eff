// Rows of activations times a matrix of 4-bit weights with group scales, on gfx950:
//   y[m][n] = sum_g s[g][n] (sum_{k in g} x[m][k] q[k][n] - z[g][n] sum_{k in g} x[m][k])  (+ bias, + residual)
// with whole q in 0 .. 15 and one scale s and zero z (bfloat16) for each column and group of 32, 64 or
// 128 rows of the matrix.
//
// The products run on the matrix cores with q itself as an operand, which 16 bits hold exactly: a byte
// 0 .. 15 read as an fp8 e4m3 number is q 2^-9 (its subnormals and first binade are one even grid), so
// two masks and four conversions with the scale 2^9 make eight operands of a word of eight nibbles.
// Activations of 16 bits are the other operand as they are, of float32 as three bfloat16 pieces of
// eight bits each, whose sum is x but for bits below 2^-133, bfloat16's smallest number (so an x below
// about 1e-33 has fewer than 24 bits).  So no product is rounded; sums, group sums of x and the
// scaling are float32, and y is rounded once.
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

// Four products with one left operand; FIRST: results, else added to.
template <bool F16, bool FIRST>
__device__ __forceinline__ void w4_mfma4(f4& a0, f4& a1, f4& a2, f4& a3, const s8& x, const s8& b0, const s8& b1, const s8& b2, const s8& b3) {
#define W4_FOUR(op, c0, c1, c2, c3)                                            \
  "s_nop 1\n\t" op " %0, %4, %5, " c0 "\n\t" op " %1, %4, %6, " c1 "\n\t" op \
  " %2, %4, %7, " c2 "\n\t" op " %3, %4, %8, " c3
  if constexpr (FIRST && F16)
    asm volatile(W4_FOUR("v_mfma_f32_16x16x32_f16", "0", "0", "0", "0") : "=&v"(a0), "=&v"(a1), "=&v"(a2), "=&v"(a3) : "v"(x), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
  else if constexpr (FIRST)
    asm volatile(W4_FOUR("v_mfma_f32_16x16x32_bf16", "0", "0", "0", "0") : "=&v"(a0), "=&v"(a1), "=&v"(a2), "=&v"(a3) : "v"(x), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
  else if constexpr (F16)
    asm volatile(W4_FOUR("v_mfma_f32_16x16x32_f16", "%0", "%1", "%2", "%3") : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3) : "v"(x), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
  else
    asm volatile(W4_FOUR("v_mfma_f32_16x16x32_bf16", "%0", "%1", "%2", "%3") : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3) : "v"(x), "v"(b0), "v"(b1), "v"(b2), "v"(b3));
#undef W4_FOUR
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

// Eight activations as loaded: 16 or (float32) 32 bytes
template <int XT>
struct W4Raw {
  static constexpr int NV = XT == W4_F32 ? 2 : 1;
  uint4 v[NV];
};
template <int XT>
__device__ __forceinline__ W4Frag<XT> w4_frag(const W4Raw<XT>& x) {
  W4Frag<XT> f;
  if constexpr (XT == W4_F32) {
    const uint32_t u[8] = {x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w, x.v[1].x, x.v[1].y, x.v[1].z, x.v[1].w};
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e]);
    w4_split(v, f);
  } else {
    f.p[0] = __builtin_bit_cast(s8, x.v[0]);
  }
  return f;
}
// Their sum
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
template <int XT>
__device__ __forceinline__ float w4_sum8(const W4Raw<XT>& x) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < W4Raw<XT>::NV; ++i) {
    const uint32_t u[4] = {x.v[i].x, x.v[i].y, x.v[i].z, x.v[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (XT == W4_F32) s += __uint_as_float(u[e]);
      else if constexpr (XT == W4_BF16)
        s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, u[e]), __builtin_bit_cast(b2v, 0x3f803f80u), s, false);
      else s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2v, u[e]), __builtin_bit_cast(h2v, 0x3c003c00u), s, false);
    }
  }
  return s;
}
// x[m][k .. k+7] element by element, zero outside M and K: rows that 16-byte accesses cannot take
template <int XT>
__device__ __forceinline__ W4Raw<XT> w4_load_odd(const W4Args& a, int m, int k) {
  W4Raw<XT> r;
  if constexpr (XT == W4_F32) {
    const float* p = static_cast<const float*>(a.x) + (size_t)min(m, a.M - 1) * a.ldx + k;
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = m < a.M && k + e < a.K ? __float_as_uint(p[e]) : 0u;
    r.v[0] = make_uint4(v[0], v[1], v[2], v[3]);
    r.v[1] = make_uint4(v[4], v[5], v[6], v[7]);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.x) + (size_t)min(m, a.M - 1) * a.ldx + k;
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = m < a.M && k + e < a.K ? p[e] : 0u;
    r.v[0] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
  return r;
}
// ... and by buffer loads from base + off: an offset past the buffer's end reads zero, without a branch
constexpr uint32_t W4_OUT = 0x60000000u;             // above any offset of a buffer (at most 2^30)
typedef unsigned u4v __attribute__((ext_vector_type(4)));
// (a buffer that the compiler does not know to be uniform costs a loop over the lanes at every load)
__device__ __forceinline__ int w4_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w4_buffer(const void* p, size_t at, int64_t bytes) {
  const uint64_t u = reinterpret_cast<uint64_t>(p) + at;
  const uint64_t base = (uint64_t)(uint32_t)w4_uniform((int)(u >> 32)) << 32 | (uint32_t)w4_uniform((int)u);
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, w4_uniform((int)bytes), 0x00027000);
}
__device__ __forceinline__ uint4 w4_buffer16(__amdgpu_buffer_rsrc_t b, uint32_t off, int uniform) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, w4_uniform(uniform), 0));
}
__device__ __forceinline__ uint32_t w4_buffer4(__amdgpu_buffer_rsrc_t b, uint32_t off, int uniform) {
  return __builtin_amdgcn_raw_buffer_load_b32(b, (int)off, w4_uniform(uniform), 0);
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

template <int N>
__device__ __forceinline__ s8 w4_down(const s8& x) {         // lane i of a row of 16 takes lane i + N's
  if constexpr (N == 0) return x;
  uint4 u = __builtin_bit_cast(uint4, x);
  auto f = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x100 | N, 0xf, 0xf, true); };
  return __builtin_bit_cast(s8, make_uint4(f(u.x), f(u.y), f(u.z), f(u.w)));
}
template <int XT, int N>
__device__ __forceinline__ W4Frag<XT> w4_frag_down(const W4Frag<XT>& x) {
  W4Frag<XT> y;
#pragma unroll
  for (int p = 0; p < W4Frag<XT>::NP; ++p) y.p[p] = w4_down<N>(x.p[p]);
  return y;
}

// Four results of a row: plus bias and residual, rounded, stored; whole where a.wide allows it
template <int XT>
__device__ __forceinline__ float4 w4_ld4(const void* p, size_t i) {
  if constexpr (XT == W4_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  if constexpr (XT == W4_BF16)
    return make_float4(bf16_val(u.x & 0xffffu), __uint_as_float(u.x & 0xffff0000u), bf16_val(u.y & 0xffffu), __uint_as_float(u.y & 0xffff0000u));
  const h2v a = __builtin_bit_cast(h2v, u.x), b = __builtin_bit_cast(h2v, u.y);
  return make_float4((float)a[0], (float)a[1], (float)b[0], (float)b[1]);
}
template <int XT>
__device__ __forceinline__ void w4_out4(const W4Args& a, int m, int n, float4 v) {
  const size_t at = (size_t)m * a.N + n;
  if (a.wide) {
    if (a.bias) v = add4(v, w4_ld4<XT>(a.bias, n));
    if (a.res) v = add4(v, w4_ld4<XT>(a.res, (size_t)m * a.ldr + n));
    if constexpr (XT == W4_F32) *reinterpret_cast<float4*>(static_cast<float*>(a.y) + at) = v;
    else {
      uint2 u;
      if constexpr (XT == W4_BF16) u = make_uint2(bf16_pack(v.x, v.y), bf16_pack(v.z, v.w));
      else u = make_uint2(__builtin_bit_cast(uint32_t, h2v{(_Float16)v.x, (_Float16)v.y}), __builtin_bit_cast(uint32_t, h2v{(_Float16)v.z, (_Float16)v.w}));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) = u;
    }
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= a.N) return;
    float y = f[e];
    if (a.bias) y += w4_ld<XT>(a.bias, n + e);
    if (a.res) y += w4_ld<XT>(a.res, (size_t)m * a.ldr + n + e);
    w4_st<XT>(a.y, at + e, y);
  }
}
__device__ __forceinline__ void w4_part4(const W4Args& a, size_t at, int n, const float4& v) {
  if (a.N % 4 == 0) {
    *reinterpret_cast<float4*>(a.part + at) = v;
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) a.part[at + e] = f[e];
}

template <int CTRL>
__device__ __forceinline__ float w4_dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float w4_quad_sum(float x) {      // over the four lanes of a quad
  x += w4_dpp<0xb1>(x);
  return x + w4_dpp<0x4e>(x);
}

// Waves of a workgroup at most
constexpr int w4_waves(int XT, int NB) { return XT != W4_F32 && NB == 1 ? 16 : 8; }

// Few rows: bound by the bytes of the weights (one row of 8192 x 28672 bfloat16, groups of 128: 23.3 us,
// 5.3 TB/s; a plain read of as much 19.8 us), small matrices by a launch (512 x 4614 float32 3.3 us).  A
// workgroup takes 16 NB columns and 16 / SP rows; its waves take the 128-deep blocks of the sum in turn, the
// next one's loads issued before the products of this one, and add their parts through LDS in wave order.
//   x is the products' left operand, so a lane's results are rows 4 (l / 16) + e of one column and it
// needs one scale.  With few rows an operand's 16 rows hold SP steps' pieces of each: row m's at rows
// SP m, SP m + 1, ...: one load then serves SP steps, the later ones after a move by lanes (whose other
// rows' products are not looked at), and only 4 / SP of a lane's four results are used.
template <int XT, int GROUP, int SP, int NB>
__global__ __launch_bounds__(w4_waves(XT, NB) * WAVE) void w4_rows_kernel(W4Args a) {
  constexpr bool F16 = XT == W4_F16;
  constexpr int NP = W4Frag<XT>::NP, NG = W4_KB / GROUP, SG = GROUP / 32, E = XT == W4_F32 ? 4 : 2;
  constexpr int XL = 4 / SP, NE = 4 / SP, MR = 16 / SP;       // loads of x a block, results a lane, rows a tile
  extern __shared__ float red[];                     // [wave][nb][e][lane]
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), W = blockDim.x / WAVE;
  const int nb0 = blockIdx.x * NB, m0 = blockIdx.y * MR;
  const s8 ones = __builtin_bit_cast(s8, F16 ? make_uint4(0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u)
                                             : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u));
  // a lane's offsets are fixed and a block's are uniform, so that a load takes no address arithmetic
  const int rows = min(MR, a.M - m0), nbs = min(NB, a.nnb - nb0);
  const __amdgpu_buffer_rsrc_t xb =
      w4_buffer(a.x, (size_t)m0 * a.ldx * E, a.vec ? ((rows - 1) * (int64_t)a.ldx + a.K) * E : 0);
  const __amdgpu_buffer_rsrc_t qb = w4_buffer(a.q, (size_t)nb0 * a.nkb * 1024, (int64_t)nbs * a.nkb * 1024);
  const __amdgpu_buffer_rsrc_t sb = w4_buffer(a.meta, (size_t)nb0 * a.nkb * (NG * 64), (int64_t)nbs * a.nkb * (NG * 64));
  const int xk = 32 * (r % SP) + 8 * c;              // the lane's first k of a load
  uint32_t xoff[XL], qoff[NB], soff[NB];
#pragma unroll
  for (int u = 0; u < XL; ++u) xoff[u] = r / SP < rows ? (uint32_t)(r / SP * a.ldx + 32 * SP * u + xk) * E : W4_OUT;
#pragma unroll
  for (int i = 0; i < NB; ++i) {                     // (columns past the last: zero codes and scales)
    qoff[i] = (uint32_t)i * a.nkb * 1024 + 16 * l;
    soff[i] = (uint32_t)i * a.nkb * (NG * 64) + 4 * r;
  }
  float tot[NB][NE];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int e = 0; e < NE; ++e) tot[i][e] = 0.f;
  struct Block {
    uint4 q[NB];
    uint32_t sz[NB][NG];
    W4Raw<XT> x[XL];
  };
  // Without a branch, behind which the compiler would wait for all loads, these included: past the last
  // block offsets go out of range for good (in place, since a register of its own may be one that a load is
  // still to write), nothing is read and nothing used.
  auto load = [&](Block& o, int kb, auto vec) __attribute__((always_inline)) {
    const uint32_t past = kb < a.nkb ? 0u : W4_OUT;
    const int at = min(kb, a.nkb - 1);               // (the uniform part of an offset stays within the buffer)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      o.q[i] = w4_buffer16(qb, qoff[i] |= past, at * 1024);
      soff[i] |= past;
#pragma unroll
      for (int g = 0; g < NG; ++g) o.sz[i][g] = w4_buffer4(sb, soff[i] + 64 * g, at * (NG * 64));
    }
#pragma unroll
    for (int u = 0; u < XL; ++u) {
      if constexpr (vec.value) {
        xoff[u] = kb * W4_KB < a.K - 32 * SP * u - xk ? xoff[u] : W4_OUT;
#pragma unroll
        for (int v = 0; v < W4Raw<XT>::NV; ++v) o.x[u].v[v] = w4_buffer16(xb, xoff[u] + 16 * v, at * (W4_KB * E));
      } else {
        o.x[u] = w4_load_odd<XT>(a, r / SP < rows ? m0 + r / SP : a.M, kb * W4_KB + 32 * SP * u + xk);
      }
    }
  };
  auto add = [&](const Block& o) __attribute__((always_inline)) {
    W4Frag<XT> x[XL];
#pragma unroll
    for (int u = 0; u < XL; ++u) x[u] = w4_frag<XT>(o.x[u]);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f4 acc[NB], xs;
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        const int j = g * SG + s;
        const W4Frag<XT>& f = x[j / SP];
        const W4Frag<XT> xj = j % SP == 0   ? f
                              : j % SP == 1 ? w4_frag_down<XT, 1>(f)
                              : j % SP == 2 ? w4_frag_down<XT, 2>(f)
                                            : w4_frag_down<XT, 3>(f);
        s8 op[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i)
          op[i] = w4_operand<F16>(j == 0 ? o.q[i].x : j == 1 ? o.q[i].y : j == 2 ? o.q[i].z : o.q[i].w);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            if (s == 0 && p == 0) w4_mfma_first<F16>(acc[i], xj.p[p], op[i]);
            else w4_mfma<F16>(acc[i], xj.p[p], op[i]);
          }
          if (s == 0 && p == 0) w4_mfma_first<F16>(xs, xj.p[p], ones);
          else w4_mfma<F16>(xs, xj.p[p], ones);
        }
      }
      drain(xs);
#pragma unroll
      for (int i = 0; i < NB; ++i) w4_hold(acc[i]);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float s = bf16_val(o.sz[i][g] & 0xffffu), z = __uint_as_float(o.sz[i][g] & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < NE; ++e) tot[i][e] = fmaf(s, fmaf(-z, xs[e * SP], acc[i][e * SP]), tot[i][e]);
      }
    }
  };
  auto run = [&](auto vec) __attribute__((always_inline)) {
    Block even, odd;
    int kb = w;
    load(even, kb, vec);
    for (;;) {
      load(odd, kb + W, vec);
      add(even);
      if ((kb += W) >= a.nkb) break;
      load(even, kb + W, vec);
      add(odd);
      if ((kb += W) >= a.nkb) break;
    }
  };
  // (the launch gives every wave a block)
  if (a.vec) run(std::true_type{});
  else run(std::false_type{});
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int e = 0; e < NE; ++e) red[((w * NB + i) * NE + e) * WAVE + l] = tot[i][e];
  __syncthreads();
  constexpr int ALL = NB * NE * WAVE;
  for (int x = threadIdx.x; x < ALL; x += blockDim.x) {
    float v = red[x];
    for (int u = 1; u < W; ++u) v += red[u * ALL + x];
    const int lane = x % WAVE, e = x / WAVE % NE, i = x / (WAVE * NE);
    const int m = m0 + NE * (lane >> 4) + e, n = (nb0 + i) * 16 + (lane & 15);
    if (m >= a.M || n >= a.N) continue;
    if (a.bias) v += w4_ld<XT>(a.bias, n);
    if (a.res) v += w4_ld<XT>(a.res, (size_t)m * a.ldr + n);
    w4_st<XT>(a.y, (size_t)m * a.N + n, v);
  }
}

// More rows: a workgroup of WM x WN x WK waves takes 16 MT WM rows and 16 NBW WN columns, and one of the
// sum's gridDim.z parts, WK 128-deep blocks of it at a time (one for each wave along WK).  The waves stage the
// blocks of x in LDS as operands (float32 split once), with each group's sum, so that x crosses the
// caches once for all the columns: a CU takes about 34 bytes a nanosecond from the L2, and with x in
// every wave's registers that was the bound.  The next blocks are loaded while these are multiplied.
// With several parts the sums go to a.part (part, M, N), which w4_join_kernel adds in order.
//   32 rows of 14336 x 4096: 13.6 us bfloat16, 13.3 float16, 20.7 float32 with the weights (32 MB) in the
// last-level cache, 14.0, 14.1 and 21.2 from HBM (2.3 TB/s), of that the join 2 to 4: a workgroup has seven
// rounds of staging, a barrier, products and scaling, one after the other (weights loaded two rounds ahead
// instead of one, bfloat16: 14.5 for 14.3).  128 rows of 4096 x 4096 15.4.
template <int XT_, int GROUP_, int MT_, int NBW_, int WM_, int WN_, int WK_>
struct W4Tile {
  static constexpr int XT = XT_, GROUP = GROUP_, MT = MT_, NBW = NBW_, WM = WM_, WN = WN_, WK = WK_;
  static constexpr int W = WM * WN * WK, NP = W4Frag<XT>::NP, NG = W4_KB / GROUP;
  static constexpr int UNITS = WK * WM * MT;         // 16 rows of a block each
  static constexpr int UNIT = 4 * NP * WAVE * 16;    // bytes of a unit's operands
  static constexpr int BUF = UNITS * (UNIT + NG * 64);
  static constexpr int BM = 16 * MT * WM, BN = 16 * NBW * WN;
  static constexpr int LDO = BN + 4;                 // floats of a row of results in LDS
  static constexpr int LDS = 2 * BUF > BM * LDO * 4 ? 2 * BUF : BM * LDO * 4;
};
template <class C>
__global__ __launch_bounds__(C::W * WAVE) void w4_tile_kernel(W4Args a) {
  constexpr int XT = C::XT, GROUP = C::GROUP, MT = C::MT, NBW = C::NBW, WM = C::WM, WN = C::WN, WK = C::WK, W = C::W;
  constexpr bool F16 = XT == W4_F16;
  constexpr int NP = C::NP, NG = C::NG, SG = GROUP / 32, E = XT == W4_F32 ? 4 : 2, NU = (C::UNITS + W - 1) / W;
  extern __shared__ char lds[];
  auto frag = [&](int buf, int unit, int p, int j) { return reinterpret_cast<uint4*>(lds + buf * C::BUF + unit * C::UNIT + (p * 4 + j) * (WAVE * 16)); };
  auto sums = [&](int buf, int unit, int g) { return reinterpret_cast<float*>(lds + buf * C::BUF + C::UNITS * C::UNIT + (unit * NG + g) * 64); };
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id();
  const int wk = w / (WM * WN), wm = w / WN % WM, wn = w % WN;
  const int nb0 = __builtin_amdgcn_readfirstlane((blockIdx.x * WN + wn) * NBW), m0 = blockIdx.y * C::BM, parts = gridDim.z;
  const int kb0 = (int)((int64_t)a.nkb * blockIdx.z / parts), kb1 = (int)((int64_t)a.nkb * (blockIdx.z + 1) / parts);
  const int rows = min(C::BM, a.M - m0), k_end = min(a.K, kb1 * W4_KB);
  const __amdgpu_buffer_rsrc_t xb =
      w4_buffer(a.x, (size_t)m0 * a.ldx * E, ((rows - 1) * (int64_t)a.ldx + (a.K + 7) / 8 * 8) * E);
  // (columns past the last: zero codes and scales)
  const int nbs = max(0, min(NBW, a.nnb - nb0));
  const size_t nbc = nbs ? nb0 : 0;
  const __amdgpu_buffer_rsrc_t qb = w4_buffer(a.q, nbc * a.nkb * 1024, (int64_t)nbs * a.nkb * 1024);
  const __amdgpu_buffer_rsrc_t sb = w4_buffer(a.meta, nbc * a.nkb * (NG * 64), (int64_t)nbs * a.nkb * (NG * 64));
  f4 tot[NBW][MT];
#pragma unroll
  for (int i = 0; i < NBW; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  struct Block {
    uint4 q[NBW];
    uint32_t sz[NBW][NG];
  };
  W4Raw<XT> xr[NU][4];
  // the wave's own block kb + wk of the weights, and its units of x of the blocks kb .. kb + WK - 1 (past the
  // part's last block: zeros of x); lane l takes rows l / 8 (+ 8) and k 8 (l % 8) (+ 64) of a unit
  uint32_t xoff[NU][4], qoff[NBW], soff[NBW];
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int unit = w + W * i;
#pragma unroll
    for (int j = 0; j < 4; ++j) {                    // rows 8 (j / 2) .., k 64 (j % 2) ..
      const int m = 16 * (unit % (MT * WM)) + (l >> 3) + 8 * (j / 2);
      xoff[i][j] = unit < C::UNITS && m < rows ? (uint32_t)(m * a.ldx + unit / (MT * WM) * W4_KB + 64 * (j % 2) + 8 * (l & 7)) * E : W4_OUT;
    }
  }
#pragma unroll
  for (int i = 0; i < NBW; ++i) {
    qoff[i] = (uint32_t)i * a.nkb * 1024 + 16 * l;
    soff[i] = (uint32_t)i * a.nkb * (NG * 64) + 4 * r;
  }
  // (past the end: as in w4_rows_kernel)
  auto load = [&](Block& o, int kb) __attribute__((always_inline)) {
    const uint32_t past = kb + wk < kb1 ? 0u : W4_OUT;
    const int at = min(kb, a.nkb - 1), qat = min(kb + wk, a.nkb - 1);
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = (w + W * i) / (MT * WM) * W4_KB + 64 * (j % 2) + 8 * (l & 7);
        xoff[i][j] = kb * W4_KB < k_end - k ? xoff[i][j] : W4_OUT;
#pragma unroll
        for (int v = 0; v < W4Raw<XT>::NV; ++v) xr[i][j].v[v] = w4_buffer16(xb, xoff[i][j] + 16 * v, at * (W4_KB * E));
      }
#pragma unroll
    for (int i = 0; i < NBW; ++i) {
      o.q[i] = w4_buffer16(qb, qoff[i] |= past, qat * 1024);
      soff[i] |= past;
#pragma unroll
      for (int g = 0; g < NG; ++g) o.sz[i][g] = w4_buffer4(sb, soff[i] + 64 * g, qat * (NG * 64));
    }
    __builtin_amdgcn_sched_barrier(0);               // issued here, not where they are used
  };
  // An operand's lane (row, c) lies at slot 16 c + (row ^ (c + 4 (step & 1))): eight lanes that hold a
  // row's 128 bytes then write to eight different banks, and a wave's reads are whole lines.
  auto stage = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int unit = w + W * i;
      if (C::UNITS % W && unit >= C::UNITS) continue;      // (uniform)
      const int ch = l & 7;
      float sum[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const W4Frag<XT> x = w4_frag<XT>(xr[i][j]);
        const int row = (l >> 3) + 8 * (j / 2);
#pragma unroll
        for (int p = 0; p < NP; ++p)
          frag(buf, unit, p, 0)[(2 * (j % 2) + (ch >> 2)) * WAVE + 16 * (ch & 3) + (row ^ ch)] = __builtin_bit_cast(uint4, x.p[p]);
        sum[j] = w4_sum8<XT>(xr[i][j]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = (l >> 3) + 8 * j;
        float s0 = sum[2 * j], s1 = sum[2 * j + 1];
        if constexpr (NG == 1) s0 += s1;
        s0 = w4_quad_sum(s0);
        if constexpr (NG > 1) s1 = w4_quad_sum(s1);
        if constexpr (NG <= 2) s0 += w4_dpp<0x141>(s0);
        if constexpr (NG == 2) s1 += w4_dpp<0x141>(s1);
        if constexpr (NG == 4) {
          if ((ch & 3) == 0) {
            sums(buf, unit, ch >> 2)[row] = s0;
            sums(buf, unit, 2 + (ch >> 2))[row] = s1;
          }
        } else if (ch == 0) {
          sums(buf, unit, 0)[row] = s0;
          if constexpr (NG == 2) sums(buf, unit, 1)[row] = s1;
        }
      }
    }
  };
  auto add = [&](const Block& o, int buf) __attribute__((always_inline)) {
    const int u0 = wk * (MT * WM) + wm * MT, slot = l ^ c;
    // operands of x in the order of their use, read AHEAD of it
    constexpr int STEPS = 4 * NP * MT, AHEAD = 4;
    auto read = [&](int i) __attribute__((always_inline)) {
      const int t = i % MT, p = i / MT % NP, j = i / (MT * NP);
      return __builtin_bit_cast(s8, frag(buf, u0 + t, p, j)[j & 1 ? slot ^ 4 : slot]);
    };
    s8 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = read(i);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f4 acc[NBW][MT];
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        const int j = g * SG + s;
        s8 op[NBW];
#pragma unroll
        for (int i = 0; i < NBW; ++i)
          op[i] = w4_operand<F16>(j == 0 ? o.q[i].x : j == 1 ? o.q[i].y : j == 2 ? o.q[i].z : o.q[i].w);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int at = (j * NP + p) * MT + t;
            const s8 xt = x[at % AHEAD];
#pragma unroll
            for (int i = 0; i < NBW; ++i) {
              if (s == 0 && p == 0) w4_mfma_first<F16>(acc[i][t], xt, op[i]);
              else w4_mfma<F16>(acc[i][t], xt, op[i]);
            }
            if (at + AHEAD < STEPS) x[at % AHEAD] = read(at + AHEAD);
            __builtin_amdgcn_sched_barrier(0x7f);    // (reads of LDS stay where they are)
          }
      }
      auto sum = [&](int t) __attribute__((always_inline)) { return *reinterpret_cast<const f4*>(sums(buf, u0 + t, g) + 4 * c); };
      f4 xs = sum(0);
      drain(acc[0][0]);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < NBW; ++i) w4_hold(acc[i][t]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const f4 next = sum(t + 1 < MT ? t + 1 : t);
#pragma unroll
        for (int i = 0; i < NBW; ++i) {
          const float s = bf16_val(o.sz[i][g] & 0xffffu), z = __uint_as_float(o.sz[i][g] & 0xffff0000u);
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[i][t][e] = fmaf(s, fmaf(-z, xs[e], acc[i][t][e]), tot[i][t][e]);
          w4_hold(tot[i][t]);                        // (before the next group's products: registers)
        }
        xs = next;
      }
    }
  };
  Block even, odd;
  int kb = kb0, buf = 0;
  load(even, kb);
  stage(0);
  __syncthreads();
  for (;;) {
    load(odd, kb + WK);
    add(even, buf);
    if ((kb += WK) >= kb1) break;
    stage(buf ^= 1);
    __syncthreads();
    load(even, kb + WK);
    add(odd, buf);
    if ((kb += WK) >= kb1) break;
    stage(buf ^= 1);
    __syncthreads();
  }
  // results through LDS, the waves along the sum one after the other, so that whole lines are written
  float* out = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int v = 0; v < WK; ++v) {
    __syncthreads();
    if (wk != v) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < NBW; ++i) {
          float& o = out[(16 * (wm * MT + t) + 4 * c + e) * C::LDO + 16 * (wn * NBW + i) + r];
          o = v ? o + tot[i][t][e] : tot[i][t][e];
        }
  }
  __syncthreads();
  const int n0 = blockIdx.x * C::BN;
  for (int x = threadIdx.x; x < C::BM * C::BN / 4; x += W * WAVE) {
    const int row = x / (C::BN / 4), col = 4 * (x % (C::BN / 4)), m = m0 + row, n = n0 + col;
    if (row >= rows || n >= a.N) continue;
    const float4 v = *reinterpret_cast<const float4*>(out + row * C::LDO + col);
    if (parts > 1) w4_part4(a, ((size_t)blockIdx.z * a.M + m) * a.N + n, n, v);
    else w4_out4<XT>(a, m, n, v);
  }
}

// Rows that 16-byte accesses cannot take, as rows that they can: ld elements, zero past K
template <typename T>
__global__ __launch_bounds__(256) void w4_align_kernel(const T* x, T* out, int K, size_t ldx, int ld) {
  const size_t m = blockIdx.x;
  for (int k = blockIdx.y * 256 + threadIdx.x; k < ld; k += 256 * gridDim.y) out[m * ld + k] = k < K ? x[m * ldx + k] : T(0);
}

// The parts of a sum, in order; four columns a thread
template <int XT>
__global__ __launch_bounds__(256) void w4_join_kernel(W4Args a, int parts) {
  const int cols = (a.N + 3) / 4, x = blockIdx.x * 256 + threadIdx.x, m = x / cols, n = 4 * (x - m * cols);
  if (m >= a.M) return;
  const size_t at = (size_t)m * a.N + n, step = (size_t)a.M * a.N;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.N % 4 == 0) {
#pragma unroll 8
    for (int p = 0; p < parts; ++p) v = add4(v, *reinterpret_cast<const float4*>(a.part + p * step + at));
  } else {
    float f[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < a.N) f[e] += a.part[p * step + at + e];
    v = make_float4(f[0], f[1], f[2], f[3]);
  }
  w4_out4<XT>(a, m, n, v);
}

// Many rows: bound by the matrix cores and by what the operands cost beside them, so nothing else is left in
// the loop.  A pass over x first (w4_prep_kernel) writes the groups' sums of x as operands, three
// bfloat16 pieces each, and where x's own rows cannot be read as they are (float32, odd strides, a last
// block that ends early) its 16-bit pieces as rows of whole blocks.  Then a workgroup of eight waves takes
// BM rows and 256 columns, a wave 16 MT rows and 64 columns: x comes into LDS by DMA, a block ahead of
// its use, the scale is one fma a group and result, and the zeros are a product of their own behind the
// sum, (sums of x) x (-s z) over the groups, 32 groups a step: s z has 16 bits, two pieces.
//   2048 rows of 4096 x 4096: 76 us bfloat16 and float16, 905 TFLOP/s (a large library product of bfloat16
// 1219), of that the pass over x 4; float32, three products each, 188.  With parts of the loop left out: products alone 55, without the DMA 64, without the
// scaling 70, without the conversions 74, without the products 59.  Zeros in the scaling instead of a product,
// x staged through registers as in w4_tile_kernel: 112.
template <int XT_, int GROUP_>
struct W4Gemm {
  static constexpr int XT = XT_, GROUP = GROUP_, NP = W4Frag<XT>::NP;
  static constexpr int WM = 2, WN = 4, MT = XT == W4_F32 ? 2 : 4, NBW = 4;
  static constexpr int BM = 16 * MT * WM, BN = 16 * NBW * WN, LDO = BN + 4;
  // a block's x, codes and scales in LDS, NBUF blocks in turn (float32: as many as fit)
  static constexpr int NBUF = XT == W4_F32 ? 2 : 3, NG = W4_KB / GROUP;
  static constexpr int XB = NP * BM * W4_KB * 2, QB = BN / 16 * 1024, BUF = XB + QB + NG * 1024;
  static constexpr int LDS = NBUF * BUF > BM * LDO * 4 ? NBUF * BUF : BM * LDO * 4;
};
struct W4GemmArgs {
  const uint16_t *x, *sums;     // NP planes of rows of ld elements; w4_sums_bytes
  size_t ld, plane;
  int ngb;                      // steps of 32 groups
};

// A wave a row: sums of the groups, and with planes (x's 16-bit pieces, Kp columns, zero past K)
template <int XT, int GROUP>
__global__ __launch_bounds__(256) void w4_prep_kernel(W4Args a, uint16_t* planes, uint16_t* sums, int ngb) {
  constexpr int NP = W4Frag<XT>::NP, LG = GROUP / 8;          // lanes of a group
  const int l = lane_id(), m = blockIdx.x * 4 + wave_id(), Kp = a.nkb * W4_KB, mt = (a.M + 15) / 16;
  if (m >= a.M) return;
  for (int k = 8 * (l + WAVE * (int)blockIdx.y); k < ngb * 32 * GROUP; k += 8 * WAVE * gridDim.y) {
    W4Raw<XT> x;
    if (a.vec && k < a.K) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(a.x) + ((size_t)m * a.ldx + k) * (XT == W4_F32 ? 4 : 2));
#pragma unroll
      for (int v = 0; v < W4Raw<XT>::NV; ++v) x.v[v] = p[v];
    } else {
      x = w4_load_odd<XT>(a, k < a.K ? m : a.M, k);
    }
    if (planes && k < Kp) {
      const W4Frag<XT> f = w4_frag<XT>(x);
#pragma unroll
      for (int p = 0; p < NP; ++p)                   // (the largest piece last, as in W4Frag)
        *reinterpret_cast<uint4*>(planes + ((size_t)p * a.M + m) * Kp + k) = __builtin_bit_cast(uint4, f.p[p]);
    }
    float s = w4_quad_sum(w4_sum8<XT>(x));
    if constexpr (LG >= 8) s += w4_dpp<0x141>(s);    // the other quad of eight lanes,
    if constexpr (LG >= 16) s += w4_dpp<0x128>(s);   // the other eight of sixteen
    if (l % LG == 0) {
      const int g = k / GROUP, gb = g / 32, gi = g % 32;
      const float h = w4_top(s), r = s - h;
      const uint32_t piece[3] = {__float_as_uint(r - w4_top(r)), __float_as_uint(r), __float_as_uint(h)};
#pragma unroll
      for (int p = 0; p < 3; ++p)
        sums[(((size_t)p * mt + m / 16) * ngb + gb) * 512 + (m % 16 + 16 * (gi / 8)) * 8 + gi % 8] = (uint16_t)(piece[p] >> 16);
    }
  }
}

template <class C>
__global__ __launch_bounds__(512) void w4_gemm_kernel(W4Args a, W4GemmArgs b) {
  constexpr int XT = C::XT, GROUP = C::GROUP, MT = C::MT, NBW = C::NBW, WN = C::WN, NP = C::NP;
  constexpr bool F16 = XT == W4_F16;
  constexpr int NG = C::NG, SG = GROUP / 32, RO = C::BM / 8, DMA = NP * RO * 2 / 8;     // octets of rows, a wave's DMAs of x
  extern __shared__ char lds[];
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), wm = w / WN, wn = w % WN;
  const int tb0 = blockIdx.x * (C::BN / 16), nb0 = tb0 + wn * NBW, m0 = blockIdx.y * C::BM;
  // A KB of x in LDS holds eight rows' 64 k: lane l's sixteen bytes are row l / 8's chunk (l % 8) ^ (l / 8), so
  // that rows come as whole lines and a wave's reads of an operand meet no bank twice.  (Rows and columns
  // past the last: the last again, and not looked at.)
  const char *src[DMA], *qsrc[2];
#pragma unroll
  for (int i = 0; i < DMA; ++i) {
    const int u = w * DMA + i, p = u / (2 * RO), ro = u / 2 % RO, h = u % 2;
    const int m = min(m0 + 8 * ro + (l >> 3), a.M - 1);
    src[i] = reinterpret_cast<const char*>(b.x + p * b.plane + (size_t)m * b.ld + 64 * h + 8 * ((l & 7) ^ (l >> 3)));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    qsrc[i] = reinterpret_cast<const char*>(a.q) + (size_t)min(tb0 + 2 * w + i, a.nnb - 1) * a.nkb * 1024 + 16 * l;
  // (sixteen columns' words of a group are 64 bytes; a wave fetches group w % NG of the block)
  const char* ssrc = reinterpret_cast<const char*>(a.meta) +
                     ((size_t)min(tb0 + (l >> 2), a.nnb - 1) * a.nkb * NG + w % NG) * 64 + 16 * (l & 3);
  auto dma = [&](const char* from, int to) __attribute__((always_inline)) {
    lds_dma16(reinterpret_cast<const float*>(from), reinterpret_cast<float*>(lds + to));
  };
  constexpr int DMAS = DMA + 3;
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < DMA; ++i) dma(src[i] + (size_t)kb * (2 * W4_KB), buf + (w * DMA + i) * 1024);
#pragma unroll
    for (int i = 0; i < 2; ++i) dma(qsrc[i] + (size_t)kb * 1024, buf + C::XB + (2 * w + i) * 1024);
    dma(ssrc + (size_t)kb * (NG * 64), buf + C::XB + C::QB + w % NG * 1024);
  };
  f4 tot[NBW][MT];
#pragma unroll
  for (int i = 0; i < NBW; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  // where the lane's operands lie in a KB, for the steps 0 | 2 and 1 | 3
  const int at0 = (r & 7) * 128 + (c ^ (r & 7)) * 16, at1 = (r & 7) * 128 + ((c + 4) ^ (r & 7)) * 16;
  auto add = [&](int buf) __attribute__((always_inline)) {
    constexpr int STEPS = 4 * NP * MT, AHEAD = 2;
    static_assert(NBW == 4 && NP * MT >= NBW, "a step of the sum leaves room for the next one's operands");
    auto read = [&](int i) __attribute__((always_inline)) {
      const int t = i % MT, p = i / MT % NP, j = i / (MT * NP);
      return *reinterpret_cast<const s8*>(lds + buf + ((p * RO + 2 * (wm * MT + t) + (r >> 3)) * 2 + j / 2) * 1024 + (j & 1 ? at1 : at0));
    };
    uint4 q[NBW];
#pragma unroll
    for (int i = 0; i < NBW; ++i) q[i] = *reinterpret_cast<const uint4*>(lds + buf + C::XB + (wn * NBW + i) * 1024 + 16 * l);
    auto word = [&](int i, int j) __attribute__((always_inline)) {
      return w4_operand<F16>(j == 0 ? q[i].x : j == 1 ? q[i].y : j == 2 ? q[i].z : q[i].w);
    };
    s8 x[AHEAD], op[2][NBW];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = read(i);
#pragma unroll
    for (int i = 0; i < NBW; ++i) op[0][i] = word(i, 0);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f4 acc[NBW][MT];
#pragma unroll
      for (int s = 0; s < SG; ++s) {
        const int j = g * SG + s;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const int i = p * MT + t, at = j * NP * MT + i;
            const s8 xt = x[at % AHEAD];
            const s8* w4 = op[j % 2];
            if (s == 0 && p == 0) w4_mfma4<F16, true>(acc[0][t], acc[1][t], acc[2][t], acc[3][t], xt, w4[0], w4[1], w4[2], w4[3]);
            else w4_mfma4<F16, false>(acc[0][t], acc[1][t], acc[2][t], acc[3][t], xt, w4[0], w4[1], w4[2], w4[3]);
            // beside the products: the operands of the next step of the sum, one column block's at a time
            if (at + AHEAD < STEPS) x[at % AHEAD] = read(at + AHEAD);
            if (j < 3 && i < NBW) op[(j + 1) % 2][i] = word(i, j + 1);
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      drain(acc[0][0]);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < NBW; ++i) w4_hold(acc[i][t]);
#pragma unroll
      for (int i = 0; i < NBW; ++i) {
        const float s = __uint_as_float(*reinterpret_cast<const uint32_t*>(lds + buf + C::XB + C::QB + g * 1024 + (wn * NBW + i) * 64 + 4 * r) << 16);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[i][t][e] = fmaf(s, acc[i][t][e], tot[i][t][e]);
          w4_hold(tot[i][t]);
        }
      }
    }
  };
  // Block kb has come when only the DMAs of the NBUF - 2 behind it are under way; then everyone's has.  (Past
  // the end the last block again, so that the counts stay the same.)
  constexpr int BEHIND = (C::NBUF - 2) * DMAS;
  static_assert(BEHIND < 16, "vmcnt's low bits");
  const int last = a.nkb - 1;
  int buf = 0, into = (C::NBUF - 1) * C::BUF;
  auto next = [&](int x) { return x == (C::NBUF - 1) * C::BUF ? 0 : x + C::BUF; };
#pragma unroll
  for (int i = 0; i < C::NBUF - 1; ++i) fetch(min(i, last), i * C::BUF);
  for (int kb = 0; kb <= last; ++kb) {
    __builtin_amdgcn_s_waitcnt(WAIT_VMCNT0 | BEHIND);
    __syncthreads();
    fetch(min(kb + C::NBUF - 1, last), into);
    add(buf);
    buf = next(buf);
    into = next(into);
  }
  __builtin_amdgcn_s_waitcnt(WAIT_VMCNT0);           // (LDS is used again below)
  // the zeros
  const int mtiles = (a.M + 15) / 16, nbs = max(0, min(NBW, a.nnb - nb0));
  const __amdgpu_buffer_rsrc_t sb = w4_buffer(a.meta, (size_t)(nbs ? nb0 : 0) * a.nkb * (NG * 64), (int64_t)nbs * a.nkb * (NG * 64));
  for (int gb = 0; gb < b.ngb; ++gb) {
    s8 z[NBW][2];
#pragma unroll
    for (int i = 0; i < NBW; ++i) {
      uint32_t lo[8], hi[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // (groups past the last: meta ends at the columns' last block, and may go on with the next columns')
        const int g = gb * 32 + 8 * c + e;
        const uint32_t off = g < a.nkb * NG ? (uint32_t)((i * a.nkb * NG + g) * 64 + 4 * r) : W4_OUT;
        const uint32_t sz = w4_buffer4(sb, off, 0);
        const float v = -(bf16_val(sz & 0xffffu) * __uint_as_float(sz & 0xffff0000u));
        hi[e] = __float_as_uint(v) >> 16;
        lo[e] = __float_as_uint(v - w4_top(v)) >> 16;
      }
      z[i][0] = __builtin_bit_cast(s8, make_uint4(lo[0] | lo[1] << 16, lo[2] | lo[3] << 16, lo[4] | lo[5] << 16, lo[6] | lo[7] << 16));
      z[i][1] = __builtin_bit_cast(s8, make_uint4(hi[0] | hi[1] << 16, hi[2] | hi[3] << 16, hi[4] | hi[5] << 16, hi[6] | hi[7] << 16));
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const size_t mt = min(m0 / 16 + wm * MT + t, mtiles - 1);
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const s8 x = *reinterpret_cast<const s8*>(b.sums + (((size_t)p * mtiles + mt) * b.ngb + gb) * 512 + 8 * l);
#pragma unroll
        for (int i = 0; i < NBW; ++i) {
          w4_mfma<false>(tot[i][t], x, z[i][0]);
          w4_mfma<false>(tot[i][t], x, z[i][1]);
        }
      }
    }
  }
  drain(tot[0][0]);
#pragma unroll
  for (int i = 0; i < NBW; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) w4_hold(tot[i][t]);
  // results through LDS, so that whole lines are written
  float* out = reinterpret_cast<float*>(lds);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < NBW; ++i) out[(16 * (wm * MT + t) + 4 * c + e) * C::LDO + 16 * (wn * NBW + i) + r] = tot[i][t][e];
  __syncthreads();
  const int n0 = blockIdx.x * C::BN, rows = min(C::BM, a.M - m0);
  for (int x = threadIdx.x; x < C::BM * C::BN / 4; x += 512) {
    const int row = x / (C::BN / 4), col = 4 * (x % (C::BN / 4)), n = n0 + col;
    if (row >= rows || n >= a.N) continue;
    w4_out4<XT>(a, m0 + row, n, *reinterpret_cast<const float4*>(out + row * C::LDO + col));
  }
}

// How a product runs: parts 0: rows; else tiles, the sum in parts.
//   rows: one launch, x and (over 16 rows) the weights read again by each tile of rows.  Up to 8 rows
//     always; more where the weights come from the caches again, 2^15 tiles of 16 rows and 128 x 16
//     weights, and the sum is not long beside the columns (bfloat16, us, rows against tiles: 64 rows of
//     2048 x 2048 5.7, 8.8; 64 of 4096 x 4096 11.8, 11.7; 128 of 4096 x 4096 20.7, 15.1; 16 of
//     4096 x 14336 12.5, 14.5; 16 of 14336 x 4096 16.8, 13.2).  Not measured against tiles: float32, and more
//     than 128 rows of small matrices (2048 float32 rows of 768 x 512 29.8 us, of 1024 x 512 32.6).
//   parts: two workgroups a CU where that leaves 14 blocks of 128 or more to each, else one, with
//     four blocks at least (64 rows of 14336 x 4096, 1 / 4 / 8 / 16 parts: 74, 25, 21, 27; 256 of
//     4096 x 4096, 1 / 2: 21.8, 23.5).
//   -1: many rows, w4_gemm_kernel, from three workgroups for four CUs on (bfloat16, us, against tiles: 2048
//     rows of 4096 x 4096 77, 103; 1024 72, 55; 512 of 4096 x 14336 73, 92; 512 of 14336 x 4096 228, 95) and
//     more than half a tile of rows, since it multiplies whole ones (rows of 4096 x 131072: 16 133, 66; 64
//     138, 131; 96 146, 190; 256 306, 487; float32, tiles of 64, 4096 x 50257: 32 83, 68; 64 89, 133).
template <int XT, int GROUP>
using W4Tiles = W4Tile<XT, GROUP, 2, 2, 1, 4, 2>;
static bool w4_many(int dtype, int M, int nnb) {
  const int bm = dtype == W4_F32 ? W4Gemm<W4_F32, 128>::BM : W4Gemm<W4_BF16, 128>::BM, bn = W4Gemm<W4_BF16, 128>::BN;
  return M > bm / 2 && (int64_t)((M + bm - 1) / bm) * ((16 * nnb + bn - 1) / bn) * 4 >= (int64_t)cu_count() * 3;
}
static int w4_parts(int dtype, int M, int nkb, int nnb) {
  using C = W4Tiles<W4_BF16, 128>;
  if (M <= 8 || (nkb <= 64 && (int64_t)nkb * nnb * ((M + 15) / 16) <= 32768)) return 0;
  const int64_t tiles = (int64_t)((16 * nnb + C::BN - 1) / C::BN) * ((M + C::BM - 1) / C::BM), cus = cu_count();
  if (w4_many(dtype, M, nnb)) return -1;
  const int64_t two = 2 * cus / tiles, one = cus / tiles;
  const int64_t p = two >= 1 && nkb / two >= 14 ? two : one < nkb / 4 ? one : nkb / 4;
  return p < 1 ? 1 : (int)p;
}

static size_t w4_align_bytes(int dtype, const W4Args& a) {
  return a.vec ? 0 : ((size_t)a.M * ((a.K + 7) / 8 * 8) * (dtype == W4_F32 ? 4 : 2) + 255) / 256 * 256;
}
static int w4_ngb(int group, const W4Args& a) { return (a.nkb * (W4_KB / group) + 31) / 32; }
static size_t w4_sums_bytes(int group, const W4Args& a) { return (size_t)3 * ((a.M + 15) / 16) * w4_ngb(group, a) * 1024; }
// whether w4_gemm_kernel can read x's own rows
static bool w4_direct(int dtype, const W4Args& a) { return dtype != W4_F32 && a.vec && a.K % W4_KB == 0; }
size_t w4_workspace_bytes(int dtype, int group, const W4Args& a) {
  const int parts = w4_parts(dtype, a.M, a.nkb, a.nnb);
  if (parts < 0)
    return w4_sums_bytes(group, a) + (w4_direct(dtype, a) ? 0 : (size_t)(dtype == W4_F32 ? 3 : 1) * a.M * a.nkb * W4_KB * 2);
  return parts ? w4_align_bytes(dtype, a) + (parts > 1 ? (size_t)parts * a.M * a.N * 4 : 0) : 0;
}

template <int XT, int GROUP, int SP, int NB>
static void w4_rows(const W4Args& a, hipStream_t s) {
  constexpr int most = w4_waves(XT, NB);
  const int W = a.nkb < most ? a.nkb : most;
  const dim3 grid((a.nnb + NB - 1) / NB, (a.M + 16 / SP - 1) / (16 / SP));
  hipLaunchKernelGGL((w4_rows_kernel<XT, GROUP, SP, NB>), grid, dim3(W * WAVE), (size_t)W * NB * (4 / SP) * WAVE * 4, s, a);
}

template <int XT, int GROUP>
static void w4_go(W4Args a, hipStream_t s) {
  const int parts = w4_parts(XT, a.M, a.nkb, a.nnb);
  if (parts == 0) {
    // two columns' blocks a wave where two workgroups a CU are left (one row of 4096 x 14336 float32:
    // 14.6 -> 11.8 us, 16 of 4096 x 11008 14.7 -> 12.5; one of 4096 x 4096 4.5 -> 5.1)
    const bool two = (int64_t)a.nnb * ((a.M + 15) / 16) >= 2 * cu_count();
    if (a.M <= 4) two ? w4_rows<XT, GROUP, 4, 2>(a, s) : w4_rows<XT, GROUP, 4, 1>(a, s);
    else if (a.M <= 8) two ? w4_rows<XT, GROUP, 2, 2>(a, s) : w4_rows<XT, GROUP, 2, 1>(a, s);
    else two ? w4_rows<XT, GROUP, 1, 2>(a, s) : w4_rows<XT, GROUP, 1, 1>(a, s);
    return;
  }
  if (parts < 0) {
    using C = W4Gemm<XT, GROUP>;
    W4GemmArgs b{};
    b.ngb = w4_ngb(GROUP, a);
    uint16_t* sums = reinterpret_cast<uint16_t*>(a.part);
    uint16_t* planes = w4_direct(XT, a) ? nullptr : sums + w4_sums_bytes(GROUP, a) / 2;
    b.sums = sums;
    b.x = planes ? planes : static_cast<const uint16_t*>(a.x);
    b.ld = planes ? (size_t)a.nkb * W4_KB : a.ldx;
    b.plane = (size_t)a.M * b.ld;
    hipLaunchKernelGGL((w4_prep_kernel<XT, GROUP>), dim3((a.M + 3) / 4, (b.ngb * GROUP + 31) / 32), dim3(256), 0, s, a, planes, sums, b.ngb);
    hipLaunchKernelGGL((w4_gemm_kernel<C>), dim3((a.N + C::BN - 1) / C::BN, (a.M + C::BM - 1) / C::BM), dim3(512), C::LDS, s, a, b);
    return;
  }
  if (!a.vec) {
    using T = std::conditional_t<XT == W4_F32, uint32_t, uint16_t>;
    const int ld = (a.K + 7) / 8 * 8;
    T* x = reinterpret_cast<T*>(a.part);
    a.part = reinterpret_cast<float*>(reinterpret_cast<char*>(a.part) + w4_align_bytes(XT, a));
    hipLaunchKernelGGL((w4_align_kernel<T>), dim3(a.M, ld < 2048 ? 1 : ld / 1024 < 64 ? ld / 1024 : 64), dim3(256), 0, s,
                       static_cast<const T*>(a.x), x, a.K, a.ldx, ld);
    a.x = x;
    a.ldx = ld;
  }
  using C = W4Tiles<XT, GROUP>;
  const dim3 grid((a.N + C::BN - 1) / C::BN, (a.M + C::BM - 1) / C::BM, parts);
  hipLaunchKernelGGL((w4_tile_kernel<C>), grid, dim3(C::W * WAVE), C::LDS, s, a);
  if (parts > 1)
    hipLaunchKernelGGL((w4_join_kernel<XT>), dim3(((int64_t)a.M * ((a.N + 3) / 4) + 255) / 256), dim3(256), 0, s, a, parts);
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
