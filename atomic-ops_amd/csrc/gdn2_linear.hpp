// Kernels of gdn2_linear.hip, instantiated for each type in a translation unit of its own (gdn2_linear_*.hip).
// Products with an epilogue, on gfx950: y = act(A B + bias) + residual, where a layer's forward pass and its two
// gradients differ in how the operands lie in memory (include/gdn2.h, gdn2_product).
//
// The matrix cores take operands whose lanes hold eight consecutive values along the sum.  An operand whose rows run
// along the sum (x; W and dz for the input's gradient) is read from LDS as it is.  One whose rows run across it (W of a
// layer; x and dz for the weight's gradient) lies in LDS as in memory and is transposed on its way to the registers
// (ds_read_b64_tr_b16), so that no pass over memory turns a matrix around.
//
// What takes a product (the rules, with both sides measured, are in gdn2_linear.hip):
//   lin_tile_kernel     tiles of 256 x 256 (float32 256 x 128), 128 x 128 or 64 x 64, operands into LDS by DMA a block ahead of
//                       their use, sums in parts where there are few tiles; float32 as three bfloat16 pieces, six
//                       products.  Bound by the matrix cores: 8192 x 4096 x 4096 bfloat16 215 to 232
//                       us by card, 1.18 to 1.28 PFLOP/s; 4096^3 float32 647 to 671, 205 to 212 TFLOP/s (a library product on
//                       the float32 matrix cores 917).  Each tile's epilogue waits for its products: with bias,
//                       activation, z and residual 260.  CUT:
//                       float32 stays as it is up to LDS and each wave cuts what it reads, no pass over memory before it:
//                       218 x 8192 x 7680 181 to 188 us (the library 208 to 216), 4096 x 2048 x 1024 103 (by a pass 128, the
//                       library 119);
//   lin_direct_kernel   small float32 products: 2048 x 768 x 512 21 us (the library's 18), 512^3 10.6 (17), bound by what
//                       its small tiles draw from the caches;
//   lin_rows_kernel, lin_columns_kernel, lin_dots_kernel   up to 8 rows, bound by W's bytes: one row of 4096 x 14336 bfloat16
//                       21.8 us, 5.4 TB/s.
#pragma once
#include "gdn2_kernels.hpp"

namespace gdn2 {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef s4 __attribute__((address_space(3)))* lds_s4;
constexpr int LIN_NONE = 0, LIN_SILU = 1, LIN_GELU = 2, LIN_TANH = 3;

template <int DT>
struct LinType {
  using T = std::conditional_t<DT == LIN_F32, float, std::conditional_t<DT == LIN_BF16, uint16_t, _Float16>>;
  static __device__ __forceinline__ float get(const void* p, size_t i) {
    if constexpr (DT == LIN_BF16) return bf16_val(static_cast<const uint16_t*>(p)[i]);
    else return (float)static_cast<const T*>(p)[i];
  }
  static __device__ __forceinline__ void put(void* p, size_t i, float v) {
    if constexpr (DT == LIN_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)bf16_bits(v);
    else static_cast<T*>(p)[i] = (T)v;
  }
  static __device__ __forceinline__ float4 get4(const void* p, size_t i) {
    if constexpr (DT == LIN_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
    if constexpr (DT == LIN_BF16)
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xffff0000u));
    const h2v a = __builtin_bit_cast(h2v, u.x), b = __builtin_bit_cast(h2v, u.y);
    return make_float4((float)a[0], (float)a[1], (float)b[0], (float)b[1]);
  }
  static __device__ __forceinline__ void put4(void* p, size_t i, const float4& v) {
    if constexpr (DT == LIN_F32) *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
    else if constexpr (DT == LIN_BF16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(bf16_pack(v.x, v.y), bf16_pack(v.z, v.w));
    else {
      const h2v a = {(_Float16)v.x, (_Float16)v.y}, b = {(_Float16)v.z, (_Float16)v.w};
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) = make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    }
  }
};
template <int DT>
struct LinVec {                                          // 16 bytes
  static constexpr int E = DT == LIN_F32 ? 4 : 8;
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
  static __device__ __forceinline__ void store8(void* p, size_t at, const float* x) {
    if constexpr (DT == LIN_F32) {
      float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
      q[0] = make_float4(x[0], x[1], x[2], x[3]);
      q[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == LIN_BF16) w[i] = bf16_pack(x[2 * i], x[2 * i + 1]);
        else {
          const h2v h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
          w[i] = __builtin_bit_cast(uint32_t, h);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  // N values from p[at] on, those before `end` (VEC: all, 16-byte aligned)
  template <int N, bool VEC>
  static __device__ __forceinline__ void load(const void* p, size_t at, int left, float* x) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < N; i += E)
        widen(*reinterpret_cast<const uint4*>(static_cast<const typename LinType<DT>::T*>(p) + at + i), x + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = LinType<DT>::get(p, at + min(i, left - 1));      // (no branch: the loads go together)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = i < left ? x[i] : 0.f;
    }
  }
};
// Four neighbouring values of a matrix as they are, aligned to themselves alone (a row of an odd stride starts anywhere): the
// types say so, and gfx950 reads 16 or 8 bytes from such places at once.
typedef uint32_t lin_u4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t lin_u2 __attribute__((ext_vector_type(2), aligned(2)));
template <bool F32>
__host__ __device__ __forceinline__ void lin_four(const void* src, size_t at, uint32_t* v) {
  if constexpr (F32) {
    const lin_u4 u = *reinterpret_cast<const lin_u4*>(static_cast<const uint32_t*>(src) + at);
    v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
  } else {
    const lin_u2 u = *reinterpret_cast<const lin_u2*>(static_cast<const uint16_t*>(src) + at);
    v[0] = u.x & 0xffffu; v[1] = u.x >> 16; v[2] = u.y & 0xffffu; v[3] = u.y >> 16;
  }
}

// by a type known at run time (wave-uniform)
__device__ __forceinline__ float lin_get(int dt, const void* p, size_t i) {
  return dt == LIN_F32 ? LinType<LIN_F32>::get(p, i) : dt == LIN_BF16 ? LinType<LIN_BF16>::get(p, i) : LinType<LIN_F16>::get(p, i);
}
__device__ __forceinline__ void lin_put(int dt, void* p, size_t i, float v) {
  if (dt == LIN_F32) LinType<LIN_F32>::put(p, i, v);
  else if (dt == LIN_BF16) LinType<LIN_BF16>::put(p, i, v);
  else LinType<LIN_F16>::put(p, i, v);
}
__device__ __forceinline__ float4 lin_get4(int dt, const void* p, size_t i) {
  return dt == LIN_F32 ? LinType<LIN_F32>::get4(p, i) : dt == LIN_BF16 ? LinType<LIN_BF16>::get4(p, i) : LinType<LIN_F16>::get4(p, i);
}
__device__ __forceinline__ void lin_put4(int dt, void* p, size_t i, const float4& v) {
  if (dt == LIN_F32) LinType<LIN_F32>::put4(p, i, v);
  else if (dt == LIN_BF16) LinType<LIN_BF16>::put4(p, i, v);
  else LinType<LIN_F16>::put4(p, i, v);
}

// ---- activations: z s(u), s the logistic function, with u = z, 1.5958 (z + 0.044715 z^3), or gelu's z Phi(z).  The
// tanh form 0.5 (1 + tanh(u / 2)) is s(u), which does not cancel where tanh goes to -1.
constexpr float LIN_TANH_C = 1.5957691216f;       // 2 sqrt(2 / pi)
// (the hardware's reciprocal: an error of one unit of the last place, and a sixth of a division)
__device__ __forceinline__ float lin_logistic(float u) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.44269504088896341f)); }
template <int ACT>
__device__ __forceinline__ float lin_act(float z) {
  if constexpr (ACT == LIN_SILU) return z * lin_logistic(z);
  else if constexpr (ACT == LIN_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  else if constexpr (ACT == LIN_TANH) return z * lin_logistic(LIN_TANH_C * (z + 0.044715f * z * z * z));
  else return z;
}
// (far out a slope is 0 or 1, and its terms 0 times an infinity: as a factor z goes no further than where that is so.  float16
// keeps a z beyond 65504 as an infinity.  NaN stays NaN by the other factors.)
template <int ACT>
__device__ __forceinline__ float lin_slope(float z) {
  const float near = __builtin_amdgcn_fmed3f(z, -1e18f, 1e18f);
  if constexpr (ACT == LIN_SILU) {
    const float s = lin_logistic(z);
    return s * (1.f + near * (1.f - s));
  } else if constexpr (ACT == LIN_GELU) {
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + near * 0.39894228040143268f * __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  } else if constexpr (ACT == LIN_TANH) {
    const float s = lin_logistic(LIN_TANH_C * (z + 0.044715f * z * z * z));
    return s + near * s * (1.f - s) * (LIN_TANH_C * (1.f + 0.134145f * near * near));
  } else {
    return 1.f;
  }
}

// ---- the product --------------------------------------------------------------------------------------------------

// Operands of lane l in a 32-deep product: eight values along the sum (group l / 16) of row or column l % 16.
template <bool F16>
__device__ __forceinline__ void lin_mfma4(f4& a0, f4& a1, f4& a2, f4& a3, const s8& n0, const s8& n1, const s8& n2, const s8& n3, const s8& m) {
#define LIN_FOUR(op)                                                                                       \
  "s_nop 1\n\t" op " %0, %4, %8, %0\n\t" op " %1, %5, %8, %1\n\t" op " %2, %6, %8, %2\n\t" op " %3, %7, %8, %3"
  if constexpr (F16)
    asm volatile(LIN_FOUR("v_mfma_f32_16x16x32_f16") : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3) : "v"(n0), "v"(n1), "v"(n2), "v"(n3), "v"(m));
  else
    asm volatile(LIN_FOUR("v_mfma_f32_16x16x32_bf16") : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3) : "v"(n0), "v"(n1), "v"(n2), "v"(n3), "v"(m));
#undef LIN_FOUR
}
__device__ __forceinline__ void lin_hold(f4& a) { asm volatile("" : "+v"(a)); }

// An operand as the kernels read it: 16-bit rows of ld elements, 16-byte aligned; planes of float32's pieces
struct LinOperand {
  const uint16_t* p;
  size_t ld, plane;
  int rows;              // across the sum: M or N; of a matrix whose rows run across it, a multiple of 8
};
struct LinArgs {
  LinOperand a, b;
  int M, N, K;           // K: up to the last whole value of the sum
  int mt, nt, parts, per;        // tiles; parts of the sum, of `per` blocks each
  int out_dtype, bias_dtype, z_dtype, vec, pairs;       // how results are written: lin_out8, lin_out_pairs
  int sums, halves;        // float32 sums go to `part`, to be joined: of parts, or of the two halves of a's rows
  size_t ldr;
  const void *bias, *residual;
  void *y, *z;
  float* part;
};

static __device__ uint4 lin_zeros;      // what lies past the end of a sum

// s_waitcnt: all but the last n of the wave's DMAs
constexpr int lin_wait(int n) { return WAIT_VMCNT0 | (n & 15) | n >> 4 << 14; }
// lds_dma16 for four bytes a lane (global_load_lds_dword), at dst + i floats
__device__ __forceinline__ void lin_dma4(const float* src, float* dst) {
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float*)dst;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}
// float32 as it is: blocks of 32 along the sum, by W waves' DMAs of 16 bytes a lane (WIDE: rows that take them) or of 4.
// In LDS, in chunks of four values:
//   rows along the sum (8 chunks): chunk c of row r at c ^ (r & 7);
//   rows across it (ROWS / 4): chunk c of value k at c ^ 4 (k / 4 & 3), so that the lanes of a read, which take k = 4 c + j
//   for c = 0 .. 3 of sixteen rows each, meet no bank twice.
template <bool R, int ROWS, int W, bool WIDE>
struct LinFloats {
  static constexpr int E = WIDE ? 4 : 1, D = ROWS * 32 / (64 * E * W);
  const char* src[D];
  int k[D];
  size_t step;
  __device__ __forceinline__ void init(const LinOperand& o, int row0, int kb0) {
    const float* p = reinterpret_cast<const float*>(o.p);
    step = (R ? 32 * o.ld : (size_t)32) * 4;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int f = ((wave_id() * D + i) * 64 + lane_id()) * E, q = f >> 2, e = f & 3;
      size_t at;
      if constexpr (R) {
        k[i] = q / (ROWS / 4);
        const int chunk = (q & (ROWS / 4 - 1)) ^ ((k[i] >> 2 & 3) << 2);
        at = (size_t)k[i] * o.ld + min(row0 + 4 * chunk + e, o.rows - E);
      } else {
        const int row = q >> 3;
        k[i] = 4 * ((q & 7) ^ (row & 7)) + e;
        at = (size_t)min(row0 + row, o.rows - 1) * o.ld + k[i];
      }
      src[i] = reinterpret_cast<const char*>(p + at) + (size_t)kb0 * step;
      k[i] += kb0 * 32;
    }
  }
  __device__ __forceinline__ void fetch(char* dst, int K, bool tail) {
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const char* s = src[i];
      if (tail) s = k[i] < K ? s : reinterpret_cast<const char*>(&lin_zeros);
      float* to = reinterpret_cast<float*>(dst) + (wave_id() * D + i) * 64 * E;
      if constexpr (WIDE) lds_dma16(reinterpret_cast<const float*>(s), to);
      else lin_dma4(reinterpret_cast<const float*>(s), to);
      src[i] += step;
      k[i] += 32;
    }
  }
};
// A lane's values of tile t (16 rows) and of sixteen along the sum, s of two: 4 c .. 4 c + 3, c = lane / 16
template <bool R, int ROWS>
__device__ __forceinline__ float4 lin_floats(const char* lds, int t, int s) {
  const int l = lane_id(), r = l & 15, c = l >> 4;
  if constexpr (R) {
    const float* p = reinterpret_cast<const float*>(lds) + (16 * s + 4 * c) * ROWS + 16 * (t ^ c) + r;
    return make_float4(p[0], p[ROWS], p[2 * ROWS], p[3 * ROWS]);
  } else {
    const int row = 16 * t + r;
    return *reinterpret_cast<const float4*>(lds + row * 128 + (((4 * s + c) ^ (row & 7)) << 4));
  }
}
// Both s of a tile as the three pieces of the whole block's operand, each the next eight bits.  The pieces behind the first are
// below 2^-7 and 2^-15 of the value, so the three products of pieces that are not formed are below 2^-21 of a product, and of its
// sign.  (An infinity leaves NaN.)
template <bool R, int ROWS>
__device__ __forceinline__ void lin_cut(const char* lds, int t, s8& hi, s8& mid, s8& lo) {
  const float4 x = lin_floats<R, ROWS>(lds, t, 0), y = lin_floats<R, ROWS>(lds, t, 1);
  float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  uint32_t piece[3][4];
#pragma unroll
  for (int p = 0; p < 3; ++p)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t a = __float_as_uint(f[e]), b = __float_as_uint(f[e + 1]);
      piece[p][e / 2] = __builtin_amdgcn_perm(b, a, 0x07060302);
      f[e] -= __uint_as_float(a & 0xffff0000u);
      f[e + 1] -= __uint_as_float(b & 0xffff0000u);
    }
  hi = __builtin_bit_cast(s8, piece[0]);
  mid = __builtin_bit_cast(s8, piece[1]);
  lo = __builtin_bit_cast(s8, piece[2]);
}

// BM x BN results a workgroup of WM x WN waves; blocks of BK along the sum, NBUF of them in LDS; NP planes; AR, BR: rows
// run across the sum
// CUT: operands are float32 in LDS, and each wave cuts what it reads (1: fetched by 16 bytes, 2: by 4)
template <int DT_, int ACT_, int NP_, bool AR_, bool BR_, int BM_, int BN_, int WM_, int WN_, int BK_, int NBUF_, int GM_, int CUT_ = 0>
struct LinTile {
  static constexpr int GM = GM_, DT = DT_, ACT = ACT_, NP = NP_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NBUF = NBUF_, W = WM * WN;
  static constexpr bool AR = AR_, BR = BR_;
  static constexpr int CUT = CUT_, LP = CUT ? 1 : NP, ES = CUT ? 4 : 2;        // planes in LDS, of elements of ES bytes
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static constexpr int AB = BM * BK * ES, BB = BN * BK * ES, BUF = LP * (AB + BB), LDO = 68, OUT = 16 * (MT < 4 ? MT : 4) * LDO * 4;
  static constexpr int LDS = NBUF * BUF > W * OUT ? NBUF * BUF : W * OUT;      // LDO: a row of a wave's results
  static constexpr int DA = LP * AB / 1024 / W * (CUT == 2 ? 4 : 1), DB = LP * BB / 1024 / W * (CUT == 2 ? 4 : 1);       // a wave's DMAs of a block
  static_assert(AB % 1024 == 0 && BB % 1024 == 0 && LP * AB % (1024 * W) == 0 && LP * BB % (1024 * W) == 0, "whole DMAs");
  static_assert(NT == 4 && (MT % 4 == 0 || MT < 4) && (CUT ? NP == 3 && BK == 32 : NP == 1 || (!AR && !BR)) && LDS <= 160 * 1024, "shapes");
};

// Where a wave's i-th DMA of an operand's block comes from.  Sixteen bytes a lane:
//   rows along the sum: row q / CH, chunk (q % CH) ^ f(row) of eight values;
//   rows across it: value q / (ROWS / 8) along the sum, the pair of chunks exchanged by its own f.
// f spreads what the lanes of a read have in common over LDS's banks.
template <int BK>
__device__ __forceinline__ int lin_turn(int row) { return BK == 64 ? row & 7 : (row >> 1) & 3; }
template <int ROWS>
__device__ __forceinline__ int lin_turn_r(int k) { return ROWS == 64 ? k & 3 : (k & 3) | (k >> 1 & 4); }

template <class C, bool R, int ROWS, int D>
struct LinSource {
  static constexpr int PLANE = ROWS * C::BK * 2 / 1024;
  const char* src[D];
  int k[D];                // along the sum, of the lane's first value
  size_t step;
  __device__ __forceinline__ void init(const LinOperand& o, int row0, int kb0) {
    const int l = lane_id(), w = wave_id();
    step = (R ? C::BK * o.ld : (size_t)C::BK) * 2;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const int u = w * D + i, p = u / PLANE, q = u % PLANE * 64 + l;
      size_t at;
      if constexpr (R) {
        k[i] = q / (ROWS / 8);
        const int c = q % (ROWS / 8), unit = (c >> 1) ^ lin_turn_r<ROWS>(k[i]);
        at = (size_t)k[i] * o.ld + min(row0 + 16 * unit + 8 * (c & 1), o.rows - 8);
      } else {
        constexpr int CH = C::BK / 8;
        const int row = q / CH;
        k[i] = 8 * (q % CH ^ lin_turn<C::BK>(row));
        at = (size_t)min(row0 + row, o.rows - 1) * o.ld + k[i];
      }
      src[i] = reinterpret_cast<const char*>(o.p + p * o.plane + at) + (size_t)kb0 * step;
      k[i] += kb0 * C::BK;
    }
  }
  // the next block into LDS at dst; tail: it may pass the end of the sum
  __device__ __forceinline__ void fetch(char* dst, int K, bool tail) {
    const int w = wave_id();
#pragma unroll
    for (int i = 0; i < D; ++i) {
      const char* s = src[i];
      if (tail) s = k[i] < K ? s : reinterpret_cast<const char*>(&lin_zeros);
      lds_dma16(reinterpret_cast<const float*>(s), reinterpret_cast<float*>(dst + (w * D + i) * 1024));
      src[i] += step;
      k[i] += C::BK;
    }
  }
};

// A lane's operands of tile t (16 rows) and step s (32 values) of a block in LDS
template <class C, bool R, int ROWS>
__device__ __forceinline__ s8 lin_read(const char* lds, int t, int s) {
  const int l = lane_id(), r = l & 15, c = l >> 4;
  if constexpr (R) {
    const int k = 8 * c + (r >> 2), at = k * ROWS * 2 + ((t ^ lin_turn_r<ROWS>(k)) << 5) + (r & 3) * 8 + s * 32 * ROWS * 2;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at + 8 * ROWS));
    return s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  } else {
    const int row = 16 * t + r;
    return *reinterpret_cast<const s8*>(lds + row * C::BK * 2 + (((4 * s + c) ^ lin_turn<C::BK>(row)) << 4));
  }
}

// Results of a row, E of them from column n on: bias, activation, residual
template <int DT, int ACT, int E>
__device__ __forceinline__ void lin_out(const LinArgs& a, int m, int n, const float* f) {
  const size_t at = (size_t)m * a.N + n;
  if (a.vec) {               // (whole groups of eight columns, and every pointer takes 16 bytes)
    static_assert(E % 4 == 0 || E == 1, "columns");
    if constexpr (E == 1) return;          // (whole rows come by fours)
#pragma unroll
    for (int q = 0; q + 3 < E; q += 4) {
      float4 v = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
      if (a.bias) {
        const float4 b = lin_get4(a.bias_dtype, a.bias, n + q);
        v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
      }
      if (a.z) lin_put4(a.z_dtype, a.z, at + q, v);
      v = make_float4(lin_act<ACT>(v.x), lin_act<ACT>(v.y), lin_act<ACT>(v.z), lin_act<ACT>(v.w));
      if (a.residual) {
        const float4 r = lin_get4(a.out_dtype, a.residual, (size_t)m * a.ldr + n + q);
        v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
      }
      lin_put4(a.out_dtype, a.y, at + q, v);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (n + e >= a.N) break;
    float z = f[e] + (a.bias ? lin_get(a.bias_dtype, a.bias, n + e) : 0.f);
    if (a.z) lin_put(a.z_dtype, a.z, at + e, z);
    z = lin_act<ACT>(z);
    if (a.residual) z += lin_get(a.out_dtype, a.residual, (size_t)m * a.ldr + n + e);
    lin_put(a.out_dtype, a.y, at + e, z);
  }
}
// The same for eight columns, with the bias loaded once and the residual ahead; as lin_out where a.vec does not hold
struct LinColumns {
  float4 b[2];
  __device__ __forceinline__ void load(const LinArgs& a, int n) {
    b[0] = b[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!a.bias || !a.vec) return;
    b[0] = lin_get4(a.bias_dtype, a.bias, n);
    b[1] = lin_get4(a.bias_dtype, a.bias, n + 4);
  }
};
struct LinResidual {
  uint4 u[2];              // eight of 16 bits, or of 32
  __device__ __forceinline__ void load(const LinArgs& a, int m, int n) {
    if (!a.residual || !a.vec) return;
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(a.residual) + ((size_t)m * a.ldr + n) * (a.out_dtype == LIN_F32 ? 4 : 2));
    u[0] = p[0];
    if (a.out_dtype == LIN_F32) u[1] = p[1];
  }
};
template <int DT, int ACT>
__device__ __forceinline__ void lin_out8(const LinArgs& a, int m, int n, float* f, const LinColumns& cols, const LinResidual& r) {
  if (!a.vec) {
    lin_out<DT, ACT, 8>(a, m, n, f);
    return;
  }
  const size_t at = (size_t)m * a.N + n;
  const float b[8] = {cols.b[0].x, cols.b[0].y, cols.b[0].z, cols.b[0].w, cols.b[1].x, cols.b[1].y, cols.b[1].z, cols.b[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] += b[e];
  if (a.z && a.z_dtype == LIN_F32) LinVec<LIN_F32>::store8(a.z, at, f);
  else if (a.z) LinVec<DT>::store8(a.z, at, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = lin_act<ACT>(f[e]);
  if (a.residual) {
    float x[8];
    if (a.out_dtype == LIN_F32) {
      LinVec<LIN_F32>::widen(r.u[0], x);
      LinVec<LIN_F32>::widen(r.u[1], x + 4);
    } else {
      LinVec<DT == LIN_F32 ? LIN_BF16 : DT>::widen(r.u[0], x);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] += x[e];
  }
  if (a.out_dtype == LIN_F32) LinVec<LIN_F32>::store8(a.y, at, f);
  else LinVec<DT>::store8(a.y, at, f);
}
// ... or of a part of the sum
template <int E>
__device__ __forceinline__ void lin_out_part(const LinArgs& a, int part, int m, int n, const float* f) {
  float* p = a.part + ((size_t)part * a.M + m) * a.N + n;
  if (a.vec) {
#pragma unroll
    for (int q = 0; q < E; q += 4) *reinterpret_cast<float4*>(p + q) = make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (n + e < a.N) p[e] = f[e];
}

// A wave's results in LDS (rows of ldo floats; more: a second part of their sum, or NULL) where rows are not whole groups of
// eight columns: a lane takes one column of COLS, so that what a wave writes at a time is whole lines all the same.
template <int DT, int ACT, int COLS>
__device__ __forceinline__ void lin_out_odd(const LinArgs& a, int part, const float* own, const float* more, int ldo, int rows, int m0, int n0) {
  const int l = lane_id(), col = l % COLS, n = n0 + col;
  constexpr int STEP = WAVE / COLS, U = 8;
  if (n >= a.N) return;
  const float bias = a.bias ? lin_get(a.bias_dtype, a.bias, n) : 0.f;
  for (int r = l / COLS; r < rows && m0 + r < a.M; r += STEP * U) {
    float res[U];
    if (a.residual && !a.sums)
#pragma unroll
      for (int u = 0; u < U; ++u) res[u] = lin_get(a.out_dtype, a.residual, (size_t)min(m0 + r + u * STEP, a.M - 1) * a.ldr + n);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = r + u * STEP, m = m0 + row;
      if (row >= rows || m >= a.M) break;
      float f = own[row * ldo + col];
      if (more) f += more[row * ldo + col];
      if (a.sums) {
        a.part[((size_t)part * a.M + m) * a.N + n] = f;
        continue;
      }
      f += bias;
      const size_t at = (size_t)m * a.N + n;
      if (a.z) lin_put(a.z_dtype, a.z, at, f);
      f = lin_act<ACT>(f);
      if (a.residual) f += res[u];
      lin_put(a.out_dtype, a.y, at, f);
    }
  }
}

// The same for results of 16 bits, which would be half a line at a time: half a wave takes a row, a lane two neighbouring
// columns from an even place in memory on (rows of odd width start at an odd one every other time: then the last lane has the
// two that are left over).  y and z take 4-byte accesses.
template <int DT, int ACT>
__device__ __forceinline__ void lin_out_pairs(const LinArgs& a, const float* own, int ldo, int rows, int m0, int n0) {
  using L = LinType<DT>;
  const int l = lane_id(), hl = l & 31;
  constexpr int U = 4;
  const int left = a.N - n0;                 // columns from here on
  if (left <= 0) return;
  float b[4] = {0.f, 0.f, 0.f, 0.f};         // of columns 2 hl .. 2 hl + 2, and 0
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 3; ++e) b[e] = lin_get(a.bias_dtype, a.bias, n0 + min(2 * hl + e, left - 1));
    b[3] = lin_get(a.bias_dtype, a.bias, n0);
  }
  for (int r = l >> 5; r < rows && m0 + r < a.M; r += 2 * U) {
    float res[U][2];
    int col[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int m = min(m0 + r + 2 * u, a.M - 1), odd = (int)(((size_t)m * a.N + n0) & 1);
      const bool over = odd && hl == 31;
      col[u][0] = over ? 63 : 2 * hl + odd;
      col[u][1] = over ? 0 : 2 * hl + odd + 1;
      if (a.residual)
#pragma unroll
        for (int e = 0; e < 2; ++e) res[u][e] = lin_get(a.out_dtype, a.residual, (size_t)m * a.ldr + n0 + min(col[u][e], left - 1));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = r + 2 * u, m = m0 + row, odd = col[u][0] & 1;
      if (row >= rows || m >= a.M) break;
      const bool over = col[u][1] < col[u][0];
      float f[2], z[2];
      z[0] = own[row * ldo + col[u][0]] + (odd ? b[1] : b[0]);
      z[1] = own[row * ldo + col[u][1]] + (over ? b[3] : odd ? b[2] : b[1]);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        f[e] = lin_act<ACT>(z[e]);
        if (a.residual) f[e] += res[u][e];
      }
      const size_t at = (size_t)m * a.N + n0;
      auto two = [&](void* p, const float* v) __attribute__((always_inline)) {
        if (!over && col[u][1] < left) {
          uint32_t w;
          if constexpr (DT == LIN_BF16) w = bf16_pack(v[0], v[1]);
          else {
            const h2v h = {(_Float16)v[0], (_Float16)v[1]};
            w = __builtin_bit_cast(uint32_t, h);
          }
          *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + at + col[u][0]) = w;
          return;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (col[u][e] < left) L::put(p, at + col[u][e], v[e]);
      };
      if (a.z) two(a.z, z);
      two(a.y, f);
    }
  }
}

// Workgroups go to the 8 dies in turn: each die gets a run of neighbouring tiles (of one part of the sum), GM rows of tiles
// high, so that what its workgroups read at a time is shared in its L2.
__device__ __forceinline__ void lin_place(const LinArgs& a, int gm, int& part, int& mi, int& ni) {
  const int tiles = a.mt * a.nt, total = tiles * a.parts, b = blockIdx.x, x = b & 7, whole = total >> 3, more = total & 7;
  const int i = x * whole + min(x, more) + (b >> 3);
  part = i / tiles;
  const int t = i - part * tiles, group = t / (gm * a.nt), m0 = group * gm, h = min(gm, a.mt - m0), in = t - m0 * a.nt;
  ni = in / h;
  mi = m0 + in - ni * h;
}

template <class C>
__global__ __launch_bounds__(C::W * WAVE) void lin_tile_kernel(LinArgs a) {
  constexpr int MT = C::MT, NT = C::NT, NP = C::NP, S = C::BK / 32;
  constexpr bool F16 = C::DT == LIN_F16;
  extern __shared__ char lds[];
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), wm = w / C::WN, wn = w % C::WN;
  int part, mi, ni;
  lin_place(a, C::GM, part, mi, ni);
  const int m0 = mi * C::BM, n0 = ni * C::BN;
  const int blocks = (a.K + C::BK - 1) / C::BK, kb0 = part * a.per, kb1 = min(blocks, kb0 + a.per);
  std::conditional_t<C::CUT != 0, LinFloats<C::AR, C::BM, C::W, C::CUT == 1>, LinSource<C, C::AR, C::BM, C::DA>> sa;
  std::conditional_t<C::CUT != 0, LinFloats<C::BR, C::BN, C::W, C::CUT == 1>, LinSource<C, C::BR, C::BN, C::DB>> sb;
  sa.init(a.a, m0, kb0);
  sb.init(a.b, n0, kb0);
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
    const bool tail = (kb + 1) * C::BK > a.K;
    sa.fetch(lds + buf, a.K, tail);
    sb.fetch(lds + buf + C::LP * C::AB, a.K, tail);
  };
  // float32: the products of the leading pieces on their own, so that the small ones are not rounded beside them
  constexpr int NA = NP > 1 ? 2 : 1;
  f4 acc[NA][NT][MT];
#pragma unroll
  for (int q = 0; q < NA; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[q][i][t] = f4{0.f, 0.f, 0.f, 0.f};
  // Operands are read ahead of their use, those of A by AHEAD tiles, those of B by one step of the sum, a few beside each
  // group of products (8192 x 4096 x 4096 bfloat16, on one card: 225 us; read where they are used 248)
  auto products = [&](int t, const s8 (&n)[NP][NT], const s8 (&m)[NP]) __attribute__((always_inline)) {
    // (float32: the smallest pieces' products first)
#pragma unroll
    for (int o = NP - 1; o >= 0; --o)
#pragma unroll
      for (int p = 0; p <= o; ++p) {
        auto& c4 = acc[o ? NA - 1 : 0];
        const auto& b4 = n[o - p];
        lin_mfma4<F16>(c4[0][t], c4[1][t], c4[2][t], c4[3][t], b4[0], b4[1], b4[2], b4[3], m[p]);
      }
  };
  // (8 values a lane cost 44 instructions beside the products: a tile of B serves four of A and the other way round)
  auto add_cut = [&](const char* at) __attribute__((always_inline)) {
    if constexpr (C::CUT) {
      s8 n[3][NT], m[3];
#pragma unroll
      for (int i = 0; i < NT; ++i) lin_cut<C::BR, C::BN>(at + C::AB, wn * NT + i, n[0][i], n[1][i], n[2][i]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        lin_cut<C::AR, C::BM>(at, wm * MT + t, m[0], m[1], m[2]);
        products(t, n, m);
      }
    }
  };
  auto add = [&](const char* at) __attribute__((always_inline)) {
    constexpr int STEPS = S * MT, AHEAD = NP == 1 ? 2 : 1, RING = AHEAD + 1;
    s8 n[2][NP][NT], m[RING][NP];
    auto read_n = [&](int s, int i) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < NP; ++p) n[s & 1][p][i] = lin_read<C, C::BR, C::BN>(at + NP * C::AB + p * C::BB, wn * NT + i, s);
    };
    auto read_m = [&](int x) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < NP; ++p) m[x % RING][p] = lin_read<C, C::AR, C::BM>(at + p * C::AB, wm * MT + x % MT, x / MT);
    };
#pragma unroll
    for (int i = 0; i < NT; ++i) read_n(0, i);
#pragma unroll
    for (int x = 0; x < (AHEAD < STEPS ? AHEAD : STEPS); ++x) read_m(x);
#pragma unroll
    for (int x = 0; x < STEPS; ++x) {
      const int s = x / MT, t = x % MT;
      if (x + AHEAD < STEPS) read_m(x + AHEAD);
      if (s + 1 < S)
#pragma unroll
        for (int i = t * NT / MT; i < (t + 1) * NT / MT; ++i) read_n(s + 1, i);
      products(t, n[s & 1], m[x % RING]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Block kb has come when only the DMAs of the NBUF - 2 behind it are under way
  constexpr int AHEAD = C::NBUF - 1, BEHIND = (C::NBUF - 2) * (C::DA + C::DB);
  static_assert(BEHIND < 64, "vmcnt");
  auto next = [&](int x) { return x == (C::NBUF - 1) * C::BUF ? 0 : x + C::BUF; };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (kb0 + i < kb1) fetch(kb0 + i, i * C::BUF);
  int buf = 0, into = AHEAD * C::BUF;
  for (int kb = kb0; kb < kb1; ++kb) {
    if (kb + C::NBUF - 2 < kb1) __builtin_amdgcn_s_waitcnt(lin_wait(BEHIND));
    else __builtin_amdgcn_s_waitcnt(WAIT_VMCNT0);
    __syncthreads();
    if (kb + AHEAD < kb1) fetch(kb + AHEAD, into);
    if constexpr (C::CUT) add_cut(lds + buf);
    else add(lds + buf);
    buf = next(buf);
    into = next(into);
  }
  drain(acc[0][0][0]);
#pragma unroll
  for (int q = 0; q < NA; ++q)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) lin_hold(acc[q][i][t]);
  // Each wave turns its results around in LDS, up to 64 rows at a time: a lane holds four columns of a row here and takes
  // eight there, so that whole lines are written (and the epilogue's code stands once, not for every register).
  __syncthreads();
  constexpr int HT = MT < 4 ? MT : 4;
  float* own = reinterpret_cast<float*>(lds) + w * (16 * HT * C::LDO);
  const int col = 8 * (l & 7), n = n0 + 64 * wn + col;
  LinColumns cols;
  if (n < a.N) cols.load(a, n);
#pragma unroll
  for (int h = 0; h < MT; h += HT) {
#pragma unroll
    for (int t = h; t < h + HT; ++t)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        f4 v = acc[0][i][t];
        if constexpr (NA == 2) v += acc[1][i][t];
        *reinterpret_cast<f4*>(own + (16 * (t - h) + r) * C::LDO + 16 * i + 4 * c) = v;
      }
    __builtin_amdgcn_wave_barrier();
    if (!a.vec) {
      const int mf = m0 + 16 * (wm * MT + h), nf = n0 + 64 * wn;
      if constexpr (C::DT == LIN_F32) lin_out_odd<C::DT, C::ACT, 64>(a, part, own, nullptr, C::LDO, 16 * HT, mf, nf);
      else if (a.pairs) lin_out_pairs<C::DT, C::ACT>(a, own, C::LDO, 16 * HT, mf, nf);
      else lin_out_odd<C::DT, C::ACT, 64>(a, part, own, nullptr, C::LDO, 16 * HT, mf, nf);
      __builtin_amdgcn_wave_barrier();
      continue;
    }
    const int mh = m0 + 16 * (wm * MT + h) + (l >> 3);
#pragma unroll 1
    for (int j = 0; j < 2 * HT; j += 2) {
      // (two rows of a lane at a time: the residual's loads are under way together)
      const int m1 = mh + 8 * j, m2 = m1 + 8;
      if (n >= a.N || m1 >= a.M) break;
      LinResidual r1, r2;
      if (!a.sums) {
        r1.load(a, m1, n);
        r2.load(a, min(m2, a.M - 1), n);
      }
      float f[2][8];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<f4*>(f[q] + e) = *reinterpret_cast<const f4*>(own + (8 * (j + q) + (l >> 3)) * C::LDO + col + e);
      if (a.sums) {
        lin_out_part<8>(a, part, m1, n, f[0]);
        if (m2 < a.M) lin_out_part<8>(a, part, m2, n, f[1]);
      } else {
        lin_out8<C::DT, C::ACT>(a, m1, n, f[0], cols, r1);
        if (m2 < a.M) lin_out8<C::DT, C::ACT>(a, m2, n, f[1], cols, r2);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The parts of a sum, in order, and the epilogue; four columns a thread, or (E 1) one where rows are not whole
template <int DT, int ACT, int E>
__global__ __launch_bounds__(256) void lin_join_kernel(LinArgs a) {
  const int cols = (a.N + E - 1) / E;
  const size_t x = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)a.M * a.N;
  const int m = (int)(x / cols), n = E * (int)(x - (size_t)m * cols);
  if (m >= a.M) return;
  const float* p = a.part + (size_t)m * a.N + n;
  float f[E];
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = 0.f;
#pragma unroll 8
  for (int i = 0; i < a.parts; ++i) {
    if constexpr (E == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i * step);
      f[0] += v.x; f[1] += v.y; f[2] += v.z; f[3] += v.w;
    } else {
      f[0] += p[i * step];
    }
  }
  lin_out<DT, ACT, E>(a, m, n, f);
}

// ---- float32 as it is ---------------------------------------------------------------------------------------------

// Small float32 products on the matrix cores' own float32 (a sixteenth of bfloat16's rate, a third of that of six products
// of pieces): no pass over the operands before it.  Tiles of 64 x 64, a wave 32 x 32 and, so that two waves a SIMD cover
// each other's waits where there is one workgroup a CU, half of each block of 32 along the sum; four blocks in LDS.  A lane
// takes four values along the sum at a time, 4 c .. 4 c + 3 of sixteen (c = lane / 16), one for each of four
// 4-deep products, of both operands: rows along the sum by 16 bytes, rows across it by four single values, their chunks
// exchanged by 64 bytes for each c.
template <int ACT_, bool AR_, bool BR_, bool WIDE_>
struct LinDirect {
  static constexpr int ACT = ACT_, BM = 64, BN = 64, BK = 32, NBUF = 4, AB = BM * BK * 4, BUF = 2 * AB, LDS = NBUF * BUF, LDO = 36;
  static constexpr bool AR = AR_, BR = BR_, WIDE = WIDE_;
};
template <class C>
__global__ __launch_bounds__(512) void lin_direct_kernel(LinArgs a) {
  extern __shared__ char lds[];
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), half = w >> 2, wm = w >> 1 & 1, wn = w & 1;
  int part, mi, ni;
  lin_place(a, 8, part, mi, ni);
  const int m0 = mi * C::BM, n0 = ni * C::BN;
  const int blocks = (a.K + C::BK - 1) / C::BK, kb0 = part * a.per, kb1 = min(blocks, kb0 + a.per);
  LinFloats<C::AR, C::BM, 8, C::WIDE> sa;
  LinFloats<C::BR, C::BN, 8, C::WIDE> sb;
  sa.init(a.a, m0, kb0);
  sb.init(a.b, n0, kb0);
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
    const bool tail = (kb + 1) * C::BK > a.K;
    sa.fetch(lds + buf, a.K, tail);
    sb.fetch(lds + buf + C::AB, a.K, tail);
  };
  f4 acc[2][2];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q >> 1][q & 1] = f4{0.f, 0.f, 0.f, 0.f};
  constexpr int AHEAD = C::NBUF - 1, BEHIND = (C::NBUF - 2) * (sa.D + sb.D);
  auto next = [&](int x) { return x == (C::NBUF - 1) * C::BUF ? 0 : x + C::BUF; };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (kb0 + i < kb1) fetch(kb0 + i, i * C::BUF);
  int buf = 0, into = AHEAD * C::BUF;
  for (int kb = kb0; kb < kb1; ++kb) {
    if (kb + C::NBUF - 2 < kb1) __builtin_amdgcn_s_waitcnt(lin_wait(BEHIND));
    else __builtin_amdgcn_s_waitcnt(WAIT_VMCNT0);
    __syncthreads();
    if (kb + AHEAD < kb1) fetch(kb + AHEAD, into);
    const char* at = lds + buf;
    float4 m[2], n[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = lin_floats<C::AR, C::BM>(at, wm * 2 + i, half);
      n[i] = lin_floats<C::BR, C::BN>(at + C::AB, wn * 2 + i, half);
    }
    // (the four tiles in turn: a product that waits for the one before it costs an eighth more)
    auto four = [&](float n0, float n1, float m0, float m1) __attribute__((always_inline)) {
      asm volatile(
          "s_nop 1\n\tv_mfma_f32_16x16x4_f32 %0, %4, %6, %0\n\tv_mfma_f32_16x16x4_f32 %1, %4, %7, %1\n\t"
          "v_mfma_f32_16x16x4_f32 %2, %5, %6, %2\n\tv_mfma_f32_16x16x4_f32 %3, %5, %7, %3"
          : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1])
          : "v"(n0), "v"(n1), "v"(m0), "v"(m1));
    };
    four(n[0].x, n[1].x, m[0].x, m[1].x);
    four(n[0].y, n[1].y, m[0].y, m[1].y);
    four(n[0].z, n[1].z, m[0].z, m[1].z);
    four(n[0].w, n[1].w, m[0].w, m[1].w);
    buf = next(buf);
    into = next(into);
  }
  drain(acc[0][0]);
#pragma unroll
  for (int q = 0; q < 4; ++q) lin_hold(acc[q >> 1][q & 1]);
  __syncthreads();
  // both halves' sums through LDS, each wave then a half of the tile's rows
  float* own = reinterpret_cast<float*>(lds) + w * (32 * C::LDO);
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<f4*>(own + (16 * t + r) * C::LDO + 16 * i + 4 * c) = acc[i][t];
  __syncthreads();
  const float* low = reinterpret_cast<const float*>(lds) + (w & 3) * (32 * C::LDO);
  if (!a.vec) {
    const float* first = low + 16 * half * C::LDO;
    lin_out_odd<LIN_F32, C::ACT, 32>(a, part, first, first + 4 * 32 * C::LDO, C::LDO, 16, m0 + 32 * wm + 16 * half, n0 + 32 * wn);
    return;
  }
  const int col = 8 * (l & 3), n = n0 + 32 * wn + col;
  if (n >= a.N) return;
  LinColumns cols;
  cols.load(a, n);
  const int row = 16 * half + (l >> 2), m = m0 + 32 * wm + row;
  if (m >= a.M) return;
  LinResidual res;
  if (!a.sums) res.load(a, m, n);
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    const float* q = low + row * C::LDO + col + e;
    *reinterpret_cast<f4*>(f + e) = *reinterpret_cast<const f4*>(q) + *reinterpret_cast<const f4*>(q + 4 * 32 * C::LDO);
  }
  if (a.sums) lin_out_part<8>(a, part, m, n, f);
  else lin_out8<LIN_F32, C::ACT>(a, m, n, f, cols, res);
}

// ---- few rows -----------------------------------------------------------------------------------------------------

// Few rows are bound by W's bytes, and the matrix cores have nothing to share: every element of W is read once, from memory
// to registers, and multiplied there, float32 as it is.  MR rows at a time; a.parts parts of `per` values of the sum.
constexpr int LIN_ROWS_W = 8, LIN_ROWS_COLS = 8;       // waves; lanes along the columns of W
// W (K, N): eight lanes take 16 bytes each of a row of W, the workgroup's 64 groups of lanes eight rows each; their sums meet
// over the wave's lanes and then in LDS.
template <int DT, int ACT, int MR>
__global__ __launch_bounds__(LIN_ROWS_W * WAVE) void lin_rows_kernel(LinArgs a) {
  using V = LinVec<DT>;
  constexpr int E = V::E, COLS = LIN_ROWS_COLS * E;
  __shared__ float sums[LIN_ROWS_W][MR][COLS];
  const int l = lane_id(), w = wave_id(), n = blockIdx.x * COLS + (l & 7) * E, m0 = blockIdx.z * MR;
  const int k0 = blockIdx.y * a.per, k1 = min(a.K, k0 + a.per);
  float acc[MR][E];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[m][e] = 0.f;
  if (n < a.N)
    for (int k = k0 + 8 * (w * 8 + (l >> 3)); k < k1; k += 64 * LIN_ROWS_W) {
      float wt[8][E], x[MR][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) V::template load<E, true>(a.b.p, (size_t)(k + j) * a.b.ld + n, E, wt[j]);
#pragma unroll
      for (int m = 0; m < MR; ++m) V::template load<8, true>(a.a.p, (size_t)min(m0 + m, a.M - 1) * a.a.ld + k, 8, x[m]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[m][e] = fmaf(x[m][j], wt[j][e], acc[m][e]);
    }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int o = 8; o < WAVE; o *= 2) acc[m][e] += __shfl_xor(acc[m][e], o);
      if (l < 8) sums[w][m][l * E + e] = acc[m][e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < MR * COLS / 4; i += LIN_ROWS_W * WAVE) {
    const int m = i / (COLS / 4), col = 4 * (i % (COLS / 4)), at = blockIdx.x * COLS + col;
    if (m0 + m >= a.M || at >= a.N) continue;
    float f[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < LIN_ROWS_W; ++v)
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] += sums[v][m][col + e];
    if (a.sums) lin_out_part<4>(a, blockIdx.y, m0 + m, at, f);
    else lin_out<DT, ACT, 4>(a, m0 + m, at, f);
  }
}

// The same for a W (or x) whose rows are not whole 16 bytes: a lane takes one column, so that a wave's loads are whole lines
// all the same, the four waves a quarter of the part each (at most 1024 values), x from LDS.
constexpr int LIN_COLUMNS_K = 1024;
template <int DT, int ACT, int MR>
__global__ __launch_bounds__(256) void lin_columns_kernel(LinArgs a) {
  __shared__ float x[MR][LIN_COLUMNS_K], sums[4][MR][64];
  const int l = lane_id(), w = wave_id(), n = blockIdx.x * 64 + l, m0 = blockIdx.z * MR;
  const int k0 = blockIdx.y * a.per, k1 = min(a.K, k0 + a.per), ks = k1 - k0;
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    const size_t row = (size_t)min(m0 + m, a.M - 1) * a.a.ld + k0;
#pragma unroll 4
    for (int k = threadIdx.x; k < ks; k += 256) x[m][k] = LinType<DT>::get(a.a.p, row + k);
  }
  __syncthreads();
  const int quarter = (ks + 3) / 4, b = w * quarter, e = min(ks, b + quarter);
  float acc[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) acc[m] = 0.f;
  const size_t at = (size_t)k0 * a.b.ld + min(n, a.N - 1);
  int k = b;
  for (; k + 8 <= e; k += 8) {
    float wt[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) wt[j] = LinType<DT>::get(a.b.p, at + (size_t)(k + j) * a.b.ld);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int m = 0; m < MR; ++m) acc[m] = fmaf(x[m][k + j], wt[j], acc[m]);
  }
  for (; k < e; ++k) {
    const float wt = LinType<DT>::get(a.b.p, at + (size_t)k * a.b.ld);
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[m] = fmaf(x[m][k], wt, acc[m]);
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) sums[w][m][l] = acc[m];
  __syncthreads();
  for (int i = threadIdx.x; i < MR * 16; i += 256) {
    const int m = i / 16, col = 4 * (i % 16), to = blockIdx.x * 64 + col;
    if (m0 + m >= a.M || to >= a.N) continue;
    float f[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) f[q] = (sums[0][m][col + q] + sums[1][m][col + q]) + (sums[2][m][col + q] + sums[3][m][col + q]);
    if (a.sums) lin_out_part<4>(a, blockIdx.y, m0 + m, to, f);
    else lin_out<DT, ACT, 4>(a, m0 + m, to, f);
  }
}

// W (N, K): a wave takes four rows of W, its lanes along the sum
template <int DT, int ACT, int MR, bool VEC>
__global__ __launch_bounds__(256) void lin_dots_kernel(LinArgs a) {
  using V = LinVec<DT>;
  constexpr int E = V::E, NR = 4;
  const int l = lane_id(), n0 = (blockIdx.x * 4 + wave_id()) * NR, m0 = blockIdx.z * MR;
  if (n0 >= a.N) return;
  const int k0 = blockIdx.y * a.per, k1 = min(a.K, k0 + a.per);
  float acc[MR][NR];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[m][i] = 0.f;
#pragma unroll 2
  for (int k = k0 + E * l; k < k1; k += E * WAVE) {
    float wt[NR][E], x[MR][E];
#pragma unroll
    for (int i = 0; i < NR; ++i) V::template load<E, VEC>(a.b.p, (size_t)min(n0 + i, a.N - 1) * a.b.ld + k, k1 - k, wt[i]);
#pragma unroll
    for (int m = 0; m < MR; ++m) V::template load<E, VEC>(a.a.p, (size_t)min(m0 + m, a.M - 1) * a.a.ld + k, k1 - k, x[m]);
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[m][i] = fmaf(x[m][e], wt[i][e], acc[m][i]);
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
      for (int o = 1; o < WAVE; o *= 2) acc[m][i] += __shfl_xor(acc[m][i], o);
    if (l != m || m0 + m >= a.M) continue;
    if (a.sums) lin_out_part<4>(a, blockIdx.y, m0 + m, n0, acc[m]);
    else lin_out<DT, ACT, 4>(a, m0 + m, n0, acc[m]);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------

// How a product runs.
struct LinPlan {
  int rows;                  // rows at a time by lin_rows_kernel or lin_dots_kernel; 0: tiles
  int tile;                  // LIN_SMALL, LIN_MID, LIN_BIG; float32 as it is: LIN_DIRECT, LIN_CUT, wide: by 16-byte accesses
  int parts, per;            // parts of the sum, of `per` blocks (rows: values)
  bool wide;
};
enum { LIN_SMALL, LIN_MID, LIN_BIG, LIN_DIRECT, LIN_CUT };      // the last two: no workspace but for the parts
constexpr int lin_bk(int dtype) { return dtype == LIN_F32 ? 32 : 64; }

template <int DT, int ACT>
static void lin_join(LinArgs a, hipStream_t s) {
  if (!a.sums) return;
  if (a.halves) {
    a.M /= 2;
    a.parts *= 2;
  }
  const size_t threads = (size_t)a.M * (a.vec ? a.N / 4 : a.N);
  const dim3 grid((threads + 255) / 256);
  if (a.vec) hipLaunchKernelGGL((lin_join_kernel<DT, ACT, 4>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((lin_join_kernel<DT, ACT, 1>), grid, dim3(256), 0, s, a);
}
template <class C>
static void lin_go(LinArgs a, const LinPlan& r, hipStream_t s) {
  a.mt = (a.M + C::BM - 1) / C::BM;
  a.nt = (a.N + C::BN - 1) / C::BN;
  a.parts = r.parts;
  a.per = r.per;
  hipLaunchKernelGGL(lin_tile_kernel<C>, dim3(a.mt * a.nt * a.parts), dim3(C::W * WAVE), C::LDS, s, a);
  lin_join<C::DT, C::ACT>(a, s);
}
template <int DT, int ACT, int NP, bool AR, bool BR>
static void lin_tiles(const LinArgs& a, const LinPlan& r, hipStream_t s) {
  if (r.tile == LIN_SMALL) lin_go<LinTile<DT, ACT, NP, AR, BR, 64, 64, 4, 1, lin_bk(DT), 3, 8>>(a, r, s);
  else if (r.tile == LIN_MID) lin_go<LinTile<DT, ACT, NP, AR, BR, 128, 128, DT == LIN_F32 ? 4 : 2, 2, lin_bk(DT), 2, 8>>(a, r, s);
  else if constexpr (DT == LIN_F32) lin_go<LinTile<DT, ACT, NP, AR, BR, 256, 128, 4, 2, lin_bk(DT), 2, 4>>(a, r, s);
  else lin_go<LinTile<DT, ACT, NP, AR, BR, 256, 256, 2, 4, lin_bk(DT), 2, 4>>(a, r, s);
}

// Few rows; whole: every row of x and W takes 16-byte accesses
template <int DT, int ACT, int MR, bool VEC>
static void lin_rows_go(const LinArgs& a, bool dots, hipStream_t s) {
  const int z = (a.M + MR - 1) / MR;
  if (dots) hipLaunchKernelGGL((lin_dots_kernel<DT, ACT, MR, VEC>), dim3((a.N + 15) / 16, a.parts, z), dim3(256), 0, s, a);
  else if constexpr (VEC) {
    constexpr int cols = LIN_ROWS_COLS * LinVec<DT>::E;
    hipLaunchKernelGGL((lin_rows_kernel<DT, ACT, MR>), dim3((a.N + cols - 1) / cols, a.parts, z), dim3(LIN_ROWS_W * WAVE), 0, s, a);
  } else {
    hipLaunchKernelGGL((lin_columns_kernel<DT, ACT, MR>), dim3((a.N + 63) / 64, a.parts, z), dim3(256), 0, s, a);
  }
  lin_join<DT, ACT>(a, s);
}
template <int DT, int ACT>
static void lin_rows_act(const LinArgs& a, const LinPlan& r, bool dots, bool whole, hipStream_t s) {
  auto go = [&](auto mr) {
    if (whole) lin_rows_go<DT, ACT, decltype(mr)::value, true>(a, dots, s);
    else lin_rows_go<DT, ACT, decltype(mr)::value, false>(a, dots, s);
  };
  if (r.rows == 1) go(std::integral_constant<int, 1>{});
  else if (r.rows == 2) go(std::integral_constant<int, 2>{});
  else if (r.rows == 4) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
}
template <int DT>
void lin_rows(const LinArgs& a, const LinPlan& r, int act, bool dots, bool whole, hipStream_t s) {
  if (act == LIN_SILU) lin_rows_act<DT, LIN_SILU>(a, r, dots, whole, s);
  else if (act == LIN_GELU) lin_rows_act<DT, LIN_GELU>(a, r, dots, whole, s);
  else if (act == LIN_TANH) lin_rows_act<DT, LIN_TANH>(a, r, dots, whole, s);
  else lin_rows_act<DT, LIN_NONE>(a, r, dots, whole, s);
}
template <int DT, int NP, bool AR, bool BR>
static void lin_acts(const LinArgs& a, const LinPlan& r, int act, hipStream_t s) {
  if (act == LIN_SILU) lin_tiles<DT, LIN_SILU, NP, AR, BR>(a, r, s);
  else if (act == LIN_GELU) lin_tiles<DT, LIN_GELU, NP, AR, BR>(a, r, s);
  else if (act == LIN_TANH) lin_tiles<DT, LIN_TANH, NP, AR, BR>(a, r, s);
  else lin_tiles<DT, LIN_NONE, NP, AR, BR>(a, r, s);
}
// float32 as it is in memory; wide: in rows that 16-byte accesses take
template <int ACT, bool AR, bool BR, bool WIDE>
static void lin_floats_go(LinArgs a, const LinPlan& r, hipStream_t s) {
  if (r.tile == LIN_CUT) return lin_go<LinTile<LIN_F32, ACT, 3, AR, BR, 128, 128, WIDE ? 2 : 4, 2, 32, 2, 8, WIDE ? 1 : 2>>(a, r, s);
  using C = LinDirect<ACT, AR, BR, WIDE>;
  a.mt = (a.M + C::BM - 1) / C::BM;
  a.nt = (a.N + C::BN - 1) / C::BN;
  hipLaunchKernelGGL(lin_direct_kernel<C>, dim3(a.mt * a.nt * a.parts), dim3(512), C::LDS, s, a);
  lin_join<LIN_F32, ACT>(a, s);
}
template <bool AR, bool BR, bool WIDE>
static void lin_floats_act(const LinArgs& a, const LinPlan& r, int act, hipStream_t s) {
  if (act == LIN_SILU) lin_floats_go<LIN_SILU, AR, BR, WIDE>(a, r, s);
  else if (act == LIN_GELU) lin_floats_go<LIN_GELU, AR, BR, WIDE>(a, r, s);
  else if (act == LIN_TANH) lin_floats_go<LIN_TANH, AR, BR, WIDE>(a, r, s);
  else lin_floats_go<LIN_NONE, AR, BR, WIDE>(a, r, s);
}
template <bool WIDE>
static void lin_floats_form(const LinArgs& a, const LinPlan& r, int form, int act, hipStream_t s) {
  if (form == LIN_XW) lin_floats_act<false, true, WIDE>(a, r, act, s);
  else if (form == LIN_XWT) lin_floats_act<false, false, WIDE>(a, r, act, s);
  else lin_floats_go<LIN_NONE, true, true, WIDE>(a, r, s);
}

template <int DT>
void lin_forms(const LinArgs& a, const LinPlan& r, int form, int act, hipStream_t s) {
  if constexpr (DT == LIN_F32) {
    if (r.tile >= LIN_DIRECT) r.wide ? lin_floats_form<true>(a, r, form, act, s) : lin_floats_form<false>(a, r, form, act, s);
    else lin_acts<DT, 3, false, false>(a, r, act, s);
  } else {
    if (form == LIN_XW) lin_acts<DT, 1, false, true>(a, r, act, s);
    else if (form == LIN_XWT) lin_acts<DT, 1, false, false>(a, r, act, s);
    else lin_tiles<DT, LIN_NONE, 1, true, true>(a, r, s);
  }
}


}  // namespace gdn2
