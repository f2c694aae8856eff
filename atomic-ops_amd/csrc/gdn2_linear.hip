// Products with an epilogue, on gfx950: y = act(A B + bias) + residual, where a layer's forward pass and its two
// gradients differ in how the operands lie in memory (include/gdn2.h, gdn2_product).
//
// The matrix cores take operands whose lanes hold eight consecutive values along the sum.  An operand whose rows run
// along the sum (x; W and dz for the input's gradient) is read from LDS as it is.  One whose rows run across it (W of a
// layer; x and dz for the weight's gradient) lies in LDS as in memory and is transposed on its way to the registers
// (ds_read_b64_tr_b16), so that no pass over memory turns a matrix around.
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
constexpr float LIN_TANH_C = 1.59576912160573072f;       // 2 sqrt(2 / pi)
__device__ __forceinline__ float lin_logistic(float u) { return 1.f / (1.f + __builtin_amdgcn_exp2f(u * -1.44269504088896341f)); }
template <int ACT>
__device__ __forceinline__ float lin_act(float z) {
  if constexpr (ACT == LIN_SILU) return z * lin_logistic(z);
  else if constexpr (ACT == LIN_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  else if constexpr (ACT == LIN_TANH) return z * lin_logistic(LIN_TANH_C * (z + 0.044715f * z * z * z));
  else return z;
}
template <int ACT>
__device__ __forceinline__ float lin_slope(float z) {
  if constexpr (ACT == LIN_SILU) {
    const float s = lin_logistic(z);
    return s * (1.f + z * (1.f - s));
  } else if constexpr (ACT == LIN_GELU) {
    return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  } else if constexpr (ACT == LIN_TANH) {
    const float s = lin_logistic(LIN_TANH_C * (z + 0.044715f * z * z * z));
    return s + z * s * (1.f - s) * (LIN_TANH_C * (1.f + 0.134145f * z * z));
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
  int out_dtype, bias_dtype, vec;
  size_t ldr;
  const void *bias, *residual;
  void *y, *z;
  float* part;
};

__device__ uint4 lin_zeros;      // what lies past the end of a sum

// BM x BN results a workgroup of WM x WN waves; blocks of BK along the sum, NBUF of them in LDS; NP planes; AR, BR: rows
// run across the sum
template <int DT_, int ACT_, int NP_, bool AR_, bool BR_, int BM_, int BN_, int WM_, int WN_, int BK_, int NBUF_>
struct LinTile {
  static constexpr int DT = DT_, ACT = ACT_, NP = NP_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NBUF = NBUF_, W = WM * WN;
  static constexpr bool AR = AR_, BR = BR_;
  static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  static constexpr int AB = BM * BK * 2, BB = BN * BK * 2, BUF = NP * (AB + BB), LDS = NBUF * BUF;
  static constexpr int DA = NP * AB / 1024 / W, DB = NP * BB / 1024 / W;       // a wave's DMAs of a block
  static_assert(AB % 1024 == 0 && BB % 1024 == 0 && NP * AB % (1024 * W) == 0 && NP * BB % (1024 * W) == 0, "whole DMAs");
  static_assert(NT == 4 && (NP == 1 || (!AR && !BR)) && LDS <= 160 * 1024, "shapes");
};

// Where a wave's i-th DMA of an operand's block comes from.  Sixteen bytes a lane:
//   rows along the sum: row q / CH, chunk (q % CH) ^ f(row) of eight values;
//   rows across it: value q / (ROWS / 8) along the sum, the pair of chunks exchanged by its own f.
// f spreads what the lanes of a read have in common over LDS's banks.
template <int BK>
__device__ __forceinline__ int lin_turn(int row) { return BK == 64 ? row & 7 : (row >> 1) & 3; }
__device__ __forceinline__ int lin_turn_r(int k) { return (k & 3) | (k >> 1 & 4); }

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
        const int c = q % (ROWS / 8), unit = (c >> 1) ^ lin_turn_r(k[i]);
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
    const int k = 8 * c + (r >> 2), at = k * ROWS * 2 + ((t ^ lin_turn_r(k)) << 5) + (r & 3) * 8 + s * 32 * ROWS * 2;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at + 8 * ROWS));
    return s8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  } else {
    const int row = 16 * t + r;
    return *reinterpret_cast<const s8*>(lds + row * C::BK * 2 + (((4 * s + c) ^ lin_turn<C::BK>(row)) << 4));
  }
}

// Four results of a row: bias, activation, residual
template <int DT, int ACT>
__device__ __forceinline__ void lin_out4(const LinArgs& a, int m, int n, float4 v) {
  const size_t at = (size_t)m * a.N + n;
  if (a.vec) {
    if (a.bias) {
      const float4 b = lin_get4(a.bias_dtype, a.bias, n);
      v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
    }
    if (a.z) LinType<DT>::put4(a.z, at, v);
    v = make_float4(lin_act<ACT>(v.x), lin_act<ACT>(v.y), lin_act<ACT>(v.z), lin_act<ACT>(v.w));
    if (a.residual) {
      const float4 r = lin_get4(a.out_dtype, a.residual, (size_t)m * a.ldr + n);
      v.x += r.x; v.y += r.y; v.z += r.z; v.w += r.w;
    }
    lin_put4(a.out_dtype, a.y, at, v);
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= a.N) break;
    float z = f[e] + (a.bias ? lin_get(a.bias_dtype, a.bias, n + e) : 0.f);
    if (a.z) LinType<DT>::put(a.z, at + e, z);
    z = lin_act<ACT>(z);
    if (a.residual) z += lin_get(a.out_dtype, a.residual, (size_t)m * a.ldr + n + e);
    lin_put(a.out_dtype, a.y, at + e, z);
  }
}

template <class C>
__global__ __launch_bounds__(C::W * WAVE) void lin_tile_kernel(LinArgs a) {
  constexpr int MT = C::MT, NT = C::NT, NP = C::NP, S = C::BK / 32;
  constexpr bool F16 = C::DT == LIN_F16;
  extern __shared__ char lds[];
  const int l = lane_id(), r = l & 15, c = l >> 4, w = wave_id(), wm = w / C::WN, wn = w % C::WN;
  const int tile = blockIdx.x, m0 = tile / a.nt * C::BM, n0 = tile % a.nt * C::BN;
  const int blocks = (a.K + C::BK - 1) / C::BK, kb0 = blockIdx.z * a.per, kb1 = min(blocks, kb0 + a.per);
  LinSource<C, C::AR, C::BM, C::DA> sa;
  LinSource<C, C::BR, C::BN, C::DB> sb;
  sa.init(a.a, m0, kb0);
  sb.init(a.b, n0, kb0);
  auto fetch = [&](int kb, int buf) __attribute__((always_inline)) {
    const bool tail = (kb + 1) * C::BK > a.K;
    sa.fetch(lds + buf * C::BUF, a.K, tail);
    sb.fetch(lds + buf * C::BUF + NP * C::AB, a.K, tail);
  };
  f4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](const char* at) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      s8 n[NP][NT];
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < NT; ++i) n[p][i] = lin_read<C, C::BR, C::BN>(at + NP * C::AB + p * C::BB, wn * NT + i, s);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        s8 m[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) m[p] = lin_read<C, C::AR, C::BM>(at + p * C::AB, wm * MT + t, s);
        // (float32: the smallest pieces' products first)
#pragma unroll
        for (int o = NP - 1; o >= 0; --o)
#pragma unroll
          for (int p = 0; p <= o; ++p)
            lin_mfma4<F16>(acc[0][t], acc[1][t], acc[2][t], acc[3][t], n[o - p][0], n[o - p][1], n[o - p][2], n[o - p][3], m[p]);
      }
    }
  };
  fetch(kb0, 0);
  int buf = 0;
  for (int kb = kb0; kb < kb1; ++kb) {
    __builtin_amdgcn_s_waitcnt(WAIT_VMCNT0);
    __syncthreads();
    if (kb + 1 < kb1) fetch(kb + 1, buf ^ 1);
    add(lds + buf * C::BUF);
    buf ^= 1;
  }
  drain(acc[0][0]);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) lin_hold(acc[i][t]);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = m0 + 16 * (wm * MT + t) + r;
    if (m >= a.M) continue;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int n = n0 + 16 * (wn * NT + i) + 4 * c;
      if (n >= a.N) continue;
      lin_out4<C::DT, C::ACT>(a, m, n, make_float4(acc[i][t][0], acc[i][t][1], acc[i][t][2], acc[i][t][3]));
    }
  }
}

// ---- operands that the product cannot read as they are ------------------------------------------------------------

// float32 into three planes of bfloat16 pieces, each the next eight bits (cut, so both differences are exact); 16 bits
// copied to rows that 16-byte accesses can take.  out: rows of ld elements, zero past the matrix; turn: transposed.
struct LinPack {
  const void* src;
  uint16_t* out;
  size_t lds, ld, plane;
  int rows, cols, turn;      // of src
  int tr, tc;                // tiles of 64 x 64
};
struct LinPacks {
  LinPack job[2];
  int start[3];
};
__device__ __forceinline__ float lin_top(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
template <bool F32>
__global__ __launch_bounds__(256) void lin_pack_kernel(LinPacks js) {
  constexpr int NP = F32 ? 3 : 1;
  const int which = blockIdx.x >= (unsigned)js.start[1];
  const LinPack& j = js.job[which];
  const int b = blockIdx.x - js.start[which], r0 = b / j.tc * 64, c0 = b % j.tc * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
  __shared__ uint16_t tile[NP][64][65];
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int row = r0 + 4 * i + y, col = c0 + x;
    const bool in = row < j.rows && col < j.cols;
    uint16_t piece[NP];
    if constexpr (F32) {
      const float v = in ? static_cast<const float*>(j.src)[(size_t)row * j.lds + col] : 0.f;
      const float v1 = v - lin_top(v), v2 = v1 - lin_top(v1);
      piece[0] = (uint16_t)(__float_as_uint(v) >> 16);
      piece[1] = (uint16_t)(__float_as_uint(v1) >> 16);
      piece[2] = (uint16_t)(__float_as_uint(v2) >> 16);
    } else {
      piece[0] = in ? static_cast<const uint16_t*>(j.src)[(size_t)row * j.lds + col] : (uint16_t)0;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if (j.turn) tile[p][4 * i + y][x] = piece[p];
      else if (row < j.rows && (size_t)col < j.ld) j.out[p * j.plane + (size_t)row * j.ld + col] = piece[p];
    }
  }
  if (!j.turn) return;
  __syncthreads();
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int row = c0 + 4 * i + y, col = r0 + x;      // of out
    if (row >= j.cols || (size_t)col >= j.ld) continue;
#pragma unroll
    for (int p = 0; p < NP; ++p) j.out[p * j.plane + (size_t)row * j.ld + col] = tile[p][x][4 * i + y];
  }
}

// ---- dz = dy act'(z) and the bias' gradient ------------------------------------------------------------------------

// A workgroup takes 64 columns of 64 rows; part: sums of its rows, [row block][N]
constexpr int SLOPE_ROWS = 64;
template <int ACT>
__global__ __launch_bounds__(256) void lin_slope_kernel(LinSlope a, float* part) {
  __shared__ float sums[4][64];
  const int n = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
  float s = 0.f;
  if (n < a.N)
    for (int i = y; i < SLOPE_ROWS; i += 4) {
      const int64_t m = (int64_t)blockIdx.y * SLOPE_ROWS + i;
      if (m >= a.M) break;
      const size_t at = (size_t)m * a.N + n;
      float d = lin_get(a.dy_dtype, a.dy, at);
      if constexpr (ACT != LIN_NONE) d *= lin_slope<ACT>(lin_get(a.dtype, a.z, at));
      if (a.dz) lin_put(a.dtype, a.dz, at, d);
      s += d;
    }
  if (!part) return;
  sums[y][threadIdx.x & 63] = s;
  __syncthreads();
  if (y == 0 && n < a.N) {
    const int x = threadIdx.x;
    part[(size_t)blockIdx.y * a.N + n] = (sums[0][x] + sums[1][x]) + (sums[2][x] + sums[3][x]);
  }
}
__global__ __launch_bounds__(256) void lin_bias_kernel(LinSlope a, const float* part, int blocks) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= a.N) return;
  float s = 0.f;
  for (int i = 0; i < blocks; ++i) s += part[(size_t)i * a.N + n];
  lin_put(a.bias_dtype, a.dbias, n, s);
}

// ---- launches -----------------------------------------------------------------------------------------------------

static size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }

// An operand's own rows, or the copy that the product reads
struct LinSide {
  bool across, pack;         // rows run across the sum; a copy is needed
  int rows, cols;            // as stored
  size_t ld, plane, bytes;   // of the copy
};
static LinSide lin_side(const LinProduct& p, bool b) {
  LinSide s{};
  const int outer = b ? p.N : p.M;
  s.across = b ? p.form != LIN_XWT : p.form == LIN_XTW;
  s.rows = s.across ? p.K : outer;
  s.cols = s.across ? outer : p.K;
  const size_t ld = b ? p.ldb : p.lda;
  const uintptr_t at = reinterpret_cast<uintptr_t>(b ? p.b : p.a);
  s.pack = p.dtype == LIN_F32 || at % 16 || ld % 8 || s.cols % 8;
  if (!s.pack) return s;
  const bool turned = p.dtype == LIN_F32 && s.across;
  s.ld = up(turned ? s.rows : s.cols, 8);
  s.plane = s.ld * (turned ? s.cols : s.rows);
  s.bytes = up(s.plane * 2 * (p.dtype == LIN_F32 ? 3 : 1), 256);
  return s;
}

size_t linear_workspace_bytes(const LinProduct& p) { return lin_side(p, false).bytes + lin_side(p, true).bytes; }

template <class C>
static void lin_go(LinArgs a, hipStream_t s) {
  a.mt = (a.M + C::BM - 1) / C::BM;
  a.nt = (a.N + C::BN - 1) / C::BN;
  a.parts = 1;
  a.per = (a.K + C::BK - 1) / C::BK;
  hipLaunchKernelGGL(lin_tile_kernel<C>, dim3(a.mt * a.nt, 1, a.parts), dim3(C::W * WAVE), C::LDS, s, a);
}
template <int DT, int ACT, int NP, bool AR, bool BR>
static void lin_tiles(const LinArgs& a, hipStream_t s) {
  lin_go<LinTile<DT, ACT, NP, AR, BR, 128, 128, 2, 2, NP == 1 ? 64 : 32, 2>>(a, s);
}
template <int DT, int NP, bool AR, bool BR>
static void lin_acts(const LinArgs& a, int act, hipStream_t s) {
  if (act == LIN_SILU) lin_tiles<DT, LIN_SILU, NP, AR, BR>(a, s);
  else if (act == LIN_GELU) lin_tiles<DT, LIN_GELU, NP, AR, BR>(a, s);
  else if (act == LIN_TANH) lin_tiles<DT, LIN_TANH, NP, AR, BR>(a, s);
  else lin_tiles<DT, LIN_NONE, NP, AR, BR>(a, s);
}
template <int DT>
static void lin_forms(const LinArgs& a, const LinProduct& p, hipStream_t s) {
  if constexpr (DT == LIN_F32) {
    lin_acts<DT, 3, false, false>(a, p.act, s);
  } else {
    if (p.form == LIN_XW) lin_acts<DT, 1, false, true>(a, p.act, s);
    else if (p.form == LIN_XWT) lin_acts<DT, 1, false, false>(a, p.act, s);
    else lin_tiles<DT, LIN_NONE, 1, true, true>(a, s);
  }
}

hipError_t launch_linear(const LinProduct& p, void* workspace, hipStream_t s) {
  LinArgs a{};
  LinPacks js{};
  char* ws = static_cast<char*>(workspace);
  int jobs = 0, blocks = 0, K = 0;
  for (int b = 0; b < 2; ++b) {
    const LinSide d = lin_side(p, b);
    LinOperand& o = b ? a.b : a.a;
    o.rows = b ? p.N : p.M;
    o.p = static_cast<const uint16_t*>(b ? p.b : p.a);
    o.ld = b ? p.ldb : p.lda;
    if (!d.pack) continue;
    LinPack& j = js.job[jobs];
    j.src = o.p;
    j.lds = o.ld;
    j.out = reinterpret_cast<uint16_t*>(ws);
    j.ld = o.ld = d.ld;
    j.plane = o.plane = d.plane;
    j.rows = d.rows;
    j.cols = d.cols;
    j.turn = p.dtype == LIN_F32 && d.across;
    if (d.across && !j.turn) o.rows = (int)d.ld;
    j.tr = (d.rows + 63) / 64;
    j.tc = (d.cols + 63) / 64;
    js.start[jobs++] = blocks;
    blocks += j.tr * j.tc;
    o.p = j.out;
    ws += d.bytes;
  }
  for (int i = jobs; i < 3; ++i) js.start[i] = blocks;
  if (blocks) {
    if (p.dtype == LIN_F32) hipLaunchKernelGGL(lin_pack_kernel<true>, dim3(blocks), dim3(256), 0, s, js);
    else hipLaunchKernelGGL(lin_pack_kernel<false>, dim3(blocks), dim3(256), 0, s, js);
  }
  a.M = p.M; a.N = p.N; a.K = p.K;
  a.out_dtype = p.out_dtype; a.bias_dtype = p.bias_dtype;
  a.ldr = p.ldr; a.bias = p.bias; a.residual = p.residual; a.y = p.y; a.z = p.z;
  auto low = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  a.vec = p.N % 4 == 0 && p.ldr % 4 == 0 && (low(p.bias) | low(p.residual) | low(p.y) | low(p.z)) % 16 == 0;
  if (p.dtype == LIN_F32) lin_forms<LIN_F32>(a, p, s);
  else if (p.dtype == LIN_BF16) lin_forms<LIN_BF16>(a, p, s);
  else lin_forms<LIN_F16>(a, p, s);
  return hipGetLastError();
}

size_t linear_slope_workspace_bytes(const LinSlope& a) {
  return a.dbias ? (size_t)((a.M + SLOPE_ROWS - 1) / SLOPE_ROWS) * a.N * 4 : 0;
}
hipError_t launch_linear_slope(const LinSlope& a, void* workspace, hipStream_t s) {
  const int blocks = (a.M + SLOPE_ROWS - 1) / SLOPE_ROWS;
  float* part = a.dbias ? static_cast<float*>(workspace) : nullptr;
  const dim3 grid((a.N + 63) / 64, blocks);
  if (a.act == LIN_SILU) hipLaunchKernelGGL(lin_slope_kernel<LIN_SILU>, grid, dim3(256), 0, s, a, part);
  else if (a.act == LIN_GELU) hipLaunchKernelGGL(lin_slope_kernel<LIN_GELU>, grid, dim3(256), 0, s, a, part);
  else if (a.act == LIN_TANH) hipLaunchKernelGGL(lin_slope_kernel<LIN_TANH>, grid, dim3(256), 0, s, a, part);
  else hipLaunchKernelGGL(lin_slope_kernel<LIN_NONE>, grid, dim3(256), 0, s, a, part);
  if (part) hipLaunchKernelGGL(lin_bias_kernel, dim3((a.N + 255) / 256), dim3(256), 0, s, a, part, blocks);
  return hipGetLastError();
}

}  // namespace gdn2
