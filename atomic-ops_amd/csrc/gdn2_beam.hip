// Beam search's selection on gfx950: of the K V continuations of a group's K beams, the n of the
// highest score, ties to the lowest k V + v:
//   c[k][v] = score[k] + ((x[k][v] - m_k) - ln sum_v exp(x[k][v] - m_k)),   m_k = max_v x[k][v];
// a finished beam has one continuation, the end token at its own score; NaN counts as -inf.
//
// One pass over the logits (beam_part_kernel): a workgroup keeps a piece of a row in registers, forms
// its maximum and sum, and its n best entries, which are the row's best whatever the row's sum is.
// beam_join_kernel then has a few hundred entries a group: it joins the sums, forms the scores in
// float32 as written above, and selects among them.
// Selection is by one 64-bit key: the value's bits in an order that compares as integers, then the
// complement of the index, so the largest key is the highest value at its lowest index.
#include "gdn2_kernels.hpp"

namespace gdn2 {

typedef unsigned long long u64;

__device__ __forceinline__ float beam_value(float x) { return x != x ? -__builtin_inff() : x + 0.f; }   // (-0 -> 0)
__device__ __forceinline__ u64 beam_key(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(x), o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return (u64)o << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ float beam_key_value(u64 k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t beam_key_index(u64 k) { return 0xffffffffu - (uint32_t)k; }

__device__ __forceinline__ u64 shfl_xor64(u64 x, int m) {
  return (u64)__shfl_xor((uint32_t)(x >> 32), m) << 32 | __shfl_xor((uint32_t)x, m);
}
__device__ __forceinline__ u64 wave_max64(u64 x) {
#pragma unroll
  for (int m = WAVE / 2; m >= 1; m >>= 1) {
    const u64 y = shfl_xor64(x, m);
    x = y > x ? y : x;
  }
  return x;
}
__device__ __forceinline__ float wave_maxf(float x) {
#pragma unroll
  for (int m = WAVE / 2; m >= 1; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
  return x;
}
__device__ __forceinline__ float wave_sumf(float x) {
#pragma unroll
  for (int m = WAVE / 2; m >= 1; m >>= 1) x += __shfl_xor(x, m);
  return x;
}
// exp(x - m) for x <= m, 1 where x is m (also at +inf)
__device__ __forceinline__ float beam_exp(float x, float m) { return x == m ? 1.f : fast_exp(x - m); }

constexpr int BEAM_T = 256, BEAM_W = BEAM_T / WAVE;

// The largest key of the workgroup, in every thread.  best: 2 BEAM_W words used in turn by parity.
__device__ __forceinline__ u64 block_max64(u64 x, u64 (*best)[BEAM_W], int parity) {
  x = wave_max64(x);
  if (lane_id() == 0) best[parity][wave_id()] = x;
  __syncthreads();
  u64 y = best[parity][0];
#pragma unroll
  for (int i = 1; i < BEAM_W; ++i) y = best[parity][i] > y ? best[parity][i] : y;
  return y;
}

template <int XT, int VW>
__device__ __forceinline__ void beam_load(const BeamArgs& a, size_t row, int i, float* v) {
  if constexpr (XT == W4_F32) {
    const float* p = static_cast<const float*>(a.logits) + row * a.ld + i;
    if constexpr (VW == 4) {
      const float4 u = *reinterpret_cast<const float4*>(p);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
      v[0] = *p;
    }
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(a.logits) + row * a.ld + i;
    uint32_t h[VW];
    if constexpr (VW == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
    } else {
      h[0] = *p;
    }
#pragma unroll
    for (int j = 0; j < VW; ++j)
      v[j] = XT == W4_BF16 ? bf16_val(h[j]) : (float)__builtin_bit_cast(_Float16, (uint16_t)h[j]);
  }
}

// Row r = blockIdx.y, entries [split PT T, ...): maximum, sum and n best keys.  VW consecutive
// entries a thread and load.
template <int XT, int VW, int PT>
__global__ __launch_bounds__(BEAM_T) void beam_part_kernel(BeamArgs a) {
  __shared__ float sm[2 * BEAM_W];
  __shared__ u64 best[2][BEAM_W];
  const int tid = threadIdx.x, split = blockIdx.x, row = blockIdx.y;
  u64* out = a.cand + ((size_t)row * a.splits + split) * a.n;
  const float score = a.scores[row];
  const bool done = a.finished && a.finished[row];
  if (done || !(score > -__builtin_inff())) {
    // no logit of this row matters: -inf at its first entries (the end token's own score apart, which
    // the join forms)
    if (split == 0 && tid == 0) {
      a.part[2 * (size_t)row * a.splits] = 0.f;
      a.part[2 * (size_t)row * a.splits + 1] = 1.f;
    }
    for (int i = tid; i < a.n; i += BEAM_T)
      out[i] = split == 0 && i < a.V ? beam_key(-__builtin_inff(), i) : 0;
    if (split != 0 && tid == 0) {
      a.part[2 * ((size_t)row * a.splits + split)] = -__builtin_inff();
      a.part[2 * ((size_t)row * a.splits + split) + 1] = 0.f;
    }
    return;
  }
  float v[PT];
  const int c0 = split * PT * BEAM_T;
#pragma unroll
  for (int i = 0; i < PT / VW; ++i) {
    const int at = c0 + (i * BEAM_T + tid) * VW;
    if (at + VW <= a.V) {
      beam_load<XT, VW>(a, row, at, v + i * VW);
    } else {
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        v[i * VW + e] = -__builtin_inff();
        if (at + e < a.V) beam_load<XT, 1>(a, row, at + e, v + i * VW + e);
      }
    }
  }
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    v[i] = beam_value(v[i]);
    m = fmaxf(m, v[i]);
  }
  m = wave_maxf(m);
  if (lane_id() == 0) sm[wave_id()] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float s = 0.f;
  if (m > -__builtin_inff()) {
#pragma unroll
    for (int i = 0; i < PT; ++i) s += beam_exp(v[i], m);
  }
  s = wave_sumf(s);
  if (lane_id() == 0) sm[BEAM_W + wave_id()] = s;
  __syncthreads();
  if (tid == 0) {
    a.part[2 * ((size_t)row * a.splits + split)] = m;
    a.part[2 * ((size_t)row * a.splits + split) + 1] = (sm[BEAM_W] + sm[BEAM_W + 1]) + (sm[BEAM_W + 2] + sm[BEAM_W + 3]);
  }
  // n rounds: each takes the best of the threads' bests, whose owner looks for its next
  auto index = [&](int i) { return c0 + ((i / VW) * BEAM_T + tid) * VW + i % VW; };
  auto next = [&](u64 below) {
    u64 k = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const u64 y = index(i) < a.V ? beam_key(v[i], index(i)) : 0;
      k = y < below && y > k ? y : k;
    }
    return k;
  };
  u64 mine = next(~0ull);
  for (int i = 0; i < a.n; ++i) {
    const u64 top = block_max64(mine, best, i & 1);
    if (tid == 0) out[i] = top;
    if (top == mine) mine = next(top);
  }
}

// One workgroup a group: the scores of the parts' entries, and the n best of them.
constexpr int BEAM_PT2 = 8;                     // entries a thread keeps at a time
__global__ __launch_bounds__(BEAM_T) void beam_join_kernel(BeamArgs a) {
  __shared__ u64 best[2][BEAM_W];
  __shared__ u64 kept[BEAM_MAX_N];
  __shared__ float sM[BEAM_MAX_K], sL[BEAM_MAX_K];
  const int tid = threadIdx.x, b = blockIdx.x, per = a.splits * a.n;
  for (int k = wave_id(); k < a.K; k += BEAM_W) {
    const float* p = a.part + 2 * (size_t)(b * a.K + k) * a.splits;
    float m = -__builtin_inff(), s = 0.f;
    for (int i = lane_id(); i < a.splits; i += WAVE) m = fmaxf(m, p[2 * i]);
    m = wave_maxf(m);
    for (int i = lane_id(); i < a.splits; i += WAVE)
      if (p[2 * i] > -__builtin_inff()) s += p[2 * i + 1] * beam_exp(p[2 * i], m);
    s = wave_sumf(s);
    if (lane_id() == 0) {
      sM[k] = m;
      sL[k] = logf(s);
    }
  }
  for (int i = tid; i < a.n; i += BEAM_T) kept[i] = 0;
  __syncthreads();
  const int total = a.K * per;
  for (int c0 = 0; c0 < total; c0 += BEAM_PT2 * BEAM_T) {
    u64 key[BEAM_PT2 + 1];
#pragma unroll
    for (int i = 0; i < BEAM_PT2; ++i) {
      const int e = c0 + i * BEAM_T + tid;
      key[i] = 0;
      if (e < total) {
        const int k = e / per;
        const u64 x = a.cand[(size_t)b * total + e];
        if (x) {
          const uint32_t v = beam_key_index(x);
          const float xv = beam_key_value(x), score = a.scores[b * a.K + k];
          float c = -__builtin_inff();
          if (a.finished && a.finished[b * a.K + k]) c = (int)v == a.eos ? beam_value(score) : c;
          else if (xv > -__builtin_inff() && score > -__builtin_inff())
            c = beam_value(score + ((xv == sM[k] ? 0.f : xv - sM[k]) - sL[k]));
          key[i] = beam_key(c, (uint32_t)k * a.V + v);
        }
      }
    }
    // the best of the entries before, and a finished beam's end token where the parts left it out
    key[BEAM_PT2] = tid < a.n ? kept[tid] : 0;
    if (c0 == 0 && a.finished && tid >= a.n && tid - a.n < a.K && a.finished[b * a.K + tid - a.n] && a.eos >= a.n)
      key[BEAM_PT2] = beam_key(beam_value(a.scores[b * a.K + tid - a.n]), (uint32_t)(tid - a.n) * a.V + a.eos);
    __syncthreads();
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i <= BEAM_PT2; ++i) mine = key[i] > mine ? key[i] : mine;
    for (int i = 0; i < a.n; ++i) {
      const u64 top = block_max64(mine, best, i & 1);
      if (tid == 0) kept[i] = top;
      if (top == mine) {
        mine = 0;
#pragma unroll
        for (int j = 0; j <= BEAM_PT2; ++j) mine = key[j] < top && key[j] > mine ? key[j] : mine;
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < a.n; i += BEAM_T) {
    const u64 x = kept[i];
    const uint32_t at = beam_key_index(x);
    const int k = at / (uint32_t)a.V, v = at - (uint32_t)k * a.V;
    const size_t o = (size_t)b * a.n + i;
    a.tokens[o] = v;
    a.rows[o] = (int64_t)b * a.K + k;
    a.out_scores[o] = beam_key_value(x);
    if (a.out_finished) a.out_finished[o] = (a.finished && a.finished[b * a.K + k]) || v == a.eos;
  }
}

template <int XT, int VW>
static void beam_go(const BeamArgs& a, int pt, hipStream_t s) {
  const dim3 grid(a.splits, a.B * a.K);
  if (pt == 8) hipLaunchKernelGGL((beam_part_kernel<XT, VW, 8>), grid, dim3(BEAM_T), 0, s, a);
  else hipLaunchKernelGGL((beam_part_kernel<XT, VW, 32>), grid, dim3(BEAM_T), 0, s, a);
}

// Entries a thread keeps: 32 when that still gives every CU four workgroups, else 8.
int beam_per_thread(int rows, int V) { return (int64_t)rows * ((V + 32 * BEAM_T - 1) / (32 * BEAM_T)) >= 1024 ? 32 : 8; }
int beam_splits(int rows, int V) {
  const int per = beam_per_thread(rows, V) * BEAM_T;
  return (V + per - 1) / per;
}

hipError_t launch_beam(int dtype, const BeamArgs& a, hipStream_t s) {
  const int pt = beam_per_thread(a.B * a.K, a.V);
  if (dtype == W4_F32) a.vec ? beam_go<W4_F32, 4>(a, pt, s) : beam_go<W4_F32, 1>(a, pt, s);
  else if (dtype == W4_BF16) a.vec ? beam_go<W4_BF16, 8>(a, pt, s) : beam_go<W4_BF16, 1>(a, pt, s);
  else a.vec ? beam_go<W4_F16, 8>(a, pt, s) : beam_go<W4_F16, 1>(a, pt, s);
  hipLaunchKernelGGL(beam_join_kernel, dim3(a.B), dim3(BEAM_T), 0, s, a);
  return hipGetLastError();
}

}  // namespace gdn2
