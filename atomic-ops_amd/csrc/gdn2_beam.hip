// Beam search's selection on gfx950: of the K V continuations of a group's K beams, the n of the
// highest score, ties to the lowest k V + v:
//   c[k][v] = score[k] + ((x[k][v] - m_k) - ln sum_v exp(x[k][v] - m_k)),   m_k = max_v x[k][v];
// a finished beam has one continuation, the end token at its own score; NaN counts as -inf.
//
// One pass over the logits, bound by their bytes (beam_part_kernel): a workgroup keeps a piece of a row
// in registers, forms its maximum and sum, its n best entries by logit, and the best logit that it leaves
// out.  beam_join_kernel then has a few hundred entries a group: it joins the sums, forms the scores in
// float32 as written above, and selects among them.  Scores rise with the logits, so what a piece leaves out
// never scores above the n-th best, but may round to the same score at a lower index: where the best
// left out scores as much as the n-th best, the join looks through the piece's logits again.
//   64 groups of 8 beams, 131072 float32: 57 us (268 MB; the join 8 of them); 16 of 4, 32000 bfloat16: 13.7 us,
// the two launches' latency (56 and 13.2 without a look at what the pieces leave out); with n rounds of a maximum in place of a threshold 112 and 19 us.
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

// Over the wave's lanes, by lane moves within rows of 16, then the four rows' results
template <int ROR>
__device__ __forceinline__ float beam_ror(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 | ROR, 0xf, 0xf, true));
}
__device__ __forceinline__ float beam_lane(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}
__device__ __forceinline__ float wave_maxf(float x) {
  x = fmaxf(x, beam_ror<8>(x));
  x = fmaxf(x, beam_ror<4>(x));
  x = fmaxf(x, beam_ror<2>(x));
  x = fmaxf(x, beam_ror<1>(x));
  return fmaxf(fmaxf(beam_lane(x, 0), beam_lane(x, 16)), fmaxf(beam_lane(x, 32), beam_lane(x, 48)));
}
__device__ __forceinline__ float wave_sumf(float x) {
  x += beam_ror<8>(x);
  x += beam_ror<4>(x);
  x += beam_ror<2>(x);
  x += beam_ror<1>(x);
  return (beam_lane(x, 0) + beam_lane(x, 16)) + (beam_lane(x, 32) + beam_lane(x, 48));
}
// exp(x - m) for x <= m, 1 where x is m (also at +inf)
__device__ __forceinline__ float beam_exp(float x, float m) { return x == m ? 1.f : fast_exp(x - m); }
// sum over v[0 .. PT) of exp(v - m), m > -inf their maximum or above
template <int PT>
__device__ __forceinline__ float beam_exps(const float* v, float m) {
  float s = 0.f;
  if (m == __builtin_inff()) {                       // (uniform)
#pragma unroll
    for (int i = 0; i < PT; ++i) s += v[i] == m ? 1.f : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < PT; ++i) s += fast_exp(v[i] - m);
  }
  return s;
}

constexpr int BEAM_T = 256, BEAM_W = BEAM_T / WAVE;
constexpr int BEAM_LIST = 1024;                 // entries that a selection ranks

struct BeamShared {
  u64 list[BEAM_LIST + 8];
  u64 best[2][BEAM_W];
  float t[2 * BEAM_W];
  int count;
};

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
// The largest key of the workgroup, in every thread; best is used in turn by parity.
__device__ __forceinline__ u64 block_max64(u64 x, u64 (*best)[BEAM_W], int parity) {
  x = wave_max64(x);
  if (lane_id() == 0) best[parity][wave_id()] = x;
  __syncthreads();
  u64 y = best[parity][0];
#pragma unroll
  for (int i = 1; i < BEAM_W; ++i) y = best[parity][i] > y ? best[parity][i] : y;
  return y;
}

// The n best of the workgroup's entries, put(0, .), ..., put(n - 1, .) in order (0: no more entries), each by
// some thread, and with NEXT in put(n, .) a key of the next one's value (-inf or 0: none).  key(i), i < PT: a
// thread's entries, 0 for none; v[i]: their values; m: the largest v of the thread.
//   Of a wave's lanes' maxima, the n-th largest bounds the n best from below, and so does the least of the
// four waves' ceil(n / 4)-th largest (n entries at least reach either).  A few times n entries reach the
// higher of the two; they are gathered and ranked by counting.  Where more than BEAM_LIST reach it (long ties, rows that are almost
// all masked), n rounds of the largest key of all take their place.
//   With NEXT the bound is n + 1's, except where a quarter more of n would reach it for that (n = 8: 52.8 us in
// place of 50.1 for the parts of 64 x 8 x 131072): there a look at what lies below it finds the next one, if only n reach it.
template <bool NEXT, int PT, class Key, class Put>
__device__ __forceinline__ void beam_select(BeamShared& sh, const float* v, float m, int n, Key key, Put put) {
  const int tid = threadIdx.x, l = lane_id();
  const int reach = n + (NEXT && n % BEAM_W != 0), share = (reach + BEAM_W - 1) / BEAM_W, rounds = reach <= 16 ? reach : share;
  float t = 0.f, ts = 0.f;
  for (int i = 0; i < rounds; ++i) {
    t = wave_maxf(m);
    if (i + 1 == share) ts = t;
    const u64 at = __ballot(m == t);
    if (l == __ffsll(at) - 1) m = -__builtin_inff();
  }
  if (l == 0) {
    sh.t[wave_id()] = ts;
    sh.t[BEAM_W + wave_id()] = rounds == reach ? t : -__builtin_inff();
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  t = fmaxf(fminf(fminf(sh.t[0], sh.t[1]), fminf(sh.t[2], sh.t[3])),
            fmaxf(fmaxf(sh.t[4], sh.t[5]), fmaxf(sh.t[6], sh.t[7])));
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    bool in = v[i] >= t;
    if (__ballot(in) == 0) continue;                 // (uniform in the wave)
    const u64 k = in ? key(i) : 0;
    in = k != 0;
    const u64 who = __ballot(in);
    if (who == 0) continue;
    int base = 0;
    if (l == __ffsll(who) - 1) base = atomicAdd(&sh.count, __popcll(who));
    base = __shfl(base, __ffsll(who) - 1);
    const int at = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (in && at < BEAM_LIST) sh.list[at] = k;
  }
  __syncthreads();
  const int count = sh.count;
  if (count <= BEAM_LIST) {
    if (tid < 8) sh.list[count + tid] = 0;           // (ranked eight at a time)
    __syncthreads();
    for (int i = tid; i < count; i += BEAM_T) {
      const u64 k = sh.list[i];
      int rank = 0;
      for (int j = 0; j < count; j += 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += sh.list[j + e] > k;
      }
      if (rank < n + NEXT) put(rank, k);
    }
    for (int i = count + tid; i < n; i += BEAM_T) put(i, (u64)0);
    if (NEXT && count <= n) {
      float below = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PT; ++i) below = fmaxf(below, v[i] < t ? v[i] : -__builtin_inff());
      below = wave_maxf(below);
      if (l == 0) sh.t[wave_id()] = below;           // (t is read, two barriers ago)
      __syncthreads();
      if (tid == 0) put(n, beam_key(fmaxf(fmaxf(sh.t[0], sh.t[1]), fmaxf(sh.t[2], sh.t[3])), 0));
    }
    return;
  }
  auto next = [&](u64 below) {
    u64 k = 0;
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const u64 y = key(i);
      k = y < below && y > k ? y : k;
    }
    return k;
  };
  u64 mine = next(~0ull);
  for (int i = 0; i < n + NEXT; ++i) {
    const u64 top = block_max64(mine, sh.best, i & 1);
    if (tid == 0) put(i, top);
    if (top == mine) mine = next(top);
  }
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

// Row r = blockIdx.y, entries [split PT T, ...): maximum, sum, the n best keys and the next
// one's logit.  VW consecutive entries a thread and load.
template <int XT, int VW, int PT>
__global__ __launch_bounds__(BEAM_T) void beam_part_kernel(BeamArgs a) {
  __shared__ float sm[2 * BEAM_W];
  __shared__ BeamShared sh;
  const int tid = threadIdx.x, split = blockIdx.x, row = blockIdx.y;
  const size_t piece = (size_t)row * a.splits + split;
  u64* out = a.cand + piece * a.n;
  float* part = a.part + 4 * piece;
  const float score = a.scores[row];
  const bool done = a.finished && a.finished[row];
  if (done || !(score > -__builtin_inff())) {
    // no logit of this row matters: -inf at its first entries (the end token's own score apart, which
    // the join forms)
    if (tid == 0) {
      part[0] = split == 0 ? 0.f : -__builtin_inff();
      part[1] = split == 0 ? 1.f : 0.f;
      part[2] = -__builtin_inff();
    }
    for (int i = tid; i < a.n; i += BEAM_T)
      out[i] = split == 0 && i < a.V ? beam_key(-__builtin_inff(), i) : 0;
    return;
  }
  float v[PT];
  const int c0 = split * PT * BEAM_T;
  if (c0 + PT * BEAM_T <= a.V) {                     // (uniform: loads without a branch at each, 58 -> 56.5 us)
#pragma unroll
    for (int i = 0; i < PT / VW; ++i) beam_load<XT, VW>(a, row, c0 + (i * BEAM_T + tid) * VW, v + i * VW);
  } else {
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
  }
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    v[i] = beam_value(v[i]);
    m = fmaxf(m, v[i]);
  }
  const float mine = m;
  m = wave_maxf(m);
  if (lane_id() == 0) sm[wave_id()] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float s = wave_sumf(m > -__builtin_inff() ? beam_exps<PT>(v, m) : 0.f);
  if (lane_id() == 0) sm[BEAM_W + wave_id()] = s;
  beam_select<true, PT>(sh, v, mine, a.n, [&](int i) {
    const int at = c0 + ((i / VW) * BEAM_T + tid) * VW + i % VW;
    return at < a.V ? beam_key(v[i], at) : 0;
  }, [&](int i, u64 k) {
    if (i < a.n) out[i] = k;
    else part[2] = k ? beam_key_value(k) : -__builtin_inff();
  });
  if (tid == 0) {                                    // (behind the selection's barriers)
    part[0] = m;
    part[1] = (sm[BEAM_W] + sm[BEAM_W + 1]) + (sm[BEAM_W + 2] + sm[BEAM_W + 3]);
  }
}

// A group's results from its keys
__device__ __forceinline__ void beam_write(const BeamArgs& a, int b, const u64* kept) {
  for (int i = threadIdx.x; i < a.n; i += BEAM_T) {
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
// The score of an entry x of a beam whose logits have the maximum m and ln sum exp(x - m) = ls
__device__ __forceinline__ float beam_score(float score, float x, float m, float ls) {
  if (!(x > -__builtin_inff() && score > -__builtin_inff())) return -__builtin_inff();
  return beam_value(score + ((x == m ? 0.f : x - m) - ls));
}
// The logits' type's next value above (d = 1) or below (-1) x; nothing lies above +inf, nor below -inf
template <int XT>
__device__ __forceinline__ float beam_near(float x, int d) {
  if (x == 0.f && d < 0) d = -2;                     // (-0 is 0)
  if constexpr (XT == W4_F32) {
    const uint32_t u = __float_as_uint(x), o = (u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u)) + d;
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
  } else {
    const uint32_t u = XT == W4_BF16 ? __float_as_uint(x) >> 16 : __builtin_bit_cast(uint16_t, (_Float16)x);
    const uint32_t o = (u ^ ((u >> 15) ? 0xffffu : 0x8000u)) + d, y = o ^ ((o >> 15) ? 0x8000u : 0xffffu);
    return XT == W4_BF16 ? bf16_val(y) : (float)__builtin_bit_cast(_Float16, (uint16_t)y);
  }
}
// Whether a piece may have left out entries of the score c that come before others of this score: x is the
// best logit that it left out, of that score.  Not where all of the row's entries of that score are x, which
// are kept and left out by their indices.
template <int XT>
__device__ __forceinline__ bool beam_unsure(float score, float x, float m, float ls, float c) {
  return (x < m && beam_score(score, beam_near<XT>(x, 1), m, ls) == c) ||
         (x > -__builtin_inff() && beam_score(score, beam_near<XT>(x, -1), m, ls) == c);
}

// One workgroup a group: the scores of the parts' entries, and the n best of them.
constexpr int BEAM_PT2 = 8;                     // entries a thread keeps at a time
template <int XT>
__global__ __launch_bounds__(BEAM_T) void beam_join_kernel(BeamArgs a) {
  __shared__ BeamShared sh;
  __shared__ u64 kept[BEAM_MAX_N];
  __shared__ float sM[BEAM_MAX_K], sL[BEAM_MAX_K], sS[BEAM_MAX_K];
  __shared__ uint8_t sF[BEAM_MAX_K];
  __shared__ float sAgain[BEAM_W];
  __shared__ u64 sPieces[BEAM_W];
  const int tid = threadIdx.x, b = blockIdx.x, per = a.splits * a.n, total = a.K * per;
  const u64* cand = a.cand + (size_t)b * total;
  u64 x[BEAM_PT2];
  auto fetch = [&](int c0) {
#pragma unroll
    for (int i = 0; i < BEAM_PT2; ++i) x[i] = c0 + i * BEAM_T + tid < total ? cand[c0 + i * BEAM_T + tid] : 0;
  };
  fetch(0);
  const float4* part = reinterpret_cast<const float4*>(a.part) + (size_t)b * a.K * a.splits;
  float again = __builtin_nanf("");                  // the wave's rows' highest score that a piece left out
  for (int k = wave_id(); k < a.K; k += BEAM_W) {
    float m = -__builtin_inff(), s = 0.f, next = -__builtin_inff();
    const float score = a.scores[b * a.K + k];
    const bool done = a.finished && a.finished[b * a.K + k];
    for (int i = lane_id(); i < a.splits; i += WAVE) {
      const float4 p = part[k * a.splits + i];
      const float mi = p.x, si = p.y;
      next = fmaxf(next, p.z);
      if (mi > m) {
        s = s * beam_exp(m, mi) + si;
        m = mi;
      } else if (mi > -__builtin_inff()) {
        s += si * beam_exp(mi, m);
      }
    }
    const float top = wave_maxf(m);
    s = wave_sumf(m > -__builtin_inff() ? s * beam_exp(m, top) : 0.f);
    const float ls = logf(s);
    next = wave_maxf(next);
    if (!done && score > -__builtin_inff()) {
      // (masked tokens alone are left out in order, unless logits above theirs have no score either)
      const float c = beam_score(score, next, top, ls);
      if (!(again >= c) && (next > -__builtin_inff() || beam_unsure<XT>(score, next, top, ls, c))) again = c;
    }
    if (lane_id() == 0) {
      sM[k] = top;
      sL[k] = ls;
      sS[k] = score;
      sF[k] = done;
    }
  }
  if (lane_id() == 0) sAgain[wave_id()] = again;
  for (int i = tid; i < a.n; i += BEAM_T) kept[i] = 0;
  __syncthreads();
  // the entries of this pass and the n best before them
  auto select = [&](u64* key) __attribute__((always_inline)) {
    float val[BEAM_PT2 + 1], m = -__builtin_inff();
#pragma unroll
    for (int i = 0; i <= BEAM_PT2; ++i) {
      val[i] = key[i] ? beam_key_value(key[i]) : -__builtin_inff();
      m = fmaxf(m, val[i]);
    }
    __syncthreads();                                 // (kept is read)
    beam_select<false, BEAM_PT2 + 1>(sh, val, m, a.n, [&](int i) { return key[i]; }, [&](int i, u64 k) { kept[i] = k; });
    __syncthreads();
  };
  for (int c0 = 0; c0 < total; c0 += BEAM_PT2 * BEAM_T) {
    u64 key[BEAM_PT2 + 1];
    if (c0) fetch(c0);
#pragma unroll
    for (int i = 0; i < BEAM_PT2; ++i) {
      key[i] = 0;
      if (x[i]) {
        const int k = (c0 + i * BEAM_T + tid) / per;
        const uint32_t v = beam_key_index(x[i]);
        const float c = sF[k] ? ((int)v == a.eos ? beam_value(sS[k]) : -__builtin_inff())
                              : beam_score(sS[k], beam_key_value(x[i]), sM[k], sL[k]);
        key[i] = beam_key(c, (uint32_t)k * a.V + v);
      }
    }
    // the best of the entries before, and a finished beam's end token where the parts left it out
    key[BEAM_PT2] = tid < a.n ? kept[tid] : 0;
    const int fk = tid - a.n;
    if (c0 == 0 && fk >= 0 && fk < a.K && sF[fk] && a.eos >= a.n)
      key[BEAM_PT2] = beam_key(beam_value(sS[fk]), (uint32_t)fk * a.V + a.eos);
    select(key);
  }
  // Equal scores on both sides of a piece's n-th place, the group's n-th score among them: what such pieces
  // left out of this score, pieces in the order of their indices.
  const float least = beam_key_value(kept[a.n - 1]);
  bool more = sAgain[0] == least || sAgain[1] == least || sAgain[2] == least || sAgain[3] == least;
  const int pieces = a.K * a.splits;
  for (int p0 = 0; more && p0 < pieces; p0 += BEAM_T) {
    bool mine = false;
    if (p0 + tid < pieces) {
      const int p = p0 + tid, k = p / a.splits;
      const float x = part[p].z, c = beam_score(sS[k], x, sM[k], sL[k]);
      mine = !sF[k] && sS[k] > -__builtin_inff() && c == least && beam_unsure<XT>(sS[k], x, sM[k], sL[k], c);
    }
    const u64 who = __ballot(mine);
    __syncthreads();                                 // (the pieces before are read)
    if (lane_id() == 0) sPieces[wave_id()] = who;
    __syncthreads();
    for (int i = 0; more && i < BEAM_T; ++i) {
      if (!(sPieces[i / WAVE] >> (i % WAVE) & 1)) continue;
      const int p = p0 + i, k = p / a.splits, first = (p - k * a.splits) * a.piece, end = min(first + a.piece, a.V);
      const u64 last = cand[(size_t)p * a.n + a.n - 1];
      // (n of this score or above lie before this piece)
      more = (uint32_t)k * a.V + first <= beam_key_index(kept[a.n - 1]);
      for (int c0 = first; more && c0 < end; c0 += BEAM_PT2 * BEAM_T) {
        u64 key[BEAM_PT2 + 1];
#pragma unroll
        for (int j = 0; j < BEAM_PT2; ++j) {
          const int at = c0 + j * BEAM_T + tid;
          key[j] = 0;
          if (at < end) {
            float x;
            beam_load<XT, 1>(a, (size_t)b * a.K + k, at, &x);
            x = beam_value(x);
            if (beam_key(x, at) < last && beam_score(sS[k], x, sM[k], sL[k]) == least)
              key[j] = beam_key(least, (uint32_t)k * a.V + at);
          }
        }
        key[BEAM_PT2] = tid < a.n ? kept[tid] : 0;
        select(key);
      }
    }
  }
  beam_write(a, b, kept);
}

// A small vocabulary in one launch: one workgroup a group, R rows a wave and PER entries a lane and row,
// all kept in registers with their scores.  One group of 4 beams, 256 float32: 3.2 us, a launch's latency
// (a call 11.2 us in two launches, 7.3 in one).
template <int XT, int R, int PER>
__global__ __launch_bounds__(BEAM_T) void beam_small_kernel(BeamArgs a) {
  __shared__ BeamShared sh;
  __shared__ u64 kept[BEAM_MAX_N];
  const int l = lane_id(), w = wave_id(), b = blockIdx.x;
  float v[R * PER], score[R], best = -__builtin_inff();
  bool done[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int k = w + BEAM_W * r;
    const size_t row = (size_t)b * a.K + min(k, a.K - 1);
    score[r] = k < a.K ? a.scores[row] : -__builtin_inff();
    done[r] = a.finished && a.finished[row];
#pragma unroll
    for (int j = 0; j < PER; ++j) beam_load<XT, 1>(a, row, min(j * WAVE + l, a.V - 1), v + r * PER + j);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float* x = v + r * PER;
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      x[j] = j * WAVE + l < a.V ? beam_value(x[j]) : -__builtin_inff();
      m = fmaxf(m, x[j]);
    }
    m = wave_maxf(m);
    const float ls = logf(wave_sumf(m > -__builtin_inff() ? beam_exps<PER>(x, m) : 0.f));
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      x[j] = done[r] ? (j * WAVE + l == a.eos ? beam_value(score[r]) : -__builtin_inff()) : beam_score(score[r], x[j], m, ls);
      best = fmaxf(best, x[j]);
    }
  }
  beam_select<false, R * PER>(sh, v, best, a.n, [&](int i) {
    const int k = w + BEAM_W * (i / PER), at = i % PER * WAVE + l;
    return k < a.K && at < a.V ? beam_key(v[i], (uint32_t)k * a.V + at) : 0;
  }, [&](int i, u64 k) { kept[i] = k; });
  __syncthreads();
  beam_write(a, b, kept);
}

template <int XT, int VW>
static void beam_go(const BeamArgs& a, int pt, hipStream_t s) {
  const dim3 grid(a.splits, a.B * a.K);
  if (pt == 8) hipLaunchKernelGGL((beam_part_kernel<XT, VW, 8>), grid, dim3(BEAM_T), 0, s, a);
  else hipLaunchKernelGGL((beam_part_kernel<XT, VW, 32>), grid, dim3(BEAM_T), 0, s, a);
}

template <int XT>
static void beam_small_go(const BeamArgs& a, hipStream_t s) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(a.B), dim3(BEAM_T), 0, s, a); };
  if (a.K <= 4) a.V <= 256 ? go(beam_small_kernel<XT, 1, 4>) : go(beam_small_kernel<XT, 1, 32>);
  else if (a.K <= 8) a.V <= 256 ? go(beam_small_kernel<XT, 2, 4>) : go(beam_small_kernel<XT, 2, 16>);
  else go(beam_small_kernel<XT, 4, 8>);
}

// Whether a group's logits fit one workgroup's registers: one launch in place of two.
static bool beam_small(int K, int V) { return K <= 4 ? V <= 2048 : K <= 8 ? V <= 1024 : K <= 16 && V <= 512; }
// Entries a thread keeps: 32 when that still gives every CU four workgroups, else 8.
static int beam_per_thread(int rows, int V) { return (int64_t)rows * ((V + 32 * BEAM_T - 1) / (32 * BEAM_T)) >= 1024 ? 32 : 8; }
int beam_piece(int rows, int V) { return beam_per_thread(rows, V) * BEAM_T; }
int beam_splits(int rows, int K, int V) {
  if (beam_small(K, V)) return 0;
  const int per = beam_piece(rows, V);
  return (V + per - 1) / per;
}

hipError_t launch_beam(int dtype, const BeamArgs& a, hipStream_t s) {
  if (a.splits == 0) {
    dtype == W4_F32 ? beam_small_go<W4_F32>(a, s) : dtype == W4_BF16 ? beam_small_go<W4_BF16>(a, s) : beam_small_go<W4_F16>(a, s);
    return hipGetLastError();
  }
  const int pt = beam_per_thread(a.B * a.K, a.V);
  if (dtype == W4_F32) a.vec ? beam_go<W4_F32, 4>(a, pt, s) : beam_go<W4_F32, 1>(a, pt, s);
  else if (dtype == W4_BF16) a.vec ? beam_go<W4_BF16, 8>(a, pt, s) : beam_go<W4_BF16, 1>(a, pt, s);
  else a.vec ? beam_go<W4_F16, 8>(a, pt, s) : beam_go<W4_F16, 1>(a, pt, s);
  auto join = dtype == W4_F32 ? beam_join_kernel<W4_F32> : dtype == W4_BF16 ? beam_join_kernel<W4_BF16> : beam_join_kernel<W4_F16>;
  hipLaunchKernelGGL(join, dim3(a.B), dim3(BEAM_T), 0, s, a);
  return hipGetLastError();
}

}  // namespace gdn2
