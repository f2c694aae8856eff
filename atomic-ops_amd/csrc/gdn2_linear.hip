// Launches of the products (gdn2_linear.hpp): which kernel takes a product, operands that are copied for it, and the
// gradients of activation and bias.
#include "gdn2_linear.hpp"

namespace gdn2 {

// (instantiated in gdn2_linear_*.hip)
extern template void lin_forms<LIN_F32>(const LinArgs&, const LinPlan&, int, int, hipStream_t);
extern template void lin_forms<LIN_BF16>(const LinArgs&, const LinPlan&, int, int, hipStream_t);
extern template void lin_forms<LIN_F16>(const LinArgs&, const LinPlan&, int, int, hipStream_t);
extern template void lin_rows<LIN_F32>(const LinArgs&, const LinPlan&, int, bool, bool, hipStream_t);
extern template void lin_rows<LIN_BF16>(const LinArgs&, const LinPlan&, int, bool, bool, hipStream_t);
extern template void lin_rows<LIN_F16>(const LinArgs&, const LinPlan&, int, bool, bool, hipStream_t);

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
  constexpr int NP = F32 ? 3 : 1, LDT = 72;
  const int which = blockIdx.x >= (unsigned)js.start[1];
  const LinPack& j = js.job[which];
  const int b = blockIdx.x - js.start[which], r0 = b / j.tc * 64, c0 = b % j.tc * 64;
  __shared__ __attribute__((aligned(16))) uint16_t tile[NP][64][LDT];       // rows of out
  auto split = [&](uint32_t u, int ry, int cx) __attribute__((always_inline)) {
    uint16_t piece[NP];
    if constexpr (F32) {
      const float f = __uint_as_float(u), f1 = f - lin_top(f), f2 = f1 - lin_top(f1);
      piece[0] = (uint16_t)(u >> 16);
      piece[1] = (uint16_t)(__float_as_uint(f1) >> 16);
      piece[2] = (uint16_t)(__float_as_uint(f2) >> 16);
    } else {
      piece[0] = (uint16_t)u;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      if (j.turn) tile[p][cx][ry] = piece[p];
      else tile[p][ry][cx] = piece[p];
    }
  };
  if (c0 + 64 <= j.cols) {
    // four neighbouring values a lane, sixteen lanes to a row of src, or to a row of out (so that their writes meet no bank twice)
    const int y = j.turn ? threadIdx.x & 15 : threadIdx.x >> 4, x = 4 * (j.turn ? threadIdx.x >> 4 : threadIdx.x & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + 16 * i + y;
      const size_t at = (size_t)min(row, j.rows - 1) * j.lds + c0 + x;
      uint32_t v[4];
      lin_four<F32>(j.src, at, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) split(row < j.rows ? v[e] : 0u, 16 * i + y, x + e);
    }
  } else {
    // a row of src a wave at a time, a value a lane
    const int y = threadIdx.x >> 6, x = threadIdx.x & 63, col = c0 + x;
#pragma unroll
    for (int g = 0; g < 16; g += 8) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const size_t at = (size_t)min(r0 + 4 * (g + i) + y, j.rows - 1) * j.lds + min(col, j.cols - 1);
        if constexpr (F32) v[i] = static_cast<const uint32_t*>(j.src)[at];
        else v[i] = static_cast<const uint16_t*>(j.src)[at];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) split(r0 + 4 * (g + i) + y < j.rows && col < j.cols ? v[i] : 0u, 4 * (g + i) + y, x);
    }
  }
  __syncthreads();
  const int ro = j.turn ? c0 : r0, co = j.turn ? r0 : c0, rows = j.turn ? j.cols : j.rows;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int ry = threadIdx.x / 8 + 32 * i, row = ro + ry, col = co + 8 * (threadIdx.x & 7);
    if (row >= rows || (size_t)col >= j.ld) continue;        // (ld: a multiple of 8)
#pragma unroll
    for (int p = 0; p < NP; ++p)
      *reinterpret_cast<uint4*>(j.out + p * j.plane + (size_t)row * j.ld + col) = *reinterpret_cast<const uint4*>(&tile[p][ry][8 * (threadIdx.x & 7)]);
  }
}

// ---- dz = dy act'(z) and the bias' gradient ------------------------------------------------------------------------

// dz = v, and what its rounding leaves out in dz's second half (nothing of what is infinite or not a number there)
__device__ __forceinline__ float lin_left(int dt, float v) {
  const float r = dt == LIN_BF16 ? bf16_val((uint16_t)bf16_bits(v)) : (float)(_Float16)v;
  return fabsf(r) < INFINITY ? v - r : 0.f;
}
template <bool LOW>
__device__ __forceinline__ void lin_dz4(const LinSlope& a, size_t at, const float4& v) {
  lin_put4(a.dtype, a.dz, at, v);
  if constexpr (LOW)
    lin_put4(a.dtype, a.dz, (size_t)a.M * a.N + at, make_float4(lin_left(a.dtype, v.x), lin_left(a.dtype, v.y), lin_left(a.dtype, v.z), lin_left(a.dtype, v.w)));
}
template <bool LOW>
__device__ __forceinline__ void lin_dz(const LinSlope& a, size_t at, float v) {
  lin_put(a.dtype, a.dz, at, v);
  if constexpr (LOW) lin_put(a.dtype, a.dz, (size_t)a.M * a.N + at, lin_left(a.dtype, v));
}

// A workgroup takes 256 columns, a wave every fourth of `rows` rows, a lane four columns; part: sums of its rows, [row
// block][N].  vec: whole groups of four columns, and every pointer takes 16 bytes.
template <int ACT, bool LOW>
__global__ __launch_bounds__(256) void lin_slope_kernel(LinSlope a, float* part, int rows, int vec) {
  __shared__ float4 sums[4][64];
  const int l = lane_id(), w = wave_id(), n = blockIdx.x * 256 + 4 * l;
  const int64_t first = (int64_t)blockIdx.y * rows, last = min((int64_t)a.M, first + rows);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (n < a.N && vec) {
#pragma unroll 4
    for (int64_t m = first + w; m < last; m += 4) {
      const size_t at = (size_t)m * a.N + n;
      const float4 d = lin_get4(a.dy_dtype, a.dy, at);
      float f[4] = {d.x, d.y, d.z, d.w};
      if constexpr (ACT != LIN_NONE) {
        const float4 z = lin_get4(a.z_dtype, a.z, at);
        f[0] *= lin_slope<ACT>(z.x); f[1] *= lin_slope<ACT>(z.y); f[2] *= lin_slope<ACT>(z.z); f[3] *= lin_slope<ACT>(z.w);
      }
      if (a.dz) lin_dz4<LOW>(a, at, make_float4(f[0], f[1], f[2], f[3]));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += f[e];
    }
  } else if (n < a.N) {
    for (int64_t m = first + w; m < last; m += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n + e >= a.N) break;
        const size_t at = (size_t)m * a.N + n + e;
        float d = lin_get(a.dy_dtype, a.dy, at);
        if constexpr (ACT != LIN_NONE) d *= lin_slope<ACT>(lin_get(a.z_dtype, a.z, at));
        if (a.dz) lin_dz<LOW>(a, at, d);
        s[e] += d;
      }
  }
  sums[w][l] = make_float4(s[0], s[1], s[2], s[3]);
  __syncthreads();
  if (w || n >= a.N) return;
  const float4 x = sums[0][l], y = sums[1][l], u = sums[2][l], v = sums[3][l];
  const float f[4] = {(x.x + y.x) + (u.x + v.x), (x.y + y.y) + (u.y + v.y), (x.z + y.z) + (u.z + v.z), (x.w + y.w) + (u.w + v.w)};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) part[(size_t)blockIdx.y * a.N + n + e] = f[e];
}
// Without a bias the rows do not matter: dy, z and dz are arrays of `total` values, whatever a row's width.  vec: every
// pointer takes 16 bytes.
template <int ACT, bool LOW>
__global__ __launch_bounds__(256) void lin_slope_flat_kernel(LinSlope a, size_t total, int vec) {
  const size_t x = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256, whole = vec ? total / 4 : 0;
#pragma unroll 4
  for (size_t i = x; i < whole; i += step) {
    float4 d = lin_get4(a.dy_dtype, a.dy, 4 * i);
    if constexpr (ACT != LIN_NONE) {
      const float4 z = lin_get4(a.z_dtype, a.z, 4 * i);
      d.x *= lin_slope<ACT>(z.x); d.y *= lin_slope<ACT>(z.y); d.z *= lin_slope<ACT>(z.z); d.w *= lin_slope<ACT>(z.w);
    }
    lin_dz4<LOW>(a, 4 * i, d);
  }
  for (size_t i = 4 * whole + x; i < total; i += step) {
    float d = lin_get(a.dy_dtype, a.dy, i);
    if constexpr (ACT != LIN_NONE) d *= lin_slope<ACT>(lin_get(a.z_dtype, a.z, i));
    lin_dz<LOW>(a, i, d);
  }
}
// Sixteen groups of sixteen threads: a group's columns, every sixteenth block each
__global__ __launch_bounds__(256) void lin_bias_kernel(LinSlope a, const float* part, int blocks) {
  __shared__ float sums[16][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4, n = blockIdx.x * 16 + x;
  float s = 0.f;
  if (n < a.N)
#pragma unroll 8
    for (int i = y; i < blocks; i += 16) s += part[(size_t)i * a.N + n];
  sums[y][x] = s;
  __syncthreads();
  if (y || n >= a.N) return;
  for (int i = 1; i < 16; ++i) s += sums[i][x];
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

// float32, up to this many operations on the matrix cores' own float32, beyond as pieces that each wave cuts (us, own, cut:
// 512^3 10.6, 16.3; 2048 x 768 x 512 21.2, 29.0; 1024^3 28, 33; 2048 x 1024 x 768 46.5, 37.4; 4096 x 2048 x 1024 160, 103); in rows
// that 16-byte accesses do not take 300 x 677 x 811 17.9, 22.0; 500 x 999 x 1001 24.9, 27.0; 2047 x 767 x 513 43.8, 33.3
constexpr double LIN_DIRECT_MOST = 2.5e9, LIN_DIRECT_ODD = 1.2e9;
// float32 as pieces that a pass over memory has cut before (cut by each wave, by the pass, on one card): large tiles over a long sum, 4096^3
// 698, 667, but 4096 x 2048 x 1024 103, 128; odd rows, where an operand is used often enough, which M N / (M + N) says: 2048 x
// 4095 x 4097 754, 535 (1365); 16383 x 255 x 513 75, 69 (497); 2047 x 767 x 513 33.3, 34.9 (410); 218 x 8190 x 7626 265, 358 (212)
constexpr int64_t LIN_PACK_K = 4096, LIN_PACK_USE = 450;
// Few rows: whether every row of x and W takes 16-byte accesses
static bool lin_whole(const LinProduct& p) {
  const size_t e = p.dtype == LIN_F32 ? 4 : 8;
  return (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0 && p.lda % e == 0 && p.ldb % e == 0 &&
         p.K % 8 == 0 && (p.form == LIN_XWT || p.N % e == 0);
}
// float32: whether every row of the operands takes 16-byte accesses
static bool lin_float(const LinProduct& p) {
  const int ca = p.form == LIN_XTW ? p.M : p.K, cb = p.form == LIN_XWT ? p.K : p.N;
  return p.dtype == LIN_F32 && (reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16 == 0 && p.lda % 4 == 0 &&
         p.ldb % 4 == 0 && ca % 4 == 0 && cb % 4 == 0;
}
static LinPlan lin_plan(const LinProduct& p) {
  LinPlan r{0, LIN_MID, 1, 0, lin_float(p)};
  const int64_t cus = cu_count();
  auto tiles = [&](int64_t bm, int64_t bn) { return ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  auto split = [&](int64_t units, int64_t parts, int64_t most) {
    parts = parts > most ? most : parts;
    r.per = (int)((units + (parts < 1 ? 1 : parts) - 1) / (parts < 1 ? 1 : parts));
    r.parts = (int)((units + r.per - 1) / r.per);
  };
  if (p.form != LIN_XTW && p.M <= 8 && p.K <= (1 << 25)) {     // (parts are a grid's y)
    r.rows = p.M == 1 ? 1 : p.M == 2 ? 2 : p.M <= 4 ? 4 : 8;
    const int64_t e = p.dtype == LIN_F32 ? 4 : 8, wide = p.form == LIN_XWT ? 16 : lin_whole(p) ? LIN_ROWS_COLS * e : 64;
    const int64_t wgs = (p.N + wide - 1) / wide * ((p.M + r.rows - 1) / r.rows), eights = (p.K + 7) / 8;
    if (p.form == LIN_XW && !lin_whole(p)) {       // (by columns: 128 values a part and more, 1024 at most)
      const int64_t least = (p.K + LIN_COLUMNS_K - 1) / LIN_COLUMNS_K, most = (p.K + 127) / 128, parts = 2 * cus / wgs;
      split(eights, parts < least ? least : parts, most);
    } else {
      split(eights, (p.form == LIN_XW ? cus : 4 * cus) / wgs, p.K / 1024);
    }
    r.per *= 8;
    return r;
  }
  const int64_t blocks = (p.K + lin_bk(p.dtype) - 1) / lin_bk(p.dtype);
  const int64_t big = p.dtype == LIN_F32 ? tiles(256, 128) : tiles(256, 256), mid = tiles(128, 128), small = tiles(64, 64);
  // The large tiles are faster where they fill the chip (16 bits 1090 TFLOP/s against 850 to 1000, one workgroup a CU against
  // two; float32 233 against 190, one each), but the last round of them may be nearly empty: rounds, in units of a tile of
  // 128 x 128 a CU (7199 x 8996 x 3131 bfloat16: two rounds of 256 x 256 666 us, three of 128 x 128 588).
  auto rounds = [&](int64_t tiles, int64_t at_once) { return (tiles + at_once - 1) / at_once; };
  const double big_rounds = p.dtype == LIN_F32 ? rounds(big, cus) * 2 * 0.82 : rounds(big, cus) * 4 * 0.86;
  const double mid_rounds = p.dtype == LIN_F32 ? rounds(mid, cus) : rounds(mid, 2 * cus) * 2;
  const bool large = big * 4 >= cus * 3 && big_rounds <= mid_rounds;
  const bool pack = r.wide ? large && p.K >= LIN_PACK_K : (int64_t)p.M * p.N >= LIN_PACK_USE * ((int64_t)p.M + p.N);
  if (p.dtype == LIN_F32 && 2.0 * p.M * p.N * p.K <= (r.wide ? LIN_DIRECT_MOST : LIN_DIRECT_ODD)) {
    r.tile = LIN_DIRECT;
    split(blocks, small * 4 >= cus * 3 ? 1 : 2 * cus / small, blocks / 4);
  } else if (p.dtype == LIN_F32 && !pack) {
    r.tile = LIN_CUT;      // (two workgroups a CU of four waves; one of eight, whose addresses take more registers)
    split(blocks, (r.wide ? 2 : 1) * cus / mid, blocks / 4);
  } else if (large) {
    r.tile = LIN_BIG;
    split(blocks, 1, 1);
  } else if (mid >= cus || blocks * mid >= 16 * cus) {
    split(blocks, 2 * cus / mid, blocks / 4);
  } else {
    r.tile = LIN_SMALL;
    split(blocks, small * 4 >= cus * 3 ? 1 : 2 * cus / small, blocks / 8);
  }
  return r;
}
// What copies operands: a grid has fewer than 2^32 threads, 256 of them a tile of 64 x 64
static bool lin_packs_fit(const LinProduct& p, const LinPlan& r) {
  int64_t tiles = 0;
  for (int b = 0; b < 2 && !r.rows && r.tile < LIN_DIRECT; ++b)
    if (const LinSide d = lin_side(p, b); d.pack) tiles += ((int64_t)d.rows + 63) / 64 * (((int64_t)d.cols + 63) / 64);
  return tiles < (int64_t)1 << 24;
}
bool linear_fits(const LinProduct& p) {
  const int64_t m = p.M / 64 + 1, k = p.K / 64 + 1, n = p.N / 64 + 1;
  return (m + n) * k < (int64_t)1 << 24 || lin_packs_fit(p, lin_plan(p));
}
static size_t lin_parts_bytes(const LinProduct& p, const LinPlan& r) { return r.parts > 1 || p.halves ? up((size_t)r.parts * p.M * p.N * 4, 256) : 0; }

size_t linear_workspace_bytes(const LinProduct& p) {
  const LinPlan r = lin_plan(p);
  return (r.rows || r.tile >= LIN_DIRECT ? 0 : lin_side(p, false).bytes + lin_side(p, true).bytes) + lin_parts_bytes(p, r);
}

hipError_t launch_linear(const LinProduct& p, void* workspace, hipStream_t s) {
  const LinPlan r = lin_plan(p);
  LinArgs a{};
  auto low = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  a.M = p.M; a.N = p.N; a.K = p.K;
  a.out_dtype = p.out_dtype; a.bias_dtype = p.bias_dtype;
  a.ldr = p.ldr; a.bias = p.bias; a.residual = p.residual; a.y = p.y; a.z = p.z;
  a.vec = p.N % 8 == 0 && p.ldr % 8 == 0 && (low(p.bias) | low(p.residual) | low(p.y) | low(p.z)) % 16 == 0;
  a.z_dtype = p.z_f32 ? LIN_F32 : p.dtype;
  a.sums = r.parts > 1 || p.halves;
  a.halves = p.halves;
  a.pairs = !a.sums && !(p.z && p.z_f32) && p.dtype != LIN_F32 && p.out_dtype == p.dtype && (low(p.y) | low(p.z)) % 4 == 0;
  a.parts = r.parts;
  a.per = r.per;
  a.a = LinOperand{static_cast<const uint16_t*>(p.a), p.lda, 0, p.M};
  a.b = LinOperand{static_cast<const uint16_t*>(p.b), p.ldb, 0, p.N};
  char* ws = static_cast<char*>(workspace);
  if (r.rows) {
    a.part = reinterpret_cast<float*>(ws);
    const bool dots = p.form == LIN_XWT;
    const bool whole = lin_whole(p);
    if (p.dtype == LIN_F32) lin_rows<LIN_F32>(a, r, p.act, dots, whole, s);
    else if (p.dtype == LIN_BF16) lin_rows<LIN_BF16>(a, r, p.act, dots, whole, s);
    else lin_rows<LIN_F16>(a, r, p.act, dots, whole, s);
    return hipGetLastError();
  }
  LinPacks js{};
  int jobs = 0, blocks = 0;
  for (int b = 0; b < 2; ++b) {
    const LinSide d = lin_side(p, b);
    LinOperand& o = b ? a.b : a.a;
    if (!d.pack || r.tile >= LIN_DIRECT) continue;
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
  a.part = reinterpret_cast<float*>(ws);
  if (p.dtype == LIN_F32) lin_forms<LIN_F32>(a, r, p.form, p.act, s);
  else if (p.dtype == LIN_BF16) lin_forms<LIN_BF16>(a, r, p.form, p.act, s);
  else lin_forms<LIN_F16>(a, r, p.form, p.act, s);
  return hipGetLastError();
}

// rows of a workgroup: four workgroups a CU and more, 32 rows at least
static int slope_rows(const LinSlope& a) {
  const int64_t wide = (a.N + 255) / 256, want = (4 * (int64_t)cu_count() + wide - 1) / wide;
  int64_t rows = (a.M + want - 1) / want;
  rows = rows < 32 ? 32 : (rows + 3) / 4 * 4;
  return (int)(rows > a.M ? a.M : rows);
}
static int slope_blocks(const LinSlope& a) {
  const int rows = slope_rows(a);
  return (a.M + rows - 1) / rows;
}
size_t linear_slope_workspace_bytes(const LinSlope& a) { return a.dbias ? (size_t)slope_blocks(a) * a.N * 4 : 0; }
template <int ACT, bool LOW>
static void slope_go(const LinSlope& a, float* part, hipStream_t s) {
  auto low = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  const bool wide = (low(a.dy) | low(a.z) | low(a.dz)) % 16 == 0;
  if (!part) {
    const size_t total = (size_t)a.M * a.N, wgs = (total + 4095) / 4096;
    hipLaunchKernelGGL((lin_slope_flat_kernel<ACT, LOW>), dim3(wgs < 16384 ? wgs : 16384), dim3(256), 0, s, a, total, wide && (!LOW || total % 4 == 0));
    return;
  }
  const int rows = slope_rows(a), blocks = slope_blocks(a);
  hipLaunchKernelGGL((lin_slope_kernel<ACT, LOW>), dim3((a.N + 255) / 256, blocks), dim3(256), 0, s, a, part, rows, a.N % 4 == 0 && wide);
  hipLaunchKernelGGL(lin_bias_kernel, dim3((a.N + 15) / 16), dim3(256), 0, s, a, part, blocks);
}
template <bool LOW>
static void slope_act(const LinSlope& a, float* part, hipStream_t s) {
  if (a.act == LIN_SILU) slope_go<LIN_SILU, LOW>(a, part, s);
  else if (a.act == LIN_GELU) slope_go<LIN_GELU, LOW>(a, part, s);
  else if (a.act == LIN_TANH) slope_go<LIN_TANH, LOW>(a, part, s);
  else slope_go<LIN_NONE, LOW>(a, part, s);
}
hipError_t launch_linear_slope(const LinSlope& a, void* workspace, hipStream_t s) {
  float* part = a.dbias ? static_cast<float*>(workspace) : nullptr;
  a.low ? slope_act<true>(a, part, s) : slope_act<false>(a, part, s);
  return hipGetLastError();
}

}  // namespace gdn2
