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

static LinPlan lin_plan(const LinProduct& p) {
  LinPlan r{0, LIN_MID, 1, 0};
  const int64_t cus = cu_count();
  auto tiles = [&](int64_t bm, int64_t bn) { return ((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  auto split = [&](int64_t units, int64_t parts, int64_t most) {
    parts = parts > most ? most : parts;
    r.per = (int)((units + (parts < 1 ? 1 : parts) - 1) / (parts < 1 ? 1 : parts));
    r.parts = (int)((units + r.per - 1) / r.per);
  };
  if (p.form != LIN_XTW && p.M <= (p.dtype == LIN_F32 ? 32 : 8)) {
    r.rows = p.M == 1 ? 1 : p.M == 2 ? 2 : p.M <= 4 ? 4 : 8;
    const int64_t e = p.dtype == LIN_F32 ? 4 : 8, wide = p.form == LIN_XW ? LIN_ROWS_COLS * e : 16;
    const int64_t wgs = (p.N + wide - 1) / wide * ((p.M + r.rows - 1) / r.rows), eights = (p.K + 7) / 8;
    split(eights, (p.form == LIN_XW ? cus : 4 * cus) / wgs, p.K / 1024);
    r.per *= 8;
    return r;
  }
  const int64_t blocks = (p.K + lin_bk(p.dtype) - 1) / lin_bk(p.dtype);
  const int64_t big = p.dtype == LIN_F32 ? tiles(256, 128) : tiles(256, 256), mid = tiles(128, 128);
  if (big * 4 >= cus * 3) r.tile = LIN_BIG;
  split(blocks, r.tile == LIN_BIG ? 1 : 2 * cus / mid, blocks / 4);
  return r;
}
static size_t lin_parts_bytes(const LinProduct& p, const LinPlan& r) { return r.parts > 1 ? up((size_t)r.parts * p.M * p.N * 4, 256) : 0; }

size_t linear_workspace_bytes(const LinProduct& p) {
  const LinPlan r = lin_plan(p);
  return (r.rows ? 0 : lin_side(p, false).bytes + lin_side(p, true).bytes) + lin_parts_bytes(p, r);
}

hipError_t launch_linear(const LinProduct& p, void* workspace, hipStream_t s) {
  const LinPlan r = lin_plan(p);
  LinArgs a{};
  auto low = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  a.M = p.M; a.N = p.N; a.K = p.K;
  a.out_dtype = p.out_dtype; a.bias_dtype = p.bias_dtype;
  a.ldr = p.ldr; a.bias = p.bias; a.residual = p.residual; a.y = p.y; a.z = p.z;
  a.vec = p.N % 8 == 0 && p.ldr % 8 == 0 && (low(p.bias) | low(p.residual) | low(p.y) | low(p.z)) % 16 == 0;
  a.parts = r.parts;
  a.per = r.per;
  a.a = LinOperand{static_cast<const uint16_t*>(p.a), p.lda, 0, p.M};
  a.b = LinOperand{static_cast<const uint16_t*>(p.b), p.ldb, 0, p.N};
  char* ws = static_cast<char*>(workspace);
  if (r.rows) {
    a.part = reinterpret_cast<float*>(ws);
    const bool dots = p.form == LIN_XWT;
    const size_t e = p.dtype == LIN_F32 ? 4 : 8;
    const bool whole = (low(p.a) | low(p.b)) % 16 == 0 && p.lda % e == 0 && p.ldb % e == 0 && p.K % 8 == 0 && (dots || p.N % e == 0);
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
  a.part = reinterpret_cast<float*>(ws);
  if (p.dtype == LIN_F32) lin_forms<LIN_F32>(a, r, p.form, p.act, s);
  else if (p.dtype == LIN_BF16) lin_forms<LIN_BF16>(a, r, p.form, p.act, s);
  else lin_forms<LIN_F16>(a, r, p.form, p.act, s);
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
