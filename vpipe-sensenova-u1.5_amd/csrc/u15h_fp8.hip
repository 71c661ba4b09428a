// u15h_fp8.hip -- gfx950 kernels of the fp8 tier: OCP e4m3 codes with one
// f32 scale for each block of 128.
//
// A block of activations is 128 columns of one row, a block of weights 128
// rows x 128 columns; the last block of a row or column may be shorter.
// For the values v of a block, all in f32:
//     a = max |v|,   s = max(a / 448, 2^-126),   code = e4m3(v * (1 / s)).
// 448 is e4m3's largest value.  The division and the reciprocal are correctly
// rounded, so |v| * (1 / s) <= 448 * (1 + 2^-24)^3, which rounds to 448: no
// clamp.  The least scale keeps 1 / s finite; a block of zeros has it, and
// codes 0.  max |v| is taken over the bit patterns, which order NaN above
// infinity above every finite value: a block that holds a NaN gets the scale
// NaN, one that holds an infinity the scale infinity and codes that are 0 or
// NaN, so its restored values are NaN either way and no such block passes for
// a finite one.
//
// Activation scales are stored block-major, sa[block][row]: the GEMM's tile
// of rows reads each block's scales as one contiguous run.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "u15h_internal.h"

namespace u15h {
namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kRsrcWord3 = 0x00020000;      // raw buffer, 32-bit data format
constexpr int kOobOffset = 0x40000000;      // any offset past every resource
constexpr int kNonTemporal = 2;             // a load's or store's cache policy
constexpr int kRowGroups = 16384;           // of a launch's y dimension
constexpr float kFp8Top = 448.0f;
constexpr float kFp8Least = 0x1p-126f;

// A buffer resource over [base, base + bytes): loads past it read zero,
// stores past it are dropped.  Explicitly wave-uniform, so it stays in SGPRs.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t
make_rsrc(const void* base, int bytes)
{
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  const int n = __builtin_amdgcn_readfirstlane(bytes);
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0, n, kRsrcWord3);
}

// A wave-uniform value made explicitly so: it stays in SGPRs.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <class T>
__device__ __forceinline__ T*
uniform(T* p)
{
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<T*>(((uint64_t)hi << 32) | lo);
}

// Two floats as packed bf16 (lo in the low half), round to nearest even.
__device__ __forceinline__ uint32_t
pack_bf16x2(float lo, float hi)
{
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_convertvector((f32x2_t){lo, hi}, bf16x2_t));
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// ---- the quantiser's steps ---------------------------------------------------
__device__ __forceinline__ uint32_t
max_bits(uint32_t m, float v)
{
  return max(m, __float_as_uint(v) & 0x7fffffffu);
}

// The largest over the 16 lanes of a row (DPP rotations: no LDS).
__device__ __forceinline__ uint32_t
row_max(uint32_t v)
{
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

__device__ __forceinline__ float
block_scale(uint32_t bits)
{
  const float s = __uint_as_float(bits) / kFp8Top;
  return s < kFp8Least ? kFp8Least : s;      // (a NaN stays)
}

// Eight values' codes.
__device__ __forceinline__ u32x2_t
codes8(const float (&v)[8], float inv)
{
  u32x2_t o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, c, true);
    o[h] = (uint32_t)c;
  }
  return o;
}

__device__ __forceinline__ void
unpack8(const u32x4_t& w, float (&v)[8])
{
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = bf16_lo(w[e]);
    v[2 * e + 1] = bf16_hi(w[e]);
  }
}

__device__ __forceinline__ u32x4_t
pack8(const float (&v)[8])
{
  return u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                 pack_bf16x2(v[6], v[7])};
}

// silu(g) * u in f32: g * rcp(1 + 2^(-g log2 e)) with the hardware's exp2 and
// reciprocal (about 1 ulp each).  The reciprocal loses results below 2^-126, as
// gates below -87.3 have; there 1 + e^g is 1, and silu(g) u = g e^g u is
// multiplied up from four quarters of e^g, each a normal number down to -349,
// so that nothing vanishes that f32 can hold (silu(-88) is -5e-37).  One test
// for a lane's eight gates (0.3 of 43 us at 4224 rows of 12288); which form a
// value takes is its own gate's matter.
constexpr float kFarGate = -87.0f;

__device__ __forceinline__ void
swiglu8(float (&v)[8], const float (&u)[8])
{
  float g[8];
  uint32_t least = 0;          // as bits, which order negative gates downwards
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    g[e] = v[e];
    least = max(least, __float_as_uint(g[e]));
    const float x = __builtin_amdgcn_exp2f(g[e] * -1.4426950408889634f);
    v[e] = (g[e] * __builtin_amdgcn_rcpf(1.0f + x)) * u[e];
  }
  if (__builtin_expect(least > __float_as_uint(kFarGate), 0)) {
    asm volatile("");          // keeps it a branch
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = __builtin_amdgcn_exp2f(g[e] * (0.25f * 1.4426950408889634f));
      if (g[e] < kFarGate) { v[e] = ((g[e] * t) * t) * ((u[e] * t) * t); }
    }
  }
}

// ---- rows: codes and block-major scales --------------------------------------
// One workgroup of four waves per 4 RPW rows x 512 columns.  A wave reads 512
// columns of a row at a time, lane l columns 8 l..8 l + 7, so a block of 128 is
// 16 neighbouring lanes; all of its loads issue first (two: RPW rows of one
// operand, or a row of two).  The scales of the workgroup's rows are gathered
// in LDS and written as runs of 4 RPW.
// Bound by memory: 2 bytes read (4 for SwiGLU) and 1 + 1/32 written per value.
// 4224 rows of 12288 take 26 us (6.0 TB/s; SwiGLU 43 us, 6.1 TB/s, with h 62
// us, 5.9 TB/s), four rows of 4096 2.3 us, a launch.  Workgroups walk a row's
// columns first, so those that run together read whole rows: walking the rows
// first takes a fifth more time (SwiGLU an eighth).  The operands are read once
// and for the last time, so past the caches' other lines (non-temporal): 1.0
// (1.2) us of it.  The codes are stored plainly: stored past the caches these
// take 2 us less and the product that reads them 2 more.
template <bool SWIGLU, int RPW>
__global__ __launch_bounds__(256) void
fp8_quant_rows_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ up, int rows,
                      int K, uint16_t* __restrict__ h, uint8_t* __restrict__ q,
                      float* __restrict__ sc)
{
  constexpr int R = 4 * RPW;
  __shared__ float scales[4][R];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int group = blockIdx.z * kRowGroups + blockIdx.y;
  const int row0 = group * R, col = blockIdx.x * 512 + lane * 8;
  if (row0 >= rows) { return; }
  const int valid = min(R, rows - row0);
  const int oob = col < K ? 0 : kOobOffset;
  const size_t base = (size_t)row0 * K;
  const __amdgpu_buffer_rsrc_t xs = make_rsrc(x + base, valid * K * 2);
  const __amdgpu_buffer_rsrc_t us = make_rsrc(SWIGLU ? up + base : x + base, valid * K * 2);
  const __amdgpu_buffer_rsrc_t qs = make_rsrc(q + base, valid * K);
  u32x4_t xv[RPW], uv[SWIGLU ? RPW : 1];
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int at = (wave * RPW + i) * K + col;
    xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xs, at * 2 + oob, 0, kNonTemporal);
    if constexpr (SWIGLU) {
      uv[i] = __builtin_amdgcn_raw_buffer_load_b128(us, at * 2 + oob, 0, kNonTemporal);
    }
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int at = (wave * RPW + i) * K + col;
    float v[8];
    unpack8(xv[i], v);
    if constexpr (SWIGLU) {
      float u[8];
      unpack8(uv[i], u);
      swiglu8(v, u);
      if (h != nullptr) {
        const __amdgpu_buffer_rsrc_t hs = make_rsrc(h + base, valid * K * 2);
        __builtin_amdgcn_raw_buffer_store_b128(pack8(v), hs, at * 2 + oob, 0, 0);
      }
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) { m = max_bits(m, v[e]); }
    const float s = block_scale(row_max(m));
    __builtin_amdgcn_raw_buffer_store_b64(codes8(v, 1.0f / s), qs, at + oob, 0, 0);
    if ((lane & 15) == 0) { scales[lane >> 4][wave * RPW + i] = s; }
  }
  __syncthreads();
  const int nb = (K + kFp8Block - 1) / kFp8Block;
  for (int t = threadIdx.x; t < 4 * R; t += 256) {
    const int b = blockIdx.x * 4 + t / R, r = t % R;
    if (b < nb && r < valid) { sc[(size_t)b * rows + row0 + r] = scales[t / R][r]; }
  }
}

// ---- weights: a scale per 128 x 128 ------------------------------------------
// One workgroup of four waves per block; a wave reads four rows' 256 bytes at a
// time (lane l: row l / 16, columns 8 (l % 16)..), eight such reads in flight.
// Bound by memory: 3 bytes per value, 12288 x 4096 in 26.4 us (5.7 TB/s).  A
// weight is read once and its codes wait for a later use, so both go past the
// caches' other lines (non-temporal); plainly it takes a tenth more.
__global__ __launch_bounds__(256) void
fp8_quant_blocks_kernel(const uint16_t* __restrict__ w, int N, int K, uint8_t* __restrict__ q,
                        float* __restrict__ sc)
{
  __shared__ uint32_t red[4];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int n0 = blockIdx.y * kFp8Block, col = blockIdx.x * kFp8Block + (lane & 15) * 8;
  const int valid = min(kFp8Block, N - n0);
  const int oob = col < K ? 0 : kOobOffset;
  const size_t base = (size_t)n0 * K;
  const __amdgpu_buffer_rsrc_t ws = make_rsrc(w + base, valid * K * 2);
  const __amdgpu_buffer_rsrc_t qs = make_rsrc(q + base, valid * K);
  const int at = (wave * 4 + (lane >> 4)) * K + col;
  u32x4_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = __builtin_amdgcn_raw_buffer_load_b128(ws, (at + i * 16 * K) * 2 + oob, 0, kNonTemporal);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m = max_bits(max_bits(m, bf16_lo(v[i][e])), bf16_hi(v[i][e]));
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { m = max(m, (uint32_t)__shfl_xor((int)m, o)); }
  if (lane == 0) { red[wave] = m; }
  __syncthreads();
  const float s = block_scale(max(max(red[0], red[1]), max(red[2], red[3])));
  const float inv = 1.0f / s;
  if (threadIdx.x == 0) { sc[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = s; }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f[8];
    unpack8(v[i], f);
    __builtin_amdgcn_raw_buffer_store_b64(codes8(f, inv), qs, at + i * 16 * K + oob, 0,
                                         kNonTemporal);
  }
}

// ---- the residual add, RMSNorm and codes -------------------------------------
// One workgroup per row, WPR waves holding the row in registers (dim <= 512 WPR
// CPL): chunk i of wave p, lane l is columns 8 (64 (i WPR + p) + l).., so a
// block of 128 is 16 neighbouring lanes of one chunk.
//   r = bf16(x + d) (stored to x_out),   n = (r * inv) * w in f32,
//   inv = rsqrt(sum(r^2) / dim + eps), the sum in f32: lane partials, the wave
//   by xor shuffles, the row through LDS.
// The codes are those of n itself, rounded once; y, where wanted, is bf16(n).
// Every store of a row follows all of its loads, so x_out may be x.
// Bound by memory: with the add 7 bytes per value (4 in, 2 and the code out),
// 4224 rows of 4096 in 22.5 us (5.4 TB/s; with y too 26.9 us, 5.8 TB/s);
// without it 3 bytes, 13.3 us (3.9 TB/s; with y 18.3 us, 4.8 TB/s).  Each row's
// workgroup also reads the weights from L2, as many bytes as its row: with them
// the four forms move 6.5 to 7.1 TB/s.  x, d and r go past the caches' other
// lines (non-temporal): d is read for the last time and x's or r's next reader
// is half a layer away; plainly each takes a twelfth more.  A row
// of 4096 has eight waves with the add, two loads each as it has with four waves
// without it: eight against four are level with the add (one row and 4224) and a
// tenth slower without.
template <int WPR, int CPL, bool ADD>
__global__ __launch_bounds__(64 * WPR) void
fp8_norm_kernel(const Fp8NormArgs A)
{
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x, dim = A.dim;
  const size_t base = (size_t)r * dim;
  const __amdgpu_buffer_rsrc_t xs = make_rsrc(A.x + base, dim * 2);
  const __amdgpu_buffer_rsrc_t ws = make_rsrc(r < A.m_und ? A.w_und : A.w_gen, dim * 2);
  u32x4_t v[CPL], g[CPL];
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int c = (i * WPR + part) * 64 + lane;
    v[i] = __builtin_amdgcn_raw_buffer_load_b128(xs, c * 16, 0, kNonTemporal);
    g[i] = __builtin_amdgcn_raw_buffer_load_b128(ws, c * 16, 0, 0);
  }
  if constexpr (ADD) {
    const __amdgpu_buffer_rsrc_t ds = make_rsrc(A.d + base, dim * 2);
    const __amdgpu_buffer_rsrc_t os = make_rsrc(A.x_out + base, dim * 2);
    u32x4_t d[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      d[i] = __builtin_amdgcn_raw_buffer_load_b128(ds, ((i * WPR + part) * 64 + lane) * 16, 0,
                                                   kNonTemporal);
    }
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][e] = pack_bf16x2(bf16_lo(v[i][e]) + bf16_lo(d[i][e]),
                              bf16_hi(v[i][e]) + bf16_hi(d[i][e]));
      }
      __builtin_amdgcn_raw_buffer_store_b128(v[i], os, ((i * WPR + part) * 64 + lane) * 16, 0,
                                             kNonTemporal);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ss += bf16_lo(v[i][e]) * bf16_lo(v[i][e]);
      ss += bf16_hi(v[i][e]) * bf16_hi(v[i][e]);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { ss += __shfl_xor(ss, o); }
  if constexpr (WPR > 1) {
    __shared__ float red[WPR];
    if (lane == 0) { red[part] = ss; }
    __syncthreads();
    ss = red[0];
#pragma unroll
    for (int p = 1; p < WPR; ++p) { ss += red[p]; }
  }
  const float inv = rsqrtf(ss / (float)dim + A.eps);
  const __amdgpu_buffer_rsrc_t qs = make_rsrc(A.q + base, dim);
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int c = (i * WPR + part) * 64 + lane;
    float n[8], w[8];
    unpack8(v[i], n);
    unpack8(g[i], w);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      n[e] = (n[e] * inv) * w[e];
      m = max_bits(m, n[e]);
    }
    // columns past the row do not count (0 * inv * 0 is a NaN where inv is
    // infinite), and no store of theirs is kept
    const float s = block_scale(row_max(c * 8 < dim ? m : 0u));
    __builtin_amdgcn_raw_buffer_store_b64(codes8(n, 1.0f / s), qs, c * 8, 0, 0);
    if (A.y != nullptr) {
      const __amdgpu_buffer_rsrc_t ys = make_rsrc(A.y + base, dim * 2);
      __builtin_amdgcn_raw_buffer_store_b128(pack8(n), ys, c * 16, 0, 0);
    }
    if ((lane & 15) == 0 && c * 8 < dim) { A.sc[(size_t)(c >> 4) * A.rows + r] = s; }
  }
}

// ---- the GEMM ------------------------------------------------------------------
// y[m][n] = sum over blocks b of K of (sa[b][m] * sw[n / 128][b]) *
//           sum_{k in b} a[m][k] * w[n][k].
// v_mfma_f32_16x16x128_f8f6f4 multiplies exactly one block of K: D starts from
// zero for every block, and the block's scale joins it to the f32 sums outside
// the matrix unit.  The weight fragment is the first operand, so a lane's four
// results are consecutive output columns of one activation row and share its
// scale.  Lane l holds row l % 16 and the 16-byte chunks l / 16 and 4 + l / 16
// of the block: both operands the same way, so which k the unit takes a byte
// for does not matter to the sum over the block.
__device__ __forceinline__ f32x4_t
mfma_block(i32x8_t w, i32x8_t a)
{
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4_t{}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ int
find_problem(const Fp8Batch& B, int tile)
{
  int p = 0;
#pragma unroll
  for (int q = 1; q < kMaxProb; ++q) {
    if (q < B.nprob && tile >= B.p[q].tile_begin) { p = q; }
  }
  return p;
}

// One work item: a tile, and with K shares which blocks of K.
struct Fp8Work {
  int tile, share, prob;
  bool is_split;
  int row0, col0;
  int kbeg, nst;
};

// Work item w: whole tiles first, then the split tiles, `split` consecutive
// items each.  Tiles of a problem go in bands of 4 row tiles, walked column by
// column, so that items that run together share rows of both operands in L2.
template <int BM, int BN>
__device__ __forceinline__ Fp8Work
fp8_work(const Fp8Batch& B, int nb, int w)
{
  Fp8Work t;
  t.is_split = w >= B.split_begin;
  t.tile = w;
  t.share = 0;
  t.kbeg = 0;
  t.nst = nb;
  if (t.is_split) {
    const unsigned v = w - B.split_begin, q = v / (unsigned)B.split;
    t.tile = B.split_begin + q;
    t.share = v - q * B.split;
    t.kbeg = (unsigned)t.share * nb / (unsigned)B.split;
    t.nst = (unsigned)(t.share + 1) * nb / (unsigned)B.split - t.kbeg;
  }
  t.prob = find_problem(B, t.tile);
  const Fp8Problem& P = B.p[t.prob];
  const unsigned at = t.tile - P.tile_begin, per = 4 * P.tiles_n;
  const unsigned band = at / per, in = at - band * per;
  const unsigned gm = min(P.tiles_m - (int)band * 4, 4);
  const unsigned col = gm == 4 ? in / 4 : in / gm;
  t.row0 = (band * 4 + (in - col * gm)) * BM;
  t.col0 = col * BN;
  return t;
}

// A workgroup's tile: WM x WN waves, each FJ fragments of activation rows by FI
// of weight rows, and LWV waves that only load (0: the others load).  Its LDS: NS
// stages of scales (the tile's rows', then its columns'), of activations and of
// weights.
template <int WM, int WN, int FJ, int FI, int NS, int LWV>
struct Fp8Tile {
  static constexpr int kWaves = WM * WN + LWV;
  static constexpr int BM = 16 * WM * FJ, BN = 16 * WN * FI;
  static constexpr int kRowScales = (BM + 63) / 64 * 64;
  static constexpr int kScales = kRowScales + 64;                // floats per stage
  static constexpr int kAct = (NS * kScales * 4 + 1023) / 1024 * 1024;
  static constexpr int kWeight = kAct + NS * BM * 128;
  static constexpr int kBytes = kWeight + NS * BN * 128;
  static constexpr int kPerCu = std::max(std::min(160 * 1024 / kBytes, 8 / (WM * WN)), 1);
};

// One stage is one block of K.  Both operands come through LDS by direct loads
// of 1 KiB (8 rows x 128 bytes: 12 cycles each; loaded to registers in a
// fragment's layout, 16 rows x 64 bytes, the same bytes take 64).
// A wave holds a stage's weight fragments and walks its activation fragments,
// read a pair ahead; the results of the step before join the sums (one
// multiply-add each) while the matrix unit works.
// One barrier a stage, before the last pair, during which the next stage's
// first pair is read: there every wave has read this stage's places, which the
// loads of the stage NS ahead refill, and the next stage's loads have landed.
//
// What bounds it: a 256 x 256 stage takes 2900 cycles on a compute unit of which
// the products need 2048 (58% of all cycles with the rest of a launch); without
// its loads it takes 2430 (they share the LDS and wait to issue), without its
// multiply-adds 2700.  With every unit busy the clock falls to 1.6 to 1.8 GHz,
// so what costs power costs time: square tiles per wave (128 x 64, two thirds
// of the LDS reads that 256 x 32 makes) gained 5%.  Products and
// multiply-adds alone, from registers, reach 3.7 to 4.0 PFLOP/s; 4096 rows of
// K 12288 and 4096 columns run at 2.35 (175 us), 4224 rows of two times 12288
// columns at 2.1 (400 us).
// The smaller tiles have few products a stage to hide its barrier, reads and
// loads behind, so they have more places (NS), their weights' fragments a stage
// ahead where registers allow, and four waves that load for four that multiply
// (a wave waits to issue a load while others' go out: 12 cycles each, 36 of
// them beside the 512 cycles of products of 128 x 128).  A stage of 64 x 128
// takes 0.26 us where it took 0.37 with four waves that do both, of 128 x 128
// 0.37 (0.49 with eight, 0.39 with eight and four more that load); 4096 rows of
// K 8192 and 4096 columns take 124 us on 128 x 256 (138 and 130).  The larger two
// have no registers to spare for more waves.
// Row r's 16-byte chunk c sits at position c ^ ((r >> 1) & 7), which spreads
// the 16 rows of a fragment read over the bank groups; the loads put it there
// by fetching the chunk that belongs at their landing position.  They also
// order the rows: fragment j of a wave takes its rows j, FJ + j, 2 FJ + j, ..,
// so a lane's FJ rows are neighbours and their scales one run; of two weight
// fragments 2 p and 2 p + 1 a lane's results are 8 consecutive columns.
//
// Persistent: the loads run ahead over the end of a tile into the next one,
// whose first stages land while this one's results are stored.
template <int WM, int WN, int FJ, int FI, int FB, int NS, int LWV>
__device__ __forceinline__ void
fp8_tiles(const Fp8Batch& B, char* lds)
{
  using L = Fp8Tile<WM, WN, FJ, FI, NS, LWV>;
  constexpr int BM = L::BM, BN = L::BN;
  constexpr int NW = LWV > 0 ? LWV : WM * WN;        // the waves that load
  constexpr int kStageA = BM * 128, kStageW = BN * 128;
  constexpr int LA = BM / 8 / NW, LW = BN / 8 / NW;  // a wave's loads per stage
  constexpr int kOps = LA + LW + 1;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NW % 2 == 0, "even shares of loads");
  static_assert(L::kRowScales / 64 < NW && FI % 2 == 0, "a wave for the columns' scales");
  float* const scales = reinterpret_cast<float*>(lds);

  const int K = B.K, nb = (K + 127) / 128, sa_pitch = B.sa_pitch;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lh = lane >> 4;
  const int wm = wave % WM, wn = wave / WM;
  const int lwave = LWV > 0 ? wave - WM * WN : wave;

  // Items go in rounds of gridDim.x; workgroups b, b + 8, .. run on XCD b % 8,
  // and of each round every XCD takes a contiguous run.
  const int items = B.split_begin + (B.total_tiles - B.split_begin) * B.split;
  const int G = gridDim.x, rounds = (items + G - 1) / G;
  auto item_of = [&](int round) {
    const int base = round * G, n = min(G, items - base), b = blockIdx.x;
    if (round >= rounds) { return -1; }
    if (G % 8 != 0) { return b < n ? base + b : -1; }
    const int x = b & 7, i = b >> 3;
    return i < (n >> 3) + (x < (n & 7) ? 1 : 0) ? base + x * (n >> 3) + min(x, n & 7) + i : -1;
  };

  // ---- loads ---------------------------------------------------------------
  // What the loads of the stage NS ahead need, stepped along with the stages;
  // past the last item they fetch its last block again, for nobody.
  struct {
    __amdgpu_buffer_rsrc_t a, w;
    const float* sc;      // this wave's scales of the block
    int pitch, count;     // floats between blocks, bytes per block
    int ko, left, last;   // the block's bytes into a row, blocks left, -1 in the last of K
    int round;
  } ld;
  const bool row_wave = lwave < L::kRowScales / 64;
  auto load_item = [&](int it) {
    const Fp8Work t = fp8_work<BM, BN>(B, nb, it);
    const Fp8Problem& P = B.p[t.prob];
    const int rows = min(BM, P.rows - t.row0), cols = min(BN, P.n - t.col0);
    ld.a = make_rsrc(P.a + (size_t)t.row0 * K, rows * K);
    ld.w = make_rsrc(P.w + (size_t)t.col0 * K, cols * K);
    if (row_wave) {
      ld.sc = P.sa + (size_t)t.kbeg * sa_pitch + t.row0 + lwave * 64;
      ld.pitch = sa_pitch;
      ld.count = max(0, min(64, rows - lwave * 64)) * 4;
    } else {
      ld.sc = P.sw + (size_t)(t.col0 / 128) * nb + t.kbeg;
      ld.pitch = 1;
      ld.count = (((cols + 127) / 128 - 1) * nb + 1) * 4;
    }
    ld.sc = uniform(ld.sc);
    ld.pitch = uniform(ld.pitch);
    ld.count = uniform(ld.count);
    ld.ko = uniform(t.kbeg * 128);
    ld.left = uniform(t.nst);
    ld.last = uniform(t.kbeg == nb - 1 ? -1 : 0);
  };
  // A load's lane l fills chunk position l % 8 of row l / 8 of its 8 LDS rows.
  // Wave w fills blocks w, w + NW, .. of 8 rows, all of one parity (a half of
  // 16), so its lanes' chunk is one.
  const int half = (lwave & 1) * 8 + (lane >> 3);     // the row of its 16
  const int chunk = (lane & 7) ^ (half >> 1);
  const int tail = (nb - 1) * 128 + (chunk << 4) < K ? 0 : kOobOffset;
  // .. and of its rows the part that differs from lane to lane
  const int alane = half * FJ * K + (chunk << 4);
  const int wlane = ((half >> 2) * 8 + (half & 3)) * K + (chunk << 4);
  const int w2 = uniform(lwave >> 1);
  // scales: a lane each; the columns' are nb apart
  constexpr int kColBlocks = (BN + 127) / 128;
  const int soff = row_wave ? lane * 4 : lane < kColBlocks ? lane * nb * 4 : kOobOffset;
  auto dma16 = [](const __amdgpu_buffer_rsrc_t& r, char* to, int v, int s) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void*)to, 16, v, s, 0, 0);
  };
  // Load op of a stage's kOps, to place `slot`: its weights, activations, scales.
  auto load = [&](int slot, int op) {
    if (op < LW) {
      const int f = w2 + NW / 2 * op;                // of the tile's fragments
      dma16(ld.w, lds + L::kWeight + slot * kStageW + (lwave + NW * op) * 1024,
            (wlane | (tail & ld.last)) + ((f >> 1) * 32 + (f & 1) * 4) * K, ld.ko);
    } else if (op < LW + LA) {
      const int o = op - LW, f = w2 + NW / 2 * o;
      dma16(ld.a, lds + L::kAct + slot * kStageA + (lwave + NW * o) * 1024,
            (alane | (tail & ld.last)) + (f / FJ * (16 * FJ) + f % FJ) * K, ld.ko);
    } else {
      const int g = row_wave ? lwave * 64 : L::kRowScales;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          make_rsrc(ld.sc, ld.count),
          (__attribute__((address_space(3))) void*)(scales + slot * L::kScales + g), 4, soff, 0,
          0, 0);
    }
  };
  auto advance = [&] {
    if (ld.left > 1) {
      --ld.left;
      ld.ko += 128;
      ld.sc += ld.pitch;
      ld.last = ld.ko == (nb - 1) * 128 ? -1 : 0;
    } else {
      const int it = item_of(ld.round + 1);
      if (it >= 0) {
        ++ld.round;
        load_item(it);
      }
    }
  };

  // Loading waves of their own: a stage's loads behind each barrier, NS stages
  // ahead, as many barriers as the others pass.
  if constexpr (LWV > 0) {
    if (wave >= WM * WN) {
      int it = item_of(0), place = 0;
      if (it < 0) { return; }
      ld.round = 0;
      load_item(it);
#pragma unroll
      for (int r = 0; r < NS; ++r) {
#pragma unroll
        for (int o = 0; o < kOps; ++o) { load(r, o); }
        advance();
      }
      static_assert((NS - 1) * kOps < 64, "the counter has 6 bits");
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * kOps) : "memory");
      __builtin_amdgcn_s_barrier();
      for (int round = 0; it >= 0; it = item_of(++round)) {
        const int nst = fp8_work<BM, BN>(B, nb, it).nst;
        for (int k = 0; k < nst; ++k) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * kOps) : "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
#pragma unroll
          for (int o = 0; o < kOps; ++o) { load(place, o); }
          advance();
          place = place + 1 == NS ? 0 : place + 1;
        }
      }
      // no load may still be writing LDS when the workgroup ends
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      return;
    }
  }

  // ---- fragments -------------------------------------------------------------
  const int key = (lr >> 1) & 7;
  const int rd0 = lr * 128 + ((lh ^ key) << 4), rd1 = lr * 128 + (((4 + lh) ^ key) << 4);
  auto read_frag = [&](const char* base) {
    const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(base + rd0);
    const i32x4_t hi = *reinterpret_cast<const i32x4_t*>(base + rd1);
    return i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto read_a = [&](int slot, int j) {
    return read_frag(lds + L::kAct + wm * (FJ * 2048) + slot * kStageA + j * 2048);
  };
  auto read_w = [&](int slot, int i) {
    return read_frag(lds + L::kWeight + wn * (FI * 2048) + slot * kStageW + i * 2048);
  };
  constexpr int SV = FJ % 4 == 0 ? 4 : 2;            // row scales read at a time
  typedef float sv_t __attribute__((ext_vector_type(SV)));

  // A step is the products of one activation fragment and FH weight fragments.
  // Activation fragments go in pairs: both with the first weight fragments, then
  // both with the next ones, so that a weight fragment's place, refilled behind
  // the pair's last product of it, is next needed three steps later.
  constexpr int FH = 2, HS = FI / FH;
  constexpr int kSteps = FJ * HS;
  auto frag_of = [](int step) { return 2 * (step / (2 * HS)) + step % 2; };
  auto half_of = [](int step) { return step % (2 * HS) / 2; };
  constexpr int kBarrier = kSteps - 2 * HS;          // the barrier's step: the last pair
  static_assert(FJ % 2 == 0 && FB >= 4 && FJ % FB == 0, "fragment buffers come round with a stage");
  // Where the multiplying waves load: a stage's loads begin behind the barrier,
  // about one a step, the last of them in the next stage's first steps, over two
  // thirds of a stage's time, as the next barrier waits for them.
  constexpr int kSpan = 2 * kSteps / 3;
  static_assert(LWV > 0 || NS == 2, "which leaves them little time to land");
  auto step_of = [](int op) { return (kBarrier + op * kSpan / kOps) % kSteps; };
  constexpr int kEarly =
      std::min(kOps, ((kSteps - kBarrier) * kOps + kSpan - 1) / kSpan);   // before its end
  static_assert((NS - 2) * kOps + kEarly < 64, "the counter has 6 bits");
  f32x4_t acc[FI][FJ], d[2][FH];
  // Weight fragments of this stage and the next; where registers are short, the
  // next one's take the places of this one's as its last products leave them.
  constexpr bool kAhead = FJ * FI <= 16;
  i32x8_t fa[kAhead ? 2 : 1][FI], fb[FB];
  float sc[FJ];                                      // the stage's scales, rows' times columns'
  sv_t sv[FJ / SV];                                  // the next stage's, apart
  float w, pending;                                  // .. and the one the last results wait for
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < FI; ++i) {
#pragma unroll
      for (int j = 0; j < FJ; ++j) { acc[i][j] = f32x4_t{}; }
    }
#pragma unroll
    for (int i = 0; i < FH; ++i) { d[1][i] = f32x4_t{}; }
    pending = 0.0f;
  };
  auto add = [&](int j, int h, int par, float s) {
#pragma unroll
    for (int i = 0; i < FH; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[h * FH + i][j][e] = fmaf(d[par][i][e], s, acc[h * FH + i][j][e]);
      }
    }
  };
  auto read_scales = [&](int slot) {
    const float* const at = scales + slot * L::kScales;
#pragma unroll
    for (int g = 0; g < FJ / SV; ++g) {
      sv[g] = *reinterpret_cast<const sv_t*>(at + wm * (16 * FJ) + lr * FJ + g * SV);
    }
    w = at[L::kRowScales + wn * (16 * FI) / 128];
  };
  // The sums so far stay where they are computed: nothing of a stage moves past
  // a branch, where it would hold its operands' registers.
  auto settle = [&] {
#pragma unroll
    for (int i = 0; i < FI; ++i) {
#pragma unroll
      for (int j = 0; j < FJ; ++j) { asm volatile("" : "+v"(acc[i][j])); }
    }
  };
  // One stage, its operands in place `cur`, the next one's in `next`, the last
  // one's in `prev`.
  auto stage = [&](auto par_c, int prev, int cur, int next) {
    constexpr int par = kAhead ? decltype(par_c)::value : 0;
#pragma unroll
    for (int j = 0; j < FJ; ++j) { sc[j] = sv[j / SV][j % SV] * w; }
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const int j = frag_of(step), h = half_of(step);
      if (step == kBarrier) {
        if constexpr (LWV > 0) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
          settle();
          advance();
          asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * kOps) : "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      if (h == 0) {
        fb[(j + 2) % FB] = j + 2 < FJ ? read_a(cur, j + 2) : read_a(next, j + 2 - FJ);
      }
      if (step == kBarrier + 1) { read_scales(next); }
      if (kAhead && step >= kBarrier) {
#pragma unroll
        for (int i = 0; i < FI; ++i) {
          if (kBarrier + i * 2 * HS / FI == step) { fa[par ^ kAhead][i] = read_w(next, i); }
        }
      }
      const int now = step & 1, before = now ^ 1;
#pragma unroll
      for (int i = 0; i < FH; ++i) {
        d[now][i] = mfma_block(fa[par][h * FH + i], fb[j % FB]);
      }
      if (step == 0) {
        add(FJ - 1, HS - 1, before, pending);
      } else {
        add(frag_of(step - 1), half_of(step - 1), before, sc[frag_of(step - 1)]);
      }
#pragma unroll
      for (int o = 0; o < kOps; ++o) {
        if (LWV == 0 && step_of(o) == step) { load(o < kEarly ? cur : prev, o); }
      }
      if (!kAhead && j == FJ - 1) {
#pragma unroll
        for (int i = 0; i < FH; ++i) { fa[0][h * FH + i] = read_w(next, h * FH + i); }
      }
#pragma unroll
      for (int i = 0; i < FH; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // a product
        if (i == 0) { __builtin_amdgcn_sched_group_barrier(0x100, 8, 0); }    // reads
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);        // the sums
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    pending = sc[FJ - 1];
    settle();
  };

  // ---- the first item's first stages -------------------------------------------
  int it = item_of(0);
  if (it < 0) { return; }
  if constexpr (LWV == 0) {
    ld.round = 0;
    load_item(it);
#pragma unroll
    for (int r = 0; r < NS; ++r) {
#pragma unroll
      for (int o = 0; o < (r < NS - 1 ? kOps : kEarly); ++o) { load(r, o); }
      if (r < NS - 1) { advance(); }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * kOps + kEarly) : "memory");   // stage 0's
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < FI; ++i) { fa[0][i] = read_w(0, i); }
#pragma unroll
  for (int j = 0; j < 2; ++j) { fb[j] = read_a(0, j); }
  read_scales(0);

  int prev = NS - 1, cur = 0, next = 1, round = 0;
  using std::integral_constant;
  auto step = [&](auto par_c) {
    stage(par_c, prev, cur, next);
    prev = cur;
    cur = next;
    next = next + 1 == NS ? 0 : next + 1;
  };
  clear();
  for (;;) {
    const Fp8Work t = fp8_work<BM, BN>(B, nb, it);
    const Fp8Problem& P = B.p[t.prob];
    int k = 0;
    if constexpr (kAhead) {
      for (; k + 1 < t.nst; k += 2) {
        step(integral_constant<int, 0>{});
        step(integral_constant<int, 1>{});
      }
    }
    for (; k < t.nst; ++k) {
      step(integral_constant<int, 0>{});
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < FI; ++i) { fa[0][i] = fa[1][i]; }
      }
    }
    add(FJ - 1, HS - 1, 1, pending);

    // ---- results -----------------------------------------------------------------
    const int rows = min(BM, P.rows - t.row0), r0 = wm * (16 * FJ) + lr * FJ;
    if (t.is_split) {
      // as they lie, 1 KiB each
      const __amdgpu_buffer_rsrc_t to = make_rsrc(
          B.ws + (size_t)((t.tile - B.split_begin) * B.split + t.share) * (BM * BN), BM * BN * 4);
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        const int at = r0 + j < rows ? lane * 16 : kOobOffset;
#pragma unroll
        for (int i = 0; i < FI; ++i) {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, acc[i][j]), to, at,
                                                 ((wave * FJ + j) * FI + i) * 1024, 0);
        }
      }
    } else {
      const __amdgpu_buffer_rsrc_t to = make_rsrc(P.y + (size_t)t.row0 * P.n, rows * P.n * 2);
#pragma unroll
      for (int p = 0; p < FI / 2; ++p) {
        const int n = t.col0 + wn * (16 * FI) + p * 32 + lh * 8;
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
          const f32x4_t &u = acc[2 * p][j], &v = acc[2 * p + 1][j];
          __builtin_amdgcn_raw_buffer_store_b128(
              u32x4_t{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]),
                      pack_bf16x2(v[2], v[3])},
              to, n < P.n ? ((r0 + j) * P.n + n) * 2 : kOobOffset, 0, 0);
        }
      }
    }
    it = item_of(++round);
    if (it < 0) { break; }
    clear();
  }
  // no load may still be writing LDS when the workgroup ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// (a tile's workgroups on a compute unit, and so its waves per SIMD, are what its
// LDS leaves room for)
template <int WM, int WN, int FJ, int FI, int NS, int LWV>
constexpr int kTileWaves =
    Fp8Tile<WM, WN, FJ, FI, NS, LWV>::kPerCu * Fp8Tile<WM, WN, FJ, FI, NS, LWV>::kWaves / 4;

template <int WM, int WN, int FJ, int FI, int FB, int NS, int LWV>
__global__ __launch_bounds__(64 * (WM * WN + LWV), (kTileWaves<WM, WN, FJ, FI, NS, LWV>)) void
fp8_tile_kernel(const Fp8Batch B)
{
  __shared__ __attribute__((aligned(1024))) char lds[Fp8Tile<WM, WN, FJ, FI, NS, LWV>::kBytes];
  fp8_tiles<WM, WN, FJ, FI, FB, NS, LWV>(B, lds);
}

// ---- few rows: the weights' stream ---------------------------------------------
// At most 16 MT rows.  A workgroup takes 16 FI columns and its NW waves the
// blocks of K, a contiguous share each, with nothing between them until their
// sums join through LDS, in wave order.  A wave streams its blocks (weights,
// rows, row scales) through D places of its own in LDS by direct loads, so all
// of D stages are in flight from the start; the weight scales are a register
// each of 64 blocks, read by lane.
// Bound by the weights' bytes where rows are few (and by latency where K is
// short): one row takes 7.1 us with 6144 columns of K 4096, 21.0 us with 24576
// (4.8 TB/s); 64 rows of 6144 columns 11.7 us.  A model's weights are read once
// a step and do not fit the caches, so they go past them (non-temporal): loaded
// plainly these take 8.0, 22.5 and 12.3 us, and only weights that stay in the
// 256 MB cache from call to call come faster so (5.7, 18.5 and 8.5 us).
template <int MT, int FI, int NW, int D>
struct Fp8NarrowLds {
  static constexpr int kSlot = FI * 2048 + MT * 2048 + (MT + 3) / 4 * 256;
  static constexpr int kBytes = NW * std::max(D * kSlot, MT * FI * 1024);
};

template <int MT, int FI, int NW, int D>
__global__ __launch_bounds__(64 * NW) void
fp8_narrow_kernel(const Fp8Batch B)
{
  using L = Fp8NarrowLds<MT, FI, NW, D>;
  __shared__ __attribute__((aligned(1024))) char lds[L::kBytes];
  constexpr int kOps = 2 * FI + 2 * MT + (MT + 3) / 4;
  static_assert(D * kOps < 64, "the counter has 6 bits");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lh = lane >> 4;
  const int prob = find_problem(B, blockIdx.x);
  const Fp8Problem& P = B.p[prob];
  const int n0 = (blockIdx.x - P.tile_begin) * (16 * FI);
  const int K = B.K, nb = (K + 127) / 128, sa_pitch = B.sa_pitch;
  const int b0 = wave * nb / NW, b1 = (wave + 1) * nb / NW;

  const __amdgpu_buffer_rsrc_t rw =
      make_rsrc(P.w + (size_t)n0 * K, min(16 * FI, P.n - n0) * K);
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(P.a, P.rows * K);
  const float* const sa = P.sa;
  const int scale_bytes = P.rows * 4;
  char* const mine = lds + wave * (D * L::kSlot);
  // a load's lane l fills chunk position l % 8 of row l / 8 of its 8 rows; the
  // chunk depends on the 8 rows' parity
  const int row = lane >> 3;
  int off[2], tail[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int chunk = (lane & 7) ^ (4 * h + (row >> 1));
    off[h] = (8 * h + row) * K + (chunk << 4);
    tail[h] = (nb - 1) * 128 + (chunk << 4) < K ? 0 : kOobOffset;
  }
  auto load = [&](int slot, int b) {
    char* const to = mine + slot * L::kSlot;
    const int kt = min(b, nb - 1), past = b < b1 ? 0 : kOobOffset;
    const int ko = __builtin_amdgcn_readfirstlane(kt * 128);
#pragma unroll
    for (int r = 0; r < 2 * (FI + MT); ++r) {
      const int h = r & 1, v = off[h] + ((kt == nb - 1 ? tail[h] : 0) | past);
      const bool weights = r < 2 * FI;
      auto* const dst = (__attribute__((address_space(3))) void*)(to + r * 1024);
      if (weights) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, dst, 16, v + r / 2 * 16 * K, ko, 0,
                                                 kNonTemporal);
      } else {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, dst, 16, v + (r - 2 * FI) / 2 * 16 * K, ko, 0, 0);
      }
    }
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(sa + (size_t)kt * sa_pitch, scale_bytes);
#pragma unroll
    for (int g = 0; g < (MT + 3) / 4; ++g) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(to + (FI + MT) * 2048 + g * 256), 4,
          g * 256 + lane * 4, 0, 0, 0);
    }
  };
  const float* const sw = P.sw + (size_t)(n0 / 128) * nb;
  float wv = b0 + lane < b1 ? sw[b0 + lane] : 0.0f;

  const int key = (lr >> 1) & 7;
  const int rd0 = lr * 128 + ((lh ^ key) << 4), rd1 = lr * 128 + (((4 + lh) ^ key) << 4);
  f32x4_t acc[FI][MT];
#pragma unroll
  for (int i = 0; i < FI; ++i) {
#pragma unroll
    for (int j = 0; j < MT; ++j) { acc[i][j] = f32x4_t{}; }
  }
#pragma unroll
  for (int r = 0; r < D; ++r) {
    load(r, b0 + r);
    __builtin_amdgcn_sched_barrier(0);
  }
  int slot = 0;
  for (int b = b0; b < b1; ++b) {
    if (((b - b0) & 63) == 0 && b != b0) {
      wv = b + lane < b1 ? sw[b + lane] : 0.0f;
      asm volatile("s_waitcnt vmcnt(0)" : "+v"(wv)::"memory");
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * kOps) : "memory");
    const char* const at = mine + slot * L::kSlot;
    i32x8_t f[FI + MT];
    float s[MT];
#pragma unroll
    for (int r = 0; r < FI + MT; ++r) {
      const i32x4_t lo = *reinterpret_cast<const i32x4_t*>(at + r * 2048 + rd0);
      const i32x4_t hi = *reinterpret_cast<const i32x4_t*>(at + r * 2048 + rd1);
      f[r] = i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      s[j] = *reinterpret_cast<const float*>(at + (FI + MT) * 2048 + (16 * j + lr) * 4);
    }
    // in registers: the place is free
#pragma unroll
    for (int r = 0; r < FI + MT; ++r) { asm volatile("" : "+v"(f[r])); }
#pragma unroll
    for (int j = 0; j < MT; ++j) { asm volatile("" : "+v"(s[j])); }
    load(slot, b + D);
    const float w = __uint_as_float(
        __builtin_amdgcn_readlane(__float_as_uint(wv), (b - b0) & 63));
    f32x4_t d[FI][MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
#pragma unroll
      for (int i = 0; i < FI; ++i) { d[i][j] = mfma_block(f[i], f[FI + j]); }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) {
#pragma unroll
      for (int i = 0; i < FI; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) { acc[i][j][e] = fmaf(d[i][j][e], s[j] * w, acc[i][j][e]); }
      }
    }
    slot = slot + 1 == D ? 0 : slot + 1;
  }
  // every load has landed before its place takes the sums
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FI; ++i) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      *reinterpret_cast<f32x4_t*>(lds + ((wave * FI + i) * MT + j) * 1024 + lane * 16) = acc[i][j];
    }
  }
  __syncthreads();
  for (int c = wave; c < FI * MT; c += NW) {
    f32x4_t v = *reinterpret_cast<const f32x4_t*>(lds + c * 1024 + lane * 16);
#pragma unroll
    for (int q = 1; q < NW; ++q) {
      v += *reinterpret_cast<const f32x4_t*>(lds + (q * FI * MT + c) * 1024 + lane * 16);
    }
    const int m = c % MT * 16 + lr, n = n0 + c / MT * 16 + lh * 4;
    if (m < P.rows && n < P.n) {
      *reinterpret_cast<u32x2_t*>(P.y + (size_t)m * P.n + n) =
          u32x2_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
    }
  }
}

// The shares of split tiles, added in their order: 256 threads take 8 results
// each, which lie as the tiles' lanes held them.
template <int WM, int WN, int FJ, int FI>
__global__ __launch_bounds__(256) void
fp8_reduce_kernel(const Fp8Batch B)
{
  constexpr int BM = 16 * WM * FJ, BN = 16 * WN * FI, kPer = BM * BN / 2048;
  const int tile = B.split_begin + blockIdx.x / kPer;
  const int nb = (B.K + 127) / 128;
  const Fp8Work t = fp8_work<BM, BN>(B, nb, B.split_begin + (tile - B.split_begin) * B.split);
  const Fp8Problem& P = B.p[t.prob];
  const int lane = threadIdx.x & 63, lr = lane & 15, lh = lane >> 4;
  // wave, fragment and pair of weight fragments
  const int c = blockIdx.x % kPer * 4 + (threadIdx.x >> 6);
  const int p = c % (FI / 2), j = c / (FI / 2) % FJ, wave = c / (FI / 2 * FJ);
  const int m = t.row0 + wave % WM * (16 * FJ) + lr * FJ + j;
  const int n = t.col0 + wave / WM * (16 * FI) + p * 32 + lh * 8;
  if (m >= P.rows || n >= P.n) { return; }
  const float* const at =
      B.ws + (size_t)(tile - B.split_begin) * B.split * (BM * BN) + c * 512 + lane * 4;
  // four shares' loads at a time; those past the last are its own again, not added
  f32x4_t u = {}, v = {};
  for (int q0 = 0; q0 < B.split; q0 += 4) {
    f32x4_t su[4], sv[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float* const from = at + (size_t)min(q0 + q, B.split - 1) * (BM * BN);
      su[q] = *reinterpret_cast<const f32x4_t*>(from);
      sv[q] = *reinterpret_cast<const f32x4_t*>(from + 256);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q0 + q < B.split) {
        u += su[q];
        v += sv[q];
      }
    }
  }
  *reinterpret_cast<u32x4_t*>(P.y + (size_t)m * P.n + n) =
      u32x4_t{pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]),
              pack_bf16x2(v[2], v[3])};
}

template <int WM, int WN, int FJ, int FI, int FB, int NS, int LWV>
hipError_t
tile_launch(const Fp8Batch& b, hipStream_t s)
{
  using L = Fp8Tile<WM, WN, FJ, FI, NS, LWV>;
  const int tail = b.total_tiles - b.split_begin;
  const int items = b.split_begin + tail * b.split;
  static_assert(L::kPerCu == fp8_tiles_per_cu(L::BM, L::BN), "the plan's rounds are the grid's");
  fp8_tile_kernel<WM, WN, FJ, FI, FB, NS, LWV>
      <<<std::min(items, b.cus * L::kPerCu), 64 * L::kWaves, 0, s>>>(b);   // all at once
  if (b.split > 1 && tail > 0) {
    fp8_reduce_kernel<WM, WN, FJ, FI><<<tail * (L::BM * L::BN / 2048), 256, 0, s>>>(b);
  }
  return hipGetLastError();
}

template <int WPR, int CPL, bool ADD>
void
norm_launch(const Fp8NormArgs& a, hipStream_t s)
{
  fp8_norm_kernel<WPR, CPL, ADD><<<a.rows, 64 * WPR, 0, s>>>(a);
}

template <bool SWIGLU, int RPW>
void
rows_launch(const uint16_t* x, const uint16_t* up, int rows, int K, uint16_t* h, uint8_t* q,
            float* sc, hipStream_t s)
{
  const int groups = (rows + 4 * RPW - 1) / (4 * RPW);
  const dim3 grid((K + 511) / 512, std::min(groups, kRowGroups),
                  (groups + kRowGroups - 1) / kRowGroups);
  fp8_quant_rows_kernel<SWIGLU, RPW><<<grid, 256, 0, s>>>(x, up, rows, K, h, q, sc);
}

}  // namespace

// The tile builds: X(WM, WN, FJ, FI, FB, NS, LWV).
#define U15H_FP8_TILES(X) \
  X(2, 4, 8, 4, 4, 2, 0)  \
  X(2, 4, 6, 4, 6, 2, 0)  \
  X(1, 4, 8, 4, 4, 3, 4)  \
  X(2, 2, 4, 4, 4, 4, 4)  \
  X(1, 4, 4, 2, 4, 3, 4)

#define U15H_FP8_NARROW(X) \
  X(1, 1, 4, 4)            \
  X(1, 2, 4, 4)            \
  X(2, 1, 4, 4)            \
  X(2, 2, 4, 4)            \
  X(4, 1, 4, 3)            \
  X(4, 2, 4, 3)            \
  X(6, 1, 4, 2)            \
  X(8, 1, 4, 2)

hipError_t
launch_fp8_gemm(const Fp8Batch& b, hipStream_t s)
{
  // whole tiles, or a tail in two shares or more that has a workspace
  const bool split = b.split_begin != b.total_tiles;
  if (b.total_tiles <= 0 || b.split_begin < 0 || b.split_begin > b.total_tiles ||
      (split ? b.narrow || b.split < 2 || b.split > (b.K + 127) / 128 || b.ws == nullptr
             : b.split != 1)) {
    return hipErrorInvalidValue;
  }
#define U15H_CASE(MT, FI, NW, D)                                                          \
  if (b.narrow && b.bm == 16 * MT && b.bn == 16 * FI) {                                \
    fp8_narrow_kernel<MT, FI, NW, D><<<b.total_tiles, 64 * NW, 0, s>>>(b);               \
    return hipGetLastError();                                                            \
  }
  U15H_FP8_NARROW(U15H_CASE)
#undef U15H_CASE
#define U15H_CASE(WM, WN, FJ, FI, FB, NS, LWV)                                                     \
  if (!b.narrow && b.bm == 16 * WM * FJ && b.bn == 16 * WN * FI) {                        \
    return tile_launch<WM, WN, FJ, FI, FB, NS, LWV>(b, s);                                         \
  }
  U15H_FP8_TILES(U15H_CASE)
#undef U15H_CASE
  return hipErrorInvalidValue;
}

hipError_t
launch_fp8_quant_rows(const uint16_t* x, const uint16_t* up, int rows, int K, uint16_t* h,
                      uint8_t* q, float* sc, hipStream_t s)
{
  if (up != nullptr) {
    rows_launch<true, 1>(x, up, rows, K, h, q, sc, s);
  } else {
    rows_launch<false, 2>(x, up, rows, K, h, q, sc, s);
  }
  return hipGetLastError();
}

hipError_t
launch_fp8_quant_blocks(const uint16_t* w, int N, int K, uint8_t* q, float* sc, hipStream_t s)
{
  const dim3 grid((K + kFp8Block - 1) / kFp8Block, (N + kFp8Block - 1) / kFp8Block);
  fp8_quant_blocks_kernel<<<grid, 256, 0, s>>>(w, N, K, q, sc);
  return hipGetLastError();
}

hipError_t
launch_fp8_norm(const Fp8NormArgs& a, hipStream_t s)
{
  const bool add = a.d != nullptr;
  if (a.dim <= 2048) {
    add ? norm_launch<4, 1, true>(a, s) : norm_launch<4, 1, false>(a, s);
  } else if (a.dim <= 4096) {
    add ? norm_launch<8, 1, true>(a, s) : norm_launch<4, 2, false>(a, s);
  } else if (a.dim <= 8192) {
    add ? norm_launch<8, 2, true>(a, s) : norm_launch<8, 2, false>(a, s);
  } else {
    add ? norm_launch<8, 4, true>(a, s) : norm_launch<8, 4, false>(a, s);
  }
  return hipGetLastError();
}

bool
fp8_kernels_loadable()
{
  const void* fns[] = {
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<false, 2>),
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<true, 1>),
      reinterpret_cast<const void*>(&fp8_quant_blocks_kernel),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 1, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 1, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 2, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 1, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 2, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 2, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 4, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 4, true>),
#define U15H_FN(MT, FI, NW, D) reinterpret_cast<const void*>(&fp8_narrow_kernel<MT, FI, NW, D>),
      U15H_FP8_NARROW(U15H_FN)
#undef U15H_FN
#define U15H_FN(WM, WN, FJ, FI, FB, NS, LWV)                                       \
  reinterpret_cast<const void*>(&fp8_tile_kernel<WM, WN, FJ, FI, FB, NS, LWV>),     \
      reinterpret_cast<const void*>(&fp8_reduce_kernel<WM, WN, FJ, FI>),
      U15H_FP8_TILES(U15H_FN)
#undef U15H_FN
  };
  for (const void* f : fns) {
    hipFuncAttributes a;
    if (hipFuncGetAttributes(&a, f) != hipSuccess) { return false; }
  }
  return true;
}

}  // namespace u15h
