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

// silu(g) * u in f32: g * rcp(1 + 2^(-g log2 e)) with the hardware's exp2
// and reciprocal (about 1 ulp each).
__device__ __forceinline__ float
swiglu_f32(float g, float u)
{
  const float e = __builtin_amdgcn_exp2f(g * -1.4426950408889634f);
  return (g * __builtin_amdgcn_rcpf(1.0f + e)) * u;
}

// ---- rows: codes and block-major scales --------------------------------------
// One workgroup of four waves per 4 RPW rows x 512 columns.  A wave reads 512
// columns of a row at a time, lane l columns 8 l..8 l + 7, so a block of 128 is
// 16 neighbouring lanes; all of its RPW rows' loads issue first.  The scales
// of the workgroup's rows are gathered in LDS and written as runs of 4 RPW.
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
  const int row0 = blockIdx.x * R, col = blockIdx.y * 512 + lane * 8;
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
    xv[i] = __builtin_amdgcn_raw_buffer_load_b128(xs, at * 2 + oob, 0, 0);
    if constexpr (SWIGLU) { uv[i] = __builtin_amdgcn_raw_buffer_load_b128(us, at * 2 + oob, 0, 0); }
  }
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    const int at = (wave * RPW + i) * K + col;
    float v[8];
    unpack8(xv[i], v);
    if constexpr (SWIGLU) {
      float u[8];
      unpack8(uv[i], u);
#pragma unroll
      for (int e = 0; e < 8; ++e) { v[e] = swiglu_f32(v[e], u[e]); }
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
    const int b = blockIdx.y * 4 + t / R, r = t % R;
    if (b < nb && r < valid) { sc[(size_t)b * rows + row0 + r] = scales[t / R][r]; }
  }
}

// ---- weights: a scale per 128 x 128 ------------------------------------------
// One workgroup of four waves per block; a wave reads four rows' 256 bytes at a
// time (lane l: row l / 16, columns 8 (l % 16)..), eight such reads in flight.
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
    v[i] = __builtin_amdgcn_raw_buffer_load_b128(ws, (at + i * 16 * K) * 2 + oob, 0, 0);
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
    __builtin_amdgcn_raw_buffer_store_b64(codes8(f, inv), qs, at + i * 16 * K + oob, 0, 0);
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
    v[i] = __builtin_amdgcn_raw_buffer_load_b128(xs, c * 16, 0, 0);
    g[i] = __builtin_amdgcn_raw_buffer_load_b128(ws, c * 16, 0, 0);
  }
  if constexpr (ADD) {
    const __amdgpu_buffer_rsrc_t ds = make_rsrc(A.d + base, dim * 2);
    const __amdgpu_buffer_rsrc_t os = make_rsrc(A.x_out + base, dim * 2);
    u32x4_t d[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      d[i] = __builtin_amdgcn_raw_buffer_load_b128(ds, ((i * WPR + part) * 64 + lane) * 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[i][e] = pack_bf16x2(bf16_lo(v[i][e]) + bf16_lo(d[i][e]),
                              bf16_hi(v[i][e]) + bf16_hi(d[i][e]));
      }
      __builtin_amdgcn_raw_buffer_store_b128(v[i], os, ((i * WPR + part) * 64 + lane) * 16, 0, 0);
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

constexpr int kTile = 64;

// 64 x 64 outputs per workgroup, 16 columns x 64 rows per wave, fragments
// straight from memory.
__global__ __launch_bounds__(256) void
fp8_gemm_kernel(const Fp8Batch B)
{
  const int tile = blockIdx.x;
  const Fp8Problem& P = B.p[find_problem(B, tile)];
  const int t = tile - P.tile_begin;
  const int row0 = t % P.tiles_m * kTile, col0 = t / P.tiles_m * kTile;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int lr = lane & 15, lh = lane >> 4, K = B.K;
  const int nb = (K + kFp8Block - 1) / kFp8Block;
  const int n = col0 + wave * 16;
  if (n >= P.n) { return; }
  auto load = [&](const uint8_t* row, int b) {
    const int k = b * kFp8Block + lh * 16;
    i32x4_t lo = {}, hi = {};
    if (k < K) { lo = *reinterpret_cast<const i32x4_t*>(row + k); }
    if (k + 64 < K) { hi = *reinterpret_cast<const i32x4_t*>(row + k + 64); }
    return i32x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  // rows past the problem repeat its last one; their results are not stored
  const uint8_t* const wr = P.w + (size_t)min(n + lr, P.n - 1) * K;
  const uint8_t* ar[4];
  int m[4];
  f32x4_t acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m[j] = min(row0 + 16 * j + lr, P.rows - 1);
    ar[j] = P.a + (size_t)m[j] * K;
    acc[j] = f32x4_t{};
  }
  for (int b = 0; b < nb; ++b) {
    const i32x8_t w = load(wr, b);
    const float sw = P.sw[(size_t)(n / kFp8Block) * nb + b];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t d = mfma_block(w, load(ar[j], b));
      const float s = P.sa[(size_t)b * B.sa_pitch + m[j]] * sw;
#pragma unroll
      for (int e = 0; e < 4; ++e) { acc[j][e] = fmaf(d[e], s, acc[j][e]); }
    }
  }
  const int c = n + lh * 4;
  if (c >= P.n) { return; }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = row0 + 16 * j + lr;
    if (r < P.rows) {
      *reinterpret_cast<u32x2_t*>(P.y + (size_t)r * P.n + c) =
          u32x2_t{pack_bf16x2(acc[j][0], acc[j][1]), pack_bf16x2(acc[j][2], acc[j][3])};
    }
  }
}

template <int WPR, int CPL>
void
norm_launch(const Fp8NormArgs& a, hipStream_t s)
{
  const dim3 grid(a.rows), block(64 * WPR);
  if (a.d != nullptr) {
    fp8_norm_kernel<WPR, CPL, true><<<grid, block, 0, s>>>(a);
  } else {
    fp8_norm_kernel<WPR, CPL, false><<<grid, block, 0, s>>>(a);
  }
}

template <bool SWIGLU, int RPW>
void
rows_launch(const uint16_t* x, const uint16_t* up, int rows, int K, uint16_t* h, uint8_t* q,
            float* sc, hipStream_t s)
{
  const dim3 grid((rows + 4 * RPW - 1) / (4 * RPW), (K + 511) / 512);
  fp8_quant_rows_kernel<SWIGLU, RPW><<<grid, 256, 0, s>>>(x, up, rows, K, h, q, sc);
}

}  // namespace

hipError_t
launch_fp8_gemm(const Fp8Batch& b0, hipStream_t s)
{
  Fp8Batch b = b0;
  long long tiles = 0;
  for (int i = 0; i < b.nprob; ++i) {
    Fp8Problem& p = b.p[i];
    p.tiles_m = (p.rows + kTile - 1) / kTile;
    p.tiles_n = (p.n + kTile - 1) / kTile;
    p.tile_begin = (int)tiles;
    tiles += (long long)p.tiles_m * p.tiles_n;
    if (tiles > (1 << 30)) { return hipErrorInvalidValue; }
  }
  b.total_tiles = (int)tiles;
  fp8_gemm_kernel<<<dim3((unsigned)tiles), 256, 0, s>>>(b);
  return hipGetLastError();
}

hipError_t
launch_fp8_quant_rows(const uint16_t* x, const uint16_t* up, int rows, int K, uint16_t* h,
                      uint8_t* q, float* sc, hipStream_t s)
{
  if (up != nullptr) {
    if (rows >= 1024) {
      rows_launch<true, 4>(x, up, rows, K, h, q, sc, s);
    } else {
      rows_launch<true, 1>(x, up, rows, K, h, q, sc, s);
    }
  } else if (rows >= 1024) {
    rows_launch<false, 8>(x, up, rows, K, h, q, sc, s);
  } else {
    rows_launch<false, 1>(x, up, rows, K, h, q, sc, s);
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
  if (a.dim <= 2048) {
    norm_launch<4, 1>(a, s);
  } else if (a.dim <= 4096) {
    norm_launch<4, 2>(a, s);
  } else if (a.dim <= 8192) {
    norm_launch<8, 2>(a, s);
  } else {
    norm_launch<8, 4>(a, s);
  }
  return hipGetLastError();
}

bool
fp8_kernels_loadable()
{
  const void* fns[] = {
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<false, 1>),
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<false, 8>),
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<true, 1>),
      reinterpret_cast<const void*>(&fp8_quant_rows_kernel<true, 4>),
      reinterpret_cast<const void*>(&fp8_quant_blocks_kernel),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 1, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 1, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 2, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<4, 2, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 2, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 2, true>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 4, false>),
      reinterpret_cast<const void*>(&fp8_norm_kernel<8, 4, true>),
      reinterpret_cast<const void*>(&fp8_gemm_kernel),
  };
  for (const void* f : fns) {
    hipFuncAttributes a;
    if (hipFuncGetAttributes(&a, f) != hipSuccess) { return false; }
  }
  return true;
}

}  // namespace u15h
