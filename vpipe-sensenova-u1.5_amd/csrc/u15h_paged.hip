// u15h_paged.hip -- gfx950 kernels for many requests at once: rotary
// positions, the paged K/V cache, attention behind a shared prefix.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "u15h_internal.h"

namespace u15h {
namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

constexpr int kRsrcWord3 = 0x00020000;      // raw buffer, 32-bit data format

// A wave-uniform value made explicitly so: it stays in SGPRs.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A buffer resource over [base, base + bytes): loads past it read zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t
make_rsrc(const void* base, int bytes)
{
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)p);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(
      reinterpret_cast<void*>(((uint64_t)hi << 32) | lo), 0, uniform(bytes), kRsrcWord3);
}

// Two floats as packed bf16 (lo in the low half), round to nearest even.
__device__ __forceinline__ uint32_t
pack_bf16x2(float lo, float hi)
{
  return __builtin_bit_cast(uint32_t,
                            __builtin_convertvector((f32x2_t){lo, hi}, bf16x2_t));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// ---- rotary positions -------------------------------------------------------
// y_a = x_a c - x_b s, y_b = x_b c + x_a s for every pair (a, b) of columns,
// c and s the cosine and sine of position * frequency, the same for all heads
// of a token.
//
// A workgroup takes `group` tokens.  It forms their cosines and sines once, a
// pair a thread, in LDS, and then goes over their heads' columns, VEC of them
// an access.  The angle is formed in 64 bits and in turns, whose whole part
// drops out exactly, so a position of 2^31 costs no precision: what is left is
// in [-1/2, 1/2] and goes through sincospif in 32 bits.
//
// Memory-bound: 4 bytes an element; the angles are 1/16 of the work at 32
// heads of 64 pairs.

// Access unit u of a head: the first column of its one or two runs of VEC
// columns (b -1: one run), and its first pair (-1: columns passed on).
struct RopeUnit {
  int a, b, pair;
};

template <int VEC>
__device__ __forceinline__ RopeUnit
rope_unit(const RopeArgs& A, int u)
{
  // units of the parts, in order, then the columns between them
#pragma unroll
  for (int p = 0; p < U15H_MAX_ROPE_PARTS; ++p) {
    if (p < A.nparts) {
      const RopePart& P = A.part[p];
      const int h = P.width / 2;
      const bool runs = !A.neighbours || VEC == 1;     // two runs a unit
      const int n = runs ? h / VEC : P.width / VEC;
      if (u < n) {
        if (!runs) { return {P.start + u * VEC, -1, P.pair + u * VEC / 2}; }
        return A.neighbours ? RopeUnit{P.start + 2 * u, P.start + 2 * u + 1, P.pair + u}
                            : RopeUnit{P.start + u * VEC, P.start + h + u * VEC,
                                       P.pair + u * VEC};
      }
      u -= n;
    }
  }
  // column u * VEC of those in no part; the parts are in ascending order
  int c = u * VEC;
#pragma unroll
  for (int p = 0; p < U15H_MAX_ROPE_PARTS; ++p) {
    if (p < A.nparts && c >= A.part[p].start) { c += A.part[p].width; }
  }
  return {c, -1, -1};
}

template <int VEC>
struct Cols {
  uint32_t w[VEC / 2 ? VEC / 2 : 1];
};

template <int VEC>
__device__ __forceinline__ Cols<VEC>
load_cols(const uint16_t* p)
{
  Cols<VEC> c;
  if constexpr (VEC == 8) {
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) { c.w[i] = v[i]; }
  } else if constexpr (VEC == 2) {
    c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    c.w[0] = *p;
  }
  return c;
}

template <int VEC>
__device__ __forceinline__ void
store_cols(uint16_t* p, const Cols<VEC>& c)
{
  if constexpr (VEC == 8) {
    *reinterpret_cast<u32x4_t*>(p) = u32x4_t{c.w[0], c.w[1], c.w[2], c.w[3]};
  } else if constexpr (VEC == 2) {
    *reinterpret_cast<uint32_t*>(p) = c.w[0];
  } else {
    *p = (uint16_t)c.w[0];
  }
}

constexpr int kRopePairs = kRopeMaxHeadDim / 2;
// Tokens of a workgroup: as many as give every thread an angle, once there are
// workgroups enough.
constexpr int kRopeGroup = 4;

template <int VEC>
__global__ __launch_bounds__(256) void
rope_kernel(const RopeArgs A, int group, int units, uint32_t units_inv)
{
  __shared__ float2 cs[kRopeGroup * kRopePairs];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * group;
  const int nt = min(group, A.tokens - t0);

  for (int i = tid; i < nt * A.pairs; i += 256) {
    const int tok = i / A.pairs, pair = i % A.pairs;
    double turns = 0.0;
#pragma unroll
    for (int p = 0; p < U15H_MAX_ROPE_PARTS; ++p) {
      if (p < A.nparts && pair >= A.part[p].pair) {
        const RopePart& P = A.part[p];
        if (pair - P.pair < P.width / 2) {
          turns = (double)P.pos[t0 + tok] * (P.freq[pair - P.pair] * 0.15915494309189535);
        }
      }
    }
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cs[i] = make_float2(c * A.scale, s * A.scale * A.sign);
  }
  __syncthreads();

  const int heads = A.q.heads + A.k.heads + A.v.heads;
  const int per = units * heads;
  for (int tok = 0; tok < nt; ++tok) {
    const int t = t0 + tok;
    long long at = 0;                    // the slot's place in head 0's page
    if (A.slot != nullptr) {
      const int slot = A.slot[t];
      if ((unsigned)slot >= (unsigned)A.slots) { continue; }
      at = (long long)(slot >> A.page_log2) * A.page_stride +
           (long long)(slot & ((1 << A.page_log2) - 1)) * A.d;
    }
    const float2* f = cs + tok * A.pairs;
    for (int i = tid; i < per; i += 256) {
      int h = units_inv != 0 ? (int)__umulhi((uint32_t)i, units_inv) : i;
      const int u = i - h * units;
      const uint16_t* x;
      uint16_t* y;
      bool turned = true;
      if (h < A.q.heads) {
        x = A.q.x + t * A.q.x_tok + h * A.q.x_head;
        y = A.q.y + t * A.q.y_tok + h * A.q.y_head;
      } else {
        h -= A.q.heads;
        turned = h < A.k.heads;
        const RopeRows& R = turned ? A.k : A.v;
        h = turned ? h : h - A.k.heads;
        x = R.x + t * R.x_tok + h * R.x_head;
        y = R.y + at + ((long long)h << A.page_log2) * A.d;
      }
      const RopeUnit U = rope_unit<VEC>(A, u);
      Cols<VEC> a = load_cols<VEC>(x + U.a);
      if (U.b >= 0) {
        Cols<VEC> b = load_cols<VEC>(x + U.b);
        if (turned && U.pair >= 0) {
#pragma unroll
          for (int e = 0; e < (VEC + 1) / 2; ++e) {
            const float2 f0 = f[U.pair + 2 * e];
            const float a0 = bf16_lo(a.w[e]), b0 = bf16_lo(b.w[e]);
            float a1 = 0.0f, b1 = 0.0f;
            float2 f1 = make_float2(0.0f, 0.0f);
            if constexpr (VEC > 1) {
              f1 = f[U.pair + 2 * e + 1];
              a1 = bf16_hi(a.w[e]);
              b1 = bf16_hi(b.w[e]);
            }
            a.w[e] = pack_bf16x2(a0 * f0.x - b0 * f0.y, a1 * f1.x - b1 * f1.y);
            b.w[e] = pack_bf16x2(b0 * f0.x + a0 * f0.y, b1 * f1.x + a1 * f1.y);
          }
        }
        store_cols<VEC>(y + U.b, b);
      } else if (turned && U.pair >= 0) {
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float2 f0 = f[U.pair + e];
          const float a0 = bf16_lo(a.w[e]), b0 = bf16_hi(a.w[e]);
          a.w[e] = pack_bf16x2(a0 * f0.x - b0 * f0.y, b0 * f0.x + a0 * f0.y);
        }
      }
      store_cols<VEC>(y + U.a, a);
    }
  }
}

template <int VEC>
hipError_t
launch_rope_vec(const RopeArgs& a, hipStream_t s)
{
  int columns = a.d, units = 0;
  for (int p = 0; p < a.nparts; ++p) {
    columns -= a.part[p].width;
    units += a.part[p].width / ((a.neighbours && VEC > 1) ? VEC : 2 * VEC);
  }
  units += columns / VEC;
  const int group = a.tokens >= 1024 ? kRopeGroup : 1;
  // i / units as a product's high word: exact while i * units < 2^32, and i <
  // 4096 heads * 512; one unit a head (2^32, so 0) needs none
  const uint32_t inv = (uint32_t)(((1ull << 32) + units - 1) / units);
  hipLaunchKernelGGL(rope_kernel<VEC>, dim3((unsigned)((a.tokens + group - 1) / group)),
                     dim3(256), 0, s, a, group, units, inv);
  return hipGetLastError();
}

// ---- attention over a paged cache --------------------------------------------
// Rows (a query head of a token) against keys in pages: the first `prefix` keys
// of prefix_table's pages, then a sequence's own.  Keys are walked in tiles of
// 32; the prefix's last tile and the own keys' first do not share one.
//
// paged_stream_kernel: up to 16 * NR rows of one kv head a workgroup, four
// waves that each take every fourth tile.  Nothing is staged: a wave's tile
// goes from memory to the registers of the matrix instructions (16x16x32).
//  - Scores are transposed, S^T = K Q^T.  The key operand is 16 keys x 32
//    columns, 8 consecutive columns of a key a lane: a 16-byte load.
//  - A lane then holds 8 scores of one row, keys 4 g + r and 16 + 4 g + r of
//    the tile (g = lane / 16, r < 4).  The output is transposed too, O^T = V^T
//    P^T, and takes the tile's keys in just that order, so the lane's own
//    probabilities are the second operand.
//  - The first operand wants 8 keys of one column a lane.  A lane loads 8 keys
//    x D / 16 consecutive columns (whole rows over 16 lanes) and transposes
//    them among its own registers, one v_perm a pair of keys and column.
// The running maximum is raised only when a score passes it by more than kLazy
// (base 2): probabilities stay <= 2^kLazy and the quotient is the same.
// The sum counts the probabilities as rounded to bf16 for the product.

constexpr float kLazy = 8.0f;

__device__ __forceinline__ f32x4_t
mma16(i32x4_t a, i32x4_t b, f32x4_t c)
{
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// max and sum over the lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float
max_groups(float v)
{
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float
sum_groups(float v)
{
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

// A sequence's queries [first, first + n) of q's rows, and its own keys.
struct Sequence {
  int first, n, keys;
};
__device__ __forceinline__ Sequence
sequence(const PagedArgs& A, int b)
{
  int s0 = b, s1 = b + 1;
  if (A.q_start != nullptr) {
    s0 = A.q_start[b];
    s1 = A.q_start[b + 1];
  }
  s0 = min(max(s0, 0), A.tokens);
  s1 = min(max(s1, s0), A.tokens);
  const long long room = (long long)A.table_stride << A.page_log2;
  const int most = (int)min((long long)A.max_kv, room);
  return {uniform(s0), uniform(min(s1 - s0, A.max_q)), uniform(min(max(A.kv_len[b], 0), most))};
}

// The tiles of 32 keys that a workgroup walks: [0, prefix_tiles) the prefix's,
// then the own keys'.
struct Walk {
  const int32_t* table;        // the sequence's pages
  int prefix, keys;            // keys of either
  int prefix_tiles;
};

template <int D, int NR>
__global__ __launch_bounds__(256) void
paged_stream_kernel(const PagedArgs A)
{
  constexpr int W = 4;                       // waves
  constexpr int RB = 16 * NR;                // rows
  constexpr int KS = D / 32;                 // matrix steps of a score
  constexpr int DPL = D / 16;                // columns of V a lane
  constexpr int VW = DPL / 2;                // ... in words
  constexpr int PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float so[W * RB * PITCH];
  __shared__ float sm[W][RB], sl[W][RB];

  const int G = A.hq / A.hkv;
  const int blocks = (A.max_q * G + RB - 1) / RB;
  const int kvh = blockIdx.x % A.hkv;
  const int rb = (blockIdx.x / A.hkv) % blocks;
  const int b = blockIdx.x / (A.hkv * blocks);
  const Sequence S = sequence(A, b);
  const int rows = S.n * G;
  const int row0 = rb * RB;
  if (row0 >= rows) { return; }

  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int lr = lane & 15;
  const int g = lane >> 4;

  Walk K;
  K.table = A.table + (long long)b * A.table_stride;
  K.prefix = A.prefix;
  K.prefix_tiles = (A.prefix + 31) / 32;
  // own keys that the block's last row sees
  const int last = (min(rows, row0 + RB) - 1) / G;
  K.keys = A.causal ? max(S.keys - S.n + last + 1, 0) : S.keys;
  const int tiles = K.prefix_tiles + (K.keys + 31) / 32;

  i32x4_t qf[NR][KS];
  int lim[NR];                               // last own key that the row sees
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = row0 + n * 16 + lr;
    const int tok = row / G, h = kvh * G + row % G;
    const uint16_t* qp = A.q + (S.first + tok) * A.q_tok + h * D + g * 8;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[n][s] = row < rows ? *reinterpret_cast<const i32x4_t*>(qp + s * 32)
                            : i32x4_t{0, 0, 0, 0};
    }
    lim[n] = A.causal ? S.keys - S.n + min(tok, S.n - 1) : S.keys - 1;
  }
  const int lim0 = A.causal ? S.keys - S.n + row0 / G : S.keys - 1;   // the first row's

  // This wave's i-th tile is wave + W * i; lane 2 (i % 32) + block holds the
  // page of its block of 16 keys, -1 where it has none.
  const int mine = (tiles - wave + W - 1) / W;
  auto pages_of = [&](int group) {
    const int tile = wave + W * (group * 32 + (lane >> 1));
    const bool pre = tile < K.prefix_tiles;
    const int key = (pre ? tile : tile - K.prefix_tiles) * 32 + (lane & 1) * 16;
    int id = -1;
    if (key < (pre ? K.prefix : K.keys)) {
      id = (pre ? A.prefix_table : K.table)[key >> A.page_log2];
    }
    return (unsigned)id < (unsigned)A.pages ? id : -1;
  };
  int ids = pages_of(0);

  const int koff = (lr * D + g * 8) * 2;
  const int voff = (4 * g * D + lr * DPL) * 2;
  i32x4_t kf[2][KS];
  uint32_t vr[8][VW];
  struct Block {
    long long at;
    int bytes;
  };
  auto block = [&](int i, int blk) {
    const int tile = wave + W * i;
    const bool pre = tile < K.prefix_tiles;
    const int key = (pre ? tile : tile - K.prefix_tiles) * 32 + blk * 16;
    const int id = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + blk);
    const int left = min((pre ? K.prefix : K.keys) - key, 16);
    Block B;
    B.bytes = id < 0 ? 0 : left * D * 2;
    B.at = max(id, 0) * A.page_stride +
           (((long long)kvh << A.page_log2) + (key & ((1 << A.page_log2) - 1))) * D;
    return B;
  };
  auto load_k = [&](int i) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const Block B = block(i, blk);
      const __amdgpu_buffer_rsrc_t r = make_rsrc(A.k + B.at, B.bytes);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        kf[blk][s] = __builtin_bit_cast(
            i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, koff + s * 64, 0, 0));
      }
    }
  };
  auto load_v = [&](int i) {
#pragma unroll
    for (int blk = 0; blk < 2; ++blk) {
      const Block B = block(i, blk);
      const __amdgpu_buffer_rsrc_t r = make_rsrc(A.v + B.at, B.bytes);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t* to = vr[blk * 4 + e];
        const int off = voff + e * D * 2;
        if constexpr (VW == 4) {
          const u32x4_t v = __builtin_bit_cast(
              u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
          to[0] = v[0];
          to[1] = v[1];
          to[2] = v[2];
          to[3] = v[3];
        } else if constexpr (VW == 2) {
          const u32x2_t v = __builtin_bit_cast(
              u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
          to[0] = v[0];
          to[1] = v[1];
        } else {
          to[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
        }
      }
    }
  };

  f32x4_t o[NR][DPL];
  float m[NR], l[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) { o[n][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}; }
  }
  const float scale = A.scale;

  if (mine > 0) {
    load_k(0);
    load_v(0);
  }
  for (int i = 0; i < mine; ++i) {
    const int tile = wave + W * i;
    const bool pre = tile < K.prefix_tiles;
    const int key0 = (pre ? tile : tile - K.prefix_tiles) * 32;
    const int id0 = __builtin_amdgcn_readlane(ids, 2 * (i & 31));
    const int id1 = __builtin_amdgcn_readlane(ids, 2 * (i & 31) + 1);
    f32x4_t sc[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        sc[n][blk] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < KS; ++s) { sc[n][blk] = mma16(kf[blk][s], qf[n][s], sc[n][blk]); }
      }
    }
    const bool more = i + 1 < mine;
    const bool refill = ((i + 1) & 31) == 0;
    if (refill && more) { ids = pages_of((i + 1) >> 5); }
    if (more) { load_k(i + 1); }

    if (key0 + 31 > (pre ? K.prefix - 1 : lim0) || (id0 | id1) < 0) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int lm = pre ? K.prefix - 1 : lim[n];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = key0 + (e >> 2) * 16 + 4 * g + (e & 3);
          const bool seen = (key <= lm) & ((e < 4 ? id0 : id1) >= 0);
          sc[n][e >> 2][e & 3] = seen ? sc[n][e >> 2][e & 3] : -INFINITY;
        }
      }
    }
    i32x4_t pf[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float mx = fmaxf(fmaxf(fmaxf(sc[n][0][0], sc[n][0][1]), fmaxf(sc[n][0][2], sc[n][0][3])),
                       fmaxf(fmaxf(sc[n][1][0], sc[n][1][1]), fmaxf(sc[n][1][2], sc[n][1][3])));
      mx *= scale;
      if (__any(mx > m[n] + kLazy)) {
        mx = fmaxf(max_groups(mx), m[n]);
        const float alpha = m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[n] - mx);
        m[n] = mx;
        l[n] *= alpha;
#pragma unroll
        for (int j = 0; j < DPL; ++j) { o[n][j] *= alpha; }
      }
      const float mc = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[n][p >> 1][(2 * p) & 3], scale, -mc));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[n][p >> 1][(2 * p + 1) & 3], scale, -mc));
        const uint32_t pk = pack_bf16x2(p0, p1);
        pf[n][p] = (int)pk;
        l[n] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pk),
                                               __builtin_bit_cast(bf16x2_t, 0x3f803f80u), l[n],
                                               false);
      }
    }
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      i32x4_t vf;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        vf[p] = (int)__builtin_amdgcn_perm(vr[2 * p + 1][j >> 1], vr[2 * p][j >> 1],
                                           (j & 1) ? 0x07060302u : 0x05040100u);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) { o[n][j] = mma16(vf, pf[n], o[n][j]); }
    }
    if (more) { load_v(i + 1); }
  }

  // the waves' shares meet in LDS
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const float lt = sum_groups(l[n]);
    if (g == 0) {
      sm[wave][n * 16 + lr] = m[n];
      sl[wave][n * 16 + lr] = lt;
    }
    float* to = so + (wave * RB + n * 16 + lr) * PITCH;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = (4 * g + r) * DPL;
#pragma unroll
      for (int j = 0; j < DPL; ++j) { to[c + j] = o[n][j][r]; }
    }
  }
  __syncthreads();
  for (int i = tid; i < RB * (D / 4); i += 256) {
    const int r = i / (D / 4), c = (i % (D / 4)) * 4;
    if (row0 + r >= rows) { break; }
    float top = sm[0][r];
#pragma unroll
    for (int w = 1; w < W; ++w) { top = fmaxf(top, sm[w][r]); }
    float sum = 0.0f;
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][r] - top);
      sum += f * sl[w][r];
      acc += f * *reinterpret_cast<const f32x4_t*>(so + (w * RB + r) * PITCH + c);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    const int row = row0 + r;
    uint16_t* op = A.out + (S.first + row / G) * A.o_tok + (kvh * G + row % G) * D + c;
    *reinterpret_cast<u32x2_t*>(op) = u32x2_t{pack_bf16x2(acc[0] * inv, acc[1] * inv),
                                              pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  }
}

template <int D>
hipError_t
launch_paged_d(const PagedArgs& a, hipStream_t s)
{
  const int rows = a.max_q * (a.hq / a.hkv);
  const long long blocks = (long long)a.batch * a.hkv * ((rows + 15) / 16);
  hipLaunchKernelGGL((paged_stream_kernel<D, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t
launch_rope(const RopeArgs& a, hipStream_t s)
{
  if (a.vec == 8) { return launch_rope_vec<8>(a, s); }
  if (a.vec == 2) { return launch_rope_vec<2>(a, s); }
  return launch_rope_vec<1>(a, s);
}

hipError_t
launch_paged_attention(const PagedArgs& a, hipStream_t s)
{
  if (a.d == 128) { return launch_paged_d<128>(a, s); }
  if (a.d == 64) { return launch_paged_d<64>(a, s); }
  return launch_paged_d<32>(a, s);
}

bool
paged_kernels_loadable()
{
  const void* fns[] = {
      reinterpret_cast<const void*>(&rope_kernel<8>),
      reinterpret_cast<const void*>(&rope_kernel<2>),
      reinterpret_cast<const void*>(&rope_kernel<1>),
      reinterpret_cast<const void*>(&paged_stream_kernel<128, 1>),
      reinterpret_cast<const void*>(&paged_stream_kernel<64, 1>),
      reinterpret_cast<const void*>(&paged_stream_kernel<32, 1>),
  };
  for (const void* f : fns) {
    hipFuncAttributes a;
    if (hipFuncGetAttributes(&a, f) != hipSuccess) { return false; }
  }
  return true;
}

}  // namespace u15h
