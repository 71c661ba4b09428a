// u15h_paged.hip -- gfx950 kernels for many requests at once: rotary
// positions, the paged K/V cache, attention behind a shared prefix.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

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
// drops out exactly: what is left is in [-1/2, 1/2] and goes through sincospif in
// 32 bits.  Three roundings in 64 bits (the constant, freq times it, the position
// times that) are 3 * 2^-53 of the turns: with freq <= 1 an angle is off by 5e-8
// radians at positions of 2^27, half of what its 32 bits are, and by 8e-7 at 2^31,
// a hundredth of a bf16 column's rounding at most.
//
// Bound by memory, 4 bytes an element.  4224 tokens of 32 heads of 128 turned as
// a whole, 69 MB: 14.4 us with inputs in the caches, 15.7 from memory, as a copy
// of as many bytes; in the model's three parts, whose runs of 32 and 64 bytes
// make more requests, 14.7 and 18.6.  Stepping addresses by addition in place of
// products took a tenth off, a third of neighbouring pairs' 24.5 us.

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
// workgroups enough.  (1, 2, 8: 21.5, 16.0, 18.4 us against 15.7.)
constexpr int kRopeGroup = 4;

struct RopeGrid {
  int group;              // tokens of a workgroup
  int heads;              // of its blockIdx.y's heads, of q, then k, then v
  int units;              // of a head, 256 of them to a blockIdx.z
  int lanes;              // threads of a unit: heads at once
};

// A thread keeps its unit and steps over the (token, head) pairs of q, then k,
// then v, `lanes` of them at a time over the workgroup; addresses go by steps.
// A pair's columns are on their way while the pair before is turned, the first
// ones while the angles are formed.
template <int VEC>
__global__ __launch_bounds__(256) void
rope_kernel(const RopeArgs A, const RopeGrid R)
{
  __shared__ float2 cs[kRopeGroup * kRopePairs];
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * R.group;
  const int nt = min(R.group, A.tokens - t0);
  const int h0 = blockIdx.y * R.heads;
  const int unit0 = blockIdx.z * 256, units = min(R.units - unit0, 256);
  const int lane = (unsigned)tid / (unsigned)units;
  const RopeUnit u = rope_unit<VEC>(A, unit0 + tid - lane * units);

  bool formed = false;
  auto angles = [&] {
    for (int i = tid; i < nt * A.pairs; i += 256) {
      const int tok = (unsigned)i / (unsigned)A.pairs, pair = i - tok * A.pairs;
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
    formed = true;
  };

  struct Item {
    Cols<VEC> a, b;
  };
  // The heads [lo, lo + n) of S, whose first is the workgroups' head `first`, to
  // strided rows or to the cache's slots.
  auto walk = [&](const RopeRows& S, int first, bool cache, bool turn) {
    const int lo = max(h0 - first, 0), n = min(h0 + R.heads - first, S.heads) - lo;
    if (n <= 0) { return; }
    const bool turned = turn && u.pair >= 0;
    // one step: `lanes` pairs on, which is dq tokens and dr heads, and where
    // that passes the last head one token more and n heads less
    const int dq = R.lanes / n, dr = R.lanes - dq * n;
    const long long step = dq * S.x_tok + dr * S.x_head, wrap = S.x_tok - n * S.x_head;
    const long long ystep = dq * S.y_tok + dr * S.y_head, ywrap = S.y_tok - n * S.y_head;
    int tok = lane / n, head = lane - tok * n;
    if (lane >= R.lanes) { tok = nt; }
    const uint16_t* x = S.x + (t0 + tok) * S.x_tok + (lo + head) * S.x_head;
    uint16_t* y = S.y + (t0 + tok) * S.y_tok + (lo + head) * S.y_head;
    auto fetch = [&](Item& I) {
      I.a = load_cols<VEC>(x + u.a);
      if (u.b >= 0) { I.b = load_cols<VEC>(x + u.b); }
    };
    Item I;
    if (tok < nt) { fetch(I); }
    if (!formed) { angles(); }
    while (tok < nt) {
      const int tok0 = tok, head0 = head;
      uint16_t* y0 = y;
      tok += dq;
      head += dr;
      x += step;
      y += ystep;
      if (head >= n) {
        head -= n;
        ++tok;
        x += wrap;
        y += ywrap;
      }
      Cols<VEC> a = I.a, b = I.b;
      if (tok < nt) { fetch(I); }

      if (A.slot != nullptr) {
        const int slot = A.slot[t0 + tok0];
        if ((unsigned)slot >= (unsigned)A.slots) { continue; }
        if (cache) {
          y0 = S.y + (slot >> A.page_log2) * A.page_stride +
               (((long long)(lo + head0) << A.page_log2) + (slot & ((1 << A.page_log2) - 1))) * A.d;
        }
      }
      const float2* f = cs + tok0 * A.pairs + (turned ? u.pair : 0);
      if (u.b >= 0) {
        if (turned) {
#pragma unroll
          for (int e = 0; e < (VEC + 1) / 2; ++e) {
            const float2 f0 = f[2 * e];
            const float a0 = bf16_lo(a.w[e]), b0 = bf16_lo(b.w[e]);
            float a1 = 0.0f, b1 = 0.0f;
            float2 f1 = make_float2(0.0f, 0.0f);
            if constexpr (VEC > 1) {
              f1 = f[2 * e + 1];
              a1 = bf16_hi(a.w[e]);
              b1 = bf16_hi(b.w[e]);
            }
            a.w[e] = pack_bf16x2(a0 * f0.x - b0 * f0.y, a1 * f1.x - b1 * f1.y);
            b.w[e] = pack_bf16x2(b0 * f0.x + a0 * f0.y, b1 * f1.x + a1 * f1.y);
          }
        }
        store_cols<VEC>(y0 + u.b, b);
      } else if (turned) {
#pragma unroll
        for (int e = 0; e < VEC / 2; ++e) {
          const float2 f0 = f[e];
          const float a0 = bf16_lo(a.w[e]), b0 = bf16_hi(a.w[e]);
          a.w[e] = pack_bf16x2(a0 * f0.x - b0 * f0.y, b0 * f0.x + a0 * f0.y);
        }
      }
      store_cols<VEC>(y0 + u.a, a);
    }
  };
  walk(A.q, 0, false, true);
  if (A.slot != nullptr) {
    walk(A.k, A.q.heads, true, true);
    walk(A.v, A.q.heads + A.k.heads, true, false);
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
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  RopeGrid g;
  g.group = a.tokens >= 1024 ? kRopeGroup : 1;
  const int groups = (a.tokens + g.group - 1) / g.group;
  // Few tokens: their heads over several workgroups, 128 units each or more;
  // of an append as many as the cache has, so that one walks q, k or v alone (64
  // tokens of 32 + 8 + 8 heads: 5.2 -> 4.1 us), or twice, thrice .. as many where
  // that makes thousands of workgroups.
  int cut = 1;
  while (groups * cut < 256 && heads * units / (cut * 2) >= 128) { cut *= 2; }
  g.heads = (heads + cut - 1) / cut;
  if (a.slot != nullptr && groups < 512) {
    const long long all = (long long)groups * (heads / a.k.heads);
    g.heads = a.k.heads * (int)((all + 4095) / 4096);
  }
  g.units = units;
  g.lanes = std::max(1, 256 / units);
  hipLaunchKernelGGL(rope_kernel<VEC>, dim3((unsigned)groups, (heads + g.heads - 1) / g.heads,
                                            (units + 255) / 256),
                     dim3(256), 0, s, a, g);
  return hipGetLastError();
}

// ---- attention over a paged cache --------------------------------------------
// Rows (a query head of a token) against keys in pages: the first `prefix` keys
// of prefix_table's pages, then a sequence's own.  Keys are walked in tiles of
// 32; the prefix's last tile and the own keys' first do not share one.
//
// stream_item: up to 16 * NR rows of one kv head a workgroup, four
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
// The running maximum, in the scores' own units, is raised only when a score
// passes it by more than kLazy / scale: probabilities stay <= 2^(2 kLazy) and the
// quotient is the same.  Where the scaled maximum is large the difference comes
// before the product (kFused).
// Probabilities are rounded to bf16, the type in which the matrix unit multiplies
// them by V at its full rate, and the sum counts them as rounded, so that a row's
// weights add up to 1: an output moves by at most 2^-8 of the spread of its values,
// as its own rounding moves it by 2^-8 of itself.
//
// Bound by the keys' bytes: the products of 16 rows take a quarter of a tile's
// time at the memory's rate.  131072 keys of 8 heads of 128 (537 MB) take 91 us,
// 5.9 TB/s, one workgroup a CU; a workgroup alone takes 1.2 us per 128 keys and
// 4.5 before and after.  Eight waves, or a second tile in registers, are level.

constexpr float kLazy = 8.0f;
// Exponents are one fma, score * scale - (max * scale), whose last product is
// rounded: to 2^10 that is at most 2^-14 of a weight, but it grows with the product
// and past 2^31 exceeds the exponential's range, 2^127 and 0 in place of 1.  So above
// 2^10 they are (score - max) * scale, 0 at the maximum whatever the scale: such a
// row takes the maximum's branch at every tile (2 to 3% of a call whose rows are all
// such), and other rows pay nothing (269 us for 4096 queries over 4096 keys, as
// without it; a test of its own: 276).
constexpr float kFused = 1024.0f;

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
sequence_at(const PagedArgs& A, int b)
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
  return {s0, min(s1 - s0, A.max_q), min(max(A.kv_len[b], 0), most)};
}
__device__ __forceinline__ Sequence
sequence(const PagedArgs& A, int b)                    // b the same in all lanes
{
  const Sequence S = sequence_at(A, b);
  return {uniform(S.first), uniform(S.n), uniform(S.keys)};
}

// The partial results of part p: row r's output, and its maximum (of the unscaled
// scores) and sum (the sum kNoKey where the part saw no key of it, kFinal in part 0
// where the row's output is written already).
constexpr float kNoKey = -1.0f, kFinal = -2.0f;
// The sum to leave of a maximum and a sum.  (Scores that are all NaN leave the
// maximum as it was and a sum that is not 0: they are passed on.)
__device__ __forceinline__ float
sum_of(float m, float l)
{
  return m == -INFINITY && l == 0.0f ? kNoKey : l;
}
struct Part {
  float* o;
  float2* ml;
};
__device__ __forceinline__ Part
part_of(const PagedArgs& A, int p)
{
  const long long rows = (long long)A.tokens * A.hq;
  return {A.ws + p * rows * A.d,
          reinterpret_cast<float2*>(A.ws + paged_parts(A) * rows * A.d) + p * rows};
}
__device__ __forceinline__ long long
part_row(const PagedArgs& A, int token, int head)
{
  return (long long)token * A.hq + head;
}
// Marks the rows [row0, row0 + n) of a kv head in the parts [from, to).
__device__ __forceinline__ void
mark_parts(const PagedArgs& A, int from, int to, int first, int G, int kvh, int row0, int n,
           float what)
{
  for (int p = from; p < to; ++p) {
    const Part P = part_of(A, p);
    for (int r = threadIdx.x; r < n; r += 256) {
      const int row = row0 + r;
      P.ml[part_row(A, first + row / G, kvh * G + row % G)] = make_float2(-INFINITY, what);
    }
  }
}

// Values that one workgroup leaves for another of the same launch: written
// through to the memory and read from there, past the dies' own L2.
__device__ __forceinline__ void
give(float* p, float x, float y)
{
  const uint64_t v = (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2
take(const float* p)
{
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// What a workgroup walks: prefix keys, then own keys, each from a tile's start,
// up to tile `end`.
struct Walk {
  const int32_t* table;        // the sequence's pages
  int prefix, keys;
  int prefix_tiles, end;
};

// One workgroup: up to RB rows of a kv head over a share of keys.  The first
// items are the prefix's shares for all rows (where the plan has them on this
// kernel), the others a sequence each.  o0 to o3: RB * D floats of LDS a wave.
template <int D, int NR>
__device__ __forceinline__ void
stream_item(const PagedArgs& A, int item, float* o0, float* o1, float* o2, float* o3,
            float (*sm)[16 * NR], float (*sl)[16 * NR])
{
  constexpr int W = 4;                       // waves
  constexpr int RB = 16 * NR;                // rows
  constexpr int KS = D / 32;                 // matrix steps of a score
  constexpr int DPL = D / 16;                // columns of V a lane
  constexpr int VW = DPL / 2;                // ... in words

  auto so = [&](int w) { return w == 0 ? o0 : w == 1 ? o1 : w == 2 ? o2 : o3; };
  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int lr = lane & 15;
  const int g = lane >> 4;

  const int G = A.hq / A.hkv;
  const int p_shares = A.p_tile ? 0 : A.p_shares;
  const int p_blocks = (A.tokens * G + RB - 1) / RB;
  const int p_items = p_shares * p_blocks * A.hkv;
  const bool phase = item < p_items;
  int kvh, row0, part, share, share_tiles, seq = 0;
  Walk K;
  if (phase) {
    // the blocks of rows of one share of one head 8 apart: one die's L2
    const int runs = p_shares * A.hkv;
    int run;
    if (runs % 8 == 0) {
      run = item / (8 * p_blocks) * 8 + item % 8;
      row0 = item / 8 % p_blocks * RB;
    } else {
      run = item / p_blocks;
      row0 = item % p_blocks * RB;
    }
    kvh = run % A.hkv;
    share = run / A.hkv;
    part = share;
    K.table = nullptr;
    K.prefix = A.prefix;
    share_tiles = A.p_chunk / 32;
  } else {
    item -= p_items;
    const int blocks = (min(A.max_q * G, kPagedShortRows) + RB - 1) / RB;
    kvh = item % A.hkv;
    item /= A.hkv;
    row0 = item % blocks * RB;
    item /= blocks;
    share = item % A.s_shares;
    seq = item / A.s_shares;
    part = A.p_shares + share;
    K.table = A.table + (long long)seq * A.table_stride;
    K.prefix = A.p_shares > 0 ? 0 : A.prefix;
    share_tiles = A.s_chunk / 32;
  }
  K.prefix_tiles = (K.prefix + 31) / 32;

  // This wave's i-th tile is tile0 + W * i; lane 2 (i % 32) + block holds the
  // page of its block of 16 keys, as the table has it (-1 past the table).
  const int tile0 = share * share_tiles + wave;
  auto number = [&](int group) {
    const int tile = tile0 + W * (group * 32 + (lane >> 1));
    const bool pre = tile < K.prefix_tiles;
    const int key = (pre ? tile : tile - K.prefix_tiles) * 32 + (lane & 1) * 16;
    const int at = key >> A.page_log2;
    int id = -1;
    if (pre ? key < K.prefix : (!phase && at < A.table_stride)) {
      id = (pre ? A.prefix_table : K.table)[at];
    }
    return id;
  };
  // the first numbers need no length and are on their way beside the lengths
  int ids = number(0);

  Sequence S = {0, A.tokens, 0};
  if (!phase) { S = sequence(A, seq); }
  const int rows = S.n * G;
  if (row0 >= rows || (!phase && rows > kPagedShortRows)) { return; }
  // own keys that the block's last row sees
  const int last = (min(rows, row0 + RB) - 1) / G;
  K.keys = phase ? 0 : A.causal ? max(S.keys - S.n + last + 1, 0) : S.keys;
  const bool direct = paged_parts(A) == 1;
  const int tiles = K.prefix_tiles + (K.keys + 31) / 32;
  const bool last_share = share == (phase ? p_shares : A.s_shares) - 1;
  K.end = last_share ? tiles : min((share + 1) * share_tiles, tiles);
  if (!phase && last_share) {
    mark_parts(A, part + 1, paged_parts(A), S.first, G, kvh, row0, min(rows - row0, RB), kNoKey);
  }

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

  // a block's page, -1 where it has no keys or its number is not a page
  const int mine = (K.end - tile0 + W - 1) / W;
  auto checked = [&](int id, int group) {
    const int tile = tile0 + W * (group * 32 + (lane >> 1));
    const bool pre = tile < K.prefix_tiles;
    const int key = (pre ? tile : tile - K.prefix_tiles) * 32 + (lane & 1) * 16;
    return key < (pre ? K.prefix : K.keys) && (unsigned)id < (unsigned)A.pages ? id : -1;
  };
  ids = checked(ids, 0);

  const int koff = (lr * D + g * 8) * 2;
  const int voff = (4 * g * D + lr * DPL) * 2;
  i32x4_t kf[2][KS];
  uint32_t vr[8][VW];
  struct Block {
    long long at;
    int bytes;
  };
  auto block = [&](int i, int blk) {
    const int tile = tile0 + W * i;
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
  float mc[NR];                              // what the exponents have subtracted
  float edge[NR];                            // scores past it raise the maximum
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = edge[n] = -INFINITY;
    l[n] = mc[n] = 0.0f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) { o[n][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}; }
  }
  const float scale = A.scale;
  const float lazy = kLazy / scale;

  if (mine > 0) {
    load_k(0);
    load_v(0);
  }
  for (int i = 0; i < mine; ++i) {
    const int tile = tile0 + W * i;
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
    if (refill && more) { ids = checked(number((i + 1) >> 5), (i + 1) >> 5); }
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
      if (__any(mx > edge[n])) {
        mx = fmaxf(max_groups(mx), m[n]);
        const float alpha =
            m[n] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m[n] - mx) * scale);
        m[n] = mx;
        l[n] *= alpha;
#pragma unroll
        for (int j = 0; j < DPL; ++j) { o[n][j] *= alpha; }
        if (mx != -INFINITY) {
          mc[n] = mx * scale;
          edge[n] = mx + lazy;
          if (fabsf(mc[n]) > kFused) {
#pragma unroll
            for (int e = 0; e < 8; ++e) { sc[n][e >> 2][e & 3] -= mx; }
            mc[n] = 0.0f;
            edge[n] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[n][p >> 1][(2 * p) & 3], scale, -mc[n]));
        const float p1 =
            __builtin_amdgcn_exp2f(fmaf(sc[n][p >> 1][(2 * p + 1) & 3], scale, -mc[n]));
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
    // row r's 16-byte chunk c at c ^ r: 16 rows' chunk c spread over the banks
    float* to = so(wave) + (n * 16 + lr) * D;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int j = 0; j < DPL; ++j) {
        const int c = (4 * g + r) * DPL + j;
        to[(((c >> 2) ^ lr) & (D / 4 - 1)) * 4 + (c & 3)] = o[n][j][r];
      }
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
      const float f =
          sm[w][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((sm[w][r] - top) * scale);
      sum += f * sl[w][r];
      acc += f * *reinterpret_cast<const f32x4_t*>(
                     so(w) + r * D + (((c >> 2) ^ (r & 15)) & (D / 4 - 1)) * 4);
    }
    const int row = row0 + r;
    if (!direct) {
      const Part P = part_of(A, part);
      const long long at = part_row(A, S.first + row / G, kvh * G + row % G);
      if (A.joins != nullptr) {
        if (c == 0) {
          give(reinterpret_cast<float*>(P.ml + at), top, sum_of(top, sum));
        }
        if (sum_of(top, sum) == kNoKey) { continue; }
        give(P.o + at * D + c, acc[0], acc[1]);
        give(P.o + at * D + c + 2, acc[2], acc[3]);
        continue;
      }
      if (c == 0) { P.ml[at] = make_float2(top, sum_of(top, sum)); }
      if (sum_of(top, sum) == kNoKey) { continue; }
      *reinterpret_cast<f32x4_t*>(P.o + at * D + c) = acc;
      continue;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    uint16_t* op = A.out + (S.first + row / G) * A.o_tok + (kvh * G + row % G) * D + c;
    *reinterpret_cast<u32x2_t*>(op) = u32x2_t{pack_bf16x2(acc[0] * inv, acc[1] * inv),
                                              pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  }
  if (A.joins == nullptr || direct) { return; }

  // The last share of this block to arrive adds them all, which a second launch
  // does 1 to 2 us slower where the shares are small (1800 keys of one request
  // 11.4 -> 9.5 us) and 1 us faster where they are large (131072 keys).  Every
  // wave waits for its own writes to have reached the memory before the block
  // counts as arrived.
  __shared__ int arrived;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const int blocks = (min(A.max_q * G, kPagedShortRows) + RB - 1) / RB;
    int* count = A.joins + (seq * blocks + row0 / RB) * A.hkv + kvh;
    arrived = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
    if (arrived == A.s_shares) {
      __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (arrived != A.s_shares) { return; }
  // A row over D / 4 threads, `groups` of those on the parts of one row (p =
  // group, group + groups, ..), whose sums meet in LDS; always in that order.
  constexpr int LPR = D / 4, kSlots = 256 / LPR, kAhead = 8;
  const int live = min(rows - row0, RB);
  int span = 1;
  while (span < live && span < kSlots) { span *= 2; }
  const int groups = kSlots / span;
  const int slot = tid / LPR, c = tid % LPR * 4;
  const int grp = slot / span;
  for (int r = slot % span; r - slot % span < live; r += span) {
    const int row = row0 + min(r, live - 1);
    const long long at = part_row(A, S.first + row / G, kvh * G + row % G);
    float m = -INFINITY, l = 0.0f;
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto add = [&](float m1, float l1, f32x4_t o1) {
      if (l1 < 0.0f) { return; }
      const float top = fmaxf(m, m1);
      const float f0 = __builtin_amdgcn_exp2f((m - top) * scale);
      const float f1 = __builtin_amdgcn_exp2f((m1 - top) * scale);
      l = __builtin_fmaf(l, f0, l1 * f1);
#pragma unroll
      for (int e = 0; e < 4; ++e) { acc[e] = __builtin_fmaf(o1[e], f1, acc[e] * f0); }
      m = top;
    };
    for (int p0 = grp; p0 < A.s_shares; p0 += groups * kAhead) {
      float2 ml[kAhead], lo[kAhead], hi[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int p = p0 + i * groups;
        ml[i] = make_float2(-INFINITY, kNoKey);
        lo[i] = hi[i] = make_float2(0.0f, 0.0f);
        if (p < A.s_shares) {
          const Part P = part_of(A, p);
          ml[i] = take(reinterpret_cast<const float*>(P.ml + at));
          lo[i] = take(P.o + at * D + c);
          hi[i] = take(P.o + at * D + c + 2);
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        add(ml[i].x, ml[i].y, f32x4_t{lo[i].x, lo[i].y, hi[i].x, hi[i].y});
      }
    }
    if (groups > 1) {
      // RB rows of D a buffer, kSlots <= 2 RB of them in the first two
      *reinterpret_cast<f32x4_t*>(so(slot / RB) + slot % RB * D + c) = acc;
      if (c == 0) {
        o3[2 * slot] = m;
        o3[2 * slot + 1] = sum_of(m, l);
      }
      __syncthreads();
      if (grp == 0) {
        for (int q = 1; q < groups; ++q) {
          const int other = slot + q * span;
          add(o3[2 * other], o3[2 * other + 1],
              *reinterpret_cast<const f32x4_t*>(so(other / RB) + other % RB * D + c));
        }
      }
    }
    if (grp == 0 && r < live) {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      uint16_t* op = A.out + (S.first + row / G) * A.o_tok + (kvh * G + row % G) * D + c;
      *reinterpret_cast<u32x2_t*>(op) = u32x2_t{pack_bf16x2(acc[0] * inv, acc[1] * inv),
                                                pack_bf16x2(acc[2] * inv, acc[3] * inv)};
    }
  }
}

// tile_item: 128 rows of one kv head a workgroup, for sequences (or
// prefixes of many) whose products outweigh their keys' bytes.  The tile loop is
// attention_kernel's: scores and output transposed on 32x32x16 products, keys
// and values of 64-key tiles copied from memory to LDS and read there by all
// four waves, one barrier a tile, the scores of tile t + 1 beside the
// exponentials of tile t.  What pages add is the address of a copy: a wave
// copies 16 keys, which lie in one page, through a buffer resource of its own
// whose range ends at the last key; so no page ends inside it and keys past the
// end read as zeros.  The page numbers of the next 16 tiles sit in a register,
// a lane each, and are read a group of 16 tiles ahead.
//
// Bound by the matrix unit under the power cap: two workgroups of a CU take 1.8
// us a tile of 64 keys (d = 128).  4096 queries of 32 heads over 4096 keys: 260
// us, 1.06 PFLOP/s, as over the contiguous cache.  A round of workgroups starts
// and ends in 13 us more: four images of 1024 queries over 333 + 1024 keys, two
// rounds, 99 us, 0.92 PFLOP/s.
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef short i16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16_t
mma32(i32x4_t a, i32x4_t b, f32x16_t c)
{
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float
max_halves(float v)
{
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float
sum_halves(float v)
{
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// Swizzle of V's 64-byte blocks: four consecutive keys at one block land on
// four different bank ranges.
template <int D>
__device__ __forceinline__ int
vswz(int r)
{
  return (r * (D / 32) / 4) % (D / 32);
}

constexpr int kTileRows = 128;

// Block `nb` of the long sequences' rows, in blocks of kTileRows: its sequence
// (-1: there is none) and its place within it.  Up to 64 sequences, those with
// the most keys come first, each with its last block, which under the causal
// mask sees the most keys, first: the longest workgroups start early.  More sequences
// are taken as they come, b's blocks from rows before it / 128 + b on, which
// leaves each one block or two that have no rows.
__device__ __forceinline__ int
sequence_of_block(const PagedArgs& A, int G, int nb, int* local, Sequence* S)
{
  const int lane = threadIdx.x & 63;
  if (A.batch <= 64) {
    Sequence mine = {0, 0, -1};
    if (lane < A.batch) { mine = sequence_at(A, lane); }
    const int rows = mine.n * G, keys = mine.keys;
    const int n = rows > kPagedShortRows ? (rows + kTileRows - 1) / kTileRows : 0;
    int start = 0;
    for (int j = 0; j < A.batch; ++j) {
      const int kj = __builtin_amdgcn_readlane(keys, j);
      const bool before = kj > keys || (kj == keys && j < lane);
      start += before ? __builtin_amdgcn_readlane(n, j) : 0;
    }
    const unsigned long long here = __ballot(nb >= start && nb < start + n);
    if (here == 0) { return -1; }
    const int seq = __builtin_ctzll(here);
    *S = {__builtin_amdgcn_readlane(mine.first, seq), __builtin_amdgcn_readlane(mine.n, seq),
          __builtin_amdgcn_readlane(keys, seq)};
    *local = __builtin_amdgcn_readlane(n, seq) - 1 - (nb - __builtin_amdgcn_readlane(start, seq));
    return seq;
  }
  int count = 0, start = 0;
  for (int b0 = 0; b0 < A.batch; b0 += 64) {
    const int b = b0 + lane;
    int f = INT_MAX;
    if (b < A.batch) {
      const int s0 = A.q_start != nullptr ? min(max(A.q_start[b], 0), A.tokens) : b;
      f = s0 * G / kTileRows + b;
    }
    const unsigned long long below = __ballot(f <= nb);
    if (below == 0) { break; }
    const int last = 63 - __builtin_clzll(below);
    count = b0 + last + 1;
    start = __builtin_amdgcn_readlane(f, last);
    if (last < 63) { break; }
  }
  *local = nb - start;
  if (count > 0) { *S = sequence(A, count - 1); }
  return count - 1;
}

template <int D>
__device__ __forceinline__ void
tile_item(const PagedArgs& A, int b, int items, uint16_t* ks0, uint16_t* ks1, uint16_t* vs0,
          uint16_t* vs1)
{
  constexpr int BK = 64;                     // keys of a tile
  constexpr int KCH = D / 8;                 // 16-byte chunks of a key
  constexpr int NDS = D / 16;                // matrix steps of the scores
  constexpr int NCB = D / 32;                // blocks of 32 columns of O
  constexpr int CPW = D / 32;                // 1 KiB copies of a wave's 16 keys

  const int G = A.hq / A.hkv;
  const int p_blocks = (A.tokens * G + kTileRows - 1) / kTileRows;
  const int p_items = A.p_tile ? A.p_shares * p_blocks * A.hkv : 0;
  const bool phase = b < p_items;
  Sequence S;
  const int32_t* table = nullptr;
  int prefix = A.prefix, kvh, row0, part, share, shares, chunk;
  if (phase) {
    // run by run of one head's keys, cut in 8 ranges, one per die
    const int item = p_items % 8 == 0 ? (b % 8) * (p_items / 8) + b / 8 : b;
    row0 = item % p_blocks * kTileRows;
    share = item / p_blocks % A.p_shares;
    kvh = item / (p_blocks * A.p_shares);
    part = share;
    shares = A.p_shares;
    chunk = A.p_chunk;
    S = {0, A.tokens, 0};
  } else {
    b -= p_items;
    items -= p_items;
    int item = items % 8 == 0 ? (b % 8) * (items / 8) + b / 8 : b;
    const int blocks = A.tokens * G / kTileRows + A.batch;
    share = item % A.t_shares;
    item /= A.t_shares;
    int local;
    const int seq = sequence_of_block(A, G, item % blocks, &local, &S);
    kvh = item / blocks;
    part = A.p_shares + share;
    shares = A.t_shares;
    chunk = A.t_chunk;
    if (seq < 0) { return; }
    row0 = uniform(local) * kTileRows;
    if (S.n * G <= kPagedShortRows) { return; }
    table = A.table + (long long)uniform(seq) * A.table_stride;
    if (A.p_shares > 0) { prefix = 0; }
  }
  const int rows = S.n * G;
  if (row0 >= rows) { return; }
  const int parts = paged_parts(A);
  const bool direct = A.p_shares == 0 && shares == 1;
  const int nrows = min(rows - row0, kTileRows);

  const int tid = threadIdx.x;
  const int wave = uniform(tid >> 6);
  const int lane = tid & 63;
  const int lq = lane & 31;
  const int half = lane >> 5;
  const int row = row0 + wave * 32 + lq;
  const bool valid = row < rows;
  const int tok = min(row, rows - 1) / G;
  const int h = kvh * G + row % G;
  const float scale = A.scale;
  const float lazy = kLazy / scale;          // in raw score units

  // own keys: the last that this row, the first row and the last row see
  const int lim = A.causal ? S.keys - S.n + tok : S.keys - 1;
  const int lim0 = A.causal ? S.keys - S.n + row0 / G : S.keys - 1;
  const int keys = A.causal ? max(S.keys - S.n + (row0 + nrows - 1) / G + 1, 0) : S.keys;
  const int ptiles = (prefix + BK - 1) / BK;
  const int all = ptiles + (keys + BK - 1) / BK;
  const int tbeg = min(share * (chunk / BK), all);
  const int ntiles = share == shares - 1 ? all : min(tbeg + chunk / BK, all);
  if (!phase) {
    if (direct) {
      if (parts > 1) { mark_parts(A, 0, 1, S.first, G, kvh, row0, nrows, kFinal); }
    } else if (share == shares - 1) {
      mark_parts(A, part + 1, parts, S.first, G, kvh, row0, nrows, kNoKey);
    }
  }

  i32x4_t qf[NDS];
  const uint16_t* qp = A.q + (S.first + tok) * A.q_tok + h * D;
#pragma unroll
  for (int ds = 0; ds < NDS; ++ds) {
    qf[ds] = valid ? *reinterpret_cast<const i32x4_t*>(qp + ds * 16 + half * 8)
                   : i32x4_t{0, 0, 0, 0};
  }

  // ---- pages ---------------------------------------------------------------
  // Lane 4 i + w: the page of keys [16 w, 16 w + 16) of tile tbeg + 16 group + i,
  // -1 where it has none; `there` has the lanes that have one.
  auto number = [&](int group) {             // as the table has it
    const int t = tbeg + group * 16 + (lane >> 2);
    const bool pre = t < ptiles;
    const int key = (pre ? t : t - ptiles) * BK + (lane & 3) * 16;
    int id = -1;
    if (t < ntiles && key < (pre ? prefix : keys)) {
      id = (pre ? A.prefix_table : table)[key >> A.page_log2];
    }
    return id;
  };
  auto checked = [&](int id) { return (unsigned)id < (unsigned)A.pages ? id : -1; };
  int ids0 = number(0), ids1 = number(1);
  ids0 = checked(ids0);
  ids1 = checked(ids1);
  unsigned long long there0 = __ballot(ids0 >= 0), there1 = __ballot(ids1 >= 0);
  int group = 0;                             // of ids0; ids1 the next one's
  auto page_of = [&](int t) {
    const int i = t - tbeg;
    const int at = 4 * (i & 15) + wave;
    const int a = __builtin_amdgcn_readlane(ids0, at), b = __builtin_amdgcn_readlane(ids1, at);
    return (i >> 4) == group ? a : b;
  };
  auto there_of = [&](int t) {
    const int i = t - tbeg;
    return (int)(((i >> 4) == group ? there0 : there1) >> (4 * (i & 15))) & 15;
  };

  // ---- copies: memory -> LDS -------------------------------------------------
  i32x4_t koffs = {}, voffs = {};
#pragma unroll
  for (int i = 0; i < CPW; ++i) {
    const int idx = i * 64 + lane;                    // landing chunk in the wave's 16 keys
    const int r = idx / KCH;
    koffs[i] = (r * D + (((idx % KCH) ^ (r % KCH)) << 3)) * 2;
    voffs[i] = (r * D + (((idx % KCH) ^ (4 * vswz<D>(r))) << 3)) * 2;
  }
  auto copy = [&](const uint16_t* pool, int t, uint16_t* dst_tile, const i32x4_t& offs) {
    const bool pre = t < ptiles;
    const int key = (pre ? t : t - ptiles) * BK + wave * 16;
    const int id = page_of(t);
    const int left = min((pre ? prefix : keys) - key, 16);
    const long long at = max(id, 0) * A.page_stride +
                         (((long long)kvh << A.page_log2) + (key & ((1 << A.page_log2) - 1))) * D;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(pool + at, id < 0 ? 0 : left * D * 2);
    char* dst = reinterpret_cast<char*>(dst_tile) + wave * CPW * 1024;
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(dst + i * 1024), 16, offs[i], 0, 0, 0);
    }
  };

  // per-lane fragment offsets (elements)
  const int koff = lq * D;                             // + swizzled chunk
  const int vrow = 4 * half + ((lane & 15) >> 2);      // transpose-read key
  const int vcol = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  f32x16_t o[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) { o[cb] = f32x16_t{}; }
  float m = -INFINITY;      // running max, raw score units
  float mc = 0.0f;          // what the exponents have subtracted
  float edge = -INFINITY;   // scores past it raise the maximum
  float l = 0.0f;           // this half's share of the running sum
  f32x16_t sc[2];           // scores of the current tile

  auto mask = [&](f32x16_t (&s)[2], int t) {
    const bool pre = t < ptiles;
    const int j0 = (pre ? t : t - ptiles) * BK;
    const int there = there_of(t);
    if (j0 + BK - 1 <= (pre ? prefix - 1 : lim0) && there == 15) { return; }
    const int last = pre ? prefix - 1 : lim;
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      const int kl = (r >> 4) * 32 + 8 * ((r & 15) >> 2) + 4 * half + (r & 3);
      const bool ok = (j0 + kl <= last) &
                      (((there >> ((r >> 4) * 2 + ((r & 15) >> 3))) & 1) != 0);
      s[r >> 4][r & 15] = ok ? s[r >> 4][r & 15] : -INFINITY;
    }
  };
  uint32_t pk[16];
  float ps;
  auto expo = [&](const f32x16_t& s, int r, int slot) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -mc));
    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], scale, -mc));
    pk[slot] = pack_bf16x2(p0, p1);
    ps = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pk[slot]),
                                         __builtin_bit_cast(bf16x2_t, 0x3f803f80u), ps, false);
  };
  auto pv = [&](const uint16_t* vread, int k4, int cb) {
    const i32x4_t pf = {(int)pk[k4 * 4 + 0], (int)pk[k4 * 4 + 1], (int)pk[k4 * 4 + 2],
                        (int)pk[k4 * 4 + 3]};
    const int r0 = k4 * 16 + vrow;
    const int c = (((cb ^ vswz<D>(r0)) << 5) | vcol);     // r0, r0 + 8 share it
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4_t*)(vread + r0 * D + c));
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4_t*)(vread + (r0 + 8) * D + c));
    const i32x4_t vf = {__builtin_bit_cast(int, (i16x2_t){lo[0], lo[1]}),
                        __builtin_bit_cast(int, (i16x2_t){lo[2], lo[3]}),
                        __builtin_bit_cast(int, (i16x2_t){hi[0], hi[1]}),
                        __builtin_bit_cast(int, (i16x2_t){hi[2], hi[3]})};
    o[cb] = mma32(vf, pf, o[cb]);
  };

  // Raises the maximum to mb, that of the scores `s` of the tile that is next, where
  // they pass it by enough.  It stands before an iteration's barrier: scores that
  // change at the start of the next would be copied there (170 -> 177 us for 4096
  // queries over 4096 keys, d = 64), and after the barrier all wait for the test.
  auto raise = [&](float mb, f32x16_t (&s)[2]) {
    if (mb > edge) {
      mb = fmaxf(mb, m);
      const float alpha = exp2f((m - mb) * scale);     // 0 while m is -inf
      l *= alpha;
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) { o[cb][r] *= alpha; }
      }
      m = mb;
      mc = m * scale;
      edge = m + lazy;
      if (fabsf(mc) > kFused) {
#pragma unroll
        for (int r = 0; r < 32; ++r) { s[r >> 4][r & 15] -= m; }
        mc = 0.0f;
        edge = -INFINITY;
      }
    }
  };

  // One iteration over tile t: A scores of tile t + 1 | exponentials of keys
  // 0..31; B P V of keys 0..31 | exponentials of keys 32..63; C P V of keys
  // 32..63 | mask and max of tile t + 1's scores.
  constexpr int EPA = 16 / NDS, EPB = 16 / (2 * NCB), MPC = 32 / (2 * NCB);
  auto iteration = [&](int t, const uint16_t* kread, uint16_t* kfill, const uint16_t* vread,
                       uint16_t* vfill) {
    ps = 0.0f;
    copy(A.k, t + 2, kfill, koffs);
    copy(A.v, t + 1, vfill, voffs);

    f32x16_t sn[2] = {f32x16_t{}, f32x16_t{}};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      const int off = koff + (((ds * 2 + half) ^ (lq % KCH)) << 3);
      const i32x4_t k0 = *reinterpret_cast<const i32x4_t*>(kread + off);
      const i32x4_t k1 = *reinterpret_cast<const i32x4_t*>(kread + 32 * D + off);
      sn[0] = mma32(k0, qf[ds], sn[0]);
#pragma unroll
      for (int e = 0; e < EPA; e += 2) { expo(sc[0], ds * EPA + e, (ds * EPA + e) >> 1); }
      sn[1] = mma32(k1, qf[ds], sn[1]);
    }
#pragma unroll
    for (int k4 = 0; k4 < 2; ++k4) {
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        pv(vread, k4, cb);
        const int r = (k4 * NCB + cb) * EPB;
#pragma unroll
        for (int e = 0; e < EPB; e += 2) { expo(sc[1], r + e, 8 + ((r + e) >> 1)); }
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);                // reads 0, 1
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);              // MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, 6 * EPA / 4, 0);    // VALU
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);              // reads +2
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);              // MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, 6 * EPA / 4, 0);    // VALU
    }
#pragma unroll
    for (int i = 0; i < 2 * NCB; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);              // MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, 6 * EPB / 4, 0);    // VALU
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);              // reads +2
      __builtin_amdgcn_sched_group_barrier(0x002, 6 * EPB / 4, 0);    // VALU
    }
    // (past the last tile the scores come from stale K and are dropped)
    if (t + 1 < ntiles) { mask(sn, t + 1); }
    float mx = -INFINITY;
#pragma unroll
    for (int k4 = 2; k4 < 4; ++k4) {
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        pv(vread, k4, cb);
        const int r = ((k4 - 2) * NCB + cb) * MPC;
#pragma unroll
        for (int e = 0; e < MPC; ++e) { mx = fmaxf(mx, sn[(r + e) >> 4][(r + e) & 15]); }
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);                // reads 0, 1
#pragma unroll
    for (int i = 0; i < 2 * NCB; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);              // MFMA
      __builtin_amdgcn_sched_group_barrier(0x002, MPC / 2, 0);        // VALU
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);              // reads +2
    }
    mx = max_halves(mx);
    l += ps;
    // Tiles t + 2 and t + 3 are next: from the end of a group on, its
    // successor.  The one after that is read here and looked at half a group
    // later; it is needed from tile 14 of the group on.
    if (((t + 1 - tbeg) & 7) == 0) {
      if (((t + 1 - tbeg) & 8) == 0) {
        ids0 = ids1;
        there0 = there1;
        ++group;
        ids1 = number(group + 1);
      } else if (group > 0) {
        ids1 = checked(ids1);
        there1 = __ballot(ids1 >= 0);
      }
    }
    if (t + 1 < ntiles) { raise(mx, sn); }
    __syncthreads();
    sc[0] = sn[0];
    sc[1] = sn[1];
  };

  if (tbeg < ntiles) {
    copy(A.k, tbeg, ks0, koffs);
    copy(A.k, tbeg + 1, ks1, koffs);
    copy(A.v, tbeg, vs0, voffs);
    __syncthreads();
    sc[0] = f32x16_t{};
    sc[1] = f32x16_t{};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      const int off = koff + (((ds * 2 + half) ^ (lq % KCH)) << 3);
      sc[0] = mma32(*reinterpret_cast<const i32x4_t*>(ks0 + off), qf[ds], sc[0]);
      sc[1] = mma32(*reinterpret_cast<const i32x4_t*>(ks0 + 32 * D + off), qf[ds], sc[1]);
    }
    mask(sc, tbeg);
    float mx = sc[0][0];
#pragma unroll
    for (int r = 1; r < 32; ++r) { mx = fmaxf(mx, sc[r >> 4][r & 15]); }
    raise(max_halves(mx), sc);
    __syncthreads();
  }
  for (int t = tbeg; t < ntiles;) {
    iteration(t, ks1, ks0, vs0, vs1);
    if (++t >= ntiles) { break; }
    iteration(t, ks0, ks1, vs1, vs0);
    ++t;
  }

  l = sum_halves(l);
  if (!valid) { return; }
  if (!direct) {
    const Part P = part_of(A, part);
    const long long at = part_row(A, S.first + tok, h);
    if (half == 0) { P.ml[at] = make_float2(m, sum_of(m, l)); }
    if (sum_of(m, l) == kNoKey) { return; }
    float* op = P.o + at * D;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        *reinterpret_cast<f32x4_t*>(op + cb * 32 + 8 * g + 4 * half) =
            f32x4_t{o[cb][4 * g], o[cb][4 * g + 1], o[cb][4 * g + 2], o[cb][4 * g + 3]};
      }
    }
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint16_t* op = A.out + (S.first + tok) * A.o_tok + h * D;
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      *reinterpret_cast<u32x2_t*>(op + cb * 32 + 8 * g + 4 * half) =
          u32x2_t{pack_bf16x2(o[cb][4 * g] * inv, o[cb][4 * g + 1] * inv),
                  pack_bf16x2(o[cb][4 * g + 2] * inv, o[cb][4 * g + 3] * inv)};
    }
  }
}

// The kernel: workgroups of tile items first, the longest, then of streaming
// ones, which fill the CUs as those end (256 sequences behind 32768 keys: 167 us
// with almost no own keys, 56 with almost no prefix, 182 with both; a streaming
// workgroup beside every tile one from the start: 212).  TILE or STREAM alone
// where a call has only those.
template <int D, int NR, bool TILE, bool STREAM>
__global__ __launch_bounds__(256, TILE ? 2 : 1) void
paged_kernel(const PagedArgs A, int tile_items)
{
  constexpr int kBuf = TILE ? 64 * D : 32 * NR * D;     // in 2 bytes
  __shared__ __attribute__((aligned(16))) uint16_t b0[kBuf];
  __shared__ __attribute__((aligned(16))) uint16_t b1[kBuf];
  __shared__ __attribute__((aligned(16))) uint16_t b2[kBuf];
  __shared__ __attribute__((aligned(16))) uint16_t b3[kBuf];
  if constexpr (TILE) {
    if (!STREAM || (int)blockIdx.x < tile_items) {
      tile_item<D>(A, blockIdx.x, tile_items, b0, b1, b2, b3);
      return;
    }
  }
  if constexpr (STREAM) {
    __shared__ float sm[4][16 * NR], sl[4][16 * NR];
    stream_item<D, NR>(A, blockIdx.x - tile_items, reinterpret_cast<float*>(b0),
                       reinterpret_cast<float*>(b1), reinterpret_cast<float*>(b2),
                       reinterpret_cast<float*>(b3), sm, sl);
  }
}

// Whether a token is a row of some sequence.
__device__ __forceinline__ bool
in_sequence(const PagedArgs& A, int token)
{
  if (A.q_start == nullptr) { return token < A.batch; }
  // the last b with q_start[b] <= token, 64 at a time
  const int lane = threadIdx.x & 63;
  int b = -1, first = 0;
  for (int b0 = 0; b0 < A.batch; b0 += 64) {
    const int s0 = b0 + lane < A.batch ? A.q_start[b0 + lane] : INT_MAX;
    const unsigned long long below = __ballot(s0 <= token);
    if (below == 0) { break; }
    const int last = 63 - __builtin_clzll(below);
    b = b0 + last;
    first = max(__builtin_amdgcn_readlane(s0, last), 0);
    if (last < 63) { break; }
  }
  return b >= 0 && token < A.q_start[b + 1] && token - first < A.max_q;
}

// Adds the parts of a row, W waves a row, in the order of the parts:
// out = sum f_p o_p / sum f_p l_p with f_p = 2^((m_p - max m) scale).  All of a lane's
// loads go out before the row is looked up.  Bound by latency and the parts'
// bytes: 2048 rows of 7 parts 4.9 us, 8192 rows of 7 (30 MB) 12.4.
template <int D, int W>
__global__ __launch_bounds__(256) void
paged_combine_kernel(const PagedArgs A)
{
  constexpr int C = D / 32;                  // columns a lane
  constexpr int kAhead = W == 1 ? 8 : 4;
  __shared__ float so[4][D];
  __shared__ float2 sml[4];
  const int wave = uniform(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int half = lane >> 5;                // parts 2 i + half
  const int c = (lane & 31) * C;
  const long long row = (long long)blockIdx.x * (4 / W) + wave / W;
  const int token = (int)(row / A.hq);
  const int n = paged_parts(A);
  const bool there = row < (long long)A.tokens * A.hq;

  float m = -INFINITY, l = 0.0f, o[C];
#pragma unroll
  for (int e = 0; e < C; ++e) { o[e] = 0.0f; }
  auto add = [&](float m1, float l1, const float* o1) {
    if (l1 < 0.0f) { return; }
    const float top = fmaxf(m, m1);
    const float f0 = __builtin_amdgcn_exp2f((m - top) * A.scale);
    const float f1 = __builtin_amdgcn_exp2f((m1 - top) * A.scale);
    l = __builtin_fmaf(l, f0, l1 * f1);
#pragma unroll
    for (int e = 0; e < C; ++e) { o[e] = __builtin_fmaf(o1[e], f1, o[e] * f0); }
    m = top;
  };
  if (there) {
    for (int p0 = (wave % W) * 2 + half; p0 < n; p0 += 2 * W * kAhead) {
      float2 ml[kAhead];
      float o1[kAhead][C];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int p = p0 + 2 * W * i;
        ml[i] = make_float2(-INFINITY, kNoKey);
        if (p < n) {
          const Part P = part_of(A, p);
          ml[i] = P.ml[row];
          typedef float vec_t __attribute__((ext_vector_type(C)));
          const vec_t v = *reinterpret_cast<const vec_t*>(P.o + row * D + c);
#pragma unroll
          for (int e = 0; e < C; ++e) { o1[i][e] = v[e]; }
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) { add(ml[i].x, ml[i].y, o1[i]); }
    }
  }
  bool live = there && in_sequence(A, token);
  if (live && A.longs) { live = part_of(A, 0).ml[row].y != kFinal; }
  // the halves, then the waves
  {
    const float m1 = __shfl_xor(m, 32), l1 = __shfl_xor(l, 32);
    float o1[C];
#pragma unroll
    for (int e = 0; e < C; ++e) { o1[e] = __shfl_xor(o[e], 32); }
    add(m1, sum_of(m1, l1), o1);
  }
  if constexpr (W > 1) {
    if (half == 0) {
#pragma unroll
      for (int e = 0; e < C; ++e) { so[wave][c + e] = o[e]; }
      if (lane == 0) { sml[wave] = make_float2(m, sum_of(m, l)); }
    }
    __syncthreads();
    if (wave % W != 0) { return; }
#pragma unroll
    for (int w = 1; w < W; ++w) {
      float o1[C];
#pragma unroll
      for (int e = 0; e < C; ++e) { o1[e] = so[wave + w][c + e]; }
      add(sml[wave + w].x, sml[wave + w].y, o1);
    }
  }
  if (!live || half != 0) { return; }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint16_t* op = A.out + token * A.o_tok + (row - (long long)token * A.hq) * D + c;
  if constexpr (C == 4) {
    *reinterpret_cast<u32x2_t*>(op) =
        u32x2_t{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
  } else if constexpr (C == 2) {
    *reinterpret_cast<uint32_t*>(op) = pack_bf16x2(o[0] * inv, o[1] * inv);
  } else {
    *op = (uint16_t)pack_bf16x2(o[0] * inv, 0.0f);
  }
}

__global__ __launch_bounds__(256) void
clear_joins_kernel(int* joins)
{
  joins[blockIdx.x * 256 + threadIdx.x] = 0;
}

template <int D>
hipError_t
launch_paged_d(const PagedArgs& a, hipStream_t s)
{
  const int G = a.hq / a.hkv, RB = 16 * a.nr;
  const long long rows = (long long)a.tokens * G;
  const long long tiles =
      (a.p_tile ? a.p_shares * a.hkv * ((rows + kTileRows - 1) / kTileRows) : 0) +
      (a.longs ? a.t_shares * a.hkv * (rows / kTileRows + a.batch) : 0);
  const int blocks = (std::min(a.max_q * G, kPagedShortRows) + RB - 1) / RB;
  const long long streams = (a.p_tile ? 0 : a.p_shares * a.hkv * ((rows + RB - 1) / RB)) +
                            (a.shorts ? (long long)a.batch * a.s_shares * blocks * a.hkv : 0);
#define U15H_RUN(NR, T, S)                                                                       \
  hipLaunchKernelGGL((paged_kernel<D, NR, T, S>), dim3((unsigned)(tiles + streams)), dim3(256), 0, \
                     s, a, (int)tiles)
  if (streams == 0) {
    U15H_RUN(1, true, false);
  } else if (tiles == 0) {
    if (a.nr == 1) { U15H_RUN(1, false, true); } else { U15H_RUN(2, false, true); }
  } else {
    if (a.nr == 1) { U15H_RUN(1, true, true); } else { U15H_RUN(2, true, true); }
  }
#undef U15H_RUN
  const hipError_t e = hipGetLastError();
  const int parts = paged_parts(a);
  if (e != hipSuccess || parts == 1 || a.joins != nullptr) { return e; }
  const unsigned outs = (unsigned)a.tokens * a.hq;
  if (parts > 8 && outs < 4096) {
    hipLaunchKernelGGL((paged_combine_kernel<D, 4>), dim3(outs), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((paged_combine_kernel<D, 1>), dim3((outs + 3) / 4), dim3(256), 0, s, a);
  }
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

hipError_t
launch_clear_joins(int* joins, hipStream_t s)
{
  static_assert(kPagedJoins % 256 == 0, "a thread a counter");
  hipLaunchKernelGGL(clear_joins_kernel, dim3(kPagedJoins / 256), dim3(256), 0, s, joins);
  return hipGetLastError();
}

bool
paged_kernels_loadable()
{
  const void* fns[] = {
      reinterpret_cast<const void*>(&clear_joins_kernel),
      reinterpret_cast<const void*>(&rope_kernel<8>),
      reinterpret_cast<const void*>(&rope_kernel<2>),
      reinterpret_cast<const void*>(&rope_kernel<1>),
#define U15H_FN(D)                                                   \
  reinterpret_cast<const void*>(&paged_kernel<D, 1, true, false>),   \
      reinterpret_cast<const void*>(&paged_kernel<D, 1, false, true>), \
      reinterpret_cast<const void*>(&paged_kernel<D, 2, false, true>), \
      reinterpret_cast<const void*>(&paged_kernel<D, 1, true, true>),  \
      reinterpret_cast<const void*>(&paged_kernel<D, 2, true, true>),  \
      reinterpret_cast<const void*>(&paged_combine_kernel<D, 1>),      \
      reinterpret_cast<const void*>(&paged_combine_kernel<D, 4>),
      U15H_FN(128) U15H_FN(64) U15H_FN(32)
#undef U15H_FN
  };
  for (const void* f : fns) {
    hipFuncAttributes a;
    if (hipFuncGetAttributes(&a, f) != hipSuccess) { return false; }
  }
  return true;
}

}  // namespace u15h
