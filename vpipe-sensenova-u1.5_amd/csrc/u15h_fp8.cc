// u15h_fp8.cc -- the fp8 tier's entry points (include/u15h.h): argument checks
// (nothing is launched on a refusal) and the batch tables of u15h_fp8.hip.
#include "u15h.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "u15h_internal.h"

namespace {

using u15h::Fp8Batch;
using u15h::Fp8Problem;

constexpr int kMaxK = 131072;
constexpr int kMaxRows = 1 << 22;    // a norm's workgroups of 512 threads: 2^31 threads
constexpr int kMaxN = 1 << 20;

u15h_status
refuse(u15h_ctx* ctx, const char* fmt, ...)
{
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return u15h::set_error(ctx, U15H_EINVAL, buf);
}

bool
usable(const void* p)
{
  return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

bool
usable_or_null(const void* p)
{
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// Rows of `width` codes: every row starts 16-byte aligned.
u15h_status
check_width(u15h_ctx* ctx, const char* what, int width, int most)
{
  if (width <= 0 || width % 16 != 0 || width > most) {
    return refuse(ctx, "%s: width %d must be a positive multiple of 16, at most %d", what, width,
                  most);
  }
  return U15H_OK;
}

u15h_status
check_rows(u15h_ctx* ctx, const char* what, int und, int gen)
{
  if (und < 0 || gen < 0 || (long long)und + gen > kMaxRows) {
    return refuse(ctx, "%s: rows=%d+%d (each >= 0, at most %d together)", what, und, gen,
                  kMaxRows);
  }
  return U15H_OK;
}

// The codes and scales of rows (up null) or of silu(x) * up.
u15h_status
quant_rows(u15h_ctx* ctx, u15h_stream stream, const char* what, const u15h_bf16* x,
           const u15h_bf16* up, int rows, int width, u15h_bf16* h, uint8_t* q, float* s)
{
  const u15h_status st = u15h::begin_call(ctx);
  if (st != U15H_OK) { return st; }
  return u15h::end_call(ctx,
                        u15h::launch_fp8_quant_rows(x, up, rows, width, h, q, s,
                                                    reinterpret_cast<hipStream_t>(stream)),
                        what);
}

void
add_problem(Fp8Batch& b, const uint8_t* a, const float* sa, const uint8_t* w, const float* sw,
            uint16_t* y, int rows, int n)
{
  if (rows <= 0) { return; }
  Fp8Problem& p = b.p[b.nprob++];
  p.a = a;
  p.sa = sa;
  p.w = w;
  p.sw = sw;
  p.y = y;
  p.rows = rows;
  p.n = n;
}

// The kinds of launch, and what a call takes on each, in us: `fixed`, then
//   narrow: `round` per workgroup of the busiest CU, `stage` per block of K of
//           those, `stream` per block of all of them over the CUs;
//   tiles:  `round` and `stage` per round of workgroups (a CU that runs two
//           takes two stages), `split` for the second launch with K shares,
//           `share` for each of them and `part` per MB of their sums;
//   and `weight` per MB of weights.
// Fitted to 7096 timings (a graph, weights rotated; M 1-4224, K 256-12288, N
// 512-24576, every kind and 1 to 16 shares), each to 5-9% on the mean; the kind
// and shares with the least estimate take 0.8% longer than the fastest of all,
// on the mean over the 338 sizes, and 18% at worst (64 rows, K 8192, N 1024:
// 13.4 against 11.4 us).
struct Kind {
  bool narrow;
  int bm, bn;
  double fixed, round, stage, stream, split, part, weight, share;
};
constexpr Kind kKinds[] = {
    {true, 16, 16, 2.39, 0.50, 0.0502, 0.0471, 0, 0, 0, 0},
    {true, 16, 32, 1.97, 1.30, 0.0822, 0.1000, 0, 0, 0, 0},
    {true, 32, 16, 1.70, 1.48, 0.0698, 0.0466, 0, 0, 0, 0},
    {true, 32, 32, 2.42, 1.12, 0.1004, 0.0987, 0, 0, 0, 0},
    {true, 64, 16, 1.40, 1.97, 0.1184, 0.0536, 0, 0, 0, 0},
    {true, 64, 32, 2.95, 0.99, 0.1478, 0.1196, 0, 0, 0, 0},
    {true, 96, 16, 1.42, 2.11, 0.1672, 0.0479, 0, 0, 0, 0},
    {true, 128, 16, 1.38, 2.48, 0.2095, 0.0507, 0, 0, 0, 0},
    {false, 64, 128, 3.67, 0.34, 0.316, 0, 2.63, 0.335, 0.130, 0.164},
    {false, 128, 128, 3.09, 1.70, 0.426, 0, 2.69, 0.364, 0.100, 0.141},
    {false, 128, 256, 3.14, 2.63, 0.674, 0, 2.76, 0.284, 0.119, 0.165},
    {false, 192, 256, 5.86, 0.98, 1.093, 0, 2.67, 0.200, 0.144, 0.198},
    {false, 256, 256, 7.82, 0, 1.307, 0, 3.91, 0.117, 0.109, 0.235},
};

// Counts a batch's tiles on a kind and cuts its last partial round in `shares`
// shares of K; false if the tiles are too many.
bool
set_tiles(Fp8Batch& b, const Kind& k, int shares)
{
  b.narrow = k.narrow;
  b.bm = k.bm;
  b.bn = k.bn;
  long long tiles = 0;
  for (int i = 0; i < b.nprob; ++i) {
    Fp8Problem& q = b.p[i];
    q.tiles_m = (q.rows + k.bm - 1) / k.bm;
    q.tiles_n = (q.n + k.bn - 1) / k.bn;
    q.tile_begin = (int)tiles;
    tiles += (long long)q.tiles_m * q.tiles_n;
    if (tiles > (1 << 28)) { return false; }
  }
  b.total_tiles = b.split_begin = (int)tiles;
  b.split = shares;
  if (shares > 1) { b.split_begin -= b.total_tiles % (u15h::fp8_tiles_per_cu(k.bm, k.bn) * b.cus); }
  return true;
}

// Chooses a batch's kind and shares by their estimates; false if the tiles are
// too many.
bool
plan(Fp8Batch& b, size_t workspace)
{
  const int C = b.cus, nb = (b.K + u15h::kFp8Block - 1) / u15h::kFp8Block;
  int rows = 0;
  double mb = 0;                                   // the weights'
  for (int i = 0; i < b.nprob; ++i) {
    rows = std::max(rows, b.p[i].rows);
    mb += 1e-6 * b.p[i].n * b.K;
  }
  const Kind* best = nullptr;
  int best_shares = 1;
  double least = 0;
  auto consider = [&](const Kind& k, int shares, double us) {
    if (best == nullptr || us < least) {
      best = &k;
      best_shares = shares;
      least = us;
    }
  };
  for (const Kind& k : kKinds) {
    if (k.narrow && rows > k.bm) { continue; }
    long long tiles = 0, valid = 0, padded = 0;
    for (int i = 0; i < b.nprob; ++i) {
      const long long tn = (b.p[i].n + k.bn - 1) / k.bn, tm = (b.p[i].rows + k.bm - 1) / k.bm;
      tiles += tm * tn;
      valid += b.p[i].rows * tn;
      padded += tm * k.bm * tn;
    }
    if (k.narrow) {
      const long long load = (tiles + C - 1) / C;
      consider(k, 1, k.fixed + load * (k.round + nb * k.stage) + (double)tiles * nb / C * k.stream);
      continue;
    }
    const int two = u15h::fp8_tiles_per_cu(k.bm, k.bn), slots = two * C;
    const long long full = tiles / slots, rem = tiles % slots;
    const double fixed = k.fixed + mb * k.weight + full * (k.round + nb * two * k.stage);
    if (best != nullptr && fixed >= least) { continue; }
    const double tile_mb = 4e-6 * k.bm * k.bn;
    for (int S = 1; S <= 16; S += S < 4 ? 1 : S < 8 ? 2 : 4) {
      if (S > 1 && (rem == 0 || S > nb / 2 || rem * S > 2 * slots ||
                    (size_t)(rem * S * k.bm * k.bn) * 4 > workspace)) {
        break;
      }
      double us = fixed;
      if (rem > 0) {
        const int nst = (nb + S - 1) / S;
        const long long rounds = (rem * S + slots - 1) / slots;
        // the last of them may have a CU to each workgroup
        const int last = rem * S - (rounds - 1) * slots > C ? two : 1;
        us += rounds * k.round + ((rounds - 1) * two + last) * nst * k.stage;
      }
      if (S > 1) { us += k.split + S * k.share + rem * S * tile_mb * valid / padded * k.part; }
      consider(k, S, us);
    }
  }
  return set_tiles(b, *best, best_shares);
}

}  // namespace

extern "C" {

u15h_status
u15h_quant_rows_fp8(u15h_ctx* ctx, u15h_stream stream, const u15h_bf16* x, int rows, int K,
                    uint8_t* q, float* s)
{
  if (ctx == nullptr) { return U15H_EINVAL; }
  u15h_status st = check_width(ctx, "quant_rows_fp8", K, kMaxK);
  if (st == U15H_OK) { st = check_rows(ctx, "quant_rows_fp8", rows, 0); }
  if (st != U15H_OK) { return st; }
  if (rows == 0) { return u15h::end_call(ctx, hipSuccess, ""); }
  if (!usable(x) || !usable(q) || !usable(s)) {
    return refuse(ctx, "quant_rows_fp8: null or misaligned operand");
  }
  return quant_rows(ctx, stream, "quant_rows_fp8", x, nullptr, rows, K, nullptr, q, s);
}

u15h_status
u15h_swiglu_quant_fp8(u15h_ctx* ctx, u15h_stream stream, const u15h_bf16* gate,
                      const u15h_bf16* up, int rows, int inter, u15h_bf16* h, uint8_t* q, float* s)
{
  if (ctx == nullptr) { return U15H_EINVAL; }
  u15h_status st = check_width(ctx, "swiglu_quant_fp8", inter, kMaxK);
  if (st == U15H_OK) { st = check_rows(ctx, "swiglu_quant_fp8", rows, 0); }
  if (st != U15H_OK) { return st; }
  if (rows == 0) { return u15h::end_call(ctx, hipSuccess, ""); }
  if (!usable(gate) || !usable(up) || !usable(q) || !usable(s) || !usable_or_null(h)) {
    return refuse(ctx, "swiglu_quant_fp8: null or misaligned operand");
  }
  return quant_rows(ctx, stream, "swiglu_quant_fp8", gate, up, rows, inter, h, q, s);
}

u15h_status
u15h_quant_blocks_fp8(u15h_ctx* ctx, u15h_stream stream, const u15h_bf16* w, int N, int K,
                      uint8_t* q, float* s)
{
  if (ctx == nullptr) { return U15H_EINVAL; }
  u15h_status st = check_width(ctx, "quant_blocks_fp8", K, kMaxK);
  if (st != U15H_OK) { return st; }
  if (N < 0 || N > kMaxN) {
    return refuse(ctx, "quant_blocks_fp8: N=%d (0 to %d)", N, kMaxN);
  }
  if (N == 0) { return u15h::end_call(ctx, hipSuccess, ""); }
  if (!usable(w) || !usable(q) || !usable(s)) {
    return refuse(ctx, "quant_blocks_fp8: null or misaligned operand");
  }
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  return u15h::end_call(
      ctx, u15h::launch_fp8_quant_blocks(w, N, K, q, s, reinterpret_cast<hipStream_t>(stream)),
      "quant_blocks_fp8");
}

u15h_status
u15h_mot_rms_norm_fp8(u15h_ctx* ctx, u15h_stream stream, const u15h_bf16* x,
                      const u15h_bf16* delta, u15h_bf16* x_out, int M_und, int M_gen, int dim,
                      const u15h_bf16* w_und, const u15h_bf16* w_gen, float eps, u15h_bf16* y,
                      uint8_t* q, float* s)
{
  if (ctx == nullptr) { return U15H_EINVAL; }
  const char* const what = "mot_rms_norm_fp8";
  u15h_status st = check_width(ctx, what, dim, 16384);
  if (st == U15H_OK) { st = check_rows(ctx, what, M_und, M_gen); }
  if (st != U15H_OK) { return st; }
  if (!(eps >= 0.0f)) { return refuse(ctx, "%s: eps must be >= 0", what); }
  if ((delta == nullptr) != (x_out == nullptr)) {
    return refuse(ctx, "%s: delta and x_out go together", what);
  }
  const int rows = M_und + M_gen;
  if (rows == 0) { return u15h::end_call(ctx, hipSuccess, ""); }
  if (!usable(x) || !usable(q) || !usable(s) || !usable_or_null(delta) ||
      !usable_or_null(x_out) || !usable_or_null(y) || (M_und > 0 && !usable(w_und)) ||
      (M_gen > 0 && !usable(w_gen))) {
    return refuse(ctx, "%s: null or misaligned operand", what);
  }
  if (y != nullptr && y == x_out) {
    return refuse(ctx, "%s: y must not be x_out (which keeps the sum)", what);
  }
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  u15h::Fp8NormArgs a;
  a.x = x;
  a.d = delta;
  a.x_out = x_out;
  a.w_und = w_und;
  a.w_gen = w_gen;
  a.y = y;
  a.q = q;
  a.sc = s;
  a.m_und = M_und;
  a.rows = rows;
  a.dim = dim;
  a.eps = eps;
  return u15h::end_call(ctx, u15h::launch_fp8_norm(a, reinterpret_cast<hipStream_t>(stream)),
                        what);
}

u15h_status
u15h_mot_gemm_fp8(u15h_ctx* ctx, u15h_stream stream, const uint8_t* xq, const float* sx,
                  int M_und, int M_gen, int K, const u15h_mot_proj_fp8* proj, int nproj)
{
  if (ctx == nullptr) { return U15H_EINVAL; }
  const char* const what = "mot_gemm_fp8";
  u15h_status st = check_width(ctx, what, K, kMaxK);
  if (st == U15H_OK) { st = check_rows(ctx, what, M_und, M_gen); }
  if (st != U15H_OK) { return st; }
  if (proj == nullptr || nproj < 1 || nproj > U15H_MAX_PROJ) {
    return refuse(ctx, "%s: nproj=%d must be in [1, %d]", what, nproj, U15H_MAX_PROJ);
  }
  for (int i = 0; i < nproj; ++i) {
    if (proj[i].N <= 0 || proj[i].N % 8 != 0 || proj[i].N > kMaxN) {
      return refuse(ctx, "%s: proj[%d].N=%d must be a positive multiple of 8, at most %d", what,
                    i, proj[i].N, kMaxN);
    }
  }
  const int M = M_und + M_gen;
  if (M == 0) { return u15h::end_call(ctx, hipSuccess, ""); }
  if (!usable(xq) || !usable(sx)) { return refuse(ctx, "%s: xq/sx null or misaligned", what); }
  for (int i = 0; i < nproj; ++i) {
    const u15h_mot_proj_fp8& p = proj[i];
    if (!usable(p.y)) { return refuse(ctx, "%s: proj[%d].y null or misaligned", what, i); }
    if (M_und > 0 && (!usable(p.wq_und) || !usable(p.sw_und))) {
      return refuse(ctx, "%s: proj[%d] und weights/scales null or misaligned", what, i);
    }
    if (M_gen > 0 && (!usable(p.wq_gen) || !usable(p.sw_gen))) {
      return refuse(ctx, "%s: proj[%d] gen weights/scales null or misaligned", what, i);
    }
  }
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  Fp8Batch b;
  std::memset(&b, 0, sizeof b);
  b.K = K;
  b.sa_pitch = M;
  // the larger group first, as the int8 tier's batches have it
  for (int i = 0; i < nproj; ++i) {
    const u15h_mot_proj_fp8& p = proj[i];
    add_problem(b, xq + (size_t)M_und * K, sx + M_und, p.wq_gen, p.sw_gen,
                p.y + (size_t)M_und * p.N, M_gen, p.N);
  }
  for (int i = 0; i < nproj; ++i) {
    const u15h_mot_proj_fp8& p = proj[i];
    add_problem(b, xq, sx, p.wq_und, p.sw_und, p.y, M_und, p.N);
  }
  b.cus = u15h::gemm_cus(ctx);
  if (!plan(b, u15h::split_workspace_bytes(ctx))) { return refuse(ctx, "%s: too many tiles", what); }
  if (b.split > 1) {
    void* ws = nullptr;
    if ((st = u15h::split_workspace(ctx, &ws)) != U15H_OK) { return st; }
    b.ws = static_cast<float*>(ws);
  }
  return u15h::end_call(ctx, u15h::launch_fp8_gemm(b, reinterpret_cast<hipStream_t>(stream)),
                        what);
}

}  // extern "C"
