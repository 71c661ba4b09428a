// u15h_fp8.cc -- the fp8 tier's entry points (include/u15h.h): argument checks
// (nothing is launched on a refusal) and the batch tables of u15h_fp8.hip.
#include "u15h.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "u15h_internal.h"

namespace {

using u15h::Fp8Batch;
using u15h::Fp8Problem;

constexpr int kMaxK = 131072;
constexpr int kMaxRows = 1 << 24;
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

// A launch of the product: `narrow` bm rows and bn columns per workgroup with K
// split over its waves, else tiles of bm x bn, the last partial round in
// `split` shares of K.
struct Plan {
  bool narrow;
  int bm, bn, waves, split;
};

// Counts the tiles of a batch; false if they are too many.
bool
set_tiles(Fp8Batch& b, const Plan& p)
{
  b.narrow = p.narrow;
  b.bm = p.bm;
  b.bn = p.bn;
  b.waves = p.waves;
  long long tiles = 0;
  for (int i = 0; i < b.nprob; ++i) {
    Fp8Problem& q = b.p[i];
    q.tiles_m = (q.rows + p.bm - 1) / p.bm;
    q.tiles_n = (q.n + p.bn - 1) / p.bn;
    q.tile_begin = (int)tiles;
    tiles += (long long)q.tiles_m * q.tiles_n;
    if (tiles > (1 << 28)) { return false; }
  }
  b.total_tiles = b.split_begin = (int)tiles;
  b.split = 1;
  return true;
}

// Cuts the last partial round of a batch's tiles into up to `shares` shares of
// K each, as many as the workspace holds.
void
set_split(Fp8Batch& b, const Plan& p, int slots, size_t workspace)
{
  const int nb = (b.K + u15h::kFp8Block - 1) / u15h::kFp8Block;
  const int tail = b.total_tiles % slots;
  if (tail == 0) { return; }
  int S = std::min(p.split, nb);
  S = std::min(S, (int)std::min<size_t>(1 << 16, workspace / ((size_t)tail * p.bm * p.bn * 4)));
  if (S < 2) { return; }
  b.split = S;
  b.split_begin = b.total_tiles - tail;
}

// Workgroups of a plan that run at once.
int
slots_of(const Plan& p, int cus)
{
  return p.waves == 4 ? 2 * cus : cus;
}

Plan
choose(const Fp8Batch& b, int cus)
{
  int rows = 0, cols = 0;
  for (int i = 0; i < b.nprob; ++i) {
    rows = std::max(rows, b.p[i].rows);
    cols += (b.p[i].n + 15) / 16;
  }
  if (rows <= 64) {
    const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    const int fi = cols > 4 * cus && mt > 1 ? 2 : 1;
    return Plan{true, 16 * mt, 16 * fi, 4, 1};
  }
  const int nb = (b.K + u15h::kFp8Block - 1) / u15h::kFp8Block;
  // us per stage with every slot busy, and per round beside its stages
  const struct { int bm, bn, waves; double stage, round; } kinds[] = {
      {256, 256, 8, 1.60, 6.0}, {192, 256, 8, 1.25, 5.0}, {128, 256, 8, 0.90, 5.0},
      {128, 128, 4, 0.95, 5.0}, {64, 128, 4, 0.65, 5.0}};
  Plan best = {};
  double least = 0;
  for (const auto& k : kinds) {
    int tiles = 0;
    for (int i = 0; i < b.nprob; ++i) {
      tiles += ((b.p[i].rows + k.bm - 1) / k.bm) * ((b.p[i].n + k.bn - 1) / k.bn);
    }
    const int slots = k.waves == 4 ? 2 * cus : cus;
    const int full = tiles / slots, rem = tiles % slots;
    const int S = rem == 0 ? 1 : std::max(1, std::min(slots / rem, nb / 4));
    double us = full * (nb * k.stage + k.round);
    if (rem > 0) { us += (nb + S - 1) / S * k.stage + k.round; }
    if (S > 1) { us += 3.0 + 0.3e-6 * rem * S * k.bm * k.bn * 4; }
    if (least == 0 || us < least) {
      least = us;
      best = Plan{false, k.bm, k.bn, k.waves, S};
    }
  }
  return best;
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
  b.cus = u15h::num_cus(ctx);
  const Plan plan = choose(b, b.cus);
  if (!set_tiles(b, plan)) { return refuse(ctx, "%s: too many tiles", what); }
  if (!plan.narrow) { set_split(b, plan, slots_of(plan, b.cus), u15h::split_workspace_bytes(ctx)); }
  if (b.split > 1) {
    void* ws = nullptr;
    if ((st = u15h::split_workspace(ctx, &ws)) != U15H_OK) { return st; }
    b.ws = static_cast<float*>(ws);
  }
  return u15h::end_call(ctx, u15h::launch_fp8_gemm(b, reinterpret_cast<hipStream_t>(stream)),
                        what);
}

}  // extern "C"
