// u15h_paged.cc -- entry points for many requests at once (include/u15h.h):
// rotary positions, the paged K/V cache, attention behind a shared prefix.
// Argument checks (nothing is launched on a refusal) and the kernels' tables.
#include "u15h.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "u15h_internal.h"

namespace {

using u15h::PagedArgs;
using u15h::RopeArgs;

constexpr int kMaxHeads = 4096;
constexpr int kMaxTokens = 1 << 22;
constexpr int kMaxBatch = 1 << 16;
constexpr int kMaxKeys = 1 << 29;
constexpr long long kMaxStride = 1LL << 40;      // elements between rows or pages
constexpr long long kMaxGroups = 1LL << 23;      // workgroups of a launch: 2^31 threads
constexpr float kLeastScale = 1e-12f, kMostScale = 1e12f;
constexpr double kPi = 3.14159265358979323846;

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
aligned(const void* p, int bytes)
{
  return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0;
}

u15h_status
done(u15h_ctx* ctx)
{
  return u15h::set_error(ctx, U15H_OK, "");
}

// The parts of a rotation into `a`, ascending; the widest access that they
// allow into a.vec.
u15h_status
take_spec(u15h_ctx* ctx, const char* what, const u15h_rope_spec* r, const int32_t* pos, int tokens,
          int head_dim, RopeArgs& a)
{
  if (r->nparts < 1 || r->nparts > U15H_MAX_ROPE_PARTS) {
    return refuse(ctx, "%s: %d parts (1 to %d)", what, r->nparts, U15H_MAX_ROPE_PARTS);
  }
  if (pos == nullptr) { return refuse(ctx, "%s: no positions", what); }
  if (!aligned(pos, 4)) { return refuse(ctx, "%s: positions must be 4-byte aligned", what); }
  if (!(std::fabs(r->scale) < INFINITY)) {
    return refuse(ctx, "%s: scale %g is not finite", what, (double)r->scale);
  }
  int order[U15H_MAX_ROPE_PARTS] = {0, 1, 2};
  std::sort(order, order + r->nparts,
            [&](int i, int j) { return r->part[i].start < r->part[j].start; });
  a.nparts = r->nparts;
  a.neighbours = r->neighbours != 0;
  a.scale = r->scale;
  a.pairs = 0;
  int end = 0;
  for (int i = 0; i < r->nparts; ++i) {
    const u15h_rope_part& p = r->part[order[i]];
    if (p.width <= 0 || p.width % 2 != 0 || p.start < end || p.width > head_dim ||
        p.start > head_dim - p.width) {
      return refuse(ctx, "%s: part [%d, %d + %d) of a head of %d (even widths, no overlap)", what,
                    p.start, p.start, p.width, head_dim);
    }
    if (p.axis < 0 || p.axis >= U15H_MAX_ROPE_PARTS) {
      return refuse(ctx, "%s: axis %d (0 to %d)", what, p.axis, U15H_MAX_ROPE_PARTS - 1);
    }
    if (p.freq == nullptr || !aligned(p.freq, 8)) {
      return refuse(ctx, "%s: frequencies must be given, 8-byte aligned", what);
    }
    a.part[i] = {p.freq, pos + (long long)p.axis * tokens, p.start, p.width, a.pairs};
    a.pairs += p.width / 2;
    end = p.start + p.width;
    const int run = a.neighbours ? p.width : p.width / 2;
    while (a.vec > 1 && (p.start % a.vec != 0 || run % a.vec != 0)) {
      a.vec = a.vec == 8 ? 2 : 1;
    }
  }
  return U15H_OK;
}

void
narrow(RopeArgs& a, const void* p, long long s0, long long s1)
{
  while (a.vec > 1 && (!aligned(p, a.vec * 2) || s0 % a.vec != 0 || s1 % a.vec != 0)) {
    a.vec = a.vec == 8 ? 2 : 1;
  }
}

u15h_status
check_cache(u15h_ctx* ctx, const char* what, const u15h_paged_kv* kv, long long* page_stride,
            int* page_log2)
{
  if (kv == nullptr) { return refuse(ctx, "%s: no cache", what); }
  if (kv->head_dim != 32 && kv->head_dim != 64 && kv->head_dim != 128) {
    return refuse(ctx, "%s: head_dim %d (32, 64 or 128)", what, kv->head_dim);
  }
  if (kv->page < 16 || kv->page > (1 << 20) || (kv->page & (kv->page - 1)) != 0) {
    return refuse(ctx, "%s: page %d (a power of two, 16 to 2^20)", what, kv->page);
  }
  if (kv->kv_heads <= 0 || kv->kv_heads > kMaxHeads || kv->pages < 0 ||
      (long long)kv->pages * kv->page >= (1LL << 31)) {
    return refuse(ctx, "%s: kv_heads=%d pages=%d page=%d", what, kv->kv_heads, kv->pages,
                  kv->page);
  }
  const long long whole = (long long)kv->kv_heads * kv->page * kv->head_dim;
  *page_stride = kv->page_stride == 0 ? whole : kv->page_stride;
  if (*page_stride < whole || *page_stride % 8 != 0 ||
      *page_stride > kMaxStride / std::max(kv->pages, 1)) {
    return refuse(ctx, "%s: page_stride %lld (at least %lld, a multiple of 8; at most 2^40 "
                  "elements over all pages)", what, (long long)kv->page_stride, whole);
  }
  if (kv->pages > 0 && (kv->k == nullptr || kv->v == nullptr)) {
    return refuse(ctx, "%s: null cache", what);
  }
  if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) {
    return refuse(ctx, "%s: the cache must be 16-byte aligned", what);
  }
  *page_log2 = __builtin_ctz((unsigned)kv->page);
  return U15H_OK;
}

// Rows of `width` elements, `stride` apart.
u15h_status
check_rows(u15h_ctx* ctx, const char* what, const char* name, const void* p, int64_t stride,
           long long width)
{
  if (p == nullptr) { return refuse(ctx, "%s: %s is null", what, name); }
  if (!aligned(p, 16)) { return refuse(ctx, "%s: %s must be 16-byte aligned", what, name); }
  if (stride < width || stride % 8 != 0 || stride > kMaxStride) {
    return refuse(ctx, "%s: %s's rows are %lld apart (at least %lld, a multiple of 8)", what,
                  name, (long long)stride, width);
  }
  return U15H_OK;
}

int
round_up(long long v, int to)
{
  return (int)((v + to - 1) / to * to);
}

// `keys` in at most `n` shares of a multiple of 128.
void
cut(long long keys, long long n, int* shares, int* chunk)
{
  *chunk = std::max(round_up((keys + n - 1) / n, 128), 128);
  *shares = (int)std::max((keys + *chunk - 1) / *chunk, 1LL);
}

// How a call is cut (PagedArgs): what the prefix's workgroups and the
// sequences' walk.  Lengths are known to their bounds only; own keys are taken
// as half of max_kv on the mean, and a share's keys are fixed here.  So a bound
// far above the lengths leaves few shares with keys: one request of 4000 keys
// takes 10.9 us where max_kv is 4000, 13.7 at 16384 and 42 at 131072, four of them
// 18, 25 and 78, 32 of 1 to 4000 keys 51, 113 and 113.  The figures below have
// max_kv at the longest sequence.  In a graph, 32 query heads over 8 of 128 unless
// said, us:
//  - the prefix once for all / by every sequence: 4 queries behind 8192 keys 13.2
//    / 19.7, 128 behind 500 25 / 35, 20 of 8 queries behind 4000 30 / 44; below
//    4096 keys walked again, 8 behind 256 11.1 / 8.0, 2 behind 600 11.0 / 11.1;
//  - shares of it that make 256 tile workgroups / 512: 128 queries behind 16384
//    keys 58 / 75, 200 behind 8192 65 / 77, 256 behind 32768 189 / 194 (384: 181);
//  - its rows on tiles / streaming: 256 rows behind 4224 keys 36 / 45, 640 rows
//    (heads of 64) behind 8192 18 / 28; 64 rows and fewer stream;
//  - a sequence of 100 queries whose 400 rows walk 3000 keys in shares / whole 39
//    / 47 (five of them), of 300 over 5000 keys 48 / 101;
//  - parts added by the last share / by a second kernel: 1800 keys of one request
//    9.5 / 11.4, three of 20000 to 40000 81 / 79.
void
plan(PagedArgs& a, int cus, void* ws, size_t bytes)
{
  const int G = a.hq / a.hkv;
  const long long rows1 = (long long)a.max_q * G;       // of a sequence, at most
  const long long rows = (long long)a.tokens * G;       // of a kv head
  a.longs = rows1 > u15h::kPagedShortRows;
  a.shorts = G <= u15h::kPagedShortRows;
  a.ws = static_cast<float*>(ws);
  a.nr = rows1 <= 16 || !a.shorts ? 1 : 2;
  const long long pieces = ws == nullptr ? 1 : 64;      // most shares of anything

  // us: a 64-key tile of one workgroup, the streaming of own keys, a part's
  // round trip (and 0.15 for its place in the sum; 32 parts are one pass)
  const double tile = a.d == 128 ? 0.94 : a.d == 64 ? 0.63 : 0.52;
  const double own = (double)a.batch * a.max_kv * 0.5 * a.hkv * a.d * 4 / 5e6;
  const double part = (double)a.tokens * a.hq * (a.d + 2) * 8 / 4e6;

  // The prefix for all rows at once: where at least 4096 keys would be walked
  // again and sequences are short.
  bool phase = ws != nullptr && a.batch >= 2 && a.prefix >= 256 &&
               (long long)a.batch * a.prefix >= 4096 && rows / a.batch <= 256;
  for (;; phase = false) {
    a.p_shares = 0;
    if (phase) {
      a.p_tile = rows > u15h::kPagedShortRows;
      if (!a.p_tile && rows > 16) { a.nr = 2; }
      const int rb = a.p_tile ? 128 : 16 * a.nr;
      const long long blocks = (rows + rb - 1) / rb * a.hkv;
      double best = 1e30;
      for (int n = 1; n <= std::min(pieces, 30LL); ++n) {
        int shares, chunk;
        cut(a.prefix, n, &shares, &chunk);
        const double items = (double)blocks * shares;
        double us;
        if (a.p_tile) {
          // A tile workgroup to a CU: the sequences' workgroups run beside it, and
          // a tile takes half as long again.  Two to a CU: those wait, and a pair
          // of tiles takes twice as long.
          const double walk = chunk / 64.0 * tile;
          const double beside = std::max(own, 1.5 * walk + 5.0);
          const double after = std::max(items / cus, 2.0) * walk + own + 5.0;
          const double full = std::min(std::max((items - cus) / cus, 0.0), 1.0);
          us = (1.0 - full) * beside + full * after + (items > cus ? 4.0 : 0.0);
        } else {
          const double walk = chunk / 128.0 * 1.2;
          us = std::max(own, std::max(walk, items / (2 * cus) * walk) + 5.0);
        }
        us += (part + 0.15) * shares;
        if (us < best) {
          best = us;
          a.p_shares = shares;
          a.p_chunk = chunk;
        }
      }
    }
    // What a sequence walks itself, in shares of 256 keys or more (128 in a
    // small call): the walk of the longest against all workgroups' work, which
    // hides it; a tail of uneven lengths; and what shares cost.  128 keys take a
    // streaming workgroup 1 us, 2 or more once the memory is at its rate.
    const long long before = a.p_shares > 0 ? 0 : round_up(a.prefix, 64);
    const long long keys = before + a.max_kv, mean = before + a.max_kv / 2;
    const int rb = 16 * a.nr;
    const long long s_items = (std::min<long long>(rows1, u15h::kPagedShortRows) + rb - 1) / rb *
                              a.hkv * a.batch;
    const long long t_items = (rows / 128 + a.batch) * a.hkv;
    const double work = a.longs ? (double)t_items * mean / 64 * tile / cus
                                : (double)a.batch * mean * a.hkv * a.d * 4 / 5e6;
    const long long most = std::max(1LL, std::min(keys / (work < 10.0 ? 128 : 256), pieces));
    auto shares_of = [&](double walk, long long most, int* shares, int* chunk) {
      double best = 1e30;
      int pick = 1;
      for (int n = 1; n <= most; ++n) {
        const double us = std::max(work, walk / n) + 0.3 * walk / n + n * part +
                          (n > 1 && a.p_shares == 0 ? 3.0 : 0.0);
        if (us < best) {
          best = us;
          pick = n;
        }
      }
      cut(keys, pick, shares, chunk);
    };
    // at most one streaming workgroup a CU for a sequence by itself (which
    // fills the memory's rate), four for several
    const long long s_most = (a.batch == 1 ? 1LL : 4LL) * cus / s_items;
    shares_of(keys / 128.0 * (work < 10.0 ? 1.0 : 2.0), std::min(most, s_most), &a.s_shares,
              &a.s_chunk);
    shares_of(keys / 64.0 * tile, std::min(most, 4LL * cus / t_items), &a.t_shares, &a.t_chunk);
    while (u15h::paged_ws_bytes(a) > bytes && a.s_shares + a.t_shares > 2) {
      cut(keys, std::max(a.s_shares - 1, 1), &a.s_shares, &a.s_chunk);
      cut(keys, std::max(a.t_shares - 1, 1), &a.t_shares, &a.t_chunk);
    }
    while (u15h::paged_ws_bytes(a) > bytes && a.p_shares > 1) {
      cut(a.prefix, a.p_shares - 1, &a.p_shares, &a.p_chunk);
    }
    if (!phase || u15h::paged_ws_bytes(a) <= bytes) { break; }
  }
  // Small calls of sequences by themselves are added by their own workgroups.
  const int rb = 16 * a.nr;
  const long long joins =
      (std::min<long long>(rows1, u15h::kPagedShortRows) + rb - 1) / rb * a.hkv * a.batch;
  const double walked = (double)a.batch * (a.prefix + a.max_kv / 2) * a.hkv * a.d * 4 / 5e6;
  a.joins = a.p_shares == 0 && !a.longs && a.s_shares > 1 && joins <= u15h::kPagedJoins &&
                    walked < 30.0
                ? reinterpret_cast<int*>(static_cast<char*>(ws) + bytes)
                : nullptr;
}

}  // namespace

extern "C" {

u15h_status
u15h_rope_freqs(int width, double theta, int scaling, double factor, double trained, double slow,
                double fast, double* freq, float* scale)
{
  const bool by_turns = scaling == U15H_ROPE_YARN || scaling == U15H_ROPE_BANDS;
  if (freq == nullptr || scale == nullptr || width <= 0 || width % 2 != 0 ||
      width > u15h::kRopeMaxHeadDim || !(theta > 1.0) || !(theta < INFINITY) ||
      scaling < U15H_ROPE_PLAIN || scaling > U15H_ROPE_BANDS) {
    return U15H_EINVAL;
  }
  if (scaling != U15H_ROPE_PLAIN && (!(factor >= 1.0) || !(factor < INFINITY))) {
    return U15H_EINVAL;
  }
  if (by_turns && (!(trained > 0.0) || !(trained < INFINITY) || !(slow > 0.0) ||
                   !(fast > slow) || !(fast < INFINITY))) {
    return U15H_EINVAL;
  }
  double base = theta;
  if (scaling == U15H_ROPE_NTK && width > 2) {
    base = theta * std::pow(factor, width / (width - 2.0));
  }
  // the pair, as a real number, that turns `turns` times within `trained`
  auto pair_of = [&](double turns) {
    return width * std::log(trained / (turns * 2.0 * kPi)) / (2.0 * std::log(theta));
  };
  double lo = 0.0, hi = 0.0;
  if (scaling == U15H_ROPE_YARN) {
    lo = std::max(std::floor(pair_of(fast)), 0.0);
    hi = std::min(std::ceil(pair_of(slow)), width - 1.0);
  }
  for (int i = 0; i < width / 2; ++i) {
    double f = std::pow(base, -2.0 * i / width);
    if (scaling == U15H_ROPE_LINEAR) { f /= factor; }
    if (by_turns) {
      // the share of the frequency that is kept as it is
      double keep;
      if (scaling == U15H_ROPE_YARN) {
        keep = 1.0 - std::min(std::max((i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
      } else {
        keep = (trained * f / (2.0 * kPi) - slow) / (fast - slow);
        keep = std::min(std::max(keep, 0.0), 1.0);
      }
      f = keep * f + (1.0 - keep) * f / factor;
    }
    freq[i] = f;
  }
  *scale = scaling == U15H_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  return U15H_OK;
}

u15h_status
u15h_rope(u15h_ctx* ctx, u15h_stream stream, const u15h_rope_spec* rope, const int32_t* pos,
          const u15h_bf16* x, int64_t x_tok, int64_t x_head, u15h_bf16* y, int64_t y_tok,
          int64_t y_head, int tokens, int heads, int head_dim, int inverse)
{
  const char* what = "rope";
  if (ctx == nullptr) { return U15H_EINVAL; }
  if (tokens < 0 || tokens > kMaxTokens || heads <= 0 || heads > kMaxHeads || head_dim <= 0 ||
      head_dim > u15h::kRopeMaxHeadDim) {
    return refuse(ctx, "%s: tokens=%d heads=%d head_dim=%d", what, tokens, heads, head_dim);
  }
  if (rope == nullptr) { return refuse(ctx, "%s: no rotation", what); }
  if (tokens == 0) { return done(ctx); }
  RopeArgs a = {};
  a.vec = head_dim % 8 == 0 ? 8 : head_dim % 2 == 0 ? 2 : 1;
  u15h_status st = take_spec(ctx, what, rope, pos, tokens, head_dim, a);
  if (st != U15H_OK) { return st; }
  if (x == nullptr || y == nullptr) { return refuse(ctx, "%s: null operand", what); }
  if (!aligned(x, 2) || !aligned(y, 2)) {
    return refuse(ctx, "%s: operands must be 2-byte aligned", what);
  }
  for (const int64_t v : {x_tok, x_head, y_tok, y_head}) {
    if (v < 0 || v > kMaxStride) {
      return refuse(ctx, "%s: stride %lld", what, (long long)v);
    }
  }
  // heads and tokens of y must not overlap: one of the two strides spans a
  // head, the other all of the first's heads (or tokens)
  {
    const bool by_head = y_head <= y_tok;
    const int64_t inner = by_head ? y_head : y_tok, outer = by_head ? y_tok : y_head;
    const int n_in = by_head ? heads : tokens, n_out = by_head ? tokens : heads;
    if ((n_in > 1 && inner < head_dim) ||
        (n_out > 1 && outer < (n_in - 1) * inner + head_dim)) {
      return refuse(ctx, "%s: heads of y overlap (strides %lld, %lld)", what, (long long)y_tok,
                    (long long)y_head);
    }
  }
  if (x == y && (x_tok != y_tok || x_head != y_head)) {
    return refuse(ctx, "%s: y over x needs equal strides", what);
  }
  narrow(a, x, x_tok, x_head);
  narrow(a, y, y_tok, y_head);
  a.q = {x, y, x_tok, x_head, y_tok, y_head, heads};
  a.sign = inverse ? -1.0f : 1.0f;
  a.tokens = tokens;
  a.d = head_dim;
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  return u15h::end_call(ctx, u15h::launch_rope(a, reinterpret_cast<hipStream_t>(stream)), what);
}

u15h_status
u15h_paged_append(u15h_ctx* ctx, u15h_stream stream, const u15h_paged_kv* kv, const int32_t* slot,
                  const u15h_rope_spec* rope, const int32_t* pos, const u15h_bf16* k,
                  int64_t k_stride, const u15h_bf16* v, int64_t v_stride, const u15h_bf16* q,
                  int64_t q_stride, u15h_bf16* q_out, int64_t q_out_stride, int hq, int tokens)
{
  const char* what = "paged_append";
  if (ctx == nullptr) { return U15H_EINVAL; }
  RopeArgs a = {};
  u15h_status st = check_cache(ctx, what, kv, &a.page_stride, &a.page_log2);
  if (st != U15H_OK) { return st; }
  if (tokens < 0 || tokens > kMaxTokens) {
    return refuse(ctx, "%s: tokens=%d (at most %d)", what, tokens, kMaxTokens);
  }
  if ((q == nullptr) != (q_out == nullptr) || (q != nullptr && rope == nullptr)) {
    return refuse(ctx, "%s: q and q_out come together, with a rotation", what);
  }
  if (q != nullptr && (hq <= 0 || hq > kMaxHeads)) { return refuse(ctx, "%s: hq=%d", what, hq); }
  if (tokens == 0) { return done(ctx); }
  if (slot == nullptr || !aligned(slot, 4)) {
    return refuse(ctx, "%s: slots must be given, 4-byte aligned", what);
  }
  const int d = kv->head_dim;
  const long long width = (long long)kv->kv_heads * d;
  if ((st = check_rows(ctx, what, "k", k, k_stride, width)) != U15H_OK ||
      (st = check_rows(ctx, what, "v", v, v_stride, width)) != U15H_OK) {
    return st;
  }
  a.vec = 8;
  if (rope != nullptr &&
      (st = take_spec(ctx, what, rope, pos, tokens, d, a)) != U15H_OK) {
    return st;
  }
  if (q != nullptr) {
    if ((st = check_rows(ctx, what, "q", q, q_stride, (long long)hq * d)) != U15H_OK ||
        (st = check_rows(ctx, what, "q_out", q_out, q_out_stride, (long long)hq * d)) !=
            U15H_OK) {
      return st;
    }
    if (q == q_out && q_stride != q_out_stride) {
      return refuse(ctx, "%s: q_out over q needs equal strides", what);
    }
    a.q = {q, q_out, q_stride, d, q_out_stride, d, hq};
  }
  a.k = {k, kv->k, k_stride, d, 0, 0, kv->kv_heads};
  a.v = {v, kv->v, v_stride, d, 0, 0, kv->kv_heads};
  a.sign = 1.0f;
  a.tokens = tokens;
  a.d = d;
  a.slot = slot;
  a.slots = kv->pages * kv->page;
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  return u15h::end_call(ctx, u15h::launch_rope(a, reinterpret_cast<hipStream_t>(stream)), what);
}

u15h_status
u15h_paged_attention(u15h_ctx* ctx, u15h_stream stream, const u15h_paged_kv* kv,
                     const u15h_paged_batch* bt, const u15h_bf16* q, int64_t q_stride,
                     u15h_bf16* out, int64_t out_stride, int hq, float scale, int causal)
{
  const char* what = "paged_attention";
  if (ctx == nullptr) { return U15H_EINVAL; }
  PagedArgs a = {};
  u15h_status st = check_cache(ctx, what, kv, &a.page_stride, &a.page_log2);
  if (st != U15H_OK) { return st; }
  if (bt == nullptr) { return refuse(ctx, "%s: no batch", what); }
  if (hq <= 0 || hq > kMaxHeads || hq % kv->kv_heads != 0) {
    return refuse(ctx, "%s: hq=%d over %d kv heads", what, hq, kv->kv_heads);
  }
  if (bt->batch < 0 || bt->batch > kMaxBatch || bt->tokens < 0 || bt->tokens > kMaxTokens ||
      bt->max_q < 0 || bt->max_kv < 0 || bt->max_kv >= kMaxKeys || bt->prefix_len < 0 ||
      bt->prefix_len >= kMaxKeys || bt->table_stride < 0) {
    return refuse(ctx, "%s: batch=%d tokens=%d max_q=%d max_kv=%d prefix_len=%d table_stride=%d",
                  what, bt->batch, bt->tokens, bt->max_q, bt->max_kv, bt->prefix_len,
                  bt->table_stride);
  }
  if (scale != 0.0f && !(scale >= kLeastScale && scale <= kMostScale)) {
    return refuse(ctx, "%s: scale %g (0 for 1/sqrt(head_dim), or %g to %g)", what, (double)scale,
                  (double)kLeastScale, (double)kMostScale);
  }
  if (bt->batch == 0 || bt->tokens == 0 || bt->max_q == 0) { return done(ctx); }
  if (bt->q_start == nullptr && bt->tokens < bt->batch) {
    return refuse(ctx, "%s: %d rows for %d sequences of one", what, bt->tokens, bt->batch);
  }
  if (bt->kv_len == nullptr || (bt->max_kv > 0 && bt->table_stride > 0 && bt->table == nullptr) ||
      (bt->prefix_len > 0 && bt->prefix_table == nullptr)) {
    return refuse(ctx, "%s: kv_len, table and prefix_table must be given", what);
  }
  for (const int32_t* p : {bt->q_start, bt->kv_len, bt->table, bt->prefix_table}) {
    if (!aligned(p, 4)) { return refuse(ctx, "%s: tables must be 4-byte aligned", what); }
  }
  // rows are counted in 32 bits; a sequence counts as 5 workgroups a kv head (at
  // most 2 streaming ones and a tile one that its rows do not fill are launched;
  // shares are planned only while they are few), its rows as whole tiles
  const long long groups =
      ((long long)bt->batch * 5 + (long long)bt->tokens * (hq / kv->kv_heads) / 128) *
      kv->kv_heads;
  if ((long long)bt->tokens * hq >= (1LL << 31) || groups > kMaxGroups) {
    return refuse(ctx, "%s: %d sequences, %d rows of %d heads: too many", what, bt->batch,
                  bt->tokens, hq);
  }
  const long long width = (long long)hq * kv->head_dim;
  if ((st = check_rows(ctx, what, "q", q, q_stride, width)) != U15H_OK ||
      (st = check_rows(ctx, what, "out", out, out_stride, width)) != U15H_OK) {
    return st;
  }
  a.q = q;
  a.out = out;
  a.q_tok = q_stride;
  a.o_tok = out_stride;
  a.k = kv->k;
  a.v = kv->v;
  a.pages = kv->pages;
  a.hkv = kv->kv_heads;
  a.d = kv->head_dim;
  a.hq = hq;
  a.q_start = bt->q_start;
  a.kv_len = bt->kv_len;
  a.table = bt->table;
  a.prefix_table = bt->prefix_table;
  a.table_stride = bt->max_kv > 0 ? bt->table_stride : 0;
  a.prefix = bt->prefix_len;
  a.batch = bt->batch;
  a.tokens = bt->tokens;
  a.max_q = std::min(bt->q_start == nullptr ? 1 : bt->max_q, bt->tokens);
  a.max_kv = bt->max_kv;
  a.causal = causal != 0;
  a.scale = (scale > 0.0f ? scale : 1.0f / std::sqrt((float)kv->head_dim)) * 1.4426950408889634f;
  size_t bytes = 0;
  void* ws = u15h::attention_scratch(ctx, &bytes);
  plan(a, u15h::compute_units(ctx), ws, bytes);
  if ((st = u15h::begin_call(ctx)) != U15H_OK) { return st; }
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a.joins != nullptr && !*u15h::joins_cleared(ctx)) {
    // The context's first call that counts.  A captured clear runs when its graph
    // does, so it says nothing about the next call's counters.
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    hipError_t e = hipStreamIsCapturing(s, &capture);
    if (e == hipSuccess) { e = u15h::launch_clear_joins(a.joins, s); }
    if (e != hipSuccess) { return u15h::end_call(ctx, e, what); }
    *u15h::joins_cleared(ctx) = capture == hipStreamCaptureStatusNone;
  }
  return u15h::end_call(ctx, u15h::launch_paged_attention(a, s), what);
}

}  // extern "C"
