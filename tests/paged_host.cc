// paged_host.cc -- the checks and plans of u15h_paged.cc on the host, for
// test_paged_host.py.
//
// The entry points' own source, with the context and the kernel launchers
// replaced by the ones below, which print what they are asked for.  Reads one
// call per line from stdin, `name key=value ..`, on operands that are never
// read; a key that is not given has the value of a call that is allowed.
// Prints its launch (or "-"), " ; " and the status: "ok" or the error.  The
// arguments: compute units, bytes of scratch.
#include "u15h_paged.cc"

#include <iostream>
#include <map>
#include <sstream>
#include <string>

struct u15h_ctx {
  std::string error;
  bool cleared = false;
};

namespace {

std::string g_out;
int g_cus = 256;
size_t g_bytes = 0;
bool g_capturing = false;

}  // namespace

hipError_t
hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* status)
{
  *status = g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}

namespace u15h {

u15h_status begin_call(u15h_ctx*) { return U15H_OK; }

u15h_status
end_call(u15h_ctx* ctx, hipError_t e, const char* what)
{
  return e == hipSuccess ? U15H_OK : set_error(ctx, U15H_ELAUNCH, what);
}

void*
attention_scratch(const u15h_ctx*, size_t* bytes)
{
  *bytes = g_bytes;
  return g_bytes > 0 ? reinterpret_cast<void*>(4096) : nullptr;
}

int compute_units(const u15h_ctx*) { return g_cus; }

bool* joins_cleared(u15h_ctx* ctx) { return &ctx->cleared; }

hipError_t
launch_clear_joins(int* joins, hipStream_t)
{
  g_out += joins == reinterpret_cast<int*>(4096 + g_bytes) ? "clear " : "clear elsewhere ";
  return hipSuccess;
}

u15h_status
set_error(u15h_ctx* ctx, u15h_status st, const char* msg)
{
  ctx->error = msg;
  return st;
}

hipError_t
launch_rope(const RopeArgs& a, hipStream_t)
{
  std::ostringstream s;
  s << "rope vec=" << a.vec << " pairs=" << a.pairs << " heads=" << a.q.heads << "+" << a.k.heads
    << "+" << a.v.heads << " sign=" << a.sign << " slots=" << a.slots << " parts";
  for (int p = 0; p < a.nparts; ++p) {
    s << " " << a.part[p].start << ":" << a.part[p].width << ":" << a.part[p].pair << ":"
      << (reinterpret_cast<uintptr_t>(a.part[p].pos) - 4096) / 4;
  }
  g_out += s.str();
  return hipSuccess;
}

hipError_t
launch_paged_attention(const PagedArgs& a, hipStream_t)
{
  // the scratch holds the parts, chunks cover what they cut, and a call that
  // joins in its own workgroups has no parts of another kind
  const long long keys = (a.p_shares > 0 ? 0 : a.prefix) + (long long)a.max_kv;
  if (paged_ws_bytes(a) > g_bytes || (paged_parts(a) > 1 && a.ws == nullptr) ||
      (a.p_shares > 0 && (long long)a.p_shares * a.p_chunk < a.prefix) ||
      (long long)a.s_shares * a.s_chunk < keys || (long long)a.t_shares * a.t_chunk < keys ||
      a.s_chunk % 128 != 0 || a.t_chunk % 128 != 0 || a.p_chunk % 128 != 0 ||
      (a.joins != nullptr && (a.p_shares > 0 || a.longs || a.s_shares < 2))) {
    return hipErrorInvalidValue;
  }
  std::ostringstream s;
  s << "attn parts=" << paged_parts(a) << " p=" << a.p_shares << "x" << a.p_chunk << " "
    << (a.p_shares == 0 ? "none" : a.p_tile ? "tile" : "stream") << " s=" << a.shorts << ":"
    << a.s_shares << "x" << a.s_chunk << " t=" << a.longs << ":" << a.t_shares << "x" << a.t_chunk
    << " nr=" << a.nr << " joins=" << (a.joins != nullptr) << " max_q=" << a.max_q << " scale=" << a.scale << " stride="
    << a.table_stride;
  g_out += s.str();
  return hipSuccess;
}

}  // namespace u15h

int
main(int argc, char** argv)
{
  if (argc > 1) { g_cus = std::stoi(argv[1]); }
  if (argc > 2) { g_bytes = std::stoull(argv[2]); }
  u15h_ctx ctx;
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    std::string name, word;
    in >> name;
    std::map<std::string, double> given;
    while (in >> word) {
      const size_t eq = word.find('=');
      given[word.substr(0, eq)] = std::stod(word.substr(eq + 1));
    }
    auto v = [&](const char* key, double other) {
      return given.count(key) ? given[key] : other;
    };
    auto n = [&](const char* key, double other) { return (int)v(key, other); };
    // an operand's address
    auto p = [&](const char* key) {
      return reinterpret_cast<void*>((uintptr_t)(long long)v(key, 4096));
    };
    g_out.clear();
    ctx.error.clear();
    g_capturing = n("capturing", 0) != 0;
    u15h_status st = U15H_OK;
    const int d = n("d", 128), heads = n("heads", 8);
    u15h_rope_spec r = {};
    r.nparts = n("nparts", 1);
    r.neighbours = n("neighbours", 0);
    r.scale = (float)v("rscale", 1.0);
    for (int i = 0; i < U15H_MAX_ROPE_PARTS; ++i) {
      const std::string k = std::to_string(i);
      r.part[i] = {static_cast<const double*>(p(("freq" + k).c_str())),
                   n(("start" + k).c_str(), 0), n(("width" + k).c_str(), i == 0 ? d : 0),
                   n(("axis" + k).c_str(), 0)};
    }
    u15h_paged_kv kv = {static_cast<u15h_bf16*>(p("kp")), static_cast<u15h_bf16*>(p("vp")),
                        (int64_t)v("page_stride", 0), n("pages", 100), n("page", 16), heads, d};
    u15h_ctx* c = n("ctx", 1) ? &ctx : nullptr;
    if (name == "rope") {
      st = u15h_rope(c, nullptr, n("spec", 1) ? &r : nullptr, static_cast<int32_t*>(p("pos")),
                     static_cast<u15h_bf16*>(p("x")), (int64_t)v("x_tok", heads * d),
                     (int64_t)v("x_head", d), static_cast<u15h_bf16*>(p("y")),
                     (int64_t)v("y_tok", heads * d), (int64_t)v("y_head", d), n("tokens", 5),
                     heads, d, n("inverse", 0));
    } else if (name == "append") {
      const int hq = n("hq", 32);
      st = u15h_paged_append(
          c, nullptr, n("kv", 1) ? &kv : nullptr, static_cast<int32_t*>(p("slot")),
          n("spec", 1) ? &r : nullptr, static_cast<int32_t*>(p("pos")),
          static_cast<u15h_bf16*>(p("k")), (int64_t)v("k_stride", heads * d),
          static_cast<u15h_bf16*>(p("v")), (int64_t)v("v_stride", heads * d),
          static_cast<u15h_bf16*>(p("q")), (int64_t)v("q_stride", hq * d),
          static_cast<u15h_bf16*>(p("q_out")), (int64_t)v("q_out_stride", hq * d), hq,
          n("tokens", 5));
    } else if (name == "attn") {
      const int hq = n("hq", 32), batch = n("batch", 3);
      u15h_paged_batch b = {batch, n("tokens", batch), n("max_q", 1), n("max_kv", 100),
                            static_cast<int32_t*>(p("q_start")),
                            static_cast<int32_t*>(p("kv_len")),
                            static_cast<int32_t*>(p("table")), n("table_stride", 7),
                            static_cast<int32_t*>(p("prefix_table")), n("prefix_len", 0)};
      st = u15h_paged_attention(c, nullptr, n("kv", 1) ? &kv : nullptr, n("batches", 1) ? &b : nullptr,
                                static_cast<u15h_bf16*>(p("q")), (int64_t)v("q_stride", hq * d),
                                static_cast<u15h_bf16*>(p("out")),
                                (int64_t)v("out_stride", hq * d), hq, (float)v("scale", 0),
                                n("causal", 1));
    }
    std::cout << (g_out.empty() ? "-" : g_out) << " ; "
              << (st == U15H_OK ? "ok" : ctx.error.empty() ? "refused" : ctx.error) << "\n";
  }
  return 0;
}
