// fp8_host.cc -- the checks and plans of u15h_fp8.cc on the host, for
// test_fp8_host.py.
//
// The entry points' own source, with the context and the kernel launchers
// replaced by the ones below, which print what they are asked for.  Reads one
// call per line from stdin, on operands that are aligned and never read:
//   gemm M_und M_gen K N..            | norm M_und M_gen dim delta x_out y
//   rows rows K | swiglu rows inter h | blocks N K
//   bad WHICH                         (a call with one wrong operand)
// and prints its launch (or "-"), " ; " and the status: "ok" or the error.  A
// batch that the kernels would refuse, or whose shares do not fit the
// workspace, is answered with hipErrorInvalidValue.  The first argument is the
// number of compute units.
#include "u15h_fp8.cc"

#include <iostream>
#include <sstream>
#include <string>
#include <vector>

struct u15h_ctx {
  int cus = 256;
  std::string error;
};

namespace {

std::string g_out;
size_t g_capacity = 0;

template <class T>
T*
fake(uintptr_t at = 4096)
{
  return reinterpret_cast<T*>(at);
}

hipError_t
emit(const std::string& s)
{
  g_out += s;
  return hipSuccess;
}

}  // namespace

namespace u15h {

u15h_status begin_call(u15h_ctx*) { return U15H_OK; }

u15h_status
end_call(u15h_ctx* ctx, hipError_t e, const char* what)
{
  return e == hipSuccess ? U15H_OK : set_error(ctx, U15H_ELAUNCH, what);
}

int gemm_cus(const u15h_ctx* ctx) { return ctx->cus; }

u15h_status
split_workspace(u15h_ctx*, void** ws)
{
  *ws = fake<void>();
  return U15H_OK;
}

size_t split_workspace_bytes(const u15h_ctx*) { return g_capacity; }

u15h_status
set_error(u15h_ctx* ctx, u15h_status st, const char* msg)
{
  ctx->error = msg;
  return st;
}

hipError_t
launch_fp8_gemm(const Fp8Batch& b, hipStream_t)
{
  long long tiles = 0;
  for (int i = 0; i < b.nprob; ++i) {
    const Fp8Problem& p = b.p[i];
    if (p.tile_begin != tiles || p.tiles_m != (p.rows + b.bm - 1) / b.bm ||
        p.tiles_n != (p.n + b.bn - 1) / b.bn || (b.narrow && p.tiles_m != 1)) {
      return hipErrorInvalidValue;
    }
    tiles += (long long)p.tiles_m * p.tiles_n;
  }
  const int tail = b.total_tiles - b.split_begin, nb = (b.K + kFp8Block - 1) / kFp8Block;
  if (tiles != b.total_tiles || tail < 0 || (tail == 0) != (b.split == 1) ||
      (tail > 0 && (b.narrow || b.split < 2 || b.split > nb || b.ws == nullptr)) ||
      (tail > 0 && (size_t)tail * b.split * b.bm * b.bn * 4 > g_capacity)) {
    return hipErrorInvalidValue;
  }
  std::ostringstream s;
  s << (b.narrow ? "narrow " : "tiles ") << b.bm << "x" << b.bn << " n=" << b.total_tiles << " tail=" << tail << " shares=" << b.split << " rows";
  for (int i = 0; i < b.nprob; ++i) { s << " " << b.p[i].rows; }
  return emit(s.str());
}

hipError_t
launch_fp8_quant_rows(const uint16_t*, const uint16_t* up, int rows, int K, uint16_t* h, uint8_t*,
                      float*, hipStream_t)
{
  std::ostringstream s;
  s << (up != nullptr ? "swiglu " : "rows ") << rows << " " << K << (h != nullptr ? " h" : "");
  return emit(s.str());
}

hipError_t
launch_fp8_quant_blocks(const uint16_t*, int N, int K, uint8_t*, float*, hipStream_t)
{
  std::ostringstream s;
  s << "blocks " << N << " " << K;
  return emit(s.str());
}

hipError_t
launch_fp8_norm(const Fp8NormArgs& a, hipStream_t)
{
  std::ostringstream s;
  s << "norm " << a.m_und << " " << a.rows << " " << a.dim << (a.d != nullptr ? " add" : "")
    << (a.y != nullptr ? " y" : "");
  return emit(s.str());
}

}  // namespace u15h

namespace {

u15h_status
gemm(u15h_ctx* c, int mu, int mg, int K, const std::vector<int>& ns)
{
  std::vector<u15h_mot_proj_fp8> p;
  for (int n : ns) {
    p.push_back({fake<uint8_t>(), fake<float>(), fake<uint8_t>(), fake<float>(),
                 fake<u15h_bf16>(), n});
  }
  return u15h_mot_gemm_fp8(c, nullptr, fake<uint8_t>(), fake<float>(), mu, mg, K, p.data(),
                           (int)p.size());
}

// A call that is right but for its operand `which`.
u15h_status
bad(u15h_ctx* c, const std::string& which)
{
  auto* const x = fake<u15h_bf16>();
  auto* const q = fake<uint8_t>();
  auto* const s = fake<float>();
  auto* const off = fake<uint8_t>(4104);           // 8 past a 16-byte border
  u15h_mot_proj_fp8 p = {q, s, q, s, x, 256};
  auto product = [&](int mu, int mg) {
    return u15h_mot_gemm_fp8(c, nullptr, q, s, mu, mg, 256, &p, 1);
  };
  if (which == "rows.x") { return u15h_quant_rows_fp8(c, nullptr, nullptr, 4, 256, q, s); }
  if (which == "rows.q") { return u15h_quant_rows_fp8(c, nullptr, x, 4, 256, off, s); }
  if (which == "rows.s") { return u15h_quant_rows_fp8(c, nullptr, x, 4, 256, q, nullptr); }
  if (which == "blocks.w") { return u15h_quant_blocks_fp8(c, nullptr, nullptr, 8, 256, q, s); }
  if (which == "blocks.q") { return u15h_quant_blocks_fp8(c, nullptr, x, 8, 256, off, s); }
  if (which == "swiglu.up") {
    return u15h_swiglu_quant_fp8(c, nullptr, x, nullptr, 4, 256, nullptr, q, s);
  }
  if (which == "swiglu.h") {
    return u15h_swiglu_quant_fp8(c, nullptr, x, x, 4, 256, (u15h_bf16*)off, q, s);
  }
  auto norm = [&](const u15h_bf16* d, u15h_bf16* xo, const u15h_bf16* wg, float eps, u15h_bf16* y) {
    return u15h_mot_rms_norm_fp8(c, nullptr, x, d, xo, 2, 2, 256, x, wg, eps, y, q, s);
  };
  if (which == "norm.delta") { return norm(x, nullptr, x, 1e-6f, nullptr); }
  if (which == "norm.x_out") { return norm(nullptr, x, x, 1e-6f, nullptr); }
  if (which == "norm.w_gen") { return norm(x, x, nullptr, 1e-6f, nullptr); }
  if (which == "norm.eps") { return norm(x, x, x, -1.0f, nullptr); }
  if (which == "norm.nan") { return norm(x, x, x, std::nanf(""), nullptr); }
  if (which == "norm.y") { return norm(x, x, x, 1e-6f, x); }
  if (which == "gemm.y") { p.y = (u15h_bf16*)off; return product(2, 2); }
  if (which == "gemm.wq_und") { p.wq_und = off; return product(2, 0); }
  if (which == "gemm.sw_gen") { p.sw_gen = nullptr; return product(0, 2); }
  if (which == "gemm.nproj") {
    return u15h_mot_gemm_fp8(c, nullptr, q, s, 2, 2, 256, &p, U15H_MAX_PROJ + 1);
  }
  if (which == "gemm.proj") { return u15h_mot_gemm_fp8(c, nullptr, q, s, 2, 2, 256, nullptr, 1); }
  if (which == "gemm.sx") { return u15h_mot_gemm_fp8(c, nullptr, q, nullptr, 2, 2, 256, &p, 1); }
  // the operands of a group without rows are not looked at
  if (which == "none.gemm") { p.wq_gen = nullptr; p.sw_gen = nullptr; return product(2, 0); }
  return u15h_mot_gemm_fp8(nullptr, nullptr, q, s, 2, 2, 256, &p, 1);
}

}  // namespace

int
main(int argc, char** argv)
{
  u15h_ctx ctx;
  if (argc > 1) { ctx.cus = std::stoi(argv[1]); }
  g_capacity = (size_t)ctx.cus * 256 * 256 * 4;
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    std::string op, word;
    in >> op;
    std::vector<int> v;
    u15h_status st;
    g_out.clear();
    ctx.error.clear();
    if (op == "bad") {
      in >> word;
      st = bad(&ctx, word);
    } else {
      for (int i; in >> i;) { v.push_back(i); }
      auto* const x = fake<u15h_bf16>();
      auto* const q = fake<uint8_t>();
      auto* const s = fake<float>();
      if (op == "gemm") {
        st = gemm(&ctx, v[0], v[1], v[2], {v.begin() + 3, v.end()});
      } else if (op == "rows") {
        st = u15h_quant_rows_fp8(&ctx, nullptr, x, v[0], v[1], q, s);
      } else if (op == "blocks") {
        st = u15h_quant_blocks_fp8(&ctx, nullptr, x, v[0], v[1], q, s);
      } else if (op == "swiglu") {
        st = u15h_swiglu_quant_fp8(&ctx, nullptr, x, x, v[0], v[1], v[2] ? x : nullptr, q, s);
      } else {
        st = u15h_mot_rms_norm_fp8(&ctx, nullptr, x, v[3] ? x : nullptr, v[4] ? x : nullptr, v[0],
                                   v[1], v[2], x, x, 1e-6f, v[5] ? fake<u15h_bf16>(8192) : nullptr,
                                   q, s);
      }
    }
    std::cout << (g_out.empty() ? "-" : g_out) << " ; "
              << (st == U15H_OK ? "ok" : st == U15H_EINVAL ? "refused: " + ctx.error
                                                           : "failed: " + ctx.error)
              << "\n";
  }
  return 0;
}
