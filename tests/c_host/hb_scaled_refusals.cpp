// Calls the 8-bit operators with arguments they have to refuse, on a context that never saw a GPU:
// every refusal is host arithmetic in front of the first CUDA call.  Prints one line per call that
// was not refused as it should be; exit status 0 when there is none.
#include <stdio.h>
#include <string.h>

#include <functional>

#include "../../habu_b200/csrc/hb_internal.h"

static int bad = 0;

static hb_tensor mat(void* p, int dt, int64_t r, int64_t c, int64_t s0, int64_t s1) {
  hb_tensor t;
  memset(&t, 0, sizeof(t));
  t.ptr = p; t.dtype = dt; t.rank = 2;
  t.shape[0] = r; t.shape[1] = c; t.stride[0] = s0; t.stride[1] = s1;
  return t;
}

static void expect(hb_ctx& ctx, const char* what, hb_status got, hb_status want, const char* text) {
  if (got == want && strstr(ctx.err.c_str(), text)) return;
  printf("%s: status %d (wanted %d), \"%s\" (wanted \"%s\")\n", what, got, want, ctx.err.c_str(), text);
  ++bad;
}

int main() {
  hb_ctx ctx;
  char* const P = reinterpret_cast<char*>(uintptr_t(1) << 20);   // never dereferenced
  const hb_status INV = HB_ERR_INVALID, UNS = HB_ERR_UNSUPPORTED;

  // ---- quantize
  struct Q { hb_tensor x, q, s; int b; };
  auto quant = [&](const char* what, std::function<void(Q&)> f, hb_status want, const char* text) {
    Q a = {mat(P, HB_BF16, 300, 264, 264, 1), mat(P, HB_E4M3, 300, 264, 272, 1), mat(P, HB_F32, 300, 3, 3, 1), 1};
    f(a);
    ctx.err.clear();
    expect(ctx, what, hb_quantize(&ctx, &a.x, &a.q, &a.s, a.b), want, text);
  };
  quant("block_rows", [](Q& a) { a.b = 64; }, UNS, "block_rows");
  quant("x type", [](Q& a) { a.x.dtype = HB_I32; }, UNS, "dtype");
  quant("x e4m3", [](Q& a) { a.x.dtype = HB_E4M3; }, UNS, "dtype");
  quant("x rank", [](Q& a) { a.x.rank = 1; }, INV, "rank");
  quant("x null", [](Q& a) { a.x.ptr = nullptr; }, INV, "null");
  quant("no rows", [](Q& a) { a.x.shape[0] = 0; }, INV, "empty");
  quant("no columns", [](Q& a) { a.x.shape[1] = 0; }, INV, "empty");
  quant("x columns strided", [](Q& a) { a.x.stride[1] = 2; a.x.stride[0] = 600; }, UNS, "contiguous");
  quant("x rows overlap", [](Q& a) { a.x.stride[0] = 200; }, INV, "stride");
  quant("x misaligned", [](Q& a) { a.x.ptr = static_cast<char*>(a.x.ptr) + 1; }, INV, "misaligned");
  quant("q type", [](Q& a) { a.q.dtype = HB_BF16; }, INV, "e4m3");
  quant("q shape", [](Q& a) { a.q.shape[1] = 256; }, INV, "300 x 264");
  quant("q rows overlap", [](Q& a) { a.q.stride[0] = 263; }, INV, "stride");
  quant("scale type", [](Q& a) { a.s.dtype = HB_BF16; }, INV, "fp32");
  quant("scale columns", [](Q& a) { a.s.shape[1] = 2; }, INV, "300 x 3");
  quant("scale rows of blocks", [](Q& a) { a.b = 128; }, INV, "3 x 3");
  quant("scale overlaps", [](Q& a) { a.s.stride[0] = 2; }, INV, "overlap");
  quant("scale broadcast", [](Q& a) { a.s.stride[0] = 0; }, INV, "overlap");
  quant("scale misaligned", [](Q& a) { a.s.ptr = static_cast<char*>(a.s.ptr) + 2; }, INV, "misaligned");
  quant("too many rows", [](Q& a) { a.x.shape[0] = a.q.shape[0] = a.s.shape[0] = int64_t(1) << 31; }, UNS, "2^31");
  quant("too many columns", [](Q& a) { a.x.shape[1] = a.q.shape[1] = int64_t(1) << 31; a.x.stride[0] = a.q.stride[0] = int64_t(1) << 32; }, UNS, "2^31");
  expect(ctx, "null x", hb_quantize(&ctx, nullptr, nullptr, nullptr, 1), INV, "null");
  if (hb_quantize(nullptr, nullptr, nullptr, nullptr, 1) != INV) { puts("null context accepted"); ++bad; }

  // ---- rmsnorm_quant
  struct N { hb_tensor x, q, s, r; const void* g; bool res; };
  auto norm = [&](const char* what, std::function<void(N&)> f, hb_status want, const char* text) {
    N a = {mat(P, HB_BF16, 30, 264, 264, 1), mat(P, HB_E4M3, 30, 264, 272, 1), mat(P, HB_F32, 30, 3, 3, 1), mat(P, HB_BF16, 30, 264, 264, 1), P, true};
    f(a);
    ctx.err.clear();
    expect(ctx, what, hb_rmsnorm_quant(&ctx, &a.x, a.g, &a.q, &a.s, a.res ? &a.r : nullptr, 1e-5f), want, text);
  };
  norm("gain null", [](N& a) { a.g = nullptr; }, INV, "null");
  norm("x fp32", [](N& a) { a.x.dtype = HB_F32; }, UNS, "bf16");
  norm("residual fp32", [](N& a) { a.r.dtype = HB_F32; }, UNS, "bf16");
  norm("residual shape", [](N& a) { a.r.shape[0] = 29; }, INV, "residual");
  norm("columns not of 8", [](N& a) { a.x.shape[1] = a.r.shape[1] = a.q.shape[1] = 260; }, UNS, "multiple of 8");
  norm("too wide", [](N& a) { a.x.shape[1] = a.x.stride[0] = 16392; }, UNS, "16384");
  norm("gain misaligned", [](N& a) { a.g = static_cast<const char*>(a.g) + 8; }, INV, "aligned");
  norm("x pitch", [](N& a) { a.x.stride[0] = 268; }, INV, "aligned");
  norm("residual pitch", [](N& a) { a.r.stride[0] = 268; }, INV, "aligned");
  norm("q pitch", [](N& a) { a.q.stride[0] = 268; }, INV, "aligned");
  norm("scale shape", [](N& a) { a.s.shape[0] = 29; }, INV, "30 x 3");
  norm("scale null", [](N& a) { a.s.ptr = nullptr; }, INV, "null");

  // ---- swiglu_quant
  struct S { hb_tensor x, q, s; };
  auto swi = [&](const char* what, std::function<void(S&)> f, hb_status want, const char* text) {
    S a = {mat(P, HB_BF16, 30, 528, 528, 1), mat(P, HB_E4M3, 30, 264, 272, 1), mat(P, HB_F32, 30, 3, 3, 1)};
    f(a);
    ctx.err.clear();
    expect(ctx, what, hb_swiglu_quant(&ctx, &a.x, &a.q, &a.s), want, text);
  };
  swi("x fp32", [](S& a) { a.x.dtype = HB_F32; }, UNS, "dtype");
  swi("odd width", [](S& a) { a.x.shape[1] = 527; }, UNS, "multiple of 8");
  swi("half not of 8", [](S& a) { a.x.shape[1] = 520; a.q.shape[1] = 260; }, UNS, "multiple of 8");
  swi("q is as wide as x", [](S& a) { a.q.shape[1] = 528; a.q.stride[0] = 528; }, INV, "30 x 264");
  swi("x pitch", [](S& a) { a.x.stride[0] = 530; }, INV, "aligned");

  // ---- matmul_scaled
  struct M { hb_tensor a, sa, b, sb, c; hb_matmul_opts o; };
  auto mm = [&](const char* what, std::function<void(M&)> f, hb_status want, const char* text) {
    M a = {mat(P, HB_E4M3, 30, 264, 272, 1), mat(P, HB_F32, 30, 3, 3, 1), mat(P, HB_E4M3, 264, 300, 1, 272), mat(P, HB_F32, 3, 3, 1, 3),
           mat(P, HB_BF16, 30, 300, 300, 1), {HB_EPI_NONE, -1, nullptr, 0}};
    f(a);
    ctx.err.clear();
    expect(ctx, what, hb_matmul_scaled(&ctx, &a.a, &a.sa, &a.b, &a.sb, &a.c, &a.o), want, text);
  };
  mm("A bf16", [](M& a) { a.a.dtype = HB_BF16; }, INV, "e4m3");
  mm("B bf16", [](M& a) { a.b.dtype = HB_BF16; }, INV, "e4m3");
  mm("C fp32", [](M& a) { a.c.dtype = HB_F32; }, UNS, "bf16");
  mm("A rank", [](M& a) { a.a.rank = 3; }, INV, "rank");
  mm("A null", [](M& a) { a.a.ptr = nullptr; }, INV, "null");
  mm("no rows", [](M& a) { a.a.shape[0] = a.c.shape[0] = 0; }, INV, "empty");
  mm("inner dimensions", [](M& a) { a.b.shape[0] = 256; }, INV, "inner");
  mm("C shape", [](M& a) { a.c.shape[1] = 299; }, INV, "30 x 300");
  mm("C column-major", [](M& a) { a.c.stride[0] = 1; a.c.stride[1] = 30; }, UNS, "row-major");
  mm("C rows overlap", [](M& a) { a.c.stride[0] = 299; }, INV, "stride");
  mm("A column-major", [](M& a) { a.a.stride[0] = 1; a.a.stride[1] = 32; }, UNS, "row-major");
  mm("B along N", [](M& a) { a.b.stride[0] = 304; a.b.stride[1] = 1; }, UNS, "along K");
  mm("A pitch", [](M& a) { a.a.stride[0] = 264; }, UNS, "16");
  mm("B pitch", [](M& a) { a.b.stride[1] = 268; }, UNS, "16");
  mm("A base", [](M& a) { a.a.ptr = static_cast<char*>(a.a.ptr) + 8; }, UNS, "16");
  mm("C base", [](M& a) { a.c.ptr = static_cast<char*>(a.c.ptr) + 1; }, INV, "misaligned");
  mm("a_scale shape", [](M& a) { a.sa.shape[1] = 2; }, INV, "30 x 3");
  mm("b_scale shape", [](M& a) { a.sb.shape[1] = 2; }, INV, "3 x 3");
  mm("b_scale type", [](M& a) { a.sb.dtype = HB_BF16; }, INV, "fp32");
  mm("a_scale strides", [](M& a) { a.sa.stride[0] = 1; }, INV, "overlap");
  mm("epilogue", [](M& a) { a.o.epilogue = 9; }, INV, "epilogue");
  mm("epilogue negative", [](M& a) { a.o.epilogue = -1; }, INV, "epilogue");
  mm("config", [](M& a) { a.o.config_id = 0; }, INV, "config_id");
  mm("swiglu odd N", [](M& a) { a.o.epilogue = HB_EPI_SWIGLU; a.b.shape[1] = 299; a.c.shape[1] = 149; }, INV, "even");
  mm("swiglu C width", [](M& a) { a.o.epilogue = HB_EPI_SWIGLU; }, INV, "30 x 150");
  mm("residual missing", [](M& a) { a.o.epilogue = HB_EPI_RESIDUAL; }, INV, "residual");
  mm("residual pitch", [&](M& a) { a.o.epilogue = HB_EPI_RESIDUAL; a.o.residual = P; a.o.residual_ld = 100; }, INV, "residual");
  mm("residual misaligned", [&](M& a) { a.o.epilogue = HB_EPI_RESIDUAL; a.o.residual = P + 1; }, INV, "misaligned");
  expect(ctx, "null tensors", hb_matmul_scaled(&ctx, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr), INV, "null");
  if (hb_matmul_scaled(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != INV) { puts("null context accepted"); ++bad; }

  // ---- graph: every other node takes its tensors' elements for two bytes or four
  hb_graph* g = nullptr;
  if (hb_graph_create(&ctx, &g) != HB_OK) { puts("no graph"); return 1; }
  const hb_tensor q = mat(P, HB_E4M3, 64, 256, 256, 1), w = mat(P, HB_BF16, 64, 256, 256, 1);
  int32_t iq = -1, iw = -1;
  hb_graph_input(g, &q, &iq);
  hb_graph_input(g, &w, &iw);
  for (int kind = HB_NODE_MATMUL; kind < HB_NODE_QUANTIZE; ++kind)
    for (int at = 0; at < 5; ++at) {
      hb_node n;
      memset(&n, 0, sizeof(n));
      n.kind = kind;
      for (int i = 0; i < 4; ++i) n.in[i] = at == i ? iq : iw;
      n.out = at == 4 ? iq : iw;
      ctx.err.clear();
      expect(ctx, "e4m3 in another node", hb_graph_add(g, &n), UNS, "e4m3");
    }
  hb_graph_destroy(g);
  if (ctx.launches) { puts("something was launched"); ++bad; }
  return bad ? 1 : 0;
}
