// Run by tests/test_host_block.py, without a GPU: the 4-bit and norm wrappers of
// miaie.hpp over entry points that record their arguments.  Operands that do not
// fit together, or buffers too short, have to be refused before an entry point is
// called; those that fit have to reach it with the sizes they stand for.
#include <cstdio>
#include <cstdlib>
#include <string>
#include <vector>

#include "miaie.hpp"

static std::string last;  // the last compute call: name and sizes
static int calls = 0;
static std::vector<const void*> pointers;  // of the last gradient

template <class... I>
static int called(const char* name, I... sizes) {
  ++calls;
  last = name;
  ((last += " " + std::to_string(sizes)), ...);
  return MIAIE_OK;
}

extern "C" {
int miaie_init(miaie_ctx** ctx, int) { return *ctx = reinterpret_cast<miaie_ctx*>(8), MIAIE_OK; }
int miaie_finish(miaie_ctx*) { return MIAIE_OK; }
const char* miaie_last_error_string(const miaie_ctx*) { return "recorded"; }
int miaie_alloc(miaie_ctx*, size_t, void** p) {  // addresses of their own, never read
  static uintptr_t next = 0;
  return *p = reinterpret_cast<void*>(next += 4096), MIAIE_OK;
}
int miaie_free(miaie_ctx*, void*) { return MIAIE_OK; }
size_t miaie_mxfp4_q_bytes(int R, int K) { return (size_t)R * ((K + 255) / 256 * 128); }
size_t miaie_mxfp4_s_bytes(int R, int K) { return (size_t)R * ((K + 511) / 512) * 16; }
int miaie_quant_mxfp4(miaie_ctx*, const void*, int, int R, int C, int ldx, uint8_t* Q, uint8_t*, uint8_t* Qt, uint8_t*) {
  return called("quant", R, C, ldx, Q != nullptr, Qt != nullptr);
}
int miaie_dequant_mxfp4(miaie_ctx*, const uint8_t*, const uint8_t*, void*, int, int R, int C, int ldy) {
  return called("dequant", R, C, ldy);
}
int miaie_gemm_mxfp4(miaie_ctx*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, int, int M, int N,
                     int K, int ldc) {
  return called("gemm", M, N, K, ldc);
}
int miaie_gemm_mxfp4_rq(miaie_ctx*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, uint8_t*, uint8_t*,
                        int M, int N, int K, int relu) {
  return called("gemm_rq", M, N, K, relu);
}
int miaie_mlp_mxfp4(miaie_ctx*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*,
                    const uint8_t*, uint8_t*, uint8_t*, void*, int, int M, int K, int F, int Nout, int ldy) {
  return called("mlp", M, K, F, Nout, ldy);
}
int miaie_norm_block(miaie_ctx*, const void*, const void* b, const void* gate, const float*, const float*, void*, void* y,
                     float*, int rows, int cols, int ldx, int ldb, int gate_rows, int, int, float, float) {
  return called("norm", rows, cols, ldx, ldb, gate_rows, b != nullptr, gate != nullptr, y != nullptr);
}
int miaie_norm_block_grad(miaie_ctx*, const void* r, const void* b, const void* gate, const float* w_after,
                          const float* w_before, const float* rstd, const void* dout, const void* dy, void* dx, void* db,
                          float* dgate, float* dw_after, float* dw_before, void* work, size_t work_bytes, int rows, int cols,
                          int ldx, int ldb, int gate_rows, int stream_dtype, int branch_dtype, float alpha) {
  pointers = {r, b, gate, w_after, w_before, rstd, dout, dy, dx, db, dgate, dw_after, dw_before, work};
  return called("grad", work_bytes, rows, cols, ldx, ldb, gate_rows, stream_dtype, branch_dtype, (int)(8 * alpha));
}
}

static int failures = 0;

static void report(bool ok, int line, const char* what) {
  if (ok) return;
  ++failures;
  std::printf("line %d: %s; last call: %s\n", line, what, last.c_str());
}

template <class F>
static void refused(int line, const char* text, F&& f) {
  const int before = calls;
  try {
    f();
    report(false, line, "not refused");
  } catch (const miaie::Error& e) {
    report(e.code() == MIAIE_EINVAL && std::string(e.what()).find(text) != std::string::npos, line, e.what());
  }
  report(calls == before, line, "an entry point was called");
}

static void same(int line, const std::vector<const void*>& want) {
  report(pointers == want, line, "the gradient's buffers are not where they belong");
}

template <class F>
static void reaches(int line, const char* want, F&& f) {
  try {
    f();
    report(last == want, line, want);
  } catch (const miaie::Error& e) {
    report(false, line, e.what());
  }
}

#define REFUSED(text, call) refused(__LINE__, text, [&] { call; })
#define REACHES(want, call) reaches(__LINE__, want, [&] { call; })
#define BUFFERS(...) same(__LINE__, {__VA_ARGS__})

int main() {
  using namespace miaie;
  Context ctx;
  MxMatrix A(ctx, 5, 300), B(ctx, 7, 300), longer(ctx, 5, 301), Y(ctx, 5, 7), Yt(ctx, 7, 5), W2(ctx, 9, 7);
  Buffer<float> c35(ctx, 35), c34(ctx, 34), c45(ctx, 45), c44(ctx, 44), x(ctx, 1500), x1(ctx, 1499);
  Buffer<uint16_t> h(ctx, 1500), h1(ctx, 1499);

  REACHES("quant 5 300 300 1 0", quant_mxfp4(x, A));
  REACHES("quant 5 300 300 1 0", quant_mxfp4(h, A));
  REFUSED("X is smaller", quant_mxfp4(x1, A));
  REACHES("quant 300 5 5 0 1", quant_mxfp4_t(x, A));
  REFUSED("X is smaller", quant_mxfp4_t(h1, A));
  MxMatrix At(ctx, 300, 5);
  REACHES("quant 5 300 300 1 1", quant_mxfp4_both(x, A, At));
  REFUSED("X is smaller", quant_mxfp4_both(h1, A, At));
  REFUSED("transpose", quant_mxfp4_both(x, A, longer));
  REACHES("dequant 5 300 300", dequant_mxfp4(A, h));
  REFUSED("Y is smaller", dequant_mxfp4(A, h1));

  REACHES("gemm 5 7 300 7", gemm_mxfp4(A, B, c35));
  REFUSED("different lengths", gemm_mxfp4(longer, B, c35));
  REFUSED("different lengths", gemm_mxfp4(B, longer, c35));
  REFUSED("C is smaller", gemm_mxfp4(A, B, c34));
  REACHES("gemm_rq 5 7 300 1", gemm_mxfp4_rq(A, B, Y, true));
  REFUSED("different lengths", gemm_mxfp4_rq(longer, B, Y));
  REFUSED("shape", gemm_mxfp4_rq(A, B, Yt));
  REACHES("mlp 5 300 7 9 9", mlp_mxfp4(A, B, W2, Y, c45));
  REFUSED("different lengths", mlp_mxfp4(longer, B, W2, Y, c45));
  REFUSED("W2", mlp_mxfp4(A, B, B, Y, c45));
  REFUSED("shape", mlp_mxfp4(A, B, W2, Yt, c45));
  REFUSED("Y is smaller", mlp_mxfp4(A, B, W2, Y, c44));

  const NormShape n{5, 300}, two{5, 300, 1.f, 1e-5f, 2};
  Buffer<float> w(ctx, 300), w1(ctx, 299), rstd(ctx, 10), rstd1(ctx, 9), out(ctx, 1500);
  Buffer<uint16_t> gate(ctx, 900), gate1(ctx, 899), next(ctx, 1500);
  REACHES("norm 5 300 300 300 5 0 0 1", norm_before(x, w, h, n, &rstd));
  REFUSED("x or y", norm_before(x1, w, h, n));
  REFUSED("x or y", norm_before(x, w, h1, n));
  REFUSED("w_before", norm_before(x, w1, h, n));
  REFUSED("rstd", norm_before(x, w, h, n, &rstd1));
  REACHES("norm 5 300 300 300 2 1 1 1", norm_block(x, h, &gate, w, &w, out, &next, two, &rstd));
  REACHES("norm 5 300 300 300 5 1 1 0",
          norm_block(x, h, &gate1, w, (const Buffer<float>*)nullptr, out, (Buffer<uint16_t>*)nullptr, n));
  REFUSED("smaller than rows", norm_block(x, h1, &gate, w, &w, out, &next, two));
  REFUSED("smaller than rows", norm_block(x, h, &gate, w, &w, x1, &next, two));
  REFUSED("smaller than rows", norm_block(x, h, &gate, w, &w, out, &h1, two));
  REFUSED("gate", norm_block(x, h, &gate1, w, &w, out, &next, two));
  REFUSED("w_after", norm_block(x, h, &gate, w1, &w, out, &next, two));
  REFUSED("w_after", norm_block(x, h, &gate, w, &w1, out, &next, two));
  REFUSED("rstd", norm_block(x, h, &gate, w, &w, out, &next, two, &rstd1));

  // the gradient: fp32 stream, bf16 branch, gates of two rows (three of them)
  const NormShape g{5, 300, 0.5f, 1e-5f, 2};
  Buffer<float> dout(ctx, 1500), dx(ctx, 1500), dgate(ctx, 900), dgate1(ctx, 899), dwa(ctx, 300), dwb(ctx, 300), work(ctx, 1024 * 300);
  Buffer<uint16_t> dy(ctx, 1500), db(ctx, 1500);
  const NormGrads<float, uint16_t> all{&dx, &db, &dgate, &dwa, &dwb};
  REACHES("grad 1228800 5 300 300 300 2 0 1 4",
          norm_block_grad(x, h, &gate, w, &w, rstd, &dout, &dy, all, &work, g));
  BUFFERS(x.data(), h.data(), gate.data(), w.data(), w.data(), rstd.data(), dout.data(), dy.data(), dx.data(), db.data(),
          dgate.data(), dwa.data(), dwb.data(), work.data());
  const Buffer<uint16_t>* none = nullptr;
  REACHES("grad 0 5 300 300 300 5 0 1 8",
          norm_block_grad(x, h, none, w, &w, rstd, &dout, none, NormGrads<float, uint16_t>{&dx, &db}, (Buffer<float>*)nullptr, n));
  BUFFERS(x.data(), h.data(), nullptr, w.data(), nullptr, rstd.data(), dout.data(), nullptr, dx.data(), db.data(), nullptr,
          nullptr, nullptr, nullptr);
  REACHES("grad 1228800 5 300 300 300 5 0 1 8", norm_before_grad(x, w, rstd, &dout, dy, &dx, &dwb, &work, n));
  BUFFERS(x.data(), nullptr, nullptr, nullptr, w.data(), rstd.data(), dout.data(), dy.data(), dx.data(), nullptr, nullptr,
          nullptr, dwb.data(), work.data());
  REFUSED("smaller than rows", norm_block_grad(x, h1, &gate, w, &w, rstd, &dout, &dy, all, &work, g));
  REFUSED("smaller than rows", norm_block_grad(x, h, &gate, w, &w, rstd, &x1, &dy, all, &work, g));
  REFUSED("dgate", norm_block_grad(x, h, &gate, w, &w, rstd, &dout, &dy, NormGrads<float, uint16_t>{&dx, &db, &dgate1}, &work, g));
  REFUSED("dw_after", norm_block_grad(x, h, &gate, w1, &w, rstd, &dout, &dy, all, &work, g));
  REFUSED("rstd", norm_block_grad(x, h, &gate, w, &w, rstd1, &dout, &dy, all, &work, g));
  REFUSED("smaller than rows", norm_before_grad(x, w, rstd, &dout, h1, &dx, &dwb, &work, n));
  REFUSED("dw_before", norm_before_grad(x, w, rstd, &dout, dy, &dx, &w1, &work, n));
  REFUSED("rstd", norm_before_grad(x, w, rstd1, &dout, dy, &dx, &dwb, &work, n));

  std::printf("%d calls, %d failures\n", calls, failures);
  return failures != 0;
}
