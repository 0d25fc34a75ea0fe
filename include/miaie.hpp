// miaie.hpp — C++ host surface over the miaie C ABI (miaie.h).
//
// Header-only; links against libmiaie.so.  Two layers:
//
//  1. RAII wrappers for the aie-rt-shaped runtime calls the reference
//     harnesses make (example/matrixmultiply/aieml_mm.cc:108-249):
//     Context (XAie_CfgInitialize / XAie_PartitionInitialize / teardown),
//     Buffer<T> (XAie_MemAllocate + XAie_MemGetDevAddr), move_in / move_out
//     (XAie_MoveData* + XAie_MemSync*), Context::wait (XAie_CoreWaitForDone,
//     with a deadline).  Failures throw miaie::Error carrying the status.
//
//  2. The aiehlc `__kernel__` launch surface.  aiehlc rewrites a kernel
//     declared `__kernel__` into a template
//       template <int Col, int Row, int colstart, int rowstart, int M, int N, int K,
//                 typename... Args> void NAME(Args&&...)
//     (src/llvm/aiehlc.cc:583-588) that harnesses call as
//       perf<1, 1, 4, 4, 256, 16, 64>(phy, phy_out);   (example/nokernelload/aie_nokernelload.cc:130)
//     Here the same template shapes launch the gfx950 kernels.  Col, Row,
//     colstart and rowstart place a kernel on AIE tiles; on one GPU the
//     placement is the grid decomposition over the CUs, so they are accepted
//     and not used.  M, N, K fix the problem shape at compile time.  Every
//     launch is asynchronous on the current context's stream.
#ifndef MIAIE_HPP
#define MIAIE_HPP

#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>
#include <vector>

#include "miaie.h"

namespace miaie {

class Error : public std::runtime_error {
 public:
  Error(int code, const std::string& what) : std::runtime_error(what), code_(code) {}
  int code() const { return code_; }

 private:
  int code_;
};

class Context;

namespace detail {
inline Context*& current() {
  static thread_local Context* c = nullptr;
  return c;
}
}  // namespace detail

// One device and one stream.  The most recently constructed Context on a
// thread is that thread's current context (used by the template launchers).
class Context {
 public:
  explicit Context(int device = 0) {
    if (int rc = miaie_init(&h_, device)) throw Error(rc, miaie_last_error_string(nullptr));
    prev_ = detail::current();
    detail::current() = this;
  }
  ~Context() {
    if (detail::current() == this) detail::current() = prev_;
    miaie_finish(h_);
  }
  Context(const Context&) = delete;
  Context& operator=(const Context&) = delete;

  miaie_ctx* get() const { return h_; }
  static Context& current() {
    if (!detail::current()) throw Error(MIAIE_EINVAL, "no current miaie::Context on this thread");
    return *detail::current();
  }

  // Throw on a non-zero status from an entry point called on this context.
  void check(int rc) const {
    if (rc != MIAIE_OK) throw Error(rc, miaie_last_error_string(h_));
  }
  // XAie_CoreWaitForDone analogue: returns false on MIAIE_ETIMEDOUT.
  bool wait(int timeout_ms = -1) const {
    const int rc = miaie_wait(h_, timeout_ms);
    if (rc == MIAIE_ETIMEDOUT) return false;
    check(rc);
    return true;
  }
  // The tiling planner: the kernel, tile and grid an int8 GEMM of this shape
  // takes, and the CU count it plans for (returns the previous one).
  miaie_gemm_plan plan_gemm_i8(int M, int N, int K) const {
    miaie_gemm_plan p{};
    check(miaie_plan_gemm_i8(h_, M, N, K, &p));
    return p;
  }
  int plan_set_cus(int cus) const {
    int prev = 0;
    check(miaie_plan_set_cus(h_, cus, &prev));
    return prev;
  }

 private:
  miaie_ctx* h_ = nullptr;
  Context* prev_ = nullptr;
};

// Device buffer of n elements of T (XAie_MemAllocate).
template <typename T>
class Buffer {
 public:
  Buffer(Context& ctx, size_t n) : ctx_(&ctx), n_(n) {
    void* p = nullptr;
    ctx.check(miaie_alloc(ctx.get(), n * sizeof(T) > 0 ? n * sizeof(T) : 1, &p));
    p_ = static_cast<T*>(p);
  }
  ~Buffer() {
    if (p_) miaie_free(ctx_->get(), p_);
  }
  Buffer(Buffer&& o) noexcept : ctx_(o.ctx_), p_(o.p_), n_(o.n_) { o.p_ = nullptr; }
  Buffer(const Buffer&) = delete;
  Buffer& operator=(const Buffer&) = delete;

  T* data() const { return p_; }
  size_t size() const { return n_; }
  size_t bytes() const { return n_ * sizeof(T); }

  // XAie_MoveDataExternal2Aie / XAie_MoveData host -> tile (+ MemSyncForDev)
  void move_in(const T* host, size_t n) { ctx_->check(miaie_copy_h2d(ctx_->get(), p_, host, n * sizeof(T))); }
  void move_in(const std::vector<T>& host) { move_in(host.data(), host.size()); }
  // XAie_MoveDataAie2External / XAie_MoveData tile -> host (+ MemSyncForCPU)
  void move_out(T* host, size_t n) const { ctx_->check(miaie_copy_d2h(ctx_->get(), host, p_, n * sizeof(T))); }
  std::vector<T> move_out() const {
    std::vector<T> h(n_);
    move_out(h.data(), n_);
    return h;
  }

 private:
  Context* ctx_;
  T* p_ = nullptr;
  size_t n_;
};

// ---------------------------------------------------------------- aiehlc launch surface
// `mm` of example/matrixmultiply/aieml_mm.cc:41-93 (window in: A[M][K] || B[N][K],
// out: C[M][N] = A . B^T, int32 wrap-around).  The window kernel is square.
template <int Col, int Row, int colstart, int rowstart, int M, int N, int K>
void mm(const int32_t* in_window, int32_t* out_window, Context& ctx = Context::current()) {
  static_assert(M == N && N == K && M >= 1 && M <= 4096, "mm: square window, n in [1, 4096]");
  ctx.check(miaie_mm_window_i32(ctx.get(), in_window, out_window, M));
}

// `perf` of example/perf/aieml_perf.cc:61-83 (uint32 variant of mm).
template <int Col, int Row, int colstart, int rowstart, int M, int N, int K>
void perf(const uint32_t* in_window, uint32_t* out_window, Context& ctx = Context::current()) {
  static_assert(M == N && N == K && M >= 1 && M <= 4096, "perf: square window, n in [1, 4096]");
  ctx.check(miaie_perf_window_u32(ctx.get(), in_window, out_window, M));
}

// `perf` of example/nokernelload/aie_nokernelload.cc:50-83, launched there as
// perf<1,1,4,4,256,16,64>(phy, phy_out): the uint8 MAC probe (in[0] =
// param_nn; out[0..4]).  M/N/K do not change the probe.
template <int Col, int Row, int colstart, int rowstart, int M, int N, int K>
void dot_probe(const uint32_t* in, uint32_t* out, Context& ctx = Context::current()) {
  ctx.check(miaie_dot_u8_probe(ctx.get(), in, out));
}

// int8 GEMM + requant, dense row-major NN: Y[M][N] = rq_shift(A[M][K] . B[K][N]).
template <int Col, int Row, int colstart, int rowstart, int M, int N, int K>
void gemm_i8(const int8_t* A, const int8_t* B, int8_t* Y, int shift, bool relu = false, int32_t* C_dbg = nullptr,
             Context& ctx = Context::current()) {
  static_assert(M >= 1 && N >= 1 && K >= 1, "gemm_i8: positive shape");
  ctx.check(miaie_gemm_i8_rq(ctx.get(), A, B, Y, M, N, K, shift, relu ? 1 : 0, C_dbg, MIAIE_B_NN));
}

// bf16 x bf16 -> fp32 GEMM, dense row-major NN (bf16 as raw uint16 bits).
template <int Col, int Row, int colstart, int rowstart, int M, int N, int K>
void gemm_bf16(const uint16_t* A, const uint16_t* B, float* C, Context& ctx = Context::current()) {
  static_assert(M >= 1 && N >= 1 && K >= 1, "gemm_bf16: positive shape");
  ctx.check(miaie_gemm_bf16_f32(ctx.get(), A, B, C, M, N, K));
}

// ---------------------------------------------------------------- runtime-shape operators
// The typed entry points with shapes known at run time, on device buffers.
// Asynchronous on the context's stream, like the launch templates above.

// Y = rq_shift(A . B) (NN or NT B, layout MIAIE_B_NN / MIAIE_B_NT); C_dbg
// (nullable) receives the int32 accumulators.
inline void gemm_i8_rq(const Buffer<int8_t>& A, const Buffer<int8_t>& B, Buffer<int8_t>& Y, int M, int N, int K,
                       int shift, bool relu = false, Buffer<int32_t>* C_dbg = nullptr, int b_layout = MIAIE_B_NN,
                       Context& ctx = Context::current()) {
  ctx.check(miaie_gemm_i8_rq(ctx.get(), A.data(), B.data(), Y.data(), M, N, K, shift, relu ? 1 : 0,
                             C_dbg ? C_dbg->data() : nullptr, b_layout));
}

// C = A . B in int32, with row pitches (elements) lda / ldb / ldc.
inline void gemm_i8_i32(const Buffer<int8_t>& A, const Buffer<int8_t>& B, Buffer<int32_t>& C, int M, int N, int K,
                        int lda, int ldb, int ldc, int b_layout = MIAIE_B_NN, Context& ctx = Context::current()) {
  ctx.check(miaie_gemm_i8_i32(ctx.get(), A.data(), B.data(), C.data(), M, N, K, lda, ldb, ldc, b_layout));
}

// C = A . B, bf16 in (raw uint16 bits), fp32 accumulate and out, NN.
inline void gemm_bf16(const Buffer<uint16_t>& A, const Buffer<uint16_t>& B, Buffer<float>& C, int M, int N, int K,
                      Context& ctx = Context::current()) {
  ctx.check(miaie_gemm_bf16_f32(ctx.get(), A.data(), B.data(), C.data(), M, N, K));
}

// Shape of an NHWC x OHWI convolution.
struct ConvShape {
  int N, H, W, Cin, Cout, R = 3, S = 3, stride = 1, pad = 1;
  int Ho() const { return (H + 2 * pad - R) / stride + 1; }
  int Wo() const { return (W + 2 * pad - S) / stride + 1; }
};

// Y[N][Ho][Wo][Cout] = per-channel rq(conv(X, Wt)), shifts[c] in [0, 31].
inline void conv2d_i8(const Buffer<int8_t>& X, const Buffer<int8_t>& Wt, const Buffer<uint8_t>& shifts,
                      Buffer<int8_t>& Y, const ConvShape& c, Context& ctx = Context::current()) {
  ctx.check(miaie_conv2d_i8_nhwc(ctx.get(), X.data(), Wt.data(), shifts.data(), Y.data(), c.N, c.H, c.W, c.Cin,
                                 c.Cout, c.R, c.S, c.stride, c.pad));
}

// H = relu(rq_s1(X . W1)), Y = rq_s2(H . W2); H is caller-provided device
// scratch of M x F.
inline void mlp_i8(const Buffer<int8_t>& X, const Buffer<int8_t>& W1, const Buffer<int8_t>& W2, Buffer<int8_t>& H,
                   Buffer<int8_t>& Y, int M, int K, int F, int Nout, int s1, int s2,
                   Context& ctx = Context::current()) {
  ctx.check(miaie_mlp_i8(ctx.get(), X.data(), W1.data(), W2.data(), H.data(), Y.data(), M, K, F, Nout, s1, s2));
}

// The 4-bit and 8-bit operators, the experts' and the norms infer sizes, and refuse (miaie::Error,
// MIAIE_EINVAL, before anything is queued) operands that do not fit together and
// buffers shorter than those sizes.
namespace detail {
inline void require(bool ok, const char* fn, const char* what) {
  if (!ok) throw Error(MIAIE_EINVAL, std::string(fn) + ": " + what);
}
// rows x cols elements fit the buffer (sizes below 1 are left to the entry point)
template <typename T>
bool holds(const Buffer<T>& b, int rows, int cols) {
  return rows < 1 || cols < 1 || b.size() / (size_t)cols >= (size_t)rows;
}
}  // namespace detail

// A packed MXFP4 matrix (miaie.h) of rows x cols.
struct MxMatrix {
  MxMatrix(Context& ctx, int rows, int cols)
      : rows(rows), cols(cols), q(ctx, miaie_mxfp4_q_bytes(rows, cols)), s(ctx, miaie_mxfp4_s_bytes(rows, cols)) {}
  int rows, cols;
  Buffer<uint8_t> q, s;
};

// MIAIE_F32 / MIAIE_BF16 of a buffer's elements (bf16 as raw uint16 bits).
inline constexpr int dtype_of(const float*) { return MIAIE_F32; }
inline constexpr int dtype_of(const uint16_t*) { return MIAIE_BF16; }

// Q = X packed along its rows (X dense, Q.rows x Q.cols).
template <typename T>
void quant_mxfp4(const Buffer<T>& X, MxMatrix& Q, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Q.rows, Q.cols), "quant_mxfp4", "X is smaller than Q");
  ctx.check(miaie_quant_mxfp4(ctx.get(), X.data(), dtype_of(X.data()), Q.rows, Q.cols, Q.cols, Q.q.data(), Q.s.data(),
                              nullptr, nullptr));
}

// Qt = the transpose of X packed along its rows (X dense, Qt.cols x Qt.rows).
template <typename T>
void quant_mxfp4_t(const Buffer<T>& X, MxMatrix& Qt, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Qt.cols, Qt.rows), "quant_mxfp4_t", "X is smaller than Qt");
  ctx.check(miaie_quant_mxfp4(ctx.get(), X.data(), dtype_of(X.data()), Qt.cols, Qt.rows, Qt.rows, nullptr, nullptr,
                              Qt.q.data(), Qt.s.data()));
}

// Both from one read of X.
template <typename T>
void quant_mxfp4_both(const Buffer<T>& X, MxMatrix& Q, MxMatrix& Qt, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Q.rows, Q.cols), "quant_mxfp4_both", "X is smaller than Q");
  detail::require(Qt.rows == Q.cols && Qt.cols == Q.rows, "quant_mxfp4_both", "Qt does not have the shape of Q's transpose");
  ctx.check(miaie_quant_mxfp4(ctx.get(), X.data(), dtype_of(X.data()), Q.rows, Q.cols, Q.cols, Q.q.data(), Q.s.data(),
                              Qt.q.data(), Qt.s.data()));
}

// Y = the values of Q.
template <typename T>
void dequant_mxfp4(const MxMatrix& Q, Buffer<T>& Y, Context& ctx = Context::current()) {
  detail::require(detail::holds(Y, Q.rows, Q.cols), "dequant_mxfp4", "Y is smaller than Q");
  ctx.check(miaie_dequant_mxfp4(ctx.get(), Q.q.data(), Q.s.data(), Y.data(), dtype_of(Y.data()), Q.rows, Q.cols, Q.cols));
}

// C = A . B^T (A M x K, B N x K).
template <typename T>
void gemm_mxfp4(const MxMatrix& A, const MxMatrix& B, Buffer<T>& C, Context& ctx = Context::current()) {
  detail::require(A.cols == B.cols, "gemm_mxfp4", "A and B have rows of different lengths");
  detail::require(detail::holds(C, A.rows, B.rows), "gemm_mxfp4", "C is smaller than A . B^T");
  ctx.check(miaie_gemm_mxfp4(ctx.get(), A.q.data(), A.s.data(), B.q.data(), B.s.data(), C.data(), dtype_of(C.data()),
                             A.rows, B.rows, A.cols, B.rows));
}

// Y = A . B^T packed again, after a ReLU if relu.
inline void gemm_mxfp4_rq(const MxMatrix& A, const MxMatrix& B, MxMatrix& Y, bool relu = false,
                          Context& ctx = Context::current()) {
  detail::require(A.cols == B.cols, "gemm_mxfp4_rq", "A and B have rows of different lengths");
  detail::require(Y.rows == A.rows && Y.cols == B.rows, "gemm_mxfp4_rq", "Y does not have the shape of A . B^T");
  ctx.check(miaie_gemm_mxfp4_rq(ctx.get(), A.q.data(), A.s.data(), B.q.data(), B.s.data(), Y.q.data(), Y.s.data(),
                                A.rows, B.rows, A.cols, relu ? 1 : 0));
}

// H = pack(relu(X . W1^T)), Y = H . W2^T.
template <typename T>
void mlp_mxfp4(const MxMatrix& X, const MxMatrix& W1, const MxMatrix& W2, MxMatrix& H, Buffer<T>& Y,
               Context& ctx = Context::current()) {
  detail::require(X.cols == W1.cols, "mlp_mxfp4", "X and W1 have rows of different lengths");
  detail::require(W1.rows == W2.cols, "mlp_mxfp4", "W2's rows do not have W1's number of rows");
  detail::require(H.rows == X.rows && H.cols == W1.rows, "mlp_mxfp4", "H does not have the shape of X . W1^T");
  detail::require(detail::holds(Y, X.rows, W2.rows), "mlp_mxfp4", "Y is smaller than H . W2^T");
  ctx.check(miaie_mlp_mxfp4(ctx.get(), X.q.data(), X.s.data(), W1.q.data(), W1.s.data(), W2.q.data(), W2.s.data(),
                            H.q.data(), H.s.data(), Y.data(), dtype_of(Y.data()), X.rows, X.cols, W1.rows, W2.rows,
                            W2.rows));
}

// Row counts, sizes and constants of the norms around a block (miaie_norm_block).
struct NormShape {
  int rows, cols;
  float alpha = 1.f, eps = 1e-5f;
  int gate_rows = 0;  // rows that share a gate row; 0: all of them
  int rows_of_a_gate() const { return gate_rows ? gate_rows : rows; }
  int gates() const { return gate_rows > 0 ? (int)(((long long)rows + gate_rows - 1) / gate_rows) : 1; }
};

// y = w_before * x / rms(x).
template <typename S, typename B>
void norm_before(const Buffer<S>& x, const Buffer<float>& w_before, Buffer<B>& y, const NormShape& n,
                 Buffer<float>* rstd = nullptr, Context& ctx = Context::current()) {
  detail::require(detail::holds(x, n.rows, n.cols) && detail::holds(y, n.rows, n.cols), "norm_before",
                  "x or y is smaller than rows x cols");
  detail::require(detail::holds(w_before, 1, n.cols), "norm_before", "w_before is shorter than a row");
  detail::require(!rstd || detail::holds(*rstd, 2, n.rows), "norm_before", "rstd is smaller than 2 x rows");
  ctx.check(miaie_norm_block(ctx.get(), x.data(), nullptr, nullptr, nullptr, w_before.data(), nullptr, y.data(),
                             rstd ? rstd->data() : nullptr, n.rows, n.cols, n.cols, n.cols, n.rows,
                             dtype_of(x.data()), dtype_of(y.data()), n.alpha, n.eps));
}

// out = alpha x + gate * w_after * b / rms(b) and, with w_before and y, the
// norm before the next block, y = w_before * out / rms(out).  gate (nullable):
// ceil(rows / gate_rows) x cols.
template <typename S, typename B>
void norm_block(const Buffer<S>& x, const Buffer<B>& b, const Buffer<B>* gate, const Buffer<float>& w_after,
                const Buffer<float>* w_before, Buffer<S>& out, Buffer<B>* y, const NormShape& n,
                Buffer<float>* rstd = nullptr, Context& ctx = Context::current()) {
  detail::require(detail::holds(x, n.rows, n.cols) && detail::holds(b, n.rows, n.cols) &&
                      detail::holds(out, n.rows, n.cols) && (!y || detail::holds(*y, n.rows, n.cols)),
                  "norm_block", "x, b, out or y is smaller than rows x cols");
  detail::require(!gate || detail::holds(*gate, n.gates(), n.cols), "norm_block", "gate is smaller than its rows x cols");
  detail::require(detail::holds(w_after, 1, n.cols) && (!w_before || detail::holds(*w_before, 1, n.cols)), "norm_block",
                  "w_after or w_before is shorter than a row");
  detail::require(!rstd || detail::holds(*rstd, 2, n.rows), "norm_block", "rstd is smaller than 2 x rows");
  ctx.check(miaie_norm_block(ctx.get(), x.data(), b.data(), gate ? gate->data() : nullptr, w_after.data(),
                             w_before ? w_before->data() : nullptr, out.data(), y ? y->data() : nullptr,
                             rstd ? rstd->data() : nullptr, n.rows, n.cols, n.cols, n.cols, n.rows_of_a_gate(),
                             dtype_of(x.data()), dtype_of(b.data()), n.alpha, n.eps));
}

// The gradients that norm_block_grad is to compute; those left NULL are not.
// dx may be the buffer of dout, db that of dy or b.
template <typename S, typename B>
struct NormGrads {
  Buffer<S>* dx = nullptr;
  Buffer<B>* db = nullptr;
  Buffer<float>* dgate = nullptr;     // the shape of gate
  Buffer<float>* dw_after = nullptr;  // cols
  Buffer<float>* dw_before = nullptr;
};

// The gradient of norm_block: r the stream that the second norm read (out of
// norm_block), rstd as norm_block kept it; dout (nullable: 0) the gradient of the
// stream from elsewhere, dy (nullable: no second norm; then w_before is not read) of
// y.  work (nullable unless dgate, dw_after or dw_before is wanted): device scratch
// of MIAIE_NORM_WORK_BYTES(cols).
template <typename S, typename B>
void norm_block_grad(const Buffer<S>& r, const Buffer<B>& b, const Buffer<B>* gate, const Buffer<float>& w_after,
                     const Buffer<float>* w_before, const Buffer<float>& rstd, const Buffer<S>* dout,
                     const Buffer<B>* dy, const NormGrads<S, B>& to, Buffer<float>* work, const NormShape& n,
                     Context& ctx = Context::current()) {
  auto fits = [](const auto* v, int rows, int cols) { return !v || detail::holds(*v, rows, cols); };
  detail::require(detail::holds(r, n.rows, n.cols) && detail::holds(b, n.rows, n.cols) && fits(dout, n.rows, n.cols) &&
                      fits(dy, n.rows, n.cols) && fits(to.dx, n.rows, n.cols) && fits(to.db, n.rows, n.cols),
                  "norm_block_grad", "r, b, dout, dy, dx or db is smaller than rows x cols");
  detail::require(fits(gate, n.gates(), n.cols) && fits(to.dgate, n.gates(), n.cols), "norm_block_grad",
                  "gate or dgate is smaller than its rows x cols");
  detail::require(detail::holds(w_after, 1, n.cols) && fits(w_before, 1, n.cols) && fits(to.dw_after, 1, n.cols) &&
                      fits(to.dw_before, 1, n.cols),
                  "norm_block_grad", "w_after, w_before, dw_after or dw_before is shorter than a row");
  detail::require(detail::holds(rstd, 2, n.rows), "norm_block_grad", "rstd is smaller than 2 x rows");
  auto data = [](auto* v) { return v ? v->data() : nullptr; };
  ctx.check(miaie_norm_block_grad(ctx.get(), r.data(), b.data(), data(gate), w_after.data(), dy ? data(w_before) : nullptr,
                                  rstd.data(), data(dout), data(dy), data(to.dx), data(to.db), data(to.dgate),
                                  data(to.dw_after), data(to.dw_before), data(work), work ? work->bytes() : 0, n.rows,
                                  n.cols, n.cols, n.cols, n.rows_of_a_gate(), dtype_of(r.data()), dtype_of(b.data()),
                                  n.alpha));
}

// The gradient of norm_before, added to dout (nullable: 0).
template <typename S, typename B>
void norm_before_grad(const Buffer<S>& x, const Buffer<float>& w_before, const Buffer<float>& rstd,
                      const Buffer<S>* dout, const Buffer<B>& dy, Buffer<S>* dx, Buffer<float>* dw_before,
                      Buffer<float>* work, const NormShape& n, Context& ctx = Context::current()) {
  auto fits = [](const auto* v, int rows, int cols) { return !v || detail::holds(*v, rows, cols); };
  detail::require(detail::holds(x, n.rows, n.cols) && fits(dout, n.rows, n.cols) && detail::holds(dy, n.rows, n.cols) &&
                      fits(dx, n.rows, n.cols),
                  "norm_before_grad", "x, dout, dy or dx is smaller than rows x cols");
  detail::require(detail::holds(w_before, 1, n.cols) && fits(dw_before, 1, n.cols), "norm_before_grad",
                  "w_before or dw_before is shorter than a row");
  detail::require(detail::holds(rstd, 2, n.rows), "norm_before_grad", "rstd is smaller than 2 x rows");
  auto data = [](auto* v) { return v ? v->data() : nullptr; };
  ctx.check(miaie_norm_block_grad(ctx.get(), x.data(), nullptr, nullptr, nullptr, w_before.data(), rstd.data(), data(dout),
                                  dy.data(), data(dx), nullptr, nullptr, nullptr, data(dw_before), data(work),
                                  work ? work->bytes() : 0, n.rows, n.cols, n.cols, n.cols, n.rows, dtype_of(x.data()),
                                  dtype_of(dy.data()), 1.f));
}

// ---- 8-bit matrices with a scale for each block of 128, routing, experts ----

namespace detail {
inline size_t times(int count, size_t bytes) {
  require(bytes > 0 && count > 0 && bytes <= SIZE_MAX / (size_t)count, "Fp8Matrix", "no packed matrices have such sizes");
  return count * bytes;
}
}  // namespace detail

// `count` packed matrices (miaie.h) of rows x cols, one after another: block 1 or
// 128; count: the experts' matrices.
struct Fp8Matrix {
  Fp8Matrix(Context& ctx, int rows, int cols, int block = 1, int count = 1)
      : rows(rows), cols(cols), block(block), count(count), q(ctx, detail::times(count, miaie_fp8_q_bytes(rows, cols))),
        s(ctx, detail::times(count, miaie_fp8_s_bytes(rows, cols, block)) / 4) {}
  int rows, cols, block, count;
  Buffer<uint8_t> q;
  Buffer<float> s;
};

namespace detail {
inline bool is(const Fp8Matrix& m, int rows, int cols, int block, int count = 1) {
  return m.rows == rows && m.cols == cols && m.block == block && m.count == count;
}
inline bool is(const Fp8Matrix* m, int rows, int cols) { return !m || is(*m, rows, cols, 1); }
inline uint8_t* codes(Fp8Matrix* m) { return m ? m->q.data() : nullptr; }
inline float* scales(Fp8Matrix* m) { return m ? m->s.data() : nullptr; }
template <typename T>
T* data(const Buffer<T>* b) { return b ? b->data() : nullptr; }
}  // namespace detail

// Q = X packed along its rows (X dense, Q.rows x Q.cols).
template <typename T>
void quant_fp8(const Buffer<T>& X, Fp8Matrix& Q, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Q.rows, Q.cols) && Q.count == 1, "quant_fp8", "X is smaller than Q, or Q several matrices");
  ctx.check(miaie_quant_fp8(ctx.get(), X.data(), dtype_of(X.data()), Q.rows, Q.cols, Q.cols, Q.block, Q.q.data(), Q.s.data(),
                            nullptr, nullptr));
}

// Qt = the transpose of X packed along its rows (X dense, Qt.cols x Qt.rows).
template <typename T>
void quant_fp8_t(const Buffer<T>& X, Fp8Matrix& Qt, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Qt.cols, Qt.rows) && Qt.count == 1, "quant_fp8_t",
                  "X is smaller than Qt, or Qt several matrices");
  ctx.check(miaie_quant_fp8(ctx.get(), X.data(), dtype_of(X.data()), Qt.cols, Qt.rows, Qt.rows, Qt.block, nullptr, nullptr,
                            Qt.q.data(), Qt.s.data()));
}

// Both from one read of X.
template <typename T>
void quant_fp8_both(const Buffer<T>& X, Fp8Matrix& Q, Fp8Matrix& Qt, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Q.rows, Q.cols) && Q.count == 1, "quant_fp8_both",
                  "X is smaller than Q, or Q several matrices");
  detail::require(detail::is(Qt, Q.cols, Q.rows, Q.block), "quant_fp8_both", "Qt does not have the shape of Q's transpose");
  ctx.check(miaie_quant_fp8(ctx.get(), X.data(), dtype_of(X.data()), Q.rows, Q.cols, Q.cols, Q.block, Q.q.data(), Q.s.data(),
                            Qt.q.data(), Qt.s.data()));
}

// Matrix e of Q, and with Qt that of the transposes: the experts' weights.
template <typename T>
void quant_fp8_at(const Buffer<T>& X, Fp8Matrix& Q, int e, Fp8Matrix* Qt = nullptr, Context& ctx = Context::current()) {
  detail::require(detail::holds(X, Q.rows, Q.cols) && e >= 0 && e < Q.count, "quant_fp8_at", "X is smaller than Q, or Q has no such matrix");
  detail::require(!Qt || detail::is(*Qt, Q.cols, Q.rows, Q.block, Q.count), "quant_fp8_at",
                  "Qt does not have the shape of Q's transposes");
  ctx.check(miaie_quant_fp8(ctx.get(), X.data(), dtype_of(X.data()), Q.rows, Q.cols, Q.cols, Q.block,
                            Q.q.data() + e * (Q.q.size() / Q.count), Q.s.data() + e * (Q.s.size() / Q.count),
                            Qt ? Qt->q.data() + e * (Qt->q.size() / Qt->count) : nullptr,
                            Qt ? Qt->s.data() + e * (Qt->s.size() / Qt->count) : nullptr));
}

// Y = the values of Q.
template <typename T>
void dequant_fp8(const Fp8Matrix& Q, Buffer<T>& Y, Context& ctx = Context::current()) {
  detail::require(detail::holds(Y, Q.rows, Q.cols) && Q.count == 1, "dequant_fp8", "Y is smaller than Q, or Q several matrices");
  ctx.check(miaie_dequant_fp8(ctx.get(), Q.q.data(), Q.s.data(), Q.block, Y.data(), dtype_of(Y.data()), Q.rows, Q.cols, Q.cols));
}

// C = A . B^T (A M x K of block 1, B N x K of either block).
template <typename T>
void gemm_fp8(const Fp8Matrix& A, const Fp8Matrix& B, Buffer<T>& C, Context& ctx = Context::current()) {
  detail::require(A.block == 1 && A.count == 1 && B.count == 1, "gemm_fp8", "A has blocks of 128 rows, or A or B several matrices");
  detail::require(A.cols == B.cols, "gemm_fp8", "A and B have rows of different lengths");
  detail::require(detail::holds(C, A.rows, B.rows), "gemm_fp8", "C is smaller than A . B^T");
  ctx.check(miaie_gemm_fp8(ctx.get(), A.q.data(), A.s.data(), B.q.data(), B.s.data(), B.block, C.data(), dtype_of(C.data()),
                           A.rows, B.rows, A.cols, B.rows));
}

// How miaie_route_experts chooses.
struct Routing {
  int tokens, top_k, experts;
  int scoring = MIAIE_SOFTMAX, groups = 1, groups_kept = 1, group_top = 1;
  bool renormalize = true;
  float scale = 1.f;
};

// idx and w (tokens x top_k) from logits (tokens x experts, dense).
template <typename T>
void route_experts(const Buffer<T>& logits, const Buffer<float>* bias, Buffer<int32_t>& idx, Buffer<float>& w, const Routing& r,
                   Context& ctx = Context::current()) {
  detail::require(detail::holds(logits, r.tokens, r.experts) && (!bias || detail::holds(*bias, 1, r.experts)), "route_experts",
                  "logits is smaller than tokens x experts, or bias shorter than experts");
  detail::require(detail::holds(idx, r.tokens, r.top_k) && detail::holds(w, r.tokens, r.top_k), "route_experts",
                  "idx or w is smaller than tokens x top_k");
  ctx.check(miaie_route_experts(ctx.get(), logits.data(), dtype_of(logits.data()), detail::data(bias), idx.data(), w.data(),
                                r.tokens, r.top_k, r.experts, r.experts, r.scoring, r.groups, r.groups_kept, r.group_top,
                                r.renormalize ? 1 : 0, r.scale));
}

template <typename T>
void route_experts_grad(const Buffer<T>& logits, const Buffer<int32_t>& idx, const Buffer<float>& dw, Buffer<float>& dlogits,
                        const Routing& r, Context& ctx = Context::current()) {
  detail::require(detail::holds(logits, r.tokens, r.experts) && detail::holds(dlogits, r.tokens, r.experts),
                  "route_experts_grad", "logits or dlogits is smaller than tokens x experts");
  detail::require(detail::holds(idx, r.tokens, r.top_k) && detail::holds(dw, r.tokens, r.top_k), "route_experts_grad",
                  "idx or dw is smaller than tokens x top_k");
  ctx.check(miaie_route_experts_grad(ctx.get(), logits.data(), dtype_of(logits.data()), idx.data(), dw.data(), dlogits.data(),
                                     r.tokens, r.top_k, r.experts, r.experts, r.experts, r.scoring, r.renormalize ? 1 : 0,
                                     r.scale));
}

// Slots of a routing (miaie_experts_order); matrices over them have rows() rows.
struct ExpertsOrder {
  ExpertsOrder(Context& ctx, int tokens, int top_k, int experts)
      : tokens(tokens), top_k(top_k), experts(experts), order(ctx, miaie_experts_order_bytes(tokens, top_k, experts) / 4) {}
  int rows() const { return (int)miaie_experts_rows(tokens, top_k, experts); }
  int tokens, top_k, experts;
  Buffer<int32_t> order;
};

inline void experts_order(const Buffer<int32_t>& idx, ExpertsOrder& o, Context& ctx = Context::current()) {
  detail::require(detail::holds(idx, o.tokens, o.top_k), "experts_order", "idx is smaller than tokens x top_k");
  ctx.check(miaie_experts_order(ctx.get(), idx.data(), o.order.data(), o.tokens, o.top_k, o.experts));
}

namespace detail {
// Y and the result of one type, or fp32 and bf16
template <typename TY, typename T>
int slots_dtype(const Buffer<TY>&, const Buffer<T>& out) {
  constexpr bool wide = std::is_same_v<TY, float> && !std::is_same_v<T, float>;
  static_assert(wide || std::is_same_v<TY, T>, "Y has the result's type, or is fp32");
  return dtype_of(out.data()) | (wide ? MIAIE_F32_SLOTS : 0);
}
}  // namespace detail

// out[t] = sum over t's experts of w (H . W2^T), H = pack(silu(gate) up) of X . W1^T.
template <typename TY, typename T>
void experts_mlp_fp8(const ExpertsOrder& o, const Buffer<float>& w, const Fp8Matrix& X, const Fp8Matrix& W1, const Fp8Matrix& W2,
                     Fp8Matrix& H, Buffer<TY>& Y, Buffer<T>& out, Context& ctx = Context::current()) {
  detail::require(detail::is(X, o.tokens, X.cols, 1), "experts_mlp_fp8", "X is not the tokens' rows");
  detail::require(W1.rows == 2l * W2.cols && detail::is(W1, W1.rows, X.cols, 128, o.experts) &&
                      detail::is(W2, W2.rows, W2.cols, 128, o.experts),
                  "experts_mlp_fp8", "W1 and W2 are not matrices of each expert that fit X and each other");
  detail::require(detail::is(H, o.rows(), W2.cols, 1), "experts_mlp_fp8", "H does not have the slots' rows of F columns");
  detail::require(detail::holds(w, o.tokens, o.top_k) && detail::holds(Y, o.rows(), W2.rows) &&
                      detail::holds(out, o.tokens, W2.rows),
                  "experts_mlp_fp8", "w, Y or out is too small");
  ctx.check(miaie_experts_mlp_fp8(ctx.get(), o.order.data(), w.data(), X.q.data(), X.s.data(), W1.q.data(), W1.s.data(),
                                  W2.q.data(), W2.s.data(), H.q.data(), H.s.data(), Y.data(), out.data(),
                                  detail::slots_dtype(Y, out), o.tokens, o.top_k, o.experts, X.cols, W2.cols, W2.rows, W2.rows));
}

// C[slot] = A[slot] . B_e^T; with gather A has the tokens' rows.
template <typename T>
void experts_gemm_fp8(const ExpertsOrder& o, const Fp8Matrix& A, const Fp8Matrix& B, Buffer<T>& C, bool gather = false,
                      Context& ctx = Context::current()) {
  detail::require(detail::is(A, gather ? o.tokens : o.rows(), A.cols, 1), "experts_gemm_fp8",
                  gather ? "A is not the tokens' rows" : "A is not the slots' rows");
  detail::require(detail::is(B, B.rows, A.cols, 128, o.experts), "experts_gemm_fp8", "B is not a matrix of each expert that fits A");
  detail::require(detail::holds(C, o.rows(), B.rows), "experts_gemm_fp8", "C is smaller than the slots' rows");
  ctx.check(miaie_experts_gemm_fp8(ctx.get(), o.order.data(), A.q.data(), A.s.data(), B.q.data(), B.s.data(), C.data(),
                                   dtype_of(C.data()), o.tokens, o.top_k, o.experts, B.rows, A.cols, B.rows, gather ? 1 : 0));
}

// Conversions over slots: Q (rows() x cols) and / or Qt (its transpose), either NULL.
template <typename T>
void experts_quant_fp8(const ExpertsOrder& o, const Buffer<T>& X, const Buffer<float>* w, Fp8Matrix* Q, Fp8Matrix* Qt, int cols,
                       Context& ctx = Context::current()) {
  detail::require(detail::holds(X, o.tokens, cols) && (!w || detail::holds(*w, o.tokens, o.top_k)), "experts_quant_fp8",
                  "X or w is too small");
  detail::require(detail::is(Q, o.rows(), cols) && detail::is(Qt, cols, o.rows()), "experts_quant_fp8",
                  "Q or Qt does not have the slots' shape");
  ctx.check(miaie_experts_quant_fp8(ctx.get(), o.order.data(), X.data(), dtype_of(X.data()), detail::data(w), detail::codes(Q),
                                    detail::scales(Q), detail::codes(Qt), detail::scales(Qt), o.tokens, o.top_k, o.experts, cols,
                                    cols));
}

template <typename T>
void experts_swiglu_fp8(const ExpertsOrder& o, const Buffer<T>& GU, Fp8Matrix* Q, Fp8Matrix* Qt, int F,
                        Context& ctx = Context::current()) {
  detail::require(F < 1 || detail::holds(GU, 2 * o.rows(), F), "experts_swiglu_fp8", "GU is smaller than the slots' 2 F columns");
  detail::require(detail::is(Q, o.rows(), F) && detail::is(Qt, F, o.rows()), "experts_swiglu_fp8",
                  "Q or Qt does not have the slots' shape");
  ctx.check(miaie_experts_swiglu_fp8(ctx.get(), o.order.data(), GU.data(), dtype_of(GU.data()), detail::codes(Q), detail::scales(Q),
                                     detail::codes(Qt), detail::scales(Qt), o.tokens, o.top_k, o.experts, F, 2 * F));
}

template <typename T>
void experts_swiglu_grad_fp8(const ExpertsOrder& o, const Buffer<T>& GU, const Buffer<float>& dH, Fp8Matrix* Q, Fp8Matrix* Qt, int F,
                             Context& ctx = Context::current()) {
  detail::require(F < 1 || (detail::holds(GU, 2 * o.rows(), F) && detail::holds(dH, o.rows(), F)), "experts_swiglu_grad_fp8",
                  "GU or dH is smaller than the slots' columns");
  detail::require(detail::is(Q, o.rows(), 2 * F) && detail::is(Qt, 2 * F, o.rows()), "experts_swiglu_grad_fp8",
                  "Q or Qt does not have the slots' shape");
  ctx.check(miaie_experts_swiglu_grad_fp8(ctx.get(), o.order.data(), GU.data(), dtype_of(GU.data()), dH.data(), detail::codes(Q),
                                          detail::scales(Q), detail::codes(Qt), detail::scales(Qt), o.tokens, o.top_k, o.experts,
                                          F, 2 * F, F));
}

// C (experts x At.rows x Bt.rows): each expert's At . Bt^T over its slots.
template <typename T>
void experts_wgrad_fp8(const ExpertsOrder& o, const Fp8Matrix& At, const Fp8Matrix& Bt, Buffer<T>& C,
                       Context& ctx = Context::current()) {
  detail::require(detail::is(At, At.rows, o.rows(), 1) && detail::is(Bt, Bt.rows, o.rows(), 1), "experts_wgrad_fp8",
                  "At or Bt is not packed along the slots");
  detail::require(At.rows < 1 || Bt.rows < 1 || C.size() / (size_t)At.rows / (size_t)Bt.rows >= (size_t)o.experts,
                  "experts_wgrad_fp8", "C is smaller than the experts' matrices");
  ctx.check(miaie_experts_wgrad_fp8(ctx.get(), o.order.data(), At.q.data(), At.s.data(), Bt.q.data(), Bt.s.data(), C.data(),
                                    dtype_of(C.data()), o.tokens, o.top_k, o.experts, At.rows, Bt.rows, Bt.rows));
}

// out[t] = sum over t's slots of w Y[slot] (w NULL: of Y[slot]).
template <typename TY, typename T>
void experts_combine(const ExpertsOrder& o, const Buffer<TY>& Y, const Buffer<float>* w, Buffer<T>& out, int cols,
                     Context& ctx = Context::current()) {
  detail::require(detail::holds(Y, o.rows(), cols) && detail::holds(out, o.tokens, cols) &&
                      (!w || detail::holds(*w, o.tokens, o.top_k)),
                  "experts_combine", "Y, out or w is too small");
  ctx.check(miaie_experts_combine(ctx.get(), o.order.data(), Y.data(), detail::data(w), out.data(),
                                  detail::slots_dtype(Y, out), o.tokens, o.top_k, o.experts, cols, cols, cols));
}

template <typename TY, typename T>
void experts_combine_grad(const ExpertsOrder& o, const Buffer<TY>& Y, const Buffer<T>& dout, Buffer<float>& dw, int cols,
                          Context& ctx = Context::current()) {
  detail::require(detail::holds(Y, o.rows(), cols) && detail::holds(dout, o.tokens, cols) &&
                      detail::holds(dw, o.tokens, o.top_k),
                  "experts_combine_grad", "Y, dout or dw is too small");
  ctx.check(miaie_experts_combine_grad(ctx.get(), o.order.data(), Y.data(), dout.data(), dw.data(), detail::slots_dtype(Y, dout),
                                       o.tokens, o.top_k, o.experts, cols, cols, cols));
}

}  // namespace miaie

#endif  // MIAIE_HPP
