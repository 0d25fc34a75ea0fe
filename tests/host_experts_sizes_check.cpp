// Run by tests/test_fp8_limits.py, without a GPU: sizes at the ends of the wrappers'
// ranges, and rows of slots of another type than the result, over the entry points that tests/host_experts_check.cpp records.
#define main shapes_that_fit
#include "host_experts_check.cpp"
#undef main

int main() {
  using namespace miaie;
  Context ctx;
  // sizes that no packed matrix has, or whose matrices have no size of 64 bits
  REFUSED("Fp8Matrix", Fp8Matrix(ctx, 0, 300));
  REFUSED("Fp8Matrix", Fp8Matrix(ctx, 300, 0));
  REFUSED("Fp8Matrix", Fp8Matrix(ctx, 5, 300, 1, 0));
  REFUSED("Fp8Matrix", Fp8Matrix(ctx, 5, 300, 1, -1));
  REFUSED("Fp8Matrix", Fp8Matrix(ctx, 1 << 30, 1 << 30, 1, 16));
  // gate and up of 2^30 columns of H are more rows than an int holds
  ExpertsOrder o(ctx, 10, 2, 8);
  Fp8Matrix X(ctx, 10, 40), W1(ctx, 256, 40, 128, 8), W2(ctx, 1, 1 << 30, 128, 8), H(ctx, o.rows(), 128);
  Buffer<float> w(ctx, 20), Y(ctx, o.rows()), out(ctx, 10);
  REFUSED("each expert", experts_mlp_fp8(o, w, X, W1, W2, H, Y, out));
  // fp32 rows of slots beside a bf16 result
  Fp8Matrix W(ctx, 256, 40, 128, 8), V(ctx, 30, 128, 128, 8);
  Buffer<float> Yf(ctx, o.rows() * 30), Yf1(ctx, o.rows() * 30 - 1);
  Buffer<uint16_t> result(ctx, 300);
  REACHES("mlp 17 10 2 8 40 128 30 30", P(o.order.data(), w.data(), M(X), M(W), M(V), M(H), Yf.data(), result.data()),
          experts_mlp_fp8(o, w, X, W, V, H, Yf, result));
  REACHES("combine 17 10 2 8 30 30 30", P(o.order.data(), Yf.data(), w.data(), result.data()), experts_combine(o, Yf, &w, result, 30));
  REACHES("combine_grad 17 10 2 8 30 30 30", P(o.order.data(), Yf.data(), result.data(), w.data()),
          experts_combine_grad(o, Yf, result, w, 30));
  REFUSED("too small", experts_mlp_fp8(o, w, X, W, V, H, Yf1, result));
  REFUSED("too small", experts_combine(o, Yf1, &w, result, 30));
  REFUSED("too small", experts_combine_grad(o, Yf1, result, w, 30));
  if (!failures) std::printf("ok\n");
  return failures ? 1 : 0;
}
