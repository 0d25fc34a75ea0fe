// Run by tests/test_fp8_limits.py, without a GPU: sizes at the ends of the wrappers'
// ranges, over the entry points that tests/host_experts_check.cpp records.
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
  if (!failures) std::printf("ok\n");
  return failures ? 1 : 0;
}
