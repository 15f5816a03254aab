// The fused products of the Newton-Schulz iteration (fp16 operands; see orthogonal.cu).
#include "fused_variant_make.cuh"

namespace rb200 {

const FusedVariant* fused_variants_ortho(int* n) {
  static const FusedVariant t[] = {
      fused_make<kOpGramWide, 2, 256, 2>(), fused_make<kOpGramWide, 2, 128, 2>(),   fused_make<kOpGramWide, 1, 256, 2>(), fused_make<kOpGramWide, 1, 128, 2>(),
      fused_make<kOpGramTall, 2, 256, 2>(), fused_make<kOpGramTall, 2, 128, 2>(),   fused_make<kOpGramTall, 1, 256, 2>(), fused_make<kOpGramTall, 1, 128, 2>(),
      fused_make<kOpPoly, 2, 256, 2>(), fused_make<kOpPoly, 2, 128, 2>(),       fused_make<kOpPoly, 1, 256, 2>(),     fused_make<kOpPoly, 1, 128, 2>(),
      fused_make<kOpUpdateWide, 2, 256, 2>(), fused_make<kOpUpdateWide, 2, 128, 2>(), fused_make<kOpUpdateWide, 1, 128, 2>(),
      fused_make<kOpUpdateTall, 2, 256, 2>(), fused_make<kOpUpdateTall, 2, 128, 2>(), fused_make<kOpUpdateTall, 1, 128, 2>(),
  };
  *n = static_cast<int>(sizeof(t) / sizeof(t[0]));
  return t;
}

}  // namespace rb200
