// The fused products of the gated feed-forward block, fp16 operands.
#include "fused_variant_make.cuh"

namespace rb200 {
const FusedVariant* fused_variants_f16(int* n) { return fused_ffn_table<2>(n); }
}  // namespace rb200
