// The fused products of the gated feed-forward block, bf16 operands.
#include "fused_variant_make.cuh"

namespace rb200 {
const FusedVariant* fused_variants_bf16(int* n) { return fused_ffn_table<1>(n); }
}  // namespace rb200
