// dm_block_ffn_gate.hip — both projections of the gated feed-forward block, the activation and the product (dm_block_gemm.hip).
#include "dm_block_gemm.hip"

namespace dmb {
template int gemm_launch<bf16, false, false, EPI_GATE>(GemmArgs, int, hipStream_t);
template int gemm_launch<f16, false, false, EPI_GATE>(GemmArgs, int, hipStream_t);
template int gemm_launch<bf16, false, false, EPI_GATE_F32>(GemmArgs, int, hipStream_t);
}  // namespace dmb
