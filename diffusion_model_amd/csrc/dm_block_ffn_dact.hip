// dm_block_ffn_dact.hip — dh = dy Wd of the gated feed-forward block, and from it dg and du (dm_block_gemm.hip).
#include "dm_block_gemm.hip"

namespace dmb {
template int gemm_launch<bf16, false, true, EPI_DACT>(GemmArgs, int, hipStream_t);
template int gemm_launch<f16, false, true, EPI_DACT>(GemmArgs, int, hipStream_t);
template int gemm_launch<bf16, false, true, EPI_DACT_F32>(GemmArgs, int, hipStream_t);
}  // namespace dmb
