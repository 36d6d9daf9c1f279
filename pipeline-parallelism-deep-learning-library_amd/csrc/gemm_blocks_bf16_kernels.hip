// gemm_blocks into bf16.
#include "gemm_blocks.h"

namespace lg {
void launch_gemm_blocks_bf16(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) { launch_gemm_blocks_into<LG_DTYPE_BF16>(ctx, s, g); }
}  // namespace lg
