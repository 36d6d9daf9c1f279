// gemm_blocks into f32.
#include "gemm_blocks.h"

namespace lg {
void launch_gemm_blocks_f32(lg_ctx* ctx, hipStream_t s, const GemmBlocksArgs& g) { launch_gemm_blocks_into<LG_DTYPE_F32>(ctx, s, g); }
}  // namespace lg
