// The paged attention kernels for bf16 pages.
#include "paged_attn.h"

namespace cljxla {

int64_t paged_attention_workspace_bf16(const PagedAttnParams& p) { return attention_workspace_of<__nv_bfloat16>(p); }
void launch_paged_attention_bf16(const PagedAttnParams& p, cudaStream_t s) { launch_attention_of<__nv_bfloat16>(p, s); }

}  // namespace cljxla
