// The paged attention kernels for f32 pages.
#include "paged_attn.h"

namespace cljxla {

int64_t paged_attention_workspace_f32(const PagedAttnParams& p) { return attention_workspace_of<float>(p); }
void launch_paged_attention_f32(const PagedAttnParams& p, cudaStream_t s) { launch_attention_of<float>(p, s); }

}  // namespace cljxla
