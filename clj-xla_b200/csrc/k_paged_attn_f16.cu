// The paged attention kernels for f16 pages.
#include "paged_attn.h"

namespace cljxla {

int64_t paged_attention_workspace_f16(const PagedAttnParams& p) { return attention_workspace_of<__half>(p); }
void launch_paged_attention_f16(const PagedAttnParams& p, cudaStream_t s) { launch_attention_of<__half>(p, s); }

}  // namespace cljxla
