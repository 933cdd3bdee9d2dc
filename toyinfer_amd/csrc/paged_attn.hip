// Attention over the paged bf16 cache (paged_attn.hpp).
#include "paged_attn.hpp"

namespace tiattn {

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    return a.head.d == 64 ? launch_attn_t<64, 16>(a, stream) : launch_attn_t<128, 16>(a, stream);
}

}  // namespace tiattn
