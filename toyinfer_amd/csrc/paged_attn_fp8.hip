// Attention over the paged 8-bit cache (paged_attn.hpp).
#include "paged_attn.hpp"

namespace tiattn {

hipError_t launch_paged_attention_fp8(const PagedAttnArgs& a, hipStream_t stream) {
    return a.head.d == 64 ? launch_attn_t<64, 8>(a, stream) : launch_attn_t<128, 8>(a, stream);
}

}  // namespace tiattn
