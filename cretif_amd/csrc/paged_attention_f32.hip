// paged_attention_f32.hip -- paged attention over a cache of this type (a unit of its own: the three compile side by side).
#include "paged_attention.hpp"

namespace cri {
namespace dev {

void run_paged_attn_f32(const PagedAttnArgs& a, bool even, int blocks, hipStream_t stream) {
    run_paged_attn_type<kKvF32>(a, even, blocks, stream);
}

void run_paged_mixed_f32(const PagedAttnArgs& a, bool even, int own_blocks, hipStream_t stream) {
    run_paged_mixed_type<kKvF32>(a, even, own_blocks, stream);
}

}  // namespace dev
}  // namespace cri
