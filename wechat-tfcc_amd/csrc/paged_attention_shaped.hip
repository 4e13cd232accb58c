// Attention over a paged cache with shaped scores.
#include "paged_attention.hpp"

namespace tfcc_rocm {

void launch_shaped_attention(const AttentionArgs& a, int type, bool wide, const PagedAttentionPlan& plan, hipStream_t s) {
  launch_attention<true>(a, type, wide, plan, s);
}

}  // namespace tfcc_rocm
