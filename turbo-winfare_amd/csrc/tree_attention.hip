// Attention of drafted trees over the quantised cache: the rows of a tree see the tokens before it and, of its own
// nodes, those whose bits their masks have. The workgroups' kernel is that of dt_attend.h with the masks.
#include "dt_attend.h"

namespace tdt {

void launch_tree_attend(const AttnArgs& a, const AttnPlan& plan, uint32_t head_dim, int dtype, hipStream_t st) {
    if (dtype == TURBO_HIDDEN_F32) launch_dtype<true, true>(a, plan, head_dim, st);
    else launch_dtype<false, true>(a, plan, head_dim, st);
    check_hip(hipGetLastError(), "tree attention");
}

}  // namespace tdt
