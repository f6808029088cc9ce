// bb_prompt_f16.hip — attention of several new tokens per sequence over an f16 cache: the kernels of bb_paged_prompt.h.
#include "bb_paged_prompt.h"

namespace bb {

hipError_t launch_prompt_f16(hipStream_t st, int wr, const PromptQuery& q, const PagedView& kv, const PagedSeqs& sq,
                            PromptPlan& pl) {
  return shape_f16(q.dt, pa_class(kv.hd), wr, [&](auto s) { return prompt_of(s, st, q, kv, sq, pl); });
}

}  // namespace bb
