// The many-rows kernel over the 8-bit cache (cbk_cache8_prompt.hip) as the dispatch in cbk_cache8_attn.hip sees it.
#pragma once
#include "cbk_cache8.h"
#include "cbk_cache_attn.h"

namespace cbk {
PromptPlan plan_prompt8(const DCache8&, const DRows&, int ratio, bool cut);
int launch_cache8_prompt(const PromptPlan&, const DCache8&, const DRows&, const AttnArgs&, hipStream_t);
}  // namespace cbk
