// The many-rows kernel over the 8-bit cache (cbk_cache8_prompt.hip) as the dispatch in cbk_cache8_attn.hip sees it.
#pragma once
#include "cbk_cache8.h"
#include "cbk_cache_attn.h"

namespace cbk {
// What a query row is divided by.  Its products are summed in float32 only, so that an fp16 row is an operand as it is (top 65504 times 57344 in 256
// channels: 2^40), and a bf16 row from 2^-6 to 2^15.
template <bool BF>
__device__ inline float row_factor8(float top, float& down) {
  if constexpr (BF) return row_factor<15>(top, down);
  down = top < __builtin_inff() ? 1.f : __builtin_nanf("");
  return 1.f;
}
PromptPlan plan_prompt8(const DCache8&, const DRows&, int ratio, bool cut);
int launch_cache8_prompt(const PromptPlan&, const DCache8&, const DRows&, const AttnArgs&, hipStream_t);
}  // namespace cbk
