// bf16 instantiation of the shared-prefix attention (prefix_attn.h).
#include "prefix_attn.h"

namespace hpmn {

template int prefix_attn_type<bf16_t>(const HpmnPrefixAttn &a, AttnPlan &p, hipStream_t st);

}  // namespace hpmn
