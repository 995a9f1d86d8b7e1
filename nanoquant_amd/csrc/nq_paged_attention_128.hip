// Attention over the 8-bit paged cache, heads of 128.
#include "nq_paged_attention.h"

namespace nq {
namespace paged {

template <>
int launch_paged_attention<128>(const AttnArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream) {
    return launch_attention_for<128>(a, plan, q_dtype, stream);
}

}  // namespace paged
}  // namespace nq
