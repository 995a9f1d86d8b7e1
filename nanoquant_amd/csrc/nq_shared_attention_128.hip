// Attention over the 8-bit paged cache with shared first rows, heads of 128.
#include "nq_paged_attention.h"

namespace nq {
namespace paged {

template <>
int launch_shared_attention<128>(const SharedArgs& a, const AttnPlan& plan, int q_dtype, hipStream_t stream) {
    return launch_shared_for<128>(a, plan, q_dtype, stream);
}

}  // namespace paged
}  // namespace nq
