// Tensor-core token attention backward, f16, head widths up to 128.
#include "token_attention_tc_bwd.cuh"

namespace nsc {
namespace tok {
template nsc_status tc_bwd_run<__half, 128>(const Params&, const Grads&, const void*,
                                         cudaStream_t);
}  // namespace tok
}  // namespace nsc
