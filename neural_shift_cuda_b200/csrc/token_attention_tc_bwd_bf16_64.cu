// Tensor-core token attention backward, bf16, head widths up to 64.
#include "token_attention_tc_bwd.cuh"

namespace nsc {
namespace tok {
template nsc_status tc_bwd_run<__nv_bfloat16, 64>(const Params&, const Grads&, const void*,
                                         cudaStream_t);
}  // namespace tok
}  // namespace nsc
