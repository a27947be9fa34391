// Tensor-core token attention forward, bf16, head widths up to 128.
#include "token_attention_tc_fwd.cuh"

namespace nsc {
namespace tok {
template nsc_status tc_fwd_run<__nv_bfloat16, 128>(const Params&, cudaStream_t);
}  // namespace tok
}  // namespace nsc
