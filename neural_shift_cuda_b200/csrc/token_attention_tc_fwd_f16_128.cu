// Tensor-core token attention forward, f16, head widths up to 128.
#include "token_attention_tc_fwd.cuh"

namespace nsc {
namespace tok {
template nsc_status tc_fwd_run<__half, 128>(const Params&, cudaStream_t);
}  // namespace tok
}  // namespace nsc
