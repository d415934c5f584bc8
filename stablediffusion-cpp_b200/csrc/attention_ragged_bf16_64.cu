// attention_ragged_bf16_64.cu - the tensor-core kernels of attention_ragged for bf16 operands
// and heads of up to 64 channels (one file per pair, so that they compile side by side).
#include "attention_ragged_tc.cuh"

namespace sdb {
namespace ragged {
template void launch_tc<64, __nv_bfloat16>(TcParams, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool);
}  // namespace ragged
}  // namespace sdb
