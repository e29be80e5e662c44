// experts_fp16.hip -- the grouped products of experts_gemm.hpp for FP16 weights.
#include "experts_gemm.hpp"

namespace cri {
namespace dev {

template void expert_rows<kFmtF16>(const ProductArgs&, bool, int, long, hipStream_t);
template void expert_few<kFmtF16>(const ProductArgs&, bool, int, int, long, hipStream_t);
template void expert_token<kFmtF16>(const ProductArgs&, const TokenArgs&, int, hipStream_t);

}  // namespace dev
}  // namespace cri
