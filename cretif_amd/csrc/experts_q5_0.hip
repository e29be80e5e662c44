// experts_q5_0.hip -- the grouped products of experts_gemm.hpp for Q5_0 weights.
#include "experts_gemm.hpp"

namespace cri {
namespace dev {

template void expert_rows<kFmtQ5_0>(const ProductArgs&, bool, int, long, hipStream_t);
template void expert_few<kFmtQ5_0>(const ProductArgs&, bool, int, int, long, hipStream_t);
template void expert_token<kFmtQ5_0>(const ProductArgs&, const TokenArgs&, int, hipStream_t);

}  // namespace dev
}  // namespace cri
