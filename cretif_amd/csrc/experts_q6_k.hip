// experts_q6_k.hip -- the grouped products of experts_gemm.hpp for Q6_K weights.
#include "experts_gemm.hpp"

namespace cri {
namespace dev {

template void expert_rows<kFmtQ6_K>(const ProductArgs&, bool, int, long, hipStream_t);
template void expert_few<kFmtQ6_K>(const ProductArgs&, bool, int, int, long, hipStream_t);
template void expert_token<kFmtQ6_K>(const ProductArgs&, const TokenArgs&, int, hipStream_t);

}  // namespace dev
}  // namespace cri
