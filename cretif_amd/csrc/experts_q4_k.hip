// experts_q4_k.hip -- the grouped products of experts_gemm.hpp for Q4_K weights.
#include "experts_gemm.hpp"

namespace cri {
namespace dev {

template void expert_rows<kFmtQ4_K>(const ProductArgs&, bool, int, long, hipStream_t);
template void expert_few<kFmtQ4_K>(const ProductArgs&, bool, int, int, long, hipStream_t);
template void expert_token<kFmtQ4_K>(const ProductArgs&, const TokenArgs&, int, hipStream_t);

}  // namespace dev
}  // namespace cri
