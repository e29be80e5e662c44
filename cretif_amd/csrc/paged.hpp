// paged.hpp -- what the kernels over a paged cache share: the cache's and the batch's description as the kernels
// take it, the place of a position in the pool, and the conversions of the cache's types.
//
// A position's row of a page is [n_kv_heads, head_dim]; page p starts `stride` elements after page p - 1.  A page
// table holds one row of max_pages page numbers per sequence.  What comes from device memory (tables, offsets,
// lengths) is never trusted with an address: a page number outside the pool or a position outside the table is
// left out by the append and read as page 0 by the attention, so no value there can reach past the buffers.
#pragma once

#include "common.hpp"
#include "internal.hpp"

namespace cri {
namespace dev {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// pos / page_size for 0 <= pos < 2^31: magic = floor(2^(31 + l) / d) + 1 with 2^l the least power of two that is
// not below d.  magic d exceeds 2^(31 + l) by at most d <= 2^l, so the quotient is exact for 31-bit numbers.
__device__ __forceinline__ int page_index(const PagePool& P, int pos) {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(pos)) * P.magic) >> P.shift);
}

template <int TYPE>
struct KvType;
template <>
struct KvType<kKvF32> {
    typedef float elem;
};
template <>
struct KvType<kKvF16> {
    typedef _Float16 elem;
};
template <>
struct KvType<kKvBF16> {
    typedef __bf16 elem;
};

}  // namespace dev
}  // namespace cri
