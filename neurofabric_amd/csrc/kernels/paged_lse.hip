// paged_lse.hip — flash_attention_paged_chunk with its rows' log-sum-exp: the same
// kernels, in a translation unit of their own.
#include "paged_attention.hpp"

namespace nfk {
namespace paged {

hipError_t chunk_lse(nfhip::EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const Operands& o,
                     const nfhip::Workspace& ws, hipStream_t s) {
  return chunk_all<kLse>(t, pool, b, n_heads, o, ws, s);
}

}  // namespace paged
}  // namespace nfk
