// paged_attention.hip — flash_attention_paged_chunk.
#include "paged_attention.hpp"

namespace nfhip {

hipError_t launch_paged_chunk(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                              const void* k_pool, const void* v_pool, void* out, float* lse, const Workspace& ws,
                              hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  const paged::Operands o{q, k_pool, v_pool, out, lse};
  return lse ? paged::chunk_lse(t, pool, b, n_heads, o, ws, s) : paged::chunk_all<paged::kChunk>(t, pool, b, n_heads, o, ws, s);
}

}  // namespace nfhip
