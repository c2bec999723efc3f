// Attention over a paged cache of f8 codes (paged_attn_q8.inc.h).
#include "paged_attn_q8.inc.h"

namespace cdml {

int paged_attn_f8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_attn_q8<F8, false>(a, k, wide, st);
}

}  // namespace cdml
