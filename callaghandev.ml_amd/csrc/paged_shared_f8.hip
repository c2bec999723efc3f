// Attention over shared prefixes in a paged cache of f8 codes (paged_attn_q8.inc.h).
#include "paged_attn_q8.inc.h"

namespace cdml {

int paged_shared_f8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_attn_q8<F8, true>(a, k, wide, st);
}

}  // namespace cdml
