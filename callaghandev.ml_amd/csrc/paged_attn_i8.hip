// Attention over a paged cache of i8 codes (paged_attn_q8.inc.h).
#include "paged_attn_q8.inc.h"

namespace cdml {

int paged_attn_i8(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_attn_q8<I8, false>(a, k, wide, st);
}

}  // namespace cdml
