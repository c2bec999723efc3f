// Attention over a paged cache of f32 values (paged_attn.inc.h).
#include "paged_attn.inc.h"

namespace cdml {

int paged_attn_f32(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_attn<float>(a, k, wide, st);
}

}  // namespace cdml
