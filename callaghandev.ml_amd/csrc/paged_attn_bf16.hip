// Attention over a paged cache of bf16 values (paged_attn.inc.h).
#include "paged_attn.inc.h"

namespace cdml {

int paged_attn_bf16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_attn<__bf16>(a, k, wide, st);
}

}  // namespace cdml
