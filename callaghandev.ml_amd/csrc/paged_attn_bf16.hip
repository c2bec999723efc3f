// Attention over a paged cache of bf16 values (paged_attn.inc.h).
#include "paged_attn.inc.h"

namespace cdml {

int paged_attn_bf16(const PagedArgs &a, bool vec, bool tile, bool wide, hipStream_t st) {
  return paged_attn<__bf16>(a, vec, tile, wide, st);
}

}  // namespace cdml
