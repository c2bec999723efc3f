// Attention over shared prefixes in a paged cache of f16 values (paged_attn.inc.h).
#include "paged_attn.inc.h"

namespace cdml {

int paged_shared_f16(const PagedArgs &a, const PagedKernels &k, bool wide, hipStream_t st) {
  return paged_shared<_Float16>(a, k, wide, st);
}

}  // namespace cdml
