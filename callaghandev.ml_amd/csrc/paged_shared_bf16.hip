// Attention over shared prefixes in a paged cache of bf16 values (paged_attn.inc.h).
#include "paged_attn_q8.inc.h"

namespace cdml {

int paged_shared_bf16(const PagedArgs &args, const PagedKernels &k, bool wide, hipStream_t st) {
  // up to four rows straight from the cache (offsets inside 16 rows of a page fit 32 bits)
  const bool direct = k.span && wide && args.most_rows <= 4 && (long long)args.kv_heads * args.hd < (1 << 24);
  if (!direct) return paged_shared<__bf16>(args, k, wide, st);
  PagedArgs a = args;
  a.wide = true;
  const int rc = launch_codes<__bf16, true>(a, st);
  if (rc) return rc;
  return k.tile ? launch_tiles<__bf16, true>(a, wide, st) : CDML_OK;
}

}  // namespace cdml
