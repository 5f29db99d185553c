// group norm forward, bf16 (groupnorm.h)
#include "../groupnorm.h"

void gn::fwd_bf16(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st) {
  if (a.q) launch<Fwd, bf16_t, 8, true, false>(p, lds, a, st);
  else launch<Fwd, bf16_t, 8, false, false>(p, lds, a, st);
}
