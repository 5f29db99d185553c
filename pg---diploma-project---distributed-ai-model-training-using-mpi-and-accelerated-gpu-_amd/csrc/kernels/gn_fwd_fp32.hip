// group norm forward, fp32 (groupnorm.h)
#include "../groupnorm.h"

void gn::fwd_fp32(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st) {
  if (a.q) launch<Fwd, float, 4, true, false>(p, lds, a, st);
  else launch<Fwd, float, 4, false, false>(p, lds, a, st);
}
