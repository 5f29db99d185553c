// group norm backward, fp32 (groupnorm.h)
#include "../groupnorm.h"

void gn::bwd_fp32(const Plan &p, size_t lds, const BwdArgs &a, hipStream_t st) {
  if (a.act == GN_SILU) {
    if (a.q) launch<Bwd, float, 4, true, true>(p, lds, a, st);
    else launch<Bwd, float, 4, false, true>(p, lds, a, st);
  } else {
    if (a.q) launch<Bwd, float, 4, true, false>(p, lds, a, st);
    else launch<Bwd, float, 4, false, false>(p, lds, a, st);
  }
}
