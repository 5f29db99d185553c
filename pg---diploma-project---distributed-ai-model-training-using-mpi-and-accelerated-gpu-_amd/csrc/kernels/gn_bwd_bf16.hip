// group norm backward, bf16 (groupnorm.h)
#include "../groupnorm.h"

void gn::bwd_bf16(const Plan &p, size_t lds, const BwdArgs &a, hipStream_t st) {
  if (a.act == GN_SILU) {
    if (a.q) launch<Bwd, bf16_t, 8, true, true>(p, lds, a, st);
    else launch<Bwd, bf16_t, 8, false, true>(p, lds, a, st);
  } else {
    if (a.q) launch<Bwd, bf16_t, 8, true, false>(p, lds, a, st);
    else launch<Bwd, bf16_t, 8, false, false>(p, lds, a, st);
  }
}
