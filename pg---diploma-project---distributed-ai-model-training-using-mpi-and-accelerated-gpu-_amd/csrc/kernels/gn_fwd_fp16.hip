// group norm forward, fp16 (groupnorm.h)
#include "../groupnorm.h"

void gn::fwd_fp16(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st) {
  if (a.q) launch<Fwd, _Float16, 8, true, false>(p, lds, a, st);
  else launch<Fwd, _Float16, 8, false, false>(p, lds, a, st);
}
