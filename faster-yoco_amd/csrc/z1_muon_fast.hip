// Products on fp16 operands.
#include "z1_muon_steps.h"

namespace z1muon {

int iterate_fast(Steps& a, int steps, const float* coefficients, Kind kind) { return iterate_of<false>(a, steps, coefficients, kind); }
void ways_fast(Plan& w, int* way) { ways_of<false>(w, way); }

}  // namespace z1muon
