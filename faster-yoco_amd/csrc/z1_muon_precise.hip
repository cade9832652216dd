// Products on pairs of fp16, three for one.
#include "z1_muon_steps.h"

namespace z1muon {

int iterate_precise(Steps& a, int steps, const float* coefficients, Kind kind) { return iterate_of<true>(a, steps, coefficients, kind); }
void ways_precise(Plan& w, int* way) { ways_of<true>(w, way); }

}  // namespace z1muon
