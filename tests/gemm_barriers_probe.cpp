// The product's barriers (csrc/gemm_barriers.h) as a small C library for the
// CPU tests, for the narrow forms (8 or 6 stages, 2 accumulators) and the wide
// one (6 stages, 1).
#include "../mxfp8-quantizer_b200/csrc/gemm_barriers.h"

using namespace mxfp8;

namespace {
template <int STAGES, int ACC>
int place(int kind, int i) {
    using B = GemmBarriers<STAGES, ACC>;
    switch (kind) {
        case 0: return B::full(i);
        case 1: return B::empty(i);
        case 2: return B::acc_full(i);
        case 3: return B::acc_empty(i);
        case 4: return B::drained();
        default: return B::bytes;
    }
}
}  // namespace

extern "C" int probe_barrier(int stages, int acc, int kind, int i) {
    return acc == 1 ? place<6, 1>(kind, i) : stages == 6 ? place<6, 2>(kind, i) : place<8, 2>(kind, i);
}
