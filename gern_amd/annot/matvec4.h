// Host mirrors of the aggregates of gernels/serving/matvec4.h; the annotations are the
// general ones of annot/pieces.h.
#pragma once

#include "annot/pieces.h"

#include <cstddef>

namespace gern {
namespace hip {

struct Activations {
    const void *x;
    int64_t pitch, rows;
};
struct Weights4 {
    const void *codes, *scales, *zeros;
    int64_t n, k;
};
struct MatvecOut {
    void *y;
    int64_t pitch, columns;
};

// The sizes and last members' places that csrc/gernel_check.hip asks of gernels::.
static_assert(sizeof(Activations) == 24 && offsetof(Activations, rows) == 16);
static_assert(sizeof(Weights4) == 40 && offsetof(Weights4, k) == 32);
static_assert(sizeof(MatvecOut) == 24 && offsetof(MatvecOut, columns) == 16);

}  // namespace hip
}  // namespace gern
