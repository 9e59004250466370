// Host mirrors of the aggregates of gernels/serving/matvec4.h; the annotations are the
// general ones of annot/pieces.h.
#pragma once

#include "annot/pieces.h"

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

}  // namespace hip
}  // namespace gern
