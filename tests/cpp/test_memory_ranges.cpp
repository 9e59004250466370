// The arithmetic by which calls refuse buffers that share memory.
#include "check.h"

#include "csrc/memory_ranges.h"

using gern_detail::overlap;
using gern_detail::Rows;

namespace {
const void *at(uintptr_t x) {
    return reinterpret_cast<const void *>(x);
}
}  // namespace

CASE("ranges") {
    REQUIRE(overlap(at(100), 10, at(109), 5));
    REQUIRE(!overlap(at(100), 10, at(110), 5));
    REQUIRE(overlap(at(109), 5, at(100), 10));
    REQUIRE(!overlap(at(110), 5, at(100), 10));
    REQUIRE(overlap(at(100), 10, at(103), 1));
    REQUIRE(!overlap(at(100), 0, at(100), 10));
    REQUIRE(!overlap(at(100), 10, at(100), 0));
}

CASE("extent of rows") {
    REQUIRE((Rows{at(1000), 1, 64, 32}.bytes()) == 32);
    REQUIRE((Rows{at(1000), 3, 64, 32}.bytes()) == 160);
    REQUIRE((Rows{at(1000), 0, 64, 32}.bytes()) == 0);
    // products beyond 64 bits
    REQUIRE((Rows{at(1000), 0x7fffffff, INT64_MAX, 32}.bytes()) == INT64_MAX);
    REQUIRE((Rows{at(UINTPTR_MAX - 100), 0x7fffffff, INT64_MAX, 32}.bytes()) == 100);
}

CASE("rows and a range") {
    const Rows rows{at(1000), 3, 64, 32};
    REQUIRE(overlap(rows, at(1159), 10));
    REQUIRE(!overlap(rows, at(1160), 10));
    REQUIRE(!overlap(rows, at(990), 10));
    REQUIRE(overlap(rows, at(990), 11));
}

CASE("rows side by side in wider rows") {
    const Rows q{at(1000), 5, 96, 32};
    REQUIRE(overlap(q, q));
    REQUIRE(!overlap(q, Rows{at(1032), 5, 96, 64}));
    REQUIRE(overlap(q, Rows{at(1032), 5, 96, 65}));   // into the next row
    REQUIRE(overlap(q, Rows{at(1031), 5, 96, 8}));
    REQUIRE(!overlap(Rows{at(1032), 5, 96, 64}, q));  // the other way round
    REQUIRE(overlap(Rows{at(1031), 5, 96, 8}, q));
    REQUIRE(overlap(q, Rows{at(1096), 5, 96, 32}));   // the same columns a row further
    REQUIRE(overlap(Rows{at(1096), 5, 96, 32}, q));
    REQUIRE(!overlap(q, Rows{at(1128), 5, 96, 32}));  // other columns a row further
    REQUIRE(overlap(q, Rows{at(1032), 5, 128, 32}));  // other strides
    REQUIRE(!overlap(q, Rows{at(1416), 5, 128, 32})); // behind
    const Rows one{at(1000), 1, 96, 32};
    REQUIRE(overlap(one, Rows{at(1016), 1, 96, 32}));
    REQUIRE(!overlap(one, Rows{at(1032), 1, 96, 32}));
}

CHECK_MAIN()
