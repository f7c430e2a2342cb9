// The shapes of products of 8-bit integers in the C++ front end (tannic_hip_functions.hpp), over the stand-in of its types: one line each.
#include <algorithm>
#include <cstdio>

#include "tannic_hip_functions.hpp"

using namespace tannic;

static void print(Shape const& shape) {
    std::printf("[");
    for (size_t dim = 0; dim < shape.rank(); ++dim) std::printf(dim ? ",%zu" : "%zu", shape[dim]);
    std::printf("]\n");
}

int main() {
    using hip::ScaledProduct;
    print(ScaledProduct::shape({4, 8}, {8, 5}));
    print(ScaledProduct::shape({2, 3, 4, 8}, {8, 5}));
    print(ScaledProduct::shape({4, 8}, {3, 8, 5}));
    print(ScaledProduct::shape({2, 3, 4, 8}, {2, 3, 8, 5}));
    print(ScaledProduct::shape({0, 4, 8}, {8, 5}));
    print(ScaledProduct::shape({0, 4, 8}, {1, 8, 5}));
    print(ScaledProduct::shape({1, 4, 8}, {0, 8, 5}));
    print(ScaledProduct::shape({2, 1, 4, 8}, {0, 8, 5}));
    print(ScaledProduct::shape({4, 8}, {0, 3, 8, 5}));
    return 0;
}
