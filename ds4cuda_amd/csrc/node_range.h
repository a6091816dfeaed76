// node_range.h — which of the packed nodes of a call two neighbouring starts name, whatever the starts hold. They come from
// device memory, unchecked, and the difference of two of them can pass 32 bits; of two that are brought into the
// call's nodes first it cannot.
#pragma once

#include <hip/hip_runtime.h>

namespace ds4hip {

__host__ __device__ inline int start_in(int start, int n_nodes) { return start < 0 ? 0 : start < n_nodes ? start : n_nodes; }

struct NodeRange {
    int first, n;   // first + n <= n_nodes
};
// None of them where the starts go back or name more than `most`.
__host__ __device__ inline NodeRange nodes_between(int a, int b, int n_nodes, int most) {
    const int first = start_in(a, n_nodes), n = start_in(b, n_nodes) - first;
    return {first, n > 0 && n <= most ? n : 0};
}

}  // namespace ds4hip
