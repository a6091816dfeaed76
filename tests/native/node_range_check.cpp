// Host check of the ranges of packed nodes (node_range.h) at starts of any value: every index that a walk reads or writes
// lies in the call's nodes, no start that goes on from one (plus a workgroup's width) passes 32 bits, and starts
// that are in order name what they say.
#include "node_range.h"

#include <climits>
#include <cstdio>
#include <vector>

using namespace ds4hip;

int main() {
    const int most = 1024, width = 1024;
    long long bad = 0, checked = 0;
    for (int n_nodes : {0, 1, 2, 9, 1023, 1024, 1025, 4096, 4097, 5000, 1 << 24}) {
        std::vector<int> starts = {0, 1, 2, 3, 8, 9, 10, 1023, 1024, 1025, 4096, 4097, 5000, 1 << 24, (1 << 24) + 1, 1 << 30};
        for (int i = 0; i < 2100; i += 7) {
            starts.push_back(INT_MAX - i);
            starts.push_back(INT_MIN + i);
            starts.push_back(-i);
        }
        for (int a : starts) {
            const long long s = start_in(a, n_nodes);
            bad += s < 0 || s > n_nodes || s + width > INT_MAX;
            bad += a >= 0 && a <= n_nodes && s != a;
            for (int b : starts) {
                const NodeRange r = nodes_between(a, b, n_nodes, most);
                bad += r.n < 0 || r.n > most || r.first < 0 || (long long)r.first + r.n > n_nodes;
                const bool in_order = 0 <= a && a <= b && b <= n_nodes;
                if (in_order) {
                    const long long n = (long long)b - a;
                    bad += r.first != a || r.n != (n <= most ? n : 0);
                }
                ++checked;
            }
        }
    }
    std::printf("%lld pairs, %lld wrong\n", checked, bad);
    return bad != 0;
}
