// Every index that the join of an attention's parts forms (join_row in yanlongvla_amd/csrc/tcq_paged_rows.h), on the host: for the rows of each
// sequence of a call, the statistics (2 a part) and outputs (D a part) that its waves read lie inside the workspace, every row is taken once, and
// rows of no sequence are not. Sequences without rows stand first, between the others and last, where their offset is the number of rows.
#define __host__
#define __device__
#include <stdio.h>

#include <algorithm>
#include <vector>

#include "tcq_paged_rows.h"

static int check(const std::vector<int>& cu, int rows, int most, int Hq, int S, int D, int per) {
    std::vector<int> taken((size_t)rows * Hq, 0);
    for (size_t b = 0; b + 1 < cu.size(); ++b) {
        const int c0 = std::max(0, std::min(cu[b], rows)), n = std::min(std::min(std::max(0, cu[b + 1] - cu[b]), most), rows - c0);
        const int64_t grid = ((int64_t)most * Hq + per - 1) / per;
        for (int64_t x = 0; x < grid * per; ++x) {
            const int64_t out = join_row(c0, n, Hq, x);
            if (out < 0) continue;
            if (out * S * 2 + 2 * S > (int64_t)rows * Hq * S * 2 || out * S * D + (int64_t)S * D > (int64_t)rows * Hq * S * D) return 1;
            ++taken[out];
        }
    }
    for (int r = 0; r < rows; ++r) {
        int in = 0;
        for (size_t b = 0; b + 1 < cu.size(); ++b) in += r >= cu[b] && r < std::min(cu[b + 1], cu[b] + most);
        for (int h = 0; h < Hq; ++h)
            if (taken[(size_t)r * Hq + h] != in) return 2;
    }
    return 0;
}

int main() {
    const std::vector<std::vector<int>> cus = {{0, 7}, {0, 0, 7}, {0, 7, 7}, {0, 3, 3, 7}, {0, 3, 7, 7, 7}, {2, 5, 5}, {0, 0, 0}, {7, 7}, {0, 5, 9}};
    for (auto& cu : cus)
        for (int most : {1, 4, 7})
            for (int Hq : {1, 3, 8})
                for (int S : {2, 9, 128})
                    for (int per : {1, 4}) {
                        const int e = check(cu, 7, most, Hq, S, 64, per);
                        if (e) {
                            printf("error %d: %zu sequences, most %d, heads %d, parts %d, rows a workgroup %d\n", e, cu.size() - 1, most, Hq, S, per);
                            return 1;
                        }
                    }
    printf("ok\n");
    return 0;
}
