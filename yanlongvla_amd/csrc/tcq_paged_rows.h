// Which of the parts' rows a wave of the join takes. Rows are (token, query head) of `rows` tokens in all, Hq heads each; a sequence has n * Hq of them from token
// c0 on, and n may be 0 with c0 == rows (a sequence without rows behind the last one), so c0 * Hq alone is no row.
#pragma once
#include <stdint.h>

// row x of the sequence, -1: it has no such row
__host__ __device__ inline int64_t join_row(int64_t c0, int n, int Hq, int64_t x) { return x < (int64_t)n * Hq ? c0 * Hq + x : -1; }
