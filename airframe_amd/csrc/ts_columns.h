// ts_columns.h -- the columns (token, head) of a chunk as operands of the matrix cores: written once by the window
// walk (ts_shared.hip), read by the sums over columns (ts_weigh.hip).
#pragma once
#include "ts_window.h"

namespace ts {

constexpr int kColBlk = 32;  // columns of one block

// One block: rotated q's high halves [k-step][lane], its low terms [group of 4 k-steps][term][3][lane][8 bytes], then
// each column's scale back of q (over kSkUnit) and the log2 sum of its softmax.  Columns past the last hold zeros.
template <int HD>
struct ColBlock {
    half8 hi[HD / 16][64];
    uint64_t lo[HD / 64][2][3][64];
    float back[kColBlk], lse[kColBlk];
};

}  // namespace ts
