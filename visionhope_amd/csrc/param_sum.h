// Sums of per-workgroup partial parameter gradients (param_sum.hip).
#pragma once

#include "vh_common.h"

namespace vh {

// Partial gradients [rows, quantities, columns] FP32, and where their sums over the rows go:
// quantity q < per_channel of a column to out0[channel * per_channel + q], quantity `padded`
// (>= per_channel) to out1[channel], the one after it to out2[channel] (outputs may be null).  Columns are
// channels, or lanes of 64-channel tiles of groups (group_tiles > 0) whose last tile is padded.
struct ParamSum {
    const float* partial;
    int64_t rows;
    int32_t quantities, columns, per_channel, padded;
    int32_t group_channels, group_tiles;
    float *out0, *out1, *out2;
};

// Workspace of the sum (0: none) and the launch; the order of the sum depends on the sizes
// alone, so results repeat bit by bit.
size_t param_sum_workspace_bytes(int64_t rows, int64_t quantities, int64_t columns);
int launch_param_sum(const ParamSum& p, void* workspace, hipStream_t stream);

}  // namespace vh
