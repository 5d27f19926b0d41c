// Column sums of partial parameter gradients, in a fixed order.
//
// A workgroup takes 64 columns, its 16 waves interleaved rows, four loads in flight each; LDS
// joins the waves.  With few columns and many rows the rows are also split over workgroups
// and a second launch of the same kernel adds the parts.  3 to 5 us a launch: mostly the
// launch's own time (1024 rows of 192 sums: 4.8 + 3.9 us).
#include "param_sum.h"

namespace vh {
namespace {

constexpr int WAVES = 16;

// Rows [blockIdx.y * part, ...) of the partials; LAST: writes the gradients, otherwise one
// row of sums a blockIdx.y.
template <bool LAST>
__global__ __launch_bounds__(64 * WAVES) void param_sum_kernel(ParamSum p, int64_t part, float* parts) {
    __shared__ float waves[WAVES][64];
    const int32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t width = static_cast<int64_t>(p.quantities) * p.columns;
    const int64_t m = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    const int64_t r0 = blockIdx.y * part;
    const int64_t r1 = r0 + part < p.rows ? r0 + part : p.rows;
    float sum = 0.f;
    if (m < width) {
        const float* at = p.partial + m;
        int64_t r = r0 + wave;
        for (; r + 3 * WAVES < r1; r += 4 * WAVES) {
            const float v0 = at[r * width], v1 = at[(r + WAVES) * width];
            const float v2 = at[(r + 2 * WAVES) * width], v3 = at[(r + 3 * WAVES) * width];
            sum += (v0 + v1) + (v2 + v3);
        }
        for (; r < r1; r += WAVES) sum += at[r * width];
    }
    waves[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || m >= width) return;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += waves[w][lane];
    if (!LAST) {
        parts[blockIdx.y * width + m] = sum;
        return;
    }
    const int32_t q = static_cast<int32_t>(m / p.columns);
    int32_t channel = static_cast<int32_t>(m - static_cast<int64_t>(q) * p.columns);
    if (p.group_tiles > 0) {
        const int32_t tile = channel >> 6, group = tile / p.group_tiles;
        const int32_t in_group = channel - group * p.group_tiles * 64;
        if (in_group >= p.group_channels) return;
        channel = group * p.group_channels + in_group;
    }
    if (q < p.per_channel) {
        if (p.out0 != nullptr) p.out0[static_cast<int64_t>(channel) * p.per_channel + q] = sum;
    } else if (q >= p.padded) {
        float* out = q == p.padded ? p.out1 : p.out2;
        if (out != nullptr) out[channel] = sum;
    }
}

// Workgroups that the rows of a 64-column strip are split over: about 512 in all, at least
// 256 rows each (16 loads a wave; a second launch costs as much as some 300 rows more).
int64_t splits(int64_t rows, int64_t width) {
    const int64_t strips = (width + 63) / 64;
    int64_t s = 512 / strips;
    if (s > rows / 256) s = rows / 256;
    return s < 2 ? 1 : s;
}

}  // namespace

size_t param_sum_workspace_bytes(int64_t rows, int64_t quantities, int64_t columns) {
    const int64_t s = splits(rows, quantities * columns);
    return s > 1 ? static_cast<size_t>(s) * quantities * columns * sizeof(float) : 0;
}

int launch_param_sum(const ParamSum& p, void* workspace, hipStream_t stream) {
    const int64_t width = static_cast<int64_t>(p.quantities) * p.columns;
    const uint32_t strips = static_cast<uint32_t>((width + 63) / 64);
    const int64_t s = splits(p.rows, width);
    if (s == 1) {
        param_sum_kernel<true><<<dim3(strips, 1), 64 * WAVES, 0, stream>>>(p, p.rows, nullptr);
        return check_launch("parameter gradient sum");
    }
    float* parts = static_cast<float*>(workspace);
    const int64_t part = (p.rows + s - 1) / s;
    param_sum_kernel<false><<<dim3(strips, static_cast<uint32_t>(s)), 64 * WAVES, 0, stream>>>(p, part, parts);
    if (int rc = check_launch("parameter gradient parts")) return rc;
    ParamSum last = p;
    last.partial = parts;
    last.rows = s;
    param_sum_kernel<true><<<dim3(strips, 1), 64 * WAVES, 0, stream>>>(last, s, nullptr);
    return check_launch("parameter gradient sum");
}

}  // namespace vh
