// LayerNorm of token rows with an optional SiLU gate: forward and backward.
//
//   y = ((x - mean) rstd w + b) silu(gate),   mean, variance (biased) over the row
//
// A row stays in registers between the statistics and the output: 2^lg lanes take it in
// vectors of 16 bytes (2 or 1 elements where sizes or alignment ask for it), a whole
// workgroup takes rows of more than 64 lanes' worth.  A workgroup walks several rows with
// weight and bias in registers.  Bound by the bytes of the activations: 54.6 us for 401,408
// rows of 96 bf16, 231 MB at 4.2 TB/s (a large copy reaches 4.90); 6.8 us for 64 rows of 1024.
//
// Backward, with g = dy silu(gate), gw = g w:
//   dx = rstd (gw - mean(gw) - xhat mean(gw xhat)),  dw = sum g xhat,  db = sum g,
//   dgate = dy (xhat w + b) silu'(gate)
// with the statistics of the forward; the sums of dw and db stay in registers over a
// workgroup's rows and are joined by param_sum.  92.2 us for the same rows, 389 MB at 4.2 TB/s.
#include "param_sum.h"

namespace vh {
namespace {

struct NormArgs {
    const void *x, *gate, *dy;
    int64_t x_ts, gate_ts, dy_ts;   // element strides of the rows
    const float *weight, *bias;
    void *y, *dx, *dgate;
    float *mean, *rstd, *partial;
    int64_t rows;
    int32_t channels, lg;           // lanes of a row: 2^lg, 64 at most, or 256 (lg = 8)
    float eps;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    T raw[VEC];
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
    else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
    else raw[0] = *p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(raw[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    T raw[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) raw[i] = from_f32<T>(v[i]);
    if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(raw);
    else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
    else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(raw);
    else *p = raw[0];
}

// Sum over the lanes of a row; `slot` is one of the LDS rows that a workgroup uses in
// turn, so one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, int lg, float* slot) {
    v = ln_lane_sum(v, lg > 6 ? 6 : lg);
    if (lg > 6) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (slot[0] + slot[1]) + (slot[2] + slot[3]);
    }
    return v;
}

template <typename T, int VEC, int CPL>
__global__ __launch_bounds__(256) void row_norm_kernel(const NormArgs a) {
    __shared__ float slots[3][4];
    const int32_t lanes = 1 << a.lg, sub = threadIdx.x & (lanes - 1), slot = threadIdx.x >> a.lg;
    const int32_t per_block = 256 >> a.lg;
    float w[CPL][VEC], b[CPL][VEC];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int32_t c = (j * lanes + sub) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            w[j][i] = c < a.channels ? a.weight[c + i] : 0.f;
            b[j][i] = c < a.channels ? a.bias[c + i] : 0.f;
        }
    }
    const float inv = 1.f / static_cast<float>(a.channels);
    const T* gate = static_cast<const T*>(a.gate);
    // every workgroup's rows are whole steps, so all its lanes meet at the barriers
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_block; base < a.rows;
         base += static_cast<int64_t>(gridDim.x) * per_block) {
        const bool live = base + slot < a.rows;
        const int64_t row = live ? base + slot : a.rows - 1;
        const T* x = static_cast<const T*>(a.x) + row * a.x_ts;
        float v[CPL][VEC], z[CPL][VEC];
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = (j * lanes + sub) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[j][i] = z[j][i] = 0.f;
            if (c < a.channels) {
                load_vec<T, VEC>(x + c, v[j]);
                if (gate != nullptr) load_vec<T, VEC>(gate + row * a.gate_ts + c, z[j]);
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < CPL; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum += v[j][i];
        float mean = row_sum(sum, a.lg, slots[0]) * inv;
        // The rounded mean leaves the centred values a common offset (up to 2^-24 of the mean,
        // much beside a small spread): it is their mean, and taken off once more.
        float off = 0.f, sq = 0.f;
#pragma unroll
        for (int j = 0; j < CPL; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[j][i] = (j * lanes + sub) * VEC < a.channels ? v[j][i] - mean : 0.f;
                off += v[j][i];
                sq = fmaf(v[j][i], v[j][i], sq);
            }
        off = row_sum(off, a.lg, slots[1]) * inv;
        const float var = fmaxf(row_sum(sq, a.lg, slots[2]) * inv - off * off, 0.f);
        const float rstd = 1.f / sqrtf(var + a.eps);
        mean += off;
        if (live && sub == 0 && a.mean != nullptr) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        T* y = static_cast<T*>(a.y) + row * a.channels;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = (j * lanes + sub) * VEC;
            float out[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                out[i] = fmaf((v[j][i] - off) * rstd, w[j][i], b[j][i]);
                if (gate != nullptr) out[i] *= z[j][i] * sigmoid_fast(z[j][i]);
            }
            if (live && c < a.channels) store_vec<T, VEC>(y + c, out);
        }
    }
}

template <typename T, int VEC, int CPL>
__global__ __launch_bounds__(256) void row_norm_backward_kernel(const NormArgs a) {
    __shared__ float slots[3][4];
    __shared__ float joined[256 * VEC];
    const int32_t lanes = 1 << a.lg, sub = threadIdx.x & (lanes - 1), slot = threadIdx.x >> a.lg;
    const int32_t per_block = 256 >> a.lg;
    float w[CPL][VEC], b[CPL][VEC], dw[CPL][VEC], db[CPL][VEC];
#pragma unroll
    for (int j = 0; j < CPL; ++j) {
        const int32_t c = (j * lanes + sub) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            w[j][i] = c < a.channels ? a.weight[c + i] : 0.f;
            b[j][i] = c < a.channels ? a.bias[c + i] : 0.f;
            dw[j][i] = db[j][i] = 0.f;
        }
    }
    const float inv = 1.f / static_cast<float>(a.channels);
    const T* gate = static_cast<const T*>(a.gate);
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * per_block; base < a.rows;
         base += static_cast<int64_t>(gridDim.x) * per_block) {
        const bool live = base + slot < a.rows;
        const int64_t row = live ? base + slot : a.rows - 1;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float xhat[CPL][VEC], g[CPL][VEC], z[CPL][VEC];
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = (j * lanes + sub) * VEC;
#pragma unroll
            for (int i = 0; i < VEC; ++i) xhat[j][i] = g[j][i] = z[j][i] = 0.f;
            if (live && c < a.channels) {
                load_vec<T, VEC>(static_cast<const T*>(a.x) + row * a.x_ts + c, xhat[j]);
                load_vec<T, VEC>(static_cast<const T*>(a.dy) + row * a.dy_ts + c, g[j]);
                if (gate != nullptr) load_vec<T, VEC>(gate + row * a.gate_ts + c, z[j]);
            }
        }
        // The rounding of `mean` leaves the centred values a common offset, which the forward takes
        // off once more; here it is summed beside the other two sums and enters behind them.
        float off = 0.f, s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const bool mine = live && (j * lanes + sub) * VEC < a.channels;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                xhat[j][i] = mine ? (xhat[j][i] - mean) * rstd : 0.f;
                off += xhat[j][i];
                if (gate != nullptr) {   // z becomes dy silu'(z)
                    const float zv = z[j][i], sig = sigmoid_fast(zv);
                    z[j][i] = g[j][i] * (sig * fmaf(zv, 1.f - sig, 1.f));
                    g[j][i] *= zv * sig;
                }
                const float gw = g[j][i] * w[j][i];
                s1 += gw;
                s2 = fmaf(gw, xhat[j][i], s2);
            }
        }
        off = row_sum(off, a.lg, slots[0]) * inv;
        s1 = row_sum(s1, a.lg, slots[1]) * inv;
        s2 = row_sum(s2, a.lg, slots[2]) * inv - off * s1;
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            const int32_t c = (j * lanes + sub) * VEC;
            float out[VEC], dz[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float xh = xhat[j][i] - off;
                dw[j][i] = fmaf(g[j][i], xh, dw[j][i]);
                db[j][i] += g[j][i];
                out[i] = rstd * (fmaf(g[j][i], w[j][i], -fmaf(xh, s2, s1)));
                dz[i] = z[j][i] * fmaf(xh, w[j][i], b[j][i]);
            }
            if (live && c < a.channels) {
                store_vec<T, VEC>(static_cast<T*>(a.dx) + row * a.channels + c, out);
                if (gate != nullptr) store_vec<T, VEC>(static_cast<T*>(a.dgate) + row * a.channels + c, dz);
            }
        }
    }
    // the row slots' sums, in order
    float* to = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.channels;
    const int32_t width = lanes * VEC;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int j = 0; j < CPL; ++j) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VEC; ++i) joined[threadIdx.x * VEC + i] = q == 0 ? dw[j][i] : db[j][i];
            __syncthreads();
            for (int32_t m = threadIdx.x; m < width; m += 256) {
                float sum = 0.f;
                for (int32_t s = 0; s < per_block; ++s) sum += joined[s * width + m];
                const int32_t c = j * width + m;
                if (c < a.channels) to[q * a.channels + c] = sum;
            }
        }
}

constexpr int MAX_LANE_ELEMENTS = 32;
constexpr int64_t MAX_CHANNELS = 8192;

// How the lanes take a row: vector width, vectors a lane (a compiled count) and 2^lg lanes.
struct Plan {
    int vec, cpl, lg;
};
// Of the ways to lay a row over lanes, the one that leaves the fewest lanes idle, then the one
// with the most lanes.  The backward of 16-bit types may also take 8-byte vectors, where that
// gives a lane 16 elements or fewer: it keeps seven values an element, and 24 elements leave
// two waves a SIMD (with the parameter sums 96.8 us against 103.3 for 401,408 rows of 96 bf16,
// 84.9 against 101.2 for 50,000 of 768).  The forward, which keeps four, takes 53.2 us with 24
// elements of 96 and 62.0 with 12.  A whole
// workgroup takes a row, and pays barriers for it, only where a wave cannot hold it.
Plan make_plan(int64_t channels, int widest, bool backward) {
    static const int wide[] = {1, 2, 3, 4, 6, 8}, narrow[] = {1, 2, 4, 8, 16, 32};
    Plan best{widest, 0, 8};
    int64_t padded = 0;
    int most = 0;
    for (int vec : {widest, 4}) {
        if (vec > widest || (vec < widest && !backward)) continue;
        const int* counts = vec >= 4 ? wide : narrow;
        const int64_t vectors = (channels + vec - 1) / vec;
        for (int lg : {6, 5, 4, 3, 2, 8}) {
            if (lg == 8 && best.cpl != 0) continue;
            for (int k = 0; k < 6; ++k) {
                const int cpl = counts[k], elements = backward && cpl * vec > 16 ? cpl * vec : 16;
                if (cpl * vec > MAX_LANE_ELEMENTS || (static_cast<int64_t>(cpl) << lg) < vectors) continue;
                const int64_t total = (static_cast<int64_t>(cpl) << lg) * vec;
                if (best.cpl == 0 || total < padded || (total == padded && elements < most)) {
                    best = {vec, cpl, lg};
                    padded = total;
                    most = elements;
                }
                break;
            }
        }
    }
    return best;
}

template <typename T, int VEC>
int launch_cpl(bool backward, const NormArgs& a, int cpl, uint32_t grid, hipStream_t s) {
    auto go = [&](auto tag) -> int {
        constexpr int CPL = decltype(tag)::value;
        if (backward) row_norm_backward_kernel<T, VEC, CPL><<<grid, 256, 0, s>>>(a);
        else row_norm_kernel<T, VEC, CPL><<<grid, 256, 0, s>>>(a);
        return check_launch("row norm");
    };
    if (cpl == 1) return go(std::integral_constant<int, 1>{});
    if (cpl == 2) return go(std::integral_constant<int, 2>{});
    if (cpl == 4) return go(std::integral_constant<int, 4>{});
    if constexpr (VEC == 4 || VEC == 8) {
        if (cpl == 3) return go(std::integral_constant<int, 3>{});
    }
    if constexpr (VEC == 4) {
        if (cpl == 6) return go(std::integral_constant<int, 6>{});
    }
    if constexpr (VEC <= 4) {
        if (cpl == 8) return go(std::integral_constant<int, 8>{});
    }
    if constexpr (VEC <= 2) {
        if (cpl == 16) return go(std::integral_constant<int, 16>{});
    }
    if constexpr (VEC == 1) {
        if (cpl == 32) return go(std::integral_constant<int, 32>{});
    }
    return set_error(VH_ERR_SHAPE, "row norm: no kernel for %d vectors a lane", cpl);
}
int dispatch(bool backward, const NormArgs& a, int32_t io, const Plan& p, uint32_t grid, hipStream_t s) {
    auto by_vec = [&](auto t, auto widest) -> int {
        using T = decltype(t);
        if (p.vec == decltype(widest)::value) return launch_cpl<T, decltype(widest)::value>(backward, a, p.cpl, grid, s);
        if (p.vec == 4) return launch_cpl<T, 4>(backward, a, p.cpl, grid, s);
        if (p.vec == 2) return launch_cpl<T, 2>(backward, a, p.cpl, grid, s);
        return launch_cpl<T, 1>(backward, a, p.cpl, grid, s);
    };
    if (io == VH_DTYPE_F32) return by_vec(float{}, std::integral_constant<int, 4>{});
    if (io == VH_DTYPE_BF16) return by_vec(bf16_t{}, std::integral_constant<int, 8>{});
    return by_vec(f16_t{}, std::integral_constant<int, 8>{});
}

// Widest vector (16 bytes, two elements or one) that the sizes, addresses and strides allow.
int vector_of(int64_t channels, int e, std::initializer_list<const void*> pointers,
              std::initializer_list<int64_t> strides) {
    for (int vec : {16 / e, 2}) {
        const uintptr_t bytes = static_cast<uintptr_t>(vec * e);
        bool ok = channels % vec == 0;
        for (const void* p : pointers) ok = ok && reinterpret_cast<uintptr_t>(p) % bytes == 0;
        for (int64_t s : strides) ok = ok && s % vec == 0;
        if (ok) return vec;
    }
    return 1;
}

int check_rows(int32_t io, int64_t rows, int64_t channels) {
    VH_REQUIRE(valid_dtype(io), VH_ERR_DTYPE, "unsupported io_dtype %d", io);
    VH_REQUIRE(rows > 0 && channels > 0, VH_ERR_SHAPE, "row norm needs nonempty rows, got %lld x %lld", (long long)rows,
               (long long)channels);
    VH_REQUIRE(channels <= MAX_CHANNELS, VH_ERR_SHAPE, "row norm supports at most %lld channels, got %lld",
               (long long)MAX_CHANNELS, (long long)channels);
    return VH_OK;
}

// Workgroups, each walking rows with the parameters in registers.  The backward leaves a row of
// partial sums a workgroup: four row steps each, as long as that gives 511 of them (whose sum
// is one launch) and no more than 1024.
uint32_t forward_grid(int64_t rows, int lg) {
    const int64_t per = 256 >> lg, steps = (rows + per - 1) / per;
    return static_cast<uint32_t>(steps < 2048 ? steps : 2048);
}
uint32_t backward_grid(int64_t rows, int lg) {
    const int64_t per = 256 >> lg, steps = (rows + per - 1) / per;
    const int64_t blocks = (steps + 3) / 4 > 511 ? (steps + 3) / 4 : 511;
    const int64_t capped = blocks < 1024 ? blocks : 1024;
    return static_cast<uint32_t>(steps < capped ? steps : capped);
}

}  // namespace
}  // namespace vh

extern "C" {

int vh_gated_layernorm_forward(const void* x, int64_t x_row, const void* gate, int64_t gate_row, int32_t io_dtype,
                               const float* weight, const float* bias, void* y, float* mean, float* rstd, int64_t rows,
                               int64_t channels, float eps, void* stream) {
    using namespace vh;
    if (int rc = check_rows(io_dtype, rows, channels)) return rc;
    VH_REQUIRE(x != nullptr && weight != nullptr && bias != nullptr && y != nullptr, VH_ERR_ARG,
               "x, weight, bias and y must not be null");
    VH_REQUIRE((mean == nullptr) == (rstd == nullptr), VH_ERR_ARG, "mean and rstd must be given together");
    NormArgs a{};
    a.x = x;
    a.x_ts = x_row;
    a.gate = gate;
    a.gate_ts = gate_row;
    a.weight = weight;
    a.bias = bias;
    a.y = y;
    a.mean = mean;
    a.rstd = rstd;
    a.rows = rows;
    a.channels = static_cast<int32_t>(channels);
    a.eps = eps;
    const Plan p = make_plan(channels, vector_of(channels, dtype_bytes(io_dtype), {x, gate, y}, {x_row, gate_row}), false);
    a.lg = p.lg;
    return dispatch(false, a, io_dtype, p, forward_grid(rows, p.lg), static_cast<hipStream_t>(stream));
}

size_t vh_gated_layernorm_backward_workspace_bytes(int64_t rows, int64_t channels) {
    using namespace vh;
    if (rows <= 0 || channels <= 0) return 0;
    size_t most = 0;   // of the numbers of workgroups that a call may take
    for (int lg : {2, 3, 4, 5, 6, 8}) {
        const int64_t blocks = backward_grid(rows, lg);
        const size_t one = static_cast<size_t>(blocks) * 2 * channels * sizeof(float) +
                           param_sum_workspace_bytes(blocks, 2, channels);
        most = one > most ? one : most;
    }
    return most;
}

int vh_gated_layernorm_backward(const void* dy, int64_t dy_row, const void* x, int64_t x_row, const void* gate,
                                int64_t gate_row, int32_t io_dtype, const float* weight, const float* bias,
                                const float* mean, const float* rstd, void* dx, void* dgate, float* dweight,
                                float* dbias, int64_t rows, int64_t channels, void* workspace, size_t workspace_bytes,
                                void* stream) {
    using namespace vh;
    if (int rc = check_rows(io_dtype, rows, channels)) return rc;
    VH_REQUIRE(dy != nullptr && x != nullptr && weight != nullptr && bias != nullptr && mean != nullptr &&
                   rstd != nullptr && dx != nullptr && (gate == nullptr) == (dgate == nullptr),
               VH_ERR_ARG, "dy, x, weight, bias, mean, rstd and dx must be given, dgate exactly with a gate");
    const size_t need = vh_gated_layernorm_backward_workspace_bytes(rows, channels);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need, VH_ERR_WORKSPACE,
               "row norm backward needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
    NormArgs a{};
    a.dy = dy;
    a.dy_ts = dy_row;
    a.x = x;
    a.x_ts = x_row;
    a.gate = gate;
    a.gate_ts = gate_row;
    a.weight = weight;
    a.bias = bias;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.dx = dx;
    a.dgate = dgate;
    a.rows = rows;
    a.channels = static_cast<int32_t>(channels);
    a.partial = static_cast<float*>(workspace);
    const Plan p = make_plan(channels, vector_of(channels, dtype_bytes(io_dtype), {dy, x, gate, dx, dgate},
                                                 {dy_row, x_row, gate_row}), true);
    a.lg = p.lg;
    const uint32_t grid = backward_grid(rows, p.lg);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (int rc = dispatch(true, a, io_dtype, p, grid, s)) return rc;
    ParamSum sum{};
    sum.partial = a.partial;
    sum.rows = grid;
    sum.quantities = 2;
    sum.columns = a.channels;
    sum.out1 = dweight;
    sum.out2 = dbias;
    return launch_param_sum(sum, a.partial + sum.rows * 2 * channels, s);
}

}  // extern "C"
