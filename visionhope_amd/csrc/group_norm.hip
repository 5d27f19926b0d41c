// Group norm of channels-last maps [B, P pixels, C] with an activation: forward and backward.
//
//   z = (x - mean) rstd w + b,  y = f(z),  mean and variance (biased) over a group's channels and
//   all pixels of an image; f the identity, SiLU or the exact GELU
//
// Backward, with dz = dy f'(z), xhat = (x - mean) rstd, n values a group:
//   db = sum dz,  dw = sum dz xhat  (over images and pixels),
//   dx = rstd (w dz - (s1 + xhat s2) / n),  s1 = sum w dz,  s2 = sum w dz xhat  over the group
//
// Where a workgroup's registers hold a bundle of an image's groups, one launch reads the map once
// (both directions).  Larger maps take two passes: partial sums of slabs of pixels, then the outputs,
// whose workgroups join their image's slabs first.  128 x 56 x 56 x 96 bf16 with GELU: 17 + 32 us forward
// (231 MB at 4.7 TB/s), 41 + 40 + 9 us backward, bound by the vector unit (33 instructions a value and
// pass: the activation's slope is formed twice).  32 x 14 x 14 x 448: 6.7 and 9 + 4 us.
//
// Statistics of slabs: a thread takes its values in runs of about 32 from registers, each run's squares
// centred about the run's own rounded mean, whose rest is summed beside them; runs, threads and slabs are
// joined by their means and centred squares in FP64.  No long sum is of squares about a value that may
// stand far from the others: about a thread's first value instead, 10^4 beside a spread of one, rstd was
// off by 2.5e-4 at 2048 x 96 x 96 x 16 (and the statistics took 15 us where they take 17).  Values of a
// map in registers are centred about their rounded mean in the same way.  Either way the mean is kept as a
// sum of two floats: an offset large beside the spread loses nothing.
#include <algorithm>

#include "param_sum.h"

namespace vh {
namespace {

constexpr int GN_NONE = 0, GN_SILU = 1, GN_GELU = 2;
// Slabs of an image, each a workgroup for every bundle; a workgroup of the second pass joins them all.  8 x
// 128 x 128 x 96 bf16 takes 23.7 us forward (64 slabs: 24.4, 256: 25.1); one or two large maps would be
// faster with more (1 x 512 x 512 x 96: 93 us, with 512 slabs 43).
constexpr int64_t GN_MAX_SLABS = 128;
constexpr int64_t GN_MAX_GROUP = 1024;    // channels of a group: a workgroup's threads
constexpr int GN_RESIDENT = 512;          // threads, at most, that hold a map in registers

struct GNArgs {
    const void *x, *dy;
    const float *weight, *bias;
    void *y, *dx;
    float* stats;        // [3, B, G]: mean, its rest, rstd
    double* partial;     // [B, slabs, G, 2]: mean and centred squares of a slab's group
    float* sums;         // [B, slabs, 2, C]: of dz xhat and of dz
    float* group_sums;   // [B, slabs, G, 2]: s1, s2
    int32_t images, pixels, channels, groups, per;   // per: channels of a group
    int32_t bundle, bundles;                         // groups of a workgroup; workgroups for all groups
    int32_t slabs, slab;                             // slab: its pixels
    int32_t lg, slabs_lg;                            // 2^lg lanes join a group's threads (or its slabs)
    int32_t activation;
    float eps;
};

template <typename T, int VEC>
__device__ __forceinline__ void gn_load(const T* p, float (&v)[VEC]) {
    if constexpr (VEC * sizeof(T) == 16) {
        if constexpr (sizeof(T) == 4) {
            const float4 r = *reinterpret_cast<const float4*>(p);
            v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w;
        } else {
            load8<T>(p, v);
        }
    } else {
        T raw[VEC];
        if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(raw) = *reinterpret_cast<const uint2*>(p);
        else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(raw) = *reinterpret_cast<const uint32_t*>(p);
        else raw[0] = *p;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = to_f32(raw[i]);
    }
}
template <typename T, int VEC>
__device__ __forceinline__ void gn_store(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        store8<T>(p, v);
    } else {
        T raw[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) raw[i] = from_f32<T>(v[i]);
        if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(raw);
        else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(raw);
        else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(raw);
        else *p = raw[0];
    }
}

// Phi(-a) for a >= 0 as t P(t) exp(-a^2 / 2), t = 1 / (1 + 0.28 a): Mills' ratio is smooth in t, and P
// (degree 8, our minimax fit, coefficients rounded to FP32) is within 1.2e-7 of it relatively up to a = 40
// (behind 14.5 the exponential is zero).  `bell` is exp(-a^2 / 2), which the derivative needs as well.  The
// 8e-6 of gelu_fast would show in the parameters' gradients, FP32 sums, and turns the rounding of
// 0.07 % of bf16 and 0.45 % of FP16 outputs (the output pass of 128 x 56 x 56 x 96 takes 33 us, 29 with it).
__device__ __forceinline__ float gn_tail(float a, float& bell) {
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.28f, 1.f));
    bell = __builtin_amdgcn_exp2f(-0.72134752044448170f * a * a);
    float p = 0.025926996022462845f;
    p = fmaf(p, t, -0.09835107624530792f);
    p = fmaf(p, t, 0.10011325776576996f);
    p = fmaf(p, t, -0.013008116744458675f);
    p = fmaf(p, t, 0.07595551759004593f);
    p = fmaf(p, t, 0.08275416493415833f);
    p = fmaf(p, t, 0.10321440547704697f);
    p = fmaf(p, t, 0.11169081926345825f);
    p = fmaf(p, t, 0.11170406639575958f);
    return p * t * bell;
}
template <int ACT>
__device__ __forceinline__ float gn_activate(float z) {
    if constexpr (ACT == GN_NONE) return z;
    if constexpr (ACT == GN_SILU) return z * sigmoid_fast(z);
    float bell;
    const float a = fabsf(z), tail = gn_tail(a, bell);
    return fmaf(-a, tail, fmaxf(z, 0.f));
}
template <int ACT>
__device__ __forceinline__ float gn_slope(float z) {
    if constexpr (ACT == GN_NONE) return 1.f;
    if constexpr (ACT == GN_SILU) {
        const float s = sigmoid_fast(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    float bell;
    const float tail = gn_tail(fabsf(z), bell);
    return fmaf(z * 0.398942280401432678f, bell, z < 0.f ? tail : 1.f - tail);
}
// Runs a loop over values with the activation a compiled choice.
template <typename F>
__device__ __forceinline__ void gn_with(int32_t activation, F&& loop) {
    if (activation == GN_NONE) loop(std::integral_constant<int, GN_NONE>{});
    else if (activation == GN_SILU) loop(std::integral_constant<int, GN_SILU>{});
    else loop(std::integral_constant<int, GN_GELU>{});
}

__device__ __forceinline__ double gn_lane_sum(double v, int32_t lg) {
    for (int32_t m = 1; m < (1 << lg); m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// (x - mean) rstd: centred first, so that a constant map far from zero comes out as zeros, then scaled
// and rid of the mean's rest at once.
struct GNCentre {
    float mean, rstd, rest;
    __device__ __forceinline__ GNCentre(float mean_, float rest_, float rstd_) : mean(mean_), rstd(rstd_), rest(-rest_ * rstd_) {}
    __device__ __forceinline__ float operator()(float v) const { return fmaf(v - mean, rstd, rest); }
};

// A thread's place: `vector` of the bundle's vectors in a pixel, pixels `row`, row + rows, ... of
// a slab; threads behind the last full row are idle.
struct GNPlace {
    int32_t vectors, rows, vector, row, channel, group;   // channel: its first; group: within the bundle
    int32_t groups;                                       // of this bundle
    int32_t first_pixel, pixels;                          // of the slab
    int32_t entry, entries;                               // of its group's threads, which stand side by side in LDS
    int32_t image, bundle, slab;
    bool live;
};
template <int VEC>
__device__ __forceinline__ GNPlace gn_place(const GNArgs& a) {
    GNPlace p;
    const uint32_t rest = blockIdx.x / static_cast<uint32_t>(a.slabs);
    p.slab = static_cast<int32_t>(blockIdx.x - rest * a.slabs);
    p.image = static_cast<int32_t>(rest / static_cast<uint32_t>(a.bundles));
    p.bundle = static_cast<int32_t>(rest) - p.image * a.bundles;
    const int32_t first = p.bundle * a.bundle;
    p.groups = a.groups - first < a.bundle ? a.groups - first : a.bundle;
    p.vectors = p.groups * a.per / VEC;
    p.rows = static_cast<int32_t>(blockDim.x) / p.vectors;
    p.row = static_cast<int32_t>(threadIdx.x) / p.vectors;
    p.vector = static_cast<int32_t>(threadIdx.x) - p.row * p.vectors;
    p.live = p.row < p.rows;
    p.channel = first * a.per + p.vector * VEC;
    p.group = p.vector * VEC / a.per;
    p.first_pixel = p.slab * a.slab;
    p.pixels = a.pixels - p.first_pixel < a.slab ? a.pixels - p.first_pixel : a.slab;
    const int32_t each = a.per / VEC, rows = p.pixels < p.rows ? p.pixels : p.rows;
    p.entries = each * rows;
    p.entry = p.group * p.entries + p.row * each + (p.vector - p.group * each);
    return p;
}

// A vector as loaded, in whole words; unpacked when it is used.
template <typename T, int VEC>
struct GNRaw {
    static constexpr int words = VEC * sizeof(T) < 4 ? 1 : VEC * sizeof(T) / 4;
    uint32_t w[words];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (words == 4) {
            const uint4 r = *reinterpret_cast<const uint4*>(p);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else if constexpr (words == 2) {
            const uint2 r = *reinterpret_cast<const uint2*>(p);
            w[0] = r.x; w[1] = r.y;
        } else if constexpr (VEC * sizeof(T) == 4) {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            w[0] = p->bits;
        }
    }
    __device__ __forceinline__ void unpack(float (&v)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(w[j]);
            else v[j] = to_f32(T{static_cast<uint16_t>(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu)});
        }
    }
    // What follows is computed from the words again: values of other places in the code are not carried
    // here in registers.
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < words; ++i) asm volatile("" : "+v"(w[i]));
    }
};

// Sums of one slab of one image: a group's mean and centred squares.
template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_stats_kernel(const GNArgs a) {
    __shared__ double means[1024];
    __shared__ float squares[1024], counts[1024];
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, slab = p.slab;
    const int64_t image = p.image;
    if (p.live && p.row < p.pixels) {
        constexpr int RUN = VEC >= 4 ? 32 / VEC : 8;   // vectors
        const T* at = static_cast<const T*>(a.x) + (image * a.pixels + p.first_pixel) * a.channels + p.channel;
        double mean = 0.0, centred = 0.0;
        float n = 0.f;
        for (int32_t i = p.row; i < p.pixels; i += RUN * p.rows) {
            GNRaw<T, VEC> raw[RUN];
#pragma unroll
            for (int k = 0; k < RUN; ++k)
                if (i + k * p.rows < p.pixels) raw[k].load(at + static_cast<int64_t>(i + k * p.rows) * a.channels);
            float sum = 0.f, count = 0.f;
#pragma unroll
            for (int k = 0; k < RUN; ++k)
                if (i + k * p.rows < p.pixels) {
                    float v[VEC];
                    raw[k].unpack(v);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum += v[j];
                    count += VEC;
                }
            const float about = sum / count;
            float off = 0.f, square = 0.f;
#pragma unroll
            for (int k = 0; k < RUN; ++k)
                if (i + k * p.rows < p.pixels) {
                    float v[VEC];
                    raw[k].unpack(v);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float d = v[j] - about;
                        off += d;
                        square = fmaf(d, d, square);
                    }
                }
            const float rest = off / count, share = count / (n + count);
            const double d = static_cast<double>(about) + static_cast<double>(rest) - mean;
            mean = fma(d, static_cast<double>(share), mean);
            centred += fma(d * d, static_cast<double>(n * share), static_cast<double>(fmaxf(fmaf(-off, rest, square), 0.f)));
            n += count;
        }
        means[p.entry] = mean;
        squares[p.entry] = static_cast<float>(centred);
        counts[p.entry] = n;
    }
    __syncthreads();
    const int32_t lanes = 1 << a.lg, sub = static_cast<int32_t>(threadIdx.x) & (lanes - 1);
    const double inv = 1.0 / (static_cast<double>(p.pixels) * a.per);
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> a.lg; g < p.groups; g += static_cast<int32_t>(blockDim.x) >> a.lg) {
        double total = 0.0, centred = 0.0;
        for (int32_t e = g * p.entries + sub; e < (g + 1) * p.entries; e += lanes) total = fma(means[e], static_cast<double>(counts[e]), total);
        const double mean = gn_lane_sum(total, a.lg) * inv;
        for (int32_t e = g * p.entries + sub; e < (g + 1) * p.entries; e += lanes) {
            const double d = means[e] - mean;
            centred += fma(d * d, static_cast<double>(counts[e]), static_cast<double>(squares[e]));
        }
        centred = gn_lane_sum(centred, a.lg);
        if (sub == 0) {
            double* to = a.partial + ((image * a.slabs + slab) * a.groups + bundle * a.bundle + g) * 2;
            to[0] = mean;
            to[1] = centred;
        }
    }
}

// Mean (two floats) and rstd of the bundle's groups from the slabs, in LDS [3][1024].
__device__ __forceinline__ void gn_join(const GNArgs& a, const GNPlace& p, int32_t bundle, int64_t image, float* out) {
    const int32_t lanes = 1 << a.slabs_lg, slab = static_cast<int32_t>(threadIdx.x) & (lanes - 1);
    const double inv = 1.0 / (static_cast<double>(a.pixels) * a.per);
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> a.slabs_lg; g < p.groups; g += static_cast<int32_t>(blockDim.x) >> a.slabs_lg) {
        const double* from = a.partial + (image * a.slabs * a.groups + bundle * a.bundle + g) * 2;
        const int64_t step = static_cast<int64_t>(a.groups) * 2;
        auto count = [&](int32_t i) {
            const int32_t left = a.pixels - i * a.slab;
            return static_cast<double>(left < a.slab ? left : a.slab) * a.per;
        };
        double total = 0.0, var = 0.0;
        for (int32_t i = slab; i < a.slabs; i += lanes) total = fma(from[i * step], count(i), total);
        const double all = gn_lane_sum(total, a.slabs_lg) * inv;
        for (int32_t i = slab; i < a.slabs; i += lanes) {
            const double d = from[i * step] - all;
            var += fma(d * d, count(i), from[i * step + 1]);
        }
        var = gn_lane_sum(var, a.slabs_lg) * inv;
        if (slab == 0) {
            const float high = static_cast<float>(all);
            out[g] = high;
            out[1024 + g] = static_cast<float>(all - static_cast<double>(high));
            out[2048 + g] = 1.f / sqrtf(static_cast<float>(var) + a.eps);
        }
    }
    __syncthreads();
}

template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_apply_kernel(const GNArgs a) {
    __shared__ float stats[3 * 1024];
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, slab = p.slab;
    const int64_t image = p.image;
    gn_join(a, p, bundle, image, stats);
    if (slab == 0 && a.stats != nullptr) {
        const int64_t all = static_cast<int64_t>(a.images) * a.groups, at = image * a.groups + bundle * a.bundle;
        for (int32_t g = static_cast<int32_t>(threadIdx.x); g < p.groups; g += static_cast<int32_t>(blockDim.x))
#pragma unroll
            for (int q = 0; q < 3; ++q) a.stats[q * all + at + g] = stats[q * 1024 + g];
    }
    if (!p.live) return;
    const GNCentre centre(stats[p.group], stats[1024 + p.group], stats[2048 + p.group]);
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        w[j] = a.weight[p.channel + j];
        b[j] = a.bias[p.channel + j];
    }
    const int64_t base = (image * a.pixels + p.first_pixel) * a.channels + p.channel;
    const T* x = static_cast<const T*>(a.x) + base;
    T* y = static_cast<T*>(a.y) + base;
    gn_with(a.activation, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll 2
        for (int32_t i = p.row; i < p.pixels; i += p.rows) {
            float v[VEC];
            gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = gn_activate<ACT>(fmaf(centre(v[j]), w[j], b[j]));
            gn_store<T, VEC>(y + static_cast<int64_t>(i) * a.channels, v);
        }
    });
}

// Sums over the rows of threads of each channel, in `parts` [rows][channels]: to `out`, and times the
// weight to `weighted`.
__device__ __forceinline__ void gn_channel_sums(const float* parts, const GNPlace& p, int32_t channels, float* out,
                                                float* weighted, const float* weight) {
    for (int32_t c = static_cast<int32_t>(threadIdx.x); c < channels; c += static_cast<int32_t>(blockDim.x)) {
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        int32_t r = 0;
        for (; r + 3 < p.rows; r += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += parts[(r + i) * channels + c];
        for (; r < p.rows; ++r) sum[0] += parts[r * channels + c];
        const float total = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        out[c] = total;
        weighted[c] = total * weight[c];
    }
}

// Sums of one slab of one image: dz xhat and dz of every channel, s1 and s2 of every group.
template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_sums_kernel(const GNArgs a) {
    extern __shared__ __align__(16) float gn_lds[];   // [threads * VEC], then [2][bundle channels]
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, slab = p.slab;
    const int64_t image = p.image;
    float dw[VEC], db[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] = db[j] = 0.f;
    if (p.live) {
        const int64_t all = static_cast<int64_t>(a.images) * a.groups, g = image * a.groups + bundle * a.bundle + p.group;
        const GNCentre centre(a.stats[g], a.stats[all + g], a.stats[2 * all + g]);
        float w[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = a.weight[p.channel + j];
            b[j] = a.bias[p.channel + j];
        }
        const int64_t base = (image * a.pixels + p.first_pixel) * a.channels + p.channel;
        const T *x = static_cast<const T*>(a.x) + base, *dy = static_cast<const T*>(a.dy) + base;
        gn_with(a.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll 2
            for (int32_t i = p.row; i < p.pixels; i += p.rows) {
                float v[VEC], d[VEC];
                gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
                gn_load<T, VEC>(dy + static_cast<int64_t>(i) * a.channels, d);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xhat = centre(v[j]);
                    const float dz = d[j] * gn_slope<ACT>(fmaf(xhat, w[j], b[j]));
                    dw[j] = fmaf(dz, xhat, dw[j]);
                    db[j] += dz;
                }
            }
        });
    }
    const int32_t channels = p.groups * a.per, first = bundle * a.bundle * a.per, tid = static_cast<int32_t>(threadIdx.x);
    const int32_t threads = static_cast<int32_t>(blockDim.x);
    float* of_channel = gn_lds + threads * VEC;
    float* to = a.sums + (image * a.slabs + slab) * 2 * a.channels + first;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) gn_lds[tid * VEC + j] = q == 0 ? dw[j] : db[j];
        __syncthreads();
        gn_channel_sums(gn_lds, p, channels, to + q * a.channels, of_channel + q * channels, a.weight + first);
    }
    __syncthreads();
    const int32_t lanes = 1 << a.lg, sub = tid & (lanes - 1);
    for (int32_t g = tid >> a.lg; g < p.groups; g += threads >> a.lg) {
        float s1 = 0.f, s2 = 0.f;
        for (int32_t c = sub; c < a.per; c += lanes) {
            s1 += of_channel[channels + g * a.per + c];
            s2 += of_channel[g * a.per + c];
        }
        s1 = ln_lane_sum(s1, a.lg);
        s2 = ln_lane_sum(s2, a.lg);
        if (sub == 0) {
            float* out = a.group_sums + ((image * a.slabs + slab) * a.groups + bundle * a.bundle + g) * 2;
            out[0] = s1;
            out[1] = s2;
        }
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_dx_kernel(const GNArgs a) {
    __shared__ float sums[2 * 1024];
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, slab = p.slab;
    const int64_t image = p.image;
    const int32_t lane = static_cast<int32_t>(threadIdx.x) & ((1 << a.slabs_lg) - 1);
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> a.slabs_lg; g < p.groups; g += static_cast<int32_t>(blockDim.x) >> a.slabs_lg) {
        float s1 = 0.f, s2 = 0.f;
        for (int32_t i = lane; i < a.slabs; i += 1 << a.slabs_lg) {
            const float* from = a.group_sums + ((image * a.slabs + i) * a.groups + bundle * a.bundle + g) * 2;
            s1 += from[0];
            s2 += from[1];
        }
        s1 = ln_lane_sum(s1, a.slabs_lg);
        s2 = ln_lane_sum(s2, a.slabs_lg);
        if (lane == 0) {
            const float n = static_cast<float>(a.pixels) * static_cast<float>(a.per);
            sums[g] = s1 / n;
            sums[1024 + g] = s2 / n;
        }
    }
    __syncthreads();
    if (!p.live) return;
    const int64_t all = static_cast<int64_t>(a.images) * a.groups, g = image * a.groups + bundle * a.bundle + p.group;
    const GNCentre centre(a.stats[g], a.stats[all + g], a.stats[2 * all + g]);
    const float s1 = sums[p.group], s2 = sums[1024 + p.group];
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        w[j] = a.weight[p.channel + j];
        b[j] = a.bias[p.channel + j];
    }
    const int64_t base = (image * a.pixels + p.first_pixel) * a.channels + p.channel;
    const T *x = static_cast<const T*>(a.x) + base, *dy = static_cast<const T*>(a.dy) + base;
    T* dx = static_cast<T*>(a.dx) + base;
    gn_with(a.activation, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll 2
        for (int32_t i = p.row; i < p.pixels; i += p.rows) {
            float v[VEC], d[VEC];
            gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
            gn_load<T, VEC>(dy + static_cast<int64_t>(i) * a.channels, d);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float xhat = centre(v[j]);
                const float dz = d[j] * gn_slope<ACT>(fmaf(xhat, w[j], b[j]));
                v[j] = centre.rstd * (fmaf(w[j], dz, -s1) - xhat * s2);
            }
            gn_store<T, VEC>(dx + static_cast<int64_t>(i) * a.channels, v);
        }
    });
}

// The whole of a bundle's map in one workgroup's registers, K vectors a thread.
template <typename T, int VEC, int K>
__global__ __launch_bounds__(GN_RESIDENT) void group_norm_resident_kernel(const GNArgs a) {
    __shared__ float first[GN_RESIDENT], second[GN_RESIDENT], stats[3 * GN_RESIDENT];
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, tid = static_cast<int32_t>(threadIdx.x);
    const int64_t image = p.image;
    const int64_t base = image * a.pixels * a.channels + p.channel;
    const T* x = static_cast<const T*>(a.x) + base;
    GNRaw<T, VEC> raw[K];
    float sum = 0.f;
    const bool mine = p.live && p.row < p.pixels;
    if (mine) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int32_t i = p.row + k * p.rows;
            if (i < p.pixels) raw[k].load(x + static_cast<int64_t>(i) * a.channels);
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (p.row + k * p.rows < p.pixels) {
                float v[VEC];
                raw[k].forget();
                raw[k].unpack(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum += v[j];
            }
        first[p.entry] = sum;
    }
    __syncthreads();
    const int32_t lanes = 1 << a.lg, sub = tid & (lanes - 1);
    const float inv = 1.f / (static_cast<float>(p.pixels) * static_cast<float>(a.per));
    for (int32_t g = tid >> a.lg; g < p.groups; g += static_cast<int32_t>(blockDim.x) >> a.lg) {
        float total = 0.f;
        for (int32_t e = g * p.entries + sub; e < (g + 1) * p.entries; e += lanes) total += first[e];
        total = ln_lane_sum(total, a.lg);
        if (sub == 0) stats[g] = total * inv;
    }
    __syncthreads();
    if (mine) {
        const float mean = stats[p.group];
        float off = 0.f, square = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (p.row + k * p.rows < p.pixels) {
                float v[VEC];
                raw[k].forget();
                raw[k].unpack(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = v[j] - mean;
                    off += d;
                    square = fmaf(d, d, square);
                }
            }
        first[p.entry] = off;
        second[p.entry] = square;
    }
    __syncthreads();
    const int64_t all = static_cast<int64_t>(a.images) * a.groups, at = image * a.groups + bundle * a.bundle;
    for (int32_t g = tid >> a.lg; g < p.groups; g += static_cast<int32_t>(blockDim.x) >> a.lg) {
        float off = 0.f, square = 0.f;
        for (int32_t e = g * p.entries + sub; e < (g + 1) * p.entries; e += lanes) {
            off += first[e];
            square += second[e];
        }
        off = ln_lane_sum(off, a.lg) * inv;
        const float var = fmaxf(ln_lane_sum(square, a.lg) * inv - off * off, 0.f);
        if (sub == 0) {
            const float mean = stats[g], rstd = 1.f / sqrtf(var + a.eps);
            stats[GN_RESIDENT + g] = off;
            stats[2 * GN_RESIDENT + g] = rstd;
            if (a.stats != nullptr) {
                a.stats[at + g] = mean;
                a.stats[all + at + g] = off;
                a.stats[2 * all + at + g] = rstd;
            }
        }
    }
    __syncthreads();
    if (!mine) return;
    const GNCentre centre(stats[p.group], stats[GN_RESIDENT + p.group], stats[2 * GN_RESIDENT + p.group]);
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        w[j] = a.weight[p.channel + j];
        b[j] = a.bias[p.channel + j];
    }
    T* y = static_cast<T*>(a.y) + base;
    gn_with(a.activation, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int32_t i = p.row + k * p.rows;
            if (i < p.pixels) {
                float v[VEC];
                raw[k].forget();
                raw[k].unpack(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = gn_activate<ACT>(fmaf(centre(v[j]), w[j], b[j]));
                gn_store<T, VEC>(y + static_cast<int64_t>(i) * a.channels, v);
            }
        }
    });
}

// The same for the backward: x and dy in registers, K vectors of each; a row of parameter sums an image.
template <typename T, int VEC, int K>
__global__ __launch_bounds__(GN_RESIDENT, sizeof(T) == 2 && K < 8 ? 4 : 2) void group_norm_resident_backward_kernel(const GNArgs a) {
    extern __shared__ __align__(16) float gn_lds[];   // [threads * VEC], then [2][bundle channels]
    __shared__ float sums[2 * GN_RESIDENT];
    const GNPlace p = gn_place<VEC>(a);
    const int32_t bundle = p.bundle, tid = static_cast<int32_t>(threadIdx.x);
    const int32_t threads = static_cast<int32_t>(blockDim.x);
    const int64_t image = p.image;
    const int64_t base = image * a.pixels * a.channels + p.channel;
    const bool mine = p.live && p.row < p.pixels;
    GNRaw<T, VEC> rx[K], rd[K];
    float dw[VEC], db[VEC], w[VEC], b[VEC];
    const int64_t all = static_cast<int64_t>(a.images) * a.groups, group = image * a.groups + bundle * a.bundle + p.group;
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] = db[j] = w[j] = b[j] = 0.f;
    GNCentre centre(0.f, 0.f, 0.f);
    if (mine) {
        const T *x = static_cast<const T*>(a.x) + base, *dy = static_cast<const T*>(a.dy) + base;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int32_t i = p.row + k * p.rows;
            if (i < p.pixels) {
                rx[k].load(x + static_cast<int64_t>(i) * a.channels);
                rd[k].load(dy + static_cast<int64_t>(i) * a.channels);
            }
        }
        centre = GNCentre(a.stats[group], a.stats[all + group], a.stats[2 * all + group]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = a.weight[p.channel + j];
            b[j] = a.bias[p.channel + j];
        }
        gn_with(a.activation, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (p.row + k * p.rows < p.pixels) {
                    float v[VEC], d[VEC];
                    rx[k].forget();
                    rd[k].forget();
                    rx[k].unpack(v);
                    rd[k].unpack(d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float xhat = centre(v[j]);
                        const float dz = d[j] * gn_slope<ACT>(fmaf(xhat, w[j], b[j]));
                        dw[j] = fmaf(dz, xhat, dw[j]);
                        db[j] += dz;
                    }
                }
        });
    }
    const int32_t channels = p.groups * a.per, first = bundle * a.bundle * a.per;
    float* of_channel = gn_lds + threads * VEC;
    float* to = a.sums + image * 2 * a.channels + first;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VEC; ++j) gn_lds[tid * VEC + j] = q == 0 ? dw[j] : db[j];
        __syncthreads();
        gn_channel_sums(gn_lds, p, channels, to + q * a.channels, of_channel + q * channels, a.weight + first);
    }
    __syncthreads();
    const int32_t lanes = 1 << a.lg, sub = tid & (lanes - 1);
    const float inv = 1.f / (static_cast<float>(p.pixels) * static_cast<float>(a.per));
    for (int32_t g = tid >> a.lg; g < p.groups; g += threads >> a.lg) {
        float s1 = 0.f, s2 = 0.f;
        for (int32_t c = sub; c < a.per; c += lanes) {
            s1 += of_channel[channels + g * a.per + c];
            s2 += of_channel[g * a.per + c];
        }
        s1 = ln_lane_sum(s1, a.lg);
        s2 = ln_lane_sum(s2, a.lg);
        if (sub == 0) {
            sums[g] = s1 * inv;
            sums[GN_RESIDENT + g] = s2 * inv;
        }
    }
    __syncthreads();
    if (!mine) return;
    const float s1 = sums[p.group], s2 = sums[GN_RESIDENT + p.group];
    T* dx = static_cast<T*>(a.dx) + base;
    gn_with(a.activation, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int32_t i = p.row + k * p.rows;
            if (i < p.pixels) {
                float v[VEC], d[VEC];
                rx[k].forget();
                rd[k].forget();
                rx[k].unpack(v);
                rd[k].unpack(d);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xhat = centre(v[j]);
                    const float dz = d[j] * gn_slope<ACT>(fmaf(xhat, w[j], b[j]));
                    v[j] = centre.rstd * (fmaf(w[j], dz, -s1) - xhat * s2);
                }
                gn_store<T, VEC>(dx + static_cast<int64_t>(i) * a.channels, v);
            }
        }
    });
}

// ---- host side -------------------------------------------------------------------------

struct GNPlan {
    int32_t vec, threads, bundle, bundles, slabs, slab, lg, slabs_lg;
    int32_t vectors;   // a thread of the resident kernels, 0: slabs
};

// 2^result lanes for a group's sum of n values: four values each, and all of the workgroup's groups at
// once where that takes no more lanes than there are.
int32_t lanes_lg(int64_t n, int64_t groups, int32_t threads) {
    int32_t lg = 0;
    while (lg < 6 && (static_cast<int64_t>(4) << lg) < n && (groups << (lg + 1)) <= threads) ++lg;
    return lg;
}

// A bundle in one workgroup's registers, with runs of 128 bytes of a pixel (or all channels): four
// vectors a thread of 256, or eight of 512.  32 x 14 x 14 x 448 bf16 take 6 us (slabs: 10), 128 of them
// 13 (19), with the backward 42 (52).  Shorter runs waste the lines that they share (128 of them 25 us
// with 32 bytes).  Runs of 64 bytes would hold 28 x 28 x 192 too: 32 of them forward 10 us (slabs 12), but
// 128 forward and backward 79 (slabs 69).
bool plan_resident(GNPlan& p, int64_t pixels, int64_t per, int64_t groups, int e) {
    const int64_t each = per / p.vec, bundle = std::min(groups, (127 + per * e) / (per * e));
    for (int threads : {256, GN_RESIDENT}) {
        if (bundle * each > threads) continue;
        const int64_t rows = threads / (bundle * each), vectors = (pixels + rows - 1) / rows;
        if (vectors > (threads == 256 ? 4 : 8)) continue;
        p.threads = threads;
        p.bundle = static_cast<int32_t>(bundle);
        p.bundles = static_cast<int32_t>((groups + bundle - 1) / bundle);
        p.vectors = vectors <= 2 ? static_cast<int32_t>(vectors) : vectors <= 4 ? 4 : 8;
        p.slabs = 1;
        p.slab = static_cast<int32_t>(pixels);
        p.lg = lanes_lg(each * std::min(rows, pixels), bundle, threads);
        return true;
    }
    return false;
}

// Vectors lie within a group, so that a thread's values share their statistics.  Maps that no
// workgroup holds are cut into slabs so that about eight workgroups a CU share them; a workgroup then
// takes as many groups as its threads have vectors for (long runs of a pixel's channels).
GNPlan make_plan(int64_t B, int64_t pixels, int64_t channels, int64_t groups, int widest, int e) {
    const int64_t per = channels / groups;
    int vec = widest;
    while (per % vec) vec /= 2;
    const int64_t each = per / vec;
    GNPlan p{};
    p.vec = vec;
    if (plan_resident(p, pixels, per, groups, e)) return p;
    p.threads = each <= 256 ? 256 : static_cast<int32_t>((each + 63) / 64 * 64);
    int64_t bundle = p.threads / each;
    bundle = bundle < groups ? bundle : groups;
    const int64_t bundles = (groups + bundle - 1) / bundle;
    bundle = (groups + bundles - 1) / bundles;
    p.bundle = static_cast<int32_t>(bundle);
    p.bundles = static_cast<int32_t>((groups + bundle - 1) / bundle);
    const int64_t rows = p.threads / (bundle * each);
    int64_t slabs = (2048 + B * p.bundles - 1) / (B * p.bundles);
    const int64_t most = (pixels + rows * 4 - 1) / (rows * 4);   // four pixels a thread at least
    slabs = slabs < most ? slabs : most;
    slabs = slabs < GN_MAX_SLABS ? slabs : GN_MAX_SLABS;
    p.slab = static_cast<int32_t>((pixels + slabs - 1) / slabs);
    p.slabs = static_cast<int32_t>((pixels + p.slab - 1) / p.slab);
    p.lg = lanes_lg(each * std::min<int64_t>(rows, p.slab), bundle, p.threads);
    p.slabs_lg = lanes_lg(static_cast<int64_t>(p.slabs) * 4, bundle, p.threads);
    return p;
}

int check_sizes(int32_t io, int64_t B, int64_t pixels, int64_t channels, int64_t groups, int32_t activation) {
    VH_REQUIRE(valid_dtype(io), VH_ERR_DTYPE, "unsupported io_dtype %d", io);
    VH_REQUIRE(B > 0 && pixels > 0 && channels > 0, VH_ERR_SHAPE, "group norm needs nonempty maps, got %lld x %lld x %lld",
               (long long)B, (long long)pixels, (long long)channels);
    VH_REQUIRE(groups > 0 && channels % groups == 0, VH_ERR_SHAPE, "group norm: %lld channels do not divide into %lld groups",
               (long long)channels, (long long)groups);
    VH_REQUIRE(channels / groups <= GN_MAX_GROUP, VH_ERR_SHAPE, "group norm supports groups of at most %lld channels, got %lld",
               (long long)GN_MAX_GROUP, (long long)(channels / groups));
    // a launch has a workgroup for every slab of a bundle of groups, of 1024 threads at most
    VH_REQUIRE(pixels < (1ll << 30) && channels < (1ll << 22) && B < (1ll << 22) && B * groups < (1ll << 22), VH_ERR_SHAPE,
               "group norm: %lld maps of %lld pixels and %lld channels are out of range", (long long)B, (long long)pixels,
               (long long)channels);
    VH_REQUIRE(activation >= GN_NONE && activation <= GN_GELU, VH_ERR_ARG, "group norm: unknown activation %d", activation);
    return VH_OK;
}

// Elements of the widest vector that the addresses and a pixel's bytes allow.
int widest_of(int64_t channels, int e, std::initializer_list<const void*> pointers) {
    int vec = 16 / e;
    for (; vec > 1; vec /= 2) {
        bool ok = channels % vec == 0;
        for (const void* p : pointers) ok = ok && reinterpret_cast<uintptr_t>(p) % (vec * e) == 0;
        if (ok) break;
    }
    return vec;
}

size_t forward_bytes(int64_t B, int64_t groups, const GNPlan& p) {
    return p.vectors > 0 ? 0 : static_cast<size_t>(B) * p.slabs * groups * 2 * sizeof(double);
}
size_t backward_bytes(int64_t B, int64_t channels, int64_t groups, const GNPlan& p) {
    const int64_t rows = B * p.slabs;
    return static_cast<size_t>(rows) * 2 * (channels + groups) * sizeof(float) + param_sum_workspace_bytes(rows, 2, channels);
}

GNArgs make_args(const GNPlan& p, const void* x, const float* weight, const float* bias, float* stats, int64_t B,
                 int64_t pixels, int64_t channels, int64_t groups, int32_t activation) {
    GNArgs a{};
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.stats = stats;
    a.images = static_cast<int32_t>(B);
    a.pixels = static_cast<int32_t>(pixels);
    a.channels = static_cast<int32_t>(channels);
    a.groups = static_cast<int32_t>(groups);
    a.per = static_cast<int32_t>(channels / groups);
    a.bundle = p.bundle;
    a.bundles = p.bundles;
    a.slabs = p.slabs;
    a.slab = p.slab;
    a.lg = p.lg;
    a.slabs_lg = p.slabs_lg;
    a.activation = activation;
    return a;
}

template <typename F>
int by_type(int32_t io, int vec, F&& go) {
    auto by_vec = [&](auto t) -> int {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            if (vec == 8) return go(t, std::integral_constant<int, 8>{});
        }
        if (vec == 4) return go(t, std::integral_constant<int, 4>{});
        if (vec == 2) return go(t, std::integral_constant<int, 2>{});
        return go(t, std::integral_constant<int, 1>{});
    };
    if (io == VH_DTYPE_F32) return by_vec(float{});
    return io == VH_DTYPE_BF16 ? by_vec(bf16_t{}) : by_vec(f16_t{});
}

template <typename F>
int by_vectors(int32_t vectors, F&& go) {
    if (vectors == 1) return go(std::integral_constant<int, 1>{});
    if (vectors == 2) return go(std::integral_constant<int, 2>{});
    if (vectors == 4) return go(std::integral_constant<int, 4>{});
    return go(std::integral_constant<int, 8>{});
}

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_group_norm_workspace_bytes(int64_t B, int64_t pixels, int64_t channels, int64_t groups, int32_t io_dtype) {
    using namespace vh;
    if (check_sizes(io_dtype, B, pixels, channels, groups, 0) != VH_OK) return 0;
    size_t most = 0;   // of the vectors that a call may take
    for (int vec = 16 / dtype_bytes(io_dtype); vec >= 1; vec /= 2) {
        const size_t one = forward_bytes(B, groups, make_plan(B, pixels, channels, groups, vec, dtype_bytes(io_dtype)));
        most = one > most ? one : most;
    }
    return most;
}

int vh_group_norm_forward(const void* x, int32_t io_dtype, const float* weight, const float* bias, int32_t activation,
                          void* y, float* stats, int64_t B, int64_t pixels, int64_t channels, int64_t groups, float eps,
                          void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vh;
    if (int rc = check_sizes(io_dtype, B, pixels, channels, groups, activation)) return rc;
    VH_REQUIRE(x != nullptr && weight != nullptr && bias != nullptr && y != nullptr, VH_ERR_ARG,
               "x, weight, bias and y must not be null");
    const GNPlan p = make_plan(B, pixels, channels, groups, widest_of(channels, dtype_bytes(io_dtype), {x, y}), dtype_bytes(io_dtype));
    const size_t need = forward_bytes(B, groups, p);
    VH_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               VH_ERR_WORKSPACE, "group norm needs an aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    GNArgs a = make_args(p, x, weight, bias, stats, B, pixels, channels, groups, activation);
    a.y = y;
    a.eps = eps;
    a.partial = static_cast<double*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t grid = static_cast<uint32_t>(B * p.bundles * p.slabs);
    return by_type(io_dtype, p.vec, [&](auto t, auto v) -> int {
        if (p.vectors > 0)
            return by_vectors(p.vectors, [&](auto k) -> int {
                group_norm_resident_kernel<decltype(t), decltype(v)::value, decltype(k)::value>
                    <<<grid, p.threads, 0, s>>>(a);
                return check_launch("group_norm");
            });
        group_norm_stats_kernel<decltype(t), decltype(v)::value><<<grid, p.threads, 0, s>>>(a);
        if (int rc = check_launch("group_norm statistics")) return rc;
        group_norm_apply_kernel<decltype(t), decltype(v)::value><<<grid, p.threads, 0, s>>>(a);
        return check_launch("group_norm");
    });
}

size_t vh_group_norm_backward_workspace_bytes(int64_t B, int64_t pixels, int64_t channels, int64_t groups, int32_t io_dtype) {
    using namespace vh;
    if (check_sizes(io_dtype, B, pixels, channels, groups, 0) != VH_OK) return 0;
    size_t most = 0;
    for (int vec = 16 / dtype_bytes(io_dtype); vec >= 1; vec /= 2) {
        const size_t one = backward_bytes(B, channels, groups, make_plan(B, pixels, channels, groups, vec, dtype_bytes(io_dtype)));
        most = one > most ? one : most;
    }
    return most;
}

int vh_group_norm_backward(const void* dy, const void* x, int32_t io_dtype, const float* weight, const float* bias,
                           int32_t activation, const float* stats, void* dx, float* dweight, float* dbias, int64_t B,
                           int64_t pixels, int64_t channels, int64_t groups, void* workspace, size_t workspace_bytes,
                           void* stream) {
    using namespace vh;
    if (int rc = check_sizes(io_dtype, B, pixels, channels, groups, activation)) return rc;
    VH_REQUIRE(dy != nullptr && x != nullptr && weight != nullptr && bias != nullptr && stats != nullptr && dx != nullptr,
               VH_ERR_ARG, "dy, x, weight, bias, stats and dx must not be null");
    const GNPlan p = make_plan(B, pixels, channels, groups, widest_of(channels, dtype_bytes(io_dtype), {dy, x, dx}),
                               dtype_bytes(io_dtype));
    const size_t need = backward_bytes(B, channels, groups, p);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               VH_ERR_WORKSPACE, "group norm's backward needs an aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    GNArgs a = make_args(p, x, weight, bias, const_cast<float*>(stats), B, pixels, channels, groups, activation);
    a.dy = dy;
    a.dx = dx;
    const int64_t rows = B * p.slabs;
    a.sums = static_cast<float*>(workspace);
    a.group_sums = a.sums + rows * 2 * channels;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const uint32_t grid = static_cast<uint32_t>(B * p.bundles * p.slabs);
    const int rc = by_type(io_dtype, p.vec, [&](auto t, auto v) -> int {
        constexpr int VEC = decltype(v)::value;
        const size_t lds = (static_cast<size_t>(p.threads) * VEC + 2 * static_cast<size_t>(p.bundle) * a.per) * sizeof(float);
        if (p.vectors > 0)
            return by_vectors(p.vectors, [&](auto k) -> int {
                group_norm_resident_backward_kernel<decltype(t), VEC, decltype(k)::value>
                    <<<grid, p.threads, lds, s>>>(a);
                return check_launch("group_norm gradient");
            });
        group_norm_sums_kernel<decltype(t), VEC><<<grid, p.threads, lds, s>>>(a);
        if (int rc = check_launch("group_norm sums")) return rc;
        group_norm_dx_kernel<decltype(t), VEC><<<grid, p.threads, 0, s>>>(a);
        return check_launch("group_norm gradient");
    });
    if (rc != VH_OK || (dweight == nullptr && dbias == nullptr)) return rc;
    ParamSum sum{};
    sum.partial = a.sums;
    sum.rows = rows;
    sum.quantities = 2;
    sum.columns = a.channels;
    sum.out1 = dweight;
    sum.out2 = dbias;
    return launch_param_sum(sum, a.group_sums + rows * 2 * groups, s);
}

}  // extern "C"
