// Group norm of channels-last maps [B, P pixels, C] with an activation: forward and backward.
//
//   z = (x - mean) rstd w + b,  y = f(z),  mean and variance (biased) over a group's channels and
//   all pixels of an image; f the identity, SiLU or the exact GELU
//
// Backward, with dz = dy f'(z), xhat = (x - mean) rstd, n values a group:
//   db = sum dz,  dw = sum dz xhat  (over images and pixels),
//   dx = rstd (w dz - (s1 + xhat s2) / n),  s1 = sum w dz,  s2 = sum w dz xhat  over the group
//
// Both directions are two passes over the map: partial sums of slabs of pixels, then the outputs,
// whose workgroups join their image's slabs first.  Bound by the bytes of the map.
//
// Statistics: a thread sums its values and their squares about its own first value, so that what
// cancels is bounded by its own share of the variance; threads and slabs are joined by their means
// and centred squares with the means in FP64, and the mean is kept as a sum of two floats (an offset
// large beside the spread loses nothing).
#include "param_sum.h"

namespace vh {
namespace {

constexpr int GN_NONE = 0, GN_SILU = 1, GN_GELU = 2;
constexpr int64_t GN_MAX_SLABS = 64;      // one lane of a wave each
constexpr int64_t GN_MAX_GROUP = 1024;    // channels of a group: a workgroup's threads

struct GNArgs {
    const void *x, *dy;
    const float *weight, *bias;
    void *y, *dx;
    float* stats;        // [3, B, G]: mean, its rest, rstd
    double* partial;     // [B, slabs, G, 2]: mean and centred squares of a slab's group
    float* sums;         // [B, slabs, 2, C]: of dz xhat and of dz
    float* group_sums;   // [B, slabs, G, 2]: s1, s2
    int32_t pixels, channels, groups, per;           // per: channels of a group
    int32_t bundle, bundles;                         // groups of a workgroup; workgroups for all groups
    int32_t slabs, slab;                             // slab: its pixels
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
// (degree 8, our minimax fit) is within 8.8e-8 of it relatively for all a.  `bell` is exp(-a^2 / 2),
// which the derivative needs as well.  The 8e-6 of gelu_fast would show in the
// parameters' gradients, FP32 sums.
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
__device__ __forceinline__ float gn_activate(float z, int32_t activation) {
    if (activation == GN_NONE) return z;
    if (activation == GN_SILU) return z * sigmoid_fast(z);
    float bell;
    const float a = fabsf(z), tail = gn_tail(a, bell);
    return fmaf(-a, tail, fmaxf(z, 0.f));
}
__device__ __forceinline__ float gn_slope(float z, int32_t activation) {
    if (activation == GN_NONE) return 1.f;
    if (activation == GN_SILU) {
        const float s = sigmoid_fast(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    float bell;
    const float tail = gn_tail(fabsf(z), bell);
    return fmaf(z * 0.398942280401432678f, bell, z < 0.f ? tail : 1.f - tail);
}

__device__ __forceinline__ double gn_wave_sum(double v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

// A thread's place: `vector` of the bundle's vectors in a pixel, pixels `row`, row + rows, ... of
// a slab; threads behind the last full row are idle.
struct GNPlace {
    int32_t vectors, rows, vector, row, channel, group;   // channel: its first; group: within the bundle
    int32_t groups;                                       // of this bundle
    int32_t first_pixel, pixels;                          // of the slab
    bool live;
};
template <int VEC>
__device__ __forceinline__ GNPlace gn_place(const GNArgs& a, int32_t bundle, int32_t slab) {
    GNPlace p;
    const int32_t first = bundle * a.bundle;
    p.groups = a.groups - first < a.bundle ? a.groups - first : a.bundle;
    p.vectors = p.groups * a.per / VEC;
    p.rows = static_cast<int32_t>(blockDim.x) / p.vectors;
    p.row = static_cast<int32_t>(threadIdx.x) / p.vectors;
    p.vector = static_cast<int32_t>(threadIdx.x) - p.row * p.vectors;
    p.live = p.row < p.rows;
    p.channel = first * a.per + p.vector * VEC;
    p.group = p.vector * VEC / a.per;
    p.first_pixel = slab * a.slab;
    p.pixels = a.pixels - p.first_pixel < a.slab ? a.pixels - p.first_pixel : a.slab;
    return p;
}

// Sums of one slab of one image: a group's mean and centred squares.
template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_stats_kernel(const GNArgs a) {
    __shared__ double means[1024];
    __shared__ float squares[1024];
    const int32_t slab = static_cast<int32_t>(blockIdx.x), bundle = static_cast<int32_t>(blockIdx.y);
    const int64_t image = blockIdx.z;
    const GNPlace p = gn_place<VEC>(a, bundle, slab);
    float pivot = 0.f, sum = 0.f, square = 0.f;
    if (p.live && p.row < p.pixels) {
        const T* at = static_cast<const T*>(a.x) + (image * a.pixels + p.first_pixel) * a.channels + p.channel;
        pivot = to_f32(at[static_cast<int64_t>(p.row) * a.channels]);
#pragma unroll 4
        for (int32_t i = p.row; i < p.pixels; i += p.rows) {
            float v[VEC];
            gn_load<T, VEC>(at + static_cast<int64_t>(i) * a.channels, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = v[j] - pivot;
                sum += d;
                square = fmaf(d, d, square);
            }
        }
        const float n = static_cast<float>((p.pixels - p.row + p.rows - 1) / p.rows * VEC), off = sum / n;
        means[threadIdx.x] = static_cast<double>(pivot) + static_cast<double>(off);
        squares[threadIdx.x] = fmaxf(fmaf(-sum, off, square), 0.f);
    }
    __syncthreads();
    const int32_t lane = threadIdx.x & 63, each = a.per / VEC, waves = static_cast<int32_t>(blockDim.x) >> 6;
    const int32_t rows = p.pixels < p.rows ? p.pixels : p.rows;
    const double n_all = static_cast<double>(p.pixels) * a.per;
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> 6; g < p.groups; g += waves) {
        double total = 0.0, centred = 0.0;
        for (int32_t e = lane; e < each * rows; e += 64) {
            const int32_t row = e / each, t = row * p.vectors + g * each + (e - row * each);
            total += means[t] * ((p.pixels - row + p.rows - 1) / p.rows * VEC);
        }
        const double mean = gn_wave_sum(total) / n_all;
        for (int32_t e = lane; e < each * rows; e += 64) {
            const int32_t row = e / each, t = row * p.vectors + g * each + (e - row * each);
            const double d = means[t] - mean;
            centred += d * d * ((p.pixels - row + p.rows - 1) / p.rows * VEC) + static_cast<double>(squares[t]);
        }
        centred = gn_wave_sum(centred);
        if (lane == 0) {
            double* to = a.partial + ((image * a.slabs + slab) * a.groups + bundle * a.bundle + g) * 2;
            to[0] = mean;
            to[1] = centred;
        }
    }
}

// Mean (two floats) and rstd of the bundle's groups from the slabs, in LDS [3][bundle].
__device__ __forceinline__ void gn_join(const GNArgs& a, const GNPlace& p, int32_t bundle, int64_t image, float* out) {
    const int32_t lane = threadIdx.x & 63, waves = static_cast<int32_t>(blockDim.x) >> 6;
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> 6; g < p.groups; g += waves) {
        double mean = 0.0, square = 0.0, n = 0.0;
        if (lane < a.slabs) {
            const double* from = a.partial + ((image * a.slabs + lane) * a.groups + bundle * a.bundle + g) * 2;
            mean = from[0];
            square = from[1];
            const int32_t left = a.pixels - lane * a.slab;
            n = static_cast<double>(left < a.slab ? left : a.slab) * a.per;
        }
        const double n_all = static_cast<double>(a.pixels) * a.per;
        const double all = gn_wave_sum(mean * n) / n_all;
        const double d = mean - all;
        const double var = gn_wave_sum(d * d * n + square) / n_all;
        if (lane == 0) {
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
    const int32_t slab = static_cast<int32_t>(blockIdx.x), bundle = static_cast<int32_t>(blockIdx.y);
    const int64_t image = blockIdx.z;
    const GNPlace p = gn_place<VEC>(a, bundle, slab);
    gn_join(a, p, bundle, image, stats);
    if (slab == 0 && a.stats != nullptr) {
        const int64_t all = static_cast<int64_t>(gridDim.z) * a.groups, at = image * a.groups + bundle * a.bundle;
        for (int32_t g = static_cast<int32_t>(threadIdx.x); g < p.groups; g += static_cast<int32_t>(blockDim.x))
#pragma unroll
            for (int q = 0; q < 3; ++q) a.stats[q * all + at + g] = stats[q * 1024 + g];
    }
    if (!p.live) return;
    const float mean = stats[p.group], rest = stats[1024 + p.group], rstd = stats[2048 + p.group];
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        w[j] = rstd * a.weight[p.channel + j];
        b[j] = a.bias[p.channel + j];
    }
    const int64_t base = (image * a.pixels + p.first_pixel) * a.channels + p.channel;
    const T* x = static_cast<const T*>(a.x) + base;
    T* y = static_cast<T*>(a.y) + base;
#pragma unroll 2
    for (int32_t i = p.row; i < p.pixels; i += p.rows) {
        float v[VEC];
        gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = gn_activate(fmaf((v[j] - mean) - rest, w[j], b[j]), a.activation);
        gn_store<T, VEC>(y + static_cast<int64_t>(i) * a.channels, v);
    }
}

// Sums of one slab of one image: dz xhat and dz of every channel, s1 and s2 of every group.
template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_sums_kernel(const GNArgs a) {
    extern __shared__ __align__(16) float gn_lds[];   // [threads * VEC], then [2][bundle channels]
    const int32_t slab = static_cast<int32_t>(blockIdx.x), bundle = static_cast<int32_t>(blockIdx.y);
    const int64_t image = blockIdx.z;
    const GNPlace p = gn_place<VEC>(a, bundle, slab);
    float dw[VEC], db[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[j] = db[j] = 0.f;
    if (p.live) {
        const int64_t all = static_cast<int64_t>(gridDim.z) * a.groups, g = image * a.groups + bundle * a.bundle + p.group;
        const float mean = a.stats[g], rest = a.stats[all + g], rstd = a.stats[2 * all + g];
        float w[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = a.weight[p.channel + j];
            b[j] = a.bias[p.channel + j];
        }
        const int64_t base = (image * a.pixels + p.first_pixel) * a.channels + p.channel;
        const T *x = static_cast<const T*>(a.x) + base, *dy = static_cast<const T*>(a.dy) + base;
#pragma unroll 2
        for (int32_t i = p.row; i < p.pixels; i += p.rows) {
            float v[VEC], d[VEC];
            gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
            gn_load<T, VEC>(dy + static_cast<int64_t>(i) * a.channels, d);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float xhat = ((v[j] - mean) - rest) * rstd;
                const float dz = d[j] * gn_slope(fmaf(xhat, w[j], b[j]), a.activation);
                dw[j] = fmaf(dz, xhat, dw[j]);
                db[j] += dz;
            }
        }
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
        for (int32_t c = tid; c < channels; c += threads) {
            float sum = 0.f;
            for (int32_t r = 0; r < p.rows; ++r) sum += gn_lds[r * channels + c];
            to[q * a.channels + c] = sum;
            of_channel[q * channels + c] = sum * a.weight[first + c];
        }
    }
    __syncthreads();
    const int32_t lane = tid & 63, waves = threads >> 6;
    for (int32_t g = tid >> 6; g < p.groups; g += waves) {
        float s1 = 0.f, s2 = 0.f;
        for (int32_t c = lane; c < a.per; c += 64) {
            s1 += of_channel[channels + g * a.per + c];
            s2 += of_channel[g * a.per + c];
        }
        s1 = ln_lane_sum(s1, 6);
        s2 = ln_lane_sum(s2, 6);
        if (lane == 0) {
            float* out = a.group_sums + ((image * a.slabs + slab) * a.groups + bundle * a.bundle + g) * 2;
            out[0] = s1;
            out[1] = s2;
        }
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(1024) void group_norm_dx_kernel(const GNArgs a) {
    __shared__ float sums[2 * 1024];
    const int32_t slab = static_cast<int32_t>(blockIdx.x), bundle = static_cast<int32_t>(blockIdx.y);
    const int64_t image = blockIdx.z;
    const GNPlace p = gn_place<VEC>(a, bundle, slab);
    const int32_t lane = threadIdx.x & 63, waves = static_cast<int32_t>(blockDim.x) >> 6;
    for (int32_t g = static_cast<int32_t>(threadIdx.x) >> 6; g < p.groups; g += waves) {
        float s1 = 0.f, s2 = 0.f;
        if (lane < a.slabs) {
            const float* from = a.group_sums + ((image * a.slabs + lane) * a.groups + bundle * a.bundle + g) * 2;
            s1 = from[0];
            s2 = from[1];
        }
        s1 = ln_lane_sum(s1, 6);
        s2 = ln_lane_sum(s2, 6);
        if (lane == 0) {
            const float n = static_cast<float>(a.pixels) * static_cast<float>(a.per);
            sums[g] = s1 / n;
            sums[1024 + g] = s2 / n;
        }
    }
    __syncthreads();
    if (!p.live) return;
    const int64_t all = static_cast<int64_t>(gridDim.z) * a.groups, g = image * a.groups + bundle * a.bundle + p.group;
    const float mean = a.stats[g], rest = a.stats[all + g], rstd = a.stats[2 * all + g];
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
#pragma unroll 2
    for (int32_t i = p.row; i < p.pixels; i += p.rows) {
        float v[VEC], d[VEC];
        gn_load<T, VEC>(x + static_cast<int64_t>(i) * a.channels, v);
        gn_load<T, VEC>(dy + static_cast<int64_t>(i) * a.channels, d);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float xhat = ((v[j] - mean) - rest) * rstd;
            const float dz = d[j] * gn_slope(fmaf(xhat, w[j], b[j]), a.activation);
            v[j] = rstd * (fmaf(w[j], dz, -s1) - xhat * s2);
        }
        gn_store<T, VEC>(dx + static_cast<int64_t>(i) * a.channels, v);
    }
}

// ---- host side -------------------------------------------------------------------------

struct GNPlan {
    int32_t vec, threads, bundle, bundles, slabs, slab;
};

// Vectors lie within a group, so that a thread's values share their statistics; a workgroup takes as
// many groups as its threads have vectors for (long runs of a pixel's channels), and slabs are cut so
// that about eight workgroups a CU share the map.
GNPlan make_plan(int64_t B, int64_t pixels, int64_t channels, int64_t groups, int widest) {
    const int64_t per = channels / groups;
    int vec = widest;
    while (per % vec) vec /= 2;
    const int64_t each = per / vec;
    GNPlan p;
    p.vec = vec;
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
    VH_REQUIRE(B < 65536 && pixels < (1ll << 30) && channels < (1ll << 22), VH_ERR_SHAPE,
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
    return static_cast<size_t>(B) * p.slabs * groups * 2 * sizeof(double);
}
size_t backward_bytes(int64_t B, int64_t channels, int64_t groups, const GNPlan& p) {
    const int64_t rows = B * p.slabs;
    return static_cast<size_t>(rows) * 2 * (channels + groups) * sizeof(float) + param_sum_workspace_bytes(rows, 2, channels);
}

GNArgs make_args(const GNPlan& p, const void* x, const float* weight, const float* bias, float* stats, int64_t pixels,
                 int64_t channels, int64_t groups, int32_t activation) {
    GNArgs a{};
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.stats = stats;
    a.pixels = static_cast<int32_t>(pixels);
    a.channels = static_cast<int32_t>(channels);
    a.groups = static_cast<int32_t>(groups);
    a.per = static_cast<int32_t>(channels / groups);
    a.bundle = p.bundle;
    a.bundles = p.bundles;
    a.slabs = p.slabs;
    a.slab = p.slab;
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

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_group_norm_workspace_bytes(int64_t B, int64_t pixels, int64_t channels, int64_t groups, int32_t io_dtype) {
    using namespace vh;
    if (check_sizes(io_dtype, B, pixels, channels, groups, 0) != VH_OK) return 0;
    size_t most = 0;   // of the vectors that a call may take
    for (int vec = 16 / dtype_bytes(io_dtype); vec >= 1; vec /= 2) {
        const size_t one = forward_bytes(B, groups, make_plan(B, pixels, channels, groups, vec));
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
    const GNPlan p = make_plan(B, pixels, channels, groups, widest_of(channels, dtype_bytes(io_dtype), {x, y}));
    const size_t need = forward_bytes(B, groups, p);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               VH_ERR_WORKSPACE, "group norm needs an aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    GNArgs a = make_args(p, x, weight, bias, stats, pixels, channels, groups, activation);
    a.y = y;
    a.eps = eps;
    a.partial = static_cast<double*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<uint32_t>(p.slabs), static_cast<uint32_t>(p.bundles), static_cast<uint32_t>(B));
    return by_type(io_dtype, p.vec, [&](auto t, auto v) -> int {
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
        const size_t one = backward_bytes(B, channels, groups, make_plan(B, pixels, channels, groups, vec));
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
    const GNPlan p = make_plan(B, pixels, channels, groups, widest_of(channels, dtype_bytes(io_dtype), {dy, x, dx}));
    const size_t need = backward_bytes(B, channels, groups, p);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               VH_ERR_WORKSPACE, "group norm's backward needs an aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    GNArgs a = make_args(p, x, weight, bias, const_cast<float*>(stats), pixels, channels, groups, activation);
    a.dy = dy;
    a.dx = dx;
    const int64_t rows = B * p.slabs;
    a.sums = static_cast<float*>(workspace);
    a.group_sums = a.sums + rows * 2 * channels;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<uint32_t>(p.slabs), static_cast<uint32_t>(p.bundles), static_cast<uint32_t>(B));
    const int rc = by_type(io_dtype, p.vec, [&](auto t, auto v) -> int {
        constexpr int VEC = decltype(v)::value;
        const size_t lds = (static_cast<size_t>(p.threads) * VEC + 2 * static_cast<size_t>(p.bundle) * a.per) * sizeof(float);
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
