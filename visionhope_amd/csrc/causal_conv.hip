// Short causal depthwise convolution of token lines: forward, backward and the single-token
// step.
//
//   y[t, c] = f(bias[c] + sum_k weight[c, k] x[t - K + 1 + k, c]),  f = identity or SiLU
//
// with the K - 1 inputs before the first token from a state (zero without one).  A thread
// takes four channels (one where the sizes or alignments ask for it) and a
// segment of tokens with the window in registers, so every input is read once but for the
// K - 1 inputs before each segment.  Bound by the bytes of x and y: 18 us for 32 x 3136 x 192
// bf16 with four taps and SiLU, 77 MB at 4.3 TB/s (a large copy reaches 4.84).
#include "param_sum.h"

namespace vh {
namespace {

struct ConvArgs {
    const void *x, *dy, *state;
    int64_t x_bs, x_ts, dy_bs, dy_ts;
    const float *weight, *bias;
    const int32_t* lengths;
    const void* dnew_state;
    void *y, *new_state, *dx, *dstate;
    float* partial;   // [B * strips, K + 1, C]; a strip is SEGMENTS segments
    int32_t strips;
    int32_t silu, tokens, channels, groups, segment, segments;
    int64_t threads;
};

// VEC consecutive elements as fp32.
template <typename T, int VEC>
struct Vec {
    T v[VEC];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(p);
        else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(p);
        else v[0] = *p;
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
        else if constexpr (VEC * sizeof(T) == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
        else if constexpr (VEC * sizeof(T) == 4) *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(v);
        else *p = v[0];
    }
    __device__ __forceinline__ float operator[](int i) const { return to_f32(v[i]); }
    __device__ __forceinline__ void set(int i, float f) { v[i] = from_f32<T>(f); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = from_f32<T>(0.f);
    }
};

struct ConvPlace {
    int64_t batch;
    int32_t segment, channel, len;
};
template <int VEC>
__device__ __forceinline__ bool conv_place(const ConvArgs& a, int32_t segments, ConvPlace& p) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.threads) return false;
    const int64_t rest = i / a.groups;
    p.channel = static_cast<int32_t>(i - rest * a.groups) * VEC;
    p.batch = rest / segments;
    p.segment = static_cast<int32_t>(rest - p.batch * segments);
    p.len = a.tokens;
    if (a.lengths != nullptr) {
        const int32_t l = a.lengths[p.batch];
        p.len = l < 0 ? 0 : l > a.tokens ? a.tokens : l;
    }
    return true;
}

// Input t of a line: before its first token the state, at and behind len zero.
template <typename T, int VEC, int K>
__device__ __forceinline__ void conv_input(const ConvArgs& a, const ConvPlace& p, int32_t t, Vec<T, VEC>& v) {
    if (t >= 0) {
        if (t < p.len) v.load(static_cast<const T*>(a.x) + p.batch * a.x_bs + t * a.x_ts + p.channel);
        else v.zero();
    } else if (a.state != nullptr) {
        v.load(static_cast<const T*>(a.state) + (p.batch * (K - 1) + (K - 1 + t)) * a.channels + p.channel);
    } else {
        v.zero();
    }
}

constexpr int ROWS = 4;   // tokens loaded together

template <typename T, int VEC, int K>
__global__ __launch_bounds__(256) void causal_conv_kernel(const ConvArgs a) {
    ConvPlace p;
    // one segment more a sequence, which writes its new state
    const int32_t places = a.segments + (a.new_state != nullptr ? 1 : 0);
    if (!conv_place<VEC>(a, places, p)) return;
    if (p.segment == a.segments) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            Vec<T, VEC> v;
            conv_input<T, VEC, K>(a, p, p.len - (K - 1) + j, v);
            v.store(static_cast<T*>(a.new_state) + (p.batch * (K - 1) + j) * a.channels + p.channel);
        }
        return;
    }
    float w[K][VEC], bias[VEC], window[K][VEC];   // window[K - 1]: the newest input
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        bias[i] = a.bias != nullptr ? a.bias[p.channel + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = a.weight[static_cast<int64_t>(p.channel + i) * K + k];
    }
    const int32_t t0 = p.segment * a.segment;
    const int32_t t1 = a.tokens - t0 < a.segment ? a.tokens : t0 + a.segment;
    const int32_t te = p.len < t0 ? t0 : p.len < t1 ? p.len : t1;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        Vec<T, VEC> v;
        conv_input<T, VEC, K>(a, p, t0 - (K - 1) + k, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) window[k + 1][i] = v[i];
    }
    const T* x = static_cast<const T*>(a.x) + p.batch * a.x_bs + p.channel;
    T* y = static_cast<T*>(a.y) + p.batch * a.tokens * a.channels + p.channel;
    for (int32_t t = t0; t < te; t += ROWS) {
        Vec<T, VEC> rows[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) rows[r].load(x + static_cast<int64_t>(t + r < te ? t + r : te - 1) * a.x_ts);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            Vec<T, VEC> out;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float sum = bias[i];
#pragma unroll
                for (int k = 0; k < K - 1; ++k) {
                    window[k][i] = window[k + 1][i];
                    sum = fmaf(w[k][i], window[k][i], sum);
                }
                window[K - 1][i] = rows[r][i];
                sum = fmaf(w[K - 1][i], window[K - 1][i], sum);
                out.set(i, a.silu ? sum * sigmoid_fast(sum) : sum);
            }
            if (t + r < te) out.store(y + static_cast<int64_t>(t + r) * a.channels);
        }
    }
    Vec<T, VEC> none;
    none.zero();
    for (int32_t t = te; t < t1; ++t) none.store(y + static_cast<int64_t>(t) * a.channels);
}

// Backward: with p[t] the sum before f and g[t] = dy[t] f'(p[t]), dx[s] = sum_j w[K - 1 - j]
// g[s + j], dw[k] = sum_t g[t] x[t - K + 1 + k].  p is formed again from x.  A segment walks
// K - 1 tokens past its end for the g that its last inputs need.  The inputs before the
// first token (the state's) belong to segment 0, and the new state's gradient is added to
// the inputs that it holds.
// A workgroup takes 16 channel groups and SEGMENTS segments that follow each other, and sums
// their weight gradients in LDS before they go to memory.  At 32 x 3136 x 192 bf16: 31 us,
// 116 MB at 3.7 TB/s; the vector unit is active for two thirds of that time (SiLU's derivative and
// three sets of products, 40 instructions an element), the rest is waits for loads.
constexpr int SEGMENTS = 16;
template <typename T, int VEC, int K>
__global__ __launch_bounds__(256) void causal_conv_backward_kernel(const ConvArgs a) {
    constexpr int BROWS = 4;
    __shared__ float sums[SEGMENTS][K + 1][16 * VEC];
    const int32_t row = threadIdx.x >> 4, column = threadIdx.x & 15;
    const int32_t across = (a.groups + 15) / 16;
    ConvPlace p;
    const int64_t rest = blockIdx.x / across;
    const int32_t group = static_cast<int32_t>(blockIdx.x - rest * across) * 16 + column;
    p.batch = rest / a.strips;
    const int32_t strip = static_cast<int32_t>(rest - p.batch * a.strips);
    p.segment = strip * SEGMENTS + row;
    // lanes and segments past the end take part in the sums with nothing
    const bool live = group < a.groups && p.segment < a.segments;
    p.channel = (group < a.groups ? group : a.groups - 1) * VEC;
    p.len = a.tokens;
    if (a.lengths != nullptr) {
        const int32_t l = a.lengths[p.batch];
        p.len = l < 0 ? 0 : l > a.tokens ? a.tokens : l;
    }
    float w[K][VEC], bias[VEC], window[K][VEC], g[K][VEC], dw[K][VEC], db[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        bias[i] = a.bias != nullptr ? a.bias[p.channel + i] : 0.f;
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            w[k][i] = a.weight[static_cast<int64_t>(p.channel + i) * K + k];
            dw[k][i] = g[k][i] = 0.f;
        }
    }
    const int32_t t0 = live ? p.segment * a.segment : a.tokens;
    const int32_t t1 = a.tokens - t0 < a.segment ? a.tokens : t0 + a.segment;
    const int32_t te = p.len < t0 ? t0 : p.len < t1 ? p.len : t1;   // tokens of the sequence
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        Vec<T, VEC> v;
        if (live) conv_input<T, VEC, K>(a, p, t0 - (K - 1) + k, v);
        else v.zero();
#pragma unroll
        for (int i = 0; i < VEC; ++i) window[k + 1][i] = v[i];
    }
    const T* x = static_cast<const T*>(a.x) + p.batch * a.x_bs + p.channel;
    const T* dy = static_cast<const T*>(a.dy) + p.batch * a.dy_bs + p.channel;
    T* dx = static_cast<T*>(a.dx) + p.batch * a.tokens * a.channels + p.channel;
    T* dstate = a.dstate != nullptr
        ? static_cast<T*>(a.dstate) + p.batch * (K - 1) * a.channels + p.channel : nullptr;
    const T* dnew = a.dnew_state != nullptr
        ? static_cast<const T*>(a.dnew_state) + p.batch * (K - 1) * a.channels + p.channel : nullptr;
    // The input s = t - (K - 1) is complete once g[t] is known.  Segment 0 begins with the
    // state's inputs, the others with the first input of their own.
    const bool own = live && (te > t0 || p.segment == 0);
    const int32_t s0 = p.segment == 0 ? -(K - 1) : t0;
    const int32_t stop = own ? te + K - 1 : t0;
    WaveTurns turns(a.segment + K - 1);
    for (int32_t t = t0; t < stop; t += BROWS) {
        turns.left(a.segment + K - 1 - __builtin_amdgcn_readfirstlane(t - t0));
        Vec<T, VEC> xr[BROWS], gr[BROWS];
#pragma unroll
        for (int r = 0; r < BROWS; ++r) {
            if (t + r < p.len) {
                xr[r].load(x + static_cast<int64_t>(t + r) * a.x_ts);
                gr[r].load(dy + static_cast<int64_t>(t + r) * a.dy_ts);
            } else {
                xr[r].zero();
                gr[r].zero();
            }
        }
#pragma unroll
        for (int r = 0; r < BROWS; ++r) {
            const int32_t tr = t + r, s = tr - (K - 1);
            float out[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float sum = bias[i];
#pragma unroll
                for (int k = 0; k < K - 1; ++k) {
                    window[k][i] = window[k + 1][i];
                    g[k][i] = g[k + 1][i];
                    sum = fmaf(w[k][i], window[k][i], sum);
                }
                window[K - 1][i] = xr[r][i];
                sum = fmaf(w[K - 1][i], window[K - 1][i], sum);
                float grad = gr[r][i];
                if (a.silu) {
                    const float sig = sigmoid_fast(sum);
                    grad *= sig * fmaf(sum, 1.f - sig, 1.f);
                }
                g[K - 1][i] = tr < p.len ? grad : 0.f;
                const float mine = tr < te ? g[K - 1][i] : 0.f;
                db[i] += mine;
                out[i] = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    dw[k][i] = fmaf(mine, window[k][i], dw[k][i]);
                    out[i] = fmaf(w[K - 1 - k][i], g[k][i], out[i]);
                }
            }
            if (s >= s0 && s < te) {
                if (dnew != nullptr && s >= p.len - (K - 1)) {
                    Vec<T, VEC> more;
                    more.load(dnew + static_cast<int64_t>(s - (p.len - (K - 1))) * a.channels);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) out[i] += more[i];
                }
                Vec<T, VEC> store;
#pragma unroll
                for (int i = 0; i < VEC; ++i) store.set(i, out[i]);
                if (s >= 0) store.store(dx + static_cast<int64_t>(s) * a.channels);
                else if (dstate != nullptr) store.store(dstate + static_cast<int64_t>(s + K - 1) * a.channels);
            }
        }
    }
    Vec<T, VEC> none;
    none.zero();
    for (int32_t t = te; t < t1; ++t) none.store(dx + static_cast<int64_t>(t) * a.channels);
#pragma unroll
    for (int k = 0; k <= K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sums[row][k][column * VEC + i] = k < K ? dw[k][i] : db[i];
    __syncthreads();
    float* to = a.partial + (p.batch * a.strips + strip) * (K + 1) * a.channels;
    const int32_t first = (static_cast<int32_t>(blockIdx.x - rest * across) * 16) * VEC;
    for (int32_t v = threadIdx.x; v < (K + 1) * 16 * VEC; v += 256) {
        const int32_t k = v / (16 * VEC), c = v % (16 * VEC);
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < SEGMENTS; ++r) sum += sums[r][k][c];
        if (first + c < a.channels) to[static_cast<int64_t>(k) * a.channels + first + c] = sum;
    }
}

// One token a sequence: the window is the state and the token.  A thread reads all of its
// channels' state before it writes, so new_state may be state.  3.0 us for 64 sequences of 1024
// channels, the time of a launch.
template <typename T, int VEC, int K>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(const ConvArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= a.threads) return;
    const int64_t batch = i / a.groups;
    const int32_t channel = static_cast<int32_t>(i - batch * a.groups) * VEC;
    Vec<T, VEC> in[K], out;
    const T* state = static_cast<const T*>(a.state) + batch * (K - 1) * a.channels + channel;
    T* next = static_cast<T*>(a.new_state) + batch * (K - 1) * a.channels + channel;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) in[k].load(state + static_cast<int64_t>(k) * a.channels);
    in[K - 1].load(static_cast<const T*>(a.x) + batch * a.x_bs + channel);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        float sum = a.bias != nullptr ? a.bias[channel + v] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) sum = fmaf(a.weight[static_cast<int64_t>(channel + v) * K + k], in[k][v], sum);
        out.set(v, a.silu ? sum * sigmoid_fast(sum) : sum);
    }
    out.store(static_cast<T*>(a.y) + batch * a.channels + channel);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) in[k + 1].store(next + static_cast<int64_t>(k) * a.channels);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tokens a thread of the forward takes: the work is cut until about 8 waves a SIMD (1024
// SIMDs) have some, down to 16 tokens (the K - 1 inputs before a segment are read twice).
int64_t segment_tokens(int64_t B, int64_t N, int64_t groups) {
    const int64_t wanted = 8 * 1024 * 64;
    int64_t segments = wanted / (B * groups);
    if (segments < 1) segments = 1;
    int64_t tokens = ceil_div(ceil_div(N, segments), ROWS) * ROWS;
    return tokens < 16 ? 16 : tokens > 256 ? 256 : tokens;
}

// Strips (16 segments each) that the backward cuts a line into: about three waves a SIMD, what
// its registers hold, of segments of at least 16 tokens.
int64_t strip_count(int64_t B, int64_t N, int64_t groups) {
    int64_t strips = 3 * 1024 / 4 / (B * ceil_div(groups, 16));
    if (strips > ceil_div(N, 16 * SEGMENTS)) strips = ceil_div(N, 16 * SEGMENTS);
    return strips < 1 ? 1 : strips;
}

// Widest access of at most `most` elements that all addresses and strides allow.
bool aligned(const void* p, int64_t bs, int64_t ts, int64_t bytes, int64_t e) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && bs * e % bytes == 0 && ts * e % bytes == 0;
}
int vec_of(int64_t C, int e, int bytes, std::initializer_list<const void*> dense,
           std::initializer_list<ConvArgs> strided) {
    const int64_t vec = bytes / e;
    if (C % vec) return 1;
    for (const void* p : dense)
        if (reinterpret_cast<uintptr_t>(p) % bytes) return 1;
    for (const ConvArgs& s : strided) {
        if (s.x != nullptr && !aligned(s.x, s.x_bs, s.x_ts, bytes, e)) return 1;
        if (s.dy != nullptr && !aligned(s.dy, s.dy_bs, s.dy_ts, bytes, e)) return 1;
    }
    return static_cast<int>(vec);
}

enum Kind { FORWARD, BACKWARD, STEP };

template <typename T, int VEC, int K>
int launch(Kind kind, const ConvArgs& a, hipStream_t s) {
    const int64_t blocks = kind == BACKWARD ? a.threads / 256 : ceil_div(a.threads, 256);
    VH_REQUIRE(blocks < (1ll << 24), VH_ERR_SHAPE, "causal convolution: too many sequences for one launch");
    const uint32_t grid = static_cast<uint32_t>(blocks);
    if (kind == FORWARD) causal_conv_kernel<T, VEC, K><<<grid, 256, 0, s>>>(a);
    else if (kind == BACKWARD) causal_conv_backward_kernel<T, VEC, K><<<grid, 256, 0, s>>>(a);
    else causal_conv_step_kernel<T, VEC, K><<<grid, 256, 0, s>>>(a);
    return check_launch("causal convolution");
}
template <typename T, int VEC>
int launch_taps(Kind kind, const ConvArgs& a, int taps, hipStream_t s) {
    switch (taps) {
        case 2: return launch<T, VEC, 2>(kind, a, s);
        case 3: return launch<T, VEC, 3>(kind, a, s);
        case 4: return launch<T, VEC, 4>(kind, a, s);
        case 5: return launch<T, VEC, 5>(kind, a, s);
        case 6: return launch<T, VEC, 6>(kind, a, s);
        case 7: return launch<T, VEC, 7>(kind, a, s);
        default: return launch<T, VEC, 8>(kind, a, s);
    }
}
// vec: channels a thread, 4 or 1.  (Eight of a 16-bit type a thread, 16 bytes, were slower:
// 21.2 us against 18.8 at 32 x 3136 x 192 bf16, fewer waves with more registers each.)
int dispatch(Kind kind, const ConvArgs& a, int32_t io, int vec, int taps, hipStream_t s) {
    if (io == VH_DTYPE_F32) {
        if (vec == 4) return launch_taps<float, 4>(kind, a, taps, s);
        return launch_taps<float, 1>(kind, a, taps, s);
    }
    if (io == VH_DTYPE_BF16) {
        if (vec == 4) return launch_taps<bf16_t, 4>(kind, a, taps, s);
        return launch_taps<bf16_t, 1>(kind, a, taps, s);
    }
    if (vec == 4) return launch_taps<f16_t, 4>(kind, a, taps, s);
    return launch_taps<f16_t, 1>(kind, a, taps, s);
}

int check_sizes(int32_t io, int64_t B, int64_t N, int64_t C, int32_t taps) {
    VH_REQUIRE(valid_dtype(io), VH_ERR_DTYPE, "unsupported io_dtype %d", io);
    VH_REQUIRE(B > 0 && N > 0 && C > 0, VH_ERR_SHAPE, "causal convolution needs nonempty sizes, got B=%lld N=%lld C=%lld",
               (long long)B, (long long)N, (long long)C);
    VH_REQUIRE(N < (1ll << 30) && C < (1ll << 24) && B < (1ll << 24), VH_ERR_SHAPE,
               "causal convolution: sizes out of range (B=%lld N=%lld C=%lld)", (long long)B, (long long)N, (long long)C);
    VH_REQUIRE(taps >= 2 && taps <= 8, VH_ERR_SHAPE, "taps must be 2 to 8, got %d", taps);
    return VH_OK;
}

}  // namespace
}  // namespace vh

extern "C" {

int vh_causal_conv_forward(const void* x, int64_t x_batch, int64_t x_token, int32_t io_dtype, const float* weight,
                           const float* bias, int32_t silu, const void* state, const int32_t* lengths, void* y,
                           void* new_state, int64_t B, int64_t N, int64_t C, int32_t taps, void* stream) {
    using namespace vh;
    if (int rc = check_sizes(io_dtype, B, N, C, taps)) return rc;
    VH_REQUIRE(x != nullptr && weight != nullptr && y != nullptr, VH_ERR_ARG, "x, weight and y must not be null");
    VH_REQUIRE(!overlapping(state, new_state, B * (taps - 1) * C * dtype_bytes(io_dtype)), VH_ERR_ARG,
               "state and new_state must not overlap");
    ConvArgs a{};
    a.x = x;
    a.x_bs = x_batch;
    a.x_ts = x_token;
    a.weight = weight;
    a.bias = bias;
    a.silu = silu;
    a.state = state;
    a.lengths = lengths;
    a.y = y;
    a.new_state = new_state;
    a.tokens = static_cast<int32_t>(N);
    a.channels = static_cast<int32_t>(C);
    const int e = dtype_bytes(io_dtype), vec = vec_of(C, e, 4 * e, {y, state, new_state}, {a});
    a.groups = static_cast<int32_t>(C / vec);
    a.segment = static_cast<int32_t>(segment_tokens(B, N, a.groups));
    a.segments = static_cast<int32_t>(ceil_div(N, a.segment));
    a.threads = B * (a.segments + (new_state != nullptr ? 1 : 0)) * a.groups;
    return dispatch(FORWARD, a, io_dtype, vec, taps, static_cast<hipStream_t>(stream));
}

size_t vh_causal_conv_backward_workspace_bytes(int64_t B, int64_t N, int64_t C, int32_t taps) {
    using namespace vh;
    if (B <= 0 || N <= 0 || C <= 0 || taps <= 0) return 0;
    // with four channels a thread or with one
    int64_t rows = 0;
    size_t sums = 0;
    for (int64_t groups : {C / 4 > 0 ? C / 4 : 1, C}) {
        const int64_t one = B * strip_count(B, N, groups);
        const size_t bytes = param_sum_workspace_bytes(one, taps + 1, C);
        rows = one > rows ? one : rows;
        sums = bytes > sums ? bytes : sums;
    }
    return static_cast<size_t>(rows) * (taps + 1) * C * sizeof(float) + sums;
}

int vh_causal_conv_backward(const void* dy, int64_t dy_batch, int64_t dy_token, const void* x, int64_t x_batch,
                            int64_t x_token, int32_t io_dtype, const float* weight, const float* bias, int32_t silu,
                            const void* state, const int32_t* lengths, const void* dnew_state, void* dx, float* dweight,
                            float* dbias, void* dstate, int64_t B, int64_t N, int64_t C, int32_t taps, void* workspace,
                            size_t workspace_bytes, void* stream) {
    using namespace vh;
    if (int rc = check_sizes(io_dtype, B, N, C, taps)) return rc;
    VH_REQUIRE(dy != nullptr && x != nullptr && weight != nullptr && dx != nullptr, VH_ERR_ARG,
               "dy, x, weight and dx must not be null");
    const size_t need = vh_causal_conv_backward_workspace_bytes(B, N, C, taps);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need, VH_ERR_WORKSPACE,
               "causal convolution backward needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
    ConvArgs a{};
    a.dy = dy;
    a.dy_bs = dy_batch;
    a.dy_ts = dy_token;
    a.x = x;
    a.x_bs = x_batch;
    a.x_ts = x_token;
    a.weight = weight;
    a.bias = bias;
    a.silu = silu;
    a.state = state;
    a.lengths = lengths;
    a.dnew_state = dnew_state;
    a.dx = dx;
    a.dstate = dstate;
    a.tokens = static_cast<int32_t>(N);
    a.channels = static_cast<int32_t>(C);
    const int e = dtype_bytes(io_dtype), vec = vec_of(C, e, 4 * e, {dx, state, dstate, dnew_state}, {a});
    a.groups = static_cast<int32_t>(C / vec);
    a.strips = static_cast<int32_t>(strip_count(B, N, a.groups));
    // whole loads of four tokens
    a.segment = static_cast<int32_t>(ceil_div(ceil_div(N, a.strips * SEGMENTS), 4) * 4);
    a.segments = static_cast<int32_t>(ceil_div(N, a.segment));
    a.threads = B * a.strips * ceil_div(a.groups, 16) * 256;
    a.partial = static_cast<float*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (int rc = dispatch(BACKWARD, a, io_dtype, vec, taps, s)) return rc;
    ParamSum sum{};
    sum.partial = a.partial;
    sum.rows = B * a.strips;
    sum.quantities = taps + 1;
    sum.columns = static_cast<int32_t>(C);
    sum.per_channel = sum.padded = taps;
    sum.out0 = dweight;
    sum.out1 = dbias;
    return launch_param_sum(sum, a.partial + sum.rows * (taps + 1) * C, s);
}

int vh_causal_conv_step(const void* x, int64_t x_batch, int32_t io_dtype, const float* weight, const float* bias,
                        int32_t silu, const void* state, void* new_state, void* y, int64_t B, int64_t C, int32_t taps,
                        void* stream) {
    using namespace vh;
    if (int rc = check_sizes(io_dtype, B, 1, C, taps)) return rc;
    VH_REQUIRE(x != nullptr && weight != nullptr && state != nullptr && new_state != nullptr && y != nullptr, VH_ERR_ARG,
               "x, weight, state, new_state and y must not be null");
    VH_REQUIRE(state == new_state || !overlapping(state, new_state, B * (taps - 1) * C * dtype_bytes(io_dtype)),
               VH_ERR_ARG, "state and new_state must be the same memory or not overlap");
    ConvArgs a{};
    a.x = x;
    a.x_bs = x_batch;
    a.weight = weight;
    a.bias = bias;
    a.silu = silu;
    a.state = state;
    a.new_state = new_state;
    a.y = y;
    a.channels = static_cast<int32_t>(C);
    const int e = dtype_bytes(io_dtype), vec = vec_of(C, e, 4 * e, {y, state, new_state}, {a});
    a.groups = static_cast<int32_t>(C / vec);
    a.threads = B * a.groups;
    return dispatch(STEP, a, io_dtype, vec, taps, static_cast<hipStream_t>(stream));
}

}  // extern "C"
