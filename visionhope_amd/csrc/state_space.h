// Device helpers and the argument block shared by the state space scan's forward
// (state_space.hip) and backward (state_space_backward.hip).
//
// Layout of the work: one lane per channel, the channel's S states in registers, tokens in
// order.  A wave takes 64 channels of one group of one sequence over one chunk of tokens, so
// B[t] and C[t] are the same for all its lanes and stand in scalar registers: the scalar
// unit loads and unpacks them while the vector unit computes.
#pragma once

#include "vh_common.h"

namespace vh {

constexpr float SS_LOG2E = 1.44269504088896341f;

// Tokens between two states that a training forward keeps for the backward.
constexpr int SS_BLOCK = 16;

struct SSTokens {   // an activation [B, N, ...]: element strides of sequence and token
    const void* data;
    int64_t bs, ts;
};

struct SSArgs {
    SSTokens x, dt, gate, b, c, dy;
    const float *A, *D, *dt_bias, *state;
    const int32_t* lengths;
    void* y;
    float* new_state;
    float* kept;     // [B, ceil(N / block), S, padded C]: states before each block of tokens
    float* slots;    // [B, chunks - 1, S, padded C]: states (or adjoints) between the chunks
    float* sums;     // [B, chunks, padded C]: sum of dt over a chunk
    int32_t softplus;
    int32_t states;   // of a channel as the tensors hold them; the kernels' S is the padded count
    int32_t batches, tokens, channels, group_channels, group_tiles, tiles;   // tiles: of 64 channels, all groups
    int32_t groups, chunk, chunks, first_chunk, launch_chunks, blocks;
    // backward
    int32_t wide_tiles, fine_chunks, fine_per_chunk;
    void *dx, *ddt, *dgate;
    float* dstate;
    float* bc_partial;     // [tiles, B, N, 2 S]
    float* param_partial;  // [B * chunks, S + 2, padded C]
    const float* dnew_state;
};

// Where a workgroup of one wave stands.  Consecutive indexes are the tiles of one chunk, which
// share B and C, and one contiguous range of them goes to each XCD.
struct SSPlace {
    int32_t batch, chunk, tile, group, lane, channel;
    int64_t column;     // of the padded channels
    // the lane has a channel of its own; the others take the group's last one too, compute and
    // store the same as its lane, and so need no branch in the token loop
    bool live;
    int32_t t0, t1, te; // tokens [t0, t1) of the chunk, of which [t0, te) belong to the sequence
};

__device__ __forceinline__ SSPlace ss_place(const SSArgs& a) {
    SSPlace p;
    const uint32_t bid = xcd_remap_any(blockIdx.x, gridDim.x);
    const uint32_t rest = bid / static_cast<uint32_t>(a.tiles);
    p.tile = static_cast<int32_t>(bid - rest * a.tiles);
    p.batch = static_cast<int32_t>(rest / static_cast<uint32_t>(a.launch_chunks));
    p.chunk = static_cast<int32_t>(rest) - p.batch * a.launch_chunks + a.first_chunk;
    p.lane = static_cast<int32_t>(threadIdx.x);
    p.group = p.tile / a.group_tiles;
    const int32_t in_group = (p.tile - p.group * a.group_tiles) * 64 + p.lane;
    p.live = in_group < a.group_channels;
    p.channel = p.group * a.group_channels + (p.live ? in_group : a.group_channels - 1);
    p.column = static_cast<int64_t>(p.tile) * 64 + p.lane;
    p.t0 = p.chunk * a.chunk;
    p.t1 = a.tokens - p.t0 < a.chunk ? a.tokens : p.t0 + a.chunk;
    int32_t len = a.tokens;
    if (a.lengths != nullptr) {
        len = __builtin_amdgcn_readfirstlane(a.lengths[p.batch]);
        len = len < 0 ? 0 : len > a.tokens ? a.tokens : len;
    }
    p.te = len < p.t0 ? p.t0 : len > p.t1 ? p.t1 : len;
    return p;
}

// An element `offset` bytes behind a uniform address.  `opaque` hides a lane's offset from the
// compiler, which would otherwise add it to the tensor's address once and keep (and step) a
// 64-bit address a lane for every tensor in vector registers.
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
template <typename T>
__device__ __forceinline__ T load_at(const T* base, uint32_t offset) {
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + offset);
}
template <typename T>
__device__ __forceinline__ void store_at(void* base, int64_t element, uint32_t offset, float v) {
    *reinterpret_cast<T*>(reinterpret_cast<char*>(static_cast<T*>(base) + element) + offset) = from_f32<T>(v);
}

// An activation at the first token of a wave's chunk.
template <typename T>
__device__ __forceinline__ const T* ss_tokens(const SSTokens& t, const SSPlace& p) {
    return static_cast<const T*>(t.data) + p.batch * t.bs + p.t0 * t.ts;
}

// Tokens that a wave loads together, one group ahead of the arithmetic.
constexpr int SS_UNROLL = 4;

// One token's row of S values of B or C, read through the scalar cache (a uniform address in
// memory that no kernel here writes): 16-bit pairs or FP32, 4-byte aligned.
template <typename T, int S>
struct SSRow {
    uint32_t w[S * sizeof(T) / 4];
    __device__ __forceinline__ void load(const void* base, int64_t elements) {
        typedef const __attribute__((address_space(4))) uint32_t* cptr;
        cptr p = (cptr)(reinterpret_cast<uintptr_t>(base) + elements * static_cast<int64_t>(sizeof(T)));
#pragma unroll
        for (int i = 0; i < static_cast<int>(S * sizeof(T) / 4); ++i) w[i] = p[i];
    }
    __device__ __forceinline__ float operator[](int n) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[n]);
        else return __uint_as_float((n & 1) ? (w[n / 2] & 0xffff0000u) : (w[n / 2] << 16));
    }
};

// softplus(v) = max(v, 0) + log1p(exp(-|v|)).  log1p(e) = 2 artanh(s) with s = e / (2 + e) <=
// 1/3, artanh(s) / s a polynomial in s^2 (least squares over [0, 1/9], 4e-9), so small steps
// keep their relative accuracy (3e-7), which log2(1 + e) would lose.
__device__ __forceinline__ float ss_softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-SS_LOG2E * fabsf(v));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e);
    const float w = s * s;
    float p = 0.14087328f;
    p = fmaf(p, w, 0.13980709f);
    p = fmaf(p, w, 0.20012426f);
    p = fmaf(p, w, 0.33333158f);
    p = fmaf(p, w, 1.f);
    return fmaf(s + s, p, fmaxf(v, 0.f));
}

inline int64_t ss_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A decay rate as an exponent of two a unit step: the rate times log2(e), kept finite, since a
// step of zero (a token behind a sequence's end, a chunk's sum of none) must decay by one and
// zero times an infinite rate has no value.  A NaN stays one.
__device__ __forceinline__ float ss_rate(float rate) {
    constexpr float most = 3.4028234664e38f;
    const float v = rate * SS_LOG2E;
    return v < -most ? -most : v > most ? most : v;
}

// A channel's decay rates times log2(e), zero for the padding (whose states stay zero, as B and
// C are zero there).
template <int S>
__device__ __forceinline__ void ss_rates(const SSArgs& a, int32_t channel, float (&A2)[S]) {
    const float* from = a.A + static_cast<int64_t>(channel) * a.states;
    if (a.states == S && (reinterpret_cast<uintptr_t>(a.A) & 15) == 0) {
#pragma unroll
        for (int n = 0; n < S; n += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + n);
            A2[n] = v.x; A2[n + 1] = v.y; A2[n + 2] = v.z; A2[n + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int n = 0; n < S; ++n) A2[n] = n < a.states ? from[n] : 0.f;
    }
#pragma unroll
    for (int n = 0; n < S; ++n) A2[n] = ss_rate(A2[n]);
}

// State count that the kernels are built for.
inline int32_t ss_padded(int32_t states) { return states <= 8 ? 8 : states <= 16 ? 16 : 32; }

// Argument checks and the geometry common to forward and backward.
int ss_fill(SSArgs& a, int32_t io_dtype, int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states);

// B and C as the kernels read them: where they stand (*bc_dtype the activations') if the states
// need no padding and every row is whole words of FP32 or bf16, otherwise as padded FP32 rows
// that this packs into `maps` (ss_maps_floats of them, always set aside).
inline int64_t ss_maps_floats(int64_t B, int64_t N, int32_t groups, int32_t states) {
    return 2 * B * N * groups * ss_padded(states);
}
int ss_maps(SSArgs& a, int32_t io_dtype, float* maps, int32_t* bc_dtype, hipStream_t stream);

// States (forward) or adjoints (backward) at the chunk boundaries from the chunks' own ones:
// slots [B, chunks - 1, S, padded C] in place, one chunk after the other.
int ss_join(const SSArgs& a, int64_t B, int32_t padded, bool backward, const float* edge, hipStream_t stream);

}  // namespace vh
