// Device pieces shared by the linear attention kernels (linear_attention.hip,
// linear_attention_backward.hip): operands as sums of bf16 values, powers of a decay, tiles of
// tokens in LDS.
//
// Matrix products run on v_mfma_f32_16x16x32_bf16 with FP32 accumulators.  An operand is a sum of
// bf16 values ("limbs"), each the rounding of what the ones before it leave: one for a bf16 tensor,
// two for FP16 (11 bits) and three for FP32 (24 bits), all exact and without FP16's range.  A
// product of two operands is the sum of the products of their limbs (a, b) with a + b up to an
// order; those behind it are below 2^-(8 order + 8) of the whole.  Six bf16 products take 96 cycles
// a 16x16x32 tile where the FP32 matrix instructions take 256.
#pragma once

#include "vh_common.h"

namespace vh {

typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef float la_f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct LAType;
// raw: limbs of a tensor's values; tokens: of a chunk; formed: limbs of weights and states as
// operands of a product that is rounded to T (2: 16 bits of them, so that the sum's one rounding
// to T is the only one that counts)
template <> struct LAType<bf16_t> { static constexpr int raw = 1, tokens = 64, formed = 2, order = 1; };
template <> struct LAType<f16_t> { static constexpr int raw = 2, tokens = 32, formed = 2, order = 1; };
template <> struct LAType<float> { static constexpr int raw = 3, tokens = 32, formed = 3, order = 2; };

// Limbs of what enters a state, an FP32 result: 24 bits.
constexpr int LA_STATE_LIMBS = 3;

struct LATokens {   // an activation [B, N, heads, dim]: element strides of sequence, token and head
    const void* data;
    int64_t bs, ts, hs;
};

__device__ __forceinline__ la_f32x4 la_mfma(const uint4& a, const uint4& b, la_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(la_bf16x8, a), __builtin_bit_cast(la_bf16x8, b), c, 0, 0, 0);
}

// c += a b over 32 values: lane l holds row (column) l % 16 of a (b), and of the contracted index
// the eight values that group l / 16 has (any order, the same for both); of the result, rows
// 4 (l / 16) .. + 3 in column l % 16.  Smallest products first.
template <int ORDER, int NA, int NB>
__device__ __forceinline__ la_f32x4 la_mm(const uint4 (&a)[NA], const uint4 (&b)[NB], la_f32x4 c) {
#pragma unroll
    for (int o = ORDER; o >= 0; --o)
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int j = o - i;
            if (j >= 0 && j < NB) c = la_mfma(a[i], b[j < 0 || j >= NB ? 0 : j], c);
        }
    return c;
}

__device__ __forceinline__ float la_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float la_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// A pair of values as NL pairs of limbs.
template <int NL>
__device__ __forceinline__ void la_split(float a, float b, uint32_t (&out)[NL]) {
#pragma unroll
    for (int l = 0; l < NL; ++l) {
        out[l] = pack_bf16x2(a, b);
        if (l + 1 < NL) {
            a -= la_low(out[l]);
            b -= la_high(out[l]);
        }
    }
}
template <int NL>
__device__ __forceinline__ void la_split8(const float (&v)[8], uint4 (&out)[NL]) {
    uint32_t w[4][NL];
#pragma unroll
    for (int i = 0; i < 4; ++i) la_split<NL>(v[2 * i], v[2 * i + 1], w[i]);
#pragma unroll
    for (int l = 0; l < NL; ++l) out[l] = make_uint4(w[0][l], w[1][l], w[2][l], w[3][l]);
}
// The eight values that raw limbs stand for (exact).
template <int NL>
__device__ __forceinline__ void la_join8(const uint4 (&in)[NL], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll
    for (int l = NL - 1; l >= 0; --l) {
        const uint32_t w[4] = {in[l].x, in[l].y, in[l].z, in[l].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = l == NL - 1 ? la_low(w[i]) : v[2 * i] + la_low(w[i]);
            v[2 * i + 1] = l == NL - 1 ? la_high(w[i]) : v[2 * i + 1] + la_high(w[i]);
        }
    }
}

// exp(m log_decay) for m >= 0.  The product m log2(e) log_decay is formed with its rounding error,
// which far powers would otherwise keep (m of 16384 at a decay of 1e-3: 2^-20 instead of 2^-24).
// A decay of minus infinity forgets at every token: kept finite, so that its power 0 is one.
struct LADecay {
    float high, low;
    __device__ __forceinline__ explicit LADecay(float log_decay) {
        const float a = log_decay < -1e5f ? -1e5f : log_decay;   // NaN stays
        high = a * 1.44269504088896341f;
        low = fmaf(a, 1.44269504088896341f, -high) + a * 1.92596299e-8f;   // log2(e) beyond FP32
    }
    __device__ __forceinline__ float power(float m) const {
        const float e = m * high;
        const float rest = fmaf(m, high, -e) + m * low;
        const float p = __builtin_amdgcn_exp2f(e);
        return fmaf(p, rest * 0.693147181f, p);
    }
};

// Four values of a tensor as loaded.
template <typename T> struct LAQuad { uint2 u; };
template <> struct LAQuad<float> { float4 f; };

// Values col .. col + 3 of a row of `dim`, zeros behind it; `wide`: one load (dim and addresses are
// multiples of four elements).
template <typename T>
__device__ __forceinline__ LAQuad<T> la_load(const T* row, int32_t col, int32_t dim, bool wide, bool live) {
    LAQuad<T> r{};
    if (!live || col >= dim) return r;
    if (wide) {
        if constexpr (sizeof(T) == 4) r.f = *reinterpret_cast<const float4*>(row + col);
        else r.u = *reinterpret_cast<const uint2*>(row + col);
        return r;
    }
    if constexpr (sizeof(T) == 4) {
        r.f.x = row[col];
        if (col + 1 < dim) r.f.y = row[col + 1];
        if (col + 2 < dim) r.f.z = row[col + 2];
        if (col + 3 < dim) r.f.w = row[col + 3];
    } else {
        r.u.x = row[col].bits;
        if (col + 1 < dim) r.u.x |= static_cast<uint32_t>(row[col + 1].bits) << 16;
        if (col + 2 < dim) r.u.y = row[col + 2].bits;
        if (col + 3 < dim) r.u.y |= static_cast<uint32_t>(row[col + 3].bits) << 16;
    }
    return r;
}

// A quad as limbs: words (0, 1) and (2, 3) of each.
template <typename T>
__device__ __forceinline__ void la_limbs(const LAQuad<T>& q, uint2 (&out)[LAType<T>::raw]) {
    if constexpr (std::is_same<T, bf16_t>::value) {
        out[0] = q.u;
    } else {
        float v[4];
        if constexpr (sizeof(T) == 4) {
            v[0] = q.f.x; v[1] = q.f.y; v[2] = q.f.z; v[3] = q.f.w;
        } else {
            v[0] = to_f32(T{static_cast<uint16_t>(q.u.x & 0xffffu)});
            v[1] = to_f32(T{static_cast<uint16_t>(q.u.x >> 16)});
            v[2] = to_f32(T{static_cast<uint16_t>(q.u.y & 0xffffu)});
            v[3] = to_f32(T{static_cast<uint16_t>(q.u.y >> 16)});
        }
        uint32_t a[LAType<T>::raw], b[LAType<T>::raw];
        la_split<LAType<T>::raw>(v[0], v[1], a);
        la_split<LAType<T>::raw>(v[2], v[3], b);
#pragma unroll
        for (int l = 0; l < LAType<T>::raw; ++l) out[l] = make_uint2(a[l], b[l]);
    }
}

// The low (high) halves of two words as one.
__device__ __forceinline__ uint32_t la_lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t la_highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Stores four values of a row.
template <typename T>
__device__ __forceinline__ void la_store(T* row, int32_t col, int32_t dim, bool wide, const float (&v)[4]) {
    if (wide) {
        if (col >= dim) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(row + col) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint2 w;
            if constexpr (std::is_same<T, bf16_t>::value) {
                w = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            } else {
                w.x = from_f32<T>(v[0]).bits | static_cast<uint32_t>(from_f32<T>(v[1]).bits) << 16;
                w.y = from_f32<T>(v[2]).bits | static_cast<uint32_t>(from_f32<T>(v[3]).bits) << 16;
            }
            *reinterpret_cast<uint2*>(row + col) = w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < dim) row[col + i] = from_f32<T>(v[i]);
}

// Tiles of a chunk in LDS, for heads padded to D.
template <typename T, int D>
struct LAShape {
    static constexpr int R = LAType<T>::raw, F = LAType<T>::formed, C = LAType<T>::tokens;
    static constexpr int waves = D / 16, threads = 64 * waves;
    // rows of LDS tiles, eight values longer than they need: 16 rows' 16-byte reads spread over all banks
    static constexpr int row_d = D + 8, row_c = C + 8;
    static constexpr int tokens_tile = C * row_d, turned_tile = D * row_c, weights_tile = C * row_c;
    static constexpr int state_lds = (2 * R * turned_tile) * 2 + 512;
    static constexpr int lds = state_lds + (2 * R * tokens_tile + F * weights_tile) * 2;
};

// Four columns 4 cu .. + 3 of C / 16 tokens (the tu-th such run) into `rows` (tokens' rows; the index
// 32 x + 16 h + 4 y + r stands at 32 x + 8 y + 4 h + r, the order in which two tiles of accumulators
// have it) and into `turned` (columns' rows); either may be null.
template <typename T, int D>
__device__ __forceinline__ void la_stage(const LAQuad<T> (&raw)[LAShape<T, D>::C / 16], uint16_t* rows, uint16_t* turned,
                                         int32_t cu, int32_t tu) {
    using P = LAShape<T, D>;
    constexpr int UNIT = P::C / 16;
    const int32_t in = (4 * cu) & 31, place = ((4 * cu) & ~31) + ((in & 15) >> 2) * 8 + (in >> 4) * 4;
    uint2 limbs[UNIT][P::R];
#pragma unroll
    for (int u = 0; u < UNIT; ++u) la_limbs<T>(raw[u], limbs[u]);
#pragma unroll
    for (int l = 0; l < P::R; ++l) {
        if (rows != nullptr) {
#pragma unroll
            for (int u = 0; u < UNIT; ++u)
                *reinterpret_cast<uint2*>(rows + l * P::tokens_tile + (tu * UNIT + u) * P::row_d + place) = limbs[u][l];
        }
        if (turned != nullptr) {
            uint16_t* to = turned + l * P::turned_tile + 4 * cu * P::row_c + tu * UNIT;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[UNIT / 2];
#pragma unroll
                for (int u = 0; u < UNIT / 2; ++u) {
                    const uint32_t x = c < 2 ? limbs[2 * u][l].x : limbs[2 * u][l].y;
                    const uint32_t y = c < 2 ? limbs[2 * u + 1][l].x : limbs[2 * u + 1][l].y;
                    w[u] = c & 1 ? la_highs(x, y) : la_lows(x, y);
                }
                if constexpr (UNIT == 4) *reinterpret_cast<uint2*>(to + c * P::row_c) = make_uint2(w[0], w[UNIT / 2 - 1]);
                else *reinterpret_cast<uint32_t*>(to + c * P::row_c) = w[0];
            }
        }
    }
}

// Eight values at `at` of every limb of a tile.
template <int R>
__device__ __forceinline__ void la_read(const uint16_t* tile, int32_t size, int32_t at, uint4 (&out)[R]) {
#pragma unroll
    for (int l = 0; l < R; ++l) out[l] = *reinterpret_cast<const uint4*>(tile + l * size + at);
}

// One pass of the recurrence over all heads: the forward, or a gradient that has its form.
struct LAPass {
    LATokens q, k, v;        // kdim, kdim and vdim wide
    void* out;               // [B, N, heads, vdim], dense
    const float* log_decay;
    // factors of the weights, of what comes from the state before a chunk, of what enters the state
    float scale_weight, scale_out, scale_in;
    const float* state;      // where the walk starts (null: zero); a head's [kdim, vdim] with these strides
    float* new_state;        // where it ends (or null), the same strides
    int64_t state_row, state_col;
    const int32_t* lengths;
    float* slots;            // [B, heads, segments - 1, D * D]: states between the segments
    int32_t batches, tokens, heads, kdim, vdim, segments, chunks_per_segment, chunk, reversed;
    bool wide_q, wide_k, wide_v, wide_out;
};

// Tokens of a sequence.
__device__ __forceinline__ int32_t la_end(const LAPass& a, int32_t batch) {
    if (a.lengths == nullptr) return a.tokens;
    const int32_t n = a.lengths[batch];
    return n < 0 ? 0 : n > a.tokens ? a.tokens : n;
}

// ---- host side -------------------------------------------------------------------------

struct LACut {   // segments of a line, and chunks of each (the last may have fewer)
    int32_t segments, each;
};
LACut la_cut(int64_t heads, int64_t N, int32_t padded, int32_t io_dtype);
size_t la_slots_bytes(int64_t heads, const LACut& cut, int32_t padded);
int la_check_sizes(int32_t io_dtype, int64_t B, int64_t N, int64_t heads, int64_t key_dim, int64_t value_dim);
// Runs a pass (sets its widths and its chunk itself); la_states: only as far as the states between
// the segments.
int la_run(LAPass& a, int32_t io_dtype, hipStream_t stream);
int la_states(LAPass& a, int32_t io_dtype, hipStream_t stream);

constexpr int64_t LA_MAX_DIM = 128;

inline int64_t la_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int32_t la_padded(int64_t key_dim, int64_t value_dim) {
    const int64_t d = key_dim > value_dim ? key_dim : value_dim;
    return d <= 32 ? 32 : d <= 64 ? 64 : 128;
}
// Whether four elements of a row are one load.
inline bool la_wide(const LATokens& t, int64_t dim, int64_t e) {
    return dim % 4 == 0 && reinterpret_cast<uintptr_t>(t.data) % (4 * e) == 0 && t.bs % 4 == 0 && t.ts % 4 == 0 && t.hs % 4 == 0;
}
inline int32_t la_chunk(int32_t io_dtype) { return io_dtype == VH_DTYPE_BF16 ? 64 : 32; }

}  // namespace vh
