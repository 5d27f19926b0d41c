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

#include <initializer_list>

#include "vh_common.h"

namespace vh {

typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef float la_f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct LAType;
// raw: limbs of a tensor's values; tokens: of a chunk
template <> struct LAType<bf16_t> { static constexpr int raw = 1, tokens = 64; };
template <> struct LAType<f16_t> { static constexpr int raw = 2, tokens = 32; };
template <> struct LAType<float> { static constexpr int raw = 3, tokens = 32; };

// Limbs of what is formed in FP32 (weights of pairs, states, what enters a state) and the order of
// its products: 24 bits for every type, so that results do not depend on what else a call returns.
// (Two limbs turn the rounding of 0.25 % of bf16 and of 2 % of FP16 results, three of 0.02 and 0.1 %:
// 197 against 210 us a bf16 training pass of 32 x 3136 x 3 heads of 64.)
constexpr int LA_FORMED = 3, LA_ORDER = 2;

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
template <int NA, int NB>
__device__ __forceinline__ la_f32x4 la_mm(const uint4 (&a)[NA], const uint4 (&b)[NB], la_f32x4 c) {
#pragma unroll
    for (int o = LA_ORDER; o >= 0; --o)
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

// Eight values of a tensor's row as loaded.
template <typename T> struct LAOct { uint4 u; };
template <> struct LAOct<float> { float4 a, b; };

// Values col .. col + 7 of a row of `dim`, zeros behind it.  `vec`: elements that one load may take
// (8, 4 or 1), by dim, strides and addresses; WIDE: 8.
template <typename T, bool WIDE>
__device__ __forceinline__ LAOct<T> la_load(const T* row, int32_t col, int32_t dim, int32_t vec) {
    LAOct<T> r{};
    if (col >= dim) return r;
    if (WIDE || vec == 8) {
        if constexpr (sizeof(T) == 4) {
            r.a = *reinterpret_cast<const float4*>(row);
            r.b = *reinterpret_cast<const float4*>(row + 4);
        } else {
            r.u = *reinterpret_cast<const uint4*>(row);
        }
        return r;
    }
    if (vec == 4) {
        if constexpr (sizeof(T) == 4) {
            r.a = *reinterpret_cast<const float4*>(row);
            if (col + 4 < dim) r.b = *reinterpret_cast<const float4*>(row + 4);
        } else {
            const uint2 lo = *reinterpret_cast<const uint2*>(row);
            uint2 hi = make_uint2(0, 0);
            if (col + 4 < dim) hi = *reinterpret_cast<const uint2*>(row + 4);
            r.u = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        return r;
    }
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < dim ? row[i] : T{};
    if constexpr (sizeof(T) == 4) {
        r.a = make_float4(v[0], v[1], v[2], v[3]);
        r.b = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = v[2 * i].bits | static_cast<uint32_t>(v[2 * i + 1].bits) << 16;
        r.u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return r;
}

// The eight values as limbs.
template <typename T>
__device__ __forceinline__ void la_limbs(const LAOct<T>& q, uint4 (&out)[LAType<T>::raw]) {
    if constexpr (std::is_same<T, bf16_t>::value) {
        out[0] = q.u;
    } else {
        float v[8];
        if constexpr (sizeof(T) == 4) {
            v[0] = q.a.x; v[1] = q.a.y; v[2] = q.a.z; v[3] = q.a.w;
            v[4] = q.b.x; v[5] = q.b.y; v[6] = q.b.z; v[7] = q.b.w;
        } else {
            const uint32_t w[4] = {q.u.x, q.u.y, q.u.z, q.u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = to_f32(T{static_cast<uint16_t>(w[i] & 0xffffu)});
                v[2 * i + 1] = to_f32(T{static_cast<uint16_t>(w[i] >> 16)});
            }
        }
        la_split8<LAType<T>::raw>(v, out);
    }
}

// Stores values col .. col + 3 of a row of `dim` at `row`; `wide`: as one.
template <typename T>
__device__ __forceinline__ void la_store(T* row, int32_t col, int32_t dim, bool wide, const float (&v)[4]) {
    if (wide) {
        if (col >= dim) return;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(row) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint2 w;
            if constexpr (std::is_same<T, bf16_t>::value) {
                w = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            } else {
                w.x = from_f32<T>(v[0]).bits | static_cast<uint32_t>(from_f32<T>(v[1]).bits) << 16;
                w.y = from_f32<T>(v[2]).bits | static_cast<uint32_t>(from_f32<T>(v[3]).bits) << 16;
            }
            *reinterpret_cast<uint2*>(row) = w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (col + i < dim) row[i] = from_f32<T>(v[i]);
}

// LDS tiles have rows of W values (32, 64 or 128) whose blocks of eight are permuted by the row: block b of
// row r stands at b ^ la_fold(r).  Sixteen rows' blocks of one index then lie in sixteen different places
// of the 256 bytes that the banks are wide, and so do the blocks that a transposing read takes from
// four rows.  (Rows eight values longer instead: 203 against 197 us a training pass of 32 x 3136 x 3
// heads of 64, with what is formed as two limbs.)
template <int W>
__device__ __forceinline__ int32_t la_fold(int32_t row) {
    const int32_t low = (row >> 2) & 3;
    return W == 128 ? (row & 3) << 2 | low : W == 64 ? ((row >> 1) & 1) << 2 | low : low;
}
// Where block b of a row starts.  Another block x of the same row is at this place ^ 8 (b ^ x).
template <int W>
__device__ __forceinline__ int32_t la_block(int32_t row, int32_t b) {
    return row * W + 8 * (b ^ la_fold<W>(row));
}

// Tiles of a chunk, for heads padded to D.
template <typename T, int D>
struct LAShape {
    static constexpr int R = LAType<T>::raw, F = LA_FORMED, C = LAType<T>::tokens;
    static constexpr int waves = D / 16, threads = 64 * waves, units = C / 32;   // units: of eight values a thread
    static constexpr int tile = C * D, weights = C * C;   // one limb
    static constexpr int head = 512;                              // bytes of small tables
    static constexpr int state_lds = head + 2 * R * tile * 2;
    static constexpr int lds = head + (3 * R * tile + F * weights) * 2;
};

// Key index of row 4 g + r of tile m of a state: two tiles together hold, for a lane, eight neighbours
// in a row, which are at once a lane's share of an operand that is contracted over the key index.
__device__ __forceinline__ int32_t la_state_row(int32_t m, int32_t g, int32_t r) {
    return 32 * (m >> 1) + 8 * g + 4 * (m & 1) + r;
}

// Eight values col .. col + 7 of token i into a tile.
template <typename T, int D>
__device__ __forceinline__ void la_stage(const LAOct<T>& raw, uint16_t* tile, int32_t col, int32_t i) {
    using P = LAShape<T, D>;
    uint4 limbs[P::R];
    la_limbs<T>(raw, limbs);
#pragma unroll
    for (int l = 0; l < P::R; ++l) *reinterpret_cast<uint4*>(tile + l * P::tile + la_block<D>(i, col / 8)) = limbs[l];
}

typedef short la_i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) la_i16x4 la_lds_i16x4;

// A column of a tile over eight tokens, of every limb: lane l gets column 16 m + l % 16 (ROWS: the key
// index of that row of a state's tile m) at tokens 32 x + 8 (l / 16) .. + 7.  The transposing read takes
// four columns of four tokens from the quarters of a 16-lane group and gives each lane one column of
// them.  `at`: la_column<D, ROWS>.
template <int D, bool ROWS>
__device__ __forceinline__ int32_t la_column(int32_t lane) {
    const int32_t row = 8 * (lane >> 4) + ((lane & 15) >> 2), c = lane & 3;
    return ROWS ? la_block<D>(row, c) : la_block<D>(row, c >> 1) + 4 * (c & 1);
}
template <typename T, int D, bool ROWS>
__device__ __forceinline__ void la_turned(const uint16_t* tile, int32_t at, int32_t x, int32_t m, uint4 (&out)[LAShape<T, D>::R]) {
    using P = LAShape<T, D>;
    const int32_t first = ROWS ? (at ^ (32 * (m >> 1))) + 4 * (m & 1) : at ^ (16 * m);
#pragma unroll
    for (int l = 0; l < P::R; ++l) {
        const uint16_t* from = tile + l * P::tile + 32 * x * D;
        const la_i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((la_lds_i16x4*)(from + first));
        const la_i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((la_lds_i16x4*)(from + (first ^ 8) + 4 * D));   // four rows on
        const uint2 ua = __builtin_bit_cast(uint2, a), ub = __builtin_bit_cast(uint2, b);
        out[l] = make_uint4(ua.x, ua.y, ub.x, ub.y);
    }
}

// s += tiles of k^T v over a chunk: v's columns (weighted, FP32) as limbs.
template <typename T, int D>
__device__ __forceinline__ void la_enter(const uint16_t* ks, int32_t at, int32_t x, const float (&v)[8], la_f32x4 (&s)[D / 16]) {
    uint4 vw[LA_FORMED];
    la_split8<LA_FORMED>(v, vw);
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
        uint4 ka[LAType<T>::raw];
        la_turned<T, D, true>(ks, at, x, m, ka);
        s[m] = la_mm(ka, vw, s[m]);
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
    bool ready, turned;      // the slots are there already; they hold the states' transposes
    int32_t batches, tokens, heads, kdim, vdim, segments, chunks_per_segment, chunk, reversed;
    int32_t vec_q, vec_k, vec_v;   // elements of one load
    bool wide_out;
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
int la_check_cut(int64_t heads, const LACut& cut, int32_t padded);   // a launch has 2^32 threads at most
int la_check_strides(std::initializer_list<int64_t> token_strides);   // below 2^24 elements
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
// Elements that one load of a row takes.
inline int32_t la_vec(const LATokens& t, int64_t dim, int64_t e) {
    for (int64_t v : {8, 4}) {
        const uintptr_t bytes = v * e < 16 ? v * e : 16;
        if (dim % v == 0 && reinterpret_cast<uintptr_t>(t.data) % bytes == 0 && t.bs % v == 0 && t.ts % v == 0 && t.hs % v == 0)
            return static_cast<int32_t>(v);
    }
    return 1;
}
inline int32_t la_chunk(int32_t io_dtype) { return io_dtype == VH_DTYPE_BF16 ? 64 : 32; }

}  // namespace vh
