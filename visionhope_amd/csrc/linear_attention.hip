// Linear attention with a decay for each head: prompts in chunks, and single tokens.
//
//   S[t] = g S[t-1] + k[t] v[t]^T,   o[t] = scale q[t]^T S[t],   g = exp(log_decay) of the head
//
// A chunk of n tokens from the state S before it:
//   o[i] = scale (sum_{j <= i} g^(i-j) (q[i] . k[j]) v[j] + g^(i+1) q[i]^T S)
//   S'   = g^n S + sum_j g^(n-1-j) k[j] v[j]^T
// All four products run on the matrix cores (linear_attention.h).  A workgroup walks the chunks of
// a segment of one head of one sequence; wave w has the value columns 16 w .. + 15 of the state in
// its accumulators, which are at once the operand of q S (the key index is stored in the order
// that they have).  The weights g^(i-j) (q . k) are shared out by tiles and pass through LDS.
//
// Few heads and sequences are cut into segments: a pass for each segment's own last state, a
// join over the segments, and the output pass.
//
// The gradients are the same form with other operands (linear_attention_backward.hip): `reversed`
// walks the tokens from the last one, where the state is the gradient of S behind a chunk and
// enters with one power of g less.
#include "linear_attention.h"

namespace vh {
namespace {

// Walks a segment's chunks.  OUT: writes outputs; otherwise the segment's last state only.
template <typename T, int D, bool OUT>
__global__ __launch_bounds__(4 * D) void linear_attention_kernel(const LAPass a) {
    using P = LAShape<T, D>;
    constexpr int R = P::R, F = P::F, C = P::C, ORDER = LAType<T>::order;
    constexpr int TILES = C / 16, STEPS_C = C / 32, STEPS_D = D / 32, UNIT = C / 16;
    extern __shared__ __align__(16) unsigned char la_lds[];
    float* powers = reinterpret_cast<float*>(la_lds);                       // [C + 1]
    uint16_t* kt = reinterpret_cast<uint16_t*>(la_lds + 512);               // [R][D][C]: keys, turned
    uint16_t* vt = kt + R * P::turned_tile;                                 // [R][D][C]: values, turned
    uint16_t* qs = vt + R * P::turned_tile;                                 // [R][C][D]: key index in the states' order
    uint16_t* ks = qs + R * P::tokens_tile;                                 // [R][C][D]: the same
    uint16_t* ws = ks + R * P::tokens_tile;                                 // [F][C][C]: weights

    const int32_t tid = static_cast<int32_t>(threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int32_t n16 = lane & 15, g = lane >> 4;
    // heads of a token stand side by side in memory: neighbours run on one XCD
    const uint32_t bid = xcd_remap_any(blockIdx.x, gridDim.x);
    const int32_t head = static_cast<int32_t>(bid % static_cast<uint32_t>(a.heads));
    const uint32_t rest = bid / static_cast<uint32_t>(a.heads);
    const int32_t count = OUT ? a.segments : a.segments - 1;
    const int32_t batch = static_cast<int32_t>(rest / static_cast<uint32_t>(count));
    // states are wanted of all segments but the walk's last one
    const int32_t segment = static_cast<int32_t>(rest % static_cast<uint32_t>(count)) + (!OUT && a.reversed ? 1 : 0);
    const int64_t bh = static_cast<int64_t>(batch) * a.heads + head;
    const int32_t end = la_end(a, batch);
    const int32_t length = a.chunks_per_segment * C;
    const int32_t from = segment * length;
    const int32_t to = a.tokens - from < length ? a.tokens : from + length;      // of all tokens
    const int32_t stop = end < from ? from : end < to ? end : to;                // of the sequence's
    const int32_t last = end > 0 ? (end - 1) / length : 0;                       // segment of the last token
    const LADecay decay(a.log_decay[head]);
    if (tid <= C) powers[tid] = decay.power(static_cast<float>(tid));
    if constexpr (OUT) {   // weights of later tokens that share 32 columns with earlier ones stay zero
        for (int32_t i = tid; i < F * P::weights_tile / 2; i += P::threads) reinterpret_cast<uint32_t*>(ws)[i] = 0;
    }

    // the state: key rows 16 m + 4 g .. + 3, value column 16 wave + n16
    la_f32x4 s[D / 16];
#pragma unroll
    for (int m = 0; m < D / 16; ++m) s[m] = la_f32x4{0.f, 0.f, 0.f, 0.f};
    const int32_t column = 16 * wave + n16;
    const bool starts = a.reversed ? segment == last : segment == 0;
    if (starts) {
        if (a.state != nullptr && column < a.vdim) {
            const float* at = a.state + bh * a.kdim * a.vdim + column * a.state_col;
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * m + 4 * g + r < a.kdim) s[m][r] = at[(16 * m + 4 * g + r) * a.state_row];
        }
    } else if (OUT && (a.reversed ? segment < last : true)) {
        const int32_t slot = a.reversed ? segment : segment - 1;
        const la_f32x4* at = reinterpret_cast<const la_f32x4*>(a.slots + (bh * (a.segments - 1) + slot) * D * D) +
                             wave * (D / 16) * 64 + lane;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) s[m] = at[m * 64];
    }

    // staging: a thread takes four columns of UNIT tokens of each tensor
    const int32_t cu = tid % (D / 4), tu = tid / (D / 4);
    const T* qp = static_cast<const T*>(a.q.data) + batch * a.q.bs + head * a.q.hs;
    const T* kp = static_cast<const T*>(a.k.data) + batch * a.k.bs + head * a.k.hs;
    const T* vp = static_cast<const T*>(a.v.data) + batch * a.v.bs + head * a.v.hs;
    LAQuad<T> rq[UNIT], rk[UNIT], rv[UNIT];
    const int32_t chunks = (stop - from + C - 1) / C;
    auto fetch = [&](int32_t chunk) {
        const int32_t t0 = from + chunk * C, nt = stop - t0 < C ? stop - t0 : C;
#pragma unroll
        for (int u = 0; u < UNIT; ++u) {
            const int32_t i = tu * UNIT + u;
            const int64_t t = a.reversed ? t0 + nt - 1 - i : t0 + i;
            const bool live = i < nt;
            if constexpr (OUT) rq[u] = la_load(qp + t * a.q.ts, 4 * cu, a.kdim, a.wide_q, live);
            rk[u] = la_load(kp + t * a.k.ts, 4 * cu, a.kdim, a.wide_k, live);
            rv[u] = la_load(vp + t * a.v.ts, 4 * cu, a.vdim, a.wide_v, live);
        }
    };
    if (chunks > 0) fetch(a.reversed ? chunks - 1 : 0);
    const int32_t shift = a.reversed ? 1 : 0;
    for (int32_t step = 0; step < chunks; ++step) {
        const int32_t chunk = a.reversed ? chunks - 1 - step : step;
        const int32_t t0 = from + chunk * C, nt = stop - t0 < C ? stop - t0 : C;
        __syncthreads();   // the last chunk's tiles have been read
        if constexpr (OUT) la_stage<T, D>(rq, qs, nullptr, cu, tu);
        la_stage<T, D>(rk, OUT ? ks : nullptr, kt, cu, tu);
        la_stage<T, D>(rv, nullptr, vt, cu, tu);
        if (step + 1 < chunks) fetch(a.reversed ? chunk - 1 : chunk + 1);
        __syncthreads();

        la_f32x4 o[TILES];
        if constexpr (OUT) {
            // weights of the pairs (query tile it, key tile jt <= it), a tile a wave
            for (int32_t tile = wave; tile < TILES * (TILES + 1) / 2; tile += P::waves) {
                int32_t it = 0;
                while ((it + 1) * (it + 2) / 2 <= tile) ++it;
                const int32_t jt = tile - it * (it + 1) / 2;
                la_f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < STEPS_D; ++x) {
                    uint4 ka[R], qa[R];
                    la_read(ks, P::tokens_tile, (16 * jt + n16) * P::row_d + 32 * x + 8 * g, ka);
                    la_read(qs, P::tokens_tile, (16 * it + n16) * P::row_d + 32 * x + 8 * g, qa);
                    w = la_mm<(R == 1 ? 0 : 2)>(ka, qa, w);
                }
                const int32_t i = 16 * it + n16, j = 16 * jt + 4 * g;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = j + r <= i ? w[r] * (powers[i - j - r < 0 ? 0 : i - j - r] * a.scale_weight) : 0.f;
                uint32_t lo[F], hi[F];
                la_split<F>(v[0], v[1], lo);
                la_split<F>(v[2], v[3], hi);
#pragma unroll
                for (int l = 0; l < F; ++l)
                    *reinterpret_cast<uint2*>(ws + l * P::weights_tile + i * P::row_c + j) = make_uint2(lo[l], hi[l]);
            }
            // what comes from the state: value rows, token columns
#pragma unroll
            for (int it = 0; it < TILES; ++it) o[it] = la_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < STEPS_D; ++x) {
                uint4 sa[F];
                const float v[8] = {s[2 * x][0], s[2 * x][1], s[2 * x][2], s[2 * x][3],
                                    s[2 * x + 1][0], s[2 * x + 1][1], s[2 * x + 1][2], s[2 * x + 1][3]};
                la_split8<F>(v, sa);
#pragma unroll
                for (int it = 0; it < TILES; ++it) {
                    uint4 qa[R];
                    la_read(qs, P::tokens_tile, (16 * it + n16) * P::row_d + 32 * x + 8 * g, qa);
                    o[it] = la_mm<ORDER>(sa, qa, o[it]);
                }
            }
#pragma unroll
            for (int it = 0; it < TILES; ++it) {
                const float p = powers[16 * it + n16 + 1 - shift] * a.scale_out;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[it][r] *= p;
            }
        }
        // the state behind the chunk
        uint4 va[STEPS_C][R];
#pragma unroll
        for (int x = 0; x < STEPS_C; ++x) la_read(vt, P::turned_tile, column * P::row_c + 32 * x + 8 * g, va[x]);
        const float whole = powers[nt];
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[m][r] *= whole;
#pragma unroll
        for (int x = 0; x < STEPS_C; ++x) {
            float v[8];
            la_join8<R>(va[x], v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int32_t m = nt - 1 - (32 * x + 8 * g + i) + shift;
                v[i] *= powers[m < 0 ? 0 : m] * a.scale_in;
            }
            uint4 vw[LA_STATE_LIMBS];
            la_split8<LA_STATE_LIMBS>(v, vw);
#pragma unroll
            for (int m = 0; m < D / 16; ++m) {
                uint4 ka[R];
                la_read(kt, P::turned_tile, (16 * m + n16) * P::row_c + 32 * x + 8 * g, ka);
                s[m] = la_mm<2>(ka, vw, s[m]);
            }
        }
        if constexpr (OUT) {
            __syncthreads();   // all weights are there
#pragma unroll
            for (int it = 0; it < TILES; ++it)
#pragma unroll
                for (int x = 0; x < STEPS_C; ++x)
                    if (32 * x < 16 * (it + 1)) {
                        uint4 wa[F];
#pragma unroll
                        for (int l = 0; l < F; ++l)
                            wa[l] = *reinterpret_cast<const uint4*>(ws + l * P::weights_tile + (16 * it + n16) * P::row_c + 32 * x + 8 * g);
                        o[it] = la_mm<ORDER>(va[x], wa, o[it]);
                    }
#pragma unroll
            for (int it = 0; it < TILES; ++it) {
                const int32_t i = 16 * it + n16;
                if (i >= nt) continue;
                const int64_t t = a.reversed ? t0 + nt - 1 - i : t0 + i;
                const float v[4] = {o[it][0], o[it][1], o[it][2], o[it][3]};
                la_store(static_cast<T*>(a.out) + ((batch * static_cast<int64_t>(a.tokens) + t) * a.heads + head) * a.vdim,
                         16 * wave + 4 * g, a.vdim, a.wide_out, v);
            }
        }
    }

    if constexpr (!OUT) {
        const int32_t slot = a.reversed ? segment - 1 : segment;
        la_f32x4* at = reinterpret_cast<la_f32x4*>(a.slots + (bh * (a.segments - 1) + slot) * D * D) + wave * (D / 16) * 64 + lane;
#pragma unroll
        for (int m = 0; m < D / 16; ++m) at[m * 64] = s[m];
    } else {
        const float zeros[4] = {0.f, 0.f, 0.f, 0.f};   // tokens behind the sequence's end
        for (int32_t t = stop + tu; t < to; t += 16)
            la_store(static_cast<T*>(a.out) + ((batch * static_cast<int64_t>(a.tokens) + t) * a.heads + head) * a.vdim, 4 * cu,
                     a.vdim, a.wide_out, zeros);
        if (a.new_state != nullptr && (a.reversed ? segment == 0 : segment == last) && column < a.vdim) {
            float* at = a.new_state + bh * a.kdim * a.vdim + column * a.state_col;
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * m + 4 * g + r < a.kdim) at[(16 * m + 4 * g + r) * a.state_row] = s[m][r];
        }
    }
}

// States at the segments' starts from the segments' own last ones, in the order of the walk.
__global__ __launch_bounds__(256) void linear_attention_join_kernel(const LAPass a, int32_t quads) {
    const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t bh = index / quads;
    if (bh >= static_cast<int64_t>(a.batches) * a.heads) return;
    const int32_t head = static_cast<int32_t>(bh % a.heads);
    const int32_t tokens = a.chunks_per_segment * a.chunk;
    const LADecay decay(a.log_decay[head]);
    const int32_t slots = a.segments - 1;
    const int32_t end = la_end(a, static_cast<int32_t>(bh / a.heads));
    float4* at = reinterpret_cast<float4*>(a.slots) + bh * slots * quads + index % quads;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int32_t i = 0; i < slots; ++i) {
        // slot i belongs to segment i + 1 of a reversed walk and to segment i of the other
        const int32_t slot = a.reversed ? slots - 1 - i : i;
        const int32_t first = (a.reversed ? slot + 1 : slot) * tokens;
        int32_t n = end - first;
        n = n < 0 ? 0 : n > tokens ? tokens : n;
        const float p = decay.power(static_cast<float>(n));
        const float4 own = at[static_cast<int64_t>(slot) * quads];
        s.x = fmaf(s.x, p, own.x);
        s.y = fmaf(s.y, p, own.y);
        s.z = fmaf(s.z, p, own.z);
        s.w = fmaf(s.w, p, own.w);
        at[static_cast<int64_t>(slot) * quads] = s;
    }
}

template <typename T, int D>
int launch_pass(const LAPass& a, bool states, hipStream_t stream) {
    using P = LAShape<T, D>;
    const int64_t heads = static_cast<int64_t>(a.batches) * a.heads;
    if (a.segments > 1) {
        linear_attention_kernel<T, D, false><<<static_cast<uint32_t>(heads * (a.segments - 1)), P::threads, P::state_lds, stream>>>(a);
        if (int rc = check_launch("linear_attention states")) return rc;
        const int32_t quads = D * D / 4;
        linear_attention_join_kernel<<<static_cast<uint32_t>(la_ceil(heads * quads, 256)), 256, 0, stream>>>(a, quads);
        if (int rc = check_launch("linear_attention join")) return rc;
    }
    if (states) return VH_OK;
    linear_attention_kernel<T, D, true><<<static_cast<uint32_t>(heads * a.segments), P::threads, P::lds, stream>>>(a);
    return check_launch("linear_attention");
}

template <typename T>
int launch_typed(const LAPass& a, bool states, hipStream_t stream) {
    const int32_t d = la_padded(a.kdim, a.vdim);
    if (d == 32) return launch_pass<T, 32>(a, states, stream);
    if (d == 64) return launch_pass<T, 64>(a, states, stream);
    return launch_pass<T, 128>(a, states, stream);
}

int run(LAPass& a, int32_t io_dtype, bool states, hipStream_t stream) {
    const int64_t e = dtype_bytes(io_dtype);
    a.wide_q = la_wide(a.q, a.kdim, e);
    a.wide_k = la_wide(a.k, a.kdim, e);
    a.wide_v = la_wide(a.v, a.vdim, e);
    a.wide_out = a.vdim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * e) == 0;
    a.chunk = la_chunk(io_dtype);
    if (io_dtype == VH_DTYPE_F32) return launch_typed<float>(a, states, stream);
    return io_dtype == VH_DTYPE_BF16 ? launch_typed<bf16_t>(a, states, stream) : launch_typed<f16_t>(a, states, stream);
}

}  // namespace

int la_run(LAPass& a, int32_t io_dtype, hipStream_t stream) { return run(a, io_dtype, false, stream); }
int la_states(LAPass& a, int32_t io_dtype, hipStream_t stream) { return run(a, io_dtype, true, stream); }

LACut la_cut(int64_t heads, int64_t N, int32_t padded, int32_t io_dtype) {
    // Workgroups that the card holds at once (LDS: four, two and one a CU), and a half more, so
    // that ragged segments even out.
    const int64_t wanted = padded == 32 ? 1536 : padded == 64 ? 768 : 384;
    const int64_t chunks = la_ceil(N, la_chunk(io_dtype));
    int64_t segments = la_ceil(wanted, heads);
    segments = segments < chunks ? segments : chunks;
    const int64_t each = la_ceil(chunks, segments);
    return {static_cast<int32_t>(la_ceil(chunks, each)), static_cast<int32_t>(each)};
}

size_t la_slots_bytes(int64_t heads, const LACut& cut, int32_t padded) {
    return static_cast<size_t>(heads) * (cut.segments - 1) * padded * padded * sizeof(float);
}

int la_check_sizes(int32_t io_dtype, int64_t B, int64_t N, int64_t heads, int64_t key_dim, int64_t value_dim) {
    VH_REQUIRE(valid_dtype(io_dtype), VH_ERR_DTYPE, "unsupported io_dtype %d", io_dtype);
    VH_REQUIRE(B > 0 && N > 0 && heads > 0 && key_dim > 0 && value_dim > 0, VH_ERR_SHAPE,
               "linear attention needs nonempty sequences, got %lld x %lld x %lld, heads of %lld and %lld", (long long)B,
               (long long)N, (long long)heads, (long long)key_dim, (long long)value_dim);
    VH_REQUIRE(key_dim <= LA_MAX_DIM && value_dim <= LA_MAX_DIM, VH_ERR_SHAPE,
               "linear attention supports heads of up to %lld, got %lld and %lld", (long long)LA_MAX_DIM,
               (long long)key_dim, (long long)value_dim);
    // token numbers and workgroup numbers are 32 bits wide
    VH_REQUIRE(N < (1ll << 30) && B < (1ll << 24) && heads < (1ll << 24) && B * heads < (1ll << 22), VH_ERR_SHAPE,
               "linear attention: %lld sequences of %lld heads and %lld tokens are out of range", (long long)B,
               (long long)heads, (long long)N);
    return VH_OK;
}

namespace {

struct LAStep {
    LATokens q, k, v;   // ts unused
    const float *log_decay, *state;
    float* new_state;
    void* out;
    float scale;
    int32_t heads, kdim, vdim;
};

// One token.  A workgroup takes up to 64 value columns of one head: 16 lanes of four columns (or
// 64 of one) by row groups that walk the key index; the row groups' sums meet in LDS.  Bound by the
// state's bytes, read and written once.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void linear_attention_step_kernel(const LAStep a) {
    constexpr int LANES = 64 / VEC, GROUPS = 256 / LANES;
    __shared__ float ks[LA_MAX_DIM], qs[LA_MAX_DIM];
    __shared__ float sums[GROUPS][64];
    const int64_t bh = blockIdx.x;
    const int32_t head = static_cast<int32_t>(bh % a.heads);
    const int64_t batch = bh / a.heads;
    const T* q = static_cast<const T*>(a.q.data) + batch * a.q.bs + head * a.q.hs;
    const T* k = static_cast<const T*>(a.k.data) + batch * a.k.bs + head * a.k.hs;
    const T* v = static_cast<const T*>(a.v.data) + batch * a.v.bs + head * a.v.hs;
    const float decay = LADecay(a.log_decay[head]).power(1.f);
    if (threadIdx.x < static_cast<uint32_t>(a.kdim)) {
        ks[threadIdx.x] = to_f32(k[threadIdx.x]);
        qs[threadIdx.x] = to_f32(q[threadIdx.x]) * a.scale;
    }
    const int32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const int32_t col = (static_cast<int32_t>(blockIdx.y) * LANES + lane) * VEC;
    const bool live = col < a.vdim;
    float vv[VEC], acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        vv[i] = live ? to_f32(v[col + i]) : 0.f;
        acc[i] = 0.f;
    }
    __syncthreads();
    const int64_t base = bh * a.kdim * a.vdim + col;
    if (live) {
#pragma unroll 4
        for (int32_t d = group; d < a.kdim; d += GROUPS) {
            const int64_t at = base + static_cast<int64_t>(d) * a.vdim;
            float s[VEC];
            if constexpr (VEC == 4) {
                const float4 r = *reinterpret_cast<const float4*>(a.state + at);
                s[0] = r.x; s[1] = r.y; s[2] = r.z; s[3] = r.w;
            } else {
                s[0] = a.state[at];
            }
            const float kd = ks[d], qd = qs[d];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                s[i] = fmaf(kd, vv[i], decay * s[i]);
                acc[i] = fmaf(qd, s[i], acc[i]);
            }
            if constexpr (VEC == 4) *reinterpret_cast<float4*>(a.new_state + at) = make_float4(s[0], s[1], s[2], s[3]);
            else a.new_state[at] = s[0];
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) sums[group][lane * VEC + i] = acc[i];
    __syncthreads();
    const int32_t out = static_cast<int32_t>(blockIdx.y) * 64 + threadIdx.x;
    if (threadIdx.x < 64 && out < a.vdim) {
        float sum = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) sum += sums[g][threadIdx.x];
        static_cast<T*>(a.out)[bh * a.vdim + out] = from_f32<T>(sum);
    }
}

template <typename T>
int launch_step(const LAStep& a, int64_t B, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(B * a.heads), static_cast<uint32_t>(la_ceil(a.vdim, 64)));
    const bool wide = a.vdim % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(a.new_state) % 16 == 0;
    if (wide) linear_attention_step_kernel<T, 4><<<grid, 256, 0, stream>>>(a);
    else linear_attention_step_kernel<T, 1><<<grid, 256, 0, stream>>>(a);
    return check_launch("linear_attention step");
}

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_linear_attention_workspace_bytes(int64_t B, int64_t N, int64_t heads, int64_t key_dim, int64_t value_dim,
                                           int32_t io_dtype) {
    using namespace vh;
    if (la_check_sizes(io_dtype, B, N, heads, key_dim, value_dim) != VH_OK) return 0;
    const int32_t padded = la_padded(key_dim, value_dim);
    return la_slots_bytes(B * heads, la_cut(B * heads, N, padded, io_dtype), padded);
}

int vh_linear_attention_forward(
    const void* q, int64_t q_batch, int64_t q_token, int64_t q_head, const void* k, int64_t k_batch, int64_t k_token,
    int64_t k_head, const void* v, int64_t v_batch, int64_t v_token, int64_t v_head, int32_t io_dtype,
    const float* log_decay, float scale, const float* state, const int32_t* lengths, void* out, float* new_state,
    int64_t B, int64_t N, int64_t heads, int64_t key_dim, int64_t value_dim, void* workspace, size_t workspace_bytes,
    void* stream) {
    using namespace vh;
    if (int rc = la_check_sizes(io_dtype, B, N, heads, key_dim, value_dim)) return rc;
    VH_REQUIRE(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr && out != nullptr, VH_ERR_ARG,
               "q, k, v, log_decay and out must not be null");
    VH_REQUIRE(!overlapping(state, new_state, B * heads * key_dim * value_dim * 4), VH_ERR_ARG,
               "state and new_state must not overlap");
    const int32_t padded = la_padded(key_dim, value_dim);
    const LACut cut = la_cut(B * heads, N, padded, io_dtype);
    const size_t need = la_slots_bytes(B * heads, cut, padded);
    VH_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               VH_ERR_WORKSPACE, "linear attention needs an aligned workspace of %zu bytes, got %zu", need, workspace_bytes);
    LAPass a{};
    a.q = {q, q_batch, q_token, q_head};
    a.k = {k, k_batch, k_token, k_head};
    a.v = {v, v_batch, v_token, v_head};
    a.out = out;
    a.log_decay = log_decay;
    a.scale_weight = a.scale_out = scale;
    a.scale_in = 1.f;
    a.state = state;
    a.new_state = new_state;
    a.state_row = value_dim;
    a.state_col = 1;
    a.lengths = lengths;
    a.slots = static_cast<float*>(workspace);
    a.batches = static_cast<int32_t>(B);
    a.tokens = static_cast<int32_t>(N);
    a.heads = static_cast<int32_t>(heads);
    a.kdim = static_cast<int32_t>(key_dim);
    a.vdim = static_cast<int32_t>(value_dim);
    a.segments = cut.segments;
    a.chunks_per_segment = cut.each;
    return la_run(a, io_dtype, static_cast<hipStream_t>(stream));
}

int vh_linear_attention_step(
    const void* q, int64_t q_batch, int64_t q_head, const void* k, int64_t k_batch, int64_t k_head, const void* v,
    int64_t v_batch, int64_t v_head, int32_t io_dtype, const float* log_decay, float scale, const float* state,
    float* new_state, void* out, int64_t B, int64_t heads, int64_t key_dim, int64_t value_dim, void* stream) {
    using namespace vh;
    if (int rc = la_check_sizes(io_dtype, B, 1, heads, key_dim, value_dim)) return rc;
    VH_REQUIRE(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr && state != nullptr &&
                   new_state != nullptr && out != nullptr, VH_ERR_ARG,
               "q, k, v, log_decay, state, new_state and out must not be null");
    VH_REQUIRE(state == new_state || !overlapping(state, new_state, B * heads * key_dim * value_dim * 4), VH_ERR_ARG,
               "state and new_state must be the same memory or not overlap");
    LAStep a{};
    a.q = {q, q_batch, 0, q_head};
    a.k = {k, k_batch, 0, k_head};
    a.v = {v, v_batch, 0, v_head};
    a.log_decay = log_decay;
    a.state = state;
    a.new_state = new_state;
    a.out = out;
    a.scale = scale;
    a.heads = static_cast<int32_t>(heads);
    a.kdim = static_cast<int32_t>(key_dim);
    a.vdim = static_cast<int32_t>(value_dim);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (io_dtype == VH_DTYPE_F32) return launch_step<float>(a, B, s);
    return io_dtype == VH_DTYPE_BF16 ? launch_step<bf16_t>(a, B, s) : launch_step<f16_t>(a, B, s);
}

}  // extern "C"
