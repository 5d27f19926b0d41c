// Linear attention with a decay for each head: prompts in chunks, and single tokens.
//
//   S[t] = g S[t-1] + k[t] v[t]^T,   o[t] = scale q[t]^T S[t],   g = exp(log_decay) of the head
//
// A chunk of n tokens from the state S before it:
//   o[i] = scale (sum_{j <= i} g^(i-j) (q[i] . k[j]) v[j] + g^(i+1) q[i]^T S)
//   S'   = g^n S + sum_j g^(n-1-j) k[j] v[j]^T
// All four products run on the matrix cores (linear_attention.h).  A workgroup walks the chunks of
// a segment of one head of one sequence; wave w has the value columns 16 w .. + 15 of the state in
// its accumulators, which are at once the operand of q S (la_state_row).  The weights g^(i-j) (q . k)
// are shared out by tiles and pass through LDS, the tensors' tiles stand there once and are turned by
// the reads, and the next chunk's values are on their way to registers meanwhile.
//
// Few heads and sequences are cut into segments: a pass for each segment's own last state, a
// join over the segments, and the output pass (la_cut).  Bound by the bytes of q, k, v and o, with vector
// work beside them: 32 x 3136 x 3 heads of 64 in bf16 take 18 + 5 + 44 us, the output pass 154 MB at
// 3.5 TB/s of a copy's 4.9; 1 x 16384 x 16 heads 16 + 9 + 40.  Heads of 128 hold one workgroup a CU and
// wait for latency (8 x 784 x 8 heads: 14 + 6 + 27 us, the output pass 51 MB at 1.9 TB/s).
//
// The gradients are the same form with other operands (linear_attention_backward.hip): `reversed`
// walks the tokens from the last one, where the state is the gradient of S behind a chunk and
// enters with one power of g less.
#include <algorithm>

#include "linear_attention.h"

namespace vh {
namespace {

// A tile (query tile, key tile) of the lower triangle by its number.
__device__ __forceinline__ void la_triangle(int32_t tile, int32_t& it, int32_t& jt) {
    it = static_cast<int32_t>((0x3333222110ull >> (4 * tile)) & 15);
    jt = tile - it * (it + 1) / 2;
}

// Walks a segment's chunks.  OUT: writes outputs; otherwise the segment's last state only.  WIDE: all
// loads take eight values, without the choice at each of them (5 % of a pass).
template <typename T, int D, bool OUT, bool WIDE>
__global__ __launch_bounds__(4 * D, D == 128 ? 2 : 3) void linear_attention_kernel(const LAPass a) {
    using P = LAShape<T, D>;
    constexpr int R = P::R, F = P::F, C = P::C;
    constexpr int TILES = C / 16, STEPS_C = C / 32, STEPS_D = D / 32, UNITS = P::units;
    extern __shared__ __align__(16) unsigned char la_lds[];
    float* entering = reinterpret_cast<float*>(la_lds);                     // [C]: weights of what enters the state
    uint16_t* ks = reinterpret_cast<uint16_t*>(la_lds + P::head);           // [R][C][D]
    uint16_t* vs = ks + R * P::tile;                                        // [R][C][D]
    uint16_t* qs = vs + R * P::tile;                                        // [R][C][D]
    uint16_t* ws = qs + R * P::tile;                                        // [F][C][C]: weights of pairs

    const int32_t tid = static_cast<int32_t>(threadIdx.x), lane = tid & 63;
    const int32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    // heads of a token stand side by side in memory: neighbours run on one XCD
    const uint32_t bid = xcd_remap_any(blockIdx.x, gridDim.x);
    const int32_t head = static_cast<int32_t>(bid % static_cast<uint32_t>(a.heads));
    const uint32_t rest = bid / static_cast<uint32_t>(a.heads);
    const int32_t count = OUT ? a.segments : a.segments - 1;
    const int32_t batch = static_cast<int32_t>(rest / static_cast<uint32_t>(count));
    // states are wanted of all segments but the walk's last one
    const int32_t segment = static_cast<int32_t>(rest % static_cast<uint32_t>(count)) + (!OUT && a.reversed ? 1 : 0);
    const int64_t bh = static_cast<int64_t>(batch) * a.heads + head;
    const int32_t end = __builtin_amdgcn_readfirstlane(la_end(a, batch));
    const int32_t length = a.chunks_per_segment * C;
    const int32_t from = segment * length;
    const int32_t to = a.tokens - from < length ? a.tokens : from + length;      // of all tokens
    const int32_t stop = end < from ? from : end < to ? end : to;                // of the sequence's
    const int32_t last = end > 0 ? (end - 1) / length : 0;                       // segment of the last token
    const int32_t chunks = (stop - from + C - 1) / C;
    const int32_t shift = a.reversed ? 1 : 0;
    const LADecay decay(a.log_decay[head]);

    // staging: a thread takes eight columns of tokens `row`, row + 32, ... of each tensor
    const int32_t col = tid % (D / 8) * 8, row = tid / (D / 8);
    const T* qp = static_cast<const T*>(a.q.data) + batch * a.q.bs + head * a.q.hs;
    const T* kp = static_cast<const T*>(a.k.data) + batch * a.k.bs + head * a.k.hs;
    const T* vp = static_cast<const T*>(a.v.data) + batch * a.v.bs + head * a.v.hs;
    LAOct<T> rq[UNITS], rk[UNITS], rv[UNITS];
    auto fetch = [&](int32_t chunk) {
        const int32_t t0 = from + chunk * C, nt = stop - t0 < C ? stop - t0 : C;
        const T *q = qp + t0 * a.q.ts, *k = kp + t0 * a.k.ts, *v = vp + t0 * a.v.ts;
        // offsets within a chunk fit 32 bits (token strides below 2^24)
        const uint32_t qt = static_cast<uint32_t>(a.q.ts), kt = static_cast<uint32_t>(a.k.ts), vt = static_cast<uint32_t>(a.v.ts);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int32_t i = row + 32 * u;
            const uint32_t t = static_cast<uint32_t>(a.reversed ? nt - 1 - i : i);
            if (OUT) rq[u] = LAOct<T>{};
            rk[u] = rv[u] = LAOct<T>{};
            if (i < nt) {
                if constexpr (OUT) rq[u] = la_load<T, WIDE>(q + (t * qt + col), col, a.kdim, a.vec_q);
                rk[u] = la_load<T, WIDE>(k + (t * kt + col), col, a.kdim, a.vec_k);
                rv[u] = la_load<T, WIDE>(v + (t * vt + col), col, a.vdim, a.vec_v);
            }
        }
    };
    if (chunks > 0) fetch(a.reversed ? chunks - 1 : 0);

    // powers of the decay that a lane needs in every chunk
    float diagonal[4], below[4], leaving[TILES];
    const float p16 = decay.power(16.f), p32 = decay.power(32.f);
    if constexpr (OUT) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t d = n16 - 4 * g - r;   // of a pair in a tile on the diagonal; 16 more in the next one
            diagonal[r] = d >= 0 ? decay.power(static_cast<float>(d)) * a.scale_weight : 0.f;
            below[r] = decay.power(static_cast<float>(d + 16)) * a.scale_weight;
        }
#pragma unroll
        for (int it = 0; it < TILES; ++it) leaving[it] = decay.power(static_cast<float>(16 * it + n16 + 1 - shift)) * a.scale_out;
        // weights of later tokens that share 32 columns with earlier ones stay zero
        for (int32_t i = tid; i < F * P::weights / 2; i += P::threads) reinterpret_cast<uint32_t*>(ws)[i] = 0;
    }

    // the state: key rows la_state_row(m, g, 0 .. 3), value column 16 wave + n16
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
                    if (la_state_row(m, g, r) < a.kdim) s[m][r] = at[la_state_row(m, g, r) * a.state_row];
        }
    } else if (OUT && (a.reversed ? segment < last : true)) {
        const int32_t slot = a.reversed ? segment : segment - 1;
        const float* at = a.slots + (bh * (a.segments - 1) + slot) * D * D;
        if (a.turned) {   // this state's column is a row there: of tile m2, group g2, its last two bits
            const int32_t m2 = 2 * (column >> 5) + ((column >> 2) & 1), g2 = (column >> 3) & 3;
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t c = la_state_row(m, g, r);
                    s[m][r] = at[(((c >> 4) * (D / 16) + m2) * 64 + 16 * g2 + (c & 15)) * 4 + (column & 3)];
                }
        } else {
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
                s[m] = reinterpret_cast<const la_f32x4*>(at)[(wave * (D / 16) + m) * 64 + lane];
        }
    }

    const int32_t at_row = la_block<D>(n16, g), at_weights = la_block<C>(n16, g), to_weights = la_block<C>(n16, g >> 1) + 4 * (g & 1);
    const int32_t k_column = la_column<D, true>(lane), v_column = la_column<D, false>(lane);
    int32_t entered = 0;   // the chunk length that `entering` stands for
    for (int32_t step = 0; step < chunks; ++step) {
        const int32_t chunk = a.reversed ? chunks - 1 - step : step;
        const int32_t t0 = from + chunk * C, nt = stop - t0 < C ? stop - t0 : C;
        __syncthreads();   // the last chunk's tiles have been read
        if (nt != entered) {
            if (tid < C) entering[tid] = tid < nt ? decay.power(static_cast<float>(nt - 1 - tid + shift)) * a.scale_in : 0.f;
            entered = nt;
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if constexpr (OUT) la_stage<T, D>(rq[u], qs, col, row + 32 * u);
            la_stage<T, D>(rk[u], ks, col, row + 32 * u);
            la_stage<T, D>(rv[u], vs, col, row + 32 * u);
        }
        if (step + 1 < chunks) fetch(a.reversed ? chunk - 1 : chunk + 1);
        __syncthreads();

        la_f32x4 o[TILES];
        if constexpr (OUT) {
            // weights of the pairs (query tile it, key tile jt <= it), a tile a wave
#pragma unroll
            for (int32_t first = 0; first < TILES * (TILES + 1) / 2; first += P::waves) {
                const int32_t tile = first + wave;
                if (tile >= TILES * (TILES + 1) / 2) break;
                int32_t it, jt;
                la_triangle(tile, it, jt);
                la_f32x4 w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < STEPS_D; ++x) {
                    uint4 ka[R], qa[R];
                    la_read(ks, P::tile, 16 * jt * D + (at_row ^ (32 * x)), ka);
                    la_read(qs, P::tile, 16 * it * D + (at_row ^ (32 * x)), qa);
                    w = la_mm(ka, qa, w);
                }
                if (it == jt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[r] = n16 < 4 * g + r ? 0.f : w[r] * diagonal[r];
                } else {
                    const float p = it - jt == 1 ? 1.f : it - jt == 2 ? p16 : p32;
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[r] *= below[r] * p;
                }
                uint32_t lo[F], hi[F];
                la_split<F>(w[0], w[1], lo);
                la_split<F>(w[2], w[3], hi);
#pragma unroll
                for (int l = 0; l < F; ++l)
                    *reinterpret_cast<uint2*>(ws + l * P::weights + 16 * it * C + (to_weights ^ (16 * jt))) = make_uint2(lo[l], hi[l]);
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
                    la_read(qs, P::tile, 16 * it * D + (at_row ^ (32 * x)), qa);
                    o[it] = la_mm(sa, qa, o[it]);
                }
            }
#pragma unroll
            for (int it = 0; it < TILES; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[it][r] *= leaving[it];
        }
        // the state behind the chunk
        uint4 va[STEPS_C][R];
#pragma unroll
        for (int x = 0; x < STEPS_C; ++x) la_turned<T, D, false>(vs, v_column, x, wave, va[x]);
        const float whole = decay.power(static_cast<float>(nt));
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[m][r] *= whole;
#pragma unroll
        for (int x = 0; x < STEPS_C; ++x) {
            float v[8];
            la_join8<R>(va[x], v);
            const float4 e0 = *reinterpret_cast<const float4*>(entering + 32 * x + 8 * g);
            const float4 e1 = *reinterpret_cast<const float4*>(entering + 32 * x + 8 * g + 4);
            v[0] *= e0.x; v[1] *= e0.y; v[2] *= e0.z; v[3] *= e0.w;
            v[4] *= e1.x; v[5] *= e1.y; v[6] *= e1.z; v[7] *= e1.w;
            la_enter<T, D>(ks, k_column, x, v, s);
        }
        if constexpr (OUT) {
            __syncthreads();   // all weights are there
#pragma unroll
            for (int it = 0; it < TILES; ++it)
#pragma unroll
                for (int x = 0; x < STEPS_C; ++x)
                    if (32 * x < 16 * (it + 1)) {
                        uint4 wa[F];
                        la_read(ws, P::weights, 16 * it * C + (at_weights ^ (32 * x)), wa);
                        o[it] = la_mm(va[x], wa, o[it]);
                    }
            T* out = static_cast<T*>(a.out) + ((batch * static_cast<int64_t>(a.tokens) + t0) * a.heads + head) * a.vdim;
#pragma unroll
            for (int it = 0; it < TILES; ++it) {
                const int32_t i = 16 * it + n16;
                if (i >= nt) continue;
                const uint32_t t = static_cast<uint32_t>(a.reversed ? nt - 1 - i : i);
                const float v[4] = {o[it][0], o[it][1], o[it][2], o[it][3]};
                la_store(out + (t * static_cast<uint32_t>(a.heads * a.vdim) + 16 * wave + 4 * g), 16 * wave + 4 * g, a.vdim,
                         a.wide_out, v);
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
        for (int32_t t = stop + row; t < to; t += 32)
#pragma unroll
            for (int c = 0; c < 8; c += 4)
                la_store(static_cast<T*>(a.out) + ((batch * static_cast<int64_t>(a.tokens) + t) * a.heads + head) * a.vdim + col + c,
                         col + c, a.vdim, a.wide_out, zeros);
        if (a.new_state != nullptr && (a.reversed ? segment == 0 : segment == last) && column < a.vdim) {
            float* at = a.new_state + bh * a.kdim * a.vdim + column * a.state_col;
#pragma unroll
            for (int m = 0; m < D / 16; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (la_state_row(m, g, r) < a.kdim) at[la_state_row(m, g, r) * a.state_row] = s[m][r];
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
    constexpr int AHEAD = 8;   // loads in flight: the chain is over them, not over memory
    for (int32_t i0 = 0; i0 < slots; i0 += AHEAD) {
        float4 own[AHEAD];
        // slot i belongs to segment i + 1 of a reversed walk and to segment i of the other
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (i0 + i < slots) own[i] = at[static_cast<int64_t>(a.reversed ? slots - 1 - i0 - i : i0 + i) * quads];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (i0 + i >= slots) break;
            const int32_t slot = a.reversed ? slots - 1 - i0 - i : i0 + i;
            int32_t n = end - (a.reversed ? slot + 1 : slot) * tokens;
            n = n < 0 ? 0 : n > tokens ? tokens : n;
            const float p = decay.power(static_cast<float>(n));
            s.x = fmaf(s.x, p, own[i].x);
            s.y = fmaf(s.y, p, own[i].y);
            s.z = fmaf(s.z, p, own[i].z);
            s.w = fmaf(s.w, p, own[i].w);
            at[static_cast<int64_t>(slot) * quads] = s;
        }
    }
}

template <typename T, int D, bool WIDE>
int launch_pass(const LAPass& a, bool states, hipStream_t stream) {
    using P = LAShape<T, D>;
    const int64_t heads = static_cast<int64_t>(a.batches) * a.heads;
    if (a.segments > 1 && !a.ready) {
        linear_attention_kernel<T, D, false, WIDE><<<static_cast<uint32_t>(heads * (a.segments - 1)), P::threads, P::state_lds, stream>>>(a);
        if (int rc = check_launch("linear_attention states")) return rc;
        const int32_t quads = D * D / 4;
        linear_attention_join_kernel<<<static_cast<uint32_t>(la_ceil(heads * quads, 256)), 256, 0, stream>>>(a, quads);
        if (int rc = check_launch("linear_attention join")) return rc;
    }
    if (states) return VH_OK;
    linear_attention_kernel<T, D, true, WIDE><<<static_cast<uint32_t>(heads * a.segments), P::threads, P::lds, stream>>>(a);
    return check_launch("linear_attention");
}

template <typename T>
int launch_typed(const LAPass& a, bool states, hipStream_t stream) {
    const int32_t d = la_padded(a.kdim, a.vdim);
    auto go = [&](auto wide) -> int {
        constexpr bool WIDE = decltype(wide)::value;
        if (d == 32) return launch_pass<T, 32, WIDE>(a, states, stream);
        if (d == 64) return launch_pass<T, 64, WIDE>(a, states, stream);
        return launch_pass<T, 128, WIDE>(a, states, stream);
    };
    if (a.vec_q == 8 && a.vec_k == 8 && a.vec_v == 8) return go(std::true_type{});
    return go(std::false_type{});
}

int run(LAPass& a, int32_t io_dtype, bool states, hipStream_t stream) {
    const int64_t e = dtype_bytes(io_dtype);
    a.vec_q = la_vec(a.q, a.kdim, e);
    a.vec_k = la_vec(a.k, a.kdim, e);
    a.vec_v = la_vec(a.v, a.vdim, e);
    a.wide_out = a.vdim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * e) == 0;
    a.chunk = la_chunk(io_dtype);
    if (io_dtype == VH_DTYPE_F32) return launch_typed<float>(a, states, stream);
    return io_dtype == VH_DTYPE_BF16 ? launch_typed<bf16_t>(a, states, stream) : launch_typed<f16_t>(a, states, stream);
}

}  // namespace

int la_run(LAPass& a, int32_t io_dtype, hipStream_t stream) { return run(a, io_dtype, false, stream); }
int la_states(LAPass& a, int32_t io_dtype, hipStream_t stream) { return run(a, io_dtype, true, stream); }

LACut la_cut(int64_t heads, int64_t N, int32_t padded, int32_t io_dtype) {
    // The time of a cut, in chunks of a workgroup that has its CU to itself: a second and a third one there
    // cost a third each; segments cost a pass for their states, 45 % of the outputs', a launch, and the
    // states' way to memory and back twice, beside chunks that take 0.57 of that time for their own bytes.
    // (bf16 heads of 64: 3.1 us a chunk of one workgroup a CU, 4.5 of two.  96 heads of 49 chunks take 151 us
    // whole, 93 in 3 segments, 71 in 5 and in 7; 304 of 13 take 59 us whole, 60 in 2 segments, 70 in 5.)  `held`: workgroups that the
    // card holds at once, by registers and LDS; more of them wait for the end of others.
    const int64_t held = padded == 32 ? 1024 : padded == 64 ? 768 : 256, cus = 256;
    const int64_t chunks = la_ceil(N, la_chunk(io_dtype));
    const double state = 4.0 * padded / (la_chunk(io_dtype) * dtype_bytes(io_dtype)) * 0.57 / cus;
    LACut best{1, static_cast<int32_t>(chunks)};
    double least = 0.0;
    // candidates: one to three segments, and as many as k workgroups on every CU are
    for (int64_t k = -2; k <= 2 * held / cus; ++k) {
        const int64_t wanted = std::min(chunks, std::max<int64_t>(1, k <= 0 ? k + 3 : k * cus / heads));
        const int64_t each = la_ceil(chunks, wanted), segments = la_ceil(chunks, each), groups = heads * segments;
        const int64_t rounds = la_ceil(groups, held), together = rounds > 1 ? held / cus : la_ceil(groups, cus);
        double cost = static_cast<double>(rounds * each) * (1.0 + (together - 1) / 3.0);
        if (segments > 1) cost = cost * 1.45 + 1.0 + state * static_cast<double>(heads * (segments - 1));
        if (k == -2 || cost < least) {
            least = cost;
            best = {static_cast<int32_t>(segments), static_cast<int32_t>(each)};
        }
    }
    return best;
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
    VH_REQUIRE(heads * value_dim < (1ll << 24) && heads * key_dim < (1ll << 24), VH_ERR_SHAPE,
               "linear attention: a token's %lld heads are out of range", (long long)heads);
    return VH_OK;
}

int la_check_cut(int64_t heads, const LACut& cut, int32_t padded) {
    // 4 padded threads a workgroup of a pass; the join has one for every four values of a head's state
    VH_REQUIRE(heads * cut.segments * 4 * padded < (1ll << 32) &&
                   (cut.segments == 1 || heads * padded * padded / 4 <= (1ll << 32) - 256), VH_ERR_SHAPE,
               "linear attention: %lld heads in %lld segments are out of range", (long long)heads, (long long)cut.segments);
    return VH_OK;
}

int la_check_strides(std::initializer_list<int64_t> token_strides) {
    for (int64_t t : token_strides)
        VH_REQUIRE(t >= 0 && t < (1ll << 24), VH_ERR_SHAPE, "linear attention: a token stride of %lld is out of range", (long long)t);
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
// state's bytes, read and written once: 200 x 8 heads of 128 x 128 take 33 us (6.3 TB/s, part of them in
// the last-level cache), 64 x 16 heads of 64 x 64 6.7 us.
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
    if (int rc = la_check_strides({q_token, k_token, v_token})) return rc;
    VH_REQUIRE(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr && out != nullptr, VH_ERR_ARG,
               "q, k, v, log_decay and out must not be null");
    VH_REQUIRE(!overlapping(state, new_state, B * heads * key_dim * value_dim * 4), VH_ERR_ARG,
               "state and new_state must not overlap");
    const int32_t padded = la_padded(key_dim, value_dim);
    const LACut cut = la_cut(B * heads, N, padded, io_dtype);
    if (int rc = la_check_cut(B * heads, cut, padded)) return rc;
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
