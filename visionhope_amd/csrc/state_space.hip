// Selective state space scan: forward of a prompt and the single-token step.
//
//   dt = softplus(dt_raw + dt_bias)                       per token and channel
//   h[n] = exp(dt A[n]) h[n] + dt x B[n]                  S states a channel, FP32
//   y = (sum_n C[n] h[n] + D x) silu(gate)
//
// A line of tokens is serial, so long lines are cut into chunks that run side by side: one
// pass gives every chunk's state from a zero start and its sum of dt (the chunk's decay is
// exp(A sum dt)), a join carries the states over the chunk boundaries, and the pass that
// computes y starts from them.  With enough sequences and channels the line stays whole and
// the first pass falls away.
//
// Bound by the issue of vector instructions.  A state of a token takes an exponential and four
// products or sums (the output pass; three in the first), so 16 states take about 75 of the
// output pass's 118 instructions a token and wave; softplus, SiLU and the conversions take the
// rest.  A prompt of 1 x 16384 x 1024, 16 states, bf16: 54 + 13 + 72 us where the bytes need 28;
// the vector unit is active for 87 and 83 % of the passes.  In training, which also writes the
// kept states: 64 + 15 + 93 us at 32 x 3136 x 192 (bytes 48).
#include "state_space.h"

namespace vh {
namespace {

// OUT: the output pass; otherwise the pass for the chunks' own states.  One lane a channel: a
// token's B and C stand in scalar registers and its sum over the states needs no other lane.
// (Of the second's time at 1 x 16384 x 1024 the exponentials are a fifth, softplus
// and SiLU an eighth.)
template <typename T, typename BCT, int S, bool OUT>
__global__ __launch_bounds__(64) void state_space_chunk_kernel(const SSArgs a) {
    const SSPlace p = ss_place(a);
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;
    float A2[S], h[S];
    ss_rates<S>(a, p.channel, A2);
    const float bias = a.dt_bias != nullptr ? a.dt_bias[p.channel] : 0.f;
    const float D = OUT && a.D != nullptr ? a.D[p.channel] : 0.f;
    if (OUT && p.chunk > 0) {
        const float* from = a.slots + (static_cast<int64_t>(p.batch) * (a.chunks - 1) + p.chunk - 1) * S * cp + p.column;
#pragma unroll
        for (int n = 0; n < S; ++n) h[n] = from[n * cp];
    } else if (OUT && a.state != nullptr) {
        const float* from = a.state + (static_cast<int64_t>(p.batch) * a.channels + p.channel) * a.states;
#pragma unroll
        for (int n = 0; n < S; ++n) h[n] = n < a.states ? from[n] : 0.f;
    } else {
#pragma unroll
        for (int n = 0; n < S; ++n) h[n] = 0.f;
    }
    const uint32_t lane_at = static_cast<uint32_t>(p.channel) * sizeof(T);
    const bool gated = OUT && a.gate.data != nullptr, soft = a.softplus != 0;
    const T* x = ss_tokens<T>(a.x, p);
    const T* dt = ss_tokens<T>(a.dt, p);
    const T* gate = gated ? ss_tokens<T>(a.gate, p) : x;
    const int64_t gate_ts = gated ? a.gate.ts : a.x.ts;
    const int64_t b0 = p.batch * a.b.bs + p.t0 * a.b.ts + static_cast<int64_t>(p.group) * S;
    const int64_t c0 = p.batch * a.c.bs + p.t0 * a.c.ts + static_cast<int64_t>(p.group) * S;
    const int64_t out0 = (static_cast<int64_t>(p.batch) * a.tokens + p.t0) * a.channels;
    const int32_t count = p.te - p.t0;
    float total = 0.f;

    // B and C of a token are loaded during the one before it where the scalar registers hold two
    // rows of each; the barrier keeps the compiler from loading the rows of all the tokens of
    // an iteration first and moving them to vector registers.
    constexpr bool AHEAD = S * sizeof(BCT) <= 64;
    SSRow<BCT, S> bn, cn;
    auto rows = [&](int32_t t) {
        bn.load(a.b.data, b0 + t * a.b.ts);
        if (OUT) cn.load(a.c.data, c0 + t * a.c.ts);
    };
    auto token = [&](T xr, T dr, T gr, int32_t t) {
        if (!AHEAD) rows(t);
        const SSRow<BCT, S> b = bn, c = cn;
        if (AHEAD) {
            rows(t + 1 < count ? t + 1 : t);
            __builtin_amdgcn_sched_barrier(0);
        }
        const float raw = to_f32(dr) + bias, xv = to_f32(xr), z = to_f32(gr);
        const float plus = ss_softplus(raw), step = soft ? plus : raw;   // no branch in the loop
        const float dtx = step * xv;
        float acc = D * xv;
        if (!OUT) total += step;
#pragma unroll
        for (int n = 0; n < S; ++n) {
            h[n] = fmaf(dtx, b[n], h[n] * __builtin_amdgcn_exp2f(step * A2[n]));
            if (OUT) acc = fmaf(c[n], h[n], acc);
        }
        const float silu = z * sigmoid_fast(z);
        if (OUT) store_at<T>(a.y, out0 + static_cast<int64_t>(t) * a.channels, lane_at, acc * (gated ? silu : 1.f));
        __builtin_amdgcn_sched_barrier(0);
    };
    T xn[SS_UNROLL], dn[SS_UNROLL], gn[SS_UNROLL];
    auto fetch = [&](int32_t t) {
        const uint32_t at = opaque(lane_at);
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) {
            const int64_t i = t + u < count ? t + u : count - 1;   // a token of the sequence
            xn[u] = load_at(x + i * a.x.ts, at);
            dn[u] = load_at(dt + i * a.dt.ts, at);
            if (OUT) gn[u] = load_at(gate + i * gate_ts, at);
        }
    };
    if (count > 0) {
        fetch(0);
        if (AHEAD) rows(0);
    }
    int32_t t = 0;
    WaveTurns turns(count);
    for (; t < count; t += SS_UNROLL) {
        turns.left(count - t);
        if (OUT && a.kept != nullptr && t % SS_BLOCK == 0) {
            float* to = a.kept + (static_cast<int64_t>(p.batch) * a.blocks + (p.t0 + t) / SS_BLOCK) * S * cp + p.column;
#pragma unroll
            for (int n = 0; n < S; ++n) to[n * cp] = h[n];
        }
        if (t + SS_UNROLL > count) break;
        T xr[SS_UNROLL], dr[SS_UNROLL], gr[SS_UNROLL];
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) { xr[u] = xn[u]; dr[u] = dn[u]; gr[u] = gn[u]; }
        fetch(t + SS_UNROLL);
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) token(xr[u], dr[u], gr[u], t + u);
    }
#pragma unroll
    for (int u = 0; u < SS_UNROLL - 1; ++u)
        if (t + u < count) token(xn[u], dn[u], gn[u], t + u);
    if (OUT) {
        for (t = count; t < p.t1 - p.t0; ++t)   // behind the sequence's end
            store_at<T>(a.y, out0 + static_cast<int64_t>(t) * a.channels, lane_at, 0.f);
        if (a.new_state != nullptr && p.chunk == a.chunks - 1) {
            float* to = a.new_state + (static_cast<int64_t>(p.batch) * a.channels + p.channel) * a.states;
#pragma unroll
            for (int n = 0; n < S; ++n)
                if (n < a.states) to[n] = h[n];
        }
    } else {
        float* to = a.slots + (static_cast<int64_t>(p.batch) * (a.chunks - 1) + p.chunk) * S * cp + p.column;
#pragma unroll
        for (int n = 0; n < S; ++n) to[n * cp] = h[n];
        a.sums[(static_cast<int64_t>(p.batch) * a.chunks + p.chunk) * cp + p.column] = total;
    }
}

// Carries states over chunk boundaries.  Forward: slots[k] holds the state that chunk k adds
// from a zero start and becomes the state at the start of chunk k + 1; chunk k's decay is
// exp(A sums[k]).  Backward: slots[k] holds the adjoint that chunk k + 1 hands to chunk k from
// a zero adjoint behind it and becomes the whole one; the order is reversed and the decay is
// that of chunk k + 1.  A workgroup takes one state of 64 channels, its waves ranges of the
// chunks: each folds its range, the ranges' results go through LDS, and each walks its range
// again from the value before it.  Ranges of up to JOIN slots stand in registers and are read
// once.  The launch is short, so its time is that of fetching its code: both walks share the
// loop's.  15 us with 49 chunks (32 sequences of 192 channels, 16 states), 13 with 256
// (one of 1024).
constexpr int JOIN = 8;
__global__ __launch_bounds__(1024) void state_space_join_kernel(const SSArgs a, const float* edge, int32_t S,
                                                                int32_t slots_n, int32_t backward) {
    __shared__ float fold_h[16][64], fold_p[16][64];
    const int32_t lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    const int32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // contiguous ranges of workgroups to each XCD: the states of a sequence share its sums there
    // (7 sequences of 448 channels, 49 chunks: 14.8 -> 12.8 us)
    const uint32_t bid = xcd_remap_any(blockIdx.x, gridDim.x);
    const int32_t rest = static_cast<int32_t>(bid / static_cast<uint32_t>(a.tiles)), tile = static_cast<int32_t>(bid) - rest * a.tiles;
    const int32_t batch = rest / S, n = rest - batch * S;
    const int32_t group = tile / a.group_tiles, in_group = (tile - group * a.group_tiles) * 64 + lane;
    // lanes without a channel carry the group's last one, as in the other passes
    const int32_t channel = group * a.group_channels + (in_group < a.group_channels ? in_group : a.group_channels - 1);
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;
    const float A2 = n < a.states ? ss_rate(a.A[static_cast<int64_t>(channel) * a.states + n]) : 0.f;
    const int32_t per = (slots_n + waves - 1) / waves;
    const int32_t i0 = wave * per, i1 = i0 + per < slots_n ? i0 + per : slots_n;
    // Step i touches slot i with the decay of chunk i, or slot slots_n - 1 - i with that of chunk
    // slots_n - i.  Uniform addresses; the lanes follow each other from there.
    const int32_t first = i0 < slots_n ? i0 : slots_n - 1;
    float* slot0 = a.slots + ((static_cast<int64_t>(batch) * slots_n + (backward ? slots_n - 1 - first : first)) * S + n) * cp +
                   static_cast<int64_t>(tile) * 64;
    const float* sum0 = a.sums + (static_cast<int64_t>(batch) * (slots_n + 1) + (backward ? slots_n - first : first)) * cp +
                        static_cast<int64_t>(tile) * 64;
    const int64_t slot_step = backward ? -S * cp : S * cp, sum_step = backward ? -cp : cp;
    const uint32_t lane_at = lane * sizeof(float);
    // exp(A sum) h, and nothing from an empty state even where the decay (A > 0) overflows
    auto decayed = [&](float p, float h) { return h == 0.f ? 0.f : h * __builtin_amdgcn_exp2f(A2 * p); };
    float v[JOIN], p[JOIN], h = 0.f, ps = 0.f;
    const int32_t first_walk = waves > 1 ? 0 : 1;
#pragma nounroll
    for (int32_t walk = first_walk; walk < 2; ++walk) {
        if (walk == 1) {
            if (waves > 1) {
                fold_h[wave][lane] = h;
                fold_p[wave][lane] = ps;
                __syncthreads();
            }
            h = edge != nullptr && n < a.states
                ? edge[(static_cast<int64_t>(batch) * a.channels + channel) * a.states + n] : 0.f;
#pragma nounroll
            for (int32_t w = 0; w < wave; ++w) h = decayed(fold_p[w][lane], h) + fold_h[w][lane];
        }
        float* slot = slot0;
        const float* sum = sum0;
#pragma nounroll
        for (int32_t from = i0; from < i1; from += JOIN) {
            if (walk == first_walk || per > JOIN) {
                const float* at = slot;
                const float* sat = sum;
#pragma unroll
                for (int i = 0; i < JOIN; ++i) {   // steps behind the range read its last slot and change nothing
                    const bool in = from + i < i1;
                    v[i] = load_at(at, lane_at);
                    p[i] = load_at(sat, lane_at);
                    v[i] = in ? v[i] : 0.f;
                    p[i] = in ? p[i] : 0.f;
                    at = from + i + 1 < i1 ? at + slot_step : at;
                    sat = from + i + 1 < i1 ? sat + sum_step : sat;
                }
            }
#pragma unroll
            for (int i = 0; i < JOIN; ++i) {
                h = decayed(p[i], h) + v[i];
                ps += p[i];
                if (walk == 1 && from + i < i1) store_at<float>(slot, i * slot_step, lane_at, h);
            }
            slot += JOIN * slot_step;
            sum += JOIN * sum_step;
        }
    }
}

// B and C as FP32 rows of the padded state count, zero in the padding.
template <typename T>
__global__ __launch_bounds__(256) void state_space_maps_kernel(const SSTokens b, const SSTokens c, float* to,
                                                               int64_t tokens, int64_t rows, int32_t groups,
                                                               int32_t states, int32_t S) {
    const int64_t total = 2 * rows * groups * S;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const bool second = i >= total / 2;
        const int64_t k = second ? i - total / 2 : i, n = k % S, rest = k / S;   // S is 8, 16 or 32
        const int64_t row = rest / groups, group = rest - row * groups, batch = row / tokens, t = row - batch * tokens;
        const SSTokens& from = second ? c : b;
        to[i] = n < states ? to_f32(static_cast<const T*>(from.data)[batch * from.bs + t * from.ts + group * states + n]) : 0.f;
    }
}

// One token of every sequence.  Four states a lane; the lanes of a channel stand side by side,
// so the states are read and written in whole rows of 16 bytes a lane (element by element
// where the state count or an address does not allow that).  Bound by the states' bytes (FP32,
// read and written) once the batch is large, by the launch before: 6.1 us for 64 sequences
// of 1024 channels and 16 states, 9 MB.
struct StepArgs {
    const void *x, *dt, *gate, *b, *c;
    int64_t x_bs, dt_bs, gate_bs, b_bs, c_bs;
    const float *A, *D, *dt_bias, *state;
    float* new_state;
    void* y;
    int64_t total;   // sequences x channels
    int32_t softplus, channels, group_channels, states, wide;
};
template <typename T, int LANES>
__global__ __launch_bounds__(256) void state_space_step_kernel(const StepArgs a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / LANES;    // sequence and channel
    if (row >= a.total) return;       // whole channels: the lanes of one stay together
    const int32_t part = static_cast<int32_t>(i % LANES) * 4;
    const int64_t batch = row / a.channels;
    const int32_t channel = static_cast<int32_t>(row - batch * a.channels);
    const int32_t group = channel / a.group_channels;
    const float* state = a.state + row * a.states + part;
    const float* rates = a.A + static_cast<int64_t>(channel) * a.states + part;
    const T* b = static_cast<const T*>(a.b) + batch * a.b_bs + static_cast<int64_t>(group) * a.states + part;
    const T* c = static_cast<const T*>(a.c) + batch * a.c_bs + static_cast<int64_t>(group) * a.states + part;
    float h[4], A[4], bv[4], cv[4];
    // of 12, 20, 24 and 28 states the last lanes have none, and the memory there is the next
    // channel's
    const bool wide = a.wide && part < a.states;
    if (wide) {
        const float4 h4 = *reinterpret_cast<const float4*>(state), A4 = *reinterpret_cast<const float4*>(rates);
        h[0] = h4.x; h[1] = h4.y; h[2] = h4.z; h[3] = h4.w;
        A[0] = A4.x; A[1] = A4.y; A[2] = A4.z; A[3] = A4.w;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const bool in = part + n < a.states;
        bv[n] = in ? to_f32(b[n]) : 0.f;
        cv[n] = in ? to_f32(c[n]) : 0.f;
        if (!wide) {
            h[n] = in ? state[n] : 0.f;
            A[n] = in ? rates[n] : 0.f;
        }
    }
    const float xv = to_f32(static_cast<const T*>(a.x)[batch * a.x_bs + channel]);
    float step = to_f32(static_cast<const T*>(a.dt)[batch * a.dt_bs + channel]);
    if (a.dt_bias != nullptr) step += a.dt_bias[channel];
    if (a.softplus) step = ss_softplus(step);
    const float dtx = step * xv;
    float acc = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        h[n] = fmaf(dtx, bv[n], h[n] * __builtin_amdgcn_exp2f(step * ss_rate(A[n])));
        acc = fmaf(cv[n], h[n], acc);
    }
    float* next = a.new_state + row * a.states + part;
    if (wide) {
        *reinterpret_cast<float4*>(next) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (part + n < a.states) next[n] = h[n];
    }
    acc = ln_lane_sum(acc, LANES == 1 ? 0 : LANES == 2 ? 1 : LANES == 4 ? 2 : 3);
    if (part == 0) {
        if (a.D != nullptr) acc = fmaf(a.D[channel], xv, acc);
        if (a.gate != nullptr) {
            const float z = to_f32(static_cast<const T*>(a.gate)[batch * a.gate_bs + channel]);
            acc *= z * sigmoid_fast(z);
        }
        static_cast<T*>(a.y)[row] = from_f32<T>(acc);
    }
}

// Tokens a chunk: whole lines, or the chunk (in whole blocks of 16 tokens) whose passes take
// the least time by a model fitted to whole passes of 16 states: about 118 vector instructions
// a token, of which a SIMD (of 1024) issues one every 9.5, 5.8, 5.2, 4.9, 4.5 cycles with 1, 2,
// 3, 4, 5 and more waves (its waits included); one pass for whole lines, 1.8 for chunks; 8
// tokens' time around a chunk's loop; 1.6 ns for every chunk of 64 channels whose states go
// through the join; and 10 us for the two launches more.  The state count does not enter: more
// states lengthen the passes and the join alike.
// Held against other chunks (16 to 128 tokens; 1 x 16384 x 1024, 32 x 3136 x 192, 8 x 784 x 1024
// and 4 x 4096 x 384, all passes): at 4, 8, 12 and 16 states it takes the best or one 1.5 %
// behind (the first with 16 states: 127 us at 64 tokens, 137 at 48, 149 at 80), at 20, 24 and 32
// one up to 5 % behind, but 13 % with 32 states at 32 x 3136 x 192 (64 tokens 303 us in
// training, 80 tokens 268).
int64_t forward_chunk(int64_t B, int64_t N, int64_t tiles) {
    const int64_t blocks = ss_ceil(N, SS_BLOCK), lines = B * tiles;
    static const double issue[] = {0., 9.5, 5.8, 5.2, 4.9, 4.5, 4.5};
    auto pass = [&](int64_t per, int64_t waves) {   // us, `waves` waves of `per` blocks
        const int64_t each = ss_ceil(waves, 1024);
        return static_cast<double>(per * SS_BLOCK + 8) * each * issue[each < 6 ? each : 6] * 118 / 2300;
    };
    int64_t best = blocks;
    double least = pass(blocks, lines);
    const int64_t most = ss_ceil(blocks * lines, 1024) + 1;   // blocks a chunk with one wave a SIMD
    const int64_t first = ss_ceil(most, 8);
    for (int64_t per = first; per <= most && per < blocks && per < first + 256; ++per) {
        const int64_t chunks = ss_ceil(blocks, per);
        const double time = 1.8 * pass(per, chunks * lines) + 1.6e-3 * chunks * lines + 10.;
        if (time < least) {
            least = time;
            best = per;
        }
    }
    return best * SS_BLOCK;
}

template <typename T, typename BCT, int S>
int launch_forward(SSArgs& a, int64_t B, hipStream_t s) {
    if (a.chunks > 1) {
        a.first_chunk = 0;
        a.launch_chunks = a.chunks - 1;
        state_space_chunk_kernel<T, BCT, S, false>
            <<<static_cast<uint32_t>(B * a.launch_chunks * a.tiles), 64, 0, s>>>(a);
        if (int rc = check_launch("state_space chunk states")) return rc;
        if (int rc = ss_join(a, B, S, false, a.state, s)) return rc;
    }
    a.first_chunk = 0;
    a.launch_chunks = a.chunks;
    state_space_chunk_kernel<T, BCT, S, true><<<static_cast<uint32_t>(B * a.chunks * a.tiles), 64, 0, s>>>(a);
    return check_launch("state_space forward");
}

template <typename T>
int launch_step(const StepArgs& a, hipStream_t s) {
    const int lanes = a.states <= 4 ? 1 : a.states <= 8 ? 2 : a.states <= 16 ? 4 : 8;
    const int64_t blocks = ss_ceil(a.total * lanes, 256);
    VH_REQUIRE(blocks < (1ll << 24), VH_ERR_SHAPE, "state space step: too many sequences and channels for one launch");
    const uint32_t grid = static_cast<uint32_t>(blocks);
    if (lanes == 1) state_space_step_kernel<T, 1><<<grid, 256, 0, s>>>(a);
    else if (lanes == 2) state_space_step_kernel<T, 2><<<grid, 256, 0, s>>>(a);
    else if (lanes == 4) state_space_step_kernel<T, 4><<<grid, 256, 0, s>>>(a);
    else state_space_step_kernel<T, 8><<<grid, 256, 0, s>>>(a);
    return check_launch("state_space step");
}

int dispatch_forward(int32_t io, int32_t bc, int32_t S, SSArgs& a, int64_t B, hipStream_t s) {
    auto by_states = [&](auto t, auto u) -> int {
        using T = decltype(t);
        using U = decltype(u);
        if (S == 8) return launch_forward<T, U, 8>(a, B, s);
        if (S == 16) return launch_forward<T, U, 16>(a, B, s);
        return launch_forward<T, U, 32>(a, B, s);
    };
    if (io == VH_DTYPE_F32) return by_states(float{}, float{});
    if (io == VH_DTYPE_F16) return by_states(f16_t{}, float{});
    if (bc == VH_DTYPE_F32) return by_states(bf16_t{}, float{});
    return by_states(bf16_t{}, bf16_t{});
}
int check_sizes(int64_t B, int64_t N, int64_t C, int32_t groups) {
    VH_REQUIRE(B > 0 && N > 0 && C > 0 && groups > 0 && C % groups == 0, VH_ERR_SHAPE,
               "state space scan needs nonempty sizes and channels divisible by groups, got B=%lld N=%lld C=%lld groups=%d",
               (long long)B, (long long)N, (long long)C, groups);
    VH_REQUIRE(N < (1ll << 30) && C < (1ll << 24) && B < (1ll << 24), VH_ERR_SHAPE,
               "state space scan: sizes out of range (B=%lld N=%lld C=%lld)", (long long)B, (long long)N, (long long)C);
    return VH_OK;
}

// The scalar unit reads whole words; the backward's offsets over a few rows are 32 bits wide.
bool whole_words(const SSTokens& t, int64_t e) {
    return reinterpret_cast<uintptr_t>(t.data) % 4 == 0 && t.bs * e % 4 == 0 && t.ts * e % 4 == 0 && t.ts < (1 << 24);
}

}  // namespace

int ss_fill(SSArgs& a, int32_t io_dtype, int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    VH_REQUIRE(valid_dtype(io_dtype), VH_ERR_DTYPE, "unsupported io_dtype %d", io_dtype);
    if (int rc = check_sizes(B, N, C, groups)) return rc;
    VH_REQUIRE(states >= 1 && states <= 32, VH_ERR_SHAPE, "states must be 1 to 32, got %d", states);
    VH_REQUIRE(a.x.data != nullptr && a.dt.data != nullptr && a.b.data != nullptr && a.c.data != nullptr &&
                   a.A != nullptr, VH_ERR_ARG, "x, dt, B, C and A must not be null");
    VH_REQUIRE(groups <= 32768, VH_ERR_SHAPE, "state space scan: at most 32768 groups, got %d", groups);
    a.states = states;
    a.groups = groups;
    a.batches = static_cast<int32_t>(B);
    a.tokens = static_cast<int32_t>(N);
    a.channels = static_cast<int32_t>(C);
    a.group_channels = static_cast<int32_t>(C / groups);
    a.group_tiles = static_cast<int32_t>(ss_ceil(a.group_channels, 64));
    a.tiles = a.group_tiles * groups;
    a.blocks = static_cast<int32_t>(ss_ceil(N, SS_BLOCK));
    // a launch has one wave for each tile of a chunk (no more chunks than the aimed-at waves
    // where there are that many sequences), and one for each state
    VH_REQUIRE(B * a.tiles < (1ll << 24), VH_ERR_SHAPE,
               "state space scan: too many sequences and channels for one launch");
    return VH_OK;
}

int ss_maps(SSArgs& a, int32_t io_dtype, float* maps, int32_t* bc_dtype, hipStream_t stream) {
    const int32_t S = ss_padded(a.states);
    const int64_t e = dtype_bytes(io_dtype);
    *bc_dtype = io_dtype;
    if (io_dtype != VH_DTYPE_F16 && a.states == S && whole_words(a.b, e) && whole_words(a.c, e)) return VH_OK;
    const int64_t rows = static_cast<int64_t>(a.batches) * a.tokens, total = 2 * rows * a.groups * S;
    const int64_t blocks = ss_ceil(total, 256);
    const uint32_t grid = static_cast<uint32_t>(blocks < 16384 ? blocks : 16384);
    auto go = [&](auto t) {
        state_space_maps_kernel<decltype(t)><<<grid, 256, 0, stream>>>(a.b, a.c, maps, a.tokens, rows, a.groups, a.states, S);
    };
    if (io_dtype == VH_DTYPE_F32) go(float{});
    else if (io_dtype == VH_DTYPE_BF16) go(bf16_t{});
    else go(f16_t{});
    const int64_t row = static_cast<int64_t>(a.groups) * S;
    a.b = {maps, a.tokens * row, row};
    a.c = {maps + total / 2, a.tokens * row, row};
    *bc_dtype = VH_DTYPE_F32;
    return check_launch("state_space maps");
}

int ss_join(const SSArgs& a, int64_t B, int32_t padded, bool backward, const float* edge, hipStream_t stream) {
    const int32_t slots = a.chunks - 1;
    const int32_t waves = slots > 16 * JOIN ? 16 : (slots + JOIN - 1) / JOIN;
    state_space_join_kernel<<<static_cast<uint32_t>(B * padded * a.tiles), 64 * waves, 0, stream>>>(a, edge, padded,
                                                                                                slots, backward);
    return check_launch("state_space join");
}

}  // namespace vh

extern "C" {

size_t vh_state_space_workspace_bytes(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    using namespace vh;
    if (B <= 0 || N <= 0 || C <= 0 || groups <= 0 || C % groups || states <= 0 || states > 32) return 0;
    const int64_t tiles = ss_ceil(C / groups, 64) * groups;
    const int64_t chunks = ss_ceil(N, forward_chunk(B, N, tiles));
    int64_t floats = ss_maps_floats(B, N, groups, states);
    if (chunks > 1) floats += B * tiles * 64 * ((chunks - 1) * ss_padded(states) + chunks);
    return static_cast<size_t>(floats) * sizeof(float);
}

size_t vh_state_space_kept_bytes(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    using namespace vh;
    if (B <= 0 || N <= 0 || C <= 0 || groups <= 0 || C % groups || states <= 0 || states > 32) return 0;
    return static_cast<size_t>(B) * ss_ceil(N, SS_BLOCK) * ss_padded(states) * ss_ceil(C / groups, 64) * groups * 64 *
           sizeof(float);
}

int vh_state_space_forward(
    const void* x, int64_t x_batch, int64_t x_token, const void* dt, int64_t dt_batch, int64_t dt_token,
    const void* gate, int64_t gate_batch, int64_t gate_token, int32_t io_dtype,
    const void* b, int64_t b_batch, int64_t b_token, const void* c, int64_t c_batch, int64_t c_token,
    const float* A, const float* D, const float* dt_bias, int32_t softplus, const float* state,
    const int32_t* lengths, void* y, float* new_state, float* kept, int64_t B, int64_t N, int64_t C, int32_t groups,
    int32_t states, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vh;
    SSArgs a{};
    a.x = {x, x_batch, x_token};
    a.dt = {dt, dt_batch, dt_token};
    a.gate = {gate, gate_batch, gate_token};
    a.b = {b, b_batch, b_token};
    a.c = {c, c_batch, c_token};
    a.A = A;
    a.D = D;
    a.dt_bias = dt_bias;
    a.softplus = softplus;
    a.state = state;
    a.lengths = lengths;
    a.y = y;
    a.new_state = new_state;
    a.kept = kept;
    if (int rc = ss_fill(a, io_dtype, B, N, C, groups, states)) return rc;
    VH_REQUIRE(y != nullptr, VH_ERR_ARG, "y must not be null");
    VH_REQUIRE(!overlapping(state, new_state, B * C * states * 4), VH_ERR_ARG, "state and new_state must not overlap");
    const int32_t S = ss_padded(states);
    a.chunk = static_cast<int32_t>(forward_chunk(B, N, a.tiles));
    a.chunks = static_cast<int32_t>(ss_ceil(N, a.chunk));
    const size_t need = vh_state_space_workspace_bytes(B, N, C, groups, states);
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need, VH_ERR_WORKSPACE,
               "state space scan needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
    float* maps = static_cast<float*>(workspace);
    a.slots = maps + ss_maps_floats(B, N, groups, states);
    a.sums = a.slots + static_cast<int64_t>(B) * (a.chunks - 1) * S * a.tiles * 64;
    int32_t bc_dtype = 0;
    if (int rc = ss_maps(a, io_dtype, maps, &bc_dtype, static_cast<hipStream_t>(stream))) return rc;
    return dispatch_forward(io_dtype, bc_dtype, S, a, B, static_cast<hipStream_t>(stream));
}

int vh_state_space_step(
    const void* x, int64_t x_batch, const void* dt, int64_t dt_batch, const void* gate, int64_t gate_batch,
    int32_t io_dtype, const void* b, int64_t b_batch, const void* c, int64_t c_batch, const float* A, const float* D,
    const float* dt_bias, int32_t softplus, const float* state, float* new_state, void* y, int64_t B, int64_t C,
    int32_t groups, int32_t states, void* stream) {
    using namespace vh;
    VH_REQUIRE(valid_dtype(io_dtype), VH_ERR_DTYPE, "unsupported io_dtype %d", io_dtype);
    if (int rc = check_sizes(B, 1, C, groups)) return rc;
    VH_REQUIRE(states >= 1 && states <= 32, VH_ERR_SHAPE, "states must be 1 to 32, got %d", states);
    VH_REQUIRE(x != nullptr && dt != nullptr && b != nullptr && c != nullptr && A != nullptr && state != nullptr &&
                   new_state != nullptr && y != nullptr, VH_ERR_ARG,
               "x, dt, B, C, A, state, new_state and y must not be null");
    VH_REQUIRE(state == new_state || !overlapping(state, new_state, B * C * states * 4), VH_ERR_ARG,
               "state and new_state must be the same memory or not overlap");
    StepArgs a{};
    a.x = x;
    a.x_bs = x_batch;
    a.dt = dt;
    a.dt_bs = dt_batch;
    a.gate = gate;
    a.gate_bs = gate_batch;
    a.b = b;
    a.b_bs = b_batch;
    a.c = c;
    a.c_bs = c_batch;
    a.A = A;
    a.D = D;
    a.dt_bias = dt_bias;
    a.state = state;
    a.new_state = new_state;
    a.y = y;
    a.total = B * C;
    a.softplus = softplus;
    a.channels = static_cast<int32_t>(C);
    a.group_channels = static_cast<int32_t>(C / groups);
    a.states = states;
    a.wide = states % 4 == 0 && reinterpret_cast<uintptr_t>(A) % 16 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0 &&
             reinterpret_cast<uintptr_t>(new_state) % 16 == 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (io_dtype == VH_DTYPE_F32) return launch_step<float>(a, s);
    return io_dtype == VH_DTYPE_BF16 ? launch_step<bf16_t>(a, s) : launch_step<f16_t>(a, s);
}

}  // extern "C"
