// Backward of the selective state space scan.
//
// With g[n] the adjoint of h[n] after token t, dz = dy silu(gate) the gradient of the ungated
// output and q[n] = exp(dt A[n]) h_before[n]:
//   g[n] = C[n] dz + exp(dt_next A[n]) g_next[n]
//   dC[n] = sum_channels dz h[n]            dB[n] = sum_channels dt x g[n]
//   dx = D dz + dt sum_n g[n] B[n]          ddt = sum_n g[n] (A[n] q[n] + x B[n])
//   dA[n] = sum_tokens dt g[n] q[n]         dD = sum dz x        dgate = dy y silu'(gate)
//
// The states are not kept for every token: the forward leaves the state before each block of
// tokens (state_space.h), and a wave walks the blocks of its chunk from the last, forms the
// states inside a block again and then the adjoints, newest token first.  The chunks' adjoints
// are joined over their boundaries as the forward joins states.
//
// At 32 x 3136 x 192, 16 states, bf16: adjoints between chunks 67 us, join 15, gradients 293,
// dB and dC 10, parameters 5, where the bytes need 72.  The gradients' pass is bound by the
// issue of vector instructions: 111 a token for a wave's 16 channels, the vector unit active
// for 87 % of the time.  (One lane a channel, as in the
// forward, spills its states: 681 us for the pass.)
#include "param_sum.h"
#include "state_space.h"

namespace vh {
namespace {

// Adjoint that each chunk hands to the one before it from a zero adjoint behind it, and the
// chunk's sum of dt.
template <typename T, typename BCT, int S>
__global__ __launch_bounds__(64) void state_space_adjoint_kernel(const SSArgs a) {
    const SSPlace p = ss_place(a);
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;
    float A2[S], carry[S];
    ss_rates<S>(a, p.channel, A2);
#pragma unroll
    for (int n = 0; n < S; ++n) carry[n] = 0.f;
    const float bias = a.dt_bias != nullptr ? a.dt_bias[p.channel] : 0.f;
    const uint32_t lane_at = static_cast<uint32_t>(p.channel) * sizeof(T);
    const bool gated = a.gate.data != nullptr, soft = a.softplus != 0;
    const T* dt = ss_tokens<T>(a.dt, p);
    const T* dy = ss_tokens<T>(a.dy, p);
    const T* gate = gated ? ss_tokens<T>(a.gate, p) : dy;
    const int64_t gate_ts = gated ? a.gate.ts : a.dy.ts;
    const int64_t c0 = p.batch * a.c.bs + p.t0 * a.c.ts + static_cast<int64_t>(p.group) * S;
    const int32_t count = p.te - p.t0;
    float total = 0.f;
    SSRow<BCT, S> cn;   // loaded a token ahead, as the forward loads B and C
    auto token = [&](T dr, T yr, T gr, int32_t t) {
        const SSRow<BCT, S> c = cn;
        cn.load(a.c.data, c0 + (t > 0 ? t - 1 : 0) * a.c.ts);
        __builtin_amdgcn_sched_barrier(0);
        const float raw = to_f32(dr) + bias, z = to_f32(gr);
        const float plus = ss_softplus(raw), step = soft ? plus : raw;   // no branch in the loop
        const float silu = z * sigmoid_fast(z), dz = to_f32(yr) * (gated ? silu : 1.f);
        total += step;
#pragma unroll
        for (int n = 0; n < S; ++n) carry[n] = fmaf(c[n], dz, carry[n]) * __builtin_amdgcn_exp2f(step * A2[n]);
        __builtin_amdgcn_sched_barrier(0);
    };
    int32_t t = count - 1;
    T dn[SS_UNROLL], yn[SS_UNROLL], gn[SS_UNROLL];
    auto fetch = [&](int32_t t) {   // tokens t, t - 1, ...
        const uint32_t at = opaque(lane_at);
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) {
            const int64_t i = t - u > 0 ? t - u : 0;
            dn[u] = load_at(dt + i * a.dt.ts, at);
            yn[u] = load_at(dy + i * a.dy.ts, at);
            gn[u] = load_at(gate + i * gate_ts, at);
        }
    };
    if (count > 0) {
        fetch(t);
        cn.load(a.c.data, c0 + t * a.c.ts);
    }
    WaveTurns turns(count);
    for (; t >= SS_UNROLL - 1; t -= SS_UNROLL) {
        turns.left(t);
        T dr[SS_UNROLL], yr[SS_UNROLL], gr[SS_UNROLL];
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) { dr[u] = dn[u]; yr[u] = yn[u]; gr[u] = gn[u]; }
        fetch(t - SS_UNROLL);
#pragma unroll
        for (int u = 0; u < SS_UNROLL; ++u) token(dr[u], yr[u], gr[u], t - u);
    }
#pragma unroll
    for (int u = 0; u < SS_UNROLL - 1; ++u)
        if (t - u >= 0) token(dn[u], yn[u], gn[u], t - u);
    float* to = a.slots + (static_cast<int64_t>(p.batch) * (a.chunks - 1) + p.chunk - 1) * S * cp + p.column;
#pragma unroll
    for (int n = 0; n < S; ++n) to[n * cp] = carry[n];
    a.sums[(static_cast<int64_t>(p.batch) * a.chunks + p.chunk) * cp + p.column] = total;
}

// The sums over lanes of four tokens' values, so that no lane holds a value twice before it must:
// exchanging one lane bit of two registers and adding leaves the sum of the first in the lanes
// with the bit clear, that of the second in the others.
__device__ __forceinline__ float fold32(float a, float b) {   // lane bit 5
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {   // lane bit 4
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
template <int CTRL>
__device__ __forceinline__ float fold_quad(float a, float b, bool upper) {   // a bit within four lanes
    const float first = a + ln_dpp<CTRL>(a), second = b + ln_dpp<CTRL>(b);
    return upper ? second : first;
}
// Sum over the channels inside a row of 16 lanes, in every lane.
template <int LANES>
__device__ __forceinline__ float row_channels(float v) {
    v += ln_dpp<0x128>(v);                          // row_ror 8
    v += ln_dpp<0x124>(v);                          // row_ror 4
    if constexpr (LANES == 2) v += ln_dpp<0x4E>(v); // lanes (2, 3, 0, 1)
    return v;
}

// An element `offset` bytes behind a uniform address, through a buffer descriptor made of it.
// (Plain loads cost more here: 415 vector instructions in part 3. below against 301, and 24
// registers; in the forward's loop it is the other way round, 107 us against 117.)  Offsets stay
// below the descriptor's 4 GiB: channels < 2^24 and at most 2^26 of them a token row.
template <typename T>
__device__ __forceinline__ T row_load(const T* base, uint32_t offset) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, -1, 0x00027000);
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rsrc, offset, 0, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rsrc, offset, 0, 0));
}
template <typename T>
__device__ __forceinline__ void row_store(void* base, int64_t element, uint32_t offset, float v) {
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(static_cast<T*>(base) + element, 0, -1, 0x00027000);
    const T out = from_f32<T>(v);
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, out), rsrc, offset, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, out), rsrc, offset, 0, 0);
}

// Waves a SIMD that the registers of the gradients' pass allow.
constexpr int backward_waves(int states) { return states <= 8 ? 3 : states <= 16 ? 4 : 2; }

// The gradients of one chunk.  LANES lanes share a channel, SPL states each, so the decays and
// states of SUB tokens stand in registers with room for four waves a SIMD (of independent vector
// instructions a wave alone issues one every 7 cycles, four together one every 4.6).  A workgroup takes
// 256 / LANES channels through blocks of SS_BLOCK tokens:
//   1. by token and channel: step, step x and dz of the block go to LDS, as do B and C;
//   2. by channel and states: the states before each sub-block from the kept ones, then from
//      the last sub-block the decays and states again and the adjoints; the sums over states
//      go to LDS in place of 1., those over a wave's channels beside them;
//   3. by token and channel: dx, ddt and dgate; and the sums of dB and dC over the waves.
template <typename T, typename BCT, int LANES, int SPL>
__global__ __launch_bounds__(256, backward_waves(LANES * SPL)) void state_space_backward_kernel(const SSArgs a) {
    constexpr int S = LANES * SPL, CHANNELS = 256 / LANES;
    constexpr int SUB = 4, SUBS = SS_BLOCK / SUB;
    constexpr int TOKENS = SS_BLOCK * CHANNELS / 256;   // of a thread in 1. and 3.
    __shared__ float4 tok[SS_BLOCK][CHANNELS];
    __shared__ float maps[SS_BLOCK][2 * S];             // C, then B
    __shared__ float parts[4][SS_BLOCK][2 * S + 4];    // (+ 4: the rows that a wave writes together in other banks)
    __shared__ float starts[SUBS - 1][SPL][256];        // states before the sub-blocks but the last, a lane's own

    const uint32_t bid = xcd_remap_any(blockIdx.x, gridDim.x);
    const uint32_t rest = bid / static_cast<uint32_t>(a.wide_tiles);
    const int32_t tile = static_cast<int32_t>(bid - rest * a.wide_tiles);
    const int32_t batch = static_cast<int32_t>(rest / static_cast<uint32_t>(a.chunks));
    const int32_t chunk = static_cast<int32_t>(rest) - batch * a.chunks;
    const int32_t tiles_of_group = a.wide_tiles / a.groups, group = tile / tiles_of_group;
    const int32_t first = (tile - group * tiles_of_group) * CHANNELS;   // in the group
    const int32_t t0 = chunk * a.chunk, t1 = a.tokens - t0 < a.chunk ? a.tokens : t0 + a.chunk;
    int32_t te = a.tokens;
    if (a.lengths != nullptr) te = __builtin_amdgcn_readfirstlane(a.lengths[batch]);
    te = te < t0 ? t0 : te > t1 ? t1 : te;
    const int32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;

    // by channel and states
    const int32_t part = tid & (LANES - 1), mine = tid / LANES;   // mine: of the workgroup's channels
    const bool live = first + mine < a.group_channels;
    const int32_t in_group = live ? first + mine : a.group_channels - 1;
    const int32_t channel = group * a.group_channels + in_group;
    const int64_t column = static_cast<int64_t>(group) * a.group_tiles * 64 + in_group;
    float A2[SPL], carry[SPL], dA[SPL];
#pragma unroll
    for (int j = 0; j < SPL; ++j) {
        const int32_t n = part * SPL + j;
        A2[j] = n < a.states ? ss_rate(a.A[static_cast<int64_t>(channel) * a.states + n]) : 0.f;
        dA[j] = 0.f;
    }
    // the adjoint behind the chunk, times the decay of the token behind it
    if (chunk < a.chunks - 1) {
        const int64_t slot = static_cast<int64_t>(batch) * (a.fine_chunks - 1) + (chunk + 1) * a.fine_per_chunk - 1;
        const float* from = a.slots + (slot * S + part * SPL) * cp + column;
#pragma unroll
        for (int j = 0; j < SPL; ++j) carry[j] = live ? from[j * cp] : 0.f;
    } else {
        const float* from = a.dnew_state != nullptr
            ? a.dnew_state + (static_cast<int64_t>(batch) * a.channels + channel) * a.states : nullptr;
#pragma unroll
        for (int j = 0; j < SPL; ++j)
            carry[j] = from != nullptr && live && part * SPL + j < a.states ? from[part * SPL + j] : 0.f;
    }

    // by token and channel
    const int32_t tc = tid % CHANNELS, tr = wave / (CHANNELS / 64) * TOKENS;   // channel and first token
    const bool tlive = first + tc < a.group_channels;
    const int32_t tchannel = group * a.group_channels + (tlive ? first + tc : a.group_channels - 1);
    const float bias = a.dt_bias != nullptr ? a.dt_bias[tchannel] : 0.f;
    const float D = a.D != nullptr ? a.D[tchannel] : 0.f;
    const T* x = static_cast<const T*>(a.x.data) + batch * a.x.bs;
    const T* dt = static_cast<const T*>(a.dt.data) + batch * a.dt.bs;
    const T* dy = static_cast<const T*>(a.dy.data) + batch * a.dy.bs;
    const bool gated = a.gate.data != nullptr, soft = a.softplus != 0;
    const T* gate = gated ? static_cast<const T*>(a.gate.data) + batch * a.gate.bs : dy;
    const int64_t gate_ts = gated ? a.gate.ts : a.dy.ts;
    const uint32_t lane_at = static_cast<uint32_t>(tchannel) * sizeof(T);
    const BCT* bmap = static_cast<const BCT*>(a.b.data) + batch * a.b.bs + static_cast<int64_t>(group) * S;
    const BCT* cmap = static_cast<const BCT*>(a.c.data) + batch * a.c.bs + static_cast<int64_t>(group) * S;
    const int64_t out0 = static_cast<int64_t>(batch) * a.tokens * a.channels;
    float* bc = a.bc_partial + (static_cast<int64_t>(tile) * a.batches + batch) * a.tokens * (2 * S);
    float dD = 0.f, dbias = 0.f;

    constexpr int MAPS = SS_BLOCK * 2 * S / 256;   // values of B and C a thread brings
    struct Raw { T x[TOKENS], dt[TOKENS], dy[TOKENS], gate[TOKENS]; };
    Raw next;
    float next_maps[MAPS];
    auto fetch = [&](int32_t tb) {
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            const int64_t t = tb + tr + i < te ? tb + tr + i : te - 1;   // a token of the sequence
            next.x[i] = row_load(x + t * a.x.ts, lane_at);
            next.dt[i] = row_load(dt + t * a.dt.ts, lane_at);
            next.dy[i] = row_load(dy + t * a.dy.ts, lane_at);
            next.gate[i] = row_load(gate + t * gate_ts, lane_at);
        }
        // a wave's values of one load are of C or of B and of rows that follow each other
        const int32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < MAPS; ++i) {
            const int32_t first = wave * 64 + i * 256;
            const bool second = first >= SS_BLOCK * S;
            const int32_t row = tb + (first - (second ? SS_BLOCK * S : 0)) / S, down = lane / S;
            const int32_t from = row < te ? row : te - 1, left = te - 1 - from;
            const int64_t ts = second ? a.b.ts : a.c.ts;
            const uint32_t at = static_cast<uint32_t>(down < left ? down : left) * static_cast<uint32_t>(ts) + lane % S;
            const float value = to_f32(row_load((second ? bmap : cmap) + from * ts, at * static_cast<uint32_t>(sizeof(BCT))));
            next_maps[i] = row + down < te ? value : 0.f;
        }
    };

    const int32_t blocks = (te - t0 + SS_BLOCK - 1) / SS_BLOCK;
    if (blocks > 0) fetch(t0 + (blocks - 1) * SS_BLOCK);
    WaveTurns turns(blocks);
    for (int32_t blk = blocks - 1; blk >= 0; --blk) {
        turns.left(blk);
        const int32_t tb = t0 + blk * SS_BLOCK;
        const Raw raw = next;
        float h[SPL];
        {
            const float* from = a.kept + (static_cast<int64_t>(batch) * a.blocks + tb / SS_BLOCK) * S * cp;
            const uint32_t at = static_cast<uint32_t>((part * SPL * cp + column) * sizeof(float));
#pragma unroll
            for (int j = 0; j < SPL; ++j) h[j] = live ? row_load(from + j * cp, at) : 0.f;
        }
        // 1.  Tokens behind the sequence decay by one and add nothing.
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            const bool in = tb + tr + i < te;
            const float v = to_f32(raw.dt[i]) + bias, plus = ss_softplus(v), step = soft ? plus : v;
            const float z = to_f32(raw.gate[i]), silu = z * sigmoid_fast(z);
            const float dz = to_f32(raw.dy[i]) * (gated ? silu : 1.f);
            const float dtx = step * to_f32(raw.x[i]);
            tok[tr + i][tc] = make_float4(in ? step : 0.f, in && tlive ? dtx : 0.f, in && tlive ? dz : 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < MAPS; ++i)
        {
            const int32_t first = wave * 64 + i * 256, lane = tid & 63;
            const bool second = first >= SS_BLOCK * S;
            maps[(first - (second ? SS_BLOCK * S : 0)) / S + lane / S][(second ? S : 0) + lane % S] = next_maps[i];
        }
        __syncthreads();
        // 2.
#pragma unroll
        for (int sub = 0; sub < SUBS - 1; ++sub) {
#pragma unroll
            for (int j = 0; j < SPL; ++j) starts[sub][j][tid] = h[j];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const float4 k = tok[sub * SUB + u][mine];
                const float* b = &maps[sub * SUB + u][S + part * SPL];
#pragma unroll
                for (int j = 0; j < SPL; ++j) h[j] = fmaf(k.y, b[j], h[j] * __builtin_amdgcn_exp2f(k.x * A2[j]));
                if (u % 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int sub = SUBS - 1; sub >= 0; --sub) {
            float decay[SUB][SPL], q[SUB][SPL];
            // the tokens' entries are read again from LDS in each walk, not kept from the last
            asm volatile("" ::: "memory");
            if (sub < SUBS - 1) {
#pragma unroll
                for (int j = 0; j < SPL; ++j) h[j] = starts[sub][j][tid];
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const float4 k = tok[sub * SUB + u][mine];
                const float* b = &maps[sub * SUB + u][S + part * SPL];
#pragma unroll
                for (int j = 0; j < SPL; ++j) {
                    decay[u][j] = __builtin_amdgcn_exp2f(k.x * A2[j]);
                    q[u][j] = decay[u][j] * h[j];
                    h[j] = fmaf(k.y, b[j], q[u][j]);
                }
                if (u % 2) __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" ::: "memory");
            // the adjoints, from the last token: each token's sums over states (y, g B, g A q)
            // and the parts of dC and dB of each of its states
            auto token = [&](int u, float (&v)[2 * SPL], float (&sum)[3]) {
                const int32_t t = sub * SUB + u;
                const float4 k = tok[t][mine];
                const float* c = &maps[t][part * SPL];
                const float* b = &maps[t][S + part * SPL];
                sum[0] = sum[1] = sum[2] = 0.f;
#pragma unroll
                for (int j = 0; j < SPL; ++j) {
                    const float hj = fmaf(k.y, b[j], q[u][j]);
                    const float g = fmaf(c[j], k.z, carry[j]);
                    sum[0] = fmaf(c[j], hj, sum[0]);
                    sum[1] = fmaf(g, b[j], sum[1]);
                    const float gq = g * q[u][j];
                    sum[2] = fmaf(gq, A2[j], sum[2]);
                    dA[j] = fmaf(gq, k.x, dA[j]);
                    carry[j] = g * decay[u][j];
                    v[j] = k.z * hj;
                    v[SPL + j] = k.y * g;
                    // formed here and not put off to the end of the walk, where each token's g q
                    // would still be needed
                    asm volatile("" : "+v"(dA[j]));
                }
            };
            float v[2][2 * SPL], w[2 * SPL], sum[2][3], late[3];
            token(3, v[1], sum[1]);
            token(2, v[0], sum[0]);
#pragma unroll
            for (int i = 0; i < 2 * SPL; ++i) w[i] = fold32(v[0][i], v[1][i]);
#pragma unroll
            for (int i = 0; i < 3; ++i) late[i] = fold_quad<0xB1>(sum[0][i], sum[1][i], part & 1);
            __builtin_amdgcn_sched_barrier(0);
            token(1, v[1], sum[1]);
            token(0, v[0], sum[0]);
#pragma unroll
            for (int i = 0; i < 2 * SPL; ++i) {
                // rows of 16 lanes 0 .. 3: tokens 0, 2, 1, 3
                w[i] = row_channels<LANES>(fold16(fold32(v[0][i], v[1][i]), w[i]));
                asm volatile("" : "+v"(w[i]));   // the sum is formed in every lane, not again in those that store
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) sum[0][i] = fold_quad<0xB1>(sum[0][i], sum[1][i], part & 1);
            // the channel's lanes have read these tokens' entries for the last time
            if constexpr (LANES == 4) {
#pragma unroll
                for (int i = 0; i < 3; ++i) sum[0][i] = fold_quad<0x4E>(sum[0][i], late[i], part & 2);
                tok[sub * SUB + part][mine] = make_float4(sum[0][0], sum[0][1], sum[0][2], 0.f);
            } else {
                tok[sub * SUB + part][mine] = make_float4(sum[0][0], sum[0][1], sum[0][2], 0.f);
                tok[sub * SUB + 2 + part][mine] = make_float4(late[0], late[1], late[2], 0.f);
            }
            const int32_t lane = tid & 63, row = lane >> 4;
            if ((lane & 15) < LANES) {
                float* to = &parts[wave][sub * SUB + (row & 1) * 2 + (row >> 1)][part * SPL];
#pragma unroll
                for (int j = 0; j < 2 * SPL; ++j) to[j < SPL ? j : S + j - SPL] = w[j];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        // 3.
        if (blk > 0) fetch(tb - SS_BLOCK);
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            const int64_t t = tb + tr + i;
            if (t >= te) continue;
            const float4 r = tok[tr + i][tc];   // C h, g B, g A q over the states
            float xv = to_f32(raw.x[i]), gy = to_f32(raw.dy[i]), v = to_f32(raw.dt[i]) + bias;
            float z = to_f32(raw.gate[i]);
            // formed again rather than kept in registers through 2.
            asm volatile("" : "+v"(v), "+v"(z), "+v"(gy), "+v"(xv));
            const float plus = ss_softplus(v), step = soft ? plus : v, sig = sigmoid_fast(z);
            const float dz = gy * (gated ? z * sig : 1.f);
            const float dgate = gy * fmaf(D, xv, r.x) * (sig * fmaf(z, 1.f - sig, 1.f));
            // A2 is A log2(e)
            const float ddt = fmaf(xv, r.y, r.z * 0.6931471805599453f) * (soft ? sigmoid_fast(v) : 1.f);
            dD = fmaf(dz, xv, dD);
            dbias += ddt;
            if (tlive) {
                const int64_t at = out0 + t * a.channels;
                row_store<T>(a.dx, at, lane_at, fmaf(step, r.y, D * dz));
                row_store<T>(a.ddt, at, lane_at, ddt);
                if (gated) row_store<T>(a.dgate, at, lane_at, dgate);
            }
        }
        for (uint32_t v = threadIdx.x; v < SS_BLOCK * 2 * S; v += 256) {
            const uint32_t r = v / (2 * S), n = v % (2 * S);
            if (tb + static_cast<int32_t>(r) < te)
                row_store<float>(bc, static_cast<int64_t>(tb) * (2 * S), v * static_cast<uint32_t>(sizeof(float)),
                                (parts[0][r][n] + parts[1][r][n]) + (parts[2][r][n] + parts[3][r][n]));
        }
    }
    // behind the sequence's end
    for (int64_t t = te + tid / CHANNELS; t < t1; t += 256 / CHANNELS) {
        if (!tlive) break;
        const int64_t at = out0 + t * a.channels + tchannel;
        static_cast<T*>(a.dx)[at] = from_f32<T>(0.f);
        static_cast<T*>(a.ddt)[at] = from_f32<T>(0.f);
        if (gated) static_cast<T*>(a.dgate)[at] = from_f32<T>(0.f);
    }
    for (int64_t v = static_cast<int64_t>(te) * (2 * S) + tid; v < static_cast<int64_t>(t1) * (2 * S); v += 256) bc[v] = 0.f;

    float* to = a.param_partial + (static_cast<int64_t>(batch) * a.chunks + chunk) * (S + 2) * cp;
    if (live) {
#pragma unroll
        for (int j = 0; j < SPL; ++j) to[(part * SPL + j) * cp + column] = dA[j];
        if (a.dstate != nullptr && chunk == 0) {
            float* ds = a.dstate + (static_cast<int64_t>(batch) * a.channels + channel) * a.states;
#pragma unroll
            for (int j = 0; j < SPL; ++j)
                if (part * SPL + j < a.states) ds[part * SPL + j] = carry[j];
        }
    }
    // dD and dbias: the threads of a channel, in order
    __syncthreads();
    tok[tid / CHANNELS][tc] = make_float4(dD, dbias, 0.f, 0.f);
    __syncthreads();
    if (tid < CHANNELS && tlive) {
        float sum_D = 0.f, sum_bias = 0.f;
#pragma unroll
        for (int i = 0; i < 256 / CHANNELS; ++i) {
            sum_D += tok[i][tc].x;
            sum_bias += tok[i][tc].y;
        }
        const int64_t at = static_cast<int64_t>(group) * a.group_tiles * 64 + first + tc;
        to[S * cp + at] = sum_D;
        to[(S + 1) * cp + at] = sum_bias;
    }
}

// dC and dB from the tiles' sums, tile after tile, four values a thread (S a power of two).
template <typename T>
__global__ __launch_bounds__(256) void state_space_bc_kernel(const float* partial, T* db, T* dc, int64_t rows,
                                                             int32_t S, int32_t states, int32_t groups,
                                                             int32_t group_tiles) {
    const int32_t quads = S / 2, lg = 31 - __builtin_clz(static_cast<uint32_t>(quads)), group = blockIdx.y;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows << lg;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = i >> lg;
        const int32_t in = static_cast<int32_t>(i & (quads - 1)) * 4, n = in < S ? in : in - S;
        const float* at = partial + (static_cast<int64_t>(group) * group_tiles * rows + row) * (2 * S) + in;
        float4 sum = *reinterpret_cast<const float4*>(at);
        for (int32_t k = 1; k < group_tiles; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(at + k * rows * (2 * S));
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        T* out = (in < S ? dc : db) + (row * groups + group) * states + n;
        alignas(16) const T v[4] = {from_f32<T>(sum.x), from_f32<T>(sum.y), from_f32<T>(sum.z), from_f32<T>(sum.w)};
        if (states % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (sizeof(v) - 1)) == 0) {
            if (n < states) {
                if constexpr (sizeof(v) == 16) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
                else *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < states) out[j] = v[j];
        }
    }
}

// How the backward cuts a line.  A workgroup of the gradients' pass takes a chunk of 256 /
// lanes channels; as many as the 256 CUs hold at once have one.  The adjoints' pass is one wave
// for 64 channels and cuts each chunk into fine ones, to give every SIMD four waves.
constexpr int64_t CUS = 256, TARGET_WAVES = 4096;

struct Cut {
    int64_t tiles, wide_tiles;               // of 64 channels, and of a workgroup's
    int64_t chunk, chunks;                   // tokens a chunk, chunks a line
    int64_t fine, fine_chunks, per_chunk;    // the same of the adjoints' pass
};
Cut make_cut(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    Cut c;
    c.tiles = ss_ceil(C / groups, 64) * groups;
    c.wide_tiles = ss_ceil(C / groups, states <= 8 ? 128 : 64) * groups;
    const int64_t blocks = ss_ceil(N, SS_BLOCK);
    int64_t chunks = CUS * backward_waves(states) / (B * c.wide_tiles);
    chunks = chunks < 1 || blocks <= 4 ? 1 : chunks > blocks ? blocks : chunks;   // few blocks: no adjoints' pass
    const int64_t per = ss_ceil(blocks, chunks);             // blocks a chunk
    c.chunk = per * SS_BLOCK;
    c.chunks = ss_ceil(N, c.chunk);
    // (a chunk is a multiple of 16 tokens, so the fine ones divide it)
    int64_t pieces = 1;
    while (pieces < 16 && c.chunks > 1 && c.chunk / pieces >= 32 && B * c.tiles * c.chunks * pieces * 2 <= TARGET_WAVES * 5 / 4)
        pieces *= 2;
    c.per_chunk = pieces;
    c.fine = c.chunk / pieces;
    c.fine_chunks = c.chunks == 1 ? 1 : ss_ceil(N, c.fine);
    return c;
}

struct Space {   // the workspace, in floats
    int64_t bc, slots, sums, params, maps, total_floats;   // bc first: it is read 16 bytes at a time
    size_t sum_bytes;
};
Space backward_space(const Cut& c, int64_t B, int64_t N, int32_t groups, int32_t states) {
    const int64_t cp = c.tiles * 64, S = ss_padded(states);
    Space s;
    s.bc = 0;
    s.slots = s.bc + c.wide_tiles * B * N * 2 * S;
    s.sums = s.slots + B * (c.fine_chunks - 1) * S * cp;
    s.params = s.sums + B * c.fine_chunks * cp;
    s.maps = s.params + B * c.chunks * (S + 2) * cp;
    s.total_floats = s.maps + ss_maps_floats(B, N, groups, states);
    s.sum_bytes = param_sum_workspace_bytes(B * c.chunks, S + 2, cp);
    return s;
}

template <typename T, typename BCT, int S>
int launch_backward(SSArgs& a, const Cut& c, int64_t B, hipStream_t s) {
    constexpr int LANES = S == 8 ? 2 : 4;
    a.wide_tiles = static_cast<int32_t>(c.wide_tiles);
    a.fine_chunks = static_cast<int32_t>(c.fine_chunks);
    a.fine_per_chunk = static_cast<int32_t>(c.per_chunk);
    if (c.chunks > 1) {
        a.chunk = static_cast<int32_t>(c.fine);
        a.chunks = static_cast<int32_t>(c.fine_chunks);
        a.first_chunk = 1;
        a.launch_chunks = a.chunks - 1;
        state_space_adjoint_kernel<T, BCT, S><<<static_cast<uint32_t>(B * a.launch_chunks * a.tiles), 64, 0, s>>>(a);
        if (int rc = check_launch("state_space chunk adjoints")) return rc;
        if (int rc = ss_join(a, B, S, true, a.dnew_state, s)) return rc;
    }
    a.chunk = static_cast<int32_t>(c.chunk);
    a.chunks = static_cast<int32_t>(c.chunks);
    state_space_backward_kernel<T, BCT, LANES, S / LANES>
        <<<static_cast<uint32_t>(B * c.chunks * c.wide_tiles), 256, 0, s>>>(a);
    return check_launch("state_space backward");
}

template <typename T, typename BCT>
int launch_states(SSArgs& a, const Cut& c, int64_t B, int32_t S, void* db, void* dc, hipStream_t s) {
    int rc = S == 8 ? launch_backward<T, BCT, 8>(a, c, B, s)
           : S == 16 ? launch_backward<T, BCT, 16>(a, c, B, s) : launch_backward<T, BCT, 32>(a, c, B, s);
    if (rc) return rc;
    const int64_t rows = B * a.tokens, blocks = ss_ceil(rows * S / 2, 256);
    const dim3 grid(static_cast<uint32_t>(blocks < 16384 ? blocks : 16384), a.groups);
    state_space_bc_kernel<T><<<grid, 256, 0, s>>>(a.bc_partial, static_cast<T*>(db), static_cast<T*>(dc), rows, S,
                                                  a.states, a.groups, a.wide_tiles / a.groups);
    return check_launch("state_space dB and dC");
}

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_state_space_backward_workspace_bytes(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    using namespace vh;
    if (B <= 0 || N <= 0 || C <= 0 || groups <= 0 || C % groups || states <= 0 || states > 32) return 0;
    const Space s = backward_space(make_cut(B, N, C, groups, states), B, N, groups, states);
    return static_cast<size_t>(s.total_floats) * sizeof(float) + s.sum_bytes;
}

int vh_state_space_backward(
    const void* dy, int64_t dy_batch, int64_t dy_token, const void* x, int64_t x_batch, int64_t x_token,
    const void* dt, int64_t dt_batch, int64_t dt_token, const void* gate, int64_t gate_batch, int64_t gate_token,
    int32_t io_dtype, const void* b, int64_t b_batch, int64_t b_token, const void* c, int64_t c_batch, int64_t c_token,
    const float* A, const float* D, const float* dt_bias, int32_t softplus, const int32_t* lengths,
    const float* kept, const float* dnew_state, void* dx, void* ddt, void* dgate, void* db, void* dc, float* dA,
    float* dD, float* ddt_bias, float* dstate, int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states,
    void* workspace, size_t workspace_bytes, void* stream) {
    using namespace vh;
    SSArgs a{};
    a.dy = {dy, dy_batch, dy_token};
    a.x = {x, x_batch, x_token};
    a.dt = {dt, dt_batch, dt_token};
    a.gate = {gate, gate_batch, gate_token};
    a.b = {b, b_batch, b_token};
    a.c = {c, c_batch, c_token};
    a.A = A;
    a.D = D;
    a.dt_bias = dt_bias;
    a.softplus = softplus;
    a.lengths = lengths;
    a.kept = const_cast<float*>(kept);
    a.dnew_state = dnew_state;
    a.dx = dx;
    a.ddt = ddt;
    a.dgate = dgate;
    a.dstate = dstate;
    if (int rc = ss_fill(a, io_dtype, B, N, C, groups, states)) return rc;
    VH_REQUIRE(dy != nullptr && kept != nullptr && dx != nullptr && ddt != nullptr && db != nullptr && dc != nullptr &&
                   (gate == nullptr) == (dgate == nullptr), VH_ERR_ARG,
               "dy, kept, dx, ddt, db and dc must be given, dgate exactly with a gate");
    const Cut cut = make_cut(B, N, C, groups, states);
    const Space sp = backward_space(cut, B, N, groups, states);
    const size_t need = static_cast<size_t>(sp.total_floats) * sizeof(float) + sp.sum_bytes;
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               VH_ERR_WORKSPACE, "state space backward needs a 16-byte aligned workspace of %zu bytes, got %zu", need,
               workspace_bytes);
    float* ws = static_cast<float*>(workspace);
    a.slots = ws + sp.slots;
    a.sums = ws + sp.sums;
    a.bc_partial = ws + sp.bc;
    a.param_partial = ws + sp.params;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int32_t S = ss_padded(states);
    int32_t bc_dtype = 0;
    int rc = ss_maps(a, io_dtype, ws + sp.maps, &bc_dtype, s);
    if (rc) return rc;
    if (io_dtype == VH_DTYPE_F32) rc = launch_states<float, float>(a, cut, B, S, db, dc, s);
    else if (io_dtype == VH_DTYPE_F16) rc = launch_states<f16_t, float>(a, cut, B, S, db, dc, s);
    else if (bc_dtype == VH_DTYPE_F32) rc = launch_states<bf16_t, float>(a, cut, B, S, db, dc, s);
    else rc = launch_states<bf16_t, bf16_t>(a, cut, B, S, db, dc, s);
    if (rc) return rc;
    ParamSum sum{};
    sum.partial = a.param_partial;
    sum.rows = B * cut.chunks;
    sum.quantities = S + 2;
    sum.padded = S;
    sum.columns = a.tiles * 64;
    sum.per_channel = states;
    sum.group_channels = a.group_channels;
    sum.group_tiles = a.group_tiles;
    sum.out0 = dA;
    sum.out1 = dD;
    sum.out2 = ddt_bias;
    return launch_param_sum(sum, ws + sp.total_floats, s);
}

}  // extern "C"
