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
#include "param_sum.h"
#include "state_space.h"

namespace vh {
namespace {

constexpr int UNROLL = 4;

// Adjoint that each chunk hands to the one before it from a zero adjoint behind it, and the
// chunk's sum of dt.
template <typename T, typename BCT, int S>
__global__ __launch_bounds__(64) void state_space_adjoint_kernel(const SSArgs a) {
    const SSPlace p = ss_place(a);
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;
    float A2[S], carry[S];
#pragma unroll
    for (int n = 0; n < S; ++n) {
        A2[n] = a.A[static_cast<int64_t>(p.channel) * S + n] * SS_LOG2E;
        carry[n] = 0.f;
    }
    const float bias = a.dt_bias != nullptr ? a.dt_bias[p.channel] : 0.f;
    const T* dt = static_cast<const T*>(a.dt.data) + p.batch * a.dt.bs + p.t0 * a.dt.ts;
    const T* dy = static_cast<const T*>(a.dy.data) + p.batch * a.dy.bs + p.t0 * a.dy.ts;
    const T* gate = a.gate.data != nullptr
        ? static_cast<const T*>(a.gate.data) + p.batch * a.gate.bs + p.t0 * a.gate.ts : nullptr;
    const int64_t c0 = p.batch * a.c.bs + p.t0 * a.c.ts + static_cast<int64_t>(p.group) * S;
    const int32_t count = p.te - p.t0;
    float total = 0.f;
    T dr[UNROLL], yr[UNROLL], gr[UNROLL], dn[UNROLL], yn[UNROLL], gn[UNROLL];
    auto fetch = [&](int32_t t) {   // tokens t, t - 1, ...
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int32_t at = t - u > 0 ? t - u : 0;
            dn[u] = dt[at * a.dt.ts + p.channel];
            yn[u] = dy[at * a.dy.ts + p.channel];
            if (gate != nullptr) gn[u] = gate[at * a.gate.ts + p.channel];
        }
    };
    if (count > 0) fetch(count - 1);
    for (int32_t t = count - 1; t >= 0; t -= UNROLL) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) { dr[u] = dn[u]; yr[u] = yn[u]; gr[u] = gn[u]; }
        if (t >= UNROLL) fetch(t - UNROLL);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (t - u < 0) break;
            SSRow<BCT, S> c;
            c.load(a.c.data, c0 + (t - u) * a.c.ts);
            float step = to_f32(dr[u]) + bias;
            if (a.softplus) step = ss_softplus(step);
            total += step;
            float dz = p.live ? to_f32(yr[u]) : 0.f;
            if (gate != nullptr) {
                const float z = to_f32(gr[u]);
                dz *= z * sigmoid_fast(z);
            }
#pragma unroll
            for (int n = 0; n < S; ++n)
                carry[n] = fmaf(c[n], dz, carry[n]) * __builtin_amdgcn_exp2f(step * A2[n]);
        }
    }
    float* to = a.slots + (static_cast<int64_t>(p.batch) * (a.chunks - 1) + p.chunk - 1) * S * cp + p.column;
#pragma unroll
    for (int n = 0; n < S; ++n) to[n * cp] = carry[n];
    a.sums[(static_cast<int64_t>(p.batch) * a.chunks + p.chunk) * cp + p.column] = total;
}

// Sums over the 64 lanes of M values a lane: each stage exchanges one bit of the lane index
// and halves the values, so lane l ends with value l * M / 64 (M = 16, 32 or 64).  The first
// two bits go by the row swaps, the others by DPP within 16 lanes.
template <int CTRL>
__device__ __forceinline__ float fold_dpp(float lo, float hi, bool upper) {
    const float keep = upper ? hi : lo, send = upper ? lo : hi;
    return keep + ln_dpp<CTRL>(send);
}
template <int M>
__device__ __forceinline__ float lane_fold(float (&v)[M]) {
    const int32_t lane = threadIdx.x & 63;
    static_assert(M == 16 || M == 32 || M == 64, "values a lane");
#pragma unroll
    for (int i = 0; i < M / 2; ++i) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 2]), false, false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 4; ++i) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 4]), false, false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 8; ++i) v[i] = fold_dpp<0x128>(v[i], v[i + M / 8], lane & 8);      // row_ror 8
#pragma unroll
    for (int i = 0; i < M / 16; ++i) v[i] = fold_dpp<0x141>(v[i], v[i + M / 16], lane & 4);    // i <-> 7 - i
    if constexpr (M >= 32) {
#pragma unroll
        for (int i = 0; i < M / 32; ++i) v[i] = fold_dpp<0x4E>(v[i], v[i + M / 32], lane & 2); // i <-> i ^ 2
    } else {
        v[0] += ln_dpp<0x4E>(v[0]);
    }
    if constexpr (M >= 64) return fold_dpp<0xB1>(v[0], v[1], lane & 1);                       // i <-> i ^ 1
    return v[0] + ln_dpp<0xB1>(v[0]);
}

template <typename T, typename BCT, int S>
__global__ __launch_bounds__(64) void state_space_backward_kernel(const SSArgs a) {
    constexpr int BLOCK = ss_block_tokens(S);
    constexpr int SUB = 64 / S, SUBS = BLOCK / SUB;   // tokens whose decays and states stand in registers
    static_assert(SUBS == 4, "a block is four sub-blocks");
    __shared__ float starts[SUBS][S][64];             // states before each sub-block
    const SSPlace p = ss_place(a);
    const int32_t lane = p.lane;
    const int64_t cp = static_cast<int64_t>(a.tiles) * 64;
    float A2[S], carry[S], dA[S];
#pragma unroll
    for (int n = 0; n < S; ++n) {
        A2[n] = a.A[static_cast<int64_t>(p.channel) * S + n] * SS_LOG2E;
        dA[n] = 0.f;
    }
    // the adjoint behind the chunk, times the decay of the token behind it
    if (p.chunk < a.chunks - 1) {
        const float* from = a.slots + (static_cast<int64_t>(p.batch) * (a.chunks - 1) + p.chunk) * S * cp + p.column;
#pragma unroll
        for (int n = 0; n < S; ++n) carry[n] = from[n * cp];
    } else {
        const float* from = a.dnew_state != nullptr
            ? a.dnew_state + (static_cast<int64_t>(p.batch) * a.channels + p.channel) * S : nullptr;
#pragma unroll
        for (int n = 0; n < S; ++n) carry[n] = from != nullptr && p.live ? from[n] : 0.f;
    }
    const float bias = a.dt_bias != nullptr ? a.dt_bias[p.channel] : 0.f;
    const float D = a.D != nullptr ? a.D[p.channel] : 0.f;
    float dD = 0.f, dbias = 0.f;
    const T* x = static_cast<const T*>(a.x.data) + p.batch * a.x.bs + p.channel;
    const T* dt = static_cast<const T*>(a.dt.data) + p.batch * a.dt.bs + p.channel;
    const T* dy = static_cast<const T*>(a.dy.data) + p.batch * a.dy.bs + p.channel;
    const T* gate = a.gate.data != nullptr
        ? static_cast<const T*>(a.gate.data) + p.batch * a.gate.bs + p.channel : nullptr;
    const int64_t b0 = p.batch * a.b.bs + static_cast<int64_t>(p.group) * S;
    const int64_t c0 = p.batch * a.c.bs + static_cast<int64_t>(p.group) * S;
    const int64_t out0 = static_cast<int64_t>(p.batch) * a.tokens * a.channels + p.channel;
    const int64_t bc_row0 = (static_cast<int64_t>(p.tile) * a.batches + p.batch) * a.tokens;

    const int32_t count = p.te - p.t0;
    for (int32_t blk = (count + BLOCK - 1) / BLOCK - 1; blk >= 0; --blk) {
        const int32_t tb = p.t0 + blk * BLOCK;                      // first token of the block
        const int32_t nb = p.te - tb < BLOCK ? p.te - tb : BLOCK;   // its tokens
        const int32_t last = (nb - 1) / SUB;
        {
            const float* from = a.kept + (static_cast<int64_t>(p.batch) * a.blocks + tb / BLOCK) * S * cp + p.column;
            float h[S];
#pragma unroll
            for (int n = 0; n < S; ++n) h[n] = from[n * cp];
            for (int32_t sub = 0; sub < last; ++sub) {
#pragma unroll
                for (int n = 0; n < S; ++n) starts[sub][n][lane] = h[n];
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const int64_t t = tb + sub * SUB + u;
                    SSRow<BCT, S> b;
                    b.load(a.b.data, b0 + t * a.b.ts);
                    float step = to_f32(dt[t * a.dt.ts]) + bias;
                    if (a.softplus) step = ss_softplus(step);
                    const float dtx = step * (p.live ? to_f32(x[t * a.x.ts]) : 0.f);
#pragma unroll
                    for (int n = 0; n < S; ++n)
                        h[n] = fmaf(dtx, b[n], h[n] * __builtin_amdgcn_exp2f(step * A2[n]));
                }
            }
#pragma unroll
            for (int n = 0; n < S; ++n) starts[last][n][lane] = h[n];
        }
        for (int32_t sub = last; sub >= 0; --sub) {
            const int32_t ts = tb + sub * SUB;
            const int32_t ns = p.te - ts < SUB ? p.te - ts : SUB;
            float decay[SUB][S], q[SUB][S], h[S];
            float raw[SUB], step[SUB], xv[SUB], gy[SUB], z[SUB];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const int64_t t = u < ns ? ts + u : ts + ns - 1;
                raw[u] = to_f32(dt[t * a.dt.ts]) + bias;
                xv[u] = to_f32(x[t * a.x.ts]);
                gy[u] = to_f32(dy[t * a.dy.ts]);
                z[u] = gate != nullptr ? to_f32(gate[t * a.gate.ts]) : 0.f;
            }
#pragma unroll
            for (int n = 0; n < S; ++n) h[n] = starts[sub][n][lane];
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                // tokens behind the sequence decay by one and add nothing
                const bool mine = p.live && u < ns;
                step[u] = a.softplus ? ss_softplus(raw[u]) : raw[u];
                step[u] = u < ns ? step[u] : 0.f;
                xv[u] = mine ? xv[u] : 0.f;
                gy[u] = mine ? gy[u] : 0.f;
                const float dtx = step[u] * xv[u];
                SSRow<BCT, S> b;
                b.load(a.b.data, b0 + static_cast<int64_t>(u < ns ? ts + u : ts + ns - 1) * a.b.ts);
#pragma unroll
                for (int n = 0; n < S; ++n) {
                    decay[u][n] = __builtin_amdgcn_exp2f(step[u] * A2[n]);
                    q[u][n] = decay[u][n] * h[n];
                    h[n] = fmaf(dtx, b[n], q[u][n]);
                }
            }
#pragma unroll
            for (int u = SUB - 1; u >= 0; --u) {
                if (u >= ns) continue;
                const int64_t t = ts + u;
                SSRow<BCT, S> b, c;
                b.load(a.b.data, b0 + t * a.b.ts);
                c.load(a.c.data, c0 + t * a.c.ts);
                float silu = 1.f, dsilu = 0.f;
                if (gate != nullptr) {
                    const float sig = sigmoid_fast(z[u]);
                    silu = z[u] * sig;
                    dsilu = sig * fmaf(z[u], 1.f - sig, 1.f);
                }
                const float dz = gy[u] * silu, dtx = step[u] * xv[u];
                float y = D * xv[u], gb = 0.f, ga = 0.f;
                float v[2 * S];
#pragma unroll
                for (int n = 0; n < S; ++n) {
                    const float hn = fmaf(dtx, b[n], q[u][n]);
                    const float g = fmaf(c[n], dz, carry[n]);
                    y = fmaf(c[n], hn, y);
                    gb = fmaf(g, b[n], gb);
                    const float gq = g * q[u][n];
                    ga = fmaf(gq, A2[n], ga);
                    dA[n] = fmaf(gq, step[u], dA[n]);
                    carry[n] = g * decay[u][n];
                    v[n] = dz * hn;
                    v[S + n] = dtx * g;
                }
                const float sum = lane_fold<2 * S>(v);
                constexpr int SHARE = 64 / (2 * S);
                if (lane % SHARE == 0) a.bc_partial[(bc_row0 + t) * (2 * S) + lane / SHARE] = sum;
                // A2 is A log2(e)
                float ddt = fmaf(xv[u], gb, ga * 0.6931471805599453f);
                if (a.softplus) ddt *= sigmoid_fast(raw[u]);
                const float dxv = fmaf(step[u], gb, D * dz);
                dD = fmaf(dz, xv[u], dD);
                dbias += ddt;
                if (p.live) {
                    const int64_t at = out0 + t * a.channels;
                    static_cast<T*>(a.dx)[at] = from_f32<T>(dxv);
                    static_cast<T*>(a.ddt)[at] = from_f32<T>(ddt);
                    if (gate != nullptr) static_cast<T*>(a.dgate)[at] = from_f32<T>(gy[u] * y * dsilu);
                }
            }
        }
    }
    // behind the sequence's end
    for (int64_t t = p.te; t < p.t1; ++t) {
        if (p.live) {
            const int64_t at = out0 + t * a.channels;
            static_cast<T*>(a.dx)[at] = from_f32<T>(0.f);
            static_cast<T*>(a.ddt)[at] = from_f32<T>(0.f);
            if (gate != nullptr) static_cast<T*>(a.dgate)[at] = from_f32<T>(0.f);
        }
        if (lane < 2 * S) a.bc_partial[(bc_row0 + t) * (2 * S) + lane] = 0.f;
    }
    float* to = a.param_partial + (static_cast<int64_t>(p.batch) * a.chunks + p.chunk) * (S + 2) * cp + p.column;
#pragma unroll
    for (int n = 0; n < S; ++n) to[n * cp] = dA[n];
    to[S * cp] = dD;
    to[(S + 1) * cp] = dbias;
    if (a.dstate != nullptr && p.chunk == 0 && p.live) {
        float* ds = a.dstate + (static_cast<int64_t>(p.batch) * a.channels + p.channel) * S;
#pragma unroll
        for (int n = 0; n < S; n += 4)
            *reinterpret_cast<float4*>(ds + n) = make_float4(carry[n], carry[n + 1], carry[n + 2], carry[n + 3]);
    }
}

// dC and dB from the tiles' sums, tile after tile.
template <typename T>
__global__ __launch_bounds__(256) void state_space_bc_kernel(const float* partial, T* db, T* dc, int64_t rows,
                                                             int32_t S, int32_t groups, int32_t group_tiles) {
    const int64_t width = 2 * S, total = rows * groups * width;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t in = i % width, group = (i / width) % groups, row = i / (width * groups);
        const float* at = partial + (group * group_tiles * rows + row) * width + in;
        float sum = 0.f;
        for (int32_t k = 0; k < group_tiles; ++k) sum += at[k * rows * width];
        T* out = in < S ? dc : db;
        out[(row * groups + group) * S + (in < S ? in : in - S)] = from_f32<T>(sum);
    }
}

// Chunks of the backward: two waves a SIMD (its registers allow no more), whole blocks.
constexpr int64_t TARGET_WAVES = 2048;

int64_t backward_chunk(int64_t B, int64_t N, int64_t tiles, int32_t states) {
    const int64_t block = ss_block_tokens(states), blocks = ss_ceil(N, block);
    int64_t chunks = TARGET_WAVES / (B * tiles);
    if (chunks < 1) chunks = 1;
    if (chunks > blocks) chunks = blocks;
    return ss_ceil(blocks, chunks) * block;
}

struct Space {   // the workspace, in floats
    int64_t slots, sums, bc, params, total_floats;
    size_t sum_bytes;
};
Space backward_space(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    const int64_t tiles = ss_ceil(C / groups, 64) * groups, cp = tiles * 64;
    const int64_t chunks = ss_ceil(N, backward_chunk(B, N, tiles, states));
    Space s;
    s.slots = 0;
    s.sums = s.slots + B * (chunks - 1) * states * cp;
    s.bc = s.sums + B * chunks * cp;
    s.params = s.bc + tiles * B * N * 2 * states;
    s.total_floats = s.params + B * chunks * (states + 2) * cp;
    s.sum_bytes = param_sum_workspace_bytes(B * chunks, states + 2, cp);
    return s;
}

template <typename T, typename BCT, int S>
int launch_backward(SSArgs& a, int64_t B, hipStream_t s) {
    if (a.chunks > 1) {
        a.first_chunk = 1;
        a.launch_chunks = a.chunks - 1;
        state_space_adjoint_kernel<T, BCT, S><<<static_cast<uint32_t>(B * a.launch_chunks * a.tiles), 64, 0, s>>>(a);
        if (int rc = check_launch("state_space chunk adjoints")) return rc;
        if (int rc = ss_join(a, B, S, true, a.dnew_state, s)) return rc;
    }
    a.first_chunk = 0;
    a.launch_chunks = a.chunks;
    state_space_backward_kernel<T, BCT, S><<<static_cast<uint32_t>(B * a.chunks * a.tiles), 64, 0, s>>>(a);
    return check_launch("state_space backward");
}

template <typename T, typename BCT>
int launch_states(SSArgs& a, int64_t B, int32_t S, void* db, void* dc, int32_t groups, hipStream_t s) {
    int rc = S == 8 ? launch_backward<T, BCT, 8>(a, B, s)
           : S == 16 ? launch_backward<T, BCT, 16>(a, B, s) : launch_backward<T, BCT, 32>(a, B, s);
    if (rc) return rc;
    const int64_t rows = B * a.tokens, blocks = ss_ceil(rows * groups * 2 * S, 256);
    state_space_bc_kernel<T><<<static_cast<uint32_t>(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(
        a.bc_partial, static_cast<T*>(db), static_cast<T*>(dc), rows, S, groups, a.group_tiles);
    return check_launch("state_space dB and dC");
}

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_state_space_backward_workspace_bytes(int64_t B, int64_t N, int64_t C, int32_t groups, int32_t states) {
    using namespace vh;
    if (B <= 0 || N <= 0 || C <= 0 || groups <= 0 || C % groups || states <= 0) return 0;
    const Space s = backward_space(B, N, C, groups, states);
    return static_cast<size_t>(s.total_floats) * sizeof(float) + s.sum_bytes;
}

int vh_state_space_backward(
    const void* dy, int64_t dy_batch, int64_t dy_token, const void* x, int64_t x_batch, int64_t x_token,
    const void* dt, int64_t dt_batch, int64_t dt_token, const void* gate, int64_t gate_batch, int64_t gate_token,
    int32_t io_dtype, const void* b, int64_t b_batch, int64_t b_token, const void* c, int64_t c_batch, int64_t c_token,
    int32_t bc_dtype, const float* A, const float* D, const float* dt_bias, int32_t softplus, const int32_t* lengths,
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
    if (int rc = ss_fill(a, io_dtype, bc_dtype, B, N, C, groups, states)) return rc;
    VH_REQUIRE(dy != nullptr && kept != nullptr && dx != nullptr && ddt != nullptr && db != nullptr && dc != nullptr &&
                   (gate == nullptr) == (dgate == nullptr), VH_ERR_ARG,
               "dy, kept, dx, ddt, db and dc must be given, dgate exactly with a gate");
    VH_REQUIRE(reinterpret_cast<uintptr_t>(dstate) % 16 == 0, VH_ERR_ARG, "dstate must be 16-byte aligned");
    const Space sp = backward_space(B, N, C, groups, states);
    const size_t need = static_cast<size_t>(sp.total_floats) * sizeof(float) + sp.sum_bytes;
    VH_REQUIRE(workspace != nullptr && workspace_bytes >= need, VH_ERR_WORKSPACE,
               "state space backward needs a workspace of %zu bytes, got %zu", need, workspace_bytes);
    float* ws = static_cast<float*>(workspace);
    a.slots = ws + sp.slots;
    a.sums = ws + sp.sums;
    a.bc_partial = ws + sp.bc;
    a.param_partial = ws + sp.params;
    a.chunk = static_cast<int32_t>(backward_chunk(B, N, a.tiles, states));
    a.chunks = static_cast<int32_t>(ss_ceil(N, a.chunk));
    hipStream_t s = static_cast<hipStream_t>(stream);
    int rc;
    if (io_dtype == VH_DTYPE_F32) rc = launch_states<float, float>(a, B, states, db, dc, groups, s);
    else if (io_dtype == VH_DTYPE_F16) rc = launch_states<f16_t, float>(a, B, states, db, dc, groups, s);
    else if (bc_dtype == VH_DTYPE_F32) rc = launch_states<bf16_t, float>(a, B, states, db, dc, groups, s);
    else rc = launch_states<bf16_t, bf16_t>(a, B, states, db, dc, groups, s);
    if (rc) return rc;
    ParamSum sum{};
    sum.partial = a.param_partial;
    sum.rows = B * a.chunks;
    sum.quantities = states + 2;
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
