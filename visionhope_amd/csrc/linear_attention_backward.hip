// Gradients of linear attention (linear_attention.hip), each the forward's form with other operands:
//
//   dq[i] = scale (sum_{j <= i} g^(i-j) (do[i] . v[j]) k[j] + g^(i+1) S do[i])
//   dv[j] = scale sum_{i >= j} g^(i-j) (q[i] . k[j]) do[i] + g^(n-1-j) G^T k[j]
//   dk[j] = scale sum_{i >= j} g^(i-j) (do[i] . v[j]) q[i] + g^(n-1-j) G v[j]
//   G'    = g^n G + scale sum_i g^(i+1) q[i] do[i]^T
//
// with S the state before a chunk of n tokens and G the gradient of the state behind it.  dq starts from
// the states that the forward left between its segments; G's are formed once, for dv, and read
// transposed for dk.  32 x 3136 x 3 heads of 64 in bf16: 45 (dq) + 17 + 6 + 43 (dv) + 43 us (dk).  dk and
// dv in one walk read a third less, but hold two workgroups a CU: with operands of two bf16 values 73 us
// instead of 77 for both there, and 141 instead of 118 for a training pass of 16 x 3136 x 6 heads of 32.
//
// A decay that is trained takes the states of both walks at every chunk, and one more pass:
//   dlog_decay = sum over chunks of  sum_{i > j} (i-j) g^(i-j) scale (q[i] . k[j]) (do[i] . v[j])
//              + <S, sum_i (i+1) g^(i+1) scale q[i] do[i]^T + n g^n G> + <G, sum_j (n-1-j) g^(n-1-j) k[j] v[j]^T>
// Powers stand beside small steps only, so nothing large cancels.  A training pass of 32 x 3136 x 3 heads of
// 64 in bf16 takes 464 us with it and 217 without, of 8 x 784 x 8 in FP32 174 and 103.
#include "linear_attention.h"

namespace vh {
namespace {

struct LADecayArgs {
    LATokens q, k, v, dout;
    const float *log_decay, *state, *dnew_state, *states, *adjoints;   // states: [B, heads, chunks - 1, D * D]
    float* partial;                                                     // [B, heads, chunks]
    const int32_t* lengths;
    float scale;
    int32_t tokens, heads, kdim, vdim, chunks;
    int32_t vec_q, vec_k, vec_v, vec_dout;   // elements of one load
};

// One chunk of one head: the share of a decay's gradient.
template <typename T, int D>
__global__ __launch_bounds__(4 * D, 2) void linear_attention_decay_kernel(const LADecayArgs a) {
    using P = LAShape<T, D>;
    constexpr int R = P::R, C = P::C, TILES = C / 16, STEPS_C = C / 32, STEPS_D = D / 32, TILE = P::tile * R;
    extern __shared__ __align__(16) unsigned char la_lds[];
    __shared__ float waves[P::waves];
    float* powers = reinterpret_cast<float*>(la_lds);
    uint16_t* tiles = reinterpret_cast<uint16_t*>(la_lds + P::head);
    const int32_t tid = static_cast<int32_t>(threadIdx.x), lane = tid & 63, wave = tid >> 6, n16 = lane & 15, g = lane >> 4;
    const int32_t chunk = static_cast<int32_t>(blockIdx.x % static_cast<uint32_t>(a.chunks));
    const int64_t bh = blockIdx.x / static_cast<uint32_t>(a.chunks);
    const int32_t head = static_cast<int32_t>(bh % a.heads);
    const int64_t batch = bh / a.heads;
    int32_t end = a.tokens;
    if (a.lengths != nullptr) end = a.lengths[batch] < 0 ? 0 : a.lengths[batch] > a.tokens ? a.tokens : a.lengths[batch];
    const int32_t t0 = chunk * C, nt = end - t0 < 0 ? 0 : end - t0 < C ? end - t0 : C;
    if (nt == 0) {
        if (tid == 0) a.partial[bh * a.chunks + chunk] = 0.f;
        return;
    }
    const LADecay decay(a.log_decay[head]);
    if (tid <= C) powers[tid] = decay.power(static_cast<float>(tid));
    const int32_t col = tid % (D / 8) * 8, row = tid / (D / 8);
    const LATokens from[4] = {a.q, a.k, a.dout, a.v};
    const int32_t vec[4] = {a.vec_q, a.vec_k, a.vec_dout, a.vec_v};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        const T* p = static_cast<const T*>(from[x].data) + batch * from[x].bs + head * from[x].hs;
#pragma unroll
        for (int u = 0; u < P::units; ++u) {
            const int32_t i = row + 32 * u;
            LAOct<T> raw{};
            if (i < nt) raw = la_load<T, false>(p + (t0 + i) * from[x].ts + col, col, x < 2 ? a.kdim : a.vdim, vec[x]);
            la_stage<T, D>(raw, tiles + x * TILE, col, i);
        }
    }
    __syncthreads();
    float sum = 0.f;
    // pairs within the chunk
    for (int32_t tile = wave; tile < TILES * (TILES + 1) / 2; tile += P::waves) {
        int32_t it = 0;
        while ((it + 1) * (it + 2) / 2 <= tile) ++it;
        const int32_t jt = tile - it * (it + 1) / 2;
        la_f32x4 w = {0.f, 0.f, 0.f, 0.f}, e = w;
#pragma unroll
        for (int x = 0; x < STEPS_D; ++x) {
            uint4 m[R], n[R];
            const int32_t at = la_block<D>(n16, g) ^ (32 * x), of_j = 16 * jt * D + at, of_i = 16 * it * D + at;
            la_read(tiles + TILE, P::tile, of_j, m);
            la_read(tiles, P::tile, of_i, n);
            w = la_mm(m, n, w);
            la_read(tiles + 3 * TILE, P::tile, of_j, m);
            la_read(tiles + 2 * TILE, P::tile, of_i, n);
            e = la_mm(m, n, e);
        }
        const int32_t d = 16 * it + n16 - (16 * jt + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (d - r > 0) sum = fmaf(w[r] * e[r], powers[d - r] * (static_cast<float>(d - r) * a.scale), sum);
    }
    // the chunk's sums over tokens in the states' layout
    const int32_t column = 16 * wave + n16, k_column = la_column<D, true>(lane), v_column = la_column<D, false>(lane);
    la_f32x4 before[D / 16], behind[D / 16];
    const int64_t all = a.chunks - 1;
    const int32_t last = (end - 1) / C;
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
        before[m] = behind[m] = la_f32x4{0.f, 0.f, 0.f, 0.f};
        const int64_t at = (wave * (D / 16) + m) * 64 + lane;
        if (chunk > 0) before[m] = reinterpret_cast<const la_f32x4*>(a.states + (bh * all + chunk - 1) * D * D)[at];
        if (chunk < last) behind[m] = reinterpret_cast<const la_f32x4*>(a.adjoints + (bh * all + chunk) * D * D)[at];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t row = la_state_row(m, g, r);
            const int64_t given = bh * a.kdim * a.vdim + row * a.vdim + column;
            if (row >= a.kdim || column >= a.vdim) continue;
            if (chunk == 0 && a.state != nullptr) before[m][r] = a.state[given];
            if (chunk == last && a.dnew_state != nullptr) behind[m][r] = a.dnew_state[given];
        }
    }
#pragma unroll
    for (int part = 0; part < 2; ++part) {   // q and do, k and v
        la_f32x4 acc[D / 16];
#pragma unroll
        for (int m = 0; m < D / 16; ++m) {
            acc[m] = la_f32x4{0.f, 0.f, 0.f, 0.f};
            if (part == 0) acc[m] = behind[m] * (static_cast<float>(nt) * powers[nt]);
        }
#pragma unroll
        for (int x = 0; x < STEPS_C; ++x) {
            uint4 va[R];
            la_turned<T, D, false>(tiles + (2 + part) * TILE, v_column, x, wave, va);
            float v[8];
            la_join8<R>(va, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int32_t t = 32 * x + 8 * g + i, m = part == 0 ? t + 1 : nt - 1 - t;
                v[i] *= m > 0 ? powers[m] * (static_cast<float>(m) * (part == 0 ? a.scale : 1.f)) : 0.f;
            }
            la_enter<T, D>(tiles + part * TILE, k_column, x, v, acc);
        }
#pragma unroll
        for (int m = 0; m < D / 16; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum = fmaf(acc[m][r], part == 0 ? before[m][r] : behind[m][r], sum);
    }
    sum = ln_lane_sum(sum, 6);
    if (lane == 0) waves[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < P::waves; ++w) total += waves[w];
        a.partial[bh * a.chunks + chunk] = total;
    }
}

// Sums of a head's shares over sequences and chunks, in a fixed order.
__global__ __launch_bounds__(256) void linear_attention_decay_sum_kernel(const float* partial, float* out, int32_t batches,
                                                                         int32_t heads, int32_t chunks) {
    __shared__ float waves[4];
    const int32_t head = static_cast<int32_t>(blockIdx.x);
    const int64_t total = static_cast<int64_t>(batches) * chunks;
    float sum = 0.f;
    for (int64_t i = threadIdx.x; i < total; i += 256) {
        const int64_t batch = i / chunks;
        sum += partial[(batch * heads + head) * chunks + (i - batch * chunks)];
    }
    sum = ln_lane_sum(sum, 6);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) out[head] = (waves[0] + waves[1]) + (waves[2] + waves[3]);
}

template <typename T>
int launch_decay(const LADecayArgs& a, int64_t B, float* out, hipStream_t stream) {
    const uint32_t grid = static_cast<uint32_t>(B * a.heads * a.chunks);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        linear_attention_decay_kernel<T, D><<<grid, 4 * D, LAShape<T, D>::head + 4 * LAShape<T, D>::R * LAShape<T, D>::tile * 2, stream>>>(a);
    };
    const int32_t padded = la_padded(a.kdim, a.vdim);
    if (padded == 32) go(std::integral_constant<int, 32>{});
    else if (padded == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    if (int rc = check_launch("linear_attention decay")) return rc;
    linear_attention_decay_sum_kernel<<<static_cast<uint32_t>(a.heads), 256, 0, stream>>>(a.partial, out, static_cast<int32_t>(B),
                                                                                     a.heads, a.chunks);
    return check_launch("linear_attention decay sum");
}

// Segments of the backward; with the decay's gradient every chunk is one, for its states.
LACut backward_cut(int64_t heads, int64_t N, int32_t padded, int32_t io_dtype, bool decay) {
    if (decay) return {static_cast<int32_t>(la_ceil(N, la_chunk(io_dtype))), 1};
    return la_cut(heads, N, padded, io_dtype);
}
size_t backward_bytes(int64_t heads, const LACut& cut, int32_t padded, bool decay) {
    const size_t slots = la_slots_bytes(heads, cut, padded);
    return decay ? 2 * slots + static_cast<size_t>(heads) * cut.segments * sizeof(float) : slots;
}

}  // namespace
}  // namespace vh

extern "C" {

size_t vh_linear_attention_backward_workspace_bytes(int64_t B, int64_t N, int64_t heads, int64_t key_dim,
                                                    int64_t value_dim, int32_t io_dtype, int32_t decay) {
    using namespace vh;
    if (la_check_sizes(io_dtype, B, N, heads, key_dim, value_dim) != VH_OK) return 0;
    const int32_t padded = la_padded(key_dim, value_dim);
    return backward_bytes(B * heads, backward_cut(B * heads, N, padded, io_dtype, decay != 0), padded, decay != 0);
}

int vh_linear_attention_backward(
    const void* dout, int64_t dout_batch, int64_t dout_token, int64_t dout_head, const void* q, int64_t q_batch,
    int64_t q_token, int64_t q_head, const void* k, int64_t k_batch, int64_t k_token, int64_t k_head, const void* v,
    int64_t v_batch, int64_t v_token, int64_t v_head, int32_t io_dtype, const float* log_decay, float scale,
    const float* state, const int32_t* lengths, const float* kept, const float* dnew_state, void* dq, void* dk, void* dv, float* dstate,
    float* dlog_decay, int64_t B, int64_t N, int64_t heads, int64_t key_dim, int64_t value_dim, void* workspace,
    size_t workspace_bytes, void* stream) {
    using namespace vh;
    if (int rc = la_check_sizes(io_dtype, B, N, heads, key_dim, value_dim)) return rc;
    if (int rc = la_check_strides({dout_token, q_token, k_token, v_token})) return rc;
    VH_REQUIRE(dout != nullptr && q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr && dq != nullptr &&
                   dk != nullptr && dv != nullptr, VH_ERR_ARG, "dout, q, k, v, log_decay, dq, dk and dv must not be null");
    VH_REQUIRE(!overlapping(dstate, dnew_state, B * heads * key_dim * value_dim * 4), VH_ERR_ARG,
               "dstate and dnew_state must not overlap");
    const int32_t padded = la_padded(key_dim, value_dim);
    const bool decay = dlog_decay != nullptr;
    const LACut cut = backward_cut(B * heads, N, padded, io_dtype, decay);
    const size_t need = backward_bytes(B * heads, cut, padded, decay);
    if (int rc = la_check_cut(B * heads, cut, padded)) return rc;
    VH_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               VH_ERR_WORKSPACE, "linear attention's backward needs an aligned workspace of %zu bytes, got %zu", need,
               workspace_bytes);
    VH_REQUIRE(decay || cut.segments == 1 || (kept != nullptr && reinterpret_cast<uintptr_t>(kept) % 16 == 0), VH_ERR_ARG,
               "linear attention's backward needs the states that the forward left in its workspace");
    const LATokens tq{q, q_batch, q_token, q_head}, tk{k, k_batch, k_token, k_head}, tv{v, v_batch, v_token, v_head};
    const LATokens tdo{dout, dout_batch, dout_token, dout_head};
    LAPass base{};
    base.log_decay = log_decay;
    base.scale_weight = scale;
    base.lengths = lengths;
    base.batches = static_cast<int32_t>(B);
    base.tokens = static_cast<int32_t>(N);
    base.heads = static_cast<int32_t>(heads);
    base.segments = cut.segments;
    base.chunks_per_segment = cut.each;
    const int32_t dk_ = static_cast<int32_t>(key_dim), dv_ = static_cast<int32_t>(value_dim);
    float* const adjoints = static_cast<float*>(workspace);
    float* const states = decay ? adjoints + la_slots_bytes(B * heads, cut, padded) / sizeof(float) : const_cast<float*>(kept);
    hipStream_t s = static_cast<hipStream_t>(stream);
    LAPass a = base;
    if (decay) {   // the forward's states are those between its segments
        a.q = a.k = tk;
        a.v = tv;
        a.kdim = dk_;
        a.vdim = dv_;
        a.scale_in = 1.f;
        a.state = state;
        a.state_row = value_dim;
        a.state_col = 1;
        a.slots = states;
        if (int rc = la_states(a, io_dtype, s)) return rc;
    }
    a = base;
    a.q = tdo;
    a.k = tv;
    a.v = tk;
    a.kdim = dv_;
    a.vdim = dk_;
    a.out = dq;
    a.scale_out = scale;
    a.scale_in = 1.f;
    a.state = state;
    a.state_row = 1;
    a.state_col = value_dim;
    a.slots = states;
    a.ready = a.turned = true;
    if (int rc = la_run(a, io_dtype, s)) return rc;

    base.reversed = 1;
    base.scale_out = 1.f;
    base.scale_in = scale;
    base.state = dnew_state;
    base.slots = adjoints;
    a = base;
    a.q = tk;
    a.k = tq;
    a.v = tdo;
    a.kdim = dk_;
    a.vdim = dv_;
    a.out = dv;
    a.state_row = value_dim;
    a.state_col = 1;
    a.new_state = dstate;
    if (int rc = la_run(a, io_dtype, s)) return rc;
    a = base;
    a.q = tv;
    a.k = tdo;
    a.v = tq;
    a.kdim = dv_;
    a.vdim = dk_;
    a.out = dk;
    a.state_row = 1;
    a.state_col = value_dim;
    a.ready = a.turned = true;
    if (int rc = la_run(a, io_dtype, s)) return rc;
    if (!decay) return VH_OK;

    LADecayArgs d{};
    d.q = tq;
    d.k = tk;
    d.v = tv;
    d.dout = tdo;
    d.log_decay = log_decay;
    d.state = state;
    d.dnew_state = dnew_state;
    d.adjoints = adjoints;
    d.states = states;
    d.partial = states + la_slots_bytes(B * heads, cut, padded) / sizeof(float);
    d.lengths = lengths;
    d.scale = scale;
    d.tokens = base.tokens;
    d.heads = base.heads;
    d.kdim = dk_;
    d.vdim = dv_;
    d.chunks = cut.segments;
    const int64_t e = dtype_bytes(io_dtype);
    d.vec_q = la_vec(tq, key_dim, e);
    d.vec_k = la_vec(tk, key_dim, e);
    d.vec_v = la_vec(tv, value_dim, e);
    d.vec_dout = la_vec(tdo, value_dim, e);
    if (io_dtype == VH_DTYPE_F32) return launch_decay<float>(d, B, dlog_decay, s);
    return io_dtype == VH_DTYPE_BF16 ? launch_decay<bf16_t>(d, B, dlog_decay, s) : launch_decay<f16_t>(d, B, dlog_decay, s);
}

}  // extern "C"
