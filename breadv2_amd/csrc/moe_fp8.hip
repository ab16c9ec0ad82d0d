// moe_fp8.hip — bread_moe_expert_block_fp8: the routed experts of a layer with
// e4m3 weights and the caller's routing,
//   hidden[t] = residual[t] + sum_k w[t][k] down_e(q(silu(gate_e x) * (up_e x))),  e = idx[t][k].
// Pairs (token, rank) are sorted by expert; gate and up are one grouped product
// that ends in codes by pair, down another (fp8_grouped.hip), and the pairs of a
// token are added in rank order.  Few pairs of experts with an inner size of
// 256, 512 or 1024 skip the sorting: a wave a row, one kernel for gate and up and
// one for the rest, whose lanes a pair (I / 16) have to divide a wave.  Other
// sizes are sorted however few the pairs are: one token, top 8, hidden 2048, takes
// 11 us with 512, 17 with 1024, but 31 with 768, 38 with 1536 and 41 with 2048.
#include "activate.h"
#include "fp8.h"

namespace {

// ---------------------------------------------------------------------------
// Pairs by expert
// ---------------------------------------------------------------------------

// offsets [E + 1], token[i] of sorted row i, place[p] of pair p (-1: no expert); an expert's pairs in their order.  A
// workgroup an expert: it reads all pairs' experts (from the L2 after the first), counts those before its own and its
// own, wave by wave, and lists its own.  us at 4096 tokens, top 8, 256 experts, some of them with 1500 pairs: one
// workgroup that counts and places by LDS atomics 36, a workgroup an expert that places by them 20, this 17 (with eight
// waves) and 14.
__global__ __launch_bounds__(1024) void k_f8_bucket(const int32_t *__restrict__ idx, int P, int K, int E,
                                                   int32_t *__restrict__ offsets, int32_t *__restrict__ token,
                                                   int32_t *__restrict__ place, uint32_t *__restrict__ err)
{
    constexpr int AT_A_TIME = 16, WAVES = 16;
    __shared__ int less_of[WAVES], own_of[WAVES];
    const int e = (int)blockIdx.x, l = lane_id(), wv = wave_id();
    // a wave's share of the pairs is contiguous, whole groups of 64 AT_A_TIME
    const int share = ((P + WAVES - 1) / WAVES + WAVE * AT_A_TIME - 1) / (WAVE * AT_A_TIME) * (WAVE * AT_A_TIME);
    const int begin = wv * share, end = min(begin + share, P);
    auto load = [&](int p0, int (&v)[AT_A_TIME]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AT_A_TIME; i++) {
            const int p = p0 + i * WAVE + l;
            v[i] = p < end ? idx[p] : INT32_MAX;
        }
    };
    int less = 0, own = 0;
    bool bad = false;
    for (int p0 = begin; p0 < end; p0 += WAVE * AT_A_TIME) {
        int v[AT_A_TIME];
        load(p0, v);
#pragma unroll
        for (int i = 0; i < AT_A_TIME; i++) {
            less += (unsigned)v[i] < (unsigned)e;
            own += v[i] == e;
            if (e == 0 && p0 + i * WAVE + l < end && (unsigned)v[i] >= (unsigned)E) {  // no expert
                bad = true;
                place[p0 + i * WAVE + l] = -1;
            }
        }
    }
    if (bad) __hip_atomic_fetch_or(err, BREAD_DEV_ERR_INDEX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    less = wave_scan_incl(less);
    own = wave_scan_incl(own);
    if (l == WAVE - 1) {
        less_of[wv] = less;
        own_of[wv] = own;
    }
    __syncthreads();
    int at = 0, first = 0, all = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        first += less_of[i];
        all += own_of[i];
        if (i < wv) at += own_of[i];
    }
    at += first;
    if (threadIdx.x == 0) {
        offsets[e] = first;
        if (e == E - 1) offsets[E] = first + all;
    }
    for (int p0 = begin; p0 < end; p0 += WAVE * AT_A_TIME) {
        int v[AT_A_TIME];
        load(p0, v);
#pragma unroll
        for (int i = 0; i < AT_A_TIME; i++) {
            const uint64_t mine = __builtin_amdgcn_ballot_w64(v[i] == e);
            if (!mine) continue;
            if (v[i] == e) {
                const int p = p0 + i * WAVE + l, o = at + __builtin_popcountll(mine & ((1ull << l) - 1));
                token[o] = (int)((uint32_t)p / (uint32_t)K);
                place[p] = o;
            }
            at += __builtin_popcountll(mine);
        }
    }
}

// ---------------------------------------------------------------------------
// A few tokens
// ---------------------------------------------------------------------------
// us of one token, top 8, hidden 2048, inter 512: gate and up 6.0 (16.8 MB of weights: 3.2 at the copy rate), down 6.4
// (8.4 MB; 11.5 with sixteen rows a workgroup and the lanes a pair not a constant); sorting and the grouped products take
// 29 together.  Their time is the chain routing, weights, sum.

typedef float f32x2 __attribute__((ext_vector_type(2)));

// sum of w[i] x[i] over sixteen codes each
__device__ __forceinline__ float dot16(const uint4 &w, const uint4 &x)
{
    const uint32_t a[4] = {w.x, w.y, w.z, w.w}, b[4] = {x.x, x.y, x.z, x.w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const f32x2 a0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], true);
        const f32x2 b0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], false), b1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)b[i], true);
        s = fmaf(a0[0], b0[0], s);
        s = fmaf(a0[1], b0[1], s);
        s = fmaf(a1[0], b1[0], s);
        s = fmaf(a1[1], b1[1], s);
    }
    return s;
}

__device__ __forceinline__ uint4 ld16(const uint8_t *p)
{
    return *reinterpret_cast<const uint4 *>(p);
}

__device__ __forceinline__ float lane_value(float v, int lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

struct FewArgs {
    const uint8_t *gate, *up, *down, *x;
    const float *gs, *us, *ds, *xs;
    const int32_t *idx;
    const float *w;
    float *h;  // [pairs][I]
    const void *residual;
    void *hidden;
    uint32_t *err;
    int H, I, K, E, type;
};

// h[pair][r] = silu(gate r) * (up r), a wave a row: lanes hold sixteen columns each, adjacent lanes adjacent ones
__global__ __launch_bounds__(256) void k_f8_few_gateup(const FewArgs a)
{
    const int pair = (int)blockIdx.y, r = (int)blockIdx.x * 4 + wave_id(), l = lane_id(), t = pair / a.K;
    const int e = a.idx[pair], nb = a.H / F8_BLOCK, nrb = a.I / F8_BLOCK;
    if ((unsigned)e >= (unsigned)a.E) {
        if (r == 0 && l == 0) __hip_atomic_fetch_or(a.err, BREAD_DEV_ERR_INDEX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    const size_t row = ((size_t)e * a.I + r) * a.H, sc = ((size_t)e * nrb + r / F8_BLOCK) * nb;
    const uint8_t *x = a.x + (size_t)t * a.H;
    float g = 0.f, u = 0.f;
#pragma unroll 2
    for (int c = 16 * l; c < a.H; c += 16 * WAVE) {
        const uint4 gq = ld16(a.gate + row + c), uq = ld16(a.up + row + c), xq = ld16(x + c);
        const int b = c / F8_BLOCK;
        const float xs = a.xs[(size_t)t * nb + b];
        g = fmaf(dot16(gq, xq), xs * a.gs[sc + b], g);
        u = fmaf(dot16(uq, xq), xs * a.us[sc + b], u);
    }
    g = wave_sum(g);
    u = wave_sum(u);
    if (l == 0) a.h[(size_t)pair * a.I + r] = activate(g, BREAD_ACT_SILU) * u;
}

constexpr int FEW_ROWS = 8;      // rows of hidden of a workgroup, one a wave

// hidden[t][r] = residual + sum_k w[k] down_k(q(h[k])) r: a workgroup quantises its token's pairs (as each does), then
// a wave a row, whose weights were requested before; in LDS K x I codes and their scales.  PER = I / 16 lanes a pair.
template <int PER>
__global__ __launch_bounds__(FEW_ROWS *WAVE) void k_f8_few_down(const FewArgs a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int t = (int)blockIdx.y, tid = (int)threadIdx.x, l = lane_id(), r = (int)blockIdx.x * FEW_ROWS + wave_id();
    const int nb = a.I / F8_BLOCK, nrb = a.H / F8_BLOCK, n = a.K * a.I;
    uint8_t *codes = lds;
    float *scales = reinterpret_cast<float *>(lds + n);
    // lane k: expert and weight of rank k (K <= 32); lanes in groups of I / 16 for a pair
    const int ek = l < a.K ? a.idx[t * a.K + l] : -1;
    const bool is = (unsigned)ek < (unsigned)a.E;
    const float wk = is ? a.w[t * a.K + l] : 0.f;
    const uint64_t valid = __builtin_amdgcn_ballot_w64(is);
    constexpr int AT_ONCE = WAVE / PER, AHEAD = 8 / AT_ONCE;  // eight pairs
    const int c = 16 * (l % PER), b = c / F8_BLOCK;
    uint4 q[AHEAD];
    float sc[AHEAD];
    auto load = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int k = k0 + i * AT_ONCE + l / PER;
            q[i] = make_uint4(0u, 0u, 0u, 0u);
            sc[i] = 0.f;
            const int e = __shfl(ek, k & 63);
            if (k < a.K && (unsigned)e < (unsigned)a.E) {
                q[i] = ld16(a.down + ((size_t)e * a.H + r) * a.I + c);
                sc[i] = a.ds[((size_t)e * nrb + r / F8_BLOCK) * nb + b];
            }
        }
    };
    load(0);
    float acc = 0.f;
    if (a.residual)
        acc = a.type == BREAD_QTYPE_F32 ? static_cast<const float *>(a.residual)[(size_t)t * a.H + r]
              : a.type == BREAD_QTYPE_F16 ? h2f(static_cast<const uint16_t *>(a.residual)[(size_t)t * a.H + r])
                                          : bf2f(static_cast<const uint16_t *>(a.residual)[(size_t)t * a.H + r]);
    // (four values a thread: 32 lanes a block)
    for (int i = 4 * tid; i < n; i += 4 * FEW_ROWS * WAVE) {
        const float4 v = *reinterpret_cast<const float4 *>(a.h + (size_t)t * n + i);
        uint32_t m = max(max(f8_mag(v.x), f8_mag(v.y)), max(f8_mag(v.z), f8_mag(v.w)));
#pragma unroll
        for (int d = 1; d < 32; d *= 2) m = max(m, (uint32_t)__shfl_xor((int)m, d));
        const float s = f8_scale(m);
        *reinterpret_cast<uint32_t *>(codes + i) = f8_pack4(v.x, v.y, v.z, v.w, 1.0f / s);
        if (tid % 32 == 0) scales[i / F8_BLOCK] = s;
    }
    __syncthreads();
    for (int k0 = 0; k0 < a.K; k0 += AHEAD * AT_ONCE) {
        if (k0) load(k0);
        float y[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int k = k0 + i * AT_ONCE + l / PER;
            y[i] = 0.f;
            if (k < a.K && (valid >> k & 1)) y[i] = dot16(q[i], ld16(codes + k * a.I + c)) * (scales[k * nb + b] * sc[i]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
#pragma unroll
            for (int d = 1; d < PER; d *= 2) y[i] += __shfl_xor(y[i], d);
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
#pragma unroll
            for (int j = 0; j < AT_ONCE; j++) {
                const int k = k0 + i * AT_ONCE + j;
                if (k < a.K && (valid >> k & 1)) acc = fmaf(lane_value(wk, k), lane_value(y[i], j * PER), acc);
            }
    }
    if (l == 0) {
        if (a.type == BREAD_QTYPE_F32) static_cast<float *>(a.hidden)[(size_t)t * a.H + r] = acc;
        else static_cast<uint16_t *>(a.hidden)[(size_t)t * a.H + r] = a.type == BREAD_QTYPE_F16 ? f2h(acc) : f2bf(acc);
    }
}

// ---------------------------------------------------------------------------
// The pairs' sum
// ---------------------------------------------------------------------------

__device__ __forceinline__ void load4(const void *p, int64_t at, int type, float (&v)[4])
{
    if (type == BREAD_QTYPE_F32) {
        const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        v[0] = f.x;
        v[1] = f.y;
        v[2] = f.z;
        v[3] = f.w;
        return;
    }
    uint16_t h[4];
    __builtin_memcpy(h, __builtin_assume_aligned(static_cast<const uint16_t *>(p) + at, 8), 8);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = type == BREAD_QTYPE_F16 ? h2f(h[i]) : bf2f(h[i]);
}

// hidden[t] = residual[t] + sum of w times the pairs' rows in rank order, rounded once
__global__ __launch_bounds__(256) void k_f8_combine(const float *__restrict__ eo, const int32_t *__restrict__ place,
                                                    const float *__restrict__ w, const void *residual, void *hidden,
                                                    int type, int H, int K)
{
    const int64_t t = blockIdx.x;
    const int c = 4 * (int)(blockIdx.y * 256 + threadIdx.x);
    if (c >= H) return;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (residual) load4(residual, t * H + c, type, acc);
#pragma unroll 8
    for (int k = 0; k < K; k++) {
        const int p = place[t * K + k];
        if (p < 0) continue;
        const float wk = w[t * K + k];
        const float4 v = *reinterpret_cast<const float4 *>(eo + (int64_t)p * H + c);
        acc[0] = fmaf(wk, v.x, acc[0]);
        acc[1] = fmaf(wk, v.y, acc[1]);
        acc[2] = fmaf(wk, v.z, acc[2]);
        acc[3] = fmaf(wk, v.w, acc[3]);
    }
    if (type == BREAD_QTYPE_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(hidden) + t * H + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    } else {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = type == BREAD_QTYPE_F16 ? f2h(acc[i]) : f2bf(acc[i]);
        __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t *>(hidden) + t * H + c, 8), h, 8);
    }
}

// Whether calls skip the sorting: by estimates of both, ns, fitted to 27 shapes of 9 to 256 experts.  Without it every pair
// reads its expert's weights (of some of them from the L2), and every token takes a wave for each of its values; with it
// four launches follow one another.  us without and with: 256 experts of 512, hidden 2048, top 8, 2 tokens 16 and 32, 4 24
// and 39, 6 33 and 46, 8 41 and 47; 10 experts of 256, hidden 2048, top 7, 8 tokens 18 and 33, 29 50 and 31; 12 of 256,
// hidden 512, top 2, 40 tokens 17 and 20, 100 34 and 20.
bool few(int64_t T, int64_t pairs, int64_t H, int64_t I)
{
    return pairs * 3 * H * I / 6250 + T * H / 4 <= 14000 + 7 * H;
}

}  // namespace

extern "C" int bread_moe_expert_block_fp8(bread_moe_ctx_t *c, const bread_fp8_experts_t *ex, const void *x,
                                          const float *x_scale, const void *residual, void *hidden, int hidden_type,
                                          int T, const int32_t *idx, const float *w, bread_stream_t stream)
{
    BREAD_REQUIRE(c && ex, BREAD_ERR_ARG, "NULL context or experts");
    BREAD_REQUIRE(T >= 0, BREAD_ERR_ARG, "n_tokens < 0");
    BREAD_REQUIRE(T <= c->max_tokens, BREAD_ERR_CAPACITY, "n_tokens > max_tokens of the context");
    BREAD_REQUIRE(f8_wide_type(hidden_type), BREAD_ERR_QTYPE, "hidden_type must be 0 (F32), 1 (F16) or 30 (BF16)");
    BREAD_REQUIRE(ex->gate && ex->up && ex->down && ex->gate_scale && ex->up_scale && ex->down_scale, BREAD_ERR_ARG,
                  "NULL weights or scales");
    BREAD_REQUIRE((((uintptr_t)ex->gate | (uintptr_t)ex->up | (uintptr_t)ex->down) & 15) == 0 &&
                      (((uintptr_t)ex->gate_scale | (uintptr_t)ex->up_scale | (uintptr_t)ex->down_scale) & 3) == 0,
                  BREAD_ERR_ALIGN, "weights must be 16-byte aligned, scales 4-byte aligned");
    if (T == 0) return BREAD_OK;
    int device;
    BREAD_HIP(hipGetDevice(&device));
    BREAD_REQUIRE(device == c->device, BREAD_ERR_ARG, "the context was made on another device than the current one");
    BREAD_REQUIRE(x && x_scale && hidden && idx && w, BREAD_ERR_ARG, "NULL pointer");
    BREAD_REQUIRE((((uintptr_t)x | (uintptr_t)hidden | (uintptr_t)residual) & 15) == 0 &&
                      (((uintptr_t)x_scale | (uintptr_t)idx | (uintptr_t)w) & 3) == 0,
                  BREAD_ERR_ALIGN, "x, residual and hidden must be 16-byte aligned, the others 4-byte aligned");
    const bread_moe_shape_t &s = c->shape;
    BREAD_REQUIRE((int64_t)T * s.hidden <= 1ll << 31, BREAD_ERR_SHAPE, "x of more than 2^31 bytes");
    const int H = s.hidden, I = s.expert_inter, K = s.top_k, P = T * K;
    const hipStream_t st = to_hip(stream);
    c->last_stream = st;
    bread_grouped_ws &g = c->gws;
    bread_clear_stale_error();
    const int few_lds = K * I + 4 * K * f8_blocks(I);
    if (few(T, P, H, I) && (I == 256 || I == 512 || I == 1024) && few_lds <= 64 * 1024) {
        FewArgs f;
        f.gate = static_cast<const uint8_t *>(ex->gate);
        f.up = static_cast<const uint8_t *>(ex->up);
        f.down = static_cast<const uint8_t *>(ex->down);
        f.x = static_cast<const uint8_t *>(x);
        f.gs = ex->gate_scale;
        f.us = ex->up_scale;
        f.ds = ex->down_scale;
        f.xs = x_scale;
        f.idx = idx;
        f.w = w;
        f.h = c->h;
        f.residual = residual;
        f.hidden = hidden;
        f.err = &c->dsync->error.v;
        f.H = H;
        f.I = I;
        f.K = K;
        f.E = s.n_experts;
        f.type = hidden_type;
        hipLaunchKernelGGL(k_f8_few_gateup, dim3((unsigned)I / 4, (unsigned)P), dim3(256), 0, st, f);
        BREAD_HIP(hipGetLastError());
        const auto down = I == 256 ? k_f8_few_down<16> : I == 512 ? k_f8_few_down<32> : k_f8_few_down<64>;
        hipLaunchKernelGGL(down, dim3((unsigned)H / FEW_ROWS, (unsigned)T), dim3(FEW_ROWS * WAVE), (unsigned)few_lds, st, f);
        BREAD_HIP(hipGetLastError());
        return BREAD_OK;
    }
    hipLaunchKernelGGL(k_f8_bucket, dim3((unsigned)s.n_experts), dim3(1024), 0, st, idx, P, K, s.n_experts, g.offsets, g.pair_tok, g.pos_of,
                       &c->dsync->error.v);
    BREAD_HIP(hipGetLastError());
    // codes and scales by pair: less than the fp32 values that c->h holds for the other paths
    uint8_t *codes = reinterpret_cast<uint8_t *>(c->h);
    float *scales = reinterpret_cast<float *>(codes + (size_t)P * I);
    F8Args a;
    a.w = static_cast<const uint8_t *>(ex->gate);
    a.up = static_cast<const uint8_t *>(ex->up);
    a.ws = ex->gate_scale;
    a.us = ex->up_scale;
    a.x = static_cast<const uint8_t *>(x);
    a.xs = x_scale;
    a.x_stride = H;
    a.xs_stride = f8_blocks(H);
    a.y = codes;
    a.ys = scales;
    a.y_stride = I;
    a.ys_stride = f8_blocks(I);
    a.bias = nullptr;
    a.res = nullptr;
    a.rows = I;
    a.cols = H;
    a.T = P;
    a.act = BREAD_ACT_SILU;
    a.y_type = BREAD_QTYPE_E4M3;
    a.G = s.n_experts;
    a.offsets = g.offsets;
    a.x_rows = g.pair_tok;
    a.n_x = T;
    a.y_rows = nullptr;
    a.n_y = 0;
    int rc = bread_launch_fp8_matmul(a, st);
    if (rc) return rc;
    a.w = static_cast<const uint8_t *>(ex->down);
    a.ws = ex->down_scale;
    a.up = nullptr;
    a.us = nullptr;
    a.x = codes;
    a.xs = scales;
    a.x_stride = I;
    a.xs_stride = f8_blocks(I);
    a.y = g.eo;
    a.ys = nullptr;
    a.y_stride = H;
    a.ys_stride = 0;
    a.rows = H;
    a.cols = I;
    a.act = BREAD_ACT_NONE;
    a.y_type = BREAD_QTYPE_F32;
    a.x_rows = nullptr;
    a.n_x = 0;
    rc = bread_launch_fp8_matmul(a, st);
    if (rc) return rc;
    hipLaunchKernelGGL(k_f8_combine, dim3((unsigned)T, (unsigned)((H / 4 + 255) / 256)), dim3(256), 0, st, g.eo, g.pos_of,
                       w, residual, hidden, hidden_type, H, K);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}
