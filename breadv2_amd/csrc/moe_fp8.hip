// moe_fp8.hip — bread_moe_expert_block_fp8: the routed experts of a layer with
// e4m3 weights and the caller's routing,
//   hidden[t] = residual[t] + sum_k w[t][k] down_e(q(silu(gate_e x) * (up_e x))),  e = idx[t][k].
// Pairs (token, rank) are sorted by expert; gate and up are one grouped product
// that ends in codes by pair, down another (fp8_matmul.hip), and the pairs of a
// token are added in rank order.
#include "fp8.h"

namespace {

// Pairs by expert: offsets [E + 1], token[i] of sorted row i, place[p] of pair p (-1: no expert).
__global__ __launch_bounds__(1024) void k_f8_bucket(const int32_t *__restrict__ idx, int P, int K, int E,
                                                    int32_t *__restrict__ offsets, int32_t *__restrict__ token,
                                                    int32_t *__restrict__ place, uint32_t *__restrict__ err)
{
    __shared__ int cnt[1024], base[1024], sums[16];
    const int tid = (int)threadIdx.x;
    cnt[tid] = 0;
    __syncthreads();
    bool bad = false;
    for (int p = tid; p < P; p += 1024) {
        const int e = idx[p];
        if ((unsigned)e < (unsigned)E) atomicAdd(&cnt[e], 1);
        else bad = true;
    }
    if (bad) __hip_atomic_fetch_or(err, BREAD_DEV_ERR_INDEX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const int c = tid < E ? cnt[tid] : 0, incl = wave_scan_incl(c);
    if (lane_id() == WAVE - 1) sums[tid / WAVE] = incl;
    __syncthreads();
    int before = incl - c;
    for (int i = 0; i < tid / WAVE; i++) before += sums[i];
    base[tid] = before;
    if (tid < E) offsets[tid] = before;
    if (tid == E - 1) offsets[E] = before + c;
    __syncthreads();
    for (int p = tid; p < P; p += 1024) {
        const int e = idx[p];
        int at = -1;
        if ((unsigned)e < (unsigned)E) {
            at = atomicAdd(&base[e], 1);
            token[at] = p / K;
        }
        place[p] = at;
    }
}

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
    hipLaunchKernelGGL(k_f8_bucket, dim3(1), dim3(1024), 0, st, idx, P, K, s.n_experts, g.offsets, g.pair_tok, g.pos_of,
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
