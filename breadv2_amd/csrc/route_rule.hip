// route_rule.hip — routing by a rule: softmax or sigmoid scores, a bias that
// only steers the choice, groups of experts, top-k and weights (renormalised,
// scaled).  route_layer's own rule (one_layer.cu:983-985) is the special case
// softmax, no bias, one group, renormalised.
//
// With l the logits of a token:
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e)),  c_e = s_e + bias_e,
//   a group's score = the sum of its group_top (1 or 2) largest c,
//   the top_groups best groups stay, the top_k largest c among them are chosen
//   (ties everywhere to the lower index), w_k = s of the k-th (/ their sum) * scale.
// Scores and choices are held in 64 bits: which of two experts comes first
// decides whole expert products, and sigmoid scores of large logits are closer
// to each other than fp32 can tell.
#include "bread_internal.h"
#include "route_dev.h"

namespace {

constexpr int RR_THREADS = 256;

// Order-preserving key of a choice: 0 taken or not allowed, 1 NaN, -inf and up above.
__device__ __forceinline__ uint64_t choice_key(double c)
{
    // (by words, without branches)
    const uint64_t u = __builtin_bit_cast(uint64_t, c);
    const uint32_t hi = (uint32_t)(u >> 32), all = (uint32_t)((int32_t)hi >> 31);
    const bool nan = c != c;
    const uint32_t kh = nan ? 0u : hi ^ (all | 0x80000000u), kl = nan ? 1u : (uint32_t)u ^ all;
    return ((uint64_t)kh << 32) | kl;
}

// The larger of two, a number against NaN
__device__ __forceinline__ double max_num(double a, double b)
{
    double d;
    asm("v_max_f64 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}

__device__ __forceinline__ double min_num(double a, double b)
{
    double d;
    asm("v_min_f64 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}

// Reductions over the L lanes (32 or 64, aligned) of a token; the result is in each of them.
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v)
{
    v = umax32(v, dpp_u32<0xB1>(v));
    v = umax32(v, dpp_u32<0x4E>(v));
    v = umax32(v, dpp_u32<0x141>(v));
    v = umax32(v, dpp_u32<0x140>(v));
    lane_pair p = swap16(v);
    v = umax32(p.a, p.b);
    if (L == 32) return v;
    p = swap32(v);
    return umax32(p.a, p.b);
}

template <int L>
__device__ __forceinline__ float group_max(float v)
{
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    v = fmaxf(v, dpp_f<0x140>(v));
    lane_pair p = swap16(__builtin_bit_cast(uint32_t, v));
    v = fmaxf(__builtin_bit_cast(float, p.a), __builtin_bit_cast(float, p.b));
    if (L == 32) return v;
    p = swap32(__builtin_bit_cast(uint32_t, v));
    return fmaxf(__builtin_bit_cast(float, p.a), __builtin_bit_cast(float, p.b));
}

struct double_pair {
    double a, b;
};

template <int W>
__device__ __forceinline__ double_pair swap_f64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const lane_pair lo = W == 16 ? swap16((uint32_t)u) : swap32((uint32_t)u);
    const lane_pair hi = W == 16 ? swap16((uint32_t)(u >> 32)) : swap32((uint32_t)(u >> 32));
    return {__builtin_bit_cast(double, ((uint64_t)hi.a << 32) | lo.a), __builtin_bit_cast(double, ((uint64_t)hi.b << 32) | lo.b)};
}

template <int L>
__device__ __forceinline__ double group_sum(double v)
{
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    v += dpp_f64<0x141>(v);
    v += dpp_f64<0x140>(v);
    double_pair p = swap_f64<16>(v);
    v = p.a + p.b;
    if (L == 32) return v;
    p = swap_f64<32>(v);
    return p.a + p.b;
}

// The rule as the kernel takes it.
struct Rule {
    const float *bias;
    int sigmoid, n_groups, per, top_groups, two, renorm;
    uint32_t inv_per;  // ceil(2^20 / per): e / per = (e * inv_per) >> 20 for e < 1024
    int lanes;         // lanes of a group where that is a power of two and a lane's experts are all of one, or 0
    float scale;
};

// 2^y for y <= 1023, to 8e-14 of itself (2^n p(y - n), n the nearest whole number, p the polynomial of degree 9
// that is 1 at 0 and has the least largest relative error on [-1/2, 1/2], by Remez exchange); 0 far below and
// for -inf.  Smooth to far less than the distance of two fp32 logits' scores.
__device__ __forceinline__ double exp2_f64(double y)
{
    const double n = __builtin_rint(fmax(y, -1100.0)), f = fmax(y, -1100.0) - n;
    double p = 0x1.89c489e9e3ae4p-24;
    p = fma(p, f, 0x1.63d0ec28f10f2p-20);
    p = fma(p, f, 0x1.fffd75179b1a0p-17);
    p = fma(p, f, 0x1.4308acc67a164p-13);
    p = fma(p, f, 0x1.5d87ebe42d79dp-10);
    p = fma(p, f, 0x1.3b2ab717fb0b6p-7);
    p = fma(p, f, 0x1.c6b08d7a95072p-5);
    p = fma(p, f, 0x1.ebfbdff823df0p-3);
    p = fma(p, f, 0x1.62e42fefa08dcp-1);
    return __builtin_amdgcn_ldexp(fma(p, f, 1.0), (int)n);
}

// 1 / x for x in [1, 2^1024): two Newton steps on the hardware's estimate
__device__ __forceinline__ double inverse(double x)
{
    double r = __builtin_amdgcn_rcp(x);
    r = fma(r, fma(-x, r, 1.0), r);
    return fma(r, fma(-x, r, 1.0), r);
}

constexpr double LOG2E = 1.4426950408889634;

// A logit's score (NaN as -inf), softmax's before its division.  Selects, no branches.
__device__ __forceinline__ double sigmoid_score(float l)
{
    // below -700 the score is under 1e-304, and 2^y of that is still a number
    const float x = fmaxf(l, -700.f);  // (NaN gives -700)
    const double s = inverse(1.0 + exp2_f64(-(double)x * LOG2E));
    return l >= -700.f ? s : 0.0;
}
__device__ __forceinline__ double softmax_score(float l, float m)
{
    const double e = exp2_f64(((double)l - (double)m) * LOG2E), s = l == m ? 1.0 : e;  // (an infinite largest one too)
    return l > -__builtin_inff() ? s : 0.0;
}

// LDS of one wave: what its lanes wrote is there for all of them
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The two largest of two pairs of (largest, second)
__device__ __forceinline__ void merge2(double &a1, double &a2, double b1, double b2)
{
    a2 = max_num(min_num(a1, b1), max_num(a2, b2));
    a1 = max_num(a1, b1);
}

// L lanes a token, MAXV consecutive experts a lane.  A lane ranks its experts (all pairs compared once) and lays
// their keys out in LDS in that order; of the lanes' best ones, the largest is then taken top_k times, by its high
// word on DPP (its low word too where two are equal), and its lane goes on to its next.  Groups whose experts fill
// a power of two of lanes are scored on DPP, others from LDS.
// Bound by the instructions.  MI355X, 256 experts, sigmoid, four of eight groups, top 8: 16384 tokens 15.4 us (the
// logits alone are 3.3 us at a copy's rate); a wave a token, with the library's exp and 64-bit maxima, took 31.
// 100 tokens 5.6 us against 9.6; one token of softmax 4.0 us.  Two tokens a wave up to 256 experts because the
// top_k rounds cost a wave the same for one.
template <int MAXV, int L>
__global__ __launch_bounds__(RR_THREADS) void k_route_rule(const float *__restrict__ logits, int64_t stride, int E,
                                                          int K, int T, const Rule rule, int32_t *__restrict__ idx,
                                                          float *__restrict__ w)
{
    constexpr int TOK = RR_THREADS / L;
    __shared__ uint64_t s_key[TOK][MAXV * L];  // choices by expert, groups' scores, keys by rank and lane
    __shared__ uint8_t s_id[TOK][MAXV * L];
    __shared__ uint16_t s_sel[TOK][32];
    const int tk = (int)threadIdx.x / L, tl = (int)threadIdx.x % L;
    const int t = min((int)blockIdx.x * TOK + tk, T - 1);  // past the end the last token again, not stored
    const float *lt = logits + (size_t)t * stride;
    const int e0 = tl * MAXV;
    float l[MAXV], bias[MAXV], m = -__builtin_inff();
    if (e0 + MAXV <= E) {
        __builtin_memcpy(l, lt + e0, sizeof(l));
        if (rule.bias) __builtin_memcpy(bias, rule.bias + e0, sizeof(bias));
    } else {
#pragma unroll
        for (int v = 0; v < MAXV; v++) {
            l[v] = e0 + v < E ? lt[e0 + v] : -__builtin_inff();
            bias[v] = rule.bias && e0 + v < E ? rule.bias[e0 + v] : 0.f;
        }
    }
    const bool sig = rule.sigmoid != 0;
    double c[MAXV], inv = 1.0;
    if (sig) {
#pragma unroll
        for (int v = 0; v < MAXV; v++) c[v] = sigmoid_score(l[v]);
    } else {
        double s = 0.0;
#pragma unroll
        for (int v = 0; v < MAXV; v++) m = fmaxf(m, l[v]);  // (NaN is passed over)
        m = group_max<L>(m);
#pragma unroll
        for (int v = 0; v < MAXV; v++) {
            c[v] = softmax_score(l[v], m);
            s += c[v];
        }
        s = group_sum<L>(s);
        inv = s > 0.0 ? 1.0 / s : 0.0;  // nothing but -inf: scores of zero
#pragma unroll
        for (int v = 0; v < MAXV; v++) c[v] *= inv;
    }
    if (rule.bias) {
#pragma unroll
        for (int v = 0; v < MAXV; v++) c[v] += (double)bias[v];
    }
    uint64_t key[MAXV];
#pragma unroll
    for (int v = 0; v < MAXV; v++) key[v] = choice_key(c[v]);
    if (e0 + MAXV > E) {
#pragma unroll
        for (int v = 0; v < MAXV; v++) key[v] = e0 + v < E ? key[v] : 0u;
    }
    if (rule.top_groups < rule.n_groups) {
        // a group's score: NaN choices count as -inf
        const int G = rule.n_groups;
        if (rule.lanes) {
            double a1 = -__builtin_inf(), a2 = -__builtin_inf();
#pragma unroll
            for (int v = 0; v < MAXV; v++) {
                const double x = max_num(c[v], -__builtin_inf());  // (a lane's experts are all there or none)
                a2 = max_num(a2, min_num(a1, x));
                a1 = max_num(a1, x);
            }
            if (rule.lanes >= 2) merge2(a1, a2, dpp_f64<0xB1>(a1), dpp_f64<0xB1>(a2));
            if (rule.lanes >= 4) merge2(a1, a2, dpp_f64<0x4E>(a1), dpp_f64<0x4E>(a2));
            if (rule.lanes >= 8) merge2(a1, a2, dpp_f64<0x141>(a1), dpp_f64<0x141>(a2));
            if (rule.lanes >= 16) merge2(a1, a2, dpp_f64<0x140>(a1), dpp_f64<0x140>(a2));
            if (rule.lanes >= 32) {
                const double_pair p = swap_f64<16>(a1), q = swap_f64<16>(a2);
                a1 = p.a;
                a2 = q.a;
                merge2(a1, a2, p.b, q.b);
            }
            const int g = tl / rule.lanes;
            const double score = rule.two && rule.per > 1 ? a1 + a2 : a1;
            if (tl % rule.lanes == 0 && g < G) s_key[tk][g] = __builtin_bit_cast(uint64_t, score);
            wave_sync();
            int better = 0;
            for (int j = 0; j < G; j++) {
                const double y = __builtin_bit_cast(double, s_key[tk][j]);
                better += y > score || (y == score && j < g);
            }
            if (better >= rule.top_groups) {
#pragma unroll
                for (int v = 0; v < MAXV; v++) key[v] = 0u;
            }
        } else {
#pragma unroll
            for (int v = 0; v < MAXV; v++) s_key[tk][e0 + v] = __builtin_bit_cast(uint64_t, c[v]);
            wave_sync();
            double score[MAXV];
#pragma unroll
            for (int v = 0; v < MAXV; v++) {
                const int g = tl + v * L;
                double a1 = -__builtin_inf(), a2 = -__builtin_inf();
#pragma unroll 1
                for (int i = 0; i < rule.per && g < G; i++) {
                    const double x = __builtin_bit_cast(double, s_key[tk][g * rule.per + i]);
                    if (x == x) {
                        a2 = fmax(a2, fmin(a1, x));
                        a1 = fmax(a1, x);
                    }
                }
                score[v] = rule.two && rule.per > 1 ? a1 + a2 : a1;
            }
            wave_sync();
#pragma unroll
            for (int v = 0; v < MAXV; v++) s_key[tk][tl + v * L] = __builtin_bit_cast(uint64_t, score[v]);
            wave_sync();
#pragma unroll
            for (int v = 0; v < MAXV; v++) {
                const int g = tl + v * L;
                int better = 0;
#pragma unroll 1
                for (int j = 0; j < G && g < G; j++) {
                    const double y = __builtin_bit_cast(double, s_key[tk][j]);
                    better += y > score[v] || (y == score[v] && j < g);
                }
                s_id[tk][g] = better < rule.top_groups;
            }
            wave_sync();
#pragma unroll
            for (int v = 0; v < MAXV; v++)
                if (e0 + v < E && !s_id[tk][((uint32_t)(e0 + v) * rule.inv_per) >> 20]) key[v] = 0u;
        }
        wave_sync();
    }
    // ranks in the lane: larger keys first, the lower expert among equals
    int rank[MAXV];
#pragma unroll
    for (int v = 0; v < MAXV; v++) rank[v] = v;
#pragma unroll
    for (int v = 0; v < MAXV; v++)
#pragma unroll
        for (int u = v + 1; u < MAXV; u++) {
            const int a = key[u] > key[v];
            rank[v] += a;
            rank[u] -= a;
        }
#pragma unroll
    for (int v = 0; v < MAXV; v++) {
        s_key[tk][rank[v] * L + tl] = key[v];
        s_id[tk][rank[v] * L + tl] = (uint8_t)v;
    }
    wave_sync();
    uint64_t head = s_key[tk][tl];
    int id = s_id[tk][tl], p = 0;
    for (int k = 0; k < K; k++) {
        const uint32_t hi = (uint32_t)(head >> 32), M = group_max<L>(hi);
        bool win = hi == M;
        uint64_t b = __builtin_amdgcn_ballot_w64(win);
        if (__builtin_popcountll(b) != WAVE / L) {
            // equal high words: by the low ones, then the lowest lane
            const uint32_t lo = win ? (uint32_t)head : 0u, N = group_max<L>(lo);  // (by all lanes)
            win = win && lo == N;
            b = __builtin_amdgcn_ballot_w64(win);
            if (L == 32) b = lane_id() < 32 ? b & 0xFFFFFFFFull : b & ~0xFFFFFFFFull;
            win = lane_id() == (int)__builtin_ctzll(b);
        }
        if (win) {
            s_sel[tk][k] = (uint16_t)(e0 + id);
            p++;
            head = 0u;
            if (p < MAXV) {
                head = s_key[tk][p * L + tl];
                id = s_id[tk][p * L + tl];
            }
        }
    }
    wave_sync();
    // weights from the scores of the chosen, the same arithmetic again
    const int e = tl < K ? (int)s_sel[tk][tl] : 0;
    const float le = lt[e];
    double s = tl < K ? (sig ? sigmoid_score(le) : softmax_score(le, m) * inv) : 0.0;
    if (rule.renorm) {
        const double sum = group_sum<L>(s);
        s = sum > 0.0 ? s / sum : 0.0;
    }
    if (tl < K && (int)blockIdx.x * TOK + tk < T) {
        idx[(size_t)t * K + tl] = e;
        w[(size_t)t * K + tl] = (float)(s * (double)rule.scale);
    }
}

template <int MAXV, int L>
void launch(const float *logits, int64_t stride, int E, int K, int T, Rule a, int32_t *idx, float *w, hipStream_t st)
{
    const int lanes = a.per / MAXV;
    a.lanes = a.per % MAXV == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    hipLaunchKernelGGL((k_route_rule<MAXV, L>), dim3((T + RR_THREADS / L - 1) / (RR_THREADS / L)), dim3(RR_THREADS), 0,
                       st, logits, stride, E, K, T, a, idx, w);
}

}  // namespace

int bread_validate_rule(const bread_route_rule_t *r, int E, int K)
{
    BREAD_REQUIRE(r, BREAD_ERR_ARG, "NULL rule");
    BREAD_REQUIRE(E > 0 && E <= 1024 && K > 0 && K <= 32 && K <= E, BREAD_ERR_SHAPE,
                  "n_experts must be 1 to 1024, top_k 1 to 32 and not above n_experts");
    BREAD_REQUIRE(r->score == BREAD_SCORE_SOFTMAX || r->score == BREAD_SCORE_SIGMOID, BREAD_ERR_ARG, "unknown score");
    BREAD_REQUIRE(r->n_groups > 0 && E % r->n_groups == 0, BREAD_ERR_SHAPE, "n_groups must divide n_experts");
    BREAD_REQUIRE(r->top_groups > 0 && r->top_groups <= r->n_groups, BREAD_ERR_ARG,
                  "top_groups must be 1 to n_groups");
    BREAD_REQUIRE((int64_t)r->top_groups * (E / r->n_groups) >= K, BREAD_ERR_SHAPE,
                  "the kept groups hold fewer than top_k experts");
    BREAD_REQUIRE(r->group_top == 1 || r->group_top == 2, BREAD_ERR_ARG, "group_top must be 1 or 2");
    BREAD_REQUIRE(((uintptr_t)r->bias & 3) == 0, BREAD_ERR_ALIGN, "bias must be 4-byte aligned");
    return BREAD_OK;
}

int bread_launch_route_rule(const bread_route_rule_t *r, const float *logits, int64_t stride, int E, int K, int T,
                            int32_t *idx, float *w, hipStream_t st)
{
    Rule a;
    a.bias = r->bias;
    a.sigmoid = r->score == BREAD_SCORE_SIGMOID;
    a.n_groups = r->n_groups;
    a.per = E / r->n_groups;
    a.top_groups = r->top_groups;
    a.two = r->group_top == 2;
    a.renorm = r->renorm != 0;
    a.inv_per = (uint32_t)(((1u << 20) + a.per - 1) / a.per);
    a.scale = r->scale;
    bread_clear_stale_error();
    if (E <= 64) launch<2, 32>(logits, stride, E, K, T, a, idx, w, st);
    else if (E <= 128) launch<4, 32>(logits, stride, E, K, T, a, idx, w, st);
    else if (E <= 256) launch<8, 32>(logits, stride, E, K, T, a, idx, w, st);
    else launch<16, 64>(logits, stride, E, K, T, a, idx, w, st);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

int bread_launch_route_by_rule(bread_moe_ctx_t *c, const bread_moe_layer_t *L, const bread_route_rule_t *r,
                               const float *x, int T, int32_t *idx, float *w, float *gsh, hipStream_t st)
{
    const bread_moe_shape_t &s = c->shape;
    bread_clear_stale_error();
    const int rc = bread_launch_route_logits(L->router, L->shexp_gate, x, c->logits, gsh, s.hidden, s.n_experts, T,
                                             true, st);
    if (rc) return rc;
    return bread_launch_route_rule(r, c->logits, s.n_experts, s.n_experts, s.top_k, T, idx, w, st);
}

extern "C" int bread_route_select(const bread_route_rule_t *rule, const float *logits, int64_t stride, int E, int K,
                                  int T, int32_t *idx, float *w, bread_stream_t stream)
{
    const int rc = bread_validate_rule(rule, E, K);
    if (rc) return rc;
    BREAD_REQUIRE(T >= 0, BREAD_ERR_ARG, "n_tokens < 0");
    // (four tokens a workgroup of 256 for many experts: 2^32 threads are one launch's limit)
    BREAD_REQUIRE(T <= (1 << 26) - 4, BREAD_ERR_SHAPE, "n_tokens above 2^26 - 4");
    BREAD_REQUIRE(stride == 0 || stride >= E, BREAD_ERR_SHAPE, "stride smaller than n_experts");
    if (T == 0) return BREAD_OK;
    BREAD_REQUIRE(logits && idx && w, BREAD_ERR_ARG, "NULL input or output");
    BREAD_REQUIRE((((uintptr_t)logits | (uintptr_t)idx | (uintptr_t)w) & 3) == 0, BREAD_ERR_ALIGN,
                  "logits, idx and w must be 4-byte aligned");
    return bread_launch_route_rule(rule, logits, stride ? stride : E, E, K, T, idx, w, to_hip(stream));
}
