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

constexpr int RR_WAVES = 4;

// Order-preserving key of a choice: 0 taken or not allowed, 1 NaN, -inf and up above.
__device__ __forceinline__ uint64_t choice_key(double c)
{
    if (c != c) return 1u;
    const uint64_t u = __builtin_bit_cast(uint64_t, c);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

__device__ __forceinline__ double wave_sum_f64(double v)
{
    for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The rule as the kernel takes it.
struct Rule {
    const float *bias;
    int sigmoid, n_groups, per, top_groups, two, renorm;
    uint32_t inv_per;  // ceil(2^20 / per): e / per = (e * inv_per) >> 20 for e < 1024
    float scale;
};

// One wave a token; expert e = lane + 64 v in slot v of its lane.
template <int MAXV>
__global__ __launch_bounds__(RR_WAVES *WAVE) void k_route_rule(const float *__restrict__ logits, int64_t stride, int E,
                                                              int K, int T, const Rule rule, int32_t *__restrict__ idx,
                                                              float *__restrict__ w)
{
    __shared__ double s_c[RR_WAVES][WAVE * MAXV];
    __shared__ double s_g[RR_WAVES][WAVE * MAXV];
    __shared__ uint8_t s_keep[RR_WAVES][WAVE * MAXV];
    const int wv = wave_id(), lane = lane_id();
    const int t = (int)blockIdx.x * RR_WAVES + wv;
    if (t >= T) return;
    const float *lt = logits + (size_t)t * stride;
    double s[MAXV], c[MAXV];
    float l[MAXV], m = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < MAXV; v++) {
        const int e = lane + WAVE * v;
        l[v] = e < E ? lt[e] : -__builtin_inff();
        if (l[v] != l[v]) l[v] = -__builtin_inff();
        m = fmaxf(m, l[v]);
    }
    if (rule.sigmoid) {
#pragma unroll
        for (int v = 0; v < MAXV; v++) s[v] = 1.0 / (1.0 + exp(-(double)l[v]));
    } else {
        m = wave_max(m);
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < MAXV; v++) {
            // equal to the largest: 1, an infinite one too; nothing but -inf: 0
            s[v] = m == -__builtin_inff() ? 0.0 : l[v] == m ? 1.0 : exp((double)l[v] - (double)m);
            sum += s[v];
        }
        sum = wave_sum_f64(sum);
#pragma unroll
        for (int v = 0; v < MAXV; v++) s[v] = sum > 0.0 ? s[v] / sum : 0.0;
    }
    uint64_t key[MAXV];
#pragma unroll
    for (int v = 0; v < MAXV; v++) {
        const int e = lane + WAVE * v;
        c[v] = s[v] + (rule.bias && e < E ? (double)rule.bias[e] : 0.0);
        key[v] = e < E ? choice_key(c[v]) : 0u;
    }
    if (rule.top_groups < rule.n_groups) {
#pragma unroll
        for (int v = 0; v < MAXV; v++) s_c[wv][lane + WAVE * v] = c[v];
        __builtin_amdgcn_wave_barrier();
        // a group's score: NaN choices count as -inf
        for (int g = lane; g < rule.n_groups; g += WAVE) {
            double a = -__builtin_inf(), b = -__builtin_inf();
            for (int i = 0; i < rule.per; i++) {
                const double x = s_c[wv][g * rule.per + i];
                if (x > a) {
                    b = a;
                    a = x;
                } else if (x > b) {
                    b = x;
                }
            }
            s_g[wv][g] = rule.two && rule.per > 1 ? a + b : a;
        }
        __builtin_amdgcn_wave_barrier();
        for (int g = lane; g < rule.n_groups; g += WAVE) {
            const double x = s_g[wv][g];
            int better = 0;
            for (int j = 0; j < rule.n_groups; j++) {
                const double y = s_g[wv][j];
                better += y > x || (y == x && j < g);
            }
            s_keep[wv][g] = better < rule.top_groups;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int v = 0; v < MAXV; v++) {
            const int e = lane + WAVE * v;
            if (e < E && !s_keep[wv][((uint32_t)e * rule.inv_per) >> 20]) key[v] = 0u;
        }
    }
    int my_idx = 0;
    double my_s = 0.0, sum = 0.0;
    for (int k = 0; k < K; k++) {
        uint64_t best = 0;
#pragma unroll
        for (int v = 0; v < MAXV; v++) best = u64_max(best, key[v]);
        best = wave_max_u64(best);
        int win = 0;
#pragma unroll
        for (int v = MAXV - 1; v >= 0; v--) {
            const uint64_t b = __builtin_amdgcn_ballot_w64(key[v] == best);
            if (b) win = WAVE * v + (int)__builtin_ctzll(b);
        }
        double sv = 0.0;
#pragma unroll
        for (int v = 0; v < MAXV; v++)
            if (win >> 6 == v) {
                sv = readlane_f64(s[v], win & 63);
                if (lane == (win & 63)) key[v] = 0u;
            }
        sum += sv;
        if (lane == k) {
            my_idx = win;
            my_s = sv;
        }
    }
    if (lane < K) {
        double x = my_s;
        if (rule.renorm) x = sum > 0.0 ? x / sum : 0.0;
        idx[(size_t)t * K + lane] = my_idx;
        w[(size_t)t * K + lane] = (float)(x * (double)rule.scale);
    }
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
    const int mv = (E + WAVE - 1) / WAVE;
    const dim3 grid((T + RR_WAVES - 1) / RR_WAVES), block(RR_WAVES * WAVE);
    bread_clear_stale_error();
    if (mv <= 4) hipLaunchKernelGGL(k_route_rule<4>, grid, block, 0, st, logits, stride, E, K, T, a, idx, w);
    else hipLaunchKernelGGL(k_route_rule<16>, grid, block, 0, st, logits, stride, E, K, T, a, idx, w);
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
    BREAD_REQUIRE(stride == 0 || stride >= E, BREAD_ERR_SHAPE, "stride smaller than n_experts");
    if (T == 0) return BREAD_OK;
    BREAD_REQUIRE(logits && idx && w, BREAD_ERR_ARG, "NULL input or output");
    BREAD_REQUIRE((((uintptr_t)logits | (uintptr_t)idx | (uintptr_t)w) & 3) == 0, BREAD_ERR_ALIGN,
                  "logits, idx and w must be 4-byte aligned");
    return bread_launch_route_rule(rule, logits, stride ? stride : E, E, K, T, idx, w, to_hip(stream));
}
