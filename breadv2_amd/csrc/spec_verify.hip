// spec_verify.hip — verification of drafted tokens by sampling: the acceptance
// of main_speculative.cu:477-497 (drafts equal to the target's greedy token)
// for requests that sample, with the random numbers given.
//
// A request's rows hold the target's logits after its last confirmed token and
// after each draft.  With p = softmax(logits / temperature) of a row, q the
// draft model's probabilities there (one-hot for drafts that were looked up)
// and u uniform in [0, 1), draft d stands when u q(d) < p(d).  The token after
// the last one that stands follows max(p - q, 0) at the first row whose draft
// falls, p itself at the last row; so the accepted tokens and it are distributed as
// the target's own.  It is drawn as the first token whose cumulative weight
// exceeds u' times the whole.
//
// Probabilities and sums are held in 64 bits: a vocabulary has 10^5 borders
// between tokens, and a cumulative sum that is off by 10^-7 moves the drawn
// token in some of a hundred draws.
#include "bread_internal.h"
#include "route_dev.h"

namespace {

constexpr int SV_THREADS = 256;
constexpr int SV_WAVES = SV_THREADS / WAVE;
// Logits a thread (PER): 32 once there is work for the whole GPU, 8 below that, where the time is one
// workgroup's chain of loads and exponentials.  A workgroup's chunk of a row is SV_THREADS times as many.
constexpr int SV_MANY = 32, SV_FEW = 8;
constexpr int SV_MAX_CHUNKS = 2048;  // of a row: 2^24 logits in chunks of 8192

// One chunk of a row: the largest logit and the sum of exp((l - max) / T).
struct SvPart {
    double sum;
    float max;
    int arg;  // lowest index of the largest logit
};

struct SvArgs {
    const void *logits;
    int64_t stride;  // elements from one row to the next
    int V, R, B, nchunk;
    const int32_t *tokens, *off;
    const float *u, *q, *temp;
    int64_t qstride;
    int32_t eos;
    SvPart *part;      // [R][nchunk]
    double *tot;       // [B][nchunk]
    uint32_t *count;   // [B], zero between calls
    uint32_t *err;
    int32_t *accepted, *next;
    float *logp;       // may be NULL
};

// A logit as a number: NaN counts as -inf
__device__ __forceinline__ float num(float v)
{
    return v != v ? -__builtin_inff() : v;
}

// 2^y for y <= 0, to 8e-14 of itself: 2^n p(y - n) with n the nearest whole number and p the polynomial of
// degree 9 that is 1 at 0 and nearest to 2^f on [-1/2, 1/2] in relative error (by Remez exchange).  1 for 0, and
// 0 below -1075, for -inf and for NaN (-inf times 1 / an infinite temperature).  18 instructions, where
// the library's exp takes twice as many.
__device__ __forceinline__ double exp2_neg(double y)
{
    y = fmax(y, -1100.0);
    const double n = __builtin_rint(y), f = y - n;
    double p = 0x1.89c489e9e3ae4p-24;
    p = fma(p, f, 0x1.63d0ec28f10f2p-20);
    p = fma(p, f, 0x1.fffd75179b1a0p-17);
    p = fma(p, f, 0x1.4308acc67a164p-13);
    p = fma(p, f, 0x1.5d87ebe42d79dp-10);
    p = fma(p, f, 0x1.3b2ab717fb0b6p-7);
    p = fma(p, f, 0x1.c6b08d7a95072p-5);
    p = fma(p, f, 0x1.ebfbdff823df0p-3);
    p = fma(p, f, 0x1.62e42fefa08dcp-1);
    p = fma(p, f, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}

constexpr double LOG2E = 1.4426950408889634;

// exp((l - m) / T) for l <= m, c2 = log2(e) / T: 1 where they are equal, infinite ones too; 0 for l = -inf
__device__ __forceinline__ double weight(float l, float m, double c2)
{
    if (__builtin_isinf(m)) return l == m && m > 0.f ? 1.0 : 0.0;
    return exp2_neg(((double)l - (double)m) * c2);
}

// Eight values from element i on, of which those at V and beyond read as `none`
template <typename LT>
__device__ __forceinline__ void load8(const LT *row, int i, int V, float none, float (&v)[8])
{
    LT h[8];
    if (i + 8 <= V) {
        __builtin_memcpy(h, row + i, sizeof(h));  // aligned to an element
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) h[k] = i + k < V ? row[i + k] : LT(0);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) {
        if constexpr (sizeof(LT) == 2) v[k] = num(h2f(h[k]));
        else v[k] = num(h[k]);
        if (i + k >= V) v[k] = none;
    }
}

__device__ __forceinline__ double sum_f64(double v)
{
    for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The request of a row: how many requests after the first start at or before it
__device__ __forceinline__ int request_of(const int32_t *off, int B, int row)
{
    int n = 0;
    for (int i = 1 + lane_id(); i < B + lane_id() + 1; i += WAVE) {
        const bool in = i < B && off[i] <= row;
        n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
    }
    return n;
}

// log2(e) / temperature; a greedy request's log-probabilities are those of temperature 1
__device__ __forceinline__ double scale2(const float *temp, int b)
{
    const float t = temp ? temp[b] : 1.0f;
    return t > 0.f ? LOG2E / (double)t : LOG2E;
}

__device__ __forceinline__ bool greedy(const float *temp, int b)
{
    return temp && !(temp[b] > 0.f);
}

// Workgroup b: chunk b % nchunk of row b / nchunk.
template <typename LT, int PER>
__global__ __launch_bounds__(SV_THREADS) void k_sv_stats(const SvArgs a)
{
    __shared__ float s_m[SV_WAVES];
    __shared__ double s_s[SV_WAVES];
    __shared__ int s_i[SV_WAVES];
    const int row = (int)blockIdx.x / a.nchunk, ch = (int)blockIdx.x % a.nchunk, tid = (int)threadIdx.x, wv = wave_id();
    const LT *z = static_cast<const LT *>(a.logits) + (size_t)row * a.stride;
    float v[PER / 8][8], m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < PER / 8; j++)
        load8<LT>(z, ch * (SV_THREADS * PER) + (j * SV_THREADS + tid) * 8, a.V, -__builtin_inff(), v[j]);
    const int b = request_of(a.off, a.B, row);
    const double c2 = scale2(a.temp, b);
#pragma unroll
    for (int j = 0; j < PER / 8; j++)
#pragma unroll
        for (int k = 0; k < 8; k++) m = fmaxf(m, v[j][k]);
    m = wave_max(m);
    if (lane_id() == 0) s_m[wv] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SV_WAVES; k++) m = fmaxf(m, s_m[k]);
    double s = 0.0;
    int arg = 0x7FFFFFFF;
    if (__builtin_isinf(m)) {
#pragma unroll
        for (int j = 0; j < PER / 8; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) s += weight(v[j][k], m, c2);
    } else {
        const double md = (double)m;
#pragma unroll
        for (int j = 0; j < PER / 8; j++)
#pragma unroll
            for (int k = 0; k < 8; k++) s += exp2_neg(((double)v[j][k] - md) * c2);
    }
#pragma unroll
    for (int j = PER / 8 - 1; j >= 0; j--)
#pragma unroll
        for (int k = 7; k >= 0; k--) {
            const int i = ch * (SV_THREADS * PER) + (j * SV_THREADS + tid) * 8 + k;
            if (v[j][k] == m && i < a.V) arg = i;
        }
    s = sum_f64(s);
    for (int o = WAVE / 2; o > 0; o >>= 1) arg = min(arg, __shfl_xor(arg, o));
    if (lane_id() == 0) {
        s_s[wv] = s;
        s_i[wv] = arg;
    }
    __syncthreads();
    if (tid == 0) {
        for (int k = 1; k < SV_WAVES; k++) {
            s += s_s[k];
            arg = min(arg, s_i[k]);
        }
        a.part[(size_t)row * a.nchunk + ch] = SvPart{s, m, arg};
    }
}

// A row's statistics from its chunks, by one wave
struct SvRow {
    double sum;
    float max;
    int arg;
};

__device__ __forceinline__ SvRow row_stats(const SvArgs &a, int row, double c2)
{
    const SvPart *p = a.part + (size_t)row * a.nchunk;
    SvRow r{0.0, -__builtin_inff(), 0x7FFFFFFF};
    for (int c = lane_id(); c < a.nchunk; c += WAVE) r.max = fmaxf(r.max, p[c].max);
    r.max = wave_max(r.max);
    for (int c = lane_id(); c < a.nchunk; c += WAVE) {
        r.sum += p[c].sum * weight(p[c].max, r.max, c2);
        if (p[c].max == r.max) r.arg = min(r.arg, p[c].arg);
    }
    r.sum = sum_f64(r.sum);
    for (int o = WAVE / 2; o > 0; o >>= 1) r.arg = min(r.arg, __shfl_xor(r.arg, o));
    return r;
}

__device__ __forceinline__ float log_p(float l, const SvRow &r, double c2)
{
    if (!(r.sum > 0.0) || l == -__builtin_inff() || (r.max == __builtin_inff() && l != r.max)) return -__builtin_inff();
    return (float)((l == r.max ? 0.0 : ((double)l - (double)r.max) * (c2 / LOG2E)) - log(r.sum));
}

// What is left of token i's weight e (its probability times the row's sum) when
// the draft falls: its own (no draft there), without the draft's q, or none for
// a looked-up draft itself
struct SvLeft {
    const float *q;  // the draft's row of probabilities, or NULL
    int one;         // the looked-up draft, or -1
    double sum;
    __device__ __forceinline__ double operator()(double e, int i, float x) const
    {
        if (q) {
            const double d = e - (x > 0.f ? (double)x * sum : 0.0);
            return d > 0.0 ? d : 0.0;
        }
        return i == one ? 0.0 : e;
    }
    // What eight tokens from i on leave (those at V and beyond: nothing)
    template <typename LT>
    __device__ __forceinline__ void eight(const LT *z, int i, int V, float m, double c2, double (&d)[8]) const
    {
        float l[8], x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        load8<LT>(z, i, V, -__builtin_inff(), l);
        if (q) load8<float>(q, i, V, 0.f, x);
#pragma unroll
        for (int k = 0; k < 8; k++) d[k] = (*this)(weight(l[k], m, c2), i + k, x[k]);
    }
};

// Workgroup i: chunk i % nchunk for request i / nchunk.  Every workgroup of a request judges its drafts, then sums
// one chunk of what is left at the row where it stopped; the last one to finish
// draws the token.
template <typename LT, int PER>
__global__ __launch_bounds__(SV_THREADS) void k_sv_finish(const SvArgs a)
{
    __shared__ int s_stop[SV_WAVES], s_pass[SV_WAVES];
    __shared__ SvRow s_row[SV_WAVES];
    __shared__ double s_d[SV_WAVES], s_tot[SV_MAX_CHUNKS];
    __shared__ int s_win, s_last;
    const int b = (int)blockIdx.x / a.nchunk, ch = (int)blockIdx.x % a.nchunk;
    const int tid = (int)threadIdx.x, wv = wave_id(), lane = lane_id();
    const int r0 = a.off[b], r1 = a.off[b + 1];
    const bool gr = greedy(a.temp, b);
    const double c2 = scale2(a.temp, b);
    const LT *z0 = static_cast<const LT *>(a.logits);
    // rows of no request's, or draft rows past the probabilities': nothing is judged
    if (r0 < b || r1 <= r0 || r1 > a.R || r1 - 2 - b >= a.R - a.B) {
        if (ch == 0 && tid == 0) {
            __hip_atomic_fetch_or(a.err, BREAD_DEV_ERR_OFFSET, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            a.accepted[b] = 0;
            a.next[b] = 0;
        }
        return;
    }
    // wave w judges the rows r0 + w, r0 + w + 4, ...; its first that stops
    int stop = 0x7FFFFFFF, pass = 0;
    SvRow mine{0.0, 0.f, 0};
    for (int r = r0 + wv; r < r1; r += SV_WAVES) {
        if (stop != 0x7FFFFFFF && !(ch == 0 && a.logp)) break;
        bool in = false;
        int d = -1;
        float l = -__builtin_inff(), qd = 1.0f, u = 0.f;
        if (r + 1 < r1) {
            d = a.tokens[r + 1];
            u = a.u[r];
            in = d >= 0 && d < a.V;
            if (in) {
                if constexpr (sizeof(LT) == 2) l = num(h2f(z0[(size_t)r * a.stride + d]));
                else l = num(z0[(size_t)r * a.stride + d]);
                if (a.q) qd = a.q[(size_t)(r - b) * a.qstride + d];
            }
        }
        const SvRow s = row_stats(a, r, c2);
        bool ok = false, ends = true;
        if (r + 1 < r1) {
            double p = in && s.sum > 0.0 ? weight(l, s.max, c2) / s.sum : 0.0;
            if (gr) p = in && d == s.arg && s.sum > 0.0 ? 1.0 : 0.0;
            ok = (double)u * (qd > 0.f ? (double)qd : 0.0) < p;
            ends = d == a.eos;
            if (ch == 0 && a.logp && lane == 0) a.logp[r] = log_p(l, s, c2);
        }
        if (stop == 0x7FFFFFFF && (!ok || ends)) {
            stop = r;
            pass = ok;
            mine = s;
        }
    }
    if (lane == 0) {
        s_stop[wv] = stop;
        s_pass[wv] = pass;
        s_row[wv] = mine;
    }
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int k = 1; k < SV_WAVES; k++)
        if (s_stop[k] < s_stop[at]) at = k;
    const int row = s_stop[at];
    const SvRow rs = s_row[at];
    const LT *z = z0 + (size_t)row * a.stride;
    const bool ended = s_pass[at];  // the end token stood
    auto answer = [&](int token) {
        a.accepted[b] = row - r0;
        a.next[b] = token;
        if (a.logp) {
            float l = -__builtin_inff();
            if (token >= 0 && token < a.V) {
                if constexpr (sizeof(LT) == 2) l = num(h2f(z[token]));
                else l = num(z[token]);
            }
            a.logp[r1 - 1] = log_p(l, rs, c2);
        }
    };
    if (ended || gr || !(rs.sum > 0.0)) {
        if (ch == 0 && tid == 0) answer(ended ? a.tokens[row + 1] : rs.sum > 0.0 ? rs.arg : 0);
        return;
    }
    SvLeft left{nullptr, -1, rs.sum};
    if (row + 1 < r1) {
        if (a.q) left.q = a.q + (size_t)(row - b) * a.qstride;
        else left.one = a.tokens[row + 1];
    }
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < PER / 8; j++) {
        double d[8];
        left.template eight<LT>(z, ch * (SV_THREADS * PER) + (j * SV_THREADS + tid) * 8, a.V, rs.max, c2, d);
#pragma unroll
        for (int k = 0; k < 8; k++) s += d[k];
    }
    s = sum_f64(s);
    if (lane == 0) s_d[wv] = s;
    __syncthreads();
    if (tid == 0) {
        for (int k = 1; k < SV_WAVES; k++) s += s_d[k];
        __hip_atomic_store(&a.tot[(size_t)b * a.nchunk + ch], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // the last workgroup of the request sees every sum, and leaves the counter at zero
        const uint32_t n = __hip_atomic_fetch_add(&a.count[b], 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        s_last = n + 1 == (uint32_t)a.nchunk;
        if (s_last) __hip_atomic_store(&a.count[b], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_win = 0x7FFFFFFF;
    }
    __syncthreads();
    if (!s_last) return;
    for (int c = tid; c < a.nchunk; c += SV_THREADS)
        s_tot[c] = __hip_atomic_load(&a.tot[(size_t)b * a.nchunk + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    // every wave sums the chunks, 64 at a time
    auto whole_sum = [&] {
        double t = 0.0;
        for (int c = lane; c < a.nchunk; c += WAVE) t += s_tot[c];
        return sum_f64(t);
    };
    double total = whole_sum();
    if (!(total > 0.0)) {  // the draft's probabilities cover the target's: draw from the target's
        left = SvLeft{nullptr, -1, rs.sum};
        __syncthreads();
        for (int c = tid; c < a.nchunk; c += SV_THREADS) {
            const SvPart &p = a.part[(size_t)row * a.nchunk + c];
            s_tot[c] = p.sum * weight(p.max, rs.max, c2);
        }
        __syncthreads();
        total = whole_sum();
    }
    // the chunk that the border lies in, and the weight before it; where rounding puts the border past the
    // end, the last chunk with any weight
    const double border = (double)a.u[r1 - 1] * total;
    double before = 0.0, sum = 0.0;
    int hit = -1, last = 0;
    double last_before = 0.0;
    for (int c0 = 0; c0 < a.nchunk && hit < 0; c0 += WAVE) {
        const double x = c0 + lane < a.nchunk ? s_tot[c0 + lane] : 0.0;
        const double inc = sum + wave_scan_incl_f64(x);
        const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0);
        const uint64_t over = __builtin_amdgcn_ballot_w64(x > 0.0 && inc > border);
        if (over) {
            hit = c0 + (int)__builtin_ctzll(over);
            before = readlane_f64(inc - x, hit & 63);
        } else if (some) {
            const int w = 63 - (int)__builtin_clzll(some);
            last = c0 + w;
            last_before = readlane_f64(inc - x, w);
        }
        sum = readlane_f64(inc, 63);
    }
    if (hit < 0) {
        hit = last;
        before = last_before;
    }
    // inside the chunk: thread t owns PER consecutive tokens
    const int i0 = hit * (SV_THREADS * PER) + tid * PER;
    double x[PER], own = 0.0;
#pragma unroll
    for (int j = 0; j < PER / 8; j++) {
        double d[8];
        left.template eight<LT>(z, i0 + 8 * j, a.V, rs.max, c2, d);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            x[8 * j + k] = d[k];
            own += d[k];
        }
    }
    const double inc = wave_scan_incl_f64(own);
    if (lane == WAVE - 1) s_d[wv] = inc;
    __syncthreads();
    double cum = before + (inc - own);
    for (int k = 0; k < wv; k++) cum += s_d[k];
    int win = 0x7FFFFFFF, some = -1;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        cum += x[k];
        if (x[k] > 0.0) {
            some = i0 + k;
            if (win == 0x7FFFFFFF && cum > border) win = i0 + k;
        }
    }
    atomicMin(&s_win, win);
    __syncthreads();
    if (s_win == 0x7FFFFFFF) {  // by rounding: the last token of the chunk with any weight
        __syncthreads();
        if (tid == 0) s_win = -1;
        __syncthreads();
        atomicMax(&s_win, some);
        __syncthreads();
    }
    if (tid == 0) answer(s_win < 0 ? rs.arg : s_win);
}

template <typename LT, int PER>
int launch(const SvArgs &a, hipStream_t st)
{
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_sv_stats<LT, PER>), dim3((unsigned)(a.R * a.nchunk)), dim3(SV_THREADS), 0, st, a);
    BREAD_HIP(hipGetLastError());
    hipLaunchKernelGGL((k_sv_finish<LT, PER>), dim3((unsigned)(a.B * a.nchunk)), dim3(SV_THREADS), 0, st, a);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

}  // namespace

extern "C" int bread_spec_verify(bread_moe_ctx_t *c, const bread_verify_t *v, bread_stream_t stream)
{
    BREAD_REQUIRE(c && v, BREAD_ERR_ARG, "NULL context or arguments");
    BREAD_REQUIRE(v->vocab > 0 && v->n_rows >= 0 && v->n_requests >= 0, BREAD_ERR_ARG,
                  "vocab must be > 0, n_rows and n_requests >= 0");
    BREAD_REQUIRE(v->vocab <= 1 << 24, BREAD_ERR_SHAPE, "vocab > 16777216");
    BREAD_REQUIRE(v->n_requests <= v->n_rows, BREAD_ERR_ARG, "every request has at least one row");
    BREAD_REQUIRE(v->logits_type == BREAD_QTYPE_F16 || v->logits_type == BREAD_QTYPE_F32, BREAD_ERR_QTYPE,
                  "logits_type must be 1 (F16) or 0 (F32)");
    BREAD_REQUIRE((v->logits_stride == 0 || v->logits_stride >= v->vocab) &&
                      (v->draft_probs_stride == 0 || v->draft_probs_stride >= v->vocab),
                  BREAD_ERR_SHAPE, "a stride is smaller than the vocabulary");
    BREAD_REQUIRE(v->n_rows <= c->max_tokens, BREAD_ERR_CAPACITY, "n_rows > max_tokens of the context");
    if (v->n_requests == 0) return BREAD_OK;
    BREAD_REQUIRE(v->logits && v->tokens && v->offsets && v->u && v->n_accept && v->next, BREAD_ERR_ARG,
                  "NULL input or output");
    const uintptr_t la = v->logits_type == BREAD_QTYPE_F32 ? 3 : 1;
    BREAD_REQUIRE(((uintptr_t)v->logits & la) == 0 &&
                      (((uintptr_t)v->tokens | (uintptr_t)v->offsets | (uintptr_t)v->u | (uintptr_t)v->draft_probs |
                        (uintptr_t)v->temperature | (uintptr_t)v->n_accept | (uintptr_t)v->next |
                        (uintptr_t)v->logprob) & 3) == 0,
                  BREAD_ERR_ALIGN, "buffers must be aligned to their elements");
    SvArgs a;
    a.logits = v->logits;
    a.V = v->vocab;
    a.stride = v->logits_stride ? v->logits_stride : v->vocab;
    a.R = v->n_rows;
    a.B = v->n_requests;
    a.tokens = v->tokens;
    a.off = v->offsets;
    a.u = v->u;
    a.q = v->draft_probs;
    a.qstride = v->draft_probs_stride ? v->draft_probs_stride : v->vocab;
    a.temp = v->temperature;
    a.eos = v->eos;
    // the partial results live in the context's SwiGLU buffer (free between MoE calls on the stream)
    const bread_moe_shape_t &s = c->shape;
    const size_t Imax = (size_t)(s.expert_inter > s.shared_inter ? s.expert_inter : s.shared_inter);
    const size_t have = (size_t)c->max_tokens * (s.top_k + 1) * Imax * sizeof(float);
    auto chunks = [&](int per) { return (int)(((int64_t)a.V + SV_THREADS * per - 1) / (SV_THREADS * per)); };
    auto bytes = [&](int per) {
        return (size_t)chunks(per) * ((size_t)a.R * sizeof(SvPart) + (size_t)a.B * sizeof(double));
    };
    BREAD_REQUIRE(bytes(SV_MANY) <= have && (int64_t)a.R * chunks(SV_MANY) < (1ll << 31), BREAD_ERR_CAPACITY,
                  "the context's scratch is too small for this vocabulary: create it for more tokens");
    const bool few = (int64_t)a.R * chunks(SV_FEW) <= 2048 && chunks(SV_FEW) <= SV_MAX_CHUNKS && bytes(SV_FEW) <= have;
    a.nchunk = chunks(few ? SV_FEW : SV_MANY);
    const size_t parts = (size_t)a.R * a.nchunk * sizeof(SvPart);
    a.part = reinterpret_cast<SvPart *>(c->h);
    a.tot = reinterpret_cast<double *>(reinterpret_cast<uint8_t *>(c->h) + parts);
    a.count = c->vcount;
    a.err = &c->dsync->error.v;
    a.accepted = v->n_accept;
    a.next = v->next;
    a.logp = v->logprob;
    const hipStream_t st = to_hip(stream);
    c->last_stream = st;
    if (v->logits_type == BREAD_QTYPE_F16) return few ? launch<uint16_t, SV_FEW>(a, st) : launch<uint16_t, SV_MANY>(a, st);
    return few ? launch<float, SV_FEW>(a, st) : launch<float, SV_MANY>(a, st);
}
