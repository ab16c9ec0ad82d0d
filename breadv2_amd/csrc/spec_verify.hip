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
// Logits a thread (PER): 32 once there is plenty of work, 8 below that, where the time is a workgroup's chain of
// loads and exponentials.  A workgroup's chunk of a row is SV_THREADS times as many.  us on MI355X with 32 and with 8,
// drafts looked up, rows of 248,320 tokens: 4 rows 27.7 and 15.6, 64 rows 36.0 and 27.7, 128 rows 46.7 and 38.5, 400
// rows 88 and 86, 1024 rows 185 and 200; of 32,000 tokens: 8 rows 27.4 and 15.4, 1024 rows 45.9 and 40.8.
// 64 requests with 8 drafts and their probabilities, 248,320 tokens: 144 and 172.
constexpr int SV_MANY = 32, SV_FEW = 8;
constexpr int SV_FEW_CHUNKS = 16384;  // in all, at 8 a thread
constexpr int SV_ROWS = 8;  // waves of k_sv_accept: rows looked at side by side
constexpr int SV_CHAINS = 2;  // exponentials side by side
constexpr int SV_MAX_CHUNKS = 2048;  // of a row: 2^24 logits in chunks of 8192

// One chunk of a row: the largest logit and the sum of exp((l - max) / T).
struct SvPart {
    double sum;
    float max;
    int arg;  // lowest index of the largest logit
};

// Where a request's draft fell against a draft model's probabilities: what is left there is drawn by k_sv_left.
struct SvStop {
    double sum;  // of the row's weights
    float max;
    int row;     // -1: the request has its token
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
    SvStop *stop;      // [B]
    double *tot;       // [B][nchunk]
    uint32_t *count;   // [B], zero between calls
    uint32_t *err;
    int32_t *accepted, *next;
    float *logp;       // may be NULL
};

// The larger of two, a number against NaN (fmaxf's rule, without the compiler's two extra instructions to quiet
// its arguments first; of a signalling NaN after nan_is_nan())
__device__ __forceinline__ float max2(float a, float b)
{
    float d;
    asm("v_max_f32 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}

// At a kernel's start: from here on the wave's maxima take a signalling NaN as any other.  With the mode register's
// IEEE bit (9), which kernels start with, v_max of one and a number is NaN; quieting the logits first would be an
// instruction for each (for each two, in fp16).
__device__ __forceinline__ void nan_is_nan()
{
    __builtin_amdgcn_s_setreg(1 | (9 << 6) | (0 << 11), 0u);  // hwreg(HW_REG_MODE, 9, 1)
}

// A logit as a number: NaN counts as -inf
__device__ __forceinline__ float num(float v)
{
    return max2(v, -__builtin_inff());
}

template <typename LT>
__device__ __forceinline__ float logit(LT v)
{
    if constexpr (sizeof(LT) == 2) return num(h2f(v));
    else return num(v);
}

// 2^y for y <= 0 by 2^n p(f), n the nearest whole number to y, f = y - n and p the polynomial of degree 9 that is 1
// at 0 and has the least largest relative error on [-1/2, 1/2], 8e-14 (by Remez exchange).  The coefficients stay
// in scalar registers: left to itself the compiler moves each to vector registers for every use, two moves for a
// multiply-add.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct Exp2 {
    double c[9];
    __device__ __forceinline__ Exp2()
        : c{0x1.62e42fefa08dcp-1, 0x1.ebfbdff823df0p-3, 0x1.c6b08d7a95072p-5, 0x1.3b2ab717fb0b6p-7, 0x1.5d87ebe42d79dp-10,
            0x1.4308acc67a164p-13, 0x1.fffd75179b1a0p-17, 0x1.63d0ec28f10f2p-20, 0x1.89c489e9e3ae4p-24}
    {
#pragma unroll
        for (int k = 0; k < 8; k++) asm("" : "+s"(c[k]));
        asm("" : "+v"(c[8]));  // an instruction takes one scalar operand
    }
    __device__ __forceinline__ double part(double f) const
    {
        double p = c[8];
#pragma unroll
        for (int k = 7; k >= 0; k--) asm("v_fma_f64 %0, %1, %2, %3" : "=v"(p) : "v"(p), "v"(f), "s"(c[k]));
        return fma(p, f, 1.0);
    }
    // any y: 1 for 0, and 0 below -1075, for -inf and for NaN (-inf times 1 / an infinite temperature)
    __device__ __forceinline__ double operator()(double y) const
    {
        y = fmax(y, -1100.0);
        const double n = __builtin_rint(y);
        return __builtin_amdgcn_ldexp(part(y - n), (int)n);
    }
};

// 2^(j / 32), rounded
__constant__ double SV_TWO[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// Many of them, each y in [-1000, 1]: 2^(k / 32) p(f) with k the nearest whole number to 32 y, f = y - k / 32 and p of
// degree 4 (to 8e-14 on [-1/64, 1/64]).  2^(j / 32), j = k % 32, comes from 32 doubles in LDS, a bank each, that
// hold j subtracted from the exponent's place, so that k is added there whole.  Bound by its 64-bit instructions,
// ten a logit; with the polynomial of degree 9 and no table they are sixteen, and k_sv_stats' 101 us below 119.
struct Exp2Table {
    double c[4];
    const double *two;
    // lanes 0 to 31 of the wave fill its table
    __device__ __forceinline__ explicit Exp2Table(double *mem)
        : c{0x1.62e42fef6d0cdp-1, 0x1.ebfbdff87b60bp-3, 0x1.c6b167d804924p-5, 0x1.3b2a9efd4ad16p-7}, two(mem)
    {
#pragma unroll
        for (int k = 0; k < 3; k++) asm("" : "+s"(c[k]));
        asm("" : "+v"(c[3]));
        const int j = lane_id();
        if (j < 32) {
            u32x2 q = __builtin_bit_cast(u32x2, SV_TWO[j]);
            q.y -= (uint32_t)j << 15;
            mem[j] = __builtin_bit_cast(double, q);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // s[i] += 2^y[i], N chains so that no instruction waits for the one before it
    template <int N>
    __device__ __forceinline__ void add(const double (&y)[N], double (&s)[N]) const
    {
        double t[N], f[N], p[N], w[N];
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = y[i] + 0x1.8p47;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t k = __builtin_bit_cast(u32x2, t[i]).x;
            u32x2 q = __builtin_bit_cast(u32x2, two[k & 31]);
            q.y += k << 15;
            w[i] = __builtin_bit_cast(double, q);
        }
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = y[i] - (t[i] - 0x1.8p47);
#pragma unroll
        for (int i = 0; i < N; i++) asm("v_fma_f64 %0, %1, %2, %3" : "=v"(p[i]) : "v"(c[3]), "v"(f[i]), "s"(c[2]));
#pragma unroll
        for (int k = 1; k >= 0; k--)
#pragma unroll
            for (int i = 0; i < N; i++) asm("v_fma_f64 %0, %1, %2, %3" : "=v"(p[i]) : "v"(p[i]), "v"(f[i]), "s"(c[k]));
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = fma(w[i], fma(p[i], f[i], 1.0), s[i]);
    }
};

constexpr double LOG2E = 1.4426950408889634;

// exp((l - m) / T) for l <= m, c2 = log2(e) / T: 1 where they are equal, infinite ones too; 0 for l = -inf
__device__ __forceinline__ double weight(const Exp2 &e2, float l, float m, double c2)
{
    if (__builtin_isinf(m)) return l == m && m > 0.f ? 1.0 : 0.0;
    return e2(((double)l - (double)m) * c2);
}

// Eight logits (or probabilities) as they are stored
template <typename LT> struct Eight;

template <> struct Eight<uint16_t> {
    uint32_t w[4];
    __device__ __forceinline__ float value(int k) const { return h2f(w[k / 2] >> (16 * (k & 1))); }
    __device__ __forceinline__ void set(int k, uint16_t v)
    {
        w[k / 2] = (k & 1) ? (w[k / 2] & 0xFFFFu) | ((uint32_t)v << 16) : v;
    }
    static constexpr uint16_t NONE = 0xFC00;  // -inf
};

template <> struct Eight<float> {
    float w[8];
    __device__ __forceinline__ float value(int k) const { return w[k]; }
    __device__ __forceinline__ void set(int k, float v) { w[k] = v; }
    static constexpr float NONE = -__builtin_inff();
};

// Eight values from element i on, of which those at V and beyond read as `none`
template <typename LT>
__device__ __forceinline__ void load8(const LT *row, int i, int V, LT none, Eight<LT> &v)
{
    if (i + 8 <= V) {
        __builtin_memcpy(&v, row + i, sizeof(v));  // aligned to an element
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v.set(k, i + k < V ? row[i + k] : none);
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

__device__ __forceinline__ uint32_t max2_f16(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(d) : "v"(a), "v"(b));
    return d;
}

// The largest of the values and m, numbers against NaN
__device__ __forceinline__ float max8(const Eight<float> &v, float m)
{
#pragma unroll
    for (int k = 0; k < 8; k++) m = max2(m, v.w[k]);
    return m;
}

__device__ __forceinline__ float max8(const Eight<uint16_t> &v, float m)
{
    const uint32_t p = max2_f16(max2_f16(v.w[0], v.w[1]), max2_f16(v.w[2], v.w[3]));
    return max2(max2(m, h2f(p)), h2f(p >> 16));
}

// The values, those below `least` and NaN raised to it
__device__ __forceinline__ Eight<float> raise8(const Eight<float> &v, float least)
{
    Eight<float> r;
#pragma unroll
    for (int k = 0; k < 8; k++) r.w[k] = max2(v.w[k], least);
    return r;
}

__device__ __forceinline__ Eight<uint16_t> raise8(const Eight<uint16_t> &v, float least)
{
    const uint32_t h = f2h(least), hh = h | (h << 16);
    Eight<uint16_t> r;
#pragma unroll
    for (int k = 0; k < 4; k++) r.w[k] = max2_f16(v.w[k], hh);
    return r;
}

// A chunk a wave (chunk i % nchunk of row i / nchunk), 32 logits a lane at a time and the next ones on their way:
// the largest so far, and in each lane its own sum relative to it; a larger one scales the sum down.
// Bound by the 64-bit instructions: 64 requests with 8 drafts over 248,320 tokens, 143M fp16 logits, 101 us on MI355X
// (2.8 TB/s; nine tenths of the issue slots are taken).  A chunk a workgroup, 32 logits a thread, spent a third of its
// instructions on two reductions (149 us before the table); several chunks a wave, one round of waves for the GPU, end
// unevenly (130 us).  Two chains leave room for four waves a SIMD, three for fp32 logits: 4 us less than four chains.
template <typename LT, int PER>
__global__ __launch_bounds__(SV_THREADS, sizeof(LT) == 2 ? 4 : 3) void k_sv_stats(const SvArgs a)
{
    constexpr int STEPS = PER * SV_WAVES / 32, STEP = 32 * WAVE;
    __shared__ double s_two[SV_WAVES][32];
    nan_is_nan();
    const Exp2 e2;
    const int lane = lane_id(), at = (int)blockIdx.x * SV_WAVES + wave_id();
    if (at >= a.R * a.nchunk) return;
    const int row = at / a.nchunk, base = (at - row * a.nchunk) * (STEPS * STEP), i0 = base + lane * 8;
    const LT *z = static_cast<const LT *>(a.logits) + (size_t)row * a.stride;
    Eight<LT> v[4], nx[4];
    auto load = [&](int step) __attribute__((always_inline)) {
        const int i = i0 + step * STEP;
        if (base + (step + 1) * STEP <= a.V) {  // (the whole wave)
#pragma unroll
            for (int j = 0; j < 4; j++) __builtin_memcpy(&nx[j], z + i + j * (8 * WAVE), sizeof(nx[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) load8<LT>(z, i + j * (8 * WAVE), a.V, Eight<LT>::NONE, nx[j]);
        }
    };
    load(0);
    const Exp2Table many(s_two[wave_id()]);
    const int b = request_of(a.off, a.B, row);
    const double c2 = scale2(a.temp, b);
    const bool gr = greedy(a.temp, b);
    float m = -__builtin_inff(), least = 0.f;
    double s[SV_CHAINS] = {}, mc = 0.0;
    bool plain = false;
    int arg = 0x7FFFFFFF;
    for (int step = 0; step < STEPS; step++) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = nx[j];
        if (step + 1 < STEPS) load(step + 1);
        float ms = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 4; j++) ms = max8(v[j], ms);
        ms = wave_max(ms);
        if (ms > m) {
            if (m > -__builtin_inff()) {
                const double down = weight(e2, m, ms, c2);
#pragma unroll
                for (int i = 0; i < SV_CHAINS; i++) s[i] *= down;
            }
            m = ms;
            arg = 0x7FFFFFFF;
            // Logits whose 2^y would have y < -1000 or so, masked ones and NaN too, are raised to `least` and count
            // as 2^-200 or less next to a sum of at least 1; above it the exponent can be added to the bits.  An
            // unusual temperature or size, where fp16 (or fp32) has no such value, takes the general form.
            least = m - 900.f / (float)c2;
            if constexpr (sizeof(LT) == 2) least = h2f(f2h(least));
            const double yl = ((double)least - (double)m) * c2;
            plain = yl >= -1000.0 && yl <= -200.0 && least > -60000.f;
            mc = -(double)m * c2;
        }
        if (plain) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const Eight<LT> r = raise8(v[j], least);
#pragma unroll
                for (int k = 0; k < 8; k += SV_CHAINS) {
                    double y[SV_CHAINS];
#pragma unroll
                    for (int i = 0; i < SV_CHAINS; i++) y[i] = fma((double)r.value(k + i), c2, mc);
                    many.add(y, s);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int k = 0; k < 8; k++) s[k % SV_CHAINS] += weight(e2, num(v[j].value(k)), m, c2);
        }
        if (gr && arg == 0x7FFFFFFF) {  // (of the lane; the first step that has the largest has the lane's lowest)
#pragma unroll
            for (int j = 3; j >= 0; j--)
#pragma unroll
                for (int k = 7; k >= 0; k--) {
                    const int i = i0 + step * STEP + j * (8 * WAVE) + k;
                    if (num(v[j].value(k)) == m && i < a.V) arg = i;
                }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < SV_CHAINS; i++) sum += s[i];
    sum = sum_f64(sum);
    if (gr)
        for (int o = WAVE / 2; o > 0; o >>= 1) arg = min(arg, __shfl_xor(arg, o));
    if (lane == 0) a.part[at] = SvPart{sum, m, arg};
}

// A row's statistics from its chunks, by one wave
struct SvRow {
    double sum;
    float max;
    int arg;
};

__device__ __forceinline__ SvRow row_stats(const SvArgs &a, const Exp2 &e2, int row, double c2)
{
    // the first chunks (all of 262144 logits in chunks of 2048) stay in registers: one trip to memory
    constexpr int KEEP = 2;
    const SvPart *p = a.part + (size_t)row * a.nchunk;
    const int lane = lane_id();
    SvRow r{0.0, -__builtin_inff(), 0x7FFFFFFF};
    SvPart k[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; i++)
        k[i] = i * WAVE + lane < a.nchunk ? p[i * WAVE + lane] : SvPart{0.0, -__builtin_inff(), 0x7FFFFFFF};
#pragma unroll
    for (int i = 0; i < KEEP; i++) r.max = fmaxf(r.max, k[i].max);
    for (int c = KEEP * WAVE + lane; c < a.nchunk; c += WAVE) r.max = fmaxf(r.max, p[c].max);
    r.max = wave_max(r.max);
    auto add = [&](const SvPart &q) __attribute__((always_inline)) {
        r.sum += q.sum * weight(e2, q.max, r.max, c2);
        if (q.max == r.max) r.arg = min(r.arg, q.arg);
    };
#pragma unroll
    for (int i = 0; i < KEEP; i++) add(k[i]);
    for (int c = KEEP * WAVE + lane; c < a.nchunk; c += WAVE) add(p[c]);
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
    __device__ __forceinline__ void eight(const Exp2 &e2, const LT *z, int i, int V, float m, double c2, double (&d)[8]) const
    {
        Eight<LT> l;
        Eight<float> x{};
        load8<LT>(z, i, V, Eight<LT>::NONE, l);
        if (q) load8<float>(q, i, V, 0.f, x);
#pragma unroll
        for (int k = 0; k < 8; k++) d[k] = (*this)(weight(e2, num(l.value(k)), m, c2), i + k, x.w[k]);
    }
};

// The chunk that the border lies in and the weight before it, from the chunks' weights in LDS; where rounding
// puts the border past the end, the last chunk with any weight.  By every wave alike.
__device__ __forceinline__ void find_chunk(const double *tot, int nchunk, double border, int &hit, double &before)
{
    const int lane = lane_id();
    double sum = 0.0, last_before = 0.0;
    int last = 0;
    for (int c0 = 0; c0 < nchunk; c0 += WAVE) {
        const double x = c0 + lane < nchunk ? tot[c0 + lane] : 0.0;
        const double inc = sum + wave_scan_incl_f64(x);
        const uint64_t some = __builtin_amdgcn_ballot_w64(x > 0.0);
        const uint64_t over = __builtin_amdgcn_ballot_w64(x > 0.0 && inc > border);
        if (over) {
            const int w = (int)__builtin_ctzll(over);
            hit = c0 + w;
            before = readlane_f64(inc - x, w);
            return;
        }
        if (some) {
            const int w = 63 - (int)__builtin_clzll(some);
            last = c0 + w;
            last_before = readlane_f64(inc - x, w);
        }
        sum = readlane_f64(inc, 63);
    }
    hit = last;
    before = last_before;
}

__device__ __forceinline__ double whole_sum(const double *tot, int nchunk)
{
    double t = 0.0;
    for (int c = lane_id(); c < nchunk; c += WAVE) t += tot[c];
    return sum_f64(t);
}

// Sum over the workgroup of W waves, in every thread (s_d: one double a wave)
template <int W>
__device__ __forceinline__ double block_sum(double v, double *s_d)
{
    v = sum_f64(v);
    __syncthreads();
    if (lane_id() == 0) s_d[wave_id()] = v;
    __syncthreads();
    v = s_d[0];
#pragma unroll
    for (int k = 1; k < W; k++) v += s_d[k];
    return v;
}

// What is left of a chunk, its parts in the first SV_THREADS threads of the workgroup
template <typename LT, int PER>
__device__ __forceinline__ double chunk_left(const Exp2 &e2, const SvLeft &left, const LT *z, int ch, int V, float max, double c2)
{
    double s = 0.0;
    if ((int)threadIdx.x >= SV_THREADS) return s;
#pragma unroll
    for (int j = 0; j < PER / 8; j++) {
        double d[8];
        left.template eight<LT>(e2, z, ch * (SV_THREADS * PER) + (j * SV_THREADS + (int)threadIdx.x) * 8, V, max, c2, d);
#pragma unroll
        for (int k = 0; k < 8; k++) s += d[k];
    }
    return s;
}

// The token at the border, by the workgroup, from the chunks' weights in tot (LDS): the first whose cumulative
// weight exceeds u times the whole; -1 where there is no weight.
template <typename LT, int PER>
__device__ __forceinline__ int draw(const Exp2 &e2, const SvLeft &left, const LT *z, const double *tot, int nchunk, double border, int V,
                                    float max, double c2, double *s_d, int *s_win)
{
    const int tid = (int)threadIdx.x;
    int hit;
    double before;
    find_chunk(tot, nchunk, border, hit, before);
    // thread t of the first SV_THREADS owns PER consecutive tokens of the chunk
    const int i0 = hit * (SV_THREADS * PER) + tid * PER;
    double x[PER] = {}, own = 0.0;
    if (tid < SV_THREADS) {
#pragma unroll
        for (int j = 0; j < PER / 8; j++) {
            double d[8];
            left.template eight<LT>(e2, z, i0 + 8 * j, V, max, c2, d);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                x[8 * j + k] = d[k];
                own += d[k];
            }
        }
    }
    const double inc = wave_scan_incl_f64(own);
    __syncthreads();
    if (lane_id() == WAVE - 1) s_d[wave_id()] = inc;
    if (tid == 0) *s_win = 0x7FFFFFFF;
    __syncthreads();
    double cum = before + (inc - own);
    for (int k = 0; k < wave_id(); k++) cum += s_d[k];
    int win = 0x7FFFFFFF, some = -1;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        cum += x[k];
        if (x[k] > 0.0) {
            some = i0 + k;
            if (win == 0x7FFFFFFF && cum > border) win = i0 + k;
        }
    }
    if (win != 0x7FFFFFFF) atomicMin(s_win, win);
    __syncthreads();
    if (*s_win == 0x7FFFFFFF) {  // by rounding: the last token of the chunk with any weight
        __syncthreads();
        if (tid == 0) *s_win = -1;
        __syncthreads();
        atomicMax(s_win, some);
        __syncthreads();
    }
    return *s_win;
}

// The request's answer, by one thread
template <typename LT>
__device__ __forceinline__ void answer(const SvArgs &a, int b, int row, const LT *z, const SvRow &rs, double c2, int token)
{
    a.accepted[b] = row - a.off[b];
    a.next[b] = token;
    if (a.logp)
        a.logp[a.off[b + 1] - 1] = log_p(token >= 0 && token < a.V ? logit(z[token]) : -__builtin_inff(), rs, c2);
}

// Workgroup b: tries request b's drafts, a row a wave, and draws its token
// unless a draft fell against a draft model's probabilities (k_sv_left then
// draws it).  Its time is a chain of loads: offsets, then tokens and chunk
// statistics, then the drafts' logits, then the chunk that holds the token:
// 10.8 us on MI355X for one request with four drafts, 16 us for 64 requests.
template <typename LT, int PER>
__global__ __launch_bounds__(SV_ROWS *WAVE) void k_sv_accept(const SvArgs a)
{
    __shared__ int s_stop[SV_ROWS], s_pass[SV_ROWS], s_token[SV_ROWS];
    __shared__ SvRow s_row[SV_ROWS];
    __shared__ double s_d[SV_ROWS], s_tot[SV_MAX_CHUNKS];
    __shared__ int s_win;
    nan_is_nan();
    const Exp2 e2;
    const int b = (int)blockIdx.x, tid = (int)threadIdx.x, wv = wave_id(), lane = lane_id();
    const int r0 = a.off[b], r1 = a.off[b + 1];
    const bool gr = greedy(a.temp, b);
    const double c2 = scale2(a.temp, b);
    const LT *z0 = static_cast<const LT *>(a.logits);
    if (tid == 0) a.stop[b].row = -1;
    // rows of no request's, or draft rows past the probabilities': nothing is done
    if (r0 < b || r1 <= r0 || r1 > a.R || r1 - 2 - b >= a.R - a.B) {
        if (tid == 0) {
            __hip_atomic_fetch_or(a.err, BREAD_DEV_ERR_OFFSET, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            a.accepted[b] = 0;
            a.next[b] = 0;
        }
        return;
    }
    const float u_last = a.u[r1 - 1];
    // wave w takes the rows r0 + w, r0 + w + 8, ...; its first that stops
    int stop = 0x7FFFFFFF, pass = 0, token = -1;
    SvRow mine{0.0, 0.f, 0};
    for (int r = r0 + wv; r < r1; r += SV_ROWS) {
        if (stop != 0x7FFFFFFF && !a.logp) break;
        bool in = false;
        int d = -1;
        float l = -__builtin_inff(), qd = 1.0f, u = 0.f;
        if (r + 1 < r1) {
            d = a.tokens[r + 1];
            u = a.u[r];
            in = d >= 0 && d < a.V;
            if (in) {
                l = logit(z0[(size_t)r * a.stride + d]);
                if (a.q) qd = a.q[(size_t)(r - b) * a.qstride + d];
            }
        }
        const SvRow s = row_stats(a, e2, r, c2);
        bool ok = false, ends = true;
        if (r + 1 < r1) {
            double p = in && s.sum > 0.0 ? weight(e2, l, s.max, c2) / s.sum : 0.0;
            if (gr) p = in && d == s.arg && s.sum > 0.0 ? 1.0 : 0.0;
            ok = (double)u * (qd > 0.f ? (double)qd : 0.0) < p;
            ends = d == a.eos;
            if (a.logp && lane == 0) a.logp[r] = log_p(l, s, c2);
        }
        if (stop == 0x7FFFFFFF && (!ok || ends)) {
            stop = r;
            pass = ok;
            token = d;
            mine = s;
        }
    }
    if (lane == 0) {
        s_stop[wv] = stop;
        s_pass[wv] = pass;
        s_token[wv] = token;
        s_row[wv] = mine;
    }
    __syncthreads();
    int at = 0;
#pragma unroll
    for (int k = 1; k < SV_ROWS; k++)
        if (s_stop[k] < s_stop[at]) at = k;
    const int row = s_stop[at];
    const SvRow rs = s_row[at];
    const LT *z = z0 + (size_t)row * a.stride;
    const int draft = s_token[at];  // (none in the last row)
    const bool ended = s_pass[at];  // the end token stood
    if (ended || gr || !(rs.sum > 0.0)) {
        if (tid == 0) answer(a, b, row, z, rs, c2, ended ? draft : rs.sum > 0.0 ? rs.arg : 0);
        return;
    }
    const bool fell = row + 1 < r1;
    if (fell && a.q) {
        if (tid == 0) a.stop[b] = SvStop{rs.sum, rs.max, row};
        return;
    }
    // the row's own weights, without the draft that was looked up
    const SvLeft left{nullptr, fell ? draft : -1, rs.sum};
    const bool one = left.one >= 0 && left.one < a.V;
    // (summed again rather than subtracted: the draft may be nearly all there was; its chunk is on its way while the
    // others' sums are)
    const int its = one ? left.one / (SV_THREADS * PER) : -1;
    const double part = one ? chunk_left<LT, PER>(e2, left, z, its, a.V, rs.max, c2) : 0.0;
    for (int c = tid; c < a.nchunk; c += SV_ROWS * WAVE) {
        const SvPart &p = a.part[(size_t)row * a.nchunk + c];
        if (c != its) s_tot[c] = p.sum * weight(e2, p.max, rs.max, c2);
    }
    double total = rs.sum;
    if (one) {
        const double x = block_sum<SV_ROWS>(part, s_d);
        if (tid == 0) s_tot[its] = x;
        __syncthreads();
        total = whole_sum(s_tot, a.nchunk);
    } else {
        __syncthreads();
    }
    SvLeft from = left;
    if (!(total > 0.0)) {  // the draft was all there was
        from.one = -1;
        __syncthreads();
        for (int c = tid; c < a.nchunk; c += SV_ROWS * WAVE) {
            const SvPart &p = a.part[(size_t)row * a.nchunk + c];
            s_tot[c] = p.sum * weight(e2, p.max, rs.max, c2);
        }
        __syncthreads();
        total = whole_sum(s_tot, a.nchunk);
    }
    const int next = draw<LT, PER>(e2, from, z, s_tot, a.nchunk, (double)u_last * total, a.V, rs.max, c2, s_d, &s_win);
    if (tid == 0) answer(a, b, row, z, rs, c2, next);
}

// Workgroup i: what is left of chunk i % nchunk at the row where a draft of
// request i / nchunk fell; the request's last one to finish draws the token.
template <typename LT, int PER>
__global__ __launch_bounds__(SV_THREADS) void k_sv_left(const SvArgs a)
{
    __shared__ double s_d[SV_WAVES], s_tot[SV_MAX_CHUNKS];
    __shared__ int s_win, s_last;
    nan_is_nan();
    const Exp2 e2;
    const int b = (int)blockIdx.x / a.nchunk, ch = (int)blockIdx.x % a.nchunk;
    const int tid = (int)threadIdx.x;
    const SvStop st = a.stop[b];
    if (st.row < 0) return;
    const double c2 = scale2(a.temp, b);
    const LT *z = static_cast<const LT *>(a.logits) + (size_t)st.row * a.stride;
    SvLeft left{a.q + (size_t)(st.row - b) * a.qstride, -1, st.sum};
    const double s = block_sum<SV_WAVES>(chunk_left<LT, PER>(e2, left, z, ch, a.V, st.max, c2), s_d);
    if (tid == 0) {
        __hip_atomic_store(&a.tot[(size_t)b * a.nchunk + ch], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // the store has reached where every workgroup sees it before the counter moves; the last workgroup of the
        // request then sees every sum, and leaves the counter at zero
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint32_t n = __hip_atomic_fetch_add(&a.count[b], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_last = n + 1 == (uint32_t)a.nchunk;
        if (s_last) __hip_atomic_store(&a.count[b], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int c = tid; c < a.nchunk; c += SV_THREADS)
        s_tot[c] = __hip_atomic_load(&a.tot[(size_t)b * a.nchunk + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    double total = whole_sum(s_tot, a.nchunk);
    if (!(total > 0.0)) {  // the draft's probabilities cover the target's: draw from the target's
        left.q = nullptr;
        __syncthreads();
        for (int c = tid; c < a.nchunk; c += SV_THREADS) {
            const SvPart &p = a.part[(size_t)st.row * a.nchunk + c];
            s_tot[c] = p.sum * weight(e2, p.max, st.max, c2);
        }
        __syncthreads();
        total = whole_sum(s_tot, a.nchunk);
    }
    const double border = (double)a.u[a.off[b + 1] - 1] * total;
    const int token = draw<LT, PER>(e2, left, z, s_tot, a.nchunk, border, a.V, st.max, c2, s_d, &s_win);
    if (tid == 0) answer(a, b, st.row, z, SvRow{st.sum, st.max, 0}, c2, token < 0 ? 0 : token);
}

template <typename LT, int PER>
int launch(const SvArgs &a, hipStream_t st)
{
    bread_clear_stale_error();
    const int all = a.R * a.nchunk;
    hipLaunchKernelGGL((k_sv_stats<LT, PER>), dim3((unsigned)((all + SV_WAVES - 1) / SV_WAVES)), dim3(SV_THREADS), 0, st, a);
    BREAD_HIP(hipGetLastError());
    hipLaunchKernelGGL((k_sv_accept<LT, PER>), dim3((unsigned)a.B), dim3(SV_ROWS * WAVE), 0, st, a);
    BREAD_HIP(hipGetLastError());
    if (!a.q) return BREAD_OK;
    hipLaunchKernelGGL((k_sv_left<LT, PER>), dim3((unsigned)(a.B * a.nchunk)), dim3(SV_THREADS), 0, st, a);
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
        return (size_t)chunks(per) * ((size_t)a.R * sizeof(SvPart) + (size_t)a.B * sizeof(double)) +
               (size_t)a.B * sizeof(SvStop);
    };
    BREAD_REQUIRE(bytes(SV_MANY) <= have && (int64_t)a.R * chunks(SV_MANY) < (1ll << 24), BREAD_ERR_CAPACITY,
                  "the context's scratch is too small for this vocabulary: create it for more tokens");
    const bool few = (int64_t)a.R * chunks(SV_FEW) <= SV_FEW_CHUNKS && chunks(SV_FEW) <= SV_MAX_CHUNKS && bytes(SV_FEW) <= have;
    a.nchunk = chunks(few ? SV_FEW : SV_MANY);
    a.part = reinterpret_cast<SvPart *>(c->h);
    a.stop = reinterpret_cast<SvStop *>(a.part + (size_t)a.R * a.nchunk);
    a.tot = reinterpret_cast<double *>(a.stop + a.B);
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
