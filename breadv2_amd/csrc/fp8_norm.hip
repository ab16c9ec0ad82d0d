// fp8_norm.hip — bread_rmsnorm_fp8: residual addition, RMSNorm and e4m3 codes
// with a scale for every 128 columns, in one pass over the rows:
//   h = x + residual;  v = h / sqrt(mean(h^2) + eps) * weight;
//   scale = max(max|v| / 448, 2^-126), code = e4m3(v / scale) per block.
// A row stays in its threads' registers from the sum of squares to the codes:
// memory is read and written once.  16384 rows of 2048, fp16 with a residual and
// fp16 results: 65.6 us, 4.6 TB/s (58 us at the copy rate).  Few rows wait for their
// own chain: a wave takes a row of 2048 in four steps of 512, loads, sum and
// codes one after the other (one row: 5.1 us); 509 rows of 4096, 256 threads and
// two steps each, take 6.0.
#include "fp8.h"

namespace {

struct NormArgs {
    const void *x, *res;
    void *h, *out;
    const float *w;
    uint8_t *codes;
    float *scales;
    int64_t xs, rs, hs, cs, ss, os;
    float eps;
    int n, T, out_type;
};

// Eight elements at an address that is aligned to one of them (one or two loads)
template <int XT>
__device__ __forceinline__ void load8(const void *base, int64_t at, float (&v)[8])
{
    if constexpr (XT == BREAD_QTYPE_F32) {
        __builtin_memcpy(v, static_cast<const float *>(base) + at, 32);
    } else {
        uint16_t h[8];
        __builtin_memcpy(h, static_cast<const uint16_t *>(base) + at, 16);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = XT == BREAD_QTYPE_F16 ? h2f(h[i]) : bf2f(h[i]);
    }
}

__device__ __forceinline__ void store8(void *base, int64_t at, int type, const float (&v)[8])
{
    if (type == BREAD_QTYPE_F32) {
        __builtin_memcpy(static_cast<float *>(base) + at, v, 32);
    } else {
        uint16_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = type == BREAD_QTYPE_F16 ? f2h(v[i]) : f2bf(v[i]);
        __builtin_memcpy(static_cast<uint16_t *>(base) + at, h, 16);
    }
}

template <int XT>
__device__ __forceinline__ float rounded(float v)
{
    return XT == BREAD_QTYPE_F32 ? v : XT == BREAD_QTYPE_F16 ? h2f(f2h(v)) : bf2f(f2bf(v));
}

// The largest of 16 lanes, in all of them (by their bits, as magnitudes: a NaN is above all)
__device__ __forceinline__ uint64_t max16(uint64_t m)
{
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        const uint64_t o = (uint64_t)(uint32_t)__shfl_xor((int)(m >> 32), d) << 32 | (uint32_t)__shfl_xor((int)m, d);
        m = max(m, o);
    }
    return m;
}

__device__ __forceinline__ uint64_t magnitude(double v)
{
    return __builtin_bit_cast(uint64_t, v) & ~(1ull << 63);
}

// v cut to 21 bits, the last of them set if any bit was lost: rounds to a code as v does
__device__ __forceinline__ float cut(double v)
{
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return (float)__builtin_bit_cast(double, ((b >> 32) | min((uint32_t)b, 1u)) << 32);
}

// TPR threads a row (whole waves), 8 columns a thread and step, at most NV steps
template <int XT, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_fp8(const NormArgs a)
{
    constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, WPR = TPR / WAVE;
    __shared__ float part[WPR > 1 ? WPR : 1];
    const int t = (int)threadIdx.x % TPR, lane = (int)threadIdx.x % WAVE;
    const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
    if (RPB > 1 && row >= a.T) return;  // (whole waves; with one row a workgroup there is no such row)
    float v[NV][8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 8 * (i * TPR + t);
        if (c < a.n) {
            load8<XT>(a.x, row * a.xs + c, v[i]);
            if (a.res) {
                float r[8];
                load8<XT>(a.res, row * a.rs + c, r);
#pragma unroll
                for (int k = 0; k < 8; k++) v[i][k] = rounded<XT>(v[i][k] + r[k]);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) sum = fmaf(v[i][k], v[i][k], sum);
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[i][k] = 0.f;
        }
    }
    if (a.h) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = 8 * (i * TPR + t);
            if (c < a.n) store8(a.h, row * a.hs + c, XT, v[i]);
        }
    }
    auto row_sum = [&](float mine) __attribute__((always_inline)) {
        mine = wave_sum(mine);
        if constexpr (WPR > 1) {
            if (lane == 0) part[threadIdx.x / WAVE] = mine;
            __syncthreads();
            mine = 0.f;
#pragma unroll
            for (int i = 0; i < WPR; i++) mine += part[i];
        }
        return mine;
    };
    sum = row_sum(sum);
    float mean = sum / (float)a.n + a.eps;
    // Squares beyond fp32, or too small for it with an eps that is no larger: the row (all its threads see the same sum)
    // times a power of two.  (In a row of numbers beyond 2^56, those below 2^-54 lose bits by it, 2^-110 of the others.)
    if (__builtin_expect(sum == INFINITY || mean < 0x1p-100f, 0)) {
        const float p = sum == INFINITY ? 0x1p-72f : 0x1p100f;
        float again = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                v[i][k] *= p;
                again = fmaf(v[i][k], v[i][k], again);
            }
        if constexpr (WPR > 1) __syncthreads();  // all have read the first sum
        mean = row_sum(again) / (float)a.n + a.eps * p * p;
    }
    const float f = 1.0f / sqrtf(mean);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = 8 * (i * TPR + t);
        if (8 * i * TPR >= a.n) break;
        // Codes are of h weight / (its largest / 448), in which the rows' factor is not: that product is exact in 64 bits,
        // and so the codes are those of exact numbers.  (In 32 bits one code of some ten million is the next one, and
        // those 16384 rows take 63.5 us.)
        float w[8];
        uint64_t m = 0;
        if (c < a.n) {
            if (a.w) __builtin_memcpy(w, a.w + c, 32);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (!a.w) w[k] = 1.0f;
                m = max(m, magnitude((double)v[i][k] * w[k]));
            }
        }
        m = max16(m);
        if (c < a.n) {
            const double largest = __builtin_bit_cast(double, m) * f;
            const float s = f8_scale(f8_mag((float)largest));
            // (a NaN scale, also where only 32 bits overflow, makes every code NaN)
            const double r = s == s ? f / fmax(largest * (1.0 / 448.0), (double)F8_MIN_SCALE) : (double)s;
            float q[8];
#pragma unroll
            for (int k = 0; k < 8; k++) q[k] = cut((double)v[i][k] * w[k] * r);
            uint2 p;
            p.x = f8_pack4(q[0], q[1], q[2], q[3], 1.0f);
            p.y = f8_pack4(q[4], q[5], q[6], q[7], 1.0f);
            *reinterpret_cast<uint2 *>(a.codes + row * a.cs + c) = p;
            if (lane % 16 == 0) a.scales[row * a.ss + c / F8_BLOCK] = s;
            if (a.out) {
#pragma unroll
                for (int k = 0; k < 8; k++) v[i][k] = v[i][k] * f * w[k];
                store8(a.out, row * a.os + c, a.out_type, v[i]);
            }
        }
    }
}

template <int XT, int TPR, int NV>
int launch(const NormArgs &a, hipStream_t st)
{
    constexpr int threads = TPR < 256 ? 256 : TPR, rpb = threads / TPR;
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_norm_fp8<XT, TPR, NV>), dim3((unsigned)((a.T + rpb - 1) / rpb)), dim3(threads), 0, st, a);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

template <int XT>
int launch_norm(const NormArgs &a, hipStream_t st)
{
    if (a.n <= 2048) return launch<XT, 64, 4>(a, st);
    if (a.n <= 8192) return launch<XT, 256, 4>(a, st);
    return launch<XT, 1024, 4>(a, st);
}

}  // namespace

extern "C" int bread_rmsnorm_fp8(const bread_rmsnorm_fp8_t *args, bread_stream_t stream)
{
    BREAD_REQUIRE(args, BREAD_ERR_ARG, "NULL arguments");
    const bread_rmsnorm_fp8_t &o = *args;
    BREAD_REQUIRE(o.n > 0 && o.n_tokens >= 0, BREAD_ERR_ARG, "n must be > 0 and n_tokens >= 0");
    BREAD_REQUIRE(f8_wide_type(o.x_type) && (!o.normed || f8_wide_type(o.normed_type)), BREAD_ERR_QTYPE,
                  "x_type and normed_type must be 0 (F32), 1 (F16) or 30 (BF16)");
    BREAD_REQUIRE(o.n % 16 == 0 && o.n <= 32768, BREAD_ERR_SHAPE, "n must be a multiple of 16, at most 32768");
    // (a launch holds fewer than 2^32 threads, of which a long row takes 1024)
    BREAD_REQUIRE(o.n_tokens < 1 << 22, BREAD_ERR_SHAPE, "n_tokens of 2^22 or more");
    const int64_t nb = f8_blocks(o.n);
    const int64_t xs = o.x_stride ? o.x_stride : o.n, rs = o.residual_stride ? o.residual_stride : o.n;
    const int64_t hs = o.hidden_stride ? o.hidden_stride : o.n, cs = o.codes_stride ? o.codes_stride : o.n;
    const int64_t ss = o.scales_stride ? o.scales_stride : nb, os = o.normed_stride ? o.normed_stride : o.n;
    BREAD_REQUIRE(xs >= o.n && rs >= o.n && hs >= o.n && cs >= o.n && ss >= nb && os >= o.n, BREAD_ERR_SHAPE,
                  "a stride is smaller than a row");
    if (o.n_tokens == 0) return BREAD_OK;
    // (with another stride a row of hidden would lie on rows that others have yet to read)
    BREAD_REQUIRE(o.n_tokens == 1 || !o.hidden || ((o.hidden != o.x || hs == xs) && (o.hidden != o.residual || hs == rs)),
                  BREAD_ERR_ARG, "hidden in place of x or residual needs its stride");
    BREAD_REQUIRE(o.x && o.codes && o.scales, BREAD_ERR_ARG, "NULL pointer");
    BREAD_REQUIRE(((uintptr_t)o.codes & 15) == 0 && cs % 16 == 0, BREAD_ERR_ALIGN,
                  "codes must be 16-byte aligned and their stride a multiple of 16");
    const uintptr_t xa = f8_type_bytes(o.x_type) - 1, oa = f8_type_bytes(o.normed_type) - 1;
    BREAD_REQUIRE((((uintptr_t)o.x | (uintptr_t)o.residual | (uintptr_t)o.hidden) & xa) == 0 &&
                      (!o.normed || ((uintptr_t)o.normed & oa) == 0) &&
                      (((uintptr_t)o.weight | (uintptr_t)o.scales) & 3) == 0,
                  BREAD_ERR_ALIGN, "tensors must be aligned to their elements");
    NormArgs a;
    a.x = o.x;
    a.res = o.residual;
    a.h = o.hidden;
    a.out = o.normed;
    a.w = o.weight;
    a.codes = o.codes;
    a.scales = o.scales;
    a.xs = xs;
    a.rs = rs;
    a.hs = hs;
    a.cs = cs;
    a.ss = ss;
    a.os = os;
    a.eps = o.eps;
    a.n = o.n;
    a.T = o.n_tokens;
    a.out_type = o.normed_type;
    const hipStream_t st = to_hip(stream);
    switch (o.x_type) {
    case BREAD_QTYPE_F32: return launch_norm<BREAD_QTYPE_F32>(a, st);
    case BREAD_QTYPE_F16: return launch_norm<BREAD_QTYPE_F16>(a, st);
    default: return launch_norm<BREAD_QTYPE_BF16>(a, st);
    }
}
