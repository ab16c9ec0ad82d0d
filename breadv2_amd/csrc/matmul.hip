// matmul.hip — bread_matmul: several tokens through one weight matrix, with
// bias, activation and residual in the epilogue:
//   y[t][r] = act(sum_c W[r][c] x[t][c] + bias[r]) + residual[t][r].
// W is Q4_K, Q6_K, Q8_0 or fp16, x fp16, sums fp32, y fp16 or fp32.  The
// reference runs one bread_matvec (kernels.cu:289) per token.
//
// k_mm_rows: a workgroup takes 16 weight rows at a time against up to 64
// tokens; its waves split the columns 256 at a time and join their sums in
// LDS.  Weights go from memory to registers once, as integers that fp16 holds
// exactly (a block's scale is applied to the fp32 sum): the products are exact.
#include "bread_internal.h"
#include "q4k_mfma.h"

namespace {

typedef q4m_half8 h8;
typedef q4m_half2 h2;
typedef q4m_f32x4 f32x4;

struct MmArgs {
    const uint8_t *w;
    const uint16_t *x;
    void *y;
    const float *bias;
    const void *res;
    int64_t xs, ys;  // elements from one token to the next
    uint64_t rb;     // bytes of a weight row
    int rows, cols, T, act, y32;
};

// ---------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------

__device__ __forceinline__ float activate(float v, int act)
{
    switch (act) {
    case BREAD_ACT_SILU: return v / (1.0f + expf(-v));
    case BREAD_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    case BREAD_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.79788456080286536f * (v + 0.044715f * v * v * v)));
    case BREAD_ACT_RELU: return v < 0.f ? 0.f : v;  // NaN stays NaN
    }
    return v;
}

__device__ __forceinline__ void put(const MmArgs &a, int t, int r, float v)
{
    if (a.bias) v += a.bias[r];
    v = activate(v, a.act);
    const size_t o = (size_t)t * a.ys + r;
    if (a.y32) {
        if (a.res) v += static_cast<const float *>(a.res)[o];
        static_cast<float *>(a.y)[o] = v;
    } else {
        if (a.res) v += h2f(static_cast<const uint16_t *>(a.res)[o]);
        static_cast<uint16_t *>(a.y)[o] = f2h(v);
    }
}

// ---------------------------------------------------------------------------
// 256 columns of a weight row as a lane holds them
// ---------------------------------------------------------------------------
// v_mfma_f32_16x16x32_f16: lane l holds row (or token) l % 16 and eight
// consecutive k of the group g = l / 16.  The columns that the eight MFMAs of a
// chunk take from each group are free as long as weights and activations agree:
// each format's order is the one that its bytes unpack in.

// 16 or 8 bytes at a 2-byte aligned address (one load)
__device__ __forceinline__ uint4 ldu16(const uint8_t *p)
{
    uint4 v;
    __builtin_memcpy(&v, reinterpret_cast<const uint16_t *>(p), 16);
    return v;
}

__device__ __forceinline__ uint2 ldu8(const uint8_t *p)
{
    uint2 v;
    __builtin_memcpy(&v, reinterpret_cast<const uint16_t *>(p), 8);
    return v;
}

__device__ __forceinline__ uint32_t ldu2(const uint8_t *p)
{
    return *reinterpret_cast<const uint16_t *>(p);
}

__device__ __forceinline__ uint32_t word(const uint4 &v, int i)
{
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Four bytes below 256 as two packed fp16 pairs of 1024 + byte
__device__ __forceinline__ h2 magic_lo(uint32_t v)
{
    return __builtin_bit_cast(h2, __builtin_amdgcn_perm(Q4M_MAGIC, v, 0x07010700u));
}

__device__ __forceinline__ h2 magic_hi(uint32_t v)
{
    return __builtin_bit_cast(h2, __builtin_amdgcn_perm(Q4M_MAGIC, v, 0x07030702u));
}

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d)
{
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ h2 both(float v)
{
    const _Float16 h = (_Float16)v;
    return h2{h, h};
}

template <int QT> struct Raw;

template <> struct Raw<BREAD_QTYPE_Q4_K> {
    Q4mRaw q;
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int)
    {
        q4m_load(q, row + (size_t)ch * Q4K_BYTES, g);
    }
};

template <> struct Raw<BREAD_QTYPE_Q6_K> {
    uint4 l0, l1, qh;
    uint2 sc;
    uint32_t d;
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int)
    {
        const uint8_t *b = row + (size_t)ch * Q6K_BYTES;
        const int h = g >> 1, o = 16 * (g & 1);
        l0 = ldu16(b + 64 * h + o);
        l1 = ldu16(b + 64 * h + 32 + o);
        qh = ldu16(b + 128 + 32 * h + o);
        sc = ldu8(b + 192 + 8 * h);
        d = ldu2(b + 208);
    }
};

template <> struct Raw<BREAD_QTYPE_Q8_0> {
    uint2 q[8];
    uint32_t d[8];
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int cols)
    {
        const int n = cols / Q80_ELEMS - 8 * ch;  // blocks left in the row: at least one
        const uint8_t *b = row + (size_t)ch * (8 * Q80_BYTES);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint8_t *p = b + (i < n ? i : 0) * Q80_BYTES;
            q[i] = ldu8(p + 2 + 8 * g);
            d[i] = i < n ? ldu2(p) : 0u;
        }
    }
};

template <> struct Raw<BREAD_QTYPE_F16> {
    uint4 q[8];
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int cols)
    {
        const int c0 = 256 * ch + 64 * g;
#pragma unroll
        for (int i = 0; i < 8; i++)
            q[i] = c0 + 8 * i < cols ? *reinterpret_cast<const uint4 *>(row + 2 * (size_t)(c0 + 8 * i))
                                     : make_uint4(0u, 0u, 0u, 0u);
    }
};

// Column (inside the chunk) of the first of the eight that MFMA i takes from group g
template <int QT>
__device__ __forceinline__ int column(int g, int i)
{
    if (QT == BREAD_QTYPE_Q6_K) return 128 * (g >> 1) + 32 * (i >> 1) + 16 * (g & 1) + 8 * (i & 1);
    if (QT == BREAD_QTYPE_Q8_0) return 32 * i + 8 * g;
    return 64 * g + 8 * i;
}

// Token row's activations for the chunk (zeros where there are no columns)
template <int QT>
__device__ __forceinline__ void load_x(uint4 (&xf)[8], const uint16_t *xt, int ch, int g, int cols)
{
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int c = 256 * ch + column<QT>(g, i);
        xf[i] = c < cols ? *reinterpret_cast<const uint4 *>(xt + c) : make_uint4(0u, 0u, 0u, 0u);
    }
}

__device__ __forceinline__ f32x4 mfma(const uint4 &x, h8 w, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), w, c, 0, 0, 0);
}

// Sum of eight fp16 values on top of s
__device__ __forceinline__ float sum_h8(const uint4 &v, float s)
{
    const h2 one{(_Float16)1.f, (_Float16)1.f};
    s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.x), one, s, false);
    s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.y), one, s, false);
    s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.z), one, s, false);
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.w), one, s, false);
}

// out[tt] += the chunk's products, tokens 16 tt + 4 g + i of weight row l % 16 in out[tt][i].
// EXACT (Q6_K): the integers sc q above 2048 that fp16 would round, by at most 2^-12 of themselves and only
// for the largest scales, are kept exact as sc (q with its low bit cleared) + sc (low bit), at twice the
// MFMAs: for fp32 results.  An fp16 result has itself half a step of 2^-11.
template <int QT, int NTT, bool EXACT>
__device__ __forceinline__ void chunk_mma(const Raw<QT> &r, const uint4 (&xf)[NTT][8], f32x4 (&out)[NTT], int g)
{
    if constexpr (QT == BREAD_QTYPE_Q4_K) {
        const Q4mRaw &b = r.q;
        const float d = h2f(b.head.x & 0xFFFFu), dmin = h2f(b.head.x >> 16);
        uint32_t sc0, m0, sc1, m1;
        scale_min_k4(2 * g, b.head.y, b.head.z, b.head.w, sc0, m0);
        scale_min_k4(2 * g + 1, b.head.y, b.head.z, b.head.w, sc1, m1);
        const h2 S0 = both((float)sc0), N0 = both(-1024.f * (float)sc0);
        const h2 S1 = both((float)sc1), N1 = both(-1024.f * (float)sc1);
        const h8 bq[8] = {q4m_b8(b.q0.x, b.q0.y, 0, S0, N0), q4m_b8(b.q0.z, b.q0.w, 0, S0, N0),
                          q4m_b8(b.q1.x, b.q1.y, 0, S0, N0), q4m_b8(b.q1.z, b.q1.w, 0, S0, N0),
                          q4m_b8(b.q0.x, b.q0.y, 1, S1, N1), q4m_b8(b.q0.z, b.q0.w, 1, S1, N1),
                          q4m_b8(b.q1.x, b.q1.y, 1, S1, N1), q4m_b8(b.q1.z, b.q1.w, 1, S1, N1)};
#pragma unroll
        for (int tt = 0; tt < NTT; tt++) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f}, accm = {0.f, 0.f, 0.f, 0.f};
            float x0 = 0.f, x1 = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                acc = mfma(xf[tt][i], bq[i], acc);
                if (i < 4) x0 = sum_h8(xf[tt][i], x0);
                else x1 = sum_h8(xf[tt][i], x1);
            }
            accm = __builtin_amdgcn_mfma_f32_16x16x4f32(x0, (float)m0, accm, 0, 0, 0);
            accm = __builtin_amdgcn_mfma_f32_16x16x4f32(x1, (float)m1, accm, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) out[tt][i] += d * acc[i] - dmin * accm[i];
        }
    } else if constexpr (QT == BREAD_QTYPE_Q6_K) {
        const float d = h2f(r.d);
        f32x4 acc[NTT];
#pragma unroll
        for (int tt = 0; tt < NTT; tt++) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        const h2 off = both(-1056.f), one = both(-1024.f);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int qd = i >> 1, k = 2 * (i & 1);
            const uint4 &lw = (qd & 1) ? r.l1 : r.l0;
            const uint32_t sb = (qd < 2 ? r.sc.x : r.sc.y) >> (16 * (qd & 1) + 8 * (g & 1));
            const h2 S = both((float)(int8_t)(sb & 0xFFu));
            uint32_t v0 = (word(lw, k) >> (4 * (qd >> 1))) & 0x0F0F0F0Fu, v1 = (word(lw, k + 1) >> (4 * (qd >> 1))) & 0x0F0F0F0Fu;
            v0 |= ((word(r.qh, k) >> (2 * qd)) & 0x03030303u) << 4;
            v1 |= ((word(r.qh, k + 1) >> (2 * qd)) & 0x03030303u) << 4;
            if constexpr (EXACT) {
                const uint32_t a0 = v0 & 0x3E3E3E3Eu, a1 = v1 & 0x3E3E3E3Eu;
                const uint32_t b0 = v0 & 0x01010101u, b1 = v1 & 0x01010101u;
                const h8 hi = join((magic_lo(a0) + off) * S, (magic_hi(a0) + off) * S, (magic_lo(a1) + off) * S,
                                   (magic_hi(a1) + off) * S);
                const h8 lo = join((magic_lo(b0) + one) * S, (magic_hi(b0) + one) * S, (magic_lo(b1) + one) * S,
                                   (magic_hi(b1) + one) * S);
#pragma unroll
                for (int tt = 0; tt < NTT; tt++) {
                    acc[tt] = mfma(xf[tt][i], hi, acc[tt]);
                    acc[tt] = mfma(xf[tt][i], lo, acc[tt]);
                }
            } else {
                const h8 w = join((magic_lo(v0) + off) * S, (magic_hi(v0) + off) * S, (magic_lo(v1) + off) * S,
                                  (magic_hi(v1) + off) * S);
#pragma unroll
                for (int tt = 0; tt < NTT; tt++) acc[tt] = mfma(xf[tt][i], w, acc[tt]);
            }
        }
#pragma unroll
        for (int tt = 0; tt < NTT; tt++)
#pragma unroll
            for (int i = 0; i < 4; i++) out[tt][i] += d * acc[tt][i];
    } else if constexpr (QT == BREAD_QTYPE_Q8_0) {
        const h2 off = both(-1152.f);  // 1024 + (q + 128) - 1152
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t v0 = r.q[i].x ^ 0x80808080u, v1 = r.q[i].y ^ 0x80808080u;
            const h8 w = join(magic_lo(v0) + off, magic_hi(v0) + off, magic_lo(v1) + off, magic_hi(v1) + off);
            const float d = h2f(r.d[i]);
#pragma unroll
            for (int tt = 0; tt < NTT; tt++) {
                const f32x4 p = mfma(xf[tt][i], w, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int j = 0; j < 4; j++) out[tt][j] += d * p[j];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int tt = 0; tt < NTT; tt++) out[tt] = mfma(xf[tt][i], __builtin_bit_cast(h8, r.q[i]), out[tt]);
    }
}

// ---------------------------------------------------------------------------
// 16 rows a workgroup at a time
// ---------------------------------------------------------------------------
constexpr int MR_WAVES = 8;
constexpr int MR_THREADS = MR_WAVES * WAVE;
constexpr int MR_MAXTT = 4;  // 16-token tiles a workgroup

// Workgroup b takes row tiles b / ny, b / ny + stride, ... against token tiles
// [yb NTT, yb NTT + NTT), yb = b % ny.  Wave v owns the chunks v, v + 8, ... of every row.
template <int QT, int NTT, bool EXACT>
__global__ __launch_bounds__(MR_THREADS) void k_mm_rows(const MmArgs a, int ny, int stride)
{
    __shared__ float part[2][MR_WAVES][NTT * 16][17];
    const int wv = wave_id(), l = lane_id(), g = l >> 4, c = l & 15;
    const int yb = (int)blockIdx.x % ny, t0 = yb * NTT * 16;
    const int nch = (a.cols + 255) / 256, ntile = (a.rows + 15) / 16;
    const int nw = nch < MR_WAVES ? nch : MR_WAVES;  // waves with columns
    const uint16_t *xt[NTT];
#pragma unroll
    for (int tt = 0; tt < NTT; tt++) {
        const int t = t0 + 16 * tt + c;  // beyond the last token: the last one again, not stored
        xt[tt] = a.x + (size_t)(t < a.T ? t : a.T - 1) * a.xs;
    }
    int buf = 0;
    for (int ti = (int)blockIdx.x / ny; ti < ntile; ti += stride, buf ^= 1) {
        const int r = 16 * ti + c;
        const uint8_t *row = a.w + (size_t)(r < a.rows ? r : a.rows - 1) * a.rb;
        f32x4 out[NTT];
#pragma unroll
        for (int tt = 0; tt < NTT; tt++) out[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int ch = wv; ch < nch; ch += MR_WAVES) {
            Raw<QT> raw;
            raw.load(row, ch, g, a.cols);
            uint4 xf[NTT][8];
#pragma unroll
            for (int tt = 0; tt < NTT; tt++) load_x<QT>(xf[tt], xt[tt], ch, g, a.cols);
            chunk_mma<QT, NTT, EXACT>(raw, xf, out, g);
        }
        if (wv < nw) {
#pragma unroll
            for (int tt = 0; tt < NTT; tt++)
#pragma unroll
                for (int i = 0; i < 4; i++) part[buf][wv][16 * tt + 4 * g + i][c] = out[tt][i];
        }
        q4m_bar();
        for (int o = threadIdx.x; o < NTT * 256; o += MR_THREADS) {
            const int t = t0 + (o >> 4), rr = 16 * ti + (o & 15);
            if (t < a.T && rr < a.rows) {
                float v = 0.f;
                for (int k = 0; k < nw; k++) v += part[buf][k][o >> 4][o & 15];
                put(a, t, rr, v);
            }
        }
    }
}

template <int QT, bool EXACT>
int launch_rows(const MmArgs &a, hipStream_t st)
{
    const int tt = (a.T + 15) / 16, ny = (tt + MR_MAXTT - 1) / MR_MAXTT, ntt = (tt + ny - 1) / ny;
    const int64_t ntile = ((int64_t)a.rows + 15) / 16;
    int64_t stride = 512 / ny;
    if (stride < 1) stride = 1;
    if (stride > ntile) stride = ntile;
    const dim3 grid((unsigned)(stride * ny)), block(MR_THREADS);
    bread_clear_stale_error();
    switch (ntt) {
    case 1: hipLaunchKernelGGL((k_mm_rows<QT, 1, EXACT>), grid, block, 0, st, a, ny, (int)stride); break;
    case 2: hipLaunchKernelGGL((k_mm_rows<QT, 2, EXACT>), grid, block, 0, st, a, ny, (int)stride); break;
    case 3: hipLaunchKernelGGL((k_mm_rows<QT, 3, EXACT>), grid, block, 0, st, a, ny, (int)stride); break;
    default: hipLaunchKernelGGL((k_mm_rows<QT, 4, EXACT>), grid, block, 0, st, a, ny, (int)stride); break;
    }
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

}  // namespace

extern "C" int bread_matmul(const void *w, const uint16_t *x, void *y, int rows, int cols, int qtype, int n_tokens,
                            const bread_matmul_opts_t *opts, bread_stream_t stream)
{
    static const bread_matmul_opts_t plain = {nullptr, nullptr, BREAD_ACT_NONE, BREAD_QTYPE_F16, 0, 0};
    const bread_matmul_opts_t &o = opts ? *opts : plain;
    BREAD_REQUIRE(rows >= 0 && cols > 0 && n_tokens >= 0, BREAD_ERR_ARG,
                  "rows and n_tokens must be >= 0 and cols > 0");
    BREAD_REQUIRE(qtype == BREAD_QTYPE_Q4_K || qtype == BREAD_QTYPE_Q6_K || qtype == BREAD_QTYPE_Q8_0 ||
                      qtype == BREAD_QTYPE_F16,
                  BREAD_ERR_QTYPE, "qtype must be 12 (Q4_K), 14 (Q6_K), 8 (Q8_0) or 1 (F16)");
    BREAD_REQUIRE(o.act >= BREAD_ACT_NONE && o.act <= BREAD_ACT_RELU, BREAD_ERR_ARG, "unknown activation");
    BREAD_REQUIRE(o.y_type == BREAD_QTYPE_F16 || o.y_type == BREAD_QTYPE_F32, BREAD_ERR_QTYPE,
                  "y_type must be 1 (F16) or 0 (F32)");
    const int unit = qtype == BREAD_QTYPE_Q8_0 ? Q80_ELEMS : qtype == BREAD_QTYPE_F16 ? 8 : QK;
    BREAD_REQUIRE(cols % unit == 0, BREAD_ERR_SHAPE,
                  "cols must be a multiple of the block size (256, Q8_0: 32, F16: 8)");
    const int64_t xs = o.x_stride ? o.x_stride : cols, ys = o.y_stride ? o.y_stride : rows;
    BREAD_REQUIRE(xs >= cols && ys >= rows, BREAD_ERR_SHAPE, "a stride is smaller than a token's row");
    if (rows == 0 || n_tokens == 0) return BREAD_OK;
    BREAD_REQUIRE(w && x && y, BREAD_ERR_ARG, "NULL pointer");
    BREAD_REQUIRE(((uintptr_t)w & (qtype == BREAD_QTYPE_Q4_K || qtype == BREAD_QTYPE_F16 ? 15 : 3)) == 0,
                  BREAD_ERR_ALIGN, "w must be 16-byte aligned (Q6_K and Q8_0: 4-byte)");
    BREAD_REQUIRE(((uintptr_t)x & 15) == 0 && xs % 8 == 0, BREAD_ERR_ALIGN,
                  "x must be 16-byte aligned and its stride a multiple of 8");
    const uintptr_t ya = o.y_type == BREAD_QTYPE_F32 ? 3 : 1;
    BREAD_REQUIRE((((uintptr_t)y | (uintptr_t)o.residual) & ya) == 0 && ((uintptr_t)o.bias & 3) == 0, BREAD_ERR_ALIGN,
                  "y, residual and bias must be aligned to their elements");
    MmArgs a;
    a.w = static_cast<const uint8_t *>(w);
    a.x = x;
    a.y = y;
    a.bias = o.bias;
    a.res = o.residual;
    a.xs = xs;
    a.ys = ys;
    a.rb = qtype == BREAD_QTYPE_Q4_K   ? (uint64_t)(cols / QK) * Q4K_BYTES
           : qtype == BREAD_QTYPE_Q6_K ? (uint64_t)(cols / QK) * Q6K_BYTES
           : qtype == BREAD_QTYPE_Q8_0 ? (uint64_t)(cols / Q80_ELEMS) * Q80_BYTES
                                       : (uint64_t)cols * 2;
    a.rows = rows;
    a.cols = cols;
    a.T = n_tokens;
    a.act = o.act;
    a.y32 = o.y_type == BREAD_QTYPE_F32;
    const hipStream_t st = to_hip(stream);
    switch (qtype) {
    case BREAD_QTYPE_Q4_K: return launch_rows<BREAD_QTYPE_Q4_K, false>(a, st);
    case BREAD_QTYPE_Q6_K:
        return a.y32 ? launch_rows<BREAD_QTYPE_Q6_K, true>(a, st) : launch_rows<BREAD_QTYPE_Q6_K, false>(a, st);
    case BREAD_QTYPE_Q8_0: return launch_rows<BREAD_QTYPE_Q8_0, false>(a, st);
    default: return launch_rows<BREAD_QTYPE_F16, false>(a, st);
    }
}
