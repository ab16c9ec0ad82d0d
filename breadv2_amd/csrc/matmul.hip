// matmul.hip — bread_matmul: several tokens through one weight matrix, with
// bias, activation and residual in the epilogue:
//   y[t][r] = act(sum_c W[r][c] x[t][c] + bias[r]) + residual[t][r].
// W is Q4_K, Q6_K, Q8_0 or fp16, x fp16, sums fp32, y fp16 or fp32.  The
// reference runs one bread_matvec (kernels.cu:289) per token.
//
// Weights are unpacked to integers that fp16 holds exactly, and a block's scale
// is applied to the fp32 sum: the products are exact.  k_mm_rows is for a few
// tokens (16 weight rows a workgroup at a time, the columns split over its
// waves), k_mm_tile for more (tiles of tokens by weight rows).
#include "activate.h"
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

// Four consecutive rows of a token (y is aligned to an element only)
__device__ __forceinline__ void put4(const MmArgs &a, int t, int r, const float (&in)[4])
{
    if (r + 4 > a.rows) {
        for (int k = 0; k < 4 && r + k < a.rows; k++) put(a, t, r + k, k == 0 ? in[0] : k == 1 ? in[1] : k == 2 ? in[2] : in[3]);
        return;
    }
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = activate(a.bias ? in[k] + a.bias[r + k] : in[k], a.act);
    const size_t o = (size_t)t * a.ys + r;
    if (a.y32) {
        float *y = static_cast<float *>(a.y) + o;
        if (a.res) {
            float x[4];
            __builtin_memcpy(x, static_cast<const float *>(a.res) + o, 16);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] += x[k];
        }
        __builtin_memcpy(y, v, 16);
    } else {
        uint16_t *y = static_cast<uint16_t *>(a.y) + o, h[4];
        if (a.res) {
            __builtin_memcpy(h, static_cast<const uint16_t *>(a.res) + o, 8);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] += h2f(h[k]);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) h[k] = f2h(v[k]);
        __builtin_memcpy(y, h, 8);
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

__device__ __forceinline__ uint32_t ldu4(const uint8_t *p)
{
    uint32_t v;
    __builtin_memcpy(&v, reinterpret_cast<const uint16_t *>(p), 4);
    return v;
}

// r[i] of the lanes of row j (16 lanes) for r[j] of the lanes of row i
__device__ __forceinline__ void transpose4(uint32_t (&r)[4])
{
    auto swap = [](uint32_t &a, uint32_t &b, bool wide) __attribute__((always_inline)) {
        const auto p = wide ? __builtin_amdgcn_permlane32_swap(a, b, false, false)
                            : __builtin_amdgcn_permlane16_swap(a, b, false, false);
        a = p[0];
        b = p[1];
    };
    swap(r[0], r[2], true);
    swap(r[1], r[3], true);
    swap(r[0], r[1], false);
    swap(r[2], r[3], false);
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

// The eight scales of a lane's half and d in one load: even lanes of a row load the scales, odd ones the eight bytes
// that end with d, and each takes the other's.
template <> struct Raw<BREAD_QTYPE_Q6_K> {
    uint4 l0, l1, qh;
    uint2 s;
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int)
    {
        const uint8_t *b = row + (size_t)ch * Q6K_BYTES;
        const int h = g >> 1, o = 16 * (g & 1);
        l0 = ldu16(b + 64 * h + o);
        l1 = ldu16(b + 64 * h + 32 + o);
        qh = ldu16(b + 128 + 32 * h + o);
        s = ldu8(b + ((g & 1) ? 202 : 192 + 8 * h));
    }
};

// Lane g loads the whole blocks 2 g and 2 g + 1, 68 bytes in five loads; the eight values of every block that it
// multiplies come from the other lanes of its row (spread).  A load for each block's eight bytes and each scale
// would be 16, at a cycle a lane each: 9 tokens by 100000 x 2048 took 122 us so, 57 now; by 2048 x 4096 14.3 and 7.9.
template <> struct Raw<BREAD_QTYPE_Q8_0> {
    uint32_t v[17];
    __device__ __forceinline__ void load(const uint8_t *row, int ch, int g, int cols)
    {
        const int n = min(cols / Q80_ELEMS - 8 * ch - 2 * g, 2);  // blocks of the two that the row has
        const uint8_t *b = row + (size_t)ch * (8 * Q80_BYTES) + 2 * Q80_BYTES * g;
        uint4 p[4] = {};
        uint32_t t = 0u;
        if (n >= 1) {
            p[0] = ldu16(b);
            p[1] = ldu16(b + 16);
            if (n == 1) p[2].x = ldu2(b + 32);
        }
        if (n >= 2) {
            p[2] = ldu16(b + 32);
            p[3] = ldu16(b + 48);
            t = ldu4(b + 64);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = word(p[i / 4], i & 3);
        v[16] = t;
    }
    // q[i]: the eight values 8 g .. of block 2 i + odd
    __device__ __forceinline__ void spread(int odd, uint2 (&q)[4]) const
    {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            lo[j] = odd ? v[9 + 2 * j] : __builtin_amdgcn_alignbyte(v[2 * j + 1], v[2 * j], 2);
            hi[j] = odd ? v[10 + 2 * j] : __builtin_amdgcn_alignbyte(v[2 * j + 2], v[2 * j + 1], 2);
        }
        transpose4(lo);
        transpose4(hi);
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = make_uint2(lo[i], hi[i]);
    }
    // d[i]: the scales of blocks 2 i and 2 i + 1 in its halves
    __device__ __forceinline__ void scales(uint32_t (&d)[4]) const
    {
#pragma unroll
        for (int j = 0; j < 4; j++) d[j] = (v[0] & 0xFFFFu) | (v[8] & 0xFFFF0000u);
        transpose4(d);
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

// A dot product's result needs three wait states before a matrix instruction reads it; the compiler leaves none
// between the two (it does before other vector instructions), and the last product is then missing.
__device__ __forceinline__ void dot_to_mfma(float &x)
{
    asm volatile("s_nop 3" : "+v"(x));
}

// out[tt] += the chunk's products, tokens 16 tt + 4 g + i of weight row l % 16 in out[tt][i].
// Q6_K: the integers sc q, up to 4096, do not fit fp16's 11 bits, and the scales of trained weights reach -128 in
// every superblock; they are multiplied as sc (q with its low bit cleared) + sc (low bit), both exact, at twice
// the MFMAs.  us on MI355X with the integers rounded to 11 bits and with both parts, tokens by weights, fp16 results:
// 9 by 248320 x 2048 102 and 113, 64 by 2048 x 4096 12.2 and 13.1, 509 by 2048 x 4096 25.7 and 30.2, 2048 by
// 8192 x 2048 104 and 139.
template <int QT, int NTT>
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
        auto operands = [&](int j, h8(&q)[4]) __attribute__((always_inline)) {
            const h2 S = j ? S1 : S0, N = j ? N1 : N0;
            q[0] = q4m_b8(b.q0.x, b.q0.y, j, S, N);
            q[1] = q4m_b8(b.q0.z, b.q0.w, j, S, N);
            q[2] = q4m_b8(b.q1.x, b.q1.y, j, S, N);
            q[3] = q4m_b8(b.q1.z, b.q1.w, j, S, N);
        };
        auto products = [&](int tt, int j, const h8(&q)[4], f32x4 &acc, f32x4 &accm) __attribute__((always_inline)) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                acc = mfma(xf[tt][4 * j + i], q[i], acc);
                x = sum_h8(xf[tt][4 * j + i], x);
            }
            dot_to_mfma(x);
            accm = __builtin_amdgcn_mfma_f32_16x16x4f32(x, (float)(j ? m1 : m0), accm, 0, 0, 0);
        };
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        if constexpr (NTT == 1) {
            // a sub-block's operands at a time: 16 registers less, for the second chunk that is held
            f32x4 acc = zero, accm = zero;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                h8 q[4];
                operands(j, q);
                products(0, j, q, acc, accm);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) out[0][i] += d * acc[i] - dmin * accm[i];
        } else {
            h8 q0[4], q1[4];
            operands(0, q0);
            operands(1, q1);
#pragma unroll
            for (int tt = 0; tt < NTT; tt++) {
                f32x4 acc = zero, accm = zero;
                products(tt, 0, q0, acc, accm);
                products(tt, 1, q1, acc, accm);
#pragma unroll
                for (int i = 0; i < 4; i++) out[tt][i] += d * acc[i] - dmin * accm[i];
            }
        }
    } else if constexpr (QT == BREAD_QTYPE_Q6_K) {
        const lane_pair top = swap16(r.s.y);
        const uint2 sc = make_uint2(swap16(r.s.x).a, top.a);
        const float d = h2f(top.b >> 16);
        f32x4 acc[NTT];
#pragma unroll
        for (int tt = 0; tt < NTT; tt++) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        const h2 off = both(-1056.f), one = both(-1024.f);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int qd = i >> 1, k = 2 * (i & 1);
            const uint4 &lw = (qd & 1) ? r.l1 : r.l0;
            const uint32_t sb = (qd < 2 ? sc.x : sc.y) >> (16 * (qd & 1) + 8 * (g & 1));
            const h2 S = both((float)(int8_t)(sb & 0xFFu));
            uint32_t v0 = (word(lw, k) >> (4 * (qd >> 1))) & 0x0F0F0F0Fu, v1 = (word(lw, k + 1) >> (4 * (qd >> 1))) & 0x0F0F0F0Fu;
            v0 |= ((word(r.qh, k) >> (2 * qd)) & 0x03030303u) << 4;
            v1 |= ((word(r.qh, k + 1) >> (2 * qd)) & 0x03030303u) << 4;
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
        }
#pragma unroll
        for (int tt = 0; tt < NTT; tt++)
#pragma unroll
            for (int i = 0; i < 4; i++) out[tt][i] += d * acc[tt][i];
    } else if constexpr (QT == BREAD_QTYPE_Q8_0) {
        const h2 off = both(-1152.f);  // 1024 + (q + 128) - 1152
        uint32_t dd[4];
        r.scales(dd);
#pragma unroll
        for (int odd = 0; odd < 2; odd++) {
            uint2 q[4];
            r.spread(odd, q);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t v0 = q[i].x ^ 0x80808080u, v1 = q[i].y ^ 0x80808080u;
                const h8 w = join(magic_lo(v0) + off, magic_hi(v0) + off, magic_lo(v1) + off, magic_hi(v1) + off);
                const float d = h2f(odd ? dd[i] >> 16 : dd[i] & 0xFFFFu);
#pragma unroll
                for (int tt = 0; tt < NTT; tt++) {
                    const f32x4 p = mfma(xf[tt][2 * i + odd], w, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int j = 0; j < 4; j++) out[tt][j] += d * p[j];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
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
// HOLD: a row has no more chunks than waves (1) or twice as many (2), and a wave keeps its activations in registers
// for all its row tiles (reading them again for every tile took the vocabulary's logits from 111 to 167 us) and loads
// the next weights while it works on one chunk.  Two workgroups a CU, so at most 128 registers (20 tokens, Q4_K: 105 us with
// one, 89 with two); fp16 rows for 17 to 32 tokens would not fit them (117 us, spilled 285).  Two chunks held spill 15
// registers for Q4_K and 3 for Q6_K, 17 to 32 tokens of Q4_K 1.
// MI355X, 9 tokens: 248320 x 2048 Q6_K 112 to 115 us (3.7 TB/s), Q4_K 66 to 76 us (4 TB/s), 8192 x 2048 Q4_K 7.1 us.  Bound by
// the loads: a lane's load from a row of its own costs the address unit a cycle, four loads and 64 lanes a chunk of
// Q6_K.  Rows brought through LDS in the order they lie in took as long (110 us; 91 without the products), and so did
// registers in turn for the weights on their way.
template <int QT, int NTT, int HOLD>
__global__ __launch_bounds__(MR_THREADS, HOLD == 0 || QT == BREAD_QTYPE_F16 || (HOLD > 1 && QT == BREAD_QTYPE_Q8_0) ? 2 : 4) void k_mm_rows(const MmArgs a, int ny, int stride)
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
    constexpr int SETS = HOLD > 1 ? HOLD : 1;
    uint4 xf[SETS][NTT][8];
    Raw<QT> raw;
    int ti = (int)blockIdx.x / ny, buf = 0;
    auto row_of = [&](int tile) __attribute__((always_inline)) {  // (past the last row: the last one again, not stored)
        const int r = 16 * tile + c;
        return a.w + (size_t)(r < a.rows ? r : a.rows - 1) * a.rb;
    };
    const bool two = HOLD > 1 && wv + MR_WAVES < nch;  // a second chunk for this wave
    if (HOLD > 0 && wv < nw) {
        raw.load(row_of(ti), wv, g, a.cols);
#pragma unroll
        for (int k = 0; k < SETS; k++)
#pragma unroll
            for (int tt = 0; tt < NTT; tt++) load_x<QT>(xf[k][tt], xt[tt], wv + MR_WAVES * k, g, a.cols);
    }
    for (; ti < ntile; ti += stride, buf ^= 1) {
        f32x4 out[NTT];
#pragma unroll
        for (int tt = 0; tt < NTT; tt++) out[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (HOLD > 1) {
            Raw<QT> second;
            // (the two chunks are kept apart: together they run out of registers)
            if (two) second.load(row_of(ti), wv + MR_WAVES, g, a.cols);
            __builtin_amdgcn_sched_barrier(0);
            if (wv < nw) {
                chunk_mma<QT, NTT>(raw, xf[0], out, g);
                __builtin_amdgcn_sched_barrier(0);
                if (ti + stride < ntile) raw.load(row_of(ti + stride), wv, g, a.cols);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (two) chunk_mma<QT, NTT>(second, xf[1], out, g);
        } else if constexpr (HOLD == 1) {
            if (wv < nw) {
                Raw<QT> next = raw;
                if (ti + stride < ntile) next.load(row_of(ti + stride), wv, g, a.cols);
                chunk_mma<QT, NTT>(raw, xf[0], out, g);
                raw = next;
            }
        } else {
            const uint8_t *row = row_of(ti);
            for (int ch = wv; ch < nch; ch += MR_WAVES) {
                raw.load(row, ch, g, a.cols);
#pragma unroll
                for (int tt = 0; tt < NTT; tt++) load_x<QT>(xf[0][tt], xt[tt], ch, g, a.cols);
                chunk_mma<QT, NTT>(raw, xf[0], out, g);
            }
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

// ---------------------------------------------------------------------------
// Tiles of tokens by weight rows
// ---------------------------------------------------------------------------
// k_mm_tile: a wave computes 32 WM tokens by 32 WN rows on v_mfma_f32_32x32x16_f16, MW by NW waves a workgroup.
// Activations go through LDS (64 columns of the workgroup's tokens at a time, two buffers); weights go from
// memory to the registers of the lanes that hold their rows, a superblock ahead, and are unpacked there: lane l
// holds row l % 32 and the half kh = l / 32 of each MFMA's 16 columns, and which columns of a superblock these
// are is free as long as the activations follow, so that a lane unpacks consecutive bytes.
//
// Operands are exact integers as above.  Q4_K and Q6_K: the accumulators are kept in units of the superblock's
// d, rescaled once a superblock (acc *= d_before / d; a superblock of d = 0 keeps the unit and adds zeros), which
// needs no second set of accumulators; the min terms sum_j m_j X_j, X_j the activations' sums over a sub-block, are
// one more MFMA a superblock, with X_j / 32 as a high and a low fp16 part (2^-22 of X_j).  Q8_0: a block of 32 is two
// MFMAs, whose sum is scaled and added.

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const uint4 &x, h8 w, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, x), w, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16()
{
    return f32x16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
}

// acc += f p, and acc *= f.  The accumulators are named as one register tuple afterwards: as loose values the
// compiler gives them new registers at every use and moves hundreds of them to memory and back.
__device__ __forceinline__ void add16(f32x16 &acc, float f, const f32x16 &p)
{
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = fmaf(f, p[e], acc[e]);
    asm volatile("" : "+v"(acc));
}

__device__ __forceinline__ void scale16(f32x16 &acc, float f)
{
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] *= f;
    asm volatile("" : "+v"(acc));
}

// Column of unit u (8 columns) of stage st inside a superblock; unit 4 kh + s is step s of half kh (Q8_0: unit
// 4 b + 2 kh + s is step 2 b + s, so that a step's halves lie in one block).
template <int QT>
__device__ __forceinline__ int unit_column(int st, int u)
{
    if (QT == BREAD_QTYPE_Q8_0) return 64 * st + 8 * u;
    return 128 * (u >> 2) + 32 * st + 8 * (u & 3);
}

template <int QT>
__device__ __forceinline__ int step_unit(int kh, int s)
{
    return QT == BREAD_QTYPE_Q8_0 ? 4 * (s >> 1) + 2 * kh + (s & 1) : 4 * kh + s;
}

// A weight row's superblock in LDS, PIECES pieces of 16 bytes as they were loaded (piece p from byte
// source(p)), STRIDE bytes from one row to the next; and what a lane keeps of it in registers, its half kh.
template <int QT> struct Share;

template <> struct Share<BREAD_QTYPE_Q4_K> {
    static constexpr int BYTES = Q4K_BYTES, PIECES = 9, STRIDE = 144;
    static __device__ __forceinline__ int source(int p) { return 16 * p; }
    uint4 q[2];      // stages 0 and 1, then 2 and 3
    uint32_t dd;     // d and dmin
    uint32_t sc, m;  // scales and mins of the half's four sub-blocks, a byte each
    h2 S, N;
    __device__ __forceinline__ void half(const uint8_t *b, int kh, int at)
    {
        q[0] = ld_b128(b + 16 + 64 * kh + 32 * at);
        q[1] = ld_b128(b + 32 + 64 * kh + 32 * at);
    }
    __device__ __forceinline__ float take(const uint8_t *b, int kh)
    {
        const uint4 head = ld_b128(b);
        half(b, kh, 0);
        dd = head.x;
        const uint32_t s0 = head.y, s1 = head.z, s2 = head.w;
        sc = kh ? (s2 & 0x0F0F0F0Fu) | ((s0 >> 2) & 0x30303030u) : s0 & 0x3F3F3F3Fu;
        m = kh ? ((s2 >> 4) & 0x0F0F0F0Fu) | ((s1 >> 2) & 0x30303030u) : s1 & 0x3F3F3F3Fu;
        return h2f(dd & 0xFFFFu);
    }
    __device__ __forceinline__ float dmin() const { return h2f(dd >> 16); }
    __device__ __forceinline__ void clear() { sc = 0u; }
    __device__ __forceinline__ void stage(int st)
    {
        S = both((float)byte_of(sc, st));
        N = S * both(-1024.f);
    }
    __device__ __forceinline__ h8 step(int st, int s) const
    {
        const uint4 &v = q[s >> 1];
        return q4m_b8(word(v, 2 * (s & 1)), word(v, 2 * (s & 1) + 1), st & 1, S, N);
    }
    // the mins as the operand against (X_j / 32 in two parts, the second times 2^11)
    __device__ __forceinline__ h8 mins() const
    {
        const h2 a = magic_lo(m) + both(-1024.f), b = magic_hi(m) + both(-1024.f), f = both(0x1p-11f);
        return join(a, b, a * f, b * f);
    }
};

template <> struct Share<BREAD_QTYPE_Q6_K> {
    // the last piece ends with the superblock (d is its last two bytes)
    static constexpr int BYTES = Q6K_BYTES, PIECES = 14, STRIDE = 224;
    static __device__ __forceinline__ int source(int p) { return p < 13 ? 16 * p : 194; }
    uint4 l[4], h[2];
    uint2 sc;
    h2 S[2];
    __device__ __forceinline__ float take(const uint8_t *b, int kh)
    {
#pragma unroll
        for (int k = 0; k < 4; k++) l[k] = ld_b128(b + 64 * kh + 16 * k);
        h[0] = ld_b128(b + 128 + 32 * kh);
        h[1] = ld_b128(b + 144 + 32 * kh);
        sc = *reinterpret_cast<const uint2 *>(b + 192 + 8 * kh);
        return h2f(*reinterpret_cast<const uint16_t *>(b + 222));
    }
    __device__ __forceinline__ void clear() { sc = make_uint2(0u, 0u); }
    // stage st is quarter st: low bytes l[2 (st & 1) ..], their high nibbles from stage 2 on
    __device__ __forceinline__ void stage(int st)
    {
        const uint32_t v = (st < 2 ? sc.x : sc.y) >> (16 * (st & 1));
        S[0] = both((float)(int8_t)(v & 0xFFu));
        S[1] = both((float)(int8_t)((v >> 8) & 0xFFu));
    }
    __device__ __forceinline__ void codes(int st, int s, uint32_t &v0, uint32_t &v1) const
    {
        const int k = 2 * (s & 1);
        const uint4 &lv = l[2 * (st & 1) + (s >> 1)], &hv = h[s >> 1];
        v0 = ((word(lv, k) >> (4 * (st >> 1))) & 0x0F0F0F0Fu) | (((word(hv, k) >> (2 * st)) & 0x03030303u) << 4);
        v1 = ((word(lv, k + 1) >> (4 * (st >> 1))) & 0x0F0F0F0Fu) | (((word(hv, k + 1) >> (2 * st)) & 0x03030303u) << 4);
    }
    __device__ __forceinline__ h8 scaled(uint32_t v0, uint32_t v1, h2 off, int s) const
    {
        const h2 f = S[s >> 1];
        return join((magic_lo(v0) + off) * f, (magic_hi(v0) + off) * f, (magic_lo(v1) + off) * f,
                    (magic_hi(v1) + off) * f);
    }
    // the codes without their low bits, and the low bits alone
    __device__ __forceinline__ void step2(int st, int s, h8 &hi, h8 &lo) const
    {
        uint32_t v0, v1;
        codes(st, s, v0, v1);
        hi = scaled(v0 & 0x3E3E3E3Eu, v1 & 0x3E3E3E3Eu, both(-1056.f), s);
        lo = scaled(v0 & 0x01010101u, v1 & 0x01010101u, both(-1024.f), s);
    }
};

template <> struct Share<BREAD_QTYPE_Q8_0> {
    // 69 dwords from one row to the next: the lanes' dwords lie in different banks
    static constexpr int BYTES = 8 * Q80_BYTES, PIECES = 17, STRIDE = 276;
    static __device__ __forceinline__ int source(int p) { return 16 * p; }
    // four blocks at a time: stages 0 and 1, then 2 and 3
    uint32_t q[4][4];
    float d[4];
    __device__ __forceinline__ void half(const uint8_t *b, int kh, int at)
    {
        const int k0 = 4 * at;
        const uint32_t *w = reinterpret_cast<const uint32_t *>(b) + 4 * kh;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // block k's bytes begin at 34 k + 2: at a dword for odd k, between two for even k
            const int at = (34 * (k0 + k) + 2) / 4;
            uint32_t v[5];
#pragma unroll
            for (int i = 0; i < 5; i++) v[i] = i < 4 || !(k & 1) ? w[at + i] : 0u;
#pragma unroll
            for (int i = 0; i < 4; i++) q[k][i] = (k & 1) ? v[i] : __builtin_amdgcn_alignbyte(v[i + 1], v[i], 2);
            d[k] = h2f(reinterpret_cast<const uint16_t *>(b)[17 * (k0 + k)]);
        }
    }
    __device__ __forceinline__ float take(const uint8_t *b, int kh)
    {
        half(b, kh, 0);
        return 1.0f;
    }
    __device__ __forceinline__ void stage(int) {}
    __device__ __forceinline__ h8 step(int st, int s) const
    {
        const uint32_t(&v)[4] = q[2 * (st & 1) + (s >> 1)];
        const uint32_t v0 = v[2 * (s & 1)] ^ 0x80808080u, v1 = v[2 * (s & 1) + 1] ^ 0x80808080u;
        const h2 off = both(-1152.f);
        return join(magic_lo(v0) + off, magic_hi(v0) + off, magic_lo(v1) + off, magic_hi(v1) + off);
    }
};

// fp16 rows go through LDS like the activations, 64 columns at a time
template <> struct Share<BREAD_QTYPE_F16> {
    static constexpr int BYTES = 512, PIECES = 8, STRIDE = 128;
};

// What a wave wrote to LDS comes before what it reads after this (the hardware keeps a wave's LDS accesses in order)
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int QT, int WM, int WN, int MW, int NW, int KW>
__global__ __launch_bounds__(WAVE *MW *NW *KW, 2) void k_mm_tile(const MmArgs a, int mt, int nt)
{
    using W = Share<QT>;
    constexpr int TM = 32 * WM * MW, TN = 32 * WN * NW, THREADS = WAVE * MW * NW;
    constexpr int XL = TM * 8 / THREADS, WP = TN * W::PIECES, WL = (WP + THREADS - 1) / THREADS;
    constexpr bool DENSE = QT == BREAD_QTYPE_F16;
    constexpr int AHEAD = WM * WN > 4 ? 1 : 2;  // stages of activations on their way, and of operands made: registers
    constexpr bool UNIT = QT == BREAD_QTYPE_Q4_K || QT == BREAD_QTYPE_Q6_K;
    constexpr bool TWO = QT == BREAD_QTYPE_Q6_K;  // a weight is two operands
    // a group of one wave needs neither a second buffer nor barriers: its LDS accesses are in order
    constexpr bool ALONE = MW * NW == 1;
    __shared__ uint4 xs_all[KW][ALONE ? 1 : 2][TM * 8];
    // Q4_K: X_j / 32 of every token by superblock parity and half, four high parts, then four low ones
    __shared__ __attribute__((aligned(16))) uint16_t xm_all[KW][2][QT == BREAD_QTYPE_Q4_K ? TM : 1][2][8];
    __shared__ __attribute__((aligned(16))) uint8_t ws_all[KW][DENSE ? 2 : 1][TN * W::STRIDE];
    const int kg = wave_id() / (MW * NW), wv = wave_id() - kg * (MW * NW);  // group of the superblocks, wave in it
    const int tid = (int)threadIdx.x - kg * THREADS, l = lane_id(), c = l & 31, kh = l >> 5;
    auto &xs = xs_all[kg];
    auto &ws = ws_all[kg];
    auto &xm = xm_all[kg];
    // the workgroups of one XCD (blockIdx % 8, each with an L2 of its own) take neighbouring tiles
    const int all = mt * nt, per = (all + 7) / 8;
    const int ti = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per || ti >= all) return;
    const int m0 = (ti % mt) * TM, n0 = (ti / mt) * TN;
    const int wm = wv % MW, wn = wv / MW;
    const int nsb = (a.cols + 255) / 256, rounds = (nsb + KW - 1) / KW;
    // activations: the thread's units i THREADS + tid of a stage, unit u of token t at u ^ (t % 8); two stages
    // on their way.  Byte offsets from the tile's first token (launch_tile checks that they fit).
    const uint8_t *xbase = reinterpret_cast<const uint8_t *>(a.x + (size_t)m0 * a.xs);
    uint32_t xo[XL];
    uint4 xr[AHEAD][XL];
#pragma unroll
    for (int i = 0; i < XL; i++) {
        const int k = i * THREADS + tid, u = (k & 7) ^ ((k >> 3) & 7);
        xo[i] = (uint32_t)(2 * (min(k >> 3, a.T - 1 - m0) * a.xs + unit_column<QT>(0, u)));
    }
    // stage `at` counted over the group's superblocks; past the end the last superblock again, not used
    auto fetch_x = [&](int at, uint4(&v)[XL]) __attribute__((always_inline)) {
        const int sb = min((at >> 2) * KW + kg, nsb - 1);
        const uint8_t *p = xbase + 512 * (size_t)sb + 2 * unit_column<QT>(at & 3, 0);
        if (!UNIT && a.cols - 256 * sb < 256) {  // the row ends in this superblock: zeros from there
#pragma unroll
            for (int i = 0; i < XL; i++) {
                const int k = i * THREADS + tid, u = (k & 7) ^ ((k >> 3) & 7);
                v[i] = unit_column<QT>(at & 3, u) < a.cols - 256 * sb ? ld_b128(p + xo[i]) : make_uint4(0u, 0u, 0u, 0u);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < XL; i++) v[i] = ld_b128(p + xo[i]);
    };
    auto keep_x = [&](int at, const uint4(&v)[XL]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < XL; i++) {
            const int k = i * THREADS + tid, t = k >> 3;
            xs[ALONE ? 0 : at & 1][k] = v[i];
            if constexpr (QT == BREAD_QTYPE_Q4_K) {
                // the sub-block's four units lie in four lanes; two of them store the parts
                float x = sum_h8(v[i], 0.f);
                x += dpp_f<0xB1>(x);  // quad_perm [1,0,3,2]
                x += dpp_f<0x4E>(x);  // quad_perm [2,3,0,1]
                x *= 1.0f / 32;
                const float hi = (float)(_Float16)x;
                if ((k & 3) < 2)
                    xm[(at >> 2) & 1][t][((k ^ t) >> 2) & 1][4 * (k & 1) + (at & 3)] = f2h((k & 1) ? (x - hi) * 2048.f : hi);
            }
        }
    };
    // weights: the thread's pieces i THREADS + tid, adjacent lanes adjacent pieces of a row (a lane a row would
    // cost the address unit a cycle a lane); rows past the last are the last one again, not stored
    uint32_t wo[WL];
    uint4 wr[WL];
    const uint8_t *wbase = a.w + (size_t)n0 * a.rb;
#pragma unroll
    for (int i = 0; i < WL; i++) {
        const int k = min(i * THREADS + tid, WP - 1), r = k / W::PIECES, piece = k % W::PIECES;
        wo[i] = (uint32_t)(min(r, a.rows - 1 - n0) * a.rb);
        if constexpr (DENSE) wo[i] += 2 * unit_column<QT>(0, piece ^ (r & 7));
        else wo[i] += W::source(piece);
    }
    auto fetch_w = [&](int round, int st) __attribute__((always_inline)) {
        const int sb = min(round * KW + kg, nsb - 1), left = a.cols - 256 * sb;
        const uint8_t *p = wbase + (size_t)sb * W::BYTES + (DENSE ? 2 * unit_column<QT>(st, 0) : 0);
        if (!UNIT && left < 256) {  // the row ends in this superblock: nothing is read beyond, the rest is zero
#pragma unroll
            for (int i = 0; i < WL; i++) {
                const int k = min(i * THREADS + tid, WP - 1), piece = k % W::PIECES;
                if constexpr (DENSE) {
                    wr[i] = unit_column<QT>(st, piece ^ ((k / W::PIECES) & 7)) < left ? ld_b128(p + wo[i])
                                                                                      : make_uint4(0u, 0u, 0u, 0u);
                } else {
                    const int bytes = left / Q80_ELEMS * Q80_BYTES - 16 * piece;
                    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int h = 0; h < 8; h++)
                        if (2 * h < bytes) v[h / 2] |= ldu2(p + wo[i] + 2 * h) << (16 * (h & 1));
                    wr[i] = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < WL; i++) {
            if constexpr (QT == BREAD_QTYPE_Q4_K || DENSE) wr[i] = ld_b128(p + wo[i]);
            else wr[i] = ldu16(p + wo[i]);
        }
    };
    auto keep_w = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < WL; i++) {
            const int k = i * THREADS + tid;
            if (WP % THREADS == 0 || k < WP) {
                uint8_t *p = ws[buf] + (k / W::PIECES) * W::STRIDE + 16 * (k % W::PIECES);
                if constexpr (W::STRIDE % 16 == 0) {
                    *reinterpret_cast<uint4 *>(p) = wr[i];
                } else {
#pragma unroll
                    for (int v = 0; v < 4; v++) reinterpret_cast<uint32_t *>(p)[v] = word(wr[i], v);
                }
            }
        }
    };
    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; i++)
#pragma unroll
        for (int j = 0; j < WN; j++) acc[i][j] = zero16();
    float unit[WN];
#pragma unroll
    for (int j = 0; j < WN; j++) unit[j] = 1.0f;
    fetch_w(0, 0);
    fetch_x(0, xr[0]);
    if constexpr (AHEAD > 1) fetch_x(1, xr[1]);
    auto group_sync = [&]() __attribute__((always_inline)) {
        if constexpr (ALONE) wave_order();
        else q4m_bar();
    };
    keep_w(0);
    keep_x(0, xr[0]);
    group_sync();
    for (int round = 0; round < rounds; round++) {
        const bool any = KW == 1 || round * KW + kg < nsb;  // a superblock for this group
        W w[DENSE ? 1 : WN];
        if constexpr (!DENSE) if (any) {
#pragma unroll
            for (int j = 0; j < WN; j++) {
                const float d = w[j].take(ws[0] + (32 * (wn * WN + j) + c) * W::STRIDE, kh);
                if constexpr (UNIT) {
                    if (d == 0.f) w[j].clear();
                    const float to = d == 0.f ? unit[j] : d, ratio = unit[j] / to;
                    unit[j] = to;
#pragma unroll
                    for (int i = 0; i < WM; i++) scale16(acc[i][j], ratio);
                }
            }
        }
#pragma unroll
        for (int st = 0; st < 4; st++) {
            const int buf = st & 1;
            // the activations of two stages on; the next superblock's weights, once for the four stages
            fetch_x(4 * round + st + AHEAD, xr[st % AHEAD]);
            if (DENSE) fetch_w(st < 3 ? round : round + 1, (st + 1) & 3);
            else if (st == 0) fetch_w(round + 1, 0);
            if (any) {
            if constexpr (!DENSE) {
#pragma unroll
                for (int j = 0; j < WN; j++) {
                    if constexpr (QT != BREAD_QTYPE_Q6_K) {
                        if (st == 2) w[j].half(ws[0] + (32 * (wn * WN + j) + c) * W::STRIDE, kh, 1);
                    }
                    w[j].stage(st);
                }
            }
            if constexpr (QT == BREAD_QTYPE_Q8_0) {
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    uint4 xa[WM][2];
#pragma unroll
                    for (int i = 0; i < WM; i++)
#pragma unroll
                        for (int s = 0; s < 2; s++)
                            xa[i][s] = xs[ALONE ? 0 : buf][(32 * (wm * WM + i) + c) * 8 + (step_unit<QT>(kh, 2 * b + s) ^ (c & 7))];
#pragma unroll
                    for (int j = 0; j < WN; j++) {
                        const h8 w0 = w[j].step(st, 2 * b), w1 = w[j].step(st, 2 * b + 1);
                        const float d = w[j].d[2 * (st & 1) + b];
#pragma unroll
                        for (int i = 0; i < WM; i++) {
                            const f32x16 p = mfma32(xa[i][1], w1, mfma32(xa[i][0], w0, zero16()));
                            add16(acc[i][j], d, p);
                        }
                        __builtin_amdgcn_sched_barrier(0);  // else all partial sums are in flight at once
                    }
                }
            } else {
                // a step's operands are read and unpacked beside the products of the step before it; the scheduler
                // is kept to that, else it makes the whole stage's operands first and runs out of registers
                uint4 xa[AHEAD][WM];
                h8 wf[AHEAD][WN][TWO ? 2 : 1];
                auto operands = [&](int s) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < WM; i++)
                        xa[s % AHEAD][i] = xs[ALONE ? 0 : buf][(32 * (wm * WM + i) + c) * 8 + (step_unit<QT>(kh, s) ^ (c & 7))];
#pragma unroll
                    for (int j = 0; j < WN; j++) {
                        if constexpr (DENSE)
                            wf[s % AHEAD][j][0] = __builtin_bit_cast(
                                h8, reinterpret_cast<const uint4 *>(
                                        ws[buf])[(32 * (wn * WN + j) + c) * 8 + (step_unit<QT>(kh, s) ^ (c & 7))]);
                        else if constexpr (TWO)
                            w[j].step2(st, s, wf[s % AHEAD][j][0], wf[s % AHEAD][j][1]);
                        else
                            wf[s % AHEAD][j][0] = w[j].step(st, s);
                    }
                };
                if constexpr (AHEAD > 1) operands(0);
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    if (AHEAD == 1) operands(s);
                    else if (s < 3) operands(s + 1);
#pragma unroll
                    for (int j = 0; j < WN; j++)
#pragma unroll
                        for (int i = 0; i < WM; i++) {
                            acc[i][j] = mfma32(xa[s % AHEAD][i], wf[s % AHEAD][j][0], acc[i][j]);
                            if constexpr (TWO) acc[i][j] = mfma32(xa[s % AHEAD][i], wf[s % AHEAD][j][1], acc[i][j]);
                        }
                    if (AHEAD > 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
            }
            // every wave has taken its share of the weights before stage 2's barrier
            if (DENSE) keep_w(buf ^ 1);
            else if (st == 3) keep_w(0);
            if (ALONE) wave_order();
            keep_x(4 * round + st + 1, xr[(st + 1) % AHEAD]);
            group_sync();
        }
        if constexpr (QT == BREAD_QTYPE_Q4_K) if (any) {
#pragma unroll
            for (int j = 0; j < WN; j++) {
                const h8 m = w[j].mins();
                const float f = -32.f * (w[j].dmin() / unit[j]);
#pragma unroll
                for (int i = 0; i < WM; i++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(xm[round & 1][32 * (wm * WM + i) + c][kh]);
                    add16(acc[i][j], f, mfma32(x, m, zero16()));
                }
            }
        }
    }
    // 32 by 32 results at a time through the wave's own part of the activations' buffers, which every wave has
    // read: lanes then hold four consecutive rows of a token, and the groups' sums are joined, each group taking
    // its part of the tokens
    static_assert(2 * WM >= NW, "4 KB a wave");
    if (ALONE) __syncthreads();
    float *all_out = reinterpret_cast<float *>(&xs_all[0][0][0]), *out = all_out + 1024 * wave_id();
#pragma unroll
    for (int j = 0; j < WN; j++)
#pragma unroll
        for (int i = 0; i < WM; i++) {
#pragma unroll
            for (int k = 0; k < 16; k++)
                out[32 * (8 * (k >> 2) + 4 * kh + (k & 3)) + c] = UNIT ? acc[i][j][k] * unit[j] : acc[i][j][k];
            if (KW > 1) __syncthreads();
            else wave_order();
            const int r = n0 + 32 * (wn * WN + j) + 4 * (l & 7);
#pragma unroll 1
            for (int k = kg * 4 / KW; k < (kg + 1) * 4 / KW; k++) {
                const int tt = 8 * k + (l >> 3), t = m0 + 32 * (wm * WM + i) + tt;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < KW; g++) {
                    const float4 f = *reinterpret_cast<const float4 *>(all_out + 1024 * (g * MW * NW + wv) + 32 * tt + 4 * (l & 7));
                    v[0] += f.x;
                    v[1] += f.y;
                    v[2] += f.z;
                    v[3] += f.w;
                }
                if (t < a.T && r < a.rows) put4(a, t, r, v);
            }
            if (KW > 1) __syncthreads();
            else wave_order();
        }
}

template <int QT, int WM, int WN, int MW, int NW, int KW>
int launch_tile(const MmArgs &a, hipStream_t st)
{
    const int64_t mt = (a.T + 32 * WM * MW - 1) / (32 * WM * MW), nt = ((int64_t)a.rows + 32 * WN * NW - 1) / (32 * WN * NW);
    BREAD_REQUIRE((mt * nt + 7) * (WAVE * MW * NW * KW) < (1ll << 32), BREAD_ERR_SHAPE, "too many tiles for a launch");
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_mm_tile<QT, WM, WN, MW, NW, KW>), dim3((unsigned)((mt * nt + 7) / 8 * 8)),
                       dim3(WAVE * MW * NW * KW), 0, st, a, (int)mt, (int)nt);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

template <int QT>
int launch_rows(const MmArgs &a, hipStream_t st)
{
    const int tt = (a.T + 15) / 16, ny = (tt + MR_MAXTT - 1) / MR_MAXTT, ntt = (tt + ny - 1) / ny;
    const int64_t ntile = ((int64_t)a.rows + 15) / 16;
    int64_t stride = 512 / ny;
    if (stride < 1) stride = 1;
    if (stride > ntile) stride = ntile;
    const dim3 grid((unsigned)(stride * ny)), block(MR_THREADS);
    bread_clear_stale_error();
    const int sets = (a.cols + 256 * MR_WAVES - 1) / (256 * MR_WAVES);  // chunks of a wave
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, st, a, ny, (int)stride); };
    // Two chunks are held for row tiles enough to make up for a workgroup less on a CU or registers at their limit.
    // 9 tokens by 40000 x 4096, not held and held: Q4_K 50 and 37 us, Q6_K 58 and 47, Q8_0 62 and 54; by 8192 x 2304
    // Q4_K, one tile a workgroup, 7.5 and 9.3.  Two fp16 chunks beside their activations would not fit the registers.
    if (ntt == 1 && sets == 1) go(k_mm_rows<QT, 1, 1>);
    else if (ntt == 1 && sets == 2 && QT != BREAD_QTYPE_F16 && ntile >= 2 * stride) go(k_mm_rows<QT, 1, QT == BREAD_QTYPE_F16 ? 0 : 2>);
    else if (ntt == 1) go(k_mm_rows<QT, 1, 0>);
    else if (ntt == 2 && sets == 1) go(k_mm_rows<QT, 2, 1>);
    else if (ntt == 2) go(k_mm_rows<QT, 2, 0>);
    else if (ntt == 3) go(k_mm_rows<QT, 3, 0>);
    else go(k_mm_rows<QT, 4, 0>);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

// The kernel and its tile.  Up to ROWS_T tokens: rows, which read a weight once and have no barrier between
// its arrival and its products.  Beyond, tiles: the largest that leave something for most of the 256 CUs, since a
// superblock takes a workgroup about as long for a small tile as for a large one; the smaller ones split the
// superblocks over groups of waves.  us on MI355X, fp16 results, tokens by
// 32 x 64, 64 x 64, 128 x 128, 128 x 256 and 256 x 256 tiles:
//   Q4_K   24 tokens, 2048 x 2048   rows 7.1   9.6   12.5   27.5    39.5    69.1
//          48         8192 x 2048       32.8  11.4   13.5   30.5    41.9    73.3
//         256         4096 x 2048       78.6  15.8   14.1   30.8    44.9    81.1
//        1024         4096 x 2048        274  56.9   55.5   39.4    50.1    84.3
//        2048         8192 x 2048       1011   220    226    141     109     102
//   Q6_K  509         2048 x 4096       81.8  44.2   30.0   68.6     104
//        1024         8192 x 2048          -   189    129   83.8    70.7
//   Q8_0 1024         4096 x 2048        219  84.0   58.7   38.2    59.9     176
//        2048         8192 x 2048        866   331    247    145     127     225
//   fp16 2048         8192 x 2048       1068   338    253    112     112    90.1
// (256 x 256 of Q6_K and Q8_0 do not fit their registers and are not built.  Q8_0's 128 x 256 and 64 x 64 are at their
// limit and spill 13 and 11.)
// Where 32 x 32 tiles are no more than the CUs, a workgroup has one, with its superblocks over eight groups and not
// four: a round fewer to wait for.  us with 32 x 64 and four groups, and with 32 x 32 and eight:
//   Q8_0   67 tokens, 2048 x 4096   19.0  12.3     Q4_K   64 tokens, 2048 x 2048   9.7   8.0
//   Q6_K   64         2048 x 4096   22.2  13.7     fp16  128         2048 x 4096  18.4  13.8
//   448 tiles, Q8_0, 200 tokens, 2048 x 4096       19.1  21.5
//   four groups for two superblocks, Q4_K, 64 tokens, 2048 x 512                   6.3   7.6
// (A group is then one wave and needs no barriers: 1.5 us of the 12.3.)
constexpr int ROWS_T = 32;
constexpr int64_t FILL = 200;  // workgroups

template <int QT>
int launch_matmul(const MmArgs &a, hipStream_t st)
{
    auto tiles = [&](int64_t m, int64_t n) { return (a.T + m - 1) / m * ((a.rows + n - 1) / n); };
    // a tile's rows and tokens are addressed by 32-bit offsets
    if (a.T <= ROWS_T || a.rb >= (1u << 23) || a.xs >= (1 << 22)) return launch_rows<QT>(a, st);
    if constexpr (QT == BREAD_QTYPE_Q4_K || QT == BREAD_QTYPE_F16) {
        if (tiles(256, 256) >= FILL) return launch_tile<QT, 4, 2, 2, 4, 1>(a, st);
    }
    if (tiles(128, 256) >= FILL) return launch_tile<QT, 4, 1, 1, 8, 1>(a, st);
    if (tiles(128, 128) >= FILL) return launch_tile<QT, 2, 1, 2, 4, 1>(a, st);
    if (tiles(64, 64) >= FILL) {
        // (Q6_K unpacks with twice the instructions: a wave's weights against twice the tokens)
        if constexpr (QT == BREAD_QTYPE_Q6_K) return launch_tile<QT, 2, 1, 1, 2, 4>(a, st);
        else return launch_tile<QT, 1, 1, 2, 2, 4>(a, st);
    }
    if (tiles(32, 32) <= 256 && a.cols > 4 * 256) return launch_tile<QT, 1, 1, 1, 1, 8>(a, st);
    return launch_tile<QT, 1, 1, 1, 2, 4>(a, st);
}

}  // namespace

extern "C" int bread_matmul(const void *w, const uint16_t *x, void *y, int rows, int cols, int qtype, int n_tokens,
                            const bread_matmul_opts_t *opts, bread_stream_t stream)
{
    static const bread_matmul_opts_t plain = {nullptr, nullptr, BREAD_ACT_NONE, BREAD_QTYPE_F16, 0, 0};
    const bread_matmul_opts_t &o = opts ? *opts : plain;
    BREAD_REQUIRE(rows >= 0 && cols > 0 && n_tokens >= 0, BREAD_ERR_ARG,
                  "rows and n_tokens must be >= 0 and cols > 0");
    BREAD_REQUIRE(rows <= 1 << 30 && cols <= 1 << 30 && n_tokens <= 1 << 28, BREAD_ERR_SHAPE,
                  "rows or cols above 2^30, or n_tokens above 2^28");
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
    case BREAD_QTYPE_Q4_K: return launch_matmul<BREAD_QTYPE_Q4_K>(a, st);
    case BREAD_QTYPE_Q6_K: return launch_matmul<BREAD_QTYPE_Q6_K>(a, st);
    case BREAD_QTYPE_Q8_0: return launch_matmul<BREAD_QTYPE_Q8_0>(a, st);
    default: return launch_matmul<BREAD_QTYPE_F16>(a, st);
    }
}
