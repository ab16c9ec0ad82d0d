// fp8_tile.h — the kernel of bread_matmul_fp8 and bread_matmul_fp8_grouped:
//   v[t][r] = sum_b xs[t][b] ws[r / 128][b] sum_{c in b} x[t][c] w[r][c]
// for tokens t and weight rows r, with the epilogue y = act(v + bias) [* v_up] + residual,
// rounded to fp16, bf16 or fp32, or quantised again by blocks of 128 rows.
//
// A block's products are summed by matrix instructions from zero, and the
// product of the two scales is applied to that sum: one fused multiply-add a
// block of 128 columns and element of y.
#pragma once

#include <type_traits>

#include "activate.h"
#include "fp8.h"

namespace {

typedef f8_f32x4 f32x4;
typedef f8_half8 h8;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Bytes that a buffer of activations holds at most, and an offset beyond every buffer
constexpr uint32_t BEYOND = 1u << 31;

// s_waitcnt vmcnt(0): this wave's direct-to-LDS loads have landed
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), lgkmcnt and expcnt at their maxima
    __builtin_amdgcn_sched_barrier(0);
}

// Sixteen codes as two operands of v_mfma_f32_16x16x32_f16 (exact)
__device__ __forceinline__ void widen(const uint4 &q, h8 &a, h8 &b)
{
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    h2 p[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        p[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, false);
        p[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.0f, true);
    }
    a = h8{p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
    b = h8{p[4][0], p[4][1], p[5][0], p[5][1], p[6][0], p[6][1], p[7][0], p[7][1]};
}

// The 128 columns of a row that a lane holds, 32 codes: which of the row's columns they are is free as long as
// weights and activations agree.
template <bool FAST> struct Frag;

template <> struct Frag<true> {
    i32x8 v;
    __device__ __forceinline__ void set(const uint4 &a, const uint4 &b)
    {
        v = i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    }
};

template <> struct Frag<false> {
    h8 v[4];
    __device__ __forceinline__ void set(const uint4 &a, const uint4 &b)
    {
        widen(a, v[0], v[1]);
        widen(b, v[2], v[3]);
    }
};

// z[t] = sums of 128 columns: weight rows 4 (l / 16) + i of lane l in element i, token l % 16 of tile t
template <int TX>
__device__ __forceinline__ void products(const Frag<true> &w, const Frag<true> (&x)[TX], f32x4 (&z)[TX])
{
#pragma unroll
    for (int t = 0; t < TX; t++)
        z[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x[t].v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

template <int TX>
__device__ __forceinline__ void products(const Frag<false> &w, const Frag<false> (&x)[TX], f32x4 (&z)[TX])
{
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int t = 0; t < TX; t++)
            z[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], x[t].v[i], i ? z[t] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------

// Rows r .. r + 3 of the token at row t of y
__device__ __forceinline__ void put4(const F8Args &a, int64_t t, int r, const float (&in)[4])
{
    const int64_t o = t * a.y_stride + r;
    float v[4] = {in[0], in[1], in[2], in[3]};
    if (r + 4 <= a.rows) {
        if (a.y_type == BREAD_QTYPE_F32) {
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
            const bool half = a.y_type == BREAD_QTYPE_F16;
            if (a.res) {
                __builtin_memcpy(h, static_cast<const uint16_t *>(a.res) + o, 8);
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] += half ? h2f(h[k]) : bf2f(h[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) h[k] = half ? f2h(v[k]) : f2bf(v[k]);
            __builtin_memcpy(y, h, 8);
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (r + k >= a.rows) return;
        if (a.y_type == BREAD_QTYPE_F32) {
            if (a.res) v[k] += static_cast<const float *>(a.res)[o + k];
            static_cast<float *>(a.y)[o + k] = v[k];
        } else {
            const bool half = a.y_type == BREAD_QTYPE_F16;
            if (a.res) {
                const uint32_t h = static_cast<const uint16_t *>(a.res)[o + k];
                v[k] += half ? h2f(h) : bf2f(h);
            }
            static_cast<uint16_t *>(a.y)[o + k] = half ? f2h(v[k]) : f2bf(v[k]);
        }
    }
}

// act(v + bias) or act(v) * u of rows r .. r + 3
__device__ __forceinline__ void finish4(const F8Args &a, int r, float (&v)[4])
{
    if (a.bias) {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] += a.bias[min(r + k, a.rows - 1)];
    }
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = activate(v[k], a.act);
}

// ---------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------
// A workgroup takes tiles of 16 TX NWX tokens by OR weight rows (of one or two matrices) in turn.  Its columns come in
// stages of KSB blocks of 128, by loads to LDS that are one stage ahead, across the tiles' ends too.  Rows lie 128 bytes
// apart, the eight pieces of 16 bytes of row r at piece ^ (r % 8), so that a read of a piece of 16 rows covers the banks.
// NWW x NWX waves have TO row tiles by TX token tiles each; NWK such sets of waves share a stage's blocks and add their
// sums through LDS.

// Where a tile lies: weights' group, first row and number of rows (of the call's T), first weight row
struct Place {
    int g, p0, n, row0;
};

template <int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST> struct Shape {
    static constexpr int WAVES = NWW * NWX * NWK, THREADS = WAVES * WAVE, M = GLU ? 2 : 1, N = M * TO;
    static constexpr int OR = 16 * NWW * TO, WR = M * OR, BX = 16 * NWX * TX, KPW = KSB / NWK;
    static constexpr int OB = OR > F8_BLOCK ? OR / F8_BLOCK : 1;  // blocks of rows that a tile meets
    static constexpr int PASS = THREADS / 8;                      // rows that the workgroup loads at a time
    static constexpr int PW = (KSB * WR + PASS - 1) / PASS, PX = (KSB * BX + PASS - 1) / PASS;
    static constexpr int XSW = (BX + WAVE - 1) / WAVE, NXS = KSB * XSW;  // loads of tokens' scales
    static constexpr int W_BYTES = KSB * WR * F8_BLOCK, X_BYTES = KSB * BX * F8_BLOCK;
    static constexpr int XS_AT = W_BYTES + X_BYTES, WS_AT = XS_AT + 4 * NXS * WAVE, STAGE = WS_AT + 4 * M * WAVE;
    static constexpr int SUMS = (NWK - 1) * NWW * NWX * N * TX * WAVE * 16;
    static_assert(KSB % NWK == 0 && OB * KSB <= WAVE && (OR % F8_BLOCK == 0 || F8_BLOCK % OR == 0), "whole blocks");
    static_assert((KSB * WR) % PASS == 0 && WR % 8 == 0 && BX % 8 == 0 && 16 * TO <= F8_BLOCK, "whole passes");
};

template <class S> struct Lds {
    __attribute__((aligned(16))) uint8_t buf[2][S::STAGE];
    __attribute__((aligned(16))) uint8_t sums[S::SUMS ? S::SUMS : 16];
    uint32_t mags[S::OR / 16][S::BX];
};

constexpr int GROUPS_MAX = 1024;

// tiles[g]: token tiles of the groups before g, for g <= G
template <int THREADS>
__device__ __forceinline__ void count_tiles(const F8Args &a, int bx, int *tiles, int *sums)
{
    const int per = (a.G + THREADS - 1) / THREADS, g0 = (int)threadIdx.x * per;
    auto of = [&](int g) __attribute__((always_inline)) {
        const int lo = min(max(a.offsets[g], 0), a.T), hi = min(max(a.offsets[g + 1], 0), a.T);
        return hi > lo ? (hi - lo + bx - 1) / bx : 0;
    };
    int mine = 0;
    for (int g = g0; g < min(g0 + per, a.G); g++) mine += of(g);
    const int incl = wave_scan_incl(mine);
    if (lane_id() == WAVE - 1) sums[threadIdx.x / WAVE] = incl;
    __syncthreads();
    int before = incl - mine;
    for (int i = 0; i < (int)threadIdx.x / WAVE; i++) before += sums[i];
    for (int g = g0; g < min(g0 + per, a.G); g++) {
        tiles[g] = before;
        before += of(g);
    }
    if (g0 < a.G && g0 + per >= a.G) tiles[a.G] = before;
    __syncthreads();
}

template <class S, int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, bool KEEP, bool GRP>
__device__ __forceinline__ void run_tiles(const F8Args &a, const int n_wt, int n_xt, Lds<S> &lds, int *gtiles, int *gsums)
{
    constexpr int M = S::M, N = S::N, OR = S::OR, BX = S::BX, WR = S::WR, PASS = S::PASS;
    const int tid = (int)threadIdx.x, wv = wave_id(), l = lane_id();
    const int wk = wv / (NWW * NWX), ww = wv % NWW, wx = wv / NWW % NWX;
    const int r = l & 15, g = l >> 4, nb = f8_blocks(a.cols), nrb = f8_blocks(a.rows), steps = (nb + KSB - 1) / KSB;
    if constexpr (GRP) {
        count_tiles<S::THREADS>(a, BX, gtiles, gsums);
        n_xt = uniform(gtiles[a.G]);
    }
    // consecutive tiles on one XCD, whose workgroups then share an L2
    const int total = n_xt * n_wt, per = (total + 7) / 8, stride = (int)gridDim.x / 8, xcd = (int)blockIdx.x % 8;
    const int end = min(per * (xcd + 1), total);
    int tile = per * xcd + (int)blockIdx.x / 8;
    if (tile >= end) return;

    auto place = [&](int i, int from) __attribute__((always_inline)) {
        Place p;
        if constexpr (GRP) {
            // the last group with tiles[g] <= xt, from one that is not behind it, 64 groups at a time
            const int xt = i / n_wt;
            int lo = from;
            for (;;) {
                const int ahead = lo + 1 + l;
                const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(ahead < a.G && gtiles[ahead] <= xt));
                lo += n;
                if (n < WAVE) break;
            }
            const int at = min(max(a.offsets[lo], 0), a.T), e = min(max(a.offsets[lo + 1], 0), a.T);
            p.g = lo;
            p.p0 = uniform(at + (xt - uniform(gtiles[lo])) * BX);
            p.n = uniform(min(e - p.p0, BX));
            p.row0 = (i - xt * n_wt) * OR;
        } else {
            // bands of eight token tiles: the tiles that an XCD works on at a time are a square
            const int band = i / (8 * n_wt), j = i - band * 8 * n_wt, high = min(8, n_xt - 8 * band), w = j / high;
            p.g = 0;
            p.p0 = (8 * band + j - w * high) * BX;
            p.n = min(a.T - p.p0, BX);
            p.row0 = w * OR;
        }
        return p;
    };

    // -------------------------------------------------------------- loads
    // Loads give zeros beyond their buffer: for rows that are none, and the columns behind a row's end.
    const int srow = tid / 8, piece = (tid % 8) ^ (srow & 7);
    uint32_t xoff[S::PX], xsoff = BEYOND;
    __amdgpu_buffer_rsrc_t wb, ub, xb, xsb, wsb, usb;
    int srb0 = 0;
    auto aim = [&](const Place &p) __attribute__((always_inline)) {
        const uint32_t bytes = (uint32_t)min(OR, a.rows - p.row0) * (uint32_t)a.cols;
        const size_t first = ((size_t)p.g * a.rows + p.row0) * a.cols, scale = (size_t)p.g * nrb * nb;
        const int64_t xr0 = GRP && a.x_rows ? 0 : p.p0;  // x row that offsets count from
        wb = rsrc(a.w + first, bytes);
        ub = rsrc(GLU ? a.up + first : a.w + first, bytes);
        wsb = rsrc(a.ws + scale, 4u * (uint32_t)nrb * (uint32_t)nb);
        usb = rsrc(GLU ? a.us + scale : a.ws + scale, 4u * (uint32_t)nrb * (uint32_t)nb);
        xb = rsrc(a.x + xr0 * a.x_stride, BEYOND);
        xsb = rsrc(a.xs + xr0 * a.xs_stride, BEYOND);
        srb0 = p.row0 / F8_BLOCK;
        auto x_row = [&](int i) __attribute__((always_inline)) {  // x row of tile row i, -1 for none
            if (i >= p.n) return -1;
            if (!GRP || !a.x_rows) return i;
            const int v = a.x_rows[p.p0 + i];
            return (unsigned)v < (unsigned)a.n_x ? v : -1;
        };
#pragma unroll
        for (int i = 0; i < S::PX; i++) {
            const int at = i * PASS + srow, v = KSB * BX % PASS && at >= KSB * BX ? -1 : x_row(at % BX);
            xoff[i] = v < 0 ? BEYOND : (uint32_t)v * (uint32_t)a.x_stride + 16 * piece;
        }
        if (wv < S::NXS) {
            const int v = x_row(wv % S::XSW * WAVE + l);
            xsoff = v < 0 ? BEYOND : 4u * (uint32_t)v * (uint32_t)a.xs_stride;
        }
    };
    uint32_t woff[S::PW];
#pragma unroll
    for (int i = 0; i < S::PW; i++) woff[i] = (uint32_t)((i * PASS + srow) % OR) * (uint32_t)a.cols + 16 * piece;
    auto stage = [&](uint8_t *to, int step) __attribute__((always_inline)) {
        uint8_t *b = to + wv * 8 * F8_BLOCK;
        const int k0 = step * KSB * F8_BLOCK;
        // scales first: the next barrier waits for all of a stage's loads
#pragma unroll
        for (int i = 0; i < (S::NXS + S::WAVES - 1) / S::WAVES; i++) {
            const int j = wv + i * S::WAVES, kb = step * KSB + j / S::XSW;  // (a wave's loads are of the same tokens)
            if (j < S::NXS)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xsb, to + S::XS_AT + 4 * j * WAVE, 4, kb < nb ? xsoff : BEYOND,
                                                         kb < nb ? 4 * kb : 0, 0, 0);
        }
        if (wv == S::WAVES - 1) {
            const int kb = step * KSB + l / S::OB, rb = srb0 + l % S::OB;
            const uint32_t off = l < KSB * S::OB && kb < nb && rb < nrb ? 4u * (uint32_t)(rb * nb + kb) : BEYOND;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wsb, to + S::WS_AT, 4, off, 0, 0, 0);
            if constexpr (GLU) __builtin_amdgcn_raw_ptr_buffer_load_lds(usb, to + S::WS_AT + 4 * WAVE, 4, off, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::PW; i++) {
            const int kk = i * PASS / WR, row = i * PASS % WR;  // (PASS divides WR or is a multiple of it)
            const int c = k0 + (PASS > WR ? (i * PASS + srow) / WR : kk) * F8_BLOCK;
            const uint32_t off = c + 16 * piece < a.cols ? woff[i] + (PASS > WR ? c - k0 : 0) : BEYOND;
            const int soff = PASS > WR ? k0 : k0 + kk * F8_BLOCK;
            if (!GLU || (PASS <= OR ? row < OR : srow % WR < OR))
                __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, b + i * PASS * F8_BLOCK, 16, off, soff, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ub, b + i * PASS * F8_BLOCK, 16, off, soff, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::PX; i++) {
            if (KSB * BX % PASS && i * PASS + wv * 8 >= KSB * BX) break;
            const int c = (i * PASS + srow) / BX * F8_BLOCK;
            const uint32_t off = k0 + c + 16 * piece < a.cols && xoff[i] != BEYOND ? xoff[i] + c : BEYOND;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, b + S::W_BYTES + i * PASS * F8_BLOCK, 16, off, k0, 0, 0);
        }
    };
    // -------------------------------------------------------------- products
    struct Ops {  // a block's operands as they lie in LDS
        uint4 x[TX][2], w[N][2];
        float xs[TX], ws[M];
    };
    f32x4 acc[N][TX];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int t = 0; t < TX; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    const int wr0 = 16 * TO * ww;  // the wave's first row in the tile
    const int at0 = r * F8_BLOCK + 16 * (g ^ (r & 7)), at1 = at0 ^ 64;
    auto read = [&](Ops &q, const uint8_t *b, int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TX; t++) {
            const uint8_t *p = b + S::W_BYTES + (kk * BX + 16 * (t * NWX + wx)) * F8_BLOCK;
            q.x[t][0] = *reinterpret_cast<const uint4 *>(p + at0);
            q.x[t][1] = *reinterpret_cast<const uint4 *>(p + at1);
            q.xs[t] = *reinterpret_cast<const float *>(b + S::XS_AT + 4 * (kk * S::XSW * WAVE + 16 * (t * NWX + wx) + r));
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint8_t *p = b + (kk * WR + i / TO * OR + wr0 + 16 * (i % TO)) * F8_BLOCK;
            q.w[i][0] = *reinterpret_cast<const uint4 *>(p + at0);
            q.w[i][1] = *reinterpret_cast<const uint4 *>(p + at1);
        }
#pragma unroll
        for (int m = 0; m < M; m++)
            q.ws[m] = *reinterpret_cast<const float *>(b + S::WS_AT + 4 * (m * WAVE + kk * S::OB + wr0 / F8_BLOCK));
    };
    // with the wave's first C token tiles; a row tile's sums are added while the next one's are made
    auto multiply = [&](const Ops &q, auto count) __attribute__((always_inline)) {
        constexpr int C = decltype(count)::value;
        Frag<FAST> x[C];
#pragma unroll
        for (int t = 0; t < C; t++) x[t].set(q.x[t][0], q.x[t][1]);
        f32x4 z[2][C];
        auto add = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < C; t++) {
                const float s = q.xs[t] * q.ws[i / TO];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][t][e] = fmaf(s, z[i & 1][t][e], acc[i][t][e]);
            }
        };
#pragma unroll
        for (int i = 0; i < N; i++) {
            Frag<FAST> w;
            w.set(q.w[i][0], q.w[i][1]);
            products(w, x, z[i & 1]);
            if (i) add(i - 1);
        }
        add(N - 1);
    };

    // -------------------------------------------------------------- results
    auto finish = [&](const Place &p) __attribute__((always_inline)) {
        if constexpr (NWK > 1) {
            f32x4 *part = reinterpret_cast<f32x4 *>(lds.sums);
            constexpr int W = NWW * NWX;
            if (wk) {
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int t = 0; t < TX; t++) part[(((wv - W) * N + i) * TX + t) * WAVE + l] = acc[i][t];
            }
            __syncthreads();
            if (wk == 0) {
#pragma unroll
                for (int k = 0; k < NWK - 1; k++)
#pragma unroll
                    for (int i = 0; i < N; i++)
#pragma unroll
                        for (int t = 0; t < TX; t++) acc[i][t] += part[(((k * W + wv) * N + i) * TX + t) * WAVE + l];
            }
        }
        auto y_row = [&](int t) __attribute__((always_inline)) {  // y row of the lane's token, -1 for none
            const int i = 16 * (t * NWX + wx) + r;
            if (i >= p.n) return -1;
            if (!GRP || !a.y_rows) return p.p0 + i;
            const int v = a.y_rows[p.p0 + i];
            return (unsigned)v < (unsigned)a.n_y ? v : -1;
        };
        auto result = [&](int o, int t, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = acc[o][t][e];
            finish4(a, p.row0 + wr0 + 16 * o + 4 * g, v);
            if constexpr (GLU) {
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] *= acc[N - TO + o][t][e];
            }
        };
        const bool quantised = OR % F8_BLOCK == 0 && a.y_type == BREAD_QTYPE_E4M3;
        if (!quantised) {
            if (wk == 0) {
#pragma unroll
                for (int t = 0; t < TX; t++) {
                    const int yr = y_row(t);
#pragma unroll
                    for (int o = 0; o < TO; o++) {
                        const int row = p.row0 + wr0 + 16 * o + 4 * g;
                        float v[4];
                        result(o, t, v);
                        if (yr >= 0 && row < a.rows) put4(a, yr, row, v);
                    }
                }
            }
        }
        if constexpr (OR % F8_BLOCK == 0) {
            if (quantised) {
                // a token's largest magnitude in its lanes, then over the waves of the block's rows.  (rows is a
                // multiple of 16, so a row tile is whole or absent.)
                constexpr int WPB = F8_BLOCK / (16 * TO);  // waves a block
                if (wk == 0) {
#pragma unroll
                    for (int t = 0; t < TX; t++) {
                        uint32_t m = 0;
#pragma unroll
                        for (int o = 0; o < TO; o++) {
                            float v[4];
                            result(o, t, v);
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                acc[o][t][e] = v[e];
                                if (p.row0 + wr0 + 16 * o < a.rows) m = max(m, f8_mag(v[e]));
                            }
                        }
                        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
                        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
                        if (g == 0) lds.mags[ww][16 * (t * NWX + wx) + r] = m;
                    }
                }
                __syncthreads();
                if (wk == 0) {
#pragma unroll
                    for (int t = 0; t < TX; t++) {
                        uint32_t m = 0;
#pragma unroll
                        for (int i = 0; i < WPB; i++) m = max(m, lds.mags[ww / WPB * WPB + i][16 * (t * NWX + wx) + r]);
                        const float s = f8_scale(m), inv = 1.0f / s;
                        const int yr = y_row(t);
                        if (yr < 0) continue;
                        if (ww % WPB == 0 && g == 0 && p.row0 + wr0 < a.rows)
                            a.ys[yr * a.ys_stride + (p.row0 + wr0) / F8_BLOCK] = s;
#pragma unroll
                        for (int o = 0; o < TO; o++) {
                            const int row = p.row0 + wr0 + 16 * o + 4 * g;
                            if (row < a.rows)
                                *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.y) + yr * a.y_stride + row) =
                                    f8_pack4(acc[o][t][0], acc[o][t][1], acc[o][t][2], acc[o][t][3], inv);
                        }
                    }
                }
            }
        }
    };

    Place now = place(tile, 0), next = now;
    aim(now);
    stage(lds.buf[0], 0);
    clear();
    int cur = 0;
    for (;;) {
        const int active = min(max((now.n - 16 * wx + 16 * NWX - 1) / (16 * NWX), 0), TX);  // token tiles of the wave
        for (int step = 0; step < steps; step++) {
            wait_loads();
            __syncthreads();
            // Every operand of the stage is read before the next stage's loads are issued: the compiler waits for all
            // loads to LDS before a read of LDS behind them.
            Ops q[S::KPW];
#pragma unroll
            for (int i = 0; i < S::KPW; i++) read(q[i], lds.buf[cur], wk + i * NWK);
            __builtin_amdgcn_sched_barrier(0);
            if (step + 1 < steps) {
                stage(lds.buf[cur ^ 1], step + 1);
            } else if (KEEP && tile + stride < end) {
                next = place(tile + stride, now.g);
                aim(next);
                stage(lds.buf[cur ^ 1], 0);
            }
#pragma unroll
            for (int i = 0; i < S::KPW; i++) {
                if (KSB > 1 && step * KSB + wk + i * NWK >= nb) break;
                if (!GRP) {
                    multiply(q[i], std::integral_constant<int, TX>());
                } else if (TX >= 4 && active <= TX / 4) {
                    if (active) multiply(q[i], std::integral_constant<int, (TX + 3) / 4>());
                } else if (TX >= 2 && active <= TX / 2) {
                    if (active) multiply(q[i], std::integral_constant<int, (TX + 1) / 2>());
                } else {
                    if (active) multiply(q[i], std::integral_constant<int, TX>());
                }
            }
            cur ^= 1;
        }
        finish(now);
        tile += stride;
        if (!KEEP || tile >= end) break;
        now = next;
        clear();
    }
}

// (a kernel that is a template and holds buffer descriptors itself is dropped by the host's compilation)
template <int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, int WPE, bool KEEP, bool GRP>
__global__ __launch_bounds__(NWW * NWX * NWK * WAVE, WPE) void k_f8_matmul(const F8Args a, const int n_wt, const int n_xt)
{
    using S = Shape<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST>;
    __shared__ Lds<S> lds;
    __shared__ int gtiles[GRP ? GROUPS_MAX + 1 : 1], gsums[GRP ? S::WAVES : 1];
    run_tiles<S, NWW, NWX, NWK, TO, TX, KSB, GLU, FAST, KEEP, GRP>(a, n_wt, n_xt, lds, gtiles, gsums);
}

// WPE: waves a SIMD, which the registers are held to
template <int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, int WPE, bool KEEP, bool GRP>
int launch(const F8Args &a, hipStream_t st)
{
    using S = Shape<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST>;
    constexpr int lds = (int)sizeof(Lds<S>) + (GRP ? 4 * (GROUPS_MAX + 1 + S::WAVES) : 8);
    constexpr int by_lds = 160 * 1024 / lds, by_waves = 4 * WPE / S::WAVES, resident = by_lds < by_waves ? by_lds : by_waves;
    static_assert(resident >= 1, "a workgroup fits");
    BREAD_REQUIRE(GLU == (a.up != nullptr) && GRP == (a.G > 0) && (a.y_type != BREAD_QTYPE_E4M3 || S::OR % F8_BLOCK == 0), BREAD_ERR_SHAPE,
                  "a kernel for other results");
    const int64_t n_wt = (a.rows + S::OR - 1) / S::OR;
    // groups: a tile more for each that ends inside one
    const int64_t n_xt = GRP ? a.T / S::BX + (a.G < a.T ? a.G : a.T) : (a.T + S::BX - 1) / S::BX;
    const int64_t total = n_wt * n_xt, most = KEEP ? 256 * resident : 1 << 22;
    BREAD_REQUIRE(total <= (KEEP ? 1 << 30 : 1 << 22), BREAD_ERR_SHAPE, "more tiles than a launch counts");
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_f8_matmul<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST, WPE, KEEP, GRP>),
                       dim3((unsigned)((total < most ? total : most) + 7) / 8 * 8), dim3(S::THREADS), 0, st, a, (int)n_wt,
                       (int)n_xt);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

}  // namespace
