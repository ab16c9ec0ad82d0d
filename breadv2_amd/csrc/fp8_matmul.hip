// fp8_matmul.hip — bread_matmul_fp8 and bread_matmul_fp8_grouped: several
// tokens through e4m3 weights,
//   v[t][r] = sum_b xs[t][b] ws[r / 128][b] sum_{c in b} x[t][c] w[r][c],
// with the epilogue y = act(v + bias) [* v_up] + residual, rounded to fp16,
// bf16 or fp32, or quantised again by blocks of 128 rows.
//
// A block's products are summed by matrix instructions from zero, and the
// product of the two scales is applied to that sum: one fused multiply-add a
// block of 128 columns and element of y.
#include "activate.h"
#include "fp8.h"

namespace {

typedef f8_f32x4 f32x4;
typedef f8_half8 h8;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// What lanes read that have no row or no columns
__device__ const uint4 f8_zeros = {0u, 0u, 0u, 0u};

// s_waitcnt vmcnt(0): this wave's direct-to-LDS loads have landed
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0), lgkmcnt and expcnt at their maxima
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ void lds_load16(const void *src, void *lds_wave_base)
{
    __builtin_amdgcn_global_load_lds(src, lds_wave_base, 16, 0, 0);
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

// Sums of 128 columns: weight rows 4 (l / 16) + i of lane l in element i, token l % 16
__device__ __forceinline__ f32x4 product(const Frag<true> &w, const Frag<true> &x)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ f32x4 product(const Frag<false> &w, const Frag<false> &x)
{
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; i++) z = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], x.v[i], z, 0, 0, 0);
    return z;
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
// Tiles
// ---------------------------------------------------------------------------

// Group g's rows p0 .. p0 + n - 1, the xt-th tile of BX rows in group order; false if there are fewer tiles.
// Each thread counts the tiles of some consecutive groups.
template <int THREADS, int BX>
__device__ __forceinline__ bool find_tile(const F8Args &a, int xt, int &g, int &p0, int &n)
{
    __shared__ int sums[THREADS / WAVE], found[3];
    const int per = (a.G + THREADS - 1) / THREADS, g0 = (int)threadIdx.x * per;
    int mine = 0;
    for (int i = g0; i < min(g0 + per, a.G); i++) {
        const int lo = min(max(a.offsets[i], 0), a.T), hi = min(max(a.offsets[i + 1], 0), a.T);
        if (hi > lo) mine += (hi - lo + BX - 1) / BX;
    }
    const int incl = wave_scan_incl(mine);
    if (lane_id() == WAVE - 1) sums[threadIdx.x / WAVE] = incl;
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    int before = incl - mine;
#pragma unroll
    for (int i = 0; i < THREADS / WAVE; i++)
        if (i < (int)threadIdx.x / WAVE) before += sums[i];
    if (xt >= before && xt < before + mine) {
        for (int i = g0; i < min(g0 + per, a.G); i++) {
            const int lo = min(max(a.offsets[i], 0), a.T), hi = min(max(a.offsets[i + 1], 0), a.T);
            const int tiles = hi > lo ? (hi - lo + BX - 1) / BX : 0;
            if (xt < before + tiles) {
                found[0] = i;
                found[1] = lo + (xt - before) * BX;
                found[2] = min(hi - found[1], BX);
                break;
            }
            before += tiles;
        }
    }
    __syncthreads();
    g = uniform(found[0]);
    p0 = uniform(found[1]);
    n = uniform(found[2]);
    return g >= 0;
}

// NWW x NWX waves, each TO row tiles (of one or two matrices) by TX token tiles of 16.  Weights and activations are
// staged through LDS 128 columns at a time, a row's eight pieces of 16 bytes at piece ^ (row % 8) so that a read of
// one piece of 16 rows covers the banks; the next columns load while these are multiplied.
template <int NWW, int NWX, int TO, int TX, bool GLU, bool FAST>
__global__ __launch_bounds__(NWW * NWX * WAVE, GLU ? 1 : 2) void k_f8_tile(const F8Args a, const int n_wt, const int total)
{
    constexpr int THREADS = NWW * NWX * WAVE, OR = 16 * NWW * TO, BX = 16 * NWX * TX, M = GLU ? 2 : 1;
    constexpr int WR = M * OR, PASS = THREADS / 8, PW = WR / PASS, PX = BX / PASS;
    static_assert(WR % PASS == 0 && BX % PASS == 0 && OR % PASS == 0, "whole passes");
    static_assert(OR % F8_BLOCK == 0 && (16 * TO) <= F8_BLOCK, "whole blocks");
    __shared__ __attribute__((aligned(16))) uint8_t buf[2][(WR + BX) * F8_BLOCK];
    __shared__ uint32_t mags[NWW][BX];

    // consecutive tiles on one XCD, whose workgroups then share an L2
    const int per = (total + 7) / 8, tile = ((int)blockIdx.x % 8) * per + (int)blockIdx.x / 8;
    if ((int)blockIdx.x / 8 >= per || tile >= total) return;
    const int xt = tile / n_wt, row0 = (tile - xt * n_wt) * OR;
    int grp = 0, p0 = xt * BX, n = min(a.T - p0, BX);
    if (a.G && !find_tile<THREADS, BX>(a, xt, grp, p0, n)) return;

    const int tid = (int)threadIdx.x, wv = wave_id(), l = lane_id(), ww = wv % NWW, wx = wv / NWW;
    const int r = l & 15, g = l >> 4, nb = f8_blocks(a.cols), nrb = f8_blocks(a.rows);
    const uint8_t *wm[2] = {a.w + (size_t)grp * a.rows * a.cols, GLU ? a.up + (size_t)grp * a.rows * a.cols : nullptr};
    const float *sm[2] = {a.ws + (size_t)grp * nrb * nb, GLU ? a.us + (size_t)grp * nrb * nb : nullptr};

    // x row of tile row i, -1 for none
    auto x_row = [&](int i) __attribute__((always_inline)) {
        if (i >= n) return -1;
        if (!a.x_rows) return p0 + i;
        const int v = a.x_rows[p0 + i];
        return (unsigned)v < (unsigned)a.n_x ? v : -1;
    };

    // what this thread stages: piece `piece` of rows tid / 8 + PASS i
    const int srow = tid / 8, piece = (tid % 8) ^ (srow & 7);
    uint32_t woff[PW];
    const uint8_t *xp[PX];
    bool xv[PX];
#pragma unroll
    for (int i = 0; i < PW; i++) {
        const int o = (i * PASS + srow) % OR;
        woff[i] = (uint32_t)(min(row0 + o, a.rows - 1) - row0) * (uint32_t)a.cols + 16 * piece;
    }
#pragma unroll
    for (int i = 0; i < PX; i++) {
        const int v = x_row(i * PASS + srow);
        xv[i] = v >= 0;
        xp[i] = a.x + (xv[i] ? (int64_t)v * a.x_stride + 16 * piece : 0);
    }
    const uint8_t *wb[2] = {wm[0] + (size_t)row0 * a.cols, GLU ? wm[1] + (size_t)row0 * a.cols : nullptr};
    const void *zeros = &f8_zeros;
    auto stage = [&](int k) __attribute__((always_inline)) {
        uint8_t *b = buf[k & 1] + wv * 8 * F8_BLOCK;
        const int k0 = k * F8_BLOCK;
        const bool in = k0 + 16 * piece < a.cols;
#pragma unroll
        for (int i = 0; i < PW; i++) {
            const uint8_t *p = wb[i * PASS / OR] + k0 + woff[i];
            lds_load16(in ? p : zeros, b + i * PASS * F8_BLOCK);
        }
#pragma unroll
        for (int i = 0; i < PX; i++)
            lds_load16(in && xv[i] ? xp[i] + k0 : zeros, b + (WR + i * PASS) * F8_BLOCK);
    };

    // scales of the tokens that this lane's columns are of, and of the wave's rows
    const float *xsp[TX];
    bool sv[TX];
#pragma unroll
    for (int t = 0; t < TX; t++) {
        const int v = x_row((wx * TX + t) * 16 + r);
        sv[t] = v >= 0;
        xsp[t] = a.xs + (sv[t] ? (int64_t)v * a.xs_stride : 0);
    }
    const int wr0 = ww * 16 * TO;  // the wave's first row in the tile
    const int srb = min((row0 + wr0) / F8_BLOCK, nrb - 1);
    float xs[TX], ws[M], xn[TX], wn[M];
    auto scales = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TX; t++) xn[t] = sv[t] ? xsp[t][k] : 0.f;
#pragma unroll
        for (int m = 0; m < M; m++) wn[m] = sm[m][srb * nb + k];
    };

    f32x4 acc[M][TO][TX];
#pragma unroll
    for (int m = 0; m < M; m++)
#pragma unroll
        for (int o = 0; o < TO; o++)
#pragma unroll
            for (int t = 0; t < TX; t++) acc[m][o][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int at0 = 16 * (g ^ (r & 7)), at1 = at0 ^ 64;
    stage(0);
    scales(0);
    for (int k = 0; k < nb; k++) {
        wait_loads();
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TX; t++) xs[t] = xn[t];
#pragma unroll
        for (int m = 0; m < M; m++) ws[m] = wn[m];
        if (k + 1 < nb) {
            stage(k + 1);
            scales(k + 1);
        }
        const uint8_t *b = buf[k & 1] + r * F8_BLOCK;
        auto frag = [&](Frag<FAST> &f, int row) __attribute__((always_inline)) {
            const uint8_t *p = b + row * F8_BLOCK;
            f.set(*reinterpret_cast<const uint4 *>(p + at0), *reinterpret_cast<const uint4 *>(p + at1));
        };
        Frag<FAST> x[TX];
#pragma unroll
        for (int t = 0; t < TX; t++) frag(x[t], WR + (wx * TX + t) * 16);
#pragma unroll
        for (int m = 0; m < M; m++) {
            float s[TX];
#pragma unroll
            for (int t = 0; t < TX; t++) s[t] = xs[t] * ws[m];
#pragma unroll
            for (int o = 0; o < TO; o++) {
                Frag<FAST> w;
                frag(w, m * OR + wr0 + 16 * o);
#pragma unroll
                for (int t = 0; t < TX; t++) {
                    const f32x4 z = product(w, x[t]);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[m][o][t][e] = fmaf(s[t], z[e], acc[m][o][t][e]);
                }
            }
        }
    }

    // y row of the lane's token in tile t, -1 for none
    auto y_row = [&](int t) __attribute__((always_inline)) {
        const int i = (wx * TX + t) * 16 + r;
        if (i >= n) return -1;
        if (!a.y_rows) return p0 + i;
        const int v = a.y_rows[p0 + i];
        return (unsigned)v < (unsigned)a.n_y ? v : -1;
    };
    auto result = [&](int o, int t, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = acc[0][o][t][e];
        finish4(a, row0 + wr0 + 16 * o + 4 * g, v);
        if constexpr (GLU) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] *= acc[M - 1][o][t][e];
        }
    };
    if (a.y_type != BREAD_QTYPE_E4M3) {
#pragma unroll
        for (int t = 0; t < TX; t++) {
            const int yr = y_row(t);
#pragma unroll
            for (int o = 0; o < TO; o++) {
                const int row = row0 + wr0 + 16 * o + 4 * g;
                float v[4];
                result(o, t, v);
                if (yr >= 0 && row < a.rows) put4(a, yr, row, v);
            }
        }
        return;
    }
    // quantised: a token's largest magnitude in its lanes, then over the waves of the block's rows.  (rows is a
    // multiple of 16, so a row tile is whole or absent.)
    constexpr int WPB = F8_BLOCK / (16 * TO);  // waves a block
#pragma unroll
    for (int t = 0; t < TX; t++) {
        uint32_t m = 0;
#pragma unroll
        for (int o = 0; o < TO; o++) {
            float v[4];
            result(o, t, v);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                acc[0][o][t][e] = v[e];
                if (row0 + wr0 + 16 * o < a.rows) m = max(m, f8_mag(v[e]));
            }
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
        if (g == 0) mags[ww][(wx * TX + t) * 16 + r] = m;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TX; t++) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < WPB; i++) m = max(m, mags[ww / WPB * WPB + i][(wx * TX + t) * 16 + r]);
        const float s = f8_scale(m), inv = 1.0f / s;
        const int yr = y_row(t);
        if (yr < 0) continue;
        if (ww % WPB == 0 && g == 0 && row0 + wr0 < a.rows)
            a.ys[yr * a.ys_stride + (row0 + wr0) / F8_BLOCK] = s;
#pragma unroll
        for (int o = 0; o < TO; o++) {
            const int row = row0 + wr0 + 16 * o + 4 * g;
            if (row < a.rows)
                *reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(a.y) + yr * a.y_stride + row) =
                    f8_pack4(acc[0][o][t][0], acc[0][o][t][1], acc[0][o][t][2], acc[0][o][t][3], inv);
        }
    }
}

template <int NWW, int NWX, int TO, int TX, bool GLU, bool FAST>
int launch_tile(const F8Args &a, hipStream_t st)
{
    constexpr int OR = 16 * NWW * TO, BX = 16 * NWX * TX;
    const int64_t n_wt = (a.rows + OR - 1) / OR;
    // groups: a tile more for each that ends inside one
    const int64_t n_xt = a.G ? a.T / BX + (a.G < a.T ? a.G : a.T) : (a.T + BX - 1) / BX;
    const int64_t total = n_wt * n_xt;
    BREAD_REQUIRE(total <= 1 << 23, BREAD_ERR_SHAPE, "more tiles than a launch takes");
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_f8_tile<NWW, NWX, TO, TX, GLU, FAST>), dim3((unsigned)((total + 7) / 8 * 8)),
                       dim3(NWW * NWX * WAVE), 0, st, a, (int)n_wt, (int)total);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

}  // namespace

int bread_launch_fp8_matmul(const F8Args &a, hipStream_t st)
{
    return a.up ? launch_tile<4, 1, 2, 4, true, false>(a, st) : launch_tile<4, 1, 2, 4, false, false>(a, st);
}

// ---------------------------------------------------------------------------
// Entry points
// ---------------------------------------------------------------------------

#define F8_REQUIRE(cond, status, detail)                                     \
    do {                                                                     \
        if (!(cond)) return bread_fail((status), where, (detail));           \
    } while (0)

// where: the entry point; none: a call without any groups
static int check_matmul(const char *where, const bread_matmul_fp8_t &o, bool none, F8Args &a)
{
    F8_REQUIRE(o.rows >= 0 && o.cols > 0 && o.n_tokens >= 0, BREAD_ERR_ARG,
               "rows and n_tokens must be >= 0 and cols > 0");
    F8_REQUIRE(f8_wide_type(o.y_type) || o.y_type == BREAD_QTYPE_E4M3, BREAD_ERR_QTYPE,
               "y_type must be 0 (F32), 1 (F16), 30 (BF16) or 0x1000 (E4M3)");
    F8_REQUIRE(o.act >= BREAD_ACT_NONE && o.act <= BREAD_ACT_RELU, BREAD_ERR_ARG, "unknown activation");
    F8_REQUIRE(o.cols % 16 == 0, BREAD_ERR_SHAPE, "cols must be a multiple of 16");
    F8_REQUIRE(o.cols <= 1 << 20 && o.rows <= 1 << 24 && o.n_tokens <= 1 << 24, BREAD_ERR_SHAPE,
               "cols above 2^20, or rows or n_tokens above 2^24");
    const bool q = o.y_type == BREAD_QTYPE_E4M3;
    const int64_t nb = f8_blocks(o.cols), nr = f8_blocks(o.rows);
    a.x_stride = o.x_stride ? o.x_stride : o.cols;
    a.xs_stride = o.x_scale_stride ? o.x_scale_stride : nb;
    a.y_stride = o.y_stride ? o.y_stride : o.rows;
    a.ys_stride = o.y_scale_stride ? o.y_scale_stride : nr;
    F8_REQUIRE(a.x_stride >= o.cols && a.xs_stride >= nb && a.y_stride >= o.rows && (!q || a.ys_stride >= nr),
               BREAD_ERR_SHAPE, "a stride is smaller than a token's row");
    F8_REQUIRE(!q || o.rows % 16 == 0, BREAD_ERR_SHAPE, "rows must be a multiple of 16 for quantised results");
    F8_REQUIRE(!q || !o.residual, BREAD_ERR_ARG, "quantised results take no residual");
    F8_REQUIRE(!o.up || !o.bias, BREAD_ERR_ARG, "a gated product takes no bias");
    if (o.rows == 0 || o.n_tokens == 0 || none) return BREAD_OK;
    F8_REQUIRE(o.w && o.w_scale && o.x && o.x_scale && o.y && (!o.up || o.up_scale) && (!q || o.y_scale),
               BREAD_ERR_ARG, "NULL pointer");
    F8_REQUIRE((((uintptr_t)o.w | (uintptr_t)o.up | (uintptr_t)o.x) & 15) == 0 && a.x_stride % 16 == 0,
               BREAD_ERR_ALIGN, "w, up and x must be 16-byte aligned and x's stride a multiple of 16");
    F8_REQUIRE(!q || (((uintptr_t)o.y & 15) == 0 && a.y_stride % 16 == 0), BREAD_ERR_ALIGN,
               "quantised y must be 16-byte aligned and its stride a multiple of 16");
    const uintptr_t ya = f8_type_bytes(o.y_type) - 1;
    F8_REQUIRE((((uintptr_t)o.y | (uintptr_t)o.residual) & ya) == 0 &&
                   (((uintptr_t)o.bias | (uintptr_t)o.w_scale | (uintptr_t)o.up_scale | (uintptr_t)o.x_scale |
                     (uintptr_t)o.y_scale) & 3) == 0,
               BREAD_ERR_ALIGN, "y, residual, bias and scales must be aligned to their elements");
    a.w = static_cast<const uint8_t *>(o.w);
    a.up = static_cast<const uint8_t *>(o.up);
    a.x = static_cast<const uint8_t *>(o.x);
    a.ws = o.w_scale;
    a.us = o.up_scale;
    a.xs = o.x_scale;
    a.y = o.y;
    a.ys = o.y_scale;
    a.bias = o.bias;
    a.res = o.residual;
    a.rows = o.rows;
    a.cols = o.cols;
    a.T = o.n_tokens;
    a.act = o.act;
    a.y_type = o.y_type;
    a.G = 0;
    a.offsets = a.x_rows = a.y_rows = nullptr;
    a.n_x = a.n_y = 0;
    return BREAD_OK;
}

extern "C" int bread_matmul_fp8(const bread_matmul_fp8_t *args, bread_stream_t stream)
{
    BREAD_REQUIRE(args, BREAD_ERR_ARG, "NULL arguments");
    F8Args a;
    const int rc = check_matmul("bread_matmul_fp8", *args, false, a);
    if (rc || args->rows == 0 || args->n_tokens == 0) return rc;
    return bread_launch_fp8_matmul(a, to_hip(stream));
}

extern "C" int bread_matmul_fp8_grouped(const bread_matmul_fp8_t *args, const bread_fp8_groups_t *groups,
                                        bread_stream_t stream)
{
    BREAD_REQUIRE(args && groups, BREAD_ERR_ARG, "NULL arguments");
    BREAD_REQUIRE(groups->n_groups >= 0 && (!groups->x_rows || groups->n_x >= 0) &&
                      (!groups->y_rows || groups->n_y >= 0),
                  BREAD_ERR_ARG, "n_groups, n_x and n_y must be >= 0");
    BREAD_REQUIRE(groups->n_groups <= 1024, BREAD_ERR_SHAPE, "n_groups above 1024");
    BREAD_REQUIRE(!args->bias && !args->residual, BREAD_ERR_ARG, "grouped products take no bias and no residual");
    F8Args a;
    const int rc = check_matmul("bread_matmul_fp8_grouped", *args, groups->n_groups == 0, a);
    if (rc || args->rows == 0 || args->n_tokens == 0 || groups->n_groups == 0) return rc;
    BREAD_REQUIRE(groups->offsets, BREAD_ERR_ARG, "NULL offsets");
    BREAD_REQUIRE((((uintptr_t)groups->offsets | (uintptr_t)groups->x_rows | (uintptr_t)groups->y_rows) & 3) == 0,
                  BREAD_ERR_ALIGN, "offsets and rows must be 4-byte aligned");
    a.G = groups->n_groups;
    a.offsets = groups->offsets;
    a.x_rows = groups->x_rows;
    a.y_rows = groups->y_rows;
    a.n_x = groups->n_x;
    a.n_y = groups->n_y;
    return bread_launch_fp8_matmul(a, to_hip(stream));
}
