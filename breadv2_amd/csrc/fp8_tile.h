// fp8_tile.h — the kernel of bread_matmul_fp8 and bread_matmul_fp8_grouped:
//   v[t][r] = sum_b xs[t][b] ws[r / 128][b] sum_{c in b} x[t][c] w[r][c]
// for tokens t and weight rows r, with the epilogue y = act(v + bias) [* v_up] + residual,
// rounded to fp16, bf16 or fp32, or quantised again by blocks of 128 rows.
//
// A block's products are summed in fp32 by matrix instructions from zero, and
// the product of the two scales is applied to that sum: one fused multiply-add
// a block of 128 columns and element of y.
// That product is fp32's: a number below 2^128, with fewer bits below 2^-126 (a sum
// is below 2^25, so a block's part is off by 2^-125 at most).  The header says so.
// Blocks beyond by sums in 64 bits were built and not kept: a test a block costs
// ordinary calls 2 to 5 %, one a tile up to 2 %, and with a second path for the
// sums it is 1 to 25 %, by the registers that the path takes.
#pragma once

#include "activate.h"
#include "fp8.h"

namespace {

typedef f8_f32x4 f32x4;
typedef f8_half8 h8;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Bytes that a buffer of activations holds at most, and an offset beyond every buffer
constexpr uint32_t BEYOND = 1u << 31;

// All of this wave's loads have landed (in registers or LDS)
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0); lgkmcnt and expcnt at their maxima
    __builtin_amdgcn_sched_barrier(0);
}

// A buffer: its first byte, and the bytes from which on loads give zeros
typedef uint32_t Buffer __attribute__((ext_vector_type(4)));

__device__ __forceinline__ Buffer buffer(const void *p, uint32_t bytes)
{
    const uint64_t at = uniform64(reinterpret_cast<uint64_t>(p));
    return Buffer{(uint32_t)at, (uint32_t)(at >> 32) & 0xffff, (uint32_t)uniform((int)bytes), BUF_WORD3};
}

// Loads to LDS, 4 or 16 bytes a lane, which lie behind one another from `to` on.  (Written out: of the builtin's loads the
// compiler doesn't see which buffer they fill, and waits for those in flight before any read of LDS.  Nothing but LDS is
// written.  The five wait states are those between a vector instruction that writes a scalar register and a load that reads
// it.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0, which nothing else here uses)
template <int BYTES>
__device__ __forceinline__ void load_lds(const Buffer &b, uint32_t to, uint32_t off, uint32_t soff)
{
    to = (uint32_t)uniform((int)to), soff = (uint32_t)uniform((int)soff);
    asm("" : "+s"(soff));  // a register, also of a constant
    const Buffer u{(uint32_t)uniform((int)b[0]), (uint32_t)uniform((int)b[1]), (uint32_t)uniform((int)b[2]),
                   (uint32_t)uniform((int)b[3])};
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(u), "s"(soff) : "m0", "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(u), "s"(soff) : "m0", "memory");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_at(const void *p)
{
    return (uint32_t)uniform((int)(uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p);
}

// A barrier for what lies in LDS, which leaves loads in flight (__syncthreads waits for them)
__device__ __forceinline__ void barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0); vmcnt and expcnt at their maxima
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The 128 columns of a row that a lane holds, 32 codes in eight words: which of the row's columns they are is free as
// long as weights and activations agree.  PARTS matrix instructions take them.  FAST: the codes themselves.  Else they are
// widened (exactly) to fp16, two at a time in STEPS steps.
template <bool FAST> struct Frag;

template <> struct Frag<true> {
    static constexpr int PARTS = 1, STEPS = 0;
    i32x8 v;
    __device__ __forceinline__ void begin(const uint4 &a, const uint4 &b)
    {
        v = i32x8{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    }
    __device__ __forceinline__ void step(int) {}
    // z: weight rows 4 (l / 16) + i of lane l in element i, token l % 16
    static __device__ __forceinline__ f32x4 product(const Frag &w, const Frag &x, int, const f32x4 &z)
    {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, z, 0, 0, 0, 0, 0, 0);
    }
};

template <> struct Frag<false> {
    static constexpr int PARTS = 4, STEPS = 16;
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    uint32_t q[8];
    Words v[4];
    __device__ __forceinline__ void begin(const uint4 &a, const uint4 &b)
    {
        q[0] = a.x, q[1] = a.y, q[2] = a.z, q[3] = a.w, q[4] = b.x, q[5] = b.y, q[6] = b.z, q[7] = b.w;
    }
    __device__ __forceinline__ void step(int i)
    {
        const int w = (int)q[i / 2];
        v[i / 4][i % 4] = __builtin_bit_cast(uint32_t, i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    }
    static __device__ __forceinline__ f32x4 product(const Frag &w, const Frag &x, int k, const f32x4 &z)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, w.v[k]), __builtin_bit_cast(h8, x.v[k]), z, 0, 0, 0);
    }
};

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

// ---------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------
// A workgroup takes tiles of 16 TX NWX tokens by OR weight rows (of one or two matrices).  Its columns come in stages of
// KSB blocks of 128, by loads to LDS that are one stage ahead, across the tiles' ends too where it takes several (KEEP).
// Rows lie 128 bytes apart, the eight pieces of 16 bytes of row r at piece ^ (r % 8), so that a read of a piece of 16 rows
// covers the banks.  NWW x NWX waves have TO row tiles by TX token tiles each; NWK such sets of waves share a stage's
// blocks and add their sums in the last stage's place.
//
// FAST, the 8-bit matrix instructions: they cut products more than 2^13 below the largest of their eight, which is
// 1.5e-5 to 2.3e-5 of a result (rms): a fourteenth to a ninth of fp16's own rounding, which is 2.1e-4, and a hundredth to a
// seventieth of bf16's.  Not for fp32 results, nor for e4m3, whose scales are fp32, nor for a few tokens, which wait for
// loads.  Else the codes are widened to fp16 (exact, and their products sum in fp32).
//
// What bounds them.  A compute unit's four SIMDs take an fp16 instruction of 16 x 16 x 32 in 16 cycles, and a widening,
// a scaled addition or any other vector instruction in 4 to 5; the widenings are 16 (N + TX), the additions 4 N TX of
// 4 N TX matrix instructions, so a wave's tiles want to be many and square: N, TX = 4 is what 256 registers hold.
// Measured over long columns, 4096 tokens: exact 1.25 PFLOP/s (the library's bf16 product of 8192^3: 1.37), FAST 1.85.
// Of an exact stage's 1.78 us (128 x 128 x 128 twice on a compute unit) the matrix instructions alone take 0.94, with the
// reads of LDS 1.23, with widening and scaling 1.37, and the loads to LDS add 0.42.  Of a FAST stage's 128 x 128 x 128 the
// matrix instructions are 512 cycles a SIMD and the scaled additions some 300, but LDS is busy for 768 (at 128 bytes a
// cycle): four waves of 64 x 64 read 64 KB, and 32 KB are written.  Larger wave tiles would read less.
// Forms that take tiles in turn keep more than the scalar registers hold: those of groups spill 36 to 92 of them to lanes
// (92: gated, 128 x 128), those of one matrix 10 to 36; those that take one tile none.  In the loop over the blocks that
// is five lane reads at most, beside 64 matrix and some 210 vector instructions.  Around its stages a tile costs 5 to
// 8 us of lookups, first loads and results, or those of the results where a workgroup takes the next one meanwhile.
// Tried and not kept: three stages (no faster: it is not latency), tokens widened once and shared as fp16 through LDS (the
// same), the loads spread over a stage's products (slower by 6 to 17 %), columns that begin elsewhere for each tile (5 %:
// weights are shared in step), a wave's token tiles one after the other, for wider tiles (15 %), forms that skip the token
// tiles of a group's rest that hold none (registers: 10 %), a group's rests behind all full tiles (2 %), a tile's residuals read together before its first store (4096 tokens, 8192 x
// 2048 to bf16 125 to 111 us, but 500, 4096 x 512 to fp16 11.7 to 16.4, and 4096 without a residual 89 to 92).

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

constexpr int GROUPS_MAX = 1024;

// begin[g]: the groups' first rows, tiles[g]: token tiles of the groups before g, for g <= G
template <int THREADS>
__device__ __forceinline__ void count_tiles(const F8Args &a, int bx, int *begin, uint32_t *tiles, int *sums)
{
    for (int g = (int)threadIdx.x; g <= a.G; g += THREADS) begin[g] = min(max(a.offsets[g], 0), a.T);
    __syncthreads();
    const int per = (a.G + THREADS - 1) / THREADS, g0 = (int)threadIdx.x * per;
    auto of = [&](int g) __attribute__((always_inline)) { return (uint32_t)((max(begin[g + 1] - begin[g], 0) + bx - 1) / bx); };
    uint32_t mine = 0;
    for (int g = g0; g < min(g0 + per, a.G); g++) mine += of(g);
    const uint32_t incl = (uint32_t)wave_scan_incl((int)mine);
    if (lane_id() == WAVE - 1) sums[threadIdx.x / WAVE] = (int)incl;
    __syncthreads();
    uint32_t before = incl - mine;
    for (int i = 0; i < (int)threadIdx.x / WAVE; i++) before += (uint32_t)sums[i];
    for (int g = g0; g < min(g0 + per, a.G); g++) {
        tiles[g] = before;
        before += of(g);
    }
    if (g0 < a.G && g0 + per >= a.G) tiles[a.G] = before;
    __syncthreads();
}

// LDS of a workgroup but for the stages
template <class S, bool GRP> struct Lds {
    int begin[GRP ? GROUPS_MAX + 1 : 1], scan[S::WAVES];
    uint32_t tiles[GRP ? GROUPS_MAX + 1 : 1];
};

template <class S, int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, bool KEEP, bool GRP>
__device__ __forceinline__ void run_tiles(const F8Args &a, const int n_wt, int n_xt, Lds<S, GRP> &lds, uint8_t *buf)
{
    constexpr int M = S::M, N = S::N, OR = S::OR, BX = S::BX, WR = S::WR, PASS = S::PASS;
    const int tid = (int)threadIdx.x, wv = wave_id(), l = lane_id();
    const int wk = wv / (NWW * NWX), ww = wv % NWW, wx = wv / NWW % NWX;
    const int r = l & 15, g = l >> 4, nb = f8_blocks(a.cols), nrb = f8_blocks(a.rows), steps = (nb + KSB - 1) / KSB;
    if constexpr (GRP) {
        count_tiles<S::THREADS>(a, BX, lds.begin, lds.tiles, lds.scan);
        // (n_xt: as many as offsets that ascend can give; others are held to it)
        n_xt = (int)min((uint32_t)uniform((int)lds.tiles[a.G]), (uint32_t)n_xt);
    }
    // consecutive tiles on one XCD, whose workgroups then share an L2
    const int total = n_xt * n_wt, per = (total + 7) / 8, stride = (int)gridDim.x / 8, xcd = (int)blockIdx.x % 8;
    const int end = min(per * (xcd + 1), total);
    int tile = per * xcd + (int)blockIdx.x / 8;
    if (tile >= end) return;

    // where tile i lies; from: a group that is not behind it
    auto place = [&](int i, int from) __attribute__((always_inline)) {
        Place p;
        if constexpr (GRP) {
            // the last group with no more than xt tiles before it, 64 groups at a time
            const int xt = i / n_wt;
            int lo = from;
            for (;;) {
                const int ahead = lo + 1 + l;
                const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(ahead < a.G && lds.tiles[ahead] <= (uint32_t)xt));
                lo += n;
                if (n < WAVE) break;
            }
            p.g = lo;
            // (held to the call's rows also where offsets fall)
            p.p0 = uniform(min(lds.begin[lo] + max(xt - (int)lds.tiles[lo], 0) * BX, a.T));
            p.n = uniform(max(min(lds.begin[lo + 1] - p.p0, BX), 0));
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
    Buffer wb, ub, xb, xsb, wsb, usb;
    int srb0 = 0, xrow[S::PX], xsrow = -1;
    // x rows of the tile rows that the thread loads, -1 for none
    auto look = [&](const Place &p) __attribute__((always_inline)) {
        auto x_row = [&](int i) __attribute__((always_inline)) {
            if (i >= p.n) return -1;
            if (!GRP || !a.x_rows) return i;
            return a.x_rows[p.p0 + i];
        };
#pragma unroll
        for (int i = 0; i < S::PX; i++) {
            const int at = i * PASS + srow;
            xrow[i] = KSB * BX % PASS && at >= KSB * BX ? -1 : x_row(at % BX);
        }
        if (wv < S::NXS) xsrow = x_row(wv % S::XSW * WAVE + l);
    };
    auto aim = [&](const Place &p) __attribute__((always_inline)) {
        const uint32_t bytes = (uint32_t)min(OR, a.rows - p.row0) * (uint32_t)a.cols;
        const size_t first = ((size_t)p.g * a.rows + p.row0) * a.cols, scale = (size_t)p.g * nrb * nb;
        const int64_t xr0 = GRP && a.x_rows ? 0 : p.p0;  // x row that offsets count from
        const int n_x = GRP && a.x_rows ? a.n_x : a.T;
        wb = buffer(a.w + first, bytes);
        ub = buffer(GLU ? a.up + first : a.w + first, bytes);
        wsb = buffer(a.ws + scale, 4u * (uint32_t)nrb * (uint32_t)nb);
        usb = buffer(GLU ? a.us + scale : a.ws + scale, 4u * (uint32_t)nrb * (uint32_t)nb);
        xb = buffer(a.x + xr0 * a.x_stride, BEYOND);
        xsb = buffer(a.xs + xr0 * a.xs_stride, BEYOND);
        srb0 = p.row0 / F8_BLOCK;
#pragma unroll
        for (int i = 0; i < S::PX; i++)
            xoff[i] = (unsigned)xrow[i] < (unsigned)n_x ? (uint32_t)xrow[i] * (uint32_t)a.x_stride + 16 * piece : BEYOND;
        xsoff = (unsigned)xsrow < (unsigned)n_x ? 4u * (uint32_t)xsrow * (uint32_t)a.xs_stride : BEYOND;
    };
    uint32_t woff[S::PW];
#pragma unroll
    for (int i = 0; i < S::PW; i++) woff[i] = (uint32_t)((i * PASS + srow) % OR) * (uint32_t)a.cols + 16 * piece;
    auto stage = [&](uint32_t to, int step) __attribute__((always_inline)) {
        const uint32_t b = to + wv * 8 * F8_BLOCK;
        const int k0 = step * KSB * F8_BLOCK;
#pragma unroll
        for (int i = 0; i < (S::NXS + S::WAVES - 1) / S::WAVES; i++) {
            const int j = wv + i * S::WAVES, kb = step * KSB + j / S::XSW;  // (a wave's loads are of the same tokens)
            if (j < S::NXS) load_lds<4>(xsb, to + S::XS_AT + 4 * j * WAVE, kb < nb ? xsoff : BEYOND, kb < nb ? 4 * kb : 0);
        }
        if (wv == S::WAVES - 1) {
            const int kb = step * KSB + l / S::OB, rb = srb0 + l % S::OB;
            const uint32_t off = l < KSB * S::OB && kb < nb && rb < nrb ? 4u * (uint32_t)(rb * nb + kb) : BEYOND;
            load_lds<4>(wsb, to + S::WS_AT, off, 0);
            if constexpr (GLU) load_lds<4>(usb, to + S::WS_AT + 4 * WAVE, off, 0);
        }
#pragma unroll
        for (int i = 0; i < S::PW; i++) {
            const int kk = i * PASS / WR, row = i * PASS % WR;  // (PASS divides WR or is a multiple of it)
            const int c = k0 + (PASS > WR ? (i * PASS + srow) / WR : kk) * F8_BLOCK;
            const uint32_t off = c + 16 * piece < a.cols ? woff[i] + (PASS > WR ? c - k0 : 0) : BEYOND;
            // (a block behind the last column: from the buffer's start, for a scalar offset beyond a short buffer would be
            // taken from its size)
            const int first = PASS > WR ? k0 : k0 + kk * F8_BLOCK, soff = first < a.cols ? first : 0;
            // (a wave's eight rows are of one matrix)
            if (!GLU || (PASS <= OR ? row < OR : wv * 8 % WR < OR))
                load_lds<16>(wb, b + i * PASS * F8_BLOCK, off, soff);
            else
                load_lds<16>(ub, b + i * PASS * F8_BLOCK, off, soff);
        }
#pragma unroll
        for (int i = 0; i < S::PX; i++) {
            if (KSB * BX % PASS && i * PASS + wv * 8 >= KSB * BX) break;
            const int c = (i * PASS + srow) / BX * F8_BLOCK;
            const uint32_t off = k0 + c + 16 * piece < a.cols && xoff[i] != BEYOND ? xoff[i] + c : BEYOND;
            load_lds<16>(xb, b + S::W_BYTES + i * PASS * F8_BLOCK, off, k0);
        }
    };
    // -------------------------------------------------------------- products
    f32x4 acc[N][TX];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int t = 0; t < TX; t++) acc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    const int wr0 = 16 * TO * ww;  // the wave's first row in the tile
    const int at0 = r * F8_BLOCK + 16 * (g ^ (r & 7)), at1 = at0 ^ 64;
    // Block kk of a stage.  Each matrix instruction is followed by vector instructions that take about its time: the next
    // row tile is widened and the last one's sums are scaled and added meanwhile.  (The compiler would put them in rows of
    // one kind, and a SIMD's two waves, which a barrier lets go together, both wait.  Token tiles that hold no tokens are
    // multiplied too: forms of fewer cost the registers that let a workgroup load its next tile ahead.)
    auto multiply = [&](const uint8_t *__restrict__ b, int kk) __attribute__((always_inline)) {
        using F = Frag<FAST>;
        auto frag = [&](F &f, const uint8_t *__restrict__ p) __attribute__((always_inline)) {
            f.begin(*reinterpret_cast<const uint4 *>(p + at0), *reinterpret_cast<const uint4 *>(p + at1));
        };
        auto weights = [&](F &f, int i) __attribute__((always_inline)) {
            frag(f, b + (kk * WR + i / TO * OR + wr0 + 16 * (i % TO)) * F8_BLOCK);
        };
        F x[TX], w[N];
        float xs[TX], ws[M];
        weights(w[0], 0);
#pragma unroll
        for (int t = 0; t < TX; t++) frag(x[t], b + S::W_BYTES + (kk * BX + 16 * (t * NWX + wx)) * F8_BLOCK);
        if constexpr (N > 1) weights(w[1], 1);
#pragma unroll
        for (int t = 0; t < TX; t++)
            xs[t] = *reinterpret_cast<const float *>(b + S::XS_AT + 4 * (kk * S::XSW * WAVE + 16 * (t * NWX + wx) + r));
#pragma unroll
        for (int m = 0; m < M; m++)
            ws[m] = *reinterpret_cast<const float *>(b + S::WS_AT + 4 * (m * WAVE + kk * S::OB + wr0 / F8_BLOCK));
        f32x4 z[2][TX];
        float s = 0.f;
        auto add = [&](int i, int j) __attribute__((always_inline)) {  // element j of the row tile's 4 TX
            const int t = j / 4, e = j % 4;
            if (e == 0) s = xs[t] * ws[i / TO];
            acc[i][t][e] = fmaf(s, z[i & 1][t][e], acc[i][t][e]);
        };
        constexpr int ALL = F::PARTS * TX;  // matrix instructions of a row tile
        auto widen = [&](int n) __attribute__((always_inline)) {  // what the n-th of them takes of the tokens
#pragma unroll
            for (int j = 0; j < F::STEPS / F::PARTS; j++) x[n % TX].step(n / TX * F::STEPS / F::PARTS + j);
        };
#pragma unroll
        for (int j = 0; j < F::STEPS; j++) w[0].step(j);
        widen(0);
        if (!GRP) __builtin_amdgcn_s_setprio(1);  // ahead of the other wave's loads: 2 to 5 % (of groups none)
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int n = 0; n < ALL; n++) {
                const int k = n / TX, t = n % TX;
                if (i + 2 < N && n == ALL / 2) weights(w[i + 2], i + 2);
                z[i & 1][t] = F::product(w[i], x[t], k, k ? z[i & 1][t] : f32x4{0.f, 0.f, 0.f, 0.f});
                if (i == 0 && n + 1 < ALL) widen(n + 1);
                if (i + 1 < N) {
#pragma unroll
                    for (int j = n * F::STEPS / ALL; j < (n + 1) * F::STEPS / ALL; j++) w[i + 1].step(j);
                }
                if (i) {
#pragma unroll
                    for (int j = n * 4 * TX / ALL; j < (n + 1) * 4 * TX / ALL; j++) add(i - 1, j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int j = 0; j < 4 * TX; j++) add(N - 1, j);
        if (!GRP) __builtin_amdgcn_s_setprio(0);
    };

    // -------------------------------------------------------------- results
    // spare: the last stage's buffer, for sums and magnitudes
    auto finish = [&](const Place &p, uint8_t *spare) __attribute__((always_inline)) {
        if constexpr (NWK > 1) {
            f32x4 *part = reinterpret_cast<f32x4 *>(spare);
            constexpr int W = NWW * NWX;
            barrier();  // all have read the last stage
            if (wk) {
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int t = 0; t < TX; t++) part[(((wv - W) * N + i) * TX + t) * WAVE + l] = acc[i][t];
            }
            barrier();
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
        // act(v + bias) [* v_up] in acc[0 .. TO - 1]; the kind of activation outside of the loops: its code once a value
        auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int o = 0; o < TO; o++)
#pragma unroll
                for (int t = 0; t < TX; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[o][t][e] = f(acc[o][t][e], o, t, e);
        };
        if (wk == 0) {
            if (!GLU && a.bias) {
                float bias[TO][4];
#pragma unroll
                for (int o = 0; o < TO; o++)
#pragma unroll
                    for (int e = 0; e < 4; e++) bias[o][e] = a.bias[min(p.row0 + wr0 + 16 * o + 4 * g + e, a.rows - 1)];
                each([&](float v, int o, int, int e) __attribute__((always_inline)) { return v + bias[o][e]; });
            }
            switch (a.act) {
            case BREAD_ACT_SILU:
                each([](float v, int, int, int) __attribute__((always_inline)) { return activate(v, BREAD_ACT_SILU); });
                break;
            case BREAD_ACT_GELU:
                each([](float v, int, int, int) __attribute__((always_inline)) { return activate(v, BREAD_ACT_GELU); });
                break;
            case BREAD_ACT_GELU_TANH:
                each([](float v, int, int, int) __attribute__((always_inline)) { return activate(v, BREAD_ACT_GELU_TANH); });
                break;
            case BREAD_ACT_RELU:
                each([](float v, int, int, int) __attribute__((always_inline)) { return activate(v, BREAD_ACT_RELU); });
                break;
            }
            if constexpr (GLU)
                each([&](float v, int o, int t, int e) __attribute__((always_inline)) { return v * acc[N - TO + o][t][e]; });
        }
        const bool quantised = OR % F8_BLOCK == 0 && a.y_type == BREAD_QTYPE_E4M3;
        if (!quantised) {
            if (wk == 0) {
#pragma unroll
                for (int t = 0; t < TX; t++) {
                    const int yr = y_row(t);
#pragma unroll
                    for (int o = 0; o < TO; o++) {
                        const int row = p.row0 + wr0 + 16 * o + 4 * g;
                        const float v[4] = {acc[o][t][0], acc[o][t][1], acc[o][t][2], acc[o][t][3]};
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
                uint32_t(*mags)[BX] = reinterpret_cast<uint32_t(*)[BX]>(spare + S::SUMS);
                static_assert(S::SUMS + 4 * NWW * BX <= S::STAGE, "fits");
                if (NWK == 1) barrier();  // all have read the last stage
                if (wk == 0) {
#pragma unroll
                    for (int t = 0; t < TX; t++) {
                        uint32_t m = 0;
#pragma unroll
                        for (int o = 0; o < TO; o++) {
                            if (p.row0 + wr0 + 16 * o >= a.rows) break;
#pragma unroll
                            for (int e = 0; e < 4; e++) m = max(m, f8_mag(acc[o][t][e]));
                        }
                        m = max(m, (uint32_t)__shfl_xor((int)m, 16));
                        m = max(m, (uint32_t)__shfl_xor((int)m, 32));
                        if (g == 0) mags[ww][16 * (t * NWX + wx) + r] = m;
                    }
                }
                barrier();
                if (wk == 0) {
#pragma unroll
                    for (int t = 0; t < TX; t++) {
                        uint32_t m = 0;
#pragma unroll
                        for (int i = 0; i < WPB; i++) m = max(m, mags[ww / WPB * WPB + i][16 * (t * NWX + wx) + r]);
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

    // Stages of columns are loaded one ahead of the products, over the ends of tiles too; a tile's x rows are looked
    // up while the one before is loaded.
    const uint32_t at = lds_at(buf);
    Place now = place(tile, 0), next = now, after = now;
    int ltile = tile, lstep = 0;  // the next stage to load
    int b = 0, lb = 0;            // buffers
    bool begun = false;
    look(now);
    aim(now);
    if (KEEP && tile + stride < end) {
        after = place(tile + stride, now.g);
        look(after);
    }
    auto load = [&]() __attribute__((always_inline)) {
        if (ltile >= end) return;
        if (KEEP && lstep == 0 && begun) {
            next = after;
            aim(next);
            if (ltile + stride < end) {
                after = place(ltile + stride, next.g);
                look(after);
            }
        }
        begun = true;
        stage(at + lb * S::STAGE, lstep);
        lb ^= 1;
        if (++lstep == steps) {
            lstep = 0;
            ltile = KEEP ? ltile + stride : end;
        }
    };
    for (bool first = true; tile < end; tile = KEEP ? tile + stride : end) {
        clear();
        bool any = true;  // whether the wave has tokens
        for (int i = first ? -1 : 0; i < steps; i++) {
            if (i >= 0) {
                wait_loads();
                barrier();
            }
            load();
            if (i < 0) continue;
            if (GRP && NWX > 1 && i == 0) any = now.n > 16 * wx;
            const uint8_t *cur = buf + b * S::STAGE;
            b ^= 1;
#pragma unroll
            for (int k = 0; k < S::KPW; k++) {
                const int kk = wk + k * NWK;
                if (i * KSB + kk >= nb) break;
                if (any) multiply(cur, kk);
            }
        }
        first = false;
        finish(now, buf + (b ^ 1) * S::STAGE);  // (nothing is loaded yet to the last stage's buffer)
        now = next;
    }
}

// (a kernel that is a template and holds buffer descriptors itself is dropped by the host's compilation)
template <int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, int WPE, bool KEEP, bool GRP>
__global__ __launch_bounds__(NWW * NWX * NWK * WAVE, WPE) void k_f8_matmul(const F8Args a, const int n_wt, const int n_xt)
{
    using S = Shape<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST>;
    __shared__ Lds<S, GRP> lds;
    __shared__ __attribute__((aligned(16))) uint8_t buf[2 * S::STAGE];
    run_tiles<S, NWW, NWX, NWK, TO, TX, KSB, GLU, FAST, KEEP, GRP>(a, n_wt, n_xt, lds, buf);
}

constexpr int64_t CUS = 256;  // compute units

// WPE: waves a SIMD, which the registers are held to; KEEP: workgroups take tiles in turn
template <int NWW, int NWX, int NWK, int TO, int TX, int KSB, bool GLU, bool FAST, int WPE, bool KEEP, bool GRP>
int launch(const F8Args &a, hipStream_t st)
{
    using S = Shape<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST>;
    constexpr int lds = (int)sizeof(Lds<S, GRP>) + 2 * S::STAGE;
    constexpr int by_lds = 160 * 1024 / lds, by_waves = 4 * WPE / S::WAVES, resident = by_lds < by_waves ? by_lds : by_waves;
    static_assert(resident >= 1, "a workgroup fits");
    BREAD_REQUIRE(GLU == (a.up != nullptr) && GRP == (a.G > 0) && (a.y_type != BREAD_QTYPE_E4M3 || S::OR % F8_BLOCK == 0), BREAD_ERR_SHAPE,
                  "a kernel for other results");
    const int64_t n_wt = (a.rows + S::OR - 1) / S::OR;
    // groups: a tile more for each that ends inside one
    const int64_t n_xt = GRP ? a.T / S::BX + (a.G < a.T ? a.G : a.T) : (a.T + S::BX - 1) / S::BX;
    const int64_t total = n_wt * n_xt, most = KEEP ? CUS * resident : 1 << 22;
    BREAD_REQUIRE(total <= (KEEP ? 1 << 30 : 1 << 22), BREAD_ERR_SHAPE, "more tiles than a launch counts");
    bread_clear_stale_error();
    hipLaunchKernelGGL((k_f8_matmul<NWW, NWX, NWK, TO, TX, KSB, GLU, FAST, WPE, KEEP, GRP>),
                       dim3((unsigned)((total < most ? total : most) + 7) / 8 * 8), dim3(S::THREADS), 0, st, a, (int)n_wt,
                       (int)n_xt);
    BREAD_HIP(hipGetLastError());
    return BREAD_OK;
}

}  // namespace
