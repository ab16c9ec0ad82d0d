// fp8_matmul.hip — bread_matmul_fp8 and bread_matmul_fp8_grouped: arguments,
// and the forms of fp8_tile.h's kernel for one matrix.  (Groups: fp8_grouped.hip.)
#include <algorithm>

#include "fp8_tile.h"

namespace {

// The tiles are those that give a compute unit the fewest rows of weights and tokens to load, over all its tiles: a unit
// has about 40 KB of loads under way, which is 40 KB a microsecond, and that is what all but the largest calls wait for.
// us and rows of a unit for tiles of 16, 32, 48, 64 tokens by 32 rows, 64 by 64 and 128 by 128 (bf16 results):
//   24 tokens, 2048 x 4096    7.2 (48)   9.3 (64)  11.1 (80)  12.2 (96)  17.4 (128)  24.7 (256)
//   40, 8192 x 2048          11.7 (144) 11.6 (128)  8.5 (80)   8.9 (96)  11.3 (128)  15.5 (256)
//   131, 2048 x 4096         17.2 (144) 16.7 (128) 11.6 (80)  12.8 (96)  17.5 (128)  26.1 (256)
//   500, 2048 x 4096         39.9 (384) 30.8 (256) 29.5 (240) 23.5 (192) 18.4 (128)  26.8 (256)
//   700, 4096 x 2048         64.5       48.1       45.4       37.9       28.7 (384)  17.5 (256)
// and 16, 32 and 128 tokens by 128 rows, to e4m3, where a workgroup needs whole blocks:
//   131, 2048 x 4096         17.1 (144) 21.4 (160) 39.3 (256);    500: 30.6 (288) 22.5 (160) 39.5 (256)
//   700, 4096 x 2048         49.1 (864) 35.5 (480) 24.6 (256)
// (gated alike; of 44 measured calls the rule took the fastest form each time).  Small tiles have two to four sets of waves
// by columns: 9 tokens, 8192 x 2048 5.9 with four, 7.6 with eight.  The largest, 4096 tokens, 8192 x 2048 to bf16: 87; of
// 4 x 2 waves with 2 x 4 tiles each 100, with 4 x 4 90.  Gated, 4096 x 2048 to e4m3 131 and to bf16 79; a wave's tiles 1 x 4
// of each matrix in place of 2 x 4 169 and 111.
template <bool GLU>
int launch_dense(const F8Args &a, hipStream_t st)
{
    const bool q = a.y_type == BREAD_QTYPE_E4M3, exact = q || a.y_type == BREAD_QTYPE_F32;
    auto load = [&](int64_t t, int64_t r) {
        const int64_t tiles = (a.T + t - 1) / t * ((a.rows + r - 1) / r);
        return (tiles + CUS - 1) / CUS * (t + (GLU ? 2 : 1) * r);
    };
    const int64_t least = q ? std::min(load(16, 128), load(32, 128))
                            : std::min({load(16, 32), load(32, 32), load(48, 32), load(64, 32), load(64, 64)});
    if (load(128, 128) <= least) {
        if constexpr (GLU)
            return exact ? launch<4, 2, 1, 2, 4, 1, true, false, 2, false, false>(a, st)
                         : launch<4, 2, 1, 2, 4, 1, true, true, 2, false, false>(a, st);
        else
            return exact ? launch<2, 2, 1, 4, 4, 1, false, false, 2, false, false>(a, st)
                         : launch<2, 2, 1, 4, 4, 1, false, true, 2, false, false>(a, st);
    }
    if (q) {
        if (load(16, 128) == least) return launch<8, 1, 2, 1, 1, GLU ? 2 : 4, GLU, false, 4, true, false>(a, st);
        if constexpr (GLU)
            return launch<8, 1, 1, 1, 2, 1, true, false, 2, true, false>(a, st);
        else
            return launch<8, 1, 2, 1, 2, 2, false, false, 4, true, false>(a, st);
    }
    if (load(16, 32) == least) return launch<2, 1, 4, 1, 1, GLU ? 4 : 8, GLU, false, 2, true, false>(a, st);
    if (load(32, 32) == least) return launch<2, 1, 4, 1, 2, 4, GLU, false, 2, true, false>(a, st);
    if (load(48, 32) == least) return launch<2, 1, 4, 1, 3, 4, GLU, false, 2, true, false>(a, st);
    if (load(64, 32) == least) return launch<2, 2, 2, 1, 2, GLU ? 2 : 4, GLU, false, 2, true, false>(a, st);
    return launch<2, 2, 2, 2, 2, 2, GLU, false, 2, true, false>(a, st);
}

}  // namespace

int bread_launch_fp8_matmul(const F8Args &a, hipStream_t st)
{
    if (a.G) return bread_launch_fp8_grouped(a, st);
    return a.up ? launch_dense<true>(a, st) : launch_dense<false>(a, st);
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
    F8_REQUIRE((int64_t)o.rows * o.n_tokens <= 1ll << 33 && (int64_t)o.rows * o.cols <= 1ll << 40, BREAD_ERR_SHAPE,
               "more than 2^33 results or 2^40 weights");
    const bool q = o.y_type == BREAD_QTYPE_E4M3;
    const int64_t nb = f8_blocks(o.cols), nr = f8_blocks(o.rows);
    a.x_stride = o.x_stride ? o.x_stride : o.cols;
    a.xs_stride = o.x_scale_stride ? o.x_scale_stride : nb;
    a.y_stride = o.y_stride ? o.y_stride : o.rows;
    a.ys_stride = o.y_scale_stride ? o.y_scale_stride : nr;
    F8_REQUIRE(a.x_stride >= o.cols && a.xs_stride >= nb && a.y_stride >= o.rows && (!q || a.ys_stride >= nr),
               BREAD_ERR_SHAPE, "a stride is smaller than a token's row");
    F8_REQUIRE(a.x_stride <= 1 << 22 && a.xs_stride <= 1 << 20, BREAD_ERR_SHAPE,
               "x_stride above 2^22 or x_scale_stride above 2^20");
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
    BREAD_REQUIRE((int64_t)args->rows * groups->n_groups <= 1 << 28, BREAD_ERR_SHAPE, "rows * n_groups above 2^28");
    F8Args a;
    const int rc = check_matmul("bread_matmul_fp8_grouped", *args, groups->n_groups == 0, a);
    if (rc || args->rows == 0 || args->n_tokens == 0 || groups->n_groups == 0) return rc;
    BREAD_REQUIRE(groups->offsets, BREAD_ERR_ARG, "NULL offsets");
    BREAD_REQUIRE((((uintptr_t)groups->offsets | (uintptr_t)groups->x_rows | (uintptr_t)groups->y_rows) & 3) == 0,
                  BREAD_ERR_ALIGN, "offsets and rows must be 4-byte aligned");
    BREAD_REQUIRE(!groups->x_rows || (groups->n_x * a.x_stride <= 1ll << 31 && groups->n_x * a.xs_stride <= 1ll << 29),
                  BREAD_ERR_SHAPE, "gathered x or scales of more than 2^31 bytes");
    a.G = groups->n_groups;
    a.offsets = groups->offsets;
    a.x_rows = groups->x_rows;
    a.y_rows = groups->y_rows;
    a.n_x = groups->n_x;
    a.n_y = groups->n_y;
    return bread_launch_fp8_matmul(a, to_hip(stream));
}
