// fp8_grouped.hip — the forms of fp8_tile.h's kernel for groups of rows.
#include <stdint.h>

#include <algorithm>

#include "fp8_tile.h"

namespace {

// The tiles are those that give a compute unit the fewest rows of weights and tokens to load, as for one matrix
// (fp8_matmul.hip), of about so many token tiles: half a tile more a group than the rows fill, and no fewer than groups.
// us and rows of a unit for tiles of 16, 32, 64 tokens by 32 rows, 64 by 64, 32 by 128 and 128 by 128, to fp32:
//   10 groups, 203 rows, 256 x 2048       6.6 (48)   7.6 (64)   9.6 (96)  11.8 (128)  14.7 (160)  24.0 (256)
//   8, 540, 512 x 2048                   12.7 (144) 11.7 (128)  9.8 (96)  12.2 (128)  14.6 (160)  24.6 (256)
//   54, 3452, 192 x 2048                 23.3 (288) 21.7 (256) 17.4 (192) 13.4 (128)  17.9 (320)  25.3 (256)
//   12, 5022, 256 x 2048                 38.4       29.9       23.7       22.0 (256)  18.4 (320)  25.8 (256)
//   256, 4096, 512 x 2048                87.0       85.2      105         78.5        44.9 (640)  67.2 (1024)
//   256, 16384, 2048 x 512              593        369        273        190         123 (6400)  108 (4096)
//   256, 32768, 2048 x 512             1114        653        451        314         213         164 (6144)
// and 16, 64 and 128 tokens by 128 rows, gated, to e4m3:
//   10, 203, 256 x 2048                  15.2 (272) 25.6 (320) 34.4 (384)
//   12, 5022, 256 x 2048                 38.1 (816) 26.6 (320) 35.3 (384)
//   29, 4936, 512 x 2048                 75.4       51.1 (640) 38.0 (384)
//   256, 4096, 512 x 2048                124        118 (1280) 129 (1536)
//   256, 32768, 512 x 2048               466        250        211 (2304)
// (Of 30 measured calls the rule took the fastest form 28 times, and lost 20 % in the others.)  Tiles of 32 by 128 are small
// enough for two workgroups a unit, which over several rounds take three quarters of the time: with that the rule takes
// them in those two calls as well.  Workgroups take tiles in turn and load the next one's first columns under the last
// one's results: a tile's two to four microseconds of lookups and first loads, 160 of 177 at 2048 x 512.  fp16 and bf16
// results of the largest tiles use the 8-bit matrix instructions (fp8_tile.h): gated, 256 groups, 32768 rows 177 of 211.
template <bool GLU>
int launch_groups(const F8Args &a, hipStream_t st)
{
    const bool q = a.y_type == BREAD_QTYPE_E4M3, exact = q || a.y_type == BREAD_QTYPE_F32;
    const int64_t groups = std::min(a.G, a.T);
    auto load = [&](int64_t t, int64_t r) {
        const int64_t tiles = std::max(groups, (2 * a.T / t + groups + 1) / 2) * ((a.rows + r - 1) / r);
        const int64_t rows = t + (GLU ? 2 : 1) * r, all = (tiles + CUS - 1) / CUS * rows;
        return t == 32 && r == 128 ? std::max(rows, 3 * all / 4) : all;
    };
    const int64_t wide = q ? INT64_MAX : std::min({load(16, 32), load(32, 32), load(64, 32), load(64, 64)});
    const int64_t least = std::min({wide, load(128, 128), GLU ? load(64, 128) : load(32, 128), q ? load(16, 128) : INT64_MAX});
    if constexpr (GLU) {
        if (load(128, 128) == least)
            return exact ? launch<4, 2, 1, 2, 4, 1, true, false, 2, true, true>(a, st)
                         : launch<4, 2, 1, 2, 4, 1, true, true, 2, true, true>(a, st);
        if (load(64, 128) == least) return launch<8, 1, 1, 1, 4, 1, true, false, 2, true, true>(a, st);
    } else {
        if (load(128, 128) == least)
            return exact ? launch<2, 2, 1, 4, 4, 1, false, false, 2, true, true>(a, st)
                         : launch<2, 2, 1, 4, 4, 1, false, true, 2, true, true>(a, st);
        if (load(32, 128) == least) return launch<4, 1, 1, 2, 2, 1, false, false, 2, true, true>(a, st);
    }
    if (q) return launch<8, 1, 2, 1, 1, GLU ? 2 : 4, GLU, false, 4, true, true>(a, st);
    if (load(16, 32) == least) return launch<2, 1, 4, 1, 1, GLU ? 4 : 8, GLU, false, 2, true, true>(a, st);
    if (load(32, 32) == least) return launch<2, 1, 4, 1, 2, 4, GLU, false, 2, true, true>(a, st);
    if (load(64, 32) == least) return launch<2, 2, 2, 1, 2, GLU ? 2 : 4, GLU, false, 2, true, true>(a, st);
    return launch<2, 2, 2, 2, 2, 2, GLU, false, 2, true, true>(a, st);
}

}  // namespace

int bread_launch_fp8_grouped(const F8Args &a, hipStream_t st)
{
    return a.up ? launch_groups<true>(a, st) : launch_groups<false>(a, st);
}
