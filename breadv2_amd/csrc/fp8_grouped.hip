// fp8_grouped.hip — the forms of fp8_tile.h's kernel for groups of rows.
#include "fp8_tile.h"

namespace {

// By the rows of a group, on average.  us of 256 groups, of tiles of 16, 32, 64 and 128 tokens by 128 rows:
//   gated, 512 x 2048, to e4m3         8 rows 113 119 -   123;  16: 134 123 129 137;  32: 188 147 135 146;
//                                      64: -  225 164 177;  128: -   -   262 233
//   2048 x 512, to fp32                8 rows 68  66  -   81;   16: 78  75  -   88;   32: 112 94  -   94;
//                                      64: -  144 -   116;  128: -   -   190 169
// (The weights alone take 103 and 52 at the copy rate.)  Small tiles hold fewer rows that are none, large ones are
// widened less often a product.  Workgroups that take tiles in turn load the next one's first columns under the last
// one's results; the largest tiles leave no registers for it.  fp16 and bf16 results of the largest tiles use the 8-bit
// matrix instructions (fp8_tile.h): 181 of 252 at 128 gated rows.
template <bool GLU>
int launch_groups(const F8Args &a, hipStream_t st)
{
    const bool exact = a.y_type == BREAD_QTYPE_E4M3 || a.y_type == BREAD_QTYPE_F32;
    const int64_t rows = a.T / a.G;
    if constexpr (GLU) {
        if (rows <= 12) return launch<8, 1, 1, 1, 1, 2, true, false, 2, true, true>(a, st);
        if (rows <= 96) return launch<8, 1, 1, 1, 4, 1, true, false, 2, true, true>(a, st);
        return exact ? launch<4, 2, 1, 2, 4, 1, true, false, 2, false, true>(a, st)
                     : launch<4, 2, 1, 2, 4, 1, true, true, 2, false, true>(a, st);
    } else {
        if (rows <= 32) return launch<4, 1, 1, 2, 2, 1, false, false, 2, true, true>(a, st);
        return exact ? launch<2, 2, 1, 4, 4, 1, false, false, 2, false, true>(a, st)
                     : launch<2, 2, 1, 4, 4, 1, false, true, 2, false, true>(a, st);
    }
}

}  // namespace

int bread_launch_fp8_grouped(const F8Args &a, hipStream_t st)
{
    return a.up ? launch_groups<true>(a, st) : launch_groups<false>(a, st);
}
