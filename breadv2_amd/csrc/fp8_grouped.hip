// fp8_grouped.hip — the forms of fp8_tile.h's kernel for groups of rows.
#include "fp8_tile.h"

namespace {

template <bool GLU>
int launch_groups(const F8Args &a, hipStream_t st)
{
    const bool exact = a.y_type == BREAD_QTYPE_E4M3 || a.y_type == BREAD_QTYPE_F32;
    const int64_t rows = a.T / a.G;  // of a group, on average
    if (rows <= 16) return launch<8, 1, 1, 1, 1, 2, GLU, false, GLU ? 2 : 4, true, true>(a, st);
    if (rows <= 48) return launch<8, 1, 1, 1, 4, GLU ? 1 : 2, GLU, false, 2, true, true>(a, st);
    if constexpr (GLU) {
        return exact ? launch<8, 1, 1, 1, 4, 1, true, false, 2, false, true>(a, st)
                     : launch<8, 1, 1, 1, 4, 1, true, true, 2, false, true>(a, st);
    } else {
        return exact ? launch<4, 2, 1, 2, 4, 1, false, false, 2, false, true>(a, st)
                     : launch<4, 2, 1, 2, 4, 1, false, true, 4, false, true>(a, st);
    }
}

}  // namespace

int bread_launch_fp8_grouped(const F8Args &a, hipStream_t st)
{
    return a.up ? launch_groups<true>(a, st) : launch_groups<false>(a, st);
}
