// Attention for many rows: its launch (cache_attention_tiled.hpp has the kernel).
#include "cache_attention_tiled.hpp"

namespace nnops_amd {

// Eight waves where their registers allow it and the rows fill more than four's
// (us, eight / four waves, 32 query and 8 KV heads; a prompt of 4096, d 128 150.7 /
// 249, d 64 107 / 122; 64 x 33 rows of 300 29.5 / 50.0; 24 sequences of 1 to 300 rows
// of 2500 121 / 177, d 64 99.6 / 97.9; f32, d 64, 64 x 64 of 300 38.5 / 54.4).
int tiled_rows(int64_t d, bool f16, int64_t page, int64_t rows)
{
    if (d > 128 && (!f16 || page < kTile)) {
        return 0;                                  // three parts of 256 channels: more registers than there are
    }
    if (d > (f16 ? 128 : 64)) {
        return 128;
    }
    return rows > 128 ? 256 : 128;
}

namespace {

template <typename T, int DP, int NW>
void launch_one(const AttnKern& k, const dim3& grid, hipStream_t s)
{
    if (DP > 128 || tiled_one_page(k.c.d, k.c.page)) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, true, kWhole>), grid, dim3(64 * NW), 0, s, k);
    } else if constexpr (DP <= 128) {
        NNOPS_LAUNCH((attention_rows_tiled<T, DP, NW, false, kWhole>), grid, dim3(64 * NW), 0, s, k);
    }
}

}  // namespace

void launch_tiled(const AttnKern& k, const dim3& grid, bool f16, hipStream_t s)
{
    const int d = k.c.d;
    if (f16 && k.tile_rows == 256) {
        d <= 64 ? launch_one<_Float16, 64, 8>(k, grid, s) : launch_one<_Float16, 128, 8>(k, grid, s);
    } else if (f16) {
        d <= 64    ? launch_one<_Float16, 64, 4>(k, grid, s)
        : d <= 128 ? launch_one<_Float16, 128, 4>(k, grid, s)
                   : launch_one<_Float16, 256, 4>(k, grid, s);
    } else if (k.tile_rows == 256) {
        launch_one<float, 64, 8>(k, grid, s);
    } else {
        d <= 64 ? launch_one<float, 64, 4>(k, grid, s) : launch_one<float, 128, 4>(k, grid, s);
    }
}

}  // namespace nnops_amd
