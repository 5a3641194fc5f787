// The tile kernel of the attention over the 8-bit paged cache (attend8_tiles.h) in its sizes and types.
#include "attend8_tiles.h"

namespace kitty {

void launch_tiles(const Attend8 &p, int DP, bool bf16, hipStream_t stream)
{
    const dim3 grid((unsigned)(p.B * p.c.H * p.nrb * p.splits)), block(64 * kTileWaves);
    auto go = [&](auto dp, auto bf) {
        constexpr int N = decltype(dp)::value;
        constexpr bool BF = decltype(bf)::value;
        if (p.c.D == N)
            hipLaunchKernelGGL((cache8_tile_kernel<N, BF, false>), grid, block, 0, stream, p);
        else
            hipLaunchKernelGGL((cache8_tile_kernel<N, BF, true>), grid, block, 0, stream, p);
    };
    auto by_size = [&](auto bf) {
        if (DP == 64)
            go(std::integral_constant<int, 64>{}, bf);
        else if (DP == 128)
            go(std::integral_constant<int, 128>{}, bf);
        else
            go(std::integral_constant<int, 256>{}, bf);
    };
    if (bf16)
        by_size(std::true_type{});
    else
        by_size(std::false_type{});
}

} // namespace kitty
