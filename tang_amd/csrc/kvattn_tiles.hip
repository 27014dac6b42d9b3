// The launch of tile items (kvattn_tiles.hpp).
#include <algorithm>
#include <type_traits>

#include "kvattn_tiles.hpp"

namespace th {

template <int D, typename E, int NP, bool PAD, bool ADD>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_attn_tiles_kernel(KvAttnArgs a) {
    __shared__ __align__(16) char lds[KvTiles<D, NP>::LDS];
    const int kvh = a.pages.n_kv_heads, h = blockIdx.x % kvh, count = a.head->n_tile_items;
    int n = blockIdx.x / kvh;
    // the first item is read before it is known to be there (the list has room for the grid)
    KvItem it = kv_item(a.tile_items, n);
    for (; n < count; it = kv_item(a.tile_items, n)) {
        kv_tiles_item<D, E, NP, PAD, ADD>(a, it, h, lds);
        n += gridDim.x / kvh;
        if (n >= count) break;
        __syncthreads();  // the next item's first block goes where this one's last may be read
    }
}

template <int D, typename E>
static void tiles_launch(const KvAttnArgs& a, unsigned grid, int flags, hipStream_t s) {
    constexpr int WIDE = kv_wide_parts<E>();
    const th_dtype own = std::is_same<E, __bf16>::value ? TH_BF16 : TH_F16;
    const bool one = a.qdt == own && a.odt == own, pad = a.pages.hd != D, far = flags & KV_PLAN_FAR;
    if (one && pad && far) TH_LAUNCH((kv_attn_tiles_kernel<D, E, 1, true, true>), dim3(grid), dim3(256), 0, s, a);
    else if (one && pad) TH_LAUNCH((kv_attn_tiles_kernel<D, E, 1, true, false>), dim3(grid), dim3(256), 0, s, a);
    else if (one && far) TH_LAUNCH((kv_attn_tiles_kernel<D, E, 1, false, true>), dim3(grid), dim3(256), 0, s, a);
    else if (one) TH_LAUNCH((kv_attn_tiles_kernel<D, E, 1, false, false>), dim3(grid), dim3(256), 0, s, a);
    else if (pad) TH_LAUNCH((kv_attn_tiles_kernel<D, E, WIDE, true, true>), dim3(grid), dim3(256), 0, s, a);
    else TH_LAUNCH((kv_attn_tiles_kernel<D, E, WIDE, false, true>), dim3(grid), dim3(256), 0, s, a);
    TH_LAUNCH_CHECK();
}

void launch_kv_attn_tiles(const KvAttnArgs& a, th_dtype cache, size_t grid, int flags, hipStream_t s) {
    if (grid == 0) return;
    const unsigned g = (unsigned)(std::min(grid, KV_MAX_BLOCKS / a.pages.n_kv_heads) * a.pages.n_kv_heads);
    auto with = [&](auto e) {
        typedef decltype(e) E;
        if (a.pages.hd <= 64) tiles_launch<64, E>(a, g, flags, s);
        else if (a.pages.hd <= 128) tiles_launch<128, E>(a, g, flags, s);
        else tiles_launch<256, E>(a, g, flags, s);
    };
    if (cache == TH_F16) with((_Float16)0);
    else with((__bf16)0.0f);
}

}  // namespace th
