// Tile and rows items in one launch: a shared prefix's tiles and the sequences' own
// keys, prompts next to decode steps.  Tiles come first (they take longest), rows items fill what
// they leave; two launches would each end with a part of the chip idle (64 rows on a shared prefix of 8192: 112 us
// against 119 in two launches, eight on one of 992: 25 against 32).
#include <algorithm>
#include <type_traits>

#include "kvattn_rows.hpp"
#include "kvattn_tiles.hpp"

namespace th {

// ADD: whether tiles' sums are added plainly (kv_tiles_item), or as the plan says.
enum { ADD_NO, ADD_YES, ADD_BY_PLAN };
template <int D, typename E, int NP, bool PAD, int ADD>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void kv_attn_both_kernel(KvAttnArgs a) {
    __shared__ __align__(16) char lds[std::max(KvTiles<D, NP>::LDS, KvRows<D>::LDS)];
    const int kvh = a.pages.n_kv_heads, h = blockIdx.x % kvh;
    const int tiles = __builtin_amdgcn_readfirstlane(a.head->n_tile_items);
    const int count = tiles + __builtin_amdgcn_readfirstlane(a.head->n_rows_items);
    const bool add = ADD == ADD_BY_PLAN && (__builtin_amdgcn_readfirstlane(a.head->flags) & KV_PLAN_FAR);
    for (int n = blockIdx.x / kvh; n < count; n += gridDim.x / kvh) {
        if (n < tiles) {
            const KvItem it = kv_item(a.tile_items, n);
            if constexpr (ADD == ADD_BY_PLAN) {
                if (add) kv_tiles_item<D, E, NP, PAD, true>(a, it, h, lds);
                else kv_tiles_item<D, E, NP, PAD, false>(a, it, h, lds);
            } else {
                kv_tiles_item<D, E, NP, PAD, ADD == ADD_YES>(a, it, h, lds);
            }
        } else {
            kv_rows_item<D, E, NP, PAD>(a, kv_item(a.rows_items, n - tiles), h, lds);
        }
        __syncthreads();  // the next item's rows go where this one's may be read
    }
}

template <int D, typename E, bool PAD>
static void both_launch(const KvAttnArgs& a, unsigned grid, int flags, hipStream_t s) {
    constexpr int WIDE = kv_wide_parts<E>();
    const th_dtype own = std::is_same<E, __bf16>::value ? TH_BF16 : TH_F16;
    if (a.qdt != own || a.odt != own) TH_LAUNCH((kv_attn_both_kernel<D, E, WIDE, PAD, ADD_YES>), dim3(grid), dim3(256), 0, s, a);
    else if (flags == KV_BY_PLAN) TH_LAUNCH((kv_attn_both_kernel<D, E, 1, PAD, ADD_BY_PLAN>), dim3(grid), dim3(256), 0, s, a);
    else if (flags & KV_PLAN_FAR) TH_LAUNCH((kv_attn_both_kernel<D, E, 1, PAD, ADD_YES>), dim3(grid), dim3(256), 0, s, a);
    else TH_LAUNCH((kv_attn_both_kernel<D, E, 1, PAD, ADD_NO>), dim3(grid), dim3(256), 0, s, a);
    TH_LAUNCH_CHECK();
}

void launch_kv_attn_both(const KvAttnArgs& a, th_dtype cache, size_t grid, int flags, hipStream_t s) {
    if (grid == 0) return;
    const unsigned g = (unsigned)(std::min(grid, KV_MAX_BLOCKS / a.pages.n_kv_heads) * a.pages.n_kv_heads);
    auto dims = [&](auto e, auto d) {
        typedef decltype(e) E;
        constexpr int D = decltype(d)::value;
        if (a.pages.hd == D) both_launch<D, E, false>(a, g, flags, s);
        else both_launch<D, E, true>(a, g, flags, s);
    };
    auto with = [&](auto e) {
        if (a.pages.hd <= 64) dims(e, std::integral_constant<int, 64>{});
        else if (a.pages.hd <= 128) dims(e, std::integral_constant<int, 128>{});
        else dims(e, std::integral_constant<int, 256>{});
    };
    if (cache == TH_F16) with((_Float16)0);
    else with((__bf16)0.0f);
}

}  // namespace th
