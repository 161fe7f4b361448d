// Shared by the layers whose weight depends on the row (routing, exchange of rows, grouped products, adapters).
#pragma once
#include "rp_common.h"

namespace rp {

// One rounding to the tensor type, nearest even (the hardware's conversions): these layers have no counterpart in the
// reference whose round-half-up they would have to follow, and nearest even keeps every NaN a NaN.
template <typename T> __device__ __forceinline__ T round_to(typename traits<T>::acc v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ double round_to<double>(double v) { return v; }
template <> __device__ __forceinline__ bf16_t round_to<bf16_t>(float v) { bf16_t r; r.bits = __builtin_bit_cast(uint16_t, (__bf16)v); return r; }
template <> __device__ __forceinline__ f16_t round_to<f16_t>(float v) { f16_t r; r.bits = __builtin_bit_cast(uint16_t, (_Float16)v); return r; }

// Rows in groups: group g holds rows [offsets[g], offsets[g + 1]) of `rows`, and its weight is number ids[g] of `weights` (ids null:
// g itself).  The offsets are device memory that no host code has seen: whatever they hold, begin and end are clamped to
// the rows there are, and a weight number out of range stands for a group without a weight.  Without offsets (null) there is one group of all rows.
struct RowGroups {
    const int* offsets;
    const int* ids;
    int groups, rows, weights;
    __device__ __forceinline__ int begin(int g) const { const int o = offsets ? offsets[g] : g ? rows : 0; return o < 0 ? 0 : o > rows ? rows : o; }
    __device__ __forceinline__ int end(int g) const { const int b = begin(g), o = offsets ? offsets[g + 1] : rows, e = o > rows ? rows : o; return e > b ? e : b; }
    __device__ __forceinline__ int weight(int g) const { const int w = ids ? ids[g] : g; return w >= 0 && w < weights ? w : -1; }
};

// f(begin, end) for every group of weight w that has rows, in order; the wave looks at 64 groups at a time (one after the other, their ids and
// offsets cost a trip to memory each: 32 adapters of 8192 rows in 48 segments, gradients of rank 64 at 4096 x 4096, 188 us, 144 here)
template <typename F>
__device__ __forceinline__ void for_groups_of(const RowGroups& gr, int w, F f) {
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < gr.groups; g0 += 64) {
        int b = 0, e = 0, own = -1;
        if (g0 + lane < gr.groups) { own = gr.weight(g0 + lane); b = gr.begin(g0 + lane); e = gr.end(g0 + lane); }      // (one trip to memory for all three)
        unsigned long long here = __builtin_amdgcn_ballot_w64(own == w && e > b);
        while (here) {
            const int l = __builtin_ctzll(here);
            here &= here - 1;
            f(__builtin_amdgcn_readlane(b, l), __builtin_amdgcn_readlane(e, l));
        }
    }
}

// Tiles of `tile` rows that `rows` rows in `groups` groups can come to, whatever the offsets hold as long as the groups do not overlap
static inline long long max_row_tiles(long long rows, long long groups, int tile) {
    const long long parted = rows / tile + (groups < rows ? groups : rows);
    return parted < rows ? parted : rows;
}

// Tile number `id` of the groups' row tiles, found by the whole wave together: 64 groups at a time, a lane each, their tile counts added up
// across the lanes.  All results are wave-uniform.
// rows [begin, end) of `group`, which ends at row `stop` and whose `tiles` tiles begin with number `first`; group < 0: there is no such tile
struct RowTile { int group, weight, begin, end, stop, first, tiles; };
__device__ __forceinline__ int wave_prefix_sum(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int below = __shfl_up(v, d);
        v += lane >= d ? below : 0;
    }
    return v;
}
__device__ __forceinline__ RowTile find_row_tile(const RowGroups& gr, int tile, int id) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int g0 = 0; g0 < gr.groups; g0 += 64) {
        const int g = g0 + lane;
        int b = 0, e = 0, w = -1;
        if (g < gr.groups) { b = gr.begin(g); e = gr.end(g); w = gr.weight(g); }
        const int tiles = w < 0 ? 0 : (e - b + tile - 1) / tile;
        const int upto = before + wave_prefix_sum(tiles, lane);
        const unsigned long long past = __builtin_amdgcn_ballot_w64(upto > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            RowTile t;
            t.tiles = __builtin_amdgcn_readlane(tiles, l);
            t.first = __builtin_amdgcn_readlane(upto, l) - t.tiles;
            t.group = g0 + l;
            t.weight = __builtin_amdgcn_readlane(w, l);
            t.begin = __builtin_amdgcn_readlane(b, l) + (id - t.first) * tile;
            t.stop = __builtin_amdgcn_readlane(e, l);
            t.end = t.begin + tile < t.stop ? t.begin + tile : t.stop;
            return t;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return RowTile{-1, -1, 0, 0, 0, 0, 0};
}

// Of more groups than this a tile is looked for by bisection, 64 ways at a time, instead of adding up all groups' tiles before it: a trip to memory for each power of 64 and not for
// each 64 groups.  The tiles are not numbered one after the other then: tile t of group g is number begin(g) / tile + g + t, which leaves out at most one number a group.
// (bf16, us, added up and bisected: adapters of a segment a row, 256 -> 1024, rank 16, 200 segments 18 / 15, 1000 59 / 33, 4000 437 / 96; groups of a row, 256 -> 520, 200 20 / 21, 1000 152 / 78)
constexpr int GROUPS_ADDED_UP = 256;
// Kernels whose workgroups look through all groups (RowTiles, the adapters' tiles) take no more than this, those of fp32 and fp64 half as many; more go to the generic kernel, which bisects.
// (us, RowTiles and generic, groups of a row, 1025 -> 521: bf16 2000 959 / 2076, 4000 3226 / 4086, of 257 -> 521 2939 / 1074; fp32 1000 1195 / 1052, 2000 3424 / 2055; 30000 groups,
// 257 -> 521: bf16 157521 / 7944)
constexpr int ROW_TILES_GROUPS = 4096;
// The last of `count` numbers g for which below(g), which does not grow again, is true; -1: none
template <typename F> __device__ __forceinline__ int last_of(int count, F below) {
    const int lane = threadIdx.x & 63;
    int from = 0;
    while (count > 0) {
        const int step = (count + 63) / 64, at = lane * step;
        const unsigned long long yes = __builtin_amdgcn_ballot_w64(at < count && below(from + at));
        if (!yes) return from ? from : -1;                    // (from itself is one of them then)
        const int l = 63 - __builtin_clzll(yes);
        if (step == 1) return from + l;
        from += l * step;
        count = count - l * step < step ? count - l * step : step;
    }
    return -1;
}
// find_row_tile for a kernel of a workgroup a tile, with row_tile_numbers() of them
static inline long long row_tile_numbers(long long rows, long long groups, int tile) { return groups > GROUPS_ADDED_UP ? rows / tile + groups : max_row_tiles(rows, groups, tile); }
__device__ __forceinline__ RowTile find_row_tile_number(const RowGroups& gr, int tile, int id) {
    if (gr.groups <= GROUPS_ADDED_UP) return find_row_tile(gr, tile, id);
    const int g = last_of(gr.groups, [&](int i) { return gr.begin(i) / tile + i <= id; });
    if (g < 0) return RowTile{-1, -1, 0, 0, 0, 0, 0};
    const int b = gr.begin(g), e = gr.end(g), w = gr.weight(g), t = id - (b / tile + g);
    if (w < 0 || t >= (e - b + tile - 1) / tile) return RowTile{-1, -1, 0, 0, 0, 0, 0};
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int begin = uniform(b + t * tile), stop = uniform(e);
    return RowTile{uniform(g), uniform(w), begin, begin + tile < stop ? begin + tile : stop, stop, uniform(id - t), uniform((e - b + tile - 1) / tile)};
}

// A launch has fewer than 2^32 threads: launch(workgroups, number of the first) as often as it takes; not 0: what one of them returned
template <typename F> static inline int in_launches(long long blocks, int threads, F launch) {
    const long long most = ((1ll << 32) / threads - 1) / 8 * 8;
    for (long long first = 0; first < blocks; first += most) {
        const int rc = launch((unsigned)(blocks - first < most ? blocks - first : most), first);
        if (rc != 0) return rc;
    }
    return 0;
}

// The same for a workgroup that looks up many tiles: up to 64 groups are read and added up once and kept a lane each.
struct RowTiles {
    RowGroups gr;
    int tile, total;                   // rows of a tile; how many tiles there are
    int b, e, w, upto, tiles;          // of this lane's group, if there are at most 64
    __device__ __forceinline__ RowTiles(const RowGroups& groups, int rows_of_tile) : gr(groups), tile(rows_of_tile), b(0), e(0), w(-1) {
        const int lane = threadIdx.x & 63;
        total = 0;
        for (int g0 = 0; g0 < gr.groups; g0 += 64) {
            b = e = 0;
            w = -1;
            if (g0 + lane < gr.groups) { b = gr.begin(g0 + lane); e = gr.end(g0 + lane); w = gr.weight(g0 + lane); }
            tiles = w < 0 ? 0 : (e - b + tile - 1) / tile;
            upto = total + wave_prefix_sum(tiles, lane);
            total = __builtin_amdgcn_readlane(upto, 63);
        }
    }
    __device__ __forceinline__ RowTile find(int id) const {
        if (gr.groups > 64) return find_row_tile(gr, tile, id);
        const unsigned long long past = __builtin_amdgcn_ballot_w64(upto > id);
        if (!past) return RowTile{-1, -1, 0, 0, 0, 0, 0};
        const int l = __builtin_ctzll(past);
        const int count = __builtin_amdgcn_readlane(tiles, l), first = __builtin_amdgcn_readlane(upto, l) - count;
        const int begin = __builtin_amdgcn_readlane(b, l) + (id - first) * tile, stop = __builtin_amdgcn_readlane(e, l);
        return RowTile{l, __builtin_amdgcn_readlane(w, l), begin, begin + tile < stop ? begin + tile : stop, stop, first, count};
    }
};

}  // namespace rp
