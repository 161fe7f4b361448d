// Grouped products of fp32 / fp64: the workgroups of one product whose waves share k (rp_gemm_wavekw.h), which take their tiles from the groups.
//
// By rows a tile lies in one group; how many row tiles there are is known on the device only, and the list of all groups' tiles is dealt
// to the XCDs in eight runs, so that the tiles of a group share its weight in one L2.  By weights the reduction runs over the group's
// rows.  Rows may start at any element.  The tile is the largest whose tiles occupy three quarters of the CUs, as for one product:
// small layers are bound by launch and latency (k goes to eight waves), 64 x 64 tiles of fp32 by the MFMAs.
// fp32, us, on scalar multiply-adds and here: 1024 rows of 4 groups, 784 -> 256, forward 43 / 12; its three gradients together 100 / 22
// (in launches of their own 28).  4096 rows of 8 groups, 1024 -> 1024: forward 122, 71 TFLOP/s, gradients 223.
#include "rp_gemm_wavekw.h"
#include "rp_grouped_sums.h"

namespace rp {

constexpr int GW_WAVES = 8;
// Rows of a group up to which its weights' gradient is written by outer products (19 rows of 12 groups, 1980 x 4035, forward and backward: 608 us, 540 so)
constexpr int GW_FEW_ROWS = 8;
constexpr int gw_waves_per_simd(int tiles) { return tiles <= 4 ? 4 : 2; }

// One tile in the block's own order of a matrix of one tile
template <typename E, bool B_KC, int TM, int TN>
__device__ __forceinline__ void rows_block(const GroupedArgs& ga, int tiles_n, int id, unsigned char* lds) {
    const RowTiles rows(ga.gr, 16 * TM);
    const int total = rows.total * tiles_n, at = run_tile(id, total);
    if (at == total) return;
    const int row = at / tiles_n;
    const RowTile rt = rows.find(row);
    const TileCoord in = chunk_tile(at - rt.first * tiles_n, rt.tiles, tiles_n);
    const int begin = rt.begin + (in.tm - (row - rt.first)) * 16 * TM;
    const GemmArgs g{(E*)ga.C + begin * ga.c_rs, (const E*)ga.A + begin * ga.a_rs, (const E*)ga.B + rt.weight * ga.b_ws, ga.bias ? (const E*)ga.bias + (long long)rt.weight * ga.n : nullptr,
                     1, begin + 16 * TM < rt.stop ? 16 * TM : rt.stop - begin, ga.k, ga.n, 0, ga.a_rs, 1, 0, B_KC ? 1 : ga.b_rs, B_KC ? ga.b_cs : 1, 0, ga.c_rs, 1, ga.accumulate};
    // (the block that its schedule gives this column tile)
    const int share = (tiles_n + 7) / 8;
    gemm_wavekw_block<E, true, B_KC, TM, TN, GW_WAVES>(g, 1, tiles_n, in.tn % share * 8 + in.tn / share, 1, lds);
}

template <typename E, int TM, int TN>
__device__ __forceinline__ void weights_block(const GroupedArgs& ga, int tiles_k, int tiles_n, int slots, int id, unsigned char* lds) {
    const int w = id / slots, b = __builtin_amdgcn_readfirstlane(ga.gr.begin(w)), e = __builtin_amdgcn_readfirstlane(ga.gr.end(w));
    if (e - b <= GW_FEW_ROWS) {
        // a few rows (or none: zeros, or what is there): the tile is written, and little else takes time.  A column a thread; its values of dy stay in registers.
        const int at = run_tile(id - w * slots, tiles_k * tiles_n), k0 = at / tiles_n * 16 * TM, c = at % tiles_n * 16 * TN + (int)threadIdx.x % (16 * TN), rows = e - b;
        if (at == tiles_k * tiles_n || c >= ga.n || (rows == 0 && ga.accumulate)) return;
        const E* x = (const E*)ga.A + b * ga.a_rs;
        const E* dy = (const E*)ga.B + b * ga.b_rs + c;
        E v[GW_FEW_ROWS];
#pragma unroll
        for (int i = 0; i < GW_FEW_ROWS; i++) v[i] = i < rows ? dy[i * ga.b_rs] : (E)0;
        E* out = (E*)ga.C + w * ga.c_ws + c;
        const int last = k0 + 16 * TM < ga.k ? k0 + 16 * TM : ga.k;
        for (int r = k0 + (int)threadIdx.x / (16 * TN); r < last; r += 64 * GW_WAVES / (16 * TN)) {
            E sum = 0;
#pragma unroll
            for (int i = 0; i < GW_FEW_ROWS; i++)
                if (i < rows) sum += x[i * ga.a_rs + r] * v[i];
            E* to = out + r * ga.c_rs;
            *to = ga.accumulate ? *to + sum : sum;
        }
        return;
    }
    const GemmArgs g{(E*)ga.C + w * ga.c_ws, (const E*)ga.A + b * ga.a_rs, (const E*)ga.B + b * ga.b_rs, nullptr,
                     1, ga.k, e - b, ga.n, 0, 1, ga.a_rs, 0, ga.b_rs, 1, 0, ga.c_rs, 1, ga.accumulate};
    gemm_wavekw_block<E, false, false, TM, TN, GW_WAVES>(g, tiles_k, tiles_n, id - w * slots, 1, lds);
}

template <typename E, bool B_KC, int TM, int TN>
__global__ void __launch_bounds__(64 * GW_WAVES, gw_waves_per_simd(TM * TN)) grouped_rows_wavek_kernel(GroupedArgs ga, int tiles_n) {
    extern __shared__ __attribute__((aligned(16))) unsigned char wkw_lds[];
    rows_block<E, B_KC, TM, TN>(ga, tiles_n, (int)blockIdx.x, wkw_lds);
}

// The input's gradient, the weights' and the bias's, as many of them as there are blocks for
template <typename E, int TX, int TW>
__global__ void __launch_bounds__(64 * GW_WAVES, gw_waves_per_simd(TX > TW ? TX * TX : TW * TW)) grouped_backward_wavek_kernel(GroupedArgs x, GroupedArgs w, GroupedSums sums, int s_blocks, int x_blocks, int x_tiles_n,
                                                                                                      int w_tiles_k, int w_tiles_n, int w_slots) {
    extern __shared__ __attribute__((aligned(16))) unsigned char wkw_lds[];
    const int id = (int)blockIdx.x;
    if (id < s_blocks) {
        if (id < sums.gr.weights * ((sums.cols + 63) / 64)) grouped_sums_block<E, GW_WAVES>(sums, id, (E*)wkw_lds);
    } else if (id - s_blocks < x_blocks) {
        rows_block<E, true, TX, TX>(x, x_tiles_n, id - s_blocks, wkw_lds);
    } else {
        weights_block<E, TW, TW>(w, w_tiles_k, w_tiles_n, w_slots, id - s_blocks - x_blocks, wkw_lds);
    }
}

template <typename E, bool B_KC, int TM, int TN>
static int launch_rows(const GroupedArgs& g) {
    constexpr size_t smem = wkw_smem<E, true, B_KC, TM, TN, GW_WAVES>();
    const int tiles_n = (g.n + 16 * TN - 1) / (16 * TN);
    const long long blocks = (max_row_tiles(g.gr.rows, g.gr.groups, 16 * TM) * tiles_n + 7) / 8 * 8;
    auto kern = grouped_rows_wavek_kernel<E, B_KC, TM, TN>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(64 * GW_WAVES), smem, current_stream(), g, tiles_n);
    return check_launch("grouped_rows_wavek_kernel") ? 0 : -1;
}

template <typename E, int TX, int TW>
static int launch_backward(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums) {
    constexpr size_t smem_x = wkw_smem<E, true, true, TX, TX, GW_WAVES>(), smem_w = wkw_smem<E, false, false, TW, TW, GW_WAVES>(), most = smem_x > smem_w ? smem_x : smem_w;
    constexpr size_t smem = most > 64 * 16 * sizeof(E) ? most : 64 * 16 * sizeof(E);
    const int x_tiles_n = (x.n + 16 * TX - 1) / (16 * TX), w_tiles_k = (w.k + 16 * TW - 1) / (16 * TW), w_tiles_n = (w.n + 16 * TW - 1) / (16 * TW), w_slots = (w_tiles_k * w_tiles_n + 7) / 8 * 8;
    const long long x_blocks = x.C ? (max_row_tiles(x.gr.rows, x.gr.groups, 16 * TX) * x_tiles_n + 7) / 8 * 8 : 0, w_blocks = w.C ? (long long)w_slots * w.gr.weights : 0;
    const long long s_blocks = sums.out ? (sum_blocks(sums) + 7) / 8 * 8 : 0;
    auto kern = grouped_backward_wavek_kernel<E, TX, TW>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)(s_blocks + x_blocks + w_blocks)), dim3(64 * GW_WAVES), smem, current_stream(), x, w, sums, (int)s_blocks, (int)x_blocks, x_tiles_n,
                       w_tiles_k, w_tiles_n, w_slots);
    return check_launch("grouped_backward_wavek_kernel") ? 0 : -1;
}

template <typename E, int TX>
static int launch_backward_weights(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums, int tw) {
    if constexpr (sizeof(E) == 4) {
        if (tw == 4) return launch_backward<E, TX, 4>(x, w, sums);
    }
    return tw == 2 ? launch_backward<E, TX, 2>(x, w, sums) : launch_backward<E, TX, 1>(x, w, sums);
}

constexpr long long GW_MAX_BLOCKS = (1ll << 32) / (64 * GW_WAVES) - 8;       // fewer than 2^32 threads a launch

// 16-row units of the largest square tile whose tiles occupy three quarters of the CUs, 0: none can be addressed.  tiles(t): how many of 16 t x 16 t; fits(t): rows of k are that wide.
template <typename Tiles, typename Fits>
static int wavek_tile(int dtype, Tiles tiles, Fits fits) {
    const long long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    if (dtype == RP_DTYPE_FLOAT32 && fits(4) && tiles(4) * 4 >= cus * 3) return tiles(4) <= GW_MAX_BLOCKS ? 4 : 0;
    if (fits(2) && tiles(2) * 4 >= cus * 3) return tiles(2) <= GW_MAX_BLOCKS ? 2 : 0;
    return fits(1) && tiles(1) <= GW_MAX_BLOCKS ? 1 : 0;
}

// The operands of a product can be addressed: unit strides, 32-bit byte offsets from a tile's first row
static bool rows_ok(const GroupedArgs& g, int dtype) {
    const long long esz = (long long)dtype_size(dtype), limit = 1ll << 31;
    const bool b_kc = g.b_cs != 1;
    if (g.a_cs != 1 || (b_kc && g.b_rs != 1) || g.gr.groups > ROW_TILES_GROUPS / 2 || path_disabled("mfma")) return false;
    return (63 * g.a_rs + g.k) * esz < limit && (b_kc ? 63 * g.b_cs + g.k : (g.k - 1) * g.b_rs + 64) * esz < limit;
}
static bool weights_ok(const GroupedArgs& g, int dtype) {
    const long long esz = (long long)dtype_size(dtype), limit = 1ll << 31;
    if (g.a_cs != 1 || g.b_cs != 1 || g.gr.ids || path_disabled("mfma")) return false;
    return ((long long)(g.gr.rows - 1) * g.a_rs + 64) * esz < limit && ((long long)(g.gr.rows - 1) * g.b_rs + 64) * esz < limit;
}
static long long rows_tiles(const GroupedArgs& g, int t) { return max_row_tiles(g.gr.rows, g.gr.groups, 16 * t) * ((g.n + 16 * t - 1) / (16 * t)); }
static long long weights_tiles(const GroupedArgs& g, int t) { return (long long)g.gr.weights * (((long long)((g.k + 16 * t - 1) / (16 * t)) * ((g.n + 16 * t - 1) / (16 * t)) + 7) / 8 * 8); }

static int rows_tile(const GroupedArgs& g, int dtype) {
    return rows_ok(g, dtype) ? wavek_tile(dtype, [&](int t) { return rows_tiles(g, t); }, [&](int t) { return g.b_cs != 1 || g.n >= 16 * t; }) : 0;
}
static int weights_tile(const GroupedArgs& g, int dtype) {
    return weights_ok(g, dtype) ? wavek_tile(dtype, [&](int t) { return weights_tiles(g, t); }, [&](int t) { return g.k >= 16 * t && g.n >= 16 * t; }) : 0;
}

bool grouped_rows_wavek_takes(const GroupedArgs& g, int dtype) { return rows_tile(g, dtype) != 0; }
bool grouped_backward_wavek_takes(const GroupedArgs& x, const GroupedArgs& w, int dtype) {
    const long long tx = x.C ? rows_tile(x, dtype) : 1, tw = w.C ? weights_tile(w, dtype) : 1;
    if (!tx || !tw || (x.C && x.b_cs == 1)) return false;
    return (x.C ? rows_tiles(x, (int)tx) : 0) + (w.C ? weights_tiles(w, (int)tw) : 0) + (long long)w.gr.weights * ((w.n + 63) / 64) + 16 <= GW_MAX_BLOCKS;
}

int launch_grouped_backward_wavek(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums, int dtype) {
    const int tx = x.C ? rows_tile(x, dtype) : 1, tw = w.C ? weights_tile(w, dtype) : 1;
    if (dtype == RP_DTYPE_FLOAT64) return tx == 2 ? launch_backward_weights<double, 2>(x, w, sums, tw) : launch_backward_weights<double, 1>(x, w, sums, tw);
    if (tx == 4) return launch_backward_weights<float, 4>(x, w, sums, tw);
    return tx == 2 ? launch_backward_weights<float, 2>(x, w, sums, tw) : launch_backward_weights<float, 1>(x, w, sums, tw);
}

template <typename E, int T>
static int launch_rows_layout(const GroupedArgs& g) { return g.b_cs == 1 ? launch_rows<E, false, T, T>(g) : launch_rows<E, true, T, T>(g); }

int launch_grouped_rows_wavek(const GroupedArgs& g, int dtype) {
    const int t = rows_tile(g, dtype);
    if (dtype == RP_DTYPE_FLOAT64) return t == 2 ? launch_rows_layout<double, 2>(g) : launch_rows_layout<double, 1>(g);
    return t == 4 ? launch_rows_layout<float, 4>(g) : t == 2 ? launch_rows_layout<float, 2>(g) : launch_rows_layout<float, 1>(g);
}

}  // namespace rp
