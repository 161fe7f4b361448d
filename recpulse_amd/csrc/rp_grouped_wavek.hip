// Grouped products of fp32 / fp64: the workgroups of one product whose waves share k (rp_gemm_wavekw.h), which take their tiles from the groups.
//
// By rows a tile lies in one group; how many row tiles there are is known on the device only, and all of them times the column tiles are dealt
// to the XCDs in eight runs, so that the tiles of a group share its weight in one L2.  By weights the reduction runs over the group's
// rows.  Rows may start at any element.  The tile is the largest whose tiles occupy three quarters of the CUs, as for one product:
// small layers are bound by launch and latency (k goes to eight waves), 64 x 64 tiles of fp32 by the MFMAs.
// fp32, us, on scalar multiply-adds and here: WAVEK_FIGURES
#include "rp_gemm_wavekw.h"
#include "rp_grouped.h"

namespace rp {

constexpr int GW_WAVES = 8;
constexpr int gw_waves_per_simd(int tiles) { return tiles <= 4 ? 4 : 2; }

template <typename E, bool B_KC, int TM, int TN>
__global__ void __launch_bounds__(64 * GW_WAVES, gw_waves_per_simd(TM * TN)) grouped_rows_wavek_kernel(GroupedArgs ga, int tiles_n) {
    extern __shared__ __attribute__((aligned(16))) unsigned char wkw_lds[];
    const RowTiles rows(ga.gr, 16 * TM);
    const int total = rows.total * tiles_n, per = (total + 7) / 8, at = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || at >= total) return;
    const RowTile rt = rows.find(at / tiles_n);
    const GemmArgs g{(E*)ga.C + rt.begin * ga.c_rs, (const E*)ga.A + rt.begin * ga.a_rs, (const E*)ga.B + rt.weight * ga.b_ws, ga.bias ? (const E*)ga.bias + (long long)rt.weight * ga.n : nullptr,
                     1, rt.end - rt.begin, ga.k, ga.n, 0, ga.a_rs, 1, 0, B_KC ? 1 : ga.b_rs, B_KC ? ga.b_cs : 1, 0, ga.c_rs, 1, ga.accumulate};
    // (the block that its schedule gives this column tile)
    const int tn = at % tiles_n, share = (tiles_n + 7) / 8;
    gemm_wavekw_block<E, true, B_KC, TM, TN, GW_WAVES>(g, 1, tiles_n, tn % share * 8 + tn / share, 1, wkw_lds);
}

template <typename E, int TM, int TN>
__global__ void __launch_bounds__(64 * GW_WAVES, gw_waves_per_simd(TM * TN)) grouped_weights_wavek_kernel(GroupedArgs ga, int tiles_k, int tiles_n, int slots) {
    extern __shared__ __attribute__((aligned(16))) unsigned char wkw_lds[];
    const int w = (int)blockIdx.x / slots, b = __builtin_amdgcn_readfirstlane(ga.gr.begin(w)), e = __builtin_amdgcn_readfirstlane(ga.gr.end(w));
    const GemmArgs g{(E*)ga.C + w * ga.c_ws, (const E*)ga.A + b * ga.a_rs, (const E*)ga.B + b * ga.b_rs, nullptr,
                     1, ga.k, e - b, ga.n, 0, 1, ga.a_rs, 0, ga.b_rs, 1, 0, ga.c_rs, 1, ga.accumulate};
    gemm_wavekw_block<E, false, false, TM, TN, GW_WAVES>(g, tiles_k, tiles_n, (int)blockIdx.x - w * slots, 1, wkw_lds);
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

template <typename E, int TM, int TN>
static int launch_weights(const GroupedArgs& g) {
    constexpr size_t smem = wkw_smem<E, false, false, TM, TN, GW_WAVES>();
    const int tiles_k = (g.k + 16 * TM - 1) / (16 * TM), tiles_n = (g.n + 16 * TN - 1) / (16 * TN), slots = (tiles_k * tiles_n + 7) / 8 * 8;
    auto kern = grouped_weights_wavek_kernel<E, TM, TN>;
    if (smem > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)((long long)slots * g.gr.weights)), dim3(64 * GW_WAVES), smem, current_stream(), g, tiles_k, tiles_n, slots);
    return check_launch("grouped_weights_wavek_kernel") ? 0 : -1;
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

static int rows_tile(const GroupedArgs& g, int dtype) {
    const long long esz = (long long)dtype_size(dtype), limit = 1ll << 31;
    const bool b_kc = g.b_cs != 1;
    if (g.a_cs != 1 || (b_kc && g.b_rs != 1) || path_disabled("mfma")) return 0;
    if ((63 * g.a_rs + g.k) * esz >= limit || (b_kc ? 63 * g.b_cs + g.k : (g.k - 1) * g.b_rs + 64) * esz >= limit) return 0;      // 32-bit byte offsets from a tile's first row
    return wavek_tile(dtype, [&](int t) { return (max_row_tiles(g.gr.rows, g.gr.groups, 16 * t)) * ((g.n + 16 * t - 1) / (16 * t)); }, [&](int t) { return b_kc || g.n >= 16 * t; });
}

static int weights_tile(const GroupedArgs& g, int dtype) {
    const long long esz = (long long)dtype_size(dtype), limit = 1ll << 31;
    if (g.a_cs != 1 || g.b_cs != 1 || g.gr.ids || path_disabled("mfma")) return 0;
    if (((long long)(g.gr.rows - 1) * g.a_rs + 64) * esz >= limit || ((long long)(g.gr.rows - 1) * g.b_rs + 64) * esz >= limit) return 0;
    return wavek_tile(dtype, [&](int t) { return (long long)g.gr.weights * (((long long)((g.k + 16 * t - 1) / (16 * t)) * ((g.n + 16 * t - 1) / (16 * t)) + 7) / 8 * 8); },
                      [&](int t) { return g.k >= 16 * t && g.n >= 16 * t; });
}

bool grouped_rows_wavek_takes(const GroupedArgs& g, int dtype) { return rows_tile(g, dtype) != 0; }
bool grouped_weights_wavek_takes(const GroupedArgs& g, int dtype) { return weights_tile(g, dtype) != 0; }

template <typename E, int T>
static int launch_rows_layout(const GroupedArgs& g) { return g.b_cs == 1 ? launch_rows<E, false, T, T>(g) : launch_rows<E, true, T, T>(g); }

int launch_grouped_rows_wavek(const GroupedArgs& g, int dtype) {
    const int t = rows_tile(g, dtype);
    if (dtype == RP_DTYPE_FLOAT64) return t == 2 ? launch_rows_layout<double, 2>(g) : launch_rows_layout<double, 1>(g);
    return t == 4 ? launch_rows_layout<float, 4>(g) : t == 2 ? launch_rows_layout<float, 2>(g) : launch_rows_layout<float, 1>(g);
}

int launch_grouped_weights_wavek(const GroupedArgs& g, int dtype) {
    const int t = weights_tile(g, dtype);
    if (dtype == RP_DTYPE_FLOAT64) return t == 2 ? launch_weights<double, 2, 2>(g) : launch_weights<double, 1, 1>(g);
    return t == 4 ? launch_weights<float, 4, 4>(g) : t == 2 ? launch_weights<float, 2, 2>(g) : launch_weights<float, 1, 1>(g);
}

}  // namespace rp
