// bf16 / fp16 rows times an adapter's narrow factor in a launch of its own, and beside the first pass of a few rows' shared projection.
#include "rp_adapter16.h"
#include "rp_grouped_stream16.h"

namespace rp {

template <typename T, int NC, int RT, bool ALONG_K, int PIECE>
__global__ void __launch_bounds__((sh_waves<NC, PIECE>() * 64)) adapter_shrink16_kernel(GroupedArgs g, int first) {
    adapter_shrink16_block<T, NC, RT, ALONG_K, PIECE, sh_waves<NC, PIECE>()>(g, first + (int)blockIdx.x);
}

template <typename T, int NC, int RT, bool ALONG_K, int PIECE>
static int launch_shrink(const GroupedArgs& g) {
    constexpr int waves = sh_waves<NC, PIECE>(), lds = sh_lds_bytes<NC, RT, waves>(ALONG_K);
    auto kern = adapter_shrink16_kernel<T, NC, RT, ALONG_K, PIECE>;
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
    return in_launches(row_tile_numbers(g.gr.rows, g.gr.groups, 16 * RT), waves * 64, [&](unsigned blocks, long long first) -> int {
        hipLaunchKernelGGL(kern, dim3(blocks), dim3(waves * 64), lds, current_stream(), g, (int)first);
        return check_launch("adapter_shrink16_kernel") ? 0 : -1;
    });
}

template <typename T, int NC, bool ALONG_K, int PIECE>
static int launch_shrink_rows(const GroupedArgs& g) {
    // 32 rows halve what the factor is read; 16 while they leave CUs without a workgroup
    return g.gr.rows / 32 >= device_cu_count() && g.gr.rows / g.gr.groups >= 32 ? launch_shrink<T, NC, 2, ALONG_K, PIECE>(g) : launch_shrink<T, NC, 1, ALONG_K, PIECE>(g);
}

template <typename T, int NC>
static int launch_shrink_layout(const GroupedArgs& g) {
    if (g.b_cs != 1) return launch_shrink_rows<T, NC, true, 8>(g);
    if (g.n % 8 == 0 && ((uintptr_t)g.B & 15) == 0) return launch_shrink_rows<T, NC, false, 8>(g);
    return launch_shrink_rows<T, NC, false, 1>(g);
}

template <typename T>
static int launch_shrink_rank(const GroupedArgs& g) {
    if (g.n <= 16) return launch_shrink_layout<T, 1>(g);
    if (g.n <= 32) return launch_shrink_layout<T, 2>(g);
    if (g.n <= 64) return launch_shrink_layout<T, 4>(g);
    return launch_shrink_layout<T, 8>(g);
}

bool adapter_shrink16_takes(const GroupedArgs& g) {
    return g.n <= SH_MAX_RANK && g.k >= 8 && g.a_rs >= 0 && g.a_rs < (1ll << 22) && (long long)g.k * g.n < (1 << 28) && g.a_cs == 1 && ((g.b_cs == 1 && g.b_rs == g.n) || g.b_rs == 1) && !path_disabled("mfma");
}

int launch_adapter_shrink16(const GroupedArgs& g, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? launch_shrink_rank<bf16_t>(g) : launch_shrink_rank<f16_t>(g); }

// ---- a few rows: the shared projection's shares of k and the rows' h side by side, then one launch that adds them up with the adapters' terms ----
// 32 rows with adapters of their own, 4096 x 4096 and rank 16 in bf16: 16.8 us and 4.0 (6.1 for the narrow products by themselves and 12.1 for the shared one).
template <typename T, int CPL, int RB, int NC>
__global__ void __launch_bounds__(GS_THREADS) adapter_first16_kernel(GroupedArgs shared, StreamGrid sg, GroupedArgs low, int low_blocks) {
    if ((int)blockIdx.x < low_blocks) adapter_shrink16_block<T, NC, 1, false, 8, GS_WAVES>(low, (int)blockIdx.x);
    else stream16_block<T, CPL, RB>(shared, sg, blockIdx.x - low_blocks);
}

template <typename T, int CPL, int RB, int NC>
static int launch_first(const GroupedArgs& shared, const StreamGrid& sg, const GroupedArgs& low) {
    constexpr int a = gs_lds_bytes<CPL>(), b = sh_lds_bytes<NC, 1, GS_WAVES>(false), lds = a > b ? a : b;
    const long long low_blocks = (row_tile_numbers(low.gr.rows, low.gr.groups, 16) + 7) / 8 * 8, blocks = low_blocks + stream16_blocks(shared, 16 * RB, CPL, sg.nsplit);
    auto kern = adapter_first16_kernel<T, CPL, RB, NC>;
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(GS_THREADS), lds, current_stream(), shared, sg, low, (int)low_blocks);
    return check_launch("adapter_first16_kernel") ? 0 : -1;
}

template <typename T, int NC>
static int launch_first_rows(const GroupedArgs& shared, const StreamGrid& sg, const GroupedArgs& low) {
    const int rb = stream16_row_blocks(shared.gr);
    if (rb == 1) return launch_first<T, 8, 1, NC>(shared, sg, low);
    if (rb == 2) return launch_first<T, 8, 2, NC>(shared, sg, low);
    return launch_first<T, 4, 4, NC>(shared, sg, low);
}

template <typename T>
static int launch_first_rank(const GroupedArgs& shared, const StreamGrid& sg, const GroupedArgs& low) {
    if (low.n <= 16) return launch_first_rows<T, 1>(shared, sg, low);
    if (low.n <= 32) return launch_first_rows<T, 2>(shared, sg, low);
    return launch_first_rows<T, 4>(shared, sg, low);
}

bool adapter_few_rows16_takes(const GroupedArgs& shared, const GroupedArgs& low, const AdapterTerm& term) {
    return grouped_stream16_takes(shared) && adapter_shrink16_takes(low) && low.b_cs == 1 && low.n % 8 == 0 && low.n <= 64 && ((uintptr_t)low.B & 15) == 0 &&
           term.b_cs == 1 && term.b_rs % 8 == 0 && ((uintptr_t)term.b & 15) == 0;
}

// Without memory for the sums: h first, then strips of 64 columns whose epilogue adds the term (the 32 rows above 42 us)
template <typename T, int RB>
__global__ void __launch_bounds__(GS_THREADS) adapter_strips16_kernel(GroupedArgs shared, StreamGrid sg, AdapterTerm term) { stream16_block<T, 4, RB, true>(shared, sg, blockIdx.x, &term); }

template <typename T, int RB>
static int launch_strips(const GroupedArgs& shared, const StreamGrid& sg, const AdapterTerm& term) {
    static_assert(gs_lds_bytes<4>() <= 64 * 1024, "no more than every launch may have");
    hipLaunchKernelGGL((adapter_strips16_kernel<T, RB>), dim3((unsigned)stream16_blocks(shared, 16 * RB, 4, 1)), dim3(GS_THREADS), gs_lds_bytes<4>(), current_stream(), shared, sg, term);
    return check_launch("adapter_strips16_kernel") ? 0 : -1;
}

template <typename T>
static int launch_strips_rows(const GroupedArgs& shared, const StreamGrid& sg, const AdapterTerm& term) {
    const int rb = stream16_row_blocks(shared.gr);
    return rb == 1 ? launch_strips<T, 1>(shared, sg, term) : rb == 2 ? launch_strips<T, 2>(shared, sg, term) : launch_strips<T, 4>(shared, sg, term);
}

int launch_adapter_few_rows16(const GroupedArgs& shared, const GroupedArgs& low, const AdapterTerm& term, int dtype) {
    StreamGrid sg{(shared.n + 127) / 128, stream16_splits(shared, CallScratch::MOST), nullptr};
    const CallScratch sums((size_t)sg.nsplit * shared.gr.rows * shared.n * sizeof(float));
    sg.partials = (float*)sums.ptr;
    if (!sg.partials) {
        sg.nsplit = 1;
        if (launch_adapter_shrink16(low, dtype) != 0) return -1;
        return dtype == RP_DTYPE_BFLOAT16 ? launch_strips_rows<bf16_t>(shared, sg, term) : launch_strips_rows<f16_t>(shared, sg, term);
    }
    const int rc = dtype == RP_DTYPE_BFLOAT16 ? launch_first_rank<bf16_t>(shared, sg, low) : launch_first_rank<f16_t>(shared, sg, low);
    return rc == 0 ? launch_stream16_combine(shared, sg, &term, dtype) : rc;
}

// ---- the term by itself, where the shared product is too small, or a tile's rows too many segments, for its tiles to take the term in ----
// The shared product leaves float32 sums of its shares of k; y = sums + bias + h . b_a is rounded once.  A wave for 16 rows of a segment (or of none: those are only rounded)
// and 128 columns, the rank 32 at a time; h in two values of T as in the gradients.  b is read as it lies, eight rows of the rank times eight
// columns a lane, and turned with byte permutes, or, where it is contiguous along the rank, as fragments.  Bound by a few loads in a row; with multiply-adds in
// float32 and h out of the scalar cache 7 rows of rank 64 took 67 us, 6.0 now; the product's sums 3.7 (128 x 94).
struct ExpandArgs {
    uint16_t* y;
    const uint16_t* bias;
    const float* sums;             // [shares][rows][n]
    int n, rows, shares, accumulate, strips;
    long long y_rs;
};

// Tile `id` of all rows: those before the first segment, each segment's whether it has an adapter or not, those behind the last
__device__ __forceinline__ RowTile find_any_tile(const RowGroups& gr, int tile, int id) {
    const int lane = threadIdx.x & 63;
    if (gr.groups > GROUPS_ADDED_UP) {                        // (numbered as find_row_tile_number's, the rows before the first segment as segment -1)
        auto begin = [&](int i) { return i == 0 ? 0 : i <= gr.groups ? gr.begin(i - 1) : gr.end(gr.groups - 1); };
        const int i = last_of(gr.groups + 2, [&](int i) { return begin(i) / tile + i <= id; });
        auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
        RowTile t;
        t.group = uniform(i - 1);
        t.weight = uniform(i > 0 && i <= gr.groups ? gr.weight(i - 1) : -1);
        t.stop = uniform(i == 0 ? gr.begin(0) : i <= gr.groups ? gr.end(i - 1) : gr.rows);
        t.first = uniform(begin(i) / tile + i);
        t.begin = uniform(begin(i)) + (id - t.first) * tile;
        t.tiles = 0;
        t.end = t.begin + tile < t.stop ? t.begin + tile : t.stop;
        return t;
    }
    int before = 0;
    for (int g0 = 0; g0 < gr.groups + 2; g0 += 64) {
        const int g = g0 + lane - 1;
        int b = 0, e = 0, w = -1;
        if (g < 0) e = gr.begin(0);
        else if (g < gr.groups) { b = gr.begin(g); e = gr.end(g); w = gr.weight(g); }
        else if (g == gr.groups) { b = gr.end(g - 1); e = gr.rows; }
        const int tiles = (e - b + tile - 1) / tile, upto = before + wave_prefix_sum(tiles, lane);
        const unsigned long long past = __builtin_amdgcn_ballot_w64(upto > id);
        if (past) {
            const int l = __builtin_ctzll(past);
            RowTile t;
            t.group = g0 + l - 1;
            t.weight = __builtin_amdgcn_readlane(w, l);
            t.tiles = __builtin_amdgcn_readlane(tiles, l);
            t.first = __builtin_amdgcn_readlane(upto, l) - t.tiles;
            t.begin = __builtin_amdgcn_readlane(b, l) + (id - t.first) * tile;
            t.stop = __builtin_amdgcn_readlane(e, l);
            t.end = t.begin + tile < t.stop ? t.begin + tile : t.stop;
            return t;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return RowTile{-1, -1, 0, 0, 0, 0, 0};
}

template <typename T, bool ALONG_RANK>
__global__ void __launch_bounds__(64) adapter_expand16_kernel(ExpandArgs ea, AdapterTerm term, int first) {
    const int id = first + (int)blockIdx.x;
    const RowTile rt = find_any_tile(term.gr, 16, id / ea.strips);
    const int lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15, n = ea.n, m = rt.end - rt.begin;
    if (m <= 0) return;
    const int col = id % ea.strips * 128 + 8 * j, left = n - col, by = pulled(left);
    const bool cut = col - 8 * j + 128 > n && n % 8;                      // (the strip's last vector ends with the row)
    f32x4_t acc[8];                                                       // rows 4q + v, column col + f
#pragma unroll
    for (int f = 0; f < 8; f++) acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ea.shares; s++) {
        const __amdgpu_buffer_rsrc_t rsrc = buffer_rsrc(ea.sums + ((long long)s * ea.rows + rt.begin) * n, (long long)m * n * 4);
        u32x4_t p[4][2];
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int h = 0; h < 2; h++) p[v][h] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(4 * q + v < m && left > 0 ? (uint32_t)(((long long)(4 * q + v) * n + col + 4 * h) * 4) : BUFFER_OOB), 0, 0);
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int f = 0; f < 8; f++) acc[f][v] += __uint_as_float(p[v][f / 4][f % 4]);
    }
    if (rt.weight >= 0) {
        const int rank = term.rank;
        const __amdgpu_buffer_rsrc_t h_rsrc = buffer_rsrc(term.h + (long long)rt.begin * rank, (long long)m * rank * 4);
        const __amdgpu_buffer_rsrc_t b_rsrc = buffer_rsrc((const uint16_t*)term.b + rt.weight * term.b_ws, ((rank - 1) * term.b_rs + (n - 1) * term.b_cs + 1) * 2);
        for (int k0 = 0; k0 < rank; k0 += 32) {
            const int kk = k0 + 8 * q;
            float hv[8];
            u32x4_t raw[8], hi, lo;
#pragma unroll
            for (int u = 0; u < 8; u++) hv[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(h_rsrc, (int)(j < m && kk + u < rank ? (uint32_t)((j * rank + kk + u) * 4) : BUFFER_OOB), 0, 0));
            if (ALONG_RANK && rank % 8 == 0) {
#pragma unroll
                for (int f = 0; f < 8; f++) raw[f] = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, (int)(col + f < n && kk < rank ? (uint32_t)(((col + f) * term.b_cs + kk) * 2) : BUFFER_OOB), 0, 0);
            } else if (ALONG_RANK) {
#pragma unroll
                for (int f = 0; f < 8; f++) {
                    uint32_t x[8];
#pragma unroll
                    for (int u = 0; u < 8; u++) x[u] = __builtin_amdgcn_raw_buffer_load_b16(b_rsrc, (int)(col + f < n && kk + u < rank ? (uint32_t)(((col + f) * term.b_cs + kk + u) * 2) : BUFFER_OOB), 0, 0);
#pragma unroll
                    for (int d = 0; d < 4; d++) raw[f][d] = x[2 * d] | x[2 * d + 1] << 16;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) raw[e] = __builtin_amdgcn_raw_buffer_load_b128(b_rsrc, (int)(left > 0 && kk + e < rank ? (uint32_t)(((kk + e) * term.b_rs + col - by) * 2) : BUFFER_OOB), 0, 0);
                if (cut) {
#pragma unroll
                    for (int e = 0; e < 8; e++) raw[e] = pull_into_place(raw[e], by);
                }
            }
            uint32_t any = 0;
#pragma unroll
            for (int f = 0; f < 8; f++)
#pragma unroll
                for (int d = 0; d < 4; d++) any |= not_finite<T>(raw[f][d]);
            const bool odd = __builtin_amdgcn_ballot_w64(any != 0) != 0;
            float down[4];                                                // of rows 4q + v
            if constexpr (std::is_same<T, f16_t>::value) {
                uint32_t bits = 0;
                largest_bits(bits, hv);
                const uint32_t top = low_exponent(bits);
                split_scaled<T>(hv, low_up(top), hi, lo);
#pragma unroll
                for (int v = 0; v < 4; v++) down[v] = __shfl(low_down(top), 4 * q + v);
            } else {
                split_low<T>(hv, hi, lo);
            }
#pragma unroll
            for (int f = 0; f < 8; f++) {
                u32x4_t b = raw[f];
                if constexpr (!ALONG_RANK) {
#pragma unroll
                    for (int d = 0; d < 4; d++) b[d] = __builtin_amdgcn_perm(raw[2 * d + 1][f / 2], raw[2 * d][f / 2], (f & 1) ? 0x07060302u : 0x05040100u);
                }
                // (an infinity of b times a lower value that is 0 or of the other sign is not what there is to add: the higher one's product is)
                const u32x4_t b_low = odd ? finite_only<T>(b) : b;
                if constexpr (std::is_same<T, f16_t>::value) {
                    const f32x4_t x = sh_ops<T>::mma(lo, b_low, sh_ops<T>::mma(hi, b, f32x4_t{0.f, 0.f, 0.f, 0.f}));
#pragma unroll
                    for (int v = 0; v < 4; v++) acc[f][v] += x[v] * down[v];
                } else {
                    acc[f] = sh_ops<T>::mma(hi, b, acc[f]);
                    acc[f] = sh_ops<T>::mma(lo, b_low, acc[f]);
                }
            }
        }
    }
    if (left <= 0) return;
    float bias[8] = {};
    if (ea.bias) {
#pragma unroll
        for (int f = 0; f < 8; f++) { T b; b.bits = ea.bias[f < left ? col + f : col]; bias[f] = widen(b); }
    }
#pragma unroll
    for (int v = 0; v < 4; v++) {
        if (4 * q + v >= m) continue;
        uint16_t* p = ea.y + (rt.begin + 4 * q + v) * ea.y_rs + col;
        T o[8];
#pragma unroll
        for (int f = 0; f < 8; f++) o[f] = round_to<T>(acc[f][v] + bias[f]);
        if (ea.accumulate) {                                              // (the product's rounding, and the sum's)
            const u32x4_t x = pull_into_place(*(const u32x4_odd_t*)(p - by), by);
            T was[8];
            __builtin_memcpy(was, &x, 16);
#pragma unroll
            for (int f = 0; f < 8; f++) o[f] = round_to<T>(widen(was[f]) + widen(o[f]));
        }
        if (left >= 8) {
            u32x4_t z;
            __builtin_memcpy(&z, o, 16);
            *(u32x4_odd_t*)p = z;
        } else {
#pragma unroll
            for (int f = 0; f < 7; f++)
                if (f < left) p[f] = o[f].bits;
        }
    }
}

bool adapter_expand16_takes(const GroupedArgs& shared, const AdapterTerm& term) {
    return shared.n >= 8 && shared.c_rs < (1ll << 22) && shared.n < (1 << 24) && (term.b_cs == 1 || term.b_rs == 1) && (long long)term.rank * shared.n < (1 << 28) && term.rank < (1 << 22) && !path_disabled("mfma");
}

template <typename T>
static int launch_expand(const ExpandArgs& ea, const AdapterTerm& term) {
    const long long segments = term.gr.groups + 2ll, tiles = term.gr.groups > GROUPS_ADDED_UP ? term.gr.rows / 16 + segments : max_row_tiles(term.gr.rows, segments, 16);
    return in_launches(tiles * ea.strips, 64, [&](unsigned blocks, long long first) -> int {
        if (term.b_cs == 1) hipLaunchKernelGGL((adapter_expand16_kernel<T, false>), dim3(blocks), dim3(64), 0, current_stream(), ea, term, (int)first);
        else hipLaunchKernelGGL((adapter_expand16_kernel<T, true>), dim3(blocks), dim3(64), 0, current_stream(), ea, term, (int)first);
        return check_launch("adapter_expand16_kernel") ? 0 : -1;
    });
}

int launch_adapter_expand16(const GroupedArgs& s, const AdapterTerm& term, bool ragged, int dtype, bool* taken) {
    ragged = ragged || s.n % 8;                               // (the sums are stored in whole vectors otherwise)
    const int rows = s.gr.rows, cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const bool large = (long long)((rows + 127) / 128) * ((s.n + 127) / 128) * 2 >= cus;
    const int shares = large ? 1 : skinny16_sums_shares(rows, s.k, s.n);
    const CallScratch memory((size_t)shares * rows * s.n * sizeof(float), ~(size_t)0);
    float* sums = (float*)memory.ptr;
    *taken = sums != nullptr;
    if (!sums) return 0;
    const GemmArgs g{nullptr, s.A, s.B, nullptr, 1, rows, s.k, s.n, 0, s.a_rs, s.a_cs, 0, s.b_rs, s.b_cs, 0, s.n, 1, 0};
    Plan p{FAM_MFMA16_SKINNY, 32, 128, false, s.b_cs == 1, true, ""};
    p.ragged = ragged;
    const int rc = large ? launch_sums16_128(g, p.b_mc, ragged, sums, dtype) : launch_skinny16_sums(g, p, sums, dtype);
    const ExpandArgs ea{(uint16_t*)s.C, (const uint16_t*)s.bias, sums, s.n, rows, shares, s.accumulate, (s.n + 127) / 128, s.c_rs};
    if (rc != 0) return rc;
    return dtype == RP_DTYPE_BFLOAT16 ? launch_expand<bf16_t>(ea, term) : launch_expand<f16_t>(ea, term);
}

}  // namespace rp
