// bf16 / fp16 rows times an adapter's narrow factor in a launch of its own, and beside the first pass of a few rows' shared projection.
#include "rp_adapter16.h"
#include "rp_grouped_stream16.h"

namespace rp {

template <typename T, int NC, int RT, bool ALONG_K, int PIECE>
__global__ void __launch_bounds__((sh_waves<NC, PIECE>() * 64)) adapter_shrink16_kernel(GroupedArgs g) {
    adapter_shrink16_block<T, NC, RT, ALONG_K, PIECE, sh_waves<NC, PIECE>()>(g, (int)blockIdx.x);
}

template <typename T, int NC, int RT, bool ALONG_K, int PIECE>
static int launch_shrink(const GroupedArgs& g) {
    constexpr int waves = sh_waves<NC, PIECE>(), lds = sh_lds_bytes<NC, RT, waves>(ALONG_K);
    auto kern = adapter_shrink16_kernel<T, NC, RT, ALONG_K, PIECE>;
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
    hipLaunchKernelGGL(kern, dim3((unsigned)max_row_tiles(g.gr.rows, g.gr.groups, 16 * RT)), dim3(waves * 64), lds, current_stream(), g);
    return check_launch("adapter_shrink16_kernel") ? 0 : -1;
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
    return g.n <= SH_MAX_RANK && g.a_cs == 1 && ((g.b_cs == 1 && g.b_rs == g.n) || g.b_rs == 1) && !path_disabled("mfma");
}

int launch_adapter_shrink16(const GroupedArgs& g, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? launch_shrink_rank<bf16_t>(g) : launch_shrink_rank<f16_t>(g); }

// ---- a few rows: the shared projection's shares of k and the rows' h side by side, then one launch that adds them up with the adapters' terms ----
// 32 rows with adapters of their own, 4096 x 4096 and rank 16 in bf16: 17.9 us and 6.9 (6.1 for the narrow products by themselves and 12.1 for the shared one).
template <typename T, int CPL, int RB, int NC>
__global__ void __launch_bounds__(GS_THREADS) adapter_first16_kernel(GroupedArgs shared, StreamGrid sg, GroupedArgs low, int low_blocks) {
    if ((int)blockIdx.x < low_blocks) adapter_shrink16_block<T, NC, 1, false, 8, GS_WAVES>(low, (int)blockIdx.x);
    else stream16_block<T, CPL, RB>(shared, sg, blockIdx.x - low_blocks);
}

template <typename T, int CPL, int RB, int NC>
static int launch_first(const GroupedArgs& shared, const StreamGrid& sg, const GroupedArgs& low) {
    constexpr int a = gs_lds_bytes<CPL>(), b = sh_lds_bytes<NC, 1, GS_WAVES>(false), lds = a > b ? a : b;
    const long long low_blocks = (max_row_tiles(low.gr.rows, low.gr.groups, 16) + 7) / 8 * 8, blocks = low_blocks + stream16_blocks(shared, 16 * RB, CPL, sg.nsplit);
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

int launch_adapter_few_rows16(const GroupedArgs& shared, const GroupedArgs& low, const AdapterTerm& term, int dtype) {
    // The sums lie in the null stream's own memory, or, as the split products of rp_hip_gemm_strided_batched do, in a block of the pool.
    constexpr size_t most = 16 << 20;
    StreamGrid sg{(shared.n + 127) / 128, stream16_splits(shared, most), nullptr};
    const size_t bytes = (size_t)sg.nsplit * shared.gr.rows * shared.n * sizeof(float);
    NullStreamScratch lease(bytes);
    void* block = nullptr;
    if (!lease.ptr && rp_hip_malloc(&block, bytes) != 0) return -1;
    sg.partials = (float*)(lease.ptr ? lease.ptr : block);
    int rc = dtype == RP_DTYPE_BFLOAT16 ? launch_first_rank<bf16_t>(shared, sg, low) : launch_first_rank<f16_t>(shared, sg, low);
    if (rc == 0) rc = launch_stream16_combine(shared, sg, &term, dtype);
    if (block) rp_hip_free(block);
    return rc;
}

// ---- the term by itself: y[i] += h[i] . b_a, where the shared product is too small for tiles that would fill the CUs ----
// 16 rows of a segment and 512 columns a workgroup (one wave), 8 columns a lane: b is read once for the 16 rows, h through the scalar cache.
template <typename T, bool ALONG_RANK>
__global__ void __launch_bounds__(64) adapter_expand16_kernel(uint16_t* y, AdapterTerm term, int n, long long y_rs, int parts) {
    const RowTile rt = find_row_tile(term.gr, 16, (int)(blockIdx.x / parts));
    if (rt.group < 0) return;
    const int col = (int)(blockIdx.x % parts) * 512 + threadIdx.x * 8, m = rt.end - rt.begin, there = n - col;
    if (there <= 0) return;
    const float* h = term.h + (long long)rt.begin * term.rank;
    const uint16_t* b = (const uint16_t*)term.b + rt.weight * term.b_ws + (long long)col * term.b_cs;
    float acc[16][8];
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
        for (int v = 0; v < 8; v++) acc[i][v] = 0.f;
    auto multiply = [&](const T (&bv)[8], int r) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (i < m) {                                                  // (uniform)
                const float hr = h[(long long)i * term.rank + r];
#pragma unroll
                for (int v = 0; v < 8; v++) acc[i][v] += hr * widen(bv[v]);
            }
        }
    };
    if constexpr (ALONG_RANK) {
        for (int r0 = 0; r0 < term.rank; r0 += 8) {
            T cols[8][8], bv[8];
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const u32x4_t x = load8(b + (v < there ? v : 0) * term.b_cs + r0, term.rank - r0);
                __builtin_memcpy(cols[v], &x, 16);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                if (r0 + u < term.rank) {
#pragma unroll
                    for (int v = 0; v < 8; v++) bv[v] = cols[v][u];
                    multiply(bv, r0 + u);
                }
            }
        }
    } else {
#pragma unroll 4
        for (int r = 0; r < term.rank; r++) {
            T bv[8];
            const u32x4_t x = load8(b + r * term.b_rs, there);
            __builtin_memcpy(bv, &x, 16);
            multiply(bv, r);
        }
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        if (i >= m) continue;
        uint16_t* p = y + (rt.begin + i) * y_rs + col;
        T o[8];
        const u32x4_t was = load8(p, there);
        __builtin_memcpy(o, &was, 16);
#pragma unroll
        for (int v = 0; v < 8; v++) o[v] = round_to<T>(widen(o[v]) + acc[i][v]);
        if (there >= 8) {
            u32x4_t x;
            __builtin_memcpy(&x, o, 16);
            *(u32x4_odd_t*)p = x;
        } else {
#pragma unroll
            for (int v = 0; v < 7; v++)
                if (v < there) p[v] = o[v].bits;
        }
    }
}

bool adapter_expand16_takes(const GroupedArgs& shared, const AdapterTerm& term) { return (term.b_cs == 1 || term.b_rs == 1) && !path_disabled("mfma"); }

template <typename T>
static int launch_expand(const GroupedArgs& shared, const AdapterTerm& term) {
    const int parts = (shared.n + 511) / 512;
    const long long blocks = max_row_tiles(term.gr.rows, term.gr.groups, 16) * parts;
    if (blocks > 0x7fffffffll) { set_error("adapters: %lld tiles are more than a launch takes", blocks); return -1; }
    if (term.b_cs == 1) hipLaunchKernelGGL((adapter_expand16_kernel<T, false>), dim3((unsigned)blocks), dim3(64), 0, current_stream(), (uint16_t*)shared.C, term, shared.n, shared.c_rs, parts);
    else hipLaunchKernelGGL((adapter_expand16_kernel<T, true>), dim3((unsigned)blocks), dim3(64), 0, current_stream(), (uint16_t*)shared.C, term, shared.n, shared.c_rs, parts);
    return check_launch("adapter_expand16_kernel") ? 0 : -1;
}

int launch_adapter_expand16(const GroupedArgs& shared, const AdapterTerm& term, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? launch_expand<bf16_t>(shared, term) : launch_expand<f16_t>(shared, term);
}

}  // namespace rp
