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
    return g.n <= SH_MAX_RANK && g.k >= 8 && g.a_rs >= 0 && g.a_rs < (1ll << 22) && (long long)g.k * g.n < (1 << 28) && g.a_cs == 1 && ((g.b_cs == 1 && g.b_rs == g.n) || g.b_rs == 1) && !path_disabled("mfma");
}

int launch_adapter_shrink16(const GroupedArgs& g, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? launch_shrink_rank<bf16_t>(g) : launch_shrink_rank<f16_t>(g); }

// ---- a few rows: the shared projection's shares of k and the rows' h side by side, then one launch that adds them up with the adapters' terms ----
// 32 rows with adapters of their own, 4096 x 4096 and rank 16 in bf16: 16.5 us and 4.1 (6.1 for the narrow products by themselves and 12.1 for the shared one).
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

// ---- the term by itself: y[i] += h[i] . b_a, where the shared product is too small, or a tile's rows too many segments, for its tiles to take the term in ----
// (There y has been rounded as the shared product's and is rounded once more as the sum: an operand of a whole product of any size and layout is not to be had unrounded.)
// A wave for 16 rows of a segment and 128 columns, the rank 32 at a time; h in two values of T as in the gradients.  b is read as it lies, eight rows of the rank times eight
// columns a lane, and turned with byte permutes, or, where it is contiguous along the rank, as fragments.  Bound by a few loads in a row; with multiply-adds in
// float32 and h out of the scalar cache 7 rows of rank 64 took 67 us, 5.4 now.
template <typename T, bool ALONG_RANK>
__global__ void __launch_bounds__(64) adapter_expand16_kernel(uint16_t* y, AdapterTerm term, int n, long long y_rs, int strips) {
    const RowTile rt = find_row_tile(term.gr, 16, (int)(blockIdx.x / strips));
    if (rt.group < 0) return;
    const int lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15, rank = term.rank;
    const int col = (int)(blockIdx.x % strips) * 128 + 8 * j, m = rt.end - rt.begin, left = n - col, by = pulled(left);
    const bool cut = col - 8 * j + 128 > n && n % 8;                      // (the strip's last vector ends with the row)
    const __amdgpu_buffer_rsrc_t h_rsrc = buffer_rsrc(term.h + (long long)rt.begin * rank, (long long)m * rank * 4);
    const __amdgpu_buffer_rsrc_t b_rsrc = buffer_rsrc((const uint16_t*)term.b + rt.weight * term.b_ws, ((rank - 1) * term.b_rs + (n - 1) * term.b_cs + 1) * 2);
    const __amdgpu_buffer_rsrc_t y_rsrc = buffer_rsrc(y + rt.begin * y_rs, ((m - 1) * y_rs + n) * 2);
    u32x4_t was[4];
#pragma unroll
    for (int v = 0; v < 4; v++) was[v] = __builtin_amdgcn_raw_buffer_load_b128(y_rsrc, (int)(4 * q + v < m && left > 0 ? (uint32_t)(((4 * q + v) * y_rs + col - by) * 2) : BUFFER_OOB), 0, 0);
    f32x4_t acc[8];
#pragma unroll
    for (int f = 0; f < 8; f++) acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
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
        split_low<T>(hv, hi, lo);
#pragma unroll
        for (int f = 0; f < 8; f++) {
            u32x4_t b = raw[f];
            if constexpr (!ALONG_RANK) {
#pragma unroll
                for (int d = 0; d < 4; d++) b[d] = __builtin_amdgcn_perm(raw[2 * d + 1][f / 2], raw[2 * d][f / 2], (f & 1) ? 0x07060302u : 0x05040100u);
            }
            acc[f] = sh_ops<T>::mma(hi, b, acc[f]);
            acc[f] = sh_ops<T>::mma(lo, b, acc[f]);
        }
    }
#pragma unroll
    for (int v = 0; v < 4; v++) {
        if (4 * q + v >= m || left <= 0) continue;
        const u32x4_t x = cut ? pull_into_place(was[v], by) : was[v];
        T o[8];
        __builtin_memcpy(o, &x, 16);
#pragma unroll
        for (int f = 0; f < 8; f++) o[f] = round_to<T>(widen(o[f]) + acc[f][v]);
        uint16_t* p = y + (rt.begin + 4 * q + v) * y_rs + col;
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
    return shared.n >= 8 && shared.c_rs < (1ll << 22) && (term.b_cs == 1 || term.b_rs == 1) && (long long)term.rank * shared.n < (1 << 28) && term.rank < (1 << 22) && !path_disabled("mfma");
}

template <typename T>
static int launch_expand(const GroupedArgs& shared, const AdapterTerm& term) {
    const int strips = (shared.n + 127) / 128;
    const long long blocks = max_row_tiles(term.gr.rows, term.gr.groups, 16) * strips;
    if (blocks > 0x7fffffffll) { set_error("adapters: %lld tiles are more than a launch takes", blocks); return -1; }
    if (term.b_cs == 1) hipLaunchKernelGGL((adapter_expand16_kernel<T, false>), dim3((unsigned)blocks), dim3(64), 0, current_stream(), (uint16_t*)shared.C, term, shared.n, shared.c_rs, strips);
    else hipLaunchKernelGGL((adapter_expand16_kernel<T, true>), dim3((unsigned)blocks), dim3(64), 0, current_stream(), (uint16_t*)shared.C, term, shared.n, shared.c_rs, strips);
    return check_launch("adapter_expand16_kernel") ? 0 : -1;
}

int launch_adapter_expand16(const GroupedArgs& shared, const AdapterTerm& term, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? launch_expand<bf16_t>(shared, term) : launch_expand<f16_t>(shared, term);
}

}  // namespace rp
