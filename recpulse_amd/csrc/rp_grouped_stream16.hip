// bf16 / fp16 rows in groups of a few rows each against row-major weights: decoding with experts, or with adapters beside a shared weight.
//
// Bound by reading the weights: every weight that has a row is read once.  As in the few-row kernel for one matrix
// (rp_gemm_mfma16_stream128.hip) they go from memory to registers to the MFMAs: lane (q, j) = (lane / 16, lane % 16) loads CPL adjacent
// columns of eight rows of k (8q .. 8q + 7), the 8 x CPL block is transposed in registers with byte permutes, and column residue c becomes the
// operand of one v_mfma_f32_16x16x32 whose column j is column CPL * j + c of the strip.  The rows of x are the other operand, 16 bytes a lane.
//
// A workgroup owns 16 * RB rows of one group and a strip of 16 * CPL columns; its eight waves share k, 32 rows of it at a time in turn, two
// rounds in flight each, and add their tiles through LDS in wave order: one launch, no workspace, repeatable bits.  Strips are as wide
// as leaves about a workgroup a CU (launch_grouped_stream16).
#include "rp_grouped.h"

#include <type_traits>

namespace rp {

constexpr int GS_WAVES = 8, GS_ROUND = 32;

template <typename T> struct gs_ops;
template <> struct gs_ops<bf16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
};
template <> struct gs_ops<f16_t> {
    static __device__ __forceinline__ f32x4_t mma(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
};

template <int CPL> struct gs_vec;                    // CPL 16-bit values
template <> struct gs_vec<8> { using type = u32x4_t; };
template <> struct gs_vec<4> { using type = u32x2_t; };
template <> struct gs_vec<2> { using type = uint32_t; };
template <int CPL> __device__ __forceinline__ uint32_t gs_word(typename gs_vec<CPL>::type v, int i) {
    if constexpr (CPL == 2) return v;
    else return v[i];
}
template <int CPL> __device__ __forceinline__ typename gs_vec<CPL>::type gs_load(__amdgpu_buffer_rsrc_t r, uint32_t off) {       // (streamed: read once)
    if constexpr (CPL == 8) return __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 2);
    else if constexpr (CPL == 4) return __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 2);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 2);
}

// ADAPT: `term` is added to the rows (one group; the rows' adapters in `term`)
template <typename T, int CPL, int RB, bool ADAPT>
__global__ void __launch_bounds__(GS_WAVES * 64, 2) grouped_stream16_kernel(GroupedArgs g, AdapterTerm term, int strips) {
    constexpr int COLS = 16 * CPL, PITCH = COLS + 4, ROWS = 16 * RB;
    extern __shared__ __attribute__((aligned(16))) float gs_sums[];       // [GS_WAVES][16][PITCH]
    const RowTile rt = find_row_tile(g.gr, ROWS, (int)(blockIdx.x / strips));
    if (rt.group < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, j = lane & 15;
    const int n0 = (int)(blockIdx.x % strips) * COLS, m = rt.end - rt.begin;
    const uint16_t* B = (const uint16_t*)g.B + rt.weight * g.b_ws + n0;
    const uint16_t* A = (const uint16_t*)g.A + rt.begin * g.a_rs;
    const __amdgpu_buffer_rsrc_t b_rsrc = buffer_rsrc(B, ((long long)(g.k - 1) * g.b_rs + g.n - n0) * 2), a_rsrc = buffer_rsrc(A, ((long long)(m - 1) * g.a_rs + g.k) * 2);
    const bool col_in = n0 + CPL * j < g.n;                               // (n is a multiple of 8)
    const uint32_t b_lane = (uint32_t)((8 * q * g.b_rs + CPL * j) * 2), b_step = (uint32_t)(g.b_rs * 2);
    uint32_t a_lane[RB];
#pragma unroll
    for (int i = 0; i < RB; i++) a_lane[i] = 16 * i + j < m ? (uint32_t)(((16 * i + j) * g.a_rs + 8 * q) * 2) : BUFFER_OOB;

    typename gs_vec<CPL>::type raw[2][8];
    u32x4_t av[2][RB];
    auto request = [&](auto slotc, int k0) {                              // (rounds past k read zeros)
        constexpr int S = decltype(slotc)::value;
#pragma unroll
        for (int e = 0; e < 8; e++) raw[S][e] = gs_load<CPL>(b_rsrc, col_in && k0 + 8 * q + e < g.k ? b_lane + (uint32_t)(k0 + e) * b_step : BUFFER_OOB);
#pragma unroll
        for (int i = 0; i < RB; i++) av[S][i] = __builtin_amdgcn_raw_buffer_load_b128(a_rsrc, (int)(k0 + 8 * q < g.k ? a_lane[i] + 2 * k0 : BUFFER_OOB), 0, 0);      // (k is a multiple of 8)
    };
    f32x4_t acc[RB][CPL];
#pragma unroll
    for (int i = 0; i < RB; i++)
#pragma unroll
        for (int c = 0; c < CPL; c++) acc[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](auto slotc) {
        constexpr int S = decltype(slotc)::value;
#pragma unroll
        for (int c = 0; c < CPL; c++) {
            u32x4_t b;
#pragma unroll
            for (int d = 0; d < 4; d++) b[d] = __builtin_amdgcn_perm(gs_word<CPL>(raw[S][2 * d + 1], c / 2), gs_word<CPL>(raw[S][2 * d], c / 2), (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int i = 0; i < RB; i++) acc[i][c] = gs_ops<T>::mma(av[S][i], b, acc[i][c]);
        }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    constexpr int TURN = GS_WAVES * GS_ROUND;
    const int first = wave * GS_ROUND;
    request(S0{}, first);
    request(S1{}, first + TURN);

    // this thread's outputs: EACH vectors of 8 columns of a row
    constexpr int VPR = COLS / 8, EACH = (ROWS * VPR + GS_WAVES * 64 - 1) / (GS_WAVES * 64);
    float extra[EACH][8];
#pragma unroll
    for (int o = 0; o < EACH; o++) {
        const int id = threadIdx.x + o * GS_WAVES * 64, row = id / VPR, col = n0 + id % VPR * 8;
        const bool in = row < m && col < g.n;
#pragma unroll
        for (int v = 0; v < 8; v++) extra[o][v] = 0.f;
        if (in && g.bias) {
            T e[8];
            const u32x4_t w = *(const u32x4_t*)((const uint16_t*)g.bias + (long long)rt.weight * g.n + col);
            __builtin_memcpy(e, &w, 16);
#pragma unroll
            for (int v = 0; v < 8; v++) extra[o][v] = widen(e[v]);
        }
        if constexpr (ADAPT) {                                            // (while the first rounds are on their way)
            const int a = in ? term.gr.weight_of_row(rt.begin + row) : -1;
            if (a >= 0) {
                const float* h = term.h + (long long)(rt.begin + row) * term.rank;
                const uint16_t* b = (const uint16_t*)term.b + a * term.b_ws + col;
#pragma unroll 4
                for (int r = 0; r < term.rank; r++) {
                    const float hr = h[r];
                    T e[8];
                    const u32x4_t w = *(const u32x4_t*)(b + r * term.b_rs);
                    __builtin_memcpy(e, &w, 16);
#pragma unroll
                    for (int v = 0; v < 8; v++) extra[o][v] += hr * widen(e[v]);
                }
            }
        }
    }

    for (int k0 = first; k0 < g.k; k0 += 2 * TURN) {
        multiply(S0{});
        request(S0{}, k0 + 2 * TURN);
        multiply(S1{});
        request(S1{}, k0 + 3 * TURN);
    }

    static_for<0, RB>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (i) __syncthreads();
#pragma unroll
        for (int v = 0; v < 4; v++)
#pragma unroll
            for (int c = 0; c < CPL; c += 2) {
                float* at = gs_sums + (wave * 16 + 4 * q + v) * PITCH + CPL * j + c;
                at[0] = acc[i][c][v];
                at[1] = acc[i][c + 1][v];
            }
        __syncthreads();
#pragma unroll
        for (int o = 0; o < EACH; o++) {
            const int id = threadIdx.x + o * GS_WAVES * 64, row = id / VPR, cv = id % VPR * 8;
            if (row / 16 != i || row >= m || n0 + cv >= g.n) continue;
            float s[8];
#pragma unroll
            for (int v = 0; v < 8; v++) s[v] = 0.f;
#pragma unroll
            for (int w = 0; w < GS_WAVES; w++) {
                const float* at = gs_sums + (w * 16 + row % 16) * PITCH + cv;
                const f32x4_t lo = *(const f32x4_t*)at, hi = *(const f32x4_t*)(at + 4);
#pragma unroll
                for (int v = 0; v < 4; v++) { s[v] += lo[v]; s[4 + v] += hi[v]; }
            }
            uint16_t* out = (uint16_t*)g.C + (rt.begin + row) * g.c_rs + n0 + cv;
            T y[8];
#pragma unroll
            for (int v = 0; v < 8; v++) y[v] = round_to<T>(s[v] + extra[o][v]);
            if (g.accumulate) {
                T was[8];
                __builtin_memcpy(was, out, 16);
#pragma unroll
                for (int v = 0; v < 8; v++) y[v] = round_to<T>(widen(was[v]) + widen(y[v]));
            }
            __builtin_memcpy(out, y, 16);
        }
    });
}

template <typename T, int CPL, int RB>
static int launch_stream(const GroupedArgs& g, const AdapterTerm* term) {
    constexpr int lds = GS_WAVES * 16 * (16 * CPL + 4) * 4;
    const int strips = (g.n + 16 * CPL - 1) / (16 * CPL);
    const long long blocks = max_row_tiles(g.gr.rows, g.gr.groups, 16 * RB) * strips;
    if (blocks > 0x7fffffffll) { set_error("grouped product: %lld tiles are more than a launch takes", blocks); return -1; }
    auto launch = [&](auto kern) {
        if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
        hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(GS_WAVES * 64), lds, current_stream(), g, term ? *term : AdapterTerm{}, strips);
        return check_launch("grouped_stream16_kernel") ? 0 : -1;
    };
    return term ? launch(grouped_stream16_kernel<T, CPL, RB, true>) : launch(grouped_stream16_kernel<T, CPL, RB, false>);
}

template <typename T, int CPL>
static int launch_stream_rows(const GroupedArgs& g, const AdapterTerm* term) {
    const int mean = (g.gr.rows + g.gr.groups - 1) / g.gr.groups;
    if (g.gr.groups == 1 ? mean <= 16 : mean <= 10) return launch_stream<T, CPL, 1>(g, term);
    if (g.gr.groups == 1 ? mean <= 32 : mean <= 20) return launch_stream<T, CPL, 2>(g, term);
    return launch_stream<T, CPL, 4>(g, term);
}

template <typename T>
static int launch_stream_width(const GroupedArgs& g, const AdapterTerm* term) {
    const long long used = g.gr.groups < g.gr.rows ? g.gr.groups : g.gr.rows;        // groups that have a row, at most
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
    if (used * ((g.n + 127) / 128) * 4 >= cus * 3) return launch_stream_rows<T, 8>(g, term);
    if (used * ((g.n + 63) / 64) * 4 >= cus * 3) return launch_stream_rows<T, 4>(g, term);
    return launch_stream_rows<T, 2>(g, term);
}

bool grouped_stream16_takes(const GroupedArgs& g) {
    if (path_disabled("stream16") || path_disabled("mfma")) return false;
    if (g.a_cs != 1 || g.b_cs != 1 || g.k % 8 || g.n % 8 || g.a_rs % 8 || g.b_rs % 8 || g.b_ws % 8 || g.c_rs % 8) return false;
    if (((uintptr_t)g.A | (uintptr_t)g.B | (uintptr_t)g.C | (uintptr_t)g.bias) & 15) return false;
    if (g.b_rs < g.n || (long long)(g.k + 2 * GS_WAVES * GS_ROUND + 64) * g.b_rs * 2 >= (1ll << 31) || (64 * g.a_rs + g.k) * 2 >= (1ll << 31)) return false;      // 32-bit offsets
    return g.gr.rows / g.gr.groups <= 48;
}

int launch_grouped_stream16(const GroupedArgs& g, const AdapterTerm* term, int dtype) {
    return dtype == RP_DTYPE_BFLOAT16 ? launch_stream_width<bf16_t>(g, term) : launch_stream_width<f16_t>(g, term);
}

}  // namespace rp
