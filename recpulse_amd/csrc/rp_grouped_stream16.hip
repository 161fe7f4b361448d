// Launches of the kernel for a few rows a group (rp_grouped_stream16.h), and the second launch that adds shares of k.
#include "rp_grouped_stream16.h"

namespace rp {

template <typename T, int CPL, int RB>
__global__ void __launch_bounds__(GS_THREADS) grouped_stream16_kernel(GroupedArgs g, StreamGrid sg, long long first) { stream16_block<T, CPL, RB>(g, sg, first + blockIdx.x); }

// y[row] = the shares' sums in order + bias + what the row's adapter adds, rounded once; rows of no group are left alone.  A workgroup does 32
// vectors of 8 columns of one row: eight threads share a vector's shares of k and its rank, and their sums are added in order.  The loads
// of a thread are two or three, so the launch takes the time of a few round trips.
template <typename T>
__global__ void __launch_bounds__(256) stream16_combine_kernel(GroupedArgs g, StreamGrid sg, AdapterTerm term, int blocks_per_row) {
    __shared__ __attribute__((aligned(16))) float parts[8][32][8];
    const int row = (int)(blockIdx.x / blocks_per_row), col = ((int)(blockIdx.x % blocks_per_row) * 32 + (threadIdx.x & 31)) * 8, part = threadIdx.x >> 5;
    const bool in = col < g.n;
    float s[8];
#pragma unroll
    for (int v = 0; v < 8; v++) s[v] = 0.f;
    for (int p = part; p < sg.nsplit && in; p += 8) {
        const float* at = sg.partials + ((long long)p * g.gr.rows + row) * g.n + col;
        const f32x4_t lo = *(const f32x4_t*)at, hi = *(const f32x4_t*)(at + 4);
#pragma unroll
        for (int v = 0; v < 4; v++) { s[v] += lo[v]; s[4 + v] += hi[v]; }
    }
    // the weight of the row's group: a wave looks at 64 groups at a time
    auto weight_of = [&](const RowGroups& gr) {
        const int lane = threadIdx.x & 63;
        for (int g0 = 0; g0 < gr.groups; g0 += 64) {
            const bool in = g0 + lane < gr.groups;
            const int b = in ? gr.begin(g0 + lane) : 0, e = in ? gr.end(g0 + lane) : 0, w = in ? gr.weight(g0 + lane) : -1;
            const unsigned long long here = __builtin_amdgcn_ballot_w64(b <= row && row < e);
            if (here) return __builtin_amdgcn_readlane(w, __builtin_ctzll(here));
        }
        return -1;
    };
    const int a = term.h ? weight_of(term.gr) : -1, w = weight_of(g.gr);
    if (w < 0) return;                                       // (the whole workgroup)
    {
        if (a >= 0 && in) {
            const float* h = term.h + (long long)row * term.rank;
            const uint16_t* b = (const uint16_t*)term.b + a * term.b_ws + col;
#pragma unroll 4
            for (int r = part; r < term.rank; r += 8) {
                const float hr = h[r];
                T e[8];
                const u32x4_t x = *(const u32x4_t*)(b + r * term.b_rs);
                __builtin_memcpy(e, &x, 16);
#pragma unroll
                for (int v = 0; v < 8; v++) s[v] += hr * widen(e[v]);
            }
        }
    }
    *(f32x4_t*)&parts[part][threadIdx.x & 31][0] = f32x4_t{s[0], s[1], s[2], s[3]};
    *(f32x4_t*)&parts[part][threadIdx.x & 31][4] = f32x4_t{s[4], s[5], s[6], s[7]};
    __syncthreads();
    // a column a thread
    const int c = threadIdx.x, gc = (int)(blockIdx.x % blocks_per_row) * 256 + c;
    if (gc >= g.n) return;
    float t = parts[0][c >> 3][c & 7];
#pragma unroll
    for (int p = 1; p < 8; p++) t += parts[p][c >> 3][c & 7];
    if (g.bias) t += widen(((const T*)g.bias)[(long long)w * g.n + gc]);
    T* out = (T*)g.C + row * g.c_rs + gc;
    T y = round_to<T>(t);
    if (g.accumulate) y = round_to<T>(widen(*out) + widen(y));
    *out = y;
}

int launch_stream16_combine(const GroupedArgs& g, const StreamGrid& sg, const AdapterTerm* term, int dtype) {
    const int per_row = (g.n + 255) / 256;
    const dim3 grid((unsigned)(g.gr.rows * per_row));
    if (dtype == RP_DTYPE_BFLOAT16) hipLaunchKernelGGL(stream16_combine_kernel<bf16_t>, grid, dim3(256), 0, current_stream(), g, sg, term ? *term : AdapterTerm{}, per_row);
    else hipLaunchKernelGGL(stream16_combine_kernel<f16_t>, grid, dim3(256), 0, current_stream(), g, sg, term ? *term : AdapterTerm{}, per_row);
    return check_launch("stream16_combine_kernel") ? 0 : -1;
}

template <typename T, int CPL, int RB>
static int launch_stream(const GroupedArgs& g, StreamGrid sg) {
    constexpr int lds = gs_lds_bytes<CPL>();
    auto kern = grouped_stream16_kernel<T, CPL, RB>;
    if (lds > 64 * 1024 && !check_hip(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, lds), "hipFuncSetAttribute")) return -1;
    return in_launches(stream16_blocks(g, 16 * RB, CPL, sg.nsplit), GS_THREADS, [&](unsigned blocks, long long first) -> int {
        hipLaunchKernelGGL(kern, dim3(blocks), dim3(GS_THREADS), lds, current_stream(), g, sg, first);
        return check_launch("grouped_stream16_kernel") ? 0 : -1;
    });
}

template <typename T, int CPL>
static int launch_stream_rows(const GroupedArgs& g, const StreamGrid& sg) {
    const int rb = stream16_row_blocks(g.gr);
    if (rb == 1) return launch_stream<T, CPL, 1>(g, sg);
    if (rb == 2) return launch_stream<T, CPL, 2>(g, sg);
    return launch_stream<T, 4, 4>(g, sg);                     // (64 rows of the wider strips do not fit the registers)
}

template <typename T>
static int launch_stream_t(const GroupedArgs& g, int dtype) {
    StreamGrid sg{(g.n + 127) / 128, 1, nullptr};
    // a second launch is worth its 4 us from about 2048 of k on (us, one weight of n = 4096 and one row, 64-column strips and shares of k: k = 1024 8.2 / 11.2, 4096 19.2 / 12.1)
    const int want = g.k < 2048 ? 1 : stream16_splits(g, CallScratch::MOST);
    if (want == 1) {
        const long long used = g.gr.groups < g.gr.rows ? g.gr.groups : g.gr.rows;
        const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
        return used * sg.pieces * 4 >= cus * 3ll ? launch_stream_rows<T, 8>(g, sg) : launch_stream_rows<T, 4>(g, sg);
    }
    const CallScratch sums((size_t)want * g.gr.rows * g.n * sizeof(float));
    sg.partials = (float*)sums.ptr;
    if (!sg.partials) return launch_stream_rows<T, 4>(g, sg);
    sg.nsplit = want;
    const int rc = launch_stream_rows<T, 8>(g, sg);
    return rc == 0 ? launch_stream16_combine(g, sg, nullptr, dtype) : rc;
}

bool grouped_stream16_takes(const GroupedArgs& g) {
    if (path_disabled("stream16") || path_disabled("mfma")) return false;
    if (g.a_cs != 1 || g.b_cs != 1 || g.k % 8 || g.n % 8 || g.a_rs % 8 || g.b_rs % 8 || g.b_ws % 8 || g.c_rs % 8) return false;
    if (((uintptr_t)g.A | (uintptr_t)g.B | (uintptr_t)g.C | (uintptr_t)g.bias) & 15) return false;
    if (g.b_rs < g.n || g.b_rs >= (1ll << 22) || g.a_rs >= (1ll << 22)) return false;      // 32-bit offsets within a round
    return g.gr.rows / g.gr.groups <= 48;
}

int launch_grouped_stream16(const GroupedArgs& g, int dtype) { return dtype == RP_DTYPE_BFLOAT16 ? launch_stream_t<bf16_t>(g, dtype) : launch_stream_t<f16_t>(g, dtype); }

}  // namespace rp
