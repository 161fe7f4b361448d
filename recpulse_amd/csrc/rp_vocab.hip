// Entry points of the cross entropy of a large vocabulary, and its pieces for any strides, sizes and types.
//
//   z = x . W + b;  m, s: the row's running largest and sum of exp(z - m);  loss_i = m + log s - z[i, t_i]
//   d[i, v] = (exp(z[i, v] - lse_i) - [v = t_i]) f_i,  dx = d . W^T,  dW = x^T . d,  db = sum of d over the rows
//
// f_i: the upstream gradient, for the mean over the rows with a target divided by their number, 0 for a row without one.  The kernels here take a piece of the vocabulary at a
// time through the plain products in the accumulate type: 16-bit operands are widened first.
#include "rp_vocab.h"

namespace rp {

constexpr long long VOCAB_PIECE_BYTES = 64ll << 20;      // of a piece's logits
// ... and of a piece of W that is widened first, and of its dW (bf16, w with a column stride of 2, us forward / backward with 64, 128 and 256 MiB and with one piece of all classes: 64 rows, 4096 -> 32768
// 613 / 1390, 602 / 1342, 574 / 1310, 625 / 1348; 512, 2048 -> 32000 760 / 1890, 544 / 1627, 565 / 1650, 564 / 1645; 8, 4096 -> 131072 2608 / 4918, 2200 / 4507, 2067 / 4325, 2016 / 4755, which take 160,
// 289, 545 and 2083 MiB)
constexpr long long VOCAB_WIDE_BYTES = 128ll << 20;
constexpr size_t VOCAB_GEMM_BYTES = 16 << 20;            // for the partial sums of its products
// Few rows: dx of a piece is split along its classes, 2048 a share, and 32 shares of 8 rows and 16384 float32 fill that memory
constexpr int VOCAB_FEW_ROWS = 8, VOCAB_FEW_PIECE = 65536;
constexpr int VOCAB_GRID = 1 << 20;                      // (of 1024 threads: fewer than 2^32)

static int vocab_piece(int rows, int classes, int elem, long long bytes) {
    const long long fits = bytes / ((long long)rows * elem) / 256 * 256, all = (classes + 255ll) / 256 * 256;
    return (int)(fits < 256 ? 256 : fits < all ? fits : all);
}

// ---- kernels of the pieces ----

// out[i, j] dense = in[i, j] widened
template <typename T>
__global__ void __launch_bounds__(256) vocab_widen_kernel(typename traits<T>::acc* out, const T* in, int rows, int cols, long long rs, long long cs) {
    const long long total = (long long)rows * cols;
    for (long long id = blockIdx.x * 256ll + threadIdx.x; id < total; id += gridDim.x * 256ll) {
        // neighbouring threads along the axis with the smaller stride
        const int i = (int)(cs <= rs ? id / cols : id % rows), j = (int)(cs <= rs ? id % cols : id / rows);
        out[(long long)i * cols + j] = widen(in[i * rs + j * cs]);
    }
}
// out[i, j] (+)= in[i, j] dense, rounded
template <typename T>
__global__ void __launch_bounds__(256) vocab_round_kernel(T* out, const typename traits<T>::acc* in, int rows, int cols, long long rs, long long cs, int accumulate) {
    const long long total = (long long)rows * cols;
    for (long long id = blockIdx.x * 256ll + threadIdx.x; id < total; id += gridDim.x * 256ll) {
        const int i = (int)(cs <= rs ? id / cols : id % rows), j = (int)(cs <= rs ? id % cols : id / rows);
        T* at = out + i * rs + j * cs;
        const auto v = in[(long long)i * cols + j];
        *at = round_to<T>(accumulate ? widen(*at) + v : v);
    }
}
static unsigned flat_grid(long long total) {
    const long long blocks = (total + 255) / 256;
    return (unsigned)(blocks < VOCAB_GRID ? blocks : VOCAB_GRID);
}

// A row of logits takes a workgroup of 1024 threads where there are few (f32, 567 x 29440, us with 256 and 1024: the state 78 / 19, d 54 / 24), each with eight values in flight
constexpr int VOCAB_AT_ONCE = 8;
static int vocab_threads(int rows) { return rows <= 4 * (device_cu_count() > 0 ? device_cu_count() : 256) ? 1024 : 256; }

// The piece's share of each row's running largest logit, sum and target's logit: state [rows][3]
template <typename A, int THREADS>
__global__ void __launch_bounds__(THREADS) vocab_state_kernel(A* state, const A* z, const int* targets, int rows, int width, int v0, int first) {
    __shared__ A room[2 * (THREADS / 64)];
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const A* zr = z + (long long)row * width;
        A* st = state + 3ll * row;
        const A was = first ? -(A)INFINITY : st[0];
        A own = -(A)INFINITY, own_sum = 0;
        for (int c0 = threadIdx.x; c0 < width; c0 += THREADS * VOCAB_AT_ONCE) {
            A v[VOCAB_AT_ONCE], most = own;
#pragma unroll
            for (int u = 0; u < VOCAB_AT_ONCE; u++) v[u] = c0 + u * THREADS < width ? zr[c0 + u * THREADS] : -(A)INFINITY;
#pragma unroll
            for (int u = 0; u < VOCAB_AT_ONCE; u++) most = larger(most, v[u]);
            const A base = most == -(A)INFINITY ? (A)0 : most;
            own_sum *= natural_exp(own - base);
#pragma unroll
            for (int u = 0; u < VOCAB_AT_ONCE; u++) own_sum += natural_exp(v[u] - base);
            own = most;
        }
        const A top = team_max<THREADS>(larger(own, was), room), base = top == -(A)INFINITY ? (A)0 : top;
        A sum[1] = {own_sum * natural_exp(own - base)};
        team_sums<THREADS>(sum, room + THREADS / 64);
        if (threadIdx.x == 0) {
            st[1] = (first || was == -(A)INFINITY ? (A)0 : st[1] * natural_exp(was - base)) + sum[0];
            st[0] = top;
            const int t = targets[row] - v0;
            if (targets[row] >= 0 && t >= 0 && t < width) st[2] = zr[t];
        }
        __syncthreads();
    }
}
// lse and loss of each row from its state
template <typename A>
__global__ void __launch_bounds__(256) vocab_rows_kernel(A* stats, const A* state, const int* targets, int rows, int classes) {
    for (int row = (int)(blockIdx.x * 256 + threadIdx.x); row < rows; row += (int)gridDim.x * 256) {
        const A* st = state + 3ll * row;
        const A lse = st[0] == -(A)INFINITY ? st[0] : st[0] + natural_log(st[1]);
        stats[row] = lse;
        stats[rows + row] = targets[row] >= 0 && targets[row] < classes ? lse - st[2] : (A)0;
    }
}
// The result, and how many rows have a target: one workgroup, in double, whose threads' sums are added in order
template <typename A>
__global__ void __launch_bounds__(1024) vocab_loss_kernel(A* out, A* stats, const int* targets, int rows, int classes, int reduction) {
    __shared__ double room[32];
    double sums[2] = {};
    for (int i = threadIdx.x; i < rows; i += 1024) {
        sums[0] += (double)stats[rows + i];
        sums[1] += targets[i] >= 0 && targets[i] < classes ? 1.0 : 0.0;
        if (reduction == 0) out[i] = stats[rows + i];
    }
    team_sums<1024>(sums, room);
    if (threadIdx.x) return;
    stats[2ll * rows] = (A)sums[1];
    if (reduction) out[0] = (A)(reduction == 1 ? sums[0] / (sums[1] > 0 ? sums[1] : 1.0) : sums[0]);
}

template <typename A> __device__ __forceinline__ A vocab_factor(const A* stats, const A* upstream, const int* targets, int row, int rows, int classes, int reduction) {
    if (targets[row] < 0 || targets[row] >= classes) return (A)0;
    A f = upstream ? upstream[reduction == 0 ? row : 0] : (A)1;
    if (reduction == 1) f /= stats[2ll * rows];
    return f;
}
// z of a piece becomes d
template <typename A, int THREADS>
__global__ void __launch_bounds__(THREADS) vocab_d_kernel(A* z, const A* stats, const A* upstream, const int* targets, int rows, int width, int v0, int classes, int reduction) {
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const A f = vocab_factor(stats, upstream, targets, row, rows, classes, reduction), lse = stats[row];
        const bool held = targets[row] >= 0 && targets[row] < classes;
        const int t = held ? targets[row] - v0 : -1;
        A* zr = z + (long long)row * width;
        for (int c0 = threadIdx.x; c0 < width; c0 += THREADS * VOCAB_AT_ONCE) {
            A v[VOCAB_AT_ONCE];
#pragma unroll
            for (int u = 0; u < VOCAB_AT_ONCE; u++) v[u] = c0 + u * THREADS < width ? zr[c0 + u * THREADS] : (A)0;
#pragma unroll
            for (int u = 0; u < VOCAB_AT_ONCE; u++) {
                const int c = c0 + u * THREADS;
                if (c < width) zr[c] = held ? (natural_exp(v[u] - lse) - (c == t ? (A)1 : (A)0)) * f : (A)0;
            }
        }
    }
}

// ---- any strides, sizes and types ----

template <typename T> struct VocabAnyRoom {
    using A = typename traits<T>::acc;
    static constexpr bool WIDE = sizeof(T) != sizeof(A);          // operands that are widened first
    int piece;
    A *state, *z, *x, *w, *bias, *dx, *dw, *db, *parts;
    char* gemm;
    VocabAnyRoom(VocabRoom& room, int rows, int k, int classes, bool backward) {
        piece = vocab_piece(rows, rows <= VOCAB_FEW_ROWS && classes > VOCAB_FEW_PIECE ? VOCAB_FEW_PIECE : classes, sizeof(A), VOCAB_PIECE_BYTES);
        if (WIDE) piece = vocab_piece(k, piece, sizeof(A), VOCAB_WIDE_BYTES);      // (of few rows the widened W is by far the larger)
        state = room.take<A>(3ll * rows);
        z = room.take<A>((long long)rows * piece);
        gemm = room.take<char>(VOCAB_GEMM_BYTES);
        x = w = bias = dx = dw = db = parts = nullptr;
        if (backward) parts = room.take<A>((long long)VOCAB_GEMM_BYTES / sizeof(A));
        if (!WIDE) return;
        x = room.take<A>((long long)rows * k);
        w = room.take<A>((long long)k * piece);
        bias = room.take<A>(piece);
        if (!backward) return;
        dx = room.take<A>((long long)rows * k);
        dw = room.take<A>((long long)k * piece);
        db = room.take<A>(piece);
    }
};

struct VocabProduct {
    void* room;
    int dtype;
    int operator()(void* C, const void* A, const void* B, const void* bias, int m, int k, int n, long long a_rs, long long a_cs, long long b_rs, long long b_cs, long long c_rs, int accumulate) const {
        int rc;
        bool refused;
        {
            const GemmWorkspaceLoan loan(room, VOCAB_GEMM_BYTES);
            rc = rp_hip_gemm_strided_batched(C, A, B, bias, 1, m, k, n, 0, a_rs, a_cs, 0, b_rs, b_cs, 0, c_rs, 1, accumulate, dtype);
            refused = loan.refused;
        }
        // (few rows and more than 16384 of x's columns: as one group of all rows, whose k is not split)
        if (refused) rc = launch_grouped_rows(GroupedArgs{C, A, B, bias, nullptr, RowGroups{nullptr, nullptr, 1, m, 1}, k, n, a_rs, a_cs, 0, b_rs, b_cs, 0, c_rs, accumulate ? ACCUMULATE : 0}, dtype);
        return rc;
    }
};

// dx of float32 on few tiles: the classes of a piece in shares, as a batch of products that fills the CUs with tiles of 128, added up by a second launch (567 rows, 29440 classes, 1064 columns: 515 us in one
// product, 392 so.  Both passes: 567, 1064 -> 74105 3493 / 3130, 300, 1024 -> 32000 939 / 753, 1000, 512 -> 10000 420 / 413; fewer columns: 600, 256 -> 100000 1510 / 1626, 200, 256 -> 4000 53.5 / 58.9)
static int vocab_dx_shares(int rows, int k, int width, int elem) {
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const long long tiles = (long long)((rows + 127) / 128) * ((k + 127) / 128);
    if (elem != 4 || rows < 128 || k < 512 || 2 * tiles > cus || path_disabled("vocab_shares")) return 1;
    long long count = cus / tiles;
    if (count > width / 1024) count = width / 1024;
    const long long fits = (long long)(VOCAB_GEMM_BYTES / 4) / ((long long)rows * k);
    if (count > fits) count = fits;
    return count > 8 ? 8 : count < 1 ? 1 : (int)count;
}

// piece by piece: f(first class, classes, logits with unit column stride and rows as long as the piece)
template <typename T, typename F>
static int vocab_pieces(const VocabArgs& g, const VocabAnyRoom<T>& r, const VocabProduct& product, F f) {
    using A = typename traits<T>::acc;
    const void* x = g.x;
    long long x_rs = g.x_rs, x_cs = g.x_cs;
    if constexpr (VocabAnyRoom<T>::WIDE) {
        hipLaunchKernelGGL((vocab_widen_kernel<T>), dim3(flat_grid((long long)g.rows * g.k)), dim3(256), 0, current_stream(), r.x, (const T*)g.x, g.rows, g.k, g.x_rs, g.x_cs);
        if (!check_launch("vocab_widen_kernel")) return -1;
        x = r.x;
        x_rs = g.k;
        x_cs = 1;
    }
    for (int v0 = 0; v0 < g.classes; v0 += r.piece) {
        const int width = g.classes - v0 < r.piece ? g.classes - v0 : r.piece;
        const void *w = (const T*)g.w + v0 * g.w_cs, *bias = g.bias ? (const T*)g.bias + v0 : nullptr;
        long long w_rs = g.w_rs, w_cs = g.w_cs;
        if constexpr (VocabAnyRoom<T>::WIDE) {
            hipLaunchKernelGGL((vocab_widen_kernel<T>), dim3(flat_grid((long long)g.k * width)), dim3(256), 0, current_stream(), r.w, (const T*)w, g.k, width, g.w_rs, g.w_cs);
            if (!check_launch("vocab_widen_kernel")) return -1;
            w = r.w;
            w_rs = width;
            w_cs = 1;
            if (bias) {
                hipLaunchKernelGGL((vocab_widen_kernel<T>), dim3(flat_grid(width)), dim3(256), 0, current_stream(), r.bias, (const T*)bias, 1, width, 0ll, 1ll);
                if (!check_launch("vocab_widen_kernel")) return -1;
                bias = r.bias;
            }
        }
        if (product(r.z, x, w, bias, g.rows, g.k, width, x_rs, x_cs, w_rs, w_cs, width, 0) != 0) return -1;
        if (f(v0, width, (A*)r.z, (const A*)x, x_rs, x_cs, (const A*)w, w_rs, w_cs) != 0) return -1;
    }
    return 0;
}

template <typename A>
static int vocab_result(void* loss_out, void* stats, const VocabArgs& g) {
    hipLaunchKernelGGL((vocab_loss_kernel<A>), dim3(1), dim3(1024), 0, current_stream(), (A*)loss_out, (A*)stats, g.targets, g.rows, g.classes, g.reduction);
    return check_launch("vocab_loss_kernel") ? 0 : -1;
}

int vocab_result_f32(float* loss_out, float* stats, const VocabArgs& g) { return vocab_result<float>(loss_out, stats, g); }

template <typename T>
static int vocab_any_forward(void* stats, const VocabArgs& g, void* workspace) {
    using A = typename traits<T>::acc;
    VocabRoom room(workspace);
    const VocabAnyRoom<T> r(room, g.rows, g.k, g.classes, false);
    const int rc = vocab_pieces<T>(g, r, VocabProduct{r.gemm, traits<A>::code}, [&](int v0, int width, A* z, const A*, long long, long long, const A*, long long, long long) {
        const int blocks = g.rows < VOCAB_GRID ? g.rows : VOCAB_GRID;
        if (vocab_threads(g.rows) == 1024) hipLaunchKernelGGL((vocab_state_kernel<A, 1024>), dim3(blocks), dim3(1024), 0, current_stream(), r.state, (const A*)z, g.targets, g.rows, width, v0, v0 == 0);
        else hipLaunchKernelGGL((vocab_state_kernel<A, 256>), dim3(blocks), dim3(256), 0, current_stream(), r.state, (const A*)z, g.targets, g.rows, width, v0, v0 == 0);
        return check_launch("vocab_state_kernel") ? 0 : -1;
    });
    if (rc != 0) return -1;
    hipLaunchKernelGGL((vocab_rows_kernel<A>), dim3(flat_grid(g.rows)), dim3(256), 0, current_stream(), (A*)stats, (const A*)r.state, g.targets, g.rows, g.classes);
    return check_launch("vocab_rows_kernel") ? 0 : -1;
}

template <typename T>
static int vocab_any_backward(const VocabGrads& o, const VocabArgs& g, const void* stats, const void* upstream, void* workspace) {
    using A = typename traits<T>::acc;
    constexpr bool WIDE = VocabAnyRoom<T>::WIDE;
    VocabRoom room(workspace);
    const VocabAnyRoom<T> r(room, g.rows, g.k, g.classes, true);
    const VocabProduct product{r.gemm, traits<A>::code};
    auto rounded = [&](void* out, const A* in, int rows, int cols, long long rs, long long cs, int accumulate) {
        hipLaunchKernelGGL((vocab_round_kernel<T>), dim3(flat_grid((long long)rows * cols)), dim3(256), 0, current_stream(), (T*)out, in, rows, cols, rs, cs, accumulate);
        return check_launch("vocab_round_kernel") ? 0 : -1;
    };
    const int rc = vocab_pieces<T>(g, r, product, [&](int v0, int width, A* z, const A* x, long long x_rs, long long x_cs, const A* w, long long w_rs, long long w_cs) {
        const int blocks = g.rows < VOCAB_GRID ? g.rows : VOCAB_GRID;
        if (vocab_threads(g.rows) == 1024) hipLaunchKernelGGL((vocab_d_kernel<A, 1024>), dim3(blocks), dim3(1024), 0, current_stream(), z, (const A*)stats, (const A*)upstream, g.targets, g.rows, width, v0, g.classes, g.reduction);
        else hipLaunchKernelGGL((vocab_d_kernel<A, 256>), dim3(blocks), dim3(256), 0, current_stream(), z, (const A*)stats, (const A*)upstream, g.targets, g.rows, width, v0, g.classes, g.reduction);
        if (!check_launch("vocab_d_kernel")) return -1;
        if (o.dx) {
            void* dx = WIDE ? (void*)r.dx : o.dx;
            const long long dx_rs = WIDE ? g.k : o.dx_rs;
            const int accumulate = v0 ? 1 : WIDE ? 0 : o.accumulate_dx, shares = dx_rs == g.k ? vocab_dx_shares(g.rows, g.k, width, sizeof(A)) : 1, share = width / shares / 64 * 64, rest = width - shares * share;
            bool done = false;
            if (shares > 1) {
                const GemmWorkspaceLoan loan(r.gemm, VOCAB_GEMM_BYTES);
                const int rc = rp_hip_gemm_strided_batched(r.parts, z, w, nullptr, shares, g.rows, share, g.k, share, width, 1, share * w_cs, w_cs, w_rs, (long long)g.rows * g.k, g.k, 1, 0, traits<A>::code);
                if (rc != 0 && !loan.refused) return -1;
                done = rc == 0;
            }
            if (done && rest && product(r.parts, z + (long long)shares * share, w + shares * share * w_cs, nullptr, g.rows, rest, g.k, width, 1, w_cs, w_rs, g.k, 1) != 0) return -1;
            if (done ? rp_hip_reduce_rows(dx, r.parts, shares, g.rows * g.k, accumulate, traits<A>::code) != 0
                     : product(dx, z, w, nullptr, g.rows, width, g.k, width, 1, w_cs, w_rs, dx_rs, accumulate) != 0) return -1;
        }
        if (o.dw) {
            char* dw = (char*)o.dw + v0 * o.dw_cs * (long long)sizeof(T);
            if (WIDE) {
                if (product(r.dw, x, z, nullptr, g.k, g.rows, width, x_cs, x_rs, width, 1, width, 0) != 0 || rounded(dw, r.dw, g.k, width, o.dw_rs, o.dw_cs, o.accumulate_dw) != 0) return -1;
            } else if (o.dw_cs == 1) {
                if (product(dw, x, z, nullptr, g.k, g.rows, width, x_cs, x_rs, width, 1, o.dw_rs, o.accumulate_dw) != 0) return -1;
            } else if (product(dw, z, x, nullptr, width, g.rows, g.k, 1, width, x_rs, x_cs, o.dw_cs, o.accumulate_dw) != 0) return -1;      // the transposed product
        }
        if (o.db) {
            if (WIDE) return rp_hip_reduce_rows(r.db, z, g.rows, width, 0, traits<A>::code) != 0 ? -1 : rounded((T*)o.db + v0, r.db, 1, width, 0, 1, o.accumulate_db);
            return rp_hip_reduce_rows((T*)o.db + v0, z, g.rows, width, o.accumulate_db, traits<A>::code);
        }
        return 0;
    });
    if (rc != 0) return -1;
    return WIDE && o.dx ? rounded(o.dx, r.dx, g.rows, g.k, o.dx_rs, 1, o.accumulate_dx) : 0;
}

static long long vocab_any_room(int rows, int k, int classes, bool backward, int dtype) {
    VocabRoom room(nullptr);
    RP_DISPATCH_DTYPE(dtype, const VocabAnyRoom<T> r(room, rows, k, classes, backward); (void)r);
    return room.used();
}

static bool vocab_args_ok(const char* who, bool pointers, int rows, int k, int classes, int reduction, std::initializer_list<long long> strides, int dtype) {
    if (!pointers || rows <= 0 || k <= 0 || classes <= 0 || rows > (1 << 29) || classes > (1 << 29)) {
        set_error("%s: null operand, non-positive extent, more than 2^29 rows or classes (rows=%d k=%d classes=%d)", who, rows, k, classes);
        return false;
    }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    if (reduction < 0 || reduction > 2) { set_error("%s: reduction must be none (0), mean (1) or sum (2)", who); return false; }
    for (long long s : strides)
        if (s < 0) { set_error("%s: negative stride", who); return false; }
    return true;
}

}  // namespace rp

using namespace rp;

extern "C" {

long long rp_hip_linear_cross_entropy_workspace(int rows, int k, int classes, int backward, int dtype) {
    if (!vocab_args_ok("rp_hip_linear_cross_entropy_workspace", true, rows, k, classes, 0, {}, dtype)) return -1;
    const long long tiles = dtype_size(dtype) == 2 ? vocab16_room(rows, k, classes, backward != 0) : 0, any = vocab_any_room(rows, k, classes, backward != 0, dtype);
    return tiles > any ? tiles : any;                         // (how the operands lie is not known here: room for either way)
}

long long rp_hip_linear_cross_entropy_workspace_strided(int rows, int k, int classes, int backward, long long x_rs, long long x_cs, long long w_rs, long long w_cs, int dtype) {
    if (!vocab_args_ok("rp_hip_linear_cross_entropy_workspace_strided", true, rows, k, classes, 0, {x_rs, x_cs, w_rs, w_cs}, dtype)) return -1;
    // (where they start decides nothing but the tiles' kind)
    const bool tiles = vocab16_takes(VocabArgs{nullptr, nullptr, nullptr, nullptr, rows, k, classes, 0, x_rs, x_cs, w_rs, w_cs}, dtype);
    return tiles ? vocab16_room(rows, k, classes, backward != 0) : vocab_any_room(rows, k, classes, backward != 0, dtype);
}

int rp_hip_linear_cross_entropy_forward(void* loss_out, void* stats, const void* x, const void* w, const void* bias, const int* targets, void* workspace, int rows, int k, int classes, int reduction,
                                        long long x_rs, long long x_cs, long long w_rs, long long w_cs, int dtype) {
    if (!vocab_args_ok("rp_hip_linear_cross_entropy_forward", loss_out && stats && x && w && targets && workspace, rows, k, classes, reduction, {x_rs, x_cs, w_rs, w_cs}, dtype)) return -1;
    const VocabArgs g{x, w, bias, targets, rows, k, classes, reduction, x_rs, x_cs, w_rs, w_cs};
    if (vocab16_takes(g, dtype)) return vocab16_forward((float*)loss_out, (float*)stats, g, workspace, dtype);
    RP_DISPATCH_DTYPE(dtype, if (vocab_any_forward<T>(stats, g, workspace) != 0) return -1);
    return dtype == RP_DTYPE_FLOAT64 ? vocab_result<double>(loss_out, stats, g) : vocab_result<float>(loss_out, stats, g);
}

int rp_hip_linear_cross_entropy_backward(void* dx, void* dw, void* db, const void* x, const void* w, const void* bias, const int* targets, const void* stats, const void* upstream_dev, void* workspace,
                                         int rows, int k, int classes, int reduction, long long x_rs, long long x_cs, long long w_rs, long long w_cs,
                                         long long dx_rs, long long dw_rs, long long dw_cs, int accumulate_dx, int accumulate_dw, int accumulate_db, int dtype) {
    const char* who = "rp_hip_linear_cross_entropy_backward";
    if (!vocab_args_ok(who, x && w && targets && stats && workspace, rows, k, classes, reduction, {x_rs, x_cs, w_rs, w_cs, dx_rs, dw_rs, dw_cs}, dtype)) return -1;
    if (dx && rows > 1 && dx_rs < k) { set_error("%s: rows of dx are %lld elements apart and hold %d", who, dx_rs, k); return -1; }
    if (dw && !(dw_cs == 1 && (k == 1 || dw_rs >= classes)) && !(dw_rs == 1 && (classes == 1 || dw_cs >= k))) {
        set_error("%s: dw has unit stride along one axis and rows that do not overlap along the other", who);
        return -1;
    }
    if (!dx && !dw && !db) return 0;
    const VocabArgs g{x, w, bias, targets, rows, k, classes, reduction, x_rs, x_cs, w_rs, w_cs};
    const VocabGrads o{dx, dw, db, dx_rs, dw_rs, dw_cs, accumulate_dx, accumulate_dw, accumulate_db};
    if (vocab16_takes(g, dtype)) return vocab16_backward(o, g, (const float*)stats, (const float*)upstream_dev, workspace, dtype);
    RP_DISPATCH_DTYPE(dtype, return vocab_any_backward<T>(o, g, stats, upstream_dev, workspace));
    return -1;
}

}  // extern "C"
