// bf16 / fp16 cross entropy of a large vocabulary on MFMA tiles: which tiles, in which pieces, and the small launches between the products.
#include "rp_vocab16.h"

namespace rp {

// A piece's d (2 bytes an element) is written once and read by two products.  The wider the pieces the fewer times dx's sums, 4 bytes an element, are read and written between them, and the
// fewer the products' last rounds of tiles that leave CUs idle.
constexpr long long VOCAB16_PIECE_BYTES = 256ll << 20;

// ---- which tiles ----

// How an operand lies: rows of whole 16-byte vectors that start on them, rows of at least a vector that do not overlap, or neither
enum { LIES_WHOLE, LIES_RAGGED, LIES_NEITHER };
static int lies16(const void* p, long long row_stride, long long length) {
    if (length < 8 || row_stride < length || row_stride >= (1ll << 22)) return LIES_NEITHER;
    return ((uintptr_t)p & 15) || row_stride % 8 || length % 8 ? LIES_RAGGED : LIES_WHOLE;
}
static int worse16(int a, int b) { return a > b ? a : b; }

// edge 256, 128 or 64 and what of it may hang over
struct VocabTile { int edge, over; };
static VocabTile vocab_tile(int m, int n, int k, bool gradient, bool a_mc, bool b_mc, int lie) {
    Plan p{FAM_MFMA16, 64, 64, a_mc, b_mc, true, ""};
    p.ragged = lie == LIES_RAGGED;
    choose_tile16(p, 1, m, k, n);
    // (a gradient's few tiles of 128 share k among workgroups, below; fp16, both passes, us with dx on 64 and 128: 1000 rows, 520 -> 10007 155 / 149, 512, 2048 -> 32000 361 / 335, 2000, 256 -> 50000 572 / 534)
    if (gradient && p.bm != 256 && m > 64 && n > 64 && k >= 16 * M16_BK) p.bm = p.bn = 128;
    // (logits of four slabs: the epilogue is most of the work, and tiles of 128 have two workgroups a CU for it; 2000 rows, 256 -> 50000, forward 176 / 167)
    if (!gradient && p.bm == 256 && k <= 4 * M16_BK) p.bm = p.bn = 128;
    if (p.ragged) return {p.bm >= 128 && p.bn >= 128 ? 128 : 64, M16_RAGGED};
    if (p.bm == 256 && p.bn == 256) return {256, m % 256 || n % 256 || k % M16_BK ? M16_EDGE : M16_WHOLE};
    return {p.bm >= 128 && p.bn >= 128 ? 128 : 64, M16_EDGE};
}

static int launch_logits(const VocabTileArgs& a, VocabStep step, bool b_mc, int lie, int dtype) {
    const VocabTile t = vocab_tile(a.g.m, a.g.n, a.g.k, false, false, b_mc, lie);
    if (t.edge == 256) return dtype == RP_DTYPE_BFLOAT16 ? launch_vocab16_logits_256_bf16(a, step, b_mc, t.over) : launch_vocab16_logits_256_f16(a, step, b_mc, t.over);
    return t.edge == 128 ? launch_vocab16_logits_128(a, step, b_mc, t.over, dtype) : launch_vocab16_logits_64x128(a, step, b_mc, t.over, dtype);
}
static int launch_grads(const VocabTileArgs& a, VocabStep step, bool b_mc, const VocabTile& t, int dtype) {
    if (t.edge == 256) return dtype == RP_DTYPE_BFLOAT16 ? launch_vocab16_grads_256_bf16(a, step, b_mc, t.over) : launch_vocab16_grads_256_f16(a, step, b_mc, t.over);
    return t.edge == 128 ? launch_vocab16_grads_128(a, step, b_mc, t.over, dtype) : launch_vocab16_grads_64(a, step, b_mc, t.over, dtype);
}
// Columns of a wave's patch of logits (what a part of a row's sum comes from) and its rows (of a column's), by the tile's edge in rows; the smallest tile has 64 rows and 128 columns
static int patch_columns(int edge) { return edge == 256 ? 128 : 64; }
static int patch_rows(int edge) { return edge / 2; }

// (d has as many columns as W, and is an operand of unaligned tiles too: fewer classes than a vector go the other way however W lies)
static int logits_lie(const VocabArgs& g) {
    if (g.classes < 8) return LIES_NEITHER;
    return worse16(lies16(g.x, g.x_rs, g.k), g.w_cs == 1 ? lies16(g.w, g.w_rs, g.classes) : lies16(g.w, g.w_cs, g.k));
}
bool vocab16_takes(const VocabArgs& g, int dtype) {
    if ((dtype != RP_DTYPE_BFLOAT16 && dtype != RP_DTYPE_FLOAT16) || g.x_cs != 1 || (g.w_cs != 1 && g.w_rs != 1) || path_disabled("mfma")) return false;
    // (the forward pass is one launch, of fewer than 2^32 threads; on 64 x 128 tiles from 2^37 logits on it would not be)
    return logits_lie(g) != LIES_NEITHER && (long long)((g.rows + 63) / 64) * ((g.classes + 127) / 128) < (1 << 24) - 64;
}

// Few tiles and a long k: k goes in shares of at least eight slabs to workgroups of their own, three a CU, or one where tiles of 128 keep seven eighths of the CUs busy so.  (fp16, 1000 rows, 520 -> 10007:
// dx on 40 tiles of 128 walks 157 slabs, 72 us; in six shares 29 and 5 for the launch that joins them.  Both passes, us with three a CU and one: 1000, 520 -> 10007 147 / 141, 512, 1024 -> 32000 231 / 217,
// 1024, 768 -> 50000 589 / 584; on tiles of 64: 16, 4096 -> 32000 247 / 268)
constexpr long long VOCAB16_SHARE_BYTES = 32ll << 20;      // of the shares' sums
struct Shares { int count, k; long long stride; };
static Shares vocab_shares(int m, int n, int k, const VocabTile& t) {
    const Shares one{1, k, 0};
    if (t.edge == 256 || path_disabled("vocab_shares")) return one;
    const long long tiles = (long long)((m + t.edge - 1) / t.edge) * ((n + t.edge - 1) / t.edge), area = tiles * t.edge * t.edge;
    const int cus = device_cu_count() > 0 ? device_cu_count() : 256, slabs = (k + M16_BK - 1) / M16_BK;
    long long count = cus / tiles;
    if (t.edge == 64 || 8 * count * tiles < 7ll * cus) count = 3ll * cus / tiles;
    if (count > slabs / 8) count = slabs / 8;
    if (count > 16) count = 16;
    if (count > VOCAB16_SHARE_BYTES / (area * 4)) count = VOCAB16_SHARE_BYTES / (area * 4);
    if (count < 2) return one;
    const int per = (int)((slabs + count - 1) / count);
    return {(slabs + per - 1) / per, per * M16_BK, area};
}
// Bytes that the sums of an output of m x n may take: the shares' where there are any, whichever tiles are taken
static long long share_bytes(long long m, long long n) {
    const long long area = (m + 127) / 128 * 128 * ((n + 127) / 128 * 128) * 4;
    return area * 16 < VOCAB16_SHARE_BYTES ? area * 16 : VOCAB16_SHARE_BYTES;
}

// ---- small launches ----

// A row's log sum and loss from its groups' parts, ROWS rows to a workgroup: 16, four lanes of every wave to a row, so that 64 groups are read at a time in whole cache lines; or 64 where there are no
// more, whose workgroup leaves the result too
// What a sum of exp(z - top) is multiplied by to be one of exp(z - base): of the difference, so that a part whose largest is the base stays as it is (exp_less rounds base log2 e, 4e-5 of a sum at 1000, at every join)
__device__ __forceinline__ float rebased(float top, float base) { return __builtin_amdgcn_exp2f((top - base) * LOG2_E); }
__device__ __forceinline__ VocabPart joined_parts(const VocabPart& p, const VocabPart& q) {
    const float top = fmaxf(p.top, q.top), base = top == -INFINITY ? 0.f : top;
    return VocabPart{top, p.sum * rebased(p.top, base) + q.sum * rebased(q.top, base)};
}
template <int ROWS>
__global__ void __launch_bounds__(1024) vocab16_rows_kernel(float* stats, const VocabPart* parts, const float* hits, const int* targets, int rows, int classes, int groups, float* out, int reduction) {
    constexpr int SLICES = 1024 / ROWS, BATCH = 8;
    __shared__ VocabPart room[16][ROWS];
    const int r = threadIdx.x % ROWS, slice = threadIdx.x / ROWS, wave = threadIdx.x / 64;
    for (int row0 = blockIdx.x * ROWS; row0 < rows; row0 += gridDim.x * ROWS) {
        const int row = row0 + r;
        VocabPart own{-INFINITY, 0.f};
        if (row < rows)
            for (int i0 = slice; i0 < groups; i0 += SLICES * BATCH) {
                VocabPart p[BATCH];
#pragma unroll
                for (int e = 0; e < BATCH; e++) p[e] = i0 + SLICES * e < groups ? parts[(long long)(i0 + SLICES * e) * rows + row] : VocabPart{-INFINITY, 0.f};
                float most = own.top;
#pragma unroll
                for (int e = 0; e < BATCH; e++) most = fmaxf(most, p[e].top);
                const float base = most == -INFINITY ? 0.f : most;
                own.sum *= rebased(own.top, base);
#pragma unroll
                for (int e = 0; e < BATCH; e++) own.sum += p[e].sum * rebased(p[e].top, base);
                own.top = most;
            }
#pragma unroll
        for (int d = ROWS; d < 64; d *= 2) own = joined_parts(own, VocabPart{__shfl_xor(own.top, d), __shfl_xor(own.sum, d)});
        __syncthreads();
        if ((threadIdx.x & 63) < ROWS) room[wave][r] = own;
        __syncthreads();
        if (threadIdx.x >= ROWS) continue;
        const bool there = row < rows;
        float top = room[0][r].top, sum = 0.f;
#pragma unroll
        for (int w = 1; w < 16; w++) top = fmaxf(top, room[w][r].top);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < 16; w++) sum += room[w][r].sum * rebased(room[w][r].top, base);
        const float lse = base + logf(sum);
        const bool held = there && targets[row] >= 0 && targets[row] < classes;
        const float loss = held ? lse - hits[row] : 0.f;
        if (there) {
            stats[row] = lse;
            stats[rows + row] = loss;
        }
        if constexpr (ROWS == 64) {
            if (reduction == 0 && there) out[row] = loss;
            const double total = wave_sum((double)loss), count = wave_sum(held ? 1.0 : 0.0);
            if (r == 0) {
                stats[2ll * rows] = (float)count;
                if (reduction) out[0] = (float)(reduction == 1 ? total / (count > 0 ? count : 1.0) : total);
            }
        }
    }
}

// Rows with an upstream gradient of their own: f of each over the largest of them, times 2^most, and what takes that back: one workgroup
__global__ void __launch_bounds__(1024) vocab16_factors_kernel(float* f, float* scale, const float* upstream, const int* targets, int rows, int classes, int most) {
    __shared__ float room[16];
    float top = 0.f;
    for (int i = threadIdx.x; i < rows; i += 1024) {
        float v = 0.f;
        if (targets[i] >= 0 && targets[i] < classes) v = upstream ? upstream[i] : 1.f;
        f[i] = v;
        top = fmaxf(top, __builtin_isfinite(v) ? fabsf(v) : 0.f);
    }
    top = team_max<1024>(top, room);
    if (!(top > 0.f)) top = 1.f;
    const float up = ldexpf(1.f, most);
    for (int i = threadIdx.x; i < rows; i += 1024) f[i] = f[i] / top * up;      // (each thread its own)
    if (threadIdx.x == 0) *scale = top / up;
}

// db of a piece from its groups' sums
template <typename T>
__global__ void __launch_bounds__(1024) vocab16_db_kernel(VocabTileArgs a, T* db, const float* parts, int groups, long long pitch, int width, int accumulate) {
    __shared__ float room[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, c = blockIdx.x * 64 + lane;
    float sum = 0.f;
    if (c < width)
#pragma unroll 8
        for (int i = wave; i < groups; i += 16) sum += parts[i * pitch + c];
    room[wave][lane] = sum;
    __syncthreads();
    if (wave || c >= width) return;
#pragma unroll
    for (int w = 1; w < 16; w++) sum += room[w][lane];
    sum *= scale_back(a);
    db[c] = round_to<T>(accumulate ? widen(db[c]) + sum : sum);
}

// ---- the workspace ----

struct Vocab16Room {
    VocabPart* parts;
    float *hits, *f, *scale, *db_parts, *sums, *dw_sums;
    uint16_t* d;
    int piece, pitch;
    Vocab16Room(VocabRoom& room, int rows, int k, int classes, bool backward) {
        // pieces of whole tiles; a last one of a few classes takes some of those before it (no operand is shorter than a vector)
        const long long fits = VOCAB16_PIECE_BYTES / (2ll * rows) / 256 * 256, all = (classes + 255ll) / 256 * 256;
        const long long reach = 1 << 21;                      // (the tiles' 32-bit offsets)
        piece = pitch = (int)(fits < 256 ? 256 : fits < all ? (fits < reach ? fits : reach) : all < reach ? all : reach);
        if (!backward) {
            hits = room.take<float>(rows);
            parts = room.take<VocabPart>((long long)rows * ((classes + 255ll) / 256 * 4));      // (a wave's patch has 64 columns or more)
            return;
        }
        f = room.take<float>(rows);
        scale = room.take<float>(1);
        d = room.take<uint16_t>((long long)rows * pitch);
        db_parts = room.take<float>(((long long)rows + 255) / 256 * 8 * pitch);
        const long long between = classes > piece ? (rows + 255ll) / 256 * 256 * ((k + 255ll) / 256 * 256) : 0, shares = share_bytes(rows, k) / 4;
        sums = room.take<float>(between > shares ? between : shares);
        dw_sums = room.take<float>(share_bytes(k, classes < piece ? classes : piece) / 4);
        hits = nullptr;
        parts = nullptr;
    }
    int width(int v0, int classes) const {
        const int left = classes - v0;
        return left <= piece ? left : left < piece + 64 ? piece - 128 : piece;
    }
};

long long vocab16_room(int rows, int k, int classes, bool backward) {
    VocabRoom forward(nullptr), both(nullptr);
    const Vocab16Room f(forward, rows, k, classes, false), b(both, rows, k, classes, true);
    (void)f;
    (void)b;
    return backward && both.used() > forward.used() ? both.used() : forward.used();      // (one workspace does for both passes)
}

// ---- the passes ----

int vocab16_forward(float* loss_out, float* stats, const VocabArgs& g, void* workspace, int dtype) {
    VocabRoom room(workspace);
    const Vocab16Room r(room, g.rows, g.k, g.classes, false);
    const bool b_mc = g.w_cs == 1;
    const int lie = logits_lie(g);
    VocabTileArgs a{};
    a.shares = 1;
    a.g = GemmArgs{nullptr, g.x, g.w, g.bias, 1, g.rows, g.k, g.classes, 0, g.x_rs, 1, 0, g.w_rs, g.w_cs};
    a.targets = g.targets;
    a.classes = g.classes;
    a.parts = r.parts;
    a.hits = r.hits;
    if (launch_logits(a, VOCAB_FORWARD, b_mc, lie, dtype) != 0) return -1;
    const int edge = vocab_tile(g.rows, g.classes, g.k, false, false, b_mc, lie).edge, bn = edge == 256 ? 256 : 128, groups = (g.classes + bn - 1) / bn * (bn / patch_columns(edge));
    if (g.rows <= 64) {
        hipLaunchKernelGGL((vocab16_rows_kernel<64>), dim3(1), dim3(1024), 0, current_stream(), stats, r.parts, r.hits, g.targets, g.rows, g.classes, groups, loss_out, g.reduction);
        return check_launch("vocab16_rows_kernel") ? 0 : -1;
    }
    const int blocks = (g.rows + 15) / 16;
    hipLaunchKernelGGL((vocab16_rows_kernel<16>), dim3(blocks < (1 << 20) ? blocks : 1 << 20), dim3(1024), 0, current_stream(), stats, r.parts, r.hits, g.targets, g.rows, g.classes, groups, loss_out, g.reduction);
    return check_launch("vocab16_rows_kernel") ? vocab_result_f32(loss_out, stats, g) : -1;
}

int vocab16_backward(const VocabGrads& o, const VocabArgs& g, const float* stats, const float* upstream, void* workspace, int dtype) {
    VocabRoom room(workspace);
    const Vocab16Room r(room, g.rows, g.k, g.classes, true);
    const bool tied = g.w_cs != 1;                            // W is the transpose of [classes, k] rows
    const int lie = logits_lie(g);
    // dx on the same tiles for every piece (their sums lie by tile); all but the last piece are whole slabs
    const int longest = g.classes < r.piece ? g.classes : r.piece;
    VocabTile dx_tile = vocab_tile(g.rows, g.k, longest, true, false, tied, worse16(lie, g.classes % 8 ? LIES_RAGGED : LIES_WHOLE));
    if (dx_tile.over == M16_WHOLE && g.classes % M16_BK) dx_tile.over = M16_EDGE;
    const Shares dx_shares = g.classes > r.piece ? Shares{1, 0, 0} : vocab_shares(g.rows, g.k, longest, dx_tile);
    // one f for all rows, or one for each
    const bool same = g.reduction != 0;
    const int most = dtype == RP_DTYPE_FLOAT16 ? 14 : 0;
    if (!same) {
        hipLaunchKernelGGL(vocab16_factors_kernel, dim3(1), dim3(1024), 0, current_stream(), r.f, r.scale, upstream, g.targets, g.rows, g.classes, most);
        if (!check_launch("vocab16_factors_kernel")) return -1;
    }
    auto weighted = [&](VocabTileArgs& a) {
        a.f = same ? nullptr : r.f;
        a.scale = same ? nullptr : r.scale;
        a.upstream = upstream;
        a.count = g.reduction == 1 ? stats + 2ll * g.rows : nullptr;
        a.most = most;
    };
    for (int v0 = 0, width; v0 < g.classes; v0 += width) {
        width = r.width(v0, g.classes);
        const char *w = (const char*)g.w + 2 * v0 * g.w_cs, *bias = g.bias ? (const char*)g.bias + 2ll * v0 : nullptr;
        VocabTileArgs a{};
        a.shares = 1;
        a.g = GemmArgs{nullptr, g.x, w, bias, 1, g.rows, g.k, width, 0, g.x_rs, 1, 0, g.w_rs, g.w_cs};
        a.targets = g.targets;
        a.v0 = v0;
        a.classes = g.classes;
        a.d = r.d;
        a.pitch = r.pitch;
        a.lse = stats;
        weighted(a);
        const int piece_lie = worse16(lie, g.w_cs == 1 && width % 8 ? LIES_RAGGED : LIES_WHOLE);
        const int patch = patch_rows(vocab_tile(g.rows, width, g.k, false, false, !tied, piece_lie).edge), groups = (g.rows + patch - 1) / patch;
        if (o.db && groups == 1) {
            a.db = (char*)o.db + 2ll * v0;
            a.accumulate_db = o.accumulate_db;
        } else if (o.db) a.db_parts = r.db_parts;
        if (launch_logits(a, VOCAB_GRADIENT, !tied, piece_lie, dtype) != 0) return -1;
        if (a.db_parts) {
            RP_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((vocab16_db_kernel<T>), dim3((width + 63) / 64), dim3(1024), 0, current_stream(), a, (T*)o.db + v0, r.db_parts, groups, (long long)r.pitch, width, o.accumulate_db));
            if (!check_launch("vocab16_db_kernel")) return -1;
        }
        VocabTileArgs p{};
        weighted(p);
        if (o.dx) {
            p.g = GemmArgs{o.dx, r.d, w, nullptr, 1, g.rows, width, g.k, 0, r.pitch, 1, 0, g.w_cs, g.w_rs, 0, o.dx_rs, 1, o.accumulate_dx};
            p.sums = r.sums;
            p.first = v0 == 0;
            p.last = v0 + width == g.classes;
            p.shares = dx_shares.count;
            p.k_share = dx_shares.k;
            p.share_stride = dx_shares.stride;
            if (launch_grads(p, VOCAB_DX, tied, dx_tile, dtype) != 0) return -1;
        }
        if (o.dw) {
            char* dw = (char*)o.dw + 2 * v0 * o.dw_cs;
            // x^T . d, or where dW lies as the transpose d^T . x
            p.g = o.dw_cs == 1 ? GemmArgs{dw, g.x, r.d, nullptr, 1, g.k, g.rows, width, 0, 1, g.x_rs, 0, r.pitch, 1, 0, o.dw_rs, 1, o.accumulate_dw}
                               : GemmArgs{dw, r.d, g.x, nullptr, 1, width, g.rows, g.k, 0, 1, r.pitch, 0, g.x_rs, 1, 0, o.dw_cs, 1, o.accumulate_dw};
            const VocabTile t = vocab_tile(p.g.m, p.g.n, p.g.k, true, true, true, worse16(lies16(g.x, g.x_rs, g.k), width % 8 ? LIES_RAGGED : LIES_WHOLE));
            const Shares shares = vocab_shares(p.g.m, p.g.n, p.g.k, t);
            p.sums = r.dw_sums;
            p.first = p.last = 1;
            p.shares = shares.count;
            p.k_share = shares.k;
            p.share_stride = shares.stride;
            if (launch_grads(p, VOCAB_DW, true, t, dtype) != 0) return -1;
        }
    }
    return 0;
}

}  // namespace rp
