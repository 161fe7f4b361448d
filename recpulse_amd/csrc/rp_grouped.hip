// Entry points and dispatch of the grouped products (experts) and of the adapters beside a shared projection.
//
// Experts: y[i] = x[i] . W_g + b_g for the rows i of group g;  dx[i] = dy[i] . W_g^T,  dW_g = sum x[i]^T dy[i],  db_g = sum dy[i].
// Adapters, a the adapter of row i's segment:  h[i] = s_a x[i] . A_a,  y[i] = x[i] . W + b + h[i] . B_a;
//   u[i] = s_a dy[i] . B_a^T,  dx[i] = dy[i] . W^T + u[i] . A_a^T,  dA_a = sum x[i]^T u[i],  dB_a = sum h[i]^T dy[i].
// h and u are in the accumulate type (float32, float64 for float64): they are sums that are multiplied on.
#include "rp_grouped_sums.h"

namespace rp {

static bool is16(int dtype) { return dtype == RP_DTYPE_BFLOAT16 || dtype == RP_DTYPE_FLOAT16; }
static int cus() {
    const int n = device_cu_count() / 8 * 8;
    return n >= 8 ? n : 256;
}

// How an operand of the tiled kernels lies: rows of whole 16-byte vectors that start on them, rows of at least a vector that do not overlap, or neither.
enum Lie { LIE_WHOLE, LIE_RAGGED, LIE_NEITHER };
static Lie lies(const void* p, long long row_stride, long long weight_stride, int length, int elem) {
    const int vec = 16 / elem;
    if (length < vec || row_stride < length || row_stride >= (1ll << 22)) return LIE_NEITHER;
    return ((uintptr_t)p & 15) || row_stride % vec || weight_stride % vec || length % vec ? LIE_RAGGED : LIE_WHOLE;
}
static Lie worse(Lie a, Lie b) { return a > b ? a : b; }

// 256 x 256 tiles go in whole rounds of the CUs, each of k / 1024 * 23.3 us + 10; tiles of 128, two to a CU at a time, in any number, 0.043 us each at k = 1024.  fp16,
// us on 256 and 128: 1024 -> 4096 in 8 groups, 3000 rows (1 round) 38 / 43, 4096 rows (2) 67 / 55, 8192 (3) 102 / 95, 16384 (5) 171 / 189; 4096 -> 4096, 4096 rows (2) 209 / 203.
static bool prefers256(long long tiles256, long long tiles128, long long k) {
    const long long rounds = (tiles256 + cus() - 1) / cus();
    return rounds * cus() * 4 * (k + 440) * 100 < tiles128 * (k + 60) * 187;
}

// Tiles of the 16-bit products: their edge, 0 for none, and how the operands lie.  How many row tiles there are is known on the device only: each group is taken to end inside a tile.
struct Tile16 { int edge; bool ragged; };

static Tile16 rows_tile16(const GroupedArgs& g, int dtype) {
    if (!is16(dtype) || g.a_cs != 1 || (g.b_cs != 1 && g.b_rs != 1) || g.gr.groups > ROW_TILES_GROUPS || path_disabled("mfma")) return {0, false};
    const bool b_mc = g.b_cs == 1;
    const Lie lie = worse(lies(g.A, g.a_rs, 0, g.k, 2), b_mc ? lies(g.B, g.b_rs, g.b_ws, g.n, 2) : lies(g.B, g.b_cs, g.b_ws, g.k, 2));
    if (lie == LIE_NEITHER) return {0, false};
    const int mean = g.gr.rows / g.gr.groups;
    auto tiles = [&](int edge) { return ((long long)(g.gr.rows + edge - 1) / edge + g.gr.groups / 2) * ((g.n + edge - 1) / edge); };
    if (lie == LIE_WHOLE && mean >= 256 && g.n >= 256 && g.k >= 256 && prefers256(tiles(256), tiles(128), g.k)) return {256, false};
    // 128 x 128 tiles from a round of the CUs on (bf16, 519 -> 1031, us on 64 and 128: 1999 rows of 6 groups, 171 tiles, 14.5 / 15.2; 4096 of 8, 324 tiles, 23.1 / 19.7)
    return {mean >= 96 && g.n > 64 && tiles(128) >= cus() ? 128 : 64, lie == LIE_RAGGED};
}

static Tile16 weights_tile16(const GroupedArgs& g, int dtype) {
    if (!is16(dtype) || g.a_cs != 1 || g.b_cs != 1 || path_disabled("mfma")) return {0, false};
    const Lie lie = worse(lies(g.A, g.a_rs, 0, g.k, 2), lies(g.B, g.b_rs, 0, g.n, 2));
    if (lie == LIE_NEITHER) return {0, false};
    auto tiles = [&](int edge) { return (long long)((g.k + edge - 1) / edge) * ((g.n + edge - 1) / edge) * g.gr.weights; };
    if (lie == LIE_WHOLE && g.k >= 256 && g.n >= 256 && prefers256(tiles(256), tiles(128), g.gr.rows / g.gr.groups)) return {256, false};
    return {g.k > 64 && g.n > 64 && tiles(128) >= cus() / 2 ? 128 : 64, lie == LIE_RAGGED};
}

static int grouped_rows(const GroupedArgs& g, int dtype) {
    if (is16(dtype) && grouped_stream16_takes(g)) return launch_grouped_stream16(g, dtype);
    const Tile16 t = rows_tile16(g, dtype);
    if (t.edge == 256) return dtype == RP_DTYPE_BFLOAT16 ? launch_grouped_rows16_256_bf16(g) : launch_grouped_rows16_256_f16(g);
    if (t.edge) return t.edge == 128 ? launch_grouped_rows16_128(g, t.ragged, dtype) : launch_grouped_rows16_64(g, t.ragged, dtype);
    if (!is16(dtype) && grouped_rows_wavek_takes(g, dtype)) return launch_grouped_rows_wavek(g, dtype);
    return launch_grouped_rows_generic(g, false, dtype);
}

static int grouped_weights(const GroupedArgs& g, int dtype) {
    const Tile16 t = weights_tile16(g, dtype);
    if (t.edge == 256) return dtype == RP_DTYPE_BFLOAT16 ? launch_grouped_weights16_256_bf16(g) : launch_grouped_weights16_256_f16(g);
    if (t.edge) return t.edge == 128 ? launch_grouped_weights16_128(g, t.ragged, dtype) : launch_grouped_weights16_64(g, t.ragged, dtype);
    return launch_grouped_weights_generic(g, dtype);
}

// The gradients of one layer in one launch unless 256 x 256 tiles, whose workgroups stay on their CU, take one of them.  bf16, us, in launches of their own and in
// one: 1999 rows of 6 groups, 519 -> 1031, 41 / 23; 4096 of 8 56 / 32; 8192 of 8, 1031 -> 2047, 187 / 150.  One tile edge for both, 128 from a round of the CUs on
// (64 and 128: 3000 rows of 4 groups, 700 -> 1031, 360 tiles of 128, 32 / 25; 1999 of 6, 350 tiles, 23 / 23), unless the weights' tiles alone leave CUs idle:
// each adds up a whole group's rows (14949 rows of 3 groups, 504 -> 427, 48 tiles of 128, 92 / 77).
static bool backward_together(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums, int dtype, int* result) {
    if (!x.C && !w.C) return false;
    if (!is16(dtype)) {
        const bool takes = grouped_backward_wavek_takes(x, w, dtype);
        if (takes) *result = launch_grouped_backward_wavek(x, w, sums, dtype);
        return takes;
    }
    if (!x.C + !w.C + !sums.out > 1 || (x.C && (grouped_stream16_takes(x) || x.b_rs != 1)) || path_disabled("grouped_backward")) return false;
    const Tile16 tx = x.C ? rows_tile16(x, dtype) : Tile16{64, false}, tw = w.C ? weights_tile16(w, dtype) : Tile16{64, false};
    if (!tx.edge || !tw.edge || tx.edge == 256 || tw.edge == 256) return false;
    const long long most = max_row_tiles(x.gr.rows, x.gr.groups, 64) * ((x.n + 63) / 64) + ((long long)((w.k + 63) / 64) * ((w.n + 63) / 64) + 8) * w.gr.weights + sum_blocks(sums);
    if (most > GROUPED_BACKWARD16_MOST) return false;
    const bool ragged = tx.ragged || tw.ragged;
    const long long tiles128 = (x.C ? (long long)((x.gr.rows + 127) / 128) * ((x.n + 127) / 128) : 0) + (w.C ? (long long)((w.k + 127) / 128) * ((w.n + 127) / 128) * w.gr.weights : 0);
    const int x_tile = tiles128 >= cus() ? 128 : 64, w_tile = tw.edge < x_tile ? tw.edge : x_tile;
    *result = dtype == RP_DTYPE_BFLOAT16 ? launch_grouped_backward16_bf16(x, x_tile, w, w_tile, sums, ragged) : launch_grouped_backward16_f16(x, x_tile, w, w_tile, sums, ragged);
    return true;
}

// An adapter's narrow product (C is h or u) and the gradients of its factors
static int narrow_rows(const GroupedArgs& g, int dtype) { return is16(dtype) && adapter_shrink16_takes(g) ? launch_adapter_shrink16(g, dtype) : launch_narrow_rows(g, dtype); }
// Each gradient goes by its own operands, so that its bits do not depend on whether the other is asked for: those on MFMAs, the others with a null C in their place
struct Grads16 { GroupedArgs da, db; };
static Grads16 grads16_of(GroupedArgs da, GroupedArgs db, int dtype) {
    if (!is16(dtype) || !adapter_grad16_takes(da, LOW_B)) da.C = nullptr;
    if (!is16(dtype) || !adapter_grad16_takes(db, LOW_A)) db.C = nullptr;
    return {da, db};
}
static int other_grads(const GroupedArgs& da, const GroupedArgs& db, const Grads16& taken, int dtype) {
    if (da.C && !taken.da.C && launch_narrow_weights(da, LOW_B, dtype) != 0) return -1;
    return db.C && !taken.db.C ? launch_narrow_weights(db, LOW_A, dtype) : 0;
}

// Tiles on which the shared product of a layer with adapters takes their term in (edge 0: none); whole: nothing hangs over
struct TermTile { int edge; bool whole, ragged, sums; int last; };       // sums: the product can be had as float32 sums instead; last: the edge to take where there is no memory for those
static TermTile term_tile(const GroupedArgs& s, const AdapterTerm& term, int dtype) {
    if (!is16(dtype) || s.a_cs != 1 || (s.b_cs != 1 && s.b_rs != 1) || path_disabled("mfma")) return {0, false, false, false, 0};
    Plan p{FAM_MFMA16, 64, 64, false, s.b_cs == 1, true, ""};
    const Lie lie = worse(lies(s.A, s.a_rs, 0, s.k, 2), p.b_mc ? lies(s.B, s.b_rs, 0, s.n, 2) : lies(s.B, s.b_cs, 0, s.k, 2));
    p.ragged = lie == LIE_RAGGED;
    choose_tile16(p, 1, s.gr.rows, s.k, s.n);
    if (p.ragged && p.bm == 256) p.bm = p.bn = 128;
    // (fp16, 2048 rows of 2048 -> 1024, rank 8, 128 tiles of 128: 26 us, on 64 x 64 tiles 22)
    if (p.bm == 128 && (long long)((s.gr.rows + 127) / 128) * ((s.n + 127) / 128) * 4 < cus() * 3) p.bm = p.bn = 64;
    const long long tiles = (long long)((s.gr.rows + p.bm - 1) / p.bm) * ((s.n + p.bn - 1) / p.bn);
    // byte offsets into h and into an adapter's factor in 32 bits
    const bool reach = (long long)s.gr.rows * term.rank < (1 << 29) && ((term.rank - 1) * term.b_rs + (s.n - 1) * term.b_cs) < (1 << 30);
    // from about a tile for every other CU on, and while a tile's rows are few segments, each of which costs it 1 to 2 us a step of the rank (bf16, 4096 rows, the layer's us in tiles of 128 and
    // apart: 7 segments, 1024 -> 4096, rank 8 50 / 86; 400 segments 77 / 100, 4096 -> 4096, rank 32 205 / 228, 1024 -> 1024, rank 64 62 / 47; 1500 segments 133 / 140, 300 / 281, 142 / 66)
    const int last = !reach || lie == LIE_NEITHER || term.gr.groups > ROW_TILES_GROUPS ? 0 : p.bm >= 128 && p.bn >= 128 ? 128 : 64;
    if (!last || p.bm != p.bn || tiles * 2 < cus() || term.gr.rows / term.gr.groups < 16 || path_disabled("adapter_tiles")) return {0, false, p.ragged, lie != LIE_NEITHER, last};
    return {p.bm, !p.edge, p.ragged, true, last};
}

// The shared product and the adapters' term
static int shared_with_term(const GroupedArgs& s, const AdapterTerm& term, int dtype) {
    const TermTile t = term_tile(s, term, dtype);
    if (t.edge == 256) return dtype == RP_DTYPE_BFLOAT16 ? launch_adapter_tiles16_256_bf16(s, term, !t.whole) : launch_adapter_tiles16_256_f16(s, term, !t.whole);
    if (t.edge) return t.edge == 128 ? launch_adapter_tiles16_128(s, term, !t.whole, t.ragged, dtype) : launch_adapter_tiles16_64(s, term, t.ragged, dtype);
    if (t.sums && adapter_expand16_takes(s, term)) {
        bool taken;
        const int rc = launch_adapter_expand16(s, term, t.ragged, dtype, &taken);
        if (rc != 0 || taken) return rc;
    }
    if (t.last) return t.last == 128 ? launch_adapter_tiles16_128(s, term, true, t.ragged, dtype) : launch_adapter_tiles16_64(s, term, t.ragged, dtype);
    // what no kernel of the adapters' own takes (float32 and float64, the narrowest widths, operands without a unit stride): the product is rounded, and the sum again
    int rc;
    bool refused;
    {
        const CallScratch memory(CallScratch::MOST);
        const GemmWorkspaceLoan loan(memory.ptr, CallScratch::MOST);
        rc = rp_hip_gemm_strided_batched(s.C, s.A, s.B, s.bias, 1, s.gr.rows, s.k, s.n, 0, s.a_rs, s.a_cs, 0, s.b_rs, s.b_cs, 0, s.c_rs, 1, s.accumulate, dtype);
        refused = loan.refused;
    }
    if (refused) rc = grouped_rows(s, dtype);                 // (k would be split, and there is no memory for that: one group of all rows needs none)
    if (rc != 0) return rc;
    return launch_grouped_rows_generic(GroupedArgs{s.C, term.h, term.b, nullptr, nullptr, term.gr, term.rank, s.n, term.rank, 1, term.b_ws, term.b_rs, term.b_cs, 0, s.c_rs, ACCUMULATE_JOINED}, true, dtype);
}

static bool grouped_args_ok(const char* who, bool pointers, int groups, int rows, int k, int n, std::initializer_list<long long> strides, int dtype) {
    if (!pointers || groups <= 0 || rows <= 0 || k <= 0 || n <= 0) { set_error("%s: null operand or non-positive extent (groups=%d rows=%d k=%d n=%d)", who, groups, rows, k, n); return false; }
    if (!dtype_size(dtype)) { set_error("%s: unsupported dtype %d", who, dtype); return false; }
    for (long long s : strides)
        if (s < 0) { set_error("%s: negative stride", who); return false; }
    return true;
}

static bool output_rows_ok(const char* who, const char* what, int rows, int width, long long rs) {
    if (rows == 1 || rs >= width) return true;
    set_error("%s: rows of %s are %lld elements apart and hold %d", who, what, rs, width);
    return false;
}

}  // namespace rp

using namespace rp;

extern "C" {

int rp_hip_grouped_linear_forward(void* y, const void* x, const void* w, const void* bias, const int* offsets, int groups, int rows, int k, int n,
                                  long long x_rs, long long x_cs, long long w_gs, long long w_rs, long long w_cs, long long y_rs, int dtype) {
    const char* who = "rp_hip_grouped_linear_forward";
    if (!grouped_args_ok(who, y && x && w && offsets, groups, rows, k, n, {x_rs, x_cs, w_gs, w_rs, w_cs, y_rs}, dtype) || !output_rows_ok(who, "y", rows, n, y_rs)) return -1;
    const RowGroups gr{offsets, nullptr, groups, rows, groups};
    return grouped_rows(GroupedArgs{y, x, w, bias, nullptr, gr, k, n, x_rs, x_cs, w_gs, w_rs, w_cs, 0, y_rs, 0}, dtype);
}

int rp_hip_grouped_linear_backward(void* dx, void* dw, void* db, const void* dy, const void* x, const void* w, const int* offsets, int groups, int rows, int k, int n,
                                   long long dy_rs, long long x_rs, long long x_cs, long long w_gs, long long w_rs, long long w_cs, long long dx_rs,
                                   int accumulate_dx, int accumulate_dw, int accumulate_db, int dtype) {
    const char* who = "rp_hip_grouped_linear_backward";
    if (!grouped_args_ok(who, dy && offsets && (!dx || w) && (!dw || x), groups, rows, k, n, {dy_rs, x_rs, x_cs, w_gs, w_rs, w_cs, dx_rs}, dtype)) return -1;
    if (dx && !output_rows_ok(who, "dx", rows, k, dx_rs)) return -1;
    const RowGroups gr{offsets, nullptr, groups, rows, groups};
    GroupedArgs xg{dx, dy, w, nullptr, nullptr, gr, n, k, dy_rs, 1, w_gs, w_cs, w_rs, 0, dx_rs, accumulate_dx ? ACCUMULATE : 0};
    const GroupedArgs wg{dw, x, dy, nullptr, nullptr, gr, k, n, x_rs, x_cs, 0, dy_rs, 1, (long long)k * n, n, accumulate_dw ? ACCUMULATE : 0};
    const GroupedSums sums{db, dy, gr, n, accumulate_db, dy_rs};
    int result;
    if (backward_together(xg, wg, sums, dtype, &result)) return result;
    if (dx) {
        if (grouped_rows(xg, dtype) != 0) return -1;
        xg.C = nullptr;
        if (backward_together(xg, wg, sums, dtype, &result)) return result;
    }
    if (dw && grouped_weights(wg, dtype) != 0) return -1;
    return db ? launch_grouped_sums(sums, dtype) : 0;
}

int rp_hip_adapter_linear_forward(void* y, void* h, const void* x, const void* w, const void* bias, const void* a, const void* b, const float* scales, const int* ids, const int* offsets,
                                  int segments, int adapters, int rows, int k, int n, int rank, long long x_rs, long long x_cs, long long w_rs, long long w_cs, long long y_rs, int dtype) {
    const char* who = "rp_hip_adapter_linear_forward";
    if (!grouped_args_ok(who, y && h && x && w && a && b && ids && offsets && adapters > 0 && rank > 0, segments, rows, k, n, {x_rs, x_cs, w_rs, w_cs, y_rs}, dtype) ||
        !output_rows_ok(who, "y", rows, n, y_rs)) return -1;
    const RowGroups gr{offsets, ids, segments, rows, adapters};
    const GroupedArgs low{h, x, a, nullptr, scales, gr, k, rank, x_rs, x_cs, (long long)k * rank, rank, 1, 0, rank, 0};
    const GroupedArgs shared{y, x, w, bias, nullptr, RowGroups{nullptr, nullptr, 1, rows, 1}, k, n, x_rs, x_cs, 0, w_rs, w_cs, 0, y_rs, 0};
    const AdapterTerm term{(const float*)h, b, gr, rank, (long long)rank * n, n, 1};
    if (is16(dtype) && adapter_few_rows16_takes(shared, low, term)) return launch_adapter_few_rows16(shared, low, term, dtype);
    if (narrow_rows(low, dtype) != 0) return -1;
    return shared_with_term(shared, term, dtype);
}

int rp_hip_adapter_linear_backward(void* dx, void* da, void* db, void* u, const void* dy, const void* x, const void* w, const void* a, const void* b, const void* h,
                                   const float* scales, const int* ids, const int* offsets, int segments, int adapters, int rows, int k, int n, int rank,
                                   long long dy_rs, long long x_rs, long long x_cs, long long w_rs, long long w_cs, long long dx_rs,
                                   int accumulate_dx, int accumulate_da, int accumulate_db, int dtype) {
    const char* who = "rp_hip_adapter_linear_backward";
    if (!grouped_args_ok(who, dy && ids && offsets && adapters > 0 && rank > 0 && (!(dx || da) || (u && b)) && (!dx || (w && a)) && (!da || x) && (!db || h), segments, rows, k, n,
                         {dy_rs, x_rs, x_cs, w_rs, w_cs, dx_rs}, dtype)) return -1;
    if (dx && !output_rows_ok(who, "dx", rows, k, dx_rs)) return -1;
    const RowGroups gr{offsets, ids, segments, rows, adapters};
    if ((dx || da) && narrow_rows(GroupedArgs{u, dy, b, nullptr, scales, gr, n, rank, dy_rs, 1, (long long)rank * n, 1, n, 0, rank, 0}, dtype) != 0) return -1;
    const GroupedArgs ga{da, x, u, nullptr, nullptr, gr, k, rank, x_rs, x_cs, 0, rank, 1, (long long)k * rank, rank, accumulate_da ? ACCUMULATE : 0};
    const GroupedArgs gb{db, h, dy, nullptr, nullptr, gr, rank, n, rank, 1, 0, dy_rs, 1, (long long)rank * n, n, accumulate_db ? ACCUMULATE : 0};
    const Grads16 g16 = grads16_of(ga, gb, dtype);
    if (dx) {
        const GroupedArgs shared{dx, dy, w, nullptr, nullptr, RowGroups{nullptr, nullptr, 1, rows, 1}, n, k, dy_rs, 1, 0, w_cs, w_rs, 0, dx_rs, accumulate_dx ? ACCUMULATE : 0};
        const AdapterTerm term{(const float*)u, a, gr, rank, (long long)k * rank, 1, rank};
        const TermTile t = term_tile(shared, term, dtype);
        // dx and the factors' gradients in one launch, unless workgroups that stay on their CU take dx
        if (t.edge && t.edge < 256 && shared.b_rs == 1 && (g16.da.C || g16.db.C)) {
            if ((dtype == RP_DTYPE_BFLOAT16 ? launch_adapter_backward16_bf16(shared, term, g16.da, g16.db, t.edge, t.ragged) : launch_adapter_backward16_f16(shared, term, g16.da, g16.db, t.edge, t.ragged)) != 0) return -1;
            return other_grads(ga, gb, g16, dtype);
        }
        if (shared_with_term(shared, term, dtype) != 0) return -1;
    }
    if ((g16.da.C || g16.db.C) && launch_adapter_grads16(g16.da, g16.db, dtype) != 0) return -1;
    return other_grads(ga, gb, g16, dtype);
}

}  // extern "C"
