// Grouped products: rows in groups, a weight for each group (or one that several groups share).
#pragma once
#include "rp_gemm.h"
#include "rp_rows.h"

namespace rp {

// By rows:     C[i, :] (+)= scale_w * A[i, :] . B_w + bias_w      for every row i of a group whose weight is w
// By weights:  C_w (+)= sum over the rows i of w's groups of A[i, :]^T . B[i, :]
// Strides in elements; B (by rows) and C (by weights) have a stride b_ws / c_ws from weight to weight.
// accumulate: added to what C holds, after the product has been rounded (as a product of its own would be) or together with it
enum { ACCUMULATE = 1, ACCUMULATE_JOINED = 2 };
struct GroupedArgs {
    void* C;
    const void* A;
    const void* B;
    const void* bias;              // [weights, n] dense, or null
    const float* scales;           // [weights] float32, or null
    RowGroups gr;
    int k, n;                      // by rows: A [rows, k], C [rows, n];  by weights: C_w [k, n], A [rows, k], B [rows, n]
    long long a_rs, a_cs, b_ws, b_rs, b_cs, c_ws, c_rs;        // C has unit column stride
    int accumulate;
};

// Slot `id` of `total` tiles that the eight XCDs take in a run each (workgroup i is XCD i % 8's); past the run's end: `total`
__device__ __forceinline__ int run_tile(int id, int total) {
    const int per = (total + 7) / 8, at = id % 8 * per + id / 8;
    return id / 8 < per && at < total ? at : total;
}
// Tile `at` of a matrix of rows x cols tiles: column by column through eight rows of tiles at a time, so that the tiles of a run that are
// at work together need a few panels of both operands.  (Row by row over all XCDs, every L2 fetched every weight: dx of 1999 rows of 6 groups, 1032 -> 520 in bf16 on
// 64 x 64 tiles 18 us, 13.7 so.)
__device__ __forceinline__ TileCoord chunk_tile(int at, int rows, int cols) {
    constexpr int CHUNK = 8;
    const int r0 = at / (CHUNK * cols) * CHUNK, h = rows - r0 < CHUNK ? rows - r0 : CHUNK, in = at - r0 * cols;
    return TileCoord{r0 + in % h, in / h, true};
}

// Which operand is in the accumulate type (float32, float64 for float64) whatever the tensors' type is: the low-rank activations of an adapter
enum GroupedLow { LOW_A, LOW_B };

// By rows, on the kernel that suits the sizes (rp_grouped.hip)
int launch_grouped_rows(const GroupedArgs& g, int dtype);
// Both gradients of a grouped layer and column sums, those whose output is not null, in as few launches as suit them
struct GroupedSums;
int launch_grouped_backward(const GroupedArgs& x, const GroupedArgs& wg, const GroupedSums& sums, int dtype);
// Any strides and sizes, all types (rp_grouped_generic.hip); low: A is.  No scales; by weights: no ids.
int launch_grouped_rows_generic(const GroupedArgs& g, bool low, int dtype);
int launch_grouped_weights_generic(const GroupedArgs& g, int dtype);
// The same for an adapter's narrow products (rp_adapter_any.hip): by rows C is, scales taken; by weights A or B, ids taken
int launch_narrow_rows(const GroupedArgs& g, int dtype);
int launch_narrow_weights(const GroupedArgs& g, GroupedLow low, int dtype);
// out[w, :] (+)= sum over the rows of group w of x[i, :]
struct GroupedSums;
int launch_grouped_sums(const GroupedSums& s, int dtype);

// fp32 / fp64 (rp_grouped_wavek.hip), rows of any length and start
bool grouped_rows_wavek_takes(const GroupedArgs& g, int dtype);
int launch_grouped_rows_wavek(const GroupedArgs& g, int dtype);
// the gradients in one launch: those of x, w and sums whose output is not null
bool grouped_backward_wavek_takes(const GroupedArgs& x, const GroupedArgs& w, int dtype);
int launch_grouped_backward_wavek(const GroupedArgs& x, const GroupedArgs& w, const GroupedSums& sums, int dtype);

// bf16 / fp16 on the tiles of the 16-bit MFMA kernel (rp_grouped_mfma16*.hip).  ragged: rows of any length and start.
int launch_grouped_rows16_256_bf16(const GroupedArgs& g);
int launch_grouped_rows16_256_f16(const GroupedArgs& g);
int launch_grouped_weights16_256_bf16(const GroupedArgs& g);
int launch_grouped_weights16_256_f16(const GroupedArgs& g);
int launch_grouped_rows16_128(const GroupedArgs& g, bool ragged, int dtype);
int launch_grouped_weights16_128(const GroupedArgs& g, bool ragged, int dtype);
int launch_grouped_rows16_64(const GroupedArgs& g, bool ragged, int dtype);
int launch_grouped_weights16_64(const GroupedArgs& g, bool ragged, int dtype);
constexpr long long GROUPED_BACKWARD16_MOST = 12 << 20;        // workgroups
// The gradients in one launch, the input's on tiles of 64 or 128, the weights' on no larger ones: those of x, w and sums whose output is not null; w row-major (rp_grouped_backward16*.hip)
int launch_grouped_backward16_bf16(const GroupedArgs& x, int x_tile, const GroupedArgs& w, int w_tile, const GroupedSums& sums, bool ragged);
int launch_grouped_backward16_f16(const GroupedArgs& x, int x_tile, const GroupedArgs& w, int w_tile, const GroupedSums& sums, bool ragged);

// + h[i] . b_a for the rows i of adapter a: what a layer's adapters add to its shared product (strides of b in elements)
struct AdapterTerm {
    const float* h;                // [rows, rank] dense
    const void* b;                 // [adapters, rank, n]
    RowGroups gr;                  // the segments
    int rank;
    long long b_ws, b_rs, b_cs;
};

// bf16 / fp16, row tiles of a few rows against a row-major weight that is streamed once (rp_grouped_stream16.hip)
bool grouped_stream16_takes(const GroupedArgs& g);
int launch_grouped_stream16(const GroupedArgs& g, int dtype);
struct StreamGrid;
int launch_stream16_combine(const GroupedArgs& g, const StreamGrid& sg, const AdapterTerm* term, int dtype);

// h[i] = scales[a] x[i] . a_a in float32 for bf16 / fp16 operands (rp_adapter16.hip); C is h
bool adapter_shrink16_takes(const GroupedArgs& g);
int launch_adapter_shrink16(const GroupedArgs& g, int dtype);
// The shared product as float32 sums, then y = sums + bias + h[i] . b_a (rp_adapter16.hip); ragged: rows of any length and start
bool adapter_expand16_takes(const GroupedArgs& shared, const AdapterTerm& term);
int launch_adapter_expand16(const GroupedArgs& shared, const AdapterTerm& term, bool ragged, int dtype, bool* taken);      // not taken: no memory for the sums
int launch_sums16_128(const GemmArgs& g, bool b_mc, bool ragged, float* sums, int dtype);      // [m][n], rp_adapter16_sums.hip
// The shared product with that term in it, on MFMA tiles (rp_adapter16_tiles*.hip)
int launch_adapter_tiles16_256_bf16(const GroupedArgs& shared, const AdapterTerm& term, bool edge);
int launch_adapter_tiles16_256_f16(const GroupedArgs& shared, const AdapterTerm& term, bool edge);
int launch_adapter_tiles16_128(const GroupedArgs& shared, const AdapterTerm& term, bool edge, bool ragged, int dtype);
int launch_adapter_tiles16_64(const GroupedArgs& shared, const AdapterTerm& term, bool ragged, int dtype);
// the gradients of an adapter's factors (rp_adapter16_grads.hip): LOW_A for dB, LOW_B for dA
bool adapter_grad16_takes(const GroupedArgs& g, GroupedLow low);
int launch_adapter_grads16(const GroupedArgs& da, const GroupedArgs& db, int dtype);       // those whose C is not null
// both, and dx with its term on tiles of 64 or 128 (w row-major), in one launch (rp_adapter16_backward*.hip)
int launch_adapter_backward16_bf16(const GroupedArgs& shared, const AdapterTerm& term, const GroupedArgs& da, const GroupedArgs& db, int tile, bool ragged);
int launch_adapter_backward16_f16(const GroupedArgs& shared, const AdapterTerm& term, const GroupedArgs& da, const GroupedArgs& db, int tile, bool ragged);
// The whole layer for a few rows: `shared` one group of all rows, `low` the product above, `term` what it adds
bool adapter_few_rows16_takes(const GroupedArgs& shared, const GroupedArgs& low, const AdapterTerm& term);
int launch_adapter_few_rows16(const GroupedArgs& shared, const GroupedArgs& low, const AdapterTerm& term, int dtype);

}  // namespace rp
