// The part of attention over many sequences that takes 16 query rows to a workgroup, as a kernel of its own
// (attention_seqs.hip) and beside tiles of many rows in one launch (attention_tiles.hip, attention_terms.hip).
#pragma once

#include "attention_seqs.h"

namespace zl {

// ---- 16 query rows on the matrix cores ---------------------------------------------------------
// Decode and short chunks: a workgroup takes 16 query rows of one kv head (or as many as there are)
// and a split of their keys, its waves the blocks of keys in turn, K and V straight from the
// cache into operand registers: the call is bound by reading the cache once. f32 calls take 16
// keys to a block and the f32 MFMA 16x16x4 (exact f32 products and sums), bf16 calls 32 keys and
// 16x16x32. Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that lane
// (n = lane % 16, g = lane / 16) keeps query row n throughout: its maximum, its sum, its rescaling
// factor, and keys 16 T + 4 g + r of score tile T, which are the second product's operand as they
// stand. V's rows are read in the order of those keys, CW columns to a lane, one MFMA a column
// (bf16: pairs of keys put together from two rows by byte permutes); columns come out as
// 16 CW c + CW (4 g + r) + j in register r of accumulator c CW + j.
// K of the next block is requested when this one's scores are formed, V when its output is: each is
// on its way through the other's product, and two workgroups share a CU, so that one's prologue and
// merge pass under the other's reads. The waves' states merge through LDS.
// Measured: 64 sequences of up to 8000 positions, 32 / 16 heads x 128 bf16, 451 us, 5.4 TB/s; 16 of up to 8192, 8 / 4 x
// 256 f32, 129 us, 5.1 TB/s; one token at 1250, f32, 14.4 us with the join: a chain of latencies.
// Heads of 512 take two waves to a block of keys, half the head size each, which exchange their sums of the
// scores through LDS (a wave that had all of it would need all of a SIMD's registers).
template <int D> constexpr int row_halves() { return D > 256 ? 2 : 1; }
constexpr int row_slots(int D) { return D > 256 ? 2 : 4; }
template <int D, int W> struct RowsLds {
    // the merge buffer; before it the query rows, and the halves' sums of the scores
    float o[row_slots(D) * 16 * (D + 4)];
    float m[W][16], l[W][16];
};
template <typename T, int D, int W>
__device__ __forceinline__ void seq_rows(const SeqArgs& a, int id, RowsLds<D, W>& lds) {
    float* const s_o = lds.o;
    auto& s_m = lds.m;
    auto& s_l = lds.l;
#include "attention_rows.inl"
}

}  // namespace zl
