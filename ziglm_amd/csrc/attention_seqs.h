// Shared by the kernels of attention over many sequences (attention_seqs.hip, attention_tiles.hip).
#pragma once

#include <math.h>
#include <algorithm>

#include "zl_common.h"
#include "zl_host.h"

namespace zl {

typedef float acc4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
constexpr float kLog2e = 1.4426950408889634f;

struct SeqArgs {
    const void* q;         // [n_tokens] rows of q_stride elements, heads of D
    const void* kc;        // rows of kv_stride elements
    const void* vc;
    void* out;             // [n_tokens][nh][D]
    float* ws;             // partials: [n_tokens][nh][nparts][D] sums, then [..][2] (max, sum) (nparts > 1)
    const int32_t* cu;     // [n_seqs + 1], or null: one token a sequence (paged), one sequence (prompt)
    const int32_t* len;    // [n_seqs] sequence lengths (paged)
    const int32_t* table;  // [n_seqs][max_pages] (paged), or null: prompt
    int64_t q_stride, kv_stride;
    int64_t cache_pages;
    int page, page_shift;  // page_shift: log2(page) or -1
    int max_pages;
    int max_len;           // of a sequence, as the caller says: the host's rules go by it
    int lim;               // positions that there can be: of max_len and of the table's width the smaller
    int n_seqs, n_tokens, nh, nkv, gq, D, window;
    int few_rows;          // sequences of at most this many query rows a kv head are k_seq_rows's, the others k_seq_tile's
    int nsplit, tile_split, nparts;  // splits of k_seq_rows's and k_seq_tile's ranges, the larger of them
    int chunk, tile_chunk;           // keys of a split
    int rows_grid, tile_grid;        // workgroups of each
    int tile_rows;         // query rows of a workgroup of k_seq_tile
    float scale, softcap, inv_cap;
    float cap_in;          // 2 log2(e) scale / softcap
    float cap_small, cap_c[4];  // scores up to this take the series, its coefficients
    float unit;            // of running maxima: log2(e); bf16: log2(e) * |scale|, or log2(e) where soft-capped
};

// The tokens of a sequence and where they stand.
struct Seq {
    int tok0, nq;  // first row of q, new tokens
    int pos0;      // position of the first
    int lim;       // positions are below this
    int64_t row0;  // prompts: row of position 0
    const int32_t* pages;
};
__device__ __forceinline__ int seq_tokens(const SeqArgs& a, int s, int& tok0) {
    if (!a.cu) {
        tok0 = a.table ? s : 0;
        return a.table ? 1 : a.n_tokens;
    }
    tok0 = min(max(a.cu[s], 0), a.n_tokens);
    return min(max(a.cu[s + 1], tok0), a.n_tokens) - tok0;
}
__device__ __forceinline__ Seq seq_of(const SeqArgs& a, int s) {
    Seq q;
    q.nq = seq_tokens(a, s, q.tok0);
    if (a.table) {
        q.pos0 = max(a.len[s], 0) - q.nq;
        q.lim = a.lim;
        q.row0 = 0;
        q.pages = a.table + (int64_t)s * a.max_pages;
    } else {
        q.pos0 = 0;
        q.lim = q.nq;
        q.row0 = q.tok0;
        q.pages = nullptr;
    }
    return q;
}
// Cache row of position t (in range), or -1.
__device__ __forceinline__ int row_of(const SeqArgs& a, const Seq& q, int t) {
    if (!a.table) return (int)q.row0 + t;
    const int e = a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
    const int id = q.pages[e];
    return id >= 0 && id < a.cache_pages ? id * a.page + (t - e * a.page) : -1;
}

// Query rows of a kv head: row r of a sequence is token r / gq, head r % gq of the group. Tiles of R
// consecutive rows; tile `tile` over the sequences of few (FEW) or many rows in order -> (sequence, tile
// of it), or -1. Every wave searches for itself, 64 sequences at a time.
template <int R, bool FEW>
__device__ __forceinline__ int find_tile(const SeqArgs& a, int tile, int& in_seq) {
    const int lane = threadIdx.x & 63;
    if (!a.cu) {  // (the host launches the one kernel that takes them)
        const int per = (int)(((int64_t)(a.table ? 1 : a.n_tokens) * a.gq + R - 1) / R);
        in_seq = tile % per;
        return tile / per < a.n_seqs ? tile / per : -1;
    }
    for (int s0 = 0; s0 < a.n_seqs; s0 += kWave) {
        int n = 0;
        if (s0 + lane < a.n_seqs) {
            int tok0;
            const int rows = seq_tokens(a, s0 + lane, tok0) * a.gq;
            n = (rows <= a.few_rows) == FEW ? (rows + R - 1) / R : 0;
        }
        int x = n;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        const uint64_t past = __ballot(x > tile);
        if (past) {
            const int l = __builtin_ctzll(past);
            in_seq = tile - __shfl(x - n, l);
            return s0 + l;
        }
        tile -= __shfl(x, kWave - 1);
    }
    return -1;
}

// The keys that a tile of rows [r0, r1] sees, [ks, ke), in `used` splits of `chunk`.
struct Range {
    int ks, ke, used;
};
__device__ __forceinline__ Range tile_range(const SeqArgs& a, const Seq& q, int r0, int r1, int chunk) {
    const int i0 = r0 / a.gq, i1 = r1 / a.gq;
    Range g;
    g.ke = min(q.pos0 + i1, q.lim - 1) + 1;
    g.ks = a.window > 0 ? max(0, q.pos0 + i0 + 1 - a.window) : 0;
    g.used = max((int)(((int64_t)(g.ke - g.ks) + chunk - 1) / chunk), 1);
    return g;
}
// The same, at most, as the host knows it: keys of a tile of R rows, and splits.
inline int64_t most_keys(const SeqArgs& a, int R) {
    return a.window > 0 ? std::min<int64_t>((int64_t)a.window + cdiv(R - 1, a.gq), a.max_len) : a.max_len;
}

// Soft-capped score of a bf16 call: cap * tanh(z) = cap - 2 cap / (exp(2 z) + 1), z = x * scale / cap. The
// difference of nearly equal terms near 0 is off by 2^-23 cap, far inside the rounding of the weights
// (2^-8); f32 calls take the form that is exact to the last places there too.
__device__ __forceinline__ float cap_bf16(const SeqArgs& a, float x) {
    return fmaf(__builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * a.cap_in) + 1.0f), -2.0f * a.softcap, a.softcap);
}
// The same where |z| <= 0.35, by tanh's series up to z^7 (off by 62 / 2835 z^9 cap, 2^-19 cap at the most).
__device__ __forceinline__ float cap_series(const SeqArgs& a, float x) {
    const float y = x * x;
    return x * fmaf(y, fmaf(y, fmaf(y, a.cap_c[3], a.cap_c[2]), a.cap_c[1]), a.cap_c[0]);
}

// 4 consecutive elements as f32
__device__ __forceinline__ f32x4 ld4(const float* p) { return ldf4(p); }
__device__ __forceinline__ f32x4 ld4(const uint16_t* p) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
    return f32x4{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
}
__device__ __forceinline__ void st4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void st4(uint16_t* p, const f32x4& v) {
    *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// Tiles of R query rows over all sequences, at most: sum of ceil(new tokens * gq / R).
inline int64_t most_tiles(const SeqArgs& a, int R) {
    return std::min<int64_t>((int64_t)a.n_tokens * a.gq / R + a.n_seqs, (int64_t)a.n_tokens * cdiv(a.gq, R));
}
// k_seq_tile (attention_tiles.hip): query rows of a workgroup for a type and head size, and the launch.
int tile_rows_of(int dtype, int D, bool small);
void launch_tiles(int dtype, const SeqArgs& a, hipStream_t s);
void launch_terms(const SeqArgs& a, hipStream_t s);  // (attention_terms.hip)

}  // namespace zl
