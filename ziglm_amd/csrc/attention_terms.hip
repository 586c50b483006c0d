// Attention of many sequences, f32: tiles of many query rows on the bf16 matrix cores by three-term products
// (attention_seqs.hip has the definition and the host side, attention_tiles.hip the form of the kernel).
//
// An f32 value is the sum of three bf16 terms, x = h + m + l: h its upper 16 bits, m the rest rounded, l what
// remains, exactly. A product is six of theirs, hh + hm + mh + mm + hl + lh; what is left out is under 2^-23 of
// it, as its f32 rounding is. Six bf16 MFMAs take 6/16 of the f32 MFMA's time. Q's terms stay in
// registers, the weights' are formed in them; K and V are split once for the 128 rows of a workgroup on
// their way to LDS, three planes each. Scores sum their largest products and the others apart. As in
// k_seq_tile both products are transposed and a lane (n = lane % 16, h = lane / 16) keeps query row n.
// LDS holds one tile of 32 keys (106 KB at heads of 256): the next one waits in registers, split already,
// between two barriers.
// Infinities have no terms. Values of V that are infinite or NaN stay out and go to the rows that see them
// at the end; keys of K with such values get their scores by a plain dot product.
// It waits at its two barriers a tile, a workgroup to a CU (512 tokens behind 1501, 8 / 4 heads x 256: 75 us with the
// join, matrix cores 25% and vector units 29% busy, by the f32 MFMA 109; a prompt of 4096, 32 / 16 x 128: 778 us,
// 177 TFLOP/s, which is past the 153 that a large f32 matrix product reaches).
#include "attention_rows.h"

namespace zl {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// Terms of 8 values, as bf16 pairs.
struct Terms {
    u32x4 h, m, l;
};
__device__ __forceinline__ Terms split8(const f32x4& a, const f32x4& b) {
    Terms t;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = e < 2 ? a[2 * e] : b[2 * e - 4], y = e < 2 ? a[2 * e + 1] : b[2 * e - 3];
        t.h[e] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        const float xr = x - __uint_as_float(__float_as_uint(x) & 0xffff0000u), yr = y - __uint_as_float(__float_as_uint(y) & 0xffff0000u);
        t.m[e] = pack_bf16x2(xr, yr);
        t.l[e] = pack_bf16x2(xr - bf16_lo(t.m[e]), yr - bf16_hi(t.m[e]));
    }
    return t;
}
__device__ __forceinline__ bf16x8 op(const u32x4& v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ acc4 mfma(const bf16x8& a, const bf16x8& b, const acc4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Over the four lanes of a query row.
template <typename F>
__device__ __forceinline__ float over_row4(float v, F f) {
    {
        const unsigned x = __builtin_bit_cast(unsigned, v), y = __builtin_bit_cast(unsigned, dpp<0xE4>(v));
        const auto p = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        v = f(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
    }
    const unsigned x = __builtin_bit_cast(unsigned, v), y = __builtin_bit_cast(unsigned, dpp<0xE4>(v));
    const auto p = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return f(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
}

constexpr int kTermWaves = 8, kTermRows = 16 * kTermWaves, kTermKeys = 32;
// LDS as in k_seq_tile: K's chunks in four planes by their index mod 4, V's rows padded by 32 bytes
template <int D> struct TermsLds {
    static constexpr int KS = D / 2 + 16, KP = kTermKeys * KS, VS = 2 * D + 32;
    static_assert(KP % 256 == 0 && KS / 16 % 2 == 1, "planes");
    uint8_t k[3][4 * KP], v[3][kTermKeys * VS];
    uint32_t gap[2], bad[2];  // keys without a row; with infinite or NaN values in K
    int wild;                 // infinite or NaN values of V were kept out of LDS
};
template <int D, bool CAP>
__device__ __forceinline__ void seq_terms(const SeqArgs& a, int id, TermsLds<D>& lds) {
    constexpr int KB = kTermKeys, TH = kTermWaves * kWave;
    constexpr int NQ = D / 32;       // chunks (8 values) of a query row to a lane
    constexpr int NB = D / 16;       // accumulators of the output
    constexpr int CR = D / 8;        // chunks of a row
    constexpr int NC = KB * CR / TH > 0 ? KB * CR / TH : 1;  // of a tile, to a thread
    constexpr int RS = TH / CR;      // rows between a thread's chunks
    constexpr float kSlack = 8.0f;   // log2
    constexpr int KS = TermsLds<D>::KS, KP = TermsLds<D>::KP, VS = TermsLds<D>::VS;
    auto& s_k = lds.k;
    auto& s_v = lds.v;
    auto& s_gap = lds.gap;
    auto& s_bad = lds.bad;
    int& s_wild = lds.wild;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = id % a.nkv;
    id /= a.nkv;
    const int split = id % a.tile_split;
    int tile;
    const int sq = __builtin_amdgcn_readfirstlane(find_tile<kTermRows, false>(a, id / a.tile_split, tile));
    if (sq < 0) return;
    const Seq q = seq_of(a, sq);
    const int rows = q.nq * a.gq;
    // the last tiles, whose ranges are the longest, first
    const int r0 = ((rows + kTermRows - 1) / kTermRows - 1 - __builtin_amdgcn_readfirstlane(tile)) * kTermRows;
    if (r0 < 0 || r0 >= rows) return;
    const int r1 = min(r0 + kTermRows, rows) - 1;
    const Range rg = tile_range(a, q, r0, r1, a.tile_chunk);
    if (split >= rg.used) return;
    const int ks = rg.ks + split * a.tile_chunk, ke = rg.ke - ks > a.tile_chunk ? ks + a.tile_chunk : rg.ke;
    const int ntile = ke > ks ? (ke - ks + KB - 1) / KB : 0;

    // the lane's query row and its keys [lo, hi], and what all of the wave's rows see
    const int w0 = r0 + wave * 16, w1 = min(w0 + 15, r1);
    const int rr = min(w0 + n, r1), i = rr / a.gq, p = q.pos0 + i;
    const int hi = p >= 0 && p < q.lim ? p : -1;  // (rows behind the last are the last once more)
    const int lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
    const int pf = q.pos0 + w0 / a.gq, pl = q.pos0 + max(w1, 0) / a.gq;
    const bool whole = pf >= 0 && pl < q.lim;
    const int any_lo = a.window > 0 ? max(0, pf + 1 - a.window) : 0, all_lo = a.window > 0 ? max(0, pl + 1 - a.window) : 0;
    const int any_hi = w0 <= r1 ? min(pl, q.lim - 1) : -1, all_hi = pf;

    const float* const qrow = (const float*)a.q + (int64_t)(q.tok0 + i) * a.q_stride + (kvh * a.gq + rr % a.gq) * D;
    Terms qt[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) qt[j] = split8(ldf4(qrow + 32 * j + 8 * h), ldf4(qrow + 32 * j + 8 * h + 4));
    acc4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = acc4{};
    float m = -INFINITY, l = 0.0f;

    // ---- the tiles' way to LDS ----
    const int sr = tid / CR, sc = tid % CR;               // the thread's first row and its chunk of V
    const int kc = sc % (CR / 4) * 4 + sc / (CR / 4);      // and of K
    const bool mine = sr < KB;                             // (heads of 64: half of the threads have none)
    const int kst = sr * KS + kc % 4 * KP + kc / 4 * 16, vst = sr * VS + sc * 16;
    const float* const kbase = (const float*)a.kc + kvh * D + 8 * kc;
    const float* const vbase = (const float*)a.vc + kvh * D + 8 * sc;
    f32x4 bk[NC][2], bv[NC][2];
    int row[NC], pg[NC];  // cache rows of the tile in bk and bv, page ids of the one behind it
    // The page ids of tile t are requested behind the loads of the tile before and looked at a tile later (a
    // wait for them is one for all loads before them).
    auto find_pages = [&](int t) {
        if (!a.table) return;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int key = min(ks + t * KB + sr + j * RS, ke - 1);
            pg[j] = q.pages[a.page_shift >= 0 ? key >> a.page_shift : key / a.page];
        }
    };
    // rows of tile t from them (-1: none, past the range or on a page that is not in the cache)
    auto find_rows = [&](int t) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int key = ks + t * KB + sr + j * RS;
            if (a.table) {
                const int in = a.page_shift >= 0 ? key & (a.page - 1) : key % a.page;
                row[j] = key < ke && pg[j] >= 0 && pg[j] < a.cache_pages ? pg[j] * a.page + in : -1;
            } else {
                row[j] = key < ke ? (int)q.row0 + key : -1;
            }
        }
    };
    auto load = [&]() {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int64_t at = (int64_t)max(row[j], 0) * a.kv_stride;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                bk[j][c] = ldf4(kbase + at + 4 * c);
                bv[j][c] = ldf4(vbase + at + 4 * c);
            }
        }
    };
    Terms tk[NC], tv[NC];
    uint32_t gap = 0, bad = 0;  // of the thread's keys
    bool wild = false;
    auto wild4 = [](const f32x4& v) {
        return !(fabsf(v[0]) < INFINITY) || !(fabsf(v[1]) < INFINITY) || !(fabsf(v[2]) < INFINITY) || !(fabsf(v[3]) < INFINITY);
    };
    auto tame = [](f32x4& v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fabsf(v[e]) < INFINITY ? v[e] : 0.0f;
    };
    auto terms = [&]() {  // of the loaded tile
        gap = bad = 0;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const uint32_t bit = 1u << ((sr + j * RS) & 31);
            const bool none = row[j] < 0, kw = wild4(bk[j][0]) || wild4(bk[j][1]), vw = wild4(bv[j][0]) || wild4(bv[j][1]);
            if (__any(none || kw || vw)) {
                if (none) {
                    gap |= bit;
                    bk[j][0] = bk[j][1] = bv[j][0] = bv[j][1] = f32x4{};
                }
                if (kw && !none) bad |= bit;
                wild |= vw && !none;
                tame(bk[j][0]);
                tame(bk[j][1]);
                tame(bv[j][0]);
                tame(bv[j][1]);
            }
            tk[j] = split8(bk[j][0], bk[j][1]);
            tv[j] = split8(bv[j][0], bv[j][1]);
        }
    };
    auto store = [&](int t) {
        if (!mine) return;
        if (__any((gap | bad) != 0 || wild)) {
            if (gap) atomicOr(&s_gap[t & 1], gap);
            if (bad) atomicOr(&s_bad[t & 1], bad);
            if (wild) s_wild = 1;
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            *reinterpret_cast<u32x4*>(&s_k[0][kst + j * RS * KS]) = tk[j].h;
            *reinterpret_cast<u32x4*>(&s_k[1][kst + j * RS * KS]) = tk[j].m;
            *reinterpret_cast<u32x4*>(&s_k[2][kst + j * RS * KS]) = tk[j].l;
            *reinterpret_cast<u32x4*>(&s_v[0][vst + j * RS * VS]) = tv[j].h;
            *reinterpret_cast<u32x4*>(&s_v[1][vst + j * RS * VS]) = tv[j].m;
            *reinterpret_cast<u32x4*>(&s_v[2][vst + j * RS * VS]) = tv[j].l;
        }
    };

    const int li = lane & 15, ka = n * KS + KP * h, va = (4 * h + (li >> 2)) * VS + 8 * (li & 3);
    float x[8];  // scores of a tile, then their weights: keys 16 z + 4 h + r
    auto scores = [&]() {
        acc4 big[2], small[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) big[z] = small[z] = acc4{};
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const bf16x8 qh = op(qt[j].h), qm = op(qt[j].m), ql = op(qt[j].l);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int at = ka + z * 16 * KS + j * 16;
                const bf16x8 kh = *reinterpret_cast<const bf16x8*>(&s_k[0][at]), km = *reinterpret_cast<const bf16x8*>(&s_k[1][at]),
                             kl = *reinterpret_cast<const bf16x8*>(&s_k[2][at]);
                small[z] = mfma(kl, qh, small[z]);
                big[z] = mfma(kh, qh, big[z]);
                small[z] = mfma(kh, ql, small[z]);
                small[z] = mfma(km, qm, small[z]);
                small[z] = mfma(km, qh, small[z]);
                small[z] = mfma(kh, qm, small[z]);
            }
        }
        // (the reads run ahead of the products)
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int z = 0; z < 2 * NQ - 1; ++z) {
            __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = big[e / 4][e % 4] + small[e / 4][e % 4];
    };
    auto weights = [&](int t) {
        const int k0 = ks + t * KB;
        const uint32_t none = __builtin_amdgcn_readfirstlane(s_gap[t & 1]);
        uint32_t odd = __builtin_amdgcn_readfirstlane(s_bad[t & 1]);
        while (odd) {  // (uniform)
            const int k = __builtin_ctz(odd);
            odd &= odd - 1;
            const float* const kp = (const float*)a.kc + (int64_t)max(row_of(a, q, k0 + k), 0) * a.kv_stride + kvh * D;
            float s = 0.0f;
#pragma unroll 1
            for (int d = 0; d < D; ++d) s = fmaf(qrow[d], kp[d], s);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = k == e / 4 * 16 + 4 * h + e % 4 ? s : x[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] *= a.scale;
            if constexpr (CAP) x[e] = a.softcap * tanh_fast(div_by_uniform(x[e], a.softcap, a.inv_cap));
        }
        if (none || !(whole && k0 >= all_lo && k0 + KB - 1 <= all_hi)) {  // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int kk = e / 4 * 16 + 4 * h + e % 4, key = k0 + kk;
                x[e] = key >= lo && key <= hi && !(none >> kk & 1) ? x[e] : -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
        mx = over_row4(mx, [](float u, float v) { return fmaxf(u, v); });
        if (__any(!((mx - m) * a.unit <= kSlack))) {
            const float mn = fmaxf(m, mx);
            const float c = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * a.unit);
            m = mn;
            l *= c;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] *= c;
        }
        const float ms = m == -INFINITY ? 0.0f : m;
        float ps = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f((x[e] - ms) * a.unit);
            ps += x[e];
        }
        l += ps;
    };
    auto output = [&]() {
        const Terms pt = split8(f32x4{x[0], x[1], x[2], x[3]}, f32x4{x[4], x[5], x[6], x[7]});
        const bf16x8 ph = op(pt.h), pm = op(pt.m), pl3 = op(pt.l);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            bf16x8 v[3];
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(&s_v[u][va + b * 32]));
                const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(&s_v[u][va + b * 32 + 16 * VS]));
                v[u] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
            }
            o[b] = mfma(v[2], ph, o[b]);
            o[b] = mfma(v[0], pl3, o[b]);
            o[b] = mfma(v[1], pm, o[b]);
            o[b] = mfma(v[1], ph, o[b]);
            o[b] = mfma(v[0], pm, o[b]);
            o[b] = mfma(v[0], ph, o[b]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
#pragma unroll
        for (int b = 0; b < NB - 1; ++b) {
            __builtin_amdgcn_sched_group_barrier(0x008, 6, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 6, 1);
    };

    if (tid == 0) s_wild = 0;
    if (tid < 2) s_gap[tid] = s_bad[tid] = 0;
    __syncthreads();
    if (ntile > 0) {  // (uniform)
        find_pages(0);
        find_rows(0);
        load();
        find_pages(1);
        terms();
        store(0);
        find_rows(1);
        load();
        find_pages(2);
        __syncthreads();
        for (int t = 0; t < ntile; ++t) {
            if (tid == 0) s_gap[(t + 1) & 1] = s_bad[(t + 1) & 1] = 0;
            if (ks + t * KB <= any_hi && ks + t * KB + KB > any_lo) {  // (uniform: some row of the wave sees some key)
                scores();
                weights(t);
                output();
            }
            // (past the last tile row 0 of the cache is loaded and split: no load under a branch)
            terms();
            __syncthreads();
            if (t + 1 < ntile) store(t + 1);
            find_rows(t + 2);
            load();
            find_pages(t + 3);
            __syncthreads();
        }
    }

    l = over_row4(l, [](float u, float v) { return u + v; });
    if (w0 + n > r1) return;
    if (s_wild) {
        // What a row sees of the values kept out: whatever its weight, the value itself.
#pragma unroll 1
        for (int k = ks; k < ke; ++k) {
            const int r = row_of(a, q, k);
            if (r < 0 || k < lo || k > hi) continue;
            const float* const vp = (const float*)a.vc + (int64_t)r * a.kv_stride + kvh * D + 4 * h;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f32x4 v = ldf4(vp + 16 * b);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[b][e] += fabsf(v[e]) < INFINITY ? 0.0f : v[e];
            }
        }
    }
    const int64_t th = (int64_t)(q.tok0 + i) * a.nh + kvh * a.gq + rr % a.gq;
    if (rg.used == 1) {
        float* const out = (float*)a.out + th * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = l == 0.0f ? 0.0f : o[b][e] / l;  // (no key: zeros)
            st4(out + 16 * b, v);
        }
    } else {
        const int64_t part = th * a.nparts + split;
        float* const w = a.ws + part * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b) st4(w + 16 * b, f32x4{o[b][0], o[b][1], o[b][2], o[b][3]});
        if (h == 0) {
            float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
            ml[0] = m;
            ml[1] = l;
        }
    }
}

template <int D, bool CAP>
__global__ __launch_bounds__(kTermWaves * kWave, 2) void k_seq_terms(SeqArgs a) {
    __shared__ __align__(16) TermsLds<D> lds;
    seq_terms<D, CAP>(a, (int)blockIdx.x, lds);
}
// (as k_seq_both of the bf16 tiles)
template <int D, bool CAP>
__global__ __launch_bounds__(kTermWaves * kWave, 2) void k_seq_terms_both(SeqArgs a) {
    __shared__ __align__(16) union Lds {
        TermsLds<D> tile;
        RowsLds<D, kTermWaves> rows;
    } lds;
    const int id = (int)blockIdx.x;
    if (id < a.tile_grid) seq_terms<D, CAP>(a, id, lds.tile);
    else seq_rows<float, D, kTermWaves>(a, id - a.tile_grid, lds.rows);
}

template <int D>
static void launch(const SeqArgs& a, hipStream_t s) {
    const unsigned grid = (unsigned)(a.tile_grid + a.rows_grid);
    auto run = [&](auto cap) {
        constexpr bool CAP = decltype(cap)::value;
        if (a.rows_grid > 0) k_seq_terms_both<D, CAP><<<grid, kTermWaves * kWave, 0, s>>>(a);
        else k_seq_terms<D, CAP><<<grid, kTermWaves * kWave, 0, s>>>(a);
    };
    if (a.softcap > 0.0f) run(std::true_type{});
    else run(std::false_type{});
}

void launch_terms(const SeqArgs& a, hipStream_t s) {
    if (a.D == 64) launch<64>(a, s);
    else if (a.D == 128) launch<128>(a, s);
    else launch<256>(a, s);
}

}  // namespace zl
