// Attention of many sequences, tiles of many query rows on the bf16 matrix cores (attention_seqs.hip has
// the definition and the host side).
//
// A workgroup takes NW * M query rows of one kv head of a sequence (row = token * heads of the group +
// head, so that the heads of a group share the keys), each wave M of them, and goes over the keys
// in tiles of KB that all its waves read from LDS: one pass, with the running maximum and sum of the
// softmax in f32. Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane
// holds one query row (n = lane % M) throughout: the row's maximum, sum and rescaling factor are
// registers of its own lanes, and its weights are the operand of the second product as they stand. Of a
// tile's scores the lane (n, h = lane / M) holds keys u * 256 / M + 4 h + {0..3}, u = 0, 1, ..: groups
// of four keys, which is also what a transposing LDS read (ds_read_b64_tr_b16: lane i of 16 gets column i
// of four rows) gives of V, row-major as it is in the cache. The two products order their keys alike.
// K and V of the next tile are on their way
// to registers while a tile is computed, and go to the other LDS buffer behind it: one barrier a tile.
// The weights round to bf16 for the second product (half a step, 2^-8 relative, as the output does); their
// sum takes them unrounded. The running maximum moves only when a row exceeds it by 8 in the exponent
// (weights up to 2^8 before the final quotient), so that tiles seldom rescale the output.
// Heads of 64 and 128 are bound by the softmax's vector instructions beside the MFMAs (a prompt of 8192, 32 / 16
// heads x 128: 562 us, 978 TFLOP/s, matrix cores 38% and vector units 46% busy; 4096: 154 us), heads of 256
// and 512 by LDS, whose rows 16-row waves read for half the products (4096, 8 / 4 x 256: 166 us, 414 TFLOP/s; 2048,
// 8 / 1 x 512: 136 us). 32 rows a wave do not fit at 256 (five prompts, 4099 tokens, window 512: 61 us against 38.7).
#include "attention_rows.h"

namespace zl {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

template <int M> struct Mfma;
template <> struct Mfma<32> {
    typedef f32x16 Acc;
    __device__ static __forceinline__ Acc run(const bf16x8& a, const bf16x8& b, const Acc& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Mfma<16> {
    typedef acc4 Acc;
    __device__ static __forceinline__ Acc run(const bf16x8& a, const bf16x8& b, const Acc& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// Of the lanes of a query row (lane % M), the maximum and the sum.
template <int M, typename F>
__device__ __forceinline__ float over_row(float v, F f) {
    if constexpr (M == 16) {
        const unsigned x = __builtin_bit_cast(unsigned, v), y = __builtin_bit_cast(unsigned, dpp<0xE4>(v));
        const auto p = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        v = f(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
    }
    const unsigned x = __builtin_bit_cast(unsigned, v), y = __builtin_bit_cast(unsigned, dpp<0xE4>(v));
    const auto p = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return f(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
}

// LDS is laid out so that no two lanes of a phase meet in a bank (a phase of a 16-byte read has 16 lanes: 0-3,
// 12-15, 20-27 or 4-11, 16-19, 28-31 of a half wave; of an 8-byte read 32). K: M 32 reads 16 rows at one
// column in a phase, rows are padded by 16 bytes; M 16 reads 8 rows at one chunk and the others at the
// next, so the chunks stand in four planes by their index mod 4, rows padded to an odd number of chunks.
// V: a transposing read has 4 rows and 32 bytes a group of 16 lanes, and in the other group the next 32
// bytes (M 32: rows padded by 64 bytes) or the next rows (M 16: by 32).
template <typename T, int D, int M, int NW, int KB, int HV>
struct TileLds {
    static constexpr bool BF = sizeof(T) == 2;
    static constexpr int RB = D * sizeof(T);  // bytes of a row
    static constexpr int PLANES = M == 32 ? 1 : 4;
    static constexpr int KS = RB / PLANES + 16, KP = KB * KS, VS = RB + (!BF ? 0 : M == 32 ? 64 : 32);
    static_assert(M == 32 || (KP % 256 == 0 && KS / 16 % 2 == 1), "planes");
    static constexpr int GW = (KB + 31) / 32, NU = KB / M * (M * M / 64) / 4;
    uint8_t k[2][PLANES * KP], v[2][KB * VS];
    f32x4 x[HV > 1 ? NW : 1][HV > 1 ? NU : 1][HV > 1 ? kWave : 1];  // the halves' sums of the scores
    uint32_t gap[3][GW];                  // keys without a row
    int wild;                             // infinite or NaN values were kept out of LDS
};
template <typename T, int D, int M, int NW, int KB, int HV, bool CAP>
__device__ __forceinline__ void seq_tile(const SeqArgs& a, int id, TileLds<T, D, M, NW, KB, HV>& lds) {
    typedef typename Mfma<M>::Acc Acc;
    constexpr bool BF = sizeof(T) == 2;
    static_assert(BF || M == 16, "f32 tiles have 16 rows a wave");
    constexpr int EL = 16 / sizeof(T);   // elements of a 16-byte chunk
    constexpr int G = 64 / M;            // lanes of a query row
    constexpr int DW = D / HV;           // of the head size, a wave's part
    constexpr int RG = NW / HV;          // groups of M query rows
    constexpr int NQ = DW / (EL * G);    // chunks of a query row to a lane
    constexpr int NT = KB / M;           // score tiles
    constexpr int SR = M * M / 64;       // registers of one
    constexpr int NU = NT * SR / 4;      // groups of four keys of a lane
    constexpr int US = 256 / M;          // keys between them
    constexpr int NB = DW / M;           // accumulators of the output
    constexpr int TH = NW * kWave;
    constexpr int CR = D / EL;           // chunks of a row
    constexpr int NC = KB * CR / TH;     // of a tile, to a thread
    constexpr int RS = TH / CR;          // rows between a thread's chunks
    constexpr float kSlack = 8.0f;       // log2
    static_assert(KB * CR % TH == 0 && TH % CR == 0, "chunks of a tile");
    typedef TileLds<T, D, M, NW, KB, HV> Lds;
    constexpr int PLANES = Lds::PLANES, KS = Lds::KS, KP = Lds::KP, VS = Lds::VS, GW = Lds::GW;
    auto& s_k = lds.k;
    auto& s_v = lds.v;
    auto& s_gap = lds.gap;
    auto& s_x = lds.x;
    int& s_wild = lds.wild;
    const int tid = threadIdx.x, lane = tid & 63, n = lane % M, h = lane / M;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = wave / RG;
    const int kvh = id % a.nkv;
    id /= a.nkv;
    const int split = id % a.tile_split;
    int tile;
    const int sq = __builtin_amdgcn_readfirstlane(find_tile<RG * M, false>(a, id / a.tile_split, tile));
    if (sq < 0) return;
    const Seq q = seq_of(a, sq);
    const int rows = q.nq * a.gq;
    // the last tiles, whose ranges are the longest, first
    const int r0 = ((rows + RG * M - 1) / (RG * M) - 1 - __builtin_amdgcn_readfirstlane(tile)) * (RG * M);
    if (r0 < 0 || r0 >= rows) return;
    const int r1 = min(r0 + RG * M, rows) - 1;
    const Range rg = tile_range(a, q, r0, r1, a.tile_chunk);
    if (split >= rg.used) return;
    const int ks = rg.ks + split * a.tile_chunk, ke = rg.ke - ks > a.tile_chunk ? ks + a.tile_chunk : rg.ke;
    const int ntile = ke > ks ? (ke - ks + KB - 1) / KB : 0;

    // the lane's query row and its keys [lo, hi], and what all of the wave's rows see
    const int w0 = r0 + wave % RG * M, w1 = min(w0 + M - 1, r1);
    const int rr = min(w0 + n, r1), i = rr / a.gq, p = q.pos0 + i;
    const int hi = p >= 0 && p < q.lim ? p : -1;  // (rows behind the last are the last once more)
    const int lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
    const int pf = q.pos0 + w0 / a.gq, pl = q.pos0 + max(w1, 0) / a.gq;
    const bool whole = pf >= 0 && pl < q.lim;
    const int any_lo = a.window > 0 ? max(0, pf + 1 - a.window) : 0, all_lo = a.window > 0 ? max(0, pl + 1 - a.window) : 0;
    const int any_hi = w0 <= r1 ? min(pl, q.lim - 1) : -1, all_hi = pf;
    // and of the workgroup's: tiles outside have keys that some rows do not see
    const int wg_lo = a.window > 0 ? max(0, q.pos0 + r1 / a.gq + 1 - a.window) : 0, wg_hi = q.pos0 + r0 / a.gq;

    u32x4 qv[NQ];
    {
        const T* qrow = (const T*)a.q + (int64_t)(q.tok0 + i) * a.q_stride + (kvh * a.gq + rr % a.gq) * D + half * DW + EL * h;
        const uint32_t flip = BF && !CAP && a.scale < 0.0f ? 0x80008000u : 0u;  // `unit` has no sign
#pragma unroll
        for (int j = 0; j < NQ; ++j) qv[j] = ld16(qrow + EL * G * j) ^ flip;
    }
    Acc o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = Acc{};
    float m = -INFINITY, l = 0.0f;

    // ---- the tiles' way to LDS ----
    const int sr = tid / CR, sc = tid % CR;  // the thread's first row and its chunk of a row
    const int kc = sc % (CR / PLANES) * PLANES + sc / (CR / PLANES);  // its chunk of K
    const int kst = sr * KS + kc % PLANES * KP + kc / PLANES * 16;
    const T* const kbase = (const T*)a.kc + kvh * D + EL * kc;
    const T* const vbase = (const T*)a.vc + kvh * D + EL * sc;
    u32x4 bk[NC], bv[NC];
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
            bk[j] = ld16(kbase + at);
            bv[j] = ld16(vbase + at);
        }
    };
    auto store = [&](int t) {
        const int k0 = ks + t * KB;
        bool none = false;
#pragma unroll
        for (int j = 0; j < NC; ++j) none |= row[j] < 0;
        if (__any(none)) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int r = sr + j * RS;
                if (row[j] < 0) bv[j] = u32x4{};
                if (row[j] < 0 && sc == 0) atomicOr(&s_gap[t % 3][r / 32], 1u << (r % 32));
            }
        }
        if (k0 < wg_lo || k0 + KB - 1 > wg_hi) {
            // Some rows do not see all of the tile's keys: infinite and NaN values, which weights of 0 would
            // carry to them, stay out of LDS, and go to the rows that see them at the end.
            auto low = [](uint32_t w) { return BF && (w & 0x7f80u) == 0x7f80u; };
            auto high = [](uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; };
            bool bad = false;
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= low(bv[j][e]) || high(bv[j][e]);
            if (__any(bad)) {
                if (lane == 0) s_wild = 1;
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t w = bv[j][e];
                        bv[j][e] = high(w) ? (BF && !low(w) ? w & 0xffffu : 0u) : low(w) ? w & 0xffff0000u : w;
                    }
            }
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int r = sr + j * RS;
            *reinterpret_cast<u32x4*>(&s_k[t & 1][kst + j * RS * KS]) = bk[j];
            *reinterpret_cast<u32x4*>(&s_v[t & 1][r * VS + 16 * sc]) = bv[j];
        }
    };
    // Behind tile t: tile t + 1 goes to LDS, the next one's loads out. (Past the last tile row 0 of the cache is
    // loaded: no load under a branch.)
    auto stage = [&](int t) {
        if (t + 1 < ntile) store(t + 1);
        find_rows(t + 2);
        load();
        find_pages(t + 3);
    };

    // The lane's LDS addresses: K, chunk j G + h of row z M + n; V, chunk b M / 8 + .. of row u US + 4 h + li / 4
    // (f32: chunk 16 c + n of row u US + 4 h + r).
    const int li = lane & 15, at_half = half * DW * (int)sizeof(T);
    const int ka = at_half / PLANES + n * KS + (M == 32 ? 16 : KP) * h;
    const int va = at_half + (BF ? (4 * h + (li >> 2)) * VS + (M == 32 ? 32 * (lane >> 4 & 1) : 0) + 8 * (li & 3) : 4 * h * VS + 16 * n);

    float x[NT * SR];          // scores of a tile, then (f32) their weights
    u32x4 pw[BF ? NU / 2 : 1]; // the weights as operands
    auto scores = [&](int t) {
        const uint8_t* const kb = &s_k[t & 1][ka];
        if constexpr (BF) {
            Acc s[NT];
#pragma unroll
            for (int z = 0; z < NT; ++z) s[z] = Acc{};
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int z = 0; z < NT; ++z) {
                    const bf16x8 kv = *reinterpret_cast<const bf16x8*>(kb + z * M * KS + j * G * 16 / PLANES);
                    s[z] = Mfma<M>::run(kv, __builtin_bit_cast(bf16x8, qv[j]), s[z]);
                }
            // (the reads run ahead of the products)
            constexpr int AHEAD = NQ * NT < 6 ? NQ * NT : 6;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int z = 0; z < NQ * NT - AHEAD; ++z) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) x[e] = s[e / SR][e % SR];
        } else {
            // 16 products at a time into a fresh accumulator, these summed in two chains (one chain is two to
            // three times as far from the exact dot product)
            acc4 s[NT][2];
#pragma unroll
            for (int z = 0; z < NT; ++z) s[z][0] = s[z][1] = acc4{};
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int z = 0; z < NT; ++z) {
                    const f32x4 kv = *reinterpret_cast<const f32x4*>(kb + z * M * KS + j * G * 16 / PLANES);
                    const f32x4 qf = __builtin_bit_cast(f32x4, qv[j]);
                    acc4 c = acc4{};
#pragma unroll
                    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], qf[e], c, 0, 0, 0);
                    s[z][j & 1] += c;
                }
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) x[e] = s[e / SR][0][e % SR] + s[e / SR][1][e % SR];
        }
    };
    auto weights = [&](int t) {
        const int k0 = ks + t * KB;
        if constexpr (HV > 1) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const f32x4 y = s_x[(wave + RG) % NW][u][lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * u + e] += y[e];
            }
        }
#pragma unroll
        for (int e = 0; e < NT * SR; ++e) {
            if constexpr (!BF) x[e] *= a.scale;
            if constexpr (CAP && !BF) x[e] = a.softcap * tanh_fast(div_by_uniform(x[e], a.softcap, a.inv_cap));
        }
        if constexpr (CAP && BF) {
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) top = fmaxf(top, fabsf(x[e]));
            if (__any(!(top <= a.cap_small))) {
#pragma unroll
                for (int e = 0; e < NT * SR; ++e) x[e] = cap_bf16(a, x[e]);
            } else {
#pragma unroll
                for (int e = 0; e < NT * SR; ++e) x[e] = cap_series(a, x[e]);
            }
        }
        uint32_t gap[GW], some = 0;
#pragma unroll
        for (int e = 0; e < GW; ++e) some |= gap[e] = s_gap[t % 3][e];
        some = __builtin_amdgcn_readfirstlane(some);
        if (some || !(whole && k0 >= all_lo && k0 + KB - 1 <= all_hi)) {  // uniform
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) {
                const int kk = e / 4 * US + 4 * h + e % 4, key = k0 + kk;
                const bool there = !(gap[e / 4 * US / 32] >> (kk % 32) & 1);
                x[e] = key >= lo && key <= hi && there ? x[e] : -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < NT * SR; ++e) mx = fmaxf(mx, x[e]);
        mx = over_row<M>(mx, [](float u, float v) { return fmaxf(u, v); });
        if (__any(!((mx - m) * a.unit <= kSlack))) {
            const float mn = fmaxf(m, mx);
            const float c = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * a.unit);
            m = mn;
            l *= c;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] *= c;
        }
        const float ms = m == -INFINITY ? 0.0f : m, mu = ms * a.unit;
        float ps = 0.0f;
#pragma unroll
        for (int e = 0; e < NT * SR; ++e) {
            // (f32: the difference first, which is nearly exact where it counts)
            x[e] = __builtin_amdgcn_exp2f(BF ? fmaf(x[e], a.unit, -mu) : (x[e] - ms) * a.unit);
            ps += x[e];
        }
        l += ps;
        if constexpr (BF) {
#pragma unroll
            for (int u = 0; u < NU / 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) pw[u][e] = pack_bf16x2(x[8 * u + 2 * e], x[8 * u + 2 * e + 1]);
        }
    };
    auto output = [&](int t) {
        if constexpr (BF) {
            // an MFMA takes key groups u and u + 1
            const uint8_t* const vb = &s_v[t & 1][va];
#pragma unroll
            for (int u = 0; u < NU; u += 2) {
                const bf16x8 pv = __builtin_bit_cast(bf16x8, pw[u / 2]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint8_t* const at = vb + b * M * 2;
                    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + u * US * VS));
                    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + (u + 1) * US * VS));
                    const bf16x8 vv = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[b] = Mfma<M>::run(vv, pv, o[b]);
                }
            }
            constexpr int ALL = NU / 2 * NB, AHEAD = ALL < 4 ? ALL : 4;
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * AHEAD, 1);
#pragma unroll
            for (int z = 0; z < ALL - AHEAD; ++z) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 1);
        } else {
            // accumulator 4 c + j takes column 64 c + 4 n + j of V, an MFMA keys u US + 4 h + r
            const uint8_t* const vb = &s_v[t & 1][va];
#pragma unroll
            for (int e = 0; e < NT * SR; ++e)
#pragma unroll
                for (int c = 0; c < NB / 4; ++c) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(vb + (e / 4 * US + e % 4) * VS + c * 256);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[4 * c + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j], x[e], o[4 * c + j], 0, 0, 0);
                }
        }
    };
    if (tid == 0) s_wild = 0;
    if (tid < 3) {
#pragma unroll
        for (int e = 0; e < GW; ++e) s_gap[tid][e] = 0;
    }
    __syncthreads();
    if (ntile > 0) {  // (uniform)
        find_pages(0);
        find_rows(0);
        load();
        find_pages(1);
        store(0);
        find_rows(1);
        load();
        find_pages(2);
        __syncthreads();
        for (int t = 0; t < ntile; ++t) {
            if (tid == 0) {  // the flags that tile t - 1 had are tile t + 2's
#pragma unroll
                for (int e = 0; e < GW; ++e) s_gap[(t + 2) % 3][e] = 0;
            }
            const bool some = ks + t * KB <= any_hi && ks + t * KB + KB > any_lo;  // (uniform: some row of the wave sees some key)
            if (some) scores(t);
            if constexpr (HV > 1) {
                if (some) {
#pragma unroll
                    for (int u = 0; u < NU; ++u) s_x[wave][u][lane] = f32x4{x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]};
                }
                __syncthreads();
            }
            if (some) {
                weights(t);
                output(t);
            }
            stage(t);
            __syncthreads();
        }
    }

    l = over_row<M>(l, [](float u, float v) { return u + v; });
    if (w0 + n > r1) return;
    // f(column, the lane's four outputs from it on) -> the four
    auto each4 = [&](auto f) {
#pragma unroll
        for (int b = 0; b < NB; b += BF ? 1 : 4)
#pragma unroll
            for (int e = 0; e < SR; e += BF ? 4 : 1) {
                if constexpr (BF) {
                    const f32x4 v = f(half * DW + b * M + 2 * e + 4 * h, f32x4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]});
#pragma unroll
                    for (int z = 0; z < 4; ++z) o[b][e + z] = v[z];
                } else {
                    const f32x4 v = f(half * DW + 16 * b + 16 * h + 4 * e, f32x4{o[b][e], o[b + 1][e], o[b + 2][e], o[b + 3][e]});
#pragma unroll
                    for (int z = 0; z < 4; ++z) o[b + z][e] = v[z];
                }
            }
    };
    if (s_wild) {
        // What a row sees of the values kept out: whatever its weight, the value itself.
#pragma unroll 1
        for (int k = ks; k < ke; ++k) {
            const int k0 = ks + (k - ks) / KB * KB;
            if (k0 >= wg_lo && k0 + KB - 1 <= wg_hi) continue;  // (uniform: the tile went whole)
            const int r = row_of(a, q, k);
            if (r < 0 || k < lo || k > hi) continue;
            const T* const vp = (const T*)a.vc + (int64_t)r * a.kv_stride + kvh * D;
            each4([&](int col, f32x4 v) {
                const f32x4 w = ld4(vp + col);
#pragma unroll
                for (int z = 0; z < 4; ++z) v[z] += fabsf(w[z]) < INFINITY ? 0.0f : w[z];
                return v;
            });
        }
    }
    if (l == 0.0f) {  // no key: zeros, whatever weights of 0 made of the values
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = Acc{};
        l = 1.0f;
    }
    const int64_t th = (int64_t)(q.tok0 + i) * a.nh + kvh * a.gq + rr % a.gq;
    if (rg.used == 1) {
        T* const out = (T*)a.out + th * D;
        const float inv = 1.0f / l;
        each4([&](int col, f32x4 v) {
#pragma unroll
            for (int z = 0; z < 4; ++z) v[z] = BF ? v[z] * inv : v[z] / l;
            st4(out + col, v);
            return v;
        });
    } else {
        const int64_t part = th * a.nparts + split;
        float* const w = a.ws + part * D;
        each4([&](int col, f32x4 v) {
            st4(w + col, v);
            return v;
        });
        if (h == 0 && half == 0) {
            float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
            ml[0] = m;
            ml[1] = l;
        }
    }
}

template <typename T, int D, int M, int NW, int KB, int HV, bool CAP>
__global__ __launch_bounds__(NW * kWave, 2) void k_seq_tile(SeqArgs a) {
    __shared__ __align__(16) TileLds<T, D, M, NW, KB, HV> lds;
    seq_tile<T, D, M, NW, KB, HV, CAP>(a, (int)blockIdx.x, lds);
}
// Tiles, and behind them 16 rows by as many waves: chunks beside sequences of a token. The rows, which wait for
// memory, take the CUs that the last tiles leave (24 sequences, three of them chunks of 288 to 492 tokens behind
// up to 3600, 32 / 16 heads x 128: 187 us in two launches one behind the other, 149 in one).
template <typename T, int D, int M, int NW, int KB, int HV, bool CAP>
__global__ __launch_bounds__(NW * kWave, 2) void k_seq_both(SeqArgs a) {
    constexpr int W = NW / row_halves<D>();
    __shared__ __align__(16) union Lds {
        TileLds<T, D, M, NW, KB, HV> tile;
        RowsLds<D, W> rows;
    } lds;
    const int id = (int)blockIdx.x;
    if (id < a.tile_grid) seq_tile<T, D, M, NW, KB, HV, CAP>(a, id, lds.tile);
    else seq_rows<T, D, W>(a, id - a.tile_grid, lds.rows);
}

template <typename T, int D, int M, int NW, int KB, int HV = 1>
static void launch(const SeqArgs& a, hipStream_t s) {
    const unsigned grid = (unsigned)(a.tile_grid + a.rows_grid);
    auto run = [&](auto cap) {
        constexpr bool CAP = decltype(cap)::value;
        // (rows stand beside the smaller tiles, where there are two sizes)
        if constexpr (NW == 4 || HV > 1) {
            if (a.rows_grid > 0) return k_seq_both<T, D, M, NW, KB, HV, CAP><<<grid, NW * kWave, 0, s>>>(a);
        }
        k_seq_tile<T, D, M, NW, KB, HV, CAP><<<grid, NW * kWave, 0, s>>>(a);
    };
    if (a.softcap > 0.0f) run(std::true_type{});
    else run(std::false_type{});
}

int tile_rows_of(int dtype, int D, bool small) {
    if (dtype == HIP_BRIDGE_F32 && D < 512) return 128;
    if (D == 512) return 64;
    return D <= 128 ? (small ? 128 : 256) : small ? 64 : 128;
}

void launch_tiles(int dtype, const SeqArgs& a, hipStream_t s) {
    const bool small = a.tile_rows < tile_rows_of(dtype, a.D, false);
    if (dtype == HIP_BRIDGE_F32) {
        if (a.D < 512) launch_terms(a, s);
        else launch<float, 512, 16, 8, 16, 2>(a, s);
    } else if (a.D == 512) {
        launch<uint16_t, 512, 16, 8, 32, 2>(a, s);
    } else if (small) {
        if (a.D == 64) launch<uint16_t, 64, 32, 4, 64>(a, s);
        else if (a.D == 128) launch<uint16_t, 128, 32, 4, 64>(a, s);
        else launch<uint16_t, 256, 16, 4, 32>(a, s);
    } else {
        if (a.D == 64) launch<uint16_t, 64, 32, 8, 64>(a, s);
        else if (a.D == 128) launch<uint16_t, 128, 32, 8, 64>(a, s);
        else launch<uint16_t, 256, 16, 8, 32>(a, s);
    }
}

}  // namespace zl
