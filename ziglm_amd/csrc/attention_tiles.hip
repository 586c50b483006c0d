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
// LDS rows are swizzled by 16-byte chunks, K's by row % 8 (16-byte reads of 8 rows at one column), V's
// by 2 (row % 4) (4 rows by 32 bytes of a transposing read). K and V of the next tile are on their way
// to registers while a tile is computed, and go to the other LDS buffer behind it: one barrier a tile.
// The weights round to bf16 for the second product (half a step, 2^-8 relative, as the output does); their
// sum takes them unrounded. The running maximum moves only when a row exceeds it by 8 in the exponent
// (weights up to 2^8 before the final quotient), so that tiles seldom rescale the output.
#include "attention_seqs.h"

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

template <int D, int M, int NW, int KB, int WPE, bool CAP>
__global__ __launch_bounds__(NW * kWave, WPE) void k_seq_tile(SeqArgs a) {
    typedef typename Mfma<M>::Acc Acc;
    constexpr int G = 64 / M;            // lanes of a query row
    constexpr int KD = 8 * G;            // depth of an MFMA
    constexpr int NQ = D / KD;           // operands of a query row
    constexpr int NT = KB / M;           // score tiles
    constexpr int SR = M * M / 64;       // registers of one
    constexpr int NU = NT * SR / 4;      // groups of four keys of a lane
    constexpr int US = 256 / M;          // keys between them
    constexpr int NB = D / M;            // column blocks of the output
    constexpr int TH = NW * kWave;
    constexpr int CR = D / 8;            // 16-byte chunks of a row
    constexpr int NC = KB * CR / TH;     // of a tile, to a thread
    constexpr int RS = TH / CR;          // rows between a thread's chunks
    constexpr float kSlack = 8.0f;       // log2
    static_assert(KB * CR % TH == 0 && TH % CR == 0 && RS % 8 == 0, "chunks of a tile");
    constexpr int TB = KB * D * 2;       // bytes of a tile of K or V
    __shared__ __align__(16) uint8_t s_kv[2][2][TB];  // [buffer][K, V]
    __shared__ uint32_t s_gap[3][KB / 32];  // keys without a row
    __shared__ int s_wild;                  // infinite or NaN values were kept out of LDS
    const int tid = threadIdx.x, lane = tid & 63, n = lane % M, h = lane / M;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = (int)blockIdx.x;
    const int kvh = id % a.nkv;
    id /= a.nkv;
    const int split = id % a.tile_split;
    int tile;
    const int sq = __builtin_amdgcn_readfirstlane(find_tile<NW * M, false>(a, id / a.tile_split, tile));
    if (sq < 0) return;
    const Seq q = seq_of(a, sq);
    const int rows = q.nq * a.gq;
    // the last tiles, whose ranges are the longest, first
    const int r0 = ((rows + NW * M - 1) / (NW * M) - 1 - __builtin_amdgcn_readfirstlane(tile)) * (NW * M);
    if (r0 < 0 || r0 >= rows) return;
    const int r1 = min(r0 + NW * M, rows) - 1;
    const Range rg = tile_range(a, q, r0, r1, a.tile_chunk);
    if (split >= rg.used) return;
    const int ks = rg.ks + split * a.tile_chunk, ke = rg.ke - ks > a.tile_chunk ? ks + a.tile_chunk : rg.ke;
    const int ntile = ke > ks ? (ke - ks + KB - 1) / KB : 0;

    // the lane's query row and its keys [lo, hi], and what all of the wave's rows see
    const int w0 = r0 + wave * M, w1 = min(w0 + M - 1, r1);
    const int rr = min(w0 + n, r1), i = rr / a.gq, p = q.pos0 + i;
    const int hi = p >= 0 && p < q.lim ? p : -1;  // (rows behind the last are the last once more)
    const int lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
    const int pf = q.pos0 + w0 / a.gq, pl = q.pos0 + max(w1, 0) / a.gq;
    const bool whole = pf >= 0 && pl < q.lim;
    const int any_lo = a.window > 0 ? max(0, pf + 1 - a.window) : 0, all_lo = a.window > 0 ? max(0, pl + 1 - a.window) : 0;
    const int any_hi = w0 <= r1 ? min(pl, q.lim - 1) : -1, all_hi = pf;
    // and of the workgroup's: tiles outside have keys that some rows do not see
    const int wg_lo = a.window > 0 ? max(0, q.pos0 + r1 / a.gq + 1 - a.window) : 0, wg_hi = q.pos0 + r0 / a.gq;

    bf16x8 qv[NQ];
    {
        const uint16_t* qrow = (const uint16_t*)a.q + (int64_t)(q.tok0 + i) * a.q_stride + (kvh * a.gq + rr % a.gq) * D + 8 * h;
        const uint32_t flip = !CAP && a.scale < 0.0f ? 0x80008000u : 0u;  // `unit` has no sign
#pragma unroll
        for (int j = 0; j < NQ; ++j) qv[j] = __builtin_bit_cast(bf16x8, ld16(qrow + KD * j) ^ flip);
    }
    Acc o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = Acc{};
    float m = -INFINITY, l = 0.0f;

    // ---- the tiles' way to LDS ----
    const int sr = tid / CR, sc = tid % CR;  // the thread's first row and its chunk of a row
    const uint16_t* const kbase = (const uint16_t*)a.kc + kvh * D + 8 * sc;
    const uint16_t* const vbase = (const uint16_t*)a.vc + kvh * D + 8 * sc;
    u32x4 bk[NC], bv[NC];
    int row[NC];
    // rows of tile `t` (-1: none, past the range or on a page that is not in the cache)
    auto find_rows = [&](int t) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int key = ks + t * KB + sr + j * RS;
            row[j] = row_of(a, q, min(key, ke - 1));
            if (key >= ke) row[j] = -1;
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
    // (rows: those of the tile being stored)
    auto store = [&](int t, const int (&rw)[NC]) {
        const int buf = t & 1, f = t % 3, k0 = ks + t * KB;
        bool none = false;
#pragma unroll
        for (int j = 0; j < NC; ++j) none |= rw[j] < 0;
        if (__any(none)) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                if (rw[j] < 0) {
                    bk[j] = bv[j] = u32x4{};
                    const int r = sr + j * RS;
                    if (sc == 0) atomicOr(&s_gap[f][r / 32], 1u << (r % 32));
                }
            }
        }
        if (k0 < wg_lo || k0 + KB - 1 > wg_hi) {
            // Some rows do not see all of the tile's keys: infinite and NaN values, which weights of 0 would
            // carry to them, stay out of LDS, and go to the rows that see them at the end.
            bool bad = false;
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    bad |= (bv[j][e] & 0x7f80u) == 0x7f80u || (bv[j][e] & 0x7f800000u) == 0x7f800000u;
            if (__any(bad)) {
                if (lane == 0) s_wild = 1;
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((bv[j][e] & 0x7f80u) == 0x7f80u) bv[j][e] &= 0xffff0000u;
                        if ((bv[j][e] & 0x7f800000u) == 0x7f800000u) bv[j][e] &= 0xffffu;
                    }
            }
        }
        uint8_t* const kd = &s_kv[buf][0][sr * D * 2 + ((sc ^ (sr & 7)) << 4)];
        uint8_t* const vd = &s_kv[buf][1][sr * D * 2 + ((sc ^ ((sr & 3) << 1)) << 4)];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            *reinterpret_cast<u32x4*>(kd + j * RS * D * 2) = bk[j];
            *reinterpret_cast<u32x4*>(vd + j * RS * D * 2) = bv[j];
        }
    };
    // The lane's LDS addresses: the swizzle is an exclusive or of the low three bits of a chunk's index,
    // so the operands lie at few bases and offsets that are known here. K: chunk j G + h of row T M + n;
    // V: chunk b M / 8 + vc (+ 8 bytes) of row u US + 4 h + lane % 16 / 4.
    constexpr int KBASES = 8 / G, VBASES = 64 / M;
    const int li = lane & 15;
    const int ky = h ^ (n & 7), vy = ((M == 32 ? 2 * (lane >> 4 & 1) : 0) + ((li & 3) >> 1)) ^ (li >> 2 << 1);
    const int kn = n * D * 2, vn = (4 * h + (li >> 2)) * D * 2 + (li & 1) * 8;

    if (tid == 0) s_wild = 0;
    if (tid < 3) {
#pragma unroll
        for (int e = 0; e < KB / 32; ++e) s_gap[tid][e] = 0;
    }
    __syncthreads();
    if (ntile > 0) {
        int rw[NC];
        find_rows(0);
        load();
#pragma unroll
        for (int j = 0; j < NC; ++j) rw[j] = row[j];
        if (ntile > 1) find_rows(1);
        store(0, rw);
    }
    __syncthreads();

    for (int t = 0; t < ntile; ++t) {
        const int buf = t & 1, f = t % 3, k0 = ks + t * KB;
        int rw[NC];
        if (t + 1 < ntile) {  // the next tile's loads, and the rows of the one behind it
            load();
#pragma unroll
            for (int j = 0; j < NC; ++j) rw[j] = row[j];
            if (t + 2 < ntile) find_rows(t + 2);
        }
        if (tid == 0) {  // the flags that tile t - 1 had are tile t + 2's
#pragma unroll
            for (int e = 0; e < KB / 32; ++e) s_gap[(t + 2) % 3][e] = 0;
        }
        if (k0 <= any_hi && k0 + KB > any_lo) {  // (uniform: some row of the wave sees some key)
            // scores
            const uint8_t* kb[KBASES];
#pragma unroll
            for (int c = 0; c < KBASES; ++c) kb[c] = &s_kv[buf][0][kn + ((c * G ^ ky) << 4)];
            Acc s[NT];
#pragma unroll
            for (int T = 0; T < NT; ++T) s[T] = Acc{};
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int T = 0; T < NT; ++T) {
                    const bf16x8 kv = *reinterpret_cast<const bf16x8*>(kb[j % KBASES] + T * M * D * 2 + (j / KBASES << 7));
                    s[T] = Mfma<M>::run(kv, qv[j], s[T]);
                }
            float x[NT * SR];
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) {
                x[e] = s[e / SR][e % SR];
                if constexpr (CAP) x[e] = a.softcap * tanh_fast(div_by_uniform(x[e] * a.scale, a.softcap, a.inv_cap));
            }
            uint32_t gap[KB / 32], some = 0;
#pragma unroll
            for (int e = 0; e < KB / 32; ++e) some |= gap[e] = s_gap[f][e];
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
            const float mu = (m == -INFINITY ? 0.0f : m) * a.unit;
            float ps = 0.0f;
#pragma unroll
            for (int e = 0; e < NT * SR; ++e) {
                x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], a.unit, -mu));
                ps += x[e];
            }
            l += ps;
            // output: MFMA t takes key groups 2 t and 2 t + 1
            const uint8_t* vb[VBASES];
#pragma unroll
            for (int c = 0; c < VBASES; ++c) vb[c] = &s_kv[buf][1][vn + ((c * (M / 8) ^ vy) << 4)];
#pragma unroll
            for (int u = 0; u < NU; u += 2) {
                u32x4 pw;
#pragma unroll
                for (int e = 0; e < 4; ++e) pw[e] = pack_bf16x2(x[4 * u + 2 * e], x[4 * u + 2 * e + 1]);
                const bf16x8 pv = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint8_t* const at = vb[b % VBASES] + (b / VBASES << 7);
                    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + u * US * D * 2));
                    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(at + (u + 1) * US * D * 2));
                    const bf16x8 vv = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[b] = Mfma<M>::run(vv, pv, o[b]);
                }
            }
        }
        if (t + 1 < ntile) store(t + 1, rw);
        __syncthreads();
    }

    l = over_row<M>(l, [](float u, float v) { return u + v; });
    if (w0 + n > r1) return;
    if (s_wild) {
        // What a row sees of the values kept out: whatever its weight, the value itself.
#pragma unroll 1
        for (int k = ks; k < ke; ++k) {
            const int k0 = ks + (k - ks) / KB * KB;
            if (k0 >= wg_lo && k0 + KB - 1 <= wg_hi) continue;  // (uniform: the tile went whole)
            const int r = row_of(a, q, k);
            if (r < 0 || k < lo || k > hi) continue;
            const uint16_t* const vp = (const uint16_t*)a.vc + (int64_t)r * a.kv_stride + kvh * D + 4 * h;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < SR; e += 4) {
                    const f32x4 v = ld4(vp + b * M + 2 * e);
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[b][e + c] += fabsf(v[c]) < INFINITY ? 0.0f : v[c];
                }
        }
    }
    if (l == 0.0f) {  // no key: zeros, whatever weights of 0 made of the values
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = Acc{};
        l = 1.0f;
    }
    const int64_t th = (int64_t)(q.tok0 + i) * a.nh + kvh * a.gq + rr % a.gq;
    if (rg.used == 1) {
        const float inv = 1.0f / l;
        uint16_t* out = (uint16_t*)a.out + th * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < SR; e += 4)
                st4(out + b * M + 2 * e, f32x4{o[b][e] * inv, o[b][e + 1] * inv, o[b][e + 2] * inv, o[b][e + 3] * inv});
    } else {
        const int64_t part = th * a.nparts + split;
        float* w = a.ws + part * D + 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < SR; e += 4) st4(w + b * M + 2 * e, f32x4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]});
        if (h == 0) {
            float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
            ml[0] = m;
            ml[1] = l;
        }
    }
}

template <int D, int M, int NW, int KB, int WPE>
static void launch(const SeqArgs& a, hipStream_t s) {
    const unsigned grid = (unsigned)(most_tiles(a, NW * M) * a.nkv * a.tile_split);
    if (a.softcap > 0.0f) k_seq_tile<D, M, NW, KB, WPE, true><<<grid, NW * kWave, 0, s>>>(a);
    else k_seq_tile<D, M, NW, KB, WPE, false><<<grid, NW * kWave, 0, s>>>(a);
}

#ifndef ZL_T256
#define ZL_T256 256, 16, 8, 32, 2
#define ZL_R256 128
#endif
#ifndef ZL_T128
#define ZL_T128 128, 32, 8, 64, 2
#define ZL_R128 256
#endif
int tile_rows_of(int D) { return D <= 64 ? 256 : D == 128 ? ZL_R128 : D == 256 ? ZL_R256 : 128; }

void launch_tiles(const SeqArgs& a, hipStream_t s) {
    if (a.D == 64) launch<64, 32, 8, 64, 2>(a, s);
    else if (a.D == 128) launch<ZL_T128>(a, s);
    else if (a.D == 256) launch<ZL_T256>(a, s);
    else launch<512, 16, 8, 32, 2>(a, s);
}

}  // namespace zl
