// Causal attention of the new tokens of many sequences: over a paged KV cache (hip_attention_paged:
// one token or a chunk of each sequence) and over packed prompts (hip_attention_prompt). No
// counterpart in the reference, which attends for one sequence over one contiguous cache
// (cuda_bridge.cu:2466-2879).
//
// Sequence s has tokens cu_s .. cu_(s+1) - 1 of q; token i of them is at position p = P_s + i (P_s
// positions were there before: sequence length minus its new tokens; 0 for a prompt) and sees
// positions [max(0, p + 1 - window), p]: score_t = (q_h . k_t) * scale, cap * tanh(score / cap) when
// cap > 0, softmax over t, out_h = sum_t w_t v_t; query head h reads kv head h / (n_heads / n_kv_heads).
// Position t of a paged sequence is cache row table[s][t / page] * page + t % page; pages outside the
// cache hold nothing and are masked. Row t of a prompt is its token cu_s + t.
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
constexpr int kRowWaves = 4;
// Heads of 512 take two waves to a block of keys, half the head size each, which exchange their sums of the
// scores through LDS (a wave that had all of it would need all of a SIMD's registers).
template <int D> constexpr int row_halves() { return D > 256 ? 2 : 1; }
template <typename T, int D>
__global__ __launch_bounds__(row_halves<D>() * kRowWaves * kWave, 2) void k_seq_rows(SeqArgs a) {
    constexpr int HV = row_halves<D>(), DW = D / HV;  // of a wave
    constexpr bool BF = sizeof(T) == 2;
    constexpr int BK = BF ? 32 : 16;             // keys of a block
    constexpr int NT = BK / 16;                  // score tiles of it
    constexpr int EL = 16 / sizeof(T);           // elements of a load
    constexpr int NI = DW / (4 * EL);            // K loads of a lane to a tile
    constexpr int CW = BF && D > 64 ? 8 : 4;     // columns of a V load
    constexpr int NC = DW / (16 * CW);           // V loads of a lane to a row
    constexpr int NR = BF ? 8 : 4;               // V rows of a lane
    constexpr int OS = D + 4;                    // row of the merge buffer
    constexpr int SLOTS = D > 256 ? 2 : 4;
    constexpr float kSlack = 8.0f;               // log2: how far scores may pass the running maximum
    // the merge buffer; before it the query rows, and the halves' sums of the scores
    __shared__ __align__(16) float s_o[SLOTS * 16 * OS];
    constexpr int XF = HV * NI * kWave * 4;  // floats of the query rows
    static_assert(HV == 1 || XF + 2 * HV * kRowWaves * 4 * NT * kWave <= SLOTS * 16 * OS, "LDS");
    __shared__ float s_m[kRowWaves][16], s_l[kRowWaves][16];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wave = wid % kRowWaves, half = wid / kRowWaves;
    int id = (int)blockIdx.x;
    const int kvh = id % a.nkv;
    id /= a.nkv;
    const int split = id % a.nsplit;
    int tile;
    const int sq = __builtin_amdgcn_readfirstlane(find_tile<16, true>(a, id / a.nsplit, tile));
    if (sq < 0) return;
    const Seq q = seq_of(a, sq);
    const int rows = q.nq * a.gq;
    // the last tiles, whose ranges are the longest, first
    const int r0 = ((rows + 15) / 16 - 1 - __builtin_amdgcn_readfirstlane(tile)) * 16, r1 = min(r0 + 16, rows) - 1;
    if (r0 < 0 || r0 >= rows) return;
    const Range rg = tile_range(a, q, r0, r1, a.chunk);
    if (split >= rg.used) return;
    const int ks = rg.ks + split * a.chunk, ke = rg.ke - ks > a.chunk ? ks + a.chunk : rg.ke;
    const int nblk = ke > ks ? (ke - ks + BK - 1) / BK : 0;
    // the lane's query row and its range of keys [lo, hi] (rows behind the last are the last once more)
    const int rr = min(r0 + n, r1), i = rr / a.gq, p = q.pos0 + i;
    const int hi = p >= 0 && p < q.lim ? p : -1;
    const int lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
    // the part of the keys that every row sees
    const int pf = q.pos0 + r0 / a.gq, pl = q.pos0 + r1 / a.gq;
    const bool whole = pf >= 0 && pl < q.lim;
    const int all_lo = a.window > 0 ? max(0, pl + 1 - a.window) : 0, all_hi = pf;

    u32x4* const s_q = reinterpret_cast<u32x4*>(s_o) + half * NI * kWave + lane;
    {
        const T* qrow = (const T*)a.q + (int64_t)(q.tok0 + i) * a.q_stride + (kvh * a.gq + rr % a.gq) * D + half * DW + EL * g;
        const uint32_t flip = BF && !(a.softcap > 0.0f) && a.scale < 0.0f ? 0x80008000u : 0u;  // `unit` has no sign
        for (int j = wave; j < NI; j += kRowWaves) s_q[kWave * j] = ld16(qrow + 4 * EL * j) ^ flip;
    }
    acc4 o[NC * CW];
#pragma unroll
    for (int j = 0; j < NC * CW; ++j) o[j] = acc4{};
    float m = -INFINITY, l = 0.0f;
    bool wild = false;  // infinite or NaN values were kept out of the product

    // The lane's key is lane % BK of a block: its row, -1 where there is none (past the range, or on
    // a page that is not in the cache).
    auto rows_of = [&](int blk) {
        const int key = ks + BK * blk + lane % BK, r = row_of(a, q, min(key, ke - 1));
        return key < ke ? r : -1;
    };
    const T* const kbase = (const T*)a.kc + kvh * D + half * DW + EL * g;
    const T* const vbase = (const T*)a.vc + kvh * D + half * DW + CW * n;
    u32x4 kk[NT][NI];
    typedef uint32_t vload __attribute__((ext_vector_type(BF ? CW / 2 : 4)));
    vload vv[NR][NC];
    auto load_k = [&](int row) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const T* kp = kbase + (int64_t)max(__shfl(row, 16 * t + n), 0) * a.kv_stride;
#pragma unroll
            for (int j = 0; j < NI; ++j) kk[t][j] = ld16(kp + 4 * EL * j);
        }
    };
    auto load_v = [&](int row) {
#pragma unroll
        for (int e = 0; e < NR; ++e) {
            const T* vp = vbase + (int64_t)max(__shfl(row, 16 * (e / 4) + 4 * g + e % 4), 0) * a.kv_stride;
#pragma unroll
            for (int c = 0; c < NC; ++c) vv[e][c] = *reinterpret_cast<const vload*>(vp + 16 * CW * c);
        }
    };
    // (past the last block, and in waves without one, row 0 of the cache is loaded: no load under a branch)
    int row = wave < nblk ? rows_of(wave) : -1, next = wave + kRowWaves < nblk ? rows_of(wave + kRowWaves) : -1;
    load_k(row);
    load_v(row);
    __syncthreads();  // the query rows
    // (where waves exchange sums all of them go as many steps)
    const int steps = HV == 1 ? nblk : (nblk + kRowWaves - 1) / kRowWaves * kRowWaves;
    for (int blk = wave; blk < steps; blk += kRowWaves) {
        const int k0 = ks + BK * blk;
        float x[4 * NT];
        if constexpr (BF) {
            acc4 s[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t] = acc4{};
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const bf16x8 qv = __builtin_bit_cast(bf16x8, s_q[kWave * j]);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk[t][j]), qv, s[t], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) x[e] = s[e / 4][e % 4];
        } else {
            // 16 products at a time into a fresh accumulator, these summed in two chains: one chain over the
            // whole row is two to three times as far from the exact dot product
            acc4 st[2] = {acc4{}, acc4{}};
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const f32x4 qv = __builtin_bit_cast(f32x4, s_q[kWave * j]), kv = __builtin_bit_cast(f32x4, kk[0][j]);
                acc4 c = acc4{};
#pragma unroll
                for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], qv[e], c, 0, 0, 0);
                st[j & 1] += c;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = st[0][e] + st[1][e];
        }
        if constexpr (HV > 1) {
            // (two buffers in turn: a wave is at most a step ahead of its other half)
            f32x4* const mine = reinterpret_cast<f32x4*>(s_o + XF) + ((blk / kRowWaves & 1) * HV * kRowWaves + wid) * NT * kWave + lane;
            const f32x4* const other = mine + (half ? -1 : 1) * kRowWaves * NT * kWave;
#pragma unroll
            for (int t = 0; t < NT; ++t) mine[t * kWave] = f32x4{x[4 * t], x[4 * t + 1], x[4 * t + 2], x[4 * t + 3]};
            __syncthreads();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f32x4 y = other[t * kWave];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * t + e] += y[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) {
            if constexpr (!BF) x[e] *= a.scale;
            if (a.softcap > 0.0f) x[e] = BF ? cap_bf16(a, x[e]) : a.softcap * tanh_fast(div_by_uniform(x[e], a.softcap, a.inv_cap));
        }
        const int row_v = row;
        __builtin_amdgcn_sched_barrier(0);  // the loads stay behind the last use of their registers
        load_k(next);
        row = next;
        if (blk + 2 * kRowWaves < nblk) next = rows_of(blk + 2 * kRowWaves);
        else next = -1;
        __builtin_amdgcn_sched_barrier(0);
        const bool none = __any(row_v < 0);
        const bool edge = none || !(whole && k0 >= all_lo && k0 + BK - 1 <= all_hi);  // uniform
        if (edge) {
#pragma unroll
            for (int e = 0; e < 4 * NT; ++e) {
                const int kb = 16 * (e / 4) + 4 * g + e % 4, key = k0 + kb;
                const bool there = __shfl(row_v, kb) >= 0;
                x[e] = key >= lo && key <= hi && there ? x[e] : -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int e = 1; e < 4 * NT; ++e) mx = fmaxf(mx, x[e]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(!((mx - m) * a.unit <= kSlack))) {
            const float mn = fmaxf(m, mx);
            const float c = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * a.unit);
            m = mn;
            l *= c;
#pragma unroll
            for (int j = 0; j < NC * CW; ++j) o[j] *= c;
        }
        const float ms = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int e = 0; e < 4 * NT; ++e) {
            x[e] = __builtin_amdgcn_exp2f((x[e] - ms) * a.unit);
            l += x[e];
        }
        if (edge) {
            // A weight of 0 must not carry an infinite or NaN value to a row that does not see it: such
            // values stay out, and go to the rows that see them at the end.
            bool bad = false;
#pragma unroll
            for (int e = 0; e < NR; ++e)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int w = 0; w < (int)(sizeof(vload) / 4); ++w) {
                        uint32_t v = vv[e][c][w];
                        if constexpr (BF) {
                            const bool b0 = (v & 0x7f80u) == 0x7f80u, b1 = (v & 0x7f800000u) == 0x7f800000u;
                            bad |= b0 || b1;
                            v &= (b0 ? 0xffff0000u : 0xffffffffu) & (b1 ? 0xffffu : 0xffffffffu);
                        } else {
                            const bool b = (v & 0x7f800000u) == 0x7f800000u;
                            bad |= b;
                            v = b ? 0u : v;
                        }
                        vv[e][c][w] = v;
                    }
            wild |= __any(bad) != 0;
        }
        if constexpr (BF) {
            // the weights as two bf16 terms (16 bits; one alone would add an error as large as the output's own
            // rounding, and the products here wait for memory anyway)
            u32x4 ph, pl;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ph[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
                pl[e] = pack_bf16x2(x[2 * e] - bf16_lo(ph[e]), x[2 * e + 1] - bf16_hi(ph[e]));
            }
            const bf16x8 pv = __builtin_bit_cast(bf16x8, ph), pr = __builtin_bit_cast(bf16x8, pl);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int w = 0; w < CW / 2; ++w) {
                    u32x4 v0, v1;  // columns 2 w and 2 w + 1 of the lane's eight keys
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v0[e] = __builtin_amdgcn_perm(vv[2 * e + 1][c][w], vv[2 * e][c][w], 0x05040100u);
                        v1[e] = __builtin_amdgcn_perm(vv[2 * e + 1][c][w], vv[2 * e][c][w], 0x07060302u);
                    }
                    const bf16x8 b0 = __builtin_bit_cast(bf16x8, v0), b1 = __builtin_bit_cast(bf16x8, v1);
                    acc4 &o0 = o[c * CW + 2 * w], &o1 = o[c * CW + 2 * w + 1];
                    o0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b0, pr, o0, 0, 0, 0);
                    o1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b1, pr, o1, 0, 0, 0);
                    o0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b0, pv, o0, 0, 0, 0);
                    o1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b1, pv, o1, 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[c * 4 + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vv[e][c][j]), x[e], o[c * 4 + j], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(row);
    }
    if (wild) {
        // What a row sees of the values kept out: whatever its weight, the value itself (which changes nothing
        // where it went in).
#pragma unroll 1
        for (int k = 0; k < nblk * BK; ++k) {
            const int key = ks + k;
            if (k / BK % kRowWaves != wave || key >= ke) continue;
            const int r = row_of(a, q, key);
            if (r < 0 || key < lo || key > hi) continue;
            const T* const vp = (const T*)a.vc + (int64_t)r * a.kv_stride + kvh * D + half * DW + 4 * CW * g;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < CW; j += 4) {
                        const f32x4 v = ld4(vp + 16 * CW * c + CW * e + j);
#pragma unroll
                        for (int z = 0; z < 4; ++z) o[c * CW + j + z][e] += fabsf(v[z]) < INFINITY ? 0.0f : v[z];
                    }
        }
    }

    // Merge: each wave's state scaled to the common maximum, SLOTS waves at a time into the slots, which
    // every thread then adds in slot order.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (l == 0.0f) {  // no key: zeros, whatever weights of 0 made of the values
#pragma unroll
        for (int j = 0; j < NC * CW; ++j) o[j] = acc4{};
    }
    if (g == 0 && half == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    __syncthreads();  // and every wave is done with the query rows
    {
        float M = s_m[0][n];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) M = fmaxf(M, s_m[w][n]);
        const float f = __builtin_amdgcn_exp2f((m - (M == -INFINITY ? 0.0f : M)) * a.unit);
#pragma unroll
        for (int j = 0; j < NC * CW; ++j) o[j] *= f;
    }
    float* const slot = s_o + (wave % SLOTS * 16 + n) * OS + half * DW + 4 * CW * g;
#pragma unroll
    for (int w0 = 0; w0 < kRowWaves; w0 += SLOTS) {
        if (wave >= w0 && wave < w0 + SLOTS && r0 + n <= r1) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < CW; j += 4) {
                        f32x4* const at = reinterpret_cast<f32x4*>(slot + 16 * CW * c + CW * e + j);
                        f32x4 v{o[c * CW + j][e], o[c * CW + j + 1][e], o[c * CW + j + 2][e], o[c * CW + j + 3][e]};
                        if (w0 > 0) v += *at;
                        *at = v;
                    }
        }
        __syncthreads();
    }
    for (int t = threadIdx.x; t < 16 * D / 4; t += HV * kRowWaves * kWave) {
        const int rw = t / (D / 4), col = t % (D / 4) * 4;
        if (r0 + rw > r1) break;
        const int64_t tok = q.tok0 + (r0 + rw) / a.gq, h = kvh * a.gq + (r0 + rw) % a.gq;
        float M = s_m[0][rw], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) M = fmaxf(M, s_m[w][rw]);
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w)
            L += s_l[w][rw] * __builtin_amdgcn_exp2f((s_m[w][rw] - (M == -INFINITY ? 0.0f : M)) * a.unit);
        f32x4 v{};
#pragma unroll
        for (int w = 0; w < SLOTS; ++w) v += *reinterpret_cast<const f32x4*>(s_o + (w * 16 + rw) * OS + col);
        if (rg.used == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = L == 0.0f ? 0.0f : v[e] / L;  // (no key: zeros)
            st4((T*)a.out + (tok * a.nh + h) * D + col, v);
        } else {
            const int64_t part = (tok * a.nh + h) * a.nparts + split;
            st4(a.ws + part * D + col, v);
            if (col == 0) {
                float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

// Joins the splits of a (token, head): out = sum_s exp(m_s - M) o_s / sum_s exp(m_s - M) l_s. W waves take
// a head, wave w splits w, w + W, ...: four where there can be many splits, one where there are few
// (and a workgroup four heads). The row's splits are those of the tile that formed them. The maxima
// and the first sums are requested before their number is known (slots behind it hold anything:
// they are dropped, not weighted by 0), which leaves one round trip to memory behind the sequence's own.
constexpr int kMaxSplits = 256;
constexpr int kJoinWaves = 4;
constexpr int kJoinFew = 16;  // (many heads: up to a wave's 64)
template <typename T, int D, int W>
__global__ __launch_bounds__(kJoinWaves * kWave) void k_seq_join(SeqArgs a) {
    constexpr int E = D / 64;  // columns of a lane
    constexpr int PER = W == 1 ? 1 : kMaxSplits / kWave;
    constexpr int PRE = 4;
    typedef float Cols __attribute__((ext_vector_type(E)));
    __shared__ float s_part[W == 1 ? 1 : W][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t th = W == 1 ? (int64_t)blockIdx.x * kJoinWaves + wave : (int64_t)blockIdx.x;
    const int w = W == 1 ? 0 : wave;
    if (th >= (int64_t)a.n_tokens * a.nh) return;  // (uniform in a wave, and in the workgroup where W > 1)
    const int64_t part = th * a.nparts;
    const int tok = (int)(th / a.nh), h = (int)(th % a.nh);
    const float* const ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
    const float* const sums = a.ws + part * D + E * lane;
    float mv[PER], lv[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int sp = min(lane + j * kWave, a.nparts - 1);
        mv[j] = ml[2 * sp];
        lv[j] = ml[2 * sp + 1];
    }
    Cols pre[PRE];
#pragma unroll
    for (int k = 0; k < PRE; ++k) pre[k] = *reinterpret_cast<const Cols*>(sums + (int64_t)min(w + k * W, a.nparts - 1) * D);
    int sq = tok;
    if (a.cu) {
        // the last sequence that begins at or before the token
        int lo = 0, hi = a.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= tok) lo = mid;
            else hi = mid;
        }
        sq = lo;
    } else if (!a.table) {
        sq = 0;
    }
    const Seq q = seq_of(a, sq);
    if (tok < q.tok0 || tok >= q.tok0 + q.nq) return;
    const int rows = q.nq * a.gq;
    const bool few = rows <= a.few_rows;
    const int R = few ? 16 : a.tile_rows;
    const int r = (tok - q.tok0) * a.gq + h % a.gq, r0 = r / R * R, r1 = min(r0 + R, rows) - 1;
    const int used = tile_range(a, q, r0, r1, few ? a.chunk : a.tile_chunk).used;
    if (used == 1) return;
    float M = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) M = fmaxf(M, lane + j * kWave < used ? mv[j] : -INFINITY);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    float L = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        mv[j] = __builtin_amdgcn_exp2f((mv[j] - (M == -INFINITY ? 0.0f : M)) * a.unit);
        if (lane + j * kWave < used) L = fmaf(lv[j], mv[j], L);
    }
    L = group_sum<kWave>(L);
    Cols acc = Cols{};
    // the weight of split sp
    auto weight = [&](int sp) {
        float c = mv[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) c = sp / kWave == j ? mv[j] : c;
        return __shfl(c, sp % kWave);
    };
    for (int s0 = w; s0 < used; s0 += PRE * W) {
        if (s0 > w) {
#pragma unroll
            for (int k = 0; k < PRE; ++k) pre[k] = *reinterpret_cast<const Cols*>(sums + (int64_t)min(s0 + k * W, used - 1) * D);
        }
#pragma unroll
        for (int k = 0; k < PRE; ++k)
            if (s0 + k * W < used) acc += pre[k] * weight(s0 + k * W);
    }
    auto put = [&](int c, float v) {
        v = L == 0.0f ? 0.0f : v / L;
        if constexpr (sizeof(T) == 4) ((T*)a.out)[th * D + c] = v;
        else ((T*)a.out)[th * D + c] = (T)(pack_bf16x2(v, 0.0f) & 0xffffu);
    };
    if constexpr (W == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            put(E * lane + e, acc[e]);
        }
    } else {
        *reinterpret_cast<Cols*>(&s_part[w][E * lane]) = acc;
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += kJoinWaves * kWave) put(c, (s_part[0][c] + s_part[1][c]) + (s_part[2][c] + s_part[3][c]));
    }
}

// ---- host --------------------------------------------------------------------------------------

// Tiles of k_seq_rows, at most: of all sequences, or of those of few rows.
static int64_t most_few(const SeqArgs& a) {
    const int64_t all = most_tiles(a, 16);
    return a.few_rows == INT32_MAX ? all : std::min<int64_t>(all, (int64_t)a.n_seqs * cdiv(a.few_rows, 16));
}
// Which kernels a call takes, and the splits of each one's ranges.
// k_seq_rows reads K and V for 16 query rows; the tile kernels (k_seq_tile; f32 heads up to 256 k_seq_terms)
// for 64 to 256 that share them. Sequences of few rows (bf16 16, f32 64) are k_seq_rows's, the others the
// tiles'; a call whose sequences are surely of one kind launches one kernel (32 queries of one sequence
// behind 4000 keys, 8 / 4 heads x 256 f32: 30 us by k_seq_rows, 46 by tiles; 512 behind 1500: 133 and 81).
// f32 prompts are k_seq_rows's until their tiles fill the chip twice, or once where a window makes them alike:
// its workgroups are an eighth of the work and even out (8 / 4 heads x 256, 1024 tokens 107 us / 203 by tiles, 4096
// 731 / 768, but with a window of 512 220 / 146; 32 / 16 heads x 128, 512 tokens 42 / 55, 2048 349 / 214).
static void choose(SeqArgs& a, int dtype) {
    const bool f32 = dtype == HIP_BRIDGE_F32;
    a.gq = a.nh / a.nkv;
    const int64_t rows = (int64_t)a.n_tokens * a.gq;
    auto tiles_of = [&](bool small) { return cdiv(rows, tile_rows_of(dtype, a.D, small)) * a.nkv; };  // if the sequences are even
    // Prompts that leave CUs idle take smaller tiles (64 tokens, 8 / 4 heads x 256 bf16 13.4 -> 10.6 us, 512 of 32
    // / 16 x 128 26 -> 23.5; over the largest, 8192, the larger ones are ahead by 8%).
    a.tile_rows = tile_rows_of(dtype, a.D, !a.table && tiles_of(false) < 256);
    const bool single = a.table && !a.cu;  // a token each
    const int few = f32 ? 64 : 16;
    const bool short32 = f32 && !a.table && (a.D == 512 || tiles_of(false) < (a.window > 0 ? 256 : 512));
    if (short32 || rows <= std::max<int64_t>(few, (int64_t)a.n_seqs * few / 2) || (single && a.gq <= few)) a.few_rows = INT32_MAX;
    else a.few_rows = single || !a.table || a.n_seqs == 1 ? 0 : few;

    // A call's splits have one size, whatever the sequences' lengths, which evens out the workgroups of a ragged
    // batch: `keys` each, or as many more as keep their number within bounds.
    auto split = [&](int R, int64_t keys, int& chunk) {
        const int64_t len = most_keys(a, R);
        keys = std::max(cdiv(keys, 64), cdiv(cdiv(len, kMaxSplits), 64)) * 64;
        chunk = (int)std::min<int64_t>(keys, INT32_MAX);
        return (int)std::max<int64_t>(cdiv(len, keys), 1);
    };
    a.nsplit = a.tile_split = 1;
    a.chunk = a.tile_chunk = INT32_MAX;
    if (a.few_rows > 0) {
        // Decode: half a megabyte of K and V, less where that leaves under 1024 workgroups (16 requests of up to
        // 8192 positions in 8 equal splits each 188 us, in splits of 256 keys 122), down to a block for each wave (one
        // token at 1250, f32: 14.6 us in splits of 64 keys, 19.4 of 128), and no more than 16384 workgroups (whose
        // partial sums take 17 MB at two heads of 128 to a kv head). Chunks: 1024 workgroups. Beside tiles: as
        // decode (a token of a sequence each, mostly), in at most 32 splits, as the tiles' rows pass the join too.
        const bool decode = a.n_tokens <= a.n_seqs || a.few_rows < INT32_MAX;
        const int64_t groups = (a.few_rows < INT32_MAX ? (int64_t)a.n_seqs * cdiv(a.gq, 16) : most_tiles(a, 16)) * a.nkv;
        const int64_t all = most_keys(a, 16) * groups, fill = cdiv(all, 1024);
        const int64_t least = std::max<int64_t>({f32 ? 64 : 128, cdiv(all, 16384), a.few_rows < INT32_MAX ? cdiv(most_keys(a, 16), 32) : 0});
        if (decode) a.nsplit = split(16, std::max(least, std::min<int64_t>((1 << 18) / (a.D * (f32 ? 4 : 2)), fill)), a.chunk);
        else if (groups < 1024) a.nsplit = split(16, std::max<int64_t>(fill, 128), a.chunk);
    }
    if (a.few_rows < INT32_MAX && a.table && tiles_of(false) < 256) {
        // Chunks whose tiles leave CUs idle: for one sequence as many splits as its tiles have room for at a
        // workgroup to a CU (256 tokens behind 8000, 32 / 16 heads x 128 bf16: 63 us at 256 workgroups, 82 at
        // 512, 116 at 1024: partial sums cost more than they even out; f32 213, 362 before it was 256 at the most),
        // for several, whose lengths differ, two or three to a CU.
        const int64_t tiles = tiles_of(false), len = most_keys(a, a.tile_rows);
        const int64_t keys = a.n_seqs == 1 ? std::max<int64_t>(128, cdiv(len, 256 / tiles))
                                           : std::max<int64_t>(256, cdiv(tiles * len, f32 ? 768 : 512));
        a.tile_split = split(a.tile_rows, keys, a.tile_chunk);
    }
    a.nparts = std::max(a.nsplit, a.tile_split);
}
static size_t split_bytes(const SeqArgs& a) {
    return a.nparts > 1 ? (size_t)a.n_tokens * a.nh * a.nparts * (a.D + 2) * sizeof(float) : 0;
}
static size_t workspace_bytes_of(SeqArgs& a, int dtype, bool paged) {
    if (a.n_seqs <= 0 || a.n_tokens <= 0 || a.nh <= 0 || a.nkv <= 0 || a.nh % a.nkv != 0 || a.D <= 0 || a.max_len <= 0) return 0;
    static const int32_t some = 0;  // (never followed)
    a.table = paged ? &some : nullptr;
    a.cu = &some;
    choose(a, dtype);
    size_t need = split_bytes(a);
    if (paged && a.n_tokens == a.n_seqs) {  // also called without d_cu
        a.cu = nullptr;
        choose(a, dtype);
        need = std::max(need, split_bytes(a));
    }
    return need;
}

template <typename T, int D>
static void launch_rows(const SeqArgs& a, hipStream_t s) {
    if (a.few_rows > 0) {
        const int64_t grid = most_few(a) * a.nkv * a.nsplit;
        k_seq_rows<T, D><<<(unsigned)grid, row_halves<D>() * kRowWaves * kWave, 0, s>>>(a);
    }
    if (a.few_rows < INT32_MAX) launch_tiles(sizeof(T) == 4 ? HIP_BRIDGE_F32 : HIP_BRIDGE_BF16, a, s);
    if (a.nparts > 1) {
        const int64_t th = (int64_t)a.n_tokens * a.nh;
        if (a.nparts <= (th > 2048 ? kWave : kJoinFew)) k_seq_join<T, D, 1><<<(unsigned)cdiv(th, kJoinWaves), kJoinWaves * kWave, 0, s>>>(a);
        else k_seq_join<T, D, kJoinWaves><<<(unsigned)th, kJoinWaves * kWave, 0, s>>>(a);
    }
    check_launch();
}
template <typename T>
static void launch_type(const SeqArgs& a, hipStream_t s) {
    if (a.D == 64) launch_rows<T, 64>(a, s);
    else if (a.D == 128) launch_rows<T, 128>(a, s);
    else if (a.D == 256) launch_rows<T, 256>(a, s);
    else launch_rows<T, 512>(a, s);
}

static void launch_seqs(int dtype, SeqArgs& a, void* ws, size_t ws_bytes, hipStream_t s) {
    if (!a.q || !a.kc || !a.vc || !a.out || a.nh <= 0 || a.nkv <= 0 || a.nh % a.nkv != 0 || a.max_len <= 0 ||
        a.q_stride < (int64_t)a.nh * a.D || a.kv_stride < (int64_t)a.nkv * a.D) {
        set_error(HIP_BRIDGE_EINVAL);
        return;
    }
    const int es = dtype == HIP_BRIDGE_F32 ? 4 : 2;
    const bool aligned = aligned16(a.q) && aligned16(a.kc) && aligned16(a.vc) && aligned16(a.out) &&
                         a.q_stride * es % 16 == 0 && a.kv_stride * es % 16 == 0;
    if ((dtype != HIP_BRIDGE_F32 && dtype != HIP_BRIDGE_BF16) || (a.D != 64 && a.D != 128 && a.D != 256 && a.D != 512) ||
        !aligned || (int64_t)a.n_tokens * a.nh > INT32_MAX) {
        set_error(HIP_BRIDGE_EUNSUPPORTED);
        return;
    }
    choose(a, dtype);
    if (a.nparts > 1 && (!ws || !aligned16(ws) || split_bytes(a) > ws_bytes)) {
        a.nsplit = a.tile_split = a.nparts = 1;
        a.chunk = a.tile_chunk = INT32_MAX;
    }
    a.ws = (float*)ws;
    a.inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    a.cap_in = a.softcap > 0.0f ? 2.0f * kLog2e * (a.scale / a.softcap) : 0.0f;
    // (never 0: a masked score of -inf times it stays -inf)
    a.unit = dtype == HIP_BRIDGE_F32 || a.softcap > 0.0f ? kLog2e : std::max(kLog2e * std::fabs(a.scale), 1e-30f);
    if (most_tiles(a, 16) * a.nkv * a.nparts > INT32_MAX) {
        set_error(HIP_BRIDGE_EUNSUPPORTED);
        return;
    }
    if (dtype == HIP_BRIDGE_F32) launch_type<float>(a, s);
    else launch_type<uint16_t>(a, s);
}

}  // namespace zl

using namespace zl;

extern "C" {

size_t hip_attention_paged_workspace_bytes(int dtype, int n_seqs, int n_tokens, int max_len, int n_heads, int n_kv_heads,
                                           int head_dim, int sliding_window) {
    SeqArgs a{};
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.max_len = max_len;
    a.nh = n_heads;
    a.nkv = n_kv_heads;
    a.D = head_dim;
    a.window = sliding_window;
    return workspace_bytes_of(a, dtype, true);
}

void hip_attention_paged(int dtype, const void* q, const void* k_cache, const void* v_cache, void* out,
                         int64_t cache_pages, int page_size, int64_t row_stride, const int32_t* d_block_table,
                         int max_pages, const int32_t* d_cu, const int32_t* d_seq_len, int n_seqs, int n_tokens,
                         int max_len, int n_heads, int n_kv_heads, int head_dim, float attn_scale, float softcap,
                         int sliding_window, void* workspace, size_t workspace_bytes, HipStream_t stream) {
    if (n_seqs <= 0 || n_tokens <= 0) return;
    if (!d_block_table || !d_seq_len || cache_pages <= 0 || page_size <= 0 || max_pages <= 0 ||
        (!d_cu && n_tokens != n_seqs)) {
        set_error(HIP_BRIDGE_EINVAL);
        return;
    }
    if (cache_pages > INT32_MAX / page_size) {  // cache rows are 32-bit
        set_error(HIP_BRIDGE_EUNSUPPORTED);
        return;
    }
    SeqArgs a{};
    a.q = q;
    a.kc = k_cache;
    a.vc = v_cache;
    a.out = out;
    a.cu = d_cu;
    a.len = d_seq_len;
    a.table = d_block_table;
    a.q_stride = (int64_t)n_heads * head_dim;
    a.kv_stride = row_stride;
    a.cache_pages = cache_pages;
    a.page = page_size;
    a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
    a.max_pages = max_pages;
    a.max_len = max_len;
    a.lim = (int)std::min<int64_t>(max_len, (int64_t)max_pages * page_size);
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.nh = n_heads;
    a.nkv = n_kv_heads;
    a.D = head_dim;
    a.window = sliding_window;
    a.scale = attn_scale;
    a.softcap = softcap;
    launch_seqs(dtype, a, workspace, workspace_bytes, stream_of(stream));
}

size_t hip_attention_prompt_workspace_bytes(int dtype, int n_seqs, int n_tokens, int n_heads, int n_kv_heads,
                                            int head_dim, int sliding_window) {
    SeqArgs a{};
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.max_len = n_tokens;
    a.nh = n_heads;
    a.nkv = n_kv_heads;
    a.D = head_dim;
    a.window = sliding_window;
    return workspace_bytes_of(a, dtype, false);
}

void hip_attention_prompt(int dtype, const void* q, const void* k, const void* v, void* out, int64_t q_stride,
                          int64_t kv_stride, const int32_t* d_cu, int n_seqs, int n_tokens, int n_heads, int n_kv_heads,
                          int head_dim, float attn_scale, float softcap, int sliding_window, void* workspace,
                          size_t workspace_bytes, HipStream_t stream) {
    if (n_seqs <= 0 || n_tokens <= 0) return;
    if (!d_cu && n_seqs != 1) {
        set_error(HIP_BRIDGE_EINVAL);
        return;
    }
    SeqArgs a{};
    a.q = q;
    a.kc = k;
    a.vc = v;
    a.out = out;
    a.cu = d_cu;
    a.q_stride = q_stride;
    a.kv_stride = kv_stride;
    a.max_len = n_tokens;
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.nh = n_heads;
    a.nkv = n_kv_heads;
    a.D = head_dim;
    a.window = sliding_window;
    a.scale = attn_scale;
    a.softcap = softcap;
    launch_seqs(dtype, a, workspace, workspace_bytes, stream_of(stream));
}

}  // extern "C"
