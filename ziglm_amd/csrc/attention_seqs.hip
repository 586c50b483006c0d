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

// ---- 16 query rows on the f32 matrix cores ---------------------------------------------------
// A workgroup takes 16 query rows of one kv head and a split of their keys, its waves the 16-key
// blocks in turn, with the f32 MFMA 16x16x4 (exact f32 products and sums; bf16 values are exact in
// f32). Scores are formed transposed, S^T = K Q^T, so that lane (n = lane % 16, g = lane / 16) holds
// query row n and keys 4 g + r in register r, the A operand of P V as it stands. The waves' online
// softmax states merge through LDS.
template <int D> constexpr int row_waves() { return D > 256 ? 4 : 8; }
template <typename T, int D>
__global__ __launch_bounds__(row_waves<D>() * kWave, D > 256 ? 1 : 2) void k_seq_rows(SeqArgs a) {
    constexpr int kRowWaves = row_waves<D>();
    constexpr int NI = D / 16;  // loads of a lane per K block and head row
    constexpr int NC = D / 64;  // and per V row
    constexpr int NH = D / 32;  // loads of half a K (V) block
    constexpr int SLOTS = D > 256 ? 2 : 4;
    __shared__ float s_o[SLOTS][D / 4 * kWave];
    __shared__ float s_m[kRowWaves][16], s_l[kRowWaves][16];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int id = (int)blockIdx.x;
    const int kvh = id % a.nkv;
    id /= a.nkv;
    const int split = id % a.nsplit;
    int tile;
    const int sq = __builtin_amdgcn_readfirstlane(find_tile<16, true>(a, id / a.nsplit, tile));
    if (sq < 0) return;
    const Seq q = seq_of(a, sq);
    const int r0 = __builtin_amdgcn_readfirstlane(tile) * 16, rows = q.nq * a.gq, r1 = min(r0 + 16, rows) - 1;
    if (r0 >= rows) return;
    const Range rg = tile_range(a, q, r0, r1, a.nsplit);
    if (split >= rg.used) return;
    const int ks = rg.ks + split * rg.chunk, ke = min(rg.ke, ks + rg.chunk);
    const int nblk = ke > ks ? (ke - ks + 15) / 16 : 0;
    // the lane's query row and its range of keys [lo, hi]
    const int rr = min(r0 + n, r1), i = rr / a.gq, p = q.pos0 + i;
    const bool valid = r0 + n <= r1 && p >= 0 && p < q.lim;
    const int hi = valid ? p : -1;
    const int lo = a.window > 0 ? max(0, p + 1 - a.window) : 0;
    // the part of the keys that every row sees
    const int pf = q.pos0 + r0 / a.gq, pl = q.pos0 + r1 / a.gq;
    const bool whole = r0 + 15 == r1 && pf >= 0 && pl < q.lim;
    const int all_lo = a.window > 0 ? max(0, pl + 1 - a.window) : 0, all_hi = pf;

    const T* const kbase = (const T*)a.kc + kvh * D + 4 * g;
    const T* const vbase = (const T*)a.vc + kvh * D + 4 * n;
    float* const s_q = &s_o[0][0] + 4 * lane;
    {
        const T* qrow = (const T*)a.q + (int64_t)(q.tok0 + i) * a.q_stride + (kvh * a.gq + rr % a.gq) * D + 4 * g;
        for (int j = wave; j < NI; j += kRowWaves) *reinterpret_cast<f32x4*>(s_q + 4 * kWave * j) = ld4(qrow + 16 * j);
    }
    __syncthreads();
    acc4 o[NC * 4];
#pragma unroll
    for (int j = 0; j < NC * 4; ++j) o[j] = acc4{};
    float m = -INFINITY, l = 0.0f;

    f32x4 bx[NH], by[NH];
    // The lane's key is n of a block: its row, -1 where there is none. Keys past the range take its last
    // row (masked).
    auto rows_of = [&](int blk) { return row_of(a, q, min(ks + 16 * blk + n, ke - 1)); };
    auto load_k = [&](f32x4 (&r)[NH], int row, int half) {
        const T* kp = kbase + (int64_t)max(row, 0) * a.kv_stride;
#pragma unroll
        for (int j = 0; j < NH; ++j) r[j] = ld4(kp + 16 * (NH * half + j));
    };
    auto load_v = [&](f32x4 (&r)[NH], int row, int half) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const T* vp = vbase + (int64_t)max(__shfl(row, 4 * g + 2 * half + j), 0) * a.kv_stride;
#pragma unroll
            for (int c = 0; c < NC; ++c) r[NC * j + c] = ld4(vp + 64 * c);
        }
    };
    int row = 0, row_next = 0;
    if (wave < nblk) {
        row = rows_of(wave);
        load_k(bx, row, 0);
    }
    for (int blk = wave; blk < nblk; blk += kRowWaves) {
        const int k0 = ks + 16 * blk;
        row_next = rows_of(min(blk + kRowWaves, nblk - 1));
        // scores: 16 products at a time into a fresh accumulator, these summed in two chains
        acc4 st[2] = {acc4{}, acc4{}};
        auto scores = [&](const f32x4 (&kr)[NH], int half) {
#pragma unroll
            for (int j = 0; j < NH; ++j) {
                const f32x4 qv = *reinterpret_cast<const f32x4*>(s_q + 4 * kWave * (NH * half + j));
                acc4 c = acc4{};
#pragma unroll
                for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[j][e], qv[e], c, 0, 0, 0);
                st[j & 1] += c;
            }
        };
        load_k(by, row, 1);
        scores(bx, 0);
        load_v(bx, row, 0);
        scores(by, 1);
        load_v(by, row, 1);
        // (row -1: keys 4 g + r of the block whose page is not in the cache)
        const bool gap = __any(row < 0);
        const bool edge = gap || !(whole && k0 >= all_lo && k0 + 15 <= all_hi);  // uniform
        float s[4], mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float v = (st[0][r] + st[1][r]) * a.scale;
            if (a.softcap > 0.0f) v = a.softcap * tanh_fast(div_by_uniform(v, a.softcap, a.inv_cap));
            const int key = k0 + 4 * g + r;
            const bool there = !gap || __shfl(row, 4 * g + r) >= 0;
            s[r] = key >= lo && key <= hi && key < ke && there ? v : -INFINITY;
            mx = fmaxf(mx, s[r]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.0f : mn;
        const float c = exp2f((m - ms) * kLog2e);
        float pr[4], ps = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            pr[r] = exp2f((s[r] - ms) * kLog2e);
            ps += pr[r];
        }
        l = l * c + ps;
        m = mn;
        if (!__all(c == 1.0f)) {  // rows 4 g + r of the output accumulators
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float cr = __shfl(c, 4 * g + r);
#pragma unroll
                for (int j = 0; j < NC * 4; ++j) o[j][r] *= cr;
            }
        }
        if (edge) {
            float z = 0.0f;  // NaN if a V value is infinite or NaN
#pragma unroll
            for (int j = 0; j < NH; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) z += bx[j][e] * 0.0f + by[j][e] * 0.0f;
            if (__any(!(z == 0.0f))) {
                // Some of the query rows may see such a row and others not: 0 * V would reach the others,
                // so each takes just the keys it sees, and the products below add zeros.
#pragma unroll 1
                for (int k = 0; k < 16; ++k) {
                    const int rk = __shfl(row, k);
                    if (k0 + k >= ke || rk < 0) continue;  // uniform
                    const T* vp = vbase + (int64_t)rk * a.kv_stride;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float pk = __shfl(k & 2 ? (k & 1 ? pr[3] : pr[2]) : (k & 1 ? pr[1] : pr[0]),
                                                4 * g + r + 16 * (k >> 2));
                        const int rlo = __shfl(lo, 4 * g + r), rhi = __shfl(hi, 4 * g + r);
                        if (k0 + k >= rlo && k0 + k <= rhi) {
#pragma unroll
                            for (int cc = 0; cc < NC; ++cc) {
                                const f32x4 v = ld4(vp + 64 * cc);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[cc * 4 + e][r] = fmaf(pk, v[e], o[cc * 4 + e][r]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) pr[r] = 0.0f;
#pragma unroll
                for (int j = 0; j < NH; ++j) bx[j] = by[j] = f32x4{};
            }
        }
        auto pv = [&](const f32x4 (&v)[NH], int half) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int cc = 0; cc < NC; ++cc)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[cc * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(pr[2 * half + j], v[NC * j + cc][e],
                                                                             o[cc * 4 + e], 0, 0, 0);
        };
        pv(bx, 0);
        load_k(bx, row_next, 0);
        pv(by, 1);
        row = row_next;
    }

    // Merge: each wave's state scaled to the common maximum, SLOTS waves at a time into the slots, which
    // every thread then adds in slot order.
    __syncthreads();  // every wave is done with the query rows
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        s_m[wave][n] = m;
        s_l[wave][n] = l;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int rw = 4 * g + r;
        float M = s_m[0][rw];
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) M = fmaxf(M, s_m[w][rw]);
        const float f = exp2f((s_m[wave][rw] - (M == -INFINITY ? 0.0f : M)) * kLog2e);
#pragma unroll
        for (int j = 0; j < NC * 4; ++j) o[j][r] *= f;
    }
    float* const slot = s_o[wave % SLOTS] + lane;
#pragma unroll
    for (int w0 = 0; w0 < kRowWaves; w0 += SLOTS) {
        if (wave >= w0 && wave < w0 + SLOTS) {
#pragma unroll
            for (int j = 0; j < NC * 4; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = (j * 4 + r) * kWave;
                    slot[at] = w0 == 0 ? o[j][r] : slot[at] + o[j][r];
                }
        }
        __syncthreads();
    }
    // row = 4 g + r, columns 64 c + 4 n + e: four of a row per thread
    for (int t = threadIdx.x; t < 16 * D / 4; t += kRowWaves * kWave) {
        const int rw = t / (D / 4), col = t % (D / 4), c = col / 16, nn = col % 16;
        if (r0 + rw > r1) continue;
        const int64_t tok = q.tok0 + (r0 + rw) / a.gq, h = kvh * a.gq + (r0 + rw) % a.gq;
        float M = s_m[0][rw], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kRowWaves; ++w) M = fmaxf(M, s_m[w][rw]);
#pragma unroll
        for (int w = 0; w < kRowWaves; ++w) L += s_l[w][rw] * exp2f((s_m[w][rw] - (M == -INFINITY ? 0.0f : M)) * kLog2e);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = 0.0f;
#pragma unroll
            for (int w = 0; w < SLOTS; ++w) x += s_o[w][((c * 4 + e) * 4 + (rw & 3)) * kWave + 16 * (rw >> 2) + nn];
            v[e] = x;
        }
        if (rg.used == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = L == 0.0f ? 0.0f : v[e] / L;  // (no key: zeros)
            st4((T*)a.out + (tok * a.nh + h) * D + 4 * col, v);
        } else {
            const int64_t part = (tok * a.nh + h) * a.nparts + split;
            st4(a.ws + part * D + 4 * col, v);
            if (col == 0) {
                float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

// Joins the splits of a (token, head): out = sum_s exp(m_s - M) o_s / sum_s exp(m_s - M) l_s, a wave
// each. The row's splits are those of the tile that formed them.
constexpr int kMaxSplits = 256;
constexpr int kJoinWaves = 4;
template <typename T, int D>
__global__ __launch_bounds__(kJoinWaves * kWave) void k_seq_join(SeqArgs a) {
    constexpr int E = D / 64;  // columns of a lane
    constexpr int PER = kMaxSplits / kWave;
    const int lane = threadIdx.x & 63;
    const int64_t th = (int64_t)blockIdx.x * kJoinWaves + (threadIdx.x >> 6);
    if (th >= (int64_t)a.n_tokens * a.nh) return;
    const int tok = __builtin_amdgcn_readfirstlane((int)(th / a.nh)), h = (int)(th % a.nh);
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
    const float unit = few ? kLog2e : a.unit;
    const int r = (tok - q.tok0) * a.gq + h % a.gq, r0 = r / R * R, r1 = min(r0 + R, rows) - 1;
    const Range rg = tile_range(a, q, r0, r1, few ? a.nsplit : a.tile_split);
    if (rg.used == 1) return;
    const int64_t part = th * a.nparts;
    const float* ml = a.ws + (int64_t)a.n_tokens * a.nh * a.nparts * D + 2 * part;
    float mv[PER], lv[PER], M = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int sp = lane + j * kWave;
        mv[j] = sp < rg.used ? ml[2 * sp] : -INFINITY;
        lv[j] = sp < rg.used ? ml[2 * sp + 1] : 0.0f;
        M = fmaxf(M, mv[j]);
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    float L = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        mv[j] = exp2f((mv[j] - (M == -INFINITY ? 0.0f : M)) * unit);
        L = fmaf(lv[j], mv[j], L);
    }
    L = group_sum<kWave>(L);
    float acc[E] = {};
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int end = min(rg.used - j * kWave, kWave);
        for (int sp = 0; sp < end; ++sp) {
            const float c = __shfl(mv[j], sp);
            const float* w = a.ws + (part + j * kWave + sp) * D + E * lane;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(w[e], c, acc[e]);
        }
    }
    T* out = (T*)a.out + th * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float v = L == 0.0f ? 0.0f : acc[e] / L;
        if constexpr (sizeof(T) == 4) out[e] = v;
        else out[e] = (T)(pack_bf16x2(v, 0.0f) & 0xffffu);
    }
}

// ---- host --------------------------------------------------------------------------------------

// Which kernels a call takes, and the splits of each one's ranges. k_seq_tile takes bf16 calls'
// sequences of more than 16 query rows; a call whose sequences all have that few (a token each), or
// surely more (a prompt, one chunk), launches one kernel only.
// Splits: as many as bring the launch to about 512 workgroups (256 of k_seq_tile), none shorter than 128
// (256) keys of the longest possible range.
static void choose(SeqArgs& a, int dtype) {
    a.gq = a.nh / a.nkv;
    a.tile_rows = tile_rows_of(a.D);
    const bool single = a.table && !a.cu;  // a token each
    if (dtype != HIP_BRIDGE_BF16 || (int64_t)a.n_tokens * a.gq <= 16 || (single && a.gq <= 16)) a.few_rows = INT32_MAX;
    else a.few_rows = single || !a.table || a.n_seqs == 1 ? 0 : 16;
    auto splits = [&](int R, int wgs, int least) {
        const int64_t len = a.window > 0 ? std::min<int64_t>((int64_t)a.window + (R - 1) / a.gq, a.max_len) : a.max_len;
        const int64_t want = cdiv(wgs, std::max<int64_t>(most_tiles(a, R) * a.nkv, 1));
        return (int)std::max<int64_t>(1, std::min<int64_t>({want, cdiv(len, least), (int64_t)kMaxSplits}));
    };
    a.nsplit = a.few_rows > 0 ? splits(16, 512, 128) : 1;
    a.tile_split = a.few_rows < INT32_MAX ? splits(a.tile_rows, 256, 256) : 1;
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
        const int64_t grid = most_tiles(a, 16) * a.nkv * a.nsplit;
        k_seq_rows<T, D><<<(unsigned)grid, row_waves<D>() * kWave, 0, s>>>(a);
    }
    if (a.few_rows < INT32_MAX) launch_tiles(a, s);
    if (a.nparts > 1) {
        const int64_t th = (int64_t)a.n_tokens * a.nh;
        k_seq_join<T, D><<<(unsigned)cdiv(th, kJoinWaves), kJoinWaves * kWave, 0, s>>>(a);
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
    if (a.nparts > 1 && (!ws || !aligned16(ws) || split_bytes(a) > ws_bytes)) a.nsplit = a.tile_split = a.nparts = 1;
    a.ws = (float*)ws;
    a.inv_cap = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    // (never 0: a masked score of -inf times it stays -inf)
    a.unit = std::max(a.softcap > 0.0f ? kLog2e : kLog2e * std::fabs(a.scale), 1e-30f);
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
    a.max_len = (int)std::min<int64_t>(max_len, (int64_t)max_pages * page_size);
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
