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
#include "attention_rows.h"

namespace zl {

constexpr int kRowWaves = 4;
template <typename T, int D>
__global__ __launch_bounds__(row_halves<D>() * kRowWaves * kWave, 2) void k_seq_rows(SeqArgs a) {
    constexpr int W = kRowWaves;
    int id = (int)blockIdx.x;
    __shared__ __align__(16) float s_o[row_slots(D) * 16 * (D + 4)];
    __shared__ float s_m[W][16], s_l[W][16];
#include "attention_rows.inl"
}

// Joins the splits of a (token, head): out = sum_s exp(m_s - M) o_s / sum_s exp(m_s - M) l_s. W waves take
// a head, wave w splits w, w + W, ...: four where there can be many splits, one where there are few
// (and a workgroup four heads). The row's splits are those of the tile that formed them. The maxima
// and the first sums are requested before their number is known (slots behind it hold anything:
// they are dropped, not weighted by 0), which leaves one round trip to memory behind the sequence's own
// (one token: 3.9 us of its 14.4; 1330 tokens of 32 heads x 128 beside chunks 23 of 245, bound by the sums' bytes).
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
    const bool single = a.table && !a.cu;  // a token each
    const int few = f32 ? 64 : 16;
    const bool short32 = f32 && !a.table && (a.D == 512 || tiles_of(false) < (a.window > 0 ? 320 : 512));
    if (short32 || rows <= std::max<int64_t>(few, (int64_t)a.n_seqs * few / 2) || (single && a.gq <= few)) a.few_rows = INT32_MAX;
    else a.few_rows = single || !a.table || a.n_seqs == 1 ? 0 : few;
    // Prompts that leave CUs idle take smaller tiles (64 tokens, 8 / 4 heads x 256 bf16 13.4 -> 10.6 us, 512 of 32
    // / 16 x 128 26 -> 23.5; over the largest, 8192, the larger ones are ahead by 8%), and so do tiles in one
    // launch with rows, two of whose workgroups share a CU then (up to 40 sequences, up to three with chunks,
    // 32 / 16 heads x 128, geometric mean of eight calls: 96 us in two launches, 95 in one, 85 with small tiles).
    const bool both = a.few_rows > 0 && a.few_rows < INT32_MAX;
    a.tile_rows = tile_rows_of(dtype, a.D, both || (!a.table && tiles_of(false) < 256));

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
        // for several, whose lengths differ, as many as would give two to a CU if all were as long as the longest
        // (of small tiles two and a half: the calls above in four to a CU 85 us, in these 79; in two 77, but others,
        // whose longest tile is then not split, up to twice as long).
        const int64_t tiles = tiles_of(false), len = most_keys(a, a.tile_rows);
        const int64_t keys = a.n_seqs == 1 ? std::max<int64_t>(128, cdiv(len, 256 / tiles))
                                           : std::max<int64_t>(256, cdiv(tiles * len, a.tile_rows < tile_rows_of(dtype, a.D, false) ? 320 : 512));
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
    if (a.tile_grid > 0) launch_tiles(sizeof(T) == 4 ? HIP_BRIDGE_F32 : HIP_BRIDGE_BF16, a, s);
    else k_seq_rows<T, D><<<(unsigned)a.rows_grid, row_halves<D>() * kRowWaves * kWave, 0, s>>>(a);
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
    const float z1 = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;  // of a raw score of 1
    const float tanh_c[4] = {1.0f, -1.0f / 3.0f, 2.0f / 15.0f, -17.0f / 315.0f};
    for (int e = 0; e < 4; ++e) a.cap_c[e] = a.softcap * tanh_c[e] * std::pow(z1, (float)(2 * e + 1));
    a.cap_small = z1 == 0.0f || !(std::fabs(a.cap_c[3]) < INFINITY) ? -1.0f : 0.35f / std::fabs(z1);
    // (never 0: a masked score of -inf times it stays -inf)
    a.unit = dtype == HIP_BRIDGE_F32 || a.softcap > 0.0f ? kLog2e : std::max(kLog2e * std::fabs(a.scale), 1e-30f);
    const int64_t rows = a.few_rows > 0 ? most_few(a) * a.nkv * a.nsplit : 0;
    const int64_t tiles = a.few_rows < INT32_MAX ? most_tiles(a, a.tile_rows) * a.nkv * a.tile_split : 0;
    if ((rows + tiles) * 512 > UINT32_MAX || (a.nparts > 1 && (int64_t)a.n_tokens * a.nh * kWave * kJoinWaves > UINT32_MAX)) {
        set_error(HIP_BRIDGE_EUNSUPPORTED);
        return;
    }
    a.rows_grid = (int)rows;
    a.tile_grid = (int)tiles;
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
    // cache rows are 32-bit, and so are positions, a tile or two past the last included
    if (cache_pages > INT32_MAX / page_size || std::min<int64_t>(max_len, (int64_t)max_pages * page_size) > 1 << 30) {
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
