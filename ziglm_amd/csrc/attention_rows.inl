// The body of seq_rows (attention_rows.h) and of k_seq_rows (attention_seqs.hip): T, D and W (waves, or pairs of them),
// SeqArgs a, the workgroup's number id, s_o, s_m and s_l in LDS. It is included into the kernel, not called from
// it: as an inlined function the same text comes out of the compiler with its loads in another order (f32 prompts
// of 2048 tokens, 8 / 4 heads x 256: 117 us included, 124 called).
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
    constexpr int SLOTS = row_slots(D);
    constexpr float kSlack = 8.0f;               // log2: how far scores may pass the running maximum
    constexpr int XF = HV * NI * kWave * 4;  // floats of the query rows
    static_assert(HV == 1 || XF + 2 * HV * W * 4 * NT * kWave <= SLOTS * 16 * OS, "LDS");
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wave = wid % W, half = wid / W;
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
        for (int j = wave; j < NI; j += W) s_q[kWave * j] = ld16(qrow + 4 * EL * j) ^ flip;
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
    int row = wave < nblk ? rows_of(wave) : -1, next = wave + W < nblk ? rows_of(wave + W) : -1;
    load_k(row);
    load_v(row);
    __syncthreads();  // the query rows
    // (where waves exchange sums all of them go as many steps)
    const int steps = HV == 1 ? nblk : (nblk + W - 1) / W * W;
    for (int blk = wave; blk < steps; blk += W) {
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
            f32x4* const mine = reinterpret_cast<f32x4*>(s_o + XF) + ((blk / W & 1) * HV * W + wid) * NT * kWave + lane;
            const f32x4* const other = mine + (half ? -1 : 1) * W * NT * kWave;
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
        if (blk + 2 * W < nblk) next = rows_of(blk + 2 * W);
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
            if (k / BK % W != wave || key >= ke) continue;
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
        for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w][n]);
        const float f = __builtin_amdgcn_exp2f((m - (M == -INFINITY ? 0.0f : M)) * a.unit);
#pragma unroll
        for (int j = 0; j < NC * CW; ++j) o[j] *= f;
    }
    float* const slot = s_o + (wave % SLOTS * 16 + n) * OS + half * DW + 4 * CW * g;
#pragma unroll
    for (int w0 = 0; w0 < W; w0 += SLOTS) {
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
    for (int t = threadIdx.x; t < 16 * D / 4; t += HV * W * kWave) {
        const int rw = t / (D / 4), col = t % (D / 4) * 4;
        if (r0 + rw > r1) break;
        const int64_t tok = q.tok0 + (r0 + rw) / a.gq, h = kvh * a.gq + (r0 + rw) % a.gq;
        float M = s_m[0][rw], L = 0.0f;
#pragma unroll
        for (int w = 1; w < W; ++w) M = fmaxf(M, s_m[w][rw]);
#pragma unroll
        for (int w = 0; w < W; ++w)
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
