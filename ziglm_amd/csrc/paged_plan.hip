// The bookkeeping of one step of many requests over a paged KV cache: which pages their new tokens
// take, the block tables, every token's position and cache row (hip_paged_plan; no counterpart in
// the reference, whose cache is one contiguous range of one sequence, cuda_model.zig:213-217).
//
// Request s has ctx_s tokens in the cache and brings new_s. In the order of the requests, with
// h_s = ceil(ctx_s / page) pages held:
//   t_s = tokens of new_s that the table's width and the token buffer leave room for,
//   n_s = ceil((ctx_s + t_s) / page) - h_s pages wanted, f_s = n_0 + ... + n_(s-1) the first of them,
//   g_s = pages got: those of f_s .. f_s + n_s - 1 that the free list still has,
//   m_s = min(t_s, (h_s + g_s) * page - ctx_s) tokens taken in, cu_s = m_0 + ... + m_(s-1).
// Three prefix sums over the requests and then independent writes: page f_s + j of the free list is
// entry h_s + j of the table, token cu_s + i has position ctx_s + i.
//
// One launch: every workgroup forms the prefix sums for itself (256 requests at a time, each scan a
// wave scan and one exchange through LDS), which costs less than a second launch that reads them,
// and writes its share of the tokens and pages, each found by bisection in LDS. It is bound by that
// chain of latencies, not by its bytes: 64 requests of a token each 5.4 us, 250 with 65000 tokens 8.0 us.
#include <algorithm>

#include "zl_common.h"
#include "zl_host.h"

namespace zl {

constexpr int kPlanThreads = 256;   // requests of a pass over them
constexpr int kPlanSlice = 1024;    // tokens of a workgroup's turn
constexpr int kPlanMaxGrid = 1024;

struct PlanArgs {
    const int32_t* ctx;
    const int32_t* fresh;
    const int32_t* free_pages;
    const int32_t* cursor;
    int32_t* table;
    int32_t* cu;
    int32_t* len;
    int32_t* pos;
    int64_t* slot;
    int32_t* state;
    int n_seqs, page, max_pages, n_free, cap;
};

// Exclusive prefix sum of v over the workgroup's threads, and the sum of all in `total`.
__device__ __forceinline__ int64_t plan_scan(int64_t v, int64_t* s_wave, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // the previous scan's sums have been read
    if (lane == kWave - 1) s_wave[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
        if (w < wave) before += s_wave[w];
        total += s_wave[w];
    }
    return before + x - v;
}

// The last i of start[0, n) with start[i] <= x (start[0] <= x).
__device__ __forceinline__ int plan_find(const int* start, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PlanArgs a) {
    __shared__ int64_t s_wave[kPlanThreads / kWave];
    __shared__ int s_cu[kPlanThreads], s_first[kPlanThreads], s_have[kPlanThreads], s_ctx[kPlanThreads];
    const int tid = threadIdx.x, bid = blockIdx.x, grid = gridDim.x;
    const bool lead = bid == 0;
    const int cursor = a.cursor ? min(max(*a.cursor, 0), a.n_free) : 0;
    const int avail = a.n_free - cursor;
    const int64_t room = (int64_t)a.max_pages * a.page;
    int64_t asked = 0, dropped = 0, pages = 0;  // tokens asked for so far, left out, pages wanted
    int taken = 0, got_all = 0;                 // tokens taken in and pages got so far
    for (int s0 = 0; s0 < a.n_seqs; s0 += kPlanThreads) {
        const int s = s0 + tid, count = min(kPlanThreads, a.n_seqs - s0);
        const bool in = s < a.n_seqs;
        const int ctx = in ? max(a.ctx ? a.ctx[s] : 0, 0) : 0;
        const int want = in ? max(a.fresh[s], 0) : 0;
        int64_t total;
        // tokens that fit the table, then the token buffer
        int64_t m = min((int64_t)want, max(room - ctx, (int64_t)0));
        const int64_t before = asked + plan_scan(m, s_wave, total);
        asked += total;
        m = min(m, max((int64_t)a.cap - before, (int64_t)0));
        // pages
        const int have = (int)(((int64_t)ctx + a.page - 1) / a.page);
        const int need = (int)((ctx + m + a.page - 1) / a.page) - have;
        const int64_t first = pages + plan_scan(need, s_wave, total);
        pages += total;
        const int got = (int)min((int64_t)need, max(avail - first, (int64_t)0));
        m = min(m, (int64_t)(have + got) * a.page - ctx);
        const int got_end = (int)min(pages, (int64_t)avail);
        // tokens taken in
        const int64_t start = taken + plan_scan(m, s_wave, total);
        const int end = taken + (int)total;
        s_cu[tid] = (int)start;
        s_first[tid] = (int)min(first, (int64_t)a.n_free);
        s_have[tid] = have;
        s_ctx[tid] = ctx;
        if (lead && in) {
            a.cu[s] = (int)start;
            a.len[s] = ctx + (int)m;
        }
        if (lead) {
            plan_scan(want - m, s_wave, total);
            dropped += total;
        }
        __syncthreads();
        for (int k = got_all + bid * kPlanThreads + tid; k < got_end; k += grid * kPlanThreads) {
            const int i = plan_find(s_first, count, k);
            a.table[(int64_t)(s0 + i) * a.max_pages + s_have[i] + k - s_first[i]] = a.free_pages[cursor + k];
        }
        for (int64_t t0 = (int64_t)bid * kPlanSlice; t0 < end; t0 += (int64_t)grid * kPlanSlice) {
            const int t1 = (int)min(t0 + kPlanSlice, (int64_t)end);
            for (int t = max((int)t0, taken) + tid; t < t1; t += kPlanThreads) {
                const int i = plan_find(s_cu, count, t);
                const int p = s_ctx[i] + t - s_cu[i], e = p / a.page;
                // a fresh page's entry may not be written yet: it is the free list's
                const int id = e >= s_have[i] ? a.free_pages[cursor + s_first[i] + e - s_have[i]]
                                              : a.table[(int64_t)(s0 + i) * a.max_pages + e];
                a.pos[t] = p;
                a.slot[t] = id < 0 ? -1 : (int64_t)id * a.page + (p - e * a.page);
            }
        }
        taken = end;
        got_all = got_end;
        __syncthreads();  // the tables in LDS are read
    }
    for (int64_t t0 = (int64_t)bid * kPlanSlice; t0 < a.cap; t0 += (int64_t)grid * kPlanSlice) {
        const int t1 = (int)min(t0 + kPlanSlice, (int64_t)a.cap);
        for (int t = max((int)t0, taken) + tid; t < t1; t += kPlanThreads) {
            a.pos[t] = -1;
            a.slot[t] = -1;
        }
    }
    if (lead && tid == 0) {
        a.cu[a.n_seqs] = taken;
        a.state[0] = cursor + got_all;
        a.state[1] = (int)min(dropped, (int64_t)INT32_MAX);
    }
}

}  // namespace zl

using namespace zl;

extern "C" void hip_paged_plan(const int32_t* d_ctx_len, const int32_t* d_new_len, int n_seqs, int page_size,
                               int max_pages, const int32_t* d_free_pages, int n_free, const int32_t* d_cursor,
                               int32_t* d_block_table, int n_tokens, int32_t* d_cu, int32_t* d_seq_len, int32_t* d_pos,
                               int64_t* d_slot, int32_t* d_state, HipStream_t stream) {
    if (n_seqs <= 0 || n_tokens <= 0) return;
    if (!d_new_len || !d_block_table || !d_cu || !d_seq_len || !d_pos || !d_slot || !d_state || page_size <= 0 ||
        max_pages <= 0 || n_free < 0 || (n_free > 0 && !d_free_pages) || d_seq_len == d_ctx_len ||
        d_seq_len == d_new_len || d_state == d_cursor) {
        set_error(HIP_BRIDGE_EINVAL);
        return;
    }
    if ((int64_t)max_pages * page_size > INT32_MAX) {  // positions are 32-bit
        set_error(HIP_BRIDGE_EUNSUPPORTED);
        return;
    }
    PlanArgs a{d_ctx_len, d_new_len, d_free_pages, d_cursor, d_block_table, d_cu,   d_seq_len, d_pos,
               d_slot,    d_state,   n_seqs,       page_size, max_pages,    n_free, n_tokens};
    const int64_t grid = std::min<int64_t>(cdiv(n_tokens, kPlanSlice), kPlanMaxGrid);
    k_paged_plan<<<(unsigned)grid, kPlanThreads, 0, stream_of(stream)>>>(a);
    check_launch();
}
