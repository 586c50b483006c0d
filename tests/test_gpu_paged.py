"""Operators of many sequences over a paged KV cache (hip_paged_plan, hip_attention_paged) and of packed
prompts (hip_attention_prompt) against plain 64-bit references (seq_ref), at ragged lengths, page sizes that
end inside every tile, windows, soft-caps, pages and rows that hold nothing, and as a serving loop runs
them together."""
import numpy as np
import pytest

import seq_ref
from ziglm_amd import bridge as B
from ziglm_amd import synth
from ziglm_amd.bridge import HipError
from ziglm_amd.device import Graph, HipDevice

pytestmark = pytest.mark.gpu
MARK = 0xAB  # bytes of buffers before a call


def rng_of(*key):
    return np.random.default_rng([int(x) for x in key])


# ---- plan ------------------------------------------------------------------------------------

def plan_on(dev, ctx, new, page, most, free, cursor, table, cap):
    n = len(new)
    o = {"cu": (n + 1, np.int32), "len": (n, np.int32), "pos": (cap, np.int32), "slot": (cap, np.int64), "state": (2, np.int32)}
    bufs = {k: dev.alloc(m * np.dtype(t).itemsize) for k, (m, t) in o.items()}
    for x in bufs.values():
        x.fill(MARK)
    d_table = dev.from_numpy(table)
    d_cursor = None if cursor is None else dev.from_numpy(np.array([cursor], np.int32))
    d_ctx = None if ctx is None else dev.from_numpy(np.array(ctx, np.int32))
    d_new, d_free = dev.from_numpy(np.array(new, np.int32)), dev.from_numpy(free) if len(free) else None
    dev.pagedPlan(d_ctx, d_new, n, page, most, d_free, len(free), d_cursor, d_table, cap, bufs["cu"], bufs["len"], bufs["pos"],
                  bufs["slot"], bufs["state"])
    got = {k: bufs[k].to_numpy((m,), t) for k, (m, t) in o.items()}
    got["table"] = d_table.to_numpy(table.shape, np.int32)
    return got


@pytest.mark.parametrize("n,most_new,page,room,share,pad", [
    (1, 1, 16, 20, 1.5, 0), (1, 5000, 1, 9000, 1.0, 3), (64, 1, 16, 400, 1.2, 0), (7, 40, 7, 30, 0.5, 9), (300, 90, 16, 20, 0.9, 100),
    (257, 3, 64, 4, 1.0, 0), (700, 200, 32, 12, 1.1, 1000), (256, 1, 1, 70, 0.0, 5), (33, 2000, 256, 10, 1.0, 1)])
@pytest.mark.parametrize("cap", ["all", "short"])
def test_plan(dev, n, most_new, page, room, share, pad, cap):
    rng = rng_of(n, most_new, page)
    most = room
    ctx = rng.integers(0, page * room // 2 + 2, n).astype(np.int32)
    new = rng.integers(0 if n > 1 else most_new, most_new + 1, n).astype(np.int32)
    if n > 6:
        ctx[1], new[2], ctx[3], new[4] = -3, -9, 0, 0
        ctx[5] = page * most  # full
    want = int(sum(-(-(max(c, 0) + max(m, 0)) // page) - -(-max(c, 0) // page) for c, m in zip(ctx, new)))
    free = rng.permutation(want + 50).astype(np.int32)[:int(want * share) + 3]
    table = rng.integers(0, 1000, (n, most)).astype(np.int32)
    table[:, -1] = -1  # (a held page that is nowhere)
    total = int(np.maximum(new, 0).sum())
    size = max(1, total + pad if cap == "all" else total * 2 // 3)
    ref = seq_ref.plan(ctx, new, page, most, free, 2, table, size)
    got = plan_on(dev, ctx, new, page, most, free, 2, table, size)
    for k, v in ref.items():
        assert np.array_equal(got[k], v), k


def test_plan_without_context_cursor_or_pages(dev):
    new = np.array([3, 0, 17, 1], np.int32)
    table = np.full((4, 2), -1, np.int32)
    for free in (np.arange(5, dtype=np.int32)[::-1].copy(), np.zeros(0, np.int32)):
        got = plan_on(dev, None, new, 16, 2, free, None, table, 30)
        ref = seq_ref.plan([0] * 4, new, 16, 2, free, 0, table, 30)
        for k, v in ref.items():
            assert np.array_equal(got[k], v), k


# ---- attention -------------------------------------------------------------------------------

TYPES = {"f32": (B.F32, np.float32), "bf16": (B.BF16, np.uint16)}


def normals(rng, shape, act, std=1.0):
    """(values as stored, as float64)"""
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    if act == "f32":
        return x, x.astype(np.float64)
    u = synth.f32_to_bf16(x)
    return u, synth.bf16_to_f32(u).astype(np.float64)


def values_of(raw, act):
    return raw.astype(np.float64) if act == "f32" else synth.bf16_to_f32(raw).astype(np.float64)


def check(got, ref, tol, what):
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.nanmax(np.where(bad, np.abs(got - ref) / tol, 0)))


class Paged:
    """A paged cache with ragged sequences on the device and their float64 values."""

    def __init__(self, dev, seed, act, nh, nkv, d, page, ctx, new, one=False, extra=2, fill=0):
        rng = rng_of(seed, nh, nkv, d, page)
        self.dev, self.act, self.nh, self.nkv, self.d, self.page, self.one = dev, act, nh, nkv, d, page, one
        self.ctx, self.new = list(ctx), list(new)
        self.n = len(ctx)
        self.len = [c + m for c, m in zip(ctx, new)]
        held = [-(-x // page) for x in self.len]
        self.pages = sum(held) + extra
        self.most = max(held + [1]) + 1
        ids = rng.permutation(self.pages)
        self.table = np.full((self.n, self.most), 2 ** 31 - 1, np.int32)  # entries behind a sequence are nonsense
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = ids[at:at + h]
            at += h
        dt = np.float32 if act == "f32" else np.uint16
        nan = np.float32(np.nan) if act == "f32" else np.uint16(0x7FC0)
        self.kc = np.full((self.pages * page, nkv * d), nan, dt)  # rows that nobody wrote
        self.vc = self.kc.copy()
        for s in range(self.n):
            rows = self.rows(s)
            self.kc[rows], _ = normals(rng, (len(rows), nkv * d), act)
            self.vc[rows], _ = normals(rng, (len(rows), nkv * d), act)
        self.tokens = sum(new)
        self.pad = 0 if one else 3
        self.q, self.q64 = normals(rng, (self.tokens + self.pad, nh, d), act)
        self.cu = np.cumsum([0] + self.new).astype(np.int32)
        self.max_len = max(self.len)

    def rows(self, s):
        t = np.arange(self.len[s])
        return self.table[s, t // self.page].astype(np.int64) * self.page + t % self.page

    def upload(self):
        f = self.dev.from_numpy
        self.d_q, self.d_k, self.d_v, self.d_table = f(self.q), f(self.kc), f(self.vc), f(self.table)
        self.d_cu, self.d_len = f(self.cu), f(np.array(self.len, np.int32))
        self.out = self.dev.alloc(self.q.nbytes)
        self.out.fill(MARK)
        return self

    def workspace(self, window, max_len=None):
        need = self.dev.attentionPagedWorkspaceBytes(TYPES[self.act][0], self.n, self.tokens + self.pad, max_len or self.max_len, self.nh, self.nkv,
                                                     self.d, window)
        ws = self.dev.alloc(max(need, 16))
        ws.fill(0xFF)  # NaN
        return ws, need

    def call(self, scale, cap, window, ws=None, need=0, max_len=None):
        self.dev.attentionPaged(TYPES[self.act][0], self.d_q, self.d_k, self.d_v, self.out, self.pages, self.page, self.nkv * self.d,
                                self.d_table, self.most, None if self.one else self.d_cu, self.d_len, self.n, self.tokens + self.pad,
                                max_len or self.max_len, self.nh, self.nkv, self.d, scale, cap, window, ws, need)
        raw = self.out.to_numpy(self.q.shape, self.q.dtype)
        if self.pad:
            assert (raw[self.tokens:].view(np.uint8) == MARK).all(), "rows behind the last sequence"
        return values_of(raw[:self.tokens], self.act)

    def reference(self, s, scale, cap, window, there=None, lim=None):
        rows = np.maximum(self.rows(s), 0)
        K, V = (values_of(c[rows], self.act).reshape(-1, self.nkv, self.d) for c in (self.kc, self.vc))
        a = self.cu[s]
        return seq_ref.attend_f64(self.q64[a:a + self.new[s]], K, V, self.ctx[s], scale, cap, window, there, lim, self.act == "bf16")

    def check(self, got, scale, cap, window, lim=None):
        for s in range(self.n):
            if self.new[s]:
                out, tol = self.reference(s, scale, cap, window, lim=lim)
                check(got[self.cu[s]:self.cu[s + 1]], out, tol, f"sequence {s}")


HEADS = [(8, 4, 256), (32, 16, 128), (8, 1, 256), (8, 1, 512), (6, 2, 64), (12, 1, 128), (5, 5, 64), (40, 2, 64)]


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("page,cap,window", [(16, 0.0, 0), (7, 20.0, 0), (32, 0.0, 33), (1, 0.0, 1), (100, 30.0, 150)])
def test_single_tokens(dev, nh, nkv, d, act, page, cap, window):
    c = Paged(dev, 1, act, nh, nkv, d, page, [0, 1, 15, 16, 17, 300, 611, 63], [1] * 8, one=True).upload()
    ws, need = c.workspace(window)
    c.check(c.call(d ** -0.5, cap, window, ws, need), d ** -0.5, cap, window)
    c.check(c.call(d ** -0.5, cap, window), d ** -0.5, cap, window)


@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("page,cap,window", [(16, 0.0, 0), (9, 20.0, 0), (64, 0.0, 40)])
def test_chunks(dev, nh, nkv, d, act, page, cap, window):
    ctx, new = [0, 130, 5, 64, 0, 333, 40, 1], [1, 37, 0, 1, 65, 2, 16, 150]
    c = Paged(dev, 2, act, nh, nkv, d, page, ctx, new).upload()
    ws, need = c.workspace(window)
    c.check(c.call(d ** -0.5, cap, window, ws, need), d ** -0.5, cap, window)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,n,longest", [(8, 1, 128, 1, 9000), (4, 2, 256, 3, 5000), (2, 2, 64, 2, 20000)])
def test_long_contexts_are_split(dev, act, nh, nkv, d, n, longest):
    rng = rng_of(longest)
    c = Paged(dev, 3, act, nh, nkv, d, 16, [longest] + list(rng.integers(0, longest, n - 1)), [1] * n, one=True).upload()
    ws, need = c.workspace(0)
    assert need > 0
    got = c.call(d ** -0.5, 0.0, 0, ws, need)
    c.check(got, d ** -0.5, 0.0, 0)
    c.check(c.call(d ** -0.5, 0.0, 0, ws, need - 1), d ** -0.5, 0.0, 0)  # too small: unsplit
    again = c.call(d ** -0.5, 0.0, 0, ws, need)
    assert np.array_equal(got, again)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,m", [(8, 2, 128, 3), (8, 1, 256, 40), (4, 4, 64, 200)])
def test_chunk_behind_a_long_context(dev, act, nh, nkv, d, m):
    c = Paged(dev, 4, act, nh, nkv, d, 16, [3000], [m]).upload()
    ws, need = c.workspace(0)
    got = c.call(d ** -0.5, 0.0, 0, ws, need)
    out, tol = c.reference(0, d ** -0.5, 0.0, 0)
    check(got, out, tol, "chunk")


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("one", [True, False])
def test_pages_that_are_nowhere(dev, act, one):
    """Pages outside the cache hold no keys; a token that sees no other gives zeros."""
    nh, nkv, d, page = 8, 4, 128, 16
    c = Paged(dev, 5, act, nh, nkv, d, page, [200, 40, 0], [1, 1, 1] if one else [70, 33, 30], one=one)
    good = c.table.copy()
    c.table[0, 3], c.table[0, 5], c.table[1, :], c.table[2, 0] = -1, c.pages, -7, 2 ** 31 - 1
    c.upload()
    ws, need = c.workspace(0)
    got = c.call(0.1, 0.0, 0, ws, need)
    c.table = good
    for s, lost in ((0, (3, 5)), (1, range(100)), (2, (0,))):
        there = ~np.isin(np.arange(c.len[s]) // page, list(lost))
        out, tol = c.reference(s, 0.1, 0.0, 0, there=there)
        g = got[c.cu[s]:c.cu[s + 1]]
        check(g, out, tol, s)
        if s == 1:
            assert (g == 0).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_positions_past_the_bounds_give_zeros(dev, act):
    c = Paged(dev, 6, act, 4, 2, 64, 16, [90, 0], [40, 12]).upload()
    ws, need = c.workspace(0)
    c.check(c.call(0.1, 0.0, 0, ws, need, max_len=100), 0.1, 0.0, 0, lim=100)
    # fewer positions than new tokens: the first of them stand before the sequence
    c.d_len.upload(np.array([130, 5], np.int32))
    got = c.call(0.1, 0.0, 0, ws, need)
    assert (got[40:47] == 0).all()
    K, V = (values_of(x[c.rows(1)[:5]], act).reshape(-1, 2, 64) for x in (c.kc, c.vc))
    out, tol = seq_ref.attend_f64(c.q64[40:52], K, V, -7, 0.1, bf16=act == "bf16")
    check(got[40:52], out, tol, "short")
    c.d_len.upload(np.array([-2 ** 31, 0], np.int32))
    assert (c.call(0.1, 0.0, 0, ws, need) == 0).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 128), (8, 1, 256), (4, 4, 64), (8, 1, 512)])
@pytest.mark.parametrize("window", [0, 24])
def test_values_that_only_some_tokens_see(dev, act, nh, nkv, d, window):
    """Infinite or NaN rows of later tokens, and of ones before the window, do not reach a token; a token
    that sees one shows it."""
    c = Paged(dev, 7, act, nh, nkv, d, 16, [100], [160])
    inf, nan = (np.inf, np.nan) if act == "f32" else (0x7F80, 0x7FC0)
    rows = c.rows(0)
    bad = 190  # position
    c.vc[rows[bad]] = inf
    c.kc[rows[bad + 1]] = nan
    c.vc[rows[5]] = 0 if not window else inf
    c.upload()
    ws, need = c.workspace(window)
    got = c.call(0.05, 0.0, window, ws, need)
    out, tol = c.reference(0, 0.05, 0.0, window)
    fine = [i for i in range(160) if 100 + i < bad or (window and 100 + i >= bad + 1 + window)]
    check(got[fine], out[fine], tol[fine], "tokens that see none")
    assert np.isinf(got[bad - 100]).all() and np.isnan(got[bad + 1 - 100]).all()


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_a_poisoned_query_stays_in_its_row(dev, act):
    c = Paged(dev, 8, act, 8, 4, 128, 16, [40, 3], [20, 5])
    c.q[3, 2], c.q64[3, 2] = (np.nan if act == "f32" else 0x7FC0), np.nan
    c.upload()
    got = c.call(0.1, 0.0, 0)
    assert np.isnan(got[3, 2]).all()
    c.q64[3, 2] = 0
    out, tol = c.reference(0, 0.1, 0.0, 0)
    keep = np.ones((20, 8), bool)
    keep[3, 2] = False
    check(got[:20][keep], out[keep], tol[keep], "others")


def test_offsets_past_32_bits(dev):
    """Pages at the far end of caches of more than 2^31 elements."""
    nkv, d, page = 16, 128, 64
    pages = 2 ** 31 // (nkv * d * page) + 3
    dev_k, dev_v = (dev.alloc(pages * page * nkv * d * 2) for _ in range(2))
    rng = rng_of(9)
    k, k64 = normals(rng, (2 * page, nkv * d), "bf16")
    v, v64 = normals(rng, (2 * page, nkv * d), "bf16")
    off = (pages - 2) * page * nkv * d * 2
    for buf, x in ((dev_k, k), (dev_v, v)):
        buf.at(off).upload(x)
    q, q64 = normals(rng, (1, 16, d), "bf16")
    table, length = dev.from_numpy(np.array([[pages - 1, pages - 2]], np.int32)), dev.from_numpy(np.array([100], np.int32))
    out = dev.alloc(q.nbytes)
    dev.attentionPaged(B.BF16, dev.from_numpy(q), dev_k, dev_v, out, pages, page, nkv * d, table, 2, None, length, 1, 1, 128, 16, nkv, d,
                       0.1, 0.0, 0)
    at = np.r_[page:2 * page, 0:36]
    ref, tol = seq_ref.attend_f64(q64, k64[at].reshape(-1, nkv, d), v64[at].reshape(-1, nkv, d), 99, 0.1, bf16=True)
    check(values_of(out.to_numpy(q.shape, np.uint16), "bf16"), ref, tol, "far pages")


# ---- packed prompts --------------------------------------------------------------------------

@pytest.mark.parametrize("nh,nkv,d", HEADS)
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("cap,window", [(0.0, 0), (20.0, 0), (0.0, 50), (0.0, 1)])
def test_prompts(dev, nh, nkv, d, act, cap, window):
    lens = [1, 70, 0, 129, 2, 16, 200]
    rng = rng_of(10, nh, d)
    T, wide = sum(lens), (nh + 2 * nkv) * d + 64
    raw, x64 = normals(rng, (T + 2, wide), act)
    dtype, es = TYPES[act][0], raw.itemsize
    buf, out = dev.from_numpy(raw), dev.alloc((T + 2) * nh * d * es)
    out.fill(MARK)
    cu = np.cumsum([0] + lens).astype(np.int32)
    need = dev.attentionPromptWorkspaceBytes(dtype, len(lens), T + 2, nh, nkv, d, window)
    ws = dev.alloc(max(need, 16))
    ws.fill(0xFF)
    # q, k and v side by side in one row
    dev.attentionPrompt(dtype, buf, buf.at(nh * d * es), buf.at((nh + nkv) * d * es), out, wide, wide, dev.from_numpy(cu), len(lens), T + 2,
                        nh, nkv, d, d ** -0.5, cap, window, ws, need)
    raw_out = out.to_numpy((T + 2, nh, d), raw.dtype)
    assert (raw_out[T:].view(np.uint8) == MARK).all()
    got = values_of(raw_out[:T], act)
    q, k, v = np.split(x64[:, :wide - 64], [nh * d, (nh + nkv) * d], 1)
    for s, m in enumerate(lens):
        if m:
            a, e = cu[s], cu[s + 1]
            ref, tol = seq_ref.attend_f64(q[a:e].reshape(m, nh, d), k[a:e].reshape(m, nkv, d), v[a:e].reshape(m, nkv, d), 0, d ** -0.5, cap,
                                          window, bf16=act == "bf16")
            check(got[a:e], ref, tol, f"prompt {s}")


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,T", [(8, 1, 256, 37), (4, 2, 128, 700), (2, 1, 64, 1100), (8, 1, 512, 150), (16, 16, 64, 400)])
def test_one_prompt(dev, act, nh, nkv, d, T):
    rng = rng_of(11, T)
    (q, q64), (k, k64), (v, v64) = (normals(rng, (T, h, d), act) for h in (nh, nkv, nkv))
    out = dev.alloc(q.nbytes)
    dev.attentionPrompt(TYPES[act][0], dev.from_numpy(q), dev.from_numpy(k), dev.from_numpy(v), out, nh * d, nkv * d, None, 1, T, nh, nkv, d,
                        d ** -0.5, 0.0, 0)
    got = values_of(out.to_numpy(q.shape, q.dtype), act)
    ref, tol = seq_ref.attend_f64(q64, k64, v64, 0, d ** -0.5, bf16=act == "bf16")
    check(got, ref, tol, "prompt")


def test_non_finite_rows_of_another_prompt(dev):
    """Prompts stand side by side in one buffer: none sees another's rows, not inside a tile either."""
    nh, nkv, d, lens = 4, 2, 128, [30, 21, 50]
    for act in ("f32", "bf16"):
        rng = rng_of(12)
        T = sum(lens)
        (q, q64), (k, k64), (v, v64) = (normals(rng, (T, h, d), act) for h in (nh, nkv, nkv))
        k[30:51], v[30:51] = (np.nan, np.inf) if act == "f32" else (0x7FC0, 0x7F80)
        cu, out = np.array([0, 30, 51, 101], np.int32), dev.alloc(q.nbytes)
        dev.attentionPrompt(TYPES[act][0], dev.from_numpy(q), dev.from_numpy(k), dev.from_numpy(v), out, nh * d, nkv * d, dev.from_numpy(cu), 3, T,
                            nh, nkv, d, 0.1, 0.0, 0)
        got = values_of(out.to_numpy(q.shape, q.dtype), act)
        for a, e in ((0, 30), (51, 101)):
            ref, tol = seq_ref.attend_f64(q64[a:e], k64[a:e], v64[a:e], 0, 0.1, bf16=act == "bf16")
            check(got[a:e], ref, tol, (act, a))
        assert np.isnan(got[30:51]).all()


# ---- together --------------------------------------------------------------------------------

@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_serving_loop(dev, act):
    """Plan, QK-norm + RoPE + append into the pages, attention, over three steps of prompts, chunks and single
    tokens, against the same requests on contiguous caches of their own through hip_qk_norm_rope_kv and a 64-bit
    attention. Requests come in late, stop, and run into the end of the free list."""
    nh, nkv, d, page, most, pool, n = 8, 4, 128, 16, 8, 16, 5
    dtype, es = TYPES[act][0], 4 if act == "f32" else 2
    rng = rng_of(13)
    wq, wk = (dev.from_numpy((rng.standard_normal(d) * 0.1).astype(np.float32)) for _ in range(2))
    cap = 64
    kc, vc = (dev.alloc(pool * page * nkv * d * es) for _ in range(2))
    kc.fill(0xFF)
    vc.fill(0xFF)
    table = dev.from_numpy(np.full((n, most), -1, np.int32))
    free = dev.from_numpy(rng.permutation(pool).astype(np.int32))
    lens = [dev.from_numpy(np.zeros(n, np.int32)), dev.alloc(4 * n)]
    states = [dev.from_numpy(np.zeros(2, np.int32)), dev.alloc(8)]
    cu, pos, slot = dev.alloc(4 * (n + 1)), dev.alloc(4 * cap), dev.alloc(8 * cap)
    ctx, at = [0] * n, 0
    alone = [(dev.alloc(most * page * nkv * d * es), dev.alloc(most * page * nkv * d * es)) for _ in range(n)]
    h_table, h_free = table.to_numpy((n, most), np.int32), free.to_numpy((pool,), np.int32)
    for step, new in enumerate(([30, 0, 7, 1, 20], [1, 40, 1, 16, 1], [1, 1, 33, 1, 0], [25, 25, 25, 25, 25])):
        ref = seq_ref.plan(ctx, new, page, most, h_free, at, h_table, cap)
        q, _ = normals(rng, (cap, nh, d), act)
        k, _ = normals(rng, (cap, nkv, d), act)
        v, _ = normals(rng, (cap, nkv, d), act)
        d_q, d_k, d_v, out = dev.from_numpy(q), dev.from_numpy(k), dev.from_numpy(v), dev.alloc(q.nbytes)
        out.fill(MARK)
        before, after = lens[step % 2], lens[1 - step % 2]
        dev.pagedPlan(before, dev.from_numpy(np.array(new, np.int32)), n, page, most, free, pool, states[step % 2], table, cap, cu, after, pos,
                      slot, states[1 - step % 2])
        dev.qkNormRopeKv(dtype, d_q, d_k, d_v, wq, wk, 0, kc, vc, pool * page, 0, pool * page, nkv * d, pos, 0, slot, cap, nh, nkv, d, 0, 10000.0,
                         1.0, 1e-6, True)
        need = dev.attentionPagedWorkspaceBytes(dtype, n, cap, most * page, nh, nkv, d, 0)
        ws = dev.alloc(max(need, 16))
        dev.attentionPaged(dtype, d_q, kc, vc, out, pool, page, nkv * d, table, most, cu, after, n, cap, most * page, nh, nkv, d, d ** -0.5, 0.0, 0,
                           ws, need)
        for name, buf, shape, t in (("cu", cu, (n + 1,), np.int32), ("len", after, (n,), np.int32), ("pos", pos, (cap,), np.int32),
                                    ("slot", slot, (cap,), np.int64), ("table", table, (n, most), np.int32)):
            assert np.array_equal(buf.to_numpy(shape, t), ref[name]), (step, name)
        assert np.array_equal(states[1 - step % 2].to_numpy((2,), np.int32), ref["state"])
        got = out.to_numpy(q.shape, q.dtype)
        assert (got[ref["cu"][-1]:].view(np.uint8) == MARK).all()
        for s in range(n):
            a, e = int(ref["cu"][s]), int(ref["cu"][s + 1])
            if e == a:
                continue
            m = e - a
            d_q1 = dev.from_numpy(q[a:e])
            dev.qkNormRopeKv(dtype, d_q1, dev.from_numpy(k[a:e]), dev.from_numpy(v[a:e]), wq, wk, 0, alone[s][0], alone[s][1], most * page, 0,
                             most * page, nkv * d, None, ctx[s], None, m, nh, nkv, d, 0, 10000.0, 1.0, 1e-6, True)
            L = ctx[s] + m
            K, V = (values_of(x.to_numpy((L, nkv, d), q.dtype), act) for x in alone[s])
            out64, tol = seq_ref.attend_f64(values_of(d_q1.to_numpy((m, nh, d), q.dtype), act), K, V, ctx[s], d ** -0.5, bf16=act == "bf16")
            check(values_of(got[a:e], act), out64, tol, (step, s))
        h_table, at, ctx = ref["table"], int(ref["state"][0]), [int(x) for x in ref["len"]]
    assert ref["state"][1] > 0  # the last step asked for more than the pool has


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_captured_step(dev, act):
    """Plan and attention captured once and replayed with other lengths, eager work in between; two graphs with a
    workspace each."""
    nh, nkv, d, page, n = 8, 2, 128, 16, 6
    dtype, es = TYPES[act][0], 4 if act == "f32" else 2
    c = Paged(dev, 14, act, nh, nkv, d, page, [0] * n, [1500] * n, extra=40)
    c.new, c.one, c.pad, c.tokens = [1] * n, True, 0, n
    c.q, c.q64, c.cu = c.q[:n], c.q64[:n], np.arange(n + 1, dtype=np.int32)
    c.upload()
    max_len = 1500
    steps, keep = [], []
    for g in range(2):
        ctx, new = dev.from_numpy(np.zeros(n, np.int32)), dev.from_numpy(np.ones(n, np.int32))
        bufs = [dev.alloc(4 * (n + 1)), dev.alloc(4 * n), dev.alloc(4 * n), dev.alloc(8 * n), dev.alloc(8)]
        table = dev.from_numpy(c.table)
        ws, need = c.workspace(0, max_len)
        assert need > 0
        out = dev.alloc(c.q.nbytes)

        def body(ctx=ctx, new=new, bufs=bufs, table=table, ws=ws, need=need, out=out):
            dev.pagedPlan(ctx, new, n, page, c.most, None, 0, None, table, n, *bufs)
            dev.attentionPaged(dtype, c.d_q, c.d_k, c.d_v, out, c.pages, page, nkv * d, table, c.most, None, bufs[1], n, n, max_len, nh, nkv, d,
                               0.1, 0.0, 0, ws, need)
        dev.sync()
        steps.append((ctx, bufs, out, Graph(dev, body)))
        keep.append((new, table, ws))  # the graph's buffers live as long as it
    rng = rng_of(15)
    for _ in range(3):
        at = [rng.integers(0, 90, n) * page + rng.integers(1, page, n) for _ in steps]  # inside a page: no new one is needed
        for (ctx, _, _, graph), x in zip(steps, at):
            ctx.upload(x.astype(np.int32))
            dev.sync()
            graph.launch()
        c.ctx = list(at[0])
        c.len = [int(x) + 1 for x in at[0]]
        c.d_len.upload(np.array(c.len, np.int32))
        ws, need = c.workspace(0, max_len)
        eager = c.call(0.1, 0.0, 0, ws, need, max_len=max_len)
        for (ctx, bufs, out, _), x in zip(steps, at):
            assert np.array_equal(bufs[1].to_numpy((n,), np.int32), x + 1)
            got = values_of(out.to_numpy(c.q.shape, c.q.dtype), act)
            if x is at[0]:
                assert np.array_equal(got, eager)
            c.ctx, c.len = [int(y) for y in x], [int(y) + 1 for y in x]
            c.check(got, 0.1, 0.0, 0)
    for *_, graph in steps:
        graph.destroy()


def test_on_another_stream(dev):
    """A second device object (a stream of its own) beside the first."""
    other = HipDevice()
    a = Paged(dev, 16, "f32", 8, 4, 128, 16, [500, 20], [1, 1], one=True).upload()
    b = Paged(other, 17, "f32", 8, 4, 128, 16, [90, 700], [1, 1], one=True).upload()
    wa, wb = a.workspace(0), b.workspace(0)
    for _ in range(3):
        ga, gb = a.call(0.1, 0.0, 0, *wa), b.call(0.1, 0.0, 0, *wb)
        a.check(ga, 0.1, 0.0, 0)
        b.check(gb, 0.1, 0.0, 0)
    other.deinit()


def test_refusals_raise(dev):
    c = Paged(dev, 18, "f32", 8, 4, 128, 16, [5], [1], one=True).upload()
    with pytest.raises(HipError):
        dev.attentionPaged(B.F16, c.d_q, c.d_k, c.d_v, c.out, c.pages, 16, 512, c.d_table, c.most, None, c.d_len, 1, 1, 6, 8, 4, 128, 0.1, 0.0, 0)
    assert (c.out.to_numpy(c.q.shape, np.uint32) == 0xABABABAB).all()
