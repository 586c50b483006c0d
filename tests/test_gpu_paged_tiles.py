"""The kernels that the many-sequence attention takes for larger calls, at sizes that reach each of them: tiles
of 256, 128 and 64 query rows, f32 products of three terms, splits of long ranges and their join, decode beside
chunks. A few tokens of every sequence are checked against float64."""
import numpy as np
import pytest

import seq_ref
from test_gpu_paged import MARK, Paged, TYPES, check, normals, rng_of, values_of
from ziglm_amd.device import Graph

pytestmark = pytest.mark.gpu


def some_tokens(m):
    return sorted({0, 1, 15, 16, 63, 64, 127, 128, 255, m // 3, m // 2, m - 2, m - 1} & set(range(m)))


def check_prompts(dev, act, nh, nkv, d, lens, cap=0.0, window=0, scale=None):
    rng = rng_of(21, nh, d, sum(lens))
    T, scale = sum(lens), scale or d ** -0.5
    (q, q64), (k, k64), (v, v64) = (normals(rng, (T, h, d), act) for h in (nh, nkv, nkv))
    cu = np.cumsum([0] + lens).astype(np.int32)
    dtype = TYPES[act][0]
    out = dev.alloc(q.nbytes)
    need = dev.attentionPromptWorkspaceBytes(dtype, len(lens), T, nh, nkv, d, window)
    ws = dev.alloc(max(need, 16))
    ws.fill(0xFF)
    dev.attentionPrompt(dtype, dev.from_numpy(q), dev.from_numpy(k), dev.from_numpy(v), out, nh * d, nkv * d, dev.from_numpy(cu), len(lens), T, nh,
                        nkv, d, scale, cap, window, ws, need)
    got = values_of(out.to_numpy(q.shape, q.dtype), act)
    assert np.isfinite(got).all()
    for s, m in enumerate(lens):
        for i in some_tokens(m):
            a = cu[s]
            lo = max(0, i + 1 - window) if window else 0
            ref, tol = seq_ref.attend_f64(q64[a + i:a + i + 1], k64[a + lo:a + i + 1], v64[a + lo:a + i + 1], i - lo, scale, cap, 0, bf16=act == "bf16")
            check(got[a + i:a + i + 1], ref, tol, (s, i))


@pytest.mark.parametrize("nh,nkv,d,lens,cap,window", [
    (16, 16, 64, [3000, 1, 1400, 99], 0.0, 0),      # 256 rows
    (32, 16, 128, [1300, 800], 0.0, 0),
    (32, 16, 128, [900, 1201], 30.0, 300),
    (8, 4, 256, [4000, 200], 0.0, 0),               # 128 rows
    (8, 4, 256, [2100, 2101], 0.0, 512),
    (8, 2, 64, [500, 77], 0.0, 0),                  # the smaller tiles
    (6, 2, 128, [333, 260], 20.0, 0),
    (10, 2, 256, [300, 41, 128], 0.0, 100),
    (8, 1, 512, [700, 65, 64], 0.0, 0),             # 64 rows, two waves each
    (3, 3, 512, [130], 0.0, 50)])
def test_bf16_prompts(dev, nh, nkv, d, lens, cap, window):
    check_prompts(dev, "bf16", nh, nkv, d, lens, cap, window)


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("nh,nkv,d", [(4, 2, 64), (4, 2, 128), (4, 2, 256), (2, 1, 512)])
@pytest.mark.parametrize("scale,cap", [(1.0, 5.0), (-0.3, 30.0), (1e-6, 1e-3), (1e12, 40.0), (0.05, 1e20)])
def test_capped_scores(dev, act, nh, nkv, d, scale, cap):
    """Small scores, scores at the cap, and some of both in one call: a few of a tile's rows are far larger."""
    check_prompts(dev, act, nh, nkv, d, [200, 70], cap, 0, scale)


@pytest.mark.parametrize("nh,nkv,d,lens,cap,window", [
    (16, 16, 64, [3500, 700], 0.0, 0),
    (32, 16, 128, [1500, 2, 600], 0.0, 0),
    (32, 16, 128, [1100, 1000], 25.0, 0),
    (8, 4, 256, [4100, 130], 0.0, 512),
    (8, 4, 256, [3000, 1300], 25.0, 200),
    (8, 1, 512, [600, 65], 0.0, 0)])
def test_f32_prompts(dev, nh, nkv, d, lens, cap, window):
    check_prompts(dev, "f32", nh, nkv, d, lens, cap, window)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,page,ctx,new,window", [
    (8, 4, 256, 16, [1501], [300], 0),
    (8, 4, 256, 7, [900, 2000, 30, 1200], [90, 1, 200, 1], 0),
    (32, 16, 128, 32, [700, 1900, 10, 64], [150, 1, 1, 33], 0),
    (16, 16, 64, 100, [3000, 5], [129, 256], 0),
    (8, 1, 512, 16, [1000, 400], [70, 1], 0),
    (40, 2, 64, 8, [100, 700], [20, 1], 0),
    (8, 4, 256, 64, [3000, 900, 100], [120, 1, 260], 333),
    (9, 3, 128, 1, [500, 0], [111, 64], 90)])
@pytest.mark.parametrize("split", [True, False])
def test_chunks_beside_decode(dev, act, nh, nkv, d, page, ctx, new, window, split):
    c = Paged(dev, 22, act, nh, nkv, d, page, ctx, new).upload()
    ws, need = c.workspace(window) if split else (None, 0)
    scale = d ** -0.5
    got = c.call(scale, 0.0, window, ws, need)
    for s in range(c.n):
        K, V = (values_of(x[c.rows(s)], act).reshape(-1, nkv, d) for x in (c.kc, c.vc))
        for i in some_tokens(c.new[s]):
            p = ctx[s] + i
            lo = max(0, p + 1 - window) if window else 0
            a = c.cu[s] + i
            ref, tol = seq_ref.attend_f64(c.q64[a:a + 1], K[lo:p + 1], V[lo:p + 1], p - lo, scale, bf16=act == "bf16")
            check(got[a:a + 1], ref, tol, (s, i))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 256), (4, 2, 128), (2, 2, 64), (8, 1, 512)])
def test_repeats_are_equal(dev, act, nh, nkv, d):
    """Sums are formed in one order: the same call gives the same bits."""
    c = Paged(dev, 23, act, nh, nkv, d, 16, [1200, 900, 40], [100, 1, 30]).upload()
    ws, need = c.workspace(0)
    first = c.call(0.07, 0.0, 0, ws, need)
    for _ in range(3):
        assert np.array_equal(first, c.call(0.07, 0.0, 0, ws, need))


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,ctx,new", [(8, 4, 128, 60, 200), (8, 1, 256, 300, 90), (4, 4, 64, 10, 300), (8, 1, 512, 50, 80), (8, 4, 128, 90, 1)])
def test_infinite_keys(dev, act, nh, nkv, d, ctx, new):
    """A key with an infinite component: where the query's component points away its score is -inf and its
    weight 0, where it points along the result is not a number. NaN keys show in every token that sees them."""
    c = Paged(dev, 24, act, nh, nkv, d, 16, [ctx], [new])
    rows = c.rows(0)
    j, bad, nan = d - 3, ctx // 2, ctx + new - 1
    inf = np.inf if act == "f32" else 0x7F80
    col = np.arange(nkv) * d + j
    c.kc[rows[bad]] = 0
    c.kc[rows[bad], col] = inf
    if new > 1:
        c.kc[rows[nan]] = np.nan if act == "f32" else 0x7FC0
    c.upload()
    ws, need = c.workspace(0)
    got = c.call(0.1, 0.0, 0, ws, need)
    K, V = (values_of(x[rows], act).reshape(-1, nkv, d) for x in (c.kc, c.vc))
    there = np.arange(ctx + new) != bad
    away = c.q64[:new, :, j] < 0
    for i in some_tokens(new):
        if new > 1 and i == new - 1:
            assert np.isnan(got[i]).all()
            continue
        p = ctx + i
        ref, tol = seq_ref.attend_f64(c.q64[i:i + 1], np.where(there[:, None, None], K, 0)[:p + 1], V[:p + 1], p, 0.1, there=there[:p + 1],
                                      bf16=act == "bf16")
        assert np.isnan(got[i][~away[i]]).all()
        check(got[i][away[i]], ref[0][away[i]], tol[0][away[i]], i)


@pytest.mark.parametrize("nh,nkv,d,ctx,new", [(8, 4, 128, 100, 200), (8, 1, 256, 40, 64), (2, 2, 64, 30, 300), (8, 4, 128, 500, 1)])
@pytest.mark.parametrize("size", [2.0 ** 60, 2.0 ** -60, 2.0 ** -110])
def test_sizes_of_f32_values(dev, nh, nkv, d, ctx, new, size):
    """Large and small values of V and, turned about, of q and K: products of terms keep their relative error."""
    c = Paged(dev, 25, "f32", nh, nkv, d, 16, [ctx], [new])
    c.vc = (c.vc * np.float32(size)).astype(np.float32)
    c.upload()
    got = c.call(d ** -0.5, 0.0, 0)
    rows = c.rows(0)
    K, V = (x[rows].astype(np.float64).reshape(-1, nkv, d) for x in (c.kc, c.vc))
    for i in some_tokens(new):
        ref, tol = seq_ref.attend_f64(c.q64[i:i + 1], K[:ctx + i + 1], V[:ctx + i + 1] / size, ctx + i, d ** -0.5)
        check(got[i:i + 1] / size, ref, tol, i)
    c.vc = (c.vc / np.float32(size)).astype(np.float32)
    c.kc = (c.kc * np.float32(size)).astype(np.float32)
    c.q = (c.q / np.float32(size)).astype(np.float32)
    c.upload()
    again = c.call(d ** -0.5, 0.0, 0)
    for i in some_tokens(new):
        ref, tol = seq_ref.attend_f64(c.q64[i:i + 1], K[:ctx + i + 1], V[:ctx + i + 1] / size, ctx + i, d ** -0.5)
        check(again[i:i + 1], ref, tol, i)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
@pytest.mark.parametrize("one", [True, False])
def test_scales(dev, act, scale, one):
    """Negative scales, none, and one that leaves a single key its weight."""
    c = Paged(dev, 26, act, 8, 4, 128, 16, [100, 400], [1, 1] if one else [40, 90], one=one).upload()
    ws, need = c.workspace(0)
    got = c.call(scale, 0.0, 0, ws, need)
    for s in range(2):
        out, tol = c.reference(s, scale, 0.0, 0)
        check(got[c.cu[s]:c.cu[s + 1]], out, tol, s)


def test_lengths_of_one_kind_told_as_many(dev):
    """As many tokens as sequences, but not one each: most have none."""
    for act in ("f32", "bf16"):
        c = Paged(dev, 27, act, 8, 2, 128, 16, [300, 20, 7, 900, 64, 3], [0, 4, 0, 2, 0, 0], extra=5)
        c.pad = 0
        c.q, c.q64 = c.q[:6], c.q64[:6]
        c.upload()
        ws, need = c.workspace(0)
        c.check(c.call(0.1, 0.0, 0, ws, need), 0.1, 0.0, 0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d,ctx,new", [(8, 4, 256, [300, 20, 512], [1, 1, 1]), (32, 16, 128, [700, 90], [100, 1]), (8, 1, 512, [80], [90])])
def test_bound_past_the_table(dev, act, nh, nkv, d, ctx, new):
    """max_len may be far past what the table can hold; the workspace is sized by it all the same."""
    c = Paged(dev, 28, act, nh, nkv, d, 16, ctx, new, one=max(new) == 1).upload()
    for most in (c.max_len + 1, 5000, 200000):
        ws, need = c.workspace(0, most)
        c.check(c.call(d ** -0.5, 0.0, 0, ws, need, most), d ** -0.5, 0.0, 0)
        c.check(c.call(d ** -0.5, 0.0, 0, ws, max(need - 1, 0), most), d ** -0.5, 0.0, 0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 256), (32, 16, 128), (8, 1, 512)])
def test_shared_pages(dev, act, nh, nkv, d):
    """Sequences that share the pages of a common beginning, and one that has a page twice."""
    c = Paged(dev, 29, act, nh, nkv, d, 16, [400, 500, 90, 300], [1, 120, 1, 40])
    c.table[1, :20] = c.table[0, :20]
    c.table[2, :5] = c.table[0, :5]
    c.table[3, 7] = c.table[3, 2]
    c.upload()
    ws, need = c.workspace(0)
    c.check(c.call(d ** -0.5, 0.0, 0, ws, need), d ** -0.5, 0.0, 0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 70, 3], [40, 150, 90]])
def test_first_rows_of_no_sequence(dev, act, new):
    """d_cu may begin past row 0: the rows before it stay as they are."""
    c = Paged(dev, 30, act, 8, 4, 128, 16, [300, 33, 5], new).upload()
    ws, need = c.workspace(0)
    c.d_cu = dev.from_numpy((c.cu + 3).astype(np.int32))
    front = c.q[:3].copy()
    c.q = np.concatenate([front, c.q])[:len(c.q)]  # the pad's rows move to the front
    c.q64 = np.concatenate([c.q64[:3], c.q64])[:len(c.q64)]
    c.d_q = dev.from_numpy(c.q)
    c.pad, pad = 0, c.pad
    c.tokens += pad
    raw = c.call(0.1, 0.0, 0, ws, need)
    mark = values_of(np.full(1, 0xABABABAB, np.uint32).view(c.q.dtype)[:1], act)[0]
    assert (raw[:3] == mark).all()
    c.q64 = c.q64[3:]
    c.check(raw[3:], 0.1, 0.0, 0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("nh,nkv,d", [(8, 4, 256), (32, 16, 128), (8, 1, 512)])
def test_chunks_beside_decode_in_a_graph(dev, act, nh, nkv, d):
    """Captured, then replayed for other lengths, positions and values in the same buffers."""
    c = Paged(dev, 31, act, nh, nkv, d, 16, [700, 40, 300], [1, 90, 1]).upload()
    ws, need = c.workspace(0, 1024)
    first = c.call(0.06, 0.0, 0, ws, need, 1024)
    call = (TYPES[act][0], c.d_q, c.d_k, c.d_v, c.out, c.pages, c.page, nkv * d, c.d_table, c.most, c.d_cu, c.d_len, c.n, c.tokens + c.pad, 1024,
            nh, nkv, d, 0.06, 0.0, 0, ws, need)
    dev.sync()
    graph = Graph(dev, lambda: dev.attentionPaged(*call))
    for shorter in (0, 25, 0, 39):
        lens = np.array([x - shorter for x in c.len], np.int32)
        c.d_len.upload(lens)
        c.out.fill(MARK)
        dev.sync()
        graph.launch()
        dev.sync()
        got = values_of(c.out.to_numpy(c.q.shape, c.q.dtype)[:c.tokens], act)
        if not shorter:
            assert np.array_equal(got, first)
            continue
        for s in range(c.n):
            rows = c.rows(s)[:lens[s]]
            K, V = (values_of(x[rows], act).reshape(-1, nkv, d) for x in (c.kc, c.vc))
            a = c.cu[s]
            ref, tol = seq_ref.attend_f64(c.q64[a:a + c.new[s]], K, V, c.ctx[s] - shorter, 0.06, bf16=act == "bf16")
            check(got[a:a + c.new[s]], ref, tol, (shorter, s))
    graph.destroy()
