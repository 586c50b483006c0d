"""Calls of the many-sequence operators that are refused before anything is launched: wrong sizes,
missing buffers, unsupported types, sizes and alignments, outputs that overlap inputs. No GPU is needed
(the pointers are never followed)."""
import pytest

from ziglm_amd import bridge as B

P = 0x10000  # an address that only looks like a buffer


@pytest.fixture(scope="module")
def b():
    return B.load()


def plan_args(**kw):
    a = dict(ctx=P, new=2 * P, n=3, page=16, most=4, free=3 * P, n_free=5, cursor=None, table=4 * P, cap=8, cu=5 * P,
             len=6 * P, pos=7 * P, slot=8 * P, state=9 * P, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [dict(new=None), dict(table=None), dict(cu=None), dict(len=None), dict(pos=None), dict(slot=None),
                                dict(state=None), dict(page=0), dict(page=-4), dict(most=0), dict(n_free=-1), dict(free=None),
                                dict(len=P), dict(len=2 * P), dict(cursor=9 * P)])
def test_plan_refuses(b, kw):
    b.hip_paged_plan(*plan_args(**kw))
    assert b.last_error() == B.EINVAL


def test_plan_refuses_positions_past_32_bits(b):
    b.hip_paged_plan(*plan_args(page=1 << 16, most=1 << 15))
    assert b.last_error() == B.EUNSUPPORTED


@pytest.mark.parametrize("kw", [dict(n=0), dict(n=-1), dict(cap=0), dict(cap=-5)])
def test_plan_of_nothing(b, kw):
    b.hip_paged_plan(*plan_args(**kw))
    assert b.last_error() == B.OK


def paged_args(**kw):
    a = dict(dtype=B.F32, q=P, k=2 * P, v=3 * P, out=4 * P, pages=10, page=16, stride=256, table=5 * P, most=4, cu=6 * P, len=7 * P,
             n=2, tokens=5, max_len=64, nh=4, nkv=2, d=128, scale=0.1, cap=0.0, window=0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), B.EINVAL), (dict(k=None), B.EINVAL), (dict(v=None), B.EINVAL), (dict(out=None), B.EINVAL), (dict(table=None), B.EINVAL),
    (dict(len=None), B.EINVAL), (dict(pages=0), B.EINVAL), (dict(page=0), B.EINVAL), (dict(most=0), B.EINVAL), (dict(max_len=0), B.EINVAL),
    (dict(cu=None), B.EINVAL), (dict(nh=0), B.EINVAL), (dict(nkv=0), B.EINVAL), (dict(nkv=3), B.EINVAL), (dict(stride=255), B.EINVAL),
    (dict(dtype=B.F16), B.EUNSUPPORTED), (dict(dtype=B.Q8_0), B.EUNSUPPORTED), (dict(d=96), B.EUNSUPPORTED), (dict(d=1024, stride=2048), B.EUNSUPPORTED),
    (dict(q=P + 4), B.EUNSUPPORTED), (dict(k=P + 8), B.EUNSUPPORTED), (dict(v=P + 2), B.EUNSUPPORTED), (dict(out=P + 4), B.EUNSUPPORTED),
    (dict(stride=257), B.EUNSUPPORTED), (dict(dtype=B.BF16, stride=260), B.EUNSUPPORTED),
    (dict(pages=1 << 28), B.EUNSUPPORTED), (dict(tokens=1 << 30), B.EUNSUPPORTED)])
def test_paged_refuses(b, kw, code):
    b.hip_attention_paged(*paged_args(**kw))
    assert b.last_error() == code


@pytest.mark.parametrize("kw", [dict(n=0), dict(tokens=0), dict(n=-2), dict(tokens=-1)])
def test_paged_of_nothing(b, kw):
    b.hip_attention_paged(*paged_args(**kw))
    assert b.last_error() == B.OK


def prompt_args(**kw):
    a = dict(dtype=B.F32, q=P, k=2 * P, v=3 * P, out=4 * P, q_stride=512, kv_stride=256, cu=6 * P, n=2, tokens=5, nh=4, nkv=2, d=128,
             scale=0.1, cap=0.0, window=0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), B.EINVAL), (dict(k=None), B.EINVAL), (dict(v=None), B.EINVAL), (dict(out=None), B.EINVAL), (dict(cu=None), B.EINVAL),
    (dict(q_stride=511), B.EINVAL), (dict(kv_stride=128), B.EINVAL), (dict(nh=5), B.EINVAL), (dict(nh=-4), B.EINVAL),
    (dict(dtype=B.F16), B.EUNSUPPORTED), (dict(d=100, q_stride=512), B.EUNSUPPORTED), (dict(q=P + 4), B.EUNSUPPORTED),
    (dict(q_stride=514), B.EUNSUPPORTED), (dict(kv_stride=258), B.EUNSUPPORTED), (dict(dtype=B.BF16, q_stride=516), B.EUNSUPPORTED),
    (dict(tokens=1 << 30), B.EUNSUPPORTED)])
def test_prompt_refuses(b, kw, code):
    b.hip_attention_prompt(*prompt_args(**kw))
    assert b.last_error() == code


def test_workspace_sizes(b):
    """None for calls of many rows or short contexts, some for few rows over long ones, nothing for nonsense."""
    paged, prompt = b.hip_attention_paged_workspace_bytes, b.hip_attention_prompt_workspace_bytes
    assert paged(B.F32, 1, 1, 32768, 8, 4, 256, 0) > 0
    assert paged(B.F32, 1, 1, 60, 8, 4, 256, 0) == 0
    assert paged(B.BF16, 1024, 1024, 32768, 32, 16, 128, 0) == 0
    assert prompt(B.BF16, 4, 65536, 32, 16, 128, 0) == 0
    for bad in ((B.F32, 0, 1, 100, 8, 4, 256, 0), (B.F32, 1, 0, 100, 8, 4, 256, 0), (B.F32, 1, 1, 0, 8, 4, 256, 0), (B.F32, 1, 1, 100, 8, 3, 256, 0),
                (B.F32, 1, 1, 100, 8, 4, -1, 0)):
        assert paged(*bad) == 0


def test_paged_refuses_positions_past_2_30(b):
    b.hip_attention_paged(*paged_args(pages=1 << 20, page=1 << 10, most=(1 << 20) + 1, max_len=(1 << 30) + 1))
    assert b.last_error() == B.EUNSUPPORTED


def test_grids_past_the_launch_limit_are_refused(b):
    """A launch holds under 2^32 threads."""
    b.hip_attention_paged(*paged_args(cu=None, n=1 << 21, tokens=1 << 21, nh=512, nkv=512, d=64, stride=512 * 64))
    assert b.last_error() == B.EUNSUPPORTED
    b.hip_attention_prompt(*prompt_args(dtype=B.BF16, cu=None, n=1, tokens=1 << 21, nh=1000, nkv=1000, d=256, q_stride=256000, kv_stride=256000))
    assert b.last_error() == B.EUNSUPPORTED
