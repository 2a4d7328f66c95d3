"""The paged key-value cache without a GPU: what the entry points refuse, what
kv_check finds in a batch, the workspace's size, and the oracle itself."""
import ctypes as C

import numpy as np
import pytest

import kv as O
import mynah_hip as M

BUF = np.zeros(4096, np.float64)           # something to point at; a refused call reads none of it
PTR = (BUF.ctypes.data + 63) // 64 * 64


def cache(**kw):
    a = dict(type=M.F16, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64, k=PTR, v=PTR)
    a.update(kw)
    return M.KvCacheC(**a)


def batch(**kw):
    a = dict(nseq=2, rows=8, max_pages=4, max_new=4, max_len=64, row_start=PTR, len=PTR, pages=PTR)
    a.update(kw)
    return M.KvBatchC(**a)


CACHES = [dict(type=1), dict(type=24), dict(n_pages=0), dict(n_pages=-1), dict(page_size=0), dict(n_kv_heads=0),
          dict(head_dim=96), dict(head_dim=0), dict(n_kv_heads=65537), dict(k=0), dict(v=0), dict(k=PTR + 8), dict(v=PTR + 2),
          dict(n_pages=2 ** 30, page_size=16)]
BATCHES = [dict(nseq=-1), dict(nseq=65536), dict(rows=-1), dict(rows=2 ** 24), dict(max_pages=-1), dict(max_new=-1),
           dict(max_len=-1), dict(max_len=2 ** 30 + 1), dict(row_start=0), dict(len=0), dict(pages=0),
           dict(row_start=PTR + 1), dict(len=PTR + 2), dict(pages=PTR + 3)]


def attention(lib, c=None, b=None, **kw):
    a = dict(q=PTR, ldq=256, n_heads=4, out=PTR, ldo=256, scale=0.125, causal=1, window=0, sinks=0, ws=0, ws_bytes=0)
    a.update(kw)
    M.kv_attention_dev(lib, c or cache(), b or batch(), **a)


def append(lib, c=None, b=None, prep=None, **kw):
    a = dict(q=PTR, ldq=256, n_heads=4, q_out=PTR, ldqo=256, k=PTR, ldk=128, v=PTR, ldv=128)
    a.update(kw)
    M.kv_append_dev(lib, c or cache(), b or batch(), prep, **a)


def refused(call, *a, **kw):
    """The call's own refusal, not the absence of a GPU."""
    with pytest.raises(RuntimeError) as e:
        call(*a, **kw)
    assert "gfx950" not in str(e.value) and str(e.value).split(": ", 1)[1], e.value


@pytest.mark.parametrize("call", [attention, append])
@pytest.mark.parametrize("bad", CACHES + BATCHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()).replace(str(PTR), "p"))
def test_refuses_bad_cache_or_batch(lib, call, bad):
    field = next(iter(bad))
    is_cache = field in [f for f, _ in M.KvCacheC._fields_]
    refused(call, lib, cache(**bad) if is_cache else None, None if is_cache else batch(**bad))


@pytest.mark.parametrize("bad", [
    dict(n_heads=0), dict(n_heads=3), dict(n_heads=-2), dict(q=0), dict(out=0), dict(q=PTR + 4), dict(out=PTR + 8),
    dict(ldq=254), dict(ldq=252), dict(ldo=128), dict(ldq=257), dict(ldq=260), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(window=-1), dict(window=5, sinks=-1), dict(window=5, causal=0), dict(sinks=4),
    dict(ws=PTR + 8), dict(ldo=2 ** 33)], ids=str)
def test_attention_refuses(lib, bad):
    refused(attention, lib, **bad)


def test_attention_refuses_small_workspace(lib):
    b = batch(max_pages=400, max_len=6400)
    need = M.kv_attention_ws_bytes(lib, cache(), b, 4)
    assert need > 0
    refused(attention, lib, None, b, ws=PTR, ws_bytes=need - 1)


def test_attention_refuses_too_many_workgroups(lib):
    for new in (16, 17, 2 ** 24 - 1):   # (two heads a K/V head: 32 rows, the most of the few-rows form)
        b = batch(nseq=65535, rows=2 ** 24 - 1, max_new=new, max_pages=2 ** 26, max_len=2 ** 30)
        c = cache(n_kv_heads=512, n_pages=1)
        refused(attention, lib, c, b, n_heads=1024, ldq=65536, ldo=65536)
        assert M.kv_attention_ws_bytes(lib, c, b, 1024) == 0


@pytest.mark.parametrize("bad", [
    dict(n_heads=-1), dict(q=0), dict(q_out=0), dict(k=0), dict(v=0), dict(k=PTR + 4), dict(ldk=127), dict(ldk=124),
    dict(ldv=64), dict(ldq=128), dict(ldqo=130), dict(ldqo=260)], ids=str)
def test_append_refuses(lib, bad):
    refused(append, lib, **bad)


@pytest.mark.parametrize("bad", [
    dict(rot=4, freq=PTR), dict(rot=-8, freq=PTR), dict(rot=72, freq=PTR), dict(rot=64), dict(rot=64, freq=PTR + 4),
    dict(q_norm=PTR + 4), dict(k_norm=PTR + 8), dict(q_norm=PTR, eps=-1.0), dict(k_norm=PTR, eps=float("nan")),
    dict(k_norm=PTR, eps=float("inf"))], ids=str)
def test_append_refuses_preparation(lib, bad):
    refused(append, lib, None, None, M.kv_prep(**bad))


def test_valid_calls_get_as_far_as_the_device(lib):
    """The arguments the tests above change one by one are right as they are."""
    if lib.available():
        pytest.skip("would launch")
    for call in (attention, append):
        with pytest.raises(RuntimeError, match="no gfx950 device"):
            call(lib)
    with pytest.raises(RuntimeError, match="no gfx950 device"):
        append(lib, n_heads=0, q=0, q_out=0)
    # nothing to do, and an empty buffer has no address
    for b in (batch(rows=0), batch(nseq=0, row_start=0, len=0, pages=0, rows=0)):
        with pytest.raises(RuntimeError, match="no gfx950 device"):
            attention(lib, b=b, q=0, out=0)
        with pytest.raises(RuntimeError, match="no gfx950 device"):
            append(lib, b=b, q=0, q_out=0, k=0, v=0)


# ------------------------------------------------------------------- workspace
def test_workspace_bytes(lib):
    c = cache(head_dim=128)
    # up to 512 keys a sequence: one chunk, no partial results
    assert M.kv_attention_ws_bytes(lib, c, batch(max_len=512, max_pages=100), 4) == 0
    assert M.kv_attention_ws_bytes(lib, c, batch(max_len=513, max_pages=100), 4) > 0
    # max_pages bounds the keys as well
    assert M.kv_attention_ws_bytes(lib, c, batch(max_len=513, max_pages=32), 4) == 0
    # grows with every bound, never shrinks
    last = 0
    for n in list(range(513, 20000, 61)) + [65536, 65600, 262144, 262208, 10 ** 6]:
        now = M.kv_attention_ws_bytes(lib, c, batch(max_len=n, max_pages=2 ** 20), 4)
        assert now >= last
        last = now
    # a window bounds it
    assert M.kv_attention_ws_bytes(lib, c, batch(max_len=10 ** 6, max_pages=2 ** 20), 4, 1, 1024, 4) < last / 100
    for b in (batch(nseq=0), batch(rows=0), batch(max_new=0), batch(max_len=0)):
        assert M.kv_attention_ws_bytes(lib, c, b, 4) == 0


@pytest.mark.parametrize("typ", [M.F32, M.F16, M.BF16])
@pytest.mark.parametrize("dk", [64, 128])
def test_prompt_workspace_is_bounded(lib, typ, dk):
    """Past 32 rows: never more than 512 workgroups' partial results of 128 rows; none where those alone fill the chip."""
    c, most = cache(type=typ, head_dim=dk), 0
    for nseq in (1, 2, 5, 31, 32, 200):
        for new in (33, 128, 500, 4000):
            for length in (new, 700, 5000, 100000, 2 ** 20):
                for window in (0, 300):
                    b = batch(nseq=nseq, rows=nseq * new, max_new=new, max_len=max(length, new), max_pages=2 ** 16)
                    n = M.kv_attention_ws_bytes(lib, c, b, 2, 1, window, 0)
                    assert n <= 262144 * (dk + 2) and n % (128 * 4 * (dk + 2)) == 0
                    if 2 * nseq * -(-new // 128) > 256:
                        assert n == 0
                    most = max(most, n)
    assert most > 0


# -------------------------------------------------------------------- kv_check
def tables(row_start, length, pages):
    t = [np.ascontiguousarray(x, np.int32) for x in (row_start, length, pages)]
    b = batch(nseq=len(length), rows=8, max_pages=t[2].shape[1], max_new=4, max_len=64, row_start=t[0].ctypes.data,
              len=t[1].ctypes.data, pages=t[2].ctypes.data)
    b.keep = t
    return b


def test_check_accepts(lib):
    M.kv_check(lib, cache(k=0, v=0), tables([0, 3, 3, 7], [20, 5, 4], [[1, 2], [2, 99], [3, -1]]))
    M.kv_check(lib, cache(), tables([0], [], np.zeros((0, 1))))
    M.kv_check(lib, cache(), batch(nseq=0, row_start=0, len=0, pages=0))


@pytest.mark.parametrize("row_start,length,pages,why", [
    ([0, 3, 2], [20, 5], [[1, 2], [3, 4]], "decreases"),
    ([-1, 3, 4], [20, 5], [[1, 2], [3, 4]], "negative"),
    ([0, 4, 9], [20, 15], [[1, 2], [3, 4]], "leaves the rows"),
    ([0, 5, 6], [20, 5], [[1, 2], [3, 4]], "max_new"),
    ([0, 3, 5], [2, 5], [[1, 2], [3, 4]], "fewer keys"),
    ([0, 3, 5], [65, 5], [[1, 2, 3, 4, 5], [3, 4, 5, 6, 7]], "max_len"),
    ([0, 3, 5], [33, 5], [[1, 2], [3, 4]], "max_pages"),
    ([0, 3, 5], [20, 5], [[1, 10], [3, 4]], "page outside"),
    ([0, 3, 5], [20, 5], [[-1, 2], [3, 4]], "page outside"),
    ([0, 3, 5], [20, 5], [[1, 2], [2, 4]], "two new rows"),     # slots 1 to 3 and 0 to 4 of page 2
])
def test_check_finds(lib, row_start, length, pages, why):
    with pytest.raises(RuntimeError, match=why):
        M.kv_check(lib, cache(), tables(row_start, length, pages))


def test_check_finds_a_page_twice_in_one_sequence(lib):
    """Keys 2 and 3 of a sequence in the page of keys 0 and 1, all four of them new."""
    with pytest.raises(RuntimeError, match="two new rows"):
        M.kv_check(lib, cache(page_size=2), tables([0, 4], [4], [[1, 1]]))
    M.kv_check(lib, cache(page_size=2), tables([0, 2], [4], [[1, 1]]))   # the older two are only read


# ------------------------------------------------------------------ the oracle
def test_oracle_attention_closed_forms():
    r = np.random.default_rng(1)
    kp, vp = r.standard_normal((4, 1, 3, 8)), r.standard_normal((4, 1, 3, 8))
    pages = np.array([[2, 0, 3]])
    flat = lambda x: x[[2, 0, 3], 0].reshape(9, 8)   # noqa: E731
    # q = 0: the mean of the values a row sees
    q = np.zeros((2, 2, 8))
    out, _, n, _ = O.attention(kp, vp, [0, 2], [7], pages, q, 1.0)
    np.testing.assert_allclose(out[0, 0], flat(vp)[:6].mean(0))
    np.testing.assert_allclose(out[1, 1], flat(vp)[:7].mean(0))
    out, _, n, _ = O.attention(kp, vp, [0, 2], [7], pages, q, 1.0, window=2, sinks=1)
    np.testing.assert_allclose(out[1, 0], flat(vp)[[0, 5, 6]].mean(0))
    out, _, n, _ = O.attention(kp, vp, [0, 2], [7], pages, q, 1.0, causal=False)
    assert (n == 7).all()
    # a dominant score: that key's value; a bad page's keys are not seen
    q[:] = 100 * flat(kp)[4] / (flat(kp)[4] ** 2).sum() * 10
    out = O.attention(kp, vp, [0, 2], [7], np.array([[2, 9, 3]]), q * 0, 1.0)[0]
    np.testing.assert_allclose(out[1, 0], flat(vp)[[0, 1, 2, 6]].mean(0))
    # no key: 0; a row of no sequence: NaN
    out = O.attention(kp, vp, [0, 1], [0], pages, np.ones((2, 1, 8)), 1.0)[0]
    assert (out[0] == 0).all() and np.isnan(out[1]).all()


def test_oracle_append_closed_forms():
    x = np.arange(1.0, 9.0)
    y = O.prepare_head(x, np.full(8, 2.0), 0.0, 0, 0, False, None)
    np.testing.assert_allclose(np.mean(y * y), 4.0)
    f = np.array([np.pi / 2, np.pi])
    y = O.prepare_head(x, None, 0.0, 1, 4, False, f)     # (0, 2) by a quarter turn, (1, 3) by half a turn
    np.testing.assert_allclose(y, [-3, -2, 1, -4, 5, 6, 7, 8], atol=1e-12)
    y = O.prepare_head(x, None, 0.0, 1, 4, True, f)      # (0, 1), (2, 3)
    np.testing.assert_allclose(y, [-2, 1, -3, -4, 5, 6, 7, 8], atol=1e-12)
    kp = np.zeros((3, 1, 2, 8))
    q, k2, v2 = O.append(kp, kp, [0, 2], [3], np.array([[1, 2]]), np.ones((3, 1, 8)), np.ones((3, 1, 8)) * 5,
                         np.ones((3, 1, 8)) * 7)
    assert np.isnan(q[2]).all() and (q[:2] == 1).all()
    assert (k2[1, 0, 1] == 5).all() and (k2[2, 0, 0] == 5).all() and k2.sum() == 80 and v2.sum() == 112
