"""cross_attend against its definition in 64 bits: types, head widths,
lengths, layouts, masks, shared heads, splits; what lies around its output."""
import numpy as np
import pytest

import seq_common as sc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    import sam3_hip
    return sam3_hip


@pytest.fixture(scope="module")
def env(hip):
    be = hip.Backend(precision="fp32")
    yield be, hip.Model(be)
    be.free()


def ints(be, a):
    return None if a is None else be.upload(np.asarray(a, np.int32).view(np.float32))


def bytes_mem(be, a):
    if a is None:
        return None
    flat = np.asarray(a, np.uint8).ravel()
    m = be.alloc(flat.size)
    be.write(m, 0, flat)
    return m


def run(hip, env, seed, dt, nb, H, KV, D, nq, nk, lay="tokens", klen=None, qlen=None, kmask=None,
        spread=2.0, ws=False, bad=np.nan, change=None, olay=None):
    be, m = env
    g = np.random.default_rng(seed)
    q = g.standard_normal((nb, nq, H, D), np.float32) * np.float32(spread)
    k = g.standard_normal((nb, nk, KV, D), np.float32)
    v = g.standard_normal((nb, nk, KV, D), np.float32)
    keep = sc.keep_of(nb, nk, None if klen is None else np.asarray(klen), kmask)
    k[~keep], v[~keep] = bad, bad
    if change:
        change(q, k, v)
    Q, K, V = (sc.Operand(hip, be, x, dt, lay) for x in (q, k, v))
    O = sc.Operand(hip, be, np.full(q.shape, -77.0, np.float32), dt, olay or lay, fill=-55.0)
    mems = [ints(be, qlen), ints(be, klen), bytes_mem(be, kmask)]
    work = None
    if ws:
        need = hip.cross_attend_ws(m, nb, H, KV, D, nq, nk, dt)
        work = be.alloc(max(need, 4))
        mems.append(work)
    scale = D ** -0.5
    print("cross_attend seed %d type %d nb %d heads %d/%d hd %d nq %d nk %d %s" %
          (seed, dt, nb, H, KV, D, nq, nk, lay), flush=True)
    hip.cross_attend(m, nb, H, KV, D, nq, nk, Q.op, K.op, V.op, O.op, mems[0], mems[1], mems[2],
                     scale, work)
    got, clean = O.read()
    for x in (Q, K, V, O):
        x.free()
    for x in mems:
        if x is not None:
            be.release(x)
    assert clean, "wrote outside its output"
    return got, Q.values, K.values, V.values, keep, scale


def check(hip, env, seed, dt, nb, H, KV, D, nq, nk, **kw):
    got, q, k, v, keep, scale = run(hip, env, seed, dt, nb, H, KV, D, nq, nk, **kw)
    o, av, top, prod = sc.cross(q, k, v, keep, scale)
    n = np.full(nb, nq) if kw.get("qlen") is None else np.clip(kw["qlen"], 0, nq)
    used = np.arange(nq)[None] < n[:, None]
    assert np.all(got[~used] == -77.0)
    lim = sc.cross_bound(o, av, top, prod, D, nk, dt, np.nan_to_num(v[keep]))
    off = np.abs(got - o)
    bad = ~(off <= lim) & used[:, :, None, None]
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], o[bad][:4], (off / lim)[bad].max())


ALL = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("D", [1, 7, 16, 20, 32, 40, 64, 72, 96, 128, 130, 200, 256])
def test_head_widths(hip, env, t, D):
    check(hip, env, D, sc.TYPES[t], 2, 2, 2, D, 37, 70)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("nq", [1, 2, 31, 32, 33, 64, 65, 127, 129, 300])
@pytest.mark.parametrize("nk", [0, 1, 31, 33, 64, 65, 129, 700])
def test_lengths(hip, env, t, nq, nk):
    check(hip, env, 100 * nq + nk, sc.TYPES[t], 1, 3, 3, 64, nq, nk)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("nq,nk", [(1, 5001), (9, 3000), (70, 2049)])
@pytest.mark.parametrize("ws", [False, True])
def test_splits(hip, env, t, D, nq, nk, ws):
    """Few rows over many keys: partial sums of splits, in the backend's
    workspace and in the caller's."""
    be, m = env
    assert hip.cross_attend_ws(m, 2, 4, 2, D, nq, nk, sc.TYPES[t]) > 0
    check(hip, env, nq + nk + D, sc.TYPES[t], 2, 4, 2, D, nq, nk, ws=ws, klen=[nk, 700])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("H,KV", [(8, 1), (8, 2), (6, 3), (12, 4)])
@pytest.mark.parametrize("nq", [1, 11, 90])
def test_shared_heads(hip, env, t, H, KV, nq):
    check(hip, env, H * nq, sc.TYPES[t], 3, H, KV, 64, nq, 200, qlen=[nq, 1, nq // 2],
          klen=[200, 3, 111])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("lay", ["heads", "wide", "odd"])
@pytest.mark.parametrize("D", [32, 40, 72, 128])
def test_layouts(hip, env, t, lay, D):
    check(hip, env, D, sc.TYPES[t], 2, 4, 4, D, 45, 99, lay=lay)
    check(hip, env, D + 1, sc.TYPES[t], 2, 4, 4, D, 3, 999, lay=lay, olay="tokens")


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("nq", [2, 50, 200])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, np.float32(-3.4e38)])
def test_ragged(hip, env, t, nq, bad):
    """Lengths of zero, one, the whole and past it, below zero; what lies
    behind them is not used."""
    check(hip, env, nq, sc.TYPES[t], 6, 2, 1, 64, nq, 300, bad=bad, klen=[300, 0, 1, 65, 1000, -4],
          qlen=[nq, nq, 1, 0, 9999, nq])


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("nq,nk", [(3, 37), (130, 37), (130, 260), (1, 4000)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_masks(hip, env, t, nq, nk, bad):
    """Masks that are no prefix, keep one key, none, all; together with
    lengths."""
    g = np.random.default_rng(nk)
    mask = (g.random((5, nk)) < 0.4).astype(np.uint8) * 255
    mask[1] = 0
    mask[2] = 0
    mask[2, nk - 1] = 1
    mask[3] = 2
    check(hip, env, nq, sc.TYPES[t], 5, 2, 2, 32, nq, nk, bad=bad, kmask=mask)
    check(hip, env, nq, sc.TYPES[t], 5, 2, 2, 128, nq, nk, bad=bad, kmask=mask,
          klen=[nk, nk, nk - 1, nk // 2, nk // 3])


@pytest.mark.parametrize("t", ALL)
def test_large_scores(hip, env, t):
    """Scores of some hundreds, growing along the keys: the maximum moves in
    every tile."""
    def grow(q, k, v):
        k *= np.linspace(0.1, 30, k.shape[1], dtype=np.float32)[None, :, None, None]

    check(hip, env, 5, sc.TYPES[t], 1, 2, 2, 64, 40, 500, change=grow)
    check(hip, env, 6, sc.TYPES[t], 1, 2, 2, 64, 2, 3000, change=grow)


@pytest.mark.parametrize("t", ALL)
def test_non_finite(hip, env, t):
    """Infinities and NaN among the keys that count reach the rows that
    softmax gives them to, and only those."""
    def change(q, k, v):
        q[0, :, 0, 0] = [1, -1, 2, 0.5]
        k[0, 7, 0] = 0
        k[0, 7, 0, 0] = np.inf          # scores +inf, -inf
        k[1, 9, 0, 3] = np.nan
        v[0, 3, 1, 2] = np.inf
        v[0, 4, 1, 5] = np.nan

    got, q, k, v, keep, scale = run(hip, env, 3, sc.TYPES[t], 2, 2, 2, 32, 4, 40, change=change)
    assert np.isnan(got[0, [0, 2, 3], 0]).all()       # exp(inf - inf)
    assert np.isfinite(got[0, 1, 0]).all()            # a weight of zero
    assert np.isnan(got[1, :, 0]).all()
    assert (got[0, :, 1, 2] == np.inf).all() and np.isnan(got[0, :, 1, 5]).all()
    fine = np.ones(32, bool)
    fine[[2, 5]] = False
    assert np.isfinite(got[0, :, 1][:, fine]).all() and np.isfinite(got[1, :, 1]).all()


def test_all_minus_infinity(hip, env):
    """A row whose every score is minus infinity gives zeros."""
    def change(q, k, v):
        q[...] = 0
        q[..., 0] = 1
        k[..., 0] = -np.inf

    got = run(hip, env, 4, sc.F32, 1, 1, 1, 32, 5, 70, change=change)[0]
    assert (got == 0).all()


def test_far_offsets(hip, env):
    """Keys more than 2^32 bytes behind the first: head strides of a long
    cache."""
    be, m = env
    D, nk, stride = 64, 130, (1 << 31) + 64
    big = be.alloc_typed(2 * stride, sc.F16)
    g = np.random.default_rng(1)
    k = [sc.store(g.standard_normal((nk, D)), sc.F16) for _ in range(4)]
    for i in range(2):
        be.write(big, 2 * i * stride, k[i][0])
        be.write(big, 2 * (i * stride + nk * D), k[2 + i][0])
    q, qv = sc.store(g.standard_normal((1, 3, 2, D)), sc.F16)
    Q, O = be.upload_typed(q, sc.F16), be.alloc_typed(q.size, sc.F16)
    hip.cross_attend(m, 1, 2, 2, D, 3, nk, hip.bmat(Q, 0, 2 * D, 0, D),
                     hip.bmat(big, 0, D, 0, stride), hip.bmat(big, nk * D, D, 0, stride),
                     hip.bmat(O, 0, 2 * D, 0, D))
    got = be.read(O).view(np.float16).astype(np.float64).reshape(1, 3, 2, D)
    kv = np.stack([k[0][1], k[1][1]], 1)[None]
    vv = np.stack([k[2][1], k[3][1]], 1)[None]
    o, av, top, prod = sc.cross(qv, kv, vv, np.ones((1, nk), bool), D ** -0.5)
    assert (np.abs(got - o) <= sc.cross_bound(o, av, top, prod, D, nk, sc.F16, vv)).all()
    for x in (big, Q, O):
        be.release(x)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,KV,nq,nk", [
    (128, 2, 1, 600, 1100), (128, 2, 2, 10000, 2000), (128, 4, 2, 5050, 2000), (72, 40, 40, 1100, 300),
    (256, 1, 1, 1030, 1537), (256, 80, 80, 257, 261), (256, 16, 8, 550, 2400), (200, 4, 4, 1291, 1090)])
def test_many_rows_wide_heads(hip, env, t, D, H, KV, nq, nk):
    """256 rows per workgroup: with and without splits, shared heads, masks,
    lengths that end inside a tile or before it."""
    g = np.random.default_rng(D)
    nb = 8 if D == 200 else 1
    check(hip, env, D, sc.TYPES[t], nb, H, KV, D, nq, nk)
    mask = (g.random((nb, nk)) < 0.5).astype(np.uint8)
    check(hip, env, D + 1, sc.TYPES[t], nb, H, KV, D, nq, nk, kmask=mask, klen=[nk - 33] * nb,
          qlen=[nq - 300] * nb)
    check(hip, env, D + 2, sc.TYPES[t], nb, H, KV, D, nq, nk, klen=[65] * nb)


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("D", [65, 72, 80, 96, 104, 160, 192, 200])
def test_three_quarters_of_a_width(hip, env, t, D):
    """Heads whose last quarter of columns is empty, and just not: whole tiles
    and others, few rows and many, splits; infinities in what is masked."""
    dt = sc.TYPES[t]
    for nq, nk, kw in ((40, 300, {}), (130, 640, {}), (1, 1500, {}), (300, 1030, {})):
        check(hip, env, D + nq, dt, 2, 2, 1, D, nq, nk, **kw)
    check(hip, env, D, dt, 2, 2, 2, D, 70, 400, klen=[399, 1], bad=np.inf)
    mask = (np.random.default_rng(D).random((2, 400)) < 0.3).astype(np.uint8)
    check(hip, env, D, dt, 2, 2, 2, D, 70, 400, kmask=mask, lay="wide")


def test_columns_of_neighbours_are_not_read(hip, env):
    """Heads of 96 side by side: a head of infinities leaves the next alone."""
    def change(q, k, v):
        k[:, :, 1], v[:, :, 1] = np.inf, np.nan

    for dt in (sc.F16, sc.F32):
        got, q, k, v, keep, scale = run(hip, env, 5, dt, 1, 3, 3, 96, 64, 512, change=change)
        for h in (0, 2):
            o, av, top, prod = sc.cross(q[:, :, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1], keep,
                                        scale)
            lim = sc.cross_bound(o, av, top, prod, 96, 512, dt, v[:, :, h:h + 1])
            assert (np.abs(got[:, :, h:h + 1] - o) <= lim).all()


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("H,KV,D,nq,nk", [(2, 2, 20, 1, 3001), (4, 2, 130, 3, 1200), (1, 1, 7, 200, 2050),
                                          (3, 1, 64, 40, 900)])
@pytest.mark.parametrize("ws", [False, True])
def test_splits_of_odd_layouts(hip, env, t, H, KV, D, nq, nk, ws):
    """Rows that do not start on 16 bytes, few of them over many keys."""
    be, m = env
    dt = sc.TYPES[t]
    assert hip.cross_attend_ws(m, 2, H, KV, D, nq, nk, dt) > 0
    check(hip, env, D, dt, 2, H, KV, D, nq, nk, lay="odd", ws=ws)
    check(hip, env, D, dt, 2, H, KV, D, nq, nk, lay="odd", klen=[nk - 1, 3], qlen=[nq, 1], ws=ws)


@pytest.mark.parametrize("H,KV,D,nq,nk", [(12, 12, 96, 449, 2533), (8, 8, 64, 500, 500),
                                          (4, 2, 32, 230, 3100), (1, 1, 256, 700, 2001),
                                          (16, 16, 128, 300, 230), (2, 2, 64, 65, 1000)])
def test_cuts_of_floats(hip, env, H, KV, D, nq, nk):
    check(hip, env, D, sc.F32, 1, H, KV, D, nq, nk)
    check(hip, env, D, sc.F32, 1, H, KV, D, nq, nk, klen=[nk // 3], lay="wide")
    mask = (np.random.default_rng(D).random((1, nk)) < 0.5).astype(np.uint8)
    check(hip, env, D, sc.F32, 1, H, KV, D, nq, nk, kmask=mask, qlen=[nq - 7], lay="heads")


@pytest.mark.parametrize("t", ALL)
@pytest.mark.parametrize("D,nq", [(32, 5), (64, 300), (96, 70), (128, 1), (128, 600), (256, 40), (256, 300),
                                  (20, 33)])
def test_long_masks(hip, env, t, D, nq):
    """Masks over more than 512 keys: empty tiles at the start, in the middle,
    at the end, more than 64 tiles of them, one key in all, none; bytes other
    than one; keys that end before the mask does, within its first four bytes
    too."""
    nb, nk = 8, 9001 if D < 128 else 2601
    g = np.random.default_rng(D + nq)
    mask = np.zeros((nb, nk), np.uint8)
    mask[0, :7], mask[0, -nk // 8:] = 255, 128
    mask[1, nk // 2:nk // 2 + 100] = g.integers(0, 3, 100)
    mask[2, -1] = 1
    mask[3, 0] = 16
    mask[5] = g.random(nk) < 0.02
    mask[6], mask[7] = 1, 1
    klen = [nk, nk, nk, nk, nk, nk - 1, 3, 700]
    check(hip, env, D, sc.TYPES[t], nb, 2, 1, D, nq, nk, kmask=mask, klen=klen)
