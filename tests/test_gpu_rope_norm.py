"""rope_table, rope_rows and groupnorm against their definitions in 64 bits,
and the operators one after another as a model runs them."""
import ctypes
import math

import numpy as np
import pytest

import seq_common as sc

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


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
    return be.upload(np.ascontiguousarray(a, np.int32).view(np.float32))


# ------------------------------------------------------------- tables

def frequencies(rot, theta, W=0, kind=0, factor=1.0, orig=0, fast=32.0, slow=1.0):
    j = np.arange(rot // 2)
    if W:
        return theta ** (-4.0 * (j % (rot // 4)) / rot), 1.0
    if kind == 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2.0 * j / rot)
    if kind == 1:
        f = f / factor
    if kind != 3:
        return f, 1.0
    g = np.clip((orig * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
    return (1 - g) * f / factor + g * f, 0.1 * math.log(factor) + 1


def table_of(pos, rot, theta, W=0, **kw):
    f, mul = frequencies(rot, theta, W, **kw)
    pos = np.asarray(pos, np.int64)
    if W:
        at = np.concatenate([np.repeat((pos % W)[:, None], rot // 4, 1),
                             np.repeat((pos // W)[:, None], rot // 4, 1)], 1)
    else:
        at = pos[:, None]
    a = at * f
    return np.stack([np.cos(a), np.sin(a)], -1) * mul, a, mul


def check_table(hip, env, npos, rot, theta=10000.0, W=0, pos=None, **kw):
    be, m = env
    t = be.upload(np.full(npos * rot + 8, -9.0, np.float32))
    p = None if pos is None else ints(be, pos)
    sc_ = None
    if kw:
        sc_ = hip.RopeScale(kind=kw["kind"], factor=kw["factor"], orig=kw.get("orig", 0),
                            beta_fast=kw.get("fast", 32.0), beta_slow=kw.get("slow", 1.0))
    print("rope_table", npos, rot, theta, W, kw, flush=True)
    hip.rope_table(m, t, npos, p, rot, W, theta, sc_)
    got = be.read(t)
    assert (got[npos * rot:] == -9).all()
    want, a, mul = table_of(np.arange(npos) if pos is None else pos, rot, theta, W, **kw)
    # The turn in 64 bits (frequency, product and reduction: 4 roundings, and
    # as many in numpy's angle), two roundings of the angle left, at most pi /
    # 4, six in the series, two of the factor.
    lim = mul * (10 * E + np.abs(a)[..., None] * 2.0 ** -50)
    off = np.abs(got[:npos * rot].reshape(want.shape).astype(np.float64) - want)
    assert (off <= lim).all(), (off / lim).max()
    be.release(t)


@pytest.mark.parametrize("rot", [2, 4, 10, 32, 64, 128, 512])
@pytest.mark.parametrize("npos", [1, 3, 577])
def test_table(hip, env, rot, npos):
    check_table(hip, env, npos, rot)


@pytest.mark.parametrize("W,npos", [(1, 5), (24, 576), (72, 72 * 50 + 3)])
def test_table_grid(hip, env, W, npos):
    check_table(hip, env, npos, 64, W=W)
    check_table(hip, env, 100, 32, W=W, pos=np.random.default_rng(1).integers(0, W * W, 100))


@pytest.mark.parametrize("kw", [
    dict(kind=1, factor=4.0), dict(kind=2, factor=7.5), dict(kind=3, factor=16.0, orig=4096),
    dict(kind=3, factor=1.0, orig=4096), dict(kind=3, factor=32.0, orig=100, fast=4.0, slow=0.5)])
@pytest.mark.parametrize("theta", [10000.0, 500000.0])
def test_table_scaled(hip, env, kw, theta):
    g = np.random.default_rng(2)
    check_table(hip, env, 300, 96, theta, pos=g.integers(0, 200000, 300), **kw)


def test_table_far_positions(hip, env):
    pos = [0, 1, -1, -7, 2 ** 20, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 131071, 999999]
    check_table(hip, env, len(pos), 128, pos=pos)


def test_table_is_the_trunks(hip, env):
    """The tables that SAM 3's trunk reads: rope_apply with one made here
    against one made on the host."""
    be, m = env
    side, E_, hd = 6, 128, 64
    want, _, _ = table_of(np.arange(36), hd, 10000.0, W=side)
    t = be.alloc(36 * hd * 4)
    hip.rope_table(m, t, 36, None, hd, side)
    host = be.upload(want.astype(np.float32))
    x = np.random.default_rng(3).standard_normal((36, 3 * E_)).astype(np.float32)
    mm = hip.Model(be, embed=E_, heads=2, hd=hd)
    out = []
    for table in (t, host):
        mm.m.qkv = be.upload(x)
        hip.rope_apply(mm, table, 36, 36)
        out.append(be.read(mm.m.qkv))
        be.release(mm.m.qkv)
        mm.m.qkv = None
    assert np.abs(out[0] - out[1]).max() <= 12 * E * 2 * np.abs(x).max()
    # The library's own rotation by the same table: the same values.
    X = be.upload(x)
    for third in (0, E_):
        o = hip.bmat(X, third, 3 * E_, 0, hd)
        hip.rope_rows(m, 1, 2, 36, hd, hd, hip.ROPE_PAIRS, o, o, t, 36)
    assert np.array_equal(be.read(X), out[0])


# --------------------------------------------------------------- rows

def rotate(x, table, pos, rot, halves):
    """64-bit definition: x [nb][rows][heads][hd], pos [nb][rows]; and the sum
    of each result's two products, for the bound."""
    npos = len(table)
    ok = (pos >= 0) & (pos < npos)
    t = table[np.where(ok, pos, 0)][:, :, None]
    t = np.where(ok[:, :, None, None, None], t, np.array([1.0, 0.0]))
    c, s = t[..., 0], t[..., 1]
    y, mag = x.copy(), np.zeros(x.shape)
    a_, b_ = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else \
        (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x[..., a_], x[..., b_]
    y[..., a_], y[..., b_] = a * c - b * s, a * s + b * c
    mag[..., a_], mag[..., b_] = np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)
    return y, mag


def check_rows(hip, env, seed, dt, nb, rows, heads, hd, rot, halves, lay="tokens", ylay=None,
               pos=None, pos0=0, npos=50, inplace=False):
    be, m = env
    g = np.random.default_rng(seed)
    X = sc.Operand(hip, be, g.standard_normal((nb, rows, heads, hd), np.float32), dt, lay)
    Y = X if inplace else sc.Operand(hip, be, np.full(X.shape, 3.0, np.float32), dt, ylay or lay,
                                     fill=-5.0)
    table, _, _ = table_of(np.arange(npos), rot, 100.0)
    table = table.astype(np.float32)
    T = be.upload(table)
    p = None if pos is None else ints(be, pos)
    print("rope_rows", dt, nb, rows, heads, hd, rot, halves, lay, flush=True)
    hip.rope_rows(m, nb, heads, rows, hd, rot, hip.ROPE_HALVES if halves else hip.ROPE_PAIRS, X.op,
                  Y.op, T, npos, p, pos0)
    got, clean = Y.read()
    at = np.asarray(pos) if pos is not None else \
        np.tile((pos0 + np.arange(rows)) % npos, (nb, 1))
    want, mag = rotate(X.values, table.astype(np.float64), at, rot, halves)
    lim = sc.HALF[dt] * np.abs(want) + 3 * E * mag + sc.TINY[dt]
    assert clean
    assert (np.abs(got - want) <= lim).all()
    assert np.array_equal(got[..., rot:], X.values[..., rot:])
    still = (at < 0) | (at >= npos)
    assert np.array_equal(got[still], X.values[still])
    for x in (X, Y) if Y is not X else (X,):
        x.free()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("hd,rot", [(2, 2), (32, 32), (64, 16), (64, 64), (80, 40), (96, 20),
                                    (128, 128), (128, 64), (72, 6), (33, 10), (256, 256)])
def test_rows(hip, env, t, halves, hd, rot):
    check_rows(hip, env, hd + rot, sc.TYPES[t], 2, 37, 3, hd, rot, halves)
    check_rows(hip, env, hd + rot, sc.TYPES[t], 2, 5, 3, hd, rot, halves, inplace=True)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("lay", ["heads", "wide", "odd"])
def test_rows_layouts(hip, env, t, halves, lay):
    check_rows(hip, env, 1, sc.TYPES[t], 3, 1, 5, 64, 32, halves, lay=lay)
    check_rows(hip, env, 2, sc.TYPES[t], 2, 70, 1, 64, 64, halves, lay=lay, ylay="tokens")
    check_rows(hip, env, 3, sc.TYPES[t], 2, 70, 2, 64, 64, halves, lay="tokens", ylay=lay)
    check_rows(hip, env, 4, sc.TYPES[t], 2, 9, 2, 64, 64, halves, lay=lay, inplace=True)


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_rows_positions(hip, env, halves, inplace):
    g = np.random.default_rng(5)
    pos = g.integers(0, 50, (3, 40)).astype(np.int32)
    pos[0, :4] = [-1, 50, 2 ** 31 - 1, -2 ** 31]
    pos[1, 5] = pos[1, 6] = 7
    for t in (0, 1, 2):
        check_rows(hip, env, 6, t, 3, 40, 4, 64, 64, halves, pos=pos, inplace=inplace)
        check_rows(hip, env, 7, t, 2, 120, 4, 64, 32, halves, pos0=2 ** 31 - 1, inplace=inplace)
        check_rows(hip, env, 8, t, 1, 1, 40, 128, 128, halves, pos=pos[:1, 9:10], inplace=inplace)


def test_rows_many(hip, env):
    check_rows(hip, env, 9, sc.BF16, 2, 5001, 8, 64, 64, True, npos=5001)


# --------------------------------------------------------------- norm

ACTS = ["none", "gelu", "relu", "silu"]


def check_norm(hip, env, seed, dt, nb, rows, C, groups, act=0, lay="tokens", affine=True, ws=False,
               inplace=False, mean=0.5, eps=1e-5, x=None):
    be, m = env
    g = np.random.default_rng(seed)
    if x is None:
        x = g.standard_normal((nb, rows, 1, C)) * (0.5 + g.random(C)) + \
            mean * g.standard_normal(C)
    X = sc.Operand(hip, be, x, dt, lay)
    Y = X if inplace else sc.Operand(hip, be, np.full(X.shape, 3.0, np.float32), dt, lay,
                                     fill=-5.0)
    ga = (1 + 0.2 * g.standard_normal(C)).astype(np.float32)
    bb = (0.2 * g.standard_normal(C)).astype(np.float32)
    G, B = (be.upload(ga), be.upload(bb)) if affine else (None, None)
    if not affine:
        ga, bb = np.ones(C), np.zeros(C)
    need = hip.groupnorm_ws(m, nb, rows, C, groups, dt)
    work = be.alloc(max(4, need)) if ws else None
    print("groupnorm", dt, nb, rows, C, groups, ACTS[act], lay, flush=True)
    hip.groupnorm(m, nb, rows, C, groups, X.op, Y.op, G, B, eps, act, work)
    got, clean = Y.read()
    assert clean
    v = X.values.reshape(nb, rows, groups, C // groups)
    mu = v.mean((1, 3), keepdims=True)
    var = ((v - mu) ** 2).mean((1, 3), keepdims=True)
    d = (v - mu) / np.sqrt(var + eps)
    # Two roundings of the difference, two of the deviation, one each of
    # its product with g and of the sum; the variance as the difference of
    # 64-bit sums (n roundings each at most, of values mean^2 / var larger).
    cond = 2.0 ** -52 * (rows * C // groups + 4) * (mu * mu + var) / (var + eps)
    part = (np.abs(v - mu) + E * np.abs(mu)) / np.sqrt(var + eps)
    pre = (d.reshape(nb, rows, C) * ga + bb)
    mag = (part * (8 * E + cond)).reshape(nb, rows, C) * np.abs(ga) + 2 * E * np.abs(pre)
    want, lim = pre, mag
    if act == 1:
        want = np.array([0.5 * math.erfc(-z / math.sqrt(2)) for z in pre.ravel()])
        want = want.reshape(pre.shape) * pre
    elif act == 2:
        want = np.maximum(pre, 0)
    elif act == 3:
        want = pre / (1 + np.exp(-pre))
    if act in (1, 3):
        # Slopes below 1.13; the exponential's argument carries |x| roundings.
        lim = 1.13 * mag + np.abs(pre) * (8 + np.abs(pre)) * 4 * E
    lim = lim + sc.HALF[dt] * np.abs(want) + sc.TINY[dt]
    off = np.abs(got.reshape(want.shape) - want)
    assert (off <= lim).all(), (off / lim).max()
    X.free()
    if Y is not X:
        Y.free()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("C,groups", [(1, 1), (8, 8), (32, 1), (30, 3), (64, 8), (256, 8),
                                      (320, 32), (21, 7), (2560, 32), (768, 24)])
@pytest.mark.parametrize("rows", [1, 2, 49, 323])
def test_norm(hip, env, t, C, groups, rows):
    check_norm(hip, env, C + rows, sc.TYPES[t], 2, rows, C, groups, act=rows % 4)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("ws", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_norm_chunks(hip, env, t, act, ws, inplace):
    """Enough elements that rows are split over workgroups."""
    be, m = env
    assert hip.groupnorm_ws(m, 2, 3001, 96, 4, sc.TYPES[t]) > 0
    check_norm(hip, env, act, sc.TYPES[t], 2, 3001, 96, 4, act=act, ws=ws, inplace=inplace)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lay", ["wide", "odd"])
@pytest.mark.parametrize("rows,C,groups", [(40, 64, 8), (2000, 72, 3), (700, 2570, 10)])
def test_norm_layouts(hip, env, t, lay, rows, C, groups):
    check_norm(hip, env, C, sc.TYPES[t], 2, rows, C, groups, act=2, lay=lay)
    check_norm(hip, env, C, sc.TYPES[t], 1, rows, C, groups, act=0, lay=lay, affine=False)


def test_norm_far_mean(hip, env):
    """A mean a thousand deviations away loses nothing but the input's own
    rounding."""
    check_norm(hip, env, 1, sc.F32, 2, 100, 32, 4, mean=1000.0)
    check_norm(hip, env, 2, sc.F32, 1, 5000, 32, 4, mean=1000.0)


def test_norm_constant(hip, env):
    """No variance: eps alone."""
    check_norm(hip, env, 3, sc.F32, 1, 64, 8, 2, x=np.full((1, 64, 1, 8), 2.5), eps=1e-3)
    check_norm(hip, env, 4, sc.F16, 1, 20000, 8, 2, x=np.zeros((1, 20000, 1, 8)), eps=1e-6)


def test_norm_non_finite_stays_in_its_group(hip, env):
    be, m = env
    for rows in (50, 20000):
        x = np.random.default_rng(7).standard_normal((1, rows, 1, 16)).astype(np.float32)
        x[0, 3, 0, 1], x[0, 4, 0, 9] = np.nan, np.inf
        X = sc.Operand(hip, be, x, sc.F32)
        hip.groupnorm(m, 1, rows, 16, 4, X.op, X.op, act=hip.ACT_RELU)
        y = X.read()[0][0, :, 0]
        assert np.isnan(y[:, :4]).all() and np.isnan(y[:, 8:12]).all()
        assert np.isfinite(y[:, 4:8]).all() and np.isfinite(y[:, 12:]).all()
        X.free()


# ----------------------------------------------------------- together

@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_run_of_operators(hip, env, t):
    """A memory's step: tables, rotation of queries and of the memory's keys
    (its pointer tokens not rotated), cross attention over a padded memory,
    group norm of the tokens with ReLU; each against the definition on the
    values that the step before left."""
    be, m = env
    dt = sc.TYPES[t]
    nb, side, H, D, nk = 2, 12, 4, 32, 301
    nq, g = side * side, np.random.default_rng(11)
    q = sc.Operand(hip, be, g.standard_normal((nb, nq, H, D)), dt)
    k = sc.Operand(hip, be, g.standard_normal((nb, nk, H, D)), dt)
    v = sc.Operand(hip, be, g.standard_normal((nb, nk, H, D)), dt)
    o = sc.Operand(hip, be, np.zeros((nb, nq, H, D)), dt)
    kpos = np.tile(np.arange(nk) % nq, (nb, 1)).astype(np.int32)
    kpos[:, -13:] = -1
    klen = [nk, 290]
    T, P, L = be.alloc(nq * D * 4), ints(be, kpos), ints(be, klen)
    hip.rope_table(m, T, nq, None, D, side)
    hip.rope_rows(m, nb, H, nq, D, D, hip.ROPE_PAIRS, q.op, q.op, T, nq)
    hip.rope_rows(m, nb, H, nk, D, D, hip.ROPE_PAIRS, k.op, k.op, T, nq, P)
    hip.cross_attend(m, nb, H, H, D, nq, nk, q.op, k.op, v.op, o.op, klen=L)
    table = be.read(T).reshape(nq, D // 2, 2).astype(np.float64)
    for op, pos in ((q, np.tile(np.arange(nq), (nb, 1))), (k, kpos)):
        want, mag = rotate(op.values, table, pos, D, False)
        got = op.read()[0]
        assert (np.abs(got - want) <= sc.HALF[dt] * np.abs(want) + 3 * E * mag + sc.TINY[dt]).all()
    qr, kr = q.read()[0], k.read()[0]
    want, av, top, prod = sc.cross(qr, kr, v.values, sc.keep_of(nb, nk, np.array(klen), None),
                                   D ** -0.5)
    got = o.read()[0]
    assert (np.abs(got - want) <= sc.cross_bound(want, av, top, prod, D, nk, dt, v.values)).all()
    x = hip.bmat(o.mem, 0, H * D, nq * H * D, 0)
    hip.groupnorm(m, nb, nq, H * D, 8, x, x, act=hip.ACT_RELU)
    y = o.read()[0].reshape(nb, nq, 8, 16)
    a = got.reshape(nb, nq, 8, 16)
    mu = a.mean((1, 3), keepdims=True)
    z = np.maximum((a - mu) / np.sqrt(a.var((1, 3), keepdims=True) + 1e-5), 0)
    assert (np.abs(y - z) <= sc.HALF[dt] * z + 12 * E * (1 + np.abs(z)) + sc.TINY[dt]).all()


# ----------------------------------------------------------- graphs, streams

def capture(hip, be, call):
    """The call captured on the backend's stream: a replay function."""
    # The runtime that the library is linked to: a process that imports torch
    # after it holds another one too, whose streams these are not.
    rt = hip.lib()
    s = ctypes.c_void_p(be._b.stream)
    graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamBeginCapture(s, 2) == 0
    call()
    assert rt.hipStreamEndCapture(s, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0

    def replay():
        assert rt.hipGraphLaunch(ex, s) == 0
    return replay


def test_captured_calls(hip, env):
    """Captured with a workspace of the caller's: every replay, between eager
    work, gives the eager call's bits on the inputs of the moment. Without
    one, the same within rounding."""
    be, m = env
    nb, H, D, nk = 2, 4, 64, 3000
    g = np.random.default_rng(13)
    x = [g.standard_normal((nb, n, H, D), np.float32) for n in (1, nk, nk)]
    q, k, v = (sc.Operand(hip, be, a, sc.F16) for a in x)
    r, o, e = (sc.Operand(hip, be, np.zeros((nb, 1, H, D)), sc.F16) for _ in range(3))
    ws = be.alloc(hip.cross_attend_ws(m, nb, H, H, D, 1, nk, sc.F16))
    rows, C = 4000, 64
    n_in = be.upload(g.standard_normal((rows, C)).astype(np.float32))
    n_out, n_ref = be.alloc(4 * rows * C), be.alloc(4 * rows * C)
    nws = be.alloc(hip.groupnorm_ws(m, 1, rows, C, 8, 0))
    T = be.alloc(4 * 64 * D)

    def call(out, nout, w, nw):
        hip.rope_table(m, T, 64, None, D)
        hip.rope_rows(m, nb, H, 1, D, D, hip.ROPE_HALVES, q.op, r.op, T, 64, None, 5)
        hip.cross_attend(m, nb, H, H, D, 1, nk, r.op, k.op, v.op, out.op, ws=w)
        hip.groupnorm(m, 1, rows, C, 8, hip.bmat(n_in, 0, C, 0, 0), hip.bmat(nout, 0, C, 0, 0),
                      act=hip.ACT_RELU, ws=nw)

    call(e, n_ref, None, None)
    be.finish()
    with_ws = capture(hip, be, lambda: call(o, n_out, ws, nws))
    for i in range(4):
        new = g.standard_normal((nb, 1, H, D)).astype(np.float16)
        be.write(q.mem, 0, new)
        be.write(n_in, 0, g.standard_normal((rows, C)).astype(np.float32))
        with_ws()
        be.finish()
        got, ngot = o.read()[0], be.read(n_out)
        call(e, n_ref, None, None)
        be.finish()
        assert np.array_equal(got, e.read()[0]) and np.array_equal(ngot, be.read(n_ref))
    without = capture(hip, be, lambda: call(o, n_out, None, None))
    for i in range(3):
        without()
        be.finish()
        call(e, n_ref, None, None)
        be.finish()
        assert np.abs(o.read()[0] - e.read()[0]).max() <= 4 * 2.0 ** -11
        assert np.abs(be.read(n_out) - be.read(n_ref)).max() <= 1e-5


def test_repeats_bit_for_bit(hip, env):
    be, m = env
    g = np.random.default_rng(17)
    x = [sc.Operand(hip, be, g.standard_normal((2, n, 2, 64)), sc.BF16) for n in (3, 4000, 4000)]
    o = sc.Operand(hip, be, np.zeros((2, 3, 2, 64)), sc.BF16)
    first = None
    for i in range(5):
        hip.cross_attend(m, 2, 2, 2, 64, 3, 4000, x[0].op, x[1].op, x[2].op, o.op)
        now = be.read(o.mem).copy()
        first = now if first is None else first
        assert np.array_equal(now, first)


def test_two_backends(hip, env):
    """Two backends (streams) at once, each with its own workspace."""
    be, m = env
    be2 = hip.Backend(precision="bf16")
    m2 = hip.Model(be2)
    g = np.random.default_rng(19)
    data = [g.standard_normal((1, n, 2, 64), np.float32) for n in (2, 5000, 5000)]
    ops = [[sc.Operand(hip, b, a, sc.F16) for a in data] +
           [sc.Operand(hip, b, np.zeros((1, 2, 2, 64)), sc.F16)] for b in (be, be2)]
    for i in range(10):
        for mm, x in ((m, ops[0]), (m2, ops[1])):
            hip.cross_attend(mm, 1, 2, 2, 64, 2, 5000, x[0].op, x[1].op, x[2].op, x[3].op)
    a, b = ops[0][3].read()[0], ops[1][3].read()[0]
    want, av, top, prod = sc.cross(*[x.values for x in ops[0][:3]], np.ones((1, 5000), bool), 0.125)
    lim = sc.cross_bound(want, av, top, prod, 64, 5000, sc.F16, ops[0][2].values)
    assert (np.abs(a - want) <= lim).all() and np.array_equal(a, b)
    be2.free()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [32, 20])
def test_slices_of_one_matrix(hip, env, t, D):
    """What is written may be columns of the matrix that is read: the results
    are those of a buffer apart, the other columns stay."""
    be, m = env
    dt, nb, H, n = sc.TYPES[t], 2, 2, 77
    g = np.random.default_rng(D)
    W = H * D
    x, _ = sc.store(g.standard_normal((nb, n, 4 * W), np.float32), dt)
    tab = be.alloc(4 * n * D)
    hip.rope_table(m, tab, n, None, D)

    def calls(run):
        src, out = be.upload_typed(x, dt), be.alloc_typed(x.size, dt)
        one = be.upload_typed(x, dt)
        rows = [hip.bmat(b, c * W, 4 * W, n * 4 * W, D)
                for b, c in ((src, 0), (src, 1), (src, 2), (out, 3), (one, 0), (one, 1), (one, 2),
                             (one, 3))]
        run(*rows[:4])
        run(*rows[4:])
        a, b = (np.frombuffer(be.read(z).tobytes(), x.dtype).reshape(x.shape) for z in (out, one))
        for z in (src, out, one):
            be.release(z)
        assert (a[..., 3 * W:] == b[..., 3 * W:]).all()
        assert (b[..., :3 * W] == x[..., :3 * W]).all() and not (b == x).all()

    calls(lambda q, k, v, o: hip.cross_attend(m, nb, H, H, D, n, n, q, k, v, o))
    for layout in (hip.ROPE_PAIRS, hip.ROPE_HALVES):
        calls(lambda q, k, v, o: hip.rope_rows(m, nb, H, n, D, D, layout, q, o, tab, n))
    calls(lambda q, k, v, o: hip.groupnorm(m, nb, n, W, 4, q, o))
    be.release(tab)


@pytest.mark.parametrize("nb,rows,C,G", [(3, 3000, 64, 8), (7, 1500, 96, 8), (1, 9000, 64, 2),
                                         (300, 129, 256, 1), (1, 2, 20000, 1), (1, 40000, 3, 1),
                                         (2, 1000, 1048, 4), (5, 2700, 256, 64)])
def test_norm_rounds(hip, env, nb, rows, C, G):
    """Chunks of rows in whole pairs and rounds, with and without XCDs that
    match, rows fewer than chunks, rows of more columns than threads."""
    check_norm(hip, env, C, sc.F16, nb, rows, C, G)
    check_norm(hip, env, G, sc.F32, nb, rows, C, G, lay="odd")
