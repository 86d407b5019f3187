"""Storage types, operands and 64-bit definitions for the tests of
cross_attend, rope_table, rope_rows and groupnorm."""
import numpy as np

F32, F16, BF16 = 0, 1, 2
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
# Half a step of each type, relative (unit roundoff).
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# Half of the smallest subnormal.
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def store(x, dt):
    """x rounded to type dt: the array as stored, and its values."""
    x = np.asarray(x, np.float32)
    if dt == F32:
        return x, x.astype(np.float64)
    if dt == F16:
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    b = x.view(np.uint32)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    r = np.where(np.isnan(x), np.uint16(0x7fc0), r)
    return r, load(r, dt)


def load(a, dt):
    """Stored values as float64."""
    if dt == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


class Operand:
    """nb x rows x heads x cols in a buffer of its own, laid out as asked:
    "tokens" [nb][rows][heads][cols], "heads" [nb][heads][rows][cols], "wide"
    (tokens with room between rows), "odd" (wide, at an odd offset and an odd
    row stride). Room is filled with `fill`."""

    def __init__(self, hip, be, x, dt, layout="tokens", fill=np.nan):
        nb, rows, heads, cols = x.shape
        room = {"tokens": 0, "heads": 0, "wide": 32, "odd": 5}[layout]
        self.off = 3 if layout == "odd" else 0
        if layout == "heads":
            self.ld, self.s1 = cols, max(rows, 1) * cols
            self.s0 = heads * self.s1
        else:
            self.ld, self.s1 = heads * cols + room, cols
            if layout == "odd" and self.ld % 2 == 0:
                self.ld += 1
            self.s0 = max(rows, 1) * self.ld
        n = self.off + nb * self.s0 + 8
        self.be, self.dt, self.shape = be, dt, x.shape
        full = np.full(n, fill, np.float32)
        view = np.lib.stride_tricks.as_strided(
            full[self.off:], x.shape,
            [4 * s for s in (self.s0, self.ld, self.s1, 1)])
        view[...] = x
        self.stored, vals = store(full, dt)
        self.values = self._view(vals)
        self.mem = be.upload_typed(self.stored, dt)
        self.op = hip.bmat(self.mem, self.off, self.ld, self.s0, self.s1)

    def _view(self, flat):
        z = flat.itemsize
        return np.lib.stride_tricks.as_strided(
            flat[self.off:], self.shape,
            [z * s for s in (self.s0, self.ld, self.s1, 1)])

    def read(self):
        """Values now, and whether what lies around the operand is as it
        was."""
        now = self.be.read(self.mem, self.stored.size, self.dt)
        if self.dt == F16:
            now = now.view(np.float16)
        raw = now.view(np.uint32 if self.dt == F32 else np.uint16)
        was = self.stored.view(raw.dtype)
        out = np.ones(raw.size, bool)
        self._view(out)[...] = False
        return self._view(load(now, self.dt)).copy(), bool(np.array_equal(raw[out], was[out]))

    def free(self):
        self.be.release(self.mem)


def keep_of(nb, nk, klen, kmask):
    k = np.ones((nb, nk), bool)
    if klen is not None:
        k &= np.arange(nk)[None] < np.clip(klen, 0, nk)[:, None]
    if kmask is not None:
        k &= kmask != 0
    return k


def cross(q, k, v, keep, scale):
    """Definition in 64 bits. q [nb][nq][H][D], k, v [nb][nk][KV][D]. Returns
    o, the sums of |weights x values|, and each row's largest |score| and
    largest sum of |products|, which the error bound takes."""
    nb, nq, H, D = q.shape
    g = H // k.shape[2]
    o, av = np.zeros(q.shape), np.zeros(q.shape)
    top, prod = np.zeros((nb, nq, H, 1)), np.zeros((nb, nq, H, 1))
    for b in range(nb):
        at = np.flatnonzero(keep[b])
        if not len(at):
            continue
        for h in range(H):
            kk, vv = k[b, at, h // g], v[b, at, h // g]
            s = q[b, :, h] @ kk.T * scale
            m = s.max(1, keepdims=True)
            w = np.exp(s - m)
            w /= w.sum(1, keepdims=True)
            o[b, :, h] = w @ vv
            av[b, :, h] = w @ np.abs(vv)
            top[b, :, h] = np.abs(s).max(1, keepdims=True)
            prod[b, :, h] = (np.abs(q[b, :, h]) @ np.abs(kk).T).max(1, keepdims=True) * scale
    return o, av, top, prod


def cross_bound(o, av, top, prod, D, nk, dt, v):
    """How far a result may be off. A score carries hd roundings of its sum
    of products and a few of the scaled difference with the maximum (of
    magnitude up to twice the largest score), the exponential two units; the
    weights' error counts twice (numerator and sum); P is rounded to the type
    (or lost below its subnormals, against a sum of at least 1, half of it
    where the maximum has not moved); sums of nk terms carry nk roundings at
    most; then the result's own."""
    e = 2.0 ** -24
    score = e * ((D + 4) * prod + 8 * top + 8)
    rel = 2 * score + (nk + 16) * e
    if dt != F32:
        rel = rel + HALF[dt]
    lost = 0.0 if dt == F32 else TINY[dt] * np.abs(v).sum() * 2
    return HALF[dt] * np.abs(o) + TINY[dt] + rel * av * (1 + 2.0 ** -6) + lost
