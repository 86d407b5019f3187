"""What the attention-to-another-sequence operators are timed on: cross
attention to an encoder's states, the rotary tables and rotation before it,
and the group norm with activation after it.

`own` chooses between the plain form (elementary torch operations in 32 bits,
rounded once at the end) and the library's operators through its ctypes
mirror, on the same device memory. One pass is one call.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# -------------------------------------------------------------- cases

def listed():
    return [
        # Detection decoder: presence + 200 queries over one padded text
        # prompt, default precision. The smallest call: latency.
        {"name": "detect_text_f32", "op": "cross", "type": "f32", "nb": 1,
         "heads": 8, "kv_heads": 8, "hd": 32, "nq": 201, "nk": 32,
         "kv": "tokens", "ragged": "mask"},
        # Fusion encoder: the 72 x 72 image tokens of 8 prompts, each over
        # its own padded text and geometry tokens.
        {"name": "fusion_text_bf16", "op": "cross", "type": "bf16", "nb": 8,
         "heads": 8, "kv_heads": 8, "hd": 32, "nq": 5184, "nk": 37,
         "kv": "tokens", "ragged": "mask"},
        # Memory of four earlier 72 x 72 frames and 15 further tokens, one
        # wide head: the longest matrix products.
        {"name": "memory_wide_bf16", "op": "cross", "type": "bf16", "nb": 1,
         "heads": 1, "kv_heads": 1, "hd": 256, "nq": 5184, "nk": 20751,
         "kv": "tokens", "ragged": "none"},
        # One new token of 16 sequences over long states of their own
        # lengths, kept per head, 4 query heads on each.
        {"name": "step_long_f16", "op": "cross", "type": "f16", "nb": 16,
         "heads": 32, "kv_heads": 8, "hd": 128, "nq": 1, "nk": 8192,
         "kv": "heads", "ragged": "keys"},
        # A batch of ragged target sequences over ragged encoder states
        # whose keys and values come out of one projection.
        {"name": "batch_ragged_f16", "op": "cross", "type": "f16", "nb": 4,
         "heads": 12, "kv_heads": 12, "hd": 64, "nq": 447, "nk": 1500,
         "kv": "packed", "ragged": "both"},
        # One new token of 64 sequences at far positions of their own.
        {"name": "rotate_step_bf16", "op": "rotate", "type": "bf16", "nb": 64,
         "rows": 1, "heads": 32, "hd": 128, "rot": 128, "layout": "halves",
         "npos": 131072, "fused": True, "far": True},
        # The keys of two long prompts, half of the head rotated.
        {"name": "rotate_prompt_f16", "op": "rotate", "type": "f16", "nb": 2,
         "rows": 16387, "heads": 8, "hd": 128, "rot": 64, "layout": "pairs",
         "npos": 32768, "fused": False, "far": False},
        # Angles of the quarter of the 72 x 72 image tokens that a memory
        # keeps (heads of 64).
        {"name": "table_kept", "op": "table", "npos": 1296, "rot": 64,
         "grid": 72, "theta": 10000.0, "scale": "none", "factor": 1.0, "orig": 0},
        # Angles of a packed batch of long sequences, stretched 16 times.
        {"name": "table_long", "op": "table", "npos": 131072, "rot": 128,
         "grid": 0, "theta": 500000.0, "scale": "yarn", "factor": 16.0,
         "orig": 8192},
        # Pixel decoder's last level: 288 x 288 positions.
        {"name": "norm_pixels_f32", "op": "norm", "type": "f32", "nb": 1,
         "rows": 82944, "channels": 256, "groups": 8, "act": "relu"},
        # The same decoder's middle level for 4 prompts.
        {"name": "norm_prompts_bf16", "op": "norm", "type": "bf16", "nb": 4,
         "rows": 20736, "channels": 256, "groups": 8, "act": "relu"},
        # A small odd map with narrow groups.
        {"name": "norm_small_f16", "op": "norm", "type": "f16", "nb": 3,
         "rows": 323, "channels": 320, "groups": 32, "act": "gelu"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cross"] * 5 + ["rotate"] * 2 + ["table"] + ["norm"] * 2)
    t = rng.choice(["f32", "f16", "bf16"])
    if op == "cross":
        kv = rng.choice([1, 2, 4, 8, 12])
        c = {"op": op, "type": t, "kv_heads": kv, "heads": kv * rng.choice([1, 1, 2, 4]),
             "hd": rng.choice([16, 32, 32, 40, 64, 64, 72, 96, 128, 128, 256]),
             "kv": rng.choice(["tokens", "heads", "packed"]),
             "ragged": rng.choice(["none", "keys", "both", "mask"])}
        form = rng.choice(["step", "prompt", "long"])
        if form == "step":       # few queries over long states
            c.update(nb=_log(rng, 1, 64), nq=rng.randint(1, 9), nk=_log(rng, 16, 32768))
        elif form == "prompt":   # many queries over a short prompt
            c.update(nb=_log(rng, 1, 16), nq=_log(rng, 8, 5184), nk=_log(rng, 1, 300))
        else:
            c.update(nb=_log(rng, 1, 8), nq=_log(rng, 32, 5184), nk=_log(rng, 64, 20000))
        # No more than the largest listed case reads or computes.
        flops, size = (8e9, 2e8) if t == "f32" else (8e10, 4e8)
        while 4.0 * c["hd"] * c["heads"] * c["nb"] * c["nq"] * c["nk"] > flops or \
                2.0 * c["nb"] * c["kv_heads"] * c["hd"] * c["nk"] * _size(t) > size:
            if c["nb"] > 1:
                c["nb"] = (c["nb"] + 1) // 2
            elif c["nk"] >= c["nq"]:
                c["nk"] = (c["nk"] + 1) // 2
            else:
                c["nq"] = (c["nq"] + 1) // 2
        return c
    if op == "rotate":
        hd = rng.choice([32, 64, 80, 96, 128, 128, 256])
        rows = rng.choice([1, rng.randint(2, 9), _log(rng, 16, 20000)])
        c = {"op": op, "type": t, "rows": rows, "nb": _log(rng, 1, 64) if rows < 16 else
             rng.randint(1, 3), "heads": rng.choice([1, 2, 5, 8, 16, 32]), "hd": hd,
             "rot": rng.choice([hd, hd, hd // 2, hd // 4]),
             "layout": rng.choice(["pairs", "halves"]), "npos": 32768,
             "fused": rng.random() < 0.5, "far": rng.random() < 0.5}
        while c["nb"] * rows * c["heads"] * hd > 34e6:
            c["rows"] = rows = rows // 2 + 1
        return c
    if op == "table":
        scale = rng.choice(["none", "none", "linear", "ntk", "yarn"])
        grid = rng.choice([0, rng.randint(7, 80)]) if scale == "none" else 0
        return {"op": op, "grid": grid,
                "npos": rng.randint(1, grid * grid) if grid else _log(rng, 64, 131072),
                "rot": rng.choice([32, 64, 64, 80, 128]),
                "theta": rng.choice([10000.0, 500000.0, 1000000.0]), "scale": scale,
                "factor": 1.0 if scale == "none" else rng.choice([2.0, 4.0, 7.5, 16.0, 32.0]),
                "orig": 0 if scale == "none" else rng.choice([2048, 4096, 8192])}
    groups = rng.choice([1, 4, 8, 8, 16, 32])
    channels = groups * rng.choice([4, 8, 10, 16, 32, 32, 40])
    rows = _log(rng, 1, 83000)
    nb = _log(rng, 1, 8)
    while nb * rows * channels > 21e6:
        rows = rows // 2 + 1
    return {"op": op, "type": t, "nb": nb, "rows": rows, "channels": channels, "groups": groups,
            "act": rng.choice(["none", "relu", "relu", "gelu", "silu"])}


def _size(t):
    return 4 if t == "f32" else 2


def _key_lengths(c):
    """Keys of each batch entry: the same for every seed, spread over 40 to
    100 % of the longest; with "both" one entry of five or more has none."""
    if c["ragged"] in ("none", "mask"):
        return [c["nk"]] * c["nb"]
    n = [max(1, round(c["nk"] * (1 - 0.6 * ((b * 0.618) % 1)))) for b in range(c["nb"])]
    if c["ragged"] == "both" and c["nb"] > 4:
        n[3] = 0
    return n


def _query_lengths(c):
    if c["ragged"] != "both":
        return [c["nq"]] * c["nb"]
    return [max(1, round(c["nq"] * (1 - 0.5 * ((b * 0.382) % 1)))) for b in range(c["nb"])]


def _kept(c):
    """What the padding mask keeps [nb][nk]: the first text tokens, then
    padding, then the last eighth (geometry tokens)."""
    j = np.arange(c["nk"])[None, :]
    text = np.array([1 + (7 * b + 5) % max(1, 3 * c["nk"] // 4) for b in range(c["nb"])])[:, None]
    return (j < text) | (j >= c["nk"] - c["nk"] // 8)


# ------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _frequencies(c):
    """Angular frequency of each pair and the factor on (cos, sin)."""
    rot, theta, s = c["rot"], c["theta"], c["factor"]
    if c["grid"]:
        return [theta ** (-4.0 * k / rot) for k in range(rot // 4)] * 2, 1.0
    if c["scale"] == "ntk":
        theta *= s ** (rot / (rot - 2.0))
    f = [theta ** (-2.0 * j / rot) for j in range(rot // 2)]
    if c["scale"] == "linear":
        f = [v / s for v in f]
    if c["scale"] != "yarn":
        return f, 1.0
    ramp = [min(1.0, max(0.0, (c["orig"] * v / (2 * math.pi) - 1.0) / 31.0)) for v in f]
    return [(1 - r) * v / s + r * v for v, r in zip(f, ramp)], 0.1 * math.log(s) + 1.0


def _positions(c):
    """Position of every row [nb][rows]: prompts count on from a start of
    their own, single tokens stand where their sequences are."""
    b = np.arange(c["nb"])[:, None]
    r = np.arange(c["rows"])[None, :]
    room = c["npos"] - c["rows"]
    start = (room - (977 * b) % max(1, room // 2)) if c["far"] else (31 * b) % (room + 1)
    return (start + r).astype(np.int32)


def _table_positions(c, seed):
    """Positions of the table's rows: tokens of the grid that were kept, or
    sequences one after another, each a stretch of a longer one."""
    r = np.random.RandomState(int(seed) % (1 << 32))
    n = c["npos"]
    if c["grid"]:
        return np.sort(r.choice(c["grid"] ** 2, n, replace=False)).astype(np.int32)
    ends = np.sort(r.choice(n, min(n, 5), replace=False))
    p = np.arange(n)
    return (p - np.concatenate([[0], ends])[np.searchsorted(ends, p, "right")] +
            r.randint(0, 131072, len(ends) + 1)[np.searchsorted(ends, p, "right")]).astype(np.int32)


def prepare(case, seed):
    c = dict(case)
    g = _gen(seed)
    s = {"case": c}
    if c["op"] == "cross":
        t = _TYPES[c["type"]]
        nb, H, KV, D, nq, nk = (c[k] for k in ("nb", "heads", "kv_heads", "hd", "nq", "nk"))
        # Scores of standard deviation 2: some keys matter, most do little.
        s["q"] = (2 * _normal(g, nb, nq, H, D)).to(t)
        s["o"] = torch.zeros(nb, nq, H, D, device=DEV, dtype=t)
        if c["kv"] == "packed":
            s["kv"] = _normal(g, nb, nk, 2, KV, D).to(t)
            k, v = s["kv"][:, :, 0], s["kv"][:, :, 1]          # [nb][nk][KV][D]
        elif c["kv"] == "heads":                               # room to grow
            cap = -(-nk // 64) * 64 + 64
            k = _normal(g, nb, KV, cap, D).to(t).permute(0, 2, 1, 3)[:, :nk]
            v = _normal(g, nb, KV, cap, D).to(t).permute(0, 2, 1, 3)[:, :nk]
        else:
            k, v = _normal(g, nb, nk, KV, D).to(t), _normal(g, nb, nk, KV, D).to(t)
        s["k"], s["v"], s["scale"] = k, v, 1.0 / math.sqrt(D)
        s["klen"] = s["qlen"] = s["mask"] = None
        if c["ragged"] in ("keys", "both"):
            n = _key_lengths(c)
            s["klen"] = torch.tensor(n, dtype=torch.int32, device=DEV)
            for b in range(nb):     # memory behind a sequence was never written
                k[b, n[b]:] = math.nan
                v[b, n[b]:] = math.nan
        if c["ragged"] == "both":
            s["qlen"] = torch.tensor(_query_lengths(c), dtype=torch.int32, device=DEV)
        if c["ragged"] == "mask":
            s["mask"] = torch.from_numpy(_kept(c).astype(np.uint8)).to(DEV)
    elif c["op"] == "rotate":
        t = _TYPES[c["type"]]
        width = 3 if c["fused"] else 1
        s["buf"] = _normal(g, c["nb"], c["rows"], width, c["heads"], c["hd"]).to(t)
        s["x"] = s["buf"][:, :, 0]
        s["y"] = torch.empty(c["nb"], c["rows"], c["heads"], c["hd"], device=DEV, dtype=t)
        f = 10000.0 ** (-2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV) / c["rot"])
        a = torch.arange(c["npos"], dtype=torch.float64, device=DEV)[:, None] * f
        s["table"] = torch.stack([a.cos(), a.sin()], -1).float()
        s["pos"] = torch.from_numpy(_positions(c)).to(DEV)
    elif c["op"] == "table":
        s["pos"] = torch.from_numpy(_table_positions(c, seed)).to(DEV)
        s["table"] = torch.empty(c["npos"], c["rot"] // 2, 2, device=DEV)
    else:
        t = _TYPES[c["type"]]
        C = c["channels"]
        x = _normal(g, c["nb"], c["rows"], C) * (0.5 + torch.rand(C, generator=g, device=DEV))
        s["x"] = (x + _normal(g, C)).to(t)
        s["y"] = torch.empty_like(s["x"])
        s["g"] = 1 + 0.1 * _normal(g, C)
        s["b"] = 0.1 * _normal(g, C)
    if own:
        _handles(s)     # the library's names for the same memory
    return s


# ------------------------------------------------------ the library's calls

_program = {}


def _library():
    """The program's backend and model of the library, made once."""
    if not _program:
        if "sam3_hip" in sys.modules:
            hip = sys.modules["sam3_hip"]
        else:
            spec = importlib.util.spec_from_file_location(
                "sam3_hip", os.path.join(_ROOT, "i.sam3.opencl_amd", "sam3_hip.py"))
            hip = importlib.util.module_from_spec(spec)
            sys.modules["sam3_hip"] = hip
            spec.loader.exec_module(hip)
        hip.lib()
        be = hip.Backend(precision="fp32")
        _program.update(hip=hip, be=be, model=hip.Model(be))
    return _program["hip"], _program["be"], _program["model"]


def _handles(s):
    hip, be, _ = _library()
    types = {torch.float32: hip.F32, torch.float16: hip.F16, torch.bfloat16: hip.BF16,
             torch.int32: hip.F32, torch.uint8: hip.F32}

    def buffer(t):
        if t is None:
            return None
        return hip.borrow(t.data_ptr(), t.untyped_storage().nbytes() -
                          t.storage_offset() * t.element_size(), types[t.dtype])

    def operand(t, rows, heads):
        """t by its row, batch (0) and head strides."""
        return hip.bmat(buffer(t), 0, t.stride(rows), t.stride(0), t.stride(heads))

    c = s["case"]
    if c["op"] == "cross":
        s["call"] = (c["nb"], c["heads"], c["kv_heads"], c["hd"], c["nq"], c["nk"]) + \
            tuple(operand(s[n], 1, 2) for n in "qkvo")
        s["masks"] = {"qlen": buffer(s["qlen"]), "klen": buffer(s["klen"]),
                      "kmask": buffer(s["mask"]), "scale": s["scale"]}
    elif c["op"] == "rotate":
        layout = hip.ROPE_PAIRS if c["layout"] == "pairs" else hip.ROPE_HALVES
        s["call"] = (c["nb"], c["heads"], c["rows"], c["hd"], c["rot"], layout,
                     operand(s["x"], 1, 2), operand(s["y"], 1, 2), buffer(s["table"]),
                     c["npos"], buffer(s["pos"]))
    elif c["op"] == "table":
        kind = {"none": hip.ROPE_PLAIN, "linear": hip.ROPE_LINEAR, "ntk": hip.ROPE_NTK,
                "yarn": hip.ROPE_YARN}[c["scale"]]
        s["call"] = (buffer(s["table"]), c["npos"], buffer(s["pos"]), c["rot"], c["grid"], c["theta"],
                     hip.RopeScale(kind=kind, factor=c["factor"], orig=c["orig"],
                                   beta_fast=32.0, beta_slow=1.0))
    else:
        act = {"none": hip.ACT_NONE, "relu": hip.ACT_RELU, "gelu": hip.ACT_GELU,
               "silu": hip.ACT_SILU}[c["act"]]
        s["call"] = (c["nb"], c["rows"], c["channels"], c["groups"],
                     hip.bmat(buffer(s["x"]), 0, s["x"].stride(1), s["x"].stride(0), 0),
                     hip.bmat(buffer(s["y"]), 0, s["y"].stride(1), s["y"].stride(0), 0),
                     buffer(s["g"]), buffer(s["b"]), 1e-5, act)


# --------------------------------------------------------- plain forms

def _plain_cross(s):
    c = s["case"]
    nb, H, KV, D, nq, nk = (c[k] for k in ("nb", "heads", "kv_heads", "hd", "nq", "nk"))
    grp = H // KV
    keep = torch.ones(nb, nk, dtype=torch.bool, device=DEV)
    if s["klen"] is not None:
        keep = torch.arange(nk, device=DEV)[None, :] < s["klen"][:, None]
    if s["mask"] is not None:
        keep = keep & (s["mask"] != 0)
    q = s["q"].float().view(nb, nq, KV, grp, D).permute(0, 2, 3, 1, 4).reshape(nb, KV, grp * nq, D)
    k = s["k"].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"].float().permute(0, 2, 1, 3)
    v = torch.where(keep[:, None, :, None], v, torch.zeros((), device=DEV)).contiguous()
    x = torch.where(keep[:, None, None, :], torch.matmul(q, k) * s["scale"], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(nb, KV, grp, nq, D).permute(0, 3, 1, 2, 4).reshape(nb, nq, H, D).to(s["o"].dtype)
    if s["qlen"] is None:
        return o
    used = torch.arange(nq, device=DEV)[None, :] < s["qlen"][:, None]
    return torch.where(used[:, :, None, None], o, s["o"])


def _plain_rotate(s):
    c = s["case"]
    rot = c["rot"]
    x = s["x"].float()
    t = s["table"][s["pos"].long()][:, :, None]          # [nb][rows][1][rot / 2][2]
    cos, sin = t[..., 0], t[..., 1]
    if c["layout"] == "pairs":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., rot:]], -1).to(s["y"].dtype)


def _plain_table(s):
    c = s["case"]
    f, mul = _frequencies(c)
    f = torch.tensor(f, dtype=torch.float64, device=DEV)
    p = s["pos"]
    if c["grid"]:
        n = c["rot"] // 4
        a = torch.cat([(p % c["grid"]).double()[:, None] * f[:n],
                       (p // c["grid"]).double()[:, None] * f[n:]], 1)
    else:
        a = p.double()[:, None] * f     # far positions: angles in 64 bits
    return (torch.stack([a.cos(), a.sin()], -1) * mul).float()


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float().view(c["nb"], c["rows"], c["groups"], -1)
    d = x - x.mean((1, 3), keepdim=True)
    y = d * torch.rsqrt((d * d).mean((1, 3), keepdim=True) + 1e-5)
    y = y.view(c["nb"], c["rows"], -1) * s["g"] + s["b"]
    if c["act"] == "relu":
        y = y.clamp_min(0)
    elif c["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif c["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["y"].dtype)


def run(state):
    s, op = state, state["case"]["op"]
    if op == "cross":
        if own:
            hip, _, m = _library()
            hip.cross_attend(m, *s["call"], **s["masks"])
            return s["o"]
        return _plain_cross(s)
    if op == "rotate":
        if own:
            hip, _, m = _library()
            hip.rope_rows(m, *s["call"])
            return s["y"]
        return _plain_rotate(s)
    if op == "table":
        if own:
            hip, _, m = _library()
            hip.rope_table(m, *s["call"])
            return s["table"]
        return _plain_table(s)
    if own:
        hip, _, m = _library()
        hip.groupnorm(m, *s["call"])
        return s["y"]
    return _plain_norm(s)


# --------------------------------------------------------------- work

def work(case):
    c, op = case, case["op"]
    if op == "cross":
        sz, D = _size(c["type"]), c["hd"]
        kn, qn = _key_lengths(c), _query_lengths(c)
        used = _kept(c).sum(1) if c["ragged"] == "mask" else kn
        return {"bytes": sz * D * (2 * c["heads"] * sum(qn) + 2 * c["kv_heads"] * sum(kn)) +
                (c["nb"] * c["nk"] if c["ragged"] == "mask" else 0),
                "flops": 4.0 * D * c["heads"] * float(sum(a * int(b) for a, b in zip(qn, used)))}
    if op == "rotate":
        n = c["nb"] * c["rows"]
        rows = len(set(_positions(c).ravel().tolist()))
        return {"bytes": 2 * n * c["heads"] * c["hd"] * _size(c["type"]) + 4 * c["rot"] * rows + 4 * n,
                "flops": 3.0 * n * c["heads"] * c["rot"]}
    if op == "table":
        return {"bytes": 4 * c["npos"] * (c["rot"] + 1), "flops": 2.0 * c["npos"] * c["rot"]}
    n = c["nb"] * c["rows"] * c["channels"]
    return {"bytes": 2 * n * _size(c["type"]) + 8 * c["channels"], "flops": 10.0 * n}


# ------------------------------------------------------ 64-bit results

def _exact_cross(s):
    c = s["case"]
    kn, qn = _key_lengths(c), _query_lengths(c)
    kept = _kept(c) if c["ragged"] == "mask" else None
    out = s["o"].double()
    grp = c["heads"] // c["kv_heads"]
    for b in range(c["nb"]):
        j = np.arange(kn[b])
        if kept is not None:
            j = j[kept[b, :kn[b]]]
        j = torch.from_numpy(j).to(DEV)
        for h in range(c["heads"]):
            if not len(j):
                out[b, :qn[b], h] = 0
                continue
            k, v = s["k"][b, j, h // grp].double(), s["v"][b, j, h // grp].double()
            w = torch.softmax(s["q"][b, :qn[b], h].double() @ k.t().contiguous() / math.sqrt(c["hd"]), -1)
            out[b, :qn[b], h] = w @ v
    return out


def _exact_rotate(s):
    c = s["case"]
    n = c["rot"]
    first = torch.arange(0, n, 2, device=DEV) if c["layout"] == "pairs" else torch.arange(n // 2, device=DEV)
    second = first + (1 if c["layout"] == "pairs" else n // 2)
    y = s["x"].double().clone()
    turn = torch.view_as_complex(s["table"].double())[s["pos"].long()][:, :, None]
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_table(c, seed):
    f, mul = _frequencies(c)
    p = _table_positions(c, seed).astype(np.int64)
    if c["grid"]:
        at = np.concatenate([np.repeat(p[:, None] % c["grid"], c["rot"] // 4, 1),
                             np.repeat(p[:, None] // c["grid"], c["rot"] // 4, 1)], 1)
    else:
        at = p[:, None]
    z = np.exp(1j * (at * np.array(f)[None, :])) * mul
    return np.stack([z.real, z.imag], -1)


def _exact_norm(s):
    c = s["case"]
    out = torch.empty(s["x"].shape, dtype=torch.float64, device=DEV)
    w = c["channels"] // c["groups"]
    for b in range(c["nb"]):
        for i in range(c["groups"]):
            at = slice(i * w, (i + 1) * w)
            x = s["x"][b, :, at].double()
            y = (x - x.mean()) / torch.sqrt(x.var(correction=0) + 1e-5)
            out[b, :, at] = y * s["g"][at].double() + s["b"][at].double()
    if c["act"] == "relu":
        out = torch.where(out > 0, out, 0.0)
    elif c["act"] == "gelu":
        out = out * 0.5 * torch.erfc(-out / math.sqrt(2.0))
    elif c["act"] == "silu":
        out = out * torch.sigmoid(out)
    return out


def exact(case, seed):
    c = dict(case)
    if c["op"] == "table":
        return _exact_table(c, seed)
    s = prepare(case, seed)
    return {"cross": _exact_cross, "rotate": _exact_rotate, "norm": _exact_norm}[c["op"]](s)
