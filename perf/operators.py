"""The transformer operators over packed voxel and token sets, as cases to measure.

Three operators that work on a packed batch: `n` rows that hold one set of voxels (or tokens)
after another, set `s` in rows `offsets[s] .. offsets[s+1]-1`.

* ``attention``: softmax(scale * q k^T) v within each set, heads in groups, optionally causal;
* ``rope``: rotary positions along several axes (a voxel's x, y, z; a video token's t, h, w);
* ``group_norm``: GroupNorm of each set over its rows and a group's channels, with SiLU.

``own`` selects what ``run`` does: False computes each operator in elementary torch operations in
32 bits (64 for angles and long sums), rounded once at the end; True calls the library.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    """The library's operator module (its folder's name has a dot, so it is loaded by path)."""
    if "trellis_cpp_b200" not in sys.modules:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trellis.cpp_b200")
        spec = importlib.util.spec_from_file_location("trellis_cpp_b200", os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["trellis_cpp_b200"] = mod
        spec.loader.exec_module(mod)
    from trellis_cpp_b200 import ops
    return ops


# ---- cases ---------------------------------------------------------------------------------
def _attention(name, dtype, q, k, heads, kv_heads, dim, causal, packed):
    """q, k: the sets' lengths as text. packed: q, k and v are views of one [n, heads, dim] product."""
    c = {"op": "attention", "dtype": dtype, "q": q, "k": k, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "causal": causal, "packed": packed}
    return dict(c, name=name) if name else c


def _rope(name, dtype, rows, heads, of_heads, dim, sections, layout, joint, extent, inverse):
    """The first `heads` of rows of `of_heads` heads are rotated; positions below `extent` an axis."""
    c = {"op": "rope", "dtype": dtype, "rows": rows, "heads": heads, "of_heads": of_heads, "dim": dim,
         "sections": sections, "layout": layout, "joint": joint, "extent": extent, "inverse": inverse}
    return dict(c, name=name) if name else c


def _group_norm(name, dtype, out_dtype, rows, channels, groups, act):
    c = {"op": "group_norm", "dtype": dtype, "out_dtype": out_dtype, "rows": rows, "channels": channels,
         "groups": groups, "act": act}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token against what 16 requests hold so far, heads in groups of four: serving,
        # bound by reading the keys and values
        _attention("attention token", "bf16", " ".join(["1"] * 16),
                   "8192 1 517 4096 7777 3001 8000 129 6144 2500 5555 900 8191 4097 64 7000", 32, 8, 128, True, False),
        # a small object's 600 active voxels, one call: latency counts
        _attention("attention 600 voxels", "f16", "600", "600", 12, 12, 64, False, True),
        # four objects of one batch, self attention of their voxels
        _attention("attention voxels", "bf16", "4096 1730 5511 2874", "4096 1730 5511 2874", 12, 12, 128, False, True),
        # a batch of prompts of different lengths, causal, heads in groups
        _attention("attention prompts", "bf16", "4096 1 2049 777 3500 128 1023 2600", "4096 1 2049 777 3500 128 1023 2600",
                   16, 4, 128, True, False),
        # voxels of four objects attend to the tokens of their conditioning images
        _attention("attention to image", "f16", "4096 1730 5511 2874", "1374 1029 1374 261", 16, 16, 64, False, False),
        # the 32-bit mode on two test-sized objects (600 and 800 voxels)
        _attention("attention f32", "f32", "800 600", "800 600", 8, 8, 64, False, True),
        # one large object
        _attention("attention 16384 voxels", "bf16", "16384", "16384", 12, 12, 128, False, True),
        # a small object's queries and keys, both of them the first heads of one product's rows
        _rope("rope 600 voxels", "f32", 600, 24, 36, 64, "10 10 10", "pairs", False, 64, False),
        # queries and keys of a batch of objects of 65,537 voxels
        _rope("rope voxels", "bf16", 65537, 24, 36, 128, "21 21 21", "pairs", False, 512, False),
        # frames of a video (time, height, width), frequencies shared by the axes, halves rotated
        # together; the inverse rotation carries the gradient back
        _rope("rope video inverse", "f16", 131072, 16, 16, 128, "16 24 24", "halves", True, 1024, True),
        # one small set, 32 bits
        _group_norm("group norm 800 voxels", "f32", "f32", "800", 128, 32, "silu"),
        # a batch of objects of very different sizes
        _group_norm("group norm voxels", "bf16", "bf16", "65536 1 130001 777 40000 8193 3 17761", 512, 32, "silu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rope", "group_norm"])
    if op == "attention":
        kind = rng.choice(["self", "self", "causal", "cross", "token"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        dim = rng.choice([64, 128]) if rng.random() < 0.7 else 8 * rng.randint(2, 16)
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        sets = _log_int(rng, 1, 16)
        top = 3000 if dtype == "f32" else 8192
        if kind == "token":
            k = [_log_int(rng, 1, 8192) for _ in range(sets)]
            q = [1] * sets
        else:
            q = [_log_int(rng, 1, top) for _ in range(sets)]
            k = list(q) if kind != "cross" else [_log_int(rng, 1, 2000) for _ in range(sets)]
        heads = kv_heads * group
        # no more scores, counted as the padded form holds them, than the largest listed case
        while len(q) * heads * max(q) * max(k) > 12 * 16384 ** 2 // (8 if dtype == "f32" else 1):
            i = q.index(max(q))
            q[i] = max(1, q[i] // 2)
            k[i] = max(1, k[i] // 2)
            if kind != "cross":
                k[i] = max(k[i], q[i])
        packed = kind in ("self", "causal") and rng.random() < 0.5
        if packed:
            k = list(q)
        return _attention("", dtype, " ".join(map(str, q)), " ".join(map(str, k)), heads, kv_heads, dim,
                          kind in ("causal", "token"), packed)
    if op == "rope":
        axes = rng.choice([1, 2, 3, 3])
        dim = rng.choice([64, 128]) if rng.random() < 0.7 else 8 * rng.randint(2, 16)
        half = dim // 2
        sections = [max(1, half // axes - rng.randint(0, 1)) for _ in range(axes)]
        heads = rng.choice([1, 2, 8, 12, 16, 24])
        of_heads = heads + rng.choice([0, 0, 1, heads])
        dtype = rng.choice(["bf16", "f16", "f32"])
        rows = _log_int(rng, 1, min(131072, (1 << 29) // (of_heads * dim * _DT[dtype].itemsize)))
        return _rope("", dtype, rows, heads, of_heads, dim, " ".join(map(str, sections)), rng.choice(["pairs", "halves"]),
                     rng.random() < 0.5, _log_int(rng, 2, 131072), rng.random() < 0.5)
    dtype = rng.choice(["bf16", "f16", "f32"])
    groups = rng.choice([1, 4, 8, 16, 32])
    channels = groups * rng.choice([8, 8, 16, 24, 32, 64])
    channels = min(channels, 2048)
    sets = _log_int(rng, 1, 24)
    top = (1 << 28) // (channels * _DT[dtype].itemsize)
    rows = [_log_int(rng, 1, max(1, top // sets)) for _ in range(sets)]
    return _group_norm("", dtype, rng.choice([dtype, "f32"]), " ".join(map(str, rows)), channels, groups,
                       rng.choice(["none", "silu"]))


# ---- inputs --------------------------------------------------------------------------------
def _lengths(text):
    return [int(v) for v in text.split()]


def _offsets(lengths):
    off = [0]
    for v in lengths:
        off.append(off[-1] + v)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, device="cuda", generator=g) * scale + mean).to(dtype)

    if case["op"] == "attention":
        ql, kl = _lengths(case["q"]), _lengths(case["k"])
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:
            qkv = normal(sum(ql), h + 2 * hk, d)
            q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        else:
            q, k, v = normal(sum(ql), h, d), normal(sum(kl), hk, d), normal(sum(kl), hk, d)
        return {"case": case, "q": q, "k": k, "v": v, "q_off": _offsets(ql), "k_off": _offsets(kl),
                "max_q": max(ql), "max_k": max(kl)}
    if case["op"] == "rope":
        x = normal(case["rows"], case["of_heads"], case["dim"])[:, :case["heads"]]
        sections = tuple(_lengths(case["sections"]))
        pos = torch.randint(0, case["extent"], (case["rows"], len(sections)), device="cuda", generator=g,
                            dtype=torch.int32)
        return {"case": case, "x": x, "pos": pos, "sections": sections}
    rows = _lengths(case["rows"])
    c = case["channels"]
    # activations of a decoder stage: channels with means and spreads of their own
    mean = normal(c, dtype=torch.float32)
    spread = 0.5 + torch.rand(c, device="cuda", generator=g)
    x = (torch.randn((sum(rows), c), device="cuda", generator=g) * spread + mean).to(dt)
    return {"case": case, "x": x, "w": normal(c, scale=0.1, mean=1.0, dtype=torch.float32),
            "b": normal(c, scale=0.1, dtype=torch.float32), "off": _offsets(rows)}


# ---- one pass ------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        ops = _ops()
        if case["op"] == "attention":
            return ops.attention(state["q"], state["k"], state["v"], state["q_off"], state["k_off"], causal=case["causal"])
        if case["op"] == "rope":
            return ops.rope(state["x"], state["pos"], state["sections"], theta=10000.0, layout=case["layout"],
                            freqs="joint" if case["joint"] else "axis", inverse=case["inverse"])
        return ops.group_norm(state["x"], case["groups"], state["w"], state["b"], state["off"], eps=1e-5, act=case["act"],
                              out_dtype=_DT[case["out_dtype"]])
    if case["op"] == "attention":
        return _attention_plain(state)
    if case["op"] == "rope":
        return _rope_plain(state)
    return _group_norm_plain(state)


def _pad(x, off, longest):
    """Packed rows [n, heads, dim] as [sets, heads, longest, dim] in 32 bits; rows past a set's end repeat others."""
    rows = off[:-1, None].long() + torch.arange(longest, device=x.device)
    return x[rows.clamp(max=x.shape[0] - 1)].float().transpose(1, 2)


def _attention_plain(state):
    case = state["case"]
    q_off, k_off = state["q_off"], state["k_off"]
    mq, mk, hk, d = state["max_q"], state["max_k"], case["kv_heads"], case["dim"]
    group, sets = case["heads"] // hk, q_off.numel() - 1
    q = _pad(state["q"], q_off, mq).reshape(sets, hk, group * mq, d)
    k, v = _pad(state["k"], k_off, mk), _pad(state["v"], k_off, mk)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(d)).view(sets, hk, group, mq, mk)
    ql, kl = (q_off[1:] - q_off[:-1])[:, None, None], (k_off[1:] - k_off[:-1])[:, None, None]
    col = torch.arange(mk, device=s.device)[None, None, :]
    gone = col >= kl
    if case["causal"]:
        row = torch.arange(mq, device=s.device)[None, :, None]
        gone = gone | (col > row + (kl - ql))
    s.masked_fill_(gone[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(sets, hk, group * mq, mk), v).view(sets, hk, group, mq, d)
    o = torch.where(total > 0, o / total, 0.0)
    # back to packed rows: row i of the batch is row i - q_off[s] of its set s
    i = torch.arange(state["q"].shape[0], device=s.device, dtype=torch.int32)
    which = torch.searchsorted(q_off[1:].contiguous(), i, right=True)
    o = o.permute(0, 3, 1, 2, 4)[which, (i - q_off[which]).long()]
    return o.reshape(-1, case["heads"], d).to(state["q"].dtype)


def _rope_plain(state):
    case, x, pos, sections = state["case"], state["x"], state["pos"], state["sections"]
    half, total = case["dim"] // 2, sum(sections)
    size = torch.tensor(sections, device=x.device)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device), size, output_size=total)
    j = torch.arange(total, device=x.device, dtype=torch.float64)
    if case["joint"]:
        power = j / half
    else:
        power = (j - (torch.cumsum(size, 0) - size)[axis]) / size[axis]
    angle = pos.double()[:, axis] * torch.exp(power * -math.log(10000.0))
    angle = torch.cat([angle, angle.new_zeros(angle.shape[0], half - total)], 1)[:, None]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    if case["inverse"]:
        s = -s
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if case["layout"] == "pairs":
        a, b, ya, yb = x[..., 0::2].float(), x[..., 1::2].float(), y[..., 0::2], y[..., 1::2]
    else:
        a, b, ya, yb = x[..., :half].float(), x[..., half:].float(), y[..., :half], y[..., half:]
    ya.copy_(a * c - b * s)
    yb.copy_(a * s + b * c)
    return y


def _group_norm_plain(state):
    case, x, off = state["case"], state["x"], state["off"]
    n, c, groups = x.shape[0], x.shape[1], case["groups"]
    i = torch.arange(n, device=x.device, dtype=torch.int32)
    which = torch.searchsorted(off[1:].contiguous(), i, right=True)
    count = ((off[1:] - off[:-1]) * (c // groups)).double()[:, None]
    xg = x.view(n, groups, c // groups)
    zero = torch.zeros((off.numel() - 1, groups), dtype=torch.float64, device=x.device)
    mean = zero.index_add(0, which, xg.double().sum(2)) / count
    d = xg.float() - mean.float()[which][:, :, None]
    var = zero.index_add(0, which, d.double().square().sum(2)) / count
    rstd = (var + 1e-5).rsqrt().float()
    y = (d * rstd[which][:, :, None]).view(n, c) * state["w"] + state["b"]
    if case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    return y.to(_DT[case["out_dtype"]])


# ---- what a pass cannot do without ------------------------------------------------------------
def _allowed(ql, kl, causal):
    """Pairs of a query row and a key it may see, in one set."""
    if not causal:
        return ql * kl
    first = kl - ql + 1                     # keys that row 0 sees; row t sees first + t
    rows = min(ql, kl)                      # rows that see any
    return rows * (max(1, first) + kl) // 2


def work(case):
    size = _DT[case["dtype"]].itemsize
    if case["op"] == "attention":
        ql, kl, d = _lengths(case["q"]), _lengths(case["k"]), case["dim"]
        pairs = sum(_allowed(a, b, case["causal"]) for a, b in zip(ql, kl))
        return {"bytes": size * d * 2 * (sum(ql) * case["heads"] + sum(kl) * case["kv_heads"]),
                "flops": 4 * pairs * case["heads"] * d}
    if case["op"] == "rope":
        values = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * size * values + 4 * case["rows"] * len(_lengths(case["sections"])), "flops": 3 * values}
    values = sum(_lengths(case["rows"])) * case["channels"]
    return {"bytes": values * (size + _DT[case["out_dtype"]].itemsize), "flops": 10 * values}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "attention":
        return _attention_exact(case, state)
    if case["op"] == "rope":
        return _rope_exact(case, state)
    return _group_norm_exact(case, state)


def _attention_exact(case, state):
    h, d = case["heads"], case["dim"]
    group = h // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for nq, nk in zip(_lengths(case["q"]), _lengths(case["k"])):
        q, k, v = state["q"][q0:q0 + nq], state["k"][k0:k0 + nk], state["v"][k0:k0 + nk]
        for a in range(h):
            kd, vd = k[:, a // group].double(), v[:, a // group].double()
            for r in range(0, nq, 4096):
                s = q[r:r + 4096, a].double() @ kd.T / d ** 0.5
                if case["causal"]:
                    last = torch.arange(r, r + s.shape[0], device="cuda")[:, None] + nk - nq
                    s[torch.arange(nk, device="cuda")[None] > last] = -math.inf
                p = torch.softmax(s, 1) @ vd
                out[q0 + r:q0 + r + s.shape[0], a] = torch.where(torch.isinf(s).all(1, keepdim=True), 0.0, p)
        q0, k0 = q0 + nq, k0 + nk
    return out


def _rope_exact(case, state):
    x, pos = state["x"].double(), state["pos"].double()
    half = case["dim"] // 2
    out = x.clone()
    pair = 0
    for axis, size in enumerate(state["sections"]):
        for j in range(size):
            freq = 10000.0 ** -(pair / half if case["joint"] else j / size)
            turn = torch.polar(torch.ones_like(pos[:, axis]), pos[:, axis] * freq * (-1 if case["inverse"] else 1))
            a, b = (2 * pair, 2 * pair + 1) if case["layout"] == "pairs" else (pair, pair + half)
            z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
            out[..., a], out[..., b] = z.real, z.imag
            pair += 1
    return out


def _group_norm_exact(case, state):
    x = state["x"]
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    r = 0
    for n in _lengths(case["rows"]):
        y = x[r:r + n].double().view(n, case["groups"], -1)
        var, mean = torch.var_mean(y, (0, 2), correction=0, keepdim=True)
        y = ((y - mean) / torch.sqrt(var + 1e-5)).view(n, -1) * state["w"].double() + state["b"].double()
        out[r:r + n] = y * torch.sigmoid(y) if case["act"] == "silu" else y
        r += n
    return out
