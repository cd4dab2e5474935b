"""Verifying drafted tokens over a cache, as measurable cases.

A case is a dict of plain values; ``path`` names the operator and the other
values are its sizes and options:

* ``q8_cache``   K and V rows of new tokens are quantised into an 8-bit cache
                 (a scale of 8 significant bits for each row of a head) and
                 positions of it are read back into dense caches, which the
                 prefill attention takes;
* ``rope_axes``  rotary positions that each token brings with it, on one axis
                 (drafted tokens stand at their depth in the tree) or several
                 (time, height and width of images and video);
* ``tree``       attention of a tree of drafted tokens (one token: a decode
                 step) over a dense f32 or f16 cache or over the 8-bit cache:
                 every draft sees the whole committed cache and those drafts
                 that its mask names.

Sizes are TinyLlama's and Llama-3-8B's heads, as in the repository's own
benchmark and tests, or generic.
"""

from __future__ import annotations

import math

import torch

own = False


def listed():
    return [
        # One decode step's K and V rows into the cache, and these rows out
        # again: the smallest call, where the launches count.
        dict(name="q8_append", path="q8_cache", tokens=1, pos=1023, t_max=2048, heads=0, kv_heads=4, dh=64,
             src="f32", dst="f32", span="new"),
        # The next 512 tokens of a prompt, then all 2048 positions as the f16
        # caches that the prefill attention reads.
        dict(name="q8_chunk", path="q8_cache", tokens=512, pos=1536, t_max=2048, heads=32, kv_heads=8, dh=128,
             src="f32", dst="f16", span="all"),
        # A long prompt at once, f16 activations.
        dict(name="q8_prompt", path="q8_cache", tokens=16384, pos=0, t_max=16384, heads=0, kv_heads=8, dh=128,
             src="f16", dst="f16", span="all"),
        # Sizes that fit no block: odd counts, start and capacity.
        dict(name="q8_ragged", path="q8_cache", tokens=777, pos=131, t_max=1111, heads=10, kv_heads=5, dh=64,
             src="f32", dst="f32", span="all"),
        # Sixteen drafted tokens' queries, at the depths of their tree.
        dict(name="rope_drafts", path="rope_axes", tokens=16, heads=32, head_dim=64, sections="32", dtype="f32"),
        # A video prompt: time, height and width of every patch.
        dict(name="rope_video", path="rope_axes", tokens=8192, heads=40, head_dim=128, sections="16,24,24",
             dtype="f16"),
        # An image with odd sizes, a partly rotated head.
        dict(name="rope_ragged", path="rope_axes", tokens=1531, heads=9, head_dim=80, sections="7,13", dtype="f32"),
        # Eight drafts on a short f32 cache (TinyLlama's heads).
        dict(name="tree_f32", path="tree", cache="f32", io="f32", tokens=8, kv_len=1016, t_max=2048, heads=32,
             kv_heads=4, dh=64, fused=False),
        # A large tree on a long f16 cache (Llama-3-8B's heads): the largest.
        dict(name="tree_f16_long", path="tree", cache="f16", io="f16", tokens=64, kv_len=32704, t_max=32768, heads=32,
             kv_heads=8, dh=128, fused=False),
        # f32 activations on an f16 cache, nothing a multiple of anything.
        dict(name="tree_mixed_ragged", path="tree", cache="f16", io="f32", tokens=25, kv_len=4999, t_max=5051,
             heads=32, kv_heads=8, dh=128, fused=True),
        # A decode step on a long 8-bit cache.
        dict(name="q8_decode", path="tree", cache="q8", io="f32", tokens=1, kv_len=32767, t_max=32768, heads=32,
             kv_heads=8, dh=128, fused=False),
        # A tree of 26 drafts on an 8-bit cache, eight queries to a head.
        dict(name="q8_tree", path="tree", cache="q8", io="f16", tokens=26, kv_len=8191, t_max=8292, heads=32,
             kv_heads=4, dh=64, fused=False),
    ]


# ------------------------------------------------------------------ drawing


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["q8_cache", "rope_axes", "tree", "tree", "tree"])
    if path == "q8_cache":
        kv_heads, dh = rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128])
        tokens = _log(rng, 1, 8192)
        pos = rng.choice([0, _log(rng, 1, 4096)])
        return dict(path=path, tokens=tokens, pos=pos, t_max=pos + tokens + rng.choice([0, 0, rng.randint(1, 200)]),
                    heads=rng.choice([0, 0, kv_heads * rng.choice([1, 2, 4])]), kv_heads=kv_heads, dh=dh,
                    src=rng.choice(["f32", "f16"]), dst=rng.choice(["f32", "f16"]), span=rng.choice(["new", "all"]))
    if path == "rope_axes":
        head_dim = 2 * rng.randint(16, 64)
        pairs = rng.choice([head_dim // 2, rng.randint(4, head_dim // 2)])
        axes = rng.choice([1, 2, 3, 3, 4])
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        return dict(path=path, tokens=_log(rng, 1, 4096), heads=rng.randint(1, 40), head_dim=head_dim,
                    sections=",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs])),
                    dtype=rng.choice(["f32", "f16"]))
    cache = rng.choice(["f32", "f16", "f16", "q8", "q8"])
    kv_heads, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 4, 8])
    tokens = _log(rng, 1, 64)
    kv_len = rng.choice([rng.randint(0, 100), _log(rng, 100, 32768), _log(rng, 100, 32768)])
    return dict(path=path, cache=cache, io="f32" if cache == "f32" else rng.choice(["f32", "f16"]), tokens=tokens,
                kv_len=kv_len, t_max=kv_len + tokens + rng.choice([0, rng.randint(1, 64)]),
                heads=kv_heads * group, kv_heads=kv_heads, dh=rng.choice([64, 128]), fused=rng.random() < 0.5)


# ------------------------------------------------------------------- inputs

_DT = {"f32": torch.float32, "f16": torch.float16}


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _rows(g, c, n):
    """Activations of n tokens as their projections leave them: one fused
    [n, (heads + 2 kv_heads) dh] tensor (heads > 0), or K and V apart.  Heads
    differ in size, and now and then a channel stands out."""
    kv = c["kv_heads"] * c["dh"]
    size = torch.exp(_normal(g, 2, c["kv_heads"], 1))
    outlier = 1.0 + 15.0 * (torch.rand((2, c["kv_heads"], c["dh"]), generator=g, device="cuda") < 0.02)
    x = _normal(g, n, 2, c["kv_heads"], c["dh"]) * size * outlier
    k, v = x[:, 0].reshape(n, kv).to(_DT[c["src"]]), x[:, 1].reshape(n, kv).to(_DT[c["src"]])
    if not c["heads"]:
        return k.contiguous(), v.contiguous()
    q = _normal(g, n, c["heads"] * c["dh"]).to(_DT[c["src"]])
    return (torch.cat([q, k, v], dim=1).contiguous(),)


def _tree(g, tokens):
    """A random tree: the words of each draft's mask, and the drafts' depths.
    A draft sees itself and its ancestors."""
    pick = torch.rand((tokens,), generator=g, device="cuda").tolist()
    words, depth = [], []
    for t in range(tokens):
        parent = int(pick[t] * (t + 1)) - 1  # -1: a root
        words.append((words[parent] if parent >= 0 else 0) | (1 << t))
        depth.append(depth[parent] + 1 if parent >= 0 else 0)
    return words, depth


def _sections(c):
    """Rotated pairs of each axis."""
    return [int(n) for n in c["sections"].split(",")]


def _positions(g, c):
    """[axes, tokens]: depths in a tree, or a grid's coordinates."""
    axes, n = len(_sections(c)), c["tokens"]
    if axes == 1:
        base = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        return torch.tensor([_tree(g, n)[1]], device="cuda") + base if n <= 64 else \
            torch.arange(n, device="cuda")[None] + base
    side = max(1, round(n ** (1.0 / axes)))
    i = torch.arange(n, device="cuda")
    grid = [i // side ** (axes - 1 - a) % (side if a else n + 1) for a in range(axes)]
    return torch.stack(grid) + torch.randint(0, 100, (axes, 1), generator=g, device="cuda")


def _rope_table(rows, pairs):
    inv = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
    theta = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return torch.stack([theta.cos(), theta.sin()], dim=-1).float()


def _inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if c["path"] == "q8_cache":
        return {"new": _rows(g, c, c["tokens"]), "old": _rows(g, {**c, "heads": 0}, c["pos"]) if c["pos"] else None}
    if c["path"] == "rope_axes":
        pos = _positions(g, c)
        return {"x": _normal(g, c["tokens"], c["heads"] * c["head_dim"]).to(_DT[c["dtype"]]), "pos": pos,
                "table": _rope_table(int(pos.max()) + 1, sum(_sections(c)))}
    n, kv, dh = c["kv_len"] + c["tokens"], c["kv_heads"], c["dh"]
    size = c["heads"] * dh
    width = size + 2 * kv * dh if c["fused"] else size
    words, _ = _tree(g, c["tokens"])
    v = {"q": _normal(g, c["tokens"], width).to(_DT[c["io"]]), "words": words}
    if c["cache"] == "q8":
        v["rows"] = _rows(g, {**c, "heads": 0, "src": "f32"}, n)
    else:
        v["kt"] = _normal(g, kv, dh, c["t_max"]).to(_DT[c["cache"]])
        v["v"] = _normal(g, kv, c["t_max"], dh).to(_DT[c["cache"]])
    return v


# ------------------------------------------------------------ library state

_ENGINE = None


def _engine():
    """The package, and one executor for the program."""
    global _ENGINE
    if _ENGINE is None:
        import sys
        from pathlib import Path

        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tensor-ash_amd"))
        import tensor_ash as ta

        torch.cuda.init()
        _ENGINE = ta, ta.Executor(ta.Context("index:0"), n_slots=2, max_calls_per_submit=64, tune=False)
    return _ENGINE


class _Memory:
    """The device memory of a library tensor, for torch (keeps it alive)."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {
            "shape": tensor.shape, "typestr": "<f2" if tensor.f16 else "<f4",
            "data": (tensor.device_address, False), "strides": None, "version": 3}


def _view(tensor):
    return torch.as_tensor(_Memory(tensor), device="cuda")


def _put(ex, value):
    t = ex.tensor(list(value.shape), value.dtype == torch.float16)
    _view(t).copy_(value)
    torch.cuda.synchronize()  # the library runs on streams of its own
    return t


def _empty(ex, shape, kind):
    t = ex.tensor(shape, kind == "f16")
    _view(t).zero_()
    torch.cuda.synchronize()
    return t


def _write_desc(ta, c, rows, tokens, pos):
    if len(rows) == 1:
        k0, kv = c["heads"] * c["dh"], c["kv_heads"] * c["dh"]
        return ta.Q8WriteDesc(tokens, pos, k_offset=k0, k_stride=k0 + 2 * kv, v_offset=k0 + kv, v_stride=k0 + 2 * kv)
    return ta.Q8WriteDesc(tokens, pos)


def _library_state(c, v):
    """The library's tensors own their memory, so a program that uses it has
    its values there (and in an 8-bit cache's handle) before the call."""
    ta, ex = _engine()
    if c["path"] == "q8_cache":
        cache = ex.q8_cache(c["kv_heads"], c["dh"], c["t_max"])
        if v["old"]:
            k, w = (_put(ex, x) for x in v["old"])
            ex.q8_cache_write(k, w, cache, ta.Q8WriteDesc(c["pos"], 0))
        rows = [_put(ex, x) for x in v["new"]]
        n = c["pos"] + c["tokens"]
        first = 0 if c["span"] == "all" else c["pos"]
        return {"cache": cache, "k": rows[0], "v": rows[-1], "write": _write_desc(ta, c, rows, c["tokens"], c["pos"]),
                "read": ta.Q8ReadDesc(n - first, first), "kt": _empty(ex, [c["kv_heads"], c["dh"], n], c["dst"]),
                "vc": _empty(ex, [c["kv_heads"], n, c["dh"]], c["dst"])}
    if c["path"] == "rope_axes":
        pos = ta.U32Cell(ex.ctx, v["pos"].numel())
        pos.write(v["pos"].reshape(-1).tolist())
        return {"x": _put(ex, v["x"]), "pos": pos, "table": _put(ex, v["table"]),
                "out": _empty(ex, list(v["x"].shape), c["dtype"]),
                "desc": ta.RopeAxesDesc(c["heads"], c["head_dim"], 2 * sum(_sections(c)), _sections(c))}
    mask = ta.U32Cell(ex.ctx, 2 * c["tokens"])
    mask.write([w >> s & 0xFFFFFFFF for w in v["words"] for s in (0, 32)])
    s = {"q": _put(ex, v["q"]), "mask": mask, "out": _empty(ex, [c["tokens"], c["heads"] * c["dh"]], c["io"]),
         "desc": ta.TreeAttentionDesc(c["kv_len"], c["tokens"], 1.0 / math.sqrt(c["dh"]),
                                      q_stride=v["q"].shape[1] if c["fused"] else 0)}
    if c["cache"] == "q8":
        s["cache"] = ex.q8_cache(c["kv_heads"], c["dh"], c["t_max"])
        k, w = (_put(ex, x) for x in v["rows"])
        ex.q8_cache_write(k, w, s["cache"], ta.Q8WriteDesc(c["kv_len"] + c["tokens"], 0))
    else:
        s["kt"], s["v"] = _put(ex, v["kt"]), _put(ex, v["v"])
    return s


# -------------------------------------------------------------- plain state


def _power(e):
    """2^e in f64 for whole e, exact on every device."""
    return (e + 1023 << 52).view(torch.float64)


def _quantise(x):
    """x [n, heads, dh] -> (int8 codes, f32 scales [n, heads]).  The scale and
    the codes next to a half are decided in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1)
    m, e = torch.frexp((top / torch.full_like(top, 127.0)).clamp_min(2.0 ** -100))  # a quotient, no reciprocal
    scale = torch.ceil(m * 256.0) * _power(e.long() - 8)
    return torch.round(x / scale[..., None]).to(torch.int8), scale.float()


def _plain_state(c, v):
    """The same in torch's tensors: an 8-bit cache is its codes and scales."""
    heads, dh = c.get("kv_heads"), c.get("dh")
    if c["path"] == "q8_cache":
        n = c["pos"] + c["tokens"]
        s = {"new": v["new"], "codes": torch.zeros((2, n, heads, dh), dtype=torch.int8, device="cuda"),
             "scales": torch.zeros((2, n, heads), device="cuda"),
             "kt": torch.zeros((heads, dh, n), dtype=_DT[c["dst"]], device="cuda"),
             "vc": torch.zeros((heads, n, dh), dtype=_DT[c["dst"]], device="cuda")}
        for i in range(2 if v["old"] else 0):
            s["codes"][i, :c["pos"]], s["scales"][i, :c["pos"]] = _quantise(v["old"][i].view(-1, heads, dh))
        return s
    if c["path"] == "tree" and c["cache"] == "q8":
        pairs = [_quantise(x.view(-1, heads, dh)) for x in v["rows"]]
        return {"q": v["q"], "words": _words(v["words"]), "codes": torch.stack([p[0] for p in pairs]),
                "scales": torch.stack([p[1] for p in pairs])}
    return {**v, "words": _words(v["words"])} if c["path"] == "tree" else v


def _words(words):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device="cuda")


def prepare(case, seed):
    v = _inputs(case, seed)
    state = {"case": case, **(_library_state(case, v) if own else _plain_state(case, v))}
    torch.cuda.synchronize()
    return state


# ---------------------------------------------------------------------- run


def _plain_q8_cache(s):
    c = s["case"]
    heads, dh, n0, n = c["kv_heads"], c["dh"], c["pos"], c["pos"] + c["tokens"]
    x = s["new"]
    if len(x) == 1:
        q0, kv = c["heads"] * dh, heads * dh
        x = x[0][:, q0:q0 + kv], x[0][:, q0 + kv:]
    for i in (0, 1):
        s["codes"][i, n0:n], s["scales"][i, n0:n] = _quantise(x[i].reshape(-1, heads, dh))
    first = 0 if c["span"] == "all" else n0
    k, v = s["codes"][:, first:n].float() * s["scales"][:, first:n, :, None]
    s["kt"][:, :, first:n] = k.permute(1, 2, 0).to(s["kt"].dtype)
    s["vc"][:, first:n] = v.permute(1, 0, 2).to(s["vc"].dtype)
    return {"kt": s["kt"], "v": s["vc"]}


def _plain_rope(s):
    c = s["case"]
    pairs = sum(_sections(c))
    x = s["x"].float().view(c["tokens"], c["heads"], c["head_dim"])
    axis = torch.repeat_interleave(torch.arange(len(_sections(c)), device=x.device),
                                   torch.tensor(_sections(c), device=x.device))
    row = s["pos"][axis].t()  # [tokens, pairs]
    cs = s["table"][row, torch.arange(pairs, device=x.device)]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    x0, x1 = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    y = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], dim=-1).flatten(-2)
    return torch.cat([y, x[..., 2 * pairs:]], dim=-1).view(s["x"].shape).to(s["x"].dtype)


def _plain_tree(s):
    c = s["case"]
    t, h, hkv, dh, n0 = c["tokens"], c["heads"], c["kv_heads"], c["dh"], c["kv_len"]
    n, group = n0 + t, h // hkv
    q = s["q"][:, :h * dh].float().view(t, hkv, group, dh).permute(1, 0, 2, 3).reshape(hkv, t * group, dh)
    if c["cache"] == "q8":
        k, v = s["codes"].float() * s["scales"][..., None]
        kt, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    else:
        kt, v = s["kt"][:, :, :n].float().contiguous(), s["v"][:, :n].float().contiguous()
    bits = (s["words"][:, None] >> torch.arange(t, device=q.device)[None, :] & 1).bool()
    sees = torch.cat([torch.ones((t, n0), dtype=torch.bool, device=q.device), bits], dim=1)
    sees = sees[:, None, :].expand(t, group, n).reshape(1, t * group, n)
    score = torch.matmul(q, kt) * (1.0 / math.sqrt(dh))
    score = torch.where(sees, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3.0e38)
    p = torch.where(sees, torch.exp(score - top), 0.0)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out.view(hkv, t, group, dh).permute(1, 0, 2, 3).reshape(t, h * dh).to(_DT[c["io"]])


def run(state):
    """One pass: the operator's call (the library's calls wait for their
    result)."""
    path, s = state["case"]["path"], state
    if not own:
        return {"q8_cache": _plain_q8_cache, "rope_axes": _plain_rope, "tree": _plain_tree}[path](s)
    _, ex = _engine()
    if path == "q8_cache":
        ex.q8_cache_write(s["k"], s["v"], s["cache"], s["write"])
        ex.q8_cache_read(s["cache"], s["kt"], s["vc"], s["read"])
        return {"kt": _view(s["kt"]), "v": _view(s["vc"])}
    if path == "rope_axes":
        ex.rope_axes(s["x"], s["table"], s["pos"], s["out"], s["desc"])
    elif "cache" in s:
        ex.q8_tree_attention(s["q"], s["cache"], s["out"], s["desc"], mask=s["mask"])
    else:
        ex.tree_attention(s["q"], s["kt"], s["v"], s["out"], s["desc"], mask=s["mask"])
    return _view(s["out"])


# --------------------------------------------------------------------- work


def work(case):
    c, item = case, {"f32": 4, "f16": 2}
    if c["path"] == "q8_cache":
        row = 2 * c["kv_heads"] * c["dh"]  # K and V values of a position
        code = 2 * c["kv_heads"] * (c["dh"] + 2)
        back = c["tokens"] + (c["pos"] if c["span"] == "all" else 0)
        old = back - c["tokens"]
        return {"bytes": c["tokens"] * (row * item[c["src"]] + code) + old * code + back * row * item[c["dst"]],
                "flops": 4 * c["tokens"] * row + back * row}
    if c["path"] == "rope_axes":
        n, pairs = c["tokens"] * c["heads"] * c["head_dim"], sum(_sections(c))
        return {"bytes": 2 * n * item[c["dtype"]] + 4 * c["tokens"] * len(_sections(c)) + 8 * pairs,
                "flops": 6 * c["tokens"] * c["heads"] * pairs}
    n = c["kv_len"] + c["tokens"]
    row = 2 * c["kv_heads"] * (c["dh"] + 2 if c["cache"] == "q8" else c["dh"] * item[c["cache"]])
    return {"bytes": n * row + 2 * c["tokens"] * c["heads"] * c["dh"] * item[c["io"]] + 8 * c["tokens"],
            "flops": 4 * c["dh"] * c["heads"] * c["tokens"] * (c["kv_len"] + 1)}


# -------------------------------------------------------------------- exact


def _stands_for(x):
    """The values that the rows [.., dh] have in the 8-bit cache, in f64: the
    scale is the smallest number of 8 significant bits that is no less than a
    127th of the row's largest magnitude."""
    x = x.double()
    top = x.abs().max(dim=-1, keepdim=True).values.clamp(min=127.0 * 2.0 ** -100)
    exponent = (top.view(torch.int64) >> 52) - 1023 - 7 - 7  # a 127th is over 2^-7: units that leave 8 or 9 bits
    unit = (exponent + 1023 << 52).view(torch.float64)
    whole = torch.ceil(top / (unit * 127.0))
    wide = whole > 256.0
    scale = torch.where(wide, torch.ceil(top / (unit * 254.0)) * 2.0, whole) * unit
    ratio = x / scale
    low = torch.floor(ratio)
    over = ratio - low
    up = (over > 0.5) | ((over == 0.5) & (torch.remainder(low, 2.0) == 1.0))
    return scale * (low + up.double())


def exact(case, seed):
    c, v = case, _inputs(case, seed)
    if c["path"] == "rope_axes":
        out = v["x"].double().view(c["tokens"], c["heads"], c["head_dim"]).clone()
        i = 0
        for a, size in enumerate(_sections(c)):
            for _ in range(size):
                angle = v["table"][v["pos"][a], i].double()
                cos, sin = angle[:, :1], angle[:, 1:]
                even, odd = out[:, :, 2 * i].clone(), out[:, :, 2 * i + 1].clone()
                out[:, :, 2 * i], out[:, :, 2 * i + 1] = even * cos - odd * sin, even * sin + odd * cos
                i += 1
        return out.view(c["tokens"], -1)
    heads, dh = c["kv_heads"], c["dh"]
    if c["path"] == "q8_cache":
        n0, n = c["pos"], c["pos"] + c["tokens"]
        kt = torch.zeros((heads, dh, n), dtype=torch.float64, device="cuda")
        vc = torch.zeros((heads, n, dh), dtype=torch.float64, device="cuda")
        kv = heads * dh
        new = v["new"] if len(v["new"]) == 2 else (v["new"][0][:, -2 * kv:-kv], v["new"][0][:, -kv:])
        parts = [(n0, n, new)] + ([(0, n0, v["old"])] if v["old"] and c["span"] == "all" else [])
        for lo, hi, (a, b) in parts:
            kt[:, :, lo:hi] = _stands_for(a.reshape(hi - lo, heads, dh)).permute(1, 2, 0)
            vc[:, lo:hi] = _stands_for(b.reshape(hi - lo, heads, dh)).permute(1, 0, 2)
        return {"kt": kt, "v": vc}
    t, n0, group = c["tokens"], c["kv_len"], c["heads"] // heads
    n = n0 + t
    blind = torch.tensor([[not w >> j & 1 for j in range(t)] for w in v["words"]], device="cuda")
    out = torch.zeros((t, c["heads"], dh), dtype=torch.float64, device="cuda")
    for h in range(heads):
        if c["cache"] == "q8":
            k, val = (_stands_for(x.view(n, heads, dh)[:, h]) for x in v["rows"])
            k = k.t().contiguous()
        else:
            k, val = v["kt"][h, :, :n].double(), v["v"][h, :n].double()
        for j in range(group):
            a = h * group + j
            s = v["q"][:, a * dh:(a + 1) * dh].double() @ k / math.sqrt(dh)
            s[:, n0:] = s[:, n0:].masked_fill(blind, -math.inf)
            out[:, a] = torch.softmax(s, dim=-1) @ val
    return out.view(t, -1)
