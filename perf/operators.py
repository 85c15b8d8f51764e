"""The 8-bit spatial cache: its write fused into the executed-row gather, its read-back, and the
attention of executed rows over it (shared prefix, visibility groups, few rows or many).

`run` computes an operator in plain torch operations where `own` is false and through the package's
binding where it is true. All sizes are those of the benchmark frames (512, 768, 1024 and 2048 pixel
sides with 512 text tokens, 24 heads of 128) or odd ones between them."""
import math
import os
import sys

import torch

own = False

D = 128
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
TOP = {"int8": 127.0, "e4m3": 448.0}
AXES = (16, 56, 56)
THETA, EPS = 10000.0, 1e-6


def listed():
    return [
        # a cursor moved over a 512 pixel frame: a handful of tokens, latency only
        {"name": "write_cursor", "op": "write", "dtype": "f16", "fmt": "e4m3", "heads": 24, "n": 1536, "m": 9},
        # an edited 1024 pixel frame: a third of the tokens run
        {"name": "write_edit", "op": "write", "dtype": "bf16", "fmt": "e4m3", "heads": 24, "n": 4608, "m": 1536},
        # the first frame of a 2048 pixel stream: every token is written
        {"name": "write_first", "op": "write", "dtype": "bf16", "fmt": "e4m3", "heads": 24, "n": 16896, "m": 16896},
        # an edit whose written rows are handed on in 16 bits (a consumer that needs them), a model of few heads
        {"name": "turn_odd", "op": "turn", "dtype": "f16", "fmt": "int8", "heads": 5, "n": 2305, "m": 577},
        # the executed rows of a 1024 pixel frame read back
        {"name": "read_edit", "op": "read", "dtype": "bf16", "fmt": "int8", "heads": 24, "n": 4608, "m": 1153},
        # a whole 2048 pixel cache turned back into 16 bits (a stream moved to a path that wants it)
        {"name": "read_all", "op": "read", "dtype": "bf16", "fmt": "e4m3", "heads": 24, "n": 16896, "m": 0},
        # one token of a 512 pixel frame
        {"name": "attend_one", "op": "attend", "dtype": "f16", "fmt": "int8", "heads": 24, "streams": 1, "prefix": 0,
         "n": 1536, "m": 1, "docs": 0},
        # a brush stroke on a 2048 pixel frame: few rows against a long cache
        {"name": "attend_stroke", "op": "attend", "dtype": "bf16", "fmt": "int8", "heads": 24, "streams": 1, "prefix": 0,
         "n": 16896, "m": 12, "docs": 0},
        # eight streams that share prompt and reference picture, each with a small edit of its own 768 pixel frame
        {"name": "attend_shared", "op": "attend", "dtype": "bf16", "fmt": "e4m3", "heads": 24, "streams": 8, "prefix": 4608,
         "n": 2304, "m": 15, "docs": 0},
        # two streams of regional prompts: documents, padded prompt, rows that see nothing; odd sizes
        {"name": "attend_regions", "op": "attend", "dtype": "f16", "fmt": "e4m3", "heads": 7, "streams": 2, "prefix": 333,
         "n": 2305, "m": 601, "docs": 4},
        # an edited 1024 pixel frame
        {"name": "attend_edit", "op": "attend", "dtype": "bf16", "fmt": "int8", "heads": 24, "streams": 1, "prefix": 0,
         "n": 4608, "m": 1536, "docs": 0},
        # a quarter of a 2048 pixel frame
        {"name": "attend_large", "op": "attend", "dtype": "bf16", "fmt": "e4m3", "heads": 24, "streams": 1, "prefix": 0,
         "n": 16896, "m": 4224, "docs": 0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["write", "turn", "read", "attend", "attend", "attend"])
    case = {"op": op, "dtype": rng.choice(["bf16", "f16"]), "fmt": rng.choice(["int8", "e4m3"]), "heads": rng.randint(1, 24)}
    if op == "write":
        case["fmt"] = "e4m3"
    if op != "attend":
        case["n"] = _spread(rng, 60, 16896)
        case["m"] = _spread(rng, 1, case["n"])
        return case
    case["streams"] = rng.choice([1, 1, 2, 3, 5, 8])
    case["n"] = _spread(rng, 60, 16896 if case["streams"] == 1 else 4608)
    case["prefix"] = rng.choice([0, _spread(rng, 1, 4608)])
    most = 4224 * 16896 * 24 // (case["heads"] * case["streams"] * (case["n"] + case["prefix"]))
    case["m"] = _spread(rng, 1, min(case["n"], 4224, most))
    case["docs"] = rng.choice([0, 0, rng.randint(1, 9)])
    return case


# ---- inputs ---------------------------------------------------------------------------------------
def _side(n):
    return max(1, math.isqrt(max(n - 1, 0)) + 1)


def _up(t, dtype):
    """t (in 64 bits) rounded up to dtype."""
    s = t.to(dtype)
    return torch.where(s.double() < t, (s.view(torch.int16) + 1).view(dtype), s)


def _quantise(x, fmt, dtype):
    """codes and scales of head vectors x [..., 128] in 32 bits."""
    top = TOP[fmt]
    s = _up(x.abs().amax(-1).double() / top, dtype)  # next to a border where the quotient is a number of dtype
    y = torch.where(s.float()[..., None] > 0, x / s.float()[..., None], torch.zeros_like(x))
    if fmt == "int8":
        return y.round().clamp(-top, top).to(torch.int8), s
    return y.clamp(-top, top).to(torch.float8_e4m3fn), s


def _cache(g, rows, heads, fmt, dtype):
    """A cache with rows of earlier frames: normed and rotated keys, plain values."""
    lanes = max(8, -(-rows // 8) * 8)
    made = {}
    for name in ("k", "v"):
        x = torch.randn(rows, heads, D, generator=g, device="cuda")
        if name == "k":
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        codes, s = _quantise(x, fmt, dtype)
        made[name] = codes.reshape(rows, heads * D).contiguous()
        made[name + "_scale"] = torch.zeros(heads, lanes, dtype=dtype, device="cuda")
        made[name + "_scale"][:, :rows] = s.t()
    return made


def _take(codes, rows):
    return codes.view(torch.int8)[rows].view(codes.dtype)


def _pick(g, n, m):
    return torch.randperm(n, generator=g, device="cuda")[:m].sort().values


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, h, n = TORCH[case["dtype"]], case["heads"], case["n"]
    m = case["m"] or n
    st = {"case": case, "t": t}
    if case["op"] in ("write", "turn"):
        for name in "qkv":
            st[name] = torch.randn(n, h * D, generator=g, device="cuda").to(t)
        st["norm_q"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
        st["norm_k"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
        at, text = torch.arange(n, device="cuda"), n // 9
        pos = torch.zeros(n, 3, dtype=torch.int32, device="cuda")
        pos[text:, 1] = ((at[text:] - text) // _side(n - text)).int()
        pos[text:, 2] = ((at[text:] - text) % _side(n - text)).int()
        st["pos"] = pos
        st["qc"] = torch.zeros(n, h * D, dtype=t, device="cuda")
    if case["op"] != "attend":
        st["rows"] = _pick(g, n, m)
        st["idx"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["idx"][:m] = st["rows"].int()
        st["count"] = torch.tensor([m], dtype=torch.int32, device="cuda")
        st["mask"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["mask"][st["rows"]] = 2
        st["cache"] = _cache(g, n, h, case["fmt"], t)
        if case["op"] != "read":  # a new stream's: nothing is in it yet
            st["cache"] = {name: torch.zeros_like(x) for name, x in st["cache"].items()}
        st["k_out"] = torch.zeros(m, h * D, dtype=t, device="cuda")
        st["v_out"] = torch.zeros(m, h * D, dtype=t, device="cuda")
        return st
    s, p, docs = case["streams"], case["prefix"], case["docs"]
    counts = [max(1, m - 3 * b) for b in range(s)]
    st["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    st["qc"] = torch.randn(s, m, h * D, generator=g, device="cuda")
    st["qc"] = (st["qc"].view(s, m, h, D) * torch.rsqrt(st["qc"].view(s, m, h, D).square().mean(-1, keepdim=True) + EPS)).view(s, m, h * D).to(t)
    st["idx"] = torch.stack([_pick(g, n, m) for _ in range(s)]).int()
    # the live rows: stream, compact row, token
    st["live"] = (torch.cat([torch.full((c,), b, device="cuda") for b, c in enumerate(counts)]),
                  torch.cat([torch.arange(c, device="cuda") for c in counts]))
    st["caches"] = [_cache(g, n, h, case["fmt"], t) for _ in range(s)]
    st["prefix"] = _cache(g, p, h, case["fmt"], t) if p else None
    st["out"] = torch.zeros(s, n, h * D, dtype=t, device="cuda")
    st["q_groups"] = st["k_groups"] = st["p_groups"] = None
    if docs:
        # each stream's tokens are `docs` documents; every 17th query sees nothing; of the shared rows
        # the last sixteenth is padding that nobody sees
        at = torch.arange(n, device="cuda")
        doc = torch.bitwise_left_shift(torch.ones_like(at), at * docs // n).int()
        st["k_groups"] = doc.expand(s, n).contiguous()
        st["q_groups"] = torch.where(at % 17 == 5, torch.zeros_like(doc), doc).expand(s, n).contiguous()
        if p:
            st["p_groups"] = torch.full((p,), -1, dtype=torch.int32, device="cuda")
            st["p_groups"][p - p // 16:] = 0
    return st


# ---- plain forms ----------------------------------------------------------------------------------
def _values(codes, scale, heads, rows=None):
    """Codes [n, heads * 128] times their scales, in 32 bits: [n, heads, 128]."""
    x, s = codes, scale[:, :codes.shape[0]].t()
    if rows is not None:
        x, s = _take(codes, rows), s[rows]
    return x.float().view(-1, heads, D) * s.float()[..., None]


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _turned(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _angles(pos):
    freq = torch.cat([THETA ** (-torch.arange(0, a, 2, device=pos.device, dtype=torch.float64) / a) for a in AXES])
    axis = torch.repeat_interleave(torch.arange(3, device=pos.device), torch.tensor([a // 2 for a in AXES], device=pos.device))
    return (pos.double()[:, axis] * freq)[:, None, :]


def _plain_write(st):
    h, t, rows, c = st["case"]["heads"], st["t"], st["rows"], st["cache"]
    ang = _angles(st["pos"][rows])
    cos, sin = ang.cos().float(), ang.sin().float()
    q, k, v = (st[x][rows].float().view(-1, h, D) for x in "qkv")
    st["qc"][:len(rows)] = _turned(_normed(q, st["norm_q"]), cos, sin).reshape(len(rows), -1).to(t)
    k = _turned(_normed(k, st["norm_k"]), cos, sin)
    codes, s = _quantise(k, st["case"]["fmt"], t)
    c["k"].view(torch.int8)[rows] = codes.reshape(len(rows), -1).view(torch.int8)
    c["k_scale"][:, rows] = s.t()
    codes, s = _quantise(v, st["case"]["fmt"], t)
    c["v"].view(torch.int8)[rows] = codes.reshape(len(rows), -1).view(torch.int8)
    c["v_scale"][:, rows] = s.t()


def _plain_read(st):
    h, c = st["case"]["heads"], st["cache"]
    rows = st["rows"] if st["case"]["m"] else None
    st["k_out"].copy_(_values(c["k"], c["k_scale"], h, rows).flatten(1))
    st["v_out"].copy_(_values(c["v"], c["v_scale"], h, rows).flatten(1))


def _plain_attend(st):
    case, h, t = st["case"], st["case"]["heads"], st["t"]
    s, n, m = case["streams"], case["n"], st["idx"].shape[1]
    codes = lambda name: torch.stack([c[name].view(torch.int8) for c in st["caches"]]).view(st["caches"][0][name].dtype)  # noqa: E731
    scales = lambda name: torch.stack([c[name] for c in st["caches"]])[:, :, :n].transpose(1, 2).float()[..., None]  # noqa: E731
    k = codes("k").float().view(s, n, h, D) * scales("k_scale")
    v = codes("v").float().view(s, n, h, D) * scales("v_scale")
    if st["prefix"]:
        p = st["prefix"]
        k = torch.cat([_values(p["k"], p["k_scale"], h).expand(s, -1, -1, -1), k], 1)
        v = torch.cat([_values(p["v"], p["v_scale"], h).expand(s, -1, -1, -1), v], 1)
    q = st["qc"].float().view(s, m, h, D).transpose(1, 2)
    x = (q @ k.permute(0, 2, 3, 1)) * (1 / math.sqrt(D))
    if st["q_groups"] is not None:
        qg = torch.gather(st["q_groups"], 1, st["idx"].long())
        kg = st["k_groups"]
        if st["p_groups"] is not None:
            kg = torch.cat([st["p_groups"].expand(s, -1), kg], 1)
        x = x.masked_fill(((qg[:, :, None] & kg[:, None, :]) == 0)[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = x.sum(-1, keepdim=True)
    o = (x @ v.transpose(1, 2)) / torch.where(total > 0, total, torch.ones_like(total))
    b, r = st["live"]
    st["out"][b, st["idx"][b, r].long()] = o.transpose(1, 2)[b, r].reshape(len(b), -1).to(t)


# ---- the package's calls --------------------------------------------------------------------------
def _handles(st):
    """What a program builds once: the frame's configuration, the caches' and streams' handles, a workspace."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fluxrt-cpp_b200"))
    import fxr
    case = st["case"]
    cfg = fxr.FrameConfig(n_tokens=case["n"], n_text=0, n_heads=case["heads"], dtype=case["dtype"], rope_axes=AXES,
                          rope_theta=THETA, eps=EPS)
    as_cache = lambda c: fxr.CacheQ8(c["k"], c["v"], c["k_scale"], c["v_scale"])  # noqa: E731
    if case["op"] != "attend":
        return fxr, cfg, as_cache(st["cache"])
    streams = fxr.q8_streams([
        {"qc": st["qc"][b], "idx": st["idx"][b], "count": st["counts"][b:b + 1], "cache": as_cache(st["caches"][b]), "out": st["out"][b],
         "q_groups": None if st["q_groups"] is None else st["q_groups"][b],
         "k_groups": None if st["k_groups"] is None else st["k_groups"][b]} for b in range(case["streams"])])
    prefix = as_cache(st["prefix"]) if st["prefix"] else None
    size = fxr.attention_q8_workspace_size(cfg, case["streams"], case["prefix"], st["idx"].shape[1])
    return fxr, cfg, (streams, prefix, torch.zeros(size, dtype=torch.uint8, device="cuda"))


def _own(st):
    if "handles" not in st:
        st["handles"] = _handles(st)
    fxr, cfg, held = st["handles"]
    case = st["case"]
    if case["op"] in ("write", "turn"):
        fxr.gather_norm_rope_q8(cfg, st["q"], st["k"], st["v"], st["mask"], st["idx"], st["count"], st["pos"], st["norm_q"],
                                st["norm_k"], st["qc"], held)
    if case["op"] in ("read", "turn"):
        listed_rows = case["m"] > 0
        fxr.cache_read_q8(cfg, held, st["k_out"], st["v_out"], idx=st["idx"] if listed_rows else None,
                          count=st["count"] if listed_rows else None)
    if case["op"] == "attend":
        streams, prefix, workspace = held
        fxr.attention_q8(cfg, streams, workspace, prefix=prefix, prefix_groups=st["p_groups"], max_rows=st["idx"].shape[1])


def run(state):
    case = state["case"]
    if own:
        _own(state)
    else:
        if case["op"] in ("write", "turn"):
            _plain_write(state)
        if case["op"] in ("read", "turn"):
            _plain_read(state)
        if case["op"] == "attend":
            _plain_attend(state)
    c = state.get("cache")
    if case["op"] == "write":
        return {"qc": state["qc"], "k": c["k"], "v": c["v"], "k_scale": c["k_scale"], "v_scale": c["v_scale"]}
    if case["op"] == "turn":
        return {"qc": state["qc"], "k": state["k_out"], "v": state["v_out"], "k_scale": c["k_scale"], "v_scale": c["v_scale"]}
    if case["op"] == "read":
        return {"k": state["k_out"], "v": state["v_out"]}
    return state["out"]


def work(case):
    c, h, n = case["heads"] * D, case["heads"], case["n"]
    m = case["m"] or n
    wr = m * (6 * c + 2 * c + 2 * c + 4 * h + 12 + 8)
    rd = m * (2 * c + 4 * h + 4 * c + 4)
    if case["op"] == "write":
        return {"bytes": wr, "flops": 40 * m * c}
    if case["op"] == "turn":
        return {"bytes": wr + rd, "flops": 42 * m * c}
    if case["op"] == "read":
        return {"bytes": rd, "flops": 2 * m * c}
    s, p, docs = case["streams"], case["prefix"], case["docs"]
    rows = sum(max(1, m - 3 * b) for b in range(s))
    seen = p - (p // 16 if docs else 0) + (n // docs if docs else n)
    return {"bytes": 4 * rows * c + (p + s * n) * (2 * c + 4 * h) + (4 * (p + s * n) + 4 * rows if docs else 0),
            "flops": 4 * D * h * rows * seen * (16 / 17 if docs else 1)}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _ceil_to(t, dtype):
    """The smallest number of dtype not below t > 0 (t = 0 stays 0), by its exponent and mantissa bits."""
    bits, low = (7, -133) if dtype == torch.bfloat16 else (10, -24)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(t, min=1e-300))) - bits, min=low))
    return torch.ceil(t / step) * step


def _exact_codes(x, fmt, dtype):
    s = _ceil_to(x.abs().amax(-1) / TOP[fmt], dtype)
    y = x / torch.where(s > 0, s, torch.ones_like(s))[..., None]
    if fmt == "e4m3":
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=1e-30))), min=-6) - 3)
        y = torch.clamp(torch.round(y / step) * step, -448, 448)
    else:
        y = torch.clamp(torch.round(y), -127, 127)
    return y, s


def exact(case, seed):
    st = prepare(case, seed)
    h, n = case["heads"], case["n"]
    if case["op"] == "attend":
        out = st["out"].double()
        for b, c in enumerate(st["caches"]):
            m = int(st["counts"][b])
            rows = st["idx"][b, :m].long()
            for head in range(h):
                cols = slice(head * D, (head + 1) * D)
                parts = [(c, n, None if st["k_groups"] is None else st["k_groups"][b])]
                if st["prefix"]:
                    parts.insert(0, (st["prefix"], case["prefix"], st["p_groups"]))
                k = torch.cat([x["k"][:, cols].double() * x["k_scale"][head, :r, None].double() for x, r, _ in parts])
                v = torch.cat([x["v"][:, cols].double() * x["v_scale"][head, :r, None].double() for x, r, _ in parts])
                w = st["qc"][b, :m, cols].double() @ k.t() / math.sqrt(D)
                if st["q_groups"] is not None:
                    seen = torch.cat([torch.full((r,), -1, dtype=torch.int32, device="cuda") if kg is None else kg for _, r, kg in parts])
                    w[(st["q_groups"][b][rows][:, None] & seen[None]) == 0] = -math.inf
                w = torch.softmax(w, -1)
                out[b, rows, cols] = torch.nan_to_num(w, nan=0.0) @ v
        return out
    c, rows = st["cache"], st["rows"]
    res = {}
    if case["op"] == "read":
        at = rows if case["m"] else torch.arange(n, device="cuda")
        for name in ("k", "v"):
            s = c[name + "_scale"].double()[:, at].t()
            res[name] = (_take(c[name], at).double().view(len(at), h, D) * s[..., None]).flatten(1)
        return res
    pos = st["pos"][rows].double()
    ang = torch.cat([pos[:, i:i + 1] * THETA ** (-torch.arange(a // 2, device="cuda").double() * 2 / a) for i, a in enumerate(AXES)], 1)
    turn = torch.polar(torch.ones_like(ang), ang)[:, None]
    made = {}
    for name in "qk":
        x = st[name][rows].double().view(len(rows), h, D)
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * st["norm_" + name].double()
        made[name] = torch.view_as_real(torch.view_as_complex(x.view(len(rows), h, D // 2, 2)) * turn).flatten(-2)
    made["v"] = st["v"][rows].double().view(len(rows), h, D)
    res["qc"] = st["qc"].double()
    res["qc"][:len(rows)] = made["q"].flatten(1)
    for name in "kv":
        codes, s = _exact_codes(made[name], case["fmt"], st["t"])
        res[name + "_scale"] = c[name + "_scale"].double()
        res[name + "_scale"][:, rows] = s.t()
        if case["op"] == "turn":
            res[name] = (codes * s[..., None]).flatten(1)
        else:
            res[name] = c[name].double()
            res[name][rows] = codes.flatten(1)
    return res
