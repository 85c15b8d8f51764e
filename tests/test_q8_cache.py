"""The 8-bit spatial cache: quantised write, read-back, attention over it, the frame of all three.

Bars, all derived before the first run, with u = finfo(T).eps / 2 (half a step of the 16-bit type):
  V codes and scales, read-back, restore: bit-exact (the definition in 64 bits on the same T values).
  Q': one rounding to T of the value, plus 4e-6 for the 32-bit norm and rotation (values up to ~6 through
  some ten roundings of 2^-24 each). K': read-back within half a code step of the value, plus the same 4e-6.
  Attention, element-wise: an output is a weighted mean sum(w v), w = p / sum(p). P and V (or P * V's
  scale) are rounded to T, at most u each, exponentials to 2^-13 (a degree-3 polynomial in part), K to
  u, which moves a score by at most ds = u * scale * max_j sum|q k_j|. Scores moved by up to ds change a
  weight by a factor within exp(+-2 ds) (its numerator by exp(+-ds), the sum by as much), so the mean by
  at most (exp(2 ds) - 1) sum(w |v|). The output is rounded once more:
      |err| <= u |o| + (2 u + 2^-13 + exp(2 ds) - 1) sum(w |v|)
  Attention, root mean square, where ds is at most 0.1, so that first order holds: the same roundings as
  independent uniform ones (u / sqrt(3) each):
      rms^2 <= 2^2 * mean(u^2 / 3 * (o^2 + sum(w^2 (2 v^2 + (v - o)^2 e_j)))),  e_j = scale^2 sum(q k_j)^2
  and 2^-13 * sum(w |v|) on top.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import fxr

D = 128
TDT = {"f16": torch.float16, "bf16": torch.bfloat16}
TOP = {"int8": 127.0, "e4m3": 448.0}


# ---- the definitions, in 64 bits -----------------------------------------------------------------
def up_to(t, dtype):
    """t >= 0 (float64) rounded up to a number of dtype."""
    bits, low = (7, -133) if dtype == torch.bfloat16 else (10, -24)
    e = torch.floor(torch.log2(torch.clamp(t, min=1e-300)))
    e = torch.where(torch.exp2(e) > t, e - 1, e)
    step = torch.exp2(torch.clamp(e - bits, min=low))
    return torch.ceil(t / step) * step


def quantise(x, fmt, dtype):
    """x [..., 128] float64 -> code values (float64) and scales (float64); not finite: NaN scale, codes 0."""
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    t = x.abs().amax(-1) / TOP[fmt]
    s = up_to(t, dtype)
    cap = torch.finfo(dtype).max / (128 if fmt == "int8" else 448)      # of the type itself for int8
    if fmt == "e4m3":
        cap = 146.125 if dtype == torch.float16 else math.floor(cap / 2.0 ** 112) * 2.0 ** 112
    s = torch.clamp(s, max=cap)
    y = x / torch.where(s > 0, s, torch.ones_like(s))[..., None]
    if fmt == "int8":
        y = torch.clamp(torch.round(y), -127, 127)
    else:
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=1e-30))), min=-6) - 3)
        y = torch.clamp(torch.round(y / step) * step, -448, 448)
    return y, torch.where(bad, torch.full_like(s, math.nan), s)


def values(cache, n=None):
    """A CacheQ8's K and V in float64: [n, heads, 128] each (codes times scales, not rounded)."""
    n = cache.n_rows if n is None else n
    h = cache.n_heads
    out = []
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = c[:n, :h * D].contiguous().view(torch.int8)
        x = x.view(c.dtype).float().double().view(n, h, D)
        out.append(x * s[:h, :n].t().double()[..., None])
    return out


def attend(q, k, v, seen, scale):
    """q [m, h, D], k / v [n, h, D], seen [m, n] bool -> (o, sum(w|v|), the variance term, ds) per element."""
    bad = ~torch.isfinite(k).all(-1).t() | ~torch.isfinite(v).all(-1).t()             # [h, n]
    kk, vv = (torch.nan_to_num(x).permute(1, 0, 2) for x in (k, v))
    qq = q.permute(1, 0, 2)
    s = qq @ kk.transpose(1, 2) * scale
    s = torch.where(bad[:, None, :], torch.full_like(s, math.nan), s)
    s = s.masked_fill(~seen[None], -math.inf)
    top = torch.nan_to_num(s, nan=-math.inf).amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    w = p / torch.where(p.sum(-1, keepdim=True) == 0, torch.ones(1, device=p.device, dtype=p.dtype), p.sum(-1, keepdim=True))
    o = w @ vv
    mean_abs = w @ vv.abs()
    e = (qq.square() @ kk.square().transpose(1, 2)) * scale * scale
    w2 = w.square()
    var = w2 @ (2 * vv.square()) + (w2 * e) @ vv.square() - 2 * o * ((w2 * e) @ vv) + (w2 * e).sum(-1, keepdim=True) * o.square()
    ds = (qq.abs() @ kk.abs().transpose(1, 2) * scale).masked_fill(~seen[None] | bad[:, None, :], 0).amax(-1, keepdim=True)   # of keys that the row sees
    return [x.permute(1, 0, 2) for x in (o, mean_abs, var, ds.expand_as(o))]


def check_attention(got, ref, dtype, what=""):
    o, mean_abs, var, ds = ref
    u = torch.finfo(dtype).eps / 2
    got = got.double().view(o.shape)
    nan = torch.isnan(o)
    assert torch.equal(torch.isnan(got), nan), what + ": NaN in other places"
    err = torch.where(nan, torch.zeros_like(o), (got - o).abs())
    o, mean_abs, var, ds = (torch.nan_to_num(x) for x in (o, mean_abs, var, ds))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps            # the smallest subnormal step
    bound = u * o.abs() + (2 * u + 2 ** -13 + torch.expm1(torch.clamp(2 * u * ds, max=600.0))) * mean_abs + tiny
    # exp(600) times a weight that 64 bits round to 0 (below exp(-745)) is not 0: there the bound says nothing
    bound = torch.where(2 * u * ds > 600, torch.full_like(bound, math.inf), bound)
    assert (err <= bound).all(), f"{what}: {float((err / bound).max()):.2f} of the bound"
    if err.numel() >= 256 and float(u * ds.max()) <= 0.1:
        rms = float(err.square().mean().sqrt())
        want = 2 * float((u * u / 3 * (o.square() + var)).mean().sqrt()) + 2 ** -13 * float(mean_abs.mean()) + tiny
        assert rms <= want, f"{what}: rms {rms:.3e}, bar {want:.3e}"


# ---- inputs ---------------------------------------------------------------------------------------
def cfg_of(n, heads, dtype, **more):
    return fxr.FrameConfig(n_tokens=n, n_text=0, n_heads=heads, dtype=dtype, **more)


def rng_of(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def filled_cache(g, cfg, rows, fmt, pad=0, extra_scale=0):
    """A cache of random rows: keys of unit mean square, plain values. pad: code columns past the heads'."""
    t, h = TDT[cfg.dtype], cfg.n_heads
    code = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    lanes = max(8, -(-rows // 8) * 8) + extra_scale
    made = []
    for kind in range(2):
        x = randn(g, rows, h, D).double()
        if kind == 0:
            x = x / x.square().mean(-1, keepdim=True).sqrt() if rows else x
        y, s = quantise(x, fmt, t) if rows else (x, x[..., 0])
        store = torch.full((rows, h * D + pad), 77, dtype=torch.int8, device="cuda")
        store[:, :h * D] = (y.to(torch.int8) if fmt == "int8" else y.float().to(code).view(torch.int8)).view(rows, h * D)
        sc = torch.full((h, lanes), math.nan, dtype=t, device="cuda")       # what lies behind the rows must not matter
        sc[:, :rows] = s.t().to(t)
        made.append((store.view(code), sc))
    return fxr.CacheQ8(made[0][0], made[1][0], made[0][1], made[1][1])


def stream_of(g, cfg, m, ld_extra=0, out_extra=0, idx=None):
    """A stream's queries (NaN behind the live rows), list, count and output, the output filled with 7 (rows
    that are not listed stay so)."""
    t, h, n = TDT[cfg.dtype], cfg.n_heads, cfg.n_tokens
    q = randn(g, m, h, D)
    q = (q / q.square().mean(-1, keepdim=True).sqrt()).view(m, h * D).to(t) if m else q.view(0, h * D).to(t)
    store = torch.full((n, h * D + ld_extra), math.nan, dtype=t, device="cuda")
    store[:m, :h * D] = q
    if idx is None:
        idx = torch.randperm(n, generator=g, device="cuda")[:m].sort().values.int()
    out = torch.full((n, h * D + out_extra), 7.0, dtype=t, device="cuda")
    return {"qc": store[:, :h * D], "idx": idx if m else torch.zeros(1, dtype=torch.int32, device="cuda"),
            "count": torch.tensor([m], dtype=torch.int32, device="cuda"), "out": out[:, :h * D], "m": m}


def workspace_for(cfg, streams, prefix=None, max_rows=0):
    size = fxr.attention_q8_workspace_size(cfg, len(streams), prefix.n_rows if prefix else 0, max_rows)
    return torch.zeros(size, dtype=torch.uint8, device="cuda")


def expected(cfg, st, prefix=None, prefix_groups=None):
    """attend() of one stream's rows."""
    n, m, h = cfg.n_tokens, st["m"], cfg.n_heads
    k, v = values(st["cache"], n)
    kg = st.get("k_groups")
    kg = torch.full((n,), -1, dtype=torch.int32, device="cuda") if kg is None else kg.view(torch.int32)[:n]
    if prefix is not None:
        pk, pv = values(prefix)
        pg = torch.full((prefix.n_rows,), -1, dtype=torch.int32, device="cuda") if prefix_groups is None else prefix_groups
        k, v, kg = torch.cat([pk, k]), torch.cat([pv, v]), torch.cat([pg.view(torch.int32), kg])
    rows = st["idx"][:m].long()
    qg = st.get("q_groups")
    qg = torch.full((m,), -1, dtype=torch.int32, device="cuda") if qg is None else qg.view(torch.int32)[rows]
    scale = cfg.softmax_scale if cfg.softmax_scale > 0 else 1 / math.sqrt(D)
    return attend(st["qc"][:m].double().view(m, h, D), k, v, (qg[:, None] & kg[None]) != 0, scale)


def check_streams(cfg, streams, prefix=None, prefix_groups=None, what=""):
    for b, st in enumerate(streams):
        rows = st["idx"][:st["m"]].long()
        if st["m"]:
            check_attention(st["out"][rows], expected(cfg, st, prefix, prefix_groups), TDT[cfg.dtype], f"{what} stream {b}")
        rest = torch.ones(cfg.n_tokens, dtype=torch.bool, device="cuda")
        rest[rows] = False
        assert (st["out"][rest] == 7.0).all(), f"{what} stream {b}: rows that are not listed changed"


def sync_ok():
    torch.cuda.synchronize()
    assert fxr.check_device_error() == 0


# ---- refusals (no GPU) ----------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    import build as B
    B.build()
    return fxr.load()


def _cache_struct(**over):
    c = fxr.Q8CacheStruct(4096, 4096, 4096, 4096, 256, 64, 64, fxr.FXR_Q8_INT8)
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("bad, word", [({"format": 2}, "format"), ({"ld": 240}, "ld"), ({"ld": 264}, "ld"), ({"ld_scale": 60}, "ld_scale"),
                                       ({"ld_scale": 68}, "ld_scale"), ({"n_rows": 63}, "rows"), ({"k": None}, "null"),
                                       ({"v_scale": None}, "null"), ({"k": 4104}, "aligned"), ({"k_scale": 4098}, "aligned")])
def test_bad_caches_are_refused(lib, bad, word):
    d = ctypes.byref(cfg_of(64, 2, "bf16").desc())
    c = _cache_struct(**bad)
    for st in (lib.fxr_gather_norm_rope_q8(d, *([4096] * 10), 256, ctypes.byref(c), None, None),
               lib.fxr_cache_write_q8(d, 4096, 4096, None, None, 64, ctypes.byref(c), None),
               lib.fxr_restore_rows_q8(d, 4096, 4096, 4096, 4096, ctypes.byref(c), None)):
        assert st == fxr.FXR_ERR_INVALID
        assert word.encode() in lib.fxr_last_error_string()
    s = fxr.Q8StreamStruct(4096, 256, 4096, 4096, 4096, None, None, c)
    assert lib.fxr_attention_q8(d, 1, ctypes.byref(s), None, None, 0, 4096, 1 << 40, None) == fxr.FXR_ERR_INVALID
    assert word.encode() in lib.fxr_last_error_string()


def test_bad_arguments_are_refused(lib):
    cfg = cfg_of(64, 2, "bf16")
    d, c = ctypes.byref(cfg.desc()), _cache_struct()
    inv, last = fxr.FXR_ERR_INVALID, lib.fxr_last_error_string
    ok = [4096] * 10
    assert lib.fxr_gather_norm_rope_q8(d, *ok, 256, None, None, None) == inv and b"null" in last()
    assert lib.fxr_gather_norm_rope_q8(d, *ok, 248, ctypes.byref(c), None, None) == inv and b"ld_qc" in last()
    assert lib.fxr_gather_norm_rope_q8(d, *ok, 260, ctypes.byref(c), None, None) == inv and b"ld_qc" in last()
    assert lib.fxr_gather_norm_rope_q8(d, *ok, 256, ctypes.byref(c), 4100, None) == inv and b"aligned" in last()
    assert lib.fxr_gather_norm_rope_q8(d, 4100, *ok[1:], 256, ctypes.byref(c), None, None) == inv and b"aligned" in last()
    assert lib.fxr_gather_norm_rope_q8(d, None, *ok[1:], 256, ctypes.byref(c), None, None) == inv and b"null" in last()
    assert lib.fxr_cache_write_q8(d, 4096, 4096, None, None, -1, ctypes.byref(c), None) == inv and b"count" in last()
    assert lib.fxr_cache_write_q8(d, 4096, 4096, None, None, 65, ctypes.byref(c), None) == inv and b"host_count" in last()
    assert lib.fxr_cache_write_q8(d, 4100, 4096, None, None, 64, ctypes.byref(c), None) == inv and b"aligned" in last()
    assert lib.fxr_cache_read_q8(d, ctypes.byref(c), None, None, 65, 4096, 4096, 256, None) == inv and b"host_count" in last()
    assert lib.fxr_cache_read_q8(d, ctypes.byref(c), None, None, -1, 4096, 4096, 256, None) == inv and b"count" in last()
    assert lib.fxr_cache_read_q8(d, ctypes.byref(c), None, None, 64, 4096, 4096, 250, None) == inv and b"ld" in last()
    assert lib.fxr_cache_read_q8(d, ctypes.byref(c), None, None, 64, 4096, 4104, 256, None) == inv and b"aligned" in last()
    assert lib.fxr_restore_rows_q8(d, 4096, 4096, 4096, None, ctypes.byref(c), None) == inv and b"null" in last()
    big = 1 << 40

    def call(s, prefix=None, pg=None, ws=4096, size=big, n=1):
        return lib.fxr_attention_q8(d, n, ctypes.byref(s) if s is not None else None,
                                    ctypes.byref(prefix) if prefix is not None else None, pg, 0, ws, size, None)
    good = lambda **o: fxr.Q8StreamStruct(*[o.get(k, v) for k, v in dict(  # noqa: E731
        qc=4096, ld_qc=256, idx=4096, count=4096, out=4096, q_groups=None, k_groups=None, cache=c).items()])
    assert call(None) == inv and call(good(), n=-1) == inv
    for over, word in (({"qc": None}, b"null"), ({"idx": None}, b"null"), ({"count": None}, b"null"), ({"out": None}, b"null"),
                       ({"qc": 4100}, b"aligned"), ({"out": 4104}, b"aligned"), ({"ld_qc": 248}, b"ld_qc"), ({"ld_qc": 257}, b"ld_qc"),
                       ({"q_groups": 4098}, b"q_groups"), ({"k_groups": 4098}, b"k_groups")):
        assert call(good(**over)) == inv and word in last(), over
    assert call(good(), ws=None) == inv and b"workspace" in last()
    assert call(good(), ws=4100) == inv and b"aligned" in last()
    assert call(good(), size=16) == fxr.FXR_ERR_WORKSPACE
    assert call(good(), prefix=_cache_struct(format=fxr.FXR_Q8_E4M3)) == inv and b"format" in last()
    assert call(good(), prefix=_cache_struct(ld=100)) == inv and b"prefix" in last()
    assert call(good(), prefix=_cache_struct(), pg=4098) == inv and b"prefix_groups" in last()
    # nothing to do: no launch, no error
    assert lib.fxr_attention_q8(d, 0, None, None, None, 0, None, 0, None) == fxr.FXR_OK
    none = ctypes.byref(cfg_of(0, 2, "bf16").desc())
    assert lib.fxr_attention_q8(none, 1, None, None, None, 0, None, 0, None) == fxr.FXR_OK
    assert lib.fxr_cache_write_q8(d, None, None, None, None, 0, ctypes.byref(c), None) == fxr.FXR_OK
    assert lib.fxr_cache_read_q8(d, ctypes.byref(c), None, None, 0, None, None, 256, None) == fxr.FXR_OK
    # other head dims and 32-bit frames are not built
    other = fxr.FrameConfig(n_tokens=64, n_text=0, n_heads=2, head_dim=64, dtype="bf16").desc()
    assert lib.fxr_cache_read_q8(ctypes.byref(other), ctypes.byref(c), None, None, 64, 4096, 4096, 256, None) == fxr.FXR_ERR_UNSUPPORTED
    wide = fxr.FrameConfig(n_tokens=64, n_text=0, n_heads=2, dtype="f32").desc()
    assert lib.fxr_cache_read_q8(ctypes.byref(wide), ctypes.byref(c), None, None, 64, 4096, 4096, 256, None) == fxr.FXR_ERR_UNSUPPORTED
    assert lib.fxr_frame_forward_q8(d, *([4096] * 8), ctypes.byref(c), None, None, None, None, 0, 4096, None, big, None) == inv
    assert lib.fxr_frame_forward_q8(d, *([4096] * 8), ctypes.byref(c), None, None, None, None, 0, 4096, 4096, 16, None) == fxr.FXR_ERR_WORKSPACE


def test_a_configuration_s_reference_follows_its_fields():
    cfg = cfg_of(8, 2, "bf16")
    first = cfg.ref()
    assert cfg.ref() is first and first._obj.n_tokens == 8
    cfg.n_tokens = 9
    assert cfg.ref()._obj.n_tokens == 9 and cfg.desc().n_tokens == 9


def test_structs_match_the_header():
    assert ctypes.sizeof(fxr.Q8CacheStruct) == 4 * 8 + 2 * 8 + 2 * 4
    assert ctypes.sizeof(fxr.Q8StreamStruct) == 7 * 8 + 56 and fxr.Q8StreamStruct.cache.offset == 56


def test_workspaces_grow_with_the_bound(lib):
    cfg = cfg_of(4608, 24, "bf16")
    one, few, all_rows = (fxr.attention_q8_workspace_size(cfg, 1, 0, r) for r in (1, 64, 0))
    assert 0 < one < few < all_rows == fxr.attention_q8_workspace_size(cfg, 1, 0, 4608)
    assert fxr.attention_q8_workspace_size(cfg, 8, 0, 16) == fxr.attention_q8_workspace_size(cfg, 20, 0, 16)   # groups reuse it
    assert fxr.attention_q8_workspace_size(cfg, 0) == 0 and fxr.attention_q8_workspace_size(cfg, 1, -1) == 0
    assert fxr.frame_q8_workspace_size(cfg, 0, 16) > fxr.attention_q8_workspace_size(cfg, 1, 0, 16)


def test_binding_refuses_other_types():
    k = torch.zeros(16, 256, dtype=torch.int8)
    s = torch.zeros(2, 16, dtype=torch.bfloat16)
    fxr.CacheQ8(k, k.clone(), s, s.clone())
    st = {"qc": torch.zeros(3, 256, dtype=torch.bfloat16), "idx": k, "count": k, "out": torch.zeros(16, 256, dtype=torch.bfloat16),
          "cache": fxr.CacheQ8(k, k, s, s)}
    with pytest.raises(fxr.FxrError, match="qc holds 3 rows"):
        fxr.Q8Streams([st]).check(cfg_of(16, 2, "bf16"), 4)
    with pytest.raises(fxr.FxrError, match="out holds 16 rows"):
        fxr.Q8Streams([st]).check(cfg_of(17, 2, "bf16"), 3)
    with pytest.raises(fxr.FxrError, match="16 rows, 2 heads"):
        fxr.Q8Streams([st]).check(cfg_of(16, 3, "bf16"), 3)
    with pytest.raises(fxr.FxrError, match="CUDA device"):
        fxr.q8_streams([st])
    with pytest.raises(fxr.FxrError, match="q_groups"):
        fxr.Q8Streams([dict(st, q_groups=torch.zeros(15, dtype=torch.int32))]).check(cfg_of(16, 2, "bf16"), 3)
    with pytest.raises(fxr.FxrError, match="one type"):
        fxr.Q8Streams([dict(st, out=k)])
    for bad in ((k.float(), k, s, s), (k, k.view(torch.float8_e4m3fn), s, s), (k, k, s.float(), s.float()), (k, k, s, s.half()),
                (k, k[:8], s, s), (k, k, s[:, :8], s[:, :8]), (k[:, :128], k[:, :128], s, s), (k.t(), k.t(), s, s)):
        with pytest.raises(fxr.FxrError):
            fxr.CacheQ8(*bad)


# ---- write, read, restore -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_every_code_reads_back_exactly(cuda, dtype, fmt):
    """All 256 codes (but e4m3's two NaN codes) times scales from the smallest to the largest that the type holds."""
    t = TDT[dtype]
    cfg = cfg_of(2, 1, dtype)
    codes = torch.arange(256, dtype=torch.int32, device="cuda").to(torch.uint8).view(torch.int8)
    if fmt == "e4m3":
        codes = torch.where((codes & 127) == 127, torch.zeros_like(codes), codes)
    scales = torch.tensor([2.0 ** -24, 3 * 2.0 ** -24, 2.0 ** -14, 1e-3, 0.37, 1.0, 5.5, 100.0, 140.0], device="cuda").to(t)
    code_t = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    for s in scales:
        c = fxr.CacheQ8(codes.view(2, 128).view(code_t), codes.view(2, 128).clone().view(code_t), s.expand(1, 8).contiguous(),
                        s.expand(1, 8).contiguous())
        k, v = torch.zeros(2, 128, dtype=t, device="cuda"), torch.zeros(2, 128, dtype=t, device="cuda")
        fxr.cache_read_q8(cfg, c, k, v)
        sync_ok()
        want = (c.k.float() * s.float()).to(t)      # exact in 32 bits, one rounding
        assert torch.equal(k, want) and torch.equal(v, want), float(s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n, heads", [(1, 1), (37, 3), (300, 24)])
def test_written_rows_are_the_definition(cuda, dtype, fmt, n, heads):
    """16-bit rows to codes and scales, bit for bit, all rows and listed ones; the rows behind stay as they were."""
    t = TDT[dtype]
    g = rng_of(n + heads)
    cfg = cfg_of(n, heads, dtype, ld_cache=heads * D + 24)
    x = [torch.zeros(n, heads * D + 24, dtype=t, device="cuda") for _ in range(2)]
    for a in x:
        a[:, :heads * D] = (randn(g, n, heads * D) * torch.exp(4 * randn(g, n, 1))).to(t)
        a[0, :D] = 0                                                        # a vector of zeros
    if n > 30:
        x[0][3, 5], x[1][4, 7], x[0][6, 9] = math.nan, math.inf, torch.finfo(t).max
        x[1][7, :D] = torch.finfo(t).smallest_normal * torch.finfo(t).eps   # the smallest value of the type
        x[1][8, :D] = randn(g, D).to(t) * 2.0 ** -13
    for listed in (False, True):
        cache = fxr.CacheQ8.empty(cfg, n + 3, fmt)
        for a in (cache.k, cache.v):
            a.view(torch.int8).fill_(33)
        for a in (cache.k_scale, cache.v_scale):
            a.fill_(3)
        rows = torch.randperm(n, generator=g, device="cuda")[:max(1, n // 2)] if listed else torch.arange(n, device="cuda")
        if listed:
            fxr.cache_write_q8(cfg, x[0], x[1], cache, idx=rows.int(), count=torch.tensor([len(rows)], dtype=torch.int32, device="cuda"))
        else:
            fxr.cache_write_q8(cfg, x[0], x[1], cache)
        sync_ok()
        rest = torch.ones(n + 3, dtype=torch.bool, device="cuda")
        rest[rows] = False
        for a, codes, scale in ((x[0], cache.k, cache.k_scale), (x[1], cache.v, cache.v_scale)):
            y, s = quantise(a[rows, :heads * D].double().view(-1, heads, D), fmt, t)
            assert torch.equal(torch.nan_to_num(scale[:, rows].t().double(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))
            got = codes.view(torch.int8)[rows].view(codes.dtype).float().double().view(-1, heads, D)
            assert torch.equal(got, y)
            assert (codes.view(torch.int8)[rest] == 33).all() and (scale[:, :n + 3][:, rest] == 3).all()
        k, v = (torch.full((n + 3, heads * D + 8), 5.0, dtype=t, device="cuda") for _ in range(2))
        fxr.cache_read_q8(cfg, cache, k[:, :heads * D], v[:, :heads * D], idx=rows.int(),
                          count=torch.tensor([len(rows)], dtype=torch.int32, device="cuda"))
        sync_ok()
        for a, got in zip(values(cache), (k, v)):
            want = a[rows].view(len(rows), -1).to(t)        # 64-bit products are exact: one rounding
            assert torch.equal(torch.nan_to_num(got[:len(rows), :heads * D], nan=-9.0), torch.nan_to_num(want, nan=-9.0))
            assert (got[len(rows):] == 5).all() and (got[:, heads * D:] == 5).all()


def rope_exact(x, w, pos, axes, theta, eps):
    n, h = x.shape[0], x.shape[1]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    ang = torch.cat([pos[:, i:i + 1].double() * theta ** (-torch.arange(a // 2, device=x.device).double() * 2 / a)
                     for i, a in enumerate(axes)]
                    + [torch.zeros(n, (D - sum(axes)) // 2, device=x.device, dtype=torch.float64)], 1)[:, None]
    a, b = y[..., 0::2], y[..., 1::2]
    return torch.stack([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).flatten(-2)


def frame_inputs(g, cfg, extra=0, far=128):
    t, n, h = TDT[cfg.dtype], cfg.n_tokens, cfg.n_heads
    f = {}
    for name in "qkv":
        store = randn(g, n, h * D + extra).to(t)
        f[name] = store[:, :h * D]
    f["pos"] = torch.randint(0, far, (n, len(cfg.rope_axes)), generator=g, device="cuda", dtype=torch.int32)
    f["norm_q"], f["norm_k"] = 1 + 0.1 * randn(g, D), 1 + 0.1 * randn(g, D)
    return f


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n, m, heads, axes", [(1, 1, 1, (16, 56, 56)), (70, 1, 5, (16, 56, 56)), (333, 201, 3, (32, 32, 32, 32)),
                                               (1536, 774, 24, (16, 56, 56)), (90, 90, 2, ())])
def test_gather_writes_quantised_rows(cuda, dtype, fmt, n, m, heads, axes):
    t = TDT[dtype]
    g = rng_of(7 * n + m)
    cfg = cfg_of(n, heads, dtype, rope_axes=axes, ld_qkv=heads * D + 8)
    f = frame_inputs(g, cfg, 8, 128 if n != 333 else 2 ** 24)
    rows = torch.randperm(n, generator=g, device="cuda")[:m].sort().values
    idx, count = rows.int(), torch.tensor([m], dtype=torch.int32, device="cuda")
    mask = torch.zeros(n, dtype=torch.int32, device="cuda")
    mask[rows] = torch.where(torch.rand(m, generator=g, device="cuda") < 0.3, 1, 2).int()
    cache = filled_cache(g, cfg, n, fmt)
    before = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
    qc = torch.full((n, heads * D + 8), 3.0, dtype=t, device="cuda")
    save = torch.zeros(n, fxr.q8_save_row_bytes(cfg), dtype=torch.uint8, device="cuda")
    fxr.gather_norm_rope_q8(cfg, f["q"], f["k"], f["v"], mask, idx, count, f["pos"], f["norm_q"], f["norm_k"], qc, cache, save)
    sync_ok()
    x = rope_exact(f["q"][rows].double().view(m, heads, D), f["norm_q"], f["pos"][rows], axes, cfg.rope_theta, cfg.eps)
    got = qc[:m, :heads * D].double().view(m, heads, D)
    assert ((got - x).abs() <= torch.finfo(t).eps / 2 * x.abs() * (1 + 2 ** -10) + 4e-6).all()
    assert (qc[m:] == 3).all() and (qc[:, heads * D:] == 3).all()
    # V: the definition, bit for bit
    y, s = quantise(f["v"][rows].double().view(m, heads, D), fmt, t)
    assert torch.equal(cache.v_scale[:, rows].t().double(), s)
    assert torch.equal(cache.v.view(torch.int8)[rows].view(cache.v.dtype).float().double().view(m, heads, D), y)
    # K': from its 32-bit value
    x = rope_exact(f["k"][rows].double().view(m, heads, D), f["norm_k"], f["pos"][rows], axes, cfg.rope_theta, cfg.eps)
    sk = cache.k_scale[:, rows].t().double()[..., None]
    assert ((sk / up_to(x.abs().amax(-1) / TOP[fmt], t)[..., None] - 1).abs() <= torch.finfo(t).eps * 1.01).all()   # one step of T at a border
    got = values(cache, n)[0][rows]
    half = sk / 2 if fmt == "int8" else torch.maximum((x / sk).abs() * 2.0 ** -4, torch.full_like(x, 2.0 ** -10)) * sk
    assert ((got - x).abs() <= half * (1 + 2 ** -10) + 4e-6).all()
    # rows that are not listed
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert torch.equal(cache.k.view(torch.int8)[rest], before[0][rest]) and torch.equal(cache.v.view(torch.int8)[rest], before[1][rest])
    assert torch.equal(cache.k_scale[:, :n][:, rest], before[2][:, :n][:, rest])
    # mask 1 rows come back whole
    fxr.restore_rows_q8(cfg, mask, idx, count, save, cache)
    sync_ok()
    kept = mask == 1
    for a, b in zip((cache.k.view(torch.int8), cache.v.view(torch.int8)), before[:2]):
        assert torch.equal(a[kept], b[kept])
    for a, b in zip((cache.k_scale, cache.v_scale), before[2:]):
        assert torch.equal(a[:, :n][:, kept], b[:, :n][:, kept])
    assert torch.equal(cache.v_scale[:, rows][:, mask[rows] == 2].t().double(), s[mask[rows] == 2])


@pytest.mark.gpu
def test_row_indices_outside_are_skipped_and_reported(cuda):
    cfg = cfg_of(40, 2, "bf16")
    g = rng_of(3)
    f = frame_inputs(g, cfg)
    t = torch.bfloat16
    idx = torch.tensor([3, -1, 40, 5, 2 ** 30], dtype=torch.int32, device="cuda")
    count = torch.tensor([5], dtype=torch.int32, device="cuda")
    mask = torch.full((40,), 2, dtype=torch.int32, device="cuda")
    cache = fxr.CacheQ8.empty(cfg, fmt="int8")
    qc = torch.zeros(40, 256, dtype=t, device="cuda")
    fxr.gather_norm_rope_q8(cfg, f["q"], f["k"], f["v"], mask, idx, count, f["pos"], f["norm_q"], f["norm_k"], qc, cache)
    with pytest.raises(fxr.FxrError) as e:
        fxr.check_device_error()
    assert e.value.status == fxr.FXR_ERR_BOUNDS
    assert sorted(torch.nonzero(cache.v.abs().sum(1)).flatten().tolist()) == [3, 5]
    k, v = (torch.full((5, 256), 9.0, dtype=t, device="cuda") for _ in range(2))
    fxr.cache_read_q8(cfg, cache, k, v, idx=idx, count=count)
    with pytest.raises(fxr.FxrError):
        fxr.check_device_error()
    assert [bool((v[i] == 9).all()) for i in range(5)] == [False, True, True, False, True]
    st = stream_of(g, cfg, 5, idx=idx)
    st["cache"] = cache
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st]))
    with pytest.raises(fxr.FxrError):
        fxr.check_device_error()
    assert sorted(torch.nonzero((st["out"] != 7).any(1)).flatten().tolist()) == [3, 5]
    sync_ok()


# ---- attention ------------------------------------------------------------------------------------
SMALL = [  # n, m, heads, prefix
    (1, 1, 1, 0), (2, 1, 3, 1), (31, 5, 2, 0), (33, 16, 1, 5), (127, 17, 2, 128), (128, 1, 5, 131), (129, 33, 1, 0),
    (300, 300, 2, 77), (1000, 3, 24, 0), (1537, 64, 3, 700), (700, 257, 2, 129)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n, m, heads, prefix", SMALL)
def test_attention_of_one_stream(cuda, dtype, fmt, n, m, heads, prefix):
    g = rng_of(n * 31 + m)
    cfg = cfg_of(n, heads, dtype, ld_out=heads * D + 16)
    st = stream_of(g, cfg, m, ld_extra=8, out_extra=16)
    st["cache"] = filled_cache(g, cfg, n + 2, fmt, pad=32, extra_scale=8)
    pre = filled_cache(g, cfg, prefix, fmt, pad=16) if prefix else None
    ws = workspace_for(cfg, [st], pre)
    for bound in (0, m):
        st["out"].fill_(7.0)
        fxr.attention_q8(cfg, [st], ws, prefix=pre, max_rows=bound)
        sync_ok()
        check_streams(cfg, [st], pre, what=f"bound {bound}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("counts, n, heads, prefix", [((3, 0, 20, 1), 100, 2, 130), ((0, 0), 64, 1, 10), ((5,) * 9, 61, 1, 33),
                                                      ((16,) * 8, 700, 3, 900), ((300, 17, 500), 600, 1, 300), ((1, 2), 150, 4, 0)])
def test_attention_of_streams_with_a_shared_prefix(cuda, dtype, fmt, counts, n, heads, prefix):
    g = rng_of(sum(counts) + n)
    cfg = cfg_of(n, heads, dtype)
    streams = []
    for m in counts:
        st = stream_of(g, cfg, m)
        st["cache"] = filled_cache(g, cfg, n, fmt)
        streams.append(st)
    pre = filled_cache(g, cfg, prefix, fmt) if prefix else None
    fxr.attention_q8(cfg, streams, workspace_for(cfg, streams, pre, max(counts)), prefix=pre, max_rows=max(counts))
    sync_ok()
    check_streams(cfg, streams, pre)


def random_groups(g, n, bits=3, empty=0.2):
    """Sets of up to `bits` groups (bit 31 among them), some empty."""
    w = torch.zeros(n, dtype=torch.int64, device="cuda")
    for b in range(bits):
        w |= (torch.rand(n, generator=g, device="cuda") < 0.4).long() << (31 if b == 0 else b)
    w[torch.rand(n, generator=g, device="cuda") < empty] = 0
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).int()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "e4m3"), ("f16", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("kind", ["random", "documents", "nothing", "prefix only", "one key", "late"])
@pytest.mark.parametrize("counts, n, heads, prefix", [((40, 7), 203, 2, 150), ((290,), 415, 1, 0), ((16, 1), 130, 3, 257), ((380, 256), 390, 2, 200)])
def test_attention_with_groups(cuda, dtype, fmt, kind, counts, n, heads, prefix):
    """Document masks, rows that see nothing, keys that nobody sees (NaN there changes nothing)."""
    g = rng_of(sum(counts) * 3 + len(kind))
    cfg = cfg_of(n, heads, dtype)
    pre = filled_cache(g, cfg, prefix, fmt) if prefix else None
    pg = None
    streams = []
    for m in counts:
        st = stream_of(g, cfg, m)
        st["cache"] = filled_cache(g, cfg, n, fmt)
        at = torch.arange(n, device="cuda")
        if kind == "random":
            st["q_groups"], st["k_groups"] = random_groups(g, n), random_groups(g, n)
        elif kind == "documents":
            st["q_groups"] = st["k_groups"] = torch.bitwise_left_shift(torch.ones_like(at), at * 5 // n).int()
        elif kind == "nothing":
            st["k_groups"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        elif kind == "prefix only":
            st["q_groups"] = torch.full((n,), 2, dtype=torch.int32, device="cuda")
            st["k_groups"] = torch.full((n,), 1, dtype=torch.int32, device="cuda")
        elif kind == "one key":
            st["k_groups"] = (at == n - 1).int()
        else:                                     # every row's first visible key comes late
            st["k_groups"] = (at >= n - 3).int() * 4
        if st.get("k_groups") is not None:        # what nobody sees may hold anything
            hidden = st["k_groups"] == 0
            for scale in (st["cache"].k_scale, st["cache"].v_scale):
                scale[:, :n][:, hidden] = math.nan
            st["cache"].v_scale[0, :n][hidden] = math.inf
        streams.append(st)
    if pre is not None:
        pg = random_groups(g, prefix) if kind in ("random", "documents") else \
            torch.full((prefix,), 2 if kind == "prefix only" else 0, dtype=torch.int32, device="cuda")
        pre.k_scale[:, :prefix][:, pg == 0] = math.nan
        pre.v_scale[:, :prefix][:, pg == 0] = math.nan
    ws = workspace_for(cfg, streams, pre, max(counts))
    fxr.attention_q8(cfg, streams, ws, prefix=pre, prefix_groups=pg, max_rows=max(counts))
    sync_ok()
    check_streams(cfg, streams, pre, pg, kind)
    if kind == "nothing":
        for st in streams:
            assert (st["out"][st["idx"][:st["m"]].long()] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m", [3, 270])
def test_nan_rows_poison_those_that_see_them(cuda, dtype, m):
    """A key whose K or V is NaN makes the rows of its group NaN in that head, and no others."""
    n, heads = 300, 2
    g = rng_of(m)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, "int8")
    st["cache"].v_scale[1, 140] = math.nan
    st["cache"].k_scale[0, 7] = math.inf
    at = torch.arange(n, device="cuda")
    st["q_groups"] = st["k_groups"] = torch.where(at % 2 == 0, 1, 2).int()
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
    sync_ok()
    check_streams(cfg, [st])
    rows = st["idx"][:m].long()
    out = st["out"][rows].view(m, heads, D)
    assert torch.equal(torch.isnan(out).all(-1), torch.stack([rows % 2 == 1, rows % 2 == 0], 1))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_large_scores(cuda, m, spread):
    """Scores in the hundreds: the running maximum moves often and most keys vanish. bf16."""
    n, heads = 700, 2
    g = rng_of(int(spread) + m)
    cfg = cfg_of(n, heads, "bf16", softmax_scale=spread / math.sqrt(D))
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, "e4m3")
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
    sync_ok()
    check_streams(cfg, [st])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 200])
def test_small_values_keep_their_precision(cuda, m):
    """f16 V of magnitude 1e-3 to 1e-5: P times a small scale would be a subnormal."""
    n, heads = 500, 2
    g = rng_of(m)
    cfg = cfg_of(n, heads, "f16")
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, "int8")
    st["cache"].v_scale[:, :n] = (st["cache"].v_scale[:, :n].float() * 2.0 ** -8).half()
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
    sync_ok()
    rows = st["idx"][:m].long()
    o, mean_abs, var, ds = expected(cfg, st)
    # an f16 below 2^-14 has steps of 2^-24: V and the output are rounded there by half of one each
    err = (st["out"][rows].double().view(o.shape) - o).abs()
    u = 2.0 ** -11
    assert (err <= u * o.abs() + (2 * u + 2 ** -13 + 2 * u * ds) * mean_abs + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("bf16", "e4m3"), ("f16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("m", [5, 30, 290])
@pytest.mark.parametrize("kind", ["spread", "unseen giants", "giants that nobody looks at", "zeros", "large"])
def test_scales_far_apart(cuda, dtype, fmt, m, kind):
    """V scales that differ by many powers of two: none may cost another key its precision. "large": e4m3 scales of 128
    and more (bf16), which the kernels decode in two steps."""
    n, heads = 333, 2
    g = rng_of(m + len(kind))
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, fmt)
    v, k, t = c.v_scale, c.k_scale, TDT[dtype]
    top = 2.0 ** 6 if dtype == "f16" else 2.0 ** 60
    if kind == "spread":       # over 2^24 (bf16), 2^12 (f16: the smallest scales stay normal numbers)
        wide = 24 if dtype == "bf16" else 6
        v[:, :n] = (v[:, :n].float() * torch.exp2(torch.randint(-wide // 2, wide // 2 + 1, (heads, n), generator=g, device="cuda").float())).to(t)
    elif kind == "unseen giants":
        st["k_groups"] = (torch.arange(n, device="cuda") % 3 != 0).int()
        v[:, 0:n:3] = top
    elif kind == "giants that nobody looks at":
        # keys of large norm opposite to every query: weights of 2^-200 and less
        q = st["qc"][:m].double().view(m, heads, D)
        q[:] = q[:1]
        st["qc"][:m] = q.view(m, heads * D).to(t)
        for key in (40, 200):
            y, s = quantise(-12 * st["qc"][0].double().view(heads, D), fmt, t)
            c.k.view(torch.int8)[key, :heads * D] = (y.to(torch.int8) if fmt == "int8" else y.float().to(c.k.dtype).view(torch.int8)).view(-1)
            k[:, key] = s.to(t)
            v[:, key] = top
    elif kind == "zeros":
        v[0, :n] = 0
        v[1, :n:2] = 0
    else:
        big = 130.0 if dtype == "f16" else 3000.0 if fmt == "e4m3" else 3e30
        v[:, 5:n:7] = big
        if dtype == "bf16":
            k[:, 3] = 1000.0
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
    sync_ok()
    if kind == "giants that nobody looks at":
        # in 64 bits their weight is below 2^-150 of the others': compared without them
        seen = torch.ones(n, dtype=torch.int32, device="cuda")
        seen[40] = seen[200] = 0
        ref = expected(cfg, dict(st, k_groups=seen))
        check_attention(st["out"][st["idx"][:m].long()], ref, t, kind)
    else:
        check_streams(cfg, [st], what=kind)


@pytest.mark.gpu
def test_one_workspace_for_calls_of_other_shapes(cuda):
    """Calls of few, more and many rows, with few heads and many, one after the other in one workspace."""
    g = rng_of(11)
    calls = []
    for n, heads, m, dtype, fmt in ((600, 2, 300, "bf16", "int8"), (900, 24, 5, "f16", "e4m3"), (2049, 48, 1900, "f16", "int8"),
                                    (700, 32, 17, "bf16", "e4m3"), (400, 1, 9, "bf16", "int8")):
        cfg = cfg_of(n, heads, dtype)
        st = stream_of(g, cfg, m)
        st["cache"] = filled_cache(g, cfg, n, fmt)
        calls.append((cfg, st, m))
    ws = torch.zeros(max(fxr.attention_q8_workspace_size(cfg, 1, 0, m) for cfg, _, m in calls), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for cfg, st, m in calls:
            st["out"].fill_(7.0)
            fxr.attention_q8(cfg, [st], ws, max_rows=m)
            sync_ok()
            check_streams(cfg, [st])


# calls of many rows without groups and prefix, which read the cache through its 16-bit rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("bf16", "e4m3"), ("f16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("counts, n, heads, bound", [((2049,), 4700, 18, 2049), ((2100, 0, 1900), 2501, 16, 2100), ((300,), 8003, 12, 0),
                                                     ((4224,), 4224, 24, 4224), ((2600,), 7003, 8, 2600)])
def test_attention_of_many_rows(cuda, dtype, fmt, counts, n, heads, bound):
    """Against 64 bits; the same buffers used again, larger rows between; rows behind the counts stay."""
    g = rng_of(sum(counts) + n)
    cfg = cfg_of(n, heads, dtype, ld_out=heads * D + 8)
    streams = []
    for m in counts:
        st = stream_of(g, cfg, m, ld_extra=8, out_extra=8)
        st["cache"] = filled_cache(g, cfg, n + 1, fmt, pad=16, extra_scale=8)
        streams.append(st)
    ws = workspace_for(cfg, streams, max_rows=bound)
    for _ in range(2):
        for st in streams:
            st["out"].fill_(7.0)
        fxr.attention_q8(cfg, streams, ws, max_rows=bound)
    sync_ok()
    check_streams(cfg, streams)
    # captured, and replayed with other counts
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fxr.attention_q8(cfg, streams, ws, max_rows=bound)
    for st in streams:
        st["m"] = st["m"] * 2 // 3
        st["count"].fill_(st["m"])
        st["out"].fill_(7.0)
    graph.replay()
    sync_ok()
    check_streams(cfg, streams)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "e4m3"), ("f16", "int8")])
def test_many_rows_with_nan_and_beyond_the_bound(cuda, dtype, fmt):
    """A key without a valid scale makes its head NaN; a count above the bound is an error, and its rows are left."""
    n, heads, m, bound = 2400, 32, 1950, 1900
    g = rng_of(5)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, fmt)
    st["cache"].k_scale[3, 3] = math.nan          # a pair of columns whose exponential is the polynomial's
    st["cache"].v_scale[5, n - 1] = math.inf
    before = st["out"].clone()
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=bound), max_rows=bound)
    with pytest.raises(fxr.FxrError) as e:
        fxr.check_device_error()
    assert e.value.status == fxr.FXR_ERR_BOUNDS
    rows = st["idx"][:m].long()
    assert torch.equal(st["out"][rows[bound:]], before[rows[bound:]])
    out = st["out"][rows[:bound]].view(bound, heads, D)
    bad = torch.zeros(heads, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.equal(torch.isnan(out).all(-1), bad.expand(bound, heads)) and torch.isnan(out).any(-1).sum() == 2 * bound
    # a call with groups in the same workspace, which the other kernel takes, and the first again
    st["cache"] = filled_cache(g, cfg, n, fmt)
    st["m"] = bound
    st["count"].fill_(bound)
    ws = workspace_for(cfg, [st], max_rows=bound)
    for groups in (None, torch.ones(n, dtype=torch.int32, device="cuda"), None):
        st["q_groups"] = st["k_groups"] = groups
        st["out"].fill_(7.0)
        fxr.attention_q8(cfg, [st], ws, max_rows=bound)
        sync_ok()
        check_streams(cfg, [st])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [6, 280])
def test_groups_of_queries_alone_and_queries_that_are_nan(cuda, m):
    """q_groups without k_groups: every key is seen but by empty sets. A NaN query spoils its own row only."""
    n, heads = 310, 2
    g = rng_of(m)
    cfg = cfg_of(n, heads, "bf16")
    pre = filled_cache(g, cfg, 70, "int8")
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, "int8")
    st["q_groups"] = torch.where(torch.arange(n, device="cuda") % 3 == 0, 0, 8).int()
    rows = st["idx"][:m].long()
    st["qc"][1, 5] = math.nan
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], pre, m), prefix=pre, max_rows=m)
    sync_ok()
    out = st["out"][rows].view(m, heads, D)
    blind = rows % 3 == 0
    assert (out[blind] == 0).all()
    if not blind[1]:
        assert torch.isnan(out[1, 0]).all()
    keep = torch.ones(m, dtype=torch.bool, device="cuda")
    keep[1] = False
    ref = expected(cfg, dict(st, qc=torch.nan_to_num(st["qc"])), pre)
    check_attention(out[keep], [x[keep] for x in ref], torch.bfloat16)


@pytest.mark.gpu
def test_a_captured_frame_replays(cuda):
    """frame_forward_q8 in a graph, replayed on new inputs in the same tensors, equals eager calls bit for bit."""
    n, heads = 500, 2
    g = rng_of(9)
    cfg = cfg_of(n, heads, "bf16")
    f = frame_inputs(g, cfg)
    mask = torch.where(torch.rand(n, generator=g, device="cuda") < 0.4, 2, 0).int()
    mask[:30] = 1
    caches = [filled_cache(rng_of(4), cfg, n, "e4m3") for _ in range(2)]
    outs = [torch.zeros(n, heads * D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ws = [torch.empty(fxr.frame_q8_workspace_size(cfg), dtype=torch.uint8, device="cuda") for _ in range(2)]
    call = lambda e: fxr.frame_forward_q8(cfg, f["q"], f["k"], f["v"], mask, None, f["pos"], f["norm_q"], f["norm_k"],  # noqa: E731
                                          caches[e], outs[e], ws[e])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    for seed in range(3):
        new = frame_inputs(rng_of(seed + 50), cfg)
        for name in "qkv":
            f[name].copy_(new[name])
        mask.copy_(torch.where(torch.rand(n, generator=g, device="cuda") < 0.1 * seed, 2, 1 if seed == 1 else 0).int())
        graph.replay()
        call(1)
        sync_ok()
        assert torch.equal(outs[0], outs[1])
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
            assert torch.equal(a.view(torch.int8), b.view(torch.int8))


@pytest.mark.gpu
def test_cpu_tensors_are_refused(cuda):
    cfg = cfg_of(16, 1, "bf16")
    cache = fxr.CacheQ8.empty(cfg)
    k = torch.zeros(16, D, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(fxr.FxrError, match="cpu"):
        fxr.cache_read_q8(cfg, cache, k, k.cpu())
    with pytest.raises(fxr.FxrError, match="cpu"):
        fxr.cache_write_q8(cfg, k.cpu(), k, cache)
    st = stream_of(rng_of(1), cfg, 2)
    st["cache"] = cache
    with pytest.raises(fxr.FxrError, match="cpu"):
        fxr.attention_q8(cfg, [st], workspace_for(cfg, [st]).cpu())
    with pytest.raises(fxr.FxrError, match="one CUDA device"):
        fxr.q8_streams([dict(st, idx=st["idx"].cpu())])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 300])
def test_rows_past_the_bound_are_reported(cuda, m):
    n = 400
    g = rng_of(m)
    cfg = cfg_of(n, 2, "bf16")
    st = stream_of(g, cfg, m + 5)
    st["cache"] = filled_cache(g, cfg, n, "int8")
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
    with pytest.raises(fxr.FxrError) as e:
        fxr.check_device_error()
    assert e.value.status == fxr.FXR_ERR_BOUNDS
    st["idx"], st["m"] = st["idx"][:m].contiguous(), m
    check_streams(cfg, [st])
    sync_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("m, prefix", [(4, 0), (16, 300), (400, 200)])
def test_calls_repeat_bit_for_bit_captured_and_on_other_streams(cuda, m, prefix):
    """Eager, captured and replayed (new inputs between), on a side stream, with a workspace reused by other shapes."""
    n, heads = 900, 3
    g = rng_of(m)
    cfg = cfg_of(n, heads, "bf16")
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, "e4m3")
    pre = filled_cache(g, cfg, prefix, "e4m3") if prefix else None
    ws = workspace_for(cfg, [st], pre)
    streams = fxr.q8_streams([st])
    call = lambda: fxr.attention_q8(cfg, streams, ws, prefix=pre, max_rows=m)  # noqa: E731
    call()
    sync_ok()
    first = st["out"].clone()
    for _ in range(5):
        st["out"].fill_(7.0)
        call()
    sync_ok()
    assert torch.equal(st["out"], first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        call()
    st["out"].fill_(7.0)
    graph.replay()
    sync_ok()
    assert torch.equal(st["out"], first)
    keep = st["qc"].clone()
    st["qc"].mul_(-1)
    st["count"].fill_(m - 1)
    st["out"].fill_(7.0)
    graph.replay()
    sync_ok()
    st["m"] = m - 1
    check_streams(cfg, [st], pre)
    st["qc"].copy_(keep)
    st["count"].fill_(m)
    st["m"] = m
    # two streams at once, a workspace each
    side = torch.cuda.Stream()
    other = dict(st, out=torch.full_like(st["out"], 7.0))
    ws2 = workspace_for(cfg, [st], pre)
    torch.cuda.synchronize()
    for _ in range(10):
        call()
        fxr.attention_q8(cfg, [other], ws2, prefix=pre, max_rows=m, stream=side)
    sync_ok()
    assert torch.equal(st["out"], first) and torch.equal(other["out"], first)


@pytest.mark.gpu
def test_caches_past_32_bit_offsets(cuda):
    """Rows whose byte offset passes 2^31 (one head of wide rows): written, read back, attended."""
    n, ld = 70000, 32768
    cfg = cfg_of(n, 1, "bf16")
    g = rng_of(1)
    codes = [torch.zeros(n, ld, dtype=torch.int8, device="cuda")[:, :D] for _ in range(2)]
    sc = [torch.zeros(1, n, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache = fxr.CacheQ8(codes[0], codes[1], sc[0], sc[1])
    x = [randn(g, n, D).bfloat16() for _ in range(2)]
    fxr.cache_write_q8(cfg, x[0], x[1], cache)
    y, s = quantise(x[1].double().view(n, 1, D), "int8", torch.bfloat16)
    sync_ok()
    assert torch.equal(cache.v_scale.t().double(), s) and torch.equal(cache.v.double(), y[:, 0])
    k, v = (torch.zeros(n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    fxr.cache_read_q8(cfg, cache, k, v)
    for m in (1, 130):
        st = stream_of(g, cfg, m)
        st["cache"] = cache
        fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], max_rows=m), max_rows=m)
        sync_ok()
        check_streams(cfg, [st])
    assert torch.equal(v, values(cache)[1].view(n, D).bfloat16())


@pytest.mark.gpu
def test_tensors_of_another_device_are_refused(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    cfg = cfg_of(16, 1, "bf16")
    cache = fxr.CacheQ8.empty(cfg, device="cuda:1")
    with pytest.raises(fxr.FxrError):
        fxr.cache_read_q8(cfg, cache, None, None)


# ---- the run of all of them -----------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("n, heads, p, prefix, bound", [(200, 2, 0.04, 0, 24), (700, 3, 0.5, 150, 0), (1536, 24, 0.25, 0, 0)])
def test_frames_over_an_8_bit_cache(cuda, dtype, fmt, n, heads, p, prefix, bound):
    """Three frames of one stream: rows executed, kept (mask 1) and skipped, a shared prefix. Each frame's output
    against the definition over the rows that its attention saw; its cache against what had to be kept."""
    t = TDT[dtype]
    g = rng_of(n)
    cfg = cfg_of(n, heads, dtype)
    cache = fxr.CacheQ8.empty(cfg, fmt=fmt)
    pre = filled_cache(g, cfg, prefix, fmt) if prefix else None
    valid = torch.zeros(n, dtype=torch.uint8, device="cuda")
    out = torch.full((n, heads * D), 7.0, dtype=t, device="cuda")
    ws = torch.empty(max(fxr.frame_q8_workspace_size(cfg, prefix, b) for b in (0, bound)), dtype=torch.uint8, device="cuda")
    ws.fill_(171)                                  # of any content
    for frame in range(3):
        f = frame_inputs(g, cfg)
        r = torch.rand(n, generator=g, device="cuda")
        mask = torch.where(r < p * 0.3, 1, torch.where(r < p, 2, 0)).int()
        old = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
        old_out = out.clone()
        given = mask.clone()
        rows_bound = 0 if frame == 0 else bound    # the first frame runs every token
        if rows_bound:
            mask[torch.nonzero(mask).flatten()[rows_bound:]] = 0
            given = mask.clone()
        fxr.frame_forward_q8(cfg, f["q"], f["k"], f["v"], mask, valid, f["pos"], f["norm_q"], f["norm_k"], cache, out, ws,
                             prefix=pre, max_rows=rows_bound)
        sync_ok()
        want_mask = torch.where(valid == 0, torch.full_like(given, 2), given)
        assert torch.equal(mask, want_mask)
        rows = torch.nonzero(mask).flatten()
        kept = mask == 1
        # the cache that the attention saw: the same write without the restore
        seen = fxr.CacheQ8(old[0].view(cache.k.dtype), old[1].view(cache.k.dtype), old[2], old[3])
        saved = [x.clone() for x in old]
        qc = torch.zeros(n, heads * D, dtype=t, device="cuda")
        save = torch.zeros(n, fxr.q8_save_row_bytes(cfg), dtype=torch.uint8, device="cuda")
        idx, count = rows.int(), torch.tensor([len(rows)], dtype=torch.int32, device="cuda")
        fxr.gather_norm_rope_q8(cfg, f["q"], f["k"], f["v"], mask, idx, count, f["pos"], f["norm_q"], f["norm_k"], qc, seen, save)
        sync_ok()
        st = {"qc": qc, "idx": idx, "m": len(rows), "cache": seen}
        check_attention(out[rows], expected(cfg, st, pre), t, f"frame {frame}")
        assert torch.equal(out[mask == 0], old_out[mask == 0])
        for now, was, new in zip((cache.k.view(torch.int8), cache.v.view(torch.int8)), saved[:2], (seen.k.view(torch.int8), seen.v.view(torch.int8))):
            assert torch.equal(now[kept], was[kept]) and torch.equal(now[~kept], new[~kept])
        for now, was, new in zip((cache.k_scale, cache.v_scale), saved[2:], (seen.k_scale, seen.v_scale)):
            assert torch.equal(now[:, :n][:, kept], was[:, :n][:, kept]) and torch.equal(now[:, :n][:, ~kept], new[:, :n][:, ~kept])
        fxr.mark_updated(mask, valid, 0)
        torch.cuda.synchronize()
