"""The 8-bit spatial cache at the edges of what its tensors may hold: e4m3 codes that other uses call NaN, scales next to
the largest, scores in the hundreds, NaN that comes late. Attention is held against K as the kernel holds it, so that its
rounding to T (many rows) drops out of the bars, which then are tight; derived before the first run, u = finfo(T).eps / 2:
  a score's 128 products are summed in 32 bits, at worst with 128 truncations of 2^-23 of a partial sum that is at most
  sum|q k|, and a few roundings of 2^-24 of the score follow: ds = (2^-16 + 2^-21) * scale * max_j sum|q k_j|, also where
  bf16 queries are held in f16 (elements below 2^-24 of the largest round to a step of 2^-35 of it, 128 of them: 2^-28);
  P and V are rounded to T (u each at most), exponentials to 2^-13, the output once:
      |err| <= u |o| + (2 u + 2^-13 + expm1(2 ds)) sum(w |v|) + small
  small: P in f16 is a subnormal below 2^-14, off by up to 2^-25. The largest P of a row is at least 1 (its running maximum
  is never above the largest score), so that is 2^-25 of the largest weight for each key: 2^-25 max(w) sum|v|. The kernel
  for few rows holds P times the V scale in f16 for every T, whose largest is at least 1: 2^-25 max(w scale) sum|code|.
"""
import copy
import dataclasses
import math
import pickle

import pytest
import torch

import fxr
from test_q8_cache import D, TDT, cfg_of, filled_cache, frame_inputs, rng_of, stream_of, sync_ok, workspace_for

FEW = 32        # rows that the kernel for few rows takes; it holds K and V exactly


def e4m3_values():
    """The 256 codes as numbers; 0x7f and 0xff are +-480."""
    b = torch.arange(256, device="cuda")
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e.double() - 7))
    return torch.where(b >= 128, -x, x)


def held(cache, n, exact):
    """K and V [n, heads, 128] in 64 bits as the attention holds them: codes times scales, exactly or rounded to T and
    finite. Keys without a valid scale: K NaN. And V's scales [n, heads, 1]."""
    h, t = cache.n_heads, cache.k_scale.dtype
    out, bad = [], None
    for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes = c[:n, :h * D].contiguous().view(torch.int8)
        x = codes.double() if c.dtype == torch.int8 else e4m3_values()[codes.view(torch.uint8).long()]
        s = s[:h, :n].t().double()
        cap = 1.9921875 * 2.0 ** 120 if t == torch.bfloat16 else 511.75
        if c.dtype != torch.int8:
            cap = 1.1328125 * 2.0 ** 119 if t == torch.bfloat16 else 146.125
        invalid = ~(s.abs() <= cap)
        bad = invalid if bad is None else bad | invalid
        x = x.view(n, h, D) * torch.where(invalid, torch.zeros_like(s), s)[..., None]
        out.append(x if exact else x.to(t).double().clamp(-torch.finfo(t).max, torch.finfo(t).max))
    out[0] = torch.where(bad[..., None], torch.full_like(out[0], math.nan), out[0])
    return out[0], out[1], torch.where(invalid, torch.zeros_like(s), s)[..., None]


def check(cfg, st, max_rows, prefix=None, prefix_groups=None, what="", rows=None, telling=0.7):
    """The stream's output against the definition (of the compact rows `rows`). telling: the share of elements whose bar
    is below their value, so that an output of zeros would fail."""
    n, m, h, t = cfg.n_tokens, st["m"], cfg.n_heads, TDT[cfg.dtype]
    u = torch.finfo(t).eps / 2
    exact = 0 < max_rows <= FEW
    k, v, vs = held(st["cache"], n, exact)
    ones = lambda r: torch.full((r,), -1, dtype=torch.int32, device="cuda")  # noqa: E731
    kg = st.get("k_groups") if st.get("k_groups") is not None else ones(n)
    if prefix is not None:
        k, v, vs = (torch.cat(x) for x in zip(held(prefix, prefix.n_rows, exact), (k, v, vs)))
        kg = torch.cat([prefix_groups if prefix_groups is not None else ones(prefix.n_rows), kg])
    at = st["idx"][:m].long()
    qg = st["q_groups"][at] if st.get("q_groups") is not None else ones(m)
    seen = (qg[:, None] & kg[None]) != 0
    scale = cfg.softmax_scale if cfg.softmax_scale > 0 else 1 / math.sqrt(D)
    q = st["qc"][:m].double().view(m, h, D).transpose(0, 1)
    k, v, vs = (x.transpose(0, 1) for x in (k, v, vs))
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen[None], -math.inf)
    nan = torch.isnan(s).any(-1)
    s = torch.nan_to_num(s, nan=-math.inf, neginf=-math.inf)
    w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)              # rows that see nothing: zeros
    o, mean_abs = w @ v, w @ v.abs()
    ds = (q.abs() @ torch.nan_to_num(k).abs().transpose(1, 2) * scale).masked_fill(~seen[None], 0).amax(-1, keepdim=True)
    bar = u * o.abs() + (2 * u + 2 ** -13 + torch.expm1(2 * (2 ** -16 + 2 ** -21) * ds)) * mean_abs
    bar = bar + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    some = seen.double()[None]
    if exact:
        vs = vs.abs()
        bar = bar + 2.0 ** -25 * (w * vs.transpose(1, 2)).amax(-1, keepdim=True) * (some @ torch.where(vs > 0, v.abs() / vs, vs))
    elif t == torch.float16:
        bar = bar + 2.0 ** -25 * w.amax(-1, keepdim=True) * (some @ v.abs())
    got = st["out"][at].double().view(m, h, D).transpose(0, 1)
    if rows is not None:
        got, o, bar, nan = got[:, rows], o[:, rows], bar[:, rows], nan[:, rows]
    assert torch.equal(torch.isnan(got), nan[..., None].expand_as(got)), what + ": NaN in other places"
    err = torch.where(nan[..., None], torch.zeros_like(o), (got - o).abs())
    assert (err <= bar).all(), f"{what}: {float((err / bar).max()):.2f} of the bar"
    told = (bar < o.abs()) | nan[..., None] | (o == 0)
    assert float(told.double().mean()) >= telling, f"{what}: the bar tells {float(told.double().mean()):.2f}"
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert (st["out"][rest] == 7.0).all(), what + ": rows that are not listed changed"


def attend(cfg, st, max_rows, prefix=None, prefix_groups=None):
    fxr.attention_q8(cfg, [st], workspace_for(cfg, [st], prefix, max_rows), prefix=prefix, prefix_groups=prefix_groups,
                     max_rows=max_rows)
    sync_ok()


def fill_codes(cache, rows, *codes):
    """The rows' K and V codes: `codes` in turn along the columns."""
    for c in (cache.k, cache.v):
        c = c.view(torch.uint8)
        c[rows] = torch.tensor(codes, dtype=torch.uint8, device="cuda").repeat(c.shape[1] // len(codes))


# ---- e4m3 codes that other uses call NaN -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m", [3, 12, 30, 300])
@pytest.mark.parametrize("scales", ["valid", "invalid"])
@pytest.mark.parametrize("prefix", [0, 200])
def test_rows_that_nobody_sees_hold_any_code(cuda, dtype, m, scales, prefix):
    """Padding rows of codes 0x7f and 0xff, in the prefix and among the own, and a key of such codes that every other row
    sees: the others must not notice, and those count them as +-480."""
    n, heads = 333, 2
    g = rng_of(m)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, "e4m3")
    at = torch.arange(n, device="cuda")
    st["q_groups"] = torch.where(at % 2 == 0, 1, 3).int()
    st["k_groups"] = torch.full((n,), 1, dtype=torch.int32, device="cuda")
    st["k_groups"][100:140] = 0
    st["k_groups"][n - 1] = 0
    st["k_groups"][7] = 2
    hidden = st["k_groups"] == 0
    fill_codes(c, hidden, 0x7f, 0xff)
    fill_codes(c, at == 7, 0xff, 0x7f, 0x38, 0x7f)
    c.k_scale[:, 7] = 2.0 ** -9        # K of about 1
    pre = pg = None
    if prefix:
        pre = filled_cache(g, cfg, prefix, "e4m3")
        pg = torch.full((prefix,), 1, dtype=torch.int32, device="cuda")
        pg[prefix - 37:] = 0
        fill_codes(pre, pg == 0, 0xff, 0x7f)
    if scales == "invalid":
        for s in (c.k_scale, c.v_scale):
            s[:, :n][:, hidden] = math.nan
        if prefix:
            pre.v_scale[:, :prefix][:, pg == 0] = math.inf
    attend(cfg, st, m, pre, pg)
    check(cfg, st, m, pre, pg)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n, heads, m", [(90, 3, 5), (400, 2, 200), (2400, 32, 1950)])
def test_every_code_counts_as_one_number(cuda, dtype, n, heads, m):
    """Visible codes 0x7f and 0xff are +-480 in the read-back and in the attention of few, many and very many rows."""
    g = rng_of(n)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, "e4m3")
    fill_codes(c, torch.arange(n, device="cuda") % 11 == 3, 0x7f, 0x30, 0xff, 0xb8)
    for s in (c.k_scale, c.v_scale):
        s[:, 3:n:11] = 2.0 ** -9
    attend(cfg, st, m)
    check(cfg, st, m)
    k, v = (torch.zeros(n, heads * D, dtype=TDT[dtype], device="cuda") for _ in range(2))
    fxr.cache_read_q8(cfg, c, k, v)
    sync_ok()
    for got, want in zip((k, v), held(c, n, True)[:2]):
        assert torch.equal(got, want.reshape(n, -1).to(TDT[dtype]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m", [3, 30, 300])
def test_codes_of_480_times_the_largest_scales(cuda, dtype, m):
    """480 times a scale next to the largest valid one passes the largest T: rows that do not see such keys must not
    notice. (f16: those that do see them too.)"""
    n, heads = 333, 2
    g = rng_of(m)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, "e4m3")
    at = torch.arange(n, device="cuda")
    st["q_groups"] = torch.where(at % 2 == 0, 1, 3).int()
    st["k_groups"] = torch.where(at % 50 == 9, 2, 1).int()
    st["k_groups"][200:230] = 0
    odd = st["k_groups"] != 1
    fill_codes(c, odd, 0x7f, 0xff)
    top = 1.1328125 * 2.0 ** 119 if dtype == "bf16" else 146.125
    for s in (c.k_scale, c.v_scale):
        s[:, :n][:, odd] = top
    if dtype == "f16":
        c.k_scale[:, :n][:, st["k_groups"] == 2] = 2.0 ** -9
    attend(cfg, st, m)
    rows = st["idx"][:m].long() % 2 == 0 if dtype == "bf16" else None
    check(cfg, st, m, rows=rows)


@pytest.mark.gpu
def test_codes_of_480_times_the_largest_scale_seen_by_very_many_rows(cuda):
    """The form that expands the cache: such a V stops at the largest f16."""
    n, heads, m = 2400, 32, 1950
    g = rng_of(8)
    cfg = cfg_of(n, heads, "f16")
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, "e4m3")
    fill_codes(c, torch.arange(n, device="cuda") == 77, 0x7f, 0xff)
    c.k_scale[:, 77], c.v_scale[:, 77] = 2.0 ** -9, 146.125
    attend(cfg, st, m)
    check(cfg, st, m)


# ---- NaN ---------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("m", [5, 30, 250])
@pytest.mark.parametrize("tiles, place", [(2, 1), (3, 1), (40, 39), (40, 20), (40, 0)])
def test_a_nan_key_that_is_the_first_that_a_row_sees(cuda, dtype, fmt, m, tiles, place):
    """Rows of one document see a single tile of 128 keys, shared with the others, and in it a key without a valid scale,
    in each of the columns whose exponentials are computed in another way: NaN in its head, whole units and cut ones."""
    n, heads = 128 * tiles, 9
    g = rng_of(m + tiles)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, fmt)
    at = torch.arange(n, device="cuda")
    st["q_groups"] = torch.where(at % 2 == 0, 1, 2).int()
    st["k_groups"] = torch.where(at // 128 == place, 3, 1).int()
    for head in range(8):
        (c.k_scale if head % 3 else c.v_scale)[head, 128 * place + 40 + head] = math.nan if head % 2 else math.inf
    attend(cfg, st, m)
    check(cfg, st, m)
    out = st["out"][st["idx"][:m].long()].view(m, heads, D)
    assert torch.isnan(out[:, :8]).all() and not torch.isnan(out[:, 8]).any()


# ---- refusals (no GPU) and what a call may write ---------------------------------------------------
def cpu_cache(rows, heads=2, fmt=torch.int8, dtype=torch.bfloat16):
    k = torch.zeros(rows, heads * D, dtype=torch.int8).view(fmt)
    s = torch.zeros(heads, max(8, -(-rows // 8) * 8), dtype=dtype)
    return fxr.CacheQ8(k, k.clone(), s, s.clone())


def test_read_back_refuses_outputs_that_do_not_hold_the_rows():
    cfg, cache = cfg_of(16, 2, "bf16"), cpu_cache(19)          # a cache may have more rows than the frame
    out = lambda rows, cols=2 * D, t=torch.bfloat16: torch.zeros(rows, cols, dtype=t)  # noqa: E731
    idx = torch.zeros(5, dtype=torch.int32)
    for k, v, more in ((out(16), out(16), {}), (out(19), out(18), {}), (out(18), out(19), {}), (out(6), out(6), {"host_count": 7}),
                       (out(19, D), out(19, D), {}), (out(19, t=torch.float16), out(19, t=torch.float16), {}),
                       (out(19, t=torch.float32), out(19, t=torch.float32), {}), (out(19, t=torch.int8), out(19, t=torch.int8), {}),
                       (out(2 * D, 19).t(), out(2 * D, 19).t(), {}), (out(19), None, {}), (None, out(19), {}),
                       (out(19).view(19, 4, 64)[:, :, :32], out(19).view(19, 4, 64)[:, :, :32], {}),
                       (out(19).flatten(), out(19).flatten(), {}), (out(9), out(9), {"idx": idx, "host_count": 9})):
        with pytest.raises(fxr.FxrError) as e:
            fxr.cache_read_q8(cfg, cache, k, v, **more)
        assert e.value.status == fxr.FXR_ERR_INVALID and "one row stride" not in str(e.value) and "the cache is on" not in str(e.value)
    # what holds the rows passes on to the device's check
    for k, more in ((out(19), {}), (out(30, 3 * D)[:, :2 * D], {}), (out(19).view(19, 2, D), {}), (out(7), {"host_count": 7}),
                    (out(3), {"count": idx[:1]}), (out(5), {"idx": idx, "host_count": 5})):
        with pytest.raises(fxr.FxrError, match="the cache is on"):
            fxr.cache_read_q8(cfg, cache, k, k, **more)


@pytest.mark.gpu
@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("rows, asked", [(5, 8), (8, 8), (9, 8), (1, 40), (5, 1000)])
def test_read_back_with_a_device_count_stays_in_its_outputs(cuda, listed, rows, asked):
    n, heads = 40, 2
    g = rng_of(rows)
    cfg = cfg_of(n, heads, "bf16")
    cache = filled_cache(g, cfg, n, "int8")
    store = [torch.full((n + 1, heads * D), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    idx = torch.randperm(n, generator=g, device="cuda").int() if listed else None
    fxr.cache_read_q8(cfg, cache, store[0][:rows], store[1][:rows], idx=idx,
                      count=torch.tensor([asked], dtype=torch.int32, device="cuda"))
    if min(asked, n) > rows:
        with pytest.raises(fxr.FxrError) as e:
            fxr.check_device_error()
        assert e.value.status == fxr.FXR_ERR_BOUNDS
    sync_ok()
    at = idx.long() if listed else torch.arange(n, device="cuda")
    written = min(rows, asked, n)
    for a, want in zip(store, held(cache, n, True)[:2]):
        assert torch.equal(a[:written], want.reshape(n, -1)[at[:written]].bfloat16()) and (a[written:] == 5).all()


def test_write_refuses_sources_that_do_not_hold_the_rows():
    cfg, cache = cfg_of(16, 2, "bf16"), cpu_cache(19)
    wide = cfg_of(16, 2, "bf16", ld_cache=3 * D)
    src = lambda rows, cols=2 * D, t=torch.bfloat16: torch.zeros(rows, cols, dtype=t)  # noqa: E731
    idx = torch.zeros(5, dtype=torch.int32)
    for c, k, v, more in ((cfg, src(15), src(16), {}), (cfg, src(16), src(15), {}), (cfg, src(6), src(6), {"host_count": 7}),
                          (cfg, src(16, D), src(16, D), {}), (cfg, src(16, t=torch.float16), src(16, t=torch.float16), {}),
                          (cfg, src(16, t=torch.float32), src(16), {}), (cfg, src(16), src(16, t=torch.int8), {}),
                          (cfg, src(15), src(15), {"idx": idx, "host_count": 5}), (cfg, src(15), src(15), {"idx": idx, "count": idx[:1]}),
                          (cfg, src(15), src(15), {"count": idx[:1]}), (wide, src(16), src(16), {}), (wide, src(15, 3 * D), src(16, 3 * D), {}),
                          (cfg, src(16), src(16), {"idx": idx, "host_count": 6})):
        with pytest.raises(fxr.FxrError) as e:
            fxr.cache_write_q8(c, k, v, cache, **more)
        assert e.value.status == fxr.FXR_ERR_INVALID and "the cache is on" not in str(e.value)
    for c, k, more in ((cfg, src(16), {}), (cfg, src(17), {}), (cfg, src(16).view(16, 2, D), {}), (cfg, src(32, D), {}),
                       (cfg, src(7), {"host_count": 7}), (cfg, src(16).flatten(), {"idx": idx, "count": idx[:1]}),
                       (wide, src(16, 3 * D)[:, :2 * D], {}), (wide, src(16, 4 * D)[:, :2 * D], {}), (cfg, src(16), {"idx": idx, "host_count": 5})):
        with pytest.raises(fxr.FxrError, match="the cache is on"):
            fxr.cache_write_q8(c, k, k, cache, **more)


def test_lists_counts_and_masks_of_other_types_are_refused(monkeypatch):
    cfg, cache = cfg_of(16, 2, "bf16"), cpu_cache(16)
    good, x = torch.zeros(48, dtype=torch.int32), torch.zeros(16, 2 * D, dtype=torch.bfloat16)
    w = torch.ones(D)
    save = torch.zeros(16, 2 * 2 * D + 16, dtype=torch.uint8)
    monkeypatch.setattr(fxr, "_device_of", lambda *t: 0)
    st = {"qc": x, "out": x, "cache": cache}
    for bad in (good.long(), good.float(), good.short(), good.to(torch.uint8)):
        for call in (lambda b: fxr.cache_read_q8(cfg, cache, x, x, idx=b, count=good), lambda b: fxr.cache_read_q8(cfg, cache, x, x, idx=good, count=b),
                     lambda b: fxr.cache_write_q8(cfg, x, x, cache, idx=b, count=good), lambda b: fxr.cache_write_q8(cfg, x, x, cache, idx=good, count=b),
                     lambda b: fxr.restore_rows_q8(cfg, b, good, good, save, cache), lambda b: fxr.restore_rows_q8(cfg, good, b, good, save, cache),
                     lambda b: fxr.gather_norm_rope_q8(cfg, x, x, x, b, good, good, good, w, w, x, cache),
                     lambda b: fxr.gather_norm_rope_q8(cfg, x, x, x, good, b, good, good, w, w, x, cache),
                     lambda b: fxr.gather_norm_rope_q8(cfg, x, x, x, good, good, b, good, w, w, x, cache),
                     lambda b: fxr.gather_norm_rope_q8(cfg, x, x, x, good, good, good, b, w, w, x, cache),
                     lambda b: fxr.frame_forward_q8(cfg, x, x, x, b, None, good, w, w, cache, x, save),
                     lambda b: fxr.q8_streams([dict(st, idx=b, count=good)]), lambda b: fxr.q8_streams([dict(st, idx=good, count=b)])):
            with pytest.raises(fxr.FxrError, match="32-bit words"):
                call(bad)
    fxr.q8_streams([dict(st, idx=good, count=good.to(torch.uint32))])


def test_frames_refuse_inputs_that_end_early_or_are_of_another_type():
    cfg, cache = cfg_of(16, 2, "bf16", ld_qkv=2 * D + 8, ld_out=2 * D + 16), cpu_cache(16)
    x = torch.zeros(16, 2 * D + 8, dtype=torch.bfloat16)
    good = {"q": x, "k": x[:, :2 * D], "v": x, "mask": torch.zeros(16, dtype=torch.int32), "pos": torch.zeros(16, 3, dtype=torch.int32),
            "norm_q": torch.ones(D), "norm_k": torch.ones(D)}
    frame = dict(good, valid=torch.zeros(16, dtype=torch.uint8), out=torch.zeros(16, 2 * D + 16, dtype=torch.bfloat16)[:, :2 * D])
    one, work = torch.zeros(16, dtype=torch.int32), torch.zeros(64, dtype=torch.uint8)

    def whole(**t):
        t = dict(frame, **t)
        fxr.frame_forward_q8(cfg, t["q"], t["k"], t["v"], t["mask"], t["valid"], t["pos"], t["norm_q"], t["norm_k"], cache, t["out"], work)

    for name in "qkv":
        for bad in (x[:15], x[:, :2 * D].contiguous(), x.half(), x.float(), torch.zeros(16, 2 * D + 16, dtype=torch.bfloat16).t()[:16]):
            with pytest.raises(fxr.FxrError, match=f"{name}: 16 rows of 256"):
                whole(**{name: bad})
    for bad, word in (({"mask": one[:15]}, "mask"), ({"mask": torch.zeros(32, dtype=torch.int32)[::2]}, "mask"), ({"pos": good["pos"][:15]}, "pos"),
                      ({"pos": torch.zeros(3, 16, dtype=torch.int32).t()}, "pos"), ({"norm_q": torch.ones(D).bfloat16()}, "norm"),
                      ({"norm_k": torch.ones(D - 1)}, "norm"), ({"norm_k": torch.ones(2 * D)[::2]}, "norm")):
        with pytest.raises(fxr.FxrError, match=word):
            whole(**bad)
    for bad, word in (({"out": frame["out"][:15]}, "out"), ({"out": torch.zeros(16, 2 * D, dtype=torch.bfloat16)}, "out"),
                      ({"out": frame["out"].half()}, "out"), ({"valid": frame["valid"][:15]}, "valid"), ({"valid": one}, "valid")):
        with pytest.raises(fxr.FxrError, match=word):
            whole(**bad)
    for more in ({}, {"valid": None}, {"valid": torch.zeros(16, dtype=torch.bool)}):
        with pytest.raises(fxr.FxrError, match="the cache is on"):
            whole(**more)


def test_attention_refuses_queries_and_outputs_that_end_early():
    cfg, cache = cfg_of(16, 2, "bf16", ld_out=2 * D + 16), cpu_cache(16)
    one = torch.zeros(16, dtype=torch.int32)
    out = torch.zeros(16, 2 * D + 16, dtype=torch.bfloat16)[:, :2 * D]
    make = lambda **t: fxr.Q8Streams([dict({"qc": torch.zeros(4, 2 * D, dtype=torch.bfloat16), "idx": one, "count": one, "out": out,  # noqa: E731
                                            "cache": cache}, **t)])
    make().check(cfg, 4)
    make(qc=torch.zeros(4, 2, D, dtype=torch.bfloat16)).check(cfg, 4)
    make(qc=torch.zeros(9, 4 * D, dtype=torch.bfloat16)[:4, :2 * D]).check(cfg, 4)
    with pytest.raises(fxr.FxrError, match="out ends"):
        make(out=torch.zeros(16, 2 * D, dtype=torch.bfloat16)).check(cfg, 4)
    with pytest.raises(fxr.FxrError, match="out ends"):
        make(out=torch.zeros(16, 2 * D + 8, dtype=torch.bfloat16)).check(cfg, 4)
    with pytest.raises(fxr.FxrError, match="qc ends"):
        make(qc=torch.zeros(4, D, dtype=torch.bfloat16)).check(cfg, 4)
    with pytest.raises(fxr.FxrError, match="qc ends"):
        make(qc=torch.zeros(4, 2 * D + 8, dtype=torch.bfloat16)[:, :D]).check(cfg, 4)


def test_a_used_configuration_is_copied_and_pickled_as_its_fields():
    cfg = cfg_of(8, 2, "bf16", rope_axes=[16, 56, 56])
    fresh = cfg_of(8, 2, "bf16", rope_axes=[16, 56, 56])
    cfg.ref()
    for other in (copy.copy(cfg), copy.deepcopy(cfg), pickle.loads(pickle.dumps(cfg)), pickle.loads(pickle.dumps(cfg, protocol=2)),
                  dataclasses.replace(cfg), fxr.FrameConfig(**vars(cfg))):
        assert other == cfg == fresh and vars(other) == vars(fresh) and repr(other) == repr(fresh)
        other.n_tokens = 9
        assert other.ref()._obj.n_tokens == 9 and cfg.ref()._obj.n_tokens == 8
    assert dataclasses.asdict(cfg) == dataclasses.asdict(fresh)


def test_a_configuration_s_reference_follows_axes_changed_in_place():
    cfg = cfg_of(8, 2, "bf16", rope_axes=[16, 56, 56])
    assert list(cfg.ref()._obj.rope_axes_dim)[:3] == [16, 56, 56]
    cfg.rope_axes[0], cfg.rope_axes[1] = 32, 40
    assert list(cfg.ref()._obj.rope_axes_dim)[:3] == list(cfg.desc().rope_axes_dim)[:3] == [32, 40, 56]
    cfg.rope_axes.append(0)
    assert cfg.ref()._obj.rope_n_axes == 4 and cfg.ref() is cfg.ref()


# ---- values that the bars of a rounded K leave open -------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("bf16", "e4m3"), ("f16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("n, heads, m", [(700, 2, 2), (333, 2, 30), (700, 2, 300), (2400, 32, 1950)])
@pytest.mark.parametrize("spread", [5.0, 30.0])
def test_scores_in_the_hundreds(cuda, dtype, fmt, n, heads, m, spread):
    """The running maximum moves often, and a row's result is that of a few keys."""
    g = rng_of(int(spread) + m)
    cfg = cfg_of(n, heads, dtype, softmax_scale=spread / math.sqrt(D))
    st = stream_of(g, cfg, m)
    st["cache"] = filled_cache(g, cfg, n, fmt)
    attend(cfg, st, m)
    check(cfg, st, m, telling=0.9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "int8"), ("bf16", "e4m3"), ("f16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("n, heads, m", [(333, 2, 5), (333, 2, 30), (333, 2, 290), (2400, 32, 1950)])
@pytest.mark.parametrize("groups", [False, True])
def test_large_scales(cuda, dtype, fmt, n, heads, m, groups):
    """Scales that the kernels decode in two steps (e4m3 from 128 and 136 on), of K (whose codes are the smallest then, so
    that scores stay plain) and of V, in tiles with smaller ones."""
    g = rng_of(m + n)
    cfg = cfg_of(n, heads, dtype)
    st = stream_of(g, cfg, m)
    st["cache"] = c = filled_cache(g, cfg, n, fmt)
    big = 140.0 if dtype == "f16" else 3000.0 if fmt == "e4m3" else 2.0 ** 90
    c.v_scale[:, 5:n:7] = big
    rows = torch.arange(3, n, 9, device="cuda")
    small = torch.randint(-4, 5, (len(rows), heads * D), generator=g, device="cuda").to(torch.int8)
    if fmt == "e4m3":               # +-4 times 2^-9
        small = torch.where(small < 0, -small - 128, small).to(torch.int8)
    c.k.view(torch.int8)[rows] = small
    c.k_scale[:, 3:n:9] = (140.0 if dtype == "f16" else 256.0) if fmt == "e4m3" else 0.25
    if groups:
        st["q_groups"] = st["k_groups"] = torch.where(torch.arange(n, device="cuda") % 3 == 0, 1, 6).int()
    attend(cfg, st, m)
    check(cfg, st, m, telling=0.8)


# ---- the frame: groups, and very many rows ----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt", [("bf16", "e4m3"), ("f16", "int8")])
@pytest.mark.parametrize("n, heads, rows, bound, prefix, groups", [(300, 3, 20, 24, 0, True), (300, 3, 20, 24, 150, True), (301, 2, 140, 0, 90, True),
                                                                   (300, 2, 0, 24, 40, True), (700, 2, 300, 310, 0, False),
                                                                   (4700, 18, 2049, 2100, 0, False), (8003, 12, 1900, 0, 0, False),
                                                                   (4700, 18, 2049, 2100, 0, True)])
def test_frames_with_groups_and_with_very_many_rows(cuda, dtype, fmt, n, heads, rows, bound, prefix, groups):
    """A frame of a stream whose cache is filled: executed rows, rows that are put back, documents, a padded prefix of
    which nobody sees the end, rows that see nothing."""
    t = TDT[dtype]
    g = rng_of(n + rows)
    cfg = cfg_of(n, heads, dtype)
    f = frame_inputs(g, cfg)
    listed = torch.randperm(n, generator=g, device="cuda")[:rows].sort().values
    mask = torch.zeros(n, dtype=torch.int32, device="cuda")
    mask[listed] = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.3, 1, 2).int()
    given = mask.clone()
    cache = filled_cache(g, cfg, n, fmt)
    pre = filled_cache(g, cfg, prefix, fmt) if prefix else None
    qg = kg = pg = None
    if groups:
        at = torch.arange(n, device="cuda")
        kg = torch.bitwise_left_shift(torch.ones_like(at), at * 3 // n).int()
        kg[n // 2:n // 2 + 9] = 0
        qg = torch.where(at % 7 == 3, torch.zeros_like(kg), kg | 1)
        if prefix:
            pg = torch.full((prefix,), -1, dtype=torch.int32, device="cuda")
            pg[prefix - prefix // 5:] = 0
            pre.k_scale[:, :prefix][:, pg == 0] = math.nan
    copy_of = lambda c: fxr.CacheQ8(*[x.clone() for x in (c.k, c.v, c.k_scale, c.v_scale)])  # noqa: E731
    old, seen = copy_of(cache), copy_of(cache)
    out = torch.full((n, heads * D), 7.0, dtype=t, device="cuda")
    ws = torch.full((fxr.frame_q8_workspace_size(cfg, prefix, bound),), 171, dtype=torch.uint8, device="cuda")
    fxr.frame_forward_q8(cfg, f["q"], f["k"], f["v"], mask, torch.ones(n, dtype=torch.uint8, device="cuda"), f["pos"], f["norm_q"],
                         f["norm_k"], cache, out, ws, prefix=pre, prefix_groups=pg, q_groups=qg, k_groups=kg, max_rows=bound)
    sync_ok()
    assert torch.equal(mask, given)
    # the same write without the rows put back: the cache that the attention saw
    qc, idx = torch.zeros(n, heads * D, dtype=t, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    idx[:rows] = listed.int()
    save = torch.zeros(n, fxr.q8_save_row_bytes(cfg), dtype=torch.uint8, device="cuda")
    fxr.gather_norm_rope_q8(cfg, f["q"], f["k"], f["v"], mask, idx, torch.tensor([rows], dtype=torch.int32, device="cuda"), f["pos"],
                            f["norm_q"], f["norm_k"], qc, seen, save)
    sync_ok()
    st = {"qc": qc, "idx": idx, "m": rows, "cache": seen, "out": out, "q_groups": qg, "k_groups": kg}
    if rows:
        check(cfg, st, bound, pre, pg)
        if groups:
            assert (out[listed[listed % 7 == 3]] == 0).all()
    else:
        assert (out == 7).all()
    kept = mask == 1
    for now, was, new in zip((cache.k, cache.v), (old.k, old.v), (seen.k, seen.v)):
        now, was, new = (x.view(torch.int8) for x in (now, was, new))
        assert torch.equal(now[kept], was[kept]) and torch.equal(now[~kept], new[~kept])
    for now, was, new in zip((cache.k_scale, cache.v_scale), (old.k_scale, old.v_scale), (seen.k_scale, seen.v_scale)):
        assert torch.equal(now[:, :n][:, kept], was[:, :n][:, kept]) and torch.equal(now[:, :n][:, ~kept], new[:, :n][:, ~kept])


def test_a_call_from_another_current_device_is_refused(monkeypatch):
    class On:
        def __init__(self, index):
            self.index, self.device = index, f"cuda:{index}"

        def get_device(self):
            return self.index
    fxr._raw_stream.__globals__["_torch_c"] = torch._C
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 77)
    assert fxr._raw_stream(0, None, On(0), None) == 77
    with pytest.raises(fxr.FxrError, match="tensor on cuda:1, the cache is on cuda:0"):
        fxr._raw_stream(0, None, On(0), On(1))
    with pytest.raises(fxr.FxrError, match="the current device is cuda:0"):
        fxr._raw_stream(1, None, On(1))
    cache = cpu_cache(16)
    with pytest.raises(fxr.FxrError, match="null"):
        fxr.cache_read_q8(cfg_of(16, 2, "bf16"), cache, None, None)
