"""The decode operators (velo_cuda_kv_append, velo_cuda_decode_attention,
velo_cuda_token_logprobs) where a loose comparison would not see a fault: bits of
the append, single tokens lost from long contexts, weights far below a dominant
one, results beside a raised device flag, lengths that change between replays.

Tolerances count the roundings: f16 results 2^-11 of the value (2^-25 below the
normal range), f32 arithmetic 2^-24 per operation."""
from decimal import Decimal, getcontext

import numpy as np
import pytest

import velo_cuda
from test_decode_gpu import ATTN, EPS, _attend, _cache, _dev, _half_step, dctx  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append

def _turned(x, cos, sin):
    """The rotation in f32: both products and their sum rounded."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate((a * cos - b * sin, a * sin + b * cos), -1)


def _append_rows(ctx, k, v, pos, D, base, kv):
    """One token per sequence at `pos`; (pool rows [T][H][D] and scales, k and v), k_out, v_out."""
    import torch
    T, H = k.shape[:2]
    width = int(pos.max()) // 16 + 1
    table = torch.full((T, width), T + 5, dtype=torch.int32, device="cuda")
    table[torch.arange(T, device="cuda"), _dev(pos // 16).long()] = torch.arange(T, dtype=torch.int32, device="cuda")
    dt = {"f16": torch.float16, "int8": torch.int8, "f32": torch.float32}[kv]
    act = torch.float32 if kv == "f32" else torch.float16
    sc = [torch.zeros(T, H, 16, dtype=torch.float16, device="cuda") for _ in range(2)] if kv == "int8" else [None] * 2
    cache = velo_cuda.KvCache(torch.zeros(T, H, 16, D, dtype=dt, device="cuda"),
                              torch.zeros(T, H, 16, D, dtype=dt, device="cuda"), table, *sc)
    ko, vo = (torch.empty(T, H, D, dtype=act, device="cuda") for _ in range(2))
    ctx.kv_append(cache, None, _dev(k), _dev(v), _dev(pos.astype(np.int32)), None, base, k_out=ko, v_out=vo)
    ctx.sync()
    i, s = np.arange(T), pos % 16
    rows = [t.cpu().numpy()[i, :, s] for t in cache.tensors[:2]]
    scales = [None if t is None else t.cpu().numpy()[i, :, s] for t in cache.tensors[3:]]
    return rows, scales, ko.cpu().numpy(), vo.cpu().numpy()


@pytest.mark.parametrize("kv", ["f32", "f16", "int8"])
@pytest.mark.parametrize("D,base", [(128, 10000.0), (64, 500000.0)])
def test_append_rounds_as_the_definition_says(dctx, kv, D, base):
    """Bit for bit: f32 cosine and sine of the exact angle, both products and their
    sum rounded to f32, then the page's rounding (INT8: 127 / max, truncation)."""
    rng = np.random.default_rng(51)
    T, H = 700, 3
    k, v = rng.normal(0, 1, (2, T, H, D)).astype(np.float32)
    pos = rng.integers(0, 120, T)
    a = pos[:, None].astype(np.longdouble) * np.longdouble(base) ** (np.longdouble(-2) * np.arange(D // 2) / D)
    # (each form is within 2^-46 of the exact angle: they part only that near to an f32 tie, with odds of 2^-22 an angle)
    cos, sin = (f(a).astype(np.float32)[:, None] for f in (np.cos, np.sin))
    rows, scales, ko, vo = _append_rows(dctx, k, v, pos, D, base, kv)
    for x, got, sc, out in ((_turned(k, cos, sin), rows[0], scales[0], ko), (v, rows[1], scales[1], vo)):
        if kv == "int8":
            m = np.abs(x).max(-1)
            assert np.array_equal(sc, (m / np.float32(127)).astype(np.float16))
            want = np.trunc(x * (np.float32(127) / m)[..., None]).astype(np.int8)
            assert np.array_equal(got, want)
            assert np.array_equal(out, (want * sc.astype(np.float32)[..., None]).astype(np.float16))
        else:
            want = x.astype(got.dtype)
            assert np.array_equal(got, want) and np.array_equal(out, want)


@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_append_angles_at_the_far_end(dctx, base):
    """The last positions of the widest table (2^30 tokens): rows of (1, 0) become
    the f32 cosine and sine of the exact angle, whose turns are off by 2^-64 a position."""
    import torch
    D, width = 64, 1 << 26
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    pos = np.asarray([16 * width - 1, 16 * width - 12345, 777777777])
    table = torch.full((1, width), 9, dtype=torch.int32, device="cuda")
    for i, p in enumerate(pos):
        table[0, int(p) // 16] = i
    z = torch.zeros(3, 1, 16, D, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), table)
    k = torch.zeros(1, 1, D, device="cuda")
    k[..., :D // 2] = 1
    for i, p in enumerate(pos):
        dctx.kv_append(cache, None, k, k, torch.tensor([int(p)], dtype=torch.int32, device="cuda"), None, base)
    dctx.sync()
    got = cache.tensors[0].cpu().numpy()
    for i, p in enumerate(pos):
        for e in range(D // 2):
            a = Decimal(int(p)) * (Decimal(base).ln() * Decimal(-2 * e) / Decimal(D)).exp() / (2 * pi)  # turns
            a = float(2 * pi * (a - a.to_integral_value()))
            for have, want in ((got[i, 0, p % 16, e], np.cos(a)), (got[i, 0, p % 16, D // 2 + e], np.sin(a))):
                # half a step of f32, 2^30 x 2^-64 turns of 2 pi, the 64-bit forms' own rounding
                assert abs(have - want) <= abs(want) * EPS + 2.0 ** -31 + 2.0 ** -50, (p, e)


@pytest.mark.parametrize("B", [3, 300])
def test_append_flags_starts_that_lose_or_move_tokens(dctx, B):
    """Starts past n_tokens, not from 0, falling or negative set the device flag, with
    a sequence per thread (B = 3) and with the search (B = 300); good ones do not."""
    import torch
    k = torch.ones(B, 1, 64, device="cuda")
    n = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    z = torch.zeros(B, 1, 16, 64, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1))
    good = np.arange(B + 1, dtype=np.int32)

    def run(start):
        dctx.kv_append(cache, None, k, k, n, None, 10000.0, seq_start=_dev(start))
        dctx.sync()
    bad = [np.append(good[:-1], B + 1), np.append(good[:-1], 2 ** 31 - 1), np.append([-2], good[1:]), np.append([1], good[1:]),
           good - 2, np.append(good[:-1], -1), np.append(good[:-1], 0)]
    bad.append(good.copy())
    bad[-1][2] = 0  # 0, 1, 0, 3: falls and rises again
    for start in bad:
        with pytest.raises(velo_cuda.VeloError) as e:
            run(start.astype(np.int32))
        assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
    short = np.minimum(good, B - 2)  # padding behind, an empty sequence at the end
    for start in (good, short, np.zeros(B + 1, np.int32)):
        run(start.astype(np.int32))


def test_append_stores_what_write_kv_stores(dctx):
    """f16 V rows appended to INT8 and f16 pages: the integers, scales and values that
    velo_cuda_write_kv stores for the same rows."""
    import synthetic
    import torch
    T, H, D = 50, 2, 128
    rng = np.random.default_rng(65)
    v = np.clip(rng.normal(0, 1, (T, H, D)) * np.exp(rng.normal(0, 4, (T, H, 1))), -6e4, 6e4).astype(np.float16)
    v[3, 1], v[7, 0], v[9, 0, 5] = 0, 2.0 ** -24, 60000
    meta, tensors = synthetic.llama_q4_model(n_vocab=512, n_embd=256, n_layer=1, n_head=2, n_head_kv=H, n_ff=512, seed=1)
    for kv in (velo_cuda.KV_INT8, velo_cuda.KV_F16):
        int8 = kv == velo_cuda.KV_INT8
        own = velo_cuda.Context(device=0, total_pages=4, max_slots=1, max_pages_per_slot=4, kv_dtype=kv)
        try:
            own.load_model(meta, tensors)
            own.bind_slot(0, np.arange(4, dtype=np.uint32))
            own.write_kv(0, 0, 0, v, v)
            stored = own.read_kv(0, 0, 0, T, H, int8=int8)
        finally:
            own.close()
        z = torch.zeros(4, H, 16, D, dtype=torch.int8 if int8 else torch.float16, device="cuda")
        sc = [torch.zeros(4, H, 16, dtype=torch.float16, device="cuda") for _ in range(2)] if int8 else []
        cache = velo_cuda.KvCache(z, z.clone(), torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), *sc)
        dctx.kv_append(cache, None, _dev(v), _dev(v), _dev(np.zeros(1, np.int32)), None, 10000.0,
                       seq_start=_dev(np.asarray([0, T], np.int32)))
        dctx.sync()
        rows = np.moveaxis(cache.tensors[1].cpu().numpy(), 1, 2).reshape(-1, H, D)[:T]
        assert np.array_equal(rows, stored[1])
        if int8:
            scales = np.moveaxis(cache.tensors[4].cpu().numpy(), 1, 2).reshape(-1, H)[:T]
            assert np.array_equal(scales.view(np.uint16), stored[3])


# ------------------------------------------------------------------ attention

TOKENS = {"f16": 16, "int8": 32, "f32": 8}  # of a step


def _exact(q, d, lens, kv, scale=None):
    """64-bit attention per head with what its rounding is measured by: out, lse,
    sum p |v| (INT8: and sum p 255 |scale|, whose values carry a bias of 128 through
    the sums), the largest |v|, and the largest sum of a score's |products|."""
    B, Hq, D = q.shape
    Hkv = d["k"].shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out, mag = np.zeros((2, B, Hq, D))
    lse, reach, mag8, vmax = np.full((B, Hq), -np.inf), *np.zeros((3, B, Hq))
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        ids = d["table"][b, :-(-n // 16)].astype(np.int64)

        def rows(name):
            x = d[name][ids].astype(np.float64).transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n]
            if kv != "int8":
                return x, None
            sc = d[name + "_scale"][ids].astype(np.float64).transpose(1, 0, 2).reshape(Hkv, -1)[:, :n]
            return x * sc[..., None], sc
        (k, ks), (v, vs) = rows("k"), rows("v")
        for h in range(Hq):
            g = h // (Hq // Hkv)
            qh = q[b, h].astype(np.float64) * scale
            x = k[g] @ qh
            reach[b, h] = (np.abs(k[g]) @ np.abs(qh)).max() if kv != "int8" else 255 * np.abs(ks[g]).max() * np.abs(qh).sum()
            m = x.max()
            e = np.exp(x - m)
            lse[b, h] = m + np.log(e.sum())
            w = e / e.sum()
            out[b, h], mag[b, h], vmax[b, h] = w @ v[g], w @ np.abs(v[g]), np.abs(v[g]).max()
            if kv == "int8":
                mag8[b, h] = 255 * (w @ np.abs(vs[g]))
    return out, lse, mag, mag8, vmax, reach


def _check_close(out, lse, q, d, lens, kv, scale=None):
    """Tolerances per sequence and head.  A score: D products added in f32 (INT8: D / 16
    matrix steps of 2^-22 of the biased sum), the change of base and the difference from
    the reference, 2^-22 of its size.  A weight: that, its exponential 2^-21, its two f16
    parts 2^-21.  The weighted sums: 2^-23 per addition of a chain through one warp's steps
    of the item, 32 tokens within a step and 64 states joined; INT8's six products of
    biased values a step.  f16 parts below the normal range: 2^-39 of a step's largest
    weight for each of 32 tokens.  f16 output: half a step."""
    want, want_lse, mag, mag8, vmax, reach = _exact(q, d, lens, kv, scale)
    Hkv, D = d["k"].shape[1], q.shape[-1]
    units = -(-np.asarray(lens, np.int64) // TOKENS[kv])
    chain = np.minimum(units / 4 + 1, units.sum() * Hkv * -(-(q.shape[1] // Hkv) // 4) / 296 + 8) + 96
    ds = reach * ((D / 16 + 8) * 2.0 ** -22 if kv == "int8" else (D + 8) * EPS) + 2.0 ** -22 * np.abs(reach)
    dw = ds + 2.0 ** -20 + chain[:, None] * 2.0 ** -23
    tol = _half_step(want, kv != "f32") + 2 * dw[..., None] * mag
    if kv != "f32":
        tol += (2.0 ** -20 * mag8 + 2.0 ** -34 * vmax)[..., None]
    assert np.isfinite(out).all()
    err = np.abs(out - want)
    assert (err <= tol).all(), ((err / tol).max(), np.unravel_index((err / tol).argmax(), err.shape))
    if lse is not None:
        empty = np.isneginf(want_lse)
        assert (lse[empty] == want_lse[empty]).all()
        err = np.abs(lse[~empty] - want_lse[~empty])
        assert (err <= (dw + 4 * EPS * (1 + np.abs(want_lse)))[~empty]).all()


def _set(d, kv, b, t, name, row, scale=None):
    """Token t of sequence b: `row` for every KV head."""
    at = d["table"][b, t // 16], slice(None), t % 16
    d[name][at] = row
    if kv == "int8":
        d[name + "_scale"][at] = scale


@pytest.mark.parametrize("group", [4, 8, 16])
@pytest.mark.parametrize("kv,n,nats", [("f16", 203, 18), ("f16", 4095, 18.5), ("f16", 30000, 12), ("f16", 30000, 16),
                                       ("f16", 30000, 20), ("f16", 100003, 23), ("int8", 203, 18), ("int8", 4095, 21),
                                       ("int8", 30000, 16), ("int8", 30000, 23), ("f32", 4095, 18.5)])
def test_attention_small_weights_beside_a_dominant_one(dctx, kv, n, nats, group):
    """One token takes nearly all of the weight and has a V of 0: the output is what the
    others, `nats` below it, add up to, and keeps its digits."""
    rng = np.random.default_rng(int(n + 10 * nats))
    D, Hkv, lens = 64, 2, [n, 40]
    d = _cache(rng, kv, lens, Hkv, D)
    for b, m in enumerate(lens):
        low = -nats * (1 + 0.02 * rng.random((m, 1)))
        ids, slots = d["table"][b, np.arange(m) // 16], np.arange(m) % 16
        v = 1 + rng.normal(0, 0.5, (m, Hkv, D))
        if kv == "int8":
            d["k"][ids, :, slots] = 0
            d["k"][ids, :, slots, 0] = -127
            d["k_scale"][ids, :, slots] = (-low / 127).astype(np.float16)
            d["v"][ids, :, slots] = np.clip(np.trunc(v * 40), -127, 127)
            d["v_scale"][ids, :, slots] = 0.025
        else:
            d["k"][ids, :, slots] = 0
            d["k"][ids, :, slots, 0] = low
            d["v"][ids, :, slots] = v
        _set(d, kv, b, int(m * 0.37), "k", 0, 0.1)
        _set(d, kv, b, int(m * 0.37), "v", 0, 0.0)
    q = np.zeros((2, group * Hkv, D), np.float32 if kv == "f32" else np.float16)
    q[:, :, 0] = 1 + 0.02 * np.arange(group * Hkv) / group
    out, lse = _attend(dctx, d, q, lens, scale=1.0)
    _check_close(out, lse, q, d, lens, kv, 1.0)


def test_attention_int8_scale_of_a_token_without_weight(dctx):
    """A V scale 2^25 above the others', on a token 60 nats below them: it costs them no digits."""
    rng = np.random.default_rng(61)
    lens, Hkv, D = [700, 33], 2, 128
    d = _cache(rng, "int8", lens, Hkv, D)
    for name in ("k", "v"):
        d[name + "_scale"][:] = np.where(np.isfinite(d[name + "_scale"]), np.float16(0.001), d[name + "_scale"])
    q = np.zeros((2, 16, D), np.float16)
    q[:, :, 0] = 1
    for b, t in ((0, 5), (0, 350), (1, 9)):
        row = np.zeros(D)
        row[0] = -127
        _set(d, "int8", b, t, "k", row, 0.5)
        _set(d, "int8", b, t, "v", 127, 60000)
    out, lse = _attend(dctx, d, q, lens, scale=1.0)
    # (the token's own e^-63.5 x 127 x 60000 is below 2^-60: vmax is the others')
    keep = dict(d, v_scale=np.where(d["v_scale"] == 60000, np.float16(0), d["v_scale"]))
    _check_close(out, lse, q, keep, lens, "int8", 1.0)


def test_attention_of_wide_page_tables(dctx):
    """What bounds the table's width is the work its rows can hold: 256 sequences of 64
    heads may have rows of 2^20 tokens; a step more than 2^30 of them is refused."""
    import ctypes

    import torch
    rng = np.random.default_rng(62)
    lens, Hq, Hkv, D = [int(n) for n in rng.integers(0, 100, 256)], 64, 8, 64
    for kv in ("f16", "int8"):
        d = _cache(rng, kv, lens, Hkv, D)
        q = rng.normal(0, 1, (256, Hq, D)).astype(np.float16)
        table = torch.full((256, 1 << 16), 1 << 30, dtype=torch.int32, device="cuda")
        table[:, :d["table"].shape[1]] = _dev(d["table"])
        scales = [None if d[n] is None else _dev(d[n]) for n in ("k_scale", "v_scale")]
        cache = velo_cuda.KvCache(_dev(d["k"]), _dev(d["v"]), table, *scales)
        out, lse = _attend(dctx, d, q, lens, cache=cache)
        _check_close(out, lse, q, d, lens, kv)
    L = velo_cuda.lib()
    for kv, n_kv, n_head, pages in (("f16", 8, 64, 1 << 15), ("f16", 8, 128, 1 << 15), ("f16", 8, 129 * 8, 3640),
                                    ("int8", 8, 64, 1 << 16), ("f32", 8, 64, 1 << 14), ("f32", 8, 72, 1 << 13)):
        # f16, 129 heads a KV head: 9 tiles of 16; f32, 9: two tiles of 8
        desc = velo_cuda.KvCacheDesc.from_buffer_copy(cache.desc)
        desc.kv_dtype = {"f16": velo_cuda.KV_F16, "int8": velo_cuda.KV_INT8, "f32": velo_cuda.KV_F32}[kv]
        desc.n_kv = n_kv
        for width, message in ((pages, "NULL buffer"), (pages + 2, "2^30")):
            desc.max_pages = width
            assert L.velo_cuda_decode_attention(dctx.handle, ctypes.byref(desc), None, 1 << 20, None, 4096, n_head, 0.0,
                                                None, None, None, 0) == velo_cuda.ERR_INVALID_ARGUMENT
            assert message in velo_cuda.last_error(), (kv, width, velo_cuda.last_error())


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,lens", ATTN + [(16, 2, 128, [30011, 1]), (32, 8, 64, [1000 + 37 * i % 500 for i in range(40)])])
def test_attention_close_per_head(dctx, kv, Hq, Hkv, D, lens):
    rng = np.random.default_rng(Hq * 1000 + D + len(lens) + 1)
    d = _cache(rng, kv, lens, Hkv, D)
    q = (rng.normal(0, 1, (len(lens), Hq, D)) * 1.5).astype(np.float32 if kv == "f32" else np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_close(out, lse, q, d, lens, kv)


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,lens", [
    (4, 4, 128, [1, 2, 15, 16, 17, 31, 32, 33, 0, 128, 1000]), (64, 8, 128, [60011]), (32, 32, 128, [203, 4097]),
    (16, 1, 64, [30011, 5, 20000]), (32, 8, 64, [1000 + 37 * i % 500 for i in range(70)]),
    (24, 1, 128, [5000, 300]), (18, 2, 64, [7 * i % 300 for i in range(300)])])
def test_attention_loses_no_token(dctx, kv, Hq, Hkv, D, lens):
    """Queries of 0 weigh all tokens alike, and token t has a V of 1 in dimension t % D
    alone: every output is that dimension's share of the tokens, which one token left
    out or taken twice moves by more than a rounding, wherever the list is cut."""
    rng = np.random.default_rng(len(lens))
    d = _cache(rng, kv, lens, Hkv, D)
    for b, n in enumerate(lens):
        t = np.arange(n)
        ids, slots = d["table"][b, t // 16], t % 16
        d["v"][ids, :, slots] = 0
        d["v"][ids, :, slots, t % D] = 64 if kv == "int8" else 1
        if kv == "int8":
            d["v_scale"][ids, :, slots] = 2.0 ** -6
    q = np.zeros((len(lens), Hq, D), np.float32 if kv == "f32" else np.float16)
    out, lse = _attend(dctx, d, q, lens)
    for b, n in enumerate(lens):
        share = np.bincount(np.arange(n) % D, minlength=D) / max(n, 1)
        # sums of ones are exact; the quotient and its product round, as does the output
        assert (np.abs(out[b] - share) <= _half_step(share, kv != "f32") + 4 * EPS * share).all(), (b, n)
        assert n or np.isneginf(lse[b]).all()
        assert n == 0 or (np.abs(lse[b] - np.log(n)) <= 8 * EPS * (1 + np.log(n))).all()


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
def test_attention_results_beside_the_flag(dctx, kv):
    """A page outside the pool leaves its tokens out, a length past the row ends with
    it, a negative one is 0: the flag is set and the results are those."""
    import torch
    rng = np.random.default_rng(63)
    D, Hkv, Hq = 64, 2, 8
    q = rng.normal(0, 1, (3, Hq, D)).astype(np.float32 if kv == "f32" else np.float16)
    lens = [64, 64, 57]
    d = _cache(rng, kv, lens, Hkv, D, spare=0, poison=False)
    d["table"] = np.ascontiguousarray(d["table"][:, :4])
    outside = d["k"].shape[0]

    def run(table, n):
        dd = dict(d, table=table)
        cache = velo_cuda.KvCache(_dev(dd["k"]), _dev(dd["v"]), _dev(table),
                                  *(None if d[x] is None else _dev(d[x]) for x in ("k_scale", "v_scale")))
        out, lse = torch.full((3, Hq, D), 7.0, dtype=_dev(q).dtype, device="cuda"), torch.full((3, Hq), 7.0, device="cuda")
        ws = torch.empty(dctx.decode_attention_workspace(Hq, Hkv, D), dtype=torch.uint8, device="cuda")
        dctx.decode_attention(cache, _dev(q), _dev(np.asarray(n, np.int32)), out, ws, lse=lse)
        with pytest.raises(velo_cuda.VeloError) as e:
            dctx.sync()
        assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
        return out.cpu().numpy(), lse.cpu().numpy()

    def check(got, table, n):
        _check_close(*got, q, dict(d, table=table), n, kv)
    check(run(d["table"], [65, -1, 57]), d["table"], [64, 0, 57])
    check(run(d["table"], [2 ** 31 - 1, -2 ** 31, 57]), d["table"], [64, 0, 57])
    for lost in range(4):
        table = d["table"].copy()
        table[:, lost] = [outside, -1, outside + 3] if lost < 3 else [outside, -1, table[2, 3]]
        rest = np.delete(d["table"], lost, 1)
        if lost == 3:  # the last sequence keeps its ragged page
            got = run(table, lens)
            want = np.where(np.arange(3)[:, None] < 2, np.pad(rest, ((0, 0), (0, 1))), d["table"])
            check(got, want, [48, 48, 57])
        else:
            check(run(table, lens), rest, [48, 48, 41])


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
def test_attention_graph_replayed_with_other_lengths(dctx, kv):
    """One captured call, replayed with lengths that are cut in other places, in
    fewer ones or not at all."""
    import torch
    rng = np.random.default_rng(64)
    full = [9000, 700, 40]
    d = _cache(rng, kv, full, 2, 128, poison=False)
    scales = [None if d[n] is None else _dev(d[n]) for n in ("k_scale", "v_scale")]
    cache = velo_cuda.KvCache(_dev(d["k"]), _dev(d["v"]), _dev(d["table"]), *scales)
    q = rng.normal(0, 1, (3, 8, 128)).astype(np.float32 if kv == "f32" else np.float16)
    qd, nd = _dev(q), torch.tensor([33, 700, 1], dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(qd), torch.zeros(3, 8, device="cuda")
    ws = torch.empty(dctx.decode_attention_workspace(8, 2, 128), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dctx.set_stream(torch.cuda.current_stream().cuda_stream)
        dctx.decode_attention(cache, qd, nd, out, ws, lse=lse)
    dctx.set_stream(velo_cuda.DEFAULT_STREAM)
    for lens in ([1, 650, 40], [9000, 0, 17], [0, 0, 0], full, [8999, 1, 0], [16, 16, 16]):
        nd.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        _check_close(out.cpu().numpy(), lse.cpu().numpy(), q, d, lens, kv)
    dctx.sync()


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (16, 2), (32, 2)])
def test_attention_keeps_nan_to_its_heads(dctx, kv, Hq, Hkv):
    """A NaN in one head's query, an infinite K and a NaN V in one KV head: the other
    heads and sequences are as without them, the touched ones hold a NaN."""
    rng = np.random.default_rng(66)
    lens, D, group = [700, 33], 64, Hq // Hkv
    d = _cache(rng, kv, lens, Hkv, D)
    q = rng.normal(0, 1, (2, Hq, D)).astype(np.float32 if kv == "f32" else np.float16)
    want = _attend(dctx, d, q, lens)
    bad = q.copy()
    bad[0, 1, 7] = np.nan
    out, lse = _attend(dctx, d, bad, lens)
    rest = np.ones((2, Hq), bool)
    rest[0, 1] = False
    assert np.array_equal(out[rest], want[0][rest]) and np.array_equal(lse[rest], want[1][rest])
    assert np.isnan(out[0, 1]).all() and np.isnan(lse[0, 1])
    for name, value in (("k", np.inf), ("v", np.nan)):
        dd = {n: None if a is None else a.copy() for n, a in d.items()}
        where = name + "_scale" if kv == "int8" else name
        dd[where][d["table"][0, 20], 1, 5] = value
        if kv == "int8":
            dd[name][d["table"][0, 20], 1, 5, 0] = 1  # (a 0 would already be NaN)
        out, lse = _attend(dctx, dd, q, lens)
        rest = np.ones((2, Hq), bool)
        rest[0, group:] = False
        assert np.array_equal(out[rest], want[0][rest]) and np.array_equal(lse[rest], want[1][rest])
        # an infinite K scores +inf, -inf (no weight) or NaN; the head's V is NaN in at least one dimension
        if name == "v":
            assert np.isnan(out[0, group:]).any(-1).all() and np.array_equal(lse, want[1])


# ------------------------------------------------------------------ far offsets

@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
def test_pages_past_32_bits(dctx, kv):
    """Pools of more than 2^32 elements: the last pages are appended to and read."""
    import torch
    Hkv, Hq, D = 8, 32, 128
    pages = (1 << 32) // (Hkv * 16 * D) + 40
    dt = {"f16": torch.float16, "int8": torch.int8, "f32": torch.float32}[kv]
    act = torch.float32 if kv == "f32" else torch.float16
    pools = [torch.empty(pages, Hkv, 16, D, dtype=dt, device="cuda") for _ in range(2)]
    sc = [torch.empty(pages, Hkv, 16, dtype=torch.float16, device="cuda") for _ in range(2)] if kv == "int8" else []
    rng = np.random.default_rng(67)
    new = [70, 33]
    ids = np.concatenate((rng.choice(20, 3, replace=False), pages - 1 - rng.choice(20, 5, replace=False)))
    table = rng.permutation(ids).reshape(2, 4).astype(np.int32)
    table = np.pad(table, ((0, 0), (0, 1)))
    table[0, 4], table[1, 3:] = pages - 30, 0
    cache = velo_cuda.KvCache(*pools, _dev(table), *sc)
    T = sum(new)
    x = _dev(rng.normal(0, 1, (T, Hq + 2 * Hkv, D)).astype(np.float32))
    q, ko, vo = (torch.empty(T, h, D, dtype=act, device="cuda") for h in (Hq, Hkv, Hkv))
    dctx.kv_append(cache, x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], _dev(np.zeros(2, np.int32)), q, 10000.0,
                   seq_start=_dev(np.asarray([0, 70, 103], np.int32)), k_out=ko, v_out=vo)
    last = q[[69, 102]].contiguous()
    out, lse = torch.empty_like(last), torch.empty(2, Hq, device="cuda")
    ws = torch.empty(dctx.decode_attention_workspace(Hq, Hkv, D), dtype=torch.uint8, device="cuda")
    dctx.decode_attention(cache, last, _dev(np.asarray(new, np.int32)), out, ws, lse=lse)
    dctx.sync()
    # the pages in use, copied to a small cache
    used, at = np.unique(table, return_inverse=True)
    small = {n: t[_dev(used).long()].cpu().numpy() for n, t in zip(("k", "v", "k_scale", "v_scale"), pools + sc)}
    small = dict({"k_scale": None, "v_scale": None}, **small, table=at.reshape(table.shape).astype(np.int32))
    for n, rows in (("k", ko), ("v", vo)):
        have = small[n][small["table"]].astype(np.float32)  # [2][5][Hkv][16][D]
        if kv == "int8":
            have = have * small[n + "_scale"][small["table"]].astype(np.float32)[..., None]
        have = np.moveaxis(have, 2, 3).reshape(2, -1, Hkv, D).astype(rows.cpu().numpy().dtype)
        assert np.array_equal(np.concatenate([have[0, :70], have[1, :33]]), rows.cpu().numpy())
    _check_close(out.cpu().numpy(), lse.cpu().numpy(), last.cpu().numpy(), small, new, kv)


@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_logits_past_32_bits(dctx, src):
    """Rows further apart than 2^32 elements in all."""
    import torch
    M, V, ldl = 17, 5000, (1 << 28) + 1
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[src]
    wide = torch.empty((M - 1) * ldl + V, dtype=dt, device="cuda").as_strided((M, V), (ldl, 1))
    x = torch.from_numpy(np.random.default_rng(68).normal(0, 3, (M, V)).astype(np.float32)).to(dt).cuda()
    wide.copy_(x)
    tok = torch.arange(M, dtype=torch.int32, device="cuda")
    lp, ids, tl = torch.empty(M, device="cuda"), torch.empty(M, 3, dtype=torch.int32, device="cuda"), torch.empty(M, 3, device="cuda")
    dctx.token_logprobs(wide, tok, lp, None, ids, tl)
    dctx.sync()
    want = torch.log_softmax(x.double(), -1)
    # (V / 256 + 64) additions, the exponential, arguments of up to 20
    tol = (V / 256 + 64) * EPS + 2.0 ** -20 + 40 * EPS
    assert (lp - want.gather(1, tok.long()[:, None])[:, 0]).abs().max() <= tol
    assert (tl - want.gather(1, ids.long())).abs().max() <= tol
    assert torch.equal(x.gather(1, ids.long()), x.sort(-1, descending=True).values[:, :3])


# ------------------------------------------------------------------ log probabilities

@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("V", [7, 70001])
def test_logprobs_of_logits_far_apart(dctx, src, V):
    """Logits whose difference passes the largest f32, under temperatures that bring
    the quotient back: a log probability of -6e8 is not -inf, a masked one is."""
    import torch
    x = torch.zeros(3, V)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = 3e38, 2e38, -3e38, -np.inf
    x = x.to({"f32": torch.float32, "bf16": torch.bfloat16}[src])
    lp, tok = torch.zeros(3, device="cuda"), torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    ids, tl = torch.zeros(3, min(V, 64), dtype=torch.int32, device="cuda"), torch.zeros(3, min(V, 64), device="cuda")
    for T in (1e30, 1e25):
        want = torch.log_softmax(x.double() / T, -1)
        dctx.token_logprobs(x.cuda(), tok, lp, None, ids, tl, temperature=T)
        dctx.sync()
        for got, w in ((lp.cpu().double(), want.gather(1, tok.cpu().long()[:, None])[:, 0]),
                       (tl.cpu().double(), want.gather(1, ids.cpu().long()))):
            finite = torch.isfinite(w)
            assert torch.equal(got[~finite], w[~finite])
            # 1 / T, its product and the difference: four roundings
            assert ((got - w)[finite].abs() <= 4 * EPS * w[finite].abs() + 1e-6).all()
