"""One-token decoding over a paged cache on the device: K/V append with
rotation, decode attention and token log probabilities against plain 64-bit
forms (decode_reference), their refusals, and a run of them together.

Tolerances count the roundings: f16 results 2^-11 of the value (2^-25 below the
normal range), f32 arithmetic 2^-24 per operation along the longest chain."""
import numpy as np
import pytest

import decode_reference as ref
import velo_cuda

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24  # half a step of f32


@pytest.fixture()
def dctx(ctx):
    """The context on torch's default stream; the device flag is clean after each test."""
    ctx.set_stream(velo_cuda.DEFAULT_STREAM)
    yield ctx
    ctx.set_stream(None)
    try:
        ctx.sync()
    except velo_cuda.VeloError:
        pass


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _half_step(x, f16):
    return np.maximum(np.abs(x) * 2.0 ** -11, 2.0 ** -25) if f16 else np.abs(x) * EPS


# ------------------------------------------------------------------ caches

def _cache(rng, kv, lens, Hkv, D, spare=2, poison=True):
    """A cache with permuted pages; slots past each length hold NaN (int8: huge
    scales), and unused table entries an id outside the pool."""
    need = [-(-int(n) // 16) for n in lens]
    pages, width = sum(need) + spare, max(max(need), 1) + 1
    perm = rng.permutation(pages)
    table = np.full((len(lens), width), pages + 7, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    d = {"table": table, "k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        x = rng.normal(0, 1, (pages, Hkv, 16, D)).astype(np.float32)
        if kv == "int8":
            m = np.abs(x).max(-1)
            d[name + "_scale"] = (m / 127).astype(np.float16)
            d[name] = np.trunc(x * (127 / m)[..., None]).astype(np.int8)
        else:
            d[name] = x.astype(np.float16 if kv == "f16" else np.float32)
    if poison:
        for b, n in enumerate(lens):
            if n % 16:
                pg = table[b, n // 16]
                if kv == "int8":
                    d["k_scale"][pg, :, n % 16:] = np.inf
                    d["v_scale"][pg, :, n % 16:] = np.nan
                else:
                    d["k"][pg, :, n % 16:] = np.nan
                    d["v"][pg, :, n % 16:] = np.inf
        for pg in perm[at:]:
            if kv != "int8":
                d["k"][pg] = np.nan
    return d


def _kv_cache(d):
    return velo_cuda.KvCache(_dev(d["k"]), _dev(d["v"]), _dev(d["table"]),
                             None if d["k_scale"] is None else _dev(d["k_scale"]),
                             None if d["v_scale"] is None else _dev(d["v_scale"]))


def _attend(ctx, d, q, lens, scale=0.0, lse=True, cache=None):
    import torch
    B, Hq, D = q.shape
    cache = cache or _kv_cache(d)
    qd = _dev(q)
    out = torch.full_like(qd, float("nan"))
    ls = torch.full((B, Hq), float("nan"), device="cuda") if lse else None
    ws = torch.full((ctx.decode_attention_workspace(Hq, cache.n_kv, D),), 0xff, dtype=torch.uint8, device="cuda")
    ctx.decode_attention(cache, qd, _dev(np.asarray(lens, np.int32)), out, ws, lse=ls, scale=scale)
    ctx.sync()
    return out.cpu().numpy(), None if ls is None else ls.cpu().numpy()


def _check_attention(out, lse, q, d, lens, kv, scale=None):
    want, want_lse, reach, vmax = ref.attention(q, d["k"], d["v"], d["table"], lens, d["k_scale"], d["v_scale"], scale)
    D = q.shape[-1]
    # a score's error: D products added in f32, the scale and the change of base; a
    # weight's: that, its exponential (2^-21) and its two-part rounding (f16 pairs
    # 2^-21, bf16 pairs of int8 pages 2^-16); weights enter numerator and denominator,
    # and sums over the longest chain add (length / 16 + 64) roundings
    ds = (D + 8) * EPS * reach
    dw = ds + 2.0 ** -20 + (2.0 ** -16 if kv == "int8" else 0) + (max(lens, default=0) / 16 + 64) * EPS
    tol = _half_step(want, kv != "f32") + 2 * dw * vmax
    assert np.isfinite(out).all()
    err = np.abs(out - want)
    assert (err <= tol).all(), (err - tol).max()
    if lse is not None:
        empty = np.isneginf(want_lse)
        assert (lse[empty] == want_lse[empty]).all()
        err = np.abs(lse[~empty] - want_lse[~empty])
        assert (err <= dw + 4 * EPS * (1 + np.abs(want_lse[~empty]))).all()


ATTN = [
    # Hq, Hkv, D, lens
    (4, 4, 128, [1]),
    (8, 1, 128, [16]),
    (8, 8, 64, [0, 1, 15, 16, 17, 31, 33]),
    (32, 8, 128, [0, 0, 640, 3]),
    (64, 8, 128, [1500, 0, 77]),
    (12, 12, 64, [1025]),
    (5, 1, 128, [100, 31]),
    (18, 2, 128, [259, 8]),          # 9 heads a KV head
    (16, 1, 64, [513]),
    (24, 1, 128, [300, 2]),          # more heads a KV head than one row tile
    (40, 1, 64, [48, 0, 129]),
    (32, 8, 128, [4099, 1, 2050, 17]),
    (4, 2, 64, [int(7 + 37 * i) % 150 for i in range(97)]),
]


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,lens", ATTN)
def test_attention_matches_plain(dctx, kv, Hq, Hkv, D, lens):
    rng = np.random.default_rng(Hq * 1000 + D + len(lens))
    d = _cache(rng, kv, lens, Hkv, D)
    q = (rng.normal(0, 1, (len(lens), Hq, D)) * 1.5).astype(np.float32 if kv == "f32" else np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_attention(out, lse, q, d, lens, kv)
    again, lse2 = _attend(dctx, d, q, lens)
    assert np.array_equal(out, again) and np.array_equal(lse, lse2)


@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
def test_attention_long_split(dctx, kv):
    rng = np.random.default_rng(3)
    lens = [30011, 1]
    d = _cache(rng, kv, lens, 2, 128)
    q = rng.normal(0, 2, (2, 16, 128)).astype(np.float32 if kv == "f32" else np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_attention(out, lse, q, d, lens, kv)


@pytest.mark.parametrize("kv,B,Hq", [("f16", 40, 32), ("int8", 96, 16)])
def test_attention_long_list_with_its_tail(dctx, kv, B, Hq):
    """Enough work for the short ranges at the list's end: items cut in both parts."""
    rng = np.random.default_rng(10)
    lens = [int(n) for n in rng.integers(1000, 1500, B)]
    d = _cache(rng, kv, lens, 8, 64)
    q = rng.normal(0, 1.5, (B, Hq, 64)).astype(np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_attention(out, lse, q, d, lens, kv)
    again, lse2 = _attend(dctx, d, q, lens)
    assert np.array_equal(out, again) and np.array_equal(lse, lse2)


def test_attention_shared_prefix_pages(dctx):
    """Sequences whose tables name the same pages, and a page named twice."""
    rng = np.random.default_rng(15)
    d = _cache(rng, "f16", [70, 70, 70], 2, 128, poison=False)
    d["table"][1, :4] = d["table"][0, :4]
    d["table"][2, :5] = d["table"][0, [0, 1, 1, 0, 4]]
    q = rng.normal(0, 1, (3, 4, 128)).astype(np.float16)
    out, lse = _attend(dctx, d, q, [70, 64, 66])
    _check_attention(out, lse, q, d, [70, 64, 66], "f16")


def test_attention_int8_scales_of_any_size(dctx):
    """V scales from subnormal to large within one context, negative and zero ones."""
    rng = np.random.default_rng(16)
    lens = [333, 90, 40]
    d = _cache(rng, "int8", lens, 2, 128, poison=False)
    for b, n in enumerate(lens):
        for t in range(n):
            f = [[1e-3, 1.0, 300.0][t % 3], 2.0 ** -20, 0.0][b] * (-1 if t % 5 == 0 else 1)
            d["v_scale"][d["table"][b, t // 16], :, t % 16] *= np.float16(f)
    q = rng.normal(0, 1, (3, 8, 128)).astype(np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_attention(out[:1], lse[:1], q[:1], dict(d, table=d["table"][:1]), lens[:1], "int8")
    _check_attention(out[1:2], lse[1:2], q[1:2], dict(d, table=d["table"][1:2]), lens[1:2], "int8")
    assert (out[2] == 0).all() and np.isfinite(lse[2]).all()


def test_attention_many_sequences(dctx):
    rng = np.random.default_rng(4)
    lens = [int(x) for x in rng.integers(0, 40, 4096)]
    d = _cache(rng, "f16", lens, 1, 64)
    q = rng.normal(0, 1, (4096, 2, 64)).astype(np.float16)
    out, lse = _attend(dctx, d, q, lens)
    _check_attention(out, lse, q, d, lens, "f16")


def test_attention_peaked_scores_and_scale(dctx):
    """One key far above the others, wherever it lies; scores growing along the
    context (the running maximum moves at every step); a given scale."""
    rng = np.random.default_rng(5)
    lens = [200, 333, 64]
    d = _cache(rng, "f16", lens, 1, 64)
    for b, n in enumerate(lens):
        for t in range(n):
            d["k"][d["table"][b, t // 16], 0, t % 16] = np.float16(0.002 * t) if b < 2 else np.float16(0)
    d["k"][d["table"][2, 2], 0, 5] = 8
    q = np.ones((3, 8, 64), np.float16) * np.linspace(0.5, 8, 8).astype(np.float16)[None, :, None]
    out, lse = _attend(dctx, d, q, lens, scale=0.5)
    _check_attention(out, lse, q, d, lens, "f16", 0.5)


def test_attention_strided_queries_and_no_lse(dctx):
    import torch
    rng = np.random.default_rng(6)
    lens = [50, 129, 0]
    d = _cache(rng, "f16", lens, 2, 128)
    wide = _dev(rng.normal(0, 1, (3, 12, 128)).astype(np.float16))
    q = wide[:, 4:12]
    out = torch.full((3, 8, 128), float("nan"), dtype=torch.float16, device="cuda")
    ws = torch.empty(dctx.decode_attention_workspace(8, 2, 128), dtype=torch.uint8, device="cuda")
    dctx.decode_attention(_kv_cache(d), q, _dev(np.asarray(lens, np.int32)), out, ws)
    dctx.sync()
    _check_attention(out.cpu().numpy(), None, q.cpu().numpy(), d, lens, "f16")


def test_attention_flags_bad_lengths_and_pages(dctx):
    rng = np.random.default_rng(7)
    lens = [40, 33]
    d = _cache(rng, "f16", lens, 1, 128)
    q = rng.normal(0, 1, (2, 4, 128)).astype(np.float16)
    bad = dict(d, table=d["table"].copy())
    bad["table"][1, 1] = d["k"].shape[0]  # one page outside the pool: its 16 tokens are left out
    with pytest.raises(velo_cuda.VeloError) as e:
        _attend(dctx, bad, q, lens)
    assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
    with pytest.raises(velo_cuda.VeloError) as e:
        _attend(dctx, d, q, [40, -1])
    assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
    full = _cache(rng, "f16", [64, 64], 1, 128, spare=0)
    full["table"] = np.ascontiguousarray(full["table"][:, :4])
    with pytest.raises(velo_cuda.VeloError) as e:
        _attend(dctx, full, q, [64, 65])
    assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
    out, lse = _attend(dctx, d, q, lens)  # the flag was read: a clean call passes
    _check_attention(out, lse, q, d, lens, "f16")


def test_attention_refusals(dctx):
    import torch
    rng = np.random.default_rng(8)
    d = _cache(rng, "f16", [20], 2, 128)
    cache = _kv_cache(d)
    q = torch.zeros(1, 4, 128, dtype=torch.float16, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(dctx.decode_attention_workspace(4, 2, 128), dtype=torch.uint8, device="cuda")

    def refused(f):
        with pytest.raises(velo_cuda.VeloError) as e:
            f()
        assert e.value.status == velo_cuda.ERR_INVALID_ARGUMENT
    refused(lambda: dctx.decode_attention(cache, q[:, :3], n, q[:, :3].contiguous(), ws))   # 3 heads over 2
    refused(lambda: dctx.decode_attention(cache, q.float(), n, q, ws))
    refused(lambda: dctx.decode_attention(cache, q, n.long(), q, ws))
    refused(lambda: dctx.decode_attention(cache, q, n, q, ws[:8]))
    refused(lambda: dctx.decode_attention(cache, q, n, q, ws, scale=float("nan")))
    refused(lambda: dctx.decode_attention(cache, q, n, q, ws, scale=-1.0))
    refused(lambda: dctx.decode_attention(cache, q.cpu(), n, q, ws))
    refused(lambda: dctx.decode_attention(cache, q.transpose(1, 2).contiguous().transpose(1, 2), n, q, ws))
    refused(lambda: dctx.decode_attention(cache, torch.zeros(2, 4, 128, dtype=torch.float16, device="cuda"),
                                          torch.ones(2, dtype=torch.int32, device="cuda"),
                                          torch.zeros(2, 4, 128, dtype=torch.float16, device="cuda"), ws))  # one table row
    odd = torch.zeros(4 * 128 + 4, dtype=torch.float16, device="cuda")[4:].view(1, 4, 128)
    refused(lambda: dctx.decode_attention(cache, odd, n, q, ws))                            # 8-byte aligned
    refused(lambda: dctx.decode_attention_workspace(3, 2, 128))
    refused(lambda: dctx.decode_attention_workspace(4, 2, 96))
    refused(lambda: velo_cuda.KvCache(_dev(d["k"]), _dev(d["v"]), _dev(d["table"]).long()))
    refused(lambda: velo_cuda.KvCache(_dev(d["k"]), _dev(d["v"][:1]), _dev(d["table"])))
    ints = torch.zeros(d["k"].shape, dtype=torch.int8, device="cuda")
    refused(lambda: velo_cuda.KvCache(ints, ints, _dev(d["table"])))                        # no scales
    wide = velo_cuda.KvCache(torch.zeros(2, 2, 16, 96, dtype=torch.float16, device="cuda"),
                             torch.zeros(2, 2, 16, 96, dtype=torch.float16, device="cuda"), _dev(d["table"]))
    q96 = torch.zeros(1, 4, 96, dtype=torch.float16, device="cuda")
    refused(lambda: dctx.decode_attention(wide, q96, n, q96, ws))
    dctx.decode_attention(cache, q[:0], n[:0], q[:0], ws)                                   # B = 0: nothing to do
    dctx.sync()


def test_attention_other_stream_and_graph(dctx):
    """A side stream; two captured calls with a workspace each, replayed after
    their inputs changed."""
    import torch
    rng = np.random.default_rng(9)
    lens = [700, 33]
    d = _cache(rng, "f16", lens, 2, 128)
    q = rng.normal(0, 1, (2, 8, 128)).astype(np.float16)
    cache = _kv_cache(d)
    want = _attend(dctx, d, q, lens, cache=cache)
    qd, nd = _dev(q), _dev(np.asarray(lens, np.int32))
    torch.cuda.synchronize()
    size = dctx.decode_attention_workspace(8, 2, 128)
    runs = []
    for _ in range(2):
        out, ls = torch.zeros_like(qd), torch.zeros(2, 8, device="cuda")
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            dctx.set_stream(torch.cuda.current_stream().cuda_stream)
            dctx.decode_attention(cache, qd, nd, out, ws, lse=ls)
        runs.append((g, out, ls, ws))
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(3):
        for (g, *_), s in zip(runs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out, ls, _ in runs:
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(ls.cpu().numpy(), want[1])
    nd.copy_(_dev(np.asarray([1, 650], np.int32)))  # the same graph, other lengths
    d2 = _cache(np.random.default_rng(9), "f16", [700, 700], 2, 128)
    for t, k in zip(cache.tensors, ("k", "v", "table")):
        assert t.shape[0] <= d2[k].shape[0]
    nd.copy_(_dev(np.asarray([17, 0], np.int32)))
    runs[0][0].replay()
    torch.cuda.synchronize()
    _check_attention(runs[0][1].cpu().numpy(), runs[0][2].cpu().numpy(), q, d, [17, 0], "f16")
    dctx.set_stream(velo_cuda.DEFAULT_STREAM)


def test_structs_of_another_size_are_refused(dctx):
    import ctypes

    import torch
    z = torch.zeros(1, 1, 16, 64, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    L, bad = velo_cuda.lib(), velo_cuda.ERR_INVALID_ARGUMENT
    batch = ctypes.create_string_buffer(velo_cuda._APPEND.size)
    assert L.velo_cuda_kv_append(dctx.handle, cache.ref, ctypes.byref(batch)) == bad and "struct_size" in velo_cuda.last_error()
    assert L.velo_cuda_kv_append(dctx.handle, cache.ref, None) == bad
    assert L.velo_cuda_kv_append(dctx.handle, None, ctypes.byref(batch)) == bad
    for field, value in (("struct_size", 8), ("kv_dtype", 3), ("head_dim", 96), ("n_kv", 0), ("pool_pages", 0), ("max_pages", -1),
                         ("max_pages", (1 << 26) + 1), ("k_pool", None), ("page_table", None)):
        d = velo_cuda.KvCacheDesc.from_buffer_copy(cache.desc)
        setattr(d, field, value)
        assert L.velo_cuda_decode_attention(dctx.handle, ctypes.byref(d), None, 0, None, 1, 1, 0.0, None, None, None, 0) == bad
    assert L.velo_cuda_decode_attention(dctx.handle, cache.ref, None, 64, None, 5000, 1, 0.0, None, None, None, 0) == bad


def test_counts_whose_product_passes_64_bits_are_refused(dctx):
    """4096 sequences x 2^30 heads x 2 x 2^21 pages is 2^64: the heads are refused
    before any product is formed."""
    import ctypes

    import torch
    z = torch.zeros(1, 1, 16, 64, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    L, bad = velo_cuda.lib(), velo_cuda.ERR_INVALID_ARGUMENT
    d = velo_cuda.KvCacheDesc.from_buffer_copy(cache.desc)
    d.max_pages = 1 << 21
    assert L.velo_cuda_decode_attention(dctx.handle, ctypes.byref(d), None, 64, None, 4096, 1 << 30, 0.0, None, None,
                                        None, 0) == bad
    assert "n_head" in velo_cuda.last_error()
    d.n_kv = 1 << 30
    assert L.velo_cuda_decode_attention(dctx.handle, ctypes.byref(d), None, 64, None, 1, 1 << 30, 0.0, None, None,
                                        None, 0) == bad
    assert "n_kv" in velo_cuda.last_error()
    assert L.velo_cuda_decode_attention_workspace(dctx.handle, 1 << 30, 1, 64) == 0


# ------------------------------------------------------------------ append

def _np_elem(rng, shape, src):
    """Random rows as `src` holds them: (torch tensor, f32 values)."""
    import torch
    t = torch.from_numpy(rng.normal(0, 1, shape).astype(np.float32))
    t = t.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[src])
    return t.cuda(), t.float().numpy()


APPEND = [
    # cached, new, Hq, Hkv, D, base
    ([0], [1], 4, 4, 64, 10000.0),
    ([15, 16, 0, 130999], [1, 1, 1, 1], 64, 8, 128, 500000.0),
    ([0, 5, 31], [33, 0, 17], 8, 2, 128, 10000.0),
    ([3, 100, 0, 7], [0, 0, 40, 0], 5, 1, 64, 10000.0),
    ([2 * i % 50 for i in range(300)], [i % 4 for i in range(300)], 2, 1, 64, 10000.0),
    ([1048000], [30], 12, 12, 128, 10000.0),
]


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv", ["f16", "int8", "f32"])
@pytest.mark.parametrize("cached,new,Hq,Hkv,D,base", APPEND)
def test_append_matches_plain(dctx, kv, src, cached, new, Hq, Hkv, D, base):
    import torch
    rng = np.random.default_rng(len(cached) * 10 + Hq)
    B, T, pad = len(cached), sum(new), 3
    # only the pages that receive tokens exist: the table names them at their places
    width = max(-(-(a + b) // 16) for a, b in zip(cached, new)) + 1
    table, at = np.full((B, width), -1, np.int64), 0
    for b in range(B):
        if new[b]:
            lo, hi = cached[b] // 16, (cached[b] + new[b] - 1) // 16
            table[b, lo:hi + 1] = np.arange(at, at + hi + 1 - lo)
            at += hi + 1 - lo
    pages = at + 2
    perm = rng.permutation(pages)
    table = np.where(table < 0, pages + 1, perm[np.maximum(table, 0)]).astype(np.int32)
    dt = {"f16": np.float16, "int8": np.int8, "f32": np.float32}[kv]
    act = np.float32 if kv == "f32" else np.float16
    pools = {n: rng.integers(-100, 100, (pages, Hkv, 16, D)).astype(dt) for n in "kv"}
    scales = {n: rng.random((pages, Hkv, 16)).astype(np.float16) if kv == "int8" else None for n in "kv"}
    cache = velo_cuda.KvCache(_dev(pools["k"]), _dev(pools["v"]), _dev(table),
                              *(None if scales[n] is None else _dev(scales[n]) for n in "kv"))
    qkv, x = _np_elem(rng, (T + pad, Hq + 2 * Hkv, D), src)
    q, k, v = x[:T, :Hq], x[:T, Hq:Hq + Hkv], x[:T, Hq + Hkv:]
    tact = torch.float32 if kv == "f32" else torch.float16
    q_out = torch.full((T + pad, Hq, D), 77.0, dtype=tact, device="cuda")
    k_out, v_out = (torch.full((T + pad, Hkv, D), 77.0, dtype=tact, device="cuda") for _ in range(2))
    start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    dctx.kv_append(cache, qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], _dev(np.asarray(cached, np.int32)), q_out,
                   base, seq_start=_dev(start), k_out=k_out, v_out=v_out)
    dctx.sync()
    seq = np.repeat(np.arange(B), new)
    pos = np.asarray(cached)[seq] + np.arange(T) - start[seq]
    # an angle is off by pos 2^-64 and its f32 remainder (2^-24 of half a turn) and sincospi by
    # about 2^-22 together; two products and a sum follow
    slack = 2.0 ** -21
    got_q = q_out.cpu().numpy()
    want = ref.rotate(q, pos, base)
    size = np.abs(q).max(initial=0)
    assert (np.abs(got_q[:T] - want) <= _half_step(want, kv != "f32") + 2 * slack * size).all()
    assert (got_q[T:] == 77).all() and (k_out[T:].cpu().numpy() == 77).all() and (v_out[T:].cpu().numpy() == 77).all()
    pg, sl = table[seq, pos // 16], pos % 16
    touched = np.zeros((pages, 16), bool)
    touched[pg, sl] = True
    for n, want, got_pool, got_scale, out in (("k", ref.rotate(k, pos, base), cache.tensors[0], cache.tensors[3], k_out),
                                              ("v", v.astype(np.float64), cache.tensors[1], cache.tensors[4], v_out)):
        got_pool, out = got_pool.cpu().numpy(), out[:T].cpu().numpy()
        rows = got_pool[pg, :, sl]
        same = np.moveaxis(got_pool, 2, 1)[~touched] == np.moveaxis(pools[n], 2, 1)[~touched]
        assert same.all()  # other slots are left as they were
        err = 2 * slack * np.abs(want).max(initial=0) if n == "k" else 0.0
        if kv == "int8":
            sc = got_scale.cpu().numpy()
            assert np.array_equal(np.moveaxis(sc, 2, 1)[~touched], np.moveaxis(scales[n], 2, 1)[~touched])
            s = sc[pg, :, sl].astype(np.float64)
            m = np.abs(want).max(-1)
            assert (np.abs(s - m / 127) <= _half_step(m / 127, True) + err / 127).all()
            y = want * (127 / m)[..., None]
            off = 127 * (err / m)[..., None] * 2 + 127 * 4 * EPS
            sure = np.abs(y - np.rint(y)) > off  # not at the edge of a step
            assert (rows == np.trunc(y))[sure].all() and (np.abs(rows - y) <= 1 + off).all()
            assert np.array_equal(out, (rows.astype(np.float32) * s[..., None].astype(np.float32)).astype(act))
        else:
            assert (np.abs(rows - want) <= _half_step(want, kv != "f32") + err).all()
            assert np.array_equal(out, rows)


def test_append_one_token_each_without_starts(dctx):
    import torch
    rng = np.random.default_rng(11)
    for B in (1, 5, 300):
        table = np.arange(B * 2).reshape(B, 2).astype(np.int32)
        cached = (np.arange(B) * 3 % 32).astype(np.int32)
        k, v = rng.normal(0, 1, (2, B, 2, 64)).astype(np.float32)
        res = []
        for start in (None, _dev(np.arange(B + 1, dtype=np.int32))):
            cache = velo_cuda.KvCache(torch.zeros(B * 2, 2, 16, 64, device="cuda"),
                                      torch.zeros(B * 2, 2, 16, 64, device="cuda"), _dev(table))
            dctx.kv_append(cache, None, _dev(k), _dev(v), _dev(cached), None, 10000.0, seq_start=start)
            dctx.sync()
            res.append([t.cpu().numpy() for t in cache.tensors[:2]])
        assert np.array_equal(res[0][0], res[1][0]) and np.array_equal(res[0][1], res[1][1])
        assert np.array_equal(res[0][1][table[np.arange(B), cached // 16], :, cached % 16], v)


def test_append_equals_write_kv_quantiser(dctx):
    """INT8 rows of f16 V quantise to the bytes velo_cuda_write_kv stores."""
    import torch

    import vo
    rng = np.random.default_rng(12)
    T, H, D = 40, 2, 128
    v = rng.normal(0, 1, (T, H, D)).astype(np.float16)
    v[3, 1] = 0  # an all-zero row: scale 0
    z = torch.zeros(3, H, 16, D, dtype=torch.int8, device="cuda")
    sc = torch.zeros(3, H, 16, dtype=torch.float16, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3), sc, sc.clone())
    dctx.kv_append(cache, None, _dev(v), _dev(v), _dev(np.zeros(1, np.int32)), None, 10000.0,
                   seq_start=_dev(np.asarray([0, T], np.int32)))
    dctx.sync()
    m = np.abs(v.astype(np.float32)).max(-1)
    inv = np.where(m > 0, np.float32(127) / np.where(m > 0, m, 1), 0).astype(np.float32)
    want = np.trunc(v.astype(np.float32) * inv[..., None]).astype(np.int8)
    got = np.moveaxis(cache.tensors[1].cpu().numpy(), 1, 2).reshape(-1, H, D)[:T]
    gs = np.moveaxis(cache.tensors[4].cpu().numpy(), 1, 2).reshape(-1, H)[:T]
    assert np.array_equal(got, want)
    assert np.array_equal(gs, (m / np.float32(127)).astype(np.float16))
    assert vo is not None


def test_append_flags_bad_places(dctx):
    import torch
    rng = np.random.default_rng(13)
    k = _dev(rng.normal(0, 1, (3, 1, 64)).astype(np.float32))

    def run(table, cached, start=None):
        cache = velo_cuda.KvCache(torch.zeros(4, 1, 16, 64, device="cuda"), torch.zeros(4, 1, 16, 64, device="cuda"),
                                  _dev(np.asarray(table, np.int32)))
        with pytest.raises(velo_cuda.VeloError) as e:
            dctx.kv_append(cache, None, k, k, _dev(np.asarray(cached, np.int32)), None, 10000.0,
                           seq_start=None if start is None else _dev(np.asarray(start, np.int32)))
            dctx.sync()
        assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
        return cache.tensors[0].cpu().numpy()
    pool = run([[0], [4], [2]], [0, 0, 15])           # page 4 lies outside the pool
    assert pool[0, 0, 0].any() and pool[2, 0, 15].any() and not pool[3].any()
    pool = run([[0], [1], [2]], [0, 16, 3])           # past the row
    assert not pool[1].any()
    pool = run([[0], [1], [2]], [0, -1, 3])
    assert not pool[1].any()
    pool = run([[0], [1]], [0, 0], [1, 2, 3])         # token 0 belongs to no sequence
    assert pool[0, 0, 0].any() and pool[1, 0, 0].any() and not pool[0, 0, 1:].any()
    pool = run([[0]], [5], [-2 ** 31, 3])             # a start far below zero puts every token past the row
    assert not pool.any()


def test_append_many_sequences_and_tiny_rows(dctx):
    """More sequences than a block has threads (the two-level search), empty ones
    among them; INT8 rows of zeros and of subnormal values."""
    import torch
    rng = np.random.default_rng(14)
    B = 3000
    new = rng.integers(0, 3, B)
    cached = rng.integers(0, 14, B).astype(np.int32)
    T = int(new.sum())
    start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    v = rng.normal(0, 1, (T, 1, 64)).astype(np.float32)
    v[::7] = 0
    v[3::7] *= np.float32(1e-41)
    table = rng.permutation(B).reshape(B, 1).astype(np.int32)
    seq = np.repeat(np.arange(B), new)
    sl = cached[seq] + np.arange(T) - start[seq]
    for kv in ("f32", "int8"):
        dt = torch.float32 if kv == "f32" else torch.int8
        sc = [torch.zeros(B, 1, 16, dtype=torch.float16, device="cuda") for _ in range(2)] if kv == "int8" else [None] * 2
        cache = velo_cuda.KvCache(torch.zeros(B, 1, 16, 64, dtype=dt, device="cuda"),
                                  torch.zeros(B, 1, 16, 64, dtype=dt, device="cuda"), _dev(table), *sc)
        dctx.kv_append(cache, None, _dev(v), _dev(v), _dev(cached), None, 10000.0, seq_start=_dev(start))
        dctx.sync()
        got = cache.tensors[1].cpu().numpy()[table[seq, 0], 0, sl].astype(np.float64)
        if kv == "f32":
            assert np.array_equal(got, v[:, 0].astype(np.float64))
        else:
            s = sc[1].cpu().numpy()[table[seq, 0], 0, sl].astype(np.float64)
            m = np.abs(v[:, 0]).max(-1).astype(np.float64)
            assert np.isfinite(s).all() and (np.abs(s - m / 127) <= _half_step(m / 127, True)).all()
            assert (np.abs(got * s[:, None] - v[:, 0]) <= m[:, None] / 127 * 1.001 + np.abs(v[:, 0]) * 2.0 ** -10 + 2.0 ** -18).all()


def test_append_refusals(dctx):
    import torch
    z = torch.zeros(2, 2, 16, 64, device="cuda")
    cache = velo_cuda.KvCache(z, z.clone(), torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    k = torch.zeros(2, 2, 64, device="cuda")
    q, qo = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")

    def refused(*a, **kw):
        with pytest.raises(velo_cuda.VeloError) as e:
            dctx.kv_append(*a, **kw)
        assert e.value.status == velo_cuda.ERR_INVALID_ARGUMENT
    refused(cache, q, k, k, n, qo, 1.0)
    refused(cache, q, k, k, n, qo, float("inf"))
    refused(cache, q, k, k, n, None, 1e4)
    refused(cache, q, k, k.half(), n, qo, 1e4)
    refused(cache, q.half(), k, k, n, qo, 1e4)
    refused(cache, q[:, :3], k, k, n, qo[:, :3].contiguous(), 1e4)
    refused(cache, q, k, k, n, qo.half(), 1e4)
    refused(cache, q, k[:1], k, n, qo, 1e4)
    refused(cache, q[:1], k[:1], k[:1], n, qo[:1], 1e4)          # one token, two sequences, no starts
    refused(cache, q, k, k, n, qo, 1e4, seq_start=n)             # needs 3 starts
    refused(cache, q, k, k, n, qo, 1e4, k_out=torch.zeros_like(k))
    refused(cache, q, k, k, torch.zeros(3, dtype=torch.int32, device="cuda"), qo, 1e4)
    wide = torch.zeros(2, 2 * 64 + 2, device="cuda")[:, :128].unflatten(1, (2, 64))
    refused(cache, q, wide, k, n, qo, 1e4)                       # row stride of 8 bytes modulo 16
    dctx.kv_append(cache, q[:0], k[:0], k[:0], n[:0], qo[:0], 1e4)
    dctx.sync()


# ------------------------------------------------------------------ log probabilities

def _logits(rng, M, V, src, spread=2.5):
    import torch
    t = torch.from_numpy((rng.normal(0, spread, (M, V))).astype(np.float32))
    t = t.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[src])
    return t


def _score(ctx, t, tokens, n, T, dev=None):
    import torch
    M = t.shape[0]
    lp, ent = (torch.full((M,), 55.0, device="cuda") for _ in range(2))
    ids = torch.full((M, n), -5, dtype=torch.int32, device="cuda")
    tlp = torch.full((M, n), 55.0, device="cuda")
    ctx.token_logprobs(t.cuda() if dev is None else dev, _dev(np.asarray(tokens, np.int32)), lp, ent, ids if n else None,
                       tlp if n else None, temperature=T)
    ctx.sync()
    return [a.cpu().numpy() for a in (lp, ent, ids, tlp)]


def _check_logprobs(got, x, tokens, n, T):
    lp, ent, ids, tlp = ref.logprobs(x, tokens, n, T)
    V = x.shape[1]
    fin = np.where(np.isfinite(x), np.abs(x), 0).max(-1).astype(np.float64) / T
    # sums of exponentials: chains of V / 256 + 64 additions; an argument x / T - m: three
    # roundings of its size; the exponential itself 2^-21
    chain = (V / 256 + 64) * EPS + 2.0 ** -20
    tol = chain + 8 * EPS * (1 + 2 * fin)
    spread = 2 + np.log(V)

    def near(a, b, t):
        ok = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and (a[~ok & ~np.isnan(b)] == b[~ok & ~np.isnan(b)]).all()
        t = np.broadcast_to(t, b.shape)
        err = np.abs(a[ok] - b[ok])
        assert (err <= t[ok]).all(), (err / t[ok]).max()
    near(got[0], lp, tol)
    near(got[1], ent, tol * spread)
    if n:
        assert np.array_equal(got[2].astype(np.int64), ids)
        near(got[3], tlp, tol[:, None])


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,V,n,T", [(1, 1, 1, 1.0), (3, 5, 5, 0.5), (2, 64, 64, 1.0), (7, 1000, 20, 0.8), (1, 128256, 5, 1.0),
                                     (33, 32000, 8, 1.0), (5, 50257, 20, 0.7), (300, 4096, 3, 1.0), (2, 131071, 33, 1.3),
                                     (700, 2049, 0, 1.0), (2, 1 << 20, 20, 1.0), (5000, 33, 20, 1.0),
                                     (700, 4093, 33, 0.9), (20, 70001, 20, 1.0), (34, 65600, 64, 0.9),
                                     (100, 20001, 20, 1.0)])
def test_logprobs_match_plain(dctx, src, M, V, n, T):
    rng = np.random.default_rng(M * 7 + V)
    t = _logits(rng, M, V, src)
    tokens = rng.integers(0, V, M)
    got = _score(dctx, t, tokens, n, T)
    _check_logprobs(got, t.float().numpy(), tokens, n, T)
    again = _score(dctx, t, tokens, n, T)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(got, again))


@pytest.mark.parametrize("V,copies", [(20011, 1), (4001, 40), (20011, 5), (66001, 2)])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
def test_logprobs_hard_rows(dctx, src, V, copies):
    """Masked, tied, ordered and non-finite rows, each among ordinary ones; many
    copies of them take the smaller blocks, a few the deeper ring of clusters of 2 and 4."""
    import torch
    n = 20
    rng = np.random.default_rng(21)
    x = rng.normal(0, 2, (17, V)).astype(np.float32)
    x[0] = -np.inf                                  # nothing left
    x[1, :] = -np.inf
    x[1, V // 3] = 3                                # one survivor
    x[2, 5:] = -np.inf                              # fewer than n survivors
    x[3] = 0                                        # all equal: the lowest indices
    x[4] = np.arange(V) * 1e-3                      # rising: every element beats all before
    x[5] = -np.arange(V) * 1e-3
    x[6] = np.rint(x[6])                            # many ties
    x[7, 100] = np.nan
    x[8, V - 12] = np.inf
    x[9] = np.nan
    x[10, ::2] = -0.0
    x[10, 1::2] = 0.0                               # -0 and 0 are equal
    x[11] = -60000                                  # the lowest values as a mask
    x[11, 11::1000] = 1
    x[12] = 0
    x[12, V // 2:V // 2 + 64] = 5                   # the best lie side by side (one thread's loads)
    x[13] = 0
    x[13, 3::256] = 9                               # ... and one to a stride
    x[14, :] = np.where(np.arange(V) % 1024 < 4, 8 + x[14], x[14] - 8)
    x[15] = np.float32(30000)                       # large and equal
    if src == "f32":
        x[16] = -3e38
        x[16, 5] = -2.9e38
    t = torch.from_numpy(x).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[src])
    tokens = np.arange(17) * 1000 % V
    tokens[1] = V // 3
    got = _score(dctx, t.repeat(copies, 1), np.tile(tokens, copies), n, 1.0)
    for c in range(copies):  # (an odd V: the copies start at different offsets, so sums may group differently)
        _check_logprobs([g[c * 17:(c + 1) * 17] for g in got], t.float().numpy(), tokens, n, 1.0)
    for i in range(17 if copies == 1 else 0):  # one row alone takes the other split of the work
        one = _score(dctx, t[i:i + 1], tokens[i:i + 1], n, 1.0)
        _check_logprobs(one, t[i:i + 1].float().numpy(), tokens[i:i + 1], n, 1.0)


def test_logprobs_entropy_of_peaked_rows(dctx):
    """A token that is nearly certain, wherever it lies: ln Z and Y / Z are both
    near 0 when measured from it, so the small entropy keeps its digits."""
    import torch
    rng = np.random.default_rng(25)
    V = 50021
    x = rng.normal(0, 1, (24, V)).astype(np.float32)
    for i in range(24):
        x[i, int(rng.integers(0, V))] = [12, 15, 20, 30][i % 4]
    tokens = x.argmax(-1)
    for rows in (slice(0, 24), slice(3, 4)):
        got = _score(dctx, torch.from_numpy(x[rows]), tokens[rows], 3, 1.0)
        lp, ent, _, _ = ref.logprobs(x[rows], tokens[rows], 3, 1.0)
        # the peak's thread adds a sum per 16 elements and its neighbours' to 1: (V / 4096 + 32)
        # roundings of 2^-25; the other terms keep 2^-17 of themselves
        tol = (V / 4096 + 32) * 2.0 ** -25
        assert (np.abs(got[0] - lp) <= np.abs(lp) * 2.0 ** -17 + tol).all()
        assert (np.abs(got[1] - ent) <= ent * 2.0 ** -17 + 2 * tol).all()


@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("pad,shift", [(3, 0), (8, 0), (5, 1), (16, 4)])
def test_logprobs_strides_and_alignment(dctx, src, pad, shift):
    import torch
    rng = np.random.default_rng(22)
    M, V = 9, 5003
    t = _logits(rng, M, V, src)
    wide = torch.full((M, V + pad), float("nan"), dtype=t.dtype, device="cuda")
    view = wide[:, shift:shift + V] if shift + V <= V + pad else wide[:, :V]
    view.copy_(t)
    tokens = rng.integers(0, V, M)
    got = _score(dctx, t, tokens, 6, 1.0, dev=view)
    _check_logprobs(got, t.float().numpy(), tokens, 6, 1.0)


def test_logprobs_flags_bad_token(dctx):
    import torch
    t = torch.zeros(3, 100, device="cuda")
    lp = torch.zeros(3, device="cuda")
    dctx.token_logprobs(t, _dev(np.asarray([1, 100, -1], np.int32)), lp)
    with pytest.raises(velo_cuda.VeloError) as e:
        dctx.sync()
    assert e.value.status == velo_cuda.ERR_DEVICE_FLAG
    got = lp.cpu().numpy()
    assert abs(got[0] + np.log(100)) < 1e-5 and np.isnan(got[1:]).all()


def test_logprobs_refusals(dctx):
    import torch
    t, tok, lp = torch.zeros(2, 100, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(
        2, device="cuda")
    ids, tl = torch.zeros(2, 65, dtype=torch.int32, device="cuda"), torch.zeros(2, 65, device="cuda")

    def refused(*a, **kw):
        with pytest.raises(velo_cuda.VeloError) as e:
            dctx.token_logprobs(*a, **kw)
        assert e.value.status == velo_cuda.ERR_INVALID_ARGUMENT
    refused(t, tok, lp, temperature=0.0)
    refused(t, tok, lp, temperature=float("inf"))
    refused(t, tok, lp, temperature=1e-45)
    refused(t, tok, lp, None, ids, tl)                      # n_top 65
    refused(t[:, :3], tok, lp, None, ids[:, :4].contiguous(), tl[:, :4].contiguous())
    refused(t, tok, lp, None, ids[:, :4].contiguous())
    refused(t, tok, None)
    refused(t, None, lp)
    refused(t.double(), tok, lp)
    refused(t, tok.long(), lp)
    refused(t.T.contiguous().T, tok, lp)
    refused(t, tok[:1], lp)
    refused(t.cpu(), tok, lp)
    dctx.token_logprobs(t[:0], tok[:0], lp[:0])
    dctx.token_logprobs(t, None, None)
    dctx.sync()


def test_logprobs_sampling_temperature_is_the_accept_distribution(dctx):
    """top_logprobs with every token of a small vocabulary add up to one."""
    import torch
    t = _logits(np.random.default_rng(23), 4, 50, "f32").cuda()
    ids, tl = torch.zeros(4, 50, dtype=torch.int32, device="cuda"), torch.zeros(4, 50, device="cuda")
    dctx.token_logprobs(t, None, None, None, ids, tl, temperature=0.8)
    dctx.sync()
    want = torch.log_softmax(t.double() / 0.8, -1).gather(1, ids.long())
    assert (tl.double() - want).abs().max() < 1e-5
    assert torch.equal(ids.long().sort(-1).values, torch.arange(50, device="cuda").expand(4, 50))


# ------------------------------------------------------------------ order on streams

def test_calls_wait_for_what_precedes_them(dctx):
    """The operators start as dependents of the kernel before them: they still see
    copies, clears, other streams' work and each other's results."""
    import torch
    rng = np.random.default_rng(41)
    B, H, D, V = 4, 2, 64, 70000
    table = torch.arange(B * 4, dtype=torch.int32, device="cuda").view(B, 4)
    cache = velo_cuda.KvCache(torch.zeros(B * 4, H, 16, D, device="cuda"), torch.zeros(B * 4, H, 16, D, device="cuda"), table)
    src = [_dev(rng.normal(0, 1, (B, 3 * H, D)).astype(np.float32)) for _ in range(3)]
    x, q = torch.empty_like(src[0]), torch.empty(B, H, D, device="cuda")
    out, ws = torch.empty_like(q), torch.empty(dctx.decode_attention_workspace(H, H, D), dtype=torch.uint8, device="cuda")
    pos, lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    logits, lp = torch.zeros(B, V, device="cuda"), torch.empty(B, device="cuda")
    tok = torch.zeros(B, dtype=torch.int32, device="cuda")
    big = torch.zeros(1 << 26, device="cuda")
    main, side = torch.cuda.Stream(), torch.cuda.Stream()

    def step(i, n):
        with torch.cuda.stream(side):
            side.wait_stream(main)
            big.add_(1.0)                       # a slow kernel before the rows are ready
            x.copy_(src[i])
        main.wait_stream(side)
        dctx.kv_append(cache, x[:, :H], x[:, H:2 * H], x[:, 2 * H:], pos, q, 10000.0)
        pos.add_(1)
        lens.copy_(pos)
        dctx.decode_attention(cache, q, lens, out, ws)
        logits.zero_()
        logits[:, :H * D].copy_(out.view(B, -1))
        dctx.token_logprobs(logits, tok, lp)
        return lp.clone(), out.clone()
    results = []
    for rounds in range(3):
        with torch.cuda.stream(main):
            dctx.set_stream(main.cuda_stream)
            pos.zero_()
            got = [step(i % 3, i) for i in range(20)]
        torch.cuda.synchronize()
        results.append(torch.cat([t.flatten() for r in got for t in r]).cpu())
    dctx.sync()
    assert all(torch.equal(r, results[0]) for r in results)
    last = results[0][-B * H * D:].view(B, H, D).numpy()
    # the last step against 64 bits, over the twenty cached rows
    k, v = cache.tensors[0].cpu().numpy(), cache.tensors[1].cpu().numpy()
    want, _, _, vmax = ref.attention(q.cpu().numpy(), k, v, table.cpu().numpy(), [20] * B)
    assert np.abs(last - want).max() <= 1e-5 * vmax
    rows = np.stack([src[i % 3].cpu().numpy()[:, 2 * H:] for i in range(20)], 1)  # [B][20][H][D]
    assert np.array_equal(np.moveaxis(v[table.cpu().numpy()], 3, 2).reshape(B, -1, H, D)[:, :20], rows)
    # the same chain captured: a clear, a copy and the operators as graph nodes
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dctx.set_stream(torch.cuda.current_stream().cuda_stream)
        pos.zero_()
        x.zero_()
        x.copy_(src[1])
        dctx.kv_append(cache, x[:, :H], x[:, H:2 * H], x[:, 2 * H:], pos, q, 10000.0)
        lens.copy_(pos).add_(1)
        dctx.decode_attention(cache, q, lens, out, ws)
    dctx.set_stream(velo_cuda.DEFAULT_STREAM)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        # one cached token: the output is its V row
        assert torch.equal(out, src[1][:, 2 * H:])


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("kv,Hq,Hkv,D", [("f16", 8, 2, 128), ("int8", 8, 8, 64), ("f32", 4, 1, 64)])
def test_decode_steps_together(dctx, kv, Hq, Hkv, D):
    """A prefill chunk and six decode steps of one layer as a server runs them,
    the steps replayed from one captured graph: append, attend, logits, scores;
    every step against 64-bit attention over the cached rows."""
    import torch
    rng = np.random.default_rng(31)
    B, V, steps, prompt = 3, 1000, 6, [30, 1, 15]
    act = torch.float32 if kv == "f32" else torch.float16
    pages, width = 12, 4
    table = rng.permutation(pages).reshape(B, width).astype(np.int32)
    dt = {"f16": torch.float16, "int8": torch.int8, "f32": torch.float32}[kv]
    sc = [torch.zeros(pages, Hkv, 16, dtype=torch.float16, device="cuda") for _ in range(2)] if kv == "int8" else [None] * 2
    cache = velo_cuda.KvCache(torch.zeros(pages, Hkv, 16, D, dtype=dt, device="cuda"),
                              torch.zeros(pages, Hkv, 16, D, dtype=dt, device="cuda"), _dev(table), *sc)
    heads = Hq + 2 * Hkv

    def cut(x):
        return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    T = sum(prompt)
    start = np.concatenate(([0], np.cumsum(prompt))).astype(np.int32)
    rows = torch.from_numpy(rng.normal(0, 1, (T, heads, D)).astype(np.float32)).cuda()
    q_pre = torch.empty(T, Hq, D, dtype=act, device="cuda")
    k_all, v_all = (torch.empty(T, Hkv, D, dtype=act, device="cuda") for _ in range(2))
    dctx.kv_append(cache, *cut(rows), _dev(np.zeros(B, np.int32)), q_pre, 10000.0, seq_start=_dev(start), k_out=k_all,
                   v_out=v_all)
    ks = [[k_all[start[b]:start[b + 1]].cpu().numpy()] for b in range(B)]
    vs = [[v_all[start[b]:start[b + 1]].cpu().numpy()] for b in range(B)]
    # one step's buffers and its graph
    x = torch.zeros(B, heads, D, device="cuda")
    cached = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    lens = cached + 1
    q = torch.empty(B, Hq, D, dtype=act, device="cuda")
    k1, v1 = (torch.empty(B, Hkv, D, dtype=act, device="cuda") for _ in range(2))
    out = torch.empty(B, Hq, D, dtype=act, device="cuda")
    head = torch.from_numpy(rng.normal(0, 0.3, (Hq * D, V)).astype(np.float32)).cuda()
    tok = torch.zeros(B, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(B, device="cuda"), torch.empty(B, device="cuda")
    ids, tlp = torch.empty(B, 4, dtype=torch.int32, device="cuda"), torch.empty(B, 4, device="cuda")
    ws = torch.empty(dctx.decode_attention_workspace(Hq, Hkv, D), dtype=torch.uint8, device="cuda")
    logits = torch.empty(B, V, device="cuda")
    torch.mm(out.float().view(B, -1), head)  # cuBLAS is set up outside the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dctx.set_stream(torch.cuda.current_stream().cuda_stream)
        dctx.kv_append(cache, *cut(x), cached, q, 10000.0, k_out=k1, v_out=v1)
        dctx.decode_attention(cache, q, lens, out, ws)
        logits.copy_(torch.mm(out.float().view(B, -1), head))
        dctx.token_logprobs(logits, tok, lp, ent, ids, tlp)
        cached += 1
        lens += 1
    dctx.set_stream(velo_cuda.DEFAULT_STREAM)
    cached.copy_(torch.tensor(prompt))
    lens.copy_(cached + 1)
    for step in range(steps):
        x.copy_(torch.from_numpy(rng.normal(0, 1, (B, heads, D)).astype(np.float32)))
        tok.copy_(torch.from_numpy(rng.integers(0, V, B).astype(np.int32)))
        g.replay()
        torch.cuda.synchronize()
        qn = q.cpu().numpy().astype(np.float64)
        for b in range(B):
            ks[b].append(k1[b:b + 1].cpu().numpy())
            vs[b].append(v1[b:b + 1].cpu().numpy())
            k, v = np.concatenate(ks[b]).astype(np.float64), np.concatenate(vs[b]).astype(np.float64)
            for h in range(Hq):
                s = k[:, h // (Hq // Hkv)] @ qn[b, h] / np.sqrt(D)
                p = np.exp(s - s.max())
                want = (p / p.sum()) @ v[:, h // (Hq // Hkv)]
                # k_out of INT8 rows is q * scale rounded to f16 (2^-11), where the pages are not
                slack = {"f32": 1e-5, "f16": 2e-4, "int8": 2.0 ** -11 * (1 + 2 * np.abs(qn[b, h]).sum() / np.sqrt(D)) * 4}[kv]
                assert np.abs(out[b, h].cpu().numpy() - want).max() <= np.abs(want).max() * 2.0 ** -11 + slack * np.abs(v).max()
        _check_logprobs([t.cpu().numpy() for t in (lp, ent, ids, tlp)], logits.cpu().numpy(), tok.cpu().numpy(), 4, 1.0)
    assert cached.tolist() == [n + steps for n in prompt]
    dctx.sync()
