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
from test_decode_gpu import EPS, _dev, dctx  # noqa: F401

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
