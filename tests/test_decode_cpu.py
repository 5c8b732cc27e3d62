"""Host side of the one-token decode entry points: NULL contexts, argument
checks of the Python view, and the rotation's angle arithmetic."""
import numpy as np
import pytest

import velo_cuda


def test_null_context_is_refused():
    L = velo_cuda.lib()
    bad = velo_cuda.ERR_INVALID_ARGUMENT
    assert L.velo_cuda_kv_append(None, None, None) == bad
    assert "NULL" in velo_cuda.last_error()
    assert L.velo_cuda_decode_attention(None, None, None, 0, None, 1, 1, 0.0, None, None, None, 0) == bad
    assert L.velo_cuda_token_logprobs(None, None, 0, 1, 1, 1, None, 1.0, None, None, 0, None, None) == bad
    assert L.velo_cuda_decode_attention_workspace(None, 8, 8, 128) == 0


def test_cache_view_refuses_wrong_tensors():
    import torch
    z = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    table = torch.zeros(1, 2, dtype=torch.int32)
    velo_cuda.KvCache(z, z, table)
    for bad in ((z[0], z, table), (z, z[:1], table), (z, z.float(), table), (z, z, table.long()), (z, z, table[0]),
                (z.transpose(0, 1).contiguous().transpose(0, 1), z, table), (z.to(torch.int8), z.to(torch.int8), table),
                (z.to(torch.bfloat16), z.to(torch.bfloat16), table), (z[:, :, :8], z[:, :, :8], table)):
        with pytest.raises(velo_cuda.VeloError) as e:
            velo_cuda.KvCache(*bad)
        assert e.value.status == velo_cuda.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("base,D", [(1e4, 128), (5e5, 128), (1e4, 64), (1.5, 64)])
def test_turn_fractions_keep_far_angles(base, D):
    """pos * f modulo 2^64, its upper 32 bits in f32 half turns: within 2^-23 of a
    half turn of the exact angle, 2^20 tokens into a context."""
    f = np.floor(np.ldexp(float(base) ** (-2.0 * np.arange(D // 2) / D) / (2 * np.pi), 64) + 0.5)
    assert (f < 2.0 ** 64).all()
    for pos in (0, 1, 4095, 131071, 1048576):
        for i in range(D // 2):
            t = (pos * int(f[i])) % 2 ** 64 >> 32
            half = np.float32(t - 2 ** 32 if t >= 2 ** 31 else t) * np.float32(2.0 ** -31)
            exact = np.longdouble(pos) * np.longdouble(base) ** (np.longdouble(-2 * i) / D) / np.longdouble(np.pi)
            off = (np.longdouble(half) - exact) % 2
            assert min(off, 2 - off) <= 2.0 ** -23


class _Share:
    """n units in k ranges, the first n % k with one more (decode_attn.cu)."""

    def __init__(self, n, k):
        self.n, self.k, self.q, self.r = n, k, n // k if k else 0, n % k if k else 0

    def at(self, c):
        return c * self.q + min(c, self.r)

    def range_of(self, u):
        head = self.r * (self.q + 1)
        return u // (self.q + 1) if u < head else self.r + (u - head) // self.q


def _ranges(units, per_seq, main, tail, least=4, share=12, tail_units=64, tail_states=24, join=24):
    """decode_attn.cu's cut of the unit list: per block its pieces (item, first,
    last + 1 unit of the item, units, slot of a partial piece), and the open item
    with its last block."""
    pre = np.concatenate(([0], np.cumsum(np.asarray(units) * per_seq)))
    total = int(pre[-1])
    n = min(main, -(-total // least))
    per = -(-int(np.count_nonzero(units)) * per_seq // n)
    uncut = 2 * (per * int(max(units)) - total // n) <= 3 * join or (per > 1 and max(units) <= 2 * join)
    if tail and total // main >= tail_units and max(units) <= tail_states * (total // share // tail):
        big, small = _Share(total - total // share, main), _Share(total // share, tail)
    else:
        big, small = _Share(total, n), _Share(0, 0)
    blocks = big.k + small.k

    def item(u):
        b = int(np.searchsorted(pre, u, "right")) - 1
        n = int(units[b])
        it = int(u - pre[b]) // n
        return (b, it), int(pre[b]) + it * n, n

    def cut(c):
        u = total if c >= blocks else big.at(c) if c <= big.k else big.n + small.at(c - big.k)
        if c == 0 or u >= total:
            return u
        _, start, n = item(u)
        return start if uncut or n <= max(join, (big.q if c <= big.k else small.q) // 4) else u

    def block_of(u):
        return big.range_of(u) if u < big.n else big.k + small.range_of(u - big.n)
    out = []
    for c in range(blocks):
        seg, u1 = cut(c), cut(c + 1)
        pieces, open_ = [], None
        while seg < u1:
            key, start, n = item(seg)
            end, stop = start + n, min(start + n, u1)
            full = seg == start and stop == end
            pieces.append((key, seg - start, stop - start, n, None if full else 2 * c + (seg == start)))
            if not full and seg == start:
                assert open_ is None
                open_ = (key, block_of(end - 1))
            seg = stop
        out.append((pieces, open_))
    return out


@pytest.mark.parametrize("seed", range(60))
def test_decode_work_list_covers_every_item_once(seed):
    """Every unit of every item is in exactly one block; an item cut between
    blocks is open in its first one, whose join reads slot 1 of that block and
    slot 0 of the following ones, each written once."""
    rng = np.random.default_rng(seed)
    B = int(rng.integers(1, 30))
    units = rng.integers(0, int(rng.choice([2, 20, 500, 3000])), B)
    if not units.any():
        units[0] = 1
    per_seq, main = int(rng.choice([1, 2, 8, 32])), int(rng.choice([1, 7, 296]))
    out = _ranges(units, per_seq, main, main * int(rng.choice([0, 1, 2])))
    got, written = {}, {}
    for pieces, _ in out:
        for key, lo, hi, n, slot in pieces:
            assert n == units[key[0]] and lo < hi
            got.setdefault(key, []).append((lo, hi))
            if slot is not None:
                assert slot not in written
                written[slot] = (key, lo)
    assert set(got) == {(b, i) for b in range(B) if units[b] for i in range(per_seq)}
    for key, parts in got.items():
        assert parts[0][0] == 0 and parts[-1][1] == units[key[0]]
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
    read = []
    for c, (_, open_) in enumerate(out):
        if open_:
            key, last = open_
            states = [2 * c + 1] + [2 * i for i in range(c + 1, last + 1)]
            assert [written.get(s, (None,))[0] for s in states] == [key] * len(states)
            assert [written[s][1] for s in states] == [p[0] for p in got[key]]
            read += states
    assert sorted(read) == sorted(written)
