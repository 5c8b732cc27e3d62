"""Host side of the one-token decode entry points: NULL contexts, argument
checks of the Python view, and the rotation's angle arithmetic."""
import numpy as np
import pytest

import velo_cuda


def test_null_context_is_refused():
    L = velo_cuda.lib()
    bad = velo_cuda.ERR_INVALID_ARGUMENT
    assert L.velo_cuda_kv_append(None, None, None, None, None, 0, 0, 0, 0, None, None, 1, 1, 1, 1e4, None, None, None) == bad
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
