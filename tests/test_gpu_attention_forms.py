"""attention against its 64-bit form where the sizes call for other forms of the
kernels: 32 columns a wave at every width of the tiles, walks that are split at
256 and more column tiles, joins of thousands of rows."""
import math

import pytest
import torch

from token_helpers import TYPES, attention_64, within

pytestmark = pytest.mark.gpu


def _check(t, B, Hq, Hkv, Tq, Tk, D, causal=False, key_lengths=None, query_start=None):
    from blitzgs_amd.attention import attention
    g = torch.Generator(device="cuda").manual_seed(Tq + Tk + D)
    make = lambda T, H: torch.randn((B, T, H, D), generator=g, device="cuda").to(t).transpose(1, 2)  # noqa: E731
    q, k, v, do = make(Tq, Hq), make(Tk, Hkv), make(Tk, Hkv), make(Tq, Hq)
    if key_lengths is not None:
        key_lengths = torch.tensor(key_lengths, dtype=torch.int32, device="cuda")
        for b in range(B):
            k[b, :, int(key_lengths[b]):] = float("nan")
            v[b, :, int(key_lengths[b]):] = float("nan")
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = attention(*leaves, causal=causal, key_lengths=key_lengths, query_start=query_start)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    want = attention_64(q, k, v, causal, key_lengths, query_start, 1.0 / math.sqrt(D), do)
    for name in got:
        within(got[name], *want[name], name)
    with torch.no_grad():
        assert torch.equal(attention(q, k, v, causal=causal, key_lengths=key_lengths, query_start=query_start),
                           got["o"])


# 512 column tiles of 128 queries and of 128 keys, the last of them nearly empty
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [32, 40, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_wide_tiles(gpu, t, D, causal):
    _check(t, 16, 16, 16, 130, 137, D, causal)


@pytest.mark.parametrize("t", TYPES)
def test_wide_tiles_of_shared_heads(gpu, t):
    # a tile's columns are the queries of several heads
    _check(t, 32, 24, 8, 45, 70, 64, True, key_lengths=[(7 * b) % 71 for b in range(32)])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_long_unequal_walks_of_many_tiles(gpu, t, D):
    # 256 column tiles: only walks of 64 steps and more are cut, over keys and over queries
    _check(t, 2, 128, 128, 5, 4200, D, True, key_lengths=[4200, 2500])
    _check(t, 2, 128, 128, 4200, 5, D, True, key_lengths=[5, 3])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [33, 64, 128])
def test_joins_of_thousands_of_rows(gpu, t, D):
    # 8000 rows of 2 splits and more, one wave each
    _check(t, 2, 8, 2, 500, 700, D, True, key_lengths=[700, 333])
    _check(t, 2, 8, 2, 500, 700, D)
