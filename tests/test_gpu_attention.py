"""attention against its 64-bit form: every type, lengths from none to several
tiles, heads that share keys, masks that leave rows empty, what lies in masked
places, strides, single queries over long contexts; its refusals."""
import math

import pytest
import torch

from token_helpers import TYPES, attention_64, within

pytestmark = pytest.mark.gpu


def _inputs(t, B, Hq, Hkv, Tq, Tk, D, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * Tq + 31 * Tk + D)
    make = lambda T, H: (torch.randn((B, T, H, D), generator=g, device="cuda") * size).to(t).transpose(1, 2)  # noqa
    return make(Tq, Hq), make(Tk, Hkv), make(Tk, Hkv), make(Tq, Hq)


def _run(q, k, v, do=None, **how):
    from blitzgs_amd.attention import attention
    if do is None:
        return dict(o=attention(q, k, v, **how))
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = attention(*leaves, **how)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def _check(q, k, v, do, causal=False, key_lengths=None, query_start=None, scale=None):
    how = dict(causal=causal, key_lengths=key_lengths, query_start=query_start, scale=scale)
    got = _run(q, k, v, do, **how)
    want = attention_64(q, k, v, causal, key_lengths, query_start,
                        1.0 / math.sqrt(q.shape[3]) if scale is None else scale, do)
    for name in got:
        assert got[name].dtype == q.dtype
        within(got[name], *want[name], name)
    # without gradients: the same bits
    with torch.no_grad():
        assert torch.equal(_run(q, k, v, **how)["o"], got["o"])
    return got


def _int(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 2), (2, 1), (5, 64), (64, 65), (63, 129), (130, 17), (200, 300),
                                   (1, 700), (300, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(gpu, t, Tq, Tk, causal):
    q, k, v, do = _inputs(t, 2, 3, 3, Tq, Tk, 64)
    _check(q, k, v, do, causal=causal)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [1, 8, 31, 32, 40, 64, 72, 80, 96, 100, 127, 128])
def test_head_dimensions(gpu, t, D):
    q, k, v, do = _inputs(t, 1, 2, 1, 70, 140, D)
    _check(q, k, v, do, causal=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Hq,Hkv", [(4, 1), (6, 2), (5, 5), (10, 2)])
def test_shared_heads(gpu, t, Hq, Hkv):
    q, k, v, do = _inputs(t, 2, Hq, Hkv, 33, 150, 64)
    _check(q, k, v, do)
    _check(q, k, v, do, causal=True)


@pytest.mark.parametrize("t", TYPES)
def test_key_lengths_leave_rows_empty_and_padding_unread(gpu, t):
    B, Tq, Tk = 5, 70, 200
    q, k, v, do = _inputs(t, B, 4, 2, Tq, Tk, 64)
    lengths = _int(0, 1, 63, 200, 129)
    for b in range(B):
        k[b, :, int(lengths[b]):] = float("nan")
        v[b, :, int(lengths[b]):] = float("inf")
    got = _check(q, k, v, do, key_lengths=lengths)
    assert not got["o"][0].any() and not got["dq"][0].any()
    for b in range(B):
        assert not got["dk"][b, :, int(lengths[b]):].any() and not got["dv"][b, :, int(lengths[b]):].any()
    # the queries are each sequence's last ones: those before its start see nothing
    _check(q, k, v, do, causal=True, key_lengths=lengths, query_start=lengths - Tq)
    # and its first ones
    _check(q, k, v, do, causal=True, key_lengths=lengths, query_start=torch.zeros_like(lengths))


def test_lengths_out_of_range_are_clamped(gpu):
    q, k, v, do = _inputs(torch.bfloat16, 3, 2, 2, 20, 50, 32)
    _check(q, k, v, do, key_lengths=_int(-3, 51, 2 ** 31 - 1))
    _check(q, k, v, do, causal=True, query_start=_int(-2 ** 31, 2 ** 31 - 1, -5))


@pytest.mark.parametrize("t", TYPES)
def test_hidden_keys_hold_the_types_extremes(gpu, t):
    # a causally hidden key's score may be as large as the type allows
    q, k, v, do = _inputs(t, 1, 1, 1, 40, 40, 32)
    big = {torch.float32: 1e30, torch.bfloat16: 1e30, torch.float16: 6e4}[t]
    k[:, :, 30:] = big
    how = dict(causal=True)
    got = _run(q, k, v, **how)["o"][:, :, :30]
    want = attention_64(q[:, :, :30], k[:, :, :30], v[:, :, :30], True, None, None, 1 / math.sqrt(32))["o"]
    within(got, *want, "o")


def test_nan_in_a_query_stays_in_its_row(gpu):
    q, k, v, _ = _inputs(torch.bfloat16, 1, 2, 2, 100, 100, 64)
    clean = _run(q, k, v)["o"]
    q[0, 1, 37, 5] = float("nan")
    o = _run(q, k, v)["o"]
    assert torch.isnan(o[0, 1, 37]).all()
    o[0, 1, 37] = clean[0, 1, 37]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("t", TYPES)
def test_peaked_rows(gpu, t):
    # large scores: nearly all weight on one key, and rescalings between tiles
    q, k, v, do = _inputs(t, 1, 2, 2, 66, 260, 64, size=3.0)
    _check(q, k, v, do, scale=0.5)


@pytest.mark.parametrize("t", TYPES)
def test_strides_and_odd_addresses(gpu, t):
    g = torch.Generator(device="cuda").manual_seed(5)
    B, T, H, D = 2, 90, 3, 40
    fused = torch.randn((B, T, 3 * H * D + 1), generator=g, device="cuda").to(t)[..., 1:].view(B, T, 3, H, D)
    q, k, v = (fused[:, :, i].transpose(1, 2) for i in range(3))
    do = torch.randn((B, H, T, D), generator=g, device="cuda").to(t)
    _check(q, k, v, do)
    _check(q, k, v, torch.ones((1, 1, 1, 1), device="cuda", dtype=t).expand(B, H, T, D))
    turned = [torch.randn((B, H, D, T), generator=g, device="cuda").to(t).transpose(2, 3) for _ in range(3)]
    _check(*turned, do)
    # one key head seen by the whole batch
    shared = torch.randn((1, 1, T, D), generator=g, device="cuda").to(t).expand(B, H, T, D)
    _check(q, shared, v, do)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Hq,Hkv,Tq,Tk", [(8, 2, 1, 5000), (8, 8, 1, 3001), (16, 1, 1, 4097), (4, 2, 5, 2500),
                                          (20, 4, 4, 900), (2, 1, 1, 33)])
def test_few_queries_over_a_long_context(gpu, t, Hq, Hkv, Tq, Tk):
    B = 3
    q, k, v, do = _inputs(t, B, Hq, Hkv, Tq, Tk, 128)
    lengths = _int(Tk, 0, Tk * 2 // 3)
    k[1], v[1] = float("nan"), float("nan")
    _check(q, k, v, do, key_lengths=lengths)
    _check(q, k, v, do, causal=True, key_lengths=lengths, query_start=lengths - Tq)


@pytest.mark.parametrize("t", TYPES)
def test_many_queries_over_few_keys(gpu, t):
    # the keys' gradients are sums over a long axis
    q, k, v, do = _inputs(t, 1, 4, 2, 3000, 40, 64)
    _check(q, k, v, do)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_many_blocks(gpu, t):
    # enough column tiles for the wide form of every kernel
    q, k, v, do = _inputs(t, 16, 16, 16, 130, 140, 64)
    _check(q, k, v, do, causal=True)


def test_no_queries_no_keys_no_batch(gpu):
    q, k, v, do = _inputs(torch.bfloat16, 2, 2, 2, 5, 7, 16)
    o = _run(q, k[:, :, :0], v[:, :, :0], do)
    assert not o["o"].any() and not o["dq"].any() and o["dk"].shape == (2, 2, 0, 16)
    o = _run(q[:, :, :0], k, v, do[:, :, :0])
    assert o["o"].shape == (2, 2, 0, 16) and not o["dk"].any() and not o["dv"].any()
    o = _run(q[:0], k[:0], v[:0], do[:0])
    assert o["dk"].shape == (0, 2, 7, 16)


def test_offsets_beyond_32_bits(gpu):
    # keys 2^26 elements apart: the last ones lie over 2^32 elements in
    t, Tk, D, apart = torch.bfloat16, 70, 64, 2 ** 26
    cache = torch.empty(Tk * apart, dtype=t, device="cuda")
    k = cache.as_strided((1, 1, Tk, D), (0, 0, apart, 1))
    v = cache.as_strided((1, 1, Tk, D), (0, 0, apart, 1), D)
    q, k0, v0, do = _inputs(t, 1, 2, 1, 3, Tk, D)
    k.copy_(k0)
    v.copy_(v0)
    got, want = _run(q, k, v, do), _run(q, k0, v0, do)
    for name in got:
        assert torch.equal(got[name], want[name]), name


def test_gradient_against_differences(gpu):
    # f = sum(o c) in fp32, central differences of step 1e-2 along a unit
    # direction: truncation about 1e-4 and noise below 1e-3 of a derivative of
    # order 1
    q, k, v, c = _inputs(torch.float32, 1, 2, 1, 30, 40, 24)
    grads = _run(q, k, v, c, causal=True)
    f = lambda *a: (_run(*a, causal=True)["o"].double() * c.double()).sum().item()  # noqa: E731
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn((q, k, v)[i].shape, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")
        d /= d.norm()
        up, down = [q, k, v], [q, k, v]
        h = 1e-2
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        along = (grads[name].double() * d.double()).sum().item()
        assert abs((f(*up) - f(*down)) / (2 * h) - along) <= 1e-2 * (1 + abs(along)), name


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 2)])
def test_some_gradients_only(gpu, wanted):
    # a frozen context, or frozen queries: the gradients asked for are the same bits
    from blitzgs_amd.attention import attention
    q, k, v, do = _inputs(torch.bfloat16, 2, 4, 2, 60, 90, 64)
    full = _run(q, k, v, do)
    leaves = [x.detach().requires_grad_(i in wanted) for i, x in enumerate((q, k, v))]
    got = torch.autograd.grad(attention(*leaves), [leaves[i] for i in wanted], do)
    for i, g in zip(wanted, got):
        assert torch.equal(g, full[("dq", "dk", "dv")[i]])


def test_equal_bits_and_another_stream(gpu):
    q, k, v, do = _inputs(torch.bfloat16, 2, 8, 2, 500, 700, 64)
    how = dict(causal=True, key_lengths=_int(700, 333))
    first = _run(q, k, v, do, **how)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = _run(q, k, v, do, **how)
    torch.cuda.current_stream().wait_stream(s)
    for name in first:
        assert torch.equal(first[name], second[name]), name


def test_graph_capture(gpu):
    # a forward inside a captured graph, replayed on new inputs with eager work between
    from blitzgs_amd.attention import attention
    q, k, v, _ = _inputs(torch.bfloat16, 1, 4, 2, 2, 3000, 64)
    lengths = _int(3000)
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            attention(q, k, v, key_lengths=lengths)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = attention(q, k, v, key_lengths=lengths)
        for n in (3000, 1, 1777, 0):
            q.copy_(torch.randn_like(q))
            lengths.fill_(n)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, attention(q, k, v, key_lengths=lengths)), n


def test_refusals(gpu):
    from blitzgs_amd.attention import attention
    q, k, v, _ = _inputs(torch.bfloat16, 2, 4, 2, 5, 7, 16)
    for args, how, words in [
            ((q.cpu(), k, v), {}, "HIP device tensor"), ((q.double(), k, v), {}, "float32, bfloat16 or float16"),
            ((q, k.float(), v), {}, "like q"), ((q[0], k, v), {}, "dimensions"), ((q, k, v[:, :, 1:]), {}, "one shape"),
            ((q[:1], k, v), {}, "one shape"), ((q[:, :3], k, v), {}, "multiple"), ((q[..., :8], k, v), {}, "one shape"),
            ((q[..., :0], k[..., :0], v[..., :0]), {}, "head dimension"), ((q, k, v), dict(scale=0.0), "scale"),
            ((q, k, v), dict(scale=math.nan), "scale"), ((q, k, v), dict(scale=-1.0), "scale"),
            ((q, k, v), dict(query_start=_int(0, 0)), "causal"),
            ((q, k, v), dict(key_lengths=torch.tensor([1, 2], device="cuda")), "int32"),
            ((q, k, v), dict(key_lengths=_int(1)), "int32"),
            ((q, k, v), dict(key_lengths=_int(1, 2).cpu()), "int32")]:
        with pytest.raises(RuntimeError, match=words):
            attention(*args, **how)
    wide = torch.zeros((1, 1, 2, 129), device="cuda")
    with pytest.raises(RuntimeError, match="head dimension"):
        attention(wide, wide, wide)


# What a NaN or an infinity in one token reaches: the queries that see the key, and
# the keys that the query sees.  Everything else is what it is without, to the bit
# where no row's scores change, else (the running base moves for several rows
# together) within the bound.
SPOILED = [float("nan"), float("inf"), float("-inf")]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Tq,D", [(1, 64), (1, 128), (5, 40), (70, 64), (3, 33)])
def test_the_unused_end_of_a_cache_is_not_read(gpu, t, Tq, D):
    B, Tk = 3, 300
    q, k, v, do = _inputs(t, B, 4, 2, Tq, Tk, D)
    start = _int(0, 17, 200)
    how = dict(causal=True, query_start=start)
    for b in range(B):
        k[b, :, int(start[b]) + Tq:] = 0
        v[b, :, int(start[b]) + Tq:] = 0
    clean = _run(q, k, v, do, **how)
    for spoil in SPOILED:
        for b in range(B):
            k[b, :, int(start[b]) + Tq:] = spoil
            v[b, :, int(start[b]) + Tq:] = spoil
        got = _run(q, k, v, do, **how)
        for name in got:
            assert torch.equal(got[name], clean[name]), (name, spoil)
        assert torch.equal(_run(q, k, v, **how)["o"], clean["o"])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,D", [(40, 32), (200, 64), (130, 128), (100, 80), (70, 31)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_what_a_later_key_holds_does_not_reach_earlier_queries(gpu, t, T, D, which):
    at = T // 2 + 3
    q, k, v, do = _inputs(t, 1, 4, 2, T, T, D)
    clean = _run(q, k, v, causal=True)["o"]
    want = attention_64(q, k, v, True, None, None, 1.0 / math.sqrt(D), do)
    for spoil in SPOILED:
        x = dict(k=k.clone(), v=v.clone())
        x[which][0, 1, at, D // 2] = spoil
        got = _run(q, x["k"], x["v"], do, causal=True)
        for name in ("o", "dq"):
            within(got[name][:, :2], *(w[:, :2] for w in want[name]), f"{spoil}: {name} of the other key head's queries")
            within(got[name][:, :, :at], *(w[:, :, :at] for w in want[name]), f"{spoil}: {name} of earlier queries")
        for name in ("dk", "dv"):
            within(got[name][:, :1], *(w[:, :1] for w in want[name]), f"{spoil}: {name} of the other key head")
        o = got["o"]
        if which == "v":
            assert torch.equal(o[:, :, :at], clean[:, :, :at])
            rest = [d for d in range(D) if d != D // 2]
            assert torch.equal(o[..., rest], clean[..., rest])
            column = o[:, 2:, at:, D // 2].float()
            assert torch.isnan(column).all() if math.isnan(spoil) else (column == spoil).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("T,D", [(40, 32), (200, 64), (130, 128), (70, 31)])
@pytest.mark.parametrize("which", ["q", "do"])
def test_what_an_earlier_query_holds_does_not_reach_later_keys(gpu, t, T, D, which):
    at = T // 2 - 5
    q, k, v, do = _inputs(t, 1, 4, 2, T, T, D)
    want = attention_64(q, k, v, True, None, None, 1.0 / math.sqrt(D), do)
    for spoil in SPOILED:
        x = dict(q=q.clone(), do=do.clone())
        x[which][0, 3, at] = spoil
        got = _run(x["q"], k, v, x["do"], causal=True)
        others = [i for i in range(T) if i != at]
        within(got["dq"][:, :, others], *(w[:, :, others] for w in want["dq"]), f"{spoil}: dq")
        for name in ("dk", "dv"):
            within(got[name][:, :1], *(w[:, :1] for w in want[name]), f"{spoil}: {name} of the other key head")
            within(got[name][:, :, at + 1:], *(w[:, :, at + 1:] for w in want[name]), f"{spoil}: {name}, later keys")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("D", [31, 64, 128])
def test_what_rows_that_see_nothing_hold_reaches_nothing(gpu, t, D):
    q, k, v, do = _inputs(t, 2, 4, 2, 50, 90, D)
    how = dict(causal=True, query_start=_int(-20, -50))             # 20 empty rows, 50 empty rows
    q[0, :, :20] = 0
    do[0, :, :20] = 0
    q[1] = 0
    do[1] = 0
    clean = _run(q, k, v, do, **how)
    for spoil in SPOILED:
        q[0, :, :20] = spoil
        do[0, :, :20] = spoil
        q[1] = spoil
        do[1] = spoil
        got = _run(q, k, v, do, **how)
        for name in got:
            assert torch.equal(got[name], clean[name]), (name, spoil)
        assert not got["o"][0, :, :20].any() and not got["dq"][0, :, :20].any()
        assert not any(got[name][1].any() for name in got)
