"""The 8-bit key/value cache on the GPU against its definition in 64 bits (tests/cache_ref.py).

Tolerances.  Stored values and scales are exact: scales are powers of two, so that bringing a 16-bit value (or a stored one)
to a scale is exact in 32 bits and only the rounding to 8 bits, which is the definition's, is left; reading back is exact
where the target type can hold the value and one rounding otherwise.

Attention: (a) the output's rounding, half a step: eps / 2 * |out|; (b) the weights are rounded to fp16, at most 2^-11 of
each (2^-25 of the largest for the smallest ones): 2^-11 * sum p|v|; (c) an error e of a score changes each weight by a
factor within e^(+-e) before and after the division by their sum: 2 e * sum p|v|, where a 32-bit sum of d products
is off by at most (d + 8) * 2^-24 * sum|q||k| * scale; (d) 32-bit exponentials, sums and scalings, 2^-18 in all.
The log-sum-exp is off by e, and by the sums' and the logarithm's rounding, 2^-20 relative to 1 and to itself.

Sums of weights: each term is off by the factor of (c), by the rounding of s * scale * log2(e) - lse * log2(e), half a step
of its larger part (2^-24 * (|s| + |lse|) * log2(e), taken with the largest |lse|, times ln 2), and by the exponential's
2^-20; the 128 terms of a tile are added in 32 bits (at most 128 * 2^-24), the tiles with compensation (2^-23).
"""
import math
import random

import pytest
import torch

import cache_ref as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _ops():
    from ring_swa import ops
    return ops


def make(kind, num_blocks, heads, bs, d, seed, garbage=True):
    """A cache on the GPU whose unused blocks hold what must not matter: arbitrary bytes, NaN scales."""
    ops = _ops()
    g = torch.Generator().manual_seed(seed)
    cache = ops.KVCache.empty(num_blocks, heads, bs, d, dtype=R.TORCH[kind])
    if garbage:
        for x in (cache.k, cache.v):
            x.view(torch.uint8).copy_(torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8))
        cache.k_scale.fill_(math.nan)
        cache.v_scale.fill_(math.nan)
    return cache


def host(cache):
    return {"k": cache.k.cpu().float().double(), "v": cache.v.cpu().float().double(),
            "k_scale": cache.k_scale.cpu().double(), "v_scale": cache.v_scale.cpu().double()}


def tables(lens, bs, max_blocks, num_blocks, seed):
    r = random.Random(seed)
    pages = r.sample(range(num_blocks), num_blocks)
    table = torch.full((len(lens), max_blocks), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range((n + bs - 1) // bs):
            table[i, j] = pages.pop()
    return table


def normal(*shape, seed, dt):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DT[dt])


def filled(kind, dt, lens, heads, bs, d, seed, v_spread=False, spare=3):
    """A cache with `lens` tokens per sequence, written by cache_append in one packed call, and its table."""
    ops = _ops()
    blocks = [(n + bs - 1) // bs for n in lens]
    total = sum(blocks) + spare
    table = tables(lens, bs, max(blocks + [1]) + 1, total, seed)
    cache = make(kind, total, heads, bs, d, seed)
    t = sum(lens)
    k, v = normal(t, heads, d, seed=seed + 1, dt=dt), normal(t, heads, d, seed=seed + 2, dt=dt)
    if v_spread:  # blocks of very different magnitudes
        v = (v.float() * torch.exp2(torch.arange(t)[:, None, None] % 40 / 4.0 - 5)).to(DT[dt])
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32)
    ops.cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.zeros(len(lens), dtype=torch.int32, device="cuda"), cu_seqlens=cu.cuda())
    return cache, table, k, v, cu


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dt,bs,d,heads", [("bf16", 16, 64, 1), ("bf16", 64, 128, 3), ("fp16", 128, 128, 2), ("fp16", 32, 64, 8), ("bf16", 128, 64, 2),
                                           ("bf16", 16, 128, 4)])
def test_append_and_read_are_exact(kind, dt, bs, d, heads):
    ops = _ops()
    first, more, last = [0, 1, bs, 3 * bs - 1, 5, 2 * bs], [bs + 3, 1, 0, 2, 2 * bs, 1], [1, 1, 1, 1, 1, 1]
    lens = [0] * 6
    room = [(a + b + 1 + bs - 1) // bs for a, b in zip(first, more)]
    table = tables([n * bs for n in room], bs, max(room) + 1, sum(room) + 2, seed=5)
    cache = make(kind, sum(room) + 2, heads, bs, d, seed=6)
    ref = host(cache)
    for step, counts in enumerate((first, more, last)):
        t = sum(counts)
        # every step's values are larger in some sequences: scales of blocks in use have to grow
        grow = torch.repeat_interleave(torch.tensor([1.0, 3.0, 0.1, 9.0, 1.0, 40.0]) ** step, torch.tensor(counts))[:, None, None]
        k, v = ((normal(t, heads, d, seed=10 * step + i, dt=dt).float() * grow).to(DT[dt]) for i in (0, 1))
        cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
        R.append(ref, kind, table.tolist(), lens, [x.double() for x in k.split(counts)], [x.double() for x in v.split(counts)], counts)
        at = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if step < 2:
            ops.cache_append(cache, k.cuda(), v.cuda(), table.cuda(), at, cu_seqlens=cu.cuda())
        else:
            ops.cache_append(cache, k.view(6, 1, heads, d).cuda(), v.view(6, 1, heads, d).cuda(), table.cuda(), at)
        lens = [a + b for a, b in zip(lens, counts)]
        got = host(cache)
        for name in ("k", "v", "k_scale", "v_scale"):  # (unused blocks and slots included: left as they were)
            torch.testing.assert_close(got[name], ref[name], rtol=0, atol=0, equal_nan=True)
    for most in (1, max(lens) - 1, max(lens), max(lens) + bs):
        for out in ("bf16", "fp16"):
            got = ops.cache_read(cache, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), most, dtype=DT[out])
            for x, name in zip(got, ("k", "v")):
                want = torch.zeros(6, most, heads, d, dtype=torch.float64)
                for i, n in enumerate(lens):
                    y = R.rows(ref, name, table[i], n)[:most]
                    want[i, :y.shape[0]] = y
                assert torch.equal(x.cpu(), want.float().to(DT[out]))


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_edges(kind):
    """Zeros, the smallest and the largest values, infinities and NaN; exact ends of the range; a slice of a fused projection."""
    ops = _ops()
    heads, bs, d = 2, 16, 64
    top = R.TOP[kind]
    x = torch.randn(6 * bs, 3 * heads, d, generator=torch.Generator().manual_seed(0)).bfloat16()
    k = x[:, heads:2 * heads]
    k[0:bs] = 0
    k[bs:2 * bs] = 1e-38
    k[2 * bs:3 * bs] = 3e38
    k[3 * bs, 0, 0], k[3 * bs, 1, 0] = math.inf, math.nan
    k[4 * bs:5 * bs].clamp_(-1, 1)[0, 0, 0] = torch.tensor(top * 2 ** 3).bfloat16()
    k[5 * bs:].clamp_(-1, 1)
    k[5 * bs, 0, 0] = torch.nextafter(torch.tensor(top).bfloat16(), torch.tensor(1e9).bfloat16())
    cache = make(kind, 8, heads, bs, d, seed=1)
    ref = host(cache)
    table = torch.tensor([[7, 0, 3, 5, 2, 1, 4]], dtype=torch.int32)
    xs = x.cuda()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    R.append(ref, kind, table.tolist(), [0], [x[:, heads:2 * heads].double()], [x[:, 2 * heads:].double()], [6 * bs])
    ops.cache_append(cache, xs[None, :, heads:2 * heads], xs[None, :, 2 * heads:], table.cuda(), zero)
    got = host(cache)
    bad = torch.isnan(ref["k_scale"])
    assert torch.equal(torch.isnan(got["k_scale"]), bad) and bad[5].all() and not bad[[7, 0, 3, 2, 1]].any()
    torch.testing.assert_close(got["k_scale"], ref["k_scale"], rtol=0, atol=0, equal_nan=True)
    for page in (7, 0, 3, 2, 1):
        assert torch.equal(got["k"][page], ref["k"][page])
    torch.testing.assert_close(got["v"], ref["v"], rtol=0, atol=0, equal_nan=True)
    # a token behind a poisoned block's: the block stays NaN, its neighbours do not care
    k2, v2 = ops.cache_read(cache, table.cuda(), torch.tensor([6 * bs], dtype=torch.int32, device="cuda"), 6 * bs)
    assert torch.isnan(k2[0, 3 * bs:4 * bs]).all() and torch.isfinite(k2[0, :2 * bs]).all() and torch.isfinite(k2[0, 4 * bs:]).all()
    assert torch.isfinite(v2).all()


def check_attn(cache, table, lens, q, window, sink, scale=None, weights=None):
    ops = _ops()
    dt = q.dtype
    ref = host(cache)
    dev = [t.cuda() for t in (q, table, torch.tensor(lens, dtype=torch.int32))]
    acc = None if weights is None else weights.cuda().clone()
    out, lse = ops.cache_attn(dev[0], cache, dev[1], dev[2], window_size=window, num_sink_tokens=sink, softmax_scale=scale, weights=acc,
                              return_lse=True)
    want, want_lse, w, size, most = R.attn(ref, table, lens, q.double(), window, sink, scale)
    e = (q.shape[-1] + 8) * 2.0 ** -24 * most
    eps = torch.finfo(dt).eps / 2
    tol = eps * want.abs() + (1 + eps) * (2.0 ** -11 + 2 * e + 2.0 ** -18) * size + 1e-30
    err = (out.cpu().double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"out: {(err / tol).max().item():.3g} of the tolerance"
    none = torch.isinf(want_lse)
    got_lse = lse.cpu().double()
    assert torch.equal(torch.isinf(got_lse), none)
    assert ((got_lse - want_lse).abs()[~none] <= e + 2.0 ** -20 * (1 + want_lse[~none].abs())).all()
    if weights is not None:
        n = w.shape[-1]
        got = acc.cpu().double()
        assert torch.equal(got[..., n:], weights[..., n:].double()), "weights behind the last slot were written"
        d = (got[..., :n] - weights[..., :n].double() - w).abs()
        rows = q.shape[1] * q.shape[2]
        assert (d <= (2 * e + 2.0 ** -18 + rows * 2.0 ** -24) * w + 2.0 ** -24 * (weights[..., :n].double() + w)).all()
    return out


CASES = [
    # lens, (hq, hkv), d, bs, queries, window, sink
    ([1], (1, 1), 64, 16, 1, None, 0),
    ([33, 1, 0, 17, 16], (4, 4), 64, 16, 1, None, 0),
    ([513], (4, 4), 64, 16, 1, None, 0),
    ([100, 31, 32, 64, 65, 0, 2], (8, 2), 128, 32, 1, None, 0),
    ([300, 1000, 7], (32, 8), 128, 64, 1, None, 0),
    ([2500, 130], (64, 8), 128, 128, 1, None, 0),
    ([777, 40], (16, 1), 128, 16, 1, None, 0),        # 16 rows: two columns of 8
    ([1029, 3, 250], (32, 4), 128, 64, 4, None, 0),   # 32 rows: two row tiles; queries before the start
    ([260, 8], (12, 4), 64, 32, 5, 100, 0),
    ([2000, 50, 700], (32, 8), 128, 128, 1, 256, 4),
    ([2000, 50, 700], (8, 2), 64, 16, 3, 33, 1),
    ([1500, 1499], (16, 16), 128, 16, 2, 31, 40),
    ([4000], (4, 1), 128, 32, 1, 0, 0),               # itself alone
    ([900], (4, 2), 128, 64, 1, 0, 1),
    ([600, 599], (40, 1), 64, 64, 7, 1 << 30, 1 << 30),
]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attn(case, kind):
    lens, (hq, hkv), d, bs, n, window, sink = CASES[case]
    dt = "fp16" if case % 3 == 1 else "bf16"
    cache, table, _, _, _ = filled(kind, dt, lens, hkv, bs, d, seed=case, v_spread=case % 2 == 0)
    q = normal(len(lens), n, hq, d, seed=100 + case, dt=dt)
    w = torch.rand(len(lens), hkv, table.shape[1] * bs + 5, generator=torch.Generator().manual_seed(case)) if case % 4 != 3 else None
    check_attn(cache, table, lens, q, window, sink, scale=0.3 if case % 5 == 2 else None, weights=w)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attn_far_apart_scores_and_query_sizes(kind):
    """Scores of +-300 and queries from 2^-60 to 2^60: the running reference and the queries' scaling."""
    lens, bs, d = [700, 345], 32, 128
    cache, table, _, _, _ = filled(kind, "bf16", lens, 2, bs, d, seed=3)
    for mul in (40.0, 2.0 ** -60, 1.0):
        q = (normal(2, 1, 8, d, seed=9, dt="bf16").float() * mul).bfloat16()
        check_attn(cache, table, lens, q, None, 0)
    q = (normal(2, 1, 8, d, seed=9, dt="bf16").float() * 2.0 ** 60).bfloat16()
    check_attn(cache, table, lens, q, None, 0, scale=d ** -0.5 * 2.0 ** -60)


def test_attn_of_a_poisoned_block():
    """NaN reaches the rows and heads that see the block, and no others."""
    lens, bs, d = [200], 16, 64
    cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=4)
    cache.v_scale[table[0, 3].item(), 1] = math.nan       # slots 48..63 of head 1
    cache.k_scale[table[0, 12].item(), 0] = math.nan      # slots 192..199 of head 0: the newest
    q = normal(1, 12, 4, d, seed=5, dt="bf16")
    args = (q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    out = _ops().cache_attn(*args)
    # head 0 (rows of q heads 0, 1): queries from slot 192 on, the last 8; head 1: every query
    assert torch.isnan(out[0, 4:, :2]).all() and torch.isfinite(out[0, :4, :2]).all() and torch.isnan(out[0, :, 2:]).all()
    out = _ops().cache_attn(*args, window_size=100)
    assert torch.isfinite(out[0, :, 2:]).all()
    out = _ops().cache_attn(*args, window_size=128)
    # query i at slot 188 + i sees from 60 + i on
    assert torch.isnan(out[0, :4, 2:]).all() and torch.isfinite(out[0, 4:, 2:]).all()


def test_attn_strided_queries_scales_and_results_do_not_depend_on_the_run():
    lens, bs, d = [5000, 3, 1234, 2048], 64, 128
    cache, table, _, _, _ = filled("int8", "bf16", lens, 4, bs, d, seed=8)
    fused = normal(4, 2, 24, d, seed=1, dt="bf16")
    q = fused[:, :, :16]
    a = check_attn(cache, table, lens, q, 3000, 2)
    b = check_attn(cache, table, lens, q.contiguous(), 3000, 2)
    assert torch.equal(a, b)
    # scales that are no powers of two
    cache.k_scale.mul_(1.37)
    cache.v_scale.mul_(0.71)
    check_attn(cache, table, lens, q, None, 0)
    # unaligned and otherwise strided queries
    odd = torch.empty(4 * 2 * 16 * d + 1, dtype=torch.bfloat16)[1:].view(4, 2, 16, d).copy_(q)
    check_attn(cache, table, lens, odd, None, 0)
    check_attn(cache, table, lens, q[:1].expand(4, 2, 16, d), None, 0)


def test_many_sequences_of_all_lengths():
    r = random.Random(0)
    lens = [r.choice((0, 1, 15, 16, 17, 31, 33, 64, 100, 200)) for _ in range(300)]
    cache, table, _, _, _ = filled("e4m3", "bf16", lens, 1, 16, 64, seed=2)
    q = normal(300, 1, 2, 64, seed=3, dt="bf16")
    w = torch.zeros(300, 1, table.shape[1] * 16)
    check_attn(cache, table, lens, q, None, 0, weights=w)
    check_attn(cache, table, lens, q, 20, 3)


def test_bad_tables_and_lengths_are_reported():
    from ring_swa import _kernels as K
    ops = _ops()
    lens, bs, d = [100, 50], 16, 64
    cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=4)
    before = host(cache)
    q = normal(2, 1, 4, d, seed=5, dt="bf16").cuda()
    new = normal(2, 1, 2, d, seed=5, dt="bf16").cuda()
    good = torch.tensor(lens, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for bad, n, code in (([[0, 2, -1], [0, 2, 1 << 30]], None, 110), (None, [[100, -1], [100, 10000]], 111)):
        for i in range(2):
            t, l = table.clone(), good.clone()
            if bad is not None:
                t[bad[i][0], bad[i][1]] = bad[i][2]
            if n is not None:
                l = torch.tensor(n[i], dtype=torch.int32, device="cuda")
            calls = [lambda: ops.cache_attn(q, cache, t.cuda(), l), lambda: ops.cache_read(cache, t.cuda(), l, 112)]
            if n is not None:
                calls.append(lambda: ops.cache_append(cache, new[1:], new[1:], t[1:].cuda(), l[1:]))
            for call in calls:
                call()
                torch.cuda.synchronize()
                with pytest.raises(RuntimeError, match=f"code {code}"):
                    ops.cache_read(cache, table.cuda(), good, 1)
                K.check_device_status()  # (cleared)
    after = host(cache)
    for name in before:
        torch.testing.assert_close(after[name], before[name], rtol=0, atol=0, equal_nan=True)
    check_attn(cache, table, lens, q.cpu(), None, 0)


def test_a_captured_step_is_replayed_with_other_lengths_and_on_another_stream():
    """append + attention captured once and replayed for five tokens; two such graphs run at the same time on two streams."""
    ops = _ops()
    bs, d, hkv, hq = 16, 128, 2, 8
    runs = []
    for seed in (0, 1):
        lens = [30 + 700 * seed, 100, 15]
        cache, table, _, _, _ = filled("int8", "bf16", [n + 8 for n in lens], hkv, bs, d, seed=seed, spare=0)
        table = table.cuda()
        runs.append(dict(cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), host=lens,
                         q=torch.zeros(3, 1, hq, d, dtype=torch.bfloat16, device="cuda"), k=torch.zeros(3, 1, hkv, d, dtype=torch.bfloat16, device="cuda"),
                         v=torch.zeros(3, 1, hkv, d, dtype=torch.bfloat16, device="cuda"), w=torch.zeros(3, hkv, table.shape[1] * bs, device="cuda"),
                         stream=torch.cuda.Stream()))
    for r in runs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            ops.cache_append(r["cache"], r["k"], r["v"], r["table"], r["lens"])
            r["lens"].add_(1)
            r["out"] = ops.cache_attn(r["q"], r["cache"], r["table"], r["lens"], window_size=600, num_sink_tokens=2, weights=r["w"])
        r["graph"] = g
        r["eager"] = ops.KVCache(*(t.clone() for t in (r["cache"].k, r["cache"].v, r["cache"].k_scale, r["cache"].v_scale)))
        r["eager_w"] = r["w"].clone()
    for step in range(5):
        for i, r in enumerate(runs):
            for j, name in enumerate(("q", "k", "v")):
                r[name].copy_(normal(*r[name].shape, seed=100 * step + 10 * i + j, dt="bf16"))
        torch.cuda.synchronize()
        for r in runs:
            with torch.cuda.stream(r["stream"]):
                r["graph"].replay()
        torch.cuda.synchronize()
        for r in runs:
            at = torch.tensor([n + step for n in r["host"]], dtype=torch.int32, device="cuda")
            ops.cache_append(r["eager"], r["k"], r["v"], r["table"], at)
            want = ops.cache_attn(r["q"], r["eager"], r["table"], at + 1, window_size=600, num_sink_tokens=2, weights=r["eager_w"])
            assert torch.equal(r["out"], want) and torch.equal(r["w"], r["eager_w"])
            assert torch.equal(r["lens"], at + 1)
            for name in ("k", "v"):
                assert torch.equal(getattr(r["cache"], name).view(torch.uint8), getattr(r["eager"], name).view(torch.uint8))


SUMS = [
    # lens, (hq, hkv), d, window, sink, packed
    ([1], (1, 1), 64, 0, 0, False),
    ([5], (4, 2), 128, None, 0, True),
    ([128], (4, 4), 64, 128, 0, False),
    ([129], (2, 1), 128, 0, 0, False),
    ([300], (8, 2), 128, 100, 0, False),
    ([777], (4, 4), 64, 1 << 30, 1 << 30, False),
    ([1000], (6, 2), 128, 129, 1, True),
    ([1, 255, 1, 256, 2, 500, 3], (4, 2), 64, 64, 4, True),
    ([700, 30, 900], (4, 1), 128, 250, 2, True),
    ([1, 1, 1, 1, 40, 128, 128], (2, 2), 64, 20, 0, True),
    ([2100], (16, 2), 128, 500, 300, False),
    ([513] * 3, (4, 4), 128, 33, 1, False),   # a batch
    ([260] * 2, (2, 1), 64, None, 0, False),
]


@pytest.mark.parametrize("case", range(len(SUMS)))
def test_weight_sums(case):
    ops = _ops()
    lens, (hq, hkv), d, window, sink, packed = SUMS[case]
    dt = "fp16" if case % 2 else "bf16"
    t = sum(lens)
    qk = normal(t, hq + hkv, d, seed=case, dt=dt)
    q, k = qk[:, :hq], qk[:, hq:]
    scale = None if case % 3 else 0.2
    # the log-sum-exp of the attention itself
    cu = [0] + torch.tensor(lens).cumsum(0).tolist()
    lse = torch.full((hq, t), -math.inf, dtype=torch.float64)
    for a, z in zip(cu, cu[1:]):
        i, j = torch.arange(z - a)[:, None], torch.arange(z - a)[None]
        seen = j <= i if window is None else (j <= i) & ((i - j <= window) | (j < sink))
        for h in range(hq):
            s = q[a:z, h].double() @ k[a:z, h // (hq // hkv)].double().T * (d ** -0.5 if scale is None else scale)
            lse[h, a:z] = s.masked_fill(~seen, -math.inf).logsumexp(1)
    lse = lse.float()
    if case == 8:
        lse[1, 3], lse[0, 900] = -math.inf, -math.inf   # queries that are said to have seen nothing
    want, most, terms = R.weight_sums(q.double(), k.double(), lse, window, sink, scale, lens)
    if packed:
        got = ops.attn_weight_sums(q.cuda(), k.cuda(), lse.cuda(), window, sink, softmax_scale=scale, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda())
    else:
        b = len(lens)
        qb, kb = (x.contiguous().cuda().view(b, t // b, -1, d) for x in (q, k))
        got = ops.attn_weight_sums(qb, kb, lse.view(hq, b, t // b).transpose(0, 1).cuda(), window, sink, softmax_scale=scale)
        got = got.transpose(0, 1).reshape(hkv, t)
    e = (d + 8) * 2.0 ** -24 * most
    big = lse[torch.isfinite(lse)].abs().max().item()
    rel = e + 2.0 ** -24 * (most + big) + 2.0 ** -20 + 128 * 2.0 ** -24 + 2.0 ** -23
    err = (got.cpu().double() - want).abs()
    assert (err <= rel * want + 1e-30).all(), f"{(err / (rel * want + 1e-30)).max().item():.3g} of the tolerance"
    if case != 8:  # (every query's weights add up to one; the log-sum-exps' own rounding is 2^-24 * |lse|)
        assert abs(want.sum().item() / (t * hq) - 1) < 2.0 ** -23 * (1 + big)


def test_weight_sums_of_the_forward_kernels_and_run_to_run():
    """With the log-sum-exp that the attention operator returns; the same bits every time."""
    import ring_swa.compiled  # noqa: F401  (registers the operator)
    ops = _ops()
    b, s, hq, hkv, d, window, sink = 2, 3000, 8, 2, 128, 700, 4
    q, k, v = (normal(b, s, h, d, seed=i, dt="bf16").cuda() for i, h in enumerate((hq, hkv, hkv)))
    _, lse = torch.ops.ring_swa.swa_fwd(q, k, v, window, sink, d ** -0.5, None)
    got = ops.attn_weight_sums(q, k, lse, window, sink)
    assert abs(got.double().sum().item() / (b * s * hq) - 1) < 2e-3  # (16-bit weights in the forward kernel's sum)
    for i in range(b):
        want, _, _ = R.weight_sums(q[i].cpu().double(), k[i].cpu().double(), lse[i].cpu(), window, sink, None, [s])
        assert ((got[i].cpu().double() - want).abs() <= 1e-4 * want).all()
    assert torch.equal(got, ops.attn_weight_sums(q, k, lse, window, sink))


@pytest.mark.parametrize("window,sink", [(300, 0), (2000, 4)])
def test_weight_sums_of_more_queries_than_l2_holds(window, sink):
    """All heads in one call, whose work is cut into rounds, against a call for each key/value head.  Tolerance: the sums of a
    step are the same; compensated sums over steps err by 2 roundings, the halves' and up to three pieces' additions by 3
    more, on either side."""
    ops = _ops()
    s, hq, hkv, d = 18500, 32, 2, 64
    q, k = normal(1, s, hq, d, seed=1, dt="bf16").cuda(), normal(1, s, hkv, d, seed=2, dt="bf16").cuda()
    lse = (normal(1, hq, s, seed=3, dt="bf16").float() + 4.0).cuda()
    got = ops.attn_weight_sums(q, k, lse, window, sink)
    g = hq // hkv
    for h in range(hkv):
        one = ops.attn_weight_sums(q[:, :, h * g:(h + 1) * g], k[:, :, h:h + 1], lse[:, h * g:(h + 1) * g], window, sink)
        torch.testing.assert_close(got[:, h], one[:, 0], rtol=10 * 2.0 ** -24, atol=0)
    assert torch.equal(got, ops.attn_weight_sums(q, k, lse, window, sink))


EVICT = [
    # lens, heads, d, bs, budget, sink, recent
    ([100], 1, 64, 16, 40, 0, 0),
    ([1500, 40, 1], 2, 64, 16, 512, 4, 128),
    ([300, 513, 64, 0], 3, 128, 64, 200, 1, 50),
    ([2000, 1999], 2, 128, 128, 1000, 0, 1000),      # the newest alone
    ([700], 4, 64, 32, 4, 4, 0),                      # the sinks alone
    ([700], 2, 128, 16, 699, 2, 3),
    ([100, 90], 2, 64, 32, 500, 4, 100),              # nothing to do
    ([5000, 33], 1, 64, 16, 1, 0, 0),
    ([70000], 1, 64, 128, 20000, 4, 1000),
    ([16000, 9100], 2, 64, 16, 9000, 100, 8900),      # sinks and newest alone, of many
    ([50000, 3, 6000], 2, 64, 64, 5000, 3, 1),        # several CTAs a head, some of them without a slot
    ([30000, 29999], 8, 64, 128, 25000, 0, 0),
    ([400000], 1, 64, 128, 1500, 4, 100),             # more than their shared memory holds
]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("case", range(len(EVICT)))
def test_evict(case, kind):
    ops = _ops()
    lens, heads, d, bs, budget, sink, recent = EVICT[case]
    cap = max(1, max((n + bs - 1) // bs for n in lens))
    new_cap = (min(budget, cap * bs) + bs - 1) // bs
    total = sum((n + bs - 1) // bs for n in lens)
    new_total = sum((min(n, budget) + bs - 1) // bs for n in lens)
    cache, table, _, _, _ = filled(kind, "bf16", lens, heads, bs, d, seed=case, v_spread=True, spare=new_total + 2)
    table = table[:, :cap]
    free = sorted(set(range(total + new_total + 2)) - set(table.flatten().tolist()))
    random.Random(case).shuffle(free)
    new_table = torch.full((len(lens), new_cap), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for j in range((min(n, budget) + bs - 1) // bs):
            new_table[i, j] = free.pop()
    g = torch.Generator().manual_seed(case)
    w = (torch.randn(len(lens), heads, cap * bs + 3, generator=g) * 2).exp()
    # all kinds of ties: a few values for most, zeros of both signs, infinities, NaN, negative ones
    w = torch.where(torch.rand(w.shape, generator=g) < 0.7, w.round().clamp(0, 3), w)
    w = torch.where(torch.rand(w.shape, generator=g) < 0.05, -w, w)
    if case % 2:
        w[..., 7::97], w[..., 11::131] = math.nan, math.inf
    ref = host(cache)
    want_lens, want_kept = R.evict(ref, kind, table, lens, w, budget, new_table, sink, recent)
    dev = torch.tensor(lens, dtype=torch.int32).cuda()
    new_lens, new_w, kept = ops.cache_evict(cache, table.cuda(), dev, w.cuda(), budget, new_table.cuda(), sink, recent)
    assert new_lens.tolist() == want_lens and new_lens.dtype == torch.int32
    assert new_w.shape == (len(lens), heads, new_cap * bs) and kept.shape == (len(lens), heads, budget)
    for b in range(len(lens)):
        for h in range(heads):
            slots = want_kept[b][h]
            assert kept[b, h].tolist() == slots + [-1] * (budget - len(slots))
            want = torch.zeros(new_cap * bs)
            want[:len(slots)] = w[b, h][slots]
            torch.testing.assert_close(new_w[b, h].cpu(), want, rtol=0, atol=0, equal_nan=True)
    got = host(cache)
    for name in ("k", "v", "k_scale", "v_scale"):  # (the old blocks and the unused ones as they were)
        torch.testing.assert_close(got[name], ref[name], rtol=0, atol=0, equal_nan=True)
    # evicting again what is within the budget now: the same values, bit for bit
    if case in (1, 2):
        room = ops.KVCache(*(torch.cat([x, torch.zeros_like(x)]) for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        third = torch.where(new_table >= 0, new_table + cache.k.shape[0], new_table)
        args = (new_lens, new_cap * bs)
        ops.cache_evict(room, new_table.cuda(), new_lens, new_w, budget, third.cuda())
        for x, y in zip(ops.cache_read(room, new_table.cuda(), *args), ops.cache_read(room, third.cuda(), *args)):
            assert torch.equal(x, y)


def test_evict_by_clusters_in_a_graph_and_on_two_streams():
    """Long contexts, several CTAs a head: a captured call replayed with other lengths and weights, and eager calls on two
    streams beside each other, give what single calls give."""
    ops = _ops()
    n, heads, bs, d, budget = 40000, 2, 64, 64, 3000
    cache, table, _, _, _ = filled("int8", "bf16", [n], heads, bs, d, seed=5, spare=2 * 47 + 1)
    used = set(table.flatten().tolist())
    free = [i for i in range(cache.k.shape[0]) if i not in used]
    table = table[:, :n // bs].contiguous().cuda()
    new = [torch.tensor([free[i * 47:(i + 1) * 47]], dtype=torch.int32).cuda() for i in range(2)]
    weights = [torch.rand(1, heads, n, generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]
    lens = [torch.tensor([m], dtype=torch.int32).cuda() for m in (n, 25000, 2999)]
    call = lambda m, w, to: ops.cache_evict(cache, table, m, w, budget, to, 4, 100)
    want = [[x.clone() for x in call(lens[i], weights[i], new[0])] + [x.clone() for x in ops.cache_read(cache, new[0], lens[2] * 0 + min(budget, int(lens[i])), budget)]
            for i in range(3)]
    m, w = lens[0].clone(), weights[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(m, w, new[0])
        back = ops.cache_read(cache, new[0], got[0], budget)
    for i in (2, 1, 0):
        m.copy_(lens[i]), w.copy_(weights[i])
        graph.replay()
        for x, y in zip([*got, *back], want[i]):
            assert torch.equal(x, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results[i] = call(lens[i], weights[i], new[i])
    torch.cuda.synchronize()
    for i in range(2):
        for x, y in zip(results[i], want[i]):
            assert torch.equal(x, y)


def test_evict_keeps_poison_and_reports_bad_tables():
    ops = _ops()
    cache, table, _, _, _ = filled("int8", "bf16", [64], 2, 16, 64, seed=1, spare=4)
    free = sorted(set(range(8)) - set(table.flatten().tolist()))
    new_table = torch.tensor([free[:2]], dtype=torch.int32)
    w = torch.arange(128.0).view(1, 2, 64) % 64
    w = torch.nn.functional.pad(w, (0, table.shape[1] * 16 - 64))
    cache.v_scale[table[0, 1].item(), 0] = math.nan     # slots 16..31
    lens = torch.tensor([64], dtype=torch.int32).cuda()
    w[0, 0, 16:18] = 100.0
    _, _, kept = ops.cache_evict(cache, table.cuda(), lens, w.cuda(), 32, new_table.cuda())
    assert kept[0, 0].tolist() == [16, 17, *range(34, 64)] and kept[0, 1].tolist() == list(range(32, 64))
    k, v = ops.cache_read(cache, new_table.cuda(), torch.tensor([32], dtype=torch.int32).cuda(), 32)
    assert torch.isnan(v[0, :16, 0]).all() and torch.isfinite(v[0, 16:, 0]).all() and torch.isfinite(v[0, :, 1]).all() and torch.isfinite(k).all()
    before = host(cache)
    for bad in (-1, 8, 1 << 30):
        ops.cache_evict(cache, table.cuda(), lens, w.cuda(), 32, torch.tensor([[new_table[0, 0].item(), bad]], dtype=torch.int32).cuda())
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="code 110"):
            ops.cache_read(cache, table.cuda(), lens, 1)
    ops.cache_evict(cache, table.cuda(), lens - 100, w.cuda(), 32, new_table.cuda())
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="code 111"):
        ops.cache_read(cache, table.cuda(), lens, 1)
    after = host(cache)
    for name in before:
        torch.testing.assert_close(after[name], before[name], rtol=0, atol=0, equal_nan=True)


def test_prompt_then_steps_then_eviction_then_steps():
    """The operators together: a packed batch of prompts through StreamingLLM attention, its weights and its keys and values into
    the cache, steps that add their weights, an eviction, further steps, and the cut prefix read back for a next turn."""
    import ring_swa
    import ring_swa.compiled  # noqa: F401
    ops = _ops()
    hq, hkv, d, bs, window, sink, budget = 8, 2, 128, 32, 400, 4, 256
    lens, steps = [600, 90, 333], 6
    t = sum(lens)
    cu = torch.tensor([0, 600, 690, 1023], dtype=torch.int32)
    q, k, v = (normal(t, h, d, seed=20 + i, dt="bf16") for i, h in enumerate((hq, hkv, hkv)))
    dev = [x.cuda() for x in (q, k, v, cu)]
    out = ring_swa.ring_streaming_llm_attn_varlen(*dev[:3], window, dev[3], cp_size=1, num_sink_tokens=sink)
    out2, lse = torch.ops.ring_swa.swa_fwd(dev[0][None], dev[1][None], dev[2][None], window, sink, d ** -0.5, dev[3])
    assert torch.equal(out, out2[0])
    cap = (max(lens) + 2 * steps + bs - 1) // bs
    table = tables([n + 2 * steps for n in lens], bs, cap, 60, seed=2)
    cache = make("int8", 60 + 30, hkv, bs, d, seed=3)
    lens_dev = torch.zeros(3, dtype=torch.int32, device="cuda")
    w = torch.zeros(3, hkv, cap * bs, device="cuda")
    ops.cache_append(cache, dev[1], dev[2], table.cuda(), lens_dev, cu_seqlens=dev[3])
    sums = ops.attn_weight_sums(dev[0], dev[1], lse[0], window, sink, cu_seqlens=dev[3])
    for i in range(3):
        w[i, :, :lens[i]] = sums[:, cu[i]:cu[i + 1]]
    lens_dev += dev[3][1:] - dev[3][:-1]
    ref, ref_w, ref_lens = host(cache), w.cpu().double(), list(lens)
    kind = "int8"

    def step(n, table, seed, cap):
        nonlocal ref_w
        x = [normal(3, 1, h, d, seed=seed + i, dt="bf16") for i, h in enumerate((hq, hkv, hkv))]
        ops.cache_append(cache, x[1].cuda(), x[2].cuda(), table.cuda(), lens_dev)
        lens_dev.add_(1)
        R.append(ref, kind, table.tolist(), ref_lens, [y.double() for y in x[1]], [y.double() for y in x[2]], [1, 1, 1])
        for i in range(3):
            ref_lens[i] += 1
        got = ops.cache_attn(x[0].cuda(), cache, table.cuda(), lens_dev, window_size=window, num_sink_tokens=sink, weights=w)
        want, _, dw, size, most = R.attn(ref, table, ref_lens, x[0].double(), window, sink)
        ref_w[..., :dw.shape[-1]] += dw
        e = (d + 8) * 2.0 ** -24 * most
        assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1.01 * (2.0 ** -11 + 2 * e + 2.0 ** -18) * size).all()

    for n in range(steps):
        step(n, table, 100 + 10 * n, cap)
    new_cap = (budget + steps + bs - 1) // bs
    new_table = torch.arange(60, 60 + 3 * new_cap, dtype=torch.int32).view(3, new_cap)
    exact_w = w.cpu()
    assert ((exact_w.double() - ref_w).abs() <= 2.0 ** -17 * ref_w).all()
    ref_lens, kept = R.evict(ref, kind, table, ref_lens, exact_w, budget, new_table, sink, 64)
    new_lens, w, got_kept = ops.cache_evict(cache, table.cuda(), lens_dev, w, budget, new_table.cuda(), sink, 64)
    assert [[x[:n].tolist() for x in y] for y, n in zip(got_kept, ref_lens)] == kept and new_lens.tolist() == ref_lens
    lens_dev.copy_(new_lens)
    ref_w = w.cpu().double()
    for n in range(steps):
        step(n, new_table, 500 + 10 * n, new_cap)
    got = ops.cache_read(cache, new_table.cuda(), lens_dev, new_cap * bs)
    for x, name in zip(got, ("k", "v")):
        for i, n in enumerate(ref_lens):
            assert torch.equal(x[i, :n].cpu(), R.rows(ref, name, new_table[i], n).bfloat16())
            assert not x[i, n:].any()


def test_blocks_beyond_32_bit_offsets():
    """A cache of 5 GB per K and V, used at its far end: every operator's addresses."""
    ops = _ops()
    blocks, heads, bs, d = 40000, 8, 128, 128
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    cache = ops.KVCache.empty(blocks, heads, bs, d, dtype=torch.float8_e4m3fn)
    lens = [300, 130]
    table = torch.tensor([[blocks - 1, 39000, blocks - 2], [32768, 17, -1]], dtype=torch.int32)
    new_table = torch.tensor([[blocks - 5], [blocks - 4]], dtype=torch.int32)
    k, v = (normal(sum(lens), heads, d, seed=i, dt="bf16") for i in (0, 1))
    cu = torch.tensor([0, 300, 430], dtype=torch.int32).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    ops.cache_append(cache, k.cuda(), v.cuda(), table.cuda(), n * 0, cu_seqlens=cu)
    # the same in a small cache
    small = ops.KVCache.empty(8, heads, bs, d, dtype=torch.float8_e4m3fn)
    names = {blocks - 1: 0, 39000: 1, blocks - 2: 2, 32768: 3, 17: 4, -1: -1, blocks - 5: 5, blocks - 4: 6}
    s_table, s_new = (torch.tensor([[names[x] for x in row] for row in t.tolist()], dtype=torch.int32).cuda() for t in (table, new_table))
    ops.cache_append(small, k.cuda(), v.cuda(), s_table, n * 0, cu_seqlens=cu)
    q = normal(2, 2, 16, d, seed=5, dt="bf16").cuda()
    w = torch.zeros(2, heads, 3 * bs, device="cuda")
    ws = w.clone()
    assert torch.equal(ops.cache_attn(q, cache, table.cuda(), n, weights=w), ops.cache_attn(q, small, s_table, n, weights=ws))
    assert torch.equal(w, ws)
    a = ops.cache_evict(cache, table.cuda(), n, w, 100, new_table.cuda(), 4, 10)
    b = ops.cache_evict(small, s_table, n, ws, 100, s_new, 4, 10)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    for t, st, ln in ((table.cuda(), s_table, n), (new_table.cuda(), s_new, a[0])):
        for x, y in zip(ops.cache_read(cache, t, ln, 300), ops.cache_read(small, st, ln, 300)):
            assert torch.equal(x, y) and torch.isfinite(x).all()


def test_calls_on_two_streams_at_once():
    """Eager calls that overlap on the GPU share nothing: long ones whose pieces are joined, on two streams, many times."""
    ops = _ops()
    lens, bs, d = [9000], 64, 128
    runs = []
    for seed in (0, 1):
        cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=seed)
        q = normal(1, 1, 8, d, seed=seed + 7, dt="bf16").cuda()
        args = (q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
        runs.append((args, ops.cache_attn(*args), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(40):
        for (args, _, stream), got in zip(runs, outs):
            with torch.cuda.stream(stream):
                got.append(ops.cache_attn(*args))
    torch.cuda.synchronize()
    for (_, want, _), got in zip(runs, outs):
        assert all(torch.equal(x, want) for x in got)


def test_a_first_call_of_a_thread_inside_a_capture():
    import threading
    ops = _ops()
    lens = [500, 20]
    cache, table, _, _, _ = filled("e4m3", "fp16", lens, 2, 32, 64, seed=3)
    q = normal(2, 1, 4, 64, seed=4, dt="fp16").cuda()
    args = (q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    want = ops.cache_attn(*args)
    torch.cuda.synchronize()
    got, errors = [], []

    def work():
        try:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=torch.cuda.Stream()):
                out = ops.cache_attn(*args)
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            got.append(out.clone())
            g.replay()
            torch.cuda.synchronize()
            got.append(out.clone())
            del g
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert not errors, errors
    assert all(torch.equal(x, want) for x in got) and len(got) == 2


def test_shared_prefix_and_empty_calls():
    ops = _ops()
    heads, bs, d = 2, 16, 64
    cache = make("int8", 10, heads, bs, d, seed=0)
    k, v = (normal(1, 2 * bs, heads, d, seed=i, dt="bf16") for i in (0, 1))
    zero = torch.zeros(1, dtype=torch.int32).cuda()
    ops.cache_append(cache, k.cuda(), v.cuda(), torch.tensor([[3, 7]], dtype=torch.int32).cuda(), zero)
    table = torch.tensor([[3, 7, 1], [3, 7, 2], [3, 7, -1]], dtype=torch.int32)  # three sequences that begin alike
    new = normal(2, 1, heads, d, seed=5, dt="bf16").cuda()
    ops.cache_append(cache, new, new, table[:2].cuda(), zero.expand(2).contiguous() + 2 * bs)
    lens = [2 * bs + 1, 2 * bs + 1, 2 * bs]
    q = normal(3, 1, 4, d, seed=6, dt="bf16")
    check_attn(cache, table, lens, q, None, 0, weights=torch.zeros(3, heads, 3 * bs))
    before = host(cache)
    none = torch.zeros(0, 3, dtype=torch.int32).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    assert ops.cache_attn(q[:0].cuda(), cache, none, n[:0]).shape == (0, 1, 4, d)
    assert ops.cache_attn(q[:, :0].cuda(), cache, table.cuda(), n).shape == (3, 0, 4, d)
    out = ops.cache_attn(q.cuda(), cache, torch.zeros(3, 0, dtype=torch.int32).cuda(), n * 0)
    assert not out.any()
    assert [x.shape[1] for x in ops.cache_read(cache, table.cuda(), n, 0)] == [0, 0]
    ops.cache_append(cache, new[:, :0], new[:, :0], table[:2].cuda(), n[:2])
    ops.cache_append(cache, new[:0, 0], new[:0, 0], table.cuda(), n, cu_seqlens=torch.zeros(4, dtype=torch.int32).cuda())
    assert ops.attn_weight_sums(q[:, :0].cuda(), q[:, :0, :2].cuda(), torch.zeros(3, 4, 0).cuda()).shape == (3, 2, 0)
    assert [x.shape[0] for x in ops.cache_evict(cache, none, n[:0], torch.zeros(0, heads, 48).cuda(), 8, none)] == [0, 0, 0]
    after = host(cache)
    for name in before:
        torch.testing.assert_close(after[name], before[name], rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_queries_that_are_not_finite_spoil_their_rows_alone(dt):
    ops = _ops()
    lens = [400]
    cache, table, _, _, _ = filled("int8", dt, lens, 2, 32, 128, seed=1)
    q = normal(1, 3, 8, 128, seed=2, dt=dt)
    args = (cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    want = ops.cache_attn(q.cuda(), *args)
    q[0, 1, 2, 5], q[0, 2, 7, 100] = math.nan, math.nan
    got = ops.cache_attn(q.cuda(), *args)
    bad = torch.zeros(1, 3, 8, dtype=torch.bool)
    bad[0, 1, 2] = bad[0, 2, 7] = True
    assert torch.isnan(got[bad.cuda()]).all() and torch.equal(got[~bad.cuda()], want[~bad.cuda()])
    # in the sums a NaN spoils the keys its query sees
    qs, ks = normal(1, 300, 2, 128, seed=3, dt=dt), normal(1, 300, 1, 128, seed=4, dt=dt)
    lse = torch.full((1, 2, 300), 5.0)
    qs[0, 200, 1, 3] = math.nan
    w = ops.attn_weight_sums(qs.cuda(), ks.cuda(), lse.cuda(), 50)
    nan = torch.isnan(w[0, 0]).cpu()
    assert nan[150:201].all() and not nan[:150].any() and not nan[201:].any()


def test_weight_sums_of_a_batch_with_strides_and_long_prompts():
    """q, k and lse as slices; a prompt whose items are cut between SMs in every way; against the attention over a cache."""
    ops = _ops()
    b, s, hq, hkv, d, window, sink = 2, 2500, 4, 2, 64, 300, 3
    fused = normal(b, s, hq + 2 * hkv, d, seed=1, dt="bf16").cuda()
    q, k = fused[:, :, :hq], fused[:, :, hq:hq + hkv]
    scores = torch.einsum("bihgd,bjhd->bhgij", q.reshape(b, s, hkv, hq // hkv, d).double(), k.double()) * d ** -0.5
    i, j = torch.arange(s, device="cuda")[:, None], torch.arange(s, device="cuda")[None]
    seen = (j <= i) & ((i - j <= window) | (j < sink))
    lse64 = scores.masked_fill(~seen, -math.inf).logsumexp(-1)                    # [b, hkv, group, i]
    lse = torch.zeros(b, hq, 2 * s, device="cuda")[:, :, 5:5 + s]
    lse.copy_(lse64.reshape(b, hq, s))
    want = (scores - lse.double().reshape(b, hkv, -1, s)[..., None]).exp().masked_fill(~seen, 0).sum((2, 3))
    got = ops.attn_weight_sums(q, k, lse, window, sink)
    assert ((got.double() - want).abs() <= 4e-5 * want).all()   # (128 terms in 32 bits: 128 * 2^-24; scores 72 * 2^-24 * 30)
    got = ops.attn_weight_sums(q[:, :, :1], k[:, :, :1].expand(b, s, 1, d), lse[:, :1], None)
    assert got.shape == (b, 1, s)
