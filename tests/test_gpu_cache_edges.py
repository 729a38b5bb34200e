"""The 8-bit key/value cache on the GPU where it could go wrong beside the listed forms: rows that are not finite, freed
blocks, block tables that share their rows, scales from elsewhere, streams from elsewhere.

Against the definitions in 64 bits (cache_ref.py), with the tolerances that test_gpu_cache.py derives; where a test needs more,
it says why.
"""
import math

import pytest
import torch

import cache_ref as R
from test_gpu_cache import _ops, filled, host, make, normal

pytestmark = pytest.mark.gpu


def same_nan(got, want, what):
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in {torch.isnan(got).sum().item()} places, wanted in {torch.isnan(want).sum().item()}"


def check_spoiled_attn(cache, table, lens, q, window, sink, more=0.0):
    """out, log-sum-exp and weights against the definition: NaN exactly where that has NaN, the rest within the tolerances."""
    n = table.shape[1] * cache.k.shape[2]
    start = torch.rand(len(lens), cache.k.shape[1], n, generator=torch.Generator().manual_seed(1))
    acc = start.cuda()
    out, lse = (x.cpu().double() for x in _ops().cache_attn(q.cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), window_size=window,
                                                            num_sink_tokens=sink, weights=acc, return_lse=True))
    acc = acc.cpu().double()
    want, want_lse, w, size, most = R.attn(host(cache), table, lens, q.double(), window, sink)
    want_acc = start.double()
    want_acc[..., :w.shape[-1]] += w
    same_nan(acc, want_acc, "weights"), same_nan(lse, want_lse, "lse"), same_nan(out, want, "out")
    e = (q.shape[-1] + 8) * 2.0 ** -24 * most + more
    eps = torch.finfo(q.dtype).eps / 2
    ok = torch.isfinite(want)
    tol = eps * want.abs() + (1 + eps) * (2.0 ** -11 + 2 * e + 2.0 ** -18) * size
    err = (out - want).abs()
    assert (err <= tol)[ok].all(), f"out: {(err / tol)[ok].max().item():.3g} of the tolerance"
    ok = torch.isfinite(want_lse)
    tol = e + 2.0 ** -20 * (1 + want_lse.abs())
    assert torch.equal(torch.isfinite(lse), ok) and ((lse - want_lse).abs() <= tol)[ok].all(), f"lse: off by {(lse - want_lse).abs()[ok].max().item():.3g}"
    ok = torch.isfinite(want_acc)
    rows = q.shape[1] * q.shape[2]
    tol = (2 * e + 2.0 ** -18 + rows * 2.0 ** -24) * (want_acc - start) + 2.0 ** -24 * want_acc
    err = (acc - want_acc).abs()
    assert (err <= tol)[ok].all(), f"weights: {(err / tol)[ok].max().item():.3g} of the tolerance"
    return ok


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("what", ["query", "key", "old key"])
def test_weights_of_slots_that_a_spoiled_row_does_not_see(what, bs, dt):
    """A row that is NaN adds NaN to the slots that it sees, and nothing to the others of the same tiles: in front of the
    window, behind the sinks, behind its own place, behind the sequence's end."""
    lens, d, window, sink = [200, 37], 64, 75, 4
    cache, table, _, _, _ = filled("int8", dt, lens, 2, bs, d, seed=4)
    q = normal(2, 3, 4, d, seed=5, dt=dt)
    if what == "query":
        q[0, 1, 2, 7] = math.nan
    else:  # the block of the newest slots, or one in the middle of the window that the last rows still see
        cache.k_scale[table[0, (199 if what == "key" else 150) // bs].item(), 0] = math.nan
    seen = check_spoiled_attn(cache, table, lens, q, window, sink)
    assert not seen[0].all() and seen[1].all() and seen[0, :, 4:32].all() and seen[0, :, 200:].all()
    check_spoiled_attn(cache, table, lens, q, None, 0)


@pytest.mark.parametrize("kind,dt", [("int8", "bf16"), ("e4m3", "fp16")])
@pytest.mark.parametrize("bs", [16, 128])
def test_values_that_are_not_finite_leave_weights_and_log_sum_exp_alone(bs, kind, dt):
    """A block of V whose scale is NaN or infinite makes the outputs NaN that see it; what depends on K alone stays."""
    lens, d, window, sink = [300, 50], 128, 135, 2
    for bad in (math.nan, math.inf):
        cache, table, _, _, _ = filled(kind, dt, lens, 2, bs, d, seed=6)
        for b, slot, h in ((0, 145, 1), (0, 299, 0), (1, 0, 0)):
            page = table[b, slot // bs].item()
            cache.v_scale[page, h] = bad
            cache.v.view(torch.uint8)[page, h] = 0  # (as cache_append stores them)
        q = normal(2, 20, 4, d, seed=7, dt=dt)
        check_spoiled_attn(cache, table, lens, q, window, sink)
        check_spoiled_attn(cache, table, lens, q[:, :1], None, 0)


@pytest.mark.parametrize("kind,bs", [("int8", 16), ("e4m3", 64)])
@pytest.mark.parametrize("small,large", [(-100, -100), (-100, 0), (-100, 60), (-60, 40), (80, 80)])
def test_values_of_very_different_magnitude(small, large, kind, bs):
    """V's scales as far apart as 2^-100 (a block of zeros, or nearly) and 2^80: the log-sum-exp and the weights do not know about V.
    `more`: exponents carry the scale's logarithm, up to 2^7 large; at most four roundings of half a step there, 2^-18 each
    (2^-17 behind an addition), times ln 2 and 2."""
    lens, d = [700, 90], 64
    cache, table, _, _, _ = filled(kind, "bf16", lens, 2, bs, d, seed=8)
    some = (torch.arange(cache.v.shape[0], device="cuda") % 3 == 0)[:, None]
    cache.v_scale.copy_(torch.where(some, 2.0 ** large, 2.0 ** small))
    q = normal(2, 2, 8, d, seed=9, dt="bf16")
    check_spoiled_attn(cache, table, lens, q, None, 0, more=2.0 ** -15)
    check_spoiled_attn(cache, table, lens, q[:, :1], 60, 1, more=2.0 ** -15)


def check_spoiled_sums(q, k, lse, window, sink, lens):
    """Packed sums against the definition: NaN exactly where that has NaN.  (Tolerance: test_gpu_cache.py.)"""
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32).cuda()
    got = _ops().attn_weight_sums(q.cuda(), k.cuda(), lse.cuda(), window, sink, cu_seqlens=cu).cpu().double()
    want, most, _ = R.weight_sums(q.double(), k.double(), lse, window, sink, None, lens)
    same_nan(got, want, "sums")
    e = (q.shape[-1] + 8) * 2.0 ** -24 * most
    rel = e + 2.0 ** -24 * (most + lse[torch.isfinite(lse)].abs().max().item()) + 2.0 ** -20 + 128 * 2.0 ** -24 + 2.0 ** -23
    ok = torch.isfinite(want)
    assert ((got - want).abs() <= rel * want)[ok].all(), f"{((got - want).abs() / want)[ok & (want > 0)].max().item():.3g} instead of {rel:.3g}"
    return got, want


@pytest.mark.parametrize("dt,d", [("bf16", 64), ("fp16", 128)])
def test_sums_of_keys_that_a_spoiled_query_does_not_see(dt, d):
    """A NaN log-sum-exp spoils the keys that its query sees: none in front of the window, behind the query or in another sequence."""
    lens, window, sink = [4, 4, 130, 600, 90], 100, 3
    t = sum(lens)
    q, k = normal(t, 4, d, seed=1, dt=dt), normal(t, 2, d, seed=2, dt=dt)
    lse = 3 + normal(4, t, seed=3, dt="bf16").float()
    for head, i in ((0, 5), (1, 60), (2, 500), (3, 137), (3, t - 1)):
        lse[head, i] = math.nan
    got, want = check_spoiled_sums(q, k, lse, window, sink, lens)
    assert torch.isfinite(got[:, :4]).all() and torch.isnan(got[0, 4:6]).all()
    # the query NaN besides, as it comes out of a model
    q[5, 0], q[500, 2, 3] = math.nan, math.nan
    check_spoiled_sums(q, k, lse, window, sink, lens)


@pytest.mark.parametrize("dt,d", [("bf16", 128), ("fp16", 64)])
def test_queries_that_saw_nothing_add_nothing(dt, d):
    """log-sum-exp -inf: nothing from that query, to the last bit and whatever its scores are (the attention's own answer
    for a row that is not finite)."""
    lens, window, sink = [700, 400], 500, 2
    t = sum(lens)
    q, k = normal(t, 4, d, seed=1, dt=dt), normal(t, 2, d, seed=2, dt=dt)
    lse = 3 + normal(4, t, seed=3, dt="bf16").float()
    lse[:, 300:] = -math.inf
    got, want = check_spoiled_sums(q, k, lse, window, sink, lens)
    assert (got[:, 300:] == 0).all() and (want[:, :300] > 0).all()
    q[320, 1, 5], q[699, 3], q[1000, 0, 0] = math.nan, math.nan, math.nan
    k[310, 0, 9] = math.nan   # (seen by queries that add nothing)
    check_spoiled_sums(q, k, lse, window, sink, lens)


def test_sums_behind_the_attention_of_a_prompt_with_a_query_that_is_not_finite():
    import ring_swa.compiled  # noqa: F401  (registers the operator)
    n, hq, hkv, d, window, sink = 500, 4, 2, 128, 90, 2
    q, k, v = (normal(1, n, h, d, seed=i, dt="bf16").cuda() for i, h in enumerate((hq, hkv, hkv)))
    q[0, 333, 2, 7] = math.nan
    _, lse = torch.ops.ring_swa.swa_fwd(q, k, v, window, sink, d ** -0.5, None)
    assert torch.isneginf(lse[0, 2, 333])
    got = _ops().attn_weight_sums(q, k, lse, window, sink)
    want, _, _ = R.weight_sums(q[0].cpu().double(), k[0].cpu().double(), lse[0].cpu(), window, sink, None, [n])
    assert torch.isfinite(want).all() and ((got[0].cpu().double() - want).abs() <= 1e-4 * want).all()  # (16-bit weights in the forward's sum)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 32, 64])
def test_blocks_behind_the_window_may_be_given_back(bs, kind):
    """Entries of blocks without a slot that any query sees are not looked at, for every block size: the same bits, nothing reported."""
    from ring_swa import _kernels as K
    ops = _ops()
    lens, d = [1000, 333, 70, 5], 64
    cache, table, _, _, _ = filled(kind, "bf16", lens, 2, bs, d, seed=2)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    for window, sink, queries in ((200, 0, 1), (111, 1, 1), (250, 17, 4), (0, 0, 1), (40, 33, 2)):
        freed = table.clone()
        for i, m in enumerate(lens):
            for j in range((m + bs - 1) // bs):
                if j * bs >= sink and (j + 1) * bs <= max(0, m - queries) - window:
                    freed[i, j] = -1
        assert (freed != table).any()
        q = normal(4, queries, 8, d, seed=3, dt="bf16").cuda()
        ws = [torch.zeros(4, 2, table.shape[1] * bs, device="cuda") for _ in range(2)]
        a, b = (ops.cache_attn(q, cache, t.cuda(), n, window_size=window, num_sink_tokens=sink, weights=w, return_lse=True)
                for t, w in ((table, ws[0]), (freed, ws[1])))
        K.check_device_status()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(*ws)
        assert torch.isfinite(a[0]).all()
        # an entry that is seen is still looked at
        bad = freed.clone()
        bad[0, (lens[0] - 1) // bs] = -1
        ops.cache_attn(q, cache, bad.cuda(), n, window_size=window, num_sink_tokens=sink)
        with pytest.raises(RuntimeError, match="code 110"):
            K.check_device_status()


def test_a_block_table_whose_rows_are_one():
    """Sequences that share all their blocks (one prompt, several questions): a row expanded over the batch, where it is only read."""
    ops = _ops()
    lens, bs, d, batch = [300], 16, 64, 5
    cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=2, spare=100)
    one, n = table.cuda(), torch.tensor([300, 17, 299, 0, 160], dtype=torch.int32).cuda()
    many, apart = one.expand(batch, -1), one.repeat(batch, 1)
    q = normal(batch, 2, 4, d, seed=3, dt="bf16").cuda()
    assert torch.equal(ops.cache_attn(q, cache, many, n), ops.cache_attn(q, cache, apart, n))
    for x, y in zip(ops.cache_read(cache, many, n, 300), ops.cache_read(cache, apart, n, 300)):
        assert torch.equal(x, y)
    free = sorted(set(range(cache.k.shape[0])) - set(table.flatten().tolist()))
    new = torch.tensor(free[:5 * batch], dtype=torch.int32).view(batch, 5).cuda()
    w = torch.rand(batch, 2, table.shape[1] * bs, generator=torch.Generator().manual_seed(0)).cuda()
    a = [x.clone() for x in ops.cache_evict(cache, many, n, w, 80, new, 1, 3)]
    kept = [x.clone() for x in ops.cache_read(cache, new, a[0], 80)]
    b = ops.cache_evict(cache, apart, n, w, 80, new, 1, 3)
    for x, y in zip([*a, *kept], [*b, *ops.cache_read(cache, new, b[0], 80)]):
        assert torch.equal(x, y)
    # where blocks are written to, rows have to be their own
    k = normal(batch, 1, 2, d, seed=4, dt="bf16").cuda()
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_append(cache, k, k, many, n)
    with pytest.raises(ValueError, match="overlap"):
        ops.cache_evict(cache, many, n, w, 80, new[:1].expand(batch, -1), 1, 3)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_scale_from_elsewhere_is_kept_while_the_new_tokens_fit(kind):
    """Blocks filled elsewhere, whose scales are no powers of two: a new token that they hold leaves scale and older tokens as
    they are; one that they do not hold moves the block to the least power of two, rounded once.  (Bytes: within half a step, and
    2^-22 for the reciprocal's and the product's roundings.)"""
    ops = _ops()
    top = R.TOP[kind]
    heads, bs, d, used = 2, 32, 64, 20
    sizes = torch.tensor([0.75, 0.9, 1.37e-3, 3.1, 2.0 ** -130, 2.0 ** -100])
    blocks = len(sizes)
    cache = make(kind, blocks, heads, bs, d, seed=1)
    g = torch.Generator().manual_seed(2)
    stored = torch.randint(-100, 101, (2, blocks, heads, bs, d), generator=g).float()
    for x, s, y in ((cache.k, cache.k_scale, stored[0]), (cache.v, cache.v_scale, stored[1])):
        x.copy_(y.to(R.TORCH[kind]))
        s.copy_(sizes[:, None])
    before = host(cache)
    table = torch.arange(blocks, dtype=torch.int32)[:, None].cuda()
    n = torch.full((blocks,), used, dtype=torch.int32).cuda()
    new = torch.rand(2, blocks, heads, d, generator=g) * 2 - 1
    new[..., 0] = 1
    # k: 0.98 of what the scale holds; v: 1.3 times as much
    k, v = ((x * m * top * sizes[:, None, None]).bfloat16() for x, m in zip(new, (0.98, 1.3)))
    ops.cache_append(cache, k[:, None].cuda(), v[:, None].cuda(), table, n)
    got = host(cache)
    for name, x in (("k", k), ("v", v)):
        for b in range(blocks):
            least = R.scale_for(x[b].double().abs().max().item(), kind)
            old = sizes[b].item()
            fits = name == "k" and old >= 2.0 ** -100
            want = old if fits else least
            assert (got[name + "_scale"][b] == want).all(), (name, old, got[name + "_scale"][b])
            held = got[name][b]
            rows = torch.cat([before[name][b][:, :used] * old / want, x[b].double()[:, None] / want], 1)
            if fits:
                assert torch.equal(held[:, :used], before[name][b][:, :used])
            step = torch.ones_like(rows) if kind == "int8" else torch.exp2((torch.frexp(rows.abs().clamp_min(2.0 ** -6)).exponent - 4).double())
            assert ((held[:, :used + 1] - rows).abs() <= 0.5 * step + 2.0 ** -22 * rows.abs()).all()
            assert torch.equal(held[:, used + 1:], before[name][b][:, used + 1:])


def test_streams_from_elsewhere_leave_nothing_behind():
    """A stream that another library made may be destroyed, and its handle given to another stream, while its work still runs:
    nothing that two calls must not share is kept under the handle."""
    import gc
    from cuda.bindings import runtime as rt
    ops = _ops()
    lens, bs, d = [9000], 64, 128
    cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=1)
    args = (normal(1, 1, 8, d, seed=2, dt="bf16").cuda(), cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    want = ops.cache_attn(*args)
    torch.cuda.synchronize()
    gc.collect()
    held = torch.cuda.memory_allocated()
    handles = []
    for _ in range(4):  # four that live at once: handles that no earlier call has seen
        err, s = rt.cudaStreamCreateWithFlags(rt.cudaStreamNonBlocking)
        assert int(err) == 0
        handles.append(s)
    for s in handles:
        with torch.cuda.stream(torch.cuda.ExternalStream(int(s))):
            outs = [ops.cache_attn(*args) for _ in range(3)]
        rt.cudaStreamSynchronize(s)
        assert all(torch.equal(x, want) for x in outs)
        del outs
    gc.collect()
    assert torch.cuda.memory_allocated() == held
    for s in handles:
        rt.cudaStreamDestroy(s)


def test_weights_laid_out_by_heads():
    ops = _ops()
    lens, bs, d = [300, 40, 77], 32, 64
    cache, table, _, _, _ = filled("int8", "bf16", lens, 2, bs, d, seed=2, spare=20)
    n, q = torch.tensor(lens, dtype=torch.int32).cuda(), normal(3, 2, 4, d, seed=3, dt="bf16").cuda()
    a = torch.rand(3, 2, table.shape[1] * bs, generator=torch.Generator().manual_seed(0)).cuda()
    b = torch.zeros(2, 3, a.shape[2] + 3, device="cuda")[..., :a.shape[2]].transpose(0, 1).copy_(a)
    for w in (a, b):
        ops.cache_attn(q, cache, table.cuda(), n, weights=w)
    assert torch.equal(a, b) and not b.is_contiguous()
    free = sorted(set(range(cache.k.shape[0])) - set(table.flatten().tolist()))
    new = torch.tensor(free[:6], dtype=torch.int32).view(3, 2).cuda()
    for x, y in zip(*([z.clone() for z in ops.cache_evict(cache, table.cuda(), n, w, 50, new, 1, 3)] for w in (a, b))):
        assert torch.equal(x, y)


def test_sums_of_one_key_head_for_all_and_of_a_prompt_without_a_window():
    """A key expanded over the heads' dimension, as a slice of a batch; against the 64-bit sums of the same."""
    b, s, hq, d = 2, 2500, 4, 64
    fused = normal(b, s, hq + 1, d, seed=1, dt="bf16")
    q, k = fused[:, :, :hq], fused[:, :, hq:]
    for heads in (1, 3):   # (an expanded dimension has to be laid out before a tensor map takes it)
        kk = k.expand(b, s, heads, d)
        qq = q[:, :, :heads]
        lse = torch.empty(b, heads, s)
        for i in range(b):
            for h in range(heads):
                x = (qq[i, :, h].double() @ k[i, :, 0].double().T) * d ** -0.5
                lse[i, h] = x.masked_fill(torch.ones(s, s).triu(1).bool(), -math.inf).logsumexp(1).float()
        got = _ops().attn_weight_sums(qq.cuda(), kk.cuda(), lse.cuda(), None).cpu().double()
        for i in range(b):
            want, most, _ = R.weight_sums(qq[i].double(), kk[i].double(), lse[i], None, 0, None, [s])
            rel = (d + 8) * 2.0 ** -24 * most + 2.0 ** -24 * (most + lse.abs().max().item()) + 2.0 ** -20 + 128 * 2.0 ** -24 + 2.0 ** -23
            assert ((got[i] - want).abs() <= rel * want).all()


def test_sums_of_a_prompt_are_what_its_attention_over_a_cache_adds_up():
    """Every query of a short prompt through cache_attn(weights=) and the prompt through attn_weight_sums, on the values that the
    cache holds.  Tolerances of both sides: 2 e + 2^-18 + rows * 2^-24 and e + 2^-20 + 2^-16 (test_gpu_cache.py), the log-sum-exp's
    e + 2^-20 (1 + |lse|) besides."""
    ops = _ops()
    n, hq, hkv, d, bs, window, sink = 150, 8, 2, 128, 32, 60, 3
    cache, table, _, _, _ = filled("int8", "bf16", [n], hkv, bs, d, seed=3)
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    k, _ = ops.cache_read(cache, table.cuda(), lens, n)      # (int8 times a power of two: exact in bf16)
    q = normal(1, n, hq, d, seed=4, dt="bf16")
    w = torch.zeros(1, hkv, table.shape[1] * bs, device="cuda")
    _, lse = ops.cache_attn(q.cuda(), cache, table.cuda(), lens, window_size=window, num_sink_tokens=sink, weights=w, return_lse=True)
    got = ops.attn_weight_sums(q.cuda(), k, lse, window, sink)
    _, want_lse, want, _, most = R.attn(host(cache), table, [n], q.double(), window, sink)
    e = (d + 8) * 2.0 ** -24 * most
    rel = 2 * e + 2.0 ** -18 + n * hq * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -20 * (1 + want_lse.abs().max().item())
    for x in (got.cpu().double(), w[..., :n].cpu().double()):
        assert ((x - want).abs() <= rel * want).all()


def test_scales_of_a_layer_among_others():
    """k_scale and v_scale as slices of one tensor for all layers: aligned to 4 bytes, no more."""
    ops = _ops()
    lens, bs, d = [70, 21], 16, 64
    cache, table, k, v, cu = filled("e4m3", "bf16", lens, 1, bs, d, seed=3, spare=6)
    blocks = cache.k.shape[0]
    both = torch.full((3, 2, blocks, 1), math.nan, device="cuda").flatten()[1:1 + 4 * blocks].view(2, 2, blocks, 1)
    layer = ops.KVCache(cache.k.clone(), cache.v.clone(), both[1, 0], both[1, 1])
    assert (layer.k_scale.data_ptr() | layer.v_scale.data_ptr()) % 16 != 0
    n, t = torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda()
    ops.cache_append(layer, k.cuda(), v.cuda(), t, n * 0, cu_seqlens=cu.cuda())
    q = normal(2, 1, 4, d, seed=4, dt="bf16").cuda()
    assert torch.equal(ops.cache_attn(q, layer, t, n), ops.cache_attn(q, cache, t, n))
    free = sorted(set(range(blocks)) - set(table.flatten().tolist()))
    new, w = torch.tensor(free[:4], dtype=torch.int32).view(2, 2).cuda(), torch.rand(2, 1, table.shape[1] * bs, device="cuda")
    a, b = (ops.cache_evict(c, t, n, w, 20, new) for c in (cache, layer))
    for x, y in zip([*a, *ops.cache_read(cache, new, a[0], 20)], [*b, *ops.cache_read(layer, new, b[0], 20)]):
        assert torch.equal(x, y)
