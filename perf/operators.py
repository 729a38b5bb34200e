"""Decoding from a key/value cache held in 8 bits, as measurable cases.

A model that was run with the sliding-window or StreamingLLM functions of ring_swa goes on token by token: its keys and
values lie in a cache of blocks in 8 bits, one scale for each block of tokens and head (int8: value = q * scale with
|q| <= 127; e4m3: the same with |q| <= 448).  A scale is the least power of two that keeps the block's values in that range:
bringing values to another scale or back to 16 bits then rounds nothing but what the coarser scale cannot hold, and a
token that moves from block to block does not lose a little each time.  The operators around that cache:

  append   quantise new tokens (one per sequence, or whole prompts) into the blocks of a block table
  read     bring a cached prefix back to 16 bits, for a prompt that continues it
  attn     attention of the newest token(s) of each sequence over its cached tokens: window, sink tokens, grouped heads;
           optionally adds the weight that every cached token received to a running sum
  sums     the same running sums for a prompt: how much weight the queries of a prompt gave to each of its keys
  evict    keep the sink tokens, the newest tokens and those of largest accumulated weight, packed into new blocks

The fields of a case:
  op                  one of the above
  batch, hq, hkv, d   sequences, query heads, key/value heads, head dimension
  lens                the sequences' lengths, as text: tokens in the cache (append: before the call; sums: of the prompts)
  new                 append: new tokens per sequence, as text; attn: queries per sequence (the newest tokens, a number)
  bs, kind            tokens per block; int8 | e4m3
  dtype               bf16 | fp16: queries, new keys and values, results
  window, sink        attention: a token sees itself, the `window` tokens before it (-1: all) and the first `sink` tokens
  weights             attn: add the weights up
  budget, recent      evict: tokens that stay, and how many of them are the newest
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_KINDS = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def _ops():
    path = os.path.join(os.getcwd(), "ring-sliding-window-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ring_swa import ops
    return ops


# ---------------------------------------------------------------- the cases

def _case(name, op, lens, heads, d, **more):
    lens = [lens] if isinstance(lens, int) else list(lens)
    c = {"name": name, "op": op, "batch": len(lens), "lens": ",".join(map(str, lens)), "hq": heads[0], "hkv": heads[1], "d": d}
    c.update(more)
    return c


def _spread(n, lo, hi):
    """n lengths between lo and hi, evenly over their logarithm, long and short ones mixed."""
    return [int(lo * (hi / lo) ** (((i * 13) % n) / max(1, n - 1))) for i in range(n)]


def listed():
    return [
        # the next token of one short chat with a small model (64-wide heads): latency is all there is
        _case("attn_one_513_d64", "attn", 513, (4, 4), 64, new=1, bs=16, kind="int8", dtype="bf16", window=-1, sink=0, weights=False),
        # one decoding step of a serving batch: 32 requests of 300 to 8192 tokens, grouped heads
        _case("attn_batch_8k", "attn", _spread(32, 300, 8192), (32, 8), 128, new=1, bs=64, kind="e4m3", dtype="bf16", window=-1, sink=0, weights=False),
        # StreamingLLM far into four long streams, four tokens verified at once: window of 8192, 4 sink tokens
        _case("attn_128k_sink_4", "attn", [131072, 131001, 99999, 65537], (32, 8), 128, new=4, bs=128, kind="int8", dtype="fp16", window=8192, sink=4, weights=False),
        # two long contexts without a window, with the weights added up for a later eviction; eight query heads per key head
        _case("attn_64k_weights", "attn", [65536, 60001], (64, 8), 128, new=1, bs=32, kind="int8", dtype="bf16", window=-1, sink=0, weights=True),
        # the cache side of a decoding step: one token for each of 64 requests, blocks filled to all degrees
        _case("append_step_64", "append", _spread(64, 5, 9000), (32, 8), 128, new=",".join(["1"] * 64), bs=32, kind="int8", dtype="bf16"),
        # four prompts of very different lengths go into the cache in one call
        _case("append_prompts_22k", "append", [0, 0, 0, 0], (32, 8), 128, new="512,2000,4000,16000", bs=64, kind="e4m3", dtype="bf16"),
        # the prefix of one short chat, read back for its next turn
        _case("read_777_d64", "read", 777, (4, 2), 64, bs=16, kind="e4m3", dtype="fp16"),
        # four long documents read back for a question about each
        _case("read_16k_batch", "read", [16384, 16001, 12000, 16384], (32, 8), 128, bs=64, kind="int8", dtype="bf16"),
        # weights of a short prompt of a small model
        _case("sums_1k_d64", "sums", 1024, (4, 4), 64, dtype="bf16", window=128, sink=0),
        # weights of a long prompt, grouped heads, window of 4096 and sink tokens
        _case("sums_16k_sink", "sums", 16384, (32, 8), 128, dtype="bf16", window=4096, sink=4),
        # one chat that outgrew its budget
        _case("evict_1500_d64", "evict", 1500, (4, 4), 64, bs=16, kind="int8", dtype="bf16", budget=512, sink=4, recent=128),
        # a batch of long requests cut to half
        _case("evict_16k_batch", "evict", [16384, 16384, 15001, 16384, 12345, 16384, 9000, 8000], (32, 8), 128, bs=64, kind="e4m3", dtype="bf16", budget=8192,
              sink=4, recent=1000),
    ]


_HEADS = [(4, 4), (8, 2), (16, 16), (16, 2), (32, 8), (32, 4), (64, 8), (12, 4)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges above: 1 to 64 sequences of one token to 131072 tokens, every head layout, block size and type."""
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(("attn", "attn", "attn", "append", "read", "sums", "evict"))
        heads, d = rng.choice(_HEADS), rng.choice((64, 128, 128))
        batch = _log_int(rng, 1, 64)
        top = _log_int(rng, 16, 131072)
        lens = [_log_int(rng, max(1, top // 16), top) for _ in range(batch)]
        more = {"bs": rng.choice((16, 32, 64, 128)), "kind": rng.choice(("int8", "e4m3")), "dtype": rng.choice(("bf16", "bf16", "fp16"))}
        if op == "attn":
            window = rng.choice((-1, -1, _log_int(rng, 16, 16384)))
            more.update(new=rng.choice((1, 1, 1, 2, 5, 8)), window=window, sink=0 if window < 0 else rng.choice((0, 1, 4)), weights=rng.random() < 0.3)
            lens = [max(n, more["new"]) for n in lens]
        elif op == "append":
            lens = [rng.choice((0, n)) for n in lens]
            step = rng.random() < 0.5
            more["new"] = ",".join(str(1 if step else _log_int(rng, 1, 4096)) for _ in lens)
        elif op == "sums":
            lens = [max(16, n) for n in lens[:rng.choice((1, 1, 2, 5))]]
            more = {"dtype": more["dtype"], "window": rng.choice((_log_int(rng, 16, 16384), max(lens))), "sink": rng.choice((0, 1, 4))}
        elif op == "evict":
            budget = max(16, int(top * rng.uniform(0.1, 0.8)))
            more.update(budget=budget, sink=rng.choice((0, 1, 4)), recent=rng.choice((0, budget // 4, budget // 8)))
        c = _case("", op, lens, heads, d, **more)
        del c["name"]
        # (a bound on what the 32-bit forms hold at once, besides the cost)
        if _cost(c) <= most[op] and _most_held(c) <= 4e9:
            return c


# ---------------------------------------------------------------- sizes

def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _blocks(n, bs):
    return (n + bs - 1) // bs


def _seen(n, q, window, sink):
    """(cached tokens that the last q of n tokens see between them, visible (query, key) pairs)."""
    q = min(q, n)
    if window < 0:
        return n, sum(n - q + i + 1 for i in range(q))
    lo = max(0, n - q - window)
    union = n - lo + min(sink, lo)
    pairs = 0
    for p in range(n - q, n):
        left = max(0, p - window)
        pairs += p + 1 - left + min(sink, left)
    return union, pairs


def _prompt_pairs(n, window, sink):
    full = min(n, window + 1)
    pairs = full * (full + 1) // 2 + (n - full) * (window + 1)
    return pairs + sum(max(0, n - (window + 1 + s)) for s in range(sink))


def work(case):
    lens, hq, hkv, d = _ints(case["lens"]), case["hq"], case["hkv"], case["d"]
    op = case["op"]
    if op == "sums":
        t = sum(lens)
        pairs = sum(_prompt_pairs(n, case["window"], case["sink"]) for n in lens)
        return {"bytes": t * (hq + hkv) * d * 2 + t * hq * 4 + t * hkv * 4, "flops": 2 * pairs * hq * d}
    bs = case["bs"]
    row = hkv * d * 2                       # K and V of a token, 8 bits
    scale = 2 * hkv * 4                     # the two scales of a block, all heads
    if op == "attn":
        n, b, f = case["new"], 0, 0
        for x in lens:
            tokens, pairs = _seen(x, n, case["window"], case["sink"])
            b += tokens * row + _blocks(tokens, bs) * (scale + 4) + 2 * n * hq * d * 2
            b += tokens * hkv * 8 if case["weights"] else 0
            f += 4 * pairs * hq * d
        return {"bytes": b, "flops": f}
    if op == "append":
        b = 0
        for x, n in zip(lens, _ints(case["new"])):
            old = x % bs
            # the new tokens in and out, the older tokens of the first block in and out, all of them read back
            b += n * row * 3 + old * row * 2 + _blocks(old + n, bs) * (scale + 4) + (old + n) * row * 2
        return {"bytes": b, "flops": 0}
    if op == "read":
        return {"bytes": sum(x * row + _blocks(x, bs) * (scale + 4) for x in lens) + len(lens) * max(lens) * row * 2, "flops": 0}
    b = 0
    for x in lens:
        keep = min(x, case["budget"])
        # weights in; kept rows in, out and read back; kept weights and indices out
        b += x * hkv * 4 + keep * row * 4 + keep * hkv * 8 + (_blocks(x, bs) + _blocks(keep, bs)) * (scale + 4)
    return {"bytes": b, "flops": 0}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _most_held(case):
    lens = _ints(case["lens"])
    if case["op"] == "sums":
        return 4 * (case["hq"] // case["hkv"]) * sum(lens) ** 2
    if case["op"] == "append":
        new = _ints(case["new"])
        return 4 * case["hkv"] * case["d"] * (len(lens) * (max(new) + 2 * case["bs"]) + sum(lens) + sum(new))
    return 4 * case["hkv"] * case["d"] * len(lens) * (max(lens) + case["bs"])


# ---------------------------------------------------------------- inputs

def _quantise(x, kind):
    """(8-bit values, scales) of blocks [..., tokens, d]."""
    scale = _scale_for(x.abs().amax(dim=(-2, -1)), kind)
    return _to8(x * (1.0 / scale)[..., None, None], kind), scale


def _scale_for(amax, kind):
    """The least power of two s with amax <= top * s."""
    m, e = torch.frexp(amax)
    top_m, top_e = math.frexp(_KINDS[kind][1])
    e = torch.where(amax > 0, e - top_e + (m > top_m), -100).clamp_min(-100)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _to8(x, kind):
    dt, top = _KINDS[kind]
    x = x.clamp(-top, top)
    return x.round().to(dt) if kind == "int8" else x.to(dt)


def _make_cache(g, blocks, hkv, bs, d, kind):
    """Blocks as a program has them after its prompts: normally distributed keys and values, some channels larger."""
    out = {}
    for name in ("k", "v"):
        x = torch.randn(blocks, hkv, bs, d, generator=g, device="cuda")
        if name == "k":
            x[..., :: max(1, d // 8)] *= 2.5
        out[name], out[name + "_scale"] = _quantise(x, kind)
    return out


def _tables(g, counts, spare=0):
    """A block table for sequences of `counts` blocks: blocks in no order, rows padded with -1."""
    total = sum(counts)
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, total + spare


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    op, lens, hq, hkv, d = case["op"], _ints(case["lens"]), case["hq"], case["hkv"], case["d"]
    st = {"case": case}
    if op == "sums":
        t = sum(lens)
        # q and k as slices of one projection
        qk = normal(t, hq + hkv, d)
        st["q"], st["k"] = qk[:, :hq], qk[:, hq:]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu"] = _i32(cu)
        st["lse"] = torch.cat([_scores(st, h).logsumexp(-1) for h in range(hkv)])
        return st
    bs, kind = case["bs"], case["kind"]
    if op == "append":
        new = _ints(case["new"])
        counts = [_blocks(a + n, bs) for a, n in zip(lens, new)]
        st["table"], blocks = _tables(g, counts, spare=1)  # (the last block is in no table)
        st["cache"] = _make_cache(g, blocks, hkv, bs, d, kind)
        st["k"], st["v"] = normal(sum(new), hkv, d), normal(sum(new), hkv, d)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        st["cu"], st["lens"] = _i32(cu), _i32(lens)
        # the blocks that the call touches, to read them back
        most = max(_blocks(a % bs + n, bs) for a, n in zip(lens, new))
        touched = torch.full((len(lens), most), -1, dtype=torch.int32, device="cuda")
        for i, (a, n) in enumerate(zip(lens, new)):
            k = _blocks(a % bs + n, bs)
            touched[i, :k] = st["table"][i, a // bs:a // bs + k]
        st["touched"], st["touched_lens"] = touched, _i32([a % bs + n for a, n in zip(lens, new)])
        return st
    st["table"], blocks = _tables(g, [_blocks(n, bs) for n in lens])
    if op == "evict":
        keep = [_blocks(min(n, case["budget"]), bs) for n in lens]
        new_table, more = _tables(g, keep, spare=1)  # (the last block is in no table)
        st["new_table"] = torch.where(new_table >= 0, new_table + blocks, new_table)
        blocks += more
        # accumulated weights: a few tokens hold most, and equal values occur
        st["weights"] = (torch.randn(len(lens), hkv, st["table"].shape[1] * bs, generator=g, device="cuda") * 2).exp().bfloat16().float()
    st["cache"] = _make_cache(g, blocks, hkv, bs, d, kind)
    st["lens"] = _i32(lens)
    if op == "attn":
        st["q"] = normal(len(lens), case["new"], hq, d)
        if case["weights"]:
            st["weights"] = torch.rand(len(lens), hkv, st["table"].shape[1] * bs, generator=g, device="cuda")
    return st


# ---------------------------------------------------------------- the plain forms

def _scores(st, h):
    """Scores of one key/value head's group in a packed batch of prompts [group, tokens, tokens], hidden ones -inf."""
    case = st["case"]
    grp, t = case["hq"] // case["hkv"], st["q"].shape[0]
    s = torch.matmul(st["q"][:, h * grp:(h + 1) * grp].float().transpose(0, 1), st["k"][:, h].float().t()) * case["d"] ** -0.5
    pos = torch.arange(t, device="cuda")
    seq = torch.searchsorted(st["cu"].long(), pos, right=True) - 1
    start = st["cu"].long()[seq]
    gap = pos[:, None] - pos[None]
    seen = (seq[:, None] == seq[None]) & (gap >= 0) & ((gap <= case["window"]) | (pos - start < case["sink"])[None])
    return s.masked_fill_(~seen, -math.inf)


def _dense(cache, table, name):
    """Cached values in 32 bits [batch, blocks * block size, heads, d]."""
    at = table.long().clamp_min(0)
    x = cache[name][at].float() * cache[name + "_scale"][at][..., None, None]
    b, n, h, bs, d = x.shape
    return x.permute(0, 1, 3, 2, 4).reshape(b, n * bs, h, d)


def _plain_read(cache, table, lens, most, dt):
    out = []
    for name in ("k", "v"):
        x = _dense(cache, table, name)[:, :most]
        seen = torch.arange(x.shape[1], device="cuda")[None] < lens[:, None]
        out.append(torch.where(seen[..., None, None], x, 0.0).to(dt))
    return tuple(out)


def _plain_append(st):
    case, cache, table = st["case"], st["cache"], st["table"]
    bs, kind = case["bs"], case["kind"]
    lens, cu = st["lens"].long(), st["cu"].long()
    first, n = lens // bs, cu[1:] - cu[:-1]
    blocks = first[:, None] + torch.arange(st["touched"].shape[1], device="cuda")[None]          # [batch, touched]
    slot = blocks[..., None] * bs + torch.arange(bs, device="cuda")                                # [batch, touched, bs]
    token = slot - lens[:, None, None]
    is_new, is_old = (token >= 0) & (token < n[:, None, None]), token < 0
    live = blocks * bs < (lens + n)[:, None]
    page = torch.where(live, table.long().gather(1, blocks.clamp_max(table.shape[1] - 1)), cache["k"].shape[0] - 1)
    source = (cu[:-1, None, None] + token).clamp(0, st["k"].shape[0] - 1)
    for name in ("k", "v"):
        x = torch.where(is_new[..., None, None], st[name][source].float(), 0.0).permute(0, 1, 3, 2, 4)   # [batch, touched, heads, bs, d]
        held, scale = cache[name][page], cache[name + "_scale"][page]
        before = torch.where(is_old.any(-1)[..., None], scale, 0.0)
        after = torch.maximum(_scale_for(x.abs().amax(dim=(-2, -1)), kind), before)
        x = torch.where(is_old[:, :, None, :, None], held.float() * before[..., None, None], x)
        x = _to8(x * (1.0 / after)[..., None, None], kind)
        written = (is_new | is_old)[:, :, None, :, None]
        # (through bytes: not every type can be selected from)
        cache[name].view(torch.uint8)[page] = torch.where(written, x.view(torch.uint8), held.view(torch.uint8))
        cache[name + "_scale"][page] = after


def _plain_attn(st):
    case, cache = st["case"], st["cache"]
    b, n, hq, d = st["q"].shape
    hkv = case["hkv"]
    k, v = _dense(cache, st["table"], "k"), _dense(cache, st["table"], "v")
    q = st["q"].float().view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, hq // hkv * n, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)).view(b, hkv, hq // hkv, n, -1) * d ** -0.5
    slot = torch.arange(k.shape[1], device="cuda")
    p = st["lens"].long()[:, None] - n + torch.arange(n, device="cuda")[None]                      # [batch, n]
    gap = p[..., None] - slot
    seen = gap >= 0
    if case["window"] >= 0:
        seen &= (gap <= case["window"]) | (slot < case["sink"])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    w = (s - s.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-38)
    v = torch.where((slot < st["lens"][:, None])[..., None, None], v, 0.0)
    out = torch.matmul(w.view(b, hkv, -1, w.shape[-1]), v.transpose(1, 2)).view(b, hkv, hq // hkv, n, d)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d).to(st["q"].dtype)
    if not case["weights"]:
        return out
    st["weights"] += w.sum(dim=(2, 3))
    return out, st["weights"]


def _plain_sums(st):
    # (a head at a time: the scores of all of them at once take too much memory)
    lse, grp = st["lse"], st["case"]["hq"] // st["case"]["hkv"]
    return torch.stack([(_scores(st, h) - lse[h * grp:(h + 1) * grp, :, None]).exp().sum(dim=(0, 1)) for h in range(st["case"]["hkv"])])


def _plain_evict(st):
    case, cache = st["case"], st["cache"]
    bs, kind, budget = case["bs"], case["kind"], case["budget"]
    lens, w = st["lens"].long(), st["weights"]
    slot = torch.arange(w.shape[-1], device="cuda")
    must = (slot < case["sink"]) | (slot >= lens[:, None] - case["recent"])
    rank = torch.where(must[:, None], math.inf, w)
    rank = torch.where((slot < lens[:, None])[:, None], rank, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]                  # [batch, heads, budget]
    new_lens = lens.clamp_max(budget)
    cap = st["new_table"].shape[1] * bs
    order = torch.nn.functional.pad(order, (0, max(0, cap - order.shape[-1])))[..., :cap]
    live = torch.arange(cap, device="cuda") < new_lens[:, None, None]
    kept = torch.where(live, order, w.shape[-1]).sort(dim=-1).values
    new_w = torch.where(live, w.gather(-1, kept.clamp_max(w.shape[-1] - 1)), 0.0)
    at = kept.clamp_max(w.shape[-1] - 1)
    page = st["table"].long().clamp_min(0)[torch.arange(len(lens), device="cuda")[:, None, None], at // bs]
    head = torch.arange(case["hkv"], device="cuda")[None, :, None]
    # (a row's padding goes to the last block, which is in no table)
    to = torch.where(st["new_table"] >= 0, st["new_table"], cache["k"].shape[0] - 1).long()
    b, h = kept.shape[:2]
    for name in ("k", "v"):
        x = cache[name][page, head, at % bs].float() * cache[name + "_scale"][page, head][..., None]
        x = torch.where(live.expand(kept.shape)[..., None], x, 0.0).view(b, h, -1, bs, case["d"]).transpose(1, 2)   # [batch, blocks, heads, bs, d]
        x, scale = _quantise(x, kind)
        written = live.view(b, 1, -1, bs).transpose(1, 2)[..., None]
        held = cache[name].view(torch.uint8)[to]
        cache[name].view(torch.uint8)[to] = torch.where(written, x.view(torch.uint8), held)
        cache[name + "_scale"][to] = scale
    kept = torch.where(live, kept, -1)[..., :budget].to(torch.int32)
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=-1)
    return new_lens.to(torch.int32), new_w, kept


# ---------------------------------------------------------------- one pass

def _handle(st, ops):
    """The cache object that a program keeps beside its tensors."""
    if "handle" not in st:
        c = st["cache"]
        st["handle"] = ops.KVCache(c["k"], c["v"], c["k_scale"], c["v_scale"])
    return st["handle"]


def run(state):
    case, st = state["case"], state
    op = case["op"]
    most = max(_ints(case["lens"])) if op == "read" else 0
    if own:
        ops = _ops()
        if op == "attn":
            out = ops.cache_attn(st["q"], _handle(st, ops), st["table"], st["lens"], window_size=None if case["window"] < 0 else case["window"],
                                 num_sink_tokens=case["sink"], weights=st.get("weights"))
            return (out, st["weights"]) if case["weights"] else out
        if op == "append":
            cache = _handle(st, ops)
            ops.cache_append(cache, st["k"], st["v"], st["table"], st["lens"], cu_seqlens=st["cu"])
            return ops.cache_read(cache, st["touched"], st["touched_lens"], st["touched"].shape[1] * case["bs"], dtype=st["k"].dtype)
        if op == "read":
            return ops.cache_read(_handle(st, ops), st["table"], st["lens"], most, dtype=_DTYPES[case["dtype"]])
        if op == "sums":
            return ops.attn_weight_sums(st["q"], st["k"], st["lse"], case["window"], num_sink_tokens=case["sink"], cu_seqlens=st["cu"])
        cache = _handle(st, ops)
        new_lens, new_w, kept = ops.cache_evict(cache, st["table"], st["lens"], st["weights"], case["budget"], st["new_table"],
                                                num_sink_tokens=case["sink"], num_recent_tokens=case["recent"])
        k, v = ops.cache_read(cache, st["new_table"], new_lens, st["new_table"].shape[1] * case["bs"], dtype=_DTYPES[case["dtype"]])
        return new_lens, new_w, kept, k, v
    if op == "attn":
        return _plain_attn(st)
    if op == "append":
        _plain_append(st)
        return _plain_read(st["cache"], st["touched"], st["touched_lens"], st["touched"].shape[1] * case["bs"], st["k"].dtype)
    if op == "read":
        return _plain_read(st["cache"], st["table"], st["lens"], most, _DTYPES[case["dtype"]])
    if op == "sums":
        return _plain_sums(st)
    new_lens, new_w, kept = _plain_evict(st)
    k, v = _plain_read(st["cache"], st["new_table"], new_lens, st["new_table"].shape[1] * case["bs"], _DTYPES[case["dtype"]])
    return new_lens, new_w, kept, k, v


# ---------------------------------------------------------------- in 64 bits, from the definitions

def _exact_block(values, before, kind):
    """What a block [tokens, heads, d] stands for once it is held in 8 bits; `before`: the scale [heads] it may not go below, or None."""
    top = _KINDS[kind][1]
    most = values.abs().amax(dim=(0, 2))
    scale = (2.0 ** ((most / top).log2().round() - 1).clamp_min(-100)).float().double()
    for _ in range(2):
        scale = torch.where(most > top * scale, 2 * scale, scale)
    if before is not None:
        scale = torch.maximum(scale, before)
    u = (values / scale[:, None]).clamp(-top, top)
    if kind == "int8":
        u = u.round()
    else:
        # 3 bits behind the leading one, and steps of 2^-9 below 2^-6; ties to even
        step = (2.0 ** (u.abs().clamp_min(2.0 ** -6).log2().floor() - 3)).float().double()
        u = (u / step).round() * step
    return u * scale[:, None]


def _exact_rows(cache, name, pages, n):
    """The first n tokens of a list of blocks [n, heads, d]."""
    pages = pages.long()
    x = cache[name][pages].double() * cache[name + "_scale"][pages].double()[:, :, None, None]
    return x.transpose(1, 2).flatten(0, 1)[:n]


def exact(case, seed):
    st = prepare(case, seed)
    op, lens, hkv, d = case["op"], _ints(case["lens"]), case["hkv"], case["d"]
    grp = case["hq"] // hkv
    if op == "sums":
        cu = st["cu"].tolist()
        out = torch.zeros(hkv, cu[-1], dtype=torch.float64, device="cuda")
        for a, z in zip(cu, cu[1:]):
            for lo in range(a, z, 2048):
                hi = min(z, lo + 2048)
                i, j = torch.arange(lo, hi, device="cuda")[:, None], torch.arange(a, z, device="cuda")[None]
                hidden = (j > i) | ((i - j > case["window"]) & (j - a >= case["sink"]))
                for h in range(case["hq"]):
                    s = st["q"][lo:hi, h].double() @ st["k"][a:z, h // grp].double().T / math.sqrt(d)
                    out[h // grp, a:z] += (s - st["lse"][h, lo:hi].double()[:, None]).exp().masked_fill(hidden, 0).sum(0)
        return out
    bs, kind, cache = case["bs"], case["kind"], st["cache"]
    if op == "append":
        cu, answer = st["cu"].tolist(), []
        for name in ("k", "v"):
            out = torch.zeros(len(lens), st["touched"].shape[1] * bs, hkv, d, dtype=torch.float64, device="cuda")
            for i, a in enumerate(lens):
                old = a % bs
                rows = st[name][cu[i]:cu[i + 1]].double()
                before = None
                if old:
                    page = st["touched"][i, :1]
                    rows = torch.cat([_exact_rows(cache, name, page, old), rows])
                    before = cache[name + "_scale"][page[0].long()].double()
                for at in range(0, rows.shape[0], bs):
                    out[i, at:min(at + bs, rows.shape[0])] = _exact_block(rows[at:at + bs], before if at == 0 else None, kind)
            answer.append(out)
        return tuple(answer)
    if op == "read":
        answer = []
        for name in ("k", "v"):
            out = torch.zeros(len(lens), max(lens), hkv, d, dtype=torch.float64, device="cuda")
            for i, n in enumerate(lens):
                out[i, :n] = _exact_rows(cache, name, st["table"][i, :_blocks(n, bs)], n)
            answer.append(out)
        return tuple(answer)
    if op == "attn":
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
        sums = st["weights"].double() if case["weights"] else None
        for i, n in enumerate(lens):
            k, v = (_exact_rows(cache, name, st["table"][i, :_blocks(n, bs)], n) for name in ("k", "v"))
            for j in range(case["new"]):
                p = n - case["new"] + j
                if p < 0:
                    continue
                left = 0 if case["window"] < 0 else max(0, p - case["window"])
                at = torch.cat([torch.arange(min(case["sink"], left), device="cuda"), torch.arange(left, p + 1, device="cuda")])
                q = st["q"][i, j].double().view(hkv, grp, d)
                w = torch.einsum("hgd,thd->hgt", q, k[at]).div(math.sqrt(d)).softmax(-1)
                out[i, j] = torch.einsum("hgt,thd->hgd", w, v[at]).reshape(-1, d)
                if sums is not None:
                    sums[i, :, at] += w.sum(1)
        return out if sums is None else (out, sums)
    budget, cap = case["budget"], st["new_table"].shape[1] * bs
    new_w = torch.zeros(len(lens), hkv, cap, dtype=torch.float64, device="cuda")
    k, v = (torch.zeros(len(lens), cap, hkv, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, n in enumerate(lens):
        rows = {name: _exact_rows(cache, name, st["table"][i, :_blocks(n, bs)], n) for name in ("k", "v")}
        keep = min(n, budget)
        for h in range(hkv):
            w = st["weights"][i, h, :n].double()
            score = w.clone()
            score[:case["sink"]] = math.inf
            score[max(0, n - case["recent"]):] = math.inf
            # the smallest weight that stays, then as many of the tokens that have it as there is room for, the first ones
            least = score.topk(keep).values[-1]
            above, equal = score > least, score == least
            chosen = above | (equal & (equal.cumsum(0) <= keep - above.sum()))
            at = chosen.nonzero()[:, 0]
            new_w[i, h, :keep] = w[at]
            for out, name in ((k, "k"), (v, "v")):
                x = torch.zeros(_blocks(keep, bs) * bs, d, dtype=torch.float64, device="cuda")
                x[:keep] = rows[name][at, h]
                # (blocks take the place of heads: each has a scale of its own)
                x = _exact_block(x.view(-1, bs, d).transpose(0, 1), None, kind).transpose(0, 1).reshape(-1, d)
                out[i, :keep, h] = x[:keep]
    return None, new_w, None, k, v
