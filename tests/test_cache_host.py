"""Host side of the operators on the 8-bit key/value cache that needs no GPU."""
import pytest
import torch

from ring_swa import _kernels as K
from ring_swa import ops
from ring_swa.ops import kv_cache


def test_a_call_that_finds_another_reported_error_is_made_again(monkeypatch):
    """False stands for a call that did nothing, and never reaches the caller: not where another call's error is reported between
    the look at the first one and the second attempt either."""
    cache = ops.KVCache.empty(4, 2, block_size=16, head_dim=64, device="cpu")
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    answers, looks = [False, False, "done"], []

    class Native:
        @staticmethod
        def cache_read(*args):
            return answers.pop(0)

    monkeypatch.setattr(kv_cache, "_native", Native)
    monkeypatch.setattr(K, "status_word", lambda device: looks.append("word"))
    monkeypatch.setattr(K, "raise_if_reported", lambda device: looks.append("look"))
    assert ops.cache_read(cache, table, lens, 1) == "done"
    assert looks == ["word", "look"] * 2 and not answers

    def report(device):
        raise RuntimeError("code 110")

    answers.append(False)
    monkeypatch.setattr(K, "raise_if_reported", report)
    with pytest.raises(RuntimeError, match="110"):
        ops.cache_read(cache, table, lens, 1)


def test_a_call_that_can_never_be_made_raises(monkeypatch):
    cache = ops.KVCache.empty(4, 2, block_size=16, head_dim=64, device="cpu")

    class Native:
        @staticmethod
        def cache_append(*args):
            return False

    monkeypatch.setattr(kv_cache, "_native", Native)
    monkeypatch.setattr(K, "status_word", lambda device: None)
    monkeypatch.setattr(K, "raise_if_reported", lambda device: None)
    kv = torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="did nothing"):
        ops.cache_append(cache, kv, kv, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_weights_in_either_order_of_sequences_and_heads():
    """[heads, batch, slots] transposed has no rows that overlap; it comes as far as the look at the device."""
    cache = ops.KVCache.empty(4, 2, block_size=16, head_dim=64, device="cpu")
    q, table, lens = torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for w in (torch.zeros(2, 3, 32).transpose(0, 1), torch.zeros(2, 3, 40)[..., 3:35].transpose(0, 1), torch.zeros(3, 4, 32)[:, ::2]):
        with pytest.raises(RuntimeError, match="no CPU path"):
            ops.cache_attn(q, cache, table, lens, weights=w)
        with pytest.raises(RuntimeError, match="no CPU path"):
            ops.cache_evict(cache, table, lens, w, 16, table)
    for w in (torch.zeros(2, 1, 32).expand(2, 3, 32).transpose(0, 1), torch.zeros(1, 3, 32).expand(2, 3, 32).transpose(0, 1),
              torch.zeros(200).as_strided((3, 2, 32), (16, 32, 1)), torch.zeros(200).as_strided((3, 2, 32), (32, 32, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops.cache_attn(q, cache, table, lens, weights=w)


def test_tables_whose_slots_come_close_to_32_bits_are_refused():
    """The kernels step up to 2^14 slots beyond a sequence's end before they compare."""
    from ring_swa import _C
    lib, call = _C.lib(), {"append": _C.CacheAppendParams, "read": _C.CacheReadParams, "attn": _C.CacheAttnParams, "evict": _C.CacheEvictParams}
    for name, params in call.items():
        for blocks, refused in (((1 << 24) - 4, True), ((1 << 24) - (1 << 13), False)):
            p = params()
            c = p.cache
            c.k = c.v = c.k_scale = c.v_scale = 4096  # (looked at no further: the call ends with the checks)
            c.num_blocks, c.n_kv_heads, c.block_size, c.head_dim = 1, 1, 128, 64
            p.lens = p.status = p.table.entries = 4096
            p.table.batch, p.table.max_blocks, p.table.stride = 1, blocks, blocks
            p.n_q_heads = 1
            if name == "evict":
                p.new_table = p.table
                p.budget = -1  # the refusal behind it
            else:
                p.dtype = 7
            assert getattr(lib, "rswa_cache_" + name)(p, None) < 0
            assert (b"overflow" in lib.rswa_last_error()) == refused, (name, blocks, lib.rswa_last_error())
