"""Calls that the operators on the 8-bit key/value cache refuse, without a GPU: shapes, types and options are looked at
before the device.  And the restatement that the GPU tests compare against (tests/cache_ref.py), against torch's formats."""
import ctypes
import math

import pytest
import torch

import cache_ref as R
from ring_swa import ops


def cpu_cache(**kw):
    return ops.KVCache.empty(4, 2, block_size=16, head_dim=64, device="cpu", **kw)


TABLE, LENS = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
Q, KV = torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16)


@pytest.mark.parametrize("kw", [dict(dtype=torch.float16), dict(block_size=48), dict(head_dim=96), dict(num_blocks=0), dict(num_kv_heads=0)])
def test_cache_shapes(kw):
    args = dict(num_blocks=4, num_kv_heads=2, block_size=16, head_dim=64, device="cpu")
    args.update(kw)
    with pytest.raises(ValueError, match="KVCache"):
        ops.KVCache.empty(**args)


def broken_caches():
    c = cpu_cache()
    yield ops.KVCache(c.k, c.v[:2], c.k_scale, c.v_scale)
    yield ops.KVCache(c.k, c.v.view(torch.float8_e4m3fn), c.k_scale, c.v_scale)
    yield ops.KVCache(c.k.to(torch.uint8), c.v.to(torch.uint8), c.k_scale, c.v_scale)
    yield ops.KVCache(c.k, c.v, c.k_scale[:, :1], c.v_scale)
    yield ops.KVCache(c.k, c.v, c.k_scale.half(), c.v_scale.half())
    yield ops.KVCache(c.k.transpose(1, 2).contiguous().transpose(1, 2), c.v, c.k_scale, c.v_scale)
    yield ops.KVCache(c.k[:, :, :8], c.v[:, :, :8], c.k_scale, c.v_scale)


def test_a_cache_that_is_none():
    for c in broken_caches():
        with pytest.raises(ValueError, match="cache"):
            ops.cache_read(c, TABLE, LENS, 1)


@pytest.mark.parametrize("change", [
    dict(q=Q.float()), dict(q=Q[0]), dict(q=Q[..., :32]), dict(q=Q[:, :, :3]), dict(q=Q[:2]), dict(q=Q[:, :, :0]),
    dict(block_table=TABLE.long()), dict(block_table=TABLE[0]), dict(block_table=TABLE.t()), dict(lens=LENS.long()), dict(lens=LENS[:2]),
    dict(window_size=-1), dict(num_sink_tokens=-1), dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=math.nan),
    dict(softmax_scale=math.inf), dict(softmax_scale=1e-60),
    dict(weights=torch.zeros(3, 2, 31)), dict(weights=torch.zeros(3, 4, 32)), dict(weights=torch.zeros(3, 2, 32).half()),
    dict(weights=torch.zeros(1, 2, 32).expand(3, 2, 32)), dict(weights=torch.zeros(3, 2, 64)[..., ::2]),
])
def test_attn_refuses(change):
    args = dict(q=Q, cache=cpu_cache(), block_table=TABLE, lens=LENS)
    args.update(change)
    with pytest.raises(ValueError):
        ops.cache_attn(**args)


@pytest.mark.parametrize("change", [
    dict(k=KV.float(), v=KV.float()), dict(v=KV.half()), dict(v=KV[:, :, :1]), dict(k=KV[:, 0], v=KV[:, 0]), dict(k=KV[:2], v=KV[:2]),
    dict(k=KV[..., :32], v=KV[..., :32]), dict(k=Q, v=Q), dict(cu_seqlens=torch.zeros(4, dtype=torch.int32)),
    dict(k=KV[:, 0], v=KV[:, 0], cu_seqlens=torch.zeros(3, dtype=torch.int32)), dict(k=KV[:, 0], v=KV[:, 0], cu_seqlens=torch.zeros(4)),
])
def test_append_refuses(change):
    args = dict(cache=cpu_cache(), k=KV, v=KV, block_table=TABLE, lens=LENS)
    args.update(change)
    with pytest.raises(ValueError):
        ops.cache_append(**args)


def test_read_refuses():
    with pytest.raises(ValueError):
        ops.cache_read(cpu_cache(), TABLE, LENS, -1)
    with pytest.raises(ValueError):
        ops.cache_read(cpu_cache(), TABLE, LENS, 1, dtype=torch.float32)
    with pytest.raises(TypeError):
        ops.cache_read(cpu_cache(), TABLE, LENS, 1.5)


W = torch.zeros(3, 2, 32)


@pytest.mark.parametrize("change", [
    dict(budget=0), dict(budget=-3), dict(num_sink_tokens=-1), dict(num_recent_tokens=-1), dict(budget=8, num_sink_tokens=4, num_recent_tokens=5),
    dict(budget=1 << 40), dict(weights=W[:, :, :31]), dict(weights=W.double()), dict(weights=W[:2]), dict(weights=W[:1].expand(3, 2, 32)),
    dict(new_block_table=TABLE[:2]), dict(new_block_table=TABLE.long()), dict(budget=17, new_block_table=TABLE[:, :1].contiguous()),
    dict(block_table=TABLE[0]), dict(lens=LENS.long()),
])
def test_evict_refuses(change):
    args = dict(cache=cpu_cache(), block_table=TABLE, lens=LENS, weights=W, budget=16, new_block_table=TABLE)
    args.update(change)
    with pytest.raises(ValueError):
        ops.cache_evict(**args)


SQ, SK, SL = torch.zeros(2, 10, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 10, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 10)


@pytest.mark.parametrize("change", [
    dict(q=SQ.float()), dict(k=SK.half()), dict(q=SQ[0], k=SK[0], softmax_lse=SL[0]), dict(k=SK[:, :9]), dict(k=SK[:1]), dict(q=SQ[:, :, :3]),
    dict(q=SQ[..., :32], k=SK[..., :32]), dict(softmax_lse=SL[:, :3]), dict(softmax_lse=SL[..., :9]), dict(softmax_lse=SL.double()), dict(softmax_lse=SL[:1]),
    dict(window_size=-1), dict(num_sink_tokens=-1), dict(softmax_scale=0.0), dict(cu_seqlens=torch.tensor([0, 10], dtype=torch.int32)),
    dict(q=SQ[0], k=SK[0], softmax_lse=SL[0], cu_seqlens=torch.tensor([0, 10])), dict(q=SQ[0], k=SK[0], softmax_lse=SL[0], cu_seqlens=torch.tensor([0], dtype=torch.int32)),
])
def test_weight_sums_refuse(change):
    args = dict(q=SQ, k=SK, softmax_lse=SL, window_size=4)
    args.update(change)
    with pytest.raises(ValueError):
        ops.attn_weight_sums(**args)


def test_no_cpu_path_no_gradient_no_other_tensors():
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cache_attn(Q, cpu_cache(), TABLE, LENS)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cache_append(cpu_cache(), KV, KV, TABLE, LENS)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.cache_attn(Q.clone().requires_grad_(True), cpu_cache(), TABLE, LENS)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.cache_append(cpu_cache(), KV, KV.clone().requires_grad_(True), TABLE, LENS)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.cache_evict(cpu_cache(), TABLE, LENS, W, 16, TABLE)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attn_weight_sums(SQ, SK, SL, 4)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.attn_weight_sums(SQ, SK.clone().requires_grad_(True), SL, 4)
    with pytest.raises(TypeError):
        ops.cache_attn(Q.float().numpy(), cpu_cache(), TABLE, LENS)

    class Other(torch.Tensor):
        pass

    with pytest.raises(TypeError):
        ops.cache_attn(Q.as_subclass(Other), cpu_cache(), TABLE, LENS)
    with pytest.raises(RuntimeError, match="no CPU path"), torch.no_grad():
        ops.cache_attn(Q.clone().requires_grad_(True), cpu_cache(), TABLE, LENS)


def test_the_c_entries_refuse():
    from ring_swa import _C
    lib = _C.lib()
    for name in ("cache_append", "cache_read", "cache_attn", "cache_evict", "weight_sums"):
        assert getattr(lib, "rswa_" + name)(None, None) == -1
    for name in ("cache_attn", "weight_sums"):
        assert getattr(lib, f"rswa_{name}_workspace_bytes")(None) == -1
    p = _C.CacheAttnParams()
    p.cache.head_dim, p.cache.block_size, p.cache.n_kv_heads = 128, 64, 8
    p.table.batch, p.table.max_blocks, p.q_len, p.n_q_heads, p.window = 32, 128, 1, 32, -1
    assert lib.rswa_cache_attn_workspace_bytes(ctypes.byref(p)) > 0
    p.n_q_heads = 31
    assert lib.rswa_cache_attn_workspace_bytes(ctypes.byref(p)) == -1
    p.n_q_heads, p.cache.head_dim = 32, 96
    assert lib.rswa_cache_attn_workspace_bytes(ctypes.byref(p)) == -2
    p.cache.head_dim, p.cache.kind = 128, 7
    assert lib.rswa_cache_attn(ctypes.byref(p), None) == -2 and b"kind" in lib.rswa_last_error()
    p.cache.kind, p.cache.num_blocks = 0, 0
    assert lib.rswa_cache_attn(ctypes.byref(p), None) == -1
    p.cache.num_blocks = 1
    assert lib.rswa_cache_attn(ctypes.byref(p), None) == -1 and b"16-byte aligned" in lib.rswa_last_error()


def test_struct_sizes_match_the_header():
    import os
    import subprocess
    import tempfile
    from ring_swa import _C
    names = [("rswa_cache_t", _C.Cache), ("rswa_block_table_t", _C.BlockTable), ("rswa_cache_append_params_t", _C.CacheAppendParams),
             ("rswa_cache_read_params_t", _C.CacheReadParams), ("rswa_cache_attn_params_t", _C.CacheAttnParams),
             ("rswa_weight_sums_params_t", _C.WeightSumsParams), ("rswa_cache_evict_params_t", _C.CacheEvictParams)]
    src = '#include <stdio.h>\n#include "rswa.h"\nint main(void) {\n' + "".join(f'  printf("%zu\\n", sizeof({n}));\n' for n, _ in names) + "  return 0;\n}\n"
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = os.path.join(tmp, "s.c"), os.path.join(tmp, "s")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), c, "-o", exe], check=True)
        sizes = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [ctypes.sizeof(t) for _, t in names]


def test_the_restated_formats_are_torchs():
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.arange(4096) % 24 - 14.0)
    x = torch.cat([x.clamp(-448, 448), torch.tensor([0.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 448.0, -448.0, 17.0, 19.0])])
    assert torch.equal(R.to_stored(x.double(), "e4m3"), x.to(torch.float8_e4m3fn).double())
    assert torch.equal(R.to_stored(x.double(), "int8"), x.double().round().clamp(-127, 127))
    for amax, kind, want in ((127.0, "int8", 1.0), (127.5, "int8", 2.0), (448.0, "e4m3", 1.0), (449.0, "e4m3", 2.0), (0.0, "int8", 2.0 ** -100),
                             (1.0, "int8", 2.0 ** -6), (0.99, "int8", 2.0 ** -7), (1.0, "e4m3", 2.0 ** -8)):
        assert R.scale_for(amax, kind) == want
    assert math.isnan(R.scale_for(math.inf, "int8"))
