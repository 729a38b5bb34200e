"""Decoding from a key/value cache held in 8 bits, one GPU.

The reference computes whole sequences; a model trained or prefilled with its attention goes on token by token, and what
bounds that is reading the cached keys and values.  Here they are stored in 8 bits in blocks of tokens, each with one
scale per head (KVCache), addressed through a block table as serving programs keep one:

    cache = KVCache.empty(num_blocks, num_kv_heads, block_size=64, head_dim=128)
    cache_append(cache, k, v, block_table, lens, cu_seqlens=cu)        # a packed batch of prompts, lens = 0
    lens += prompt_lens
    ...
    cache_append(cache, k, v, block_table, lens)                       # a step: k, v [batch, 1, heads, 128]
    lens += 1
    out = cache_attn(q, cache, block_table, lens, window_size=4096, num_sink_tokens=4)

and, for a cache that is kept to a number of tokens by what the model has attended to:

    weights[b, :, :n] = attn_weight_sums(q, k, softmax_lse, window)    # of a prompt
    out = cache_attn(q, cache, block_table, lens, weights=weights)     # every step adds its own
    lens, weights, kept = cache_evict(cache, block_table, lens, weights, budget, new_block_table, 4, 512)

block_table [batch, max_blocks] and lens [batch] are int32 tensors of the caller's on the cache's device: slot t of
sequence b is token t % block_size of block block_table[b, t // block_size]; a row may be expanded over the batch where its
blocks are only read.  Nothing here changes lens, copies it to the
host or waits for the device, so that a step can be captured into a CUDA graph and replayed with other lengths.  Positions
are slots: after an eviction the tokens that stayed count as neighbours.

A sequence whose table or length cannot be right (a block that is none, a length beyond the table) makes the kernels
raise the device's status word and leave that sequence alone; the next call of a public function raises.

The operators have no derivative.  Tensors of any stream may be used as with torch's own operators: the call runs on the
current stream of the cache's device.
"""
from typing import Optional, Tuple, Union

import torch

from .. import _kernels as K

_native = None


def _call(name: str, device: torch.device, *args):
    global _native
    if _native is None:
        _native = K.native_module()
    fn = getattr(_native, name)
    for _ in range(8):  # (more than twice where other threads' calls are reported meanwhile)
        result = fn(*args)
        if result is not False:
            return result
        # no status word yet, or an error of an earlier call to raise
        K.status_word(device)
        K.raise_if_reported(device)
    raise RuntimeError(f"ring_swa.ops.{name}: errors of earlier calls on {device} are being reported; this call did nothing")


def _call_cache(name: str, cache: "KVCache", *args):
    return _call(name, cache.k.device, cache.k, cache.v, cache.k_scale, cache.v_scale, *args)


class KVCache:
    """Keys and values of cached tokens in 8 bits.

    k, v [num_blocks, num_kv_heads, block_size, head_dim], int8 or float8_e4m3fn; k_scale, v_scale [num_blocks,
    num_kv_heads] float32: value = stored * scale.  block_size 16, 32, 64 or 128; head_dim 64 or 128.  All contiguous
    and on one device.

    cache_append and cache_evict write scales that are powers of two, the least ones that hold a block's values: moving
    a token to another block or reading it back rounds nothing that the other scale can hold.  int8 has the smaller error
    where a block's values are of one magnitude, float8_e4m3fn where they are not.  Tensors filled elsewhere may have
    any positive scales (V's from 2^-100 to 2^80, a smaller one counts as 2^-100 in cache_attn; and no NaN among float8_e4m3fn
    values: a NaN belongs into the scale).
    """
    __slots__ = ("k", "v", "k_scale", "v_scale")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, num_blocks: int, num_kv_heads: int, block_size: int = 64, head_dim: int = 128,
              dtype: torch.dtype = torch.int8, device: Union[str, torch.device] = "cuda") -> "KVCache":
        if dtype not in (torch.int8, torch.float8_e4m3fn):
            raise ValueError(f"KVCache: dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
        if block_size not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError(f"KVCache: block_size must be 16, 32, 64 or 128 and head_dim 64 or 128, got {block_size} and {head_dim}")
        if num_blocks <= 0 or num_kv_heads <= 0:
            raise ValueError("KVCache: num_blocks and num_kv_heads must be positive")
        shape = (num_blocks, num_kv_heads, block_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.ones(shape[:2], dtype=torch.float32, device=device),
                   torch.ones(shape[:2], dtype=torch.float32, device=device))

    @property
    def block_size(self) -> int:
        return self.k.shape[2]


def cache_append(cache: KVCache, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                 cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Stores new tokens behind the lens[b] ones that sequence b has (lens is not changed).

    k, v bf16 or fp16: [batch, tokens, num_kv_heads, head_dim], or packed [tokens, num_kv_heads, head_dim] with
    cu_seqlens (int32 [batch + 1], on the device).  A block that already holds tokens keeps its scale if the new ones fit;
    otherwise the scale grows and the older tokens are rounded to it.  A block that is given an infinity or a NaN reads as
    NaN.  The blocks written to must belong to one sequence each; blocks that are only read (a shared prefix that ends
    with a full block) may be shared.
    """
    _call_cache("cache_append", cache, k, v, block_table, lens, cu_seqlens)


def cache_read(cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, max_len: int,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of the first min(lens[b], max_len) tokens of every sequence in 16 bits, for a prompt that
    continues a cached prefix: k, v [batch, max_len, num_kv_heads, head_dim], zero behind a sequence's end."""
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"cache_read: dtype must be torch.bfloat16 or torch.float16, got {dtype}")
    return _call_cache("cache_read", cache, block_table, lens, max_len, dtype == torch.bfloat16)


def cache_attn(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor,
               window_size: Optional[int] = None, num_sink_tokens: int = 0, softmax_scale: Optional[float] = None,
               weights: Optional[torch.Tensor] = None, return_lse: bool = False
               ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest tokens of every sequence over its cached tokens, themselves included.

    q [batch, queries, num_q_heads, head_dim], bf16 or fp16; num_q_heads a multiple of the cache's heads.  Query i of
    sequence b is the token in slot p = lens[b] - queries + i (lens counts the new tokens, which cache_append has stored);
    it sees slot t <= p if p - t <= window_size or t < num_sink_tokens, with window_size None every t <= p.  The mask is that
    of ring_sliding_window_attn and ring_streaming_llm_attn.  Returns out like q, and with return_lse also the log-sum-exp
    [batch, num_q_heads, queries] float32; a query that sees nothing (an empty sequence, or one shorter than
    `queries`) gives zeros and -inf.  At most 8192 queries and heads of one key/value head together.  Blocks none of whose slots
    any query sees may have been given back: their entries of block_table are not looked at.

    weights: float32 [batch, num_kv_heads, at least max_blocks * block_size], added to in place: the softmax weights that
    every slot got from the queries and heads of its key/value head (what cache_evict goes by; start it with
    attn_weight_sums of the prompt, or zeros).  Such a call holds, while it runs, 32 bytes per slot of block_table (of the window
    and the sinks where there is a window), sequence, head and 8 queries and heads of a key/value head: a table much wider than
    the sequences costs memory.

    NaN reaches the rows that see it and no others: from a query or a block of keys the output, the log-sum-exp and the weights of
    the slots which the row sees, from a block of values the output alone.
    """
    return _call_cache("cache_attn", cache, q, block_table, lens, window_size, num_sink_tokens, softmax_scale, weights, return_lse)


def attn_weight_sums(q: torch.Tensor, k: torch.Tensor, softmax_lse: torch.Tensor, window_size: Optional[int] = None,
                     num_sink_tokens: int = 0, softmax_scale: Optional[float] = None,
                     cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The softmax weight that every key of a prompt got, summed over the queries that see it and the query heads of
    its key/value head: float32 [batch, num_kv_heads, tokens], packed [num_kv_heads, tokens].

    q [batch, tokens, num_q_heads, head_dim], k [batch, tokens, num_kv_heads, head_dim], bf16 or fp16, head_dim 64 or 128;
    packed [tokens, heads, head_dim] with cu_seqlens (int32, on the device).  The mask is that of cache_attn (and of
    ring_streaming_llm_attn on one GPU); softmax_lse [batch, num_q_heads, tokens] (packed [num_q_heads, tokens]) float32 is
    the log-sum-exp of the same attention, as wrapped_flash_attn_fwd and torch.ops.ring_swa.swa_fwd return it (for heads of
    64 elements: of q, k and v padded with zeros to 128, at the scale of 64).
    """
    return _call("weight_sums", q.device, q, k, softmax_lse, window_size, num_sink_tokens, softmax_scale, cu_seqlens)


def cache_evict(cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor, budget: int,
                new_block_table: torch.Tensor, num_sink_tokens: int = 0, num_recent_tokens: int = 0
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts every sequence to at most `budget` tokens: its first num_sink_tokens, its last num_recent_tokens, and those in
    between with the largest weights, chosen for each key/value head (equal weights: the earlier token; NaN counts as the
    largest).  The tokens keep their order.

    weights float32 [batch, num_kv_heads, at least max_blocks * block_size], as cache_attn adds them up.  The kept keys and
    values go to the blocks named by new_block_table ([batch, blocks for min(budget, tokens of block_table)], int32), which
    must be other blocks than those of block_table and belong to one sequence each; the old ones are only read, so that a
    prefix may be shared, and are free afterwards.  A sequence within the budget is moved as it is.
    Returns (new_lens [batch] int32, new_weights [batch, num_kv_heads, tokens of new_block_table], kept [batch,
    num_kv_heads, budget] int32: the old slots of the kept tokens, -1 behind them).
    """
    return _call_cache("cache_evict", cache, block_table, lens, weights, budget, new_block_table, num_sink_tokens, num_recent_tokens)
