"""Python faces of the kernels of the 8-bit cache of keys and values; see ``ops/__init__.py``.

A page holds, for every KV head, ``page_size`` rows of ``head_dim`` e4m3 numbers for the keys and as many for the values, then one
scale byte to a row: its values are the numbers times ``2^(byte - 127)``, the smallest power of two between 2^-60 and 2^40 under
which no number of the row exceeds 448.  Pages are flat: ``cache_layer`` is uint8 ``[pages, kv8_page_bytes(...)]``, numbers
``[2, kv_heads, page_size, head_dim]`` then scales ``[2, kv_heads, page_size]``.  What no row was written to is never read.
"""
from __future__ import annotations

import functools
import itertools
import random
from typing import Optional, Sequence, Tuple

import torch

from . import AP_BF16, AP_F32, KernelError, call, core, library, stream_handle

# (a CUDA tensor is there before it is asked: nothing is left to initialise)
_here = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

_CODES = {torch.float32: AP_F32, torch.bfloat16: AP_BF16}


@functools.lru_cache(maxsize=None)
def kv8_page_bytes(num_kv_heads: int, page_size: int, head_dim: int) -> int:
    """Bytes of one page of one layer's 8-bit cache (numbers, scales, padding to 16)."""
    return -(-2 * num_kv_heads * page_size * (head_dim + 1) // 16) * 16


def _take(what: str, t: torch.Tensor, name: str, dtype, dims: int, device: int):
    """Checks a tensor; returns its shape."""
    shape = t.shape
    if t.dtype is not dtype or len(shape) != dims or t.get_device() != device or not t.is_contiguous():
        raise KernelError(f"{what}: {name} must be a contiguous {dims}-dimensional tensor of {dtype} on the cache's device, is "
                          f"{tuple(shape)} {t.dtype} on {t.device}")
    return shape


def _take_cache(what: str, cache_layer: torch.Tensor, num_kv_heads: int, head_dim: int, page_size: int, positions: torch.Tensor,
                token_seq: torch.Tensor, block_table: torch.Tensor):
    """Checks the cache and the rows' metadata; returns the device, the number of rows, what the C entry points take of the cache
    (address, pages, bytes of one) and of the block table (address, blocks to a sequence, sequences)."""
    if head_dim <= 0 or head_dim % 16 or head_dim > 256 or num_kv_heads <= 0 or page_size <= 0:
        raise KernelError(f"{what}: {num_kv_heads} KV heads of {head_dim} in pages of {page_size} are not taken (head sizes are "
                          f"multiples of 16 up to 256)")
    device = cache_layer.get_device()
    if device < 0 or device != _here():
        raise KernelError(f"{what}: the cache must be a CUDA tensor on the current device, is on {cache_layer.device}")
    pages, page_bytes = _take(what, cache_layer, "cache_layer", torch.uint8, 2, device)
    cache = cache_layer.data_ptr()
    if page_bytes != kv8_page_bytes(num_kv_heads, page_size, head_dim) or cache % 16:
        raise KernelError(f"{what}: the cache must be 16-byte aligned pages of {kv8_page_bytes(num_kv_heads, page_size, head_dim)} "
                          f"bytes, is {tuple(cache_layer.shape)}")
    given, = _take(what, positions, "positions", torch.int32, 1, device)
    T, = _take(what, token_seq, "token_seq", torch.int32, 1, device)
    sequences, blocks = _take(what, block_table, "block_table", torch.int32, 2, device)
    if given < T or not sequences or not blocks:
        raise KernelError(f"{what}: fewer positions than rows, or an empty block table")
    return device, T, (cache, pages, page_bytes), (block_table.data_ptr(), blocks, sequences)


def rope_kv8_store(qkv: torch.Tensor, q_out: torch.Tensor, cache_layer: torch.Tensor, positions: torch.Tensor,
                   token_seq: torch.Tensor, block_table: torch.Tensor, cos_sin: Optional[torch.Tensor], pairing: int,
                   num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> None:
    """The rows of a stacked Q, K, V projection (``[T, (nh + 2 nkv) hd]`` in the type of ``q_out`` or 32-bit, or 32-bit partial sums
    ``[S, T, ...]`` added in order): Q rotated into ``q_out [T, nh*hd]``, K rotated and V rounded to 8 bits into slot
    ``positions[t] % page_size`` of page ``block_table[token_seq[t], positions[t] // page_size]``.  All in 32 bits, each result
    rounded once.  ``cos_sin [T, hd/2, 2]`` (None: no rotation); ``pairing`` as for :func:`rope_kv_store` (0: element i with
    i + hd/2; 1: neighbours; 2: neighbours in the input, halves in the result).  A row without a page (position or sequence outside
    the block table, page id outside the cache) is not kept, its query is written all the same.  A number that is not finite is kept as
    NaN.  Two rows of one step must not name the same slot."""
    what = "rope_kv8_store"
    device, T, cache, table = _take_cache(what, cache_layer, num_kv_heads, head_dim, page_size, positions, token_seq, block_table)
    width = (num_heads + 2 * num_kv_heads) * head_dim
    act, dt = _CODES.get(q_out.dtype), _CODES.get(qkv.dtype)
    if act is None or dt is None or (dt == AP_BF16 and act == AP_F32) or num_heads <= 0:
        raise KernelError(f"{what}: types {qkv.dtype} and {q_out.dtype} (float32 or bfloat16, the input no narrower than 32 bits "
                          f"where the queries are)")
    S = 1
    if qkv.dim() == 3:
        S, rows, wide = _take(what, qkv, "qkv", torch.float32, 3, device)
    else:
        rows, wide = _take(what, qkv, "qkv", qkv.dtype, 2, device)
    q_rows, q_width = _take(what, q_out, "q_out", q_out.dtype, 2, device)
    if rows != T or wide != width or (S == 0 and T) or q_rows < T or q_width != num_heads * head_dim:
        raise KernelError(f"{what}: shapes disagree: qkv {tuple(qkv.shape)}, q_out {tuple(q_out.shape)}, {T} rows of {num_heads} + "
                          f"2 x {num_kv_heads} heads of {head_dim}")
    x, q, cs = qkv.data_ptr(), q_out.data_ptr(), 0
    if cos_sin is not None:
        angles, pairs, two = _take(what, cos_sin, "cos_sin", torch.float32, 3, device)
        cs = cos_sin.data_ptr()
        if angles < T or pairs != head_dim // 2 or two != 2:
            raise KernelError(f"{what}: cos_sin must be [T, head_dim/2, 2], is {tuple(cos_sin.shape)}")
    if (x | q | cs) % 16:
        raise KernelError(f"{what}: qkv, q_out and cos_sin must be 16-byte aligned")
    if pairing not in (0, 1, 2):
        raise KernelError(f"{what}: unknown pairing {pairing}")
    if T:
        call(core(), "ap_rope_kv8_store", x, dt, S, T * width, q, act, *cache, positions.data_ptr(), token_seq.data_ptr(), *table, cs,
             int(pairing), T, num_heads, num_kv_heads, head_dim, page_size, stream_handle())


def kv8_read(cache_layer: torch.Tensor, positions: torch.Tensor, token_seq: torch.Tensor, block_table: torch.Tensor,
             k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor], num_kv_heads: int, head_dim: int,
             page_size: int) -> None:
    """The keys and values of cached rows: row ``r`` of ``k_out`` and ``v_out`` (float32 or bfloat16 ``[rows, nkv*hd]``, either may be
    None) gets position ``positions[r]`` of sequence ``token_seq[r]``, exactly what the cache stands for (bfloat16 holds it too).
    A row without a page reads as zeros."""
    what = "kv8_read"
    device, T, cache, table = _take_cache(what, cache_layer, num_kv_heads, head_dim, page_size, positions, token_seq, block_table)
    some = k_out if k_out is not None else v_out
    if some is None:
        return
    dtype, width = some.dtype, num_kv_heads * head_dim
    code = _CODES.get(dtype)
    if code is None:
        raise KernelError(f"{what}: outputs of {dtype} are not taken (float32, bfloat16)")
    ptr = [0, 0]
    for i, t in enumerate((k_out, v_out)):
        if t is not None:
            rows, wide = _take(what, t, "an output", dtype, 2, device)
            ptr[i] = t.data_ptr()
            if rows < T or wide != width or ptr[i] % 16:
                raise KernelError(f"{what}: outputs must be 16-byte aligned [rows, {width}], one is {tuple(t.shape)}")
    if T:
        call(core(), "ap_kv8_read", *cache, positions.data_ptr(), token_seq.data_ptr(), *table, *ptr, code, T, num_kv_heads, head_dim,
             page_size, stream_handle())


_nonces = itertools.count(random.getrandbits(61))


@functools.lru_cache(maxsize=None)
def _sms(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


@functools.lru_cache(maxsize=None)
def _machine(device: int, num_heads: int, num_kv_heads: int, head_dim: int):
    """What the kernel for single rows runs on: its library, the SMs, ((CTAs to a cluster, such clusters that run at a time), ...), and the
    pairs that a row makes (a KV head and up to eight of its query heads each)."""
    lib = library.attention(head_dim)
    clusters = tuple((c, lib.ap_attention_kv8_decode_clusters(num_heads, num_kv_heads, c)) for c in (1, 2, 4, 8, 16))
    return lib, _sms(device), clusters, num_kv_heads * -(-(num_heads // num_kv_heads) // 8)


@functools.lru_cache(maxsize=4096)
def _rows_cost(pairs: int, longest: int, mean: int, sms: int, clusters):
    """(us, CTAs, CTAs to a cluster) of the kernel for single rows: ``pairs`` of a row and a KV head, of up to ``longest`` tiles of 64 keys,
    ``mean`` on average; ``clusters`` as from :func:`_machine`.  Clusters (0: none) give every pair CTAs of its own.

    Measured (one B200, pages scattered, us; a tile takes a CTA some 0.38 once its loads run): shared work costs 6 and five tiles' time for
    each pair beside its tiles where the CTAs hold several (64 rows of 2048 keys on 8 KV heads: 54.6, in clusters of one 69.9; 100 rows
    of a prompt: 21.3), 16 where nearly every pair is cut (20 rows of 2000 keys: 31; 8 rows of
    4096: 28.1; clusters of two 20.7).  A pair to a cluster costs 5.5, and 1.2 for putting parts together (1 row of 4096 keys: clusters
    of eight 9.9, shared 13.9; on one KV head of sixteen 8.5, of eight 9.7), but a CTA to an SM it leaves SMs idle (1 row of 32768: shared
    25.7, of eight 30.5), the longest row sets its time, and what does not fit at once takes a second turn (2 rows of 4096: of
    eight 20.1, of four 13.0; the 148 SMs hold 15 of eight, 33 of four)."""
    best = (16.0 + 0.39 * pairs * mean / sms if pairs < 2 * sms else 6.0 + 0.39 * pairs * (mean + 5) / sms, max(1, min(sms, pairs * mean // 2)), 0)
    for cluster, most in clusters:
        if pairs <= most and (cluster == 1 or longest >= cluster):
            best = min(best, (5.5 + 0.38 * -(-longest // cluster) + (1.2 if cluster > 1 else 0.0), pairs * cluster, cluster))
    return best


def plan_rows(*work):
    """(CTAs, CTAs to a cluster) for :func:`_rows_cost`'s work."""
    return _rows_cost(*work)[1:]


@functools.lru_cache(maxsize=None)
def _single_rows_taken(head_dim: int, page_size: int) -> bool:
    return bool(library.attention(head_dim).ap_attention_kv8_decode_takes(page_size))


@functools.lru_cache(maxsize=4096)
def _scratch_bytes(num_heads: int, num_kv_heads: int, head_dim: int, ctas: int) -> int:
    return library.attention(head_dim).ap_attention_kv8_decode_scratch(num_heads, num_kv_heads, ctas)


def _rows(q, out, cache, table, token_seq, positions, rows, num_heads, num_kv_heads, head_dim, page_size, scale, window, longest, mean,
          scratch, device) -> None:
    """The first ``rows`` rows one by one, up to ``longest`` keys to a row and some ``mean``."""
    lib, sms, clusters, sets = _machine(device, num_heads, num_kv_heads, head_dim)
    if window:
        longest, mean = min(longest, window + 64), min(mean, window + 64)
    step = 512
    x, y, seq, pos, width = q.data_ptr(), out.data_ptr(), token_seq.data_ptr(), positions.data_ptr(), num_heads * head_dim
    for r in range(0, rows, step):
        n = min(step, rows - r)
        ctas, cluster = plan_rows(n * sets, -(-longest // 64), -(-mean // 64), sms, clusters)
        at, need, nonce = 0, 0, 0
        if not cluster:
            nonce = next(_nonces) % (1 << 62) + 1
            need = _scratch_bytes(num_heads, num_kv_heads, head_dim, ctas)
            buf = scratch("attn.kv8", (need // 4,), torch.float32) if scratch is not None else \
                torch.empty(need // 4, dtype=torch.float32, device=q.device)
            at = buf.data_ptr()
        call(lib, "ap_attention_kv8_decode", x + 2 * r * width, y + 2 * r * width, *cache, *table, seq + 4 * r, pos + 4 * r, n,
             num_heads, num_kv_heads, head_dim, page_size, float(scale), int(window), ctas, cluster, at, need,
             nonce, stream_handle())


@functools.lru_cache(maxsize=None)
def _portions_taken(num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> int:
    """Tokens of a sequence in a query tile of the kernel for portions (0: it does not take the shape)."""
    lib = library.attention(head_dim)
    if not lib.ap_attention_kv8_tcgen05_takes(num_heads, num_kv_heads, head_dim, page_size):
        return 0
    return int(lib.ap_attention_kv8_tcgen05_tokens(num_heads, num_kv_heads))


def plan_portions(query_lens: Sequence[int], per_tile: int, num_kv_heads: int, keys: int, sms: int):
    """(query tiles to a CTA, CTAs to a KV head, key slices) of the kernel for portions: query tiles of ``per_tile`` tokens, rows that see
    some ``keys`` keys on average.

    Measured (one B200, 32 heads on 8 KV heads of 128, us).  Two query tiles share every key tile, and where only one of them is filled
    a CTA alone on its SM walks two key tiles at once (2048 rows behind nothing: 58, one tile 67; 17 behind 8191: 31, one tile 35); but
    two CTAs of one tile fit an SM, so one tile is taken where CTAs outnumber the SMs and a tenth of the second tiles would lie empty
    (32 sequences of 2 rows and 2000 keys: 123, two tiles 136; twelve prompts of 21 to 515 on heads of 64: 31, two tiles 35).  The
    keys are cut while CTAs are fewer than SMs and a slice keeps some two tiles of 128 keys (512 rows behind 4096 keys: 59 in two,
    88 whole; behind nothing: 24 in two, 22 whole; 64 behind 32000: 112 in eight, 170 in four; 12 sequences of 32 rows and 1000 keys: 54 in
    two, 42 whole)."""
    single = sum(-(-n // per_tile) for n in query_lens)
    ctas = sum(-(-n // (2 * per_tile)) for n in query_lens)
    if ctas * num_kv_heads > sms and 10 * single <= 19 * ctas:
        return 1, single, 1
    slices = 1
    while slices < 8 and ctas * num_kv_heads * slices * 2 <= sms and keys >= 480 * slices:
        slices *= 2
    return 2, ctas, slices


@functools.lru_cache(maxsize=4096)
def rows_are_faster(rows_us: float, sequences: int, longest: int, numbers: int, query_tiles: int, at_once: int, waves: int) -> bool:
    """Whether portions are better taken row by row, which costs ``rows_us``.  The kernel for portions costs its start and end, the
    widening of ``longest`` keys of ``numbers`` numbers to a sequence, and rounds of a key tile each.

    Measured (one B200, 32 heads on 8 KV heads of 128, us; row by row, as portions): 17 rows behind 1000 keys 11.2, 16.8; behind 4000 28.2,
    22.9; 64 rows behind 300 29.0, 17.5; 2 rows behind 30000 33.0, 69.3; 32 sequences of 2 rows and 2000 keys 54.5, 121; of 8 rows and 500
    keys (64 sequences) 120, 72; 12 of 32 rows and 1000 keys 148, 40."""
    rounds = -(-(-(-longest // 128)) // at_once)
    return rows_us < 14.0 + 1e-6 * sequences * longest * numbers + (2.0 if query_tiles == 2 else 2.5) * rounds * waves


# bytes of scratch for widened keys and values up to which sequences go together
WIDE_SCRATCH = 1 << 30


@functools.lru_cache(maxsize=256)
def step_lengths(query_lens: Tuple[int, ...], ones: int, contexts: Optional[Tuple[int, ...]], max_context: int, mean_context: int,
                 widest: int):
    """What a step with portions from sequence ``ones`` on is planned by: (longest context from there on, longest and average context of all
    rows).  Where ``contexts`` does not say, ``max_context`` counts only if there are no one-row sequences that it may stand for,
    else the width of the block table."""
    if contexts is None:
        longest = min(max_context if max_context and not ones and 1 not in query_lens else widest, widest)
        return longest, longest, min(mean_context or longest, longest)
    longest = min(max(contexts), widest)
    mean = sum(c * n for c, n in zip(contexts, query_lens)) // max(1, sum(query_lens))
    return max(1, min(max(contexts[ones:]), widest)), max(1, longest), max(1, min(mean, longest))


@functools.lru_cache(maxsize=256)
def _row_by_row(plan, faster, query_lens, per_tile, num_heads, num_kv_heads, head_dim, window, longest, device) -> bool:
    """Whether the portions of ``query_lens`` go to the kernel for single rows."""
    if window:
        longest = min(longest, window + max(query_lens))
    _, sms, clusters, sets = _machine(device, num_heads, num_kv_heads, head_dim)
    rows_us = _rows_cost(sum(query_lens) * sets, -(-longest // 64), -(-longest // 64), sms, clusters)[0]
    query_tiles, ctas, slices = plan(query_lens, per_tile, num_kv_heads, longest - max(query_lens) // 2, sms)
    at_once = slices * (2 if slices > 1 and max(query_lens) <= per_tile else 1)
    return faster(rows_us, len(query_lens), longest, num_kv_heads * head_dim, query_tiles, at_once,
                  -(-ctas * num_kv_heads * slices // (sms * (3 - query_tiles))))


def dense_tiles(rows: int, keys: int, window: int) -> int:
    """Tiles of 128 keys that a sequence of ``keys`` keys has among those that its last ``rows`` rows see."""
    tiles = -(-keys // 128)
    return max(1, min(tiles, (window + rows + 125) // 128 + 1) if window else tiles)      # (window + rows - 1 keys from anywhere on)


def group_portions(query_lens: Sequence[int], contexts: Sequence[int], window: int, most: int):
    """[(first sequence, one past the last, tiles of each), ...]: neighbours go together while their dense tiles, as many for each as the
    longest needs, are no more than ``most``; one alone always goes."""
    groups, first, widest = [], 0, 0
    for i, (rows, keys) in enumerate(zip(query_lens, contexts)):
        tiles = dense_tiles(rows, keys, window)
        if i > first and max(widest, tiles) * (i + 1 - first) > most:
            groups.append((first, i, widest))
            first, widest = i, 0
        widest = max(widest, tiles)
    return groups + [(first, len(query_lens), widest)]


def portions_scratch_bytes(num_kv_heads: int, head_dim: int, tokens: int, rows: int, sequences: int, window: int = 0) -> int:
    """Bytes of scratch that portions take at most in a step of up to ``rows`` rows and ``sequences`` sequences of up to ``tokens`` tokens:
    what one sequence needs, more only up to ``WIDE_SCRATCH``."""
    if head_dim not in (64, 128):
        return 0
    tile = num_kv_heads * (4 * 128 * head_dim + 4)
    one = dense_tiles(rows, tokens, window)
    return -(-tile * max(one, min(sequences * one, WIDE_SCRATCH // tile)) // 16) * 16


@functools.lru_cache(maxsize=256)
def _portions_plan(lib, plan, most, sms, query_lens, contexts, longest, widest, window, per_tile, num_kv_heads):
    """(bytes of scratch, [(first sequence, sequences, dense tiles of each, query tiles to a CTA, CTAs to a KV head, key slices), ...]), the same
    for every layer of a step."""
    keys = [widest] * len(query_lens) if contexts is None else [max(1, min(c, widest)) for c in contexts]
    groups, need = [], 0
    for at, end, tiles in group_portions(query_lens, keys, window, most // lib.ap_attention_kv8_tcgen05_scratch(1, num_kv_heads)):
        lens, seen = query_lens[at:end], longest if contexts is None else max(keys[at:end])
        if window:
            seen = min(seen, window + max(lens))
        groups.append((at, end - at, tiles, *plan(lens, per_tile, num_kv_heads, seen - max(lens) // 2, sms)))
        need = max(need, lib.ap_attention_kv8_tcgen05_scratch((end - at) * tiles, num_kv_heads))
    return need, groups


def _portions(q, out, cache, table, seq_start, positions, first_seq, query_lens, T, num_heads, num_kv_heads, head_dim, page_size, scale,
              window, per_tile, longest, contexts, scratch, device) -> None:
    """The sequences from ``first_seq`` on, by their ``query_lens``, of ``contexts`` keys each, or (None) some ``longest``; their rows follow
    those of the sequences before."""
    (blocks, width, _), lib = table, library.attention(head_dim)
    need, groups = _portions_plan(lib, plan_portions, WIDE_SCRATCH, _sms(device), query_lens, contexts, longest, width * page_size, window,
                                  per_tile, num_kv_heads)
    buf = scratch("attn.kv8_wide", (need // 2,), torch.bfloat16) if scratch is not None else \
        torch.empty(need // 2, dtype=torch.bfloat16, device=q.device)
    for at, sequences, tiles, query_tiles, ctas, slices in groups:
        if ctas:
            call(lib, "ap_attention_kv8_tcgen05", q.data_ptr(), out.data_ptr(), *cache, blocks + 4 * (first_seq + at) * width, width,
                 seq_start.data_ptr() + 4 * (first_seq + at), positions.data_ptr(), sequences, T, num_heads, num_kv_heads, head_dim,
                 page_size, float(scale), int(window), query_tiles, ctas, slices, tiles, buf.data_ptr(), need, stream_handle())


def attention_kv8(q: torch.Tensor, out: torch.Tensor, cache_layer: torch.Tensor, block_table: torch.Tensor,
                  token_seq: torch.Tensor, positions: torch.Tensor, num_heads: int, num_kv_heads: int, head_dim: int,
                  page_size: int, scale: float, window: int = 0, seq_start: Optional[torch.Tensor] = None,
                  query_lens: Optional[Sequence[int]] = None, max_context: int = 0, scratch=None,
                  mean_context: int = 0, contexts: Optional[Sequence[int]] = None) -> None:
    """Causal attention of every row of ``q [T, nh*hd]`` over its sequence's keys in the 8-bit cache; arguments as for
    :func:`attention`, with ``page_size`` beside the flat pages.  ``max_context`` and ``mean_context`` only say how to cut the work.
    ``contexts`` (host, one to a sequence of ``query_lens``): the sequences' keys, the newest row's among them (none may have
    more).  Without it portions are planned by ``max_context`` where no sequence brings one row, else by the width of the block
    table, and their scratch is as wide as the table.

    Scores, softmax and sums are 32-bit; in bfloat16 a weight is rounded to eight bits before it meets its value (single rows: together
    with the value's scale, and to 2^-18 of the largest such weight among 32 neighbours).  A row sees the keys at and before its
    position (the last ``window`` of them, 0: all) whose page is there; one that sees none gets zeros.  A key that is not finite makes
    the rows that see it NaN, a value their columns of it, no other row.

    The rows of a sequence follow one another and so do their positions; ``out`` is another tensor than ``q``.  Calls that may run
    at the same time need scratch of their own (None: each allocates it)."""
    what = "attention_kv8"
    device, T, cache, table = _take_cache(what, cache_layer, num_kv_heads, head_dim, page_size, positions, token_seq, block_table)
    code = _CODES.get(q.dtype)
    if code is None or num_heads <= 0 or num_heads % num_kv_heads or window < 0:
        raise KernelError(f"{what}: {num_heads} heads on {num_kv_heads} KV heads in {q.dtype}, window {window}")
    rows, width = shape = _take(what, q, "q", q.dtype, 2, device)
    if _take(what, out, "out", q.dtype, 2, device) != shape or rows < T or width != num_heads * head_dim \
            or (q.data_ptr() | out.data_ptr()) % 16:
        raise KernelError(f"{what}: q {tuple(q.shape)} and out {tuple(out.shape)} must be 16-byte aligned rows of {num_heads} heads of "
                          f"{head_dim}, {T} at least")
    by_sequence = seq_start is not None and query_lens is not None
    if by_sequence:
        starts, = _take(what, seq_start, "seq_start", torch.int32, 1, device)
        if starts != len(query_lens) + 1 or sum(query_lens) != T or table[2] < len(query_lens):
            raise KernelError(f"{what}: seq_start, query_lens and the block table do not describe the rows")
    if contexts is not None and (not by_sequence or len(contexts) != len(query_lens)):
        raise KernelError(f"{what}: contexts must name one number to a sequence of query_lens")
    if not T:
        return
    if code == AP_BF16 and 0 < cache[1] * cache[2] < 1 << 36 and _single_rows_taken(head_dim, page_size):
        # sequences that bring one row each, then portions (one-row sequences further back ride along with them)
        widest = table[1] * page_size
        ones, rows = 0, T
        longest = min(max_context or widest, widest)
        mean = min(mean_context or longest, longest)
        if by_sequence:
            # (as many sequences as rows: one each, or none and several here and there, which the rows' own metadata says as well)
            ones = next((i for i, n in enumerate(query_lens) if n != 1), len(query_lens)) if len(query_lens) != T else T
            if ones < len(query_lens):
                query_lens, contexts = tuple(query_lens), tuple(contexts) if contexts is not None else None
                behind, all_longest, all_mean = step_lengths(query_lens, ones, contexts, max_context, mean_context, widest)
                per_tile = _portions_taken(num_heads, num_kv_heads, head_dim, page_size) if scale > 0 else 0
                if per_tile and not (T <= 512 and _row_by_row(plan_portions, rows_are_faster, query_lens[ones:], per_tile, num_heads,
                                                              num_kv_heads, head_dim, window, behind, device)):
                    _portions(q, out, cache, table, seq_start, positions, ones, query_lens[ones:], T, num_heads, num_kv_heads, head_dim,
                              page_size, scale, window, per_tile, behind, None if contexts is None else contexts[ones:], scratch, device)
                    rows = ones
                else:
                    longest, mean = all_longest, all_mean
        if rows:
            _rows(q, out, cache, table, token_seq, positions, rows, num_heads, num_kv_heads, head_dim, page_size, scale, window,
                  longest, mean, scratch, device)
        return
    call(library.attention(head_dim), "ap_attention_kv8_rows", q.data_ptr(), out.data_ptr(), code, *cache, *table,
         token_seq.data_ptr(), positions.data_ptr(), T, num_heads, num_kv_heads, head_dim, page_size, float(scale), int(window),
         stream_handle())
