"""Keys and values in 8 bits: the operators of a quantised paged cache, as cases that can be timed and compared.

A cache page holds, for every key/value head, ``page`` rows of ``head_dim`` numbers of 8 bits (e4m3) for the keys and as many
for the values, then one scale to a row, a power of two held as its exponent plus 127 in a byte.  A pass is one call's work:

* ``append``: the rows of a step are rotated, their keys and values are rounded to 8 bits and put into their pages, and the
  same rows are read back as the values that the pages now stand for (queries, keys and values come back);
* ``read``: cached rows of whole conversations come back as keys and values;
* ``decode``: sequences that bring one row each attend to their cached keys;
* ``chunk``: sequences that bring several new rows attend, each row to the keys at and before its own position.

Where ``own`` is false the operators run in their plain form, elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

LOWEST, HIGHEST = -60, 40           # exponents of a row's scale
LARGEST = 448.0                     # of the numbers of 8 bits
PAGE = 16


def _case(name, op, heads, dtype="bfloat16", page=PAGE, pages="scattered", window=0, **more):
    nh, nkv, hd = heads
    return {"name": name, "op": op, "heads": nh, "kv_heads": nkv, "head_dim": hd, "dtype": dtype, "page": page,
            "pages": pages, "window": window, **more}


L8B, L1B = (32, 8, 128), (32, 8, 64)        # the head layouts of the two Llama shapes of the benchmark
LAYOUTS = (L8B, L8B, L1B, L1B, (16, 2, 64), (8, 8, 64), (16, 1, 128))


def listed():
    return [
        # a token of one conversation: the projection's 32-bit partial sums, latency of two small launches
        _case("append one row, 1b", "append", L1B, rows=1, slices=4, pairing=0, behind=300),
        # a decode step of 64 conversations
        _case("append 64 rows, 8b", "append", L8B, rows=64, slices=1, pairing=2, behind=2000),
        # a portion of a prompt
        _case("append 2048 rows, 8b", "append", L8B, rows=2048, slices=1, pairing=2, behind=0),
        # one conversation's keys and values, to be looked at or kept elsewhere
        _case("read one conversation, 8b", "read", L8B, sequences=1, shortest=777, longest=777, out="bfloat16"),
        # the cache of many conversations of unequal length
        _case("read sixteen ragged, 8b", "read", L8B, sequences=16, shortest=200, longest=8000, out="bfloat16"),
        # a question to a small model: latency
        _case("decode one short, 1b", "decode", L1B, sequences=1, shortest=300, longest=300),
        # a long document behind one answer: few rows, so the keys are what can be split
        _case("decode one long, 8b", "decode", L8B, pages="rising", sequences=1, shortest=32768, longest=32768),
        # a busy server, contexts of unequal length
        _case("decode 64 ragged, 8b", "decode", L8B, sequences=64, shortest=150, longest=4096),
        # the 32-bit engine
        _case("decode four, 1b float32", "decode", L1B, dtype="float32", sequences=4, shortest=20, longest=700),
        # a short question behind a document that is cached already
        _case("chunk of 17 behind 8191, 8b", "chunk", L8B, sequences=1, shortest=17, longest=17, behind=8191),
        # several whole prompts of a small model in one step
        _case("chunk of twelve prompts, 1b", "chunk", L1B, sequences=12, shortest=21, longest=515, behind=0),
        # a large portion of a long document
        _case("chunk of 2048 behind 30000, 8b", "chunk", L8B, pages="rising", sequences=1, shortest=2048, longest=2048,
              behind=30000),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "read", "decode", "decode", "chunk", "chunk"))
    heads = rng.choice(LAYOUTS)
    more = {"page": rng.choice((16, 16, 16, 32, 64, 128)), "pages": rng.choice(("scattered", "rising"))}
    if op == "append":
        rows = _log_uniform(rng, 1, 4096)
        return _case("", op, heads, dtype=rng.choice(("bfloat16", "bfloat16", "float32")), rows=rows,
                     slices=rng.choice((1, 2, 4)) if rows <= 64 else 1, pairing=rng.choice((0, 1, 2)),
                     behind=_log_uniform(rng, 1, 30000), **more)
    if op == "read":
        n = _log_uniform(rng, 1, 32)
        longest = _log_uniform(rng, 1, 131072 // n)
        return _case("", op, heads, sequences=n, longest=longest, shortest=_log_uniform(rng, 1, longest),
                     out=rng.choice(("bfloat16", "float32")), **more)
    more["window"] = rng.choice((0, 0, 0, 500, 1024))
    if op == "decode":
        n = _log_uniform(rng, 1, 128)
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "bfloat16", "float32"))
        longest = _log_uniform(rng, 1, min(65536, 262144 // n) if dtype == "bfloat16" else 2000)
        return _case("", op, heads, dtype=dtype, sequences=n, longest=longest, shortest=_log_uniform(rng, 1, longest), **more)
    n = _log_uniform(rng, 1, 16)
    longest = _log_uniform(rng, 2, 2048 // n)
    return _case("", op, heads, sequences=n, longest=longest, shortest=_log_uniform(rng, 2, longest),
                 behind=rng.choice((0, _log_uniform(rng, 1, 16384 // n))), **more)


# ---- lengths and pages, the same for every seed --------------------------------------------------------------------
def _spread(n, lo, hi, salt):
    """``n`` lengths from ``lo`` to ``hi``, even over their logarithm, in a fixed disorder."""
    at = [1.0 if n == 1 else i / (n - 1) for i in range(n)]
    out = [int(round(math.exp(math.log(lo) + a * (math.log(hi) - math.log(lo))))) for a in at]
    random.Random(salt).shuffle(out)
    return out


def _lengths(c):
    """(new rows, keys) of every sequence: its rows are the last of its keys."""
    if c["op"] == "append":
        n = c["rows"] if c["rows"] <= 64 else 1          # a decode step's rows, or one prompt's portion
        new = [c["rows"] // n] * n
        return new, [b + w for b, w in zip(_spread(n, max(1, c["behind"] // 8), max(1, c["behind"]), 3), new)]
    if c["op"] == "chunk":
        new = _spread(c["sequences"], c["shortest"], c["longest"], 5)
        behind = _spread(c["sequences"], max(1, c["behind"] // 4), c["behind"], 7) if c["behind"] else [0] * len(new)
        return new, [b + w for b, w in zip(behind, new)]
    keys = _spread(c["sequences"], c["shortest"], c["longest"], 9)
    return ([1] * len(keys) if c["op"] == "decode" else keys), keys


def _page_bytes(c):
    n = 2 * c["kv_heads"] * c["page"] * (c["head_dim"] + 1)
    return -(-n // 16) * 16


def _table(c, keys):
    """Block table [sequences, blocks] (-1: no page) and the number of pages."""
    P = c["page"]
    counts = [-(-k // P) for k in keys]
    total = sum(counts)
    ids = list(range(total))
    if c["pages"] == "scattered":
        random.Random(11).shuffle(ids)
    rows, at, widest = [], 0, max(counts)
    for n in counts:
        rows.append(ids[at:at + n] + [-1] * (widest - n))
        at += n
    return rows, total


# ---- numbers of 8 bits, in plain torch -------------------------------------------------------------------------------
def _power(e):
    """2^e in 32 bits, exactly (e an int tensor from -126 to 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """Rows [..., n] in 32 bits -> (e4m3 [..., n], exponents [...]): the smallest power of two under which no number is
    above the largest one of 8 bits."""
    amax = x.abs().amax(-1)
    m, e = torch.frexp(amax)                                  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), torch.full_like(e, LOWEST)).clamp(LOWEST, HIGHEST)
    y = (x * _power(-e).unsqueeze(-1)).clamp(-LARGEST, LARGEST)
    return y.to(torch.float8_e4m3fn), e


def _split_pages(c, pages):
    """(numbers [pages, 2, kv_heads, page, head_dim] uint8, scales [pages, 2, kv_heads, page] uint8), views."""
    nkv, P, hd = c["kv_heads"], c["page"], c["head_dim"]
    n = 2 * nkv * P * hd
    return (pages[:, :n].unflatten(1, (2, nkv, P, hd)), pages[:, n:n + 2 * nkv * P].unflatten(1, (2, nkv, P)))


def _rows_of(c, pages, page, slot):
    """The rows ``slot`` of ``page`` (index tensors of one shape) as values in 32 bits, [..., 2, kv_heads, head_dim]."""
    data, scale = _split_pages(c, pages)
    x = data[page, :, :, slot].view(torch.float8_e4m3fn).float()
    return x * _power(scale[page, :, :, slot].to(torch.int32) - 127).unsqueeze(-1)


class _State(dict):
    __getattr__ = dict.__getitem__


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    nh, nkv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    dtype = getattr(torch, c["dtype"])

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)
    new, keys = _lengths(c)
    rows, total = _table(c, keys)
    T = sum(new)
    token_seq = [s for s, n in enumerate(new) for _ in range(n)]
    positions = [k - n + i for n, k in zip(new, keys) for i in range(n)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)
    s = _State(case=c, T=T, query_lens=new, table=ints(rows), token_seq=ints(token_seq), positions=ints(positions),
               seq_start=ints(starts), longest=max(keys), longest_new=max(new), mean=sum(keys) // len(keys),
               pages=torch.zeros((total, _page_bytes(c)), dtype=torch.uint8, device=dev))
    # channels of unequal size, as norms and projections leave them; some tokens are louder than others
    channel = torch.exp(0.5 * randn(2, nkv, 1, hd))
    if c["op"] == "append":
        x = randn(T, (nh + 2 * nkv), hd)
        x[:, nh:nh + nkv] *= channel[0, :, 0]
        x[:, nh + nkv:] *= channel[1, :, 0] * torch.exp(0.5 * randn(T, nkv, 1))
        if c["slices"] > 1:
            x = x / math.sqrt(c["slices"])
            s["qkv"] = torch.stack([x] + [randn(*x.shape) * x.abs().mean() for _ in range(c["slices"] - 1)]).flatten(2)
        else:
            s["qkv"] = x.flatten(1).to(dtype)
        inv = 500000.0 ** (-torch.arange(hd // 2, dtype=torch.float64, device=dev) / (hd // 2))
        angle = s.positions.double()[:, None] * inv
        s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float()
        s["q"] = torch.empty((T, nh * hd), dtype=dtype, device=dev)
        s["k"], s["v"] = (torch.empty((T, nkv * hd), dtype=torch.bfloat16, device=dev) for _ in range(2))
        return s
    data, scale = _split_pages(c, s.pages)
    step = max(1, (1 << 27) // (2 * nkv * P * hd))
    for a in range(0, total, step):
        n = min(step, total - a)
        x = randn(n, 2, nkv, P, hd) * channel
        x[:, 1] *= torch.exp(0.7 * randn(n, nkv, P, 1))
        codes, e = _quantise(x)
        data[a:a + n] = codes.view(torch.uint8)
        scale[a:a + n] = (e + 127).to(torch.uint8)
    if c["op"] == "read":
        out = getattr(torch, c["out"])
        s["k"], s["v"] = (torch.empty((T, nkv * hd), dtype=out, device=dev) for _ in range(2))
        return s
    s["q"] = randn(T, nh * hd).to(dtype)
    s["out"] = torch.empty_like(s.q)
    s["scale"] = 1.0 / math.sqrt(hd)
    kept = {}

    def scratch(name, shape, dt):
        key = (name, tuple(shape), dt)
        if key not in kept:
            kept[key] = torch.empty(shape, dtype=dt, device=dev)
        return kept[key]
    s["scratch"] = scratch
    return s


def run(s):
    c = s.case
    nh, nkv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    if own:
        from allpaca_b200 import ops
        if c["op"] == "append":
            ops.rope_kv8_store(s.qkv, s.q, s.pages, s.positions, s.token_seq, s.table, s.cos_sin, c["pairing"], nh, nkv, hd, P)
            ops.kv8_read(s.pages, s.positions, s.token_seq, s.table, s.k, s.v, nkv, hd, P)
            return s.q, s.k, s.v
        if c["op"] == "read":
            ops.kv8_read(s.pages, s.positions, s.token_seq, s.table, s.k, s.v, nkv, hd, P)
            return s.k, s.v
        ops.attention_kv8(s.q, s.out, s.pages, s.table, s.token_seq, s.positions, nh, nkv, hd, P, s.scale, c["window"],
                          seq_start=s.seq_start, query_lens=s.query_lens, max_context=s.longest, scratch=s.scratch,
                          mean_context=s.mean)
        return s.out
    seq, pos = s.token_seq.long(), s.positions.long()
    if c["op"] == "append":
        return _plain_append(s, seq, pos)
    if c["op"] == "read":
        kv = _rows_of(c, s.pages, s.table[seq, pos // P].long(), pos % P).to(s.k.dtype)
        return kv[:, 0].flatten(1), kv[:, 1].flatten(1)
    return _plain_attention(s, seq, pos)


def _plain_append(s, seq, pos):
    c = s.case
    nh, nkv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    x = s.qkv.float()
    x = (x.sum(0) if x.dim() == 3 else x).unflatten(1, (nh + 2 * nkv, hd))
    qk, v = x[:, :nh + nkv], x[:, nh + nkv:]
    a, b = (qk[..., :hd // 2], qk[..., hd // 2:]) if c["pairing"] == 0 else (qk[..., 0::2], qk[..., 1::2])
    cos, sin = s.cos_sin[:, None, :, 0], s.cos_sin[:, None, :, 1]
    ra, rb = a * cos - b * sin, a * sin + b * cos
    qk = torch.stack([ra, rb], -1).flatten(2) if c["pairing"] == 1 else torch.cat([ra, rb], -1)
    page, slot = s.table[seq, pos // P].long(), pos % P
    codes, e = _quantise(torch.stack([qk[:, nh:], v], 1))
    data, scale = _split_pages(c, s.pages)
    data[page, :, :, slot] = codes.view(torch.uint8)
    scale[page, :, :, slot] = (e + 127).to(torch.uint8)
    kv = _rows_of(c, s.pages, page, slot).to(torch.bfloat16)
    return qk[:, :nh].flatten(1).to(s.q.dtype), kv[:, 0].flatten(1), kv[:, 1].flatten(1)


def _plain_attention(s, seq, pos):
    """All sequences at once: the rows padded to the longest portion, the keys to the longest context."""
    c = s.case
    nh, nkv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    n, L = s.table.shape[0], s.table.shape[1] * P
    at = torch.arange(L, device=pos.device)
    kv = _rows_of(c, s.pages, s.table[:, at // P].clamp(min=0).long(), (at % P).expand(n, L))     # [n, L, 2, nkv, hd]
    k, v = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)                               # [n, nkv, L, hd]
    place = torch.arange(s.T, device=pos.device) - s.seq_start.long()[seq]
    q = torch.zeros((n, s.longest_new, nh, hd), device=pos.device)
    q[seq, place] = s.q.float().unflatten(1, (nh, hd))
    where = torch.full((n, s.longest_new), -1, dtype=torch.long, device=pos.device)
    where[seq, place] = pos
    group = nh // nkv
    q = q.unflatten(2, (nkv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)                         # [n, nkv, group * rows, hd]
    score = (q @ k.transpose(2, 3)).unflatten(2, (group, s.longest_new)) * s.scale
    seen = at <= where[..., None]
    if c["window"]:
        seen &= at > where[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).unflatten(2, (group, s.longest_new)) / total                      # [n, nkv, group, rows, hd]
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, place].flatten(1).to(s.q.dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    c = case
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    new, keys = _lengths(c)
    T, wide = sum(new), 2 if c["dtype"] == "bfloat16" else 4
    row = 2 * nkv * (hd + 1)                                   # a token's keys and values with their scales
    if c["op"] == "append":
        into = T * (nh + 2 * nkv) * hd * (wide if c["slices"] == 1 else 4 * c["slices"])
        return {"bytes": into + T * (nh * hd * wide + row + hd * 4 + 2 * nkv * hd * 2 + 8),
                "flops": T * (3 * (nh + nkv) * hd + 6 * nkv * hd + (c["slices"] - 1) * (nh + 2 * nkv) * hd)}
    if c["op"] == "read":
        return {"bytes": T * (row + 2 * nkv * hd * (2 if c["out"] == "bfloat16" else 4) + 8), "flops": T * 2 * nkv * hd}
    window = c["window"] or max(keys)
    seen = sum(min(k - n + i + 1, window) for n, k in zip(new, keys) for i in range(n))
    read = sum(min(k, window + n - 1) for n, k in zip(new, keys))
    return {"bytes": read * row + 2 * T * nh * hd * wide + 8 * T, "flops": 4 * seen * nh * hd}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _values64(byte):
    """What the 256 numbers of 8 bits stand for: sign, four bits of exponent (bias 7), three of fraction; 127 is no number."""
    t = []
    for i in range(256):
        e, f = (i >> 3) & 15, i & 7
        x = f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        t.append(math.nan if i & 127 == 127 else -x if i & 128 else x)
    return torch.tensor(t, dtype=torch.float64, device=byte.device)[byte.long()]


def _power64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _rounded64(x):
    """Rows in 64 bits -> the values that 8 bits and a power of two keep of them."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True) / 448)
    e = torch.where(m > 0, e - (m == 0.5).to(e.dtype), torch.full_like(e, -60)).clamp(-60, 40)
    y = x / _power64(e)
    unit = _power64(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.round(y / unit) * unit).clamp(-448, 448) * _power64(e)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    nh, nkv, hd, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    half, number = hd // 2, 2 * nkv * P * hd
    if c["op"] == "append":
        x = s.qkv.double()
        x = x.reshape(-1, s.T, nh + 2 * nkv, hd).sum(0)
        rot = torch.zeros(nh + nkv, s.T, hd, dtype=torch.float64, device=x.device)
        for i in range(half):
            a, b = (x[:, :nh + nkv, i], x[:, :nh + nkv, i + half]) if c["pairing"] == 0 else \
                (x[:, :nh + nkv, 2 * i], x[:, :nh + nkv, 2 * i + 1])
            turn = s.positions.double() * 500000.0 ** (-i / half)
            to = (2 * i, 2 * i + 1) if c["pairing"] == 1 else (i, i + half)
            rot[:, :, to[0]] = (a * turn.cos()[:, None] - b * turn.sin()[:, None]).T
            rot[:, :, to[1]] = (a * turn.sin()[:, None] + b * turn.cos()[:, None]).T
        rot = rot.transpose(0, 1)
        return rot[:, :nh].flatten(1), _rounded64(rot[:, nh:]).flatten(1), _rounded64(x[:, nh + nkv:]).flatten(1)
    new, keys = _lengths(c)
    outs, row = [], 0
    for i, (n, length) in enumerate(zip(new, keys)):
        pages = s.pages[s.table[i, :-(-length // P)].long()]
        x = _values64(pages[:, :number]).reshape(-1, 2, nkv, P, hd)
        x = x * _power64(pages[:, number:number + 2 * nkv * P].reshape(-1, 2, nkv, P, 1).int() - 127)
        k, v = x.permute(1, 2, 0, 3, 4).reshape(2, nkv, -1, hd)[:, :, :length]
        if c["op"] == "read":
            outs.append(torch.stack([k, v]).permute(0, 2, 1, 3).reshape(2, length, nkv * hd))
            continue
        at = torch.arange(length, device=x.device)
        mine = torch.arange(length - n, length, device=x.device)[:, None]
        hidden = (at > mine) | (at <= mine - (c["window"] or length + 1))
        out = torch.empty(n, nh, hd, dtype=torch.float64, device=x.device)
        for h in range(nh):
            q = s.q[row:row + n, h * hd:(h + 1) * hd].double()
            score = (q @ k[h // (nh // nkv)].T) / math.sqrt(hd)
            out[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[h // (nh // nkv)]
        outs.append(out.flatten(1))
        row += n
    if c["op"] == "read":
        both = torch.cat(outs, 1)
        return both[0], both[1]
    return torch.cat(outs)
