"""From a token's projection to attention over a cache held in 8 bits.

Four operators of ``lsa_rocm_lab.port.pipeline`` that stand around the selection:

* ``rotate``: norms of the heads of queries and keys and their rotary positions, in one pass;
* ``byte_append``: the same, and keys and values into a cache of 8-bit codes with a scale for each
  block of tokens and kv-head;
* ``byte_values``: what such a cache holds, as numbers (the index is built over these);
* ``byte_read``: attention over read lists of it.

Where ``own`` is false ``run`` computes them from elementary torch operations. Inputs come from
the seed alone; ``exact`` states the results in 64 bits.
"""

import math
import pathlib
import sys

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
LEAST = 2.0 ** -100  # the smallest scale
EPS = 1e-6
DEV = "cuda"


# ------------------------------------------------------------------------------- the cases


def listed():
    full = dict(heads_q=32, heads_kv=8, head_dim=128, dtype="bf16")
    turn = dict(interleaved=False, turned=128, norm=True)
    return [
        # one token of one request: the launch is all of it
        dict(name="rotate_b1", op="rotate", batch=1, tokens=1, start=30000, **full, **turn),
        # pieces of three prompts; pairs side by side, half of each head turned, no norm
        dict(name="rotate_3x1237_fp16", op="rotate", batch=3, tokens=1237, start=2048, heads_q=32, heads_kv=8, head_dim=128,
             dtype="fp16", interleaved=True, turned=64, norm=False),
        # a whole 32k prompt
        dict(name="rotate_32k", op="rotate", batch=1, tokens=32768, start=0, **full, **turn),
        # a decode step of a serving batch: one token a row into its open page
        dict(name="append_b32", op="append", batch=32, tokens=1, cache=2048, block=64, code="e4m3", page=64, ragged=False,
             **full, **turn),
        # pieces of five prompts, padded to one length, into a paged pool
        dict(name="append_5x300_fp16", op="append", batch=5, tokens=300, cache=2048, block=16, code="int8", page=16,
             ragged=True, heads_q=32, heads_kv=8, head_dim=128, dtype="fp16", interleaved=True, turned=128, norm=True),
        # a whole 32k prompt
        dict(name="append_32k", op="append", batch=1, tokens=32768, cache=32768, block=64, code="int8", page=0, ragged=False,
             **full, **turn),
        # the open parts of five paged caches, for their index
        dict(name="values_5x2050", op="values", batch=5, rows=2050, cache=4096, block=16, code="e4m3", page=16, heads_kv=8,
             head_dim=64, dtype="fp16"),
        # a 32k cache
        dict(name="values_32k", op="values", batch=1, rows=0, cache=32768, block=64, code="int8", page=0, heads_kv=8,
             head_dim=128, dtype="bf16"),
        # the single-stream decode at 32k: 32 spans of about 64 keys a kv-head
        dict(name="read_32k", op="read", batch=1, tokens=1, cache=32768, block=16, code="e4m3", page=0, lists="heads",
             spans=32, **full),
        # of a full batch
        dict(name="read_b32_32k", op="read", batch=32, tokens=1, cache=32768, block=64, code="int8", page=0, lists="heads",
             spans=32, **full),
        # four draft tokens of five requests over a paged pool, lists of about 4600 keys shared by the heads
        dict(name="read_5x4_paged_fp16", op="read", batch=5, tokens=4, cache=12300, block=16, code="e4m3", page=16,
             lists="shared", spans=72, heads_q=32, heads_kv=8, head_dim=128, dtype="fp16"),
        # every key of sixteen paged 32k caches
        dict(name="read_whole_b16_32k", op="read", batch=16, tokens=1, cache=32768, block=64, code="int8", page=64,
             lists="whole", spans=0, **full),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "append", "values", "read", "read", "read"])
    heads_kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 64, 128, 128, 128, 256])
    heads = dict(heads_q=heads_kv * rng.choice([1, 2, 3, 4, 8]), heads_kv=heads_kv, head_dim=dim,
                 dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    e = 4 if heads["dtype"] == "fp32" else 2
    turn = dict(interleaved=rng.random() < 0.4, turned=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                norm=rng.random() < 0.7)
    block = rng.choice([1, 16, 16, 32, 64, 64])
    held = dict(block=block, code=rng.choice(["int8", "e4m3"]), page=rng.choice([0, 0, max(16, block)]))
    if op == "rotate":
        row = (heads["heads_q"] + heads_kv) * dim * e
        tokens = _log_int(rng, 1, min(32768, (1 << 28) // row))
        batch = rng.choice([1, 1, 3]) if tokens > 64 else _log_int(rng, 1, 32)
        return dict(op=op, batch=batch, tokens=-(-tokens // batch), start=_log_int(rng, 1, 131072), **heads, **turn)
    if op == "append":
        one = rng.random() < 0.4
        batch = _log_int(rng, 1, 64) if one else _log_int(rng, 1, 8)
        row = (heads["heads_q"] + 2 * heads_kv) * dim * e
        tokens = 1 if one else _log_int(rng, 2, min(8192, (1 << 28) // row) // batch)
        return dict(op=op, batch=batch, tokens=tokens, cache=tokens + _log_int(rng, 1, 2048), **held,
                    ragged=not one and rng.random() < 0.5, **heads, **turn)
    if op == "values":
        heads.pop("heads_q")
        batch = _log_int(rng, 1, 8)
        cache = _log_int(rng, 64, min(8192, (1 << 26) // (batch * heads_kv * dim)))
        whole = not held["page"] and rng.random() < 0.4
        return dict(op=op, batch=batch, rows=0 if whole else _log_int(rng, 1, cache), cache=cache, **held, **heads)
    lists = rng.choice(["heads", "heads", "shared", "whole"])
    tokens = rng.choice([1, 1, 1, 2, 4, 17])
    spans = 0 if lists == "whole" else _log_int(rng, 1, 72)
    cache = _log_int(rng, 64, 32768) + 64 * spans
    most = (1 << 28) // (heads_kv * dim * (cache if lists == "whole" else 64 * spans))  # of listed codes
    batch = _log_int(rng, 1, max(1, min(32, most // tokens, (1 << 28) // (heads_kv * dim * cache))))
    return dict(op=op, batch=batch, tokens=min(tokens, max(1, most // batch)), cache=cache, lists=lists, spans=spans,
                **held, **heads)


# ------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys(lead, T, Hkv, D, dtype, gen):
    """[lead, T, Hkv, D]: runs of 64 tokens a cluster, center ~ N(0, 1) plus 0.3 N(0, 1)."""
    centers = torch.randn(lead, -(-T // 64), 1, Hkv, D, device=DEV, generator=gen, dtype=dtype)
    k = centers.expand(-1, -1, 64, -1, -1).reshape(lead, -1, Hkv, D)[:, :T]
    return (k + 0.3 * torch.randn(lead, T, Hkv, D, device=DEV, generator=gen, dtype=dtype)).contiguous()


def _coded(x, code):
    kind, most = CODES[code]
    x = x.clamp(-most, most)
    return (torch.round(x) if code == "int8" else x).to(kind)


def _held(x, block, code):
    """Codes and block scales of x [T, Hkv, D]."""
    T, H, D = x.shape
    pad = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, -T % block)).view(-1, block, H, D)
    scale = (pad.abs().amax((1, 3)) / CODES[code][1]).clamp(min=LEAST)
    return _coded(pad / scale[:, None, :, None], code).view(-1, H, D)[:T], scale


def _cache(c, gen, filled=None):
    """Codes [B or 1, T, Hkv, D], scales [B or 1, blocks, Hkv, 2] and, paged, the slot table [B, T].
    Positions of a row from ``filled`` on hold nothing yet."""
    B, T, H, D, block, page = (c[n] for n in ("batch", "cache", "heads_kv", "head_dim", "block", "page"))
    kind = CODES[c["code"]][0]
    whole = -(-T // page) * page if page else T
    blocks = -(-whole // block)
    k8, v8 = (torch.zeros(B, whole, H, D, device=DEV, dtype=kind) for _ in range(2))
    scales = torch.zeros(B, blocks, H, 2, device=DEV)
    for b in range(B):
        for i, (x, into) in enumerate(((_keys(1, whole, H, D, torch.bfloat16, gen)[0], k8),
                                       (torch.randn(whole, H, D, device=DEV, generator=gen, dtype=torch.bfloat16), v8))):
            if filled is not None:
                x = x * (torch.arange(whole, device=DEV) < filled[b])[:, None, None]
            into[b], scales[b, :, :, i] = _held(x, block, c["code"])
    if not page:
        return dict(k8=k8, v8=v8, scales=scales, table=None, block=block, code=c["code"])
    pages = whole // page
    where = torch.randperm(B * pages, device=DEV, generator=gen)
    table = (where.view(B, pages, 1) * page + torch.arange(page, device=DEV)).reshape(B, whole)
    back = torch.empty_like(where).index_copy_(0, where, torch.arange(B * pages, device=DEV))  # a pool page's place
    k8, v8, scales = (x.reshape(B * pages, -1).view(torch.uint8)[back].view(x.dtype).view(1, -1, *x.shape[2:])
                      for x in (k8, v8, scales))
    return dict(k8=k8, v8=v8, scales=scales, table=table[:, :T].to(torch.int32).contiguous(), block=block, code=c["code"])


def _heads(c, gen, tokens, with_v):
    """q, k (and v) as views of one projection's rows, the norms' weights and the frequencies."""
    B, Hq, Hkv, D, dt = (c[n] for n in ("batch", "heads_q", "heads_kv", "head_dim", "dtype"))
    rows = torch.randn(B, tokens, Hq + 2 * Hkv, D, device=DEV, generator=gen, dtype=DTYPES[dt])
    half = c["turned"] // 2
    s = dict(q=rows[:, :, :Hq], k=rows[:, :, Hq:Hq + Hkv], interleaved=c["interleaved"], wq=None, wk=None,
             freq=(10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)).float())
    if with_v:
        s["v"] = rows[:, :, Hq + Hkv:]
    if c["norm"]:
        s["wq"], s["wk"] = (torch.rand(D, device=DEV, generator=gen).add(0.5).to(DTYPES[dt]) for _ in range(2))
    return s


def _rotate_inputs(c, seed):
    gen = _gen(seed)
    s = _heads(c, gen, c["tokens"], False)
    first = torch.randint(c["start"] // 2, c["start"] + 1, (c["batch"], 1), device=DEV, generator=gen)
    s["pos"] = (first + torch.arange(c["tokens"], device=DEV)).to(torch.int32)
    return s


def _append_inputs(c, seed):
    gen = _gen(seed)
    B, n, T, block = c["batch"], c["tokens"], c["cache"], c["block"]
    s = _heads(c, gen, n, True)
    s["starts"] = torch.randint(0, T - n + 1, (B,), device=DEV, generator=gen).to(torch.int32)
    s["lens"] = torch.randint(0, n + 1, (B,), device=DEV, generator=gen).to(torch.int32) if c["ragged"] else None
    s.update(_cache(c, gen, s["starts"]))
    # the rows from the first block that is written to, up to the last token
    base = s["starts"].long() // block * block
    end = s["starts"] + (n if s["lens"] is None else s["lens"])
    at = base[:, None] + torch.arange(min(n + block, T), device=DEV)
    s["ids"] = (s["table"].long().gather(1, at.clamp(max=T - 1)) if c["page"] else at).to(torch.int32).contiguous()
    s["nids"] = (end - base).to(torch.int32)
    return s


def _values_inputs(c, seed):
    gen = _gen(seed)
    s = dict(_cache(c, gen), dtype=DTYPES[c["dtype"]], ids=None, nids=None)
    if c["rows"]:
        B, T, n = c["batch"], c["cache"], c["rows"]
        at = torch.randint(0, T - n + 1, (B, 1), device=DEV, generator=gen) + torch.arange(n, device=DEV)
        s["ids"] = (s["table"].long().gather(1, at) if c["page"] else at).to(torch.int32).contiguous()
        s["nids"] = torch.randint(n // 2, n + 1, (B,), device=DEV, generator=gen).to(torch.int32)
    return s


SPAN = 88  # the longest span of a list; 40 to 88 keys, 64 on average


def _read_inputs(c, seed):
    gen = _gen(seed)
    B, Tq, T, n, Hkv = c["batch"], c["tokens"], c["cache"], c["spans"], c["heads_kv"]
    s = _cache(c, gen)
    if c["lists"] == "whole":  # the first keys of each row
        lens = torch.randint(-(-T // 2), T + 1, (B, 1), device=DEV, generator=gen).expand(B, Tq)
        ids = torch.arange(T, device=DEV).expand(B, Tq, T)
    else:
        lead = (B, Tq, Hkv) if c["lists"] == "heads" else (B, Tq)
        cells = max(n, T // SPAN)  # a span begins in a cell of its own
        width = T // cells
        start = torch.rand(*lead, cells, device=DEV, generator=gen).argsort(-1)[..., :n] * width
        size = torch.randint(40, SPAN + 1, (*lead, n), device=DEV, generator=gen).clamp(max=width)
        slot = torch.arange(SPAN, device=DEV)
        ids = torch.where(slot < size[..., None], start[..., None] + slot, -1).flatten(-2)
        ids = ids.gather(-1, (ids < 0).to(torch.int8).argsort(dim=-1, stable=True))  # the listed first
        lens = size.sum(-1)
    if c["page"]:
        table = s["table"].long().view(B, *[1] * (ids.dim() - 2), T).expand(*ids.shape[:-1], T)
        ids = torch.where(ids >= 0, table.gather(-1, ids.clamp(min=0)), -1)
    q = torch.randn(B, Tq, c["heads_q"], c["head_dim"], device=DEV, generator=gen, dtype=DTYPES[c["dtype"]])
    return dict(s, q=q, ids=ids.to(torch.int32).contiguous(), lens=lens.to(torch.int32).contiguous(),
                scale=c["head_dim"] ** -0.5)


INPUTS = {"rotate": _rotate_inputs, "append": _append_inputs, "values": _values_inputs, "read": _read_inputs}


def prepare(case, seed):
    return dict(INPUTS[case["op"]](case, seed), op=case["op"])


# ------------------------------------------------------------------------------- one pass, as a user calls it


def _pipeline():
    path = str(pathlib.Path(__file__).resolve().parents[1] / "latent-sparse-attention-rocm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from lsa_rocm_lab.port import pipeline

    return pipeline


def _own_pass(s):
    p = _pipeline()
    if s["op"] == "rotate":
        return p.rotate(s["q"], s["k"], s["pos"], s["freq"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                        interleaved=s["interleaved"])
    cache = p.ByteCache(s["k8"], s["v8"], s["scales"], s["block"])
    if s["op"] == "append":
        q = p.byte_append(cache, s["k"], s["v"], s["starts"], lengths=s["lens"], slot_table=s["table"], q=s["q"],
                          frequencies=s["freq"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS,
                          interleaved=s["interleaved"])
        return (q, *p.byte_values(cache, s["ids"], s["nids"], dtype=s["k"].dtype if s["k"].dtype.itemsize == 2 else
                                  torch.bfloat16), s["scales"])
    if s["op"] == "values":
        return p.byte_values(cache, s["ids"], s["nids"], dtype=s["dtype"])
    return p.byte_read(s["q"], cache, s["ids"], s["lens"], scale=s["scale"])


# ------------------------------------------------------------------------------- the plain forms


def _turned(x, pos, freq, weight, interleaved):
    """The rows of x [B, T, H, D] normed and rotated by pos [B, T], in 32 bits; the angles in 64."""
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()
    angle = pos.double()[:, :, None, None] * freq.double()
    cos, sin = angle.cos().float(), angle.sin().float()
    n = freq.numel()
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    pair = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat([torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1), y[..., 2 * n:]], -1)


def _plain_rotate(s):
    return tuple(_turned(s[x], s["pos"], s["freq"], s[w], s["interleaved"]).to(s[x].dtype) for x, w in
                 (("q", "wq"), ("k", "wk")))


def _bytes(x):
    """8-bit floats are moved as bytes."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _fetch(x, at):
    """Rows at [B, n] (clamped) of x [B or 1, T, ...]."""
    b = torch.arange(at.shape[0], device=x.device)[:, None] if x.shape[0] == at.shape[0] else 0
    return _bytes(x)[b, at.clamp(0, x.shape[1] - 1)].view(x.dtype)


def _numbers(s, at, n):
    """The values that rows at [B, m] of the cache stand for, zeros from n [B] on: K's, V's in 32 bits."""
    here = (torch.arange(at.shape[1], device=DEV) < n[:, None])[..., None, None]
    sc = _fetch(s["scales"], at.long() // s["block"])
    return tuple((_fetch(s[x], at.long()).float() * sc[..., i, None]).masked_fill(~here, 0.0) for i, x in
                 enumerate(("k8", "v8")))


def _plain_values(s):
    at, n = s["ids"], s["nids"]
    if at is None:
        B, T = s["k8"].shape[:2]
        at = torch.arange(T, device=DEV).expand(B, T)
        n = torch.full((B,), T, device=DEV)
    return tuple(x.to(s["dtype"]) for x in _numbers(s, at, n))


def _plain_append(s):
    k, v, starts, block, most = s["k"], s["v"], s["starts"].long(), s["block"], CODES[s["code"]][1]
    B, n, Hkv, D = k.shape
    lens = torch.full((B,), n, device=DEV) if s["lens"] is None else s["lens"].long()
    live = torch.arange(n, device=DEV) < lens[:, None]
    pos = starts[:, None] + torch.arange(n, device=DEV)
    q = _turned(s["q"], pos, s["freq"], s["wq"], s["interleaved"]).masked_fill(~live[..., None, None], 0.0).to(k.dtype)
    # whole blocks of every row, from the one that its first token falls in
    m = (n + 2 * block - 2) // block * block
    at = (starts // block * block)[:, None] + torch.arange(m, device=DEV)  # positions
    new = (at >= starts[:, None]) & (at < (starts + lens)[:, None])
    old = (at < starts[:, None]) & new.view(B, -1, block).any(-1).repeat_interleave(block, 1)
    T = s["table"].shape[1] if s["table"] is not None else s["k8"].shape[1]
    row = s["table"].long().gather(1, at.clamp(max=T - 1)) if s["table"] is not None else at.clamp(max=T - 1)
    from_ = (at - starts[:, None]).clamp(0, n - 1)
    b = torch.arange(B, device=DEV)[:, None]
    cache_row = (b if s["k8"].shape[0] == B else torch.zeros_like(b)).expand(B, m)
    lead = row.view(B, -1, block)[:, :, 0] // block  # every block's place in the scales
    touched = new.view(B, -1, block).any(-1)
    old_scale = _fetch(s["scales"], lead)  # [B, blocks, Hkv, 2]
    had = old.view(B, -1, block).any(-1)[..., None]
    for_k = _turned(k, pos, s["freq"], s["wk"], s["interleaved"])
    for i, (x, c8) in enumerate(((for_k, s["k8"]), (v.float(), s["v8"]))):
        x = x[b, from_].masked_fill(~new[..., None, None], 0.0)  # [B, m, Hkv, D]
        grown = x.view(B, -1, block, Hkv, D).abs().amax((2, 4)) / most
        was = old_scale[..., i]
        scale = torch.maximum(grown.clamp(min=LEAST), torch.where(had, was, 0.0))
        each = scale.repeat_interleave(block, 1)[..., None]
        kept = _fetch(c8, row).float() * (was / scale).repeat_interleave(block, 1)[..., None]
        codes = _coded(torch.where(new[..., None, None], x / each, kept), s["code"])
        out = new | old
        c8.view(torch.uint8)[cache_row[out], row[out]] = codes.view(torch.uint8)[out]
        s["scales"][cache_row[:, ::block][touched], lead[touched], :, i] = scale[touched]
    to = k.dtype if k.dtype.itemsize == 2 else torch.bfloat16
    return (q, *(x.to(to) for x in _numbers(s, s["ids"], s["nids"])), s["scales"])


def _plain_read(s):
    q, ids = s["q"], s["ids"]
    B, Tq, Hq, D = q.shape
    T, Hkv = s["k8"].shape[1:3]
    W = ids.shape[-1]
    ids = ids if ids.dim() == 4 else ids[:, :, None].expand(B, Tq, Hkv, W)
    lens = s["lens"].view(B, Tq, -1, 1)
    ok = (ids >= 0) & (torch.arange(W, device=DEV) < lens)
    at = ids.long().clamp(0, T - 1)
    b = torch.arange(B, device=DEV).view(B, 1, 1, 1) if s["k8"].shape[0] == B else 0
    h = torch.arange(Hkv, device=DEV).view(1, 1, Hkv, 1)
    sc = s["scales"][b, at // s["block"], h]  # [B, Tq, Hkv, W, 2]

    def rows(c8, i):
        return _bytes(c8)[b, at, h].view(c8.dtype).float() * sc[..., i, None]

    qf = q.float().view(B, Tq, Hkv, Hq // Hkv, D) * s["scale"]
    w = torch.matmul(qf, rows(s["k8"], 0).transpose(-1, -2).contiguous()).masked_fill(~ok[:, :, :, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    return (torch.matmul(w, rows(s["v8"], 1)) / w.sum(-1, keepdim=True)).reshape(B, Tq, Hq, D).to(q.dtype)


PLAIN = {"rotate": _plain_rotate, "append": _plain_append, "values": _plain_values, "read": _plain_read}


def run(s):
    if own:
        return _own_pass(s)
    return PLAIN[s["op"]](s)


# ------------------------------------------------------------------------------- what a pass needs


def work(case):
    c = case
    e = 4 if c["dtype"] == "fp32" else 2
    held = c["heads_kv"] * c["head_dim"]
    if c["op"] == "values":
        rows = c["batch"] * (0.75 * c["rows"] or c["cache"])
        written = c["batch"] * (c["rows"] or c["cache"])
        return {"bytes": 2 * held * (rows + e * written) + 8 * c["heads_kv"] * rows / c["block"], "flops": 0}
    wide = c["heads_q"] * c["head_dim"]
    rows = c["batch"] * c["tokens"]
    if c["op"] == "rotate":
        return {"bytes": rows * (2 * e * (wide + held) + 4), "flops": 10.0 * rows * (wide + held)}
    if c["op"] == "append":  # q read and written, k and v read, their codes written, read again and written as numbers
        live = rows * (0.5 if c["ragged"] else 1.0)
        seen = c["batch"] * min(c["tokens"] + c["block"], c["cache"])
        back = live + c["batch"] * (c["block"] - 1) / 2
        return {"bytes": live * (e * wide + 2 * held * (e + 1)) + e * rows * wide + 2 * held * (back + 2 * seen),
                "flops": 10.0 * live * (wide + held)}
    keys = 0.75 * c["cache"] if c["lists"] == "whole" else 64 * c["spans"]
    read = c["batch"] * (keys if c["lists"] == "whole" else
                         c["cache"] * (1.0 - (1.0 - min(1.0, keys / c["cache"])) ** c["tokens"]))
    lists = 4 * rows * keys * (c["heads_kv"] if c["lists"] == "heads" else 1)
    return {"bytes": read * 2 * held + 8 * c["heads_kv"] * read / c["block"] + lists + 2 * e * rows * wide,
            "flops": 4.0 * rows * wide * keys}


# ------------------------------------------------------------------------------- 64 bits


def _spin(x, pos, freq, weight, interleaved):
    """Rows x [n, H, D] at positions pos [n], as complex numbers turned by their angle."""
    y = x.double()
    if weight is not None:
        y = weight.double() * y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS)
    n = freq.numel()
    even, odd = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(y[..., even], y[..., odd])
    z = z * torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[:, None, None] * freq.double())
    out = y.clone()
    out[..., even], out[..., odd] = z.real, z.imag
    return out


def _exact_rotate(s):
    return tuple(torch.stack([_spin(s[x][b], s["pos"][b], s["freq"], s[w], s["interleaved"]) for b in
                              range(s[x].shape[0])]) for x, w in (("q", "wq"), ("k", "wk")))


def _nearest(x, code):
    """The nearest number that a code holds, ties to even, saturating."""
    if code == "int8":
        return torch.round(x).clamp(-127, 127)
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())  # 3 bits behind the leading one, down to 2^-9
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_values(s, rows=None):
    """By row: codes times their block's scale."""
    k8, ids = s["k8"], s["ids"]
    B = s["scales"].shape[0] if ids is None else ids.shape[0]
    T = k8.shape[1]
    found = []
    for i, x in enumerate(("k8", "v8")):
        out = []
        for b in range(B):
            at = torch.arange(T, device=DEV) if ids is None else ids[b].long()
            live = T if ids is None else int(s["nids"][b])
            c = b if k8.shape[0] == B else 0
            at = at[:live]
            y = torch.zeros(T if ids is None else ids.shape[1], *k8.shape[2:], dtype=torch.float64, device=DEV)
            y[:live] = _bytes(s[x])[c][at].view(s[x].dtype).double() * s["scales"][c, at // s["block"], :, i, None].double()
            out.append(y)
        found.append(torch.stack(out))
    return tuple(found)


def _exact_append(s):
    B, n, Hkv, D = s["k"].shape
    block, most = s["block"], CODES[s["code"]][1]
    lens = [n] * B if s["lens"] is None else s["lens"].tolist()
    k8, v8, scales = s["k8"].double(), s["v8"].double(), s["scales"].double()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, first in enumerate(s["starts"].tolist()):
        m = lens[b]
        pos = first + torch.arange(m, device=DEV)
        c = b if k8.shape[0] == B else 0
        if m:
            q[b, :m] = _spin(s["q"][b, :m], pos, s["freq"], s["wq"], s["interleaved"])
            k = _spin(s["k"][b, :m], pos, s["freq"], s["wk"], s["interleaved"])
        at = first
        while at < first + m:  # the tokens of one block after another
            last = min(at // block * block + block, first + m)
            lead = at // block * block
            where = s["table"][b, lead:last].long() if s["table"] is not None else torch.arange(lead, last, device=DEV)
            place = int(where[0]) // block
            for i, (x, c8) in enumerate(((k, k8), (s["v"][b].double(), v8))):
                x = x[at - first:last - first]
                was = scales[c, place, :, i] if at > lead else torch.zeros(Hkv, dtype=torch.float64, device=DEV)
                scale = torch.maximum(torch.maximum(x.abs().amax((0, 2)) / most, was), torch.tensor(LEAST, device=DEV))
                if at > lead:
                    before = where[: at - lead]
                    c8[c, before] = _nearest(c8[c, before] * (was / scale)[:, None], s["code"])
                c8[c, where[at - lead:]] = _nearest(x / scale[:, None], s["code"])
                scales[c, place, :, i] = scale
            at = last
    return (q, *_exact_values(dict(s, k8=k8, v8=v8, scales=scales)), scales)


def _exact_read(s):
    B, Tq, Hq, D = s["q"].shape
    Hkv = s["k8"].shape[2]
    G = Hq // Hkv
    out = torch.zeros(B, Tq, Hq, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        c = b if s["k8"].shape[0] == B else 0
        for t in range(Tq):
            for g in range(Hkv):
                per = s["ids"].dim() == 4
                n = int(s["lens"][b, t, g] if per else s["lens"][b, t])
                at = (s["ids"][b, t, g] if per else s["ids"][b, t])[:n].long()
                at = at[at >= 0]
                sc = s["scales"][c, at // s["block"], g].double()
                k, v = (_bytes(s[x])[c, at, g].view(s[x].dtype).double() * sc[:, i, None] for i, x in
                        enumerate(("k8", "v8")))
                w = torch.softmax(s["scale"] * (s["q"][b, t, g * G:(g + 1) * G].double() @ k.T), 1)
                out[b, t, g * G:(g + 1) * G] = w @ v
    return out


EXACT = {"rotate": _exact_rotate, "append": _exact_append, "values": _exact_values, "read": _exact_read}


def exact(case, seed):
    s = prepare(case, seed)
    return EXACT[case["op"]](s)
