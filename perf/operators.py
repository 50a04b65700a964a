"""Cases of the 4-bit paged KV cache and of the page-table operators.

Five operators, each in a plain torch form (``own`` false) and through this
package (``own`` true):

* ``store``   rows of K and V into 4-bit pages and the values they then hold;
* ``decode``  attention of one query row per sequence over its 4-bit pages;
* ``chunk``   causal attention of ragged chunks of rows over their 4-bit pages;
* ``fork``    forked sequences dropped and forked again (pages shared and copied);
* ``compact`` sequences dropped, the live pages moved to the front of every pool.

Page layout (uint8), per page and KV head, hd the head dim, 16 tokens:
K nibbles (8 hd bytes), V nibbles (8 hd), K scales (hd), V scales (hd).
A scale is 16 bits per token and block of 32 dims: the bits 0x7ff0 are an fp16
step d, the low 4 bits the zero point z, and a value is d * (q - z).
K: token r's row of hd/2 bytes is 4 chunks t of one 32-bit word per block b;
nibble e of the word is dim 32 b + 8 t + e.  V: words ordered [group][g 8][t 4]
[tile], tile = 16 dims; byte 2 u + w of a word is token 2 t + u + 8 w, its low
nibble dim 16 tile + g, its high nibble dim 16 tile + g + 8.
"""
import math

import torch

own = False

PAGE = 16          # tokens per page
BLOCK = 32         # dims per scale
LIMIT = 32768.0    # values are clamped to it, so that every stored value is an fp16 number

# Llama-3-8B head layout (32 query, 8 KV heads of 128) and TinyLlama's (32, 4, 64)
# are the ones of this repository's benchmark and tests.


def listed():
    return [
        # the K/V of one decode step of 64 sequences
        {"name": "store_step_b64", "op": "store", "seqs": 64, "rows": 1, "start": 2047, "ragged": True, "kv": 8, "hd": 128},
        # one prefill chunk of 4096 rows, three prompts that begin inside a page
        {"name": "store_chunk_4096", "op": "store", "seqs": 3, "rows": 1365, "start": 21, "ragged": False, "kv": 8, "hd": 128},
        # a single user's decode step
        {"name": "decode_b1_257", "op": "decode", "seqs": 1, "ctx": 257, "ragged": False, "heads": 32, "kv": 4, "hd": 64},
        # the benchmark's decode step: 64 sequences of 2176 tokens
        {"name": "decode_b64_2176", "op": "decode", "seqs": 64, "ctx": 2176, "ragged": False, "heads": 32, "kv": 8, "hd": 128},
        # one long document
        {"name": "decode_b1_131072", "op": "decode", "seqs": 1, "ctx": 131072, "ragged": False, "heads": 32, "kv": 8, "hd": 128},
        # a batch of very different lengths, groups of 7 heads
        {"name": "decode_b37_ragged", "op": "decode", "seqs": 37, "ctx": 8191, "ragged": True, "heads": 14, "kv": 2, "hd": 64},
        # a few draft tokens of each sequence checked at once
        {"name": "chunk_draft_b24", "op": "chunk", "seqs": 24, "rows": 5, "past": 1499, "ragged": True, "heads": 32, "kv": 8, "hd": 128},
        # prompts from their start
        {"name": "chunk_prompt_4x2048", "op": "chunk", "seqs": 4, "rows": 2048, "past": 0, "ragged": False, "heads": 32, "kv": 8, "hd": 128},
        # two prompts, each sampled four times
        {"name": "fork_2x4", "op": "fork", "parents": 2, "each": 4, "tokens": 77, "ragged": True, "pools": 4, "kv": 4, "hd": 64},
        # 16 prompts, each sampled four times
        {"name": "fork_16x4", "op": "fork", "parents": 16, "each": 4, "tokens": 2040, "ragged": True, "pools": 16, "kv": 8, "hd": 128},
        # a small cache after two of nine sequences ended
        {"name": "compact_9", "op": "compact", "seqs": 9, "tokens": 190, "ragged": True, "drop": 4, "pools": 4, "kv": 4, "hd": 64},
        # a full cache after every third of 64 sequences ended
        {"name": "compact_64", "op": "compact", "seqs": 64, "tokens": 2080, "ragged": False, "drop": 3, "pools": 8, "kv": 8, "hd": 128},
    ]


def _between(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "chunk", "chunk", "fork", "compact"])
    kv = rng.choice([1, 2, 3, 4, 8])
    hd = rng.choice([32, 64, 128, 128])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    c = {"op": op, "ragged": rng.random() < 0.6, "kv": kv, "hd": hd}
    if op == "store":
        c["seqs"] = _between(rng, 1, 64)
        c["rows"] = _between(rng, 1, 4096 // c["seqs"])
        c["start"] = _between(rng, 1, 2048) - 1
    elif op == "decode":
        c["heads"] = kv * group
        c["seqs"] = _between(rng, 1, 64)
        c["ctx"] = _between(rng, 1, 131072 // c["seqs"])
    elif op == "chunk":
        c["heads"] = kv * group
        c["seqs"] = _between(rng, 1, 24)
        most = min(4096 // c["seqs"], math.isqrt((1 << 28) // (c["seqs"] * c["heads"])))
        c["rows"] = _between(rng, 1, max(2, most))
        # the plain form holds every score, seen or not: keep them to 2^28
        room = (1 << 28) // (c["seqs"] * c["heads"] * c["rows"])
        c["past"] = max(0, min(_between(rng, 1, 16384) - 1, room - c["rows"]))
    elif op == "fork":
        c["hd"] = rng.choice([64, 128])
        c["parents"] = _between(rng, 1, 16)
        c["each"] = _between(rng, 1, 8)
        c["tokens"] = _between(rng, 1, 2048)
        c["pools"] = 2 * rng.randint(1, 8)
    else:
        c["hd"] = rng.choice([64, 128])
        c["seqs"] = _between(rng, 2, 64)
        c["tokens"] = _between(rng, 16, 2080)
        c["drop"] = rng.randint(2, 5)
        c["pools"] = 2 * rng.randint(1, 4)
    return c


def _lens(n, most, ragged, least=1):
    """n lengths up to `most`: all alike, or spread over least..most (the first is the longest)."""
    if not ragged:
        return [most] * n
    return [most - (i * 2654435761 >> 7) % (most - least + 1) if i else most for i in range(n)]


def _blocks(tokens):
    return (tokens + PAGE - 1) // PAGE


# ---- the 4-bit format in elementary torch operations --------------------------------

def _steps(device):
    """Every step d by its code: fp16 with the low 4 mantissa bits clear."""
    return (torch.arange(0x7C0, dtype=torch.int16, device=device) << 4).view(torch.float16).float()


def _quantize(x):
    """x [..., 32 m] fp32 -> (q, code, z): whole numbers, q like x, code and z per block."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    b = torch.where(b.isnan(), torch.zeros_like(b), b).clamp(-LIMIT, LIMIT)
    lo, hi = b.amin(-1).clamp(max=0), b.amax(-1).clamp(min=0)
    steps = _steps(x.device)
    code = torch.searchsorted(15 * steps, (hi - lo).contiguous())
    d = steps[code].double()
    d = torch.where(d == 0, torch.ones_like(d), d)      # an all-zero block: every q - z is 0
    z = -torch.floor(lo.double() / d + 0.5)
    q = (torch.floor(b.double() / d[..., None] + 0.5) + z[..., None]).clamp(0, 15)
    return q.to(torch.int64).reshape(x.shape), code, z.to(torch.int64)


def _value(q, code, z):
    b = q.reshape(*q.shape[:-1], -1, BLOCK)
    return (_steps(q.device)[code][..., None] * (b - z[..., None]).float()).reshape(q.shape)


def _scale_bytes(code, z):
    """[..., 16, nb] -> [..., 16 * nb * 2] bytes."""
    w = ((code << 4) | z).to(torch.int16).contiguous()
    return w.view(torch.uint8).reshape(*w.shape[:-2], -1)


def _pack(k, v):
    """k, v [pages, kv, 16, hd] fp32 -> page bytes [pages, kv, 18 hd]."""
    P, H, _, hd = k.shape
    nb, tiles = hd // 32, hd // 16
    per = min(4, tiles)
    kq, kc, kz = _quantize(k)
    vq, vc, vz = _quantize(v)
    a = kq.reshape(P, H, 16, nb, 4, 4, 2).permute(0, 1, 2, 4, 3, 5, 6)        # [.. r, t, b, byte, nibble]
    kb = (a[..., 0] | (a[..., 1] << 4)).to(torch.uint8).reshape(P, H, -1)
    # tokens 2 t + u + 8 w, dims 16 (group per + tile) + 8 n + g
    a = vq.reshape(P, H, 2, 4, 2, tiles // per, per, 2, 8).permute(0, 1, 5, 8, 3, 6, 4, 2, 7)
    vb = (a[..., 0] | (a[..., 1] << 4)).to(torch.uint8).reshape(P, H, -1)
    return torch.cat([kb, vb, _scale_bytes(kc, kz), _scale_bytes(vc, vz)], -1)


def _unpack(pages, hd):
    """page bytes [..., 18 hd] -> k, v [..., 16, hd] fp32."""
    lead = pages.shape[:-1]
    nb, tiles = hd // 32, hd // 16
    per = min(4, tiles)
    kb, vb, ks, vs = pages.split([8 * hd, 8 * hd, hd, hd], -1)

    def steps(s):
        w = s.contiguous().view(torch.int16).reshape(*lead, 16, nb, 1)
        return (w & 0x7FF0).view(torch.float16).float(), (w & 15).float()

    n = len(lead)
    a = torch.stack([kb & 15, kb >> 4], -1).reshape(*lead, 16, 4, nb, 8)     # [r, t, b, e]
    k = a.permute(*range(n), n, n + 2, n + 1, n + 3).reshape(*lead, 16, nb, 32).float()
    a = torch.stack([vb & 15, vb >> 4], -1).reshape(*lead, tiles // per, 8, 4, per, 2, 2, 2)
    # [group, g, t, tile, u, w, n] -> [w, t, u, group, tile, n, g]
    v = a.permute(*range(n), n + 5, n + 2, n + 4, n, n + 3, n + 6, n + 1).reshape(*lead, 16, nb, 32).float()
    (kd, kz), (vd, vz) = steps(ks), steps(vs)
    return (kd * (k - kz)).reshape(*lead, 16, hd), (vd * (v - vz)).reshape(*lead, 16, hd)


# ---- inputs ------------------------------------------------------------------------

def _gen(seed, part):
    g = torch.Generator(device="cuda")
    return g.manual_seed(seed * 1000003 + part)


def _rows(seed, part, n, kv, hd):
    """K and V rows [n, kv, hd]: normal values, a few K channels four times as large."""
    g = _gen(seed, part)
    k = torch.randn(n, kv, hd, device="cuda", generator=g)
    v = torch.randn(n, kv, hd, device="cuda", generator=g)
    k[:, :, ::29] *= 4
    return k, v


def _table(seed, n_seqs, blocks, max_blocks):
    """A block table whose sequences hold blocks[i] pages of a shuffled pool, and the pool's size."""
    need = sum(blocks)
    order = torch.randperm(need, device="cuda", generator=_gen(seed, 7)).to(torch.int32)
    table = torch.full((n_seqs, max_blocks), -1, dtype=torch.int32, device="cuda")
    j = torch.arange(max_blocks, device="cuda")
    held = torch.tensor(blocks + [0] * (n_seqs - len(blocks)), device="cuda")
    table[j[None] < held[:, None]] = order
    return table, need


def _cache(seed, lens, kv, hd):
    """A filled 4-bit cache: pages, table and the fp32 rows it was filled from.  Slots past a
    sequence's end hold whatever was in memory."""
    blocks = [_blocks(n) for n in lens]
    table, n_pages = _table(seed, len(lens), blocks, max(blocks))
    pages = torch.randint(0, 256, (n_pages, kv, 18 * hd), dtype=torch.uint8, device="cuda", generator=_gen(seed, 8))
    for s, n in enumerate(lens):
        k, v = _rows(seed, 100 + s, blocks[s] * PAGE, kv, hd)
        at = table[s, :blocks[s]].long()
        for a in range(0, blocks[s], 512):       # in pieces: packing takes 64-bit temporaries
            b = min(blocks[s], a + 512)
            kk, vv = (x[a * PAGE:b * PAGE].reshape(b - a, PAGE, kv, hd).transpose(1, 2) for x in (k, v))
            new = _pack(kk, vv)
            if b == blocks[s] and n % PAGE:      # keep the unused slots' bytes of the last page
                full = pages[at[b - 1]]
                uk, uv = full.clone(), new[-1].clone()
                new[-1] = _merge(uk, uv, n % PAGE, hd)
            pages[at[a:b]] = new
    return pages, table, n_pages


def _merge(old, new, used, hd):
    """Page bytes with the first `used` tokens of `new`, the rest of `old` ([kv, 18 hd])."""
    tiles = hd // 16
    per = min(4, tiles)
    tok = torch.arange(PAGE, device=old.device)
    krow = (tok < used).repeat_interleave(hd // 2)
    t, u, w = (torch.arange(4, device=old.device), torch.arange(2, device=old.device), torch.arange(2, device=old.device))
    token = 2 * t[:, None, None, None] + u[None, None, :, None] + 8 * w[None, None, None, :]   # [t, tile, u, w]
    vword = (token < used).expand(4, per, 2, 2).reshape(1, 1, -1).expand(tiles // per, 8, -1).reshape(-1)
    srow = (tok < used).repeat_interleave(hd // 16)
    return torch.where(torch.cat([krow, vword, srow, srow]), new, old)


def prepare(case, seed):
    c = dict(case)
    op = c["op"]
    s = {"case": c}
    if op == "store":
        kv, hd = c["kv"], c["hd"]
        rows = _lens(c["seqs"], c["rows"], c["ragged"])
        first = _lens(c["seqs"], c["start"], c["ragged"], 0)
        blocks = [_blocks(a + n) for a, n in zip(first, rows)]
        s["table"], n_pages = _table(seed, c["seqs"], blocks, max(blocks))
        s["pages"] = torch.zeros(n_pages, kv, 18 * hd, dtype=torch.uint8, device="cuda")
        k, v = _rows(seed, 1, sum(rows), kv, hd)
        s["k"], s["v"] = k.reshape(-1, kv * hd), v.reshape(-1, kv * hd)
        s["row_seq"] = torch.tensor([i for i, n in enumerate(rows) for _ in range(n)], dtype=torch.int32, device="cuda")
        s["row_pos"] = torch.tensor([a + j for a, n in zip(first, rows) for j in range(n)], dtype=torch.int32, device="cuda")
    elif op == "decode":
        lens = _lens(c["seqs"], c["ctx"], c["ragged"])
        s["pages"], s["table"], _ = _cache(seed, lens, c["kv"], c["hd"])
        s["q"] = torch.randn(c["seqs"], c["heads"] * c["hd"], device="cuda", generator=_gen(seed, 2))
        s["q_pos"] = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    elif op == "chunk":
        rows = _lens(c["seqs"], c["rows"], c["ragged"])
        past = _lens(c["seqs"], c["past"], c["ragged"], 0)
        s["pages"], s["table"], _ = _cache(seed, [a + n for a, n in zip(past, rows)], c["kv"], c["hd"])
        start = [sum(rows[:i]) for i in range(len(rows) + 1)]
        s["q"] = torch.randn(start[-1], c["heads"] * c["hd"], device="cuda", generator=_gen(seed, 2))
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
        s["q_pos"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        s["max_rows"] = max(rows)
    elif op == "fork":
        lens = _lens(c["parents"], c["tokens"], c["ragged"])
        kids = c["parents"] * c["each"]
        blocks = [_blocks(n) for n in lens]
        table, need = _table(seed, c["parents"] + kids, blocks, max(blocks))
        s["parents"] = torch.arange(c["parents"], dtype=torch.int32, device="cuda").repeat_interleave(c["each"])
        s["children"] = torch.arange(c["parents"], c["parents"] + kids, dtype=torch.int32, device="cuda")
        s["tokens"] = torch.tensor(lens, dtype=torch.int32, device="cuda").repeat_interleave(c["each"])
        n_pages = need + kids
        ref = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        ref[:need] = 1
        s["pools"] = _pools(seed, c, n_pages)
        s["table"], s["ref"] = table, ref
        _fork(s)                                  # the children of the last round
    else:
        lens = _lens(c["seqs"], c["tokens"], c["ragged"])
        blocks = [_blocks(n) for n in lens]
        s["table"], n_pages = _table(seed, c["seqs"], blocks, max(blocks))
        s["ref"] = torch.ones(n_pages, dtype=torch.int32, device="cuda")
        s["pools"] = _pools(seed, c, n_pages)
        s["gone"] = torch.arange(0, c["seqs"], c["drop"], dtype=torch.int32, device="cuda")
        s["table_now"], s["ref_now"] = s["table"].clone(), s["ref"].clone()
    return s


def _pools(seed, c, n_pages):
    """fp16 K and V pages of pools / 2 layers, one tensor [pools, pages, kv, 16, hd]."""
    return torch.randn(c["pools"], n_pages, c["kv"], PAGE, c["hd"], dtype=torch.float16, device="cuda", generator=_gen(seed, 9))


# ---- plain forms -------------------------------------------------------------------

def _store(s):
    c = s["case"]
    k, v = (s[n].reshape(-1, c["kv"], c["hd"]) for n in ("k", "v"))
    return [_value(*_quantize(x)).reshape(-1, c["kv"] * c["hd"]) for x in (k, v)]


def _gather(s):
    """Every sequence's K and V [seqs, kv, tokens, hd]; unused slots are zero."""
    c = s["case"]
    table = s["table"]
    k, v = _unpack(s["pages"][table.clamp(min=0).long()], c["hd"])            # [S, blocks, kv, 16, hd]
    n = table.shape[1] * PAGE
    return [x.transpose(1, 2).reshape(table.shape[0], c["kv"], n, c["hd"]) for x in (k, v)]


def _attend(q, k, v, seen):
    """q [S, kv, rows, hd], seen [S, 1, rows or 1, tokens]: softmax(q k / sqrt(hd)) v in 32 bits."""
    used = seen.any(2).transpose(1, 2)[:, None]   # [S, 1, tokens, 1]: slots that some row sees
    k, v = torch.where(used, k, 0), torch.where(used, v, 0)
    score = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    score = torch.where(seen, score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    return (p @ v) / p.sum(-1, keepdim=True)


def _decode(s):
    c = s["case"]
    k, v = _gather(s)
    S, group = c["seqs"], c["heads"] // c["kv"]
    at = torch.arange(k.shape[2], device="cuda")
    seen = (at[None] <= s["q_pos"][:, None])[:, None, None]
    return _attend(s["q"].reshape(S, c["kv"], group, c["hd"]), k, v, seen).reshape(S, -1)


def _chunk(s):
    c = s["case"]
    k, v = _gather(s)
    S, group, T = c["seqs"], c["heads"] // c["kv"], s["max_rows"]
    start = s["q_start"].long()
    i = torch.arange(T, device="cuda")
    row = start[:-1, None] + i                                                # [S, T], padded
    live = row < start[1:, None]
    q = s["q"][row.clamp(max=s["q"].shape[0] - 1)].reshape(S, T, c["kv"], group, c["hd"])
    q = q.permute(0, 2, 3, 1, 4).reshape(S, c["kv"], group * T, c["hd"])
    at = torch.arange(k.shape[2], device="cuda")
    last = (start[1:] - start[:-1] - 1).clamp(min=0)
    seen = at[None, None] <= (s["q_pos"][:, None] + torch.minimum(i[None], last[:, None]))[..., None]   # [S, T, n]
    o = _attend(q, k, v, seen.repeat(1, group, 1)[:, None])
    o = o.reshape(S, c["kv"], group, T, c["hd"]).permute(0, 3, 1, 2, 4).reshape(S, T, -1)
    return o[live]


def _free(s, table, ref, seqs):
    gone = table[seqs.long()]
    ref.sub_(torch.bincount(gone[gone >= 0].long(), minlength=ref.numel()).to(torch.int32))
    table[seqs.long()] = -1


def _fork(s):
    table, ref = s["table"], s["ref"]
    full, part = s["tokens"] // PAGE, (s["tokens"] % PAGE) > 0
    parent, child = s["parents"].long(), s["children"].long()
    free = torch.nonzero(ref == 0).reshape(-1)
    kids = torch.nonzero(part).reshape(-1)
    new, old = free[:kids.numel()], table[parent[kids], full[kids].long()].long()
    j = torch.arange(table.shape[1], device="cuda")
    rows = torch.where(j[None] < full[:, None], table[parent], -1)
    rows[kids, full[kids].long()] = new.to(torch.int32)
    table[child] = rows
    ref.add_(torch.bincount(rows[rows >= 0].long(), minlength=ref.numel()).to(torch.int32))
    s["pools"][:, new] = s["pools"][:, old]


def _compact(s, table, ref):
    live = ref > 0
    n = live.sum()
    at = torch.arange(ref.numel(), device="cuda")
    src, dst = torch.nonzero(live & (at >= n)).reshape(-1), torch.nonzero(~live & (at < n)).reshape(-1)
    to = at.to(torch.int32)
    to[src] = dst.to(torch.int32)
    s["pools"][:, dst] = s["pools"][:, src]
    ref[dst] = ref[src]
    ref[src] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    return n.to(torch.int32).reshape(1)


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if op in ("store", "decode", "chunk"):
        if own:
            kv = _handle(s)
            if op == "store":
                kv.append_rows(s["k"], s["v"], s["row_seq"], s["row_pos"])
                return list(kv.read_rows(s["row_seq"], s["row_pos"]))
            if op == "decode":
                return kv.decode_attention(s["q"], c["heads"], s["q_pos"])
            return kv.chunk_attention(s["q"], c["heads"], s["q_start"], s["q_pos"], s["max_rows"])
        return {"store": _store, "decode": _decode, "chunk": _chunk}[op](s)
    if op == "fork":
        if own:
            pages = _page_handle(s, s["table"], s["ref"])
            pages.free(s["children"])
            pages.fork(s["parents"], s["children"], s["tokens"])
        else:
            _free(s, s["table"], s["ref"], s["children"])
            _fork(s)
        return {"table": s["table"], "ref": s["ref"], "pools": s["pools"]}
    # the sources of the moves stay as they were, so the same cache can be compacted again
    table, ref = s["table_now"].copy_(s["table"]), s["ref_now"].copy_(s["ref"])
    if own:
        pages = _page_handle(s, table, ref)
        pages.free(s["gone"])
        n = pages.compact()
    else:
        _free(s, table, ref, s["gone"])
        n = _compact(s, table, ref)
    return {"live": n, "table": table, "ref": ref, "pools": s["pools"]}


def _handle(s):
    """The cache object over the state's pages, kept as a program keeps it."""
    if "handle" not in s:
        from axion_b200.paged_kv import PagedKVCache4
        c = s["case"]
        s["handle"] = PagedKVCache4(c["kv"], c["hd"], pages=s["pages"], block_table=s["table"])
    return s["handle"]


def _page_handle(s, table, ref):
    if "handle" not in s:
        from axion_b200.kv_pages import KVPages
        s["handle"] = KVPages(list(s["pools"]), table, ref)
    return s["handle"]


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    c = case
    op = c["op"]
    if op == "store":
        n = sum(_lens(c["seqs"], c["rows"], c["ragged"])) * c["kv"] * c["hd"]
        return {"bytes": n * 2 * (4 + 0.5625 + 4), "flops": n * 2 * 6}
    if op == "decode":
        lens = _lens(c["seqs"], c["ctx"], c["ragged"])
        rows = c["seqs"] * c["heads"] * c["hd"]
        return {"bytes": sum(lens) * c["kv"] * c["hd"] * 1.125 + rows * 8, "flops": 4 * sum(lens) * c["heads"] * c["hd"]}
    if op == "chunk":
        rows, past = _lens(c["seqs"], c["rows"], c["ragged"]), _lens(c["seqs"], c["past"], c["ragged"], 0)
        pairs = sum(n * a + n * (n + 1) // 2 for n, a in zip(rows, past))
        held = sum(a + n for a, n in zip(past, rows))
        return {"bytes": held * c["kv"] * c["hd"] * 1.125 + sum(rows) * c["heads"] * c["hd"] * 8,
                "flops": 4 * pairs * c["heads"] * c["hd"]}
    page = c["pools"] * c["kv"] * PAGE * c["hd"] * 2
    if op == "fork":
        lens = _lens(c["parents"], c["tokens"], c["ragged"])
        copies = c["each"] * sum(n % PAGE > 0 for n in lens)
        entries = c["each"] * sum(_blocks(n) for n in lens)
        return {"bytes": 2 * copies * page + entries * 4 * 6, "flops": 0}
    lens = [_blocks(n) for n in _lens(c["seqs"], c["tokens"], c["ragged"])]
    total = sum(lens)
    live = total - sum(lens[::c["drop"]])
    moves = live * (total - live) / total        # live pages past the live count, in a shuffled pool
    return {"bytes": 2 * moves * page + total * 4 * 6, "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------

def _exact_value(x):
    """The value a 4-bit cache holds for x [n, kv, hd], in 64 bits from the format's definition."""
    b = x.double().clamp(-LIMIT, LIMIT).reshape(*x.shape[:-1], -1, BLOCK)
    low = torch.minimum(b.min(-1, keepdim=True).values, b.new_zeros(()))
    high = torch.maximum(b.max(-1, keepdim=True).values, b.new_zeros(()))
    need = (high.float() - low.float()).double() / 15          # the least step
    exponent = torch.floor(torch.log2(need.clamp(min=2.0 ** -30))).clamp(min=-14)
    grain = torch.exp2(exponent - 6)                            # 7 significant bits
    d = torch.ceil(need / grain) * grain
    d1 = torch.where(d > 0, d, torch.ones_like(d))
    below = -torch.floor(low / d1 + 0.5)
    q = torch.minimum(torch.floor(b / d1 + 0.5) + below, b.new_tensor(15.0))
    return (d * (q - below)).reshape(x.shape)


def exact(case, seed):
    c = case
    op = c["op"]
    if op == "store":
        n = sum(_lens(c["seqs"], c["rows"], c["ragged"]))
        return [_exact_value(x).reshape(n, -1) for x in _rows(seed, 1, n, c["kv"], c["hd"])]
    if op in ("fork", "compact"):
        return None                                             # whole numbers and copies
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    if op == "decode":
        rows, past = [1] * c["seqs"], [n - 1 for n in _lens(c["seqs"], c["ctx"], c["ragged"])]
    else:
        rows, past = _lens(c["seqs"], c["rows"], c["ragged"]), _lens(c["seqs"], c["past"], c["ragged"], 0)
    q = torch.randn(sum(rows), heads * hd, device="cuda", generator=_gen(seed, 2)).double()
    out = torch.empty_like(q)
    r0 = 0
    for s, (T, a) in enumerate(zip(rows, past)):
        n = a + T
        k, v = (_exact_value(x)[:n] for x in _rows(seed, 100 + s, _blocks(n) * PAGE, kv, hd))
        ahead = torch.arange(n, device="cuda")[None] > a + torch.arange(T, device="cuda")[:, None]
        for h in range(heads):
            g = h // (heads // kv)
            w = (q[r0:r0 + T, h * hd:(h + 1) * hd] @ k[:, g].T) / hd ** 0.5
            w.masked_fill_(ahead, -math.inf)
            out[r0:r0 + T, h * hd:(h + 1) * hd] = torch.softmax(w, -1) @ v[:, g]
        r0 += T
    return out
