"""More serving operators of the Transformer stack: the key/value cache in 4 bits, reading a cache back, and the attention of packed chunks.

Each case is one step of a user's program on device tensors:
  store    `serving.KVCache.append` and `.read`: new tokens' keys and values go into a 4-bit cache, rotated on the way, and what
           the cache then holds of them (or of the whole sequences) comes back as rows, as a chunk's attention takes it
  read     `serving.KVCache.read`: cached keys and values of a range of every sequence, as packed bf16 rows
  cache    `serving.KVCache.attend`: the newest token (or few) of every sequence over its 4-bit keys and values
  packed   `serving.packed_attention`: causal attention of packed sequences of different lengths, of whole prompts or of
           chunks behind the keys and values that the cache gave back

Four bits: 32 neighbouring elements of a head of one token share a step and a middle, both bf16, and code c of 0 ... 15 stands
for middle + (c - 8) * step: step is (most - least) / 15, the middle least + 8 steps, c - 8 the whole number next to
(value - middle) * (1 / step), that factor in bf16 too. A token's row of head_dim / 2 bytes holds, for g = 0 ... 7 and each group,
the codes of elements 4 g ... 4 g + 3 of the group, two to a byte, the first in the low half; its parameters are the groups'
steps, then their middles.
"""

import math

import torch

own = False

GROUP = 32  # elements that share a step and a middle
_LEAST_STEP = 2.0**-100  # steps below it count as zero


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # One new token in each of 64 conversations of 8192 tokens: a call of a few microseconds.
        dict(name="store_step", op="store", batch=64, new=1, past=8191, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, page_size=64, ragged=True, keep_k=False, back="new"),
        # A batch of ragged prompts entering the cache (16 heads of 64).
        dict(name="store_prompts", op="store", batch=16, new=2048, past=0, heads=16, kv_heads=16, head_dim=64, rotary_dim=64,
             interleaved=False, page_size=32, ragged=True, keep_k=True, back="new"),
        # Chunks of three long documents behind what the cache holds, all of which comes back; a quarter of each head rotated.
        dict(name="store_chunks", op="store", batch=3, new=2003, past=15001, heads=16, kv_heads=4, head_dim=128, rotary_dim=32,
             interleaved=True, page_size=16, ragged=True, keep_k=False, back="all"),
        # The cached part of 16 conversations in 8 bits, from an odd token on.
        dict(name="read_e4m3", op="read", kind="e4m3", batch=16, kv=4096, skip=77, kv_heads=16, head_dim=64, page_size=64,
             ragged=True),
        # Four long documents in 4 bits (1.1 GB of rows).
        dict(name="read_long", op="read", kind="int4", batch=4, kv=65536, skip=0, kv_heads=8, head_dim=128, page_size=128,
             ragged=False),
        # One sequence of about a thousand tokens, every head with its own keys: latency.
        dict(name="cache_one", op="cache", batch=1, kv=1001, q_len=1, heads=12, kv_heads=12, head_dim=64, page_size=16,
             window=0, sinks=0, ragged=False),
        # An ordinary serving batch: 64 sequences of up to 8192 tokens, four query heads to a key head.
        dict(name="cache_batch", op="cache", batch=64, kv=8192, q_len=1, heads=32, kv_heads=8, head_dim=128, page_size=64,
             window=0, sinks=0, ragged=True),
        # Long documents: 8 sequences of 131072 tokens (1.3 GB of 4-bit keys and values).
        dict(name="cache_long", op="cache", batch=8, kv=131072, q_len=1, heads=32, kv_heads=8, head_dim=128, page_size=128,
             window=0, sinks=0, ragged=False),
        # Streaming with a window and sinks, a token and one draft behind it, five query heads to a key head.
        dict(name="cache_streaming", op="cache", batch=32, kv=20011, q_len=2, heads=20, kv_heads=4, head_dim=128,
             page_size=32, window=4096, sinks=4, ragged=True),
        # Three short odd prompts: latency.
        dict(name="packed_short", op="packed", batch=3, new=41, past=0, heads=4, kv_heads=4, head_dim=64, window=0, sinks=0,
             ragged=True, slack=0),
        # Ragged prompts without their padding (16 heads of 64).
        dict(name="packed_prompts", op="packed", batch=24, new=2048, past=0, heads=16, kv_heads=16, head_dim=64, window=0,
             sinks=0, ragged=True, slack=0),
        # Chunks of four long documents behind what the cache gave back, four query heads of 128 to a key head.
        dict(name="packed_chunks", op="packed", batch=4, new=2048, past=14336, heads=16, kv_heads=4, head_dim=128, window=0,
             sinks=0, ragged=True, slack=0),
    ]


_ELEMENTS = 8 * 131072 * 8 * 128  # of cache_long's keys
_SCORES = 4 * 2048 * 16384 * 16  # of packed_chunks


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["store", "read", "cache", "cache", "packed", "packed"])
    head_dim = rng.choice([32, 64, 64, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    page = rng.choice([16, 32, 64, 128])
    if op == "store":
        head_dim = rng.choice([head_dim, 256])
        batch = _log(rng, 1, 128)
        width = kv_heads * (group + 2) * head_dim
        new = _log(rng, 1, max(1, min(8192, 2048 * 16 * 48 * 64 // (batch * width))))
        past = rng.choice([0, rng.randint(1, 5000)])
        back = "all" if past and batch * past * kv_heads * head_dim < 2**24 and rng.random() < 0.5 else "new"
        return dict(op=op, batch=batch, new=new, past=past, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice([0, 16 * rng.randint(1, head_dim // 16), head_dim]),
                    interleaved=rng.random() < 0.5, page_size=page, ragged=batch > 1 and rng.random() < 0.7,
                    keep_k=rng.random() < 0.5, back=back)
    if op == "read":
        batch = _log(rng, 1, 128)
        kv = _log(rng, 1, min(65536, 4 * 65536 * 8 * 128 // (batch * kv_heads * head_dim)))
        return dict(op=op, kind=rng.choice(["int4", "int4", "e4m3", "bf16"]), batch=batch, kv=kv,
                    skip=rng.choice([0, rng.randint(0, kv - 1)]), kv_heads=kv_heads, head_dim=head_dim, page_size=page,
                    ragged=batch > 1 and rng.random() < 0.7)
    window = rng.choice([0, 0, _log(rng, 1, 8192), _log(rng, 64, 8192)])
    sinks = rng.choice([0, 1, 4, rng.randint(1, 200)]) if window else 0
    if op == "cache":
        batch = _log(rng, 1, 256)
        q_len = rng.choice([1, 1, 1, 2, 4])
        return dict(op=op, batch=batch, kv=max(q_len, _log(rng, 1, min(131072, _ELEMENTS // (batch * kv_heads * head_dim)))),
                    q_len=q_len, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, page_size=page, window=window,
                    sinks=sinks, ragged=batch > 1 and rng.random() < 0.6)
    heads = kv_heads * group
    batch = _log(rng, 1, 64)
    new = _log(rng, 1, min(8192, math.isqrt(_SCORES // (heads * batch))))
    past = rng.choice([0, _log(rng, 1, max(1, min(32768, _SCORES // (heads * batch * new) - new)))])
    if (new + past) * new * heads * batch > _SCORES:
        past = 0
    return dict(op=op, batch=batch, new=new, past=past, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window,
                sinks=sinks, ragged=batch > 1 and rng.random() < 0.8, slack=rng.choice([0, 0, rng.randint(1, 200)]))


# --------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case, most, least=1):
    """Lengths of the case's sequences: all `most`, or ragged between a quarter of it and it (the first one is `most`)."""
    batch, low = case["batch"], max(least, most // 4)
    if not case["ragged"]:
        return [most] * batch
    return [most] + [low + (7919 * b + 104729 * b * b) % (max(low, most) - low + 1) for b in range(1, batch)]


def _starts(lengths):
    """First row of each of some packed sequences, and the row behind the last."""
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _activations(shape, head_dim, g):
    """Projection outputs: unit variance, with a few channels of each head several times larger, as trained keys have."""
    x = torch.randn(shape, device="cuda", generator=g)
    boost = torch.ones(head_dim, device="cuda")
    boost[:: max(1, head_dim // 4)] = 5.0
    return (x.view(-1, head_dim) * boost).view(shape).bfloat16()


def _table(positions, rotary_dim):
    """cos and sin of position * 10000^(-2i / rotary_dim), from 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cuda") / rotary_dim)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _pages(lengths, page, seed):
    """Page table [batch, most pages] with -1 where a sequence has no page, pages in random order; and their number."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + 3
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed + 1)).int()
    table = torch.full((len(lengths), max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return table.cuda(), total


def _cache(pages, kv_heads, page, head_dim, kind, g):
    """Full pages of keys or values (what was in a page before stays in its unused slots), with their scales."""
    shape = (pages, kv_heads, page, head_dim)
    if kind == "bf16":
        return _activations(shape, head_dim, g), None
    if kind == "int4":
        codes = torch.empty(*shape[:3], head_dim // 2, device="cuda", dtype=torch.uint8)
        params = torch.empty(*shape[:3], 2, head_dim // GROUP, device="cuda", dtype=torch.bfloat16)
        some = max(1, 2**27 // (kv_heads * page * head_dim))  # pages at a time, for the room that 32 bits take
        for i in range(0, pages, some):
            codes[i:i + some], params[i:i + some] = _quantise(_activations((min(some, pages - i), *shape[1:]), head_dim, g).float())
        return codes, params
    x = _activations(shape, head_dim, g)
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().float().amax((2, 3)) / 448.0)))
    return (x.float() / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = _generator(seed)
    hd, hk, state = case["head_dim"], case["kv_heads"], {"case": case}
    to = dict(device="cuda", dtype=torch.int32)
    rows = dict(device="cuda", dtype=torch.bfloat16)
    if case["op"] == "store":
        h, r = case["heads"], case["rotary_dim"]
        new, past = _lengths(case, case["new"]), _lengths(case, case["past"], 0)[::-1]
        table, pages = _pages([n + p for n, p in zip(new, past)], case["page_size"], seed)
        k, ks = _cache(pages, hk, case["page_size"], hd, "int4", g)
        v, vs = _cache(pages, hk, case["page_size"], hd, "int4", g)
        start = _starts(new)
        back = [n + p for n, p in zip(new, past)] if case["back"] == "all" else new
        first = [0] * case["batch"] if case["back"] == "all" else past
        at = _starts(back)
        return state | dict(
            qkv=_activations((start[-1], (h + 2 * hk) * hd), hd, g), new_start=torch.tensor(start[:-1], **to),
            new_len=torch.tensor(new, **to), past_len=torch.tensor(past, **to), page_table=table, max_new=max(new),
            k=k, v=v, k_scale=ks, v_scale=vs, table=_table(case["new"] + case["past"] + 1, r) if r else None,
            q_out=torch.empty(start[-1], h * hd, **rows) if r else None,
            k_out=torch.empty(start[-1], hk * hd, **rows) if r and case["keep_k"] else None,
            out_start=torch.tensor(at[:-1], **to), length=torch.tensor(back, **to), start=torch.tensor(first, **to),
            max_len=max(back), k_rows=torch.empty(at[-1], hk * hd, **rows), v_rows=torch.empty(at[-1], hk * hd, **rows))
    if case["op"] == "read":
        lengths = _lengths(case, case["kv"])
        table, pages = _pages(lengths, case["page_size"], seed)
        k, ks = _cache(pages, hk, case["page_size"], hd, case["kind"], g)
        v, vs = _cache(pages, hk, case["page_size"], hd, case["kind"], g)
        first = [min(case["skip"], n) for n in lengths]
        take = [n - f for n, f in zip(lengths, first)]
        at = _starts(take)
        return state | dict(
            k=k, v=v, k_scale=ks, v_scale=vs, page_table=table, out_start=torch.tensor(at[:-1], **to),
            length=torch.tensor(take, **to), start=torch.tensor(first, **to), max_len=max(take),
            k_rows=torch.empty(at[-1], hk * hd, **rows), v_rows=torch.empty(at[-1], hk * hd, **rows))
    h = case["heads"]
    if case["op"] == "cache":
        lengths = _lengths(case, case["kv"], case["q_len"])
        table, pages = _pages(lengths, case["page_size"], seed)
        k, ks = _cache(pages, hk, case["page_size"], hd, "int4", g)
        v, vs = _cache(pages, hk, case["page_size"], hd, "int4", g)
        q = torch.randn(case["batch"] * case["q_len"], h * hd, device="cuda", generator=g).bfloat16()
        return state | dict(q=q, page_table=table, kv_len=torch.tensor(lengths, **to), k=k, v=v, k_scale=ks, v_scale=vs,
                            scale=hd**-0.5, out=torch.empty_like(q))
    new, past = _lengths(case, case["new"]), _lengths(case, case["past"], 0)[::-1]
    q_at, kv_at = _starts(new), _starts([n + p for n, p in zip(new, past)])
    total = q_at[-1] + case["slack"]
    out = torch.zeros(total, h * hd, **rows)
    q_start = torch.tensor(q_at, **to)
    if not case["past"]:  # whole prompts: columns of one projection
        qkv = torch.randn(total, (h + 2 * hk) * hd, device="cuda", generator=g).bfloat16()
        q, k, v = qkv.split([h * hd, hk * hd, hk * hd], 1)
        return state | dict(q=q, k=k, v=v, q_start=q_start, kv_start=None, scale=hd**-0.5, out=out)
    q = torch.randn(total, h * hd, device="cuda", generator=g).bfloat16()
    k, v = (torch.randn(kv_at[-1] + case["slack"], hk * hd, device="cuda", generator=g).bfloat16() for _ in range(2))
    return state | dict(q=q, k=k, v=v, q_start=q_start, kv_start=torch.tensor(kv_at, **to), scale=hd**-0.5, out=out)


# --------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return {"store": _own_store, "read": _own_read, "cache": _own_cache, "packed": _own_packed}[case["op"]](state)
    return {"store": _store, "read": _read, "cache": _attend, "packed": _packed}[case["op"]](state)


def _kv_cache(state):
    """The cache object that a user's program keeps around its pages."""
    if "cache" not in state:
        from tiktoktechjam2026track3_b200 import serving

        state["cache"] = serving.KVCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state["cache"]


def _own_store(s):
    c, cache = s["case"], _kv_cache(s)
    cache.append(s["qkv"], c["heads"], s["new_start"], s["new_len"], s["past_len"], s["page_table"], s["max_new"],
                 table=s["table"], interleaved=c["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
    cache.read(s["out_start"], s["length"], s["start"], s["page_table"], s["max_len"], k_out=s["k_rows"], v_out=s["v_rows"])
    return _stored(s)


def _stored(s):
    got = dict(k=s["k_rows"], v=s["v_rows"])
    for name in ("q_out", "k_out"):
        if s[name] is not None:
            got[name] = s[name]
    return got


def _own_read(s):
    _kv_cache(s).read(s["out_start"], s["length"], s["start"], s["page_table"], s["max_len"], k_out=s["k_rows"],
                      v_out=s["v_rows"])
    return dict(k=s["k_rows"], v=s["v_rows"])


def _own_cache(s):
    c = s["case"]
    return _kv_cache(s).attend(s["q"], s["page_table"], s["kv_len"], q_len=c["q_len"], scale=s["scale"],
                               window=c["window"], sinks=c["sinks"], out=s["out"])


def _own_packed(s):
    from tiktoktechjam2026track3_b200 import serving

    c = s["case"]
    return serving.packed_attention(s["q"], s["k"], s["v"], s["q_start"], s["kv_start"], c["head_dim"], window=c["window"],
                                    sinks=c["sinks"], scale=s["scale"], out=s["out"])


# --------------------------------------------------------------------------------------------- plain forms
def _quantise(x):
    """(codes, parameters) of values [..., head_dim] in 32 bits: every operation rounded by itself, as the codes at a border need."""
    hd = x.shape[-1]
    y = x.unflatten(-1, (hd // GROUP, GROUP))
    lo, hi = y.aminmax(dim=-1)
    step = ((hi - lo) / torch.full((), 15.0, device="cuda")).bfloat16().float()  # (by a number it would multiply by 1 / 15)
    step = torch.where(step < _LEAST_STEP, 0.0, step)
    mid = (lo + 8.0 * step).bfloat16().float()
    inverse = torch.where(step > 0, 1.0 / step, 0.0).bfloat16().float()
    code = (((y - mid[..., None]) * inverse[..., None]).clamp(-8.0, 7.0).round() + 8.0).to(torch.uint8)
    code = code.unflatten(-1, (8, 4)).transpose(-3, -2).flatten(-3)  # [..., g, group, 4]
    return code[..., 0::2] | code[..., 1::2] << 4, torch.stack([step, mid], -2).bfloat16()


def _values(codes, params):
    """Values [..., head_dim] in 32 bits."""
    groups = params.shape[-1]
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (8, groups, 4)).transpose(-3, -2).flatten(-2)
    p = params.float()
    return (p[..., 1, :, None] + (c.float() - 8.0) * p[..., 0, :, None]).flatten(-2)


def _rotate(x, c, s, rotary_dim, interleaved):
    """x [rows, heads, head_dim] in 32 bits, c and s [rows, 1, rotary_dim / 2]."""
    half = rotary_dim // 2
    x1, x2 = (x[..., 0:rotary_dim:2], x[..., 1:rotary_dim:2]) if interleaved else (x[..., :half], x[..., half:rotary_dim])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., rotary_dim:]], -1)


def _owner(start, rows):
    """The sequence of each of some packed rows, and the row's number in it."""
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(start, at, right=True) - 1
    return b, at - start[b]


def _store(st):
    c, qkv = st["case"], st["qkv"]
    h, hk, hd, page, r = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"], c["rotary_dim"]
    b, i = _owner(st["new_start"], qkv.shape[0])
    pos = st["past_len"][b] + i
    x = qkv.float().view(-1, h + 2 * hk, hd)
    k, v = x[:, h:h + hk], x[:, h + hk:]
    if r:
        cs = st["table"][pos][:, None]
        qk = _rotate(x[:, :h + hk], cs[..., 0], cs[..., 1], r, c["interleaved"])
        st["q_out"].copy_(qk[:, :h].flatten(1))
        k = qk[:, h:]
        if st["k_out"] is not None:
            st["k_out"].copy_(k.flatten(1))
    pages, slot = st["page_table"][b, pos // page].long(), pos % page
    st["k"][pages, :, slot], st["k_scale"][pages, :, slot] = _quantise(k)
    st["v"][pages, :, slot], st["v_scale"][pages, :, slot] = _quantise(v)
    _read(st)
    return _stored(st)


def _read(st):
    page = st["case"]["page_size"]
    b, i = _owner(st["out_start"], st["k_rows"].shape[0])
    pos = st["start"][b] + i
    pages, slot = st["page_table"][b, pos // page].long(), (pos % page).long()

    def rows(x, scale):
        if scale is None:
            return x[pages, :, slot]
        if x.dtype == torch.uint8:
            return _values(x[pages, :, slot], scale[pages, :, slot])
        return x.view(torch.uint8)[pages, :, slot].view(torch.float8_e4m3fn).float() * scale[pages][..., None]

    st["k_rows"].copy_(rows(st["k"], st["k_scale"]).flatten(1))
    st["v_rows"].copy_(rows(st["v"], st["v_scale"]).flatten(1))
    return dict(k=st["k_rows"], v=st["v_rows"])


def _softmax(s, seen):
    """Weights of the scores s where `seen` (rows that see nothing: zeros), in s's memory."""
    s.masked_fill_(~seen, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp(min=1e-30))


def _attend(st):
    c, q_len, window = st["case"], st["case"]["q_len"], st["case"]["window"]
    h, hk, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    table = st["page_table"].clamp(min=0).long()
    batch, most = table.shape[0], table.shape[1] * page

    def dense(x, params):
        return _values(x[table], params[table]).transpose(1, 2).reshape(batch, hk, most, hd)

    q = st["q"].float().view(batch, q_len, hk, h // hk, hd).permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, hd)
    s = (q @ dense(st["k"], st["k_scale"]).transpose(2, 3)).mul_(st["scale"])
    p = (st["kv_len"][:, None] - q_len + torch.arange(q_len, device="cuda"))[:, :, None]
    j = torch.arange(most, device="cuda")
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < c["sinks"])
    w = _softmax(s.view(batch, hk, q_len, h // hk, most), seen[:, None, :, None]).view(batch, hk, -1, most)
    o = (w @ dense(st["v"], st["v_scale"])).view(batch, hk, q_len, h // hk, hd)
    return o.permute(0, 2, 1, 3, 4).reshape(batch * q_len, h * hd).bfloat16()


def _packed(st):
    """Sequences laid out side by side with room for the longest."""
    c = st["case"]
    h, hk, hd, window, batch = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["batch"]
    q_start = st["q_start"]
    kv_start = st["kv_start"] if st["kv_start"] is not None else q_start
    most_q, most_kv = c["new"], c["new"] + c["past"]
    n_q, n_kv = q_start.diff(), kv_start.diff()
    i, j = torch.arange(most_q, device="cuda"), torch.arange(most_kv, device="cuda")
    at_q = (q_start[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    at_kv = (kv_start[:-1, None] + j).clamp(max=st["k"].shape[0] - 1)
    p = ((n_kv - n_q)[:, None] + i)[:, :, None]
    seen = (j <= p) & (j < n_kv[:, None, None]) & (i < n_q[:, None])[:, :, None]
    if window:
        seen &= (p - j < window) | (j < c["sinks"])
    q = st["q"][at_q].float().view(batch, most_q, hk, h // hk, hd).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, hd)
    k = st["k"][at_kv].float().view(batch, most_kv, hk, hd).permute(0, 2, 3, 1)
    s = (q @ k).mul_(st["scale"]).view(batch, hk, h // hk, most_q, most_kv)
    w = _softmax(s, seen[:, None, None]).view(batch, hk, -1, most_kv)
    v = st["v"][at_kv].float().view(batch, most_kv, hk, hd).transpose(1, 2)
    o = (w @ v).view(batch, hk, h // hk, most_q, hd).permute(0, 3, 1, 2, 4).reshape(batch, most_q, h * hd)
    b, row = _owner(q_start, st["q"].shape[0])
    inside = b < batch  # rows behind the last sequence stay as they are
    got = o[b.clamp(max=batch - 1), row.clamp(max=most_q - 1)].bfloat16()
    return torch.where(inside[:, None], got, st["out"])


# --------------------------------------------------------------------------------------------- floors
def _visible(i, window, sinks):
    """How many keys a query at position i sees."""
    if i < 0:
        return 0
    return i + 1 if not window else min(i + 1, window + min(sinks, max(0, i + 1 - window)))


def _visible_sum(first, last, window, sinks):
    """The same, over positions first ... last - 1."""
    return sum(_visible(i, window, sinks) for i in range(first, last))


def work(case):
    hd, hk = case["head_dim"], case["kv_heads"]
    packed = hd // 2 + 4 * hd // GROUP  # bytes of a token and key head in 4 bits
    if case["op"] == "store":
        h, r = case["heads"], case["rotary_dim"]
        new, past = _lengths(case, case["new"]), _lengths(case, case["past"], 0)
        n = sum(new)
        wrote = n * (2 * hk * packed + (2 * h * hd + (2 * hk * hd if case["keep_k"] else 0) if r else 0))
        read = n * ((2 * hk + (h if r else 0)) * hd * 2 + 4 * r)
        held = sum(past) if case["back"] == "all" else 0
        return {"bytes": read + wrote + held * 2 * hk * packed + (n + held) * 4 * hk * hd,
                "flops": n * (3 * (h + hk) * r + 10 * hk * hd) + (n + held) * 4 * hk * hd}
    if case["op"] == "read":
        n = sum(m - min(case["skip"], m) for m in _lengths(case, case["kv"]))
        size = {"int4": packed, "e4m3": hd, "bf16": 2 * hd}[case["kind"]]
        return {"bytes": n * 2 * hk * (size + 2 * hd), "flops": n * 4 * hk * hd}
    h, window, sinks, total, flops = case["heads"], case["window"], case["sinks"], 0, 0
    if case["op"] == "cache":
        q_len = case["q_len"]
        for kv in _lengths(case, case["kv"], q_len):
            read = min(kv, _visible(kv - 1, window, sinks) + q_len - 1)
            total += 2 * read * hk * packed + 4 * -(-read // case["page_size"]) + 4 * q_len * h * hd
            flops += 4 * h * hd * _visible_sum(kv - q_len, kv, window, sinks)
        return {"bytes": total, "flops": flops}
    for n, p in zip(_lengths(case, case["new"]), _lengths(case, case["past"], 0)[::-1]):
        first = min(n + p, _visible(p, window, sinks) + n - 1)  # keys that some query sees
        total += 4 * n * h * hd + 4 * first * hk * hd
        flops += 4 * h * hd * _visible_sum(p, n + p, window, sinks)
    return {"bytes": total, "flops": flops}


# --------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "read": _exact_read, "cache": _exact_cache, "packed": _exact_packed}[case["op"]](s)


def _exact_turn(x, cos, sin, rotary_dim, interleaved):
    """Rotates the last axis of x by matrices of angles: pairs as complex numbers."""
    y = x.clone()
    a = torch.arange(rotary_dim // 2, device=x.device)
    first, second = (2 * a, 2 * a + 1) if interleaved else (a, a + rotary_dim // 2)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sin)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_round(x):
    """x [rows, heads, head_dim] as the values that 4 bits hold of it."""
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    step = ((hi - lo) / 15).bfloat16().double()
    mid = (lo + 8 * step).bfloat16().double()
    inverse = (1 / step.clamp(min=_LEAST_STEP)).bfloat16().double()
    code = torch.round((y - mid) * inverse).clamp(-8, 7)
    return torch.where(step >= _LEAST_STEP, mid + code * step, mid).reshape(x.shape)


def _exact_values(codes, params, hd):
    """Values [tokens, head_dim] of rows of codes [tokens, head_dim / 2]: each element looked up by its number."""
    d = torch.arange(hd, device="cuda")
    group, inside = d // GROUP, d % GROUP
    byte = (inside // 4) * (2 * (hd // GROUP)) + 2 * group + (inside % 4) // 2
    c = (codes[:, byte].int() >> (4 * (d % 2)).int()) & 15
    p = params.double()
    return p[:, 1, group] + (c - 8).double() * p[:, 0, group]


def _exact_rows(s, b, first, last, x, scale):
    """Tokens first ... last - 1 of sequence b, [tokens, kv_heads, head_dim]."""
    page, hd, hk = s["case"]["page_size"], s["case"]["head_dim"], s["case"]["kv_heads"]
    if first >= last:
        return torch.zeros(0, hk, hd, device="cuda", dtype=torch.float64)
    low = first // page
    ids = s["page_table"][b, low:(last - 1) // page + 1].long()
    heads = []
    for g in range(hk):
        if scale is None:
            y = x[ids, g].double()
        elif x.dtype == torch.uint8:
            y = _exact_values(x[ids, g].flatten(0, 1), scale[ids, g].flatten(0, 1), hd)
        else:
            y = x.view(torch.uint8)[ids, g].view(torch.float8_e4m3fn).double() * scale[ids, g].double()[:, None, None]
        heads.append(y.reshape(-1, hd)[first - low * page:last - low * page])
    return torch.stack(heads, 1)


def _exact_store(s):
    c = s["case"]
    h, hk, hd, r = c["heads"], c["kv_heads"], c["head_dim"], c["rotary_dim"]
    x = s["qkv"].double().reshape(-1, h + 2 * hk, hd)
    start, new, past = s["new_start"].tolist(), s["new_len"].tolist(), s["past_len"].tolist()
    k_rows, v_rows = [], []
    for b in range(c["batch"]):
        rows = slice(start[b], start[b] + new[b])
        if r:
            cs = s["table"].double()[past[b]:past[b] + new[b], None]
            x[rows, :h + hk] = _exact_turn(x[rows, :h + hk], cs[..., 0], cs[..., 1], r, c["interleaved"])
        if c["back"] == "all":
            k_rows.append(_exact_rows(s, b, 0, past[b], s["k"], s["k_scale"]))
            v_rows.append(_exact_rows(s, b, 0, past[b], s["v"], s["v_scale"]))
        k_rows.append(_exact_round(x[rows, h:h + hk]))
        v_rows.append(_exact_round(x[rows, h + hk:]))
    got = dict(k=torch.cat(k_rows).reshape(-1, hk * hd), v=torch.cat(v_rows).reshape(-1, hk * hd))
    if r:
        got["q_out"] = x[:, :h].reshape(-1, h * hd)
        if s["k_out"] is not None:
            got["k_out"] = x[:, h:h + hk].reshape(-1, hk * hd)
    return got


def _exact_read(s):
    got = {}
    first, n = s["start"].tolist(), s["length"].tolist()
    for name in ("k", "v"):
        rows = [_exact_rows(s, b, first[b], first[b] + n[b], s[name], s[name + "_scale"]) for b in range(s["case"]["batch"])]
        got[name] = torch.cat(rows).flatten(1)
    return got


def _exact_seen(p, window, sinks, n):
    """Keys that a query at position p sees, of n."""
    low = max(0, p - window + 1) if window else 0
    at = torch.cat([torch.arange(min(sinks, low) if window else 0), torch.arange(low, min(p + 1, n))])
    return at.cuda()


def _exact_cache(s):
    c = s["case"]
    h, hk, hd, q_len = c["heads"], c["kv_heads"], c["head_dim"], c["q_len"]
    out = torch.zeros(c["batch"], q_len, h, hd, device="cuda", dtype=torch.float64)
    q = s["q"].double().view(c["batch"], q_len, hk, h // hk, hd)
    for b, n in enumerate(s["kv_len"].tolist()):
        k, v = (_exact_rows(s, b, 0, n, s[x], s[x + "_scale"]) for x in ("k", "v"))
        for t in range(q_len):
            if n - q_len + t < 0:
                continue
            at = _exact_seen(n - q_len + t, c["window"], c["sinks"], n)
            a = torch.softmax(torch.einsum("gid,jgd->gij", q[b, t], k[at]) * s["scale"], -1)
            out[b, t] = torch.einsum("gij,jgd->gid", a, v[at]).reshape(h, hd)
    return out.reshape(c["batch"] * q_len, h * hd)


def _exact_packed(s):
    c = s["case"]
    h, hk, hd, window, sinks = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
    if 4 * h * hd * sum(n * (n + p) for n, p in zip(_lengths(c, c["new"]), _lengths(c, c["past"], 0)[::-1])) > 4e13:
        return None
    q_at = s["q_start"].tolist()
    kv_at = s["kv_start"].tolist() if s["kv_start"] is not None else q_at
    out = s["out"].double()
    for b in range(c["batch"]):
        k, v = (s[x][kv_at[b]:kv_at[b + 1]].double().view(-1, hk, hd).transpose(0, 1) for x in ("k", "v"))
        n = k.shape[1]
        past = n - (q_at[b + 1] - q_at[b])
        for r0 in range(q_at[b], q_at[b + 1], 1024):
            r1 = min(r0 + 1024, q_at[b + 1])
            i = past + torch.arange(r0 - q_at[b], r1 - q_at[b], device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            hidden = j > i
            if window:
                hidden |= (i - j >= window) & (j >= sinks)
            q = s["q"][r0:r1].double().view(r1 - r0, hk, h // hk, hd).permute(1, 2, 0, 3).reshape(hk, -1, hd)
            a = (q @ k.transpose(1, 2) * s["scale"]).view(hk, h // hk, r1 - r0, n).masked_fill(hidden, -math.inf)
            o = torch.softmax(a, -1).view(hk, -1, n) @ v
            out[r0:r1] = o.view(hk, h // hk, r1 - r0, hd).permute(2, 0, 1, 3).reshape(r1 - r0, h * hd)
    return out
