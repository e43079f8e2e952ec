"""Serving operators of the Transformer stack: rotary positions, the paged key/value cache and the two attentions that read it.

Each case is one call of one operator on device tensors:
  rotary   `serving.rotary`: q and k rows of a step, or the gradient of a long prompt's rotation
  append   `serving.KVCache.append`: rotates q and k of new tokens and stores their keys and values in the cache's pages
  cache    `serving.KVCache.attend`: the newest token (or few) of every sequence over its cached keys and values
  window   `serving.window_attention`: causal prompt attention with a sliding window and first tokens that stay visible
"""

import math

import torch

own = False

_SCALE_MIN, _SCALE_MAX = -40, 40  # exponents of a page's scale
_E4M3_MAX = 448.0


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # The q and k heads of one decoding step of 8 sequences (12 heads of 64): a call of a few microseconds.
        dict(name="rotary_step", op="rotary", tokens=8, heads=24, head_dim=64, rotary_dim=64, interleaved=False,
             inverse=False, pad=768, max_positions=4096),
        # Gradient through the positions of a long prompt: neighbouring pairs, half of each head, a strided input.
        dict(name="rotary_prompt_gradient", op="rotary", tokens=32771, heads=32, head_dim=128, rotary_dim=64,
             interleaved=True, inverse=True, pad=2048, max_positions=65536),
        # One new token in each of 64 conversations, 8-bit pages of 64 tokens.
        dict(name="append_step", op="append", batch=64, new=1, past=8191, heads=32, kv_heads=8, head_dim=128,
             rotary_dim=128, interleaved=False, page_size=64, kind="e4m3", ragged=True, keep_k=False),
        # A batch of ragged prompts entering an 8-bit cache (16 heads of 64), rotated keys kept for the prompt's attention.
        dict(name="append_prompts", op="append", batch=16, new=2048, past=0, heads=16, kv_heads=16, head_dim=64,
             rotary_dim=64, interleaved=False, page_size=32, kind="e4m3", ragged=True, keep_k=True),
        # Chunks of three long documents behind what the cache already holds, bf16 pages, a quarter of each head rotated.
        dict(name="append_chunks_bf16", op="append", batch=3, new=5003, past=7001, heads=16, kv_heads=4, head_dim=128,
             rotary_dim=32, interleaved=True, page_size=16, kind="bf16", ragged=True, keep_k=False),
        # One sequence of about a thousand tokens, every head with its own keys: latency.
        dict(name="cache_one", op="cache", batch=1, kv=1001, q_len=1, heads=12, kv_heads=12, head_dim=64, page_size=16,
             kind="e4m3", window=0, sinks=0, ragged=False),
        # An ordinary serving batch: 64 sequences of up to 8192 tokens, four query heads to a key head.
        dict(name="cache_batch", op="cache", batch=64, kv=8192, q_len=1, heads=32, kv_heads=8, head_dim=128,
             page_size=64, kind="e4m3", window=0, sinks=0, ragged=True),
        # Long documents: 8 sequences of 131072 tokens (2.1 GB of 8-bit keys and values).
        dict(name="cache_long", op="cache", batch=8, kv=131072, q_len=1, heads=32, kv_heads=8, head_dim=128,
             page_size=128, kind="e4m3", window=0, sinks=0, ragged=False),
        # Streaming with a window and sinks over bf16 pages, a token and one draft behind it, five query heads to a key head.
        dict(name="cache_streaming_bf16", op="cache", batch=32, kv=20011, q_len=2, heads=20, kv_heads=4, head_dim=128,
             page_size=32, kind="bf16", window=4096, sinks=4, ragged=True),
        # A short odd prompt: latency.
        dict(name="window_short", op="window", batch=1, seq=77, heads=4, kv_heads=4, head_dim=64, window=32, sinks=4,
             ragged=False),
        # A batch of ragged prompts (16 heads of 64).
        dict(name="window_batch", op="window", batch=16, seq=2048, heads=16, kv_heads=16, head_dim=64, window=512,
             sinks=4, ragged=True),
        # One long prompt, four query heads of 128 to a key head.
        dict(name="window_long", op="window", batch=1, seq=32768, heads=16, kv_heads=4, head_dim=128, window=4096,
             sinks=16, ragged=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "cache", "cache", "window"])
    head_dim = rng.choice([32, 64, 64, 128, 128, 128])
    if op == "rotary":
        head_dim = rng.choice([head_dim, 256])
        heads = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, min(65536, 32768 * 32 * 128 // (heads * head_dim))))
        return dict(op=op, tokens=tokens, heads=heads, head_dim=head_dim, rotary_dim=16 * rng.randint(1, head_dim // 16),
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.4, pad=8 * rng.randint(0, 200),
                    max_positions=rng.choice([8192, 131072]))
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
    kind = rng.choice(["e4m3", "e4m3", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        batch = _log(rng, 1, 128)
        width = (kv_heads * (group + 2)) * head_dim
        new = _log(rng, 1, max(1, min(8192, 2048 * 16 * 48 * 64 // (batch * width))))
        past = rng.choice([0, rng.randint(1, 5000)])
        return dict(op=op, batch=batch, new=new, past=past, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rng.choice([0, 16 * rng.randint(1, head_dim // 16), head_dim]),
                    interleaved=rng.random() < 0.5, page_size=page, kind=kind, ragged=batch > 1 and rng.random() < 0.7,
                    keep_k=rng.random() < 0.5)
    window = rng.choice([0, _log(rng, 1, 8192), _log(rng, 64, 8192)])
    sinks = rng.choice([0, 1, 4, rng.randint(1, 200)]) if window else 0
    if op == "cache":
        batch = _log(rng, 1, 256)
        most = 8 * 131072 * 8 * 128 // (batch * kv_heads * head_dim * (2 if kind == "bf16" else 1))
        q_len = rng.choice([1, 1, 1, 2, 4])
        return dict(op=op, batch=batch, kv=max(q_len, _log(rng, 1, min(131072, most))), q_len=q_len,
                    heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, page_size=page, kind=kind,
                    window=window, sinks=sinks, ragged=batch > 1 and rng.random() < 0.6)
    # window: the score matrix of the plain form bounds the sizes
    heads = kv_heads * group
    seq = _log(rng, 1, 32768)
    seen = min(seq, window or seq) + 128
    batch = max(1, min(_log(rng, 1, 32), 32768 * 4224 * 16 // (seq * seen * heads)))
    if seq * seen * heads * batch > 32768 * 4224 * 16:
        seq, batch = 2048, 1
    return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window,
                sinks=sinks, ragged=batch > 1 and rng.random() < 0.6)


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
    x = _activations((pages, kv_heads, page, head_dim), head_dim, g)
    if kind == "bf16":
        return x, None
    scale = torch.exp2(_exponent(x.abs().float().amax((2, 3))).float())
    return (x.float() / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = _generator(seed)
    hd, state = case["head_dim"], {"case": case}
    if case["op"] == "rotary":
        width = case["heads"] * hd
        rows = torch.randn(case["tokens"], width + case["pad"], device="cuda", generator=g).bfloat16()
        most = case["max_positions"]
        start = int(torch.randint(0, max(1, most - case["tokens"]), (1,), generator=torch.Generator().manual_seed(seed)))
        positions = (torch.arange(case["tokens"], device="cuda") + start) % most
        return state | dict(x=rows[:, :width], positions=positions.int(), table=_table(most, case["rotary_dim"]),
                            out=torch.empty(case["tokens"], width, device="cuda", dtype=torch.bfloat16))
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "append":
        batch, kind, page = case["batch"], case["kind"], case["page_size"]
        new, past = _lengths(case, case["new"]), _lengths(case, case["past"], 0)[::-1]
        table, pages = _pages([n + p for n, p in zip(new, past)], page, seed)
        k, ks = _cache(pages, hk, page, hd, kind, g)
        v, vs = _cache(pages, hk, page, hd, kind, g)
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        tokens = start[-1]
        to = dict(device="cuda", dtype=torch.int32)
        r = case["rotary_dim"]
        out = dict(device="cuda", dtype=torch.bfloat16)
        return state | dict(
            qkv=_activations((tokens, (h + 2 * hk) * hd), hd, g), new_start=torch.tensor(start[:-1], **to),
            new_len=torch.tensor(new, **to), past_len=torch.tensor(past, **to), page_table=table, max_new=max(new),
            k=k, v=v, k_scale=ks, v_scale=vs, table=_table(case["new"] + case["past"] + 1, r) if r else None,
            q_out=torch.empty(tokens, h * hd, **out) if r else None,
            k_out=torch.empty(tokens, hk * hd, **out) if r and case["keep_k"] else None)
    if case["op"] == "cache":
        batch, page = case["batch"], case["page_size"]
        lengths = _lengths(case, case["kv"], case["q_len"])
        table, pages = _pages(lengths, page, seed)
        k, ks = _cache(pages, hk, page, hd, case["kind"], g)
        v, vs = _cache(pages, hk, page, hd, case["kind"], g)
        rows = batch * case["q_len"]
        q = torch.randn(rows, h * hd, device="cuda", generator=g).bfloat16()
        return state | dict(q=q, page_table=table, kv_len=torch.tensor(lengths, device="cuda", dtype=torch.int32), k=k,
                            v=v, k_scale=ks, v_scale=vs, scale=hd**-0.5, out=torch.empty_like(q))
    rows = case["batch"] * case["seq"]
    qkv = torch.randn(rows, (h + 2 * hk) * hd, device="cuda", generator=g).bfloat16()
    lengths = _lengths(case, case["seq"])
    return state | dict(q=qkv[:, :h * hd], k=qkv[:, h * hd:(h + hk) * hd], v=qkv[:, (h + hk) * hd:],
                        kv_len=torch.tensor(lengths, device="cuda", dtype=torch.int32) if case["ragged"] else None,
                        scale=hd**-0.5, out=torch.empty(rows, h * hd, device="cuda", dtype=torch.bfloat16))


# --------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "cache": _own_cache, "window": _own_window}[case["op"]](state)
    return {"rotary": _rotary, "append": _append, "cache": _attend, "window": _window}[case["op"]](state)


def _kv_cache(state):
    """The cache object that a user's program keeps around its pages."""
    if "cache" not in state:
        from tiktoktechjam2026track3_b200 import serving

        state["cache"] = serving.KVCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state["cache"]


def _own_rotary(s):
    from tiktoktechjam2026track3_b200 import serving

    c = s["case"]
    return serving.rotary(s["x"], s["positions"], s["table"], c["head_dim"], out=s["out"], interleaved=c["interleaved"],
                          inverse=c["inverse"])


def _own_append(s):
    c, cache = s["case"], _kv_cache(s)
    cache.append(s["qkv"], c["heads"], s["new_start"], s["new_len"], s["past_len"], s["page_table"], s["max_new"],
                 table=s["table"], interleaved=c["interleaved"], q_out=s["q_out"], k_out=s["k_out"])
    return _appended(s)


def _appended(s):
    got = dict(k=s["k"], v=s["v"])
    for name in ("k_scale", "v_scale", "q_out", "k_out"):
        if s[name] is not None:
            got[name] = s[name]
    return got


def _own_cache(s):
    c = s["case"]
    return _kv_cache(s).attend(s["q"], s["page_table"], s["kv_len"], q_len=c["q_len"], scale=s["scale"],
                               window=c["window"], sinks=c["sinks"], out=s["out"])


def _own_window(s):
    from tiktoktechjam2026track3_b200 import serving

    c = s["case"]
    return serving.window_attention(s["q"], s["k"], s["v"], c["batch"], c["seq"], c["head_dim"], window=c["window"],
                                    sinks=c["sinks"], kv_len=s["kv_len"], scale=s["scale"], out=s["out"])


# --------------------------------------------------------------------------------------------- plain forms
def _rotate(x, c, s, rotary_dim, interleaved):
    """x [rows, heads, head_dim] in 32 bits, c and s [rows, 1, rotary_dim / 2]."""
    half = rotary_dim // 2
    x1, x2 = (x[..., 0:rotary_dim:2], x[..., 1:rotary_dim:2]) if interleaved else (x[..., :half], x[..., half:rotary_dim])
    y1, y2 = x1 * c - x2 * s, x2 * c + x1 * s
    y = torch.stack([y1, y2], -1).flatten(-2) if interleaved else torch.cat([y1, y2], -1)
    return torch.cat([y, x[..., rotary_dim:]], -1)


def _rotary(st):
    c = st["case"]
    x = st["x"].float().view(c["tokens"], c["heads"], c["head_dim"])
    cs = st["table"][st["positions"]][:, None]
    y = _rotate(x, cs[..., 0], -cs[..., 1] if c["inverse"] else cs[..., 1], c["rotary_dim"], c["interleaved"])
    return y.flatten(1).bfloat16()


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, kept in range (a page of zeros has the least)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x - 9 + (m > 0.875), _SCALE_MIN).clamp(_SCALE_MIN, _SCALE_MAX)


def _e4m3(x, scale):
    y = (x / scale).clamp(-_E4M3_MAX, _E4M3_MAX)
    return torch.where(x.isfinite(), y, math.nan).to(torch.float8_e4m3fn)


def _append(st):
    c, qkv, past = st["case"], st["qkv"], st["past_len"]
    h, hk, hd, page, r = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"], c["rotary_dim"]
    rows = torch.arange(qkv.shape[0], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(st["new_start"], rows, right=True) - 1
    pos = past[b] + rows - st["new_start"][b]
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
    if c["kind"] == "bf16":
        st["k"][pages, :, slot] = k.bfloat16()
        st["v"][pages, :, slot] = v.bfloat16()
        return _appended(st)
    # A page that holds earlier tokens of its sequence keeps at least its scale; they are rounded again if it grows.
    first = st["page_table"].gather(1, (past // page).long().clamp(max=st["page_table"].shape[1] - 1)[:, None])[:, 0]
    first = first.clamp(min=0).long()
    held = past % page
    for new, store, scale in ((k, st["k"], st["k_scale"]), (v, st["v"], st["v_scale"])):
        most = torch.where(new.isfinite(), new, 0.0).abs().amax(-1)
        amax = torch.zeros_like(scale).index_reduce_(0, pages, most, "amax")
        e = _exponent(amax)
        old = torch.log2(scale[first]).to(e.dtype)
        e = e.index_reduce(0, first, torch.where((held > 0)[:, None], old, _SCALE_MIN), "amax")
        touched = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, pages, True)
        grown = torch.exp2((old - e[first]).float())[:, :, None, None]
        block = store[first].float()
        again = (block * grown).to(torch.float8_e4m3fn).float()
        inside = torch.arange(page, device="cuda")[None, :] < held[:, None]
        block = torch.where(inside[:, None, :, None], again, block)
        store.view(torch.uint8)[first] = block.to(torch.float8_e4m3fn).view(torch.uint8)
        scale.copy_(torch.where(touched[:, None], torch.exp2(e.float()), scale))
        store.view(torch.uint8)[pages, :, slot] = _e4m3(new, scale[pages][:, :, None]).view(torch.uint8)
    return _appended(st)


def _attend(st):
    c, q_len, window = st["case"], st["case"]["q_len"], st["case"]["window"]
    h, hk, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    table = st["page_table"].clamp(min=0).long()
    batch, most = table.shape[0], table.shape[1] * page

    def dense(x, scale):
        x = x.view(torch.uint8)[table].view(torch.float8_e4m3fn) if scale is not None else x[table]
        x = x.float() * scale[table][..., None, None] if scale is not None else x.float()
        return x.transpose(1, 2).reshape(batch, hk, most, hd)

    q = st["q"].float().view(batch, q_len, hk, h // hk, hd).permute(0, 2, 1, 3, 4).reshape(batch, hk, -1, hd)
    s = (q @ dense(st["k"], st["k_scale"]).transpose(2, 3)) * st["scale"]
    p = (st["kv_len"][:, None] - q_len + torch.arange(q_len, device="cuda"))[:, :, None]
    j = torch.arange(most, device="cuda")
    seen = j <= p
    if window:
        seen &= (p - j < window) | (j < c["sinks"])
    s = s.view(batch, hk, q_len, h // hk, most).masked_fill(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    w = (s - top).exp()
    w = (w / w.sum(-1, keepdim=True).clamp(min=1e-30)).view(batch, hk, -1, most)
    o = (w @ dense(st["v"], st["v_scale"])).view(batch, hk, q_len, h // hk, hd)
    return o.permute(0, 2, 1, 3, 4).reshape(batch * q_len, h * hd).bfloat16()


def _window(st):
    """Blocks of queries against the keys that any of a block may see: the first tokens, then the band before it."""
    c = st["case"]
    batch, seq, h, hk, hd = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["head_dim"]
    window, block = c["window"] or seq, 128
    blocks = -(-seq // block)
    i = torch.arange(blocks, device="cuda")[:, None] * block + torch.arange(block, device="cuda")
    band = min(blocks * block, window + block - 1)
    j = i[:, -1:] - torch.arange(band, device="cuda")  # [blocks, band], newest first
    sinks = torch.arange(min(c["sinks"], seq), device="cuda").expand(blocks, -1)
    keys = torch.cat([sinks, j], 1)
    first = torch.cat([torch.ones_like(sinks, dtype=torch.bool), j >= c["sinks"]], 1)  # a sink inside the band counts once
    n = st["kv_len"] if st["kv_len"] is not None else torch.full((batch,), seq, device="cuda", dtype=torch.int32)
    d = i[:, :, None] - keys[:, None]
    seen = (d >= 0) & ((d < window) | (keys < c["sinks"])[:, None]) & (first & (keys >= 0))[:, None]
    seen = seen & (i[None] < n[:, None, None])[..., None]  # [batch, blocks, block, keys]
    q = st["q"].float().view(batch, seq, h, hd)
    q = torch.nn.functional.pad(q, (0, 0, 0, 0, 0, blocks * block - seq))
    q = q.view(batch, blocks, block, hk, h // hk, hd).permute(0, 1, 3, 4, 2, 5).flatten(3, 4)
    at = keys.clamp(0, seq - 1)
    k = st["k"].float().view(batch, seq, hk, hd)[:, at].permute(0, 1, 3, 4, 2)
    s = (q @ k).mul_(st["scale"]).view(batch, blocks, hk, h // hk, block, -1)
    s.masked_fill_(~seen[:, :, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    s.div_(s.sum(-1, keepdim=True).clamp(min=1e-30))
    v = st["v"].float().view(batch, seq, hk, hd)[:, at].transpose(2, 3)
    o = (s.flatten(3, 4) @ v).view(batch, blocks, hk, h // hk, block, hd).permute(0, 1, 4, 2, 3, 5)
    return o.reshape(batch, blocks * block, h * hd)[:, :seq].reshape(batch * seq, h * hd).bfloat16()


# --------------------------------------------------------------------------------------------- floors
def _visible(i, window, sinks):
    """How many keys a query at position i sees."""
    if i < 0:
        return 0
    return i + 1 if not window else min(i + 1, window + min(sinks, max(0, i + 1 - window)))


def work(case):
    hd = case["head_dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"] * hd
        return {"bytes": 4 * n + 4 * case["tokens"] * case["rotary_dim"], "flops": 6 * n * case["rotary_dim"] // hd // 2}
    h, hk = case["heads"], case["kv_heads"]
    size = 1 if case.get("kind") == "e4m3" else 2
    if case["op"] == "append":
        n, r = sum(_lengths(case, case["new"])), case["rotary_dim"]
        wrote = n * (2 * hk * hd * size + (2 * h * hd + (2 * hk * hd if case["keep_k"] else 0) if r else 0))
        read = n * ((2 * hk + (h if r else 0)) * hd * 2 + 4 * r)
        return {"bytes": read + wrote, "flops": n * (3 * (h + hk) * r + 4 * hk * hd)}
    window, sinks, total, flops = case["window"], case["sinks"], 0, 0
    if case["op"] == "cache":
        q_len = case["q_len"]
        for kv in _lengths(case, case["kv"], q_len):
            read = min(kv, _visible(kv - 1, window, sinks) + q_len - 1)
            pages = -(-read // case["page_size"])
            total += 2 * read * hk * hd * size + (8 * hk * pages if size == 1 else 0) + 4 * pages + 4 * q_len * h * hd
            flops += 4 * h * hd * sum(_visible(kv - q_len + t, window, sinks) for t in range(q_len))
        return {"bytes": total, "flops": flops}
    for n in _lengths(case, case["seq"]):
        total += n * (2 * h + 2 * hk) * hd * 2
        flops += 4 * h * hd * sum(_visible(i, window, sinks) for i in range(n))
    return {"bytes": total, "flops": flops}


# --------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "append": _exact_append, "cache": _exact_cache, "window": _exact_window}[case["op"]](s)


def _exact_turn(x, cos, sin, rotary_dim, interleaved):
    """Rotates the last axis of x by matrices of angles: pairs as complex numbers."""
    y = x.clone()
    a = torch.arange(rotary_dim // 2, device=x.device)
    first, second = (2 * a, 2 * a + 1) if interleaved else (a, a + rotary_dim // 2)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(cos, sin)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(s):
    c = s["case"]
    cs = s["table"].double()[s["positions"].long()]
    sign = -1.0 if c["inverse"] else 1.0
    x = s["x"].double().reshape(c["tokens"], c["heads"], c["head_dim"])
    return _exact_turn(x, cs[:, None, :, 0], sign * cs[:, None, :, 1], c["rotary_dim"], c["interleaved"]).reshape(
        c["tokens"], -1)


def _exact_code(x):
    """Nearest value of 4 exponent and 3 mantissa bits, ties to even, for |x| <= 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-60))).clamp(min=-6.0)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(s):
    c = s["case"]
    h, hk, hd, page, r = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"], c["rotary_dim"]
    got = {n: s[n].double() for n in ("k", "v", "k_scale", "v_scale") if s[n] is not None}
    x = s["qkv"].double().reshape(-1, h + 2 * hk, hd)
    start, new, past = s["new_start"].tolist(), s["new_len"].tolist(), s["past_len"].tolist()
    table = s["page_table"].tolist()
    for b in range(c["batch"]):
        rows = slice(start[b], start[b] + new[b])
        if r:
            cs = s["table"].double()[past[b]:past[b] + new[b], None]
            x[rows, :h + hk] = _exact_turn(x[rows, :h + hk], cs[..., 0], cs[..., 1], r, c["interleaved"])
    if r:
        got["q_out"] = x[:, :h].reshape(-1, h * hd)
        if s["k_out"] is not None:
            got["k_out"] = x[:, h:h + hk].reshape(-1, hk * hd)
    for b in range(c["batch"]):
        at = past[b]
        while at < past[b] + new[b]:
            stop = min((at // page + 1) * page, past[b] + new[b])
            row, p, slot = start[b] + at - past[b], table[b][at // page], at % page
            for name, first in (("k", h), ("v", h + hk)):
                fresh = x[row:row + stop - at, first:first + hk].transpose(0, 1)  # [heads, tokens, head_dim]
                store = got[name]
                if c["kind"] == "bf16":
                    store[p, :, slot:slot + stop - at] = fresh
                    continue
                most = torch.log2(fresh.abs().amax((1, 2)).clamp(min=2.0**-100) / 448.0)
                e = torch.ceil(most - 1e-9).clamp(-40, 40)  # a maximum of exactly 448 * 2^e takes e
                if slot:
                    before = torch.log2(got[name + "_scale"][p])
                    e = torch.maximum(e, before)
                    store[p, :, :slot] = _exact_code(store[p, :, :slot] * torch.exp2(before - e)[:, None, None])
                got[name + "_scale"][p] = torch.exp2(e)
                store[p, :, slot:slot + stop - at] = _exact_code(fresh * torch.exp2(-e)[:, None, None])
            at = stop
    return got


def _exact_cache(s):
    c = s["case"]
    h, hk, hd, q_len, window = c["heads"], c["kv_heads"], c["head_dim"], c["q_len"], c["window"]
    out = torch.zeros(c["batch"], q_len, h, hd, device="cuda", dtype=torch.float64)
    q = s["q"].double().view(c["batch"], q_len, hk, h // hk, hd)
    lengths = s["kv_len"].tolist()
    for b in range(c["batch"]):
        n = lengths[b]
        ids = s["page_table"][b, :-(-n // c["page_size"])].long().tolist()
        for g in range(hk):
            def rows(x, scale):
                if scale is None:
                    return x[ids, g].double().reshape(-1, hd)[:n]
                y = x.view(torch.uint8)[ids, g].view(torch.float8_e4m3fn).double()
                return (y * scale[ids, g].double()[:, None, None]).reshape(-1, hd)[:n]

            k, v = rows(s["k"], s["k_scale"]), rows(s["v"], s["v_scale"])
            for t in range(q_len):
                p = n - q_len + t
                if p < 0:
                    continue
                low = max(0, p - window + 1) if window else 0
                at = torch.cat([torch.arange(min(c["sinks"], low) if window else 0), torch.arange(low, p + 1)]).cuda()
                a = torch.softmax(q[b, t, g] @ k[at].T * s["scale"], -1)
                out[b, t, g * (h // hk):(g + 1) * (h // hk)] = a @ v[at]
    return out.reshape(c["batch"] * q_len, h * hd)


def _exact_window(s):
    c = s["case"]
    seq, h, hk, hd, window = c["seq"], c["heads"], c["kv_heads"], c["head_dim"], c["window"]
    out = torch.zeros(c["batch"], seq, h, hd, device="cuda", dtype=torch.float64)
    lengths = s["kv_len"].tolist() if s["kv_len"] is not None else [seq] * c["batch"]
    heads = [x.view(c["batch"], seq, -1, hd) for x in (s["q"], s["k"], s["v"])]
    for b in range(c["batch"]):
        q, k, v = (x[b].double().transpose(0, 1) for x in heads)
        for i0 in range(0, lengths[b], 1024):
            i1 = min(i0 + 1024, lengths[b])
            low = max(0, i0 - window + 1) if window else 0
            j = torch.cat([torch.arange(min(c["sinks"], low)), torch.arange(low, i1)]).cuda()
            i = torch.arange(i0, i1, device="cuda")[:, None]
            seen = (j <= i) & ((i - j < window) | (j < c["sinks"])) if window else j <= i
            a = q[:, i0:i1].reshape(hk, -1, hd) @ k[:, j].transpose(1, 2) * s["scale"]
            a = a.view(hk, h // hk, i1 - i0, -1).masked_fill(~seen, -math.inf)
            o = torch.softmax(a, -1).view(hk, -1, len(j)) @ v[:, j]
            out[b, i0:i1] = o.view(h, i1 - i0, hd).transpose(0, 1)
    return out.reshape(c["batch"] * seq, h * hd)
