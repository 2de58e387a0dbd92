"""Cases of the cache-side operators of large-model serving: query / key norms with the rotation,
the block-scaled 8-bit KV cache (write, decode, chunked prefill) and attention over selected pages.

`run` computes a pass in plain torch (`own` false) or through b200attn's ops (`own` true).
`exact` computes the same outputs from the definitions in 64 bits.

Shapes: Llama-3.2-1B attention (32 query heads, 8 KV heads, head size 64), Llama-3.1-8B (32 / 8 /
128) and Llama-3.1-70B (64 / 8 / 128) as the repository's benchmark configurations name them.
"""
import math
import sys

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
QMAX = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
EPS = 1e-6


def _ops():
    if "tt-xla_b200" not in sys.path:
        sys.path.insert(0, "tt-xla_b200")
    from b200attn import ops

    return ops


# ------------------------------------------------------------------------------------- cases
def listed():
    c1 = dict(nq=32, nkv=8, hd=64, bs=32)
    c8 = dict(nq=32, nkv=8, hd=128, bs=64)
    c70 = dict(nq=64, nkv=8, hd=128, bs=64)
    return [
        # one decode step of eight users: latency is all there is
        dict(name="norm_rope_decode", op="norm_rope", tokens=8, rotary=64, neox=True, cache="bf16",
             pos_hi=1024, **c1),
        # four prompts of 2048 tokens
        dict(name="norm_rope_prompt", op="norm_rope", tokens=8192, rotary=128, neox=True,
             cache="bf16", pos_hi=2048, **c8),
        # a decode step appends one token to each of 64 sequences
        dict(name="write_int8_append", op="write", fmt="int8", seqs=64, q_lo=1, q_hi=1, start_hi=63,
             bounds=True, nkv=8, hd=128, bs=64),
        # four prompts of 2048 tokens fill a cache in e4m3
        dict(name="write_e4m3_prompt", op="write", fmt="e4m3", seqs=4, q_lo=2048, q_hi=2048,
             start_hi=0, bounds=False, nkv=8, hd=128, bs=64),
        # eight short users, head size 64
        dict(name="decode_int8_short", op="decode", fmt="int8", users=8, ctx_lo=128, ctx_hi=1024,
             window=0, sinks=False, **c1),
        # 64 users of mixed lengths
        dict(name="decode_e4m3_mixed", op="decode", fmt="e4m3", users=64, ctx_lo=1024, ctx_hi=8192,
             window=0, sinks=False, **c8),
        # long contexts, 32 users
        dict(name="decode_int8_long", op="decode", fmt="int8", users=32, ctx_lo=32768, ctx_hi=32768,
             window=0, sinks=False, **c70),
        # one user with a long context: the work has to be split over it
        dict(name="decode_int8_single", op="decode", fmt="int8", users=1, ctx_lo=30000,
             ctx_hi=32768, window=0, sinks=True, **c70),
        # two chunks of 512 tokens behind 4096 cached ones
        dict(name="prefill_int8_chunks", op="prefill", fmt="int8", seqs=2, q_lo=512, q_hi=512,
             start_lo=4096, start_hi=4096, **c8),
        # short ragged chunks, head size 64
        dict(name="prefill_e4m3_ragged", op="prefill", fmt="e4m3", seqs=5, q_lo=3, q_hi=200,
             start_lo=0, start_hi=700, **c1),
        # few pages of short contexts
        dict(name="pages_bf16_short", op="pages", fmt="bf16", users=8, ctx_lo=128, ctx_hi=1024,
             pages=8, first=1, last=1, **c1),
        # an eighth of long contexts
        dict(name="pages_int8_long", op="pages", fmt="int8", users=32, ctx_lo=30000, ctx_hi=32768,
             pages=64, first=1, last=2, **c70),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "write", "decode", "prefill", "pages"])
    nkv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128])
    bs = rng.choice([32, 64])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    heads = dict(nq=nkv * group, nkv=nkv, hd=hd, bs=bs)
    if op == "norm_rope":
        return dict(op=op, tokens=_log_int(rng, 1, 8192), rotary=rng.choice([16, 32, 48, hd, hd]),
                    neox=rng.random() < 0.7, cache=rng.choice(["bf16", "bf16", "e4m3"]),
                    pos_hi=_log_int(rng, 64, 1 << 20), **heads)
    if op == "write":
        q_hi = _log_int(rng, 1, 2048)
        return dict(op=op, fmt=rng.choice(["int8", "e4m3", "bf16"]),
                    seqs=_log_int(rng, 1, max(1, 8192 // (q_hi + 64))), q_lo=max(1, q_hi // 3),
                    q_hi=q_hi, start_hi=rng.randrange(0, 300), bounds=True, nkv=nkv, hd=hd, bs=bs)
    if op == "decode":
        ctx_hi = _log_int(rng, 1, 32768)
        users = _log_int(rng, 1, max(1, min(64, 400000 // ctx_hi)))
        return dict(op=op, fmt=rng.choice(["int8", "e4m3"]), users=users, ctx_lo=max(1, ctx_hi // 4),
                    ctx_hi=ctx_hi, window=rng.choice([0, 0, 1, 100, 1000]),
                    sinks=rng.random() < 0.3, **heads)
    if op == "prefill":
        heads = dict(nq=nkv * min(group, 8), nkv=nkv, hd=hd, bs=bs)
        q_hi = _log_int(rng, 2, 512)
        return dict(op=op, fmt=rng.choice(["int8", "e4m3"]), seqs=rng.randrange(1, 4),
                    q_lo=max(1, q_hi // 2), q_hi=q_hi, start_lo=0,
                    start_hi=_log_int(rng, 1, 4096), **heads)
    ctx_hi = _log_int(rng, 64, 32768)
    users = _log_int(rng, 1, max(1, min(32, 400000 // ctx_hi)))
    return dict(op=op, fmt=rng.choice(["bf16", "int8", "e4m3"]), users=users,
                ctx_lo=max(1, ctx_hi // 8), ctx_hi=ctx_hi, pages=_log_int(rng, 4, 128),
                first=rng.randrange(0, 3), last=rng.randrange(1, 3), **heads)


# ------------------------------------------------------------------------------------ inputs
def _ints(gen, n, lo, hi):
    return torch.randint(lo, hi + 1, (n,), generator=gen)


def _spread(gen, n, *ranges):
    """For each range n whole numbers spread over it, the same ones for every seed (the outputs'
    sizes go by them), in an order that goes by the seed."""
    order = torch.randperm(n, generator=gen)
    return [(lo + (torch.arange(n) * 0.6180339887 * (i + 1) % 1 * (hi - lo + 1)).long())[order]
            for i, (lo, hi) in enumerate(ranges)]


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _page_table(gen, lens, bs, spare=1):
    """A random permutation of the pool's pages; rows beyond a sequence's pages hold page 0."""
    need = [(n + bs - 1) // bs for n in lens]
    nb = sum(need) + spare
    perm = torch.randperm(nb, generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table.to(DEV), nb


def _key_pages(g, n, nkv, bs, hd):
    """Keys: a few strong channels and a direction of their own for every page."""
    x = _randn(g, n, nkv, bs, hd)
    x += 0.5 * _randn(g, n, nkv, 1, hd)
    x[..., : hd // 16] *= 3.0
    return x.to(torch.bfloat16)


def _pool(g, fmt, nb, nkv, bs, hd, with_bounds):
    """K / V caches filled page by page as the writes leave them."""
    kind = CODE.get(fmt, torch.bfloat16)
    s = dict(k_cache=torch.empty(nb, nkv, bs, hd, dtype=kind, device=DEV),
             v_cache=torch.empty(nb, nkv, bs, hd, dtype=kind, device=DEV))
    if fmt != "bf16":
        s["k_scale"] = torch.empty(nb, nkv, device=DEV)
        s["v_scale"] = torch.empty(nb, nkv, device=DEV)
    if with_bounds:
        s["k_bounds"] = torch.empty(nb, nkv, 2, hd, dtype=torch.bfloat16, device=DEV)
    for a in range(0, nb, 2048):
        b = min(nb, a + 2048)
        for which in "kv":
            x = _key_pages(g, b - a, nkv, bs, hd) if which == "k" else \
                _randn(g, b - a, nkv, bs, hd).to(torch.bfloat16)
            if with_bounds and which == "k":
                s["k_bounds"][a:b, :, 0] = x.amin(2)
                s["k_bounds"][a:b, :, 1] = x.amax(2)
            if fmt == "bf16":
                s[which + "_cache"][a:b] = x
            else:
                scale = x.float().abs().amax((2, 3)) / QMAX[fmt]
                s[which + "_scale"][a:b] = scale
                codes = x.float() / scale[:, :, None, None]
                s[which + "_cache"][a:b] = \
                    (codes.round() if fmt == "int8" else codes).to(kind)
    return s


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=c)
    nkv, hd, bs = c["nkv"], c["hd"], c["bs"]
    if c["op"] == "norm_rope":
        t, nq = c["tokens"], c["nq"]
        # the rows of a fused projection: query, key and value side by side
        qkv = (_randn(g, t, (nq + 2 * nkv) * hd) * 2.0).to(torch.bfloat16)
        s["query"], s["key"], s["value"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
        s["q_weight"] = (1.0 + 0.2 * _randn(g, hd)).to(torch.bfloat16)
        s["k_weight"] = (1.0 + 0.2 * _randn(g, hd)).to(torch.bfloat16)
        s["positions"] = torch.randint(0, c["pos_hi"], (t,), generator=g, device=DEV)
        r = c["rotary"]
        s["inv_freq"] = (1.0 / 500000.0 ** (torch.arange(0, r, 2) / r)).to(DEV)
        nb = (t + bs - 1) // bs + 1
        slots = torch.randperm(nb * bs, generator=gen)[:t]
        slots[torch.rand(t, generator=gen) < 0.02] = -1        # padding rows
        s["slots"] = slots.to(DEV)
        kind = torch.bfloat16 if c["cache"] == "bf16" else torch.float8_e4m3fn
        s["k_cache"] = torch.zeros(nb, nkv, bs, hd, dtype=kind, device=DEV)
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        s["out_query"] = torch.empty(t, nq * hd, dtype=torch.bfloat16, device=DEV)
        s["out_key"] = torch.empty(t, nkv * hd, dtype=torch.bfloat16, device=DEV)
    elif c["op"] == "write":
        lens, start = _spread(gen, c["seqs"], (c["q_lo"], c["q_hi"]), (0, c["start_hi"]))
        s["page_table"], nb = _page_table(gen, (lens + start).tolist(), bs)
        s.update(_pool(g, c["fmt"], nb, nkv, bs, hd, c["bounds"]))
        cu = torch.zeros(c["seqs"] + 1, dtype=torch.int32)
        cu[1:] = lens.cumsum(0)
        n = int(cu[-1])
        s["cu_q"], s["q_start"] = cu.to(DEV), start.to(torch.int32).to(DEV)
        s["one_each"] = c["q_hi"] == 1
        kv = _randn(g, n, 2 * nkv * hd)
        kv *= torch.exp(0.5 * _randn(g, n, 1))                 # rows of different strength
        s["key"], s["value"] = kv.to(torch.bfloat16).view(n, 2, nkv, hd).unbind(1)
    elif c["op"] in ("decode", "pages"):
        lens = _ints(gen, c["users"], c["ctx_lo"], c["ctx_hi"])
        s["page_table"], nb = _page_table(gen, lens.tolist(), bs)
        s["cur_pos"] = (lens - 1).to(torch.int32).to(DEV)
        s.update(_pool(g, c["fmt"], nb, nkv, bs, hd, c["op"] == "pages"))
        s["query"] = _randn(g, c["users"], c["nq"], hd).to(torch.bfloat16)
        s["sinks"] = _randn(g, c["nq"]) if c.get("sinks") else None
        s["max_len"] = int(lens.max())
    else:
        lens, start = _spread(gen, c["seqs"], (c["q_lo"], c["q_hi"]),
                              (c["start_lo"], c["start_hi"]))
        s["page_table"], nb = _page_table(gen, (lens + start).tolist(), bs)
        s.update(_pool(g, c["fmt"], nb, nkv, bs, hd, False))
        cu = torch.zeros(c["seqs"] + 1, dtype=torch.int32)
        cu[1:] = lens.cumsum(0)
        s["cu_host"], s["cu_q"] = cu, cu.to(DEV)
        s["q_start"] = start.to(torch.int32).to(DEV)
        s["query"] = _randn(g, int(cu[-1]), c["nq"], hd).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------- passes
def _values(cache, scale):
    """What the codes of an 8-bit cache stand for."""
    if cache.dtype == torch.bfloat16:
        return cache
    codes = cache.float() if cache.dtype == torch.float8_e4m3fn else cache
    return codes * scale[:, :, None, None]


def _context(s, width):
    """Keys and values of the users' first `width` pages: [users, nkv, width * bs, hd], 32 bits."""
    pages = s["page_table"][:, :width].long()
    got = []
    for which in "kv":
        x = s[which + "_cache"][pages].float()                  # [users, pages, nkv, bs, hd]
        if which + "_scale" in s:
            x = x * s[which + "_scale"][pages][..., None, None]
        got.append(x.transpose(1, 2).flatten(2, 3))
    return got


def _attend(q, k, v, mask, sinks, out_type):
    """softmax(q k / sqrt(hd)) v with `mask` true where a key is attended: q [u, h, g, hd]; a row
    whose mask leaves nothing is zero."""
    logits = (q @ k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    logits = logits.masked_fill(~mask, -math.inf)
    top = logits.amax(-1, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks)
    top = top.clamp_min(torch.finfo(top.dtype).min)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    return ((p @ v) / total.clamp_min(1e-30)).to(out_type)


def _plain_norm_rope(s):
    c = s["case"]
    hd, r, t = c["hd"], c["rotary"], c["tokens"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    got = []
    for name in ("query", "key"):
        x = s[name].reshape(t, -1, hd).float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s[name[0] + "_weight"].float()
        if c["neox"]:
            a, b = x[..., : r // 2], x[..., r // 2: r]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
        else:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2),
                           x[..., r:]], -1)
        got.append(y.to(torch.bfloat16))
    slots = s["slots"].clamp_min(0)
    blk, off = slots // c["bs"], slots % c["bs"]
    keep = (s["slots"] >= 0)[:, None, None]
    for cache, new in (("k_cache", got[1]), ("v_cache", s["value"].reshape(t, -1, hd))):
        x = s[cache]
        if x.dtype != torch.bfloat16:
            new = new.float().clamp(-448.0, 448.0).to(x.dtype)
            x, new = x.view(torch.uint8), new.view(torch.uint8)
        # a padding row goes to a row that is thrown away
        grown = torch.cat([x.transpose(1, 2).flatten(0, 1), x.new_zeros(1, *new.shape[1:])])
        grown[torch.where(keep[:, 0, 0], blk * c["bs"] + off, grown.shape[0] - 1)] = new
        x.copy_(grown[:-1].view(x.shape[0], x.shape[2], x.shape[1], hd).transpose(1, 2))
    return got[0].flatten(1), got[1].flatten(1), s["k_cache"], s["v_cache"]


def _rows_of(s):
    """Of every new token: its page and its offset in the page."""
    bs, n = s["case"]["bs"], s["key"].shape[0]
    t = torch.arange(n, device=s["key"].device)
    seq = torch.searchsorted(s["cu_q"][1:].long(), t, right=True)
    pos = s["q_start"].long()[seq] + t - s["cu_q"].long()[seq]
    return s["page_table"].long()[seq, pos // bs], pos % bs


def _plain_write(s):
    c = s["case"]
    nkv, bs, hd = c["nkv"], c["bs"], c["hd"]
    page, off = _rows_of(s)
    nb = s["k_cache"].shape[0]
    dev = page.device
    first = torch.full((nb,), bs, device=dev).scatter_reduce_(0, page, off, "amin")
    fresh, touched = (first == 0)[:, None], (first < bs)[:, None]
    got = []
    for which, new in (("k", s["key"]), ("v", s["value"])):
        cache = s[which + "_cache"]
        if c["fmt"] == "bf16":
            cache[page, :, off] = new
            continue
        qmax, scale = QMAX[c["fmt"]], s[which + "_scale"]
        top = new.float().abs().amax(-1)                                    # [tokens, nkv]
        need = torch.zeros(nb, nkv, device=dev).scatter_reduce_(
            0, page[:, None].expand(-1, nkv), top, "amax") / qmax
        # a page that goes on keeps its scale, or grows it by the smallest power of two that is enough
        (ms, es), (mn, en) = torch.frexp(scale), torch.frexp(need)
        up = (en - es + (mn > ms)).clamp_min(0)
        kept = torch.where(scale > 0, torch.ldexp(scale, torch.where(need > scale, up, 0)), need)
        now = torch.where(touched, torch.where(fresh, need, kept), scale)
        shrink = torch.where(touched & ~fresh & (scale > 0), scale / now.clamp_min(1e-45), 1.0)
        old = (torch.arange(bs, device=dev) < first[:, None])[:, None, :, None]   # rows that stay
        codes = cache.float()
        less = codes * shrink[:, :, None, None]
        less = less.round() if c["fmt"] == "int8" else less.to(cache.dtype).float()
        codes = torch.where(old & (shrink < 1)[:, :, None, None], less, codes)
        row = now[page][..., None]
        q = torch.where(row > 0, new.float() / row, 0.0).clamp(-qmax, qmax)
        codes[page, :, off] = q.round() if c["fmt"] == "int8" else q
        cache.copy_(codes.to(cache.dtype))
        scale.copy_(now)
    if c["bounds"]:
        b = s["k_bounds"]
        at = page[:, None, None].expand(-1, nkv, hd)
        for i, how, none in ((0, "amin", math.inf), (1, "amax", -math.inf)):
            seen = torch.full((nb, nkv, hd), none, device=dev).scatter_reduce_(
                0, at, s["key"].float(), how)
            was = b[:, :, i].float()
            both = torch.minimum(was, seen) if how == "amin" else torch.maximum(was, seen)
            b[:, :, i] = torch.where(touched[..., None], torch.where(fresh[..., None], seen, both),
                                     was).to(b.dtype)
        got = [b]
    return _written(s) + got


def _written(s):
    if s["case"]["fmt"] == "bf16":
        return [s["k_cache"], s["v_cache"]]
    return [_values(s["k_cache"], s["k_scale"]), _values(s["v_cache"], s["v_scale"]),
            s["k_scale"], s["v_scale"]]


def _plain_decode(s):
    c = s["case"]
    u, nkv, hd = c["users"], c["nkv"], c["hd"]
    k, v = _context(s, (s["max_len"] + c["bs"] - 1) // c["bs"])
    j = torch.arange(k.shape[2], device=k.device)
    pos = s["cur_pos"].long()[:, None]
    mask = j <= pos
    if c["window"]:
        mask = mask & (j > pos - c["window"])
    q = s["query"].float().view(u, nkv, -1, hd)
    sinks = None if s["sinks"] is None else s["sinks"].view(nkv, -1, 1)
    return _attend(q, k, v, mask[:, None, None], sinks, torch.bfloat16).view(u, c["nq"], hd)


def _plain_prefill(s):
    c = s["case"]
    nkv, hd, n = c["nkv"], c["hd"], s["query"].shape[0]
    k, v = _context(s, s["page_table"].shape[1])
    t = torch.arange(n, device=k.device)
    seq = torch.searchsorted(s["cu_q"][1:].long(), t, right=True)
    row = t - s["cu_q"].long()[seq]
    # rows of every sequence side by side: [seqs, longest, nq, hd]
    q = k.new_zeros(c["seqs"], c["q_hi"], c["nq"], hd)
    q[seq, row] = s["query"].float()
    at = s["q_start"].long()[:, None] + torch.arange(c["q_hi"], device=k.device)
    mask = torch.arange(k.shape[2], device=k.device) <= at[..., None]       # [seqs, rows, keys]
    group = c["nq"] // nkv
    q = q.transpose(1, 2).reshape(c["seqs"], nkv, group * c["q_hi"], hd)
    mask = mask.repeat(1, group, 1)[:, None]
    out = _attend(q, k, v, mask, None, torch.bfloat16)
    out = out.view(c["seqs"], c["nq"], c["q_hi"], hd).transpose(1, 2)
    return out[seq, row]


def _plain_pages(s):
    c = s["case"]
    u, nkv, hd, bs, want = c["users"], c["nkv"], c["hd"], c["bs"], c["pages"]
    width = (s["max_len"] + bs - 1) // bs
    pages = s["page_table"][:, :width].long()
    n = (s["cur_pos"].long() + bs) // bs                                    # [users] pages in use
    # in 64 bits: which page is the last one in is decided between scores that may be near
    b = s["k_bounds"][pages].double().transpose(1, 2)                       # [u, nkv, p, 2, hd]
    q = s["query"].double().view(u, nkv, -1, hd)
    score = q.clamp_max(0) @ b[..., 0, :].transpose(-1, -2) + \
        q.clamp_min(0) @ b[..., 1, :].transpose(-1, -2)                     # [u, nkv, g, p]
    score = score.amax(2)
    p = torch.arange(width, device=score.device)
    forced = (p < c["first"]) | (p >= (n - c["last"])[:, None])
    score = score.masked_fill(forced[:, None], math.inf)
    score = score.masked_fill((p >= n[:, None])[:, None], -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :want]
    count = n.clamp_max(want)[:, None, None]
    slot = torch.arange(order.shape[-1], device=order.device)
    order = torch.where(slot < count, order, width).sort(-1).values
    used = order < width
    ids = s["page_table"].long()[:, None].expand(-1, nkv, -1).gather(
        -1, order.clamp_max(width - 1))
    table = torch.zeros(u, nkv, want, dtype=torch.int32, device=order.device)
    table[..., : ids.shape[-1]] = torch.where(used, ids, 0).int()
    pos = (count[..., 0] - 1) * bs + s["cur_pos"].long()[:, None] % bs
    head = torch.arange(nkv, device=order.device)[:, None]
    got = []
    for which in "kv":
        x = s[which + "_cache"][ids, head].float()                          # [u, nkv, want, bs, hd]
        if which + "_scale" in s:
            x = x * s[which + "_scale"][ids, head][..., None, None]
        got.append(x.flatten(2, 3))
    mask = torch.arange(got[0].shape[2], device=order.device) <= pos[..., None]
    out = _attend(q.float(), got[0], got[1], mask[:, :, None], None, torch.bfloat16)
    return out.view(u, c["nq"], hd), table, pos.expand(-1, nkv).int()


def _own_norm_rope(s):
    c = s["case"]
    q, k = _ops().qk_norm_rope_kv_scatter_slots(
        s["query"], s["key"], s["value"], s["positions"], s["inv_freq"], c["rotary"], c["hd"],
        s["q_weight"], s["k_weight"], EPS, s["k_cache"], s["v_cache"], s["slots"],
        is_neox_style=c["neox"], out_query=s["out_query"], out_key=s["out_key"])
    return q, k, s["k_cache"], s["v_cache"]


def _own_write(s):
    _ops().paged_write(s["k_cache"], s["v_cache"], s["key"], s["value"], s["page_table"],
                       s["q_start"], cu_q=None if s["one_each"] else s["cu_q"],
                       k_scale=s.get("k_scale"), v_scale=s.get("v_scale"),
                       k_bounds=s.get("k_bounds"))
    return _written(s) + ([s["k_bounds"]] if s["case"]["bounds"] else [])


def _own_decode(s):
    return _ops().paged_decode(s["query"], s["k_cache"], s["v_cache"], s["page_table"],
                               s["cur_pos"], max_context_len=s["max_len"],
                               sliding_window=s["case"]["window"], sinks=s["sinks"],
                               k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_prefill(s):
    return _ops().prefill(s["query"], s["k_cache"], s["v_cache"], s["cu_host"],
                          page_table=s["page_table"], q_start=s["q_start"], cu_q=s["cu_q"],
                          k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_pages(s):
    c, ops = s["case"], _ops()
    table, pos = ops.select_pages(s["query"], s["k_bounds"], s["page_table"], s["cur_pos"],
                                  c["bs"], c["pages"], keep_first=c["first"],
                                  keep_last=c["last"], max_context_len=s["max_len"])
    out = ops.paged_decode(s["query"], s["k_cache"], s["v_cache"], table, pos,
                           k_scale=s.get("k_scale"), v_scale=s.get("v_scale"))
    return out, table, pos


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm_rope": _own_norm_rope, "write": _own_write, "decode": _own_decode,
                "prefill": _own_prefill, "pages": _own_pages}[op](state)
    return {"norm_rope": _plain_norm_rope, "write": _plain_write, "decode": _plain_decode,
            "prefill": _plain_prefill, "pages": _plain_pages}[op](state)


# --------------------------------------------------------------------------------------- work
def work(case):
    c = case
    nkv, hd, bs = c["nkv"], c["hd"], c["bs"]
    if c["op"] == "norm_rope":
        t, nq = c["tokens"], c["nq"]
        row = (nq + nkv) * hd
        cache = 2 * nkv * hd * (2 if c["cache"] == "bf16" else 1)
        return dict(bytes=t * (2 * (row + nkv * hd) + 2 * row + cache + 16), flops=8 * t * row)
    if c["op"] == "write":
        t = c["seqs"] * (c["q_lo"] + c["q_hi"]) / 2
        pages = c["seqs"] * ((c["start_hi"] / 2 + t / c["seqs"]) / bs + 1)
        if c["fmt"] == "bf16":
            total = t * nkv * hd * 8
        else:                      # codes written, and the values that come back
            total = t * nkv * hd * 6 + pages * bs * nkv * hd * 2 * 5
        return dict(bytes=total + (pages * nkv * hd * 8 if c["bounds"] else 0),
                    flops=4 * t * nkv * hd)
    size = 2 if c["fmt"] == "bf16" else 1
    if c["op"] == "decode":
        ctx = (c["ctx_lo"] + c["ctx_hi"]) / 2
        ctx = min(ctx, c["window"]) if c["window"] else ctx
        keys = c["users"] * ctx
        return dict(bytes=2 * keys * nkv * hd + 8 * keys * nkv / bs + 4 * c["users"] * c["nq"] * hd,
                    flops=4 * keys * c["nq"] * hd)
    if c["op"] == "prefill":
        q, start = (c["q_lo"] + c["q_hi"]) / 2, (c["start_lo"] + c["start_hi"]) / 2
        keys = start + q / 2
        return dict(bytes=c["seqs"] * (2 * (start + q) * nkv * hd + 4 * q * c["nq"] * hd),
                    flops=4 * c["seqs"] * q * keys * c["nq"] * hd)
    ctx = (c["ctx_lo"] + c["ctx_hi"]) / 2
    near = min(ctx, c["pages"] * bs)
    return dict(bytes=c["users"] * (ctx / bs * nkv * hd * 4 + 2 * near * nkv * hd * size
                                    + 4 * c["nq"] * hd + 4 * nkv * c["pages"]),
                flops=c["users"] * c["nq"] * hd * (4 * ctx / bs + 4 * near))


# -------------------------------------------------------------------------------------- exact
def _exact_row(q, k, v, sink=None):
    """Attention of the rows q [g, hd] over k, v [keys, hd], all in 64 bits."""
    if not k.shape[0]:
        return torch.zeros_like(q)
    w = torch.einsum("gd,jd->gj", q, k) / math.sqrt(q.shape[-1])
    if sink is not None:
        w = torch.cat([w, sink[:, None]], 1)
        v = torch.cat([v, torch.zeros_like(v[:1])])
    return torch.einsum("gj,jd->gd", torch.softmax(w, -1), v)


def _exact_page_values(s, which, ids, head):
    x = s[which + "_cache"][ids, head].double()
    if which + "_scale" in s:
        x = x * s[which + "_scale"][ids, head].double()[:, None, None]
    return x.reshape(-1, x.shape[-1])


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "write": _exact_write, "decode": _exact_decode,
            "prefill": _exact_prefill, "pages": _exact_pages}[case["op"]](s)


def _exact_norm_rope(s):
    c = s["case"]
    t, hd, r, bs = c["tokens"], c["hd"], c["rotary"], c["bs"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       s["positions"].double()[:, None] * s["inv_freq"].double()[None])
    done = {}
    for name, weight in (("query", "q_weight"), ("key", "k_weight")):
        x = s[name].double().reshape(t, -1, hd)
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * s[weight].double()
        i = torch.arange(r // 2, device=DEV)
        a, b = (i, i + r // 2) if c["neox"] else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., a], x[..., b]) * turn[:, None]
        x[..., a], x[..., b] = z.real, z.imag
        done[name] = x
    caches = []
    live = (s["slots"] >= 0).nonzero()[:, 0]
    for new in (done["key"], s["value"].double().reshape(t, -1, hd)):
        x = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device=DEV)
        at = s["slots"][live]
        x[at // bs, :, at % bs] = new[live].clamp(-448, 448) if c["cache"] != "bf16" else new[live]
        caches.append(x)
    return [done["query"].reshape(t, -1), done["key"].reshape(t, -1)] + caches


def _exact_write(s):
    """The scales by their rule; a row's value is the row's own (what quantising loses is a choice
    of the format and has no exact value, so the values are left out)."""
    c = s["case"]
    bs, page_table = c["bs"], s["page_table"].tolist()
    cu, start = s["cu_q"].tolist(), s["q_start"].tolist()
    out = []
    scales = {w: s[w + "_scale"].double() for w in "kv"} if c["fmt"] != "bf16" else {}
    bounds = s["k_bounds"].double() if c["bounds"] else None
    caches = {w: s[w + "_cache"].clone() for w in "kv"} if c["fmt"] == "bf16" else {}
    if sum(-(-(b - a) // bs) + 1 for a, b in zip(cu, cu[1:])) > 4096:
        return None
    for i in range(c["seqs"]):
        lo = start[i]
        end = lo + cu[i + 1] - cu[i]
        while lo < end:
            blk, fresh, hi = page_table[i][lo // bs], lo % bs == 0, min(end, lo // bs * bs + bs)
            a = cu[i] + lo - start[i]
            for which, new in (("k", s["key"]), ("v", s["value"])):
                rows = new[a:a + hi - lo]
                if caches:
                    caches[which][blk, :, lo % bs: lo % bs + hi - lo] = rows.transpose(0, 1)
                    continue
                need = rows.double().abs().amax((0, 2)) / QMAX[c["fmt"]]
                was = scales[which][blk]
                # the rule compares in 32 bits
                steps = torch.ceil(torch.log2((need.float().double() / was).clamp_min(1e-300)))
                grown = was * 2.0 ** steps.clamp_min(0)
                scales[which][blk] = need if fresh else torch.where(was > 0, grown, need)
            if bounds is not None:
                rows = s["key"][a:a + hi - lo].double()
                least, most = rows.amin(0), rows.amax(0)
                if not fresh:
                    least = torch.minimum(least, bounds[blk, :, 0])
                    most = torch.maximum(most, bounds[blk, :, 1])
                bounds[blk, :, 0], bounds[blk, :, 1] = least, most
            lo = hi
    out = [caches["k"].double(), caches["v"].double()] if caches else \
        [None, None, scales["k"], scales["v"]]
    return out + ([bounds] if bounds is not None else [])


def _exact_decode(s):
    c = s["case"]
    group, out = c["nq"] // c["nkv"], torch.zeros(c["users"], c["nq"], c["hd"], dtype=torch.float64,
                                                  device=DEV)
    for u, last in enumerate(s["cur_pos"].tolist()):
        ids = s["page_table"][u, : last // c["bs"] + 1].long()
        a = max(0, last + 1 - c["window"]) if c["window"] else 0
        for h in range(c["nkv"]):
            k = _exact_page_values(s, "k", ids, h)[a:last + 1]
            v = _exact_page_values(s, "v", ids, h)[a:last + 1]
            mine = slice(h * group, (h + 1) * group)
            sink = None if s["sinks"] is None else s["sinks"][mine].double()
            out[u, mine] = _exact_row(s["query"][u, mine].double(), k, v, sink)
    return out


def _exact_prefill(s):
    c = s["case"]
    group, out = c["nq"] // c["nkv"], torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    cu = s["cu_host"].tolist()
    for i, start in enumerate(s["q_start"].tolist()):
        rows = cu[i + 1] - cu[i]
        ids = s["page_table"][i, : (start + rows + c["bs"] - 1) // c["bs"]].long()
        ahead = torch.ones(rows, start + rows, dtype=torch.bool, device=DEV).triu(start + 1)
        for h in range(c["nkv"]):
            k = _exact_page_values(s, "k", ids, h)[: start + rows]
            v = _exact_page_values(s, "v", ids, h)[: start + rows]
            for q in range(h * group, (h + 1) * group):
                w = s["query"][cu[i]:cu[i + 1], q].double() @ k.T / math.sqrt(c["hd"])
                out[cu[i]:cu[i + 1], q] = torch.softmax(w.masked_fill(ahead, -math.inf), -1) @ v
    return out


def _exact_pages(s):
    c = s["case"]
    group, bs = c["nq"] // c["nkv"], c["bs"]
    out = torch.zeros(c["users"], c["nq"], c["hd"], dtype=torch.float64, device=DEV)
    for u, last in enumerate(s["cur_pos"].tolist()):
        n = last // bs + 1
        ids = s["page_table"][u, :n].long()
        for h in range(c["nkv"]):
            mine = slice(h * group, (h + 1) * group)
            q = s["query"][u, mine].double()
            chosen = torch.arange(n, device=DEV)
            if n > c["pages"]:
                b = s["k_bounds"][ids, h].double()
                most = torch.maximum(q[:, None] * b[None, :, 0], q[:, None] * b[None, :, 1])
                score = most.sum(-1).amax(0)
                score[: c["first"]] = math.inf
                score[n - c["last"]:] = math.inf
                chosen = score.sort(dim=0, descending=True, stable=True).indices[: c["pages"]]
                chosen = chosen.sort().values
            at = (chosen[:, None] * bs + torch.arange(bs, device=DEV)).flatten() <= last
            k = _exact_page_values(s, "k", ids[chosen], h)[at]
            v = _exact_page_values(s, "v", ids[chosen], h)[at]
            out[u, mine] = _exact_row(q, k, v)
    return [out, None, None]
