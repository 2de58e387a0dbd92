"""Random shapes, lengths, strides and options of the cache-side operators against the plain
restatements; small, so that every case is compared in full."""
import random

import pytest
import torch

from oracle import blocks

pytestmark = pytest.mark.gpu


def _heads(r):
    nkv = r.choice([1, 2, 3, 4])
    group = r.randrange(1, 17)
    return nkv * group, nkv, r.choice([64, 128]), r.choice([32, 64])


def _cache(r, nb, nkv, bs, hd, kind, g):
    c = {}
    for w in "kv":
        x = torch.randn(nb, nkv, bs, hd, generator=g)
        if kind == torch.bfloat16:
            c[w + "_cache"], c[w + "_scale"] = x.bfloat16(), None
            continue
        scale = x.abs().amax((2, 3)) / blocks.QMAX[kind].item()
        q = x / scale[:, :, None, None]
        c[w + "_cache"] = (q.round() if kind == torch.int8 else q).to(kind)
        c[w + "_scale"] = scale * torch.exp2(torch.randint(-6, 7, scale.shape, generator=g).float())
    return c


@pytest.mark.parametrize("seed", range(30))
def test_decode(clean_error_word, seed):
    from b200attn import ops

    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    nq, nkv, hd, bs = _heads(r)
    kind = r.choice([torch.int8, torch.float8_e4m3fn])
    lists = r.random() < 0.4
    users = r.randrange(1, 7)
    shape = (users, nkv) if lists else (users,)
    ctx = torch.randint(0, r.choice([5, 130, 700]), shape, generator=g)
    ctx[torch.rand(shape, generator=g) < 0.15] = 0
    width = max(1, (int(ctx.max()) + bs - 1) // bs) + r.randrange(0, 3)
    nb = r.randrange(1, 40)
    table = torch.randint(0, nb, shape + (width,), generator=g).int()      # shared pages
    c = _cache(r, nb, nkv, bs, hd, kind, g)
    q = torch.randn(users, nq, hd, generator=g).bfloat16() * r.choice([0.1, 1.0, 4.0])
    window = 0 if lists else r.choice([0, 0, 1, 50, 200])
    sinks = torch.randn(nq, generator=g) if r.random() < 0.4 else None
    scale = r.choice([None, 0.3])
    pos = (ctx - 1).int()
    wide = torch.full(shape + (width + 5,), -7, dtype=torch.int32)         # strided rows
    wide[..., 2:2 + width] = table
    got = ops.paged_decode(
        q.cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), wide.cuda()[..., 2:2 + width],
        pos.cuda(), scale=scale, num_splits=r.choice([0, 0, 1, 2, 7]),
        max_context_len=r.choice([0, 64, 5000]), sliding_window=window,
        sinks=None if sinks is None else sinks.cuda(), k_scale=c["k_scale"].cuda(),
        v_scale=c["v_scale"].cuda()).cpu().double()
    args = dict(scale=scale, k_scale=c["k_scale"], v_scale=c["v_scale"], window=window, sinks=sinks)
    want = blocks.decode(q, c["k_cache"], c["v_cache"], table, pos, **args)
    size = blocks.decode(q, c["k_cache"], c["v_cache"].float().abs(), table, pos, **args)
    # scores: fp32 sums of q.k are off by up to hd 2^-23 of the sum of magnitudes, a weight by as
    # much again relative; 2^-11 for its rounding
    mag = q.float().abs().reshape(users, nkv, -1, hd).amax((2, 3)).max() * hd * 130
    top = float((c["k_scale"].max() * mag * (hd ** -0.5 if scale is None else scale)))
    # f16 weights have a smallest step of 2^-24 of the largest weight times V scale: where the keys
    # that carry a row have a value of exactly zero, what is left is the others' rounding, at most
    # half a step each times the largest |v|
    v_max = float((c["v_cache"].float().abs().amax((2, 3)) * c["v_scale"]).max())
    floor = int(ctx.max()) * 2.0 ** -25 * v_max
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -10 + 2 * top * hd * 2.0 ** -24) * size + floor
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("seed", range(30))
def test_write(clean_error_word, seed):
    from b200attn import ops

    r, g = random.Random(seed), torch.Generator().manual_seed(100 + seed)
    _, nkv, hd, bs = _heads(r)
    kind = r.choice([torch.int8, torch.float8_e4m3fn, torch.bfloat16])
    seqs = r.randrange(1, 40)
    lens = torch.randint(0, r.choice([2, 9, 150]), (seqs,), generator=g)
    start = torch.randint(-1, r.choice([3, 70, 300]), (seqs,), generator=g)
    need = torch.where(start >= 0, (start + lens + bs - 1) // bs, 0).tolist()
    nb = sum(need) + 1
    perm = torch.randperm(nb, generator=g).int()
    table = torch.full((seqs, max(need) + 1), nb + 3, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    c = _cache(r, nb, nkv, bs, hd, kind, g)
    bounds = torch.randn(nb, nkv, 2, hd, generator=g).sort(dim=2).values.bfloat16() \
        if kind == torch.bfloat16 or r.random() < 0.5 else None
    cu = torch.cat([torch.zeros(1), lens.cumsum(0)]).int()
    rows = int(cu[-1]) + r.randrange(0, 3)
    if rows == 0:
        pytest.skip("no rows")
    kv = torch.randn(rows, 2 * nkv * hd + 8, generator=g) * \
        torch.exp2(torch.randint(-6, 7, (rows, 1), generator=g).float())
    kv = kv.bfloat16()
    key, value = kv[:, : nkv * hd], kv[:, nkv * hd: 2 * nkv * hd]
    qlen = torch.randint(-1, 160, (seqs,), generator=g).int() if r.random() < 0.5 else None
    host = {n: t.clone() for n, t in dict(c, k_bounds=bounds).items() if t is not None}
    dev = {n: t.cuda() for n, t in host.items()}
    dkv = kv.cuda()
    extra = ("k_scale", "v_scale", "k_bounds")
    ops.paged_write(dev["k_cache"], dev["v_cache"], dkv[:, : nkv * hd],
                    dkv[:, nkv * hd: 2 * nkv * hd], table.cuda(), start.int().cuda(),
                    cu_q=cu.cuda(), q_len=None if qlen is None else qlen.cuda(),
                    **{n: dev[n] for n in extra if n in dev})
    blocks.paged_write(host["k_cache"], host["v_cache"], key.reshape(rows, nkv, hd),
                       value.reshape(rows, nkv, hd), table, start.int(), cu, qlen,
                       **{n: host[n] for n in extra if n in host})
    for n in host:
        assert torch.equal(dev[n].cpu().float(), host[n].float()), n


@pytest.mark.parametrize("seed", range(30))
def test_select(clean_error_word, seed):
    from b200attn import ops

    r, g = random.Random(seed), torch.Generator().manual_seed(200 + seed)
    nq, nkv, hd, bs = _heads(r)
    users = r.randrange(1, 6)
    ctx = torch.randint(0, r.choice([60, 3000, 30000]), (users,), generator=g)
    width = max(1, (int(ctx.max()) + bs - 1) // bs) + r.randrange(0, 3)
    nb = r.randrange(1, 700)
    table = torch.randint(0, nb, (users, width), generator=g).int()        # shared pages: ties
    bounds = torch.randn(nb, nkv, 2, hd, generator=g).sort(dim=2).values.bfloat16()
    q = torch.randn(users, nq, hd, generator=g).bfloat16()
    first, last = r.randrange(0, 4), r.randrange(1, 4)
    k = first + last + r.randrange(0, 60)
    pos = (ctx - 1).int()
    got_t, got_p = ops.select_pages(q.cuda(), bounds.cuda(), table.cuda(), pos.cuda(), bs, k, first,
                                    last, max_context_len=r.choice([0, 100, 1 << 17]))
    want_t, want_p = blocks.select_pages(q, bounds, table, pos, bs, k, first, last)
    assert torch.equal(got_p.cpu(), want_p) and torch.equal(got_t.cpu(), want_t)


@pytest.mark.parametrize("seed", range(20))
def test_norm_rope(clean_error_word, seed):
    from b200attn import ops

    r, g = random.Random(seed), torch.Generator().manual_seed(300 + seed)
    nq, nkv, hd, bs = _heads(r)
    tokens = r.randrange(1, 70)
    rotary = 16 * r.randrange(1, hd // 16 + 1)
    neox = r.random() < 0.6
    x = (torch.randn(tokens, (nq + nkv) * hd, generator=g) * 3).bfloat16()
    pos = torch.randint(-5, 1 << r.randrange(4, 31), (tokens,), generator=g)
    inv = 1.0 / 10000.0 ** (torch.arange(0, rotary, 2).float() / rotary)
    w = [torch.randn(hd, generator=g).to(r.choice([torch.float32])) for _ in range(2)]
    eps = r.choice([0.0, 1e-6, 1e-2])
    d = x.cuda()
    rq, rk = ops.qk_norm_rope_kv_scatter_slots(
        d[:, : nq * hd], d[:, nq * hd:], None, pos.cuda(), inv.cuda(), rotary, hd, w[0].cuda(),
        w[1].cuda(), eps, is_neox_style=neox)
    for got, y, weight in ((rq, x[:, : nq * hd], w[0]), (rk, x[:, nq * hd:], w[1])):
        want = blocks.qk_norm_rope(y, pos, inv, rotary, hd, weight, eps, neox).reshape(-1, hd)
        top = want.abs().amax(-1, keepdim=True)
        err = (got.double().cpu().reshape(-1, hd) - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * top).all()
