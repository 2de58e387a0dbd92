"""Block-scaled 8-bit KV cache: the write bit for bit, attention over it against fp64."""
import math

import pytest
import torch

from oracle import blocks

pytestmark = pytest.mark.gpu

KINDS = [torch.int8, torch.float8_e4m3fn]


def _bits(t):
    return t.cpu().view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.cpu()


def _same(a, b):
    """Equal values, -0 = +0 for e4m3, NaN equal to NaN."""
    a, b = a.cpu().float(), b.cpu().float()
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def _filled(nb, nkv, bs, hd, kind, seed):
    """A cache whose every page was written from its first row on."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for which in "kv":
        x = torch.randn(nb, nkv, bs, hd, generator=g)
        scale = x.abs().amax((2, 3)) / blocks.QMAX[kind].item()
        q = x / scale[:, :, None, None]
        out[which + "_cache"] = (q.round() if kind == torch.int8 else q).to(kind)
        out[which + "_scale"] = scale
    out["k_bounds"] = torch.randn(nb, nkv, 2, hd, generator=g).sort(dim=2).values.bfloat16()
    return out


def _run_write(state, key, value, table, start, cu=None, qlen=None, bounds=True):
    from b200attn import ops

    dev = {n: t.cuda() for n, t in state.items()}
    host = {n: t.clone() for n, t in state.items()}
    if not bounds:
        dev.pop("k_bounds"), host.pop("k_bounds")
    args = [key, value, table, start]
    ops.paged_write(dev["k_cache"], dev["v_cache"], *[a.cuda() for a in args],
                    cu_q=None if cu is None else cu.cuda(),
                    q_len=None if qlen is None else qlen.cuda(),
                    **{n: dev[n] for n in ("k_scale", "v_scale", "k_bounds") if n in dev})
    blocks.paged_write(host["k_cache"], host["v_cache"], *args, cu_q=cu, q_len=qlen,
                       **{n: host[n] for n in ("k_scale", "v_scale", "k_bounds") if n in host})
    return dev, host


def _check(dev, host):
    for n in host:
        assert _same(dev[n], host[n]), n


@pytest.mark.parametrize("kind", KINDS + [torch.bfloat16])
@pytest.mark.parametrize("hd,bs,nkv", [(64, 32, 1), (64, 64, 3), (128, 32, 2), (128, 64, 8)])
@pytest.mark.parametrize("lens,starts", [
    ([1], [0]), ([1, 1, 1], [0, 31, 64]), ([5, 0, 64, 130, 2], [0, 9, 64, 33, 63]),
    ([200, 1, 31, 32, 33, 63, 64, 65], [0, 0, 1, 32, 31, 1, 0, 7]),
])
def test_write_matches_the_plain_write(clean_error_word, kind, hd, bs, nkv, lens, starts):
    g = torch.Generator().manual_seed(sum(lens) + hd)
    need = [(a + b + bs - 1) // bs for a, b in zip(lens, starts)]
    nb = sum(need) + 1
    perm = torch.randperm(nb, generator=g).int()
    table = torch.zeros(len(lens), max(need) + 1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    if kind == torch.bfloat16:
        state = _filled(nb, nkv, bs, hd, torch.int8, 1)
        state = dict(k_cache=state["k_cache"].bfloat16(), v_cache=state["v_cache"].bfloat16(),
                     k_bounds=state["k_bounds"])
    else:
        state = _filled(nb, nkv, bs, hd, kind, 1)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    n = int(cu[-1])
    # rows of very different strength, so that pages that go on grow their scales
    kv = torch.randn(n, 2, nkv, hd, generator=g) * torch.exp2(torch.randint(-3, 6, (n, 2, nkv, 1),
                                                                           generator=g).float())
    kv = kv.bfloat16()
    dev, host = _run_write(state, kv[:, 0], kv[:, 1], table, torch.tensor(starts).int(), cu)
    _check(dev, host)


@pytest.mark.parametrize("kind", KINDS)
def test_appending_token_by_token_stays_within_a_step(clean_error_word, kind):
    """A page filled one token at a time: the same bits as the plain write after every step, and
    every value within what the format and the re-roundings allow."""
    from b200attn import ops

    g = torch.Generator().manual_seed(9)
    bs, hd, nkv, users = 32, 64, 2, 3
    rows = (torch.randn(bs, users, 2, nkv, hd, generator=g) *
            torch.linspace(0.2, 6.0, bs)[:, None, None, None, None]).bfloat16()
    dev = {n: t.cuda() for n, t in _filled(4, nkv, bs, hd, kind, 2).items()}
    host = {n: t.cpu().clone() for n, t in dev.items()}
    table = torch.tensor([[2], [0], [3]], dtype=torch.int32)
    for i in range(bs):
        pos = torch.full((users,), i, dtype=torch.int32)
        k, v = rows[i, :, 0], rows[i, :, 1]
        names = ("k_scale", "v_scale", "k_bounds")
        ops.paged_write(dev["k_cache"], dev["v_cache"], k.cuda(), v.cuda(), table.cuda(),
                        pos.cuda(), **{n: dev[n] for n in names})
        blocks.paged_write(host["k_cache"], host["v_cache"], k, v, table, pos,
                           **{n: host[n] for n in names})
    _check(dev, host)
    for u in range(users):
        for h in range(nkv):
            blk = int(table[u, 0])
            scale = dev["k_scale"][blk, h].item()
            got = dev["k_cache"][blk, h].float().cpu() * scale
            err = (got - rows[:, u, 0, h].float()).abs()
            if kind == torch.int8:      # half a step at first, then at most s/2 + s/4 + ... + s/2
                assert (err <= scale * 1.0001).all()
            else:                       # 2^-4 relative, or a subnormal's steps as above
                x = rows[:, u, 0, h].float().abs()
                assert (err <= torch.maximum(x * 2.0 ** -4, torch.tensor(scale * 2.0 ** -9 * 1.001))).all()


@pytest.mark.parametrize("kind", KINDS)
def test_write_special_values(clean_error_word, kind):
    """Zero rows, tiny and huge rows, NaN and infinities: scales and codes as documented."""
    bs, hd, nkv = 32, 64, 1
    state = _filled(8, nkv, bs, hd, kind, 3)
    state["k_scale"][2] = 0.0
    state["k_cache"][2] = torch.zeros(1).to(kind)
    state["k_scale"][3] = float("nan")
    state["k_scale"][6] = 1e-30
    n = 8
    kv = torch.randn(n, 2, nkv, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    kv[0] = 0.0                              # fresh, all zero
    kv[1, :, :, 3] = float("inf")            # fresh, not finite
    kv[4, 0, 0, 0] = float("nan")            # goes on, not finite
    kv[5] *= 1e-38                           # fresh, subnormal scale
    kv[6] = 3e38                             # goes on with a scale far too small
    kv[7] *= 1e-30                           # goes on with a scale far larger than needed
    start = torch.tensor([0, 0, 5, 5, 7, 0, 9, 31], dtype=torch.int32)
    table = torch.arange(8, dtype=torch.int32)[:, None]
    dev, host = _run_write(state, kv[:, 0], kv[:, 1], table, start)
    _check(dev, host)
    s = dev["k_scale"][:, 0].cpu()
    assert s[0] == 0 and s[1].isnan() and s[3].isnan() and s[4].isnan() and s[2] > 0
    assert dev["k_bounds"][4, 0, 0, 0].isnan()


def test_write_skips_and_reports(clean_error_word):
    """Negative starts and q_len limits write nothing; rows behind the last sequence stay."""
    kind, bs, hd, nkv = torch.int8, 32, 64, 2
    state = _filled(6, nkv, bs, hd, kind, 5)
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
    kv = torch.randn(100, 2, nkv, hd, generator=torch.Generator().manual_seed(6)).bfloat16()
    cu = torch.tensor([0, 40, 60, 90], dtype=torch.int32)
    start = torch.tensor([0, -1, 10], dtype=torch.int32)
    qlen = torch.tensor([33, 20, 0], dtype=torch.int32)
    dev, host = _run_write(state, kv[:, 0], kv[:, 1], table, start, cu, qlen)
    _check(dev, host)
    for n in ("k_cache", "v_cache"):
        assert torch.equal(_bits(dev[n][2:]), _bits(state[n][2:]))
        assert torch.equal(_bits(dev[n][1, :, 1:]), _bits(state[n][1, :, 1:]))


def test_write_bad_pages_are_skipped_and_reported():
    from b200attn import ops

    ops.read_error_word()
    kind, bs, hd, nkv = torch.float8_e4m3fn, 32, 128, 2
    state = _filled(3, nkv, bs, hd, kind, 7)
    table = torch.tensor([[3], [-1], [1], [2]], dtype=torch.int32)
    kv = torch.randn(4, 2, nkv, hd, generator=torch.Generator().manual_seed(8)).bfloat16()
    start = torch.tensor([0, 0, 4, 32], dtype=torch.int32)       # the last: beyond the table
    dev, host = _run_write(state, kv[:, 0], kv[:, 1], table, start)
    assert ops.read_error_word() == 2
    _check(dev, host)


def test_write_with_malformed_offsets_is_reported():
    """cu_q out of order or past the rows: nothing out of range is read or written."""
    from b200attn import ops

    ops.read_error_word()
    state = _filled(4, 1, 32, 64, torch.int8, 1)
    dev = {n: t.cuda() for n, t in state.items()}
    kv = torch.randn(20, 2, 1, 64).bfloat16().cuda()
    table = torch.zeros(2, 2, dtype=torch.int32).cuda()
    for cu in ([0, 10, 50], [0, 30, 20], [-5, 10, 20]):
        ops.paged_write(dev["k_cache"], dev["v_cache"], kv[:, 0], kv[:, 1], table,
                        torch.zeros(2, dtype=torch.int32).cuda(),
                        cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), k_scale=dev["k_scale"],
                        v_scale=dev["v_scale"])
        assert ops.read_error_word() == 2, cu


# ------------------------------------------------------------------------------------- decode
def _decode_case(users, nq, nkv, hd, bs, ctx, kind, seed, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    need = [(c + bs - 1) // bs for c in ctx]
    nb = sum(need) + 1
    c = _filled(nb, nkv, bs, hd, kind, seed)
    if spread:      # scales that differ by orders of magnitude from page to page
        c["v_scale"] *= torch.exp2(torch.randint(-20, 21, c["v_scale"].shape, generator=g).float()
                                   * spread)
    perm = torch.randperm(nb, generator=g).int()
    table = torch.zeros(users, max(max(need), 1), dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    c["table"] = table
    c["pos"] = torch.tensor(ctx, dtype=torch.int32) - 1
    c["query"] = torch.randn(users, nq, hd, generator=g).bfloat16()
    return c


def _decode(c, **kw):
    from b200attn import ops

    return ops.paged_decode(c["query"].cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(),
                            c["table"].cuda(), c["pos"].cuda(), k_scale=c["k_scale"].cuda(),
                            v_scale=c["v_scale"].cuda(), **kw).cpu()


def _attention_close(got, c, **kw):
    """One rounding to bf16 (half a step relative), and weights rounded to f16 (2^-11 relative
    each) against an unrounded sum: at most 2^-11 of the weighted mean of |v|; as much again for
    the fp32 sums, exponentials and scores."""
    want = blocks.decode(c["query"], c["k_cache"], c["v_cache"], c["table"], c["pos"],
                         k_scale=c["k_scale"], v_scale=c["v_scale"], **kw)
    size = dict(c, v_cache=c["v_cache"].float().abs())
    mean_abs = blocks.decode(c["query"], c["k_cache"], size["v_cache"], c["table"], c["pos"],
                             k_scale=c["k_scale"], v_scale=c["v_scale"], **kw)
    err = (got.double() - want).abs()
    tol = torch.finfo(torch.bfloat16).eps / 2 * want.abs() + 2.0 ** -10 * mean_abs
    assert (err <= tol).all(), f"{(err - tol).max():.3e} over; max err {err.max():.3e}"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd,bs", [(4, 4, 64, 32), (32, 8, 64, 64), (32, 8, 128, 64),
                                          (64, 8, 128, 32), (16, 1, 128, 64), (27, 3, 64, 32),
                                          (10, 2, 128, 32), (24, 2, 64, 64)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_decode_matches_fp64(clean_error_word, kind, nq, nkv, hd, bs, splits):
    c = _decode_case(6, nq, nkv, hd, bs, [1, 16, 63, 64, 129, 777], kind, seed=nq + hd)
    _attention_close(_decode(c, num_splits=splits), c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_with_scales_far_apart(clean_error_word, kind, hd):
    """V scales from 2^-20 to 2^20 between pages: every page keeps its precision."""
    c = _decode_case(4, 8, 2, hd, 32, [40, 200, 333, 64], kind, seed=3, spread=1.0)
    _attention_close(_decode(c, num_splits=2), c)
    # a page with a huge scale whose keys score low next to one with a tiny scale
    c["k_scale"][c["table"][2, 3].long()] = 0.0
    _attention_close(_decode(c, num_splits=1), c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, False), (17, False), (64, True), (1000, True), (0, True)])
def test_decode_window_and_sinks(clean_error_word, kind, window, sinks):
    c = _decode_case(5, 16, 4, 128, 64, [1, 70, 128, 300, 1000], kind, seed=window + 1)
    s = torch.randn(16, generator=torch.Generator().manual_seed(1)) * 2 if sinks else None
    got = _decode(c, sliding_window=window, sinks=None if s is None else s.cuda())
    _attention_close(got, c, window=window, sinks=s)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_empty_rows_zero_scales_and_extreme_queries(clean_error_word, kind):
    c = _decode_case(5, 8, 2, 128, 32, [100, 50, 40, 33, 90], kind, seed=12)
    c["pos"][1] = -1                                     # a padding row
    c["v_scale"][c["table"][0, 1].long()] = 0.0          # values of a whole page are zero
    c["k_scale"][c["table"][0, 2].long()] = 0.0
    c["query"][2] *= 1e30                                # one key takes everything
    c["query"][3] = 0.0                                  # uniform weights
    c["query"][4] *= 1e-30
    got = _decode(c)
    assert not got[1].any()
    _attention_close(got, c)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("splits", [1, 2])
def test_decode_ignores_what_is_behind_the_context(clean_error_word, kind, splits):
    """Dead rows of the last page hold anything (e4m3 NaN codes included), and so do the pages and
    scales that no context reaches."""
    c = _decode_case(3, 8, 2, 64, 32, [5, 40, 95], kind, seed=8)
    want = _decode(c, num_splits=splits)
    for u, n in enumerate([5, 40, 95]):
        blk = int(c["table"][u, (n - 1) // 32])
        for name in ("k_cache", "v_cache"):
            c[name].view(torch.uint8)[blk, :, (n - 1) % 32 + 1:] = 0x7F
    used = {int(c["table"][u, i]) for u, n in enumerate([5, 40, 95]) for i in range((n + 31) // 32)}
    for blk in set(range(c["k_cache"].shape[0])) - used:
        c["k_scale"][blk] = c["v_scale"][blk] = float("nan")
        c["v_cache"].view(torch.uint8)[blk] = 0x7F
    assert torch.equal(_decode(c, num_splits=splits), want)


@pytest.mark.parametrize("splits", [1, 2, 4])
def test_decode_nan_scales_come_out(clean_error_word, splits):
    c = _decode_case(3, 8, 2, 128, 32, [64, 100, 64], torch.int8, seed=8)
    c["k_scale"][int(c["table"][0, 1]), 0] = float("nan")
    c["v_scale"][int(c["table"][1, 0]), 1] = float("nan")
    got = _decode(c, num_splits=splits)
    assert got[0, :4].isnan().all() and not got[0, 4:].isnan().any()
    assert got[1, 4:].isnan().all() and not got[1, :4].isnan().any()
    assert not got[2].isnan().any()


def test_decode_bad_page_is_reported():
    from b200attn import ops

    ops.read_error_word()
    c = _decode_case(2, 8, 2, 128, 32, [64, 100], torch.int8, seed=8)
    c["table"][0, 1] = 99
    c["table"][1, 0] = -3
    _decode(c)
    assert ops.read_error_word() == 2


@pytest.mark.parametrize("splits", [0, 2])
def test_decode_positions_behind_the_table_are_reported(splits):
    """Up to the largest int: the keys of the table's pages are attended, nothing else is read."""
    from b200attn import ops

    ops.read_error_word()
    c = _decode_case(3, 8, 2, 64, 32, [64, 96, 64], torch.int8, seed=8)
    full = dict(c, pos=torch.tensor([95, 95, 95], dtype=torch.int32))
    want = _decode(full, num_splits=splits)
    assert ops.read_error_word() == 0
    got = _decode(dict(c, pos=torch.tensor([96, 95, 2 ** 31 - 1], dtype=torch.int32)),
                  num_splits=splits)
    assert ops.read_error_word() == 2
    assert torch.equal(got, want)


@pytest.mark.parametrize("splits", [0, 1, 5])
def test_decode_shares_of_uneven_pairs(clean_error_word, splits):
    """One long context among short and empty ones: shares begin and end inside pairs."""
    ctx = [1, 0, 9000, 3, 0, 130, 257, 1]
    c = _decode_case(8, 6, 3, 64, 64, ctx, torch.float8_e4m3fn, seed=4)
    got = _decode(c, num_splits=splits)
    _attention_close(got, c)
    assert not got[1].any() and not got[4].any()


def test_decode_one_pair_uses_many_ctas(clean_error_word):
    c = _decode_case(1, 4, 1, 128, 64, [20000], torch.int8, seed=4)
    _attention_close(_decode(c), c)
    _attention_close(_decode(c, num_splits=200), c)


def test_decode_writes_into_out_rows_and_nothing_else(clean_error_word):
    """A strided `out`, a strided query and fewer users than table rows."""
    from b200attn import ops

    c = _decode_case(4, 8, 2, 64, 32, [64, 100, 7, 33], torch.int8, seed=8)
    d = {n: t.cuda() for n, t in c.items()}
    buf = torch.full((5, 3, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(4, 12, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10] = d["query"]
    out = buf[:3, 1]
    r = ops.paged_decode(wide[:3, 2:10], d["k_cache"], d["v_cache"], d["table"], d["pos"][:3],
                         out=out, k_scale=d["k_scale"], v_scale=d["v_scale"])
    assert r is out
    assert torch.equal(out.cpu(), _decode(c)[:3])
    assert (buf[:, 0] == 3).all() and (buf[:, 2] == 3).all() and (buf[3:] == 3).all()


def test_many_users_are_cut_between_pairs(clean_error_word):
    """More (user, KV head) pairs than arrival counters: no pair is shared by two CTAs."""
    users, nkv = 2100, 8
    c = _decode_case(users, 8, nkv, 64, 32, [1 + i % 70 for i in range(users)], torch.int8, seed=2)
    one, two = _decode(c, num_splits=1), _decode(c, num_splits=2)
    assert users * nkv > 16384
    sub = [0, 69, 1000, 2099]
    small = {n: (t[sub] if n in ("table", "pos", "query") else t) for n, t in c.items()}
    _attention_close(one[sub], small)
    _attention_close(two[sub], small)


@pytest.mark.parametrize("hd,bs", [(64, 32), (128, 64)])
@pytest.mark.parametrize("splits", [0, 1, 2])
@pytest.mark.parametrize("window", [1, 13, 40])
def test_decode_ignores_nan_codes_in_front_of_the_window(clean_error_word, hd, bs, splits, window):
    """e4m3 NaN codes in rows that a sliding window has left behind."""
    ctx = [20, 64, 139, 300]
    c = _decode_case(4, 8, 2, hd, bs, ctx, torch.float8_e4m3fn, seed=8)
    want = _decode(c, num_splits=splits, sliding_window=window)
    for u, n in enumerate(ctx):
        for j in range(max(0, n - window)):
            blk = int(c["table"][u, j // bs])
            for name in ("k_cache", "v_cache"):
                c[name].view(torch.uint8)[blk, :, j % bs] = 0x7F
    assert torch.equal(_decode(c, num_splits=splits, sliding_window=window), want)


@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("value", [-0.01, float("-inf"), float("inf"), float("nan")])
def test_what_is_no_scale_comes_out_as_nan(clean_error_word, which, value):
    """Negative and infinite scales in decode and in prefill: NaN for who attends the page and no
    one else, as a NaN scale."""
    from b200attn import ops

    n, bs, nq, nkv, hd = 150, 32, 8, 2, 64
    c = _decode_case(2, nq, nkv, hd, bs, [n, n], torch.int8, seed=6)
    q = torch.randn(n, nq, hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int32)

    def prefill():
        return ops.prefill(q.cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), cu,
                           page_table=c["table"][:1].cuda(), k_scale=c["k_scale"].cuda(),
                           v_scale=c["v_scale"].cuda()).cpu()

    good = [[_decode(c, num_splits=s) for s in (0, 1, 3)], prefill()]
    c[which][int(c["table"][0, 2]), 1] = value
    for got, want in zip([_decode(c, num_splits=s) for s in (0, 1, 3)], good[0]):
        assert got[0, 4:].isnan().all()
        assert torch.equal(got[0, :4], want[0, :4]) and torch.equal(got[1], want[1])
    got = prefill()
    assert got[2 * bs:, 4:].isnan().all()
    assert torch.equal(got[: 2 * bs], good[1][: 2 * bs]) and torch.equal(got[:, :4], good[1][:, :4])


# ------------------------------------------------------------------------------------ prefill
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd,bs", [(8, 2, 64, 32), (8, 8, 128, 64), (12, 3, 128, 32)])
@pytest.mark.parametrize("window", [0, 50])
def test_prefill_over_scaled_pages(clean_error_word, kind, nq, nkv, hd, bs, window):
    """Against fp64 attention over code * scale.  Weights are bf16: 2^-8 of the weighted mean of |v|,
    as much again for the fp32 scores and exponentials, and the rounding of the result."""
    from b200attn import ops

    lens, starts = [1, 37, 130], [0, 64, 15]
    ctx = [a + b for a, b in zip(lens, starts)]
    c = _decode_case(3, nq, nkv, hd, bs, ctx, kind, seed=5)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    q = torch.randn(int(cu[-1]), nq, hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    out = ops.prefill(q.cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), cu,
                      page_table=c["table"].cuda(),
                      q_start=torch.tensor(starts, dtype=torch.int32).cuda(),
                      sliding_window=window, k_scale=c["k_scale"].cuda(),
                      v_scale=c["v_scale"].cuda()).cpu()
    for s in range(3):
        for i in range(lens[s]):
            want, size = [blocks.decode(q[cu[s] + i][None], c["k_cache"], v, c["table"][s][None],
                                        torch.tensor([starts[s] + i]), window=window,
                                        k_scale=c["k_scale"], v_scale=c["v_scale"])[0]
                          for v in (c["v_cache"], c["v_cache"].float().abs())]
            err = (out[cu[s] + i].double() - want).abs()
            assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all(), (s, i, err.max())


@pytest.mark.parametrize("bs", [32, 64])
def test_prefill_scales_far_apart_zero_and_nan(clean_error_word, bs):
    """Scales of any size between the pages of a tile; a page of zeros; a NaN scale reaches the rows
    that attend its page and no others."""
    from b200attn import ops

    n, nq, nkv, hd = 150, 4, 2, 64
    c = _decode_case(1, nq, nkv, hd, bs, [n], torch.int8, seed=5, spread=1.0)
    ids = c["table"][0].long()
    c["v_scale"][ids[1]] = 0.0
    c["k_scale"][ids[0], 1] = 0.0
    q = torch.randn(n, nq, hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    cu = torch.tensor([0, n], dtype=torch.int32)

    def run():
        return ops.prefill(q.cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), cu,
                           page_table=c["table"].cuda(), k_scale=c["k_scale"].cuda(),
                           v_scale=c["v_scale"].cuda()).cpu()

    out = run()
    for i in range(n):
        want, size = [blocks.decode(q[i][None], c["k_cache"], v, c["table"], torch.tensor([i]),
                                    k_scale=c["k_scale"], v_scale=c["v_scale"])[0]
                      for v in (c["v_cache"], c["v_cache"].float().abs())]
        err = (out[i].double() - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all(), (i, err.max())
    last = (n - 1) // bs
    for which in ("k_scale", "v_scale"):
        keep = c[which].clone()
        c[which][ids[last], 0] = float("nan")
        got = run()
        assert got[last * bs:, : nq // 2].isnan().all()
        assert torch.equal(got[: last * bs], out[: last * bs])
        assert torch.equal(got[:, nq // 2:], out[:, nq // 2:])
        c[which] = keep


@pytest.mark.parametrize("bad", [99, -3, 2 ** 31 - 1])
def test_prefill_bad_page_is_reported_and_comes_out_as_nan(bad):
    """For the rows that attend it and no others; no row shows what memory held before."""
    from b200attn import ops

    n, nq, nkv, hd, bs = 150, 4, 2, 64, 32
    c = _decode_case(2, nq, nkv, hd, bs, [n, n], torch.int8, seed=5)
    q = torch.randn(2 * n, nq, hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32)

    def run():
        return ops.prefill(q.cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), cu,
                           page_table=c["table"].cuda(), k_scale=c["k_scale"].cuda(),
                           v_scale=c["v_scale"].cuda()).cpu()

    ops.read_error_word()
    want = run()
    assert ops.read_error_word() == 0
    c["table"][1, 2] = bad
    for fill in (float("nan"), 1.0, 0.0):
        junk = torch.full((1 << 22,), fill, device="cuda")      # what the allocator hands out next
        del junk
        got = run()
        assert ops.read_error_word() == 2
        assert torch.equal(got[: n + 2 * bs], want[: n + 2 * bs])
        assert got[n + 2 * bs:].isnan().all()


def test_prefill_through_a_table_much_wider_than_its_contexts(clean_error_word):
    """The columns of the longest context count, for the result and for the memory."""
    from b200attn import ops

    lens, starts = [33, 1, 130], [0, 64, 15]
    c = _decode_case(3, 8, 2, 128, 64, [a + b for a, b in zip(lens, starts)], torch.int8, seed=5)
    cu = torch.tensor([0] + lens).cumsum(0).int()
    q = torch.randn(int(cu[-1]), 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    wide = torch.full((3, 2048), 10 ** 8, dtype=torch.int32)
    wide[:, : c["table"].shape[1]] = c["table"]
    d = {n: t.cuda() for n, t in c.items()}

    def run(table, **kw):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = ops.prefill(q, d["k_cache"], d["v_cache"], cu, page_table=table,
                          q_start=torch.tensor(starts, dtype=torch.int32).cuda(),
                          k_scale=d["k_scale"], v_scale=d["v_scale"], **kw)
        torch.cuda.synchronize()
        return out, torch.cuda.max_memory_allocated() - before

    want, _ = run(d["table"])
    for hint in (145, 192, 1000, 0):
        got, used = run(wide.cuda(), max_context_len=hint)
        assert torch.equal(got, want)
        if hint:         # bf16 K and V of 2 heads of 128, and room for the rest
            assert used < 3 * (hint // 64 + 1) * 2 * 64 * 128 * 4 + (4 << 20)


@pytest.mark.parametrize("hint", [1, 64, 144])
def test_prefill_of_a_context_longer_than_promised_is_reported(hint):
    from b200attn import ops

    c = {n: t.cuda() for n, t in _decode_case(2, 8, 2, 64, 32, [40, 145], torch.int8, seed=5).items()}
    cu = torch.tensor([0, 40, 75], dtype=torch.int32)
    q = torch.zeros(75, 8, 64, dtype=torch.bfloat16, device="cuda")

    def run(n):
        ops.prefill(q, c["k_cache"], c["v_cache"], cu, page_table=c["table"], max_context_len=n,
                    q_start=torch.tensor([0, 110], dtype=torch.int32).cuda(), k_scale=c["k_scale"],
                    v_scale=c["v_scale"])
        return ops.read_error_word()

    ops.read_error_word()
    assert run(145) == 0 and run(hint) == 2 and run(0) == 0


# ----------------------------------------------------------------------------------- refusals
def test_refusals():
    from b200attn import ops
    from b200attn._lib import B200AttnError

    c = {n: t.cuda() for n, t in _decode_case(2, 8, 2, 64, 32, [40, 50], torch.int8, 1).items()}
    scales = dict(k_scale=c["k_scale"], v_scale=c["v_scale"])

    def dec(table=c["table"], pos=c["pos"], q=c["query"], k=c["k_cache"], v=c["v_cache"], **kw):
        return ops.paged_decode(q, k, v, table, pos, **{**scales, **kw})

    dec()
    new = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(v_scale=None), dict(k_scale=c["k_scale"].double()),
                dict(k_scale=c["k_scale"][:1]), dict(k=c["k_cache"].bfloat16()),
                dict(k=c["k_cache"].bfloat16(), v=c["v_cache"].bfloat16()),
                dict(k_scale=None, v_scale=None), dict(new_key=new, new_value=new),
                dict(pos=c["pos"][:1]), dict(table=c["table"][:1]), dict(table=c["table"].long())):
        with pytest.raises(ValueError):
            dec(**bad)
    with pytest.raises(B200AttnError):
        dec(q=torch.zeros(2, 34, 64, dtype=torch.bfloat16, device="cuda"))    # 17 per KV head
    with pytest.raises(B200AttnError, match="workspace"):
        dec(num_splits=2, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        dec(k_scale=c["k_scale"].cpu())

    def write(key=new, value=new, start=torch.zeros(2, dtype=torch.int32, device="cuda"),
              table=c["table"], k=c["k_cache"], v=c["v_cache"], **kw):
        ops.paged_write(k, v, key, value, table, start, **{**scales, **kw})

    write()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(key=new.float()), dict(key=new[:1]), dict(value=new[:, :1]),
                dict(start=cu), dict(cu_q=cu[:2]), dict(cu_q=cu.long()), dict(q_len=cu),
                dict(k_scale=None), dict(k_scale=None, v_scale=None), dict(table=c["table"][:1]),
                dict(k_bounds=torch.zeros(2, 2, 2, 64, device="cuda")),
                dict(k=c["k_cache"].bfloat16(), v=c["v_cache"].bfloat16(), k_scale=None,
                     v_scale=None)):
        with pytest.raises(ValueError):
            write(**bad)
    with pytest.raises(ValueError, match="paged cache"):
        ops.prefill(c["query"], new, new, torch.tensor([0, 2], dtype=torch.int32), **scales)
