"""Page selection against fp64 scores (equal integers), and decode over the lists it gives."""
import pytest
import torch

from oracle import blocks

pytestmark = pytest.mark.gpu


def _case(users, nq, nkv, hd, bs, ctx, seed, cache=False):
    g = torch.Generator().manual_seed(seed)
    need = [max(0, (c + bs - 1) // bs) for c in ctx]
    nb = sum(need) + 1
    perm = torch.randperm(nb, generator=g).int()
    table = torch.zeros(users, max(max(need), 1) + 2, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = perm[at:at + n]
        at += n
    c = dict(table=table, pos=torch.tensor(ctx, dtype=torch.int32) - 1,
             query=torch.randn(users, nq, hd, generator=g).bfloat16())
    if cache:
        c["k_cache"] = (torch.randn(nb, nkv, bs, hd, generator=g)
                        + torch.randn(nb, nkv, 1, hd, generator=g)).bfloat16()
        c["v_cache"] = torch.randn(nb, nkv, bs, hd, generator=g).bfloat16()
        c["k_bounds"] = torch.stack([c["k_cache"].amin(2), c["k_cache"].amax(2)], 2)
    else:
        c["k_bounds"] = torch.randn(nb, nkv, 2, hd, generator=g).sort(dim=2).values.bfloat16()
    return c


def _select(c, bs, k, first, last, **kw):
    from b200attn import ops

    return ops.select_pages(c["query"].cuda(), c["k_bounds"].cuda(), c["table"].cuda(),
                            c["pos"].cuda(), bs, k, first, last, **kw)


def _check(c, bs, k, first, last, **kw):
    table, pos = _select(c, bs, k, first, last, **kw)
    want_t, want_p = blocks.select_pages(c["query"], c["k_bounds"], c["table"], c["pos"], bs, k,
                                         first, last)
    assert torch.equal(pos.cpu(), want_p)
    assert torch.equal(table.cpu(), want_t)
    return table, pos


@pytest.mark.parametrize("nq,nkv,hd,bs", [(8, 8, 64, 32), (32, 8, 128, 64), (16, 1, 128, 32),
                                          (27, 3, 64, 64), (10, 2, 128, 64)])
@pytest.mark.parametrize("k,first,last", [(1, 0, 1), (4, 1, 1), (9, 2, 3), (16, 0, 2), (64, 1, 1),
                                          (3, 2, 1)])
def test_selection_matches_fp64(clean_error_word, nq, nkv, hd, bs, k, first, last):
    ctx = [1, bs, bs + 1, 5 * bs - 3, 17 * bs, 300 * bs + 7]
    _check(_case(6, nq, nkv, hd, bs, ctx, seed=nq + k), bs, k, first, last)


@pytest.mark.parametrize("hint", [0, 32, 1 << 20])
def test_the_length_hint_does_not_change_the_choice(clean_error_word, hint):
    c = _case(2, 8, 2, 64, 32, [900 * 32, 70], seed=4)
    _check(c, 32, 20, 1, 1, max_context_len=hint)


@pytest.mark.parametrize("pages", [4097, 9000])
def test_more_pages_than_stay_in_shared_memory(clean_error_word, pages):
    c = _case(2, 4, 1, 64, 32, [pages * 32 - 5, 4096 * 32], seed=pages)
    _check(c, 32, 200, 2, 3)
    c["k_bounds"][:] = c["k_bounds"][0]
    _check(c, 32, 300, 1, 2)


def test_many_users(clean_error_word):
    """More (user, KV head) pairs than arrival counters."""
    users = 2100
    c = _case(users, 8, 8, 64, 32, [1 + (i * 37) % 400 for i in range(users)], seed=2)
    table, pos = _select(c, 32, 4, 1, 1)
    sub = [0, 10, 777, 2099]
    small = dict(c, query=c["query"][sub], table=c["table"][sub], pos=c["pos"][sub])
    want_t, want_p = blocks.select_pages(small["query"], c["k_bounds"], small["table"], small["pos"],
                                         32, 4, 1, 1)
    assert torch.equal(table.cpu()[sub], want_t) and torch.equal(pos.cpu()[sub], want_p)


def test_ties_go_to_the_lower_page(clean_error_word):
    """Equal bounds everywhere, two values of bounds, and a zero query."""
    c = _case(3, 8, 2, 64, 32, [700 * 32, 50 * 32, 400 * 32], seed=4)
    c["k_bounds"][:] = c["k_bounds"][0]
    _check(c, 32, 33, 1, 2)
    c["k_bounds"][::3] *= 2
    _check(c, 32, 300, 1, 2)
    c["query"][:] = 0
    _check(c, 32, 10, 0, 1)


def test_scores_that_differ_in_the_last_bits(clean_error_word):
    """Pages whose scores differ by less than fp32 sums resolve: the exact order decides.  Large
    terms that cancel hide a small one."""
    c = _case(1, 4, 1, 128, 32, [200 * 32], seed=6)
    c["query"][:] = 1.0
    c["k_bounds"][:] = 0.0
    n = c["k_bounds"].shape[0]
    small = torch.randperm(n, generator=torch.Generator().manual_seed(1)).float()
    c["k_bounds"][:, 0, 1, 0] = 3.0e7
    c["k_bounds"][:, 0, 1, 5] = -3.0e7
    c["k_bounds"][:, 0, 1, 9] = (small * 2.0 ** -7).bfloat16()
    _check(c, 32, 50, 1, 1)


def test_nan_and_infinite_bounds(clean_error_word):
    c = _case(2, 4, 2, 64, 32, [100 * 32, 60 * 32], seed=7)
    c["k_bounds"][int(c["table"][0, 40]), 0, 0, 3] = float("nan")
    c["k_bounds"][int(c["table"][0, 50]), 1, 1, 3] = float("inf")
    c["k_bounds"][int(c["table"][1, 20]), 0, 0, 5] = float("-inf")
    table, _ = _check(c, 32, 8, 1, 1)
    assert int(c["table"][0, 40]) in table[0, 0].tolist()


def test_padding_rows_and_contexts_beyond_the_table(clean_error_word):
    c = _case(4, 4, 2, 64, 32, [0, 500, 33, 0], seed=8)
    c["pos"][3] = -7
    table, pos = _check(c, 32, 5, 1, 1)
    assert (pos[0] == -1).all() and not table[0].any() and (pos[3] == -1).all()


def test_bad_pages_are_reported_and_rank_last():
    from b200attn import ops

    ops.read_error_word()
    c = _case(1, 4, 2, 64, 32, [40 * 32], seed=9)
    bad = [7, 13]
    c["table"][0, bad[0]] = 10 ** 6
    c["table"][0, bad[1]] = -2
    table, _ = _select(c, 32, 20, 1, 1)
    assert ops.read_error_word() == 2
    assert 10 ** 6 not in table.cpu()[0].flatten().tolist()
    assert -2 not in table.cpu()[0].flatten().tolist()


@pytest.mark.parametrize("pages", [6, 64])
@pytest.mark.parametrize("behind", [0, 5, 2 ** 31])
def test_positions_behind_the_table_are_reported(pages, behind):
    """The choice is the one at the table's last key, whether every page is taken or some are."""
    from b200attn import ops

    ops.read_error_word()
    c = _case(2, 4, 2, 64, 32, [20 * 32, 20 * 32], seed=8)
    c["table"] = c["table"][:, :20].contiguous()
    want = _check(c, 32, pages, 1, 1)
    assert ops.read_error_word() == 0
    c["pos"][1] = min(20 * 32 + behind, 2 ** 31 - 1)
    got = _check(c, 32, pages, 1, 1)
    assert ops.read_error_word() == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("q_exp,b_exp", [(-70, -75), (-100, -30), (-76, -76), (-85, -66)])
def test_scores_below_the_normal_range(clean_error_word, q_exp, b_exp):
    """Products and sums that fp32 flushes or holds in a few bits: the exact order decides."""
    c = _case(2, 8, 2, 64, 32, [100 * 32, 37 * 32 + 5], seed=12)
    c["query"] *= 2.0 ** q_exp
    c["k_bounds"] *= 2.0 ** b_exp
    _check(c, 32, 20, 1, 1)


@pytest.mark.parametrize("nq,nkv,hd,bs", [(8, 2, 64, 32), (32, 8, 128, 64), (32, 2, 128, 32)])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
def test_decode_over_the_chosen_pages(clean_error_word, nq, nkv, hd, bs, splits, kind):
    """bf16 weights: 2^-8 of the weighted mean of |v| (f16 in the scaled kernels), as much again for
    the fp32 part, and one rounding of the result."""
    from b200attn import ops

    c = _case(5, nq, nkv, hd, bs, [1, bs, 9 * bs + 5, 33 * bs - 1, 20 * bs], seed=3, cache=True)
    c["pos"][4] = -1
    scales = {}
    if kind != torch.bfloat16:
        for w in "kv":
            x = c[w + "_cache"].float()
            s = x.abs().amax((2, 3)) / blocks.QMAX[kind].item()
            q = x / s[:, :, None, None]
            c[w + "_cache"] = (q.round() if kind == torch.int8 else q).to(kind)
            scales[w + "_scale"] = s
    table, pos = _select(c, bs, 6, 1, 1)
    got = ops.paged_decode(c["query"].cuda(), c["k_cache"].cuda(), c["v_cache"].cuda(), table, pos,
                           num_splits=splits, **{n: s.cuda() for n, s in scales.items()}).cpu()
    args = (c["query"], c["k_cache"])
    want = blocks.decode(*args, c["v_cache"], table.cpu(), pos.cpu(), **scales)
    size = blocks.decode(*args, c["v_cache"].float().abs(), table.cpu(), pos.cpu(), **scales)
    err = (got.double() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all(), err.max()
    assert not got[4].any()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("splits", [1, 4])
def test_lists_of_any_length_per_head(clean_error_word, kind, splits):
    """Lists the caller made: another length for every head, empty ones, a page twice; bf16 and
    unscaled e4m3 caches."""
    from b200attn import ops

    g = torch.Generator().manual_seed(11)
    users, nq, nkv, hd, bs, nb = 3, 12, 3, 128, 32, 20
    k = torch.randn(nb, nkv, bs, hd, generator=g).to(kind)
    v = torch.randn(nb, nkv, bs, hd, generator=g).to(kind)
    q = torch.randn(users, nq, hd, generator=g).bfloat16()
    table = torch.randint(0, nb, (users, nkv, 9), generator=g).int()
    pos = torch.tensor([[0, 31, 287], [-1, 32, 100], [5, -1, 250]], dtype=torch.int32)
    got = ops.paged_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), pos.cuda(),
                           num_splits=splits).cpu()
    want = blocks.decode(q, k, v, table, pos)
    size = blocks.decode(q, k, v.float().abs(), table, pos)
    err = (got.double() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all(), err.max()
    assert not got[1, :4].any() and not got[2, 4:8].any()


def test_a_list_of_every_page_is_the_dense_decode(clean_error_word):
    from b200attn import ops

    c = {n: t.cuda() for n, t in _case(3, 8, 2, 128, 64, [64, 700, 129], seed=3,
                                       cache=True).items()}
    table, pos = ops.select_pages(c["query"], c["k_bounds"], c["table"], c["pos"], 64, 16)
    a = ops.paged_decode(c["query"], c["k_cache"], c["v_cache"], table, pos, num_splits=2)
    b = ops.paged_decode(c["query"], c["k_cache"], c["v_cache"], c["table"], c["pos"], num_splits=2)
    assert torch.equal(a, b)


def test_refusals():
    from b200attn import ops
    from b200attn._lib import B200AttnError

    c = {n: t.cuda() for n, t in _case(2, 8, 2, 64, 32, [300, 200], seed=3, cache=True).items()}

    def sel(q=c["query"], b=c["k_bounds"], t=c["table"], p=c["pos"], bs=32, k=4, **kw):
        return ops.select_pages(q, b, t, p, bs, k, **kw)

    table, pos = sel()
    for bad in (dict(b=c["k_bounds"].float()), dict(b=c["k_bounds"][:, :, :1]),
                dict(q=c["query"][:, :3]), dict(q=c["query"][..., :32]), dict(t=c["table"].long()),
                dict(p=c["pos"][:1]), dict(t=c["table"][:1]), dict(k=1), dict(keep_last=0),
                dict(keep_first=-1), dict(k=4, keep_first=2, keep_last=3)):
        with pytest.raises(ValueError):
            sel(**bad)
    with pytest.raises(B200AttnError):
        sel(bs=48)
    with pytest.raises(B200AttnError, match="workspace"):
        sel(workspace=torch.zeros(1024, dtype=torch.uint8, device="cuda"))

    def dec(t=table, p=pos, **kw):
        return ops.paged_decode(c["query"], c["k_cache"], c["v_cache"], t, p, **kw)

    dec()
    new = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(p=c["pos"]), dict(t=table[:1]), dict(t=table[:, :1]), dict(sliding_window=8),
                dict(new_key=new, new_value=new), dict(t=table.long()),
                dict(t=table[:, :1].expand(2, 2, 4))):
        with pytest.raises(ValueError):
            dec(**bad)
