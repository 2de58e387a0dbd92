"""The cache-side operators as a layer uses them: norms + rotation, block-scaled or bf16 cache with
key bounds, page selection and attention, in both metadata forms, over several steps, against the
plain restatement; and the calls around them: captured graphs, side streams, replays side by side."""
import pytest
import torch

from oracle import blocks

pytestmark = pytest.mark.gpu

NQ, NKV, HD, BS = 8, 2, 64, 32
DTYPES = {"int8_block": torch.int8, "fp8_block": torch.float8_e4m3fn, "auto": torch.bfloat16}


class Reference:
    """A layer's cache and outputs, one operator after the other, on the CPU in fp64."""

    def __init__(self, kind, nb, bounds):
        self.kind = DTYPES[kind]
        shape = (nb, NKV, BS, HD)
        self.k, self.v = torch.zeros(shape).to(self.kind), torch.zeros(shape).to(self.kind)
        scaled = kind != "auto"
        self.ks = torch.zeros(nb, NKV) if scaled else None
        self.vs = torch.zeros(nb, NKV) if scaled else None
        self.bounds = torch.zeros(nb, NKV, 2, HD).bfloat16() if bounds else None

    def write(self, key, value, table, start, cu=None):
        blocks.paged_write(self.k, self.v, key.reshape(-1, NKV, HD), value.reshape(-1, NKV, HD),
                           table, start, cu, k_scale=self.ks, v_scale=self.vs,
                           k_bounds=self.bounds)

    def decode(self, query, table, pos, sparse=None):
        q = query.reshape(-1, NQ, HD)
        if sparse:
            table, pos = blocks.select_pages(q, self.bounds, table, pos, BS, *sparse)
        return [blocks.decode(q, self.k, v, table, pos, k_scale=self.ks, v_scale=self.vs)
                for v in (self.v, self.v.float().abs())]


def _close(got, want, size):
    """Weights of 8 bits or more (2^-8 of the weighted mean of |v|), as much again for fp32 scores
    and exponentials, one rounding of the result."""
    err = (got.reshape(want.shape).double().cpu() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all(), err.max()


def _layer(kind, sparse, norm=True):
    from b200attn import B200Attention

    g = torch.Generator().manual_seed(3)
    w = [(1 + 0.2 * torch.randn(HD, generator=g)).bfloat16() for _ in range(2)]
    kw = dict(sparse_pages=sparse[0], sparse_keep_first=sparse[1], sparse_keep_last=sparse[2]) \
        if sparse else {}
    norms = dict(q_norm_weight=w[0], k_norm_weight=w[1], norm_eps=1e-5) if norm else {}
    layer = B200Attention(NQ, HD, HD ** -0.5, NKV, rotary_dim=HD, rope_theta=10000.0,
                          kv_cache_dtype=kind, **norms, **kw)
    return layer, w


def _qkv(n, seed):
    return torch.randn(n, (NQ + 2 * NKV) * HD, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _split(x):
    return x.split([NQ * HD, NKV * HD, NKV * HD], 1)


def _caches(kind, nb, bounds):
    from b200attn import sharding

    return sharding.allocate_kv_caches(1, nb, NKV, BS, HD, dtype=DTYPES[kind], device="cuda",
                                       block_scales=kind != "auto",
                                       page_bounds=bounds)["layers.0.attn"]


def _check_cache(cache, ref):
    pairs = [(cache[0], ref.k), (cache[1], ref.v)]
    if ref.ks is not None:
        pairs += [(cache[2], ref.ks), (cache[3], ref.vs)]
    if ref.bounds is not None:
        pairs.append((cache[4], ref.bounds))
    for a, b in pairs:
        assert torch.equal(a.cpu().float(), b.float())


@pytest.mark.parametrize("kind", ["int8_block", "fp8_block", "auto"])
@pytest.mark.parametrize("sparse", [None, (3, 1, 1)])
def test_varlen_steps(clean_error_word, kind, sparse):
    """Prompts, then a mixed step, then decode steps, through the layer in vLLM's varlen form."""
    from b200attn.backend import build_varlen_metadata

    if kind == "auto" and not sparse:
        pytest.skip("the plain bf16 cache has tests of its own")
    layer, w = _layer(kind, sparse)
    nb = 40
    layer.kv_cache = _caches(kind, nb, bool(sparse))
    ref = Reference(kind, nb, bool(sparse))
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(1))[:36].int().reshape(3, 12)
    steps = [[150, 70, 1], [1, 40, 1], [1, 1, 1], [1, 1, 1]]
    done = [0, 0, 0]
    # vLLM orders one-token rows first
    for n, lens in enumerate(steps):
        order = sorted(range(3), key=lambda s: lens[s] != 1)
        q_lens = [lens[s] for s in order]
        start = torch.tensor([done[s] for s in order]).int()
        cu = torch.tensor([0] + q_lens).cumsum(0).int()
        seq = start + torch.tensor(q_lens).int()
        rows = table[order]
        pos = torch.cat([torch.arange(a, b) for a, b in zip(start.tolist(), seq.tolist())])
        slots = torch.cat([rows[i, torch.arange(int(a), int(b)) // BS].long() * BS
                           + torch.arange(int(a), int(b)) % BS
                           for i, (a, b) in enumerate(zip(start, seq))])
        x = _qkv(int(cu[-1]), 10 + n)
        md = build_varlen_metadata(cu.cuda(), cu, seq.cuda(), rows.cuda(), slots.cuda(),
                                   max_seq_len=int(seq.max()))
        dev = x.cuda()
        out = layer(*_split(dev), attn_metadata=md, positions=pos.cuda())
        q, k, v = _split(dev.cpu())                 # rotated in place
        hq, hk, hv = _split(x)
        for got, y, weight in ((q, hq, w[0]), (k, hk, w[1])):
            want = blocks.qk_norm_rope(y, pos, layer.inv_freq.cpu(), HD, HD, weight, 1e-5, True)
            top = want.reshape(-1, HD).abs().amax(-1).repeat_interleave(HD).reshape(want.shape)
            assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * top).all()
        ref.write(k, v, rows, start, cu)
        _check_cache(layer.kv_cache, ref)
        for i in range(3):
            for t in range(q_lens[i]):
                at = int(cu[i]) + t
                one = torch.tensor([int(start[i]) + t])
                use = sparse if q_lens[i] == 1 else None
                want, size = ref.decode(q[at:at + 1], rows[i:i + 1], one, use)
                _close(out[at], want[0].reshape(-1), size[0].reshape(-1))
        for s in range(3):
            done[s] += lens[s]


@pytest.mark.parametrize("kind", ["int8_block", "fp8_block"])
def test_plugin_form_padded_prompt_chunk_and_decode(clean_error_word, kind):
    """[users x tokens] form: padded prompts (padding written nowhere, whatever it holds), a chunk on
    top, then decode with a padding row."""
    from b200attn import B200AttentionBackendImpl, B200Metadata

    nb, users, tokens = 24, 3, 64
    impl = B200AttentionBackendImpl(NQ, HD, HD ** -0.5, NKV, None, None, kind)
    cache = _caches(kind, nb, True)
    ref = Reference(kind, nb, True)
    table = torch.randperm(nb, generator=torch.Generator().manual_seed(1))[:18].int().reshape(3, 6)
    valid = [64, 37, 0]
    x = _qkv(users * tokens, 4)
    x3 = x.reshape(users, tokens, -1)
    for u, n in enumerate(valid):
        x3[u, n:] = float("nan") if u else 3e38
    pos = torch.tensor(valid).int() - 1
    md = B200Metadata(cache_position=pos.cuda(), page_table=table.cuda(), num_users=users,
                      batch_idx=torch.arange(users).int().cuda())
    out = torch.empty(users * tokens, NQ * HD, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, *[t.contiguous().cuda() for t in _split(x)], cache, md, output=out)
    for u, n in enumerate(valid):
        q, k, v = _split(x3[u, :n].contiguous())
        ref.write(k, v, table[u:u + 1], torch.zeros(1).int(), torch.tensor([0, n]).int())
    _check_cache(cache, ref)
    # a chunk of 32 tokens on top of a 64-token prefix for users 0 and (all dead) 1, 2
    y = _qkv(users * 32, 5)
    total = torch.tensor([96, 0, 0]).int()
    fill = torch.cat([table[:, 2:], table[:, :2]], 1).contiguous()
    md = B200Metadata(cache_position=(total - 1).cuda(), page_table=table.cuda(), num_users=users,
                      fill_page_table=fill.cuda(), batch_idx=torch.arange(users).int().cuda(),
                      chunk_start_idx=torch.tensor([64]).int().cuda())
    out = torch.empty(users * 32, NQ * HD, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, *[t.contiguous().cuda() for t in _split(y)], cache, md, output=out)
    q, k, v = _split(y[:32].contiguous())
    ref.write(k, v, table[:1], torch.tensor([64]).int(), torch.tensor([0, 32]).int())
    _check_cache(cache, ref)
    for t in range(32):
        want, size = ref.decode(q[t:t + 1], table[:1], torch.tensor([64 + t]))
        _close(out[t], want[0].reshape(-1), size[0].reshape(-1))
    # decode: user 0 at 96, user 1 at 37, user 2 is padding
    z = _qkv(users, 6)
    pos = torch.tensor([96, 37, -1]).int()
    md = B200Metadata(cache_position=pos.cuda(), page_table=table.cuda(), num_users=users,
                      batch_idx=torch.arange(users).int().cuda())
    out = torch.empty(users, NQ * HD, dtype=torch.bfloat16, device="cuda")
    impl.forward(None, *[t.contiguous().cuda() for t in _split(z)], cache, md, output=out)
    q, k, v = _split(z)
    ref.write(k, v, table, pos)
    _check_cache(cache, ref)
    want, size = ref.decode(q, table, pos)
    _close(out, want.reshape(users, -1), size.reshape(users, -1))
    assert not out[2].any()


def _decode_setup(kind, users, ctx, seed):
    from b200attn import ops

    g = torch.Generator().manual_seed(seed)
    per = (ctx + BS) // BS + 1
    nb = users * per
    cache = _caches(kind, nb, True)
    table = torch.randperm(nb, generator=g).int().reshape(users, per).cuda()
    kv = torch.randn(users * ctx, 2, NKV, HD, generator=g).bfloat16().cuda()
    cu = (torch.arange(users + 1) * ctx).int().cuda()
    ops.paged_write(cache[0], cache[1], kv[:, 0], kv[:, 1], table, torch.zeros(users).int().cuda(),
                    cu_q=cu, k_scale=cache[2], v_scale=cache[3], k_bounds=cache[4])
    return cache, table


def _step(cache, table, x, pos, count):
    """One decode step as a runner issues it; returns its output."""
    from b200attn import ops

    q, k, v = _split(x)
    scales = dict(k_scale=cache[2], v_scale=cache[3])
    ops.paged_write(cache[0], cache[1], k, v, table, pos, k_bounds=cache[4], **scales)
    t, p = ops.select_pages(q.unflatten(1, (NQ, HD)), cache[4], table, pos, BS, count)
    return ops.paged_decode(q.unflatten(1, (NQ, HD)), cache[0], cache[1], t, p, **scales)


@pytest.mark.parametrize("kind", ["int8_block", "fp8_block"])
def test_captured_steps_replay_like_eager_ones(clean_error_word, kind):
    users, ctx = 4, 700
    cache, table = _decode_setup(kind, users, ctx, 1)
    eager = [None if c is None else c.clone() for c in cache]
    x = torch.empty(users, (NQ + 2 * NKV) * HD, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(users, dtype=torch.int32, device="cuda")
    x.copy_(_qkv(users, 0))
    pos.fill_(ctx)
    spare = [None if c is None else c.clone() for c in cache]
    for _ in range(2):
        _step(spare, table, x, pos, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(cache, table, x, pos, 5)
    for i in range(4):
        x.copy_(_qkv(users, 20 + i))
        pos.copy_(torch.tensor([ctx + i, ctx + i, -1 if i == 2 else ctx + i, ctx + i]).int())
        graph.replay()
        want = _step(eager, table, x, pos, 5)
        assert torch.equal(out, want)
        for a, b in zip(cache, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_two_graphs_replayed_side_by_side(clean_error_word):
    """Captured on the same stream, replayed at the same time on two: no scratch in common."""
    users, ctx = 2, 6000
    sides = []
    for i in range(2):
        cache, table = _decode_setup("int8_block", users, ctx, i)
        x = _qkv(users, 30 + i).cuda()
        pos = torch.full((users,), ctx, dtype=torch.int32, device="cuda")
        want = _step([c.clone() for c in cache], table, x, pos, 40).clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = _step(cache, table, x, pos, 40)
        inputs = (cache, table, x, pos)          # a graph does not keep what it reads alive
        sides.append((graph, out, want, torch.cuda.Stream(), inputs))
    torch.cuda.synchronize()
    for _ in range(50):
        for graph, _, _, stream, _ in sides:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in sides:
        assert torch.equal(out, want)


def test_eager_calls_on_two_streams(clean_error_word):
    users, ctx = 2, 5000
    sides = []
    for i in range(2):
        cache, table = _decode_setup("int8_block", users, ctx, i)
        x = _qkv(users, 40 + i).cuda()
        pos = torch.full((users,), ctx, dtype=torch.int32, device="cuda")
        want = _step([c.clone() for c in cache], table, x, pos, 30).clone()
        sides.append((cache, table, x, pos, want, torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(30):
        for cache, table, x, pos, _, stream, outs in sides:
            with torch.cuda.stream(stream):
                outs.append(_step(cache, table, x, pos, 30))
    torch.cuda.synchronize()
    for *_, want, _, outs in sides:
        assert all(torch.equal(o, want) for o in outs)


def test_captured_prefill_over_a_scaled_cache(clean_error_word):
    from b200attn import ops

    cache, table = _decode_setup("fp8_block", 2, 200, 3)
    cu = torch.tensor([0, 40, 90], dtype=torch.int32)
    q = torch.randn(90, NQ, HD, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    start = torch.tensor([100, 150], dtype=torch.int32).cuda()
    cu_dev = cu.cuda()

    def run():
        return ops.prefill(q, cache[0], cache[1], cu, page_table=table, q_start=start, cu_q=cu_dev,
                           k_scale=cache[2], v_scale=cache[3])

    want = run().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


def test_a_run_is_the_same_bits_every_time(clean_error_word):
    """Partials are merged in a fixed order whoever merges them."""
    cache, table = _decode_setup("int8_block", 3, 5000, 5)
    x = _qkv(3, 50).cuda()
    pos = torch.full((3,), 5000, dtype=torch.int32, device="cuda")
    first = _step(cache, table, x, pos, 60).clone()
    for _ in range(20):
        assert torch.equal(_step(cache, table, x, pos, 60), first)


def test_a_layer_widens_by_the_longest_sequence(clean_error_word, monkeypatch):
    """A runner's block table is as wide as its longest allowed context."""
    from b200attn import B200AttentionBackendImpl, ops
    from b200attn.backend import build_varlen_metadata

    impl = B200AttentionBackendImpl(NQ, HD, HD ** -0.5, NKV, None, None, "int8_block")
    table = torch.zeros(2, 1024, dtype=torch.int32)
    table[:, :4] = torch.randperm(8, generator=torch.Generator().manual_seed(1)).view(2, 4).int()
    cu, seq = torch.tensor([0, 50, 150]).int(), torch.tensor([50, 100]).int()
    slots = torch.zeros(150, dtype=torch.int64)             # positions come from the block table
    x = _qkv(150, 3).cuda()
    outs, columns = [], []
    widen = ops._widen_scaled_pages

    def note(*a, **kw):
        got = widen(*a, **kw)
        columns.append(got[5])
        return got

    monkeypatch.setattr(ops, "_widen_scaled_pages", note)
    for longest in (100, 0):
        cache = _caches("int8_block", 8, False)
        md = build_varlen_metadata(cu.cuda(), cu, seq.cuda(), table.cuda(), slots.cuda(),
                                   max_seq_len=longest)
        out = torch.empty(150, NQ * HD, dtype=torch.bfloat16, device="cuda")
        impl.forward(None, *[t.contiguous() for t in _split(x)], cache, md, output=out)
        outs.append(out)
    assert columns == [4, 1024] and torch.equal(*outs)


def test_layer_refusals():
    from b200attn import B200AttentionBackendImpl, B200Attention, sharding

    for kw in (dict(sparse_pages=1), dict(sparse_pages=4, sparse_keep_last=0)):
        with pytest.raises(ValueError):
            B200AttentionBackendImpl(NQ, HD, 0.1, NKV, **kw)
    for kw in (dict(sparse_pages=4, sliding_window=64), dict(sparse_pages=4, kv_cache_dtype="fp8")):
        with pytest.raises(NotImplementedError):
            B200AttentionBackendImpl(NQ, HD, 0.1, NKV, **kw)
    w = torch.ones(HD)
    for kw in (dict(q_norm_weight=w), dict(q_norm_weight=w, k_norm_weight=w)):
        with pytest.raises(ValueError):
            B200Attention(NQ, HD, 0.1, NKV, **kw)
    with pytest.raises(NotImplementedError):
        B200Attention(NQ, HD, 0.1, NKV, rotary_dim=HD, is_neox_style=False)
    for kw in (dict(dtype=torch.float16), dict(block_scales=True),
               dict(dtype=torch.float8_e4m3fn, page_bounds=True)):
        with pytest.raises(ValueError):
            sharding.allocate_kv_caches(1, 4, NKV, BS, HD, **kw)
    impl = B200AttentionBackendImpl(NQ, HD, 0.1, NKV, None, None, "int8_block")
    kv = [torch.zeros(1, NKV, BS, HD, dtype=torch.int8)] * 2
    with pytest.raises(ValueError, match="block-scaled"):
        impl._page_values(kv, tuple(kv))
    plain = B200AttentionBackendImpl(NQ, HD, 0.1, NKV)
    with pytest.raises(ValueError, match="scales"):
        plain._page_values(kv + [w, w], tuple(kv))
    sparse = B200AttentionBackendImpl(NQ, HD, 0.1, NKV, sparse_pages=4)
    with pytest.raises(ValueError, match="bounds"):
        sparse._page_values(kv, tuple(kv))


def test_a_captured_prefill_serves_longer_contexts_than_it_was_captured_with(clean_error_word):
    """A bound on the contexts holds for the eager call only."""
    from b200attn import ops

    cache, table = _decode_setup("int8_block", 2, 400, 8)
    cu = torch.tensor([0, 40, 70], dtype=torch.int32)
    q = torch.randn(70, NQ, HD, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    start = torch.zeros(2, dtype=torch.int32).cuda()
    cu_dev = cu.cuda()

    def run(longest):
        return ops.prefill(q, cache[0], cache[1], cu, page_table=table, q_start=start, cu_q=cu_dev,
                           k_scale=cache[2], v_scale=cache[3], max_context_len=longest)

    run(40)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(40)
    for a, b in ((0, 0), (100, 7), (360, 370)):
        start.copy_(torch.tensor([a, b], dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, run(max(a + 40, b + 30)))


def test_prefills_of_two_threads_on_one_stream(clean_error_word):
    """Each attends over the pages it widened, whatever the other enqueues in between."""
    import threading

    from b200attn import ops

    cases = []
    for i in range(2):
        cache, table = _decode_setup("int8_block", 2, 300, 60 + i)
        cu = torch.tensor([0, 33, 97], dtype=torch.int32)
        q = torch.randn(97, NQ, HD, generator=torch.Generator().manual_seed(i)).bfloat16().cuda()
        args = (q, cache[0], cache[1], cu)
        kw = dict(page_table=table, q_start=torch.tensor([200, 230], dtype=torch.int32).cuda(),
                  cu_q=cu.cuda(), k_scale=cache[2], v_scale=cache[3])
        cases.append((args, kw, ops.prefill(*args, **kw).clone()))
    torch.cuda.synchronize()
    outs = [[], []]

    def run(i):
        args, kw, _ = cases[i]
        outs[i] += [ops.prefill(*args, **kw) for _ in range(200)]

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for mine, (_, _, want) in zip(outs, cases):
        assert len(mine) == 200 and all(torch.equal(o, want) for o in mine)


def test_head_norm_weights_on_another_device_are_followed(clean_error_word):
    """Weights on the host, changed in place between two forwards."""
    from b200attn import B200Attention, B200Metadata

    w = [torch.ones(HD).bfloat16(), torch.ones(HD).bfloat16()]
    layer = B200Attention(NQ, HD, HD ** -0.5, NKV, rotary_dim=HD, q_norm_weight=w[0],
                          k_norm_weight=w[1])
    layer.kv_cache = _caches("auto", 2, False)
    md = B200Metadata(cache_position=torch.zeros(1).int().cuda(), num_users=1,
                      page_table=torch.ones(1, 1).int().cuda(), batch_idx=torch.zeros(1).int().cuda())
    for by in (1.0, 2.0, 0.5):
        w[0].mul_(by)
        w[1].mul_(by)
        x = _qkv(1, 3).cuda()
        q, k, v = [t.contiguous() for t in _split(x)]
        before = q.clone()
        layer(q, k, v, attn_metadata=md, positions=torch.zeros(1).long().cuda())
        rows = before.float().view(NQ, HD)
        want = rows * torch.rsqrt(rows.square().mean(-1, keepdim=True) + 1e-6) * w[0].cuda().float()
        err = (q.float().view(NQ, HD) - want).abs()
        assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().amax()).all()
