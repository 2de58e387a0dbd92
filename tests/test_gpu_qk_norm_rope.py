"""Per-head norms + rotation + cache write in one launch, against fp64."""
import pytest
import torch

from oracle import blocks

pytestmark = pytest.mark.gpu

HALF_STEP = torch.finfo(torch.bfloat16).eps / 2     # rounding of the result, relative


def _case(tokens, nq, nkv, hd, rotary, seed, pos_hi=4096, w_dtype=torch.bfloat16, fused=True):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, (nq + 2 * nkv) * hd, generator=g) * 2).bfloat16()
    c = dict(positions=torch.randint(0, pos_hi, (tokens,), generator=g),
             inv_freq=1.0 / 10000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float32) / rotary),
             wq=(1 + 0.3 * torch.randn(hd, generator=g)).to(w_dtype),
             wk=(1 + 0.3 * torch.randn(hd, generator=g)).to(w_dtype))
    dev = qkv.cuda()
    c["host"] = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    c["dev"] = dev.split([nq * hd, nkv * hd, nkv * hd], 1)
    if not fused:
        c["dev"] = tuple(x.contiguous() for x in c["dev"])
    return c


def _close(got, want):
    """One rounding to bf16 of an fp32 result.  fp32 part: the norm and each product are off by a
    few 2^-24 relative to the head's entries, the angle by 2^-22 of a radian, so the rotated sum is
    off by less than 2^-20 of the largest entry of its head."""
    got = got.double().cpu()
    head_max = want.abs().amax(-1, keepdim=True)
    err = (got - want).abs()
    assert (err <= HALF_STEP * want.abs() + 2.0 ** -20 * head_max).all(), err.max()


@pytest.mark.parametrize("tokens,nq,nkv,hd,rotary,neox", [
    (1, 1, 1, 64, 64, True), (1, 32, 8, 128, 128, True), (7, 32, 8, 64, 64, True),
    (33, 5, 5, 128, 32, True), (16, 6, 2, 64, 48, True), (9, 64, 8, 128, 128, False),
    (130, 24, 3, 64, 16, False), (5, 7, 1, 128, 96, False), (257, 8, 8, 64, 32, True),
])
@pytest.mark.parametrize("fused", [True, False])
def test_norm_and_rotation(clean_error_word, tokens, nq, nkv, hd, rotary, neox, fused):
    from b200attn import ops

    c = _case(tokens, nq, nkv, hd, rotary, seed=tokens + nq, fused=fused)
    q, k, _ = c["dev"]
    before = [x.clone() for x in c["dev"]]
    oq = torch.full((tokens, nq * hd), 7.0, dtype=torch.bfloat16, device="cuda")
    ok = torch.full((tokens, nkv * hd), 7.0, dtype=torch.bfloat16, device="cuda")
    rq, rk = ops.qk_norm_rope_kv_scatter_slots(
        q, k, None, c["positions"].cuda(), c["inv_freq"].cuda(), rotary, hd, c["wq"].cuda(),
        c["wk"].cuda(), 1e-5, is_neox_style=neox, out_query=oq, out_key=ok)
    assert rq is oq and rk is ok
    for x, b in zip(c["dev"], before):
        assert torch.equal(x, b), "an input changed"
    for got, x, w in ((oq, c["host"][0], c["wq"]), (ok, c["host"][1], c["wk"])):
        want = blocks.qk_norm_rope(x, c["positions"], c["inv_freq"], rotary, hd, w, 1e-5, neox)
        _close(got.reshape(tokens, -1, hd), want.reshape(tokens, -1, hd))
    # in place: the same bits
    iq, ik = ops.qk_norm_rope_kv_scatter_slots(
        q, k, None, c["positions"].cuda(), c["inv_freq"].cuda(), rotary, hd, c["wq"].cuda(),
        c["wk"].cuda(), 1e-5, is_neox_style=neox)
    assert iq.data_ptr() == q.data_ptr() and ik.data_ptr() == k.data_ptr()
    assert torch.equal(iq, oq) and torch.equal(ik, ok)
    assert torch.equal(c["dev"][2], before[2]), "value changed"


def test_far_positions_and_fp32_weights(clean_error_word):
    from b200attn import ops

    c = _case(64, 4, 2, 128, 128, seed=5, w_dtype=torch.float32)
    c["positions"] = torch.arange(64) * 33333331 + 7            # up to 2.1e9
    q, k, _ = c["dev"]
    rq, rk = ops.qk_norm_rope_kv_scatter_slots(
        q, k, None, c["positions"].cuda(), c["inv_freq"].cuda(), 128, 128, c["wq"].cuda(),
        c["wk"].cuda(), 0.0)
    for got, x, w in ((rq, c["host"][0], c["wq"]), (rk, c["host"][1], c["wk"])):
        want = blocks.qk_norm_rope(x, c["positions"], c["inv_freq"], 128, 128, w, 0.0, True)
        _close(got.reshape(64, -1, 128), want.reshape(64, -1, 128))


def test_zero_rows_stay_zero(clean_error_word):
    from b200attn import ops

    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(3, 2 * 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, device="cuda")
    rq, rk = ops.qk_norm_rope_kv_scatter_slots(
        q, k, None, torch.arange(3).cuda(), torch.ones(32, device="cuda"), 64, 64, w, w)
    assert not rq.any() and not rk.any()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("hd,bs,rotary", [(64, 32, 64), (128, 64, 64), (128, 32, 128)])
def test_cache_write_is_the_scatter_of_the_results(clean_error_word, kind, hd, bs, rotary):
    from b200attn import ops

    tokens, nq, nkv = 45, 8, 4
    c = _case(tokens, nq, nkv, hd, rotary, seed=hd + bs)
    nb = 5
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(3))[:tokens]
    slots[::7] = -1
    kc = torch.zeros(nb, nkv, bs, hd, device="cuda").to(kind)
    vc, kc2, vc2 = kc.clone(), kc.clone(), kc.clone()
    q, k, v = c["dev"]
    rq, rk = ops.qk_norm_rope_kv_scatter_slots(
        q, k, v, c["positions"].cuda(), c["inv_freq"].cuda(), rotary, hd, c["wq"].cuda(),
        c["wk"].cuda(), 1e-6, kc, vc, slots.cuda())
    ops.kv_scatter_slots(kc2, vc2, rk.reshape(tokens, nkv, hd), v.reshape(tokens, nkv, hd),
                         slots.cuda())
    assert torch.equal(kc.view(torch.uint8), kc2.view(torch.uint8))
    assert torch.equal(vc.view(torch.uint8), vc2.view(torch.uint8))


def test_outputs_side_by_side_in_one_buffer(clean_error_word):
    from b200attn import ops

    c = _case(9, 4, 2, 64, 64, seed=8)
    q, k, v = c["dev"]
    args = (c["positions"].cuda(), c["inv_freq"].cuda(), 64, 64, c["wq"].cuda(), c["wk"].cuda())
    both = torch.zeros(9, 6 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    ops.qk_norm_rope_kv_scatter_slots(q, k, None, *args, out_query=both[:, : 4 * 64],
                                      out_key=both[:, 4 * 64: 6 * 64])
    assert not both[:, 6 * 64:].any()
    iq, ik = ops.qk_norm_rope_kv_scatter_slots(q, k, None, *args)
    assert torch.equal(both[:, : 4 * 64], iq) and torch.equal(both[:, 4 * 64: 6 * 64], ik)


def test_a_slot_twice_takes_one_of_the_rows(clean_error_word):
    from b200attn import ops

    c = _case(2, 2, 1, 64, 64, seed=1)
    q, k, v = c["dev"]
    kc = torch.zeros(2, 1, 32, 64, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    ops.qk_norm_rope_kv_scatter_slots(
        q, k, v, c["positions"].cuda(), c["inv_freq"].cuda(), 64, 64, c["wq"].cuda(),
        c["wk"].cuda(), 1e-6, kc, vc, torch.tensor([7, 7]).cuda())
    got = torch.stack([kc[0, 0, 7], vc[0, 0, 7]])
    assert ((got[0] == k[0]) | (got[0] == k[1])).all() and ((got[1] == v[0]) | (got[1] == v[1])).all()
    kc[0, 0, 7] = 0
    assert not kc.any()


def test_slots_outside_the_cache_are_skipped_and_reported():
    from b200attn import ops

    ops.read_error_word()
    c = _case(3, 2, 1, 64, 64, seed=1)
    kc = torch.zeros(2, 1, 32, 64, dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    q, k, v = c["dev"]
    ops.qk_norm_rope_kv_scatter_slots(
        q, k, v, c["positions"].cuda(), c["inv_freq"].cuda(), 64, 64, c["wq"].cuda(),
        c["wk"].cuda(), 1e-6, kc, vc, torch.tensor([64, 1 << 40, 5]).cuda())
    assert ops.read_error_word() == 2
    assert torch.equal(kc[0, 0, 5], k[2]) and torch.equal(vc[0, 0, 5], v[2])
    kc[0, 0, 5] = 0
    vc[0, 0, 5] = 0
    assert not kc.any() and not vc.any()


def test_refusals():
    from b200attn import ops
    from b200attn._lib import B200AttnError

    c = _case(4, 4, 2, 64, 64, seed=2, fused=False)
    q, k, v = c["dev"]
    pos, inv, wq, wk = c["positions"].cuda(), c["inv_freq"].cuda(), c["wq"].cuda(), c["wk"].cuda()

    def call(q=q, k=k, v=v, pos=pos, inv=inv, rotary=64, hd=64, wq=wq, wk=wk, **kw):
        return ops.qk_norm_rope_kv_scatter_slots(q, k, v, pos, inv, rotary, hd, wq, wk, **kw)

    for bad in (dict(q=q.float()), dict(q=q[:3]), dict(pos=pos.int()), dict(inv=inv[:8]),
                dict(wq=wq[:32], wk=wk[:32]), dict(wq=wq.float()), dict(q=q[:, :100]),
                dict(out_query=q[:, :64]), dict(slot_mapping=pos), dict(inv=inv.half())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="overlap"):
        call(out_key=q[:, : 2 * 64])
    with pytest.raises(ValueError, match="overlap"):                   # shifted by one head
        big = torch.zeros(4, 5 * 64, dtype=torch.bfloat16, device="cuda")
        call(q=big[:, : 4 * 64], out_query=big[:, 64:])
    with pytest.raises(ValueError, match="overlap"):                   # both in place, one memory
        call(q=k, k=k)
    row = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device="cuda").expand(4, -1)
    with pytest.raises(B200AttnError):                                 # rows on top of each other
        call(q=row, out_query=torch.empty_like(q))
    with pytest.raises(B200AttnError):
        call(q=row, out_query=row)
    with pytest.raises(B200AttnError):                                 # not a multiple of 16
        call(rotary=24, inv=inv[:12].clone())
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(wq=wq.cpu())
    call()


def test_value_rows_under_an_output_are_refused():
    """The value is read while rows are stored: it may not lie under a result, in place or not."""
    from b200attn import ops

    c = _case(4, 4, 2, 64, 64, seed=2, fused=False)
    q, k, v = c["dev"]
    args = (c["positions"].cuda(), c["inv_freq"].cuda(), 64, 64, c["wq"].cuda(), c["wk"].cuda())
    kc = torch.zeros(2, 2, 32, 64, dtype=torch.bfloat16, device="cuda")
    write = dict(eps=1e-6, k_cache=kc, v_cache=kc.clone(), slot_mapping=torch.arange(4).cuda())
    before = q.clone(), k.clone()
    for value, outs in ((k, {}), (k, dict(out_query=torch.empty_like(q))), (q[:, :128], {}),
                        (q[:, 64:192], dict(out_key=torch.empty_like(k))),
                        (v, dict(out_query=torch.empty_like(q), out_key=v))):
        with pytest.raises(ValueError, match="overlap"):
            ops.qk_norm_rope_kv_scatter_slots(q, k, value, *args, **write, **outs)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1]) and not kc.any()
    ops.qk_norm_rope_kv_scatter_slots(q, k, k, *args)        # nothing reads the value here
