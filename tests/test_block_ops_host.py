"""Refusals of the block-scaled / page-list / norm entry points, and the shapes that
allocate_kv_caches makes for them: no GPU needed, nothing is launched."""
import functools
import threading
import time
from types import SimpleNamespace

import pytest
import torch

from b200attn import _lib, sharding

OK, NULL, UNSUPPORTED, MISALIGNED, WORKSPACE, BAD, NO_DEVICE = 0, -1, -2, -3, -4, -5, -6
BF16, FP8, INT8 = 0, 1, 2


@pytest.fixture()
def L(built_library):
    return _lib.lib()


def _call(fn, args, **changes):
    args = dict(args)
    for name, value in changes.items():
        assert name in args, name
        args[name] = value
    return fn(*args.values())


WRITE = dict(k=16, v=16, ks=16, vs=16, bounds=None, kind=INT8, kn=16, kstride=256, vn=16,
             vstride=256, table=16, tstride=4, width=4, cu=None, qlen=None, start=16, seqs=2,
             tokens=2, nkv=2, hd=128, bs=32, nb=8, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(k=None), NULL), (dict(start=None), NULL), (dict(ks=None), NULL), (dict(table=None), NULL),
    (dict(kind=BF16), BAD), (dict(kind=7), BAD), (dict(seqs=-1), BAD), (dict(width=0), BAD),
    (dict(tokens=3), BAD), (dict(kstride=128), BAD), (dict(nkv=0), BAD), (dict(nb=0), BAD),
    (dict(hd=96), UNSUPPORTED), (dict(bs=16), UNSUPPORTED), (dict(kn=8), MISALIGNED),
    (dict(vstride=260), MISALIGNED), (dict(bounds=4), MISALIGNED),
])
def test_paged_write_refusals(L, changes, status):
    assert _call(L.b200attn_paged_write, WRITE, **changes) == status


DECODE = dict(out=16, ostride=1024, q=16, qstride=1024, k=16, v=16, ks=16, vs=16, kind=INT8,
              table=16, tstride=4, hstride=0, width=4, pos=16, users=2, nq=8, nkv=2, hd=128, bs=32,
              nb=8, scale=1.0, window=0, sinks=None, ctx=0, splits=0, ws=None, wsbytes=0,
              stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(vs=None), NULL), (dict(q=None), NULL), (dict(kind=BF16), BAD), (dict(kind=9), BAD),
    (dict(ks=None, vs=None, kind=INT8), BAD), (dict(ks=None, vs=None, kind=FP8, hd=64), UNSUPPORTED),
    (dict(hstride=4, window=8), UNSUPPORTED), (dict(hstride=-4), BAD), (dict(scale=0.0), BAD),
    (dict(nq=34, qstride=8192, ostride=8192), UNSUPPORTED), (dict(nq=7), BAD),
    (dict(splits=-1), BAD), (dict(splits=300), -8), (dict(qstride=512), BAD), (dict(q=8), MISALIGNED),
    (dict(window=-1), BAD),
])
def test_paged_decode_blocks_refusals(L, changes, status):
    assert _call(L.b200attn_paged_decode_blocks, DECODE, **changes) == status


SELECT = dict(table_out=16, pos_out=16, q=16, qstride=1024, bounds=16, table=16, tstride=8, width=8,
              pos=16, users=2, nq=8, nkv=2, hd=128, bs=64, nb=8, pages=4, first=1, last=1, ctx=0,
              ws=None, wsbytes=0, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(q=None), NULL), (dict(bounds=None), NULL), (dict(pages=0), BAD), (dict(last=0), BAD),
    (dict(first=-1), BAD), (dict(first=3, last=2), BAD), (dict(nq=9), BAD), (dict(width=0), BAD),
    (dict(nq=40, qstride=8192), UNSUPPORTED), (dict(hd=32), UNSUPPORTED), (dict(bs=128), UNSUPPORTED),
    (dict(bounds=8), MISALIGNED), (dict(qstride=512), BAD), (dict(pages=1 << 30, first=0), -8),
    (dict(first=2 ** 31 - 1, last=2 ** 31 - 1), BAD),
])
def test_select_pages_refusals(L, changes, status):
    assert _call(L.b200attn_select_pages, SELECT, **changes) == status


NORM = dict(oq=16, oqs=512, ok=16, oks=128, q=16, qs=512, k=16, ks=128, v=16, vs=128, wq=16, wk=16,
            f32=0, eps=1e-6, pos=16, inv=16, rotary=64, neox=1, kc=16, vc=16, kind=BF16, slots=16,
            tokens=3, nq=8, nkv=2, hd=64, bs=32, nb=4, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(oq=None), NULL), (dict(wk=None), NULL), (dict(kc=None), NULL), (dict(v=None), NULL),
    (dict(eps=-1.0), BAD), (dict(eps=float("nan")), BAD), (dict(rotary=24), UNSUPPORTED),
    (dict(rotary=80), UNSUPPORTED), (dict(rotary=0), UNSUPPORTED), (dict(hd=80), UNSUPPORTED),
    (dict(kind=INT8), BAD), (dict(bs=48), UNSUPPORTED), (dict(tokens=-1), BAD), (dict(qs=504), BAD),
    (dict(qs=516), MISALIGNED), (dict(wq=8), MISALIGNED), (dict(vs=64), BAD),
])
def test_qk_norm_rope_refusals(L, changes, status):
    assert _call(L.b200attn_qk_norm_rope_kv_scatter_slots, NORM, **changes) == status


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_nothing_runs_without_a_device(L):
    for fn, args in ((L.b200attn_paged_write, WRITE), (L.b200attn_paged_decode_blocks, DECODE),
                     (L.b200attn_select_pages, SELECT),
                     (L.b200attn_qk_norm_rope_kv_scatter_slots, NORM)):
        assert fn(*args.values()) == NO_DEVICE


def test_workspace_sizes(L):
    small = L.b200attn_decode_scaled_workspace_bytes(2, 8, 2, 128, 0)
    assert small >= 65536 + 2 * 2 * 64 * 4 * (128 * 4 + 8)
    # more users do not grow it beyond the launch's CTAs; explicit splits do
    assert L.b200attn_decode_scaled_workspace_bytes(4096, 8, 2, 128, 0) == \
        L.b200attn_decode_scaled_workspace_bytes(1024, 8, 2, 128, 0)
    assert L.b200attn_decode_scaled_workspace_bytes(1024, 8, 2, 128, 8) >= \
        65536 + 1024 * 2 * 8 * 4 * (128 * 4 + 8)
    assert L.b200attn_decode_scaled_workspace_bytes(0, 8, 2, 128, 0) == 0
    assert L.b200attn_select_pages_workspace_bytes(3, 2, 100) == 65536 + 600 * 16


def test_allocated_caches():
    def shapes(**kw):
        pair = sharding.allocate_kv_caches(2, 6, 4, 32, 64, tp_size=2, **kw)["layers.1.attn"]
        return [None if t is None else (tuple(t.shape), t.dtype) for t in pair]

    scale = ((6, 2), torch.float32)
    bounds = ((6, 2, 2, 64), torch.bfloat16)
    rows = (6, 2, 32, 64)
    assert shapes() == [(rows, torch.bfloat16)] * 2
    assert shapes(dtype=torch.int8) == [(rows, torch.int8)] * 2 + [scale] * 2
    assert shapes(dtype=torch.float8_e4m3fn) == [(rows, torch.float8_e4m3fn)] * 2
    assert shapes(dtype=torch.float8_e4m3fn, block_scales=True, page_bounds=True) == \
        [(rows, torch.float8_e4m3fn)] * 2 + [scale] * 2 + [bounds]
    assert shapes(page_bounds=True) == [(rows, torch.bfloat16)] * 2 + [None] * 2 + [bounds]


def test_ops_refuse_cpu_tensors():
    from b200attn import ops

    kc = torch.zeros(4, 2, 32, 64, dtype=torch.int8)
    s = torch.zeros(4, 2)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    table, pos = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    w = torch.ones(64)
    for call in (lambda: ops.paged_write(kc, kc, x, x, table, pos, k_scale=s, v_scale=s),
                 lambda: ops.paged_decode(x, kc, kc, table, pos, k_scale=s, v_scale=s),
                 lambda: ops.select_pages(x, torch.zeros(4, 2, 2, 64).bfloat16(), table, pos, 32, 4),
                 lambda: ops.qk_norm_rope_kv_scatter_slots(
                     x.flatten(1), x.flatten(1), None, torch.zeros(1, dtype=torch.int64),
                     torch.ones(32), 64, 64, w, w)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def _row_sets():
    """40 tokens of 4 query heads and 2 + 2 KV heads of 64 side by side in rows of 512 elements, and
    memory apart, as (pointer, row stride, row width) in bytes."""
    step = 2 * 8 * 64
    q, k, v = (4096, step, 512), (4096 + 512, step, 256), (4096 + 768, step, 256)
    far = 1 << 20
    return q, k, v, (far, 512, 512), (far + 40 * 512, 256, 256)


def test_outputs_that_overlap_nothing_they_may_not_are_taken():
    from b200attn.ops import _check_outputs

    q, k, v, oq, ok = _row_sets()
    unread = (0, 0, 256)
    for outs in ((q, k), (oq, ok), (q, ok), (oq, k)):
        for val in (v, unread):
            _check_outputs(40, *outs, q, k, val)
    # value where a key goes is nothing to a call that does not read it
    _check_outputs(40, q, k, q, k, unread)
    for n in (1, 40):                                    # memory side by side, strides apart
        _check_outputs(n, (0, 512, 512), (n * 512, 256, 256), (0, 512, 512), (n * 512, 256, 256),
                       (n * 768, 256, 256))


@pytest.mark.parametrize("tokens", [1, 40])
def test_outputs_that_overlap_what_is_still_read_are_refused(tokens):
    """In place or not: an output on the value's rows, on the other input's, on the other output's,
    or on part of its own input's."""
    from b200attn.ops import _check_outputs

    q, k, v, oq, ok = _row_sets()
    half = (k[0] + 128, k[1], k[2])
    for outs, ins in (((q, k), (q, k, k)),               # value is the key, both in place
                      ((oq, k), (q, k, k)), ((q, ok), (q, k, q)), ((q, k), (q, k, q)),
                      ((q, v), (q, k, v)), ((v, ok), (q, k, v)), ((oq, k), (q, k, half)),
                      ((q, ok), (q, q, v)), ((oq, k), (k, k, v)), ((q, k), (q, half, v)),
                      ((oq, half), (q, k, v)), ((k, ok), (q, k, v)), ((oq, oq), (q, k, v))):
        with pytest.raises(ValueError, match="overlap"):
            _check_outputs(tokens, *outs, *ins)


class _RecordingLibrary:
    """Stands in for the library: notes which memory each launch is given; a `meet` barrier holds
    every thread between its two launches until all of them are there."""

    def __init__(self, meet=None):
        self.meet, self.widened, self.attended, self.order = meet, {}, {}, []

    def _note_widened(self, spans):
        self.widened[threading.get_ident()] = spans
        if self.meet is not None:
            self.meet.wait(30)
        return 0

    def b200attn_dequant_pages_scaled_ex(self, k, v, factors, *rest):
        width, limit, seqs, nkv, hd, bs = rest[7], *rest[10:15]
        self.columns = (width, limit)
        pages = seqs * width
        half = pages * nkv * bs * hd * 2
        return self._note_widened([(k, half), (v, half), (factors, pages * nkv * 8)])

    def b200attn_dequant_pages_fp8(self, k, v, *rest):
        self.order.append(("widen", threading.get_ident()))
        if self.meet is not None:
            time.sleep(0.05)                     # time for another thread to come in between
        return 0

    def b200attn_prefill_ex(self, *args):
        self.order.append(("attend", threading.get_ident()))
        return 0

    def b200attn_prefill_scaled(self, out, ostride, q, qstride, k, v, factors, *rest):
        assert rest[2] == self.columns[0]
        self.attended[threading.get_ident()] = [k, v, factors]
        return 0


@pytest.fixture()
def stubbed(monkeypatch):
    """ops on CPU tensors against a recording library."""
    from b200attn import ops

    def use(library):
        monkeypatch.setattr(ops._lib, "lib", lambda: library)
        for name, value in (("_need_cuda", lambda *t: None), ("_device_of", lambda *t: 0),
                            ("_current_device", lambda: 0), ("_raw_stream", lambda index: 7),
                            ("_stream", lambda t: 7)):
            monkeypatch.setattr(ops, name, value)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        return ops

    return use


def _prefill_call(ops, kind, seqs=2, width=4, scaled=True, **kw):
    cache = torch.zeros(8, 2, 32, 128).to(kind)
    scales = dict(k_scale=torch.ones(8, 2), v_scale=torch.ones(8, 2)) if scaled else {}
    cu = torch.arange(seqs + 1, dtype=torch.int32) * 3
    return ops.prefill(torch.zeros(3 * seqs, 4, 128, dtype=torch.bfloat16), cache, cache.clone(), cu,
                       page_table=torch.zeros(seqs, width, dtype=torch.int32), cu_q=cu,
                       q_start=torch.zeros(seqs, dtype=torch.int32), **scales, **kw)


def _check_each_thread_attends_what_it_widened(lib, threads):
    spans = []
    assert len(lib.widened) == len(lib.attended) == threads
    for thread, mine in lib.widened.items():
        assert lib.attended[thread] == [at for at, _ in mine]
        spans += mine
    spans.sort()
    assert all(a + n <= b for (a, n), (b, _) in zip(spans, spans[1:]))


def _in_threads(n, call):
    errors = []

    def run():
        try:
            call()
        except Exception as e:                   # noqa: BLE001  (reported by the caller's thread)
            errors.append(e)

    threads = [threading.Thread(target=run) for _ in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_prefills_on_one_stream_widen_into_pools_of_their_own(stubbed):
    """Three threads have all widened their pages before the first of them attends."""
    lib = _RecordingLibrary(threading.Barrier(3))
    ops = stubbed(lib)
    _in_threads(3, lambda: _prefill_call(ops, torch.int8))
    _check_each_thread_attends_what_it_widened(lib, 3)


def test_unscaled_e4m3_prefills_do_not_come_between_each_other(stubbed, monkeypatch):
    """The pool of a stream is shared: who has widened into it attends before anyone else widens."""
    lib = _RecordingLibrary(threading.Barrier(1))
    ops = stubbed(lib)
    monkeypatch.setattr(ops, "_fp8_scratch", {})
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: SimpleNamespace(cuda_stream=7))
    _in_threads(3, lambda: _prefill_call(ops, torch.float8_e4m3fn, scaled=False))
    assert len(lib.order) == 6
    for first, second in zip(lib.order[::2], lib.order[1::2]):
        assert first == ("widen", first[1]) and second == ("attend", first[1])


@pytest.mark.parametrize("hint,columns", [(0, 2048), (1, 1), (32, 1), (33, 2), (100, 4),
                                          (65536, 2048), (1 << 30, 2048)])
def test_widening_goes_by_the_longest_context(stubbed, monkeypatch, hint, columns):
    """Not by the width of the page table, where the caller says how long contexts are; a captured
    call keeps all columns."""
    lib = _RecordingLibrary()
    ops = stubbed(lib)
    sizes = []
    new_empty = torch.Tensor.new_empty
    monkeypatch.setattr(torch.Tensor, "new_empty",
                        lambda t, *a, **kw: sizes.append(a) or new_empty(t, *a, **kw))
    _prefill_call(ops, torch.int8, width=2048, max_context_len=hint)
    assert lib.columns == (columns, hint)
    assert (2 * columns * 2 * 32 * 128 * 4 + 2 * columns * 2 * 8,) in sizes
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    _prefill_call(ops, torch.int8, width=2048, max_context_len=hint)
    assert lib.columns == (2048, 0)


def test_a_negative_longest_context_is_refused(stubbed):
    with pytest.raises(ValueError, match="max_context_len"):
        _prefill_call(stubbed(_RecordingLibrary()), torch.int8, max_context_len=-1)


WIDEN = dict(kd=16, vd=16, f=16, k=16, v=16, ks=16, vs=16, kind=INT8, table=16, tstride=4, width=4,
             cu=16, start=16, ctx=0, seqs=2, nkv=2, hd=128, bs=32, nb=8, stream=None)


@pytest.mark.parametrize("changes,status", [
    (dict(kd=None), NULL), (dict(f=None), NULL), (dict(ks=None), NULL), (dict(cu=None), NULL),
    (dict(kind=BF16), BAD), (dict(width=0), BAD), (dict(seqs=-1), BAD), (dict(ctx=-1), BAD),
    (dict(hd=96), UNSUPPORTED), (dict(vd=8), MISALIGNED), (dict(seqs=1 << 30), -8),
])
def test_dequant_pages_scaled_refusals(L, changes, status):
    assert _call(L.b200attn_dequant_pages_scaled_ex, WIDEN, **changes) == status
    if "ctx" not in changes:
        old = {n: x for n, x in {**WIDEN, **changes}.items() if n != "ctx"}
        assert L.b200attn_dequant_pages_scaled(*old.values()) == status


def test_identity_tables(monkeypatch):
    """One per stream, whatever sizes ask for it; a capture makes its own."""
    from b200attn import ops

    monkeypatch.setattr(ops, "_identity_tables", {})
    dev = torch.device("cpu")
    for pages in (1, 15, 4096, 4097, 10000, 18):
        got = ops._identity_table(dev, 1, pages, False)
        assert got.dtype == torch.int32 and got.numel() >= pages
        assert torch.equal(got, torch.arange(got.numel(), dtype=torch.int32))
    assert list(ops._identity_tables) == [(None, 1)] and ops._identity_tables[(None, 1)] is got
    own = ops._identity_table(dev, 1, 6, True)
    assert own is not got and own.tolist() == list(range(6))
    assert ops._identity_table(dev, 2, 6, False) is not got
    assert list(ops._identity_tables) == [(None, 1), (None, 2)]


@pytest.mark.parametrize("kw", [dict(dtype=torch.int8), dict(page_bounds=True),
                                dict(dtype=torch.float8_e4m3fn, block_scales=True),
                                dict(dtype=torch.float8_e4m3fn, block_scales=True, page_bounds=True)])
def test_write_to_kv_cache_refuses_what_it_would_leave_stale(stubbed, kw):
    """A slot write knows nothing of a page's scales or bounds."""
    from b200attn.backend import write_to_kv_cache

    stubbed(SimpleNamespace(b200attn_kv_scatter_slots_ex=lambda *a: 0,
                            b200attn_kv_scatter_slots=lambda *a: 0))
    cache = sharding.allocate_kv_caches(1, 6, 2, 32, 64, **kw)["layers.0.attn"]
    rows = torch.ones(3, 2 * 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="paged_write"):
        write_to_kv_cache(rows, rows, cache, torch.arange(3))


@pytest.mark.parametrize("extra", [[], [None, None], [None, None, None]])
def test_write_to_kv_cache_takes_plain_caches(stubbed, extra, monkeypatch):
    from b200attn import backend

    calls = []
    monkeypatch.setattr(backend.ops, "kv_scatter_slots", lambda *a: calls.append(a))
    pair = sharding.allocate_kv_caches(1, 6, 2, 32, 64)["layers.0.attn"]
    rows = torch.ones(3, 2 * 64, dtype=torch.bfloat16)
    backend.write_to_kv_cache(rows, rows, list(pair) + extra, torch.arange(3))
    backend.write_to_kv_cache(rows, rows, torch.stack(pair), torch.arange(3))
    assert len(calls) == 2 and calls[0][0] is pair[0] and calls[0][2].shape == (3, 2, 64)


class _NormCalls(list):
    """Takes the place of ops.qk_norm_rope_kv_scatter_slots: keeps the weights of every call."""

    def __call__(self, q, k, v, positions, inv_freq, rotary, hd, wq, wk, *rest, **kw):
        self.append((wq, wk, wq.clone(), wk.clone()))
        return q, k


def _norm_layer(monkeypatch, wq, wk):
    from b200attn import B200Attention, backend

    calls = _NormCalls()
    monkeypatch.setattr(backend.ops, "qk_norm_rope_kv_scatter_slots", calls)
    layer = B200Attention(4, 64, 0.125, 2, rotary_dim=64, q_norm_weight=wq, k_norm_weight=wk)
    monkeypatch.setattr(layer.impl, "forward", lambda *a, output, **kw: output.zero_())
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16)
    kv = torch.zeros(3, 2, 2 * 64, dtype=torch.bfloat16)
    return calls, lambda pos=torch.arange(3): layer(q, kv[:, 0], kv[:, 1], positions=pos)


def test_a_layer_with_head_norms_refuses_a_call_without_positions(monkeypatch):
    calls, forward = _norm_layer(monkeypatch, torch.ones(64), torch.ones(64))
    with pytest.raises(ValueError, match="positions"):
        forward(None)
    assert not calls
    forward()
    assert len(calls) == 1


@pytest.mark.parametrize("make", [lambda: torch.ones(64), lambda: torch.nn.Parameter(torch.ones(64)),
                                  lambda: torch.ones(128)[::2]])
def test_a_layer_sees_head_norm_weights_that_change(monkeypatch, make):
    """Loaded after the layer was made, or again later; a copy, where one is needed, keeps its
    address."""
    wq, wk = make(), make()
    calls, forward = _norm_layer(monkeypatch, wq, wk)
    with torch.inference_mode():
        forward()
    with torch.no_grad():
        wq.copy_(torch.arange(64.0))
    forward()
    with torch.no_grad():
        wk.mul_(3.0)
    forward()
    want_q = [torch.ones(64), torch.arange(64.0), torch.arange(64.0)]
    want_k = [torch.ones(64), torch.ones(64), torch.full((64,), 3.0)]
    for call, q, k in zip(calls, want_q, want_k):
        assert torch.equal(call[2], q) and torch.equal(call[3], k)
        assert call[0].is_contiguous() and call[1].is_contiguous()
    assert len({c[0].data_ptr() for c in calls}) == 1 and len({c[1].data_ptr() for c in calls}) == 1
    if isinstance(wq, torch.nn.Parameter):               # a module that is moved swaps the data
        wq.data = torch.full((64,), 5.0)
        forward()
        assert torch.equal(calls[-1][2], torch.full((64,), 5.0))


def test_a_layer_takes_head_norm_weights_made_in_inference_mode(monkeypatch):
    with torch.inference_mode():
        w = torch.ones(128)[::2]
    calls, forward = _norm_layer(monkeypatch, w, w)
    forward()
    forward()
    assert len(calls) == 2 and torch.equal(calls[1][2], torch.ones(64))


@pytest.mark.parametrize("which", ["key", "query", "part"])
def test_a_layer_with_head_norms_refuses_a_value_that_is_rotated_away(monkeypatch, which):
    """Also where the cache write comes later (block-scaled caches): the value would be read after
    the key was normed and rotated in place."""
    from b200attn import B200Attention, backend

    calls = _NormCalls()
    monkeypatch.setattr(backend.ops, "qk_norm_rope_kv_scatter_slots", calls)
    w = torch.ones(64)
    layer = B200Attention(4, 64, 0.125, 2, rotary_dim=64, q_norm_weight=w, k_norm_weight=w)
    monkeypatch.setattr(layer.impl, "forward", lambda *a, output, **kw: output.zero_())
    rows = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    q, k, v = rows.split([256, 128, 128], 1)
    bad = {"key": k, "query": q[:, :128], "part": rows[:, 320:448]}[which]
    with pytest.raises(ValueError, match="shares memory"):
        layer(q, k, bad, positions=torch.arange(3))
    assert not calls
    layer(q, k, v, positions=torch.arange(3))
    assert len(calls) == 1


def test_split_counts_of_page_lists_are_kept_per_device(stubbed, monkeypatch):
    """They go by the SM count of the device that is current."""
    at, splits = [0], []
    library = SimpleNamespace(
        b200attn_decode_auto_splits=lambda *a: 1 + at[0],
        b200attn_decode_workspace_bytes=lambda *a: 0,
        b200attn_paged_decode_blocks=lambda *a: splits.append(a[24]) or 0)
    ops = stubbed(library)
    monkeypatch.setattr(ops, "_device_of", lambda *t: at[0])
    monkeypatch.setattr(ops, "_current_device", lambda: at[0])
    for kept in (ops._list_splits, ops._decode_bytes):
        monkeypatch.setattr(ops, kept.__name__, functools.lru_cache(kept.__wrapped__))
    cache = torch.zeros(4, 2, 32, 64, dtype=torch.bfloat16)
    for device in (0, 3, 0):
        at[0] = device
        ops.paged_decode(torch.zeros(1, 2, 64, dtype=torch.bfloat16), cache, cache,
                         torch.zeros(1, 2, 3, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32))
    assert splits == [1, 4, 1]


def test_prefill_over_a_scaled_cache_refuses_cpu_tensors():
    from b200attn import ops

    with pytest.raises(RuntimeError, match="no CPU path"):
        _prefill_call(ops, torch.int8)
    with pytest.raises(ValueError, match="paged cache"):
        x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
        ops.prefill(x, x, x, torch.tensor([0, 2], dtype=torch.int32), k_scale=torch.ones(1, 2),
                    v_scale=torch.ones(1, 2))
