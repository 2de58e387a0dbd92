"""Plain restatements of the cache-side operators that have no counterpart in the reference: norms
with the rotation, the block-scaled cache write, attention over block-scaled pages and page
selection.  fp64 on the CPU, one page / head / row at a time (test infrastructure only); the parts
that the operators define in fp32 (scales and codes) are computed in fp32, so they are bit-exact."""
from __future__ import annotations

import math

import numpy as np
import torch

QMAX = {torch.int8: np.float32(127.0), torch.float8_e4m3fn: np.float32(448.0)}


def qk_norm_rope(x, positions, inv_freq, rotary, head_size, weight, eps, neox):
    """[tokens, heads * head_size] -> fp64 rows after norm and rotation."""
    t = x.shape[0]
    y = x.double().reshape(t, -1, head_size)
    y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / head_size + eps) * weight.double()
    f = positions.double()[:, None] * inv_freq.double()[None, :]
    c, s = torch.cos(f)[:, None, :], torch.sin(f)[:, None, :]
    i = torch.arange(rotary // 2)
    ia, ib = (i, i + rotary // 2) if neox else (2 * i, 2 * i + 1)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia] = a * c - b * s
    y[..., ib] = b * c + a * s
    return y.reshape(t, -1)


def encode(x: np.ndarray, scale: np.float32, kind) -> torch.Tensor:
    """fp32 values -> codes (NaN scale or zero scale: zeros)."""
    if not scale > 0:
        return torch.zeros(x.shape, dtype=torch.float32).to(kind)
    with np.errstate(over="ignore"):
        q = torch.from_numpy((x / scale).astype(np.float32))
    if kind == torch.int8:
        return q.round().clamp(-127, 127).to(torch.int8)
    return q.clamp(-448.0, 448.0).to(kind)


def _write_page(codes, scale, rows, r0, kind):
    """codes [bs, hd] and scale (np.float32) of one page and head after `rows` ([n, hd] bf16) were
    written at row r0."""
    x = rows.float().numpy()
    qmax = QMAX[kind]
    finite = np.isfinite(x).all()
    need = np.float32(np.abs(x).max()) * (np.float32(1.0) / qmax) if finite else np.float32(np.nan)
    codes = codes.clone()
    if r0 == 0 or not finite:
        now = np.float32(need)
    elif not (scale >= 0 and np.isfinite(scale)):
        now = np.float32(np.nan)
    elif scale == 0:
        now = need
    else:
        now = scale
        n = 0
        # compared in fp64: exact for fp32 values
        while float(now) < float(need):
            n += 1
            now = np.float32(math.ldexp(float(scale), n))
        if n:
            old = codes[:r0].float() * (2.0 ** -n)
            codes[:r0] = old.round().to(kind) if kind == torch.int8 else old.to(kind)
    codes[r0:r0 + len(rows)] = encode(x, now, kind)
    return codes, now


def paged_write(k_cache, v_cache, key, value, page_table, q_start, cu_q=None, q_len=None,
                k_scale=None, v_scale=None, k_bounds=None):
    """In place, on CPU tensors."""
    nb, nkv, bs, hd = k_cache.shape
    seqs = q_start.numel()
    for s in range(seqs):
        a, b = (s, s + 1) if cu_q is None else (int(cu_q[s]), int(cu_q[s + 1]))
        n = b - a if q_len is None else max(0, min(b - a, int(q_len[s])))
        start = int(q_start[s])
        if start < 0:
            continue
        at = start
        while at < start + n:
            col, r0 = divmod(at, bs)
            m = min(bs - r0, start + n - at)
            blk = int(page_table[s, col]) if col < page_table.shape[1] else -1
            rows = slice(a + at - start, a + at - start + m)
            if 0 <= blk < nb:
                for h in range(nkv):
                    for cache, scale, new in ((k_cache, k_scale, key), (v_cache, v_scale, value)):
                        x = new[rows, h]
                        if scale is None:
                            cache[blk, h, r0:r0 + m] = x
                        else:
                            c, now = _write_page(cache[blk, h], np.float32(scale[blk, h].item()), x,
                                                 r0, cache.dtype)
                            cache[blk, h] = c
                            scale[blk, h] = float(now)
                    if k_bounds is not None:
                        lo, hi = key[rows, h].float().amin(0), key[rows, h].float().amax(0)
                        if r0:
                            lo = torch.minimum(lo, k_bounds[blk, h, 0].float())
                            hi = torch.maximum(hi, k_bounds[blk, h, 1].float())
                        k_bounds[blk, h, 0], k_bounds[blk, h, 1] = lo.bfloat16(), hi.bfloat16()
            at += m


def page_values(cache, scale, ids, head):
    """[len(ids) * bs, hd] fp64 values of a page list of one head."""
    x = cache[ids, head].double()
    if scale is not None:
        x = x * scale[ids, head].double()[:, None, None]
    return x.reshape(-1, x.shape[-1])


def attend_row(q, k, v, scale, sink=None):
    """softmax(q k^T scale) v for q [g, hd], k / v [n, hd], in fp64; no keys: zeros."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    w = q @ k.T * scale
    if sink is not None:
        w = torch.cat([w, sink.double()[:, None]], 1)
    w = torch.softmax(w, -1)[:, : k.shape[0]]
    return w @ v


def decode(query, k_cache, v_cache, page_table, cur_pos, scale=None, k_scale=None, v_scale=None,
           window=0, sinks=None):
    """[users, nq, hd] fp64; page_table [users, w] or [users, nkv, w]."""
    users, nq, hd = query.shape
    nkv, bs = k_cache.shape[1], k_cache.shape[2]
    g = nq // nkv
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(users, nq, hd, dtype=torch.float64)
    for u in range(users):
        for h in range(nkv):
            row = page_table[u] if page_table.dim() == 2 else page_table[u, h]
            ctx = int(cur_pos[u] if cur_pos.dim() == 1 else cur_pos[u, h]) + 1
            if ctx <= 0:
                continue
            ids = row[: (ctx + bs - 1) // bs].long()
            lo = max(0, ctx - window) if window else 0
            k = page_values(k_cache, k_scale, ids, h)[lo:ctx]
            v = page_values(v_cache, v_scale, ids, h)[lo:ctx]
            mine = slice(h * g, (h + 1) * g)
            out[u, mine] = attend_row(query[u, mine].double(), k, v, scale,
                                      None if sinks is None else sinks[mine])
    return out


def select_pages(query, k_bounds, page_table, cur_pos, bs, num_pages, keep_first, keep_last):
    users, nq, hd = query.shape
    nkv = k_bounds.shape[1]
    g = nq // nkv
    table = torch.zeros(users, nkv, num_pages, dtype=torch.int32)
    pos = torch.full((users, nkv), -1, dtype=torch.int32)
    for u in range(users):
        p = min(int(cur_pos[u]), page_table.shape[1] * bs - 1)      # behind the table: its last key
        n = p // bs + 1 if p >= 0 else 0
        for h in range(nkv):
            if n == 0:
                continue
            chosen = list(range(n))
            if n > num_pages:
                b = k_bounds[page_table[u, :n].long(), h].double()
                q = query[u, h * g:(h + 1) * g].double()
                s = q.clamp(max=0) @ b[:, 0].T + q.clamp(min=0) @ b[:, 1].T
                s = torch.where(s.isnan(), math.inf, s).amax(0)
                inner = list(range(keep_first, n - keep_last))
                inner.sort(key=lambda i: (-s[i].item(), i))
                chosen = list(range(keep_first)) + \
                    sorted(inner[: num_pages - keep_first - keep_last]) + \
                    list(range(n - keep_last, n))
            table[u, h, : len(chosen)] = page_table[u, chosen]
            pos[u, h] = (len(chosen) - 1) * bs + p % bs
    return table, pos
