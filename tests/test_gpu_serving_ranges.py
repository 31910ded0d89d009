"""Batched serving on the GPU at the ends of its ranges: values at the limits of their type, batches of more sequences than
a wave has lanes, prompts that fill the chip, against 64 bits.

Tolerances count U = 2^-24, half a step of fp32, and E(kind), that of a type (see test_gpu_serving)."""
import ctypes as C
import time

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import kx  # noqa: E402

from test_gpu_serving import (E, KINDS, NAMES, U, Cache, check_decode, check_prompt, close, exact_attention,  # noqa: E402
                              exact_rope, rope_tables, rounded)

TYPES = [kx.F32, kx.F16, kx.BF16]


# ------------------------------------------------------------------ a weighted mean is a mean
def equal_columns(rng, n, kv_heads, hs, kind):
    """Values that are alike in all rows: the largest of fp16 with both signs, or any."""
    row = np.where(np.arange(kv_heads * hs) % 2, -1.0, 1.0) * 65504 if kind == kx.F16 else rng.standard_normal(kv_heads * hs)
    return np.broadcast_to(rounded(row.astype(np.float32), kind).reshape(1, kv_heads, hs), (n, kv_heads, hs)).copy()


def assert_means(got, v, g, kind, keys):
    """got [rows][heads][hs] of rows that see something, v [rows][kv_heads][hs] alike in all rows.  The weights that are
    summed are those that multiply the values, so the quotient of both sums is off by their roundings alone, 8 sqrt(keys) U
    of the value: nothing that a 16-bit type shows (half a step is 2^-9 or 2^-12 at least)."""
    want = np.repeat(v[:1], g, axis=1)
    if kind == kx.F32:
        assert (np.abs(got - want) <= (8 * np.sqrt(keys) * U + 2.0 ** -20) * np.abs(want)).all()
    else:
        np.testing.assert_array_equal(got, np.broadcast_to(want, got.shape))


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("paged", [False, True])
def test_prompt_means_of_equal_values(kind, hs, paged):
    rng = np.random.default_rng(hs + kind)
    n, heads, kv_heads = 460, 6, 2
    cache = Cache(rng, [n], kv_heads, hs, 16, kind)
    q = rounded(rng.standard_normal((n, heads, hs)).astype(np.float32) * 4, kind)  # few keys carry most of the weight
    k, v = cache.k[0], equal_columns(rng, n, kv_heads, hs, kind)
    if paged:
        pool = kx.PagePool(*(a[np.arange(480) % n].reshape(30, 16, kv_heads, hs) for a in (k, v)), kind)
        table = np.arange(30, dtype=np.int32)[None]
        got = kx.prompt_attention(q, [0, n], pool=pool, table=table, seq_lens=[n], kind=kind)
        one = kx.paged_decode(pool, table, [n], q[-1:], q_kind=kind)
        assert_means(one, v, 3, kind, n)
    else:
        got = kx.prompt_attention(q, [0, n], k, v, kind=kind)
    assert_means(got, v, 3, kind, n)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
def test_prompt_mean_with_one_key_far_above_the_first(kind):
    """One key at score zero in the first tile and one 256 keys on (in a later tile of the same waves), 6 to 8 powers of two
    above it, nearly alone with each other: the running maximum stays with the first, so the second one's weight is among
    the largest that are held."""
    rng = np.random.default_rng(7)
    rows, keys, hs = 256, 300, 64
    q = np.zeros((rows, 1, hs), np.float32)
    q[:, 0, 0] = np.linspace(6, 8, rows) * np.log(2)
    q[:, 0, 1] = 1
    k = np.zeros((keys, 1, hs), np.float32)
    k[:, 0, 1] = -60
    k[[0, 262], 0, 1] = 0
    k[262, 0, 0] = 1
    q, k, v = rounded(q, kind), rounded(k, kind), equal_columns(rng, keys, 1, hs, kind)
    got = kx.prompt_attention(q, [0, rows], k, v, cu_k=[0, keys], causal=False, scale=1.0, kind=kind)
    assert_means(got, v, 1, kind, keys)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
def test_prompt_mean_of_a_strong_key_and_many_weak_ones(kind):
    """20 000 keys of 2^-22 of the weight of one: they are half a percent of the sum, though each is next to nothing."""
    rng = np.random.default_rng(8)
    rows, keys, hs = 3, 20000, 32
    q, k = np.zeros((rows, 1, hs), np.float32), np.zeros((keys, 1, hs), np.float32)
    q[:, 0, 0] = 1
    k[:, 0, 0] = np.where(np.arange(keys) == 11, 15.25, 0)  # 15.25 = 22 ln 2
    v = np.full((keys, 1, hs), 3.0, np.float32)
    v[11] = 1.0
    got = kx.prompt_attention(q, [0, rows], k, v, cu_k=[0, keys], causal=False, scale=1.0, kind=kind)
    w = np.exp(-15.25) * (keys - 1)
    want = (1 + 3 * w) / (1 + w)
    # the weak weights round to a type by half a step of it at most (fp16 holds them with 2^-10 there)
    relative = {kx.F32: 2.0 ** -18, kx.F16: 2.0 ** -10, kx.BF16: 2.0 ** -8}[kind] * w * 3
    half = {kx.F32: U, kx.F16: 2.0 ** -11, kx.BF16: 2.0 ** -8}[kind] * want
    assert (np.abs(got - want) <= relative + half + 8 * np.sqrt(keys) * U * want).all()
    v[:] = equal_columns(rng, 1, 1, hs, kx.BF16) if kind == kx.BF16 else 1000.0
    got = kx.prompt_attention(q, [0, rows], k, v, cu_k=[0, keys], causal=False, scale=1.0, kind=kind)
    assert_means(got, v, 1, kind, keys)


@pytest.mark.parametrize("kind", [kx.F16, kx.BF16], ids=lambda k: NAMES[k])
def test_prompt_means_beside_hidden_nan_and_seen_infinity(kind):
    """Rows ahead of a NaN are computed from what they see alone; an infinity that is seen stays one."""
    rng = np.random.default_rng(9)
    n, hs = 200, 64
    q, k = (rounded(rng.standard_normal((n, m, hs)).astype(np.float32), kind) for m in (4, 2))
    v = equal_columns(rng, n, 2, hs, kind)
    want = v.copy()
    v[190, :, 3], v[193, :, 5], v[195] = np.inf, -np.inf, np.nan
    got = kx.prompt_attention(q, [0, n], k, v, kind=kind)
    assert_means(got[:190], want, 2, kind, n)
    assert np.isposinf(got[190:195, :, 3]).all() and np.isneginf(got[193:195, :, 5]).all() and np.isnan(got[195:]).all()


# ------------------------------------------------------------------ values that are not finite
def check_around(q, cu, ks, vs, got, kind, scale, window, first, broken):
    """broken: (sequence, key, column, value) of values that are not finite in vs; `first`: the sequences' first key that is
    there.  Rows that see one have it in that column of the heads that share its kv head, all else is as without it."""
    g, got, vs = q.shape[1] // ks[0].shape[1], got.copy(), [v.copy() for v in vs]
    for b, key, column, value in broken:
        n, m = cu[b + 1] - cu[b], len(ks[b])
        p = m - n + np.arange(n)
        rows = cu[b] + np.nonzero((key <= p) & (key > p - (window or m)) & (key >= first[b]))[0]
        assert len(rows)
        mine = got[rows, :, column]
        assert (np.isnan(mine) if np.isnan(value) else mine == value).all()
        got[rows, :, column] = 0
        vs[b][key, :, column] = 0
        vs[b][:, :, column] = np.where(np.isfinite(vs[b][:, :, column]), vs[b][:, :, column], 0)
    for b in range(len(cu) - 1):
        n, m = cu[b + 1] - cu[b], len(ks[b])
        p, at = (m - n + np.arange(n))[:, None], np.arange(m)[None]
        seen = (at <= p) & (at > p - (window or m)) & (at >= first[b])
        for h in range(q.shape[1]):
            want, spread, size = exact_attention(q[cu[b]:cu[b + 1], h], ks[b][:, h // g], vs[b][:, h // g], seen, scale)
            mine = got[cu[b]:cu[b + 1], h].copy()
            for c, key, column, _ in broken:
                if c == b:
                    hit = seen[:, key]
                    want[hit, column], spread[hit, column], mine[hit, column] = 0, 0, 0
            close(mine, want, spread, size, E[kind] if kind != kx.F32 else 0, kind)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,kv_heads,hs,page,window", [
    (4, 2, 32, 0, 0), (7, 1, 64, 0, 90), (8, 2, 128, 16, 0), (6, 2, 64, 24, 90), (4, 4, 32, 5, 200), (3, 1, 128, 7, 40)])
def test_prompt_values_that_are_not_finite(kind, heads, kv_heads, hs, page, window):
    """A NaN and infinities in single columns, in tiles of which some rows see a part; pages that are not there hold NaN, and so
    does the page that stands in for them."""
    rng = np.random.default_rng(heads + hs + page)
    new, lens = [330, 40, 129], [330, 210, 300] if page else [330, 40, 129]
    cu = np.cumsum([0] + new)
    cache = Cache(rng, lens, kv_heads, hs, page or 16, kind)
    broken = [(0, 100, 3, np.nan), (0, 131, 9, np.inf), (0, 300, 5, -np.inf), (2, lens[2] - 1, 0, np.nan), (1, lens[1] - 3, 7, np.inf)]
    q = rounded(rng.standard_normal((cu[-1], heads, hs)).astype(np.float32), kind)
    vs, first = [v.copy() for v in cache.v], [0, 0, 0]
    for b, key, column, value in broken:
        vs[b][key, :, column] = value
    if not page:
        got = kx.prompt_attention(q, cu, np.concatenate(cache.k), np.concatenate(vs), window=window, kind=kind)
    else:
        pages, free = cache.pool.shape[0], int(cache.spare[0])
        key, value = (np.full(cache.pool.shape, np.nan, np.float32) for _ in range(2))
        # page 0, which stands in for those that are not there, is one that nobody has
        moved = np.where(cache.table == 0, free, np.where(cache.table == free, 0, cache.table))
        for b, n in enumerate(lens):
            for t in range(n):
                at = moved[b, t // page], t % page
                key[at], value[at] = cache.k[b][t], vs[b][t]
        for b in (1, 2):
            gone = (lens[b] - new[b]) // 2 // page
            moved[b, :gone] = -1
            first[b] = gone * page
        assert pages == len(key) and np.isnan(value[0]).all()
        got = kx.prompt_attention(q, cu, pool=kx.PagePool(key, value, kind), table=moved, seq_lens=lens, window=window, kind=kind)
    check_around(q, cu, cache.k, vs, got, kind, 1 / np.sqrt(hs), window, first, broken)


@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows", [700, 1500])
@pytest.mark.parametrize("broken", [False, True])
def test_attention_over_its_own_queries(kind, rows, broken):
    """Results that lie over the queries: the same bits as beside them, with values that are not finite as well (some waves of
    a workgroup see those, others do not)."""
    rng = np.random.default_rng(rows)
    heads, kv_heads, hs = 64, 8, 128
    q = kx.to_kind(rng.standard_normal((rows, heads, hs)).astype(np.float32), kind)
    cache = Cache(rng, [rows], kv_heads, hs, 16, kind)
    k, v = cache.k[0], cache.v[0].copy()
    if broken:
        v[[40, rows // 2, rows - 6], :, 3] = np.nan
    dk, dv = (kx.Buf.from_numpy(kx.to_kind(a, kind)) for a in (k, v))
    cu = kx.Buf.from_numpy(np.array([0, rows], np.int32))
    got = []
    for over in (False, True):
        dq = kx.Buf.from_numpy(q)
        out = dq if over else kx.Buf.zeros(q.shape, q.dtype)
        d = kx.PromptAttnDesc(type=kind, head_num=heads, kv_head_num=kv_heads, head_size=hs, batch=1, q_rows=rows, k_rows=rows,
                              causal=1, scale=hs ** -0.5, q=dq.ptr, q_stride=heads * hs, k=dk.ptr, k_stride=kv_heads * hs, v=dv.ptr,
                              v_stride=kv_heads * hs, out=out.ptr, out_stride=heads * hs, cu_q=cu.ptr, cu_k=cu.ptr)
        kx.check(kx.lib().kx_prompt_attention(C.byref(d), None))
        got.append(kx.from_kind(out.numpy(q.dtype, q.shape), kind))
    np.testing.assert_array_equal(got[0], got[1])
    assert np.isnan(got[0][40:, :, 3]).all() == broken and np.isfinite(got[0][:40]).all() and np.isfinite(got[0][:, :, 4:]).all()
    # single tokens, in chunks that several workgroups join
    lens, table = kx.Buf.from_numpy(np.array([rows], np.int32)), kx.Buf.from_numpy(cache.table)
    ws = kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(1, heads, kv_heads, hs), np.uint8)
    one = []
    for over in (False, True):
        dq = kx.Buf.from_numpy(q[-1:])
        out = dq if over else kx.Buf.zeros(q[-1:].shape, q.dtype)
        d = kx.PagedDecodeDesc(kv=cache.pool.desc(table, lens), q_type=kind, head_num=heads, scale=hs ** -0.5, q=dq.ptr,
                               q_stride=heads * hs, out=out.ptr, out_stride=heads * hs, workspace=ws.ptr, workspace_bytes=ws.nbytes)
        kx.check(kx.lib().kx_paged_decode(C.byref(d), None))
        one.append(kx.from_kind(out.numpy(q.dtype, q[-1:].shape), kind))
    np.testing.assert_array_equal(one[0], one[1])


@pytest.mark.parametrize("paged", [False, True])
def test_prompt_values_that_are_not_finite_cost_little(paged):
    """One broken value does not hold up its batch: only a tile that is partly seen is taken key by key, which adds less than this
    call's own time.  (Pairs of a row and a head computed anew, one by one, took 200 times as long: the limit lies between.)"""
    rng = np.random.default_rng(3)
    n, heads, kv_heads, hs, page = 2048, 32, 8, 128, 16
    q, k, v = (kx.to_kind(rng.standard_normal((n, m, hs)).astype(np.float32), kx.BF16) for m in (heads, kv_heads, kv_heads))
    cu, lens = kx.Buf.from_numpy(np.array([0, n], np.int32)), kx.Buf.from_numpy(np.array([n], np.int32))
    dq, out = kx.Buf.from_numpy(q), kx.Buf.zeros(q.shape, np.uint16)
    table = np.arange(n // page, dtype=np.int32)[None]
    took = []
    for broken in (False, True):
        if broken and paged:
            v[:page], table = 0x7FC0, table.copy()
            table[0, :20] = -1
        elif broken:
            v[n - 40, :, 3] = 0x7FC0
        dk, dv, dt = (kx.Buf.from_numpy(a) for a in (k, v, table))
        kv = kx.PagedKv(type=kx.BF16, kv_head_num=kv_heads, head_size=hs, page_size=page, num_pages=n // page,
                        table_pages=n // page, batch=1, key=dk.ptr, value=dv.ptr, page_stride=page * kv_heads * hs,
                        row_stride=kv_heads * hs, head_stride=hs, table=dt.ptr, table_stride=n // page, seq_lens=lens.ptr)
        d = kx.PromptAttnDesc(type=kx.BF16, head_num=heads, kv_head_num=kv_heads, head_size=hs, batch=1, q_rows=n, causal=1,
                              scale=hs ** -0.5, q=dq.ptr, q_stride=heads * hs, out=out.ptr, out_stride=heads * hs, cu_q=cu.ptr)
        if paged:
            d.pages = C.addressof(kv)
        else:
            d.k, d.v, d.cu_k, d.k_rows, d.k_stride, d.v_stride = dk.ptr, dv.ptr, cu.ptr, n, kv_heads * hs, kv_heads * hs
        times = []
        for _ in range(6):
            kx.sync()
            start = time.perf_counter()
            for _ in range(4):
                kx.check(kx.lib().kx_prompt_attention(C.byref(d), None))
            kx.sync()
            times.append(time.perf_counter() - start)
        took.append(min(times))
    got = kx.from_kind(out.numpy(), kx.BF16)
    assert np.isfinite(got[320:n - 40]).all() and np.isnan(got[n - 40:, :, 3]).all() != paged
    assert took[1] < 20 * took[0], took


# ------------------------------------------------------------------ sure tokens
@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows,vocab", [(3, 40000), (64, 128256), (1100, 20000), (2, 37)])
def test_logprobs_of_sure_tokens(kind, rows, vocab):
    """Three logits that are not banned: one at the start, one further on and the likeliest behind both, up to 17 above the
    first.  No probability passes one and no entropy falls below zero, and both hold to the last bits:
    relative to the largest logit, d = x - max rounds to U |d|, e^d to U (2 |d| + 4) of itself, the sum z of 1 and two others
    to 2 U z, ln z to U (2 + 2 ln z), the last difference to U of its result; a share p of the entropy likewise."""
    rng = np.random.default_rng(rows + vocab)
    x = np.full((rows, vocab), -np.inf, np.float32)
    at = np.array([0, 5, 20]) if vocab < 100 else np.array([1, vocab // 3, vocab - 7])
    gap = rng.uniform(0.5, 17, (rows, 2)).astype(np.float32)
    x[:, at[2]] = rng.uniform(-4, 4, rows)
    x[:, at[0]], x[:, at[1]] = x[:, at[2]] - gap[:, 0], x[:, at[2]] - gap[:, 1]
    x[0, at] = [-3.0, -12.75, 12.875]
    x = rounded(x, kind)
    order = np.argsort(-x[:, at].astype(np.float64), axis=1, kind="stable")
    lp, en, ids, tl = kx.token_logprobs(x, np.full(rows, at[2]), 3, kind)
    np.testing.assert_array_equal(ids, at[order])
    d = x[:, at].astype(np.float64)
    d -= d.max(1, keepdims=True)
    z = np.exp(d).sum(1)
    off_e = np.exp(d) * U * (2 * np.abs(d) + 4)
    off_lz = off_e.sum(1) / z + 2 * U + U * (2 + 2 * np.log(z))
    want = d - np.log(z)[:, None]
    off = off_lz[:, None] + U * np.abs(d) + U * np.abs(want)
    assert (tl <= 0).all() and (lp <= 0).all()
    assert (np.abs(tl - np.take_along_axis(want, order, 1)) <= np.take_along_axis(off, order, 1)).all()
    assert (np.abs(lp - want[:, 2]) <= off[:, 2]).all()
    p = np.exp(want)
    h = -(p * want).sum(1)
    off_h = off_lz + (np.exp(d) * np.abs(d) * U * (2 * np.abs(d) + 8)).sum(1) / z + 4 * U * h
    assert (en >= 0).all() and (np.abs(en - h) <= off_h).all()


# ------------------------------------------------------------------ more sequences than a wave has lanes
BATCHES = [63, 64, 65, 129, 200]


def ragged(rng, batch, most):
    """Lengths of 0 .. most, with sequences of none and of one on both sides of every 64th."""
    n = rng.integers(0, most + 1, batch)
    for edge in range(64, batch + 1, 64):
        for i, at in enumerate(range(edge - 2, min(edge + 2, batch))):
            n[at] = (0, 1, 0, 2)[(i + edge // 64) % 4]
    n[-1] = most
    return n


@pytest.mark.parametrize("batch", BATCHES + [4096, 4097, 4300])
@pytest.mark.parametrize("src,kind", [(kx.F32, kx.F16), (kx.BF16, kx.BF16)], ids=lambda k: NAMES[k])
def test_write_many_sequences(src, kind, batch):
    rng = np.random.default_rng(batch)
    hs, page, variant = 32, 4, batch % 2
    new = ragged(rng, batch, 5)
    lens = new + rng.integers(0, 9, batch)
    held = -(-lens // page)
    pages = rng.permutation(held.sum() + 2)
    table = np.full((batch, held.max()), -1, np.int32)
    table[np.arange(held.max())[None] < held[:, None]] = pages[:held.sum()]
    key = np.full((len(pages), page, 1, hs), np.nan, np.float32)
    pool = kx.PagePool(key, key, kind)
    cu = 1 + np.concatenate([[0], np.cumsum(new)])
    rows = cu[-1] + 2
    q, k, v = (rounded(rng.standard_normal((rows, n, hs)).astype(np.float32), src) for n in (2, 1, 1))
    tables = rope_tables(16, hs)
    got_q = kx.paged_write(pool, table, lens, cu, k, v, q, tables, variant, src, in_place=True)
    got_k, got_v = pool.read()
    seq = np.repeat(np.arange(batch), new)
    row = np.arange(cu[0], cu[-1])
    pos = row - cu[seq + 1] + lens[seq]
    at = (table[seq, pos // page], pos % page)
    want_v = key.copy()
    want_v[at] = rounded(v[row], kind)
    np.testing.assert_array_equal(got_v, want_v)
    assert (np.isnan(got_k) == np.isnan(want_v)).all()
    for x, got, kind_of in ((q, got_q[row], src), (k, got_k[at], kind)):
        pairs = [exact_rope(x[r], p, tables, variant) for r, p in zip(row, pos)]
        want, size = np.stack([y for y, _ in pairs]), np.stack([z for _, z in pairs])
        # two products and a sum in fp32, then the type's rounding, as in test_write
        assert (np.abs(got - want) <= 3 * U * size + E[kind_of] * np.abs(want) * (1 + 2 ** -7) + (2.0 ** -25 if kind_of == kx.F16 else 0)).all()
    outside = np.setdiff1d(np.arange(rows), row)
    np.testing.assert_array_equal(got_q[outside], q[outside])


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("q_kind,kind", KINDS, ids=lambda k: NAMES[k])
def test_decode_many_sequences(q_kind, kind, batch):
    """Long sequences, which are cut over workgroups, ahead of the 64th, behind it and at both ends."""
    rng = np.random.default_rng(batch + kind)
    lens = ragged(rng, batch, 40)
    for at in (0, 3, 62, 66, 70, 127, 130, batch - 1):
        if at < batch:
            lens[at] = 2000 + 37 * (at % 50)
    heads, kv_heads, hs, page = [(3, 1, 32, 16), (4, 2, 64, 5)][batch % 2]
    cache = Cache(rng, lens.tolist(), kv_heads, hs, page, kind)
    q = rounded(rng.standard_normal((batch, heads, hs)).astype(np.float32), q_kind)
    got = kx.paged_decode(cache.pool, cache.table, lens, q, q_kind=q_kind)
    assert (got[lens == 0] == 0).all()
    check_decode(cache, q, got, 0, 1 / np.sqrt(hs), q_kind)
    got = kx.paged_decode(cache.pool, cache.table, lens, q, window=1000, q_kind=q_kind)
    check_decode(cache, q, got, 1000, 1 / np.sqrt(hs), q_kind)


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
def test_prompts_of_many_sequences(kind, batch):
    rng = np.random.default_rng(batch + kind)
    heads, kv_heads, hs = [(3, 1, 32), (4, 2, 64)][batch % 2]
    new = ragged(rng, batch, 20)
    new[[5, batch // 2]] = 150, 70
    cu = 2 + np.concatenate([[0], np.cumsum(new)])
    rows = cu[-1] + 3
    q, k, v = (rounded(rng.standard_normal((rows, n, hs)).astype(np.float32), kind) for n in (heads, kv_heads, kv_heads))
    got = kx.prompt_attention(q, cu, k, v, kind=kind, fill=7.0)
    assert (got[:2] == 7).all() and (got[-3:] == 7).all()
    check_prompt(q, cu, [k[a:b] for a, b in zip(cu, cu[1:])], [v[a:b] for a, b in zip(cu, cu[1:])], got, kind, 1 / np.sqrt(hs))
    lens = new + rng.integers(0, 30, batch)
    for page in (16, 7):
        cache = Cache(rng, lens.tolist(), kv_heads, hs, page, kind)
        got = kx.prompt_attention(q, cu, pool=cache.pool, table=cache.table, seq_lens=lens, window=25, kind=kind, fill=7.0)
        assert (got[:2] == 7).all() and (got[-3:] == 7).all()
        check_prompt(q, cu, cache.k, cache.v, got, kind, 1 / np.sqrt(hs), window=25)


# ------------------------------------------------------------------ prompts that fill the chip
def check_sample(rng, q, cu, ks, vs, got, kind, scale, window, hidden=None):
    """A sample of rows and heads against 64 bits; hidden: key positions of each sequence that are not there."""
    g = q.shape[1] // ks[0].shape[1]
    for b in range(len(cu) - 1):
        n, m = cu[b + 1] - cu[b], len(ks[b])
        if not n:
            continue
        sample = np.unique(np.concatenate([[0, n - 1, min(n - 1, 63), min(n - 1, 64)], rng.integers(0, n, 6)]))
        for h in np.unique(np.concatenate([[0, q.shape[1] - 1], rng.integers(0, q.shape[1], 4)])):
            at, p = np.arange(m)[None], (m - n + sample)[:, None]
            seen = at <= p
            if window:
                seen &= at > p - window
            if hidden is not None:
                seen &= ~hidden[b][None]
            want, spread, size = exact_attention(q[cu[b] + sample, h], ks[b][:, h // g], vs[b][:, h // g], seen, scale)
            close(got[cu[b] + sample, h], want, spread, size, E[kind], kind)


@pytest.mark.parametrize("kind", [kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,hs", [(64, 128), (128, 64), (128, 32)])
@pytest.mark.parametrize("page", [0, 16, 5])
def test_prompts_that_fill_the_chip(kind, heads, hs, page):
    """Enough rows and heads that a workgroup keeps its keys to itself (256 pairs of a row and a head each: 320 such workgroups
    for 128-wide heads, 800 for 64, 600 for 32): packed rows, pages of whole blocks, others; windows, missing pages, and a NaN
    in a value that rows ahead of it do not see."""
    rng = np.random.default_rng(heads + hs + page)
    kv_heads, scale = 8, hs ** -0.5
    new = [800, 1, 0, 60, 870]
    cu = np.cumsum([0] + new)
    assert cu[-1] * heads / 256 >= {128: 320, 64: 800, 32: 600}[hs]
    q = rounded(rng.standard_normal((cu[-1], heads, hs)).astype(np.float32), kind)
    if not page:
        k, v = (rounded(rng.standard_normal((cu[-1], kv_heads, hs)).astype(np.float32), kind) for _ in range(2))
        ks, vs = ([a[i:j] for i, j in zip(cu, cu[1:])] for a in (k, v))
        for window in (0, 100):
            got = kx.prompt_attention(q, cu, k, v, window=window, kind=kind)
            check_sample(rng, q, cu, ks, vs, got, kind, scale, window)
        broken = v.copy()
        broken[cu[4] - 3] = np.nan  # the third last row of the fourth sequence
        got = kx.prompt_attention(q, cu, k, broken, kind=kind)
        assert np.isnan(got[cu[4] - 3:cu[4]]).all() and np.isfinite(got[:cu[4] - 3]).all() and np.isfinite(got[cu[4]:]).all()
        check_sample(rng, q, [cu[3], cu[4] - 3], [ks[3][:-3]], [vs[3][:-3]], got, kind, scale, 0)
        return
    lens = [n + c for n, c in zip(new, [200, 0, 20, 333, 90])]
    cache = Cache(rng, lens, kv_heads, hs, page, kind)
    for window in (0, 150):
        got = kx.prompt_attention(q, cu, pool=cache.pool, table=cache.table, seq_lens=lens, window=window, kind=kind)
        check_sample(rng, q, cu, cache.k, cache.v, got, kind, scale, window)
    table = cache.table.copy()
    hidden = [np.zeros(n, bool) for n in lens]
    for b, col in ((0, 3), (0, 1000 // page - 1), (3, 0), (4, 20)):
        table[b, col] = [-1, 1 << 30][col % 2]
        hidden[b][col * page:(col + 1) * page] = True
    got = kx.prompt_attention(q, cu, pool=cache.pool, table=table, seq_lens=lens, kind=kind)
    check_sample(rng, q, cu, cache.k, cache.v, got, kind, scale, 0, hidden)


# ------------------------------------------------------------------ rows wider than what is in them
@pytest.mark.parametrize("kind", TYPES, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("page,head_major", [(16, False), (5, True)])
def test_strides_wider_than_rows(kind, page, head_major):
    """q, k and v beside each other in padded rows, pages with room between their rows, tables with columns that no sequence has:
    filed, attended as a prompt and as single tokens; the room between is left alone."""
    rng = np.random.default_rng(page)
    heads, kv_heads, hs, pad = 6, 2, 64, 8
    lens = [70, 1, 33]
    wide, es = kx.KIND_DTYPE[kind], 4 if kind == kx.F32 else 2
    cu, rows = np.cumsum([0] + lens), sum(lens)
    width = (heads + 2 * kv_heads) * hs + pad
    src = rounded(rng.standard_normal((rows, width)).astype(np.float32), kind)
    columns = -(-max(lens) // page) + 3
    pages = max(40, 3 * columns)
    table = np.full((3, columns + 2), 1 << 30, np.int32)
    table[:, :columns] = rng.permutation(pages)[:3 * columns].reshape(3, columns)
    # [page][row or head][head or row][hs] with `pad` elements behind each row of a page and of a head
    inner = hs + pad
    row_stride, head_stride = (inner, page * inner) if head_major else (kv_heads * inner, inner)
    page_stride = page * kv_heads * inner + pad
    mark = kx.to_kind(np.full(pages * page_stride, 3.0, np.float32), kind)
    dk, dv = kx.Buf.from_numpy(mark), kx.Buf.from_numpy(mark)
    qkv, dt = kx.Buf.from_numpy(kx.to_kind(src, kind)), kx.Buf.from_numpy(table)
    sl, dcu = kx.Buf.from_numpy(np.array(lens, np.int32)), kx.Buf.from_numpy(cu.astype(np.int32))
    out_stride = heads * hs + pad
    out = kx.Buf.from_numpy(kx.to_kind(np.full((rows, out_stride), 5.0, np.float32), kind))
    tables = rope_tables(max(lens), hs)
    sin, cos = (kx.Buf.from_numpy(t) for t in tables)
    kv = kx.PagedKv(type=kind, kv_head_num=kv_heads, head_size=hs, page_size=page, num_pages=pages, table_pages=columns, batch=3,
                    key=dk.ptr, value=dv.ptr, page_stride=page_stride, row_stride=row_stride, head_stride=head_stride,
                    table=dt.ptr, table_stride=columns + 2, seq_lens=sl.ptr)
    w = kx.PagedWriteDesc(kv=kv, src_type=kind, rows=rows, head_num=heads, rope_variant=1, table_rows=max(lens), cu_rows=dcu.ptr,
                          k=qkv.at(heads * hs * es), k_stride=width, v=qkv.at((heads + kv_heads) * hs * es), v_stride=width,
                          q=qkv.ptr, q_stride=width, q_out=qkv.ptr, q_out_stride=width, sin_cache=sin.ptr, cos_cache=cos.ptr)
    kx.check(kx.lib().kx_paged_write(C.byref(w), None))
    now = kx.from_kind(qkv.numpy(wide, src.shape), kind)
    np.testing.assert_array_equal(now[:, heads * hs:], src[:, heads * hs:])
    key, value = (kx.from_kind(b.numpy(wide, mark.shape), kind) for b in (dk, dv))
    ks, vs, filed = [], [], np.zeros(mark.shape, bool)
    for b, n in enumerate(lens):
        at = np.array([[table[b, t // page] * page_stride + t % page * row_stride + h * head_stride for h in range(kv_heads)]
                       for t in range(n)])[..., None] + np.arange(hs)
        ks.append(key[at])
        vs.append(value[at])
        filed[at] = True
        np.testing.assert_array_equal(value[at].reshape(n, -1), src[cu[b]:cu[b + 1], (heads + kv_heads) * hs:-pad])
        for t in range(n):
            want, size = exact_rope(src[cu[b] + t, heads * hs:(heads + kv_heads) * hs].reshape(kv_heads, hs), t, tables, 1)
            assert (np.abs(ks[b][t] - want) <= 3 * U * size + E[kind] * np.abs(want) * (1 + 2 ** -7) + 2.0 ** -25).all()
    assert (key[~filed] == 3).all() and (value[~filed] == 3).all()
    q = now[:, :heads * hs].reshape(rows, heads, hs)
    p = kx.PromptAttnDesc(type=kind, head_num=heads, kv_head_num=kv_heads, head_size=hs, batch=3, q_rows=rows, causal=1,
                          scale=0.125, q=qkv.ptr, q_stride=width, out=out.ptr, out_stride=out_stride, cu_q=dcu.ptr, pages=C.addressof(kv))
    kx.check(kx.lib().kx_prompt_attention(C.byref(p), None))
    got = kx.from_kind(out.numpy(wide, (rows, out_stride)), kind)
    assert (got[:, heads * hs:] == 5).all()
    check_prompt(q, cu, ks, vs, got[:, :heads * hs].reshape(rows, heads, hs), kind, 0.125)
    ws = kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(3, heads, kv_heads, hs), np.uint8)
    last = qkv.numpy(wide, src.shape)[cu[1:] - 1]
    dq, one = kx.Buf.from_numpy(last), kx.Buf.from_numpy(kx.to_kind(np.full((3, out_stride), 5.0, np.float32), kind))
    d = kx.PagedDecodeDesc(kv=kv, q_type=kind, head_num=heads, scale=0.125, q=dq.ptr, q_stride=width, out=one.ptr,
                           out_stride=out_stride, workspace=ws.ptr, workspace_bytes=ws.nbytes)
    kx.check(kx.lib().kx_paged_decode(C.byref(d), None))
    got = kx.from_kind(one.numpy(wide, (3, out_stride)), kind)
    assert (got[:, heads * hs:] == 5).all()
    cache = Cache.__new__(Cache)
    cache.k, cache.v, cache.lens, cache.kind, cache.page = ks, vs, lens, kind, page
    check_decode(cache, q[cu[1:] - 1], got[:, :heads * hs].reshape(3, heads, hs), 0, 0.125, kind)
