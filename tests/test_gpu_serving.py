"""Batched serving on the GPU: kx_paged_write, kx_paged_decode, kx_prompt_attention and kx_token_logprobs against
plain implementations in 64 bits, at the sizes, masks and page layouts where they can go wrong.

Tolerances.  U = 2^-24 is half a step of fp32, E(kind) = eps / 2 that of a type.  Attention: a score is a sum of hs
products, off by at most 4 sqrt(hs) U sum |q k| (rounding errors of random sign; the products of 16-bit operands are
exact), a weight by twice that and 2^-21 for the exponential, a sum over n keys by 4 sqrt(n) U of what it adds up;
all of it relative to sum p |v|.  Decode holds its weights in 16 bits or more (2^-16 where the cache is bf16, 2^-21
else); the prompt kernel rounds them to the type, E of each.  A result of a 16-bit type is rounded once, E of it."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import kx  # noqa: E402

U = 2.0 ** -24
E = {kx.F32: U, kx.F16: 2.0 ** -11, kx.BF16: 2.0 ** -8}
KINDW = {kx.F32: 4, kx.F16: 2, kx.BF16: 2}
NAMES = {kx.F32: "f32", kx.F16: "f16", kx.BF16: "bf16"}


def rounded(a, kind):
    return kx.from_kind(kx.to_kind(a, kind), kind)


def exact_attention(q, k, v, seen, scale):
    """q [m][hs], k, v [n][hs], seen [m][n]: (out, bound of the sums' error as above without the weights' own)"""
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    out, spread, size = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros((len(q), 1))
    for i in range(len(q)):
        at = np.nonzero(seen[i])[0]
        if not len(at):
            continue
        s = scale * (k[at] @ q[i])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ v[at]
        spread[i] = p @ np.abs(v[at])
        size[i] = 8 * np.sqrt(q.shape[1]) * U * (abs(scale) * (np.abs(k[at]) @ np.abs(q[i]))).max() + 8 * np.sqrt(len(at)) * U
    return out, spread, size


def close(got, want, spread, size, weight, kind):
    bound = (size + 2.0 ** -20 + weight) * spread + E[kind] * np.abs(want) * (1 if kind != kx.F32 else 4) + 1e-30
    if kind == kx.F16:
        bound = bound + 2.0 ** -25
    worst = (np.abs(got - want) / bound).max()
    assert np.isfinite(got).all() and worst <= 1, worst


class Cache:
    """Sequences with their rows, dealt over shuffled pages; what is in no sequence is NaN."""

    def __init__(self, rng, lens, kv_heads, hs, page, kind, head_major=False, spare=3, columns=None, new=None):
        held = [-(-n // page) for n in lens]
        self.columns = columns or max(max(held), 1)
        self.lens, self.page, self.kind = list(lens), page, kind
        total = sum(held) + spare
        order = rng.permutation(total)
        key = np.full((total, page, kv_heads, hs), np.nan, np.float32)
        value = key.copy()
        self.table = np.full((len(lens), self.columns), -1, np.int32)
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(lens):
            mine = order[at:at + held[b]]
            at += held[b]
            self.table[b, :held[b]] = mine
            k, v = (rounded(rng.standard_normal((n, kv_heads, hs)).astype(np.float32), kind) for _ in range(2))
            filed = n - (new[b] if new else 0)
            for t in range(filed):
                key[mine[t // page], t % page], value[mine[t // page], t % page] = k[t], v[t]
            self.k.append(k)
            self.v.append(v)
        self.spare = order[at:]
        self.pool = kx.PagePool(key, value, kind, head_major)


def check_decode(cache, q, got, window, scale, q_kind, lens=None, hidden=()):
    batch, heads, hs = q.shape
    g = heads // cache.k[0].shape[1]
    for b in range(batch):
        n = (lens or cache.lens)[b]
        lo = max(0, n - window) if window else 0
        for h in range(heads):
            seen = np.zeros((1, len(cache.k[b])), bool)
            seen[0, lo:n] = True
            for page in hidden:
                seen[0, page * cache.page:(page + 1) * cache.page] = False
            want, spread, size = exact_attention(q[b, h][None], cache.k[b][:, h // g], cache.v[b][:, h // g], seen, scale)
            close(got[b, h][None], want, spread, size, 2.0 ** -16 if cache.kind == kx.BF16 else 2.0 ** -20, q_kind)


# ------------------------------------------------------------------ writing
def rope_tables(n, hs, theta=5e5):
    angle = np.arange(n)[:, None] * theta ** (-np.arange(hs) / hs)[None]
    return np.sin(angle).astype(np.float32), np.cos(angle).astype(np.float32)


def exact_rope(x, pos, tables, variant):
    """x [heads][hs]; (value, sum of the two products' sizes)"""
    hs = x.shape[1]
    i = np.arange(hs // 2)
    a, b = (2 * i, 2 * i + 1) if variant == 0 else (i, i + hs // 2)
    sin, cos = (t[pos, 2 * i].astype(np.float64) for t in tables)
    x = x.astype(np.float64)
    y, size = np.empty_like(x), np.empty_like(x)
    y[:, a], y[:, b] = x[:, a] * cos - x[:, b] * sin, x[:, a] * sin + x[:, b] * cos
    size[:, a] = np.abs(x[:, a] * cos) + np.abs(x[:, b] * sin)
    size[:, b] = np.abs(x[:, a] * sin) + np.abs(x[:, b] * cos)
    return y, size


@pytest.mark.parametrize("src,kind", [(kx.F32, kx.F32), (kx.F32, kx.F16), (kx.F32, kx.BF16), (kx.F16, kx.F16),
                                      (kx.BF16, kx.BF16)], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,kv_heads,hs,page,variant,head_major", [
    (4, 2, 32, 16, 0, False), (7, 1, 64, 1, 1, False), (4, 4, 128, 24, 1, True), (32, 8, 128, 64, 0, False)])
def test_write(src, kind, heads, kv_heads, hs, page, variant, head_major):
    rng = np.random.default_rng(heads * 100 + page + kind)
    new, lens = [1, 0, 19, 3, 1], [1, 5, 40, 3, 77]
    cache = Cache(rng, lens, kv_heads, hs, page, kind, head_major, new=new)
    before = cache.pool.read()
    first, behind = 2, 3  # rows of no sequence at both ends
    cu = first + np.cumsum([0] + new)
    rows = cu[-1] + behind
    q, k, v = (rounded(rng.standard_normal((rows, n, hs)).astype(np.float32), src) for n in (heads, kv_heads, kv_heads))
    tables = rope_tables(80, hs)
    got_q = kx.paged_write(cache.pool, cache.table, lens, cu, k, v, q, tables, variant, src, in_place=True)
    key, value = cache.pool.read()
    want_k, want_v = (a.copy() for a in before)
    size_k = np.zeros_like(key)
    want_q, size_q = q.astype(np.float64), np.zeros(q.shape)
    want_k = want_k.astype(np.float64)
    for b, n in enumerate(new):
        for i in range(n):
            pos, row = lens[b] - n + i, cu[b] + i
            at = (cache.table[b, pos // page], pos % page)
            want_k[at], size_k[at] = exact_rope(k[row], pos, tables, variant)
            want_v[at] = rounded(v[row], kind)
            want_q[row], size_q[row] = exact_rope(q[row], pos, tables, variant)
    np.testing.assert_array_equal(value, want_v)
    assert (np.isnan(key) == np.isnan(want_k)).all()
    # two products and a sum in fp32 (3 roundings of at most U each), then the type's
    ok = np.abs(key - want_k) <= 3 * U * size_k + E[kind] * np.abs(want_k) * (1 + 2 ** -7) + (2.0 ** -25 if kind == kx.F16 else 0)
    assert (ok | np.isnan(want_k)).all()
    assert (np.abs(got_q - want_q) <= 3 * U * size_q + E[src] * np.abs(want_q) * (1 + 2 ** -7) * (size_q > 0) +
            (2.0 ** -25 * (size_q > 0) if src == kx.F16 else 0)).all()


def test_write_without_rotation_and_saturating():
    rng = np.random.default_rng(5)
    cache = Cache(rng, [9, 30], 2, 64, 8, kx.F16, new=[9, 2])
    k, v = (rng.standard_normal((11, 2, 64)).astype(np.float32) * 40000 for _ in range(2))
    kx.paged_write(cache.pool, cache.table, [9, 30], [0, 9, 11], k, v)
    key, value = cache.pool.read()
    with np.errstate(over="ignore"):
        for row, (b, pos) in enumerate([(0, i) for i in range(9)] + [(1, 28), (1, 29)]):
            at = (cache.table[b, pos // 8], pos % 8)
            np.testing.assert_array_equal(key[at], np.clip(k[row], -65504, 65504).astype(np.float16).astype(np.float32))
            np.testing.assert_array_equal(value[at], np.clip(v[row], -65504, 65504).astype(np.float16).astype(np.float32))


def test_write_leaves_alone_what_has_no_place():
    """Missing pages, positions below zero, behind the table of pages and behind the sin/cos tables."""
    rng = np.random.default_rng(6)
    hs, page = 32, 4
    cache = Cache(rng, [12, 12, 12, 12], 1, hs, page, kx.F32, new=[12] * 4)
    table = cache.table.copy()
    table[0, 1], table[1, 2] = -1, 10 ** 6
    before = cache.pool.read()
    lens, new = [12, 12, 2, 50], [12, 12, 5, 12]
    cu = np.cumsum([0] + new)
    k, v = (rng.standard_normal((cu[-1], 1, hs)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((cu[-1], 3, hs)).astype(np.float32)
    tables = rope_tables(10, hs)
    got_q = kx.paged_write(cache.pool, table, lens, cu, k, v, q, tables, 1, in_place=True)
    key, value = cache.pool.read()
    want_v = before[1].copy()
    for b in range(4):
        n = new[b]
        for i in range(n):
            pos, row = lens[b] - n + i, cu[b] + i
            if 0 <= pos < 10:
                assert np.abs(got_q[row] - exact_rope(q[row], pos, tables, 1)[0]).max() < 1e-5
                if 0 <= table[b, pos // page] < 15:
                    want_v[table[b, pos // page], pos % page] = v[row]
            else:
                np.testing.assert_array_equal(got_q[row], q[row])
    np.testing.assert_array_equal(value, want_v)
    assert (np.isnan(key) == np.isnan(want_v)).all()


def test_lengths_past_the_table():
    """A sequence that has outgrown its table of pages: what lies in it is filed, read and attended at its own
    position, the rest is not there."""
    rng = np.random.default_rng(8)
    hs, page, window, length, n = 64, 4, 9, 23, 7  # the table holds 20 rows, the new ones are 16 .. 22
    cache = Cache(rng, [20], 1, hs, page, kx.F32, new=[4])
    k, v = (rng.standard_normal((n, 1, hs)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n, 2, hs)).astype(np.float32)
    before = cache.pool.read()
    tables = rope_tables(40, hs)
    got_q = kx.paged_write(cache.pool, cache.table, [length], [0, n], k, v, q, tables, 1)
    key, value = cache.pool.read()
    pos = length - n + np.arange(n)
    assert np.abs(got_q - np.stack([exact_rope(q[i], pos[i], tables, 1)[0] for i in range(n)])).max() < 1e-5
    last = cache.table[0, 4]
    np.testing.assert_array_equal(value[last, :, 0], v[:4, 0])
    others = np.arange(len(key)) != last
    np.testing.assert_array_equal(value[others], before[1][others])
    np.testing.assert_array_equal(key[others], before[0][others])
    ks, vs = (a.reshape(-1, 1, hs)[[t * page + i for t in cache.table[0] for i in range(page)]] for a in (key, value))
    seen = (np.arange(20)[None] <= pos[:, None]) & (np.arange(20)[None] > pos[:, None] - window)
    got = kx.prompt_attention(got_q, [0, n], pool=cache.pool, table=cache.table, seq_lens=[length], window=window, kind=kx.F32)
    one = kx.paged_decode(cache.pool, cache.table, [length], got_q[-1:], window=window)
    for h in range(2):
        want, spread, size = exact_attention(got_q[:, h], ks[:, 0], vs[:, 0], seen, hs ** -0.5)
        close(got[:, h], want, spread, size, 0, kx.F32)
        close(one[:, h], want[-1:], spread[-1:], size[-1:], 2.0 ** -20, kx.F32)
    one = kx.paged_decode(cache.pool, cache.table, [20 + window], got_q[-1:], window=window)
    assert (one == 0).all()


# ------------------------------------------------------------------ one new token per sequence
KINDS = [(kx.F32, kx.F32), (kx.F32, kx.F16), (kx.F32, kx.BF16), (kx.F16, kx.F16), (kx.BF16, kx.BF16)]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257]


@pytest.mark.parametrize("q_kind,kind", KINDS, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,kv_heads,hs,page,window,head_major", [
    (4, 2, 32, 16, 0, False), (7, 1, 64, 48, 0, True), (8, 2, 128, 1, 0, False), (3, 3, 64, 5, 20, False),
    (40, 2, 128, 64, 33, False), (16, 1, 128, 32, 0, True), (64, 1, 32, 7, 1, False)])
def test_decode_edges(q_kind, kind, heads, kv_heads, hs, page, window, head_major):
    rng = np.random.default_rng(heads + page + 10 * kind)
    cache = Cache(rng, EDGES, kv_heads, hs, page, kind, head_major)
    q = rounded(rng.standard_normal((len(EDGES), heads, hs)).astype(np.float32), q_kind)
    got = kx.paged_decode(cache.pool, cache.table, EDGES, q, window=window, q_kind=q_kind)
    assert (got[0] == 0).all()
    check_decode(cache, q, got, window, 1 / np.sqrt(hs), q_kind)


@pytest.mark.parametrize("q_kind,kind", KINDS, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("lens,heads,kv_heads,hs,page,window", [
    ([9001], 8, 2, 128, 16, 0), ([1, 7000, 3, 260, 1999], 4, 1, 64, 24, 0), ([5000, 4100], 28, 4, 128, 128, 4090),
    ([20000], 2, 1, 32, 3, 0)])
def test_decode_long(q_kind, kind, lens, heads, kv_heads, hs, page, window):
    rng = np.random.default_rng(lens[0] + kind)
    cache = Cache(rng, lens, kv_heads, hs, page, kind)
    q = rounded(rng.standard_normal((len(lens), heads, hs)).astype(np.float32) * 3, q_kind)
    got = kx.paged_decode(cache.pool, cache.table, lens, q, window=window, q_kind=q_kind)
    check_decode(cache, q, got, window, 1 / np.sqrt(hs), q_kind)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("page", [16, 5, 64])
def test_decode_missing_pages(kind, page):
    """Pages that are not there (freed behind a window, or simply unset) are not read and get no weight."""
    rng = np.random.default_rng(page)
    lens = [300, 5 * page, page]
    cache = Cache(rng, lens, 2, 64, page, kind)
    q = rounded(rng.standard_normal((3, 8, 64)).astype(np.float32), kind)
    table = cache.table.copy()
    table[:, 0] = [-1, 1 << 30, -7]
    table[0, 3] = cache.pool.shape[0]
    got = kx.paged_decode(cache.pool, table, lens, q, q_kind=kind)
    assert (got[2] == 0).all()
    check_decode(cache, q[:1], got[:1], 0, 0.125, kind, hidden=(0, 3))
    cache.k, cache.v, cache.lens = cache.k[1:], cache.v[1:], cache.lens[1:]
    check_decode(cache, q[1:2], got[1:2], 0, 0.125, kind, hidden=(0,))


def test_decode_lengths_out_of_range_are_bounded():
    rng = np.random.default_rng(2)
    cache = Cache(rng, [32, 48, 48], 2, 64, 16, kx.F16)
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    got = kx.paged_decode(cache.pool, cache.table, [-5, 10 ** 9, 48], q)
    assert (got[0] == 0).all()
    cache.lens = [0, 48, 48]
    check_decode(cache, q, got, 0, 0.125, kx.F32)


@pytest.mark.parametrize("q_kind,kind", KINDS, ids=lambda k: NAMES[k])
def test_decode_large_scores_and_values(q_kind, kind):
    """One key far above the others, queries and values of very different sizes: the weights are all but 0 and 1."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [700, 40], 1, 128, 16, kind)
    q = rng.standard_normal((2, 4, 128)).astype(np.float32)
    q[0, 0] *= 300
    q[0, 1] *= 1e-6
    q[1, 2, :64] *= 1000
    q = rounded(q, q_kind)
    got = kx.paged_decode(cache.pool, cache.table, [700, 40], q, q_kind=q_kind)
    check_decode(cache, q, got, 0, 1 / np.sqrt(128), q_kind)


@pytest.mark.parametrize("q_kind,kind", KINDS, ids=lambda k: NAMES[k])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
def test_decode_scales(q_kind, kind, scale):
    rng = np.random.default_rng(10)
    lens = [77, 1, 300]
    cache = Cache(rng, lens, 2, 64, 16, kind)
    q = rounded(rng.standard_normal((3, 6, 64)).astype(np.float32), q_kind)
    got = kx.paged_decode(cache.pool, cache.table, lens, q, scale=scale, window=50, q_kind=q_kind)
    check_decode(cache, q, got, 50, scale, q_kind)


def test_decode_offsets_past_32_bits():
    """A pool of more than 2^31 elements: the last pages are reached (rows sit at a page stride of 2^26 elements)."""
    pages, stride, hs = 70, 1 << 26, 128
    rng = np.random.default_rng(3)
    key, value = kx.Buf(pages * stride * 2), kx.Buf(pages * stride * 2)
    order = rng.permutation(pages)[:20].astype(np.int32)
    order[0] = pages - 1
    k, v = (rounded(rng.standard_normal((20 * 16, hs)).astype(np.float32), kx.F16) for _ in range(2))
    for i, p in enumerate(order):
        key.upload(kx.to_kind(k[16 * i:16 * i + 16], kx.F16), int(p) * stride * 2)
        value.upload(kx.to_kind(v[16 * i:16 * i + 16], kx.F16), int(p) * stride * 2)
    table, lens = kx.Buf.from_numpy(order[None]), kx.Buf.from_numpy(np.array([315], np.int32))
    q = rng.standard_normal((1, 4, hs)).astype(np.float32)
    dq, out = kx.Buf.from_numpy(q), kx.Buf.zeros(q.shape)
    ws = kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(1, 4, 1, hs), np.uint8)
    kv = kx.PagedKv(type=kx.F16, kv_head_num=1, head_size=hs, page_size=16, num_pages=pages, table_pages=20, batch=1,
                    key=key.ptr, value=value.ptr, page_stride=stride, row_stride=hs, head_stride=hs, table=table.ptr,
                    table_stride=20, seq_lens=lens.ptr)
    d = kx.PagedDecodeDesc(kv=kv, q_type=kx.F32, head_num=4, scale=hs ** -0.5, q=dq.ptr, q_stride=4 * hs, out=out.ptr,
                           out_stride=4 * hs, workspace=ws.ptr, workspace_bytes=ws.nbytes)
    kx.check(kx.lib().kx_paged_decode(C.byref(d), None))
    got = out.numpy()
    for h in range(4):
        want, spread, size = exact_attention(q[0, h][None], k[:315], v[:315], np.ones((1, 315), bool), hs ** -0.5)
        close(got[0, h][None], want, spread, size, 2.0 ** -20, kx.F32)
    # the same pages for a prompt of two rows, and a row filed in the last of them
    q16 = kx.Buf.from_numpy(kx.to_kind(q.reshape(2, 2, hs), kx.F16))
    out16, cu = kx.Buf.zeros((2, 2, hs), np.float16), kx.Buf.from_numpy(np.array([0, 2], np.int32))
    p = kx.PromptAttnDesc(type=kx.F16, head_num=2, kv_head_num=1, head_size=hs, batch=1, q_rows=2, causal=1,
                          scale=hs ** -0.5, q=q16.ptr, q_stride=2 * hs, out=out16.ptr, out_stride=2 * hs, cu_q=cu.ptr,
                          pages=C.addressof(kv))
    kx.check(kx.lib().kx_prompt_attention(C.byref(p), None))
    got = out16.numpy().astype(np.float32)
    qr = rounded(q, kx.F16).reshape(2, 2, hs)
    seen = np.arange(315)[None] <= np.array([[313], [314]])
    for h in range(2):
        want, spread, size = exact_attention(qr[:, h], k[:315], v[:315], seen, hs ** -0.5)
        close(got[:, h], want, spread, size, E[kx.F16], kx.F16)


def test_decode_repeats_bit_for_bit_and_leaves_its_workspace_ready():
    rng = np.random.default_rng(11)
    heads, hs = 8, 128
    ws = kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(40, heads, 2, hs), np.uint8)
    first = {}
    for turn in range(3):
        for seed, lens in enumerate([[6000], [1] * 40, [3000, 0, 17, 5], [200] * 9]):
            r = np.random.default_rng(seed)
            cache = Cache(r, lens, 2, hs, 16, kx.F16)
            q = r.standard_normal((len(lens), heads, hs)).astype(np.float32)
            got = kx.paged_decode(cache.pool, cache.table, lens, q, workspace=ws)
            np.testing.assert_array_equal(got, first.setdefault(seed, got))
            if turn == 0:
                check_decode(cache, q, got, 0, 1 / np.sqrt(hs), kx.F32)


def test_decode_captured_and_replayed_as_the_sequences_grow():
    rng = np.random.default_rng(12)
    lens, heads, hs, page = [700, 5, 64, 1500], 8, 64, 16
    cache = Cache(rng, [n + 40 for n in lens], 2, hs, page, kx.BF16)
    q = rounded(rng.standard_normal((4, heads, hs)).astype(np.float32), kx.BF16)
    dq, out = kx.Buf.from_numpy(kx.to_kind(q, kx.BF16)), kx.Buf.zeros(q.shape, np.uint16)
    table, dl = kx.Buf.from_numpy(cache.table), kx.Buf.from_numpy(np.array(lens, np.int32))
    ws = kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(4, heads, 2, hs), np.uint8)
    d = kx.PagedDecodeDesc(kv=cache.pool.desc(table, dl), q_type=kx.BF16, head_num=heads, scale=0.125, q=dq.ptr,
                           q_stride=heads * hs, out=out.ptr, out_stride=heads * hs, workspace=ws.ptr,
                           workspace_bytes=ws.nbytes)
    stream, graph = kx.Stream(), C.c_void_p()
    kx.check(kx.lib().kx_paged_decode(C.byref(d), stream.ptr))
    stream.sync()
    kx.check(kx.lib().kx_graph_begin_capture(stream.ptr))
    kx.check(kx.lib().kx_paged_decode(C.byref(d), stream.ptr))
    kx.check(kx.lib().kx_graph_end_capture(stream.ptr, C.byref(graph)))
    for step in range(5):
        now = [n + 8 * step for n in lens]
        dl.upload(np.array(now, np.int32))
        kx.check(kx.lib().kx_graph_launch(graph, stream.ptr))
        stream.sync()
        got = kx.from_kind(out.numpy(np.uint16, q.shape), kx.BF16)
        check_decode(cache, q, got, 0, 0.125, kx.BF16, lens=now)
        eager = kx.paged_decode(cache.pool, cache.table, now, q, scale=0.125, q_kind=kx.BF16, workspace=ws)
        np.testing.assert_array_equal(got, eager)
    kx.lib().kx_graph_destroy(graph)


# ------------------------------------------------------------------ packed prompts
def check_prompt(q, cu, ks, vs, got, kind, scale, causal=True, window=0):
    g = q.shape[1] // ks[0].shape[1]
    for b in range(len(cu) - 1):
        n, m = cu[b + 1] - cu[b], len(ks[b])
        p = (m - n + np.arange(n))[:, None]
        at = np.arange(m)[None]
        seen = (at <= p) if causal else np.ones((n, m), bool)
        if window:
            seen = seen & (at > p - window)
        for h in range(q.shape[1]):
            want, spread, size = exact_attention(q[cu[b]:cu[b + 1], h], ks[b][:, h // g], vs[b][:, h // g], seen, scale)
            if n:
                close(got[cu[b]:cu[b + 1], h], want, spread, size, E[kind] if kind != kx.F32 else 0, kind)


LENS = [1, 0, 33, 2, 64, 65, 31, 130, 17, 200]


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,kv_heads,hs,causal,window", [
    (4, 2, 32, True, 0), (7, 1, 64, True, 0), (8, 2, 128, True, 0), (3, 3, 128, False, 0), (6, 1, 64, True, 19),
    (20, 1, 128, True, 64), (2, 2, 32, False, 0)])
def test_prompts_packed(kind, heads, kv_heads, hs, causal, window):
    rng = np.random.default_rng(heads * 7 + kind)
    cu = np.cumsum([3] + LENS)  # three rows ahead of the first sequence, two behind the last
    rows = cu[-1] + 2
    q, k, v = (rounded(rng.standard_normal((rows, n, hs)).astype(np.float32), kind) for n in (heads, kv_heads, kv_heads))
    k[:3], v[:3], k[cu[-1]:], v[cu[-1]:] = np.nan, np.nan, np.nan, np.nan
    got = kx.prompt_attention(q, cu, k, v, causal=causal, window=window, kind=kind, fill=7.0)
    assert (got[:3] == 7).all() and (got[cu[-1]:] == 7).all()
    parts = [(k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]]) for b in range(len(LENS))]
    check_prompt(q, cu, [p[0] for p in parts], [p[1] for p in parts], got, kind, 1 / np.sqrt(hs), causal, window)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 50)])
def test_prompts_with_other_keys(kind, causal, window):
    """More keys than queries (a piece of a prompt), fewer (rows that see nothing), none at all."""
    rng = np.random.default_rng(21 + kind)
    hs, heads, kv_heads = 64, 4, 2
    nq, nk = [5, 40, 70, 3, 0, 150], [300, 10, 70, 0, 9, 151]
    cu, ck = np.cumsum([0] + nq), np.cumsum([1] + nk)
    q = rounded(rng.standard_normal((cu[-1], heads, hs)).astype(np.float32), kind)
    k, v = (rounded(rng.standard_normal((ck[-1], kv_heads, hs)).astype(np.float32), kind) for _ in range(2))
    got = kx.prompt_attention(q, cu, k, v, cu_k=ck, causal=causal, window=window, kind=kind, fill=7.0)
    parts = [(k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]]) for b in range(len(nq))]
    if causal:
        assert (got[cu[1]:cu[1] + 30] == 0).all()
    assert (got[cu[3]:cu[4]] == 0).all()
    check_prompt(q, cu, [p[0] for p in parts], [p[1] for p in parts], got, kind, 0.125, causal, window)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("heads,kv_heads,hs,page,window,head_major", [
    (4, 2, 64, 16, 0, False), (8, 1, 128, 5, 0, True), (4, 4, 32, 1, 0, False), (6, 2, 128, 64, 40, False),
    (4, 2, 64, 24, 300, True)])
def test_prompts_over_pages(kind, heads, kv_heads, hs, page, window, head_major):
    rng = np.random.default_rng(page + kind)
    new, lens = [1, 60, 0, 129, 33], [500, 60, 20, 140, 700]
    cache = Cache(rng, lens, kv_heads, hs, page, kind, head_major)
    cu = np.cumsum([0] + new)
    q = rounded(rng.standard_normal((cu[-1], heads, hs)).astype(np.float32), kind)
    got = kx.prompt_attention(q, cu, pool=cache.pool, table=cache.table, seq_lens=lens, window=window, kind=kind)
    check_prompt(q, cu, cache.k, cache.v, got, kind, 1 / np.sqrt(hs), True, window)


@pytest.mark.parametrize("hs", [32, 64, 128])
def test_prompts_of_many_heads(hs):
    """fp32 calls that fill the chip (others are cut into smaller workgroups): packed rows, pages of whole blocks and others."""
    rng = np.random.default_rng(hs + 5)
    heads, lens = 24, [1, 40, 33, 2, 64, 65, 31, 90, 17, 100, 129]
    cu = np.cumsum([0] + lens)
    q = rng.standard_normal((cu[-1], heads, hs)).astype(np.float32)
    for page in (16, 5):
        cache = Cache(rng, lens, heads, hs, page, kx.F32)
        got = kx.prompt_attention(q, cu, pool=cache.pool, table=cache.table, seq_lens=lens, kind=kx.F32)
        check_prompt(q, cu, cache.k, cache.v, got, kx.F32, 1 / np.sqrt(hs))
    np.testing.assert_array_equal(kx.prompt_attention(q, cu, np.concatenate(cache.k), np.concatenate(cache.v), kind=kx.F32), got)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("page", [16, 6])
def test_prompts_missing_pages(kind, page):
    """The pages that a window has left behind are gone; their entries say so."""
    rng = np.random.default_rng(31)
    new, lens, window = [40, 7], [400, 90], 64
    cache = Cache(rng, lens, 2, 64, page, kind)
    table = cache.table.copy()
    for b in range(2):
        table[b, :max(0, lens[b] - new[b] - window + 1) // page] = [-1, 1 << 29][b]
    cu = np.cumsum([0] + new)
    q = rounded(rng.standard_normal((cu[-1], 4, 64)).astype(np.float32), kind)
    got = kx.prompt_attention(q, cu, pool=cache.pool, table=table, seq_lens=lens, window=window, kind=kind)
    check_prompt(q, cu, cache.k, cache.v, got, kind, 0.125, True, window)
    table[:, -3:] = -1  # and without a single page: zeros
    table[1] = -1
    got = kx.prompt_attention(q, cu, pool=cache.pool, table=table, seq_lens=lens, window=window, kind=kind)
    assert np.isfinite(got).all() and (got[cu[1]:] == 0).all()


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
def test_prompt_rows_do_not_see_what_is_masked(kind):
    """Infinities and NaN in later rows of a sequence, in keys and in values, reach no row ahead of them."""
    rng = np.random.default_rng(41)
    n, hs = 150, 64
    q, k, v = (rounded(rng.standard_normal((n, m, hs)).astype(np.float32), kind) for m in (4, 2, 2))
    k[100], v[90, 1, 5], v[97, 0] = np.nan, np.inf, np.nan
    got = kx.prompt_attention(q, [0, n], k, v, kind=kind)
    check_prompt(q[:90], [0, 90], [k[:90]], [v[:90]], got[:90], kind, 0.125)
    assert np.isposinf(got[90:97, 2:, 5]).all() and np.isfinite(got[90:97, :2]).all()
    assert np.isnan(got[97:, :2]).all() and np.isnan(got[100:]).all()


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 1.0])
def test_prompt_scales(kind, scale):
    rng = np.random.default_rng(42)
    cu = [0, 100, 133]
    q, k, v = (rounded(rng.standard_normal((133, m, 64)).astype(np.float32), kind) for m in (4, 2, 2))
    got = kx.prompt_attention(q, cu, k, v, scale=scale, window=70, kind=kind)
    check_prompt(q, cu, [k[:100], k[100:]], [v[:100], v[100:]], got, kind, scale, True, 70)


@pytest.mark.parametrize("kind", [kx.F16, kx.BF16, kx.F32], ids=lambda k: NAMES[k])
def test_prompt_long_and_strided(kind):
    """q, k and v beside each other in one row, a long sequence and a short one; large scores."""
    rng = np.random.default_rng(51)
    heads, kv_heads, hs = 4, 2, 128
    cu = [0, 1111, 1131]
    qkv = rounded(rng.standard_normal((1131, heads + 2 * kv_heads, hs)).astype(np.float32) * 2, kind)
    buf, es = kx.Buf.from_numpy(kx.to_kind(qkv, kind)), 4 if kind == kx.F32 else 2
    out = kx.Buf.zeros((1131, heads + 1, hs), kx.KIND_DTYPE[kind])
    dc = kx.Buf.from_numpy(np.array(cu, np.int32))
    row = (heads + 2 * kv_heads) * hs
    d = kx.PromptAttnDesc(type=kind, head_num=heads, kv_head_num=kv_heads, head_size=hs, batch=2, q_rows=1131,
                          k_rows=1131, causal=1, scale=hs ** -0.5, q=buf.ptr, q_stride=row, k=buf.at(heads * hs * es),
                          k_stride=row, v=buf.at((heads + kv_heads) * hs * es), v_stride=row, out=out.ptr,
                          out_stride=(heads + 1) * hs, cu_q=dc.ptr, cu_k=dc.ptr)
    kx.check(kx.lib().kx_prompt_attention(C.byref(d), None))
    got = kx.from_kind(out.numpy(), kind)
    assert (got[:, heads] == 0).all()
    k, v = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    check_prompt(qkv[:, :heads], cu, [k[:1111], k[1111:]], [v[:1111], v[1111:]], got[:, :heads], kind, hs ** -0.5)


# ------------------------------------------------------------------ log probabilities
def check_logprobs(x, tokens, top_n, got, kind):
    """Against 64 bits.  A difference x - max is exact to U of its size, the sum of n exponentials to 4 sqrt(n) U + 2^-21
    relative; log of it and the last difference round to U of their sizes."""
    x = rounded(x, kind).astype(np.float64)
    rows, vocab = x.shape
    lp, en, ids, tl = got
    tol_z = 4 * np.sqrt(vocab) * U + 2.0 ** -20
    for r in range(rows):
        m = x[r].max()
        order = np.lexsort((np.arange(vocab), -np.where(np.isnan(x[r]), -np.inf, x[r]), np.isnan(x[r])))[:top_n]
        np.testing.assert_array_equal(ids[r], order)
        if not np.isfinite(m):
            assert np.isnan(tl[r]).all() and (en is None or np.isnan(en[r]))
            assert lp is None or np.isnan(lp[r]) or (tokens[r] < 0 and lp[r] == 0)
            continue
        e = np.exp(x[r] - m)
        p, lse = e / e.sum(), m + np.log(e.sum())
        size = tol_z + 4 * U * (np.abs(m) + np.log(vocab) + 1)
        np.testing.assert_array_less(np.abs(tl[r] - (x[r][order] - lse))[np.isfinite(x[r][order])],
                                     (size + 4 * U * np.abs(x[r][order] - lse))[np.isfinite(x[r][order])])
        assert np.isneginf(tl[r][np.isneginf(x[r][order])]).all()
        if lp is not None:
            t = tokens[r]
            if t < 0:
                assert lp[r] == 0
            elif t >= vocab:
                assert np.isnan(lp[r])
            elif np.isneginf(x[r, t]):
                assert np.isneginf(lp[r])
            else:
                assert abs(lp[r] - (x[r, t] - lse)) <= size + 4 * U * abs(x[r, t] - lse)
        if en is not None:
            at = p > 0
            terms = -p[at] * np.log(p[at])
            assert abs(en[r] - terms.sum()) <= 4 * tol_z * (terms.sum() + np.log(vocab) + 1), (en[r], terms.sum())


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows,vocab,top_n,extra", [
    (1, 1, 1, 0), (3, 2, 2, 1), (5, 31, 20, 0), (2, 33, 32, 7), (7, 1000, 5, 1), (1, 128256, 20, 0), (3, 50257, 32, 0),
    (300, 5003, 3, 2), (4, 32000, 0, 5), (2, 151936, 1, 0), (2500, 517, 2, 0)])
def test_logprobs(kind, rows, vocab, top_n, extra):
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[:, rng.integers(vocab)] += 9
    tokens = rng.integers(0, vocab, rows)
    tokens[-1] = -1 if rows > 1 else tokens[-1]
    tokens[0] = vocab if rows > 2 else tokens[0]
    got = kx.token_logprobs(x, tokens, top_n, kind, row_stride=vocab + extra)
    check_logprobs(x, tokens, top_n, got, kind)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows", [6, 600])
def test_logprobs_orders(kind, rows):
    """Rising, falling, all alike, few different values, both zeros, huge values: the order among equals is the index."""
    vocab, rng = 20011, np.random.default_rng(8)
    x = np.zeros((rows, vocab), np.float32)
    ramp = np.linspace(-40, 40, vocab).astype(np.float32)
    for r in range(rows):
        x[r] = [ramp, ramp[::-1], np.full(vocab, -3.25), rng.integers(0, 4, vocab), rng.choice([0.0, -0.0], vocab),
                np.where(rng.random(vocab) < 0.5, 60000, -60000)][r % 6]
    got = kx.token_logprobs(x, np.arange(rows) * 7 % vocab, 32, kind)
    check_logprobs(x, np.arange(rows) * 7 % vocab, 32, got, kind)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows,top_n", [(5, 32), (5, 5), (520, 5), (520, 32)])
def test_logprobs_few_above_many_alike(kind, rows, top_n):
    """A vocabulary of which next to nothing is allowed, or nearly all is alike, with the few at the ends, in the middle,
    behind each other and in rising order; some rows hold NaN."""
    vocab = 30011
    x = np.full((rows, vocab), -np.inf, np.float32)
    at = np.array([0, 1, 255, 256, 4099, 8191, 8192, 20000, vocab - 9, vocab - 1])
    for r in range(rows):
        case = r % 5
        if case in (1, 3, 4):
            x[r] = 1.5
        if case == 0:
            x[r, at[[0, 5, 9]]] = 1.0
        elif case == 1:
            x[r, at] = 2.0 + np.arange(10)  # rising: each is above all ahead of it
        elif case == 2:
            x[r, vocab - 40:] = np.arange(40) * 0.25
        elif case == 3:
            x[r, at] = 1.5 - 0.5 * np.arange(10)
            x[r, 777] = np.nan
        else:
            x[r, ::3] = -np.inf
            x[r, at[::2]] = 3.0
    tokens = np.where(np.arange(rows) % 2, vocab - 1, 8192)
    got = kx.token_logprobs(x, tokens, top_n, kind, row_stride=vocab + 3)
    check_logprobs(x, tokens, top_n, got, kind)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
@pytest.mark.parametrize("rows", [8, 800])
def test_logprobs_banned_and_broken_rows(kind, rows):
    vocab, rng = 4099, np.random.default_rng(18)
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    for r in range(rows):
        case = r % 8
        if case == 0:
            x[r, rng.random(vocab) < 0.9] = -np.inf
        elif case == 1:
            x[r] = -np.inf
        elif case == 2:
            x[r] = -np.inf
            x[r, 4000] = 1.5  # one choice left
        elif case == 3:
            x[r, 77] = np.nan
        elif case == 4:
            x[r, 88] = np.inf
        elif case == 5:
            x[r, :] = np.finfo(np.float32).min if kind == kx.F32 else -65504 if kind == kx.F16 else -3.3e38
        elif case == 6:
            x[r] = np.nan
    got = kx.token_logprobs(x, tokens, 5, kind)
    check_logprobs(x, tokens, 5, got, kind)


def test_logprobs_parts_and_workspace():
    """Each output by itself, two rows' counts with one workspace, and bit for bit again."""
    rng = np.random.default_rng(28)
    ws = kx.Buf.zeros(max(kx.lib().kx_token_logprobs_workspace_bytes(r, 70000, 20) for r in (1, 3, 64)), np.uint8)
    for rows in (1, 64, 3, 1):
        x = (rng.standard_normal((rows, 70000)) * 3).astype(np.float32)
        t = rng.integers(0, 70000, rows)
        all_of = kx.token_logprobs(x, t, 20, workspace=ws)
        check_logprobs(x, t, 20, all_of, kx.F32)
        again = kx.token_logprobs(x, t, 20, workspace=ws)
        for a, b in zip(all_of, again):
            np.testing.assert_array_equal(a, b)
        only_lp = kx.token_logprobs(x, t, 0, entropy=False, workspace=ws)
        np.testing.assert_allclose(only_lp[0], all_of[0], rtol=1e-5, atol=1e-5)
        none = kx.token_logprobs(x, None, 3, entropy=False, workspace=ws)
        np.testing.assert_array_equal(none[2], all_of[2][:, :3])


# ------------------------------------------------------------------ as they are used, one after the other
@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
def test_a_batch_is_served(kind):
    """Prompts of a batch are filed and attended, continued in pieces, then tokens one by one: every step equals the
    attention over all rows so far, in 64 bits; and the flat-cache entries say the same of a single sequence."""
    rng = np.random.default_rng(61)
    heads, kv_heads, hs, page = 8, 2, 64, 16
    prompt, piece, tokens = [70, 1, 33], [20, 50, 0], 3
    total = [p + c + tokens for p, c in zip(prompt, piece)]
    cache = Cache(rng, total, kv_heads, hs, page, kind, new=total)
    rows = [rounded(rng.standard_normal((n, heads + 2 * kv_heads, hs)).astype(np.float32), kind) for n in total]
    tables = rope_tables(max(total), hs)
    done = [0, 0, 0]
    for step, new in enumerate([prompt, piece] + [[1, 1, 1]] * tokens):
        cu, lens = np.cumsum([0] + new), [d + n for d, n in zip(done, new)]
        packed = np.concatenate([r[d:d + n] for r, d, n in zip(rows, done, new)])
        q, k, v = packed[:, :heads], packed[:, heads:heads + kv_heads], packed[:, heads + kv_heads:]
        q = kx.paged_write(cache.pool, cache.table, lens, cu, k, v, q, tables, 1, kind)
        key, value = cache.pool.read()
        ks = [key.reshape(-1, kv_heads, hs)[[t * page + i for t in cache.table[b] for i in range(page)][:n]] for b, n in enumerate(lens)]
        vs = [value.reshape(-1, kv_heads, hs)[[t * page + i for t in cache.table[b] for i in range(page)][:n]] for b, n in enumerate(lens)]
        assert all(np.isfinite(a).all() for a in ks + vs)
        over_pages = kx.prompt_attention(q, cu, pool=cache.pool, table=cache.table, seq_lens=lens, kind=kind)
        check_prompt(q, cu, ks, vs, over_pages, kind, 0.125)
        if step == 0:  # packed rows, ahead of any cache
            got = kx.prompt_attention(q, cu, np.concatenate(ks), np.concatenate(vs), kind=kind)
            check_prompt(q, cu, ks, vs, got, kind, 0.125)
        if step >= 2:
            got = kx.paged_decode(cache.pool, cache.table, lens, q, scale=0.125, q_kind=kind)
            cache.k, cache.v = ks, vs
            check_decode(cache, q, got, 0, 0.125, kind, lens=lens)
            flat = kx.mha_decode(q[0].reshape(-1), ks[0].reshape(1, -1, kv_heads * hs), vs[0].reshape(1, -1, kv_heads * hs),
                                 lens[0] - 1, heads, heads // kv_heads, hs, 0)
            assert np.abs(got[0] - flat).max() <= E[kind] * 4 * np.abs(flat).max() + 2e-5
        done = lens
    logits = rounded((got.reshape(3, -1) @ rng.standard_normal((heads * hs, 997))).astype(np.float32), kind)
    best = [int(np.argmax(row)) for row in logits]
    out = kx.token_logprobs(logits, best, 4, kind)
    np.testing.assert_array_equal(out[2][:, 0], best)
    check_logprobs(logits, best, 4, out, kind)


def test_calls_on_two_streams():
    """Two batches on two streams, each with its own workspace, in flight together."""
    rng = np.random.default_rng(71)
    jobs = []
    for n in (5000, 3000):
        cache = Cache(rng, [n, 17, n // 3], 2, 64, 16, kx.F16)
        q = rng.standard_normal((3, 8, 64)).astype(np.float32)
        x = (rng.standard_normal((2, 40000)) * 3).astype(np.float32)
        b = dict(q=kx.Buf.from_numpy(q), out=kx.Buf.zeros(q.shape), t=kx.Buf.from_numpy(cache.table),
                 l=kx.Buf.from_numpy(np.array(cache.lens, np.int32)), x=kx.Buf.from_numpy(x), e=kx.Buf.zeros(2),
                 ids=kx.Buf.zeros((2, 4), np.int32), tl=kx.Buf.zeros((2, 4)),
                 w=kx.Buf.zeros(kx.lib().kx_paged_decode_workspace_bytes(3, 8, 2, 64), np.uint8),
                 w2=kx.Buf.zeros(kx.lib().kx_token_logprobs_workspace_bytes(2, 40000, 4), np.uint8))
        d = kx.PagedDecodeDesc(kv=cache.pool.desc(b["t"], b["l"]), q_type=kx.F32, head_num=8, scale=0.125, q=b["q"].ptr,
                               q_stride=512, out=b["out"].ptr, out_stride=512, workspace=b["w"].ptr, workspace_bytes=b["w"].nbytes)
        lp = kx.LogprobsDesc(type=kx.F32, rows=2, vocab=40000, top_n=4, logits=b["x"].ptr, row_stride=40000,
                             entropy=b["e"].ptr, top_ids=b["ids"].ptr, top_logprobs=b["tl"].ptr,
                             workspace=b["w2"].ptr, workspace_bytes=b["w2"].nbytes)
        jobs.append((cache, q, x, b, d, lp, kx.Stream()))
    kx.sync()
    for _ in range(20):
        for *_, d, lp, s in jobs:
            kx.check(kx.lib().kx_paged_decode(C.byref(d), s.ptr))
            kx.check(kx.lib().kx_token_logprobs(C.byref(lp), s.ptr))
    kx.sync()
    for cache, q, x, b, *_ in jobs:
        check_decode(cache, q, b["out"].numpy(), 0, 0.125, kx.F32)
        check_logprobs(x, None, 4, (None, b["e"].numpy(), b["ids"].numpy(), b["tl"].numpy()), kx.F32)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16], ids=lambda k: NAMES[k])
def test_windows_longer_than_anything(kind):
    """A window of 2^31 - 1 is none, with rows ahead of the first key as well."""
    rng = np.random.default_rng(81)
    cu, ck = [0, 90, 160], [0, 20, 220]
    q, k, v = (rounded(rng.standard_normal((n, m, 64)).astype(np.float32), kind) for n, m in ((160, 4), (220, 2), (220, 2)))
    parts = [(k[a:b], v[a:b]) for a, b in ((0, 20), (20, 220))]
    got = kx.prompt_attention(q, cu, k, v, cu_k=ck, window=2 ** 31 - 1, kind=kind)
    check_prompt(q, cu, [p[0] for p in parts], [p[1] for p in parts], got, kind, 0.125)
    assert (got[:70] == 0).all() and (got[70:90] != 0).all()
    cache = Cache(rng, [1, 300], 2, 64, 16, kind)
    got = kx.paged_decode(cache.pool, cache.table, cache.lens, q[:2], window=2 ** 31 - 1, q_kind=kind)
    check_decode(cache, q[:2], got, 0, 0.125, kind)


def test_one_workspace_for_all_that_meet_in_it():
    """Decode and log probabilities of several sizes take turns in one workspace."""
    rng = np.random.default_rng(82)
    L = kx.lib()
    ws = kx.Buf.zeros(max(L.kx_paged_decode_workspace_bytes(9, 40, 8, 128), L.kx_paged_decode_workspace_bytes(1, 4, 1, 64),
                          L.kx_token_logprobs_workspace_bytes(512, 5000, 32)), np.uint8)
    wide, one = Cache(rng, [900, 40, 7000] + [5] * 6, 8, 128, 16, kx.BF16), Cache(rng, [9000], 1, 64, 16, kx.F16)
    q, q1 = rng.standard_normal((9, 40, 128)).astype(np.float32), rng.standard_normal((1, 4, 64)).astype(np.float32)
    few, many = (rng.standard_normal((2, 90000)) * 3).astype(np.float32), rng.standard_normal((512, 5000)).astype(np.float32)
    first = None
    for turn in range(3):
        got = (kx.paged_decode(wide.pool, wide.table, wide.lens, q, workspace=ws),
               *kx.token_logprobs(many, None, 32, workspace=ws)[1:],
               kx.paged_decode(one.pool, one.table, one.lens, q1, workspace=ws),
               *kx.token_logprobs(few, None, 5, workspace=ws)[1:])
        if turn == 0:
            first = got
            check_decode(wide, q, got[0], 0, 128 ** -0.5, kx.F32)
            check_decode(one, q1, got[4], 0, 0.125, kx.F32)
            check_logprobs(many, None, 32, (None, *got[1:4]), kx.F32)
            check_logprobs(few, None, 5, (None, *got[5:]), kx.F32)
        for a, b in zip(first, got):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("kind", [kx.F32, kx.F16, kx.BF16], ids=lambda k: NAMES[k])
def test_a_step_captured_and_replayed(kind):
    """Filing, attention of the new rows, attention of the last one and the log probabilities as one graph, replayed as
    the rows' dealing over the sequences, the lengths and the pages change; each replay against eager calls."""
    rng = np.random.default_rng(83)
    heads, kv_heads, hs, page, rows, batch, vocab = 8, 2, 64, 16, 48, 3, 40000
    width, wide = KINDW[kind], kx.KIND_DTYPE[kind]
    pages = np.zeros((60, page, kv_heads, hs), np.float32)
    pool, other = kx.PagePool(pages, pages, kind), kx.PagePool(pages, pages, kind)
    tables = rope_tables(400, hs)
    sin, cos = (kx.Buf.from_numpy(t) for t in tables)
    b = dict(k=kx.Buf(rows * kv_heads * hs * width), v=kx.Buf(rows * kv_heads * hs * width), q=kx.Buf(rows * heads * hs * width),
             qo=kx.Buf.zeros((rows, heads, hs), wide), o=kx.Buf.zeros((rows, heads, hs), wide), d=kx.Buf.zeros((batch, heads, hs), wide),
             x=kx.Buf(batch * vocab * width), lp=kx.Buf.zeros(batch), en=kx.Buf.zeros(batch), ids=kx.Buf.zeros((batch, 4), np.int32),
             tl=kx.Buf.zeros((batch, 4)))
    table, lens, cu = kx.Buf.zeros((batch, 20), np.int32), kx.Buf.zeros(batch, np.int32), kx.Buf.zeros(batch + 1, np.int32)
    token = kx.Buf.zeros(batch, np.int32)
    L = kx.lib()
    ws = kx.Buf.zeros(max(L.kx_paged_decode_workspace_bytes(batch, heads, kv_heads, hs), L.kx_token_logprobs_workspace_bytes(batch, vocab, 4)), np.uint8)
    kv = pool.desc(table, lens)
    n, m = heads * hs, kv_heads * hs
    w = kx.PagedWriteDesc(kv=kv, src_type=kind, rows=rows, head_num=heads, rope_variant=1, table_rows=400, cu_rows=cu.ptr,
                          k=b["k"].ptr, k_stride=m, v=b["v"].ptr, v_stride=m, q=b["q"].ptr, q_stride=n, q_out=b["qo"].ptr,
                          q_out_stride=n, sin_cache=sin.ptr, cos_cache=cos.ptr)
    p = kx.PromptAttnDesc(type=kind, head_num=heads, kv_head_num=kv_heads, head_size=hs, batch=batch, q_rows=rows, causal=1,
                          scale=0.125, q=b["qo"].ptr, q_stride=n, out=b["o"].ptr, out_stride=n, cu_q=cu.ptr, pages=C.addressof(kv))
    d = kx.PagedDecodeDesc(kv=kv, q_type=kind, head_num=heads, scale=0.125, q=b["qo"].ptr, q_stride=n, out=b["d"].ptr,
                           out_stride=n, workspace=ws.ptr, workspace_bytes=ws.nbytes)
    x = kx.LogprobsDesc(type=kind, rows=batch, vocab=vocab, top_n=4, logits=b["x"].ptr, row_stride=vocab, tokens=token.ptr,
                        logprob=b["lp"].ptr, entropy=b["en"].ptr, top_ids=b["ids"].ptr, top_logprobs=b["tl"].ptr,
                        workspace=ws.ptr, workspace_bytes=ws.nbytes)
    stream, graph = kx.Stream(), C.c_void_p()
    kx.check(L.kx_graph_begin_capture(stream.ptr))
    for f, what in ((L.kx_paged_write, w), (L.kx_prompt_attention, p), (L.kx_paged_decode, d), (L.kx_token_logprobs, x)):
        kx.check(f(C.byref(what), stream.ptr))
    kx.check(L.kx_graph_end_capture(stream.ptr, C.byref(graph)))
    have = np.zeros(batch, int)
    where = rng.permutation(60).reshape(batch, 20).astype(np.int32)
    table.upload(where)
    for new in ([16, 16, 16], [48, 0, 0], [1, 1, 1], [0, 40, 8], [3, 20, 25], [1, 0, 2]):
        have += new
        bounds = np.cumsum([0] + new)
        q, k, v = (rounded(rng.standard_normal((rows, g, hs)).astype(np.float32), kind) for g in (heads, kv_heads, kv_heads))
        logits, tokens = rounded((rng.standard_normal((batch, vocab)) * 3).astype(np.float32), kind), rng.integers(0, vocab, batch)
        for name, a in (("q", q), ("k", k), ("v", v), ("x", logits)):
            b[name].upload(kx.to_kind(a, kind))
        cu.upload(bounds.astype(np.int32))
        lens.upload(have.astype(np.int32))
        token.upload(tokens.astype(np.int32))
        kx.check(L.kx_graph_launch(graph, stream.ptr))
        stream.sync()
        last = bounds[-1]
        eager_q = kx.paged_write(other, where, have, bounds, k, v, q, tables, 1, kind)
        for a, c in zip(pool.read(), other.read()):
            np.testing.assert_array_equal(a, c)
        got_q, out = (kx.from_kind(b[name].numpy(wide, (rows, heads, hs)), kind) for name in ("qo", "o"))
        np.testing.assert_array_equal(got_q[:last], eager_q[:last])
        eager = kx.prompt_attention(eager_q, bounds, pool=other, table=where, seq_lens=have, scale=0.125, kind=kind)
        np.testing.assert_array_equal(out[:last], eager[:last])
        one = kx.paged_decode(other, where, have, got_q[:batch], scale=0.125, q_kind=kind)
        np.testing.assert_array_equal(kx.from_kind(b["d"].numpy(wide, (batch, heads, hs)), kind), one)
        said = kx.token_logprobs(logits, tokens, 4, kind)
        for a, c in zip(said, (b["lp"].numpy(), b["en"].numpy(), b["ids"].numpy(), b["tl"].numpy())):
            np.testing.assert_array_equal(a, c)
        check_logprobs(logits, tokens, 4, said, kind)
    L.kx_graph_destroy(graph)
