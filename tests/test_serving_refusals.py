"""What the entries of batched serving refuse, found on the host before anything is launched (no GPU needed)."""
import ctypes as C

import pytest

import kx

EINVAL, EUNSUPPORTED, EWORKSPACE, ELIMIT = -1, -2, -3, -4
P = 1 << 20  # a 16-byte aligned address that nothing reads


def pages(**kw):
    d = dict(type=kx.F16, kv_head_num=2, head_size=64, page_size=16, num_pages=8, table_pages=4, batch=2, key=P,
             value=P, page_stride=16 * 128, row_stride=128, head_stride=64, table=P, table_stride=4, seq_lens=P)
    d.update(kw)
    return kx.PagedKv(**d)


BAD_PAGES = [(dict(type=3), EINVAL), (dict(type=-1), EINVAL), (dict(kv_head_num=0), EINVAL), (dict(page_size=0), EINVAL),
             (dict(num_pages=0), EINVAL), (dict(table_pages=0), EINVAL), (dict(key=None), EINVAL),
             (dict(value=None), EINVAL), (dict(key=P + 8), EINVAL), (dict(value=P + 2), EINVAL), (dict(table=None), EINVAL),
             (dict(table=P + 1), EINVAL), (dict(seq_lens=None), EINVAL), (dict(head_size=48), EUNSUPPORTED),
             (dict(head_size=0), EUNSUPPORTED), (dict(page_stride=32), EINVAL), (dict(row_stride=132), EINVAL),
             (dict(head_stride=0), EINVAL), (dict(table_stride=3), EINVAL), (dict(batch=-1), EINVAL),
             (dict(page_size=1 << 16, table_pages=1 << 15, table_stride=1 << 15), EINVAL),
             (dict(page_size=0x7FFFFF01, table_pages=1), EINVAL)]


def write(kv=None, **kw):
    d = dict(kv=kv or pages(), src_type=kx.F32, rows=5, head_num=4, rope_variant=1, table_rows=64, cu_rows=P, k=P,
             k_stride=128, v=P, v_stride=128, q=P, q_stride=256, q_out=P, q_out_stride=256, sin_cache=P, cos_cache=P)
    d.update(kw)
    return kx.lib().kx_paged_write(C.byref(kx.PagedWriteDesc(**d)), None)


def decode(kv=None, **kw):
    d = dict(kv=kv or pages(), q_type=kx.F32, head_num=4, window=0, scale=1.0, q=P, q_stride=256, out=P, out_stride=256,
             workspace=P, workspace_bytes=1 << 30)
    d.update(kw)
    return kx.lib().kx_paged_decode(C.byref(kx.PagedDecodeDesc(**d)), None)


def prompt(**kw):
    d = dict(type=kx.F16, head_num=4, kv_head_num=2, head_size=64, batch=2, q_rows=5, k_rows=5, causal=1, window=0,
             scale=1.0, q=P, q_stride=256, k=P, k_stride=128, v=P, v_stride=128, out=P, out_stride=256, cu_q=P, cu_k=P)
    d.update(kw)
    return kx.lib().kx_prompt_attention(C.byref(kx.PromptAttnDesc(**d)), None)


def logprobs(**kw):
    d = dict(type=kx.F32, rows=3, vocab=100, top_n=5, logits=P, row_stride=100, tokens=P, logprob=P, entropy=P,
             top_ids=P, top_logprobs=P, workspace=P, workspace_bytes=1 << 30)
    d.update(kw)
    return kx.lib().kx_token_logprobs(C.byref(kx.LogprobsDesc(**d)), None)


@pytest.mark.parametrize("bad,code", BAD_PAGES)
def test_pages(bad, code):
    assert write(kv=pages(**bad)) == code
    assert decode(kv=pages(**bad)) == code
    if "batch" not in bad:
        p = pages(**bad)
        assert prompt(k=None, v=None, cu_k=None, pages=C.addressof(p)) == code


@pytest.mark.parametrize("bad,code", [
    (dict(rows=-1), EINVAL), (dict(src_type=7), EINVAL), (dict(src_type=kx.BF16), EUNSUPPORTED), (dict(cu_rows=None), EINVAL),
    (dict(cu_rows=P + 2), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(k=P + 4), EINVAL), (dict(k_stride=126), EINVAL),
    (dict(k_stride=130), EINVAL), (dict(v_stride=0), EINVAL), (dict(q_out=None), EINVAL), (dict(q=None), EINVAL),
    (dict(q_stride=252), EINVAL), (dict(q_out_stride=258), EINVAL), (dict(q=P + 8), EINVAL), (dict(q_out=P + 8), EINVAL), (dict(head_num=0), EINVAL),
    (dict(sin_cache=None), EINVAL), (dict(cos_cache=None), EINVAL), (dict(sin_cache=None, cos_cache=None), EINVAL),
    (dict(table_rows=0), EINVAL), (dict(rope_variant=2), EINVAL), (dict(q_out_stride=264), EINVAL), (dict(rows=1 << 25), ELIMIT),
    (dict(sin_cache=P + 2), EINVAL), (dict(cos_cache=P + 2), EINVAL),
    (dict(head_num=1 << 24, q_stride=1 << 30, q_out_stride=1 << 30), ELIMIT)])
def test_write(bad, code):
    assert write(**bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(q_type=5), EINVAL), (dict(q_type=kx.BF16), EUNSUPPORTED), (dict(head_num=3), EINVAL), (dict(head_num=0), EINVAL),
    (dict(window=-1), EINVAL), (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(q=P + 4), EINVAL),
    (dict(out=P + 8), EINVAL), (dict(q_stride=255), EINVAL), (dict(q_stride=258), EINVAL), (dict(out_stride=128), EINVAL),
    (dict(workspace=None), EWORKSPACE), (dict(workspace=P + 16), EINVAL), (dict(workspace_bytes=64), EWORKSPACE), (dict(scale=float("nan")), EINVAL), (dict(scale=float("inf")), EINVAL)])
def test_decode(bad, code):
    assert decode(**bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(type=4), EINVAL), (dict(head_num=5), EINVAL), (dict(kv_head_num=0), EINVAL), (dict(head_size=256), EUNSUPPORTED),
    (dict(batch=-1), EINVAL), (dict(q_rows=-1), EINVAL), (dict(k_rows=-1), EINVAL), (dict(window=-4), EINVAL),
    (dict(window=4, causal=0), EINVAL), (dict(q=None), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL),
    (dict(out=None), EINVAL), (dict(cu_q=None), EINVAL), (dict(cu_k=None), EINVAL), (dict(cu_q=P + 2), EINVAL),
    (dict(q=P + 2), EINVAL), (dict(v=P + 8), EINVAL), (dict(q_stride=260), EINVAL), (dict(k_stride=120), EINVAL),
    (dict(v_stride=132), EINVAL), (dict(out_stride=0), EINVAL), (dict(scale=float("nan")), EINVAL),
    (dict(k_stride=1 << 22), EUNSUPPORTED), (dict(v_stride=1 << 22), EUNSUPPORTED), (dict(q_rows=1 << 30), ELIMIT),
    (dict(k_rows=0x7FFFFF01), ELIMIT), (dict(q_rows=1 << 30, head_num=2), ELIMIT), (dict(batch=1 << 22), ELIMIT)])
def test_prompt(bad, code):
    assert prompt(**bad) == code


@pytest.mark.parametrize("bad", [dict(page_stride=1 << 31), dict(row_stride=1 << 26)])
def test_prompt_over_pages_far_apart(bad):
    p = pages(**bad)
    assert prompt(k=None, v=None, cu_k=None, pages=C.addressof(p)) == EUNSUPPORTED


@pytest.mark.parametrize("heads,batch,code", [(1025, 2, EUNSUPPORTED), (2, 1 << 23, ELIMIT)])
def test_decode_limits(heads, batch, code):
    assert decode(kv=pages(kv_head_num=heads, batch=batch), head_num=heads, q_stride=heads * 64, out_stride=heads * 64) == code


@pytest.mark.parametrize("bad,code", [
    (dict(), EINVAL), (dict(type=kx.BF16), EUNSUPPORTED), (dict(kv_head_num=4), EINVAL), (dict(batch=3), EINVAL),
    (dict(head_size=32, q_stride=128), EINVAL)])
def test_prompt_over_pages(bad, code):
    p = pages()
    kw = dict(pages=C.addressof(p), **({} if not bad else dict(k=None, v=None, cu_k=None)))  # {}: both sources
    assert prompt(**kw, **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(type=3), EINVAL), (dict(rows=-1), EINVAL), (dict(vocab=0), EINVAL), (dict(row_stride=99), EINVAL),
    (dict(logits=None), EINVAL), (dict(logits=P + 2), EINVAL), (dict(tokens=None), EINVAL), (dict(logprob=None), EINVAL),
    (dict(top_n=-1), EINVAL), (dict(top_n=33), EINVAL), (dict(top_n=6, vocab=5), EINVAL), (dict(top_ids=None), EINVAL),
    (dict(top_logprobs=None), EINVAL), (dict(workspace=None), EWORKSPACE), (dict(workspace=P + 8), EINVAL),
    (dict(workspace_bytes=16), EWORKSPACE), (dict(rows=1 << 24), ELIMIT), (dict(tokens=P + 2), EINVAL),
    (dict(logprob=P + 1), EINVAL), (dict(entropy=P + 2), EINVAL), (dict(top_ids=P + 2), EINVAL), (dict(top_logprobs=P + 3), EINVAL),
    (dict(vocab=0x7FFFFF01, row_stride=0x7FFFFF01), ELIMIT)])
def test_logprobs(bad, code):
    assert logprobs(**bad) == code


def test_nothing_to_do():
    assert write(rows=0) == 0 and write(kv=pages(batch=0)) == 0 and decode(kv=pages(batch=0)) == 0
    assert prompt(batch=0) == 0 and prompt(q_rows=0) == 0 and logprobs(rows=0) == 0


def test_no_description():
    L = kx.lib()
    assert [f(None, None) for f in (L.kx_paged_write, L.kx_paged_decode, L.kx_prompt_attention, L.kx_token_logprobs)] \
        == [EINVAL] * 4


def test_workspace_sizes():
    L = kx.lib()
    assert L.kx_paged_decode_workspace_bytes(0, 8, 2, 64) == 0 and L.kx_paged_decode_workspace_bytes(1, 8, 3, 64) == 0
    one, many = L.kx_paged_decode_workspace_bytes(1, 32, 8, 128), L.kx_paged_decode_workspace_bytes(512, 32, 8, 128)
    assert 0 < one <= many < 256 << 20
    assert L.kx_token_logprobs_workspace_bytes(0, 10, 5) == 0
    assert 0 < L.kx_token_logprobs_workspace_bytes(1, 128256, 20) < 64 << 20
