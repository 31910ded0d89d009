"""The operators of batched serving -- a paged key/value cache, the attention that reads it, the attention over
packed prompts, and the log probabilities of an answer's tokens -- as a user's program calls them, beside their
plain form in elementary torch operations.

  own = False   run() computes the plain form: 32-bit arithmetic, rounded once at the end
  own = True    run() makes the calls of this framework (package `kx`)

listed() names the cases that stand for the range of real use, draw() gives further ones, prepare() makes what a
program has in hand before the call, work() says what a pass cannot do without, and exact() computes the
definition in 64 bits.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
ROPE_THETA = 5e5
WORKSPACE_BYTES = 64 << 20  # scratch that a serving program keeps for its stream


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat, a short context: a serving program at its least load, where latency counts.  Llama-3-8B heads,
        # the framework's own fp32 queries over its 16-bit cache
        dict(name="decode one short chat", op="decode", heads=32, kv_heads=8, head_size=128, q="f32", kv="f16",
             page=16, batch=1, short=137, long=137, window=0, shape=1),
        # a loaded server: 48 chats between a few tokens and 8k, one of them just begun
        dict(name="decode ragged batch", op="decode", heads=32, kv_heads=8, head_size=128, q="bf16", kv="bf16",
             page=64, batch=48, short=1, long=8192, window=0, shape=2),
        # few long documents: the cache is read at the memory's rate, the split over its length carries it.
        # Llama-3-70B heads
        dict(name="decode long documents", op="decode", heads=64, kv_heads=8, head_size=128, q="f16", kv="f16",
             page=32, batch=3, short=60000, long=131072, window=0, shape=3),
        # the reference's cache type, Qwen2.5-7B heads (seven per kv head), pages of a size that is no power of two
        dict(name="decode fp32 cache", op="decode", heads=28, kv_heads=4, head_size=128, q="f32", kv="f32",
             page=48, batch=16, short=500, long=4400, window=0, shape=4),
        # the benchmark's prompt: 4096 tokens, Llama-3-8B heads
        dict(name="prompt of 4096", op="prompt", heads=32, kv_heads=8, head_size=128, type="bf16", batch=1,
             short=4096, long=4096, cached=0, window=0, page=0, shape=5),
        # prompts of very different lengths packed into one pass, Llama-3.2-1B heads
        dict(name="prompts packed", op="prompt", heads=32, kv_heads=8, head_size=64, type="f16", batch=12,
             short=1, long=2500, cached=0, window=0, page=0, shape=6),
        # the next pieces of long prompts, read from the pages that hold what came before
        dict(name="prompt pieces over pages", op="prompt", heads=32, kv_heads=8, head_size=128, type="bf16", batch=6,
             short=100, long=1024, cached=6000, window=0, page=32, shape=7),
        # short prompts in the reference's type
        dict(name="prompts fp32", op="prompt", heads=12, kv_heads=12, head_size=64, type="f32", batch=7,
             short=3, long=300, cached=0, window=0, page=0, shape=8),
        # one new token of each of 64 chats, from the fp32 projections into a 16-bit cache
        dict(name="write one row each", op="write", heads=32, kv_heads=8, head_size=128, src="f32", kv="f16",
             page=16, batch=64, new=1, long=2048, variant=1, shape=9),
        # whole prompts into the cache
        dict(name="write prompts", op="write", heads=32, kv_heads=8, head_size=128, src="bf16", kv="bf16",
             page=64, batch=9, new=1500, long=4096, variant=1, shape=10),
        # the next token of one chat with its 20 best alternatives, Llama-3 vocabulary
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=128256, type="f32", top=20, masked=False, shape=11),
        # the scoring of a text: every position of 2048, Qwen2.5 vocabulary
        dict(name="logprobs of a text", op="logprobs", rows=2048, vocab=152064, type="bf16", top=5, masked=True,
             shape=12),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "write", "logprobs"])
    shape = rng.randrange(1 << 30)
    if op == "logprobs":
        vocab = _spread(rng, 320, 152064)
        rows = _spread(rng, 1, min(4096, 2048 * 152064 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, type=rng.choice(["f32", "f16", "bf16"]) if rows * vocab < 150e6
                    else "bf16", top=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.5, shape=shape)
    heads, kv_heads, hs = rng.choice([(32, 8, 128), (32, 8, 64), (28, 4, 128), (64, 8, 128), (12, 12, 64), (8, 1, 128),
                                      (4, 2, 32), (40, 2, 128)])
    page = rng.choice([1, 16, 16, 24, 32, 64, 128])
    if op == "decode":
        batch = _spread(rng, 1, 200)
        longest = _spread(rng, 16, min(65536, 300000 * 4 // (batch * kv_heads) + 16))
        q, kv = rng.choice([("f32", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_size=hs, q=q, kv=kv, page=page, batch=batch,
                    short=_spread(rng, 1, longest), long=longest,
                    window=rng.choice([0, 0, 0, _spread(rng, 4, longest)]), shape=shape)
    if op == "prompt":
        batch = _spread(rng, 1, 16)
        longest = _spread(rng, 8, min(4096, int(4096 / math.sqrt(batch * max(heads, 32) / 32))))
        kind = rng.choice(["f32", "f16", "bf16", "bf16"])
        if kind == "f32":
            longest = min(longest, 1500)
        paged = rng.random() < 0.4
        return dict(op=op, heads=heads, kv_heads=kv_heads, head_size=hs, type=kind, batch=batch,
                    short=_spread(rng, 1, longest), long=longest, cached=_spread(rng, 1, 2000) if paged else 0,
                    window=rng.choice([0, 0, 0, _spread(rng, 4, longest)]), page=page if paged else 0, shape=shape)
    src, kv = rng.choice([("f32", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    batch = _spread(rng, 1, 64)
    new = rng.choice([1, _spread(rng, 2, 4000 // batch + 2)])
    return dict(op=op, heads=heads, kv_heads=kv_heads, head_size=hs, src=src, kv=kv, page=page, batch=batch, new=new,
                long=new + _spread(rng, 1, 2048), variant=rng.choice([0, 1]), shape=shape)


def _lengths(c):
    """The lengths of a case's sequences: (new rows, rows of the cache with the new ones), a list each."""
    r = random.Random(c["shape"])
    if c["op"] == "write":
        new = [c["new"] if c["new"] == 1 else r.randint(1, c["new"]) for _ in range(c["batch"])]
        return new, [n + r.randint(0, c["long"] - n) for n in new]
    some = [_spread(r, c["short"], c["long"]) for _ in range(c["batch"])]
    some[0] = c["long"]
    if c["op"] == "decode":
        return [1] * c["batch"], some
    return some, [n + r.randint(0, c["cached"]) for n in some]


def _seen(new, total, window):
    """Key rows that the `new` last positions of a sequence of `total` see."""
    if not window:
        return new * total - new * (new - 1) // 2
    full = total - new + 1
    return sum(min(window, full + i) for i in range(new))


def work(c):
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * BYTES[c["type"]] + c["rows"] * (12 + 8 * c["top"]), "flops": 6 * n}
    new, total = _lengths(c)
    h, kvh, hs = c["heads"], c["kv_heads"], c["head_size"]
    if c["op"] == "write":
        b = sum(new) * hs * (2 * h * BYTES[c["src"]] + 2 * kvh * (BYTES[c["src"]] + BYTES[c["kv"]]) + 4)
        return {"bytes": b, "flops": 3 * sum(new) * hs * (h + kvh)}
    w = c["window"]
    kv = c["kv"] if c["op"] == "decode" else c["type"]
    rows = sum(min(t, w + n - 1) if w else t for n, t in zip(new, total))
    b = 2 * rows * kvh * hs * BYTES[kv] + 2 * sum(new) * h * hs * BYTES[c["q"] if c["op"] == "decode" else c["type"]]
    return {"bytes": b, "flops": 4 * h * hs * sum(_seen(n, t, w) for n, t in zip(new, total))}


# ------------------------------------------------------------------ what a program has in hand
def _cumulated(lengths, device):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).to(torch.int32).to(device)


def _pages(c, total, kind, gen, device):
    """A pool of pages with random rows in it, and a table that deals its pages out in no order."""
    page = c["page"]
    columns = max((t + page - 1) // page for t in total)
    count = sum((t + page - 1) // page for t in total)
    order = torch.randperm(count + 3, generator=gen, device=device).to(torch.int32)
    table = torch.zeros(len(total), columns, dtype=torch.int32, device=device)
    held = torch.tensor([(t + page - 1) // page for t in total], device=device)
    table[torch.arange(columns, device=device)[None] < held[:, None]] = order[:count]
    shape = (count + 3, page, c["kv_heads"], c["head_size"])
    key = torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(kind)
    value = torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(kind)
    return key, value, table


def prepare(case, seed):
    c = dict(case)
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)

    def rand(*shape, kind=torch.float32):
        return torch.randn(shape, generator=gen, device=device, dtype=torch.float32).to(kind)

    s = {"case": c, "workspace": torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=device)}
    if c["op"] == "logprobs":
        rows, vocab, top = c["rows"], c["vocab"], c["top"]
        x = rand(rows, vocab).mul_(2.5)
        likely = torch.randint(vocab, (rows,), generator=gen, device=device)
        x[torch.arange(rows, device=device), likely] += 11.0
        taken = torch.where(torch.rand(rows, generator=gen, device=device) < 0.7, likely,
                            torch.randint(vocab, (rows,), generator=gen, device=device))
        if c["masked"]:  # a grammar that forbids half of the vocabulary in every third row
            even = (torch.arange(vocab, device=device) % 2 == 0)[None] & (torch.arange(rows, device=device) % 3 == 0)[:, None]
            even[torch.arange(rows, device=device), taken] = False
            x.masked_fill_(even, float("-inf"))
        s.update(logits=x.to(TYPES[c["type"]]), tokens=taken.to(torch.int32),
                 logprob=torch.empty(rows, device=device), entropy=torch.empty(rows, device=device),
                 top_ids=torch.empty(rows, top, dtype=torch.int32, device=device),
                 top_logprobs=torch.empty(rows, top, device=device))
        return s
    new, total = _lengths(c)
    h, kvh, hs = c["heads"], c["kv_heads"], c["head_size"]
    rows = sum(new)
    s.update(rows=rows, longest_new=max(new), longest=max(total), cu_q=_cumulated(new, device),
             seq_lens=torch.tensor(total, dtype=torch.int32, device=device), scale=1.0 / math.sqrt(hs))
    if c["op"] == "decode":
        s["key"], s["value"], s["table"] = _pages(c, total, TYPES[c["kv"]], gen, device)
        s["q"] = rand(rows, h, hs, kind=TYPES[c["q"]])
        s["out"] = torch.empty_like(s["q"])
    elif c["op"] == "prompt":
        kind = TYPES[c["type"]]
        if c["page"]:
            s["key"], s["value"], s["table"] = _pages(c, total, kind, gen, device)
            s["q"] = rand(rows, h, hs, kind=kind)
        else:  # as the projection leaves them: q, k and v beside each other in one row
            s["qkv"] = rand(rows, h + 2 * kvh, hs, kind=kind)
            s["q"], s["key"], s["value"] = s["qkv"].split([h, kvh, kvh], dim=1)
        s["out"] = torch.empty(rows, h, hs, dtype=kind, device=device)
    else:
        s["key"], s["value"], s["table"] = _pages(c, total, TYPES[c["kv"]], gen, device)
        kind = TYPES[c["src"]]
        s["q"], s["k"], s["v"] = rand(rows, h, hs, kind=kind), rand(rows, kvh, hs, kind=kind), rand(rows, kvh, hs, kind=kind)
        s["q_out"] = torch.empty_like(s["q"])
        angle = torch.arange(max(total), device=device, dtype=torch.float64)[:, None] \
            * ROPE_THETA ** (-torch.arange(hs, device=device, dtype=torch.float64) / hs)[None]
        s["sin"], s["cos"] = angle.sin().float(), angle.cos().float()
    return s


# ------------------------------------------------------------------ the plain forms
def _paged_rows(pool, table, page, longest):
    """[sequence][position] of the rows that a table names, with those of the table's end repeated behind it."""
    used = table[:, :(longest + page - 1) // page].long()
    return pool[used].flatten(1, 2)[:, :longest]


def _attend(q, k, v, seen, scale):
    """q [B, G, M, d], k and v [B, G, L, d] in 32 bits, seen [B, 1, M, L]: softmax(scale q k^T) v over what is seen."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(scale).masked_fill_(~seen, float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    return torch.matmul(x, v) / x.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_decode(s):
    c = s["case"]
    b, kvh, hs, w = c["batch"], c["kv_heads"], c["head_size"], c["window"]
    g = c["heads"] // kvh
    k = _paged_rows(s["key"], s["table"], c["page"], s["longest"]).float().transpose(1, 2).contiguous()
    v = _paged_rows(s["value"], s["table"], c["page"], s["longest"]).float().transpose(1, 2).contiguous()
    at = torch.arange(s["longest"], device=k.device)[None]
    last = s["seq_lens"][:, None] - 1
    seen = at <= last
    if w:
        seen &= at > last - w
    o = _attend(s["q"].float().view(b, kvh, g, hs), k, v, seen[:, None, None], s["scale"])
    return o.reshape(b, c["heads"], hs).to(s["q"].dtype)


def _plain_prompt(s):
    c = s["case"]
    b, kvh, hs, w = c["batch"], c["kv_heads"], c["head_size"], c["window"]
    g, device, cu = c["heads"] // kvh, s["out"].device, s["cu_q"].long()
    n, total = cu[1:] - cu[:-1], s["seq_lens"].long()
    row = torch.arange(s["longest_new"], device=device)[None]
    inside = row < n[:, None]
    rows = (cu[:-1, None] + row).clamp_max(s["rows"] - 1)
    q = s["q"][rows].float()  # [B, M, H, d]
    q = q.view(b, -1, kvh, g, hs).permute(0, 2, 3, 1, 4).reshape(b, kvh, -1, hs).contiguous()
    if c["page"]:
        k = _paged_rows(s["key"], s["table"], c["page"], s["longest"]).float()
        v = _paged_rows(s["value"], s["table"], c["page"], s["longest"]).float()
    else:
        k, v = s["key"][rows].float(), s["value"][rows].float()
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    at = torch.arange(k.shape[2], device=device)[None, None]
    position = (total - n)[:, None, None] + row[..., None]
    seen = (at <= position) & (at < total[:, None, None])
    if w:
        seen &= at > position - w
    o = _attend(q, k, v, seen[:, None].repeat(1, 1, g, 1), s["scale"])
    o = o.view(b, kvh, g, -1, hs).permute(0, 3, 1, 2, 4).reshape(b, -1, c["heads"], hs)
    return o[inside].to(s["out"].dtype)


def _rotate(x, sin, cos, variant):
    """Pairs (2i, 2i+1) with variant 0, (i, i + d/2) with variant 1, turned by the angle of column 2i."""
    sin, cos = sin[:, None, 0::2], cos[:, None, 0::2]
    if variant == 0:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _slots(s):
    """The position of each new row, and its row in the pool."""
    c, cu = s["case"], s["cu_q"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(c["batch"], device=cu.device), n, output_size=s["rows"])
    position = torch.arange(s["rows"], device=cu.device) - cu[1:][seq] + s["seq_lens"].long()[seq]
    return position, s["table"][seq, position // c["page"]].long() * c["page"] + position % c["page"]


def _plain_write(s):
    c = s["case"]
    position, slot = _slots(s)
    sin, cos = s["sin"][position], s["cos"][position]
    q = _rotate(s["q"].float(), sin, cos, c["variant"]).to(s["q"].dtype)
    s["key"].flatten(0, 1)[slot] = _rotate(s["k"].float(), sin, cos, c["variant"]).to(s["key"].dtype)
    s["value"].flatten(0, 1)[slot] = s["v"].to(s["value"].dtype)
    return q, s["key"], s["value"]


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    logprob = (x.gather(1, s["tokens"].long()[:, None]) - lse)[:, 0]
    entropy = (z.log() - (e * torch.where(e > 0, x - m, 0.0)).sum(-1, keepdim=True) / z)[:, 0]
    if not top:
        return logprob, entropy
    # the order of the values as whole numbers, the lower index ahead among equal ones
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits) << 32
    ids = order.add_(0xffffffff - torch.arange(x.shape[1], device=x.device)).topk(top, -1).indices
    return logprob, entropy, ids.to(torch.int32), x.gather(1, ids) - lse


# ------------------------------------------------------------------ the framework's calls
def _kx():
    path = os.path.join(os.getcwd(), "llm-inference-engine_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import kx
    return kx


def _call(s):
    """The call that a program makes of an operator again and again: its description is filled in once."""
    kx, c = _kx(), s["case"]
    if c["op"] == "logprobs":
        d = kx.LogprobsDesc(type=CODES[c["type"]], rows=c["rows"], vocab=c["vocab"], top_n=c["top"],
                            logits=s["logits"].data_ptr(), row_stride=c["vocab"], tokens=s["tokens"].data_ptr(),
                            logprob=s["logprob"].data_ptr(), entropy=s["entropy"].data_ptr(),
                            top_ids=s["top_ids"].data_ptr(), top_logprobs=s["top_logprobs"].data_ptr(),
                            workspace=s["workspace"].data_ptr(), workspace_bytes=WORKSPACE_BYTES)
        out = (s["logprob"], s["entropy"]) + ((s["top_ids"], s["top_logprobs"]) if c["top"] else ())
        return kx, kx.lib().kx_token_logprobs, ctypes.byref(d), d, out
    h, kvh, hs = c["heads"], c["kv_heads"], c["head_size"]
    pages = None
    if c["page"]:
        pages = kx.PagedKv(type=CODES[c["type"] if c["op"] == "prompt" else c["kv"]], kv_head_num=kvh, head_size=hs,
                           page_size=c["page"], num_pages=s["key"].shape[0], table_pages=s["table"].shape[1],
                           batch=c["batch"], key=s["key"].data_ptr(), value=s["value"].data_ptr(),
                           page_stride=c["page"] * kvh * hs, row_stride=kvh * hs, head_stride=hs,
                           table=s["table"].data_ptr(), table_stride=s["table"].shape[1],
                           seq_lens=s["seq_lens"].data_ptr())
    if c["op"] == "decode":
        d = kx.PagedDecodeDesc(kv=pages, q_type=CODES[c["q"]], head_num=h, q=s["q"].data_ptr(), q_stride=h * hs,
                               out=s["out"].data_ptr(), out_stride=h * hs, scale=s["scale"], window=c["window"],
                               workspace=s["workspace"].data_ptr(), workspace_bytes=WORKSPACE_BYTES)
        return kx, kx.lib().kx_paged_decode, ctypes.byref(d), d, s["out"]
    if c["op"] == "prompt":
        d = kx.PromptAttnDesc(type=CODES[c["type"]], head_num=h, kv_head_num=kvh, head_size=hs, batch=c["batch"],
                              q_rows=s["rows"], causal=1, window=c["window"], scale=s["scale"],
                              q=s["q"].data_ptr(), q_stride=s["q"].stride(0), out=s["out"].data_ptr(),
                              out_stride=h * hs, cu_q=s["cu_q"].data_ptr())
        if pages is not None:
            d.pages = ctypes.addressof(pages)
        else:
            d.k, d.v, d.cu_k, d.k_rows = s["key"].data_ptr(), s["value"].data_ptr(), s["cu_q"].data_ptr(), s["rows"]
            d.k_stride, d.v_stride = s["key"].stride(0), s["value"].stride(0)
        return kx, kx.lib().kx_prompt_attention, ctypes.byref(d), (d, pages), s["out"]
    d = kx.PagedWriteDesc(kv=pages, src_type=CODES[c["src"]], rows=s["rows"], cu_rows=s["cu_q"].data_ptr(),
                          k=s["k"].data_ptr(), k_stride=kvh * hs, v=s["v"].data_ptr(), v_stride=kvh * hs,
                          q=s["q"].data_ptr(), q_stride=h * hs, q_out=s["q_out"].data_ptr(), q_out_stride=h * hs,
                          head_num=h, sin_cache=s["sin"].data_ptr(), cos_cache=s["cos"].data_ptr(),
                          table_rows=s["sin"].shape[0], rope_variant=c["variant"])
    return kx, kx.lib().kx_paged_write, ctypes.byref(d), d, (s["q_out"], s["key"], s["value"])


def run(s):
    if own:
        if "call" not in s:
            s["call"] = _call(s)
        kx, entry, desc, _, out = s["call"]
        kx.check(entry(desc, torch.cuda.current_stream().cuda_stream), s["case"]["op"])
        return out
    return {"decode": _plain_decode, "prompt": _plain_prompt, "write": _plain_write,
            "logprobs": _plain_logprobs}[s["case"]["op"]](s)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rows(s, b, total):
    """Key and value rows 0..total-1 of sequence b, [kv head][position][d] in 64 bits."""
    c = s["case"]
    if c["page"]:
        at = torch.arange(total, device=s["key"].device)
        rows = s["table"][b, at // c["page"]].long() * c["page"] + at % c["page"]
        return [p.reshape(-1, *p.shape[2:])[rows].double().permute(1, 0, 2) for p in (s["key"], s["value"])]
    lo = int(s["cu_q"][b])
    return [p[lo:lo + total].double().permute(1, 0, 2) for p in (s["key"], s["value"])]


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "logprobs":
        outs = []
        for r in range(0, c["rows"], 64):
            x = s["logits"][r:r + 64].double()
            p = torch.log_softmax(x, -1)
            outs.append((p.gather(1, s["tokens"][r:r + 64].long()[:, None])[:, 0],
                         -torch.where(p > -1e300, p.exp() * p, 0.0).sum(-1), p.sort(-1, descending=True).values[:, :c["top"]]))
        logprob, entropy, top = (torch.cat(o) for o in zip(*outs))
        return (logprob, entropy, None, top) if c["top"] else (logprob, entropy)
    new, total = _lengths(c)
    if c["op"] == "write":
        position, slot = _slots(s)
        half = c["head_size"] // 2

        def turned(x):
            y = x.double().clone()
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if c["variant"] == 0 else (i, i + half)
                sin, cos = s["sin"][position, 2 * i].double()[:, None], s["cos"][position, 2 * i].double()[:, None]
                y[..., a] = x[..., a].double() * cos - x[..., b].double() * sin
                y[..., b] = x[..., a].double() * sin + x[..., b].double() * cos
            return y

        key, value = s["key"].double(), s["value"].double()
        key.view(-1, *key.shape[2:])[slot] = turned(s["k"])
        value.view(-1, *value.shape[2:])[slot] = s["v"].double()
        return turned(s["q"]), key, value
    if sum(_seen(n, t, 0) for n, t in zip(new, total)) * c["heads"] * c["head_size"] > 4e12:
        return None
    g, out, first = c["heads"] // c["kv_heads"], [], 0
    for b, (n, t) in enumerate(zip(new, total)):
        q = s["q"][first:first + n].double()
        first += n
        k, v = _exact_rows(s, b, t)
        at = torch.arange(t, device=q.device)[None]
        position = torch.arange(t - n, t, device=q.device)[:, None]
        hidden = at > position
        if c["window"]:
            hidden |= at <= position - c["window"]
        o = torch.empty_like(q)
        for h in range(c["heads"]):
            x = (q[:, h] @ k[h // g].T.contiguous()) * s["scale"]
            o[:, h] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ v[h // g]
        out.append(o)
    return torch.cat(out)
