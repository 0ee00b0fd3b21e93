"""The attention operators of the prompt encoder's language model: what they compute, and calls to measure.

    packed   causal attention of packed sequences of different lengths with grouped heads
    write    new keys and values into the 8-bit cache, and the cache's rows read back
    attend   attention of new rows over the 8-bit cache

``run`` computes them from elementary torch operations, or, with ``own`` true, through libexn_b200's entry
points (Attention.packed, .cache_write, .cache_read, .cache_attend).  Head dimension 128 throughout, as the encoder.

The cache holds 64 tokens a page; a page has, for each key/value head, 64 x 128 codes of 8 bits and one scale, a
power of two: the smallest with max |x| <= 127 scale over the tokens the page has held so far.
"""
import math
import os
import random
import sys

import torch

own = False

DIM = 128
PAGE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

_handle = None


def _library():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ex-nihilo_b200"))
    import exn_b200
    return exn_b200


def _attention():
    """One Attention handle a process, as a serving program keeps one."""
    global _handle
    if _handle is None:
        _handle = _library().Attention(device=0)
    return _handle


def _ints(text):
    return [int(t) for t in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


def _spread(rng, n, lo, hi):
    """N lengths between LO and HI, spread over their logarithm."""
    return [int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) for _ in range(n)]


# ------------------------------------------------------------------------------------------------ the cases


def listed():
    r = random.Random(20)
    prompts = _spread(r, 14, 20, 300)
    decode = _spread(r, 64, 500, 8192)
    small = _spread(r, 64, 20, 120)
    return [
        # one short prompt of the encoder (32 query heads on 8): the call's latency
        dict(name="packed_short", op="packed", type="bf16", heads=32, kv_heads=8, q="27", k="", pad=0, fused=True),
        # a batch of picture prompts, an empty one and a single token among them, rows behind the last
        dict(name="packed_prompts", op="packed", type="bf16", heads=32, kv_heads=8, q=_text(prompts + [0, 1]), k="",
             pad=37, fused=False),
        # long prompts packed with short ones: the tensor cores' rate
        dict(name="packed_long", op="packed", type="bf16", heads=32, kv_heads=8, q="8192,5001,130,2999", k="", pad=0,
             fused=True),
        # every query head its own keys, in fp16, odd lengths
        dict(name="packed_mha", op="packed", type="fp16", heads=16, kv_heads=16, q="1025,63,2047,512", k="", pad=0,
             fused=False),
        # the last rows of longer sequences (a prompt whose first part is known): more keys than queries, and a
        # sequence with fewer keys than queries, whose first rows see nothing
        dict(name="packed_tail", op="packed", type="bf16", heads=28, kv_heads=4, q="300,77,512,9", k="4100,900,513,5",
             pad=3, fused=False),
        # one new token for each of 64 short prompts, pages partly filled
        dict(name="write_token", op="write", type="bf16", heads=32, kv_heads=8, new=_text([1] * 64),
             len=_text(small), fused=True),
        # whole prompts into the cache, odd starts and lengths
        dict(name="write_prompts", op="write", type="fp16", heads=32, kv_heads=8, new="1500,63,1,4096,700",
             len="1500,100,128,4096,1333", fused=False),
        # one new token of one prompt: latency
        dict(name="attend_one", op="attend", type="bf16", heads=32, kv_heads=8, new="1", len="1001", fused=True),
        # one new token for each of 64 prompts of 500 to 8192 tokens: memory
        dict(name="attend_batch", op="attend", type="bf16", heads=32, kv_heads=8, new=_text([1] * 64),
             len=_text(decode), fused=False),
        # one new token over a long cache
        dict(name="attend_long", op="attend", type="bf16", heads=32, kv_heads=8, new="1", len="130001", fused=False),
        # a few new tokens each, 7 query heads on a key/value head, fp16, one sequence with nothing new
        dict(name="attend_few", op="attend", type="fp16", heads=28, kv_heads=4, new="2,1,5,3,0,2,1,4",
             len="2000,1,777,4095,64,65,12001,300", fused=False),
        # chunks of a prompt over what is kept: the tensor cores' rate
        dict(name="attend_chunk", op="attend", type="bf16", heads=32, kv_heads=8, new="512,300,1024",
             len="8192,300,5555", fused=False),
    ]


def draw(rng):
    heads, kv = rng.choice([(32, 8), (32, 8), (16, 16), (28, 4), (8, 2), (24, 8), (16, 1)])
    base = dict(type=rng.choice(["bf16", "bf16", "fp16"]), heads=heads, kv_heads=kv, fused=rng.random() < 0.5)
    op = rng.choice(["packed", "packed", "write", "attend", "attend"])
    n = int(round(math.exp(rng.uniform(0, math.log(48)))))
    if op == "packed":
        q = _spread(rng, n, 1, max(2, 4000 // n))
        if n > 2:
            q[rng.randrange(n)] = 0
        k = [c + rng.choice([0, 0, 1, 64, 500]) for c in q] if rng.random() < 0.4 else []
        return dict(base, op=op, q=_text(q), k=_text(k), pad=rng.choice([0, 5]))
    if op == "write":
        new = _spread(rng, n, 1, max(2, 4000 // n))
        return dict(base, op=op, new=_text(new), len=_text([c + rng.randrange(0, 100) for c in new]))
    if rng.random() < 0.7:  # tokens
        new = [rng.choice([1, 1, 1, 2, 4]) for _ in range(n)]
        old = _spread(rng, n, 1, max(64, 150000 // n))
    else:  # chunks
        new = _spread(rng, n, 1, max(2, 1500 // n))
        old = _spread(rng, n, 1, max(64, 12000 // n))
    return dict(base, op=op, new=_text(new), len=_text([o + c for o, c in zip(old, new)]))


def _starts(counts):
    s = [0]
    for c in counts:
        s.append(s[-1] + c)
    return s


def work(case):
    h, kv = case["heads"], case["kv_heads"]
    if case["op"] == "packed":
        q = _ints(case["q"])
        k = _ints(case["k"]) if case["k"] else q
        pairs = sum(sum(max(0, i + nk - nq + 1) for i in range(nq)) for nq, nk in zip(q, k))
        return {"bytes": 2 * DIM * (2 * h * sum(q) + 2 * kv * sum(k)), "flops": 4 * DIM * h * pairs}
    new, total = _ints(case["new"]), _ints(case["len"])
    rows, cached = sum(new), sum(total)
    pages = sum((t + PAGE - 1) // PAGE for t in total)
    if case["op"] == "write":
        # the new rows in and their codes out, every row of the cache in 8 bits in and in 16 out
        return {"bytes": 2 * kv * DIM * (2 * rows + rows + cached + 2 * cached) + 8 * kv * pages,
                "flops": 2 * kv * DIM * (2 * rows + cached)}
    pairs = sum(sum(t - c + i + 1 for i in range(c)) for c, t in zip(new, total))
    live = sum(t for c, t in zip(new, total) if c)  # a sequence with no new row is not read
    return {"bytes": 2 * kv * DIM * live + 8 * kv * ((live + PAGE - 1) // PAGE) + 2 * 2 * DIM * h * rows,
            "flops": 4 * DIM * h * pairs}


# ------------------------------------------------------------------------------------------------ the inputs


def _scale_exponent(amax):
    """The smallest e >= -126 with amax <= 127 2^e (amax float64, any shape)."""
    _, e = torch.frexp(amax / 127.0)
    e = e.to(torch.float64)
    e = torch.where(amax <= 127.0 * torch.exp2(e - 1.0), e - 1.0, e)
    return torch.clamp(e, min=-126.0)


def _rows(gen, rows, heads, unit):
    """Keys as the encoder makes them (each head's row of unit mean square times the norm's weights), or values
    (heads of different sizes)."""
    x = torch.randn(rows, heads, DIM, generator=gen, device="cuda")
    if unit:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        x = x * (1 + 0.25 * torch.randn(DIM, generator=gen, device="cuda"))
    else:
        x = x * torch.exp(0.7 * torch.randn(heads, 1, generator=gen, device="cuda"))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    t = TYPES[case["type"]]
    h, kv = case["heads"], case["kv_heads"]
    st = dict(case)
    st["scale"] = 1.0 / math.sqrt(DIM)
    if case["op"] == "packed":
        q = _ints(case["q"])
        k = _ints(case["k"]) if case["k"] else q
        st["nq"], st["nk"] = q, k
        rq, rk = sum(q) + case["pad"], sum(k) + case["pad"]
    else:
        st["new"], st["total"] = _ints(case["new"]), _ints(case["len"])
        q, k = st["new"], st["new"]
        rq = rk = sum(q)
    qs, ks, vs = _rows(gen, rq, h, True).to(t), _rows(gen, rk, kv, True).to(t), _rows(gen, rk, kv, False).to(t)
    qs, ks, vs = qs.view(rq, h * DIM), ks.view(rk, kv * DIM), vs.view(rk, kv * DIM)
    if case["fused"] and rq == rk:  # the three as columns of one matrix, as a fused projection leaves them
        both = torch.cat([qs, ks, vs], 1)
        qs, ks, vs = both[:, :h * DIM], both[:, h * DIM:(h + kv) * DIM], both[:, (h + kv) * DIM:]
    st["q"], st["k"], st["v"] = qs, ks, vs
    st["rows_q"], st["rows_k"] = rq, rk
    st["out"] = torch.full((rq, h * DIM), 7.0, device="cuda", dtype=t)  # rows behind the last sequence stay as they are
    st["q_off"] = torch.tensor(_starts(q), dtype=torch.int32, device="cuda")
    st["k_off"] = torch.tensor(_starts(k), dtype=torch.int32, device="cuda")
    if case["op"] != "packed":
        _prepare_cache(st, gen, t)
    if own:
        _prepare_own(st)
    return st


def _prepare_cache(st, gen, t):
    """A pool of pages in random order, the tokens before the call's (for attend, the call's too) written to it."""
    kv, new, total = st["kv_heads"], st["new"], st["total"]
    npages = [(n + PAGE - 1) // PAGE for n in total]
    pool = sum(npages) + 1
    ld = max(npages) + 1
    order = torch.randperm(pool, generator=gen, device="cuda").tolist()
    table = [[-1] * ld for _ in total]
    for s, n in enumerate(npages):
        table[s][:n] = order[sum(npages[:s]):sum(npages[:s + 1])]
    st["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
    st["lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    for name, unit in (("k", True), ("v", False)):
        codes = torch.zeros(pool, kv, PAGE, DIM, dtype=torch.int8, device="cuda")
        scales = torch.full((pool, kv), 2.0 ** -126, dtype=torch.float32, device="cuda")
        for s, (c, n) in enumerate(zip(new, total)):
            have = n - c if st["op"] == "write" else n
            if have == 0:
                continue
            x = _rows(gen, have, kv, unit).to(t).double()
            full = torch.zeros(npages[s] * PAGE, kv, DIM, dtype=torch.float64, device="cuda")
            full[:have] = x
            full = full.view(npages[s], PAGE, kv, DIM).transpose(1, 2)
            e = _scale_exponent(full.abs().amax((2, 3)))
            at = torch.tensor(table[s][:npages[s]], device="cuda")
            codes[at] = torch.round(full / torch.exp2(e)[..., None, None]).to(torch.int8)
            scales[at] = torch.exp2(e).float()
        st[name + "_codes"], st[name + "_scales"] = codes, scales
    if st["op"] == "write":
        st["all_off"] = torch.tensor(_starts(total), dtype=torch.int32, device="cuda")
        st["k_rows"] = torch.zeros(sum(total), kv * DIM, dtype=t, device="cuda")
        st["v_rows"] = torch.zeros(sum(total), kv * DIM, dtype=t, device="cuda")


def _prepare_own(st):
    """The handle, and for a cache its description and the call's workspace."""
    E = _library()
    st["att"] = _attention()
    st["dtype"] = {"bf16": E.GGML_BF16, "fp16": E.GGML_F16}[st["type"]]
    if st["op"] != "packed":
        st["cache"] = E.KvCache(kv_heads=st["kv_heads"], nseq=len(st["new"]), pages=st["k_codes"].shape[0],
                                table_ld=st["table"].shape[1], k=st["k_codes"].data_ptr(), v=st["v_codes"].data_ptr(),
                                k_scale=st["k_scales"].data_ptr(), v_scale=st["v_scales"].data_ptr(),
                                table=st["table"].data_ptr(), lens=st["lens"].data_ptr())
        if st["op"] == "attend":
            n = st["att"].cache_workspace(st["cache"], st["rows_q"], st["heads"])
            st["space"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
            st["space_bytes"] = n


# ------------------------------------------------------------------------------------------------ the passes


def run(st):
    if own:
        return _run_own(st)
    if st["op"] == "packed":
        return _plain_packed(st)
    if st["op"] == "write":
        return _plain_write(st)
    return _plain_attend(st)


def _run_own(st):
    stream = torch.cuda.current_stream().cuda_stream
    att = st["att"]
    if st["op"] == "packed":
        att.packed(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["out"].data_ptr(),
                   st["q_off"].data_ptr(), len(st["nq"]), st["rows_q"], st["heads"], st["kv_heads"], dtype=st["dtype"],
                   ld_q=st["q"].stride(0), ld_k=st["k"].stride(0), ld_v=st["v"].stride(0),
                   kv_offsets=st["k_off"].data_ptr(), kv_rows=st["rows_k"], stream=stream)
        return st["out"]
    if st["op"] == "write":
        att.cache_write(st["cache"], st["k"].data_ptr(), st["v"].data_ptr(), st["q_off"].data_ptr(), st["rows_k"],
                        dtype=st["dtype"], ld_k=st["k"].stride(0), ld_v=st["v"].stride(0), stream=stream)
        att.cache_read(st["cache"], st["k_rows"].data_ptr(), st["v_rows"].data_ptr(), st["all_off"].data_ptr(),
                       st["k_rows"].shape[0], dtype=st["dtype"], stream=stream)
        return st["k_rows"], st["v_rows"], st["k_scales"], st["v_scales"]
    att.cache_attend(st["cache"], st["q"].data_ptr(), st["out"].data_ptr(), st["q_off"].data_ptr(), st["rows_q"],
                     st["heads"], dtype=st["dtype"], ld_q=st["q"].stride(0), workspace=st["space"].data_ptr(),
                     workspace_bytes=st["space_bytes"], stream=stream)
    return st["out"]


def _plain_rows(q, k, v, scale):
    """Causal attention of the last rows q [nq][kv][g][128] over k, v [nk][kv][128], 32 bits: [nq][kv][g][128]."""
    nq, kv, g, _ = q.shape
    nk = k.shape[0]
    out = torch.zeros(nq, kv, g, DIM, device="cuda")
    if nk == 0:
        return out
    kt = k.float().permute(1, 2, 0)[:, None]                     # [kv][1][128][nk]
    vt = v.float().permute(1, 0, 2)[:, None]                     # [kv][1][nk][128]
    step = max(1, (1 << 28) // (kv * g * nk))
    j = torch.arange(nk, device="cuda")
    for a in range(0, nq, step):
        b = min(nq, a + step)
        s = torch.matmul(q[a:b].float().permute(1, 2, 0, 3), kt) * scale  # [kv][g][rows][nk]
        hidden = j > (torch.arange(a, b, device="cuda") + (nk - nq))[:, None]
        s = s.masked_fill(hidden, float("-inf"))
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        p = torch.exp(s - m)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, vt) / torch.where(total == 0, torch.ones_like(total), total)
        out[a:b] = o.permute(2, 0, 1, 3)
    return out


def _plain_packed(st):
    kv, g = st["kv_heads"], st["heads"] // st["kv_heads"]
    qa, ka = 0, 0
    for nq, nk in zip(st["nq"], st["nk"]):
        if nq:
            o = _plain_rows(st["q"][qa:qa + nq].reshape(nq, kv, g, DIM), st["k"][ka:ka + nk].reshape(nk, kv, DIM),
                            st["v"][ka:ka + nk].reshape(nk, kv, DIM), st["scale"])
            st["out"][qa:qa + nq] = o.reshape(nq, kv * g * DIM).to(st["out"].dtype)
        qa, ka = qa + nq, ka + nk
    return st["out"]


def _plain_cached(st, s, name):
    """Sequence s's rows of the cache: [len][kv][128] float32."""
    n = st["total"][s]
    at = st["table"][s, :(n + PAGE - 1) // PAGE].long()
    x = st[name + "_codes"][at].float() * st[name + "_scales"][at][..., None, None]
    return x.transpose(1, 2).reshape(-1, st["kv_heads"], DIM)[:n]


def _positions(st, offsets, rows):
    """For the rows that OFFSETS packs, the last ones of their sequences: position, first position, page."""
    counts = offsets[1:] - offsets[:-1]
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=rows)
    start = (st["lens"] - counts)[seq]
    pos = start + torch.arange(rows, device="cuda") - offsets[seq]
    return pos, start, st["table"][seq, pos // PAGE].long()


def _plain_write(st):
    kv, rows = st["kv_heads"], st["rows_k"]
    pos, start, page = _positions(st, st["q_off"], rows)
    anew = torch.zeros(st["k_codes"].shape[0], dtype=torch.bool, device="cuda")
    anew[page] = pos // PAGE * PAGE >= start
    for name in "kv":
        x = st[name].reshape(rows, kv, DIM).float()
        codes, scales = st[name + "_codes"], st[name + "_scales"]
        amax = torch.zeros_like(scales).scatter_reduce_(0, page[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
        scale = torch.exp2(_scale_exponent(amax.double())).float()
        scale = torch.where(anew[:, None], scale, torch.maximum(scale, scales))
        touched = torch.zeros_like(anew)
        touched[page] = True
        shrink = torch.where(touched[:, None], scales / scale, torch.ones_like(scales))
        scales.copy_(torch.where(touched[:, None], scale, scales))
        old = codes.float() * torch.where(anew[:, None], torch.zeros_like(shrink), shrink)[..., None, None]
        codes.copy_(torch.round(old).to(torch.int8))
        codes[page, :, pos % PAGE] = torch.round(x / scales[page][..., None]).to(torch.int8)
        at, _, pages = _positions(st, st["all_off"], st[name + "_rows"].shape[0])
        back = codes[pages, :, at % PAGE].float() * scales[pages][..., None]
        st[name + "_rows"].copy_(back.reshape(-1, kv * DIM))
    return st["k_rows"], st["v_rows"], st["k_scales"], st["v_scales"]


def _plain_attend(st):
    kv, g = st["kv_heads"], st["heads"] // st["kv_heads"]
    row = 0
    for s, c in enumerate(st["new"]):
        if c:
            o = _plain_rows(st["q"][row:row + c].reshape(c, kv, g, DIM), _plain_cached(st, s, "k"),
                            _plain_cached(st, s, "v"), st["scale"])
            st["out"][row:row + c] = o.reshape(c, kv * g * DIM).to(st["out"].dtype)
        row += c
    return st["out"]


# ------------------------------------------------------------------------------------------------ in 64 bits


def _exact_head(q, k, v):
    """One head: q [n][128], k, v [m][128] float64; row i sees keys 0 .. i + m - n."""
    n, m = q.shape[0], k.shape[0]
    out = torch.zeros(n, DIM, dtype=torch.float64, device=q.device)
    first = max(0, n - m)  # rows before it see no key
    for a in range(first, n, 4096):
        b = min(n, a + 4096)
        last = b + m - n
        logits = (q[a:b] @ k[:last].T) / DIM ** 0.5
        seen = torch.ones(b - a, last, dtype=torch.bool, device=q.device).tril(a + m - n)
        logits = torch.where(seen, logits, torch.full_like(logits, -torch.inf))
        out[a:b] = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True)) @ v[:last]
    return out


def _exact_sequences(st, keys, values, counts):
    g = st["heads"] // st["kv_heads"]
    out = st["out"].double().reshape(st["rows_q"], st["heads"], DIM)
    row = 0
    for s, c in enumerate(counts):
        if c:
            q = st["q"][row:row + c].double().reshape(c, st["heads"], DIM)
            ks, vs = keys(s), values(s)
            for h in range(st["heads"]):
                out[row:row + c, h] = _exact_head(q[:, h], ks[:, h // g], vs[:, h // g])
        row += c
    return out.reshape(st["rows_q"], -1)


def exact(case, seed):
    st = prepare(case, seed)
    kv = st["kv_heads"]
    if case["op"] == "packed":
        at = _starts(st["nk"])

        def part(name):
            return lambda s: st[name][at[s]:at[s + 1]].double().reshape(-1, kv, DIM)

        return _exact_sequences(st, part("k"), part("v"), st["nq"])

    def held(name):
        values = st[name + "_codes"].double() * st[name + "_scales"].double()[:, :, None, None]

        def rows(s):
            pages = [p for p in st["table"][s].tolist() if p >= 0]
            return torch.cat([values[p].permute(1, 0, 2) for p in pages])[:st["total"][s]]

        return rows

    if case["op"] == "attend":
        return _exact_sequences(st, held("k"), held("v"), st["new"])
    # write: page by page on the values the page stands for
    results = []
    for name in "kv":
        codes, scales = st[name + "_codes"].double(), st[name + "_scales"].double()
        x = st[name].double().reshape(-1, kv, DIM)
        rows, row = [], 0
        for s, (c, n) in enumerate(zip(st["new"], st["total"])):
            start = n - c
            got = torch.zeros(n, kv, DIM, dtype=torch.float64, device="cuda")
            for b in range((n + PAGE - 1) // PAGE):
                page = int(st["table"][s, b])
                lo, hi = b * PAGE, min(n, (b + 1) * PAGE)
                first = min(max(start, lo), hi)  # the page's first new position
                old = codes[page, :, :first - lo] * scales[page][:, None, None]
                if first < hi:
                    fresh = x[row + first - start:row + hi - start].permute(1, 0, 2)
                    amax = fresh.abs().amax((1, 2))
                    unit = torch.exp2(torch.ceil(torch.log2(amax / 127.0)).clamp(min=-126.0))
                    unit = torch.where((amax <= 63.5 * unit) & (unit > 2.0 ** -126), unit / 2, unit)  # log2 rounded up
                    if first > lo:
                        unit = torch.maximum(unit, scales[page])
                    unit = unit[:, None, None]
                    old = torch.round(old / unit) * unit
                    got[first:hi] = (torch.round(fresh / unit) * unit).permute(1, 0, 2)
                    scales[page] = unit[:, 0, 0]
                got[lo:first] = old.permute(1, 0, 2)
            rows.append(got)
            row += c
        results.append((torch.cat(rows).reshape(-1, kv * DIM), scales))
    return results[0][0], results[1][0], results[0][1], results[1][1]
