"""The attention operators (include/exn_b200.h, exn_attn_*) on a B200 where inputs are at the ends of their range.
The bounds of what an output may be off stand in test_gpu_attn.py, whose helpers these tests use."""
import math

import pytest

import exn_b200 as E
from test_gpu_attn import (D, GGML, TYPES, Cache, att, check, check_packed, offsets, reference, rows,  # noqa: F401
                           run_packed)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# --------------------------------------------------------------------------- items whose keys blocks share


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("heads,kv_heads,nq,nk", [(32, 8, 64, 800), (8, 2, 64, 900), (16, 16, 200, 1100), (28, 4, 36, 1040)])
def test_a_query_that_is_not_finite_beside_shared_keys(att, t, value, heads, kv_heads, nq, nk):
    """A block's part of the keys may be one that only the item's second tile sees; a query row of the first
    tile that is not finite stays in its own output row, whatever the parts."""
    q, k, v = rows(nq, heads, 1, t), rows(nk, kv_heads, 2, t), rows(nk, kv_heads, 3, t)
    good = run_packed(att, q, k, v, [nq], heads, kv_heads, t, nk=[nk])
    check_packed(good, q, k, v, [nq], heads, kv_heads, t, nk=[nk])
    for row, head in ((0, 0), (nq // 3, heads - 1), (nq - 1, 1)):
        bad = q.clone()
        bad[row, head * D + 7] = value
        out = run_packed(att, bad, k, v, [nq], heads, kv_heads, t, nk=[nk])
        touched = torch.zeros_like(good, dtype=torch.bool)
        touched[row, head * D:(head + 1) * D] = True
        assert torch.equal(out[~touched], good[~touched])
        assert value == value or torch.isnan(out[touched]).all()


# --------------------------------------------------------------------------- offsets that decrease


# offsets that decrease once or again and again, and how many sequences stand before the first decrease; those
# behind it claim rows, pages and work of the ones before
DECREASING = [([0, 640, 10, 700], 1), ([0, 30, 300, 299, 700, 5, 640], 2), ([0] + [64] * 1 + [128, 0, 700] * 20, 2),
              ([0, 640] + [10, 700] * 35, 1), ([8 * i for i in range(81)] + [3, 640] * 110, 80)]


def in_the_middle(n, width, t, value=7.0):
    """N rows with 128 rows of VALUE before and behind them: the whole and the rows."""
    x = torch.full((n + 256, width), value, dtype=TYPES[t], device="cuda")
    return x, x[128:128 + n]


@pytest.mark.parametrize("bad,good", DECREASING)
def test_packed_with_offsets_that_decrease(att, bad, good):
    """The sequences before the first decrease are right, and nothing is written beside the rows."""
    heads, kv_heads, n = 8, 2, 700
    q, k, v = rows(n, heads, 1, "bf16"), rows(n, kv_heads, 2, "bf16"), rows(n, kv_heads, 3, "bf16")
    counts = [b - a for a, b in zip(bad[:good], bad[1:good + 1])]
    end = bad[good]
    want = run_packed(att, q[:end], k[:end], v[:end], counts, heads, kv_heads, "bf16")
    o = torch.tensor(bad, dtype=torch.int32, device="cuda")
    whole, out = in_the_middle(n, heads * D, "bf16")
    att.packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), o.data_ptr(), len(bad) - 1, n, heads, kv_heads)
    with pytest.raises(E.ExnError) as e:
        att.sync()
    assert e.value.code == 1 and "decrease" in str(e.value)
    assert torch.equal(out[:end], want)
    assert (whole[:128] == 7).all() and (whole[-128:] == 7).all() and (out[end:] == 7).all()


@pytest.mark.parametrize("bad,good", DECREASING)
def test_cache_calls_with_offsets_that_decrease(att, bad, good):
    """Write, read and both kinds of attention: as above; the pages that no sequence before the decrease has
    stay as they are."""
    heads, kv_heads, n, nseq = 8, 2, 700, len(bad) - 1
    c = Cache(nseq, 12, kv_heads)
    counts = [b - a for a, b in zip(bad[:good], bad[1:good + 1])]
    end = bad[good]
    # every sequence starts inside a page: 23 positions before the call's
    held = [23] * good + [0] * (nseq - good)
    c.write(att, held, rows(23 * good, kv_heads, 4, "bf16"), rows(23 * good, kv_heads, 5, "bf16"), "bf16")
    lens = [23 + max(b - a, 0) for a, b in zip(bad, bad[1:])]
    c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    before = {x: (c.codes[x].clone(), c.scales[x].clone()) for x in "kv"}
    whole_k, k = in_the_middle(n, kv_heads * D, "bf16", math.nan)
    whole_v, v = in_the_middle(n, kv_heads * D, "bf16", math.nan)
    k.copy_(rows(n, kv_heads, 2, "bf16"))
    v.copy_(rows(n, kv_heads, 3, "bf16"))
    o = torch.tensor(bad, dtype=torch.int32, device="cuda")
    att.cache_write(c.c, k.data_ptr(), v.data_ptr(), o.data_ptr(), n)
    with pytest.raises(E.ExnError):
        att.sync()
    mine = torch.zeros(c.c.pages, dtype=torch.bool, device="cuda")
    for s in range(good):
        for name, x in (("k", k), ("v", v)):
            c._model_write(s, name, x[bad[s]:bad[s + 1]].double().cpu().reshape(-1, kv_heads, D))
        mine[c.table[s, :(lens[s] + 63) // 64].long()] = True
    for x in "kv":
        assert torch.equal(c.codes[x][~mine], before[x][0][~mine]) and torch.equal(c.scales[x][~mine], before[x][1][~mine])
    whole_k, got_k = in_the_middle(n, kv_heads * D, "bf16")
    whole_v, got_v = in_the_middle(n, kv_heads * D, "bf16")
    att.cache_read(c.c, got_k.data_ptr(), got_v.data_ptr(), o.data_ptr(), n)
    with pytest.raises(E.ExnError):
        att.sync()
    for name, whole, got in (("k", whole_k, got_k), ("v", whole_v, got_v)):
        want = c.expect(name, counts + [0] * (nseq - good)).flatten(1)
        assert torch.equal(got[:end].double(), want)
        assert (whole[:128] == 7).all() and (whole[-128:] == 7).all() and (got[end:] == 7).all()
    q = rows(n, heads, 6, "bf16")
    few = torch.tensor(list(range(good + 1)) + [(good + 1) * (i % 2) for i in range(nseq - good)], dtype=torch.int32,
                       device="cuda")
    for off, last in ((o, n), (few, good + 2)):
        at = [x.item() for x in off[:good + 1]]
        whole, out = in_the_middle(last, heads * D, "bf16")
        space = torch.empty(att.cache_workspace(c.c, last, heads), dtype=torch.uint8, device="cuda")
        att.cache_attend(c.c, q.data_ptr(), out.data_ptr(), off.data_ptr(), last, heads, workspace=space.data_ptr(),
                         workspace_bytes=space.numel())
        with pytest.raises(E.ExnError):
            att.sync()
        c.dense = last * (heads // kv_heads) > 64 * (nseq + 1)
        for s in range(good):
            ref = reference(q[at[s]:at[s + 1]], c.model[s]["k"].cuda().flatten(1), c.model[s]["v"].cuda().flatten(1),
                            heads, kv_heads)
            check(out[at[s]:at[s + 1]], ref, "bf16", p16="same" if c.dense else "fp16")
        assert (whole[:128] == 7).all() and (whole[-128:] == 7).all() and (out[at[good]:] == 7).all()


def test_what_a_kernel_on_another_stream_finds_is_reported_once(att):
    """Syncs on one stream while a bad call waits behind slow work on another: one of them, or the sync of
    that stream, reports it, and one only."""
    q, k, v = rows(64, 8, 1, "bf16"), rows(64, 2, 2, "bf16"), rows(64, 2, 3, "bf16")
    out = torch.zeros_like(q)
    bad = torch.tensor([0, 65], dtype=torch.int32, device="cuda")
    slow, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        big = torch.randn(2048, 2048, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(slow):
            for _ in range(3):
                big = big @ big * 1e-3
            att.packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), bad.data_ptr(), 1, 64, 8, 2,
                       stream=slow.cuda_stream)
        reports = 0
        for st in [other] * 30 + [slow, other]:
            try:
                att.sync(st.cuda_stream)
            except E.ExnError as e:
                assert e.code == 1
                reports += 1
        assert reports == 1
