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


# --------------------------------------------------------------------------- pages of values of very different sizes


def pages_of_sizes(t, heads, kv_heads, v_exponents, k_levels, seed, few=0):
    """A cache of one sequence whose page i has values of the size 2^v_exponents[i] and keys whose scores are
    about k_levels[i] (natural logarithms), and rows of q; all numbers small multiples of powers of two, so
    that the cache holds them exactly and the scores' sums are exact.  The last page has FEW positions (0: all)."""
    n = 64 * len(v_exponents) - (64 - few if few else 0)
    g = torch.Generator(device="cuda").manual_seed(seed)
    side = torch.randint(0, 2, (1, 1, D), generator=g, device="cuda") * 2.0 - 1
    q = side.expand(1, heads, D) * torch.tensor([1.0, 0.5, 1.0, 2.0], device="cuda").repeat(heads)[:heads, None]
    page = torch.arange(n, device="cuda") // 64
    # side . k = 128 level: the score is level * 128 / sqrt(128); one more key dim turned over changes it a little
    level = torch.tensor([round(x * 64 / 11.3137) / 64 for x in k_levels], device="cuda")[page]
    turned = torch.rand(n, kv_heads, D, generator=g, device="cuda") < 0.02
    k = level[:, None, None] * side * torch.where(turned, -1.0, 1.0)
    size = torch.exp2(torch.tensor([float(x) for x in v_exponents], device="cuda"))[page]
    v = torch.randint(-96, 97, (n, kv_heads, D), generator=g, device="cuda") * size[:, None, None]
    c = Cache(1, len(v_exponents), kv_heads)
    return c, [x.to(TYPES[t]).reshape(len(x), -1) for x in (q, k, v)]


def check_wide(out, c, q, heads, kv_heads, t, p_step):
    """As check of test_gpu_attn.py, with what the weights' 16 bits drop measured by the row's largest product
    of a weight and a page's scale: each of N positions loses a code of up to 127 times 2^-25 of it."""
    v = c.model[0]["v"].cuda()
    n = v.shape[0]
    o, a, _ = reference(q, c.model[0]["k"].cuda().flatten(1), v.flatten(1), heads, kv_heads)
    scales = torch.tensor([[2.0 ** c.units[0]["v"][j // 64, h] for h in range(kv_heads)] for j in range(n)], device="cuda").double()
    w = reference(q, c.model[0]["k"].cuda().flatten(1), scales[:, :, None].expand(n, kv_heads, D).flatten(1), heads, kv_heads)
    # w[0] is the sum of weights times scales, at least the largest of them
    tol = 2 ** -8 * o.abs() if t == "bf16" else 2 ** -11 * o.abs() + 2.0 ** -25
    tol = tol + (p_step + 2 ** -11.5) * a + n * 127 * 2.0 ** -25 * w[0]
    assert torch.isfinite(out).all()
    worst = ((out.double() - o).abs() / tol).max().item()
    assert worst <= 1, "an output is %.3g of its bound off" % worst


def attend_copies(att, c, q, heads, t, copies):
    """c's attention for COPIES sequences of the same pages, [copies][rows of q]: so many items that a warp
    takes several pages of each."""
    n = q.shape[0]
    table, lens = c.table[:1].repeat(copies, 1), c.lens[:1].repeat(copies)
    one = E.KvCache.from_buffer_copy(c.c)
    one.nseq, one.table, one.lens = copies, table.data_ptr(), lens.data_ptr()
    o = offsets([n] * copies)
    qs = q.repeat(copies, 1)
    out = torch.full_like(qs, 7.0)
    space = torch.empty(att.cache_workspace(one, n * copies, heads), dtype=torch.uint8, device="cuda")
    att.cache_attend(one, qs.data_ptr(), out.data_ptr(), o.data_ptr(), n * copies, heads, dtype=GGML[t],
                     workspace=space.data_ptr(), workspace_bytes=space.numel())
    att.sync()
    assert n * (heads // c.kv) <= 64  # the kernel that reads the codes
    return out.reshape(copies, n, heads * D)


WIDE = [  # sizes of the pages' values and levels of their scores
    ([0, 30], [20, 0]),                  # a weight of 2^-29 on values 2^30 times as large
    ([0] * 9 + [30] * 9, [20] * 9 + [0] * 9),
    ([30] * 9 + [0] * 9, [0] * 9 + [20] * 9),
    ([0, 34, 0, 33] * 5, [23, 0, 22, 1] * 5),
    ([-60] * 7 + [60] * 7, [0] * 14),    # the larger pages are the output, in either order
    ([60] * 7 + [-60] * 7, [0] * 14),
    ([-40, -80, -60, 10, -50, -41] * 4, [30, 60, 45, 0, 38, 31] * 4),
    ([100] * 6 + [-100] * 6 + [0] * 6, [0] * 6 + [80] * 6 + [40] * 6),  # as far apart as bf16 allows
    ([7 * (i % 9) - 30 for i in range(40)], [1.5 * (i % 7) for i in range(40)]),
]


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (8, 2), (16, 1)])
@pytest.mark.parametrize("sizes,levels", WIDE)
@pytest.mark.parametrize("few,copies", [(0, 1), (5, 1), (40, 400)])
def test_attention_over_pages_of_very_different_sizes(att, heads, kv_heads, sizes, levels, few, copies):
    """A small weight on large values counts as much as a large one on small values, whichever page comes
    first, in one warp or in several."""
    c, (q, k, v) = pages_of_sizes("bf16", heads, kv_heads, sizes, levels, 1, few)
    c.write(att, [k.shape[0]], k, v, "bf16")
    out = attend_copies(att, c, q, heads, "bf16", copies)
    check_wide(out[:, 0], c, q, heads, kv_heads, "bf16", 2 ** -11)
    assert torch.equal(out, attend_copies(att, c, q, heads, "bf16", copies))


def test_one_token_and_a_chunk_agree_over_pages_of_different_sizes(att):
    """The same rows by either path of cached attention."""
    heads, kv_heads = 8, 2
    c, (q, k, v) = pages_of_sizes("bf16", heads, kv_heads, [0, 30, 1, 31] * 4, [20, 0, 19, 1] * 4, 2)
    c.write(att, [k.shape[0]], k, v, "bf16")
    one = attend_copies(att, c, q, heads, "bf16", 400)[:, 0]
    many = q.repeat(40, 1)
    chunk = c.attend(att, [40], many, heads, "bf16")
    assert c.dense
    check_wide(one, c, q, heads, kv_heads, "bf16", 2 ** -11)
    check_wide(chunk[-1:], c, q, heads, kv_heads, "bf16", 2 ** -8)


def test_rows_of_a_tile_keep_their_own_unit(att):
    """Rows that share a tile and see different pages: the ones that a page of huge values is hidden from, or
    has no weight for, keep theirs."""
    heads, kv_heads = 4, 1
    c, (q, k, v) = pages_of_sizes("bf16", heads, kv_heads, [-100] * 8 + [20], [0] * 9, 3, few=2)
    # the last two positions have huge values; row 0 sees neither, row 1 the first, row 2 both
    c.write(att, [k.shape[0]], k, v, "bf16")
    for copies in (1, 400):
        out = attend_copies(att, c, q.repeat(3, 1), heads, "bf16", copies)
        check_wide(out[:, 2], c, q, heads, kv_heads, "bf16", 2 ** -11)
        c.lens -= 2
        model, c.model[0]["v"] = c.model[0]["v"], c.model[0]["v"][:-2]
        keys, c.model[0]["k"] = c.model[0]["k"], c.model[0]["k"][:-2]
        check_wide(out[:, 0], c, q, heads, kv_heads, "bf16", 2 ** -11)
        c.lens += 2
        c.model[0] = dict(k=keys, v=model)
    # a head that turns away from the huge pages: scores of -100, weights of 2^-144 times values of 2^120 times as large
    for sizes in ([-100] * 8 + [20] * 8, [20] * 8 + [-100] * 8):
        c, (q, k, v) = pages_of_sizes("bf16", heads, kv_heads, sizes, [25 * (x > 0) for x in sizes], 4)
        c.write(att, [k.shape[0]], k, v, "bf16")
        q[:, D:2 * D] *= -8
        for copies in (1, 400):
            check_wide(attend_copies(att, c, q, heads, "bf16", copies)[:, 0], c, q, heads, kv_heads, "bf16", 2 ** -11)


@pytest.mark.parametrize("t,fraction", [("fp16", 0.5 - 2 ** -12), ("fp16", 0.5 + 2 ** -10), ("bf16", 0.5 - 2 ** -9),
                                        ("fp16", -0.5 + 2 ** -12), ("fp16", 1.5 - 2 ** -10), ("fp16", -63.5 + 2 ** -5)])
def test_small_query_elements_are_rounded_to_nearest(att, t, fraction):
    """Rows of q of 127 equal elements beside one of 127, which no key sees: each of the 127 may be off by 1/512
    (half of 1/256 of the unit 1), which moves a score of equal keys of 8 by 127 * 8 / 512 times the scale and,
    between keys of 8 and of -8, a weight by twice that relatively."""
    c = Cache(1, 3, 1)
    k = torch.full((130, D), 8.0, device="cuda")
    k[::2] *= -1
    k[:, 5] = 0
    v = torch.ones(130, D, dtype=TYPES[t], device="cuda")  # the output is the two kinds' weights' difference
    v[::2] *= -1
    q = torch.full((1, 2 * D), fraction, device="cuda")
    q[0, 5] = 127
    q[0, D + 5] = -127
    q, k = q.to(TYPES[t]), k.to(TYPES[t])
    assert q[0, 0].item() == fraction
    c.write(att, [130], k, v, t)
    scale = 2.0 ** -10 / max(1.0, abs(fraction))  # scores of about -1 .. 1: the weights stay of one size
    out = torch.zeros_like(q)
    o = offsets([1])
    space = torch.empty(att.cache_workspace(c.c, 1, 2), dtype=torch.uint8, device="cuda")
    att.cache_attend(c.c, q.data_ptr(), out.data_ptr(), o.data_ptr(), 1, 2, dtype=GGML[t], scale=scale,
                     workspace=space.data_ptr(), workspace_bytes=space.numel())
    att.sync()
    ref, a, absv = reference(q, c.model[0]["k"].cuda().flatten(1), c.model[0]["v"].cuda().flatten(1), 2, 1, scale)
    u = 2 ** -8 if t == "bf16" else 2 ** -11
    err = max(abs(math.remainder(fraction, 1 / 256)), 2 ** -24)  # what the nearest multiple of 1/256 is off
    assert err <= 1 / 512
    tol = u * ref.abs() + 2.0 ** -25 + (2 ** -11 + 2 ** -11.5 + 2.1 * 127 * 8 * err * scale) * a + 2.0 ** -25 * absv
    worst = ((out.double() - ref).abs() / tol).max().item()
    assert worst <= 1, "an output is %.3g of its bound off" % worst


# --------------------------------------------------------------------------- the largest numbers of a type


@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_the_largest_numbers_stay_finite(att, t):
    """Values up to the type's largest are held off by less than their scale, by at most half of it below 63.5
    times it, and come back finite, by reading and by attention, also after a page's scale has grown to them."""
    biggest = torch.finfo(TYPES[t]).max
    unit = 2.0 ** (10 if t == "fp16" else 122)
    x = torch.zeros(80, D, device="cuda")
    x[:64] = torch.linspace(-1, 1, 64, device="cuda")[:, None] * biggest
    x[64:72] = 0.49 * biggest  # a scale of half of UNIT, then the largest: it grows
    x[72:76, ::2], x[76:] = biggest, -biggest
    x = x.to(TYPES[t])
    c = Cache(1, 2, 1)
    for part in (x[:64], x[64:72], x[72:]):
        c.lens += len(part)
        o = offsets([len(part)])
        att.cache_write(c.c, part.data_ptr(), part.data_ptr(), o.data_ptr(), len(part), dtype=GGML[t])
        att.sync()
    k, v = c.read(att, [80], t)
    assert torch.equal(k, v) and torch.isfinite(k).all()
    for page in (0, 1):
        assert c.scales["k"][c.table[0, page], 0].item() == unit
    off = (k.double() - x.double()).abs()
    assert (off < unit).all() and (off[x.double().abs() <= 63.5 * unit] <= unit / 2).all()
    zero = torch.zeros(1, D, dtype=TYPES[t], device="cuda")  # equal weights for all positions
    c.lens.fill_(1)
    out = c.attend(att, [1], zero, 1, t)
    assert torch.equal(out[0], k[0])
    many = torch.zeros(129, 1 * D, dtype=TYPES[t], device="cuda")
    out = c.attend(att, [129], many, 1, t)
    assert c.dense and torch.equal(out[-1], k[0])


# --------------------------------------------------------------------------- tables with room for very many positions


def test_chunks_over_tables_with_room_for_2_31_positions(att):
    """More positions than one launch turns into 16 bits: the codes are read, with as little workspace."""
    heads, kv_heads, lens, counts = 4, 1, [200, 70], [60, 70]
    c = Cache(2, 4, kv_heads)
    c.write(att, lens, rows(270, kv_heads, 1, "bf16"), rows(270, kv_heads, 2, "bf16"), "bf16")
    few = att.cache_workspace(c.c, 1, heads)
    ld = 2 ** 24 + 1
    table = torch.full((2, ld), -1, dtype=torch.int32, device="cuda")
    table[:, :4] = c.table
    c.c.table, c.c.table_ld = table.data_ptr(), ld
    q = rows(130, heads, 3, "bf16")
    assert att.cache_workspace(c.c, 130, heads) == few
    out = torch.full_like(q, 7.0)
    space = torch.empty(few, dtype=torch.uint8, device="cuda")
    o = offsets(counts)
    att.cache_attend(c.c, q.data_ptr(), out.data_ptr(), o.data_ptr(), 130, heads, workspace=space.data_ptr(),
                     workspace_bytes=few)
    att.sync()
    c.dense = False
    c.check_attend(out, counts, q, heads, "bf16")


def test_work_next_to_2_31(att):
    """As much work as one call may have (2^26 half pages a run of the sequences, 2^31 in all): every sequence
    is the same page again and again, so its rows are those over the page alone.

    A warp adds up a fifth of an item, 2^20 / 5 half pages, in two products each, and the tensor core cuts what
    is behind the last bit of a sum, up to 2^-23 of it, where other units round: 2 * 2^20 / 5 * 2^-23 = 5 % of A
    at most, beside the usual bound."""
    heads = kv_heads = 64
    c = Cache(1, 1, kv_heads)
    c.write(att, [64], rows(64, kv_heads, 1, "bf16"), rows(64, kv_heads, 2, "bf16"), "bf16")
    q = rows(1, heads, 3, "bf16")
    want = c.attend(att, [1], q, heads, "bf16")
    c.check_attend(want, [1], q, heads, "bf16")
    nseq, pages = 32, 2 ** 19 - 7  # 64 items of 2^20 - 14 + 12 a sequence
    table = c.table[0, 0].repeat(nseq, pages)
    lens = torch.full((nseq,), 64 * pages, dtype=torch.int32, device="cuda")
    c.c.nseq, c.c.table_ld, c.c.table, c.c.lens = nseq, pages, table.data_ptr(), lens.data_ptr()
    out = torch.full((nseq, heads * D), 7.0, dtype=torch.bfloat16, device="cuda")
    o = offsets([1] * nseq)
    qs = q.repeat(nseq, 1)
    space = torch.empty(att.cache_workspace(c.c, nseq, heads), dtype=torch.uint8, device="cuda")
    att.cache_attend(c.c, qs.data_ptr(), out.data_ptr(), o.data_ptr(), nseq, heads, workspace=space.data_ptr(),
                     workspace_bytes=space.numel())
    att.sync()
    ref, a, absv = reference(q, c.model[0]["k"].cuda().flatten(1), c.model[0]["v"].cuda().flatten(1), heads, kv_heads)
    tol = 2 ** -8 * ref.abs() + (2 ** -11 + 2 ** -11.5 + 0.05) * a + 2.0 ** -25 * (1 + absv)
    worst = ((out.double() - ref).abs() / tol).max().item()
    assert worst <= 1, "an output is %.3g of its bound off" % worst


# --------------------------------------------------------------------------- what is not finite in a cache or beside one


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("copies,tokens", [(1, 3), (400, 3), (1, 200)])
def test_a_page_of_nan_reaches_the_rows_that_see_it(att, t, name, copies, tokens):
    """A page whose keys or values were given a NaN after the first rows' positions, with a page of other
    sizes before it: rows before its first position are right, the others NaN in its head, right in the next."""
    heads, kv_heads, n = 4, 2, 64 * 6 + 1
    c = Cache(1, 7, kv_heads)
    k, v = rows(n, kv_heads, 1, t), rows(n, kv_heads, 2, t)
    v[:128] *= 2.0 ** -6
    c.write(att, [n], k, v, t)
    page = c.table[0, 6].item()  # of the last position alone
    c.scales[name][page, 0] = math.nan
    q = rows(tokens, heads, 3, t)
    if tokens > 64:
        out = c.attend(att, [tokens], q, heads, t).reshape(1, tokens, -1)
        assert c.dense
    else:
        out = attend_copies(att, c, q, heads, t, copies)
    half = heads // 2 * D
    assert torch.isnan(out[:, -1, :half]).all() and torch.isfinite(out[:, :-1]).all() and torch.isfinite(out[:, -1, half:]).all()
    c.model[0] = {x: y[:-1] for x, y in c.model[0].items()}
    c.scales[name][page, 0] = 1.0
    c.lens.fill_(n - 1)
    ref = reference(q[:-1], c.model[0]["k"].cuda().flatten(1), c.model[0]["v"].cuda().flatten(1), heads, kv_heads)
    for x in out:
        check(x[:-1], ref, t, p16="same" if tokens > 64 else "fp16")


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("tokens", [1, 3, 80])
def test_a_query_that_is_not_finite_over_a_cache(att, value, tokens):
    """It stays in its own output row and head, by either path."""
    heads, kv_heads = 8, 2
    c = Cache(2, 9, kv_heads)
    lens = [500, 130]
    c.write(att, lens, rows(630, kv_heads, 1, "bf16"), rows(630, kv_heads, 2, "bf16"), "bf16")
    q = rows(2 * tokens, heads, 3, "bf16")
    good = c.attend(att, [tokens] * 2, q, heads, "bf16")
    assert c.dense == (tokens == 80)
    for row, head in ((0, 1), (tokens, 6), (2 * tokens - 1, 0)):
        bad = q.clone()
        bad[row, head * D + 9] = value
        out = c.attend(att, [tokens] * 2, bad, heads, "bf16")
        touched = torch.zeros_like(good, dtype=torch.bool)
        touched[row, head * D:(head + 1) * D] = True
        assert torch.equal(out[~touched], good[~touched])
        assert value == value or torch.isnan(out[touched]).all()


def test_rows_without_any_sequence(att):
    """Rows of which the offsets give none away: every call leaves its outputs as they are."""
    c = Cache(3, 2, 2)
    c.write(att, [70, 1, 0], rows(71, 2, 1, "bf16"), rows(71, 2, 2, "bf16"), "bf16")
    before = [c.codes[x].clone() for x in "kv"]
    x = rows(300, 8, 3, "bf16")
    for n in (5, 300):
        out = torch.full((n, 8 * D), 7.0, dtype=torch.bfloat16, device="cuda")
        assert (c.attend(att, [0, 0, 0], x[:n], 8, "bf16", out=out) == 7).all()
        assert (run_packed(att, x[:n], x[:n, :2 * D], x[:n, :2 * D], [0, 0], 8, 2, "bf16", out=out) == 7).all()
        o = offsets([0, 0, 0])
        att.cache_write(c.c, x.data_ptr(), x.data_ptr(), o.data_ptr(), n)
        att.cache_read(c.c, out.data_ptr(), out.data_ptr(), o.data_ptr(), n)
        att.sync()
        assert (out == 7).all() and all(torch.equal(c.codes[y], z) for y, z in zip("kv", before))
