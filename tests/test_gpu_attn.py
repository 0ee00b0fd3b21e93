"""The attention operators (include/exn_b200.h, exn_attn_*) on a B200 against their formulas in 64 bits.

How far an output may be off, with u the type's half step (2^-8 for bf16, 2^-11 for fp16), w the softmax
weights and A = sum_j w_j |v_j| of the same row and dim:
  * the output's own rounding: u |o|;
  * P rounded to 16 bits before the second product: u A at most; in fp16 also 2^-25 for each P below
    2^-14, whose largest is at least 1: 2^-25 sum_j |v_j|;
  * the fp32 arithmetic: a score of 128 products is off by at most 130 2^-24 scale sum |q k|, and scale
    sum |q k| <= scale |q| |k| stays below 31 for the rows below (|q|, |k| <= 18.5), so the weights by
    130 * 31 * 2^-24 = 2^-12 relatively; sums of weights and outputs add less than 2^-16: 2^-11.5 A;
  * an output below the type's normal range: its smallest step.

Where a cache's codes are read directly, the scores' sums are exact integers and q is what is rounded, to two
int8 numbers, q = 2^a (hi + lo / 256) with 127 2^a < 2 M for the row's largest |q| = M: an element from M / 128
(bf16) or M / 16 (fp16) on is exact, a smaller one off by at most 2^-15 M, evenly spread.  M stays below 4.5 for
the rows below (1.6 times that where they are spread), and of 128 normal elements fewer than 60 lie below M / 16,
so with independent errors a score has a deviation of at most 2^-15 4.5 / sqrt(3) sqrt(60) / sqrt(128) = 2^-14.1
and stays below 2^-11.5 at six of them: the fp32 term above covers it, its score part not being needed.
"""
import ctypes
import math

import pytest

import exn_b200 as E

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

D = 128
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GGML = {"bf16": E.GGML_BF16, "fp16": E.GGML_F16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


@pytest.fixture(scope="module")
def att():
    with E.Attention() as a:
        yield a


def rows(n, heads, seed, t, spread=1.0, ld=0):
    """N rows of HEADS heads, a view of row stride LD (0: contiguous)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, heads, D, generator=g, device="cuda")
    x = (spread * x.clamp(-4, 4) / x.square().mean(-1, keepdim=True).sqrt()).reshape(n, heads * D).to(TYPES[t])
    if not ld:
        return x
    wide = torch.full((n, ld), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :heads * D] = x
    return wide[:, :heads * D]


def offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts, dtype=torch.int64).cumsum(0)) if counts else [0],
                        dtype=torch.int32, device="cuda")


def reference(q, k, v, heads, kv_heads, scale=1 / math.sqrt(D)):
    """One sequence in 64 bits: (o, A, sum |v|) as [nq][heads * 128]; q's rows are its last positions."""
    nq, nk, g = q.shape[0], k.shape[0], heads // kv_heads
    q = q.double().reshape(nq, heads, D).transpose(0, 1)
    k = k.double().reshape(nk, kv_heads, D).transpose(0, 1).repeat_interleave(g, 0)
    v = v.double().reshape(nk, kv_heads, D).transpose(0, 1).repeat_interleave(g, 0)
    seen = torch.arange(nk, device="cuda") <= torch.arange(nq, device="cuda")[:, None] + (nk - nq)
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    w = torch.softmax(s, -1).masked_fill(~seen, 0.0)
    w = torch.where(seen.any(-1)[:, None], w, torch.zeros_like(w))
    vis = torch.where(seen, 1.0, 0.0).double()

    def flat(x):
        return x.transpose(0, 1).reshape(nq, heads * D)
    return flat(w @ v), flat(w @ v.abs()), flat((vis @ v.abs()))


def check(out, ref, t, p16="same"):
    """P16: the type of the second product's weights (the rows' own, or fp16)."""
    o, a, absv = ref
    p16 = t if p16 == "same" else p16
    u = HALF_STEP[t]
    tol = u * o.abs() + (HALF_STEP[p16] + 2 ** -11.5) * a + 2.0 ** -25
    if p16 == "fp16":
        tol = tol + 2.0 ** -25 * absv
    err = (out.double() - o).abs()
    assert torch.isfinite(out).all()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1, "an output is %.3g of its bound off (%.3g)" % (worst, err.max().item())


def run_packed(att, q, k, v, nq, heads, kv_heads, t, nk=None, pad=0, out=None, scale=0.0, stream=0):
    if out is None:
        out = torch.full((q.shape[0], heads * D), 7.0, dtype=q.dtype, device="cuda")
    qo = offsets(nq)
    ko = offsets(nk) if nk is not None else None
    att.packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qo.data_ptr(), len(nq), q.shape[0], heads,
               kv_heads, dtype=GGML[t], ld_q=q.stride(0), ld_k=k.stride(0), ld_v=v.stride(0), ld_out=out.stride(0),
               kv_offsets=ko.data_ptr() if ko is not None else None, kv_rows=k.shape[0], scale=scale, stream=stream)
    att.sync(stream)
    return out


def check_packed(out, q, k, v, nq, heads, kv_heads, t, nk=None, scale=1 / math.sqrt(D)):
    nk = nk or nq
    a = b = 0
    for n, m in zip(nq, nk):
        if n:
            check(out[a:a + n], reference(q[a:a + n], k[b:b + m], v[b:b + m], heads, kv_heads, scale), t)
        a, b = a + n, b + m
    assert (out[a:] == 7).all()


# --------------------------------------------------------------------------- packed sequences


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (4, 4), (14, 2), (6, 2), (16, 1), (128, 1)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("nq", [[1], [31, 0, 33], [64, 65, 1, 127], [128, 129], [0, 0, 300, 0]])
def test_packed_matches_formula(att, heads, kv_heads, t, nq):
    """Lengths around the query tiles (128 rows of tokens times heads), the 64-key units and the 128-key
    loads; empty sequences first, last and between; groups that divide 128 and that do not."""
    n = sum(nq)
    q, k, v = rows(n, heads, 1, t), rows(n, kv_heads, 2, t), rows(n, kv_heads, 3, t)
    out = run_packed(att, q, k, v, nq, heads, kv_heads, t)
    check_packed(out, q, k, v, nq, heads, kv_heads, t)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_packed_long_and_ragged(att, t):
    nq = [1500, 3, 700, 64, 1]
    n = sum(nq)
    q, k, v = rows(n, 8, 1, t), rows(n, 2, 2, t), rows(n, 2, 3, t)
    check_packed(run_packed(att, q, k, v, nq, 8, 2, t), q, k, v, nq, 8, 2, t)


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (7, 1), (2, 2)])
@pytest.mark.parametrize("nq,nk", [([1], [400]), ([5, 64, 0, 130], [5, 100, 7, 1000]), ([9, 70, 200], [5, 0, 131]),
                                   ([3, 3], [0, 0])])
def test_packed_with_other_key_rows(att, heads, kv_heads, nq, nk):
    """The queries are the last positions of longer sequences; where there are fewer keys than queries the
    first rows see nothing and are 0."""
    q, k, v = rows(sum(nq), heads, 1, "bf16"), rows(sum(nk), kv_heads, 2, "bf16"), rows(sum(nk), kv_heads, 3, "bf16")
    out = run_packed(att, q, k, v, nq, heads, kv_heads, "bf16", nk=nk)
    check_packed(out, q, k, v, nq, heads, kv_heads, "bf16", nk=nk)


def test_packed_strides_and_rows_behind(att):
    """q, k, v as columns of one matrix, other strides, an output with a stride of its own, and rows behind
    the last sequence, in the tensors (NaN) and the output (kept)."""
    nq, heads, kv_heads = [70, 33], 8, 2
    n = sum(nq) + 6
    both = torch.full((n, 12 * D + 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    for at, h, seed in ((0, 8, 1), (8 * D, 2, 2), (10 * D + 8, 2, 3)):
        both[:sum(nq), at:at + h * D] = rows(sum(nq), h, seed, "bf16")
    q, k, v = both[:, :8 * D], both[:, 8 * D:10 * D], both[:, 10 * D + 8:12 * D + 8]
    wide = torch.full((n, 8 * D + 40), 7.0, dtype=torch.bfloat16, device="cuda")
    out = run_packed(att, q, k, v, nq, heads, kv_heads, "bf16", out=wide[:, :8 * D])
    check_packed(out, q, k, v, nq, heads, kv_heads, "bf16")
    assert (wide[:, 8 * D:] == 7).all()


def test_packed_scale(att):
    nq = [90]
    q, k, v = rows(90, 4, 1, "bf16"), rows(90, 2, 2, "bf16"), rows(90, 2, 3, "bf16")
    out = run_packed(att, q, k, v, nq, 4, 2, "bf16", scale=0.03)
    check_packed(out, q, k, v, nq, 4, 2, "bf16", scale=0.03)


def test_packed_peaked_scores(att):
    """Scores far apart: a row's running maximum grows past the rescaling threshold again and again, and
    the weights of all but a few keys are 0."""
    n = 700
    q, k, v = rows(n, 4, 1, "bf16", spread=1.6), rows(n, 1, 2, "bf16"), rows(n, 1, 3, "bf16")
    k = (k * torch.linspace(0.02, 1.1, n, device="cuda")[:, None]).to(torch.bfloat16)
    check_packed(run_packed(att, q, k, v, [n], 4, 1, "bf16"), q, k, v, [n], 4, 1, "bf16")


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("at", [52, 127])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_packed_not_finite_rows_reach_only_those_who_see_them(att, t, at, value):
    """A value or key row that is not finite, within a unit of the sequence before (52) or among later
    tokens of the same one (127): the rows that do not see it are right, the rows that see a bad value
    are not finite in its dim, and only there."""
    nq, heads, kv_heads = [50, 200, 40], 8, 2
    q, k, v = rows(290, heads, 1, t), rows(290, kv_heads, 2, t), rows(290, kv_heads, 3, t)
    good = run_packed(att, q, k, v, nq, heads, kv_heads, t)
    sees = torch.zeros(290, dtype=torch.bool, device="cuda")
    sees[at:250] = True
    bad_v = v.clone()
    bad_v[at, 5] = value  # head 0, dim 5
    out = run_packed(att, q, k, bad_v, nq, heads, kv_heads, t)
    check(out[:50], reference(q[:50], k[:50], v[:50], heads, kv_heads), t)
    ref = reference(q[50:250], k[50:250], v[50:250], heads, kv_heads)
    check(out[50:at], tuple(x[:at - 50] for x in ref), t)
    touched = torch.zeros(290, heads * D, dtype=torch.bool, device="cuda")
    for h in range(heads // kv_heads):
        touched[at:250, h * D + 5] = True
    assert not torch.isfinite(out[touched]).any()
    rest = sees[:, None] & ~touched
    assert torch.equal(out[rest], good[rest]) and torch.equal(out[250:], good[250:])
    assert torch.equal(out[:, 4 * D:], good[:, 4 * D:])
    bad_k = k.clone()
    bad_k[at, 5] = value
    out = run_packed(att, q, bad_k, v, nq, heads, kv_heads, t)
    assert torch.equal(out[~sees], good[~sees]) and torch.equal(out[:, 4 * D:], good[:, 4 * D:])
    if value != value:
        assert torch.isnan(out[sees][:, :4 * D]).all()


def test_packed_deterministic_and_independent_of_the_packing(att):
    """A sequence's rows have the same bits alone and among others, call after call."""
    nq, heads, kv_heads = [37, 150, 260], 8, 2
    q, k, v = rows(447, heads, 1, "bf16"), rows(447, kv_heads, 2, "bf16"), rows(447, kv_heads, 3, "bf16")
    a = run_packed(att, q, k, v, nq, heads, kv_heads, "bf16")
    assert torch.equal(a, run_packed(att, q, k, v, nq, heads, kv_heads, "bf16"))
    b = run_packed(att, q[37:187], k[37:187], v[37:187], [150], heads, kv_heads, "bf16")
    assert torch.equal(a[37:187], b)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (28, 4), (5, 1), (16, 16)])
@pytest.mark.parametrize("nq,nk", [([64], [5000]), ([1], [1024]), ([70, 3, 40], [4200, 0, 1500]), ([129, 0], [2049, 63]),
                                   ([300, 77], [4100, 900]), ([20, 290, 1, 33], [1500, 300, 9, 2500]),
                                   ([200] * 4, [5000, 1030, 600, 1])])
def test_packed_few_rows_over_long_keys(att, heads, kv_heads, t, nq, nk):
    """Few work items of long sequences, whose keys several blocks share: from a share of one load to many,
    a last share that only the item's later rows see, a sequence without keys beside long ones; more items
    than clusters, of which the long ones are shared."""
    q, k, v = rows(sum(nq), heads, 1, t), rows(sum(nk), kv_heads, 2, t), rows(sum(nk), kv_heads, 3, t)
    out = run_packed(att, q, k, v, nq, heads, kv_heads, t, nk=nk)
    check_packed(out, q, k, v, nq, heads, kv_heads, t, nk=nk)
    assert torch.equal(out, run_packed(att, q, k, v, nq, heads, kv_heads, t, nk=nk))


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_packed_shared_keys_that_are_not_finite(att, t, value):
    """As above for a value row that is not finite among the last tokens of a long sequence, and for a key
    row in the middle: rows that do not see the value row keep their bits, those that do are not finite in
    its dim; a key row that is NaN reaches every row of its heads."""
    nq, nk, heads, kv_heads = [70, 40], [2050, 1500], 8, 2
    q, k, v = rows(110, heads, 1, t), rows(3550, kv_heads, 2, t), rows(3550, kv_heads, 3, t)
    good = run_packed(att, q, k, v, nq, heads, kv_heads, t, nk=nk)
    bad = v.clone()
    bad[2050 - 20, 5] = value  # row 50's own token
    out = run_packed(att, q, k, bad, nq, heads, kv_heads, t, nk=nk)
    check(out[:50], tuple(x[:50] for x in reference(q[:70], k[:2050], v[:2050], heads, kv_heads)), t)
    dims = torch.zeros(heads * D, dtype=torch.bool, device="cuda")
    dims[torch.arange(4, device="cuda") * D + 5] = True
    assert not torch.isfinite(out[50:70][:, dims]).any()
    assert torch.equal(out[50:70][:, ~dims], good[50:70][:, ~dims]) and torch.equal(out[70:], good[70:])
    bad = k.clone()
    bad[700, 5] = value
    out = run_packed(att, q, bad, v, nq, heads, kv_heads, t, nk=nk)
    assert torch.equal(out[:, 4 * D:], good[:, 4 * D:]) and torch.equal(out[70:], good[70:])
    if value != value:
        assert torch.isnan(out[:70, :4 * D]).all()


@pytest.mark.parametrize("nseq", [33, 70, 1100])
def test_packed_many_sequences(att, nseq):
    """More sequences than a warp has lanes, empty ones among them, with rows of their own and as the last
    rows of longer ones."""
    heads, kv_heads = 4, 2
    nq = [(7 * i) % 11 * (i % 3 > 0) + (40 if i % 29 == 0 else 0) for i in range(nseq)]
    for nk in (nq, [n + i % 5 for i, n in enumerate(nq)]):
        q, k, v = rows(sum(nq), heads, 1, "bf16"), rows(sum(nk), kv_heads, 2, "bf16"), rows(sum(nk), kv_heads, 3, "bf16")
        out = run_packed(att, q, k, v, nq, heads, kv_heads, "bf16", nk=nk)
        check_packed(out, q, k, v, nq, heads, kv_heads, "bf16", nk=nk)


def test_packed_captured_with_shared_items(att):
    """Calls whose blocks share items, captured one after another and replayed with other inputs."""
    heads, kv_heads = 8, 2
    sets = []
    for nq, nk in (([64], [5000]), ([30, 70], [1100, 3000]), ([300, 77, 20, 5], [4100, 900, 1500, 200])):
        q, k, v = rows(sum(nq), heads, 1, "bf16"), rows(sum(nk), kv_heads, 2, "bf16"), rows(sum(nk), kv_heads, 3, "bf16")
        sets.append((nq, nk, q, k, v, torch.empty_like(q), offsets(nq), offsets(nk)))
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        st = torch.cuda.current_stream().cuda_stream
        for nq, nk, q, k, v, out, qo, ko in sets:
            att.packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), qo.data_ptr(), len(nq), sum(nq), heads,
                       kv_heads, kv_offsets=ko.data_ptr(), kv_rows=sum(nk), stream=st)
    for seed in (5, 6):
        for nq, nk, q, k, v, _, _, _ in sets:
            q.copy_(rows(sum(nq), heads, seed, "bf16"))
            v.copy_(rows(sum(nk), kv_heads, seed + 10, "bf16"))
        g.replay()
        g.replay()
        torch.cuda.synchronize()
        att.sync()
        for nq, nk, q, k, v, out, _, _ in sets:
            check_packed(out, q, k, v, nq, heads, kv_heads, "bf16", nk=nk)


def test_packed_past_32_bits(att):
    """Thousands of sequences whose rows reach past 2^31 elements: those around the border and the last."""
    heads, kv_heads, each, nseq = 32, 8, 61, 8700
    n = each * nseq
    assert n * heads * D > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.empty(n, heads * D, dtype=torch.bfloat16, device="cuda")
    q[-40 * each:] = rows(40 * each, heads, 1, "bf16")
    border = 2 ** 31 // (heads * D) // each * each
    q[:border - each].fill_(0.5)
    q[border - each:border + 2 * each] = rows(3 * each, heads, 2, "bf16")
    q[border + 2 * each:-40 * each].fill_(0.5)
    k = torch.randn(n, kv_heads * D, generator=g, device="cuda", dtype=torch.bfloat16).clamp_(-1.4, 1.4)
    v = torch.randn(n, kv_heads * D, generator=g, device="cuda", dtype=torch.bfloat16)
    out = run_packed(att, q, k, v, [each] * nseq, heads, kv_heads, "bf16")
    for a in (0, border - each, border, border + each, n - 3 * each, n - each):
        check(out[a:a + each], reference(q[a:a + each], k[a:a + each], v[a:a + each], heads, kv_heads), "bf16")


# --------------------------------------------------------------------------- the cache


class Cache:
    """A pool of pages in a shuffled order with a description, and a model of it in 64 bits."""

    def __init__(self, nseq, pages_each, kv_heads, seed=0):
        n = nseq * pages_each + 2
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.kv = kv_heads
        self.codes = {x: torch.randint(-127, 128, (n, kv_heads, 64, D), generator=g, dtype=torch.int8, device="cuda")
                      for x in "kv"}
        self.scales = {x: torch.full((n, kv_heads), 2.0 ** 40, device="cuda") for x in "kv"}  # of a former use
        self.table = torch.randperm(n, generator=g, device="cuda")[:nseq * pages_each].int().reshape(nseq, pages_each)
        self.lens = torch.zeros(nseq, dtype=torch.int32, device="cuda")
        self.c = E.KvCache(kv_heads=kv_heads, nseq=nseq, pages=n, table_ld=pages_each, k=self.codes["k"].data_ptr(),
                           v=self.codes["v"].data_ptr(), k_scale=self.scales["k"].data_ptr(),
                           v_scale=self.scales["v"].data_ptr(), table=self.table.data_ptr(), lens=self.lens.data_ptr())
        self.model = [dict(k=torch.zeros(0, kv_heads, D, dtype=torch.float64), v=torch.zeros(0, kv_heads, D, dtype=torch.float64))
                      for _ in range(nseq)]
        self.units = [dict(k={}, v={}) for _ in range(nseq)]

    def write(self, att, counts, k, v, t):
        self.lens += torch.tensor(counts, dtype=torch.int32, device="cuda")
        o = offsets(counts)
        att.cache_write(self.c, k.data_ptr(), v.data_ptr(), o.data_ptr(), k.shape[0], dtype=GGML[t], ld_k=k.stride(0),
                        ld_v=v.stride(0))
        att.sync()
        at = 0
        for s, c in enumerate(counts):
            for name, x in (("k", k), ("v", v)):
                self._model_write(s, name, x[at:at + c].double().cpu().reshape(c, self.kv, D))
            at += c

    def _model_write(self, s, name, x):
        held = self.model[s][name]
        start, end = held.shape[0], held.shape[0] + x.shape[0]
        held = torch.cat([held, x])
        for b in range(start // 64, (end + 63) // 64 if len(x) else 0):
            lo, hi = max(start, 64 * b), min(end, 64 * b + 64)
            for h in range(self.kv):
                amax = held[lo:hi, h].abs().max().item()
                e = -126
                while amax > 127 * 2.0 ** e:
                    e += 1
                if lo > 64 * b:
                    e = max(e, self.units[s][name][b, h])
                self.units[s][name][b, h] = e
                top = 63 if e == 122 else 127  # 64 * 2^122 is no bf16 number
                held[64 * b:hi, h] = torch.round(held[64 * b:hi, h] / 2.0 ** e).clamp(-top, top) * 2.0 ** e
        self.model[s][name] = held

    def read(self, att, counts, t, ld=0):
        n = sum(counts)
        o = offsets(counts)
        k = torch.full((n + 2, (ld or self.kv * D)), 7.0, dtype=TYPES[t], device="cuda")
        v = k.clone()
        att.cache_read(self.c, k.data_ptr(), v.data_ptr(), o.data_ptr(), n + 2, dtype=GGML[t], ld_k=ld, ld_v=ld)
        att.sync()
        assert (k[n:] == 7).all() and (v[n:] == 7).all() and (k[:, self.kv * D:] == 7).all()
        return k[:n, :self.kv * D], v[:n, :self.kv * D]

    def expect(self, name, counts):
        return torch.cat([self.model[s][name][self.model[s][name].shape[0] - c:] for s, c in enumerate(counts)]).cuda()

    def attend(self, att, counts, q, heads, t, stream=0, out=None, workspace=None):
        o = offsets(counts)
        if out is None:
            out = torch.full((q.shape[0], heads * D), 7.0, dtype=q.dtype, device="cuda")
        n = att.cache_workspace(self.c, q.shape[0], heads)
        w = torch.full((max(n, 256),), 0xff, dtype=torch.uint8, device="cuda")  # NaN in every type
        att.cache_attend(self.c, q.data_ptr(), out.data_ptr(), o.data_ptr(), q.shape[0], heads, dtype=GGML[t],
                         ld_q=q.stride(0), ld_out=out.stride(0), workspace=w.data_ptr(), workspace_bytes=n, stream=stream)
        att.sync(stream)
        self.dense = q.shape[0] * (heads // self.kv) > 64 * (self.c.nseq + 1)  # keys and values in 16 bits
        assert n >= att.cache_workspace(self.c, 1, heads)
        assert not self.dense or n >= self.c.nseq * self.c.table_ld * 64 * self.kv * D * 2 * 2
        return out

    def check_attend(self, out, counts, q, heads, t):
        a = 0
        for s, c in enumerate(counts):
            if c:
                ref = reference(q[a:a + c], self.model[s]["k"].cuda().flatten(1), self.model[s]["v"].cuda().flatten(1),
                                heads, self.kv)
                # P is fp16 in the kernel that reads the codes, the rows' type in the one that reads 16 bits
                check(out[a:a + c], ref, t, p16="same" if self.dense else "fp16")
            a += c
        assert (out[a:] == 7).all()


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("steps", [[[1, 64, 200]], [[63, 0, 5], [1, 1, 70], [2, 130, 64], [0, 64, 1]],
                                   [[1, 1, 1]] * 4])
def test_cache_write_and_read_exactly(att, t, steps):
    """Whole prompts, continued pages (with growing values, so that pages change their scale), odd starts
    and ends: what the cache stands for is the definition's value to the bit, in codes and scales."""
    c = Cache(3, 8, 2, seed=5)
    for i, counts in enumerate(steps):
        n = sum(counts)
        k, v = rows(n, 2, 10 + i, t, spread=1.5 ** i, ld=264), rows(n, 2, 20 + i, t, spread=0.01 * 3 ** i)
        c.write(att, counts, k, v, t)
    total = [m["k"].shape[0] for m in c.model]
    for counts in (total, [min(3, n) for n in total]):
        k, v = c.read(att, counts, "bf16")
        assert torch.equal(k.double().reshape(-1, 2, D), c.expect("k", counts))
        assert torch.equal(v.double().reshape(-1, 2, D), c.expect("v", counts))
    k, _ = c.read(att, total, "fp16", ld=272)
    assert torch.equal(k.reshape(-1, 2, D), c.expect("k", total).half())
    for s in range(3):
        for name in "kv":
            for (b, h), e in c.units[s][name].items():
                assert c.scales[name][c.table[s, b], h].item() == 2.0 ** e


def test_cache_write_extremes(att):
    """Zeros, the largest and the smallest numbers of bf16, 127 times a power of two, and a tie."""
    c = Cache(1, 2, 1)
    x = torch.zeros(70, D, dtype=torch.bfloat16, device="cuda")
    c.write(att, [1], x[:1], x[:1], "bf16")
    assert c.scales["k"][c.table[0, 0], 0].item() == 2.0 ** -126
    x[1, 0], x[1, 1], x[1, 2] = 127 * 2.0 ** -3, 0.5 * 2.0 ** -3, 1.5 * 2.0 ** -3
    c.write(att, [1], x[1:2], x[1:2], "bf16")
    assert c.scales["k"][c.table[0, 0], 0].item() == 2.0 ** -3
    x[2, 0], x[2, 3] = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    c.write(att, [68], x[2:], x[2:], "bf16")
    k, v = c.read(att, [70], "bf16")
    assert torch.equal(k.double().reshape(-1, 1, D), c.expect("k", [70])) and torch.equal(k, v)
    assert c.scales["k"][c.table[0, 1], 0].item() == 2.0 ** -126


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_cache_page_with_a_value_that_is_not_finite(att, value):
    """Its page reads as NaN, also after more tokens, the pages and heads beside it as before; the page is
    whole again when its first position is written anew."""
    c = Cache(1, 3, 2)
    k, v = rows(130, 2, 1, "bf16"), rows(130, 2, 2, "bf16")
    k[70, 3] = value
    c.write(att, [71], k[:71], v[:71], "bf16")
    c.write(att, [59], k[71:], v[71:], "bf16")
    a, b = c.read(att, [130], "bf16")
    assert torch.isnan(a[64:128, :D]).all() and torch.isfinite(a[:64]).all() and torch.isfinite(a[128:]).all()
    assert torch.isfinite(a[:, D:]).all() and torch.isfinite(b).all()
    q = rows(130, 4, 3, "bf16")
    out = torch.full((3, 4 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    c.lens.fill_(66)  # positions 63, 64, 65: the first does not see the page
    c.attend(att, [3], q[:3], 4, "bf16", out=out)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1:, :2 * D]).all() and torch.isfinite(out[1:, 2 * D:]).all()
    c.lens.fill_(64)
    c.model[0] = {n: x[:64] for n, x in c.model[0].items()}
    k = rows(66, 2, 7, "bf16")
    c.write(att, [66], k, k, "bf16")
    a, _ = c.read(att, [66], "bf16")
    assert torch.equal(a.double().reshape(-1, 2, D), c.expect("k", [66]))


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (4, 4), (14, 2), (16, 1), (40, 1), (6, 2)])
@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,counts", [([1], [1]), ([64, 65, 1000], [1, 1, 1]), ([3, 700, 9, 130], [2, 0, 4, 1]),
                                         ([200, 20], [16, 3])])
def test_cache_attend_matches_formula(att, heads, kv_heads, t, lens, counts):
    """Single tokens and a few, lengths of one token, of whole pages and one more, groups of 1 to 40 query
    heads, a sequence with nothing new."""
    c = Cache(len(lens), 17, kv_heads)
    c.write(att, lens, rows(sum(lens), kv_heads, 1, t), rows(sum(lens), kv_heads, 2, t, spread=0.3), t)
    q = rows(sum(counts) + 1, heads, 3, t)
    out = c.attend(att, counts, q, heads, t)
    c.check_attend(out, counts, q, heads, t)


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (7, 1)])
def test_cache_attend_long(att, heads, kv_heads):
    """Sequences of many pages, split over the warps and CTAs of a cluster (more than 32 pages a warp)."""
    lens, counts = [33000, 4097, 130], [1, 2, 1]
    c = Cache(3, 520, kv_heads)
    for part in ([30000, 4000, 100], [3000, 97, 30]):
        n = sum(part)
        c.write(att, part, rows(n, kv_heads, n, "bf16"), rows(n, kv_heads, n + 1, "bf16"), "bf16")
    q = rows(4, heads, 3, "bf16")
    out = c.attend(att, counts, q, heads, "bf16")
    c.check_attend(out, counts, q, heads, "bf16")
    assert torch.equal(out, c.attend(att, counts, q, heads, "bf16"))


@pytest.mark.parametrize("heads,tokens", [(4, 1), (8, 2)])
def test_cache_attend_one_item_in_hundreds_of_parts(att, heads, tokens):
    """One key/value head and one long sequence: every CTA of the device has a part of the same item."""
    c = Cache(1, 800, 1)
    for i in range(2):
        c.write(att, [25500], rows(25500, 1, 2 * i, "bf16"), rows(25500, 1, 2 * i + 1, "bf16"), "bf16")
    q = rows(tokens, heads, 3, "bf16")
    for _ in range(3):
        out = c.attend(att, [tokens], q, heads, "bf16")
        c.check_attend(out, [tokens], q, heads, "bf16")


@pytest.mark.parametrize("t", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,counts", [([200, 64, 500], [100, 64, 1]), ([129, 300], [129, 0])])
def test_cache_attend_chunks(att, t, lens, counts):
    """Many new rows a sequence (the tensor-core tiles over the cache in 16 bits)."""
    c = Cache(len(lens), 9, 2)
    c.write(att, lens, rows(sum(lens), 2, 1, t), rows(sum(lens), 2, 2, t), t)
    q = rows(sum(counts) + 1, 8, 3, t)
    out = c.attend(att, counts, q, 8, t)
    assert c.dense
    c.check_attend(out, counts, q, 8, t)


def test_cache_attend_query_ranges(att):
    """bf16 rows of q far above and below fp16's range, and rows of zeros."""
    c = Cache(1, 2, 1)
    c.write(att, [70], rows(70, 1, 1, "bf16"), rows(70, 1, 2, "bf16"), "bf16")
    q = rows(1, 8, 3, "bf16").reshape(8, D)
    q[0] *= 2.0 ** -100
    q[1] = 0
    q[2] *= 2.0 ** -20
    k, v = c.model[0]["k"][:, 0].cuda(), c.model[0]["v"][:, 0].cuda()
    q[3] = 0
    q[3, 0] = 1e6 * (1 if k[5, 0] > 0 else -1)  # the largest key values of dim 0 take all the weight
    q = q.reshape(1, 8 * D)
    out = c.attend(att, [1], q, 8, "bf16")
    ref = reference(q, k, v, 8, 1)
    sel = torch.cat([torch.arange(h * D, h * D + D) for h in range(8) if h != 3]).cuda()
    check(out[:, sel], tuple(x[:, sel] for x in ref), "bf16", p16="fp16")
    # row 3's scores are single products, its weights equal among the ties: the output's rounding is all
    assert (out.double() - ref[0])[0, 3 * D:4 * D].abs().max() <= 2 ** -7 * v.abs().max()


# --------------------------------------------------------------------------- together, graphs, streams


def test_prompts_then_tokens(att):
    """As a program uses them: prompts packed through attention and into the cache, then single tokens over
    the cache, against the formula on what the cache stands for."""
    heads, kv_heads, nq = 8, 2, [100, 63, 1]
    c = Cache(3, 4, kv_heads)
    n = sum(nq)
    q, k, v = rows(n, heads, 1, "bf16"), rows(n, kv_heads, 2, "bf16"), rows(n, kv_heads, 3, "bf16")
    check_packed(run_packed(att, q, k, v, nq, heads, kv_heads, "bf16"), q, k, v, nq, heads, kv_heads, "bf16")
    c.write(att, nq, k, v, "bf16")
    for step in range(3):
        q, k, v = rows(3, heads, 4 + step, "bf16"), rows(3, kv_heads, 14 + step, "bf16"), rows(3, kv_heads, 24 + step, "bf16")
        c.write(att, [1, 1, 1], k, v, "bf16")
        out = c.attend(att, [1, 1, 1], q, heads, "bf16")
        c.check_attend(out, [1, 1, 1], q, heads, "bf16")


@pytest.mark.parametrize("chunk", [1, 40])
def test_captured_steps_follow_lengths_on_the_device(att, chunk):
    """Write and attention captured once, replayed as the sequences grow: lengths and tokens are read from
    the device; a second graph with its own workspace, replayed between, changes nothing."""
    heads, kv_heads = 8, 2
    two = []
    for seed in (0, 1):
        c = Cache(2, 8, kv_heads, seed=seed)
        k, v = rows(130, kv_heads, seed + 1, "bf16"), rows(130, kv_heads, seed + 2, "bf16")
        c.write(att, [100, 30], k, v, "bf16")
        q, k, v = (rows(2 * chunk, h, seed + 3, "bf16") for h in (heads, kv_heads, kv_heads))
        o = offsets([chunk, chunk])
        out = torch.zeros(2 * chunk, heads * D, dtype=torch.bfloat16, device="cuda")
        n = att.cache_workspace(c.c, 2 * chunk, heads)
        w = torch.empty(max(n, 256), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            st = torch.cuda.current_stream().cuda_stream
            att.cache_write(c.c, k.data_ptr(), v.data_ptr(), o.data_ptr(), 2 * chunk, stream=st)
            att.cache_attend(c.c, q.data_ptr(), out.data_ptr(), o.data_ptr(), 2 * chunk, heads, workspace=w.data_ptr(),
                             workspace_bytes=n, stream=st)
        two.append((c, q, k, v, out, g, w, o))
    for step in range(3):
        for c, q, k, v, out, g, _, _ in two:
            k.copy_(rows(2 * chunk, kv_heads, 50 + step, "bf16"))
            v.copy_(rows(2 * chunk, kv_heads, 60 + step, "bf16"))
            c.lens += chunk
            g.replay()
        torch.cuda.synchronize()
        att.sync()
        for c, q, k, v, out, g, _, _ in two:
            for s in range(2):
                for name, x in (("k", k), ("v", v)):
                    c._model_write(s, name, x[s * chunk:(s + 1) * chunk].double().cpu().reshape(chunk, kv_heads, D))
            c.dense = chunk > 1
            c.check_attend(out, [chunk, chunk], q, heads, "bf16")


def test_calls_on_other_streams_and_after_slow_work(att):
    """Each call is ordered on its own stream: inputs made there by earlier work are waited for."""
    nq = [300]
    q, k, v = rows(300, 8, 1, "bf16"), rows(300, 2, 2, "bf16"), rows(300, 2, 3, "bf16")
    want = run_packed(att, q, k, v, nq, 8, 2, "bf16")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    o = offsets(nq)
    torch.cuda.synchronize()
    for s in (s1, s2):
        with torch.cuda.stream(s):
            late = torch.zeros_like(q)
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = big @ big * 1e-3
            late.copy_(q)
            out = torch.empty_like(q)
            att.packed(late.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), o.data_ptr(), 1, 300, 8, 2,
                       stream=s.cuda_stream)
            outs.append((out, late, big))
    for s, (out, _, _) in zip((s1, s2), outs):
        att.sync(s.cuda_stream)
        assert torch.equal(out, want)


@pytest.mark.parametrize("tokens", [1, 3, 40])
def test_attention_over_a_cache_twice_at_once(att, tokens):
    """The same call on two streams that wait for the same slow work, with a workspace each: both have the
    bits of a call alone; afterwards one workspace serves calls of other sizes and the first again."""
    heads, kv_heads, lens = 8, 2, [3000, 70, 900]
    c = Cache(3, 47, kv_heads)
    k, v = rows(sum(lens), kv_heads, 1, "bf16"), rows(sum(lens), kv_heads, 2, "bf16")
    c.write(att, lens, k, v, "bf16")
    q = rows(3 * tokens, heads, 3, "bf16")
    want = c.attend(att, [tokens] * 3, q, heads, "bf16")
    c.check_attend(want, [tokens] * 3, q, heads, "bf16")
    n = att.cache_workspace(c.c, 3 * tokens, heads)
    o, one = offsets([tokens] * 3), offsets([1, 1, 1])
    n1 = att.cache_workspace(c.c, 3, heads)
    spaces = [torch.zeros(max(n, n1), dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(4):
        big = big @ big * 1e-3
    ready = torch.cuda.Event()
    ready.record()
    for st, w, out in zip(streams, spaces, outs):
        st.wait_event(ready)
        for _ in range(5):
            att.cache_attend(c.c, q.data_ptr(), out.data_ptr(), o.data_ptr(), 3 * tokens, heads, workspace=w.data_ptr(),
                             workspace_bytes=n, stream=st.cuda_stream)
    for st, out in zip(streams, outs):
        att.sync(st.cuda_stream)
        assert torch.equal(out, want)
    small = torch.zeros(3, heads * D, dtype=torch.bfloat16, device="cuda")
    st = streams[0].cuda_stream
    att.cache_attend(c.c, q.data_ptr(), small.data_ptr(), one.data_ptr(), 3, heads, workspace=spaces[0].data_ptr(),
                     workspace_bytes=n1, stream=st)
    outs[0].zero_()
    torch.cuda.synchronize()
    att.cache_attend(c.c, q.data_ptr(), outs[0].data_ptr(), o.data_ptr(), 3 * tokens, heads, workspace=spaces[0].data_ptr(),
                     workspace_bytes=n, stream=st)
    att.sync(st)
    assert torch.equal(outs[0], want)
    c.dense = False
    c.check_attend(small, [1, 1, 1], q[:3], heads, "bf16")


@pytest.mark.parametrize("nseq", [70, 300])
def test_cache_of_many_sequences(att, nseq):
    """More sequences than lanes, and than a block's threads: written, read and attended, some with nothing
    new, some without any position."""
    heads, kv_heads = 4, 2
    c = Cache(nseq, 2, kv_heads)
    lens = [(13 * i) % 127 * (i % 7 > 0) for i in range(nseq)]
    k, v = rows(sum(lens), kv_heads, 1, "bf16"), rows(sum(lens), kv_heads, 2, "bf16")
    c.write(att, lens, k, v, "bf16")
    new = [i % 2 for i in range(nseq)]
    k, v, q = rows(sum(new), kv_heads, 3, "bf16"), rows(sum(new), kv_heads, 4, "bf16"), rows(sum(new), heads, 5, "bf16")
    c.write(att, new, k, v, "bf16")
    out = c.attend(att, new, q, heads, "bf16")
    c.check_attend(out, new, q, heads, "bf16")
    total = [a + b for a, b in zip(lens, new)]
    got_k, got_v = c.read(att, total, "bf16")
    assert torch.equal(got_k.double(), c.expect("k", total).flatten(1))
    assert torch.equal(got_v.double(), c.expect("v", total).flatten(1))


@pytest.mark.parametrize("extra", [2, 300])
def test_rows_before_the_first_position_are_zero(att, extra):
    """More rows than a sequence has positions: the first ones see nothing and are 0, by either path."""
    heads, kv_heads, lens = 4, 2, [100, 0, 3]
    c = Cache(3, 2, kv_heads)
    k, v = rows(103, kv_heads, 1, "bf16"), rows(103, kv_heads, 2, "bf16")
    c.write(att, lens, k, v, "bf16")
    counts = [100 + extra, 2, 3 + extra]
    q = rows(sum(counts), heads, 3, "bf16")
    out = c.attend(att, counts, q, heads, "bf16")
    c.check_attend(out, counts, q, heads, "bf16")
    assert (out[:extra] == 0).all() and (out[100 + extra:102 + extra] == 0).all()


@pytest.mark.parametrize("tokens", [1, 5, 150])
def test_cache_past_32_bits(att, tokens):
    """A pool of more than 4 GB of codes whose last pages are the sequences': written, read and attended."""
    heads, kv_heads = 16, 8
    c = Cache(2, 5, kv_heads)
    pages = 2 ** 32 // (kv_heads * 64 * D) + 11
    codes = {x: torch.empty(pages, kv_heads, 64, D, dtype=torch.int8, device="cuda") for x in "kv"}
    scales = {x: torch.full((pages, kv_heads), 2.0 ** 40, device="cuda") for x in "kv"}
    c.codes, c.scales = codes, scales
    c.c.k, c.c.v = codes["k"].data_ptr(), codes["v"].data_ptr()
    c.c.k_scale, c.c.v_scale, c.c.pages = scales["k"].data_ptr(), scales["v"].data_ptr(), pages
    c.table.copy_((pages - 1 - torch.arange(10, device="cuda")).int().reshape(2, 5))
    lens = [161, 99]
    k, v = rows(260, kv_heads, 1, "bf16"), rows(260, kv_heads, 2, "bf16")
    c.write(att, lens, k, v, "bf16")
    new = [tokens, min(tokens, 2)]
    k, v, q = rows(sum(new), kv_heads, 3, "bf16"), rows(sum(new), kv_heads, 4, "bf16"), rows(sum(new), heads, 5, "bf16")
    c.write(att, new, k, v, "bf16")
    total = [a + b for a, b in zip(lens, new)]
    got_k, got_v = c.read(att, total, "bf16")
    assert torch.equal(got_k.double(), c.expect("k", total).flatten(1))
    assert torch.equal(got_v.double(), c.expect("v", total).flatten(1))
    c.check_attend(c.attend(att, new, q, heads, "bf16"), new, q, heads, "bf16")


# --------------------------------------------------------------------------- refusals


def test_refusals(att):
    x = torch.zeros(64, 8 * D, dtype=torch.bfloat16, device="cuda")
    o = offsets([64])
    p, po = x.data_ptr(), o.data_ptr()
    good = dict(q=p, k=p, v=p, out=p, offsets=po, nseq=1, rows=64, heads=8, kv_heads=8)
    for change in (dict(dtype=E.GGML_F32), dict(heads=7, kv_heads=2), dict(heads=0), dict(kv_heads=0), dict(q=None),
                   dict(out=None), dict(k=p + 8), dict(v=None), dict(ld_q=1000), dict(ld_k=1025), dict(ld_out=1028),
                   dict(offsets=None), dict(nseq=-1), dict(rows=-1), dict(rows=1 << 31), dict(scale=-1.0),
                   dict(scale=math.nan), dict(scale=math.inf), dict(kv_rows=60), dict(offsets=po + 2),
                   dict(heads=129 * 8, kv_heads=8)):
        with pytest.raises(E.ExnError) as e:
            att.packed(**dict(good, **change))
        assert e.value.code == 1 and "exn_attn_packed" in str(e.value), change
    c = Cache(1, 2, 8)
    for field, value in (("kv_heads", 0), ("pages", 0), ("table_ld", 0), ("k", None), ("lens", None), ("v", c.c.v + 8)):
        bad = E.KvCache.from_buffer_copy(c.c)
        setattr(bad, field, value)
        for call in (lambda: att.cache_write(bad, p, p, po, 64), lambda: att.cache_read(bad, p, p, po, 64),
                     lambda: att.cache_attend(bad, p, p, po, 64, 8), lambda: att.cache_workspace(bad, 64, 8)):
            with pytest.raises(E.ExnError) as e:
                call()
            assert e.value.code == 1
    with pytest.raises(E.ExnError):
        att.cache_attend(c.c, p, p, po, 64, 12)
    wide = torch.zeros(130, 8 * D, dtype=torch.bfloat16, device="cuda")
    n = att.cache_workspace(c.c, 130, 8)
    assert n > 0
    with pytest.raises(E.ExnError) as e:
        att.cache_attend(c.c, wide.data_ptr(), wide.data_ptr(), po, 130, 8, workspace=p, workspace_bytes=n - 1)
    assert "workspace" in str(e.value)
    att.packed(**dict(good, nseq=0))
    att.packed(**dict(good, rows=0))
    att.sync()


def test_bad_device_contents_are_left_out_and_reported(att):
    """Offsets, lengths and page numbers that only the kernels can see: reported by sync, the other
    sequences right, the handle usable."""
    heads, kv_heads, nq = 8, 2, [40, 50]
    q, k, v = rows(90, heads, 1, "bf16"), rows(90, kv_heads, 2, "bf16"), rows(90, kv_heads, 3, "bf16")
    want = run_packed(att, q, k, v, nq, heads, kv_heads, "bf16")
    for bad in ([0, 40, 91], [0, 40, 30], [-1, 40, 90]):
        o = torch.tensor(bad, dtype=torch.int32, device="cuda")
        out = torch.full_like(want, 7.0)
        att.packed(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), o.data_ptr(), 2, 90, heads, kv_heads)
        with pytest.raises(E.ExnError) as e:
            att.sync()
        assert e.value.code == 1 and "offsets" in str(e.value)
        part = slice(40, 90) if bad[0] < 0 else slice(0, 40)
        assert torch.equal(out[part], want[part])
    att.sync()
    c = Cache(2, 2, kv_heads)
    c.write(att, [70, 20], k, v, "bf16")
    one = offsets([1, 1])
    page = c.table[0, 1].item()
    for wrong in (-1, c.c.pages, 1 << 30):
        good = c.attend(att, [1, 1], q[:2], heads, "bf16")  # sequence 1 is written to below
        c.table[0, 1] = wrong
        out = torch.full_like(good, 7.0)
        with pytest.raises(E.ExnError):
            c.attend(att, [1, 1], q[:2], heads, "bf16", out=out)
        assert torch.equal(out[1], good[1])
        for call in (att.cache_write, att.cache_read):
            call(c.c, k.data_ptr(), v.data_ptr(), one.data_ptr(), 2)
            with pytest.raises(E.ExnError):
                att.sync()
        c.table[0, 1] = page
    for lens in ([200, 20], [0, 20]):  # more than the table has, fewer than the call's rows
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        att.cache_write(c.c, k.data_ptr(), v.data_ptr(), one.data_ptr(), 2)
        with pytest.raises(E.ExnError):
            att.sync()
    att.sync()


def test_current_device_and_errors_of_a_closed_gate():
    """The current device is the caller's after every call; a device that is not there is refused."""
    before = torch.cuda.current_device()
    with pytest.raises(E.ExnError) as e:
        E.Attention(device=99)
    assert e.value.code == 2 and "no CUDA device 99" in str(e.value)
    with E.Attention() as a:
        a.sync()
    assert torch.cuda.current_device() == before
    assert ctypes.sizeof(E.KvCache) == 64
