"""The encoder's passes of several prompts (exn_enc_states_packed) and over kept keys and values
(exn_enc_extend), against the oracle.

Tolerance as tests/test_gpu_encoder.py: bf16 operands of every product with fp32 sums, two blocks held to
rel-L2 <= 2e-2; the cached pass is compared with an oracle that rounds keys and values to 8 bits by the
cache's rule at the same steps.  There the products' own error moves keys and values over rounding borders,
each by one unit U: a value off by d changes its code with probability |d| / U, so codes differ by
sqrt(mean |d| U) in the root mean square.  U <= 2/127 of the page's largest of 64 x 128 values, about 4.3 of
their rms, so 0.068 rms; d comes from three roundings to bf16 (the row, the matrix, the result), each 2^-8 /
sqrt(3) / 1.4 relatively, so mean |d| <= 0.8 * sqrt(3) * 0.0016 = 0.0022 rms, and codes differ by sqrt(0.0022 *
0.068) = 1.2 % of the rms.  Keys move the weights by that much and values their sums by that much, 2.4 % of an
attention's output at most, so two blocks add 5 % at most to the 2e-2."""
import numpy as np
import pytest

import exn_b200 as E
from oracle import dit_oracle as O
from oracle import encoder_oracle as EO

pytestmark = pytest.mark.gpu
TOL = 2e-2
TOL_CACHED = TOL + 2 * 2.4e-2
SMALL = dict(width=EO.SMALL.width, layers=EO.SMALL.layers, heads=EO.SMALL.heads, kv_heads=EO.SMALL.kv_heads,
             ffn=EO.SMALL.ffn, vocab=EO.SMALL.vocab)


@pytest.fixture(scope="module")
def small():
    e = E.Encoder(**SMALL)
    e.load_synthetic(1)
    yield e
    e.close()


@pytest.fixture(scope="module")
def small_wt():
    return EO.SynthEncoder(EO.SMALL, seed=1)


@pytest.mark.parametrize("counts", [[1], [20, 0, 141, 33], [64, 65, 1], [300, 280, 77]])
def test_packed_prompts_match_oracle(small, small_wt, counts):
    """Prompts of different lengths in one pass (up to 512 tokens in all the GEMMs run split along K, beyond
    with the epilogues fused), each against the oracle alone."""
    prompts = [EO.synth_ids(EO.SMALL, n, seed=n) for n in counts]
    got = small.states_packed(prompts)
    assert [len(g) for g in got] == counts
    for g, ids in zip(got, prompts):
        if len(ids):
            err = O.rel_l2(g, EO.states(small_wt, EO.SMALL, ids))
            print("\npacked prompt of %d tokens: rel-L2 %.4g" % (len(ids), err))
            assert err < TOL


def test_packed_edit_positions(small, small_wt):
    a, b = EO.edit_positions(6, 4, 6, 9), EO.text_positions(31)
    prompts = [EO.synth_ids(EO.SMALL, len(p), seed=5) for p in (a, b)]
    got = small.states_packed(prompts, [a, b])
    for g, ids, pos in zip(got, prompts, (a, b)):
        assert O.rel_l2(g, EO.states(small_wt, EO.SMALL, ids, pos)) < TOL


def test_packed_device_feeds_a_batch_of_pictures(small):
    """Prompts of one length, the system turn's rows cut, straight into the contexts' memory: the rows of the
    host call."""
    import torch
    prompts = [EO.synth_ids(EO.SMALL, 24, seed=s) for s in (1, 2, 3)]
    want = np.stack([g[5:] for g in small.states_packed(prompts)])
    d = torch.full((3, 19, EO.SMALL.width), float("nan"), device="cuda")
    small.states_packed_device(prompts, d.data_ptr(), skip=5)
    assert np.array_equal(d.cpu().numpy(), want)


class CachedOracle:
    """The oracle's blocks over keys and values kept in 8 bits: pages of 64 tokens, a power-of-two unit a page
    and head that grows with what the page is given, codes rounded half to even."""

    def __init__(self, wt, sh):
        self.wt, self.sh, self.n = wt, sh, 0
        self.kept = [dict(k=np.zeros((0, sh.kv_heads, 128)), v=np.zeros((0, sh.kv_heads, 128)), ku={}, vu={})
                     for _ in range(sh.layers)]

    def _keep(self, li, name, x):
        c = self.kept[li]
        start, held = len(c[name]), np.concatenate([c[name], x.astype(np.float64)])
        for b in range(start // 64, (len(held) + 63) // 64):
            lo, hi = max(start, 64 * b), min(len(held), 64 * b + 64)
            for h in range(self.sh.kv_heads):
                amax, e = np.abs(held[lo:hi, h]).max(), -126
                while amax > 127 * 2.0 ** e:
                    e += 1
                if lo > 64 * b:
                    e = max(e, c[name + "u"][b, h])
                c[name + "u"][b, h] = e
                held[64 * b:hi, h] = np.rint(held[64 * b:hi, h] / 2.0 ** e) * 2.0 ** e
        c[name] = held
        return held

    def extend(self, ids, positions=None):
        sh, n = self.sh, len(ids)
        pos = np.repeat(np.arange(self.n, self.n + n)[:, None], 3, 1) if positions is None else positions
        ang = EO.mrope_angles(sh, pos)
        cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        x = self.wt("token_embd.weight")[ids].astype(np.float32)
        seen = np.arange(self.n + n) <= self.n + np.arange(n)[:, None]
        for li in range(sh.layers):
            b = "blk.%d." % li
            wt = self.wt
            h = EO.rms(x, wt(b + "attn_norm.weight"), sh.eps)
            q, k, v = ((h @ wt(b + "attn_%s.weight" % w).T).reshape(n, -1, 128) for w in "qkv")
            q = EO.rope_halves(EO.rms(q, wt(b + "attn_q_norm.weight"), sh.eps), cos, sin)
            k = EO.rope_halves(EO.rms(k, wt(b + "attn_k_norm.weight"), sh.eps), cos, sin)
            ks, vs = self._keep(li, "k", k), self._keep(li, "v", v)
            a = np.empty_like(q)
            for hd in range(sh.heads):
                kv = hd // (sh.heads // sh.kv_heads)
                s = np.where(seen, q[:, hd].astype(np.float64) @ ks[:, kv].T / np.sqrt(128.0), -np.inf)
                s = np.exp(s - s.max(-1, keepdims=True))
                a[:, hd] = (s / s.sum(-1, keepdims=True)) @ vs[:, kv]
            x = x + a.reshape(n, -1) @ wt(b + "attn_output.weight").T
            h = EO.rms(x, wt(b + "ffn_norm.weight"), sh.eps)
            g, u = h @ wt(b + "ffn_gate.weight").T, h @ wt(b + "ffn_up.weight").T
            x = (x + ((g / (1 + np.exp(-g))) * u) @ wt(b + "ffn_down.weight").T).astype(np.float32)
        self.n += n
        return x


def test_growing_prompts_match_the_oracle_over_8_bits(small, small_wt):
    """Prompts begun with different lengths, grown by single tokens and chunks, one waiting a while."""
    oracles = [CachedOracle(small_wt, EO.SMALL) for _ in range(3)]
    with small.cache(3, 300) as c:
        for i, counts in enumerate([[60, 5, 130], [1, 1, 1], [1, 0, 1], [70, 2, 33], [1, 1, 1]]):
            tokens = [EO.synth_ids(EO.SMALL, n, seed=10 * i + s) for s, n in enumerate(counts)]
            got = c.extend(tokens)
            for g, o, t in zip(got, oracles, tokens):
                if len(t):
                    err = O.rel_l2(g, o.extend(t))
                    print("\n%d tokens after %d: rel-L2 %.4g" % (len(t), o.n - len(t), err))
                    assert err < TOL_CACHED
            assert c.lengths() == [o.n for o in oracles]


def test_trimmed_prompt_continues_from_its_prefix(small):
    """A prompt edited from some word on: trimmed to whole pages and continued it gives, to the bit, the same
    whatever stood behind them before; the other sequence is as it was.  (Passes of the same sizes: the
    split of the GEMMs along K, so their fp32 order, goes by the pass's tokens.)"""
    sys_turn, old, new = (EO.synth_ids(EO.SMALL, n, seed=n) for n in (64, 90, 41))
    with small.cache(2, 256) as c:
        c.extend([sys_turn, sys_turn])
        c.extend([old, old[:7]])
        c.trim(0, 64)
        assert c.lengths() == [64, 71]
        a = c.extend([new, old[7:9]])
    with small.cache(2, 256) as c:
        c.extend([sys_turn, sys_turn])
        c.extend([old[::-1], old[:7]])
        c.trim(0, 64)
        b = c.extend([new, old[7:9]])
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_extend_is_near_the_uncached_states(small):
    """Eight bits against sixteen: a whole prompt through the cache and without it.  A page's unit is at most
    2/127 of its largest value, so a code is off by at most 1/127 of it; per-head rows of 128 values whose
    largest of 64 x 128 is about 4 of their rms are off by 4/127/sqrt(3) ~ 2 % of their rms at most, and
    weights and values each carry that once a block, averaged over the keys: two blocks stay below 6 %."""
    ids = EO.synth_ids(EO.SMALL, 150, seed=8)
    with small.cache(1, 150) as c:
        a = np.concatenate([c.extend([ids[:100]])[0], c.extend([ids[100:]])[0]])
    err = O.rel_l2(a, small.states(ids))
    print("\n8-bit keys and values against bf16: rel-L2 %.4g" % err)
    assert 0 < err < 6e-2


def test_refusals(small):
    for call in (lambda: small.states_packed([]), lambda: small.states_packed([[], []]),
                 lambda: small.states_packed([[0, EO.SMALL.vocab]]), lambda: small.states_packed([[-1]]),
                 lambda: small.states_packed([np.zeros(20000), np.zeros(20000)]),
                 lambda: small.states_packed([[1, 2]], [np.zeros((3, 3))]),
                 lambda: small.states_packed_device([[1, 2], [3]], 0, skip=0),
                 lambda: small.states_packed_device([[1, 2], [3]], 256, skip=1),
                 lambda: small.cache(0, 10), lambda: small.cache(1, 0), lambda: small.cache(1 << 20, 1 << 20)):
        with pytest.raises(E.ExnError) as e:
            call()
        assert e.value.code == 1
    with small.cache(2, 100) as c:
        c.extend([[1, 2, 3], []])
        for call in (lambda: c.extend([[], []]), lambda: c.extend([[1]]), lambda: c.extend([[1], list(range(129))]),
                     lambda: c.trim(0, 4), lambda: c.trim(2, 0), lambda: c.trim(0, -1), lambda: c.extend([[-5], []])):
            with pytest.raises(E.ExnError) as e:
                call()
            assert e.value.code == 1
        assert c.lengths() == [3, 0]
        with E.Encoder(**SMALL) as other:
            assert E.lib().exn_enc_cache_trim(other.h, c.h, 0, 0) == 1
    with E.Encoder(**SMALL) as bare:
        with pytest.raises(E.ExnError) as e:
            bare.states_packed([[1]])
        assert e.value.code == 4


def test_a_cache_of_a_closed_encoder_is_refused(small):
    """Another encoder, which may have got the closed one's address, does not take its cache."""
    first = E.Encoder(**SMALL)
    cache = first.cache(2, 64)
    address = first.h.value
    first.close()
    others = []
    for _ in range(8):
        others.append(E.Encoder(**SMALL))
        if others[-1].h.value == address:
            break
    for other in others + [small]:
        other.load_synthetic(1)
        cache.encoder = other
        with pytest.raises(E.ExnError) as e:
            cache.trim(0, 0)
        assert e.value.code == 1 and "another encoder" in str(e.value)
        with pytest.raises(E.ExnError) as e:
            cache.extend([[1], [2, 3]])
        assert e.value.code == 1 and "another encoder" in str(e.value)
    assert cache.lengths() == [0, 0]
    cache.close()
    for other in others:
        other.close()
