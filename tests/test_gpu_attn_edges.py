"""The attention operators (include/exn_b200.h, exn_attn_*) on a B200 where inputs are at the ends of their range.
The bounds of what an output may be off stand in test_gpu_attn.py, whose helpers these tests use."""
import math

import pytest

import exn_b200 as E
from test_gpu_attn import D, GGML, TYPES, Cache, att, check_packed, offsets, reference, rows, run_packed  # noqa: F401

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
