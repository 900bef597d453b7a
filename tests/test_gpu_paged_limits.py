"""The paged key/value cache where it is easily wrong: precision of fp32 outputs, sizes near the ends of their types, tables and
caches of unusual form.  The oracle and the helpers are those of test_gpu_paged.py."""
import math

import pytest
import torch

from oracle import hpu_oracle as O
from test_gpu_paged import BF16, E4M3, E5M2, F32, _close, _i32, _one, _Paged, _status  # noqa: F401 (_status: device status after each test)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- attention: precision
@pytest.mark.parametrize("cache", [E4M3, E5M2, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (20, 1, 128), (24, 2, 64), (8, 2, 64), (16, 1, 256), (4, 2, 80)])
def test_fp32_output_has_more_bits_than_a_half(cache, heads, kv, dim):
    """Queries and keys are small integers, so that scores are exact.  What is left: three roundings of a score's factor (scale, its
    inverse scale of the keys, log2 e), 3 * 2^-24 of an exponent below 2^5 in absolute value: 2^-17 of a probability, and again of the sum; the
    two terms of a probability, 2^-16 for bf16 and 2^-21 for f16 terms; ex2, 2^-22; and sums over up to 257 keys, 16 at a time: 33 additions at
    2^-23.  Together below 2^-14 (bf16) and 2^-15 of sum p |v|.  A probability of one f16 would be off by up to 2^-11."""
    p = _Paged([0, 1, 2, 3, 17, 40, 100, 257], kv, dim, cache, 16, seed=dim)
    k = torch.randint(-2, 3, p.k.shape, generator=p.g).float()
    p.k = torch.where(p.k.float().isnan(), math.nan, k).to(cache)
    q = torch.randint(-3, 4, (8, heads, dim), generator=p.g).to(BF16)
    scale = 2.0 / dim
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, scale)
    assert float(lse[lse.isfinite()].abs().max()) < 16
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.k.cuda(), p.vd, p.table.cuda(), p.lens.cuda(), scale, out_dtype=F32)
    _close(got, want, 2.0 ** -23 * want.abs() + 2.0 ** (-14 if cache == BF16 else -15) * size)
    _close(got_lse, lse, 2.0 ** -16 + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), 0.0))


# ----------------------------------------------------------------------------- append
@pytest.mark.parametrize("rot", [8, 64])
def test_append_with_a_table_of_no_positions(rot):
    """Every position is outside such a table: what turns becomes NaN, values are stored as ever."""
    x = torch.randn(4, 3, 64).to(BF16).cuda()
    kc, vc = torch.zeros(2, 1, 16, 1, 64, dtype=BF16).cuda()
    at = torch.arange(4).cuda()
    q = torch.ops.b200q.qk_norm_rope_append(x[:, :1], x[:, 1:2], x[:, 2:], None, None, 1e-6, torch.empty(0, rot).cuda(), at, False, at, kc, vc)
    for t in (q, kc[0, :4]):
        assert bool(t[..., :rot].isnan().all()) and bool(t[..., rot:].isfinite().all())
    assert torch.equal(vc[0, :4], x[:, 2:])
