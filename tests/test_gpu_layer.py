"""The norm before, the adapters beside and the experts in place of the FP8 products, on the GPU against the oracle in 64 bits.

Tolerances.  A value that is rounded once to a type is off by at most half a step of it (bf16 2^-8, fp32 2^-24, e4m3 2^-4, e5m2 2^-3
relative; below the smallest normal half of 2^-9 and 2^-16).  On top of that comes the arithmetic in fp32, where an operation is off by 2^-24
and an addition inside the tensor cores by 2^-23:
norm: a sum of squares by threads of up to 64 values and a tree of up to 10 levels, half of it after the root, three products: below 2^-17.
adapters: sums over k and rank, 16 products at a time, (k + rank) / 16 + 32 additions, and the rounding of a x before it meets b, 2^-16 (y in
bf16) or 2^-23, all of scale |b| (|a| |x|).
experts: sums over hidden and inner, 32 products at a time at most, that is n / 32 + 32 additions, of the sums of absolute values; h by 2^-12 of itself
and 2^-26 of the largest of its token and expert; the oracle carries these through the gate and the second product."""
import ctypes as C
import math

import pytest
import torch

from oracle import hpu_oracle as O

pytestmark = pytest.mark.gpu
E4M3, E5M2, BF16, F32 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24, E4M3: 2.0 ** -4, E5M2: 2.0 ** -3}
FLOOR = {BF16: 2.0 ** -134, F32: 2.0 ** -149, E4M3: 2.0 ** -10, E5M2: 2.0 ** -17}
LIMIT = {BF16: math.inf, F32: math.inf, E4M3: 448.0, E5M2: 57344.0}
EPS = 1e-6


@pytest.fixture(autouse=True)
def _status():
    import b200_hpu_ops
    yield
    assert b200_hpu_ops.device_status() == 0


def _gen(*seed):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * int(v) for i, v in enumerate(seed)) % (1 << 31))


def _randn(g, *shape, std=1.0, dtype=BF16):
    x = torch.randn(*shape, generator=g) * std
    return x.clamp(-LIMIT[dtype], LIMIT[dtype]).to(dtype)


def _cu(t):
    return None if t is None else t.cuda()


def _one(v):
    return torch.tensor([v], dtype=F32)


def _close(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    off = torch.where(got == want, 0.0, (got - want).abs()) - tol  # (equal infinities are no distance)
    off = off[~want.isnan()]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max()):.3g} beyond the tolerance"


# ----------------------------------------------------------------------------- norm
NORM = 2.0 ** -17


def _check_norm(out, inv, kept, y, dtype, scale, keep):
    """out, scale_inv and kept against the oracle's y."""
    dynamic = dtype != BF16 and scale is None
    factor = torch.ones(y.shape[0], 1, dtype=torch.float64) * (1.0 if scale is None else float(scale))
    if dynamic:
        top = y.abs().amax(-1, keepdim=True) if y.shape[1] else torch.zeros(y.shape[0], 1, dtype=torch.float64)
        factor = torch.where(top == 0, 1.0, LIMIT[dtype] / top).clamp(max=torch.finfo(F32).max)
        want = torch.where(top == 0, 1.0, top / LIMIT[dtype])
        _close(inv, want, 2 * NORM * want.abs() + 2.0 ** -149)
    else:
        assert inv.shape == (0,)
    v = (y * factor).clamp(-LIMIT[dtype], LIMIT[dtype])
    _close(out.float(), v, (HALF_STEP[dtype] + 2 * NORM) * v.abs() + FLOOR[dtype])
    if keep:
        _close(kept.float(), y, (HALF_STEP[BF16] + NORM) * y.abs() + FLOOR[BF16])
    else:
        assert kept.shape == (0,)


def _norm_case(tokens, dim, src, residual, weight, dtype, scale, keep, seed=0):
    g = _gen(tokens, dim, seed)
    x, r = _randn(g, tokens, dim, dtype=src), _randn(g, tokens, dim, std=2.0, dtype=src) if residual else None
    w = None if weight is None else (1 + 0.1 * torch.randn(dim, generator=g)).to(weight)
    z, y = O.add_rms_norm(x, r, w, EPS)
    rd = _cu(r)
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(x.cuda(), rd, _cu(w), EPS, dtype, _cu(scale), keep)
    assert out.shape == x.shape and out.dtype == dtype
    if residual:
        assert torch.equal(rd.cpu(), z)
    _check_norm(out, inv, kept, y, dtype, scale, keep)


NORM_SIZES = [(1, 1), (1, 8), (3, 7), (2, 256), (5, 257), (4, 1000), (9, 1024), (2, 1032), (3, 2056), (7, 4096), (1, 8192), (160, 8192), (2, 8200), (2, 16384),
              (3, 13433), (1, 32768), (2, 32776), (1, 50001), (300, 264), (1200, 72), (2000, 1), (171, 3)]
NORM_FORMS = [(BF16, True, BF16, E4M3, None, True), (F32, False, BF16, E4M3, None, False), (BF16, False, None, E5M2, None, False), (F32, True, F32, E5M2, 200.0, True),
              (BF16, True, F32, E4M3, 74.6, False), (F32, True, None, BF16, None, False), (BF16, False, BF16, BF16, 0.5, True)]


@pytest.mark.parametrize("form", range(len(NORM_FORMS)))
@pytest.mark.parametrize("tokens,dim", NORM_SIZES)
def test_norm(tokens, dim, form):
    src, residual, weight, dtype, scale, keep = NORM_FORMS[form]
    _norm_case(tokens, dim, src, residual, weight, dtype, None if scale is None else _one(scale), keep)


def test_norm_static_scale_saturates():
    _norm_case(4, 512, BF16, True, BF16, E4M3, _one(1000.0), False)
    _norm_case(4, 512, F32, False, BF16, E5M2, _one(1e5), True)


@pytest.mark.parametrize("dim", [64, 61, 4096, 40000])
@pytest.mark.parametrize("src", [BF16, F32])
def test_norm_special_rows(src, dim):
    """Zeros; one value; a NaN; an infinity; squares that pass the end of fp32; squares below its beginning."""
    x = torch.zeros(7, dim, dtype=src)
    x[1, dim // 2] = 3.0
    x[2], x[2, dim - 1] = 1.0, math.nan
    x[3], x[3, 0] = 1.0, -math.inf
    x[4] = 1e25
    x[5] = 1e-30
    x[6] = -2.0
    w = torch.ones(dim, dtype=BF16)
    w[0] = -1.5
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(x.cuda(), None, w.cuda(), EPS, E4M3, None, True)
    out, inv, kept = out.float().cpu(), inv.cpu()[:, 0], kept.float().cpu()
    assert bool((out[[0, 4]] == 0).all()) and inv[[0, 4]].tolist() == [1.0, 1.0] and bool((kept[[0, 4]] == 0).all())
    assert out[1].tolist() == [448.0 if i == dim // 2 else 0.0 for i in range(dim)]
    assert bool(inv[[2, 3]].isnan().all()) and bool(out[[2, 3]].isnan().all())
    assert bool(kept[2].isnan().all()) and bool(kept[3, 0].isnan()) and bool((kept[3, 1:] == 0).all())
    assert out[5].abs().max() == 448.0  # 1e-30 / sqrt(eps): small, not nothing
    _, y = O.add_rms_norm(x[5:], None, w, EPS)
    want = y.abs().amax(-1) / 448
    _close(inv[5:], want, 2 * NORM * want)
    z = torch.full((1, dim), 1e-42, dtype=F32)  # the quotient 448 / max passes the end of fp32
    out, inv, _ = torch.ops.b200q.add_rms_norm_cast(z.cuda(), None, None, 1.0, E4M3)
    assert bool(out.float().isfinite().all()) and float(inv) == 2 * 2.0 ** -149  # 1e-42 / 448 is 1.6 of fp32's smallest steps


@pytest.mark.parametrize("dim", [128, 125, 2056])
def test_norm_strided_rows(dim):
    """Rows of wider matrices: what lies between stays as it is, and x and the residual may be columns of one matrix."""
    g = _gen(dim)
    both = _randn(g, 9, 2 * dim + 24)
    keep, x, r = both.clone(), both[:, 8:8 + dim], both[:, dim + 16:2 * dim + 16]
    d = both.cuda()
    z, y = O.add_rms_norm(x, r, None, EPS)
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(d[:, 8:8 + dim], d[:, dim + 16:2 * dim + 16], None, EPS, E4M3)
    keep[:, dim + 16:2 * dim + 16] = z
    assert torch.equal(d.cpu(), keep)
    _check_norm(out, inv, kept, y, E4M3, None, False)
    t = _randn(g, dim, 5)  # values that are not contiguous
    _check_norm(*torch.ops.b200q.add_rms_norm_cast(t.cuda().t(), None, None, EPS, E4M3), O.add_rms_norm(t.t(), None, None, EPS)[1], E4M3, None, False)
    row = _randn(g, 1, dim)  # one row for all tokens
    _check_norm(*torch.ops.b200q.add_rms_norm_cast(row.cuda().expand(4, dim), None, None, EPS, E4M3), O.add_rms_norm(row.expand(4, dim), None, None, EPS)[1], E4M3, None, False)


def test_norm_of_nothing():
    for shape in ((0, 64), (3, 0), (0, 0)):
        out, inv, kept = torch.ops.b200q.add_rms_norm_cast(torch.zeros(*shape, dtype=BF16).cuda(), None, None, EPS, E4M3, None, True)
        assert out.shape == kept.shape == shape and inv.cpu().tolist() == [[1.0]] * shape[0]


def test_norm_refuses():
    op = torch.ops.b200q.add_rms_norm_cast
    x = torch.zeros(4, 64, dtype=BF16).cuda()
    one = torch.ones(1).cuda()
    for args, why in [((x.half(), None, None, EPS, E4M3), "float or bfloat16"), ((x[0], None, None, EPS, E4M3), "tokens, dim"), ((x, None, None, EPS, F32), "dtype must be"),
                      ((x, x.float(), None, EPS, E4M3), "dtype and shape"), ((x, x[:2], None, EPS, E4M3), "dtype and shape"), ((x, x, None, EPS, E4M3), "must not overlap x"),
                      ((x, x[:1].clone().expand(4, 64), None, EPS, E4M3), "must not overlap"), ((x, x.clone().t().contiguous().t(), None, EPS, E4M3), "contiguous"),
                      ((x, None, one, EPS, E4M3), "64 values"), ((x, None, None, EPS, E4M3, torch.ones(4).cuda()), "one element"), ((x, None, None, EPS, E4M3, one.double()), "float tensor"),
                      ((x, x.cpu(), None, EPS, E4M3), "must be on")]:
        with pytest.raises(RuntimeError, match=why):
            op(*args)


# ----------------------------------------------------------------------------- adapters
def _lora_case(tokens, k, n, rank, adapters, dtype, seed=0, which=None, scaled=True):
    g = _gen(tokens, k, n, rank, adapters, seed)
    y, x = _randn(g, tokens, n, dtype=dtype), _randn(g, tokens, k)
    a, b = _randn(g, adapters, rank, k, std=k ** -0.5), _randn(g, adapters, n, rank, std=rank ** -0.5)
    if which is None:
        which = torch.randint(-1, adapters + 1, (tokens,), generator=g)  # (one is behind the last)
    return y, x, a, b, which.to(torch.int32), 0.5 + torch.rand(adapters, generator=g) if scaled else None


def _lora_tol(want, size, k, rank, dtype):
    return (HALF_STEP[dtype] * (1 + 2.0 ** -10)) * want.abs() + size * (((k + rank) / 16 + 32) * 2.0 ** -23 + (2.0 ** -16 if dtype == BF16 else 2.0 ** -23)) + FLOOR[dtype]


def _check_lora(got, y, x, a, b, which, scales):
    want, size, live = O.lora_add(y, x, a, b, which, scales)
    assert torch.equal(got.cpu()[~live], y[~live])
    _close(got.float(), want, _lora_tol(want, size, x.shape[1], a.shape[1], y.dtype))


def _run_lora(y, x, a, b, which, scales):
    yd = y.cuda()
    assert torch.ops.b200q.lora_add_(yd, x.cuda(), a.cuda(), b.cuda(), which.cuda(), _cu(scales)) is yd
    return yd


LORA_SIZES = [(1, 8, 8, 8, 1), (1, 256, 128, 16, 3), (2, 264, 136, 24, 2), (5, 1024, 512, 64, 4), (8, 512, 1416, 128, 3), (9, 520, 264, 8, 70), (17, 2056, 256, 40, 5),
              (33, 128, 1032, 256, 2), (64, 1024, 1024, 32, 64), (65, 256, 512, 16, 1), (130, 640, 392, 48, 7), (300, 384, 520, 32, 40), (1030, 128, 136, 16, 3),
              (200, 256, 520, 128, 2), (260, 136, 264, 64, 1), (129, 72, 136, 192, 2), (300, 64, 1416, 256, 3), (70, 4104, 128, 128, 1),
              (3, 7, 5, 3, 2), (4, 100, 61, 4, 3), (6, 129, 64, 8, 2), (7, 64, 99, 16, 2), (11, 64, 64, 20, 2), (2, 1, 1, 1, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n,rank,adapters", LORA_SIZES)
def test_lora(tokens, k, n, rank, adapters, dtype):
    c = _lora_case(tokens, k, n, rank, adapters, dtype)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("tokens,runs", [(200, [200]), (200, [64, 64, 72]), (257, [1, 255, 1]), (700, [16] * 20 + [300, 80]), (2100, [2100])])
@pytest.mark.parametrize("rank", [16, 64])
def test_lora_runs_of_tokens(tokens, runs, rank):
    """Prompts beside single tokens; some without an adapter."""
    which = torch.repeat_interleave((torch.arange(len(runs)) * 7) % 5 - (torch.arange(len(runs)) % 4 == 1).long() * 9, torch.tensor(runs))
    c = _lora_case(tokens, 192, 264, rank, 5, BF16, which=which)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("value", [-1, 7, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("rank", [16, 3])
def test_lora_without_adapters(value, rank):
    c = list(_lora_case(40, 64, 72, rank, 7, BF16))
    c[4] = torch.full((40,), value, dtype=torch.int32)
    assert torch.equal(_run_lora(*c).cpu(), c[0])


def test_lora_more_tokens_than_are_taken_at_once():
    g = _gen(1)
    which = torch.full((8192 + 8192 + 70,), -1)
    some = torch.randperm(which.numel(), generator=g)[:150]
    some[:3] = torch.tensor([8191, 8192, which.numel() - 1])
    which[some] = torch.randint(0, 6, (150,), generator=g)
    c = _lora_case(which.numel(), 64, 72, 16, 6, BF16, which=which)
    _check_lora(_run_lora(*c), *c)


def test_lora_last_tokens_in_more_parts_than_those_before():
    """85 adapters: 8192 tokens leave no room for parts of k, the 7936 behind them do."""
    g = _gen(2)
    which = torch.randint(-1, 85, (8192 + 7936,), generator=g)
    c = _lora_case(which.numel(), 512, 32, 8, 85, BF16, which=which)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("many", [2048, 1500])
def test_lora_many_adapters(many):
    c = _lora_case(50, 64, 64, 8, many, F32)
    _check_lora(_run_lora(*c), *c)


def test_lora_without_scales():
    c = _lora_case(9, 128, 64, 16, 3, F32, scaled=False)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("tokens", [1, 20, 300])
def test_lora_x_between_boundaries(tokens):
    y, x, a, b, which, scales = _lora_case(tokens, 64, 72, 16, 3, BF16)
    wide = torch.full((tokens, 70), math.nan, dtype=BF16)
    wide[:, 3:67] = x
    yd = y.cuda()
    torch.ops.b200q.lora_add_(yd, wide.cuda()[:, 3:67], a.cuda(), b.cuda(), which.cuda(), scales.cuda())
    _check_lora(yd, y, x, a, b, which, scales)


@pytest.mark.parametrize("pad", [8, 3])
def test_lora_strided(pad):
    """y a column block of a wider product, x rows of another, adapters of one layer in a stack of layers."""
    y, x, a, b, which, scales = _lora_case(21, 128, 96, 16, 4, BF16)
    wide = torch.zeros(21, 96 + 2 * pad, dtype=BF16).cuda()
    wide[:, pad:96 + pad] = y.cuda()
    xs = torch.zeros(21, 128 + pad, dtype=BF16).cuda()
    xs[:, pad:] = x.cuda()
    stack_a, stack_b = torch.zeros(4, 3, 16, 128, dtype=BF16).cuda(), torch.zeros(4, 3, 96, 16 + pad, dtype=BF16).cuda()
    stack_a[:, 1], stack_b[:, 1, :, :16] = a.cuda(), b.cuda()
    torch.ops.b200q.lora_add_(wide[:, pad:96 + pad], xs[:, pad:], stack_a[:, 1], stack_b[:, 1, :, :16], which.cuda(), scales.cuda())
    _check_lora(wide[:, pad:96 + pad], y, x, a, b, which, scales)
    assert bool((wide[:, :pad] == 0).all()) and bool((wide[:, 96 + pad:] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,at", [(5, 1), (200, 3), (200, 8)])
def test_lora_y_between_boundaries(tokens, at, dtype):
    """y from a column of a wider matrix on whose rows lie on no 16 bytes."""
    y, x, a, b, which, scales = _lora_case(tokens, 64, 272, 16, 2, dtype)
    wide = torch.zeros(tokens, 272 + 13, dtype=dtype).cuda()
    wide[:, at:at + 272] = y.cuda()
    torch.ops.b200q.lora_add_(wide[:, at:at + 272], x.cuda(), a.cuda(), b.cuda(), which.cuda(), scales.cuda())
    _check_lora(wide[:, at:at + 272], y, x, a, b, which, scales)
    assert bool((wide[:, :at] == 0).all()) and bool((wide[:, at + 272:] == 0).all())


def test_lora_one_row_for_all_tokens():
    y, x, a, b, which, scales = _lora_case(40, 64, 72, 16, 3, F32)
    yd = y.cuda()
    torch.ops.b200q.lora_add_(yd, x[:1].cuda().expand(40, 64), a.cuda(), b.cuda(), which.cuda(), scales.cuda())
    _check_lora(yd, y, x[:1].expand(40, 64), a, b, which, scales)


def test_lora_fp32_sums():
    """Sums over 8192 products of one sign, in which an addition that drops bits adds up.  256 products at a time are added inside the tensor core, 16 by 16: each
    addition may drop up to 2^-23 of the sum so far, half the last sum on average, 8.5 * 2^-23 in all, and 2^-23 for the products of a step; 32 such sums are added
    in fp32, 31 * 2^-24; b and its three terms add 4 * 2^-23: below 2^-18 of the sum of the absolute values.  A row of 512 such additions inside could be off by
    2^-15."""
    y, x, a, b, which, scales = _lora_case(40, 8192, 64, 8, 1, F32, which=torch.zeros(40))
    x, a, b, y = x.abs(), a.abs(), b.abs(), torch.zeros_like(y)
    want, size, _ = O.lora_add(y, x, a, b, which, scales)
    _close(_run_lora(y, x, a, b, which, scales), want, 2.0 ** -18 * size)


def test_lora_other_tokens_do_not_matter():
    """Infinities and NaN in other tokens, in other adapters, and in y's rows that are left alone."""
    y, x, a, b, which, scales = _lora_case(30, 128, 64, 16, 4, BF16)
    which[:] = torch.arange(30) % 4
    clean = _run_lora(y, x, a, b, which, scales).cpu()
    bad = which == 2
    x[bad], y[bad], a[2], b[2] = math.nan, math.inf, math.nan, -math.inf
    which[4] = -1
    y[4] = math.nan
    got = _run_lora(y, x, a, b, which, scales).cpu()
    fine = ~bad
    fine[4] = False
    assert torch.equal(got[fine], clean[fine]) and bool(got[bad].isnan().all()) and bool(got[4].isnan().all())


def test_lora_of_nothing():
    z = lambda *s: torch.zeros(*s, dtype=BF16).cuda()  # noqa: E731
    for t, k, n, r, ad in [(0, 8, 8, 8, 2), (3, 0, 8, 8, 2), (3, 8, 0, 8, 2), (3, 8, 8, 0, 2), (3, 8, 8, 8, 0)]:
        y = torch.ones(t, n, dtype=BF16).cuda()
        torch.ops.b200q.lora_add_(y, z(t, k), z(ad, r, k), z(ad, n, r), torch.zeros(t, dtype=torch.int32).cuda())
        assert bool((y == 1).all())


def test_lora_refuses():
    y, x, a, b, which, scales = (t.cuda() for t in _lora_case(4, 64, 32, 8, 2, BF16))
    op = torch.ops.b200q.lora_add_
    pool = torch.zeros(4, 128, dtype=BF16).cuda()
    for args, why in [((y.half(), x, a, b, which), "float or bfloat16"), ((y, x.float(), a, b, which), "bfloat16"), ((y, x, a.float(), b, which), "bfloat16"),
                      ((y[0], x, a, b, which), "wanted"), ((y, x[:3], a, b, which), "wanted"), ((y, x, a, b[:, :, :4], which), "wanted"), ((y, x, a[:1], b, which), "wanted"),
                      ((y, x, a, b, which.long()), "int32"), ((y, x, a, b, which[:3]), "int32"), ((y, x, a, b, which, scales[:1]), "per adapter"), ((y, x, a, b, which, scales.double()), "float"),
                      ((y[:1].expand(4, 32), x, a, b, which), "overlap"), ((y.t().contiguous().t(), x, a, b, which), "contiguous"), ((y, x.cpu(), a, b, which), "must be on"),
                      ((pool[:, 32:64], pool[:, :64], a, b, which), "must not overlap"), ((a.view(-1)[:128].view(4, 32), x, a, b, which), "must not overlap")]:
        with pytest.raises(RuntimeError, match=why):
            op(*args)
    op(pool[:, 64:96], pool[:, :64], a, b, which)  # columns of one matrix that lie apart
    big = torch.zeros(1, 257, 8, dtype=BF16).cuda()
    with pytest.raises(RuntimeError, match="maximum"):
        op(y[:, :8], x[:, :8], big, big.transpose(1, 2).contiguous(), which)


# ----------------------------------------------------------------------------- experts
def _moe_case(tokens, hidden, inner, experts, weights, seed=0, scaled=True, router=BF16):
    g = _gen(tokens, hidden, inner, experts, seed)
    fp8 = weights == E4M3
    x, r = _randn(g, tokens, hidden), _randn(g, experts, hidden, std=1.5 * max(1, hidden) ** -0.5, dtype=router)
    gu = _randn(g, experts, 2 * inner, hidden, std=64.0 if fp8 else max(1, hidden) ** -0.5, dtype=weights)
    down = _randn(g, experts, hidden, inner, std=64.0 if fp8 else max(1, inner) ** -0.5, dtype=weights)
    s = [None, None]
    if scaled:
        s = [(0.5 + torch.rand(experts, n, generator=g)) * (max(1, m) ** -0.5 / 64 if fp8 else 1.0) for n, m in ((2 * inner, hidden), (hidden, inner))]
    return x, r, gu, down, s[0], s[1]


def _check_moe(got, case, top_k, renormalize=True, count=None, dtype=BF16):
    x, r, gu, down, s1, s2 = case
    out, weights, ids = got
    w, i = O.moe_route(x, r, top_k, renormalize, count)
    assert torch.equal(ids.cpu(), i)
    _close(weights, w, 2.0 ** -20 * w.abs())
    n = max(x.shape[1], down.shape[2])
    want, bound = O.moe_experts(x, w, i, gu, down, s1, s2, rel_sum=(n / 32 + 32) * 2.0 ** -23, rel_hidden=2.0 ** -12, abs_hidden=2.0 ** -26)
    assert out.dtype == dtype
    _close(out.float(), want, HALF_STEP[dtype] * (1 + 2.0 ** -10) * want.abs() + bound + FLOOR[dtype])


def _run_moe(case, top_k, renormalize=True, count=None, dtype=None):
    x, r, gu, down, s1, s2 = (_cu(t) for t in case)
    n = None if count is None else torch.tensor([count], dtype=torch.int32).cuda()
    return torch.ops.b200q.moe_layer(x, r, gu, down, s1, s2, top_k, renormalize, n, dtype)


MOE_SIZES = [(1, 64, 64, 4, 2), (1, 512, 256, 16, 8), (2, 128, 96, 3, 1), (3, 272, 144, 8, 8), (7, 256, 128, 5, 2), (8, 128, 128, 33, 4), (9, 640, 272, 16, 3), (16, 256, 512, 2, 1),
             (29, 384, 160, 64, 8), (33, 128, 64, 2, 2), (64, 256, 128, 32, 4), (70, 64, 64, 1, 1), (100, 128, 256, 9, 3), (5, 1024, 688, 12, 6)]


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", MOE_SIZES)
def test_moe(tokens, hidden, inner, experts, top_k, weights):
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k), case, top_k)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 1, 1, 1, 1), (3, 7, 5, 4, 2), (2, 100, 33, 6, 3), (4, 64, 40, 3, 2), (5, 36, 64, 3, 3)])
def test_moe_sizes_off_the_tiles(tokens, hidden, inner, experts, top_k, weights):
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k), case, top_k)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("renormalize,dtype,scaled,router", [(False, None, True, BF16), (True, F32, True, F32), (False, F32, False, F32)])
def test_moe_forms(weights, renormalize, dtype, scaled, router):
    case = _moe_case(6, 256, 128, 12, weights, scaled=scaled, router=router)
    if weights == E4M3 and not scaled:
        case = (case[0], case[1], (case[2].float() / 512).to(E4M3), (case[3].float() / 512).to(E4M3), None, None)
    _check_moe(_run_moe(case, 3, renormalize, dtype=dtype), case, 3, renormalize, dtype=dtype or BF16)


@pytest.mark.parametrize("count", [-5, 0, 1, 6, 11, 12, 100])
@pytest.mark.parametrize("hidden", [128, 100])
def test_moe_padded(count, hidden):
    case = _moe_case(12, hidden, 64, 8, E4M3)
    case[0][max(0, count):] = math.nan  # (nothing is made of what lies there)
    live = min(max(count, 0), 12)
    got = _run_moe(case, 2, count=count)
    _check_moe(got, case, 2, count=live)
    assert bool((got[0][live:] == 0).all())


@pytest.mark.parametrize("tokens,count", [(257, None), (600, 300), (520, 256)])
def test_moe_more_tokens_than_are_taken_at_once(tokens, count):
    case = _moe_case(tokens, 64, 32, 4, E4M3)
    _check_moe(_run_moe(case, 2, count=count), case, 2, count=count)


@pytest.mark.parametrize("tokens", [3, 40])
def test_moe_all_tokens_to_the_same_experts(tokens):
    case = _moe_case(tokens, 128, 96, 10, E4M3)
    case[0][:, 0] = case[0][:, 0].abs() + 4
    case[1][4], case[1][7] = 0, 0
    case[1][4, 0], case[1][7, 0] = 8, 4
    got = _run_moe(case, 2)
    assert bool((got[2].cpu() == torch.tensor([4, 7])).all())
    _check_moe(got, case, 2)


def test_moe_equal_logits_go_to_the_lower_index():
    case = _moe_case(5, 64, 32, 40, BF16)
    case[1][:] = case[1][0]
    got = _run_moe(case, 6)
    assert bool((got[2].cpu() == torch.arange(6)).all())
    _check_moe(got, case, 6)
    case[1][[39, 33, 2]] = -case[1][0]
    got = _run_moe(case, 3)
    _check_moe(got, case, 3)


def test_moe_neighbours_in_the_order_of_experts():
    """Logits that differ by 2^-40 of their terms: a sum in fp32 would order them by its roundings."""
    x = torch.full((1, 512), 1.0)
    x[0, 1::2] = -1.0
    router = torch.full((20, 512), 1.0, dtype=F32)
    router += torch.randn(512, generator=_gen(5))  # the same for all experts
    order = torch.randperm(20, generator=_gen(6))
    router[:, 0] = 0.0
    router[order, 0] = torch.arange(20, 0, -1).float() * 2.0 ** -40
    case = (x.to(BF16), router, *_moe_case(1, 512, 64, 20, E4M3)[2:])
    got = _run_moe(case, 16)
    assert torch.equal(got[2].cpu()[0].long(), order[:16])
    _check_moe(got, case, 16)


def test_moe_a_token_of_nan_leaves_the_others_alone():
    case = _moe_case(10, 256, 128, 8, E4M3)
    clean = [t.cpu() for t in _run_moe(case, 2)]
    case[0][3, 7] = math.nan
    case[0][5, 0] = math.inf
    out, weights, ids = (t.cpu() for t in _run_moe(case, 2))
    others = [t for t in range(10) if t not in (3, 5)]
    for got, want in zip((out, weights, ids), clean):
        assert torch.equal(got[others], want[others])
    assert ids[3].tolist() == [0, 1] and bool(weights[3].isnan().all()) and bool(out[3].isnan().all())
    assert bool(((ids >= 0) & (ids < 8)).all())


def test_moe_values_of_uneven_size():
    """Tokens and experts whose values lie many powers of two apart, within a token too."""
    case = list(_moe_case(9, 256, 128, 6, E4M3))
    size = 2.0 ** torch.tensor([-60, -20, -3, 0, 1, 9, 20, 40, -120.0])
    case[0] = (case[0].float() * size[:, None]).to(BF16)
    case[0][:, 100:] = (case[0][:, 100:].float() * 2.0 ** -12).to(BF16)
    case[4] = case[4] * (2.0 ** torch.randint(-6, 7, (6, 1), generator=_gen(9)))
    case = tuple(case)
    x, r, gu, down, s1, s2 = case
    out, weights, ids = _run_moe(case, 2, dtype=F32)
    w, i = O.moe_route(x, r, 2, True)
    assert torch.equal(ids.cpu(), i)
    _close(weights, w, 2.0 ** -20 * w.abs() + 2.0 ** -126)
    want, bound = O.moe_experts(x, w, i, gu, down, s1, s2, rel_sum=40 * 2.0 ** -23, rel_hidden=2.0 ** -12, abs_hidden=2.0 ** -26)
    # (what a term of x is off by, 2^-22 of the token's largest value, against that of the sum of all terms, enters like a sum's error)
    ok = want.abs() < 1e37
    _close(torch.where(ok, out.cpu().double(), 0.0), torch.where(ok, want, 0.0), torch.where(ok, 2.0 ** -18 * want.abs() + 4 * bound + 1e-37, 1.0))


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("form", ["columns", "between", "expanded", "reversed"])
def test_moe_views_of_x(form, weights):
    case = list(_moe_case(11, 128, 64, 6, weights))
    x = case[0]
    if form == "expanded":
        case[0] = x[:1].expand(11, 128)
        xd = x[:1].cuda().expand(11, 128)
    elif form == "reversed":
        case[0] = x.t().contiguous().t()
        xd = x.t().contiguous().cuda().t()
    else:
        wide = torch.full((11, 160), math.nan, dtype=BF16)
        at = 16 if form == "columns" else 3
        wide[:, at:at + 128] = x
        xd = wide.cuda()[:, at:at + 128]
    out = torch.ops.b200q.moe_layer(xd, *(_cu(t) for t in case[1:]), 2)
    _check_moe(out, case, 2)


@pytest.mark.parametrize("experts,top_k,tokens", [(512, 16, 3), (512, 16, 40), (300, 7, 64), (129, 16, 256), (16, 16, 256), (1, 1, 256)])
def test_moe_largest_numbers_of_experts(experts, top_k, tokens):
    case = _moe_case(tokens, 64, 32, experts, E4M3)
    _check_moe(_run_moe(case, top_k), case, top_k)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 4096, 128, 4, 1), (3, 128, 4096, 3, 2), (20, 2176, 272, 40, 2), (9, 1280, 1280, 8, 1), (12, 1024, 640, 148, 3), (1, 8192, 32, 1, 1), (100, 1536, 1280, 4, 2), (256, 1184, 144, 5, 1)])
def test_moe_cut_tiles(tokens, hidden, inner, experts, top_k, weights):
    """Long rows on few tiles, and numbers of tiles around those of the SMs: all tiles cut into parts, some, or none."""
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k), case, top_k)


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k,weights", [(100, 4352, 160, 4, 2, E4M3), (70, 160, 4400, 3, 1, E4M3), (4, 4480, 144, 80, 16, E4M3), (9, 5120, 4224, 2, 1, E4M3),
                                                                     (100, 2176, 144, 4, 2, BF16), (24, 2304, 320, 60, 8, BF16), (2, 2112, 2120, 5, 3, BF16)])
def test_moe_cut_long_rows(tokens, hidden, inner, experts, top_k, weights):
    """Rows of more than 4096 bytes, whose tiles are cut where they do not come out even: few tiles, more than the SMs, several groups of an expert, both products."""
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k), case, top_k)


def test_moe_of_nothing():
    z = lambda *s: torch.zeros(*s, dtype=BF16).cuda()  # noqa: E731
    out, weights, ids = torch.ops.b200q.moe_layer(z(0, 64), z(4, 64), z(4, 64, 64), z(4, 64, 32), None, None, 2)
    assert out.shape == (0, 64) and weights.shape == ids.shape == (0, 2)
    out, weights, ids = torch.ops.b200q.moe_layer(z(3, 64), z(4, 64), z(4, 0, 64), z(4, 64, 0), None, None, 2)
    assert bool((out == 0).all()) and ids.cpu().tolist() == [[0, 1]] * 3 and weights.cpu().tolist() == [[0.5, 0.5]] * 3


def test_moe_refuses():
    x, r, gu, down, s1, s2 = (t.cuda() for t in _moe_case(4, 64, 32, 5, E4M3))
    op = torch.ops.b200q.moe_layer
    for args, why in [((x.float(), r, gu, down, s1, s2, 2), "bfloat16 tensor"), ((x[0], r, gu, down, s1, s2, 2), "bfloat16 tensor"), ((x, r.half(), gu, down, s1, s2, 2), "router"),
                      ((x, r, gu.to(E5M2), down, s1, s2, 2), "both be"), ((x, r, gu, down.float().to(BF16), s1, s2, 2), "both be"), ((x, r[:4], gu, down, s1, s2, 2), "wanted"),
                      ((x, r, gu[:, :62], down, s1, s2, 2), "wanted"), ((x, r, gu, down[:, :60], s1, s2, 2), "wanted"), ((x, r, gu, down, s1, s2, 0), "top_k"), ((x, r, gu, down, s1, s2, 6), "top_k"),
                      ((x, r, gu, down, s1[:, :3], s2, 2), "gate_up_scale_inv"), ((x, r, gu, down, s1, s2.double(), 2), "down_scale_inv"), ((x, r, gu, down, s1, s2, 2, True, torch.ones(1).cuda()), "num_tokens"),
                      ((x, r, gu, down, s1, s2, 2, True, None, E4M3), "out_dtype"), ((x, r.cpu(), gu, down, s1, s2, 2), "must be on"),
                      ((x, r, gu.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3), down, s1, s2, 2), "contiguous")]:
        with pytest.raises(RuntimeError, match=why):
            op(*args)


# ----------------------------------------------------------------------------- all of them
def _step(x, residual, w):
    """A decoder layer's products for a few tokens: norm, FP8 projection with adapters, norm, experts."""
    ops = torch.ops.b200q
    x8, inv, kept = ops.add_rms_norm_cast(x, residual, w["norm1"], EPS, E4M3, None, True)
    y = torch.ops.hpu.fp8_gemm_v2(x8, False, w["proj"], True, None, BF16, inv, w["proj_scale"])
    ops.lora_add_(y, kept, w["a"], w["b"], w["which"], w["scales"])
    z, _, _ = ops.add_rms_norm_cast(y, residual, w["norm2"], EPS, BF16)
    return ops.moe_layer(z, w["router"], w["gate_up"], w["down"], w["s1"], w["s2"], 2, True, w["count"])


def _step_inputs(tokens, dim, seed=0):
    g = _gen(tokens, dim, seed)
    _, r, gu, down, s1, s2 = _moe_case(tokens, dim, 128, 6, E4M3)
    w = dict(norm1=(1 + 0.1 * torch.randn(dim, generator=g)).to(BF16), norm2=(1 + 0.1 * torch.randn(dim, generator=g)).to(BF16), proj=_randn(g, dim, dim, std=64.0, dtype=E4M3),
             proj_scale=torch.rand(1, dim, generator=g) * dim ** -0.5 / 64, a=_randn(g, 3, 16, dim, std=dim ** -0.5), b=_randn(g, 3, dim, 16, std=0.25),
             which=torch.randint(-1, 3, (tokens,), generator=g).to(torch.int32), scales=torch.rand(3, generator=g), router=r, gate_up=gu, down=down, s1=s1, s2=s2,
             count=torch.tensor([tokens - 1], dtype=torch.int32))
    return _randn(g, tokens, dim), _randn(g, tokens, dim, std=2.0), w


@pytest.mark.parametrize("tokens", [2, 19])
def test_a_layer_of_them(tokens):
    """Each operator on what the one before has left, against the oracle on the same."""
    dim = 256
    x, residual, w = _step_inputs(tokens, dim)
    d = {k: v.cuda() for k, v in w.items()}
    res = residual.cuda()
    ops = torch.ops.b200q
    x8, inv, kept = ops.add_rms_norm_cast(x.cuda(), res, d["norm1"], EPS, E4M3, None, True)
    z, y = O.add_rms_norm(x, residual, w["norm1"], EPS)
    assert torch.equal(res.cpu(), z)
    _check_norm(x8, inv, kept, y, E4M3, None, True)
    p = torch.ops.hpu.fp8_gemm_v2(x8, False, d["proj"], True, None, BF16, inv, d["proj_scale"])
    want = (x8.cpu().double() * inv.cpu().double()) @ (w["proj"].double() * w["proj_scale"].double().T).T
    _close(p.float(), want, 2.0 ** -8 * want.abs() + 2.0 ** -16)
    base = p.cpu()
    ops.lora_add_(p, kept, d["a"], d["b"], d["which"], d["scales"])
    _check_lora(p, base, kept.cpu(), w["a"], w["b"], w["which"], w["scales"])
    mid, zero, _ = ops.add_rms_norm_cast(p, res, d["norm2"], EPS, BF16)
    z2, y2 = O.add_rms_norm(p.cpu(), z, w["norm2"], EPS)
    assert torch.equal(res.cpu(), z2) and zero.numel() == 0
    _close(mid.float(), y2, (2.0 ** -8 + NORM) * y2.abs())
    got = ops.moe_layer(mid, d["router"], d["gate_up"], d["down"], d["s1"], d["s2"], 2, True, d["count"])
    _check_moe(got, (mid.cpu(), w["router"], w["gate_up"], w["down"], w["s1"], w["s2"]), 2, count=tokens - 1)


@pytest.mark.parametrize("tokens", [2, 19])
def test_a_captured_layer(tokens):
    """The step as a graph on a stream of its own, replayed on other inputs; two graphs that were captured one behind the other, and eager calls between."""
    x, residual, w = _step_inputs(tokens, 256)
    d = {k: v.cuda() for k, v in w.items()}
    ins = [(x, residual), (-0.5 * x, residual.flip(0).contiguous())]
    eager = []
    for a, b in ins:
        r = b.cuda()
        eager.append([*(t.cpu() for t in _step(a.cuda(), r, d)), r.cpu()])
    xs, rs, outs, graphs = [], [], [], []
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(2):
        xs.append(torch.zeros_like(x).cuda())
        rs.append(torch.zeros_like(residual).cuda())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(_step(xs[-1], rs[-1], d))
        graphs.append(graph)
    for which in (0, 1, 1, 0):
        for i in range(2):
            a, b = ins[which ^ i]
            xs[i].copy_(a.cuda())
            rs[i].copy_(b.cuda())
        for graph in graphs:
            graph.replay()
        _step(x.cuda(), residual.cuda(), d)
        torch.cuda.synchronize()
        for i in range(2):
            for got, want in zip([*outs[i], rs[i]], eager[which ^ i]):
                assert torch.equal(got.cpu(), want)
    for graph in graphs:
        graph.reset()


def test_the_same_call_gives_the_same_bytes():
    x, residual, w = _step_inputs(37, 256)
    d = {k: v.cuda() for k, v in w.items()}
    first = None
    for _ in range(4):
        r = residual.cuda()
        got = [*(t.cpu() for t in _step(x.cuda(), r, d)), r.cpu()]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("tokens,n,adapters", [(1, 4096, 2), (20, 1032, 7), (128, 2048, 60), (400, 512, 90), (1500, 256, 3)])
def test_adapters_one_behind_the_other(tokens, n, adapters):
    """Kernels begin before those in front of them are done, and fetch y early: a chain of calls on one y, between kernels that change y and x, has the bytes of calls that are waited for."""
    y, x, a, b, which, scales = (t.cuda() for t in _lora_case(tokens, 256, n, 16, adapters, BF16))

    def chain(y, x, wait):
        for i in range(12):
            torch.ops.b200q.lora_add_(y, x, a, b, which, scales)
            wait()
            if i % 3 == 1:
                y.mul_(0.75)
                wait()
            if i % 4 == 2:
                x.neg_()
                wait()
            which.copy_(which.roll(1))
            wait()
        return y

    first = which.clone()
    want = chain(y.clone(), x.clone(), torch.cuda.synchronize)
    for _ in range(5):
        which.copy_(first)
        assert torch.equal(chain(y.clone(), x.clone(), lambda: None), want)
    ys, xs = y.clone(), x.clone()
    which.copy_(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(ys, xs, lambda: None)
    for _ in range(3):
        which.copy_(first)
        ys.copy_(y)
        xs.copy_(x)
        graph.replay()
        assert torch.equal(ys, want)
    graph.reset()


def test_two_streams_at_once():
    x, residual, w = _step_inputs(19, 256)
    d = {k: v.cuda() for k, v in w.items()}
    want = [t.cpu() for t in _step(x.cuda(), residual.cuda(), d)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    inputs = [[(x.cuda(), residual.cuda()) for _ in range(6)] for _ in streams]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        for s, pairs in zip(streams, inputs):
            with torch.cuda.stream(s):
                outs.append(_step(*pairs[i], d))
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(out, want))


def test_plain_and_fast_kernels_agree():
    """The C ABI's force_plain on sizes that have tensor-core kernels: within the same bounds."""
    from b200_hpu_ops import abi
    case = _moe_case(6, 256, 128, 8, E4M3)
    x, r, gu, down, s1, s2 = (t.cuda() for t in case)
    for plain in (0, 1):
        out, weights, ids = torch.empty(6, 256, dtype=BF16).cuda(), torch.empty(6, 2).cuda(), torch.empty(6, 2, dtype=torch.int32).cuda()
        n = abi.lib.b200q_moe_workspace_bytes(6, 256, 128, 8, 2)
        ws = torch.empty(n, dtype=torch.uint8).cuda()
        a = abi.MoeArgs(x=x.data_ptr(), x_stride=256, tokens=6, hidden=256, inner=128, experts=8, top_k=2, renormalize=1, router=r.data_ptr(), router_dtype=abi.BF16,
                        gate_up=gu.data_ptr(), down=down.data_ptr(), weight_dtype=abi.E4M3, gate_up_scale=s1.data_ptr(), down_scale=s2.data_ptr(), out=out.data_ptr(),
                        out_dtype=abi.BF16, weights=weights.data_ptr(), ids=ids.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=n, force_plain=plain, stream=abi.stream_ptr())
        abi.check(abi.lib.b200q_moe_layer(C.byref(a)))
        _check_moe((out, weights, ids), case, 2)
    y, x, a_w, b_w, which, scales = _lora_case(40, 128, 96, 16, 4, F32)
    d = [t.cuda() for t in (x, a_w, b_w, which, scales)]
    for plain in (0, 1):
        yd = y.cuda()
        n = abi.lib.b200q_lora_workspace_bytes(40, 128, 96, 16, 4)
        ws = torch.empty(n, dtype=torch.uint8).cuda()
        a = abi.LoraArgs(x=d[0].data_ptr(), x_stride=128, y=yd.data_ptr(), y_dtype=abi.F32, y_stride=96, a=d[1].data_ptr(), b=d[2].data_ptr(), a_stride=2048, a_row_stride=128,
                         b_stride=1536, b_row_stride=16, adapter=d[3].data_ptr(), scales=d[4].data_ptr(), tokens=40, k=128, n=96, rank=16, adapters=4,
                         workspace=ws.data_ptr(), workspace_bytes=n, force_plain=plain, stream=abi.stream_ptr())
        abi.check(abi.lib.b200q_lora_add(C.byref(a)))
        _check_lora(yd, y, x, a_w, b_w, which, scales)
