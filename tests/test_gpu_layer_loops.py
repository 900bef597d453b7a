"""The norm, the adapters and the experts where a block takes more than one row, tile or unit: the turns of rings, of barriers and of accumulators.

Tolerances as in test_gpu_layer.py, whose helpers these tests use."""
import pytest
import torch

from oracle import hpu_oracle as O
from test_gpu_layer import (BF16, E4M3, E5M2, EPS, F32, FLOOR, HALF_STEP, LIMIT, NORM, _check_lora, _check_moe, _close, _lora_case, _lora_tol, _moe_case, _run_lora, _run_moe,  # noqa: F401
                            _status)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- norm: several rows to a block
def _off(got, want, tol, what):
    off = (got.double() - want).abs() - tol
    assert bool(got.isfinite().all()) and float(off.max()) <= 0, f"{what}: {float(off.max()):.3g} beyond the tolerance"


# Rows of each instance of the ring (12, 6, 6, 4, 2, 2 and 1 blocks of an SM) and of the kernel that has a row in a warp or block, so many that each block has the
# ring's places twice and some have a row more: (dim, tokens).
ROWS = [(200, 12001), (400, 9000), (600, 16005), (1500, 6301), (2300, 4447), (3000, 4501), (4000, 5003), (8192, 1301), (12000, 1201), (20000, 601), (32768, 303)]


@pytest.mark.parametrize("odd", [0, 1, 3])
@pytest.mark.parametrize("src,residual,dtype,scale,keep", [(BF16, True, E4M3, None, True), (F32, False, E5M2, None, False), (F32, True, BF16, 0.5, True), (BF16, False, E4M3, 74.6, False)])
@pytest.mark.parametrize("dim,tokens", ROWS)
def test_norm_several_rows_to_a_block(dim, tokens, src, residual, dtype, scale, keep, odd):
    """Even rows, and packed rows of odd lengths, which begin between boundaries; the last one ends where the tensor does."""
    dim = dim - odd if dim > 32700 else dim + odd  # (rows of more values are a kernel of their own)
    g = torch.Generator(device="cuda").manual_seed(dim + tokens)
    x = torch.randn(tokens, dim, generator=g, device="cuda").to(src)
    r = (2 * torch.randn(tokens, dim, generator=g, device="cuda")).to(src) if residual else None
    w = (1 + 0.1 * torch.randn(dim, generator=g, device="cuda")).to(BF16)
    size = torch.logspace(-3, 3, tokens, device="cuda")[torch.randperm(tokens, generator=g, device="cuda")]
    x = (x.float() * size[:, None]).to(src)  # (a row's neighbours are of another size)
    z, y = O.add_rms_norm(x, r, w, EPS)
    s = None if scale is None else torch.tensor(scale, device="cuda")
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(x, r, w, EPS, dtype, s, keep)
    if residual:
        assert torch.equal(r, z)
    factor = 1.0 if scale is None else float(s)
    if dtype != BF16 and scale is None:
        top = y.abs().amax(-1, keepdim=True)
        factor = LIMIT[dtype] / top
        _off(inv, top / LIMIT[dtype], 2 * NORM * top / LIMIT[dtype], "scale_inv")
    v = (y * factor).clamp(-LIMIT[dtype], LIMIT[dtype])
    _off(out.float(), v, (HALF_STEP[dtype] + 2 * NORM) * v.abs() + FLOOR[dtype], "out")
    if keep:
        _off(kept.float(), y, (HALF_STEP[BF16] + NORM) * y.abs() + FLOOR[BF16], "kept")


@pytest.mark.parametrize("dim,step,tokens", [(4096, 4104, 1500), (4093, 4101, 1500), (605, 613, 5400), (8189, 8197, 700), (2301, 2317, 2000)])
def test_norm_rows_of_wider_matrices_several_to_a_block(dim, step, tokens):
    """Rows that lie alike in x and the outputs, with values between them that are neither read into a sum nor written."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    wide = torch.full((2, tokens, step), float("nan"), device="cuda", dtype=BF16)
    wide[:, :, :dim] = torch.randn(2, tokens, dim, generator=g, device="cuda").to(BF16)
    x, r = wide[0, :, :dim], wide[1, :, :dim]
    z, y = O.add_rms_norm(x, r, None, EPS)
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(x, r, None, EPS, E4M3)
    assert torch.equal(r, z) and bool(wide[:, :, dim:].isnan().all())
    top = y.abs().amax(-1, keepdim=True)
    v = y * (448.0 / top)
    _off(inv, top / 448.0, 2 * NORM * top / 448.0, "scale_inv")
    _off(out.float(), v, (HALF_STEP[E4M3] + 2 * NORM) * v.abs() + FLOOR[E4M3], "out")


# ----------------------------------------------------------------------------- adapters: several tiles to a block
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n,rank,adapters", [(6000, 72, 264, 16, 2048), (4000, 320, 136, 72, 1500), (2000, 136, 72, 256, 700), (8192, 72, 264, 16, 340), (8192, 200, 136, 64, 330)])
def test_lora_more_tiles_than_blocks(tokens, k, n, rank, adapters, dtype):
    """Tiles of 16 tokens, some two to four to each block of both kernels, so that the terms, the accumulators and their barriers turn."""
    c = _lora_case(tokens, k, n, rank, adapters, dtype)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("order", ["runs", "scattered"])
@pytest.mark.parametrize("tokens,k,n,rank,adapters", [(400, 2056, 136, 16, 2), (300, 4104, 72, 128, 1), (1024, 4104, 136, 64, 8), (2048, 8192, 64, 24, 16)])
def test_lora_long_rows_of_many_tokens(tokens, k, n, rank, adapters, order, dtype):
    """Rows of k that are cut into parts, of more than four steps of 64 values each."""
    which = torch.arange(tokens) * adapters // tokens
    if order == "scattered":
        which = which[torch.randperm(tokens, generator=torch.Generator().manual_seed(tokens))]
    c = _lora_case(tokens, k, n, rank, adapters, dtype, which=which)
    _check_lora(_run_lora(*c), *c)


@pytest.mark.parametrize("tokens,rank,adapters", [(40, 8, 1), (300, 8, 1), (400, 128, 2), (3000, 16, 100)])
def test_lora_fp32_sums_of_many_tokens(tokens, rank, adapters):
    """As test_lora_fp32_sums: 8192 products of one sign, off by less than 2^-18 of their sum; with rank products of one sign behind them, rank / 16 * 3 + 1 additions more of
    half the last sum on average, 25 * 2^-24 at most: below 2^-17."""
    y, x, a, b, which, scales = _lora_case(tokens, 8192, 64, rank, adapters, F32, which=torch.arange(tokens) % adapters)
    x, a, b, y = x.abs(), a.abs(), b.abs(), torch.zeros_like(y)
    want, size, _ = O.lora_add(y, x, a, b, which, scales)
    _close(_run_lora(y, x, a, b, which, scales), want, 2.0 ** -17 * size)


# ----------------------------------------------------------------------------- experts: several units to a block
@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(64, 1024, 640, 64, 8), (256, 512, 272, 96, 8), (8, 1024, 1040, 40, 8)])
def test_moe_several_units_to_a_block(tokens, hidden, inner, experts, top_k, weights):
    """More tiles than three times the SMs: units from the counter, accumulators and rings that turn many times."""
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k), case, top_k)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(1, 2048, 640, 4, 1), (3, 1280, 1536, 3, 2), (12, 2048, 160, 5, 2), (100, 1408, 128, 2, 2), (1, 4096, 2048, 2, 1)])
def test_moe_cut_short_rows(tokens, hidden, inner, experts, top_k, dtype, weights):
    """Rows of 9 to 32 steps, whose tiles are cut where they are fewer than a third of the SMs."""
    case = _moe_case(tokens, hidden, inner, experts, weights)
    _check_moe(_run_moe(case, top_k, dtype=dtype), case, top_k, dtype=dtype)


# ----------------------------------------------------------------------------- adapters: tiles of 128 tokens, which only long batches have
def _order(order, tokens, adapters):
    if order == "runs":
        return torch.arange(tokens) * adapters // tokens
    if order == "scattered":
        return torch.randint(-1, adapters + 1, (tokens,), generator=torch.Generator().manual_seed(tokens))
    lens = [1, 255, 1, 16, 64, 127, 128, 129, 700, 3]  # prompts beside single tokens
    which = torch.repeat_interleave(torch.arange(len(lens)) * 7 % (adapters + 1), torch.tensor(lens))
    return which.repeat(-(-tokens // len(which)))[:tokens]


def _check_long(got, y, x, a, b, which, scales):
    """_check_lora with the oracle's sums adapter by adapter, which for thousands of tokens is quicker than token by token."""
    want, size = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    live = (which >= 0) & (which < a.shape[0])
    for i in which[live].unique().tolist():
        rows, s = (which == i).nonzero()[:, 0], float(scales[i])
        u, v, t = a[i].double(), b[i].double(), x[rows].double()
        want[rows] += s * (t @ u.T @ v.T)
        size[rows] = abs(s) * (t.abs() @ u.abs().T @ v.abs().T)
    assert torch.equal(got.cpu()[~live], y[~live])
    _close(got.float(), want, _lora_tol(want, size, x.shape[1], a.shape[1], y.dtype))


LARGE = [(3200, 4104, 4104, 16, 8), (8192, 2056, 1416, 64, 84), (4000, 6400, 264, 40, 3), (6001, 200, 4304, 8, 20), (2048, 264, 136, 192, 3), (3000, 72, 1032, 136, 100), (6400, 4104, 2056, 128, 5)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("order", ["runs", "scattered", "mixed"])
@pytest.mark.parametrize("tokens,k,n,rank,adapters", LARGE)
def test_lora_long_batches(tokens, k, n, rank, adapters, order, dtype):
    c = _lora_case(tokens, k, n, rank, adapters, dtype, which=_order(order, tokens, adapters))
    _check_long(_run_lora(*c), *c)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("at", [3, 8])
def test_lora_long_batches_between_boundaries(at, dtype):
    """y from a column of a wider matrix on, x of another."""
    y, x, a, b, which, scales = c = _lora_case(4000, 6400, 264, 16, 6, dtype, which=_order("mixed", 4000, 6))
    wide, xs = torch.zeros(4000, 264 + 13, dtype=dtype).cuda(), torch.zeros(4000, 6416, dtype=BF16).cuda()
    wide[:, at:at + 264], xs[:, 8:6408] = y.cuda(), x.cuda()
    torch.ops.b200q.lora_add_(wide[:, at:at + 264], xs[:, 8:6408], a.cuda(), b.cuda(), which.cuda(), scales.cuda())
    _check_long(wide[:, at:at + 264], *c)
    assert bool((wide[:, :at] == 0).all()) and bool((wide[:, at + 264:] == 0).all())


def test_lora_long_batches_fp32_sums():
    """As test_lora_fp32_sums_of_many_tokens."""
    y, x, a, b, which, scales = _lora_case(3300, 8192, 64, 8, 4, F32, which=torch.arange(3300) % 4)
    x, a, b, y = x.abs(), a.abs(), b.abs(), torch.zeros_like(y)
    want, size, _ = O.lora_add(y, x, a, b, which, scales)
    _close(_run_lora(y, x, a, b, which, scales), want, 2.0 ** -17 * size)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lora_long_batches_one_behind_the_other(dtype):
    """A chain of calls on one y, between kernels that change y and x, has the bytes of calls that are waited for."""
    y, x, a, b, which, scales = (t.cuda() for t in _lora_case(4096, 4096, 2056, 16, 8, dtype, which=_order("mixed", 4096, 8)))

    def chain(wait):
        ys, xs, ws = y.clone(), x.clone(), which.clone()
        for i in range(6):
            torch.ops.b200q.lora_add_(ys, xs, a, b, ws, scales)
            wait()
            ys.mul_(0.75)
            wait()
            xs.neg_()
            wait()
            ws.copy_(ws.roll(1))
            wait()
        return ys

    want = chain(torch.cuda.synchronize)
    for _ in range(3):
        assert torch.equal(chain(lambda: None), want)


def test_lora_long_batches_infinities():
    import math
    y, x, a, b, which, scales = _lora_case(4000, 6400, 264, 16, 3, BF16, which=torch.arange(4000) % 3)
    a, b = a.abs() + 2.0 ** -10, b.abs() + 2.0 ** -10
    x[[0, 1, 300], 3] = math.inf
    x[7, 5], x[8, 6399], x[9, 0] = -math.inf, math.nan, math.inf
    want, _, _ = O.lora_add(y, x, a, b, which, scales)
    got = _run_lora(y, x, a, b, which, scales).cpu().float()
    bad = ~want.isfinite()
    assert int(bad.any(-1).sum()) == 6 and torch.equal(got[bad].nan_to_num(nan=7.0), want[bad].float().nan_to_num(nan=7.0))
    assert bool(got[~bad].isfinite().all())
