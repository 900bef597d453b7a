"""The norm, the adapters and the experts where something does not come, or does not fit: waits that run out, infinities, views that share memory, fp32 outputs.

Tolerances as in test_gpu_layer.py, whose helpers these tests use, or where they stand."""
import ctypes as C
import math

import pytest
import torch

from oracle import hpu_oracle as O
from test_gpu_layer import BF16, E4M3, E5M2, EPS, F32, FLOOR, HALF_STEP, _check_lora, _check_moe, _close, _cu, _lora_case, _moe_case, _randn, _run_lora, _run_moe, _status  # noqa: F401

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------- waits that run out
def _moe_args(case, top_k, out_dtype=BF16, plain=0):
    """The C ABI's arguments, and what has to stay alive: out, weights, ids, and the rest."""
    from b200_hpu_ops import abi
    x, r, gu, down, s1, s2 = d = [_cu(t) for t in case]
    tokens, hidden, experts, inner = x.shape[0], x.shape[1], r.shape[0], down.shape[2]
    out, weights = torch.zeros(tokens, hidden, dtype=out_dtype, device="cuda"), torch.zeros(tokens, top_k, device="cuda")
    ids = torch.full((tokens, top_k), 0x7FFF, dtype=torch.int32, device="cuda")
    n = abi.lib.b200q_moe_workspace_bytes(tokens, hidden, inner, experts, top_k)
    ws = torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda")
    a = abi.MoeArgs(x=x.data_ptr(), x_stride=hidden, tokens=tokens, hidden=hidden, inner=inner, experts=experts, top_k=top_k, renormalize=1, router=r.data_ptr(),
                    router_dtype=abi.DTYPE[r.dtype], gate_up=gu.data_ptr(), down=down.data_ptr(), weight_dtype=abi.DTYPE[gu.dtype],
                    gate_up_scale=None if s1 is None else s1.data_ptr(), down_scale=None if s2 is None else s2.data_ptr(), out=out.data_ptr(), out_dtype=abi.DTYPE[out_dtype],
                    weights=weights.data_ptr(), ids=ids.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=n, force_plain=plain, stream=abi.stream_ptr())
    return a, out, weights, ids, (d, ws)


@pytest.mark.parametrize("lost", [0, 1, 2, 3])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(45, 256, 128, 16, 2), (200, 4352, 160, 6, 3)])
def test_moe_that_waits_in_vain(tokens, hidden, inner, experts, top_k, lost):
    """The wait runs out (no GPU fault), the status says so, nothing finite is left in out, and the next call is as it should be."""
    import b200_hpu_ops
    from b200_hpu_ops import abi
    case = _moe_case(tokens, hidden, inner, experts, E4M3)
    want = [t.cpu() for t in _run_moe(case, top_k)]
    _check_moe(want, case, top_k)
    for _ in range(2):
        a, out, weights, ids, held = _moe_args(case, top_k)
        abi.check(abi.lib.b200q_selftest_moe_wait_timeout(C.byref(a), lost))
        code = b200_hpu_ops.device_status()
        assert code == 825 if lost < 2 else 821 <= code <= 825
        assert bool(out.isnan().all())
        assert torch.equal(weights.cpu(), want[1]) and torch.equal(ids.cpu(), want[2])  # (these are there before anything is waited for)
        for got, w in zip(_run_moe(case, top_k), want):
            assert torch.equal(got.cpu(), w)
    assert b200_hpu_ops.device_status() == 0


def _lora_args(y, x, a, b, which, scales, plain=0):
    from b200_hpu_ops import abi
    d = [_cu(t) for t in (y.clone(), x, a, b, which, scales)]
    (tokens, n), k, adapters, rank = y.shape, x.shape[1], a.shape[0], a.shape[1]
    size = abi.lib.b200q_lora_workspace_bytes(tokens, k, n, rank, adapters)
    ws = torch.full((size,), 0x3F, dtype=torch.uint8, device="cuda")  # (as fp32: finite)
    args = abi.LoraArgs(x=d[1].data_ptr(), x_stride=k, y=d[0].data_ptr(), y_dtype=abi.DTYPE[y.dtype], y_stride=n, a=d[2].data_ptr(), b=d[3].data_ptr(), a_stride=rank * k, a_row_stride=k,
                        b_stride=n * rank, b_row_stride=rank, adapter=d[4].data_ptr(), scales=None if scales is None else d[5].data_ptr(), tokens=tokens, k=k, n=n, rank=rank,
                        adapters=adapters, workspace=ws.data_ptr(), workspace_bytes=size, force_plain=plain, stream=abi.stream_ptr())
    return args, d[0], (d, ws)


@pytest.mark.parametrize("lost", [0, 1])
@pytest.mark.parametrize("tokens,k,n,rank,adapters", [(1, 256, 128, 16, 1), (40, 4104, 520, 32, 5), (300, 520, 264, 16, 40), (6000, 264, 136, 16, 1900)])
def test_lora_that_waits_in_vain(tokens, k, n, rank, adapters, lost):
    """A copy never comes: the wait runs out (no GPU fault), the status says so, a value of y that missed something is NaN or as it was, the others have an undisturbed
    call's bytes, and the next call is as it should be."""
    import b200_hpu_ops
    from b200_hpu_ops import abi
    c = _lora_case(tokens, k, n, rank, adapters, BF16, which=torch.arange(tokens) % (adapters + 1))
    y, which = c[0], c[4]
    want = _run_lora(*c).cpu()
    _check_lora(want, *c)
    for _ in range(2):
        a, got, held = _lora_args(*c)
        abi.check(abi.lib.b200q_selftest_lora_wait_timeout(C.byref(a), lost))
        assert 831 <= b200_hpu_ops.device_status() <= 833
        got = got.cpu()
        missed = got.isnan() if lost == 0 else (got != want) & (got == y)
        assert torch.equal(got[~missed], want[~missed])
        rows = missed.any(-1)
        assert bool(rows.any()) and bool((which[rows] < adapters).all()) and (tokens == 1 or not bool(rows[which < adapters].all()))
        if lost == 0:
            assert torch.equal(missed.all(-1), rows)
        assert torch.equal(_run_lora(*c).cpu(), want)
    assert b200_hpu_ops.device_status() == 0


@pytest.mark.parametrize("tokens,dim,residual", [(149, 4104, True), (1300, 8192, True), (1300, 5000, False)])
def test_norm_that_waits_in_vain(tokens, dim, residual):
    """The first row never comes: the wait runs out (no GPU fault), the status says so, that row and those behind it of its block are not written, the others have an
    undisturbed call's bytes, and the next call is as it should be."""
    import b200_hpu_ops
    from b200_hpu_ops import abi
    g = torch.Generator(device="cuda").manual_seed(dim)
    x, r = (torch.randn(tokens, dim, generator=g, device="cuda").to(BF16) for _ in range(2))
    run = lambda res: torch.ops.b200q.add_rms_norm_cast(x, res if residual else None, None, EPS, E4M3, None, True)  # noqa: E731
    after = r.clone()
    want = [*run(after), after]
    mine = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    mine[::2 * 148] = True  # block 0's rows
    for _ in range(2):
        got = [torch.full((tokens, dim), 2.0, device="cuda").to(E4M3), torch.full((tokens, 1), 2.0, device="cuda"), torch.full((tokens, dim), 2.0, device="cuda", dtype=BF16), r.clone()]
        before = [t.clone() for t in got]
        a = abi.NormArgs(x=x.data_ptr(), x_dtype=abi.BF16, tokens=tokens, dim=dim, x_stride=dim, residual=got[3].data_ptr() if residual else None, residual_stride=dim, eps=EPS,
                         out=got[0].data_ptr(), out_dtype=abi.E4M3, scale_inv=got[1].data_ptr(), kept=got[2].data_ptr(), stream=abi.stream_ptr())
        abi.check(abi.lib.b200q_selftest_norm_wait_timeout(C.byref(a)))
        assert b200_hpu_ops.device_status() == 811
        for t, b, w in zip(got, before, want):
            t, b, w = t.float(), b.float(), w.float()
            assert torch.equal(t[mine], b[mine]) and torch.equal(t[~mine], w[~mine])
        after = r.clone()
        assert all(torch.equal(t.float(), w.float()) for t, w in zip([*run(after), after], want))
    assert b200_hpu_ops.device_status() == 0


# ----------------------------------------------------------------------------- infinities
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens,k,n,rank", [(9, 64, 72, 16), (200, 264, 136, 72), (9, 60, 71, 12), (200, 61, 72, 3)])
def test_lora_infinities(tokens, k, n, rank, dtype):
    """Infinities of x and a, by tensor-core kernels (the first two sizes) and plain ones: what products and sums make of them, in either; and a x behind the end of bf16, but not of fp32."""
    y, x, a, b, which, scales = _lora_case(tokens, k, n, rank, 3, dtype, which=torch.arange(tokens) % 3)
    a, b = a.abs() + 2.0 ** -10, b.abs() + 2.0 ** -10  # (no zeros)
    a[2, 1, 5] = math.inf   # one rank of an adapter
    b[0, 7] = 0             # a column that an infinity meets with zeros
    x[:, 5] = x[:, 5].abs() + 1
    x[0, 3], x[3, k - 1], x[4, 3], x[6, 3], x[6, 4] = math.inf, -math.inf, math.inf, math.inf, -math.inf
    x[7] = 0
    x[7, 0] = 3.3e38
    a[1, :, 0], b[1, :, :] = 1.0234375, 2.0 ** -12  # 3.377e38, and with the scale below as much as fp32 holds
    scales[1] = 1.0058
    want, size, live = O.lora_add(y, x, a, b, which, scales)
    assert bool(want[0, :7].isposinf().all()) and bool(want[0, 7].isnan()) and bool(want[3, 0].isneginf()) and bool(want[4].isposinf().all()) and bool(want[6].isnan().all())
    assert bool(want[2].isposinf().all()) and 3.3895313892515355e38 < float((a[1].double() @ x[7].double() * scales[1]).max()) < 3.4e38 and bool(want[7].isfinite().all())
    got = _run_lora(y, x, a, b, which, scales).cpu().float()
    finite = want.isfinite()
    assert torch.equal(got[~finite].nan_to_num(nan=7.0), want[~finite].float().nan_to_num(nan=7.0))
    tol = (HALF_STEP[dtype] * (1 + 2.0 ** -10)) * want.abs() + size * (((k + rank) / 16 + 32) * 2.0 ** -23 + 2.0 ** -16) + FLOOR[dtype]
    _close(torch.where(finite, got, 0.0), torch.where(finite, want, 0.0), torch.where(finite, tol, 0.0))


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("hidden,inner", [(64, 32), (272, 160), (60, 33)])
@pytest.mark.parametrize("tokens", [6, 12])
def test_moe_h_at_the_end_of_fp32(tokens, hidden, inner, weights):
    """An h of 3.397e38, which bf16 has no finite value for, and one beyond fp32: that makes its token NaN, by tensor-core kernels (the first two sizes) and plain ones alike."""
    x, r, gu, down, s1, s2 = _moe_case(tokens, hidden, inner, 2, weights)
    gu, down = torch.zeros(gu.shape), torch.full(down.shape, 2.0 ** -6).to(weights)
    gu[:, 1, 0] = gu[:, inner + 1, 0] = 1.0  # of unit 1 alone: g = 8 x[0], u = 31.95 x[0]
    s1, s2 = torch.ones_like(s1), torch.full_like(s2, 2.0 ** -13)
    s1[:, 1], s1[:, inner + 1] = 8.0, 31.95
    x[:, 0] = x[:, 0].abs() + 1
    x[2, 0], x[4, 0] = 2.0 ** 60, 2.0 ** 64
    assert 3.3895313892515355e38 < 2.0 ** 123 * float(s1[0, inner + 1]) < 3.402e38
    case = (x, r, gu.to(weights), down, s1, s2)
    w, i = O.moe_route(x, r, 1, True)
    want, bound = O.moe_experts(x, w, i, *case[2:], rel_sum=40 * 2.0 ** -23, rel_hidden=2.0 ** -12, abs_hidden=2.0 ** -26)
    want[4], bound[4] = math.nan, 0
    out, weights_of, ids = _run_moe(case, 1)
    assert torch.equal(ids.cpu(), i) and bool((weights_of == 1).all())
    _close(out.float(), want, HALF_STEP[BF16] * (1 + 2.0 ** -10) * want.abs() + bound + FLOOR[BF16])


# ----------------------------------------------------------------------------- fp32 outputs of the experts
@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,inner", [(8, 1792), (30, 1792), (70, 4352), (5, 4352)])
def test_moe_fp32_h(tokens, inner, weights):
    """h is the same in all units of a token, so that what its terms drop adds up.  h itself: g and u one rounding each, 2^-24, expf, addition, division and two products, below
    2^-21 where g is positive; its terms 2^-24.  The second sum is of one sign: 256 products at a time inside the tensor core, 9.5 * 2^-23 (as test_lora_fp32_sums has it), a tenth
    more for the terms behind the first, inner / 256 additions of 2^-24, and three products: below 25 * 2^-23 for 4352 units, all together below 2^-18."""
    hidden = 256
    x, r, gu, down, s1, s2 = _moe_case(tokens, hidden, inner, 1, weights)
    x[:, 1:], x[:, 0] = 0, x[:, 0].abs() + 0.5
    gu, down = torch.ones(gu.shape).to(weights), torch.ones(down.shape).to(weights)
    s1, s2 = torch.full_like(s1, 1 / 3), torch.full_like(s2, 1 / 7)
    case = (x, r, gu, down, s1, s2)
    want, _ = O.moe_experts(x, torch.ones(tokens, 1), torch.zeros(tokens, 1, dtype=torch.int32), gu, down, s1, s2)
    out, _, _ = _run_moe(case, 1, dtype=F32)
    _close(out, want, 2.0 ** -18 * want)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden", [(8, 8192), (40, 8192), (20, 2176)])
def test_moe_fp32_sums(tokens, hidden, weights):
    """Sums of one sign over hidden.  g and u are off by (9.5 + 1) * 2^-23 + hidden / 256 * 2^-24, below 28 * 2^-23, and with what follows as above: silu makes at most 1.3 of
    it, that is 2.3 * 28 * 2^-23 in h, and 2^-19 behind: below 2^-16."""
    x, r, gu, down, s1, s2 = _moe_case(tokens, hidden, 64, 2, weights)
    x, gu, down = x.abs(), gu.float().abs().to(weights), down.float().abs().to(weights)
    s1 = s1 * (3 * hidden ** -0.5)
    case = (x, r, gu, down, s1, s2)
    w, i = O.moe_route(x, r, 1, True)
    want, _ = O.moe_experts(x, w, i, gu, down, s1, s2)
    out, _, ids = _run_moe(case, 1, dtype=F32)
    assert torch.equal(ids.cpu(), i)
    _close(out, want, 2.0 ** -16 * want)


@pytest.mark.parametrize("weights", [E4M3, BF16])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(7, 512, 272, 16, 8), (45, 4352, 160, 6, 2), (256, 128, 96, 20, 4), (256, 64, 32, 129, 16), (20, 160, 4400, 40, 8), (300, 272, 144, 512, 16)])
def test_moe_fp32(tokens, hidden, inner, experts, top_k, weights):
    """Against the oracle with h to 2^-23 of itself and 2^-40 of the largest of its token and expert, where outputs in bf16 have 2^-12 and 2^-26."""
    case = _moe_case(tokens, hidden, inner, experts, weights)
    out, weights_of, ids = _run_moe(case, top_k, dtype=F32)
    w, i = O.moe_route(case[0], case[1], top_k, True)
    assert torch.equal(ids.cpu(), i)
    n = max(hidden, inner)
    want, bound = O.moe_experts(case[0], w, i, *case[2:], rel_sum=(min(n, 256) / 16 + n / 256 + 16) * 2.0 ** -23, rel_hidden=2.0 ** -23, abs_hidden=2.0 ** -40)
    _close(out, want, 2.0 ** -22 * want.abs() + bound + FLOOR[F32])


# ----------------------------------------------------------------------------- memory that is shared
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lora_in_one_allocation(dtype):
    """All of a call's tensors as parts of one allocation, as a program that divides up its memory itself has them."""
    y, x, a, b, which, scales = c = _lora_case(40, 64, 72, 16, 3, dtype)
    pool, at = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"), 0

    def place(t):
        nonlocal at
        part = pool[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
        at += -(-part.numel() * part.element_size() // 256) * 256
        return part.copy_(t)

    ad, sd, xd, yd, bd, wd = (place(t) for t in (a, scales, x, y, b, which))
    torch.ops.b200q.lora_add_(yd, xd, ad, bd, wd, sd)
    _check_lora(yd, *c)
    wide = torch.zeros(40, 512, dtype=torch.uint8, device="cuda")  # y beside x in the rows of one buffer
    ys, xs = wide[:, :72 * y.element_size()].view(dtype), wide[:, 384:512].view(BF16)
    ys.copy_(y)
    xs.copy_(x)
    torch.ops.b200q.lora_add_(ys, xs, ad, bd, wd, sd)
    _check_lora(ys, *c)


def test_lora_refuses_to_write_its_inputs():
    y, x, a, b, which, scales = (t.cuda() for t in _lora_case(4, 64, 32, 8, 2, F32))
    op = torch.ops.b200q.lora_add_
    for args in [(y, x, a, b, y.view(torch.int32)[1, 3:7]), (y, x, a, b, which, y[3, 30:]), (a.view(-1).view(F32)[:128].view(4, 32), x, a, b, which), (b.view(-1).view(F32)[128:256].view(4, 32), x, a, b, which)]:
        with pytest.raises(RuntimeError, match="must not overlap"):
            op(*args)


def test_norm_refuses_to_write_its_inputs():
    x, r = torch.ones(4, 64, dtype=BF16, device="cuda"), torch.ones(4, 64, dtype=BF16, device="cuda")
    op = torch.ops.b200q.add_rms_norm_cast
    for weight, scale in [(r[1], None), (r.view(F32).view(-1)[10:74], None), (None, r.view(F32)[3, 5])]:
        with pytest.raises(RuntimeError, match="must not overlap weight or scale"):
            op(x, r, weight, EPS, BF16, scale)
    both = torch.ones(6, 64, dtype=BF16, device="cuda")  # one allocation
    op(x, both[:4], both[4], EPS, BF16, both[5].view(F32)[7])
    assert bool((both[:4] == 2).all()) and bool((both[4:] == 1).all())


@pytest.mark.parametrize("dim,step", [(525, 5), (521, 1), (1000, 8), (8189, 5), (261, 5)])
def test_norm_rows_that_overlap(dim, step):
    """Windows of one long row, up to its end."""
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn(400 * step + dim, generator=g, device="cuda").to(BF16).as_strided((401, dim), (step, 1))
    _, y = O.add_rms_norm(x, None, None, EPS)
    out, inv, kept = torch.ops.b200q.add_rms_norm_cast(x, None, None, EPS, E4M3, None, True)
    top = y.abs().amax(-1, keepdim=True)
    v = y * (448.0 / top)
    _close(inv, (top / 448.0).cpu(), 2.0 ** -16 * (top / 448.0).cpu())
    _close(out.float(), v.cpu(), ((HALF_STEP[E4M3] + 2.0 ** -16) * v.abs() + FLOOR[E4M3]).cpu())
    _close(kept.float(), y.cpu(), ((HALF_STEP[BF16] + 2.0 ** -17) * y.abs() + FLOOR[BF16]).cpu())
