"""The paged key/value cache on the GPU (plan of a step, append, attention of one new token) against the oracle in 64 bits.

Tolerances.  A value that is rounded once to a type is off by at most half a step of it (bf16 2^-8, e4m3 2^-4, e5m2 2^-3 relative;
below the smallest normal half of 2^-9 and 2^-16).  On top of that comes the arithmetic in fp32: a head's norm is a sum of
at most 256 squares (2^-24 each, in a tree: below 2^-20), the rotation adds two products: 2^-20 of the head's largest value in all.
Attention: probabilities are rounded to 11 bits or more before the product with the values (2^-12 of sum p |v|, here 2^-11), a score's
sum of up to 256 products is off by at most 2^-15 in these inputs (sum of |products| below 2^7, 2^-22 of it), which changes p by as
much, twice with the normalisation; sums over a thousand keys in fp32 2^-14: 2^-11 + 2^-13 of sum p |v| holds them all."""
import ctypes as C
import math

import pytest
import torch

from oracle import hpu_oracle as O

pytestmark = pytest.mark.gpu
E4M3, E5M2, BF16, F32 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24, E4M3: 2.0 ** -4, E5M2: 2.0 ** -3}
FLOOR = {BF16: 0.0, F32: 0.0, E4M3: 2.0 ** -10, E5M2: 2.0 ** -17}
LIMIT = {BF16: math.inf, F32: math.inf, E4M3: 448.0, E5M2: 57344.0}


@pytest.fixture(autouse=True)
def _status():
    import b200_hpu_ops
    yield
    assert b200_hpu_ops.device_status() == 0


def _cu(t):
    return None if t is None else t.cuda()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32)


def _one(v):
    return torch.tensor([v], dtype=F32)


def _close(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    off = torch.where(got == want, 0.0, (got - want).abs()) - tol  # (equal infinities are no distance)
    off = off[~want.isnan()]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max()):.3g} beyond the tolerance"


# ----------------------------------------------------------------------------- plan
def _plan_case(requests, context, new, page, width, spare, seed, padded=3, head=None):
    g = torch.Generator().manual_seed(seed)
    ctx = torch.randint(-1, context + 1, (requests,), generator=g, dtype=torch.int32)
    add = torch.randint(-1, new + 1, (requests,), generator=g, dtype=torch.int32)
    table = torch.randint(0, 1 << 20, (requests, width), generator=g, dtype=torch.int32)
    need = sum(max(0, -(-(max(c, 0) + max(n, 0)) // page) - -(-max(c, 0) // page)) for c, n in zip(ctx.tolist(), add.tolist()))
    free = torch.randperm(1 << 16, generator=g)[:max(0, need + spare + (head or 0))].to(torch.int32)
    tokens = max(0, int(add.clamp(min=0).sum()) + padded)
    return ctx, add, table, free, None if head is None else _i32([head]), page, tokens


def _plan_check(case):
    ctx, add, table, free, head, page, tokens = case
    want = O.paged_plan(ctx, add, table, free, head, page, tokens)
    dev = table.cuda()
    got = torch.ops.b200q.paged_plan(ctx.cuda(), add.cuda(), dev, free.cuda(), _cu(head), page, tokens)
    for name, x, y in zip(("slot_map", "positions", "query_start", "kv_lens", "free_head", "block_table"), (*got, dev), want):
        assert x.dtype == y.dtype and torch.equal(x.cpu(), y), name


@pytest.mark.parametrize("requests,context,new,page,width", [
    (1, 0, 1, 16, 1), (1, 100, 1, 16, 8), (3, 0, 40, 16, 4), (7, 50, 1, 1, 60), (33, 300, 77, 7, 60), (256, 500, 1, 16, 40), (257, 100, 30, 64, 4),
    (1000, 64, 9, 32, 5), (8192, 20, 2, 16, 3), (2, 5000, 9000, 128, 120)])
@pytest.mark.parametrize("spare,padded,head", [(0, 0, None), (5, 700, 3), (-4, -2, 0)])
def test_plan(requests, context, new, page, width, spare, padded, head):
    _plan_check(_plan_case(requests, context, new, page, width, spare, requests + spare, padded, head))


def test_plan_of_nothing_and_of_narrow_tables():
    empty = torch.empty(0, dtype=torch.int32)
    _plan_check((empty, empty, torch.empty(0, 4, dtype=torch.int32), empty, _i32([5]), 16, 3))
    _plan_check((_i32([4, 9]), _i32([2, 3]), torch.empty(2, 0, dtype=torch.int32), _i32([1, 2]), None, 4, 5))   # no table at all
    _plan_check((_i32([15, 33]), _i32([40, 3]), torch.full((2, 2), 6, dtype=torch.int32), _i32([1, 2]), None, 16, 43))  # rows that end too early
    _plan_check((_i32([3]), _i32([2]), _i32([[8, -1]]), empty, None, 4, 2))                                        # no free page


def test_plan_lengths_near_the_type():
    """Lengths whose sums pass 31 bits: the sums saturate, nothing is written outside the outputs."""
    ctx, add = _i32([2 ** 31 - 1, 5, 7]), _i32([2 ** 31 - 1, 3, 2 ** 31 - 1])
    table = _i32([[3, 4], [5, 6], [8, 9]]).cuda()
    slots, pos, start, lens, head = torch.ops.b200q.paged_plan(ctx.cuda(), add.cuda(), table, _i32([1]).cuda(), _i32([-9]).cuda(), 16, 6)
    assert slots.tolist() == [-1] * 6 and pos.tolist() == [2 ** 31 - 1 + i for i in range(6)]
    assert start.tolist() == [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1] and lens.tolist() == [2 ** 31 - 1, 8, 2 ** 31 - 1]
    assert head.tolist() == [1] and table.tolist() == [[3, 4], [5, 6], [8, 1]]


def test_plan_is_repeatable_and_keeps_strided_rows():
    ctx, add, table, free, head, page, tokens = _plan_case(20, 90, 30, 16, 9, 3, 5)
    whole = torch.full((20, 13), 77, dtype=torch.int32).cuda()
    view = whole[:, 2:11]
    view.copy_(table)
    args = (ctx.cuda(), add.cuda(), view, free.cuda(), None, page, tokens)
    first = [t.clone() for t in torch.ops.b200q.paged_plan(*args)]
    again = torch.ops.b200q.paged_plan(*args)
    want = O.paged_plan(ctx, add, table, free, head, page, tokens)
    for x, y, z in zip(first, again, want):
        assert torch.equal(x, y) and torch.equal(x.cpu(), z)
    assert torch.equal(view.cpu(), want[5]) and int((whole[:, :2] != 77).sum() + (whole[:, 11:] != 77).sum()) == 0


def test_plan_refusals():
    z, t = torch.zeros(2, dtype=torch.int32).cuda(), torch.zeros(2, 4, dtype=torch.int32).cuda()
    plan = torch.ops.b200q.paged_plan
    for bad in ((z.long(), z, t, z, None, 16, 1), (z, z.float(), t, z, None, 16, 1), (z, z, t.long(), z, None, 16, 1), (z, z, t, z.long(), None, 16, 1),
                (z, z, t, z, z, 16, 1), (z, z, t, z, None, 0, 1), (z, z, t, z, None, 16, -1), (z[:1], z, t, z, None, 16, 1), (z, z, t[:1], z, None, 16, 1),
                (z, z, t.t().contiguous().t(), z, None, 16, 1), (z, z, t[:1].expand(2, 4), z, None, 16, 1), (z.reshape(1, 2), z, t, z, None, 16, 1),
                (z, z.cpu(), t, z, None, 16, 1)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            plan(*bad)


# ----------------------------------------------------------------------------- append
def _table(rot, positions=600):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _append_check(tokens, heads, kv, dim, rot, interleaved, norm, src, cache, q_dtype, page, seed=0, w_dtype=BF16, layout="packed", skip=2, extra=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=g).to(src)
    if extra is not None:
        extra(qkv)
    qw, kw = (torch.randn(dim, generator=g).to(w_dtype) for _ in range(2)) if norm else (None, None)
    cos_sin = _table(rot) if rot else None
    positions = torch.randint(0, 600, (tokens,), generator=g)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[:min(skip, tokens)] = torch.tensor([-1, pages * page, -5])[:min(skip, tokens)]
    fp8 = cache != BF16
    ks, vs, qs = (30.0, 50.0, 40.0 if q_dtype in (E4M3, E5M2) else None) if fp8 else (None, None, None)
    if layout == "packed":
        dev = qkv.cuda()
        q, k, v = dev[:, :heads], dev[:, heads:heads + kv], dev[:, heads + kv:]
    elif layout == "heads first":  # [heads, tokens, dim] tensors
        q, k, v = (t.transpose(0, 1).contiguous().cuda().transpose(0, 1) for t in (qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]))
    else:  # rows that start at no multiple of four values
        wide = torch.zeros(tokens, heads + 2 * kv, dim + 3, dtype=src).cuda()
        wide[..., 1:dim + 1] = qkv.cuda()
        q, k, v = (t[..., 1:dim + 1] for t in (wide[:, :heads], wide[:, heads:heads + kv], wide[:, heads + kv:]))
    before = (torch.randn(2, pages, page, kv, dim, generator=g) * 8).to(cache)
    if layout == "heads first":
        caches = before.transpose(2, 3).contiguous().cuda().transpose(2, 3)
    else:
        caches = before.cuda()
    kc, vc = caches[0], caches[1]
    got = torch.ops.b200q.qk_norm_rope_append(q, k, v, _cu(qw), _cu(kw), 1e-5, _cu(cos_sin), _cu(positions) if rot else None, interleaved, slots.cuda(), kc, vc,
                                              None if ks is None else _one(ks).cuda(), None if vs is None else _one(vs).cuda(),
                                              None if qs is None else _one(qs).cuda(), q_dtype)
    assert got.dtype == q_dtype and got.is_contiguous()

    def rounded(x, y, scale, dtype):  # y: fp64, before the rounding
        y = y * (scale or 1.0)
        top = torch.where(y.isfinite(), y.abs(), 0.0).amax(-1, keepdim=True)
        want = y.clamp(-LIMIT[dtype], LIMIT[dtype])
        _close(x.float(), want, HALF_STEP[dtype] * want.abs().nan_to_num() + FLOOR[dtype] + 2.0 ** -20 * top)

    rounded(got, O.norm_rope(qkv[:, :heads], qw, 1e-5, cos_sin, positions, interleaved), qs, q_dtype)
    kept = (slots >= 0) & (slots < pages * page)
    for new, old, x, scale in ((kc, before[0], O.norm_rope(qkv[:, heads:heads + kv], kw, 1e-5, cos_sin, positions, interleaved), ks),
                               (vc, before[1], qkv[:, heads + kv:].double(), vs)):
        new = new.cpu().reshape(-1, kv, dim)
        rounded(new[slots[kept]], x[kept], scale, cache)
        rest = torch.ones(pages * page, dtype=torch.bool)
        rest[slots[kept]] = False
        as_bytes = (lambda t: t.view(torch.int16)) if cache == BF16 else (lambda t: t.view(torch.uint8))  # noqa: E731
        assert torch.equal(as_bytes(new)[rest], as_bytes(old.reshape(-1, kv, dim))[rest]), "a slot that no token has was written"


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,interleaved,norm,page", [
    (1, 8, 1, 128, 128, False, True, 16), (1, 1, 1, 8, 8, True, True, 1), (5, 7, 3, 64, 32, True, False, 16), (33, 64, 8, 128, 128, False, True, 16),
    (17, 16, 2, 256, 256, False, True, 64), (9, 6, 2, 80, 24, False, True, 5), (3, 5, 5, 248, 0, False, True, 16), (130, 4, 4, 96, 96, True, True, 32),
    (700, 9, 1, 64, 64, False, True, 128), (2, 40, 40, 128, 64, False, False, 16)])
@pytest.mark.parametrize("src,cache,q_dtype", [(BF16, E4M3, BF16), (BF16, BF16, BF16), (F32, E4M3, E4M3), (F32, E5M2, E5M2), (F32, BF16, E4M3)])
def test_append(tokens, heads, kv, dim, rot, interleaved, norm, page, src, cache, q_dtype):
    _append_check(tokens, heads, kv, dim, rot, interleaved, norm, src, cache, q_dtype, page, seed=tokens + dim)


@pytest.mark.parametrize("layout", ["heads first", "odd"])
@pytest.mark.parametrize("src,cache", [(BF16, E4M3), (F32, BF16)])
def test_append_layouts(layout, src, cache):
    _append_check(37, 8, 2, 128, 128, False, True, src, cache, BF16, 16, layout=layout, w_dtype=F32)


def test_append_many_tokens():
    _append_check(3001, 10, 2, 128, 128, False, True, BF16, E4M3, BF16, 16, skip=3)


def test_append_infinities_and_nan():
    """Without a norm a NaN spoils the pair that it turns with and nothing else; values saturate in an fp8 cache."""
    def spoil(x):
        x[3, 1, 5] = x[5, 8, 0] = x[7, 10, 2] = math.nan
        x[8, 10, 3], x[9, 11, 4] = math.inf, -math.inf
    _append_check(12, 8, 2, 64, 64, False, False, BF16, E4M3, BF16, 16, extra=spoil)


def test_append_extreme_sizes_of_values():
    def sizes(x):
        x[0] *= 1e18
        x[1] *= 1e-18
        x[2] = 0.0
    _append_check(8, 4, 2, 128, 128, False, True, F32, E4M3, BF16, 16, extra=sizes, skip=0)


def test_append_positions_outside_the_table():
    x = torch.randn(4, 3, 64).to(BF16).cuda()
    kc, vc = torch.zeros(2, 1, 16, 1, 64, dtype=BF16).cuda()
    pos = torch.tensor([0, 600, -1, 599]).cuda()
    q = torch.ops.b200q.qk_norm_rope_append(x[:, :1], x[:, 1:2], x[:, 2:], None, None, 1e-6, _table(32).cuda(), pos, False, torch.arange(4).cuda(), kc, vc)
    for t in (q, kc[0, :4]):
        assert t[1, :, :32].isnan().all() and t[2, :, :32].isnan().all() and t[1:3, :, 32:].isfinite().all() and t[[0, 3]].isfinite().all()
    assert torch.equal(vc[0, :4], x[:, 2:])


def test_append_of_nothing():
    kc, vc = torch.ones(2, 2, 16, 2, 64, dtype=BF16).cuda()
    e = torch.empty(0, 6, 64, dtype=BF16).cuda()
    none = torch.empty(0, dtype=torch.int64).cuda()
    assert torch.ops.b200q.qk_norm_rope_append(e[:, :2], e[:, 2:4], e[:, 4:], None, None, 1e-6, _table(64).cuda(), none, False, none, kc, vc).shape == (0, 2, 64)
    x = torch.randn(3, 6, 64).to(BF16).cuda()
    no_pages = torch.empty(0, 16, 2, 64, dtype=BF16).cuda()
    q = torch.ops.b200q.qk_norm_rope_append(x[:, :2], x[:, 2:4], x[:, 4:], None, None, 1e-6, None, None, False, torch.arange(3).cuda(), no_pages, no_pages.clone())
    assert torch.equal(q, x[:, :2]) and bool((kc == 1).all())


def test_append_offsets_beyond_32_bits():
    pages, page, kv, dim = 1100000, 16, 2, 128  # 4.5e9 elements in each cache
    kc, vc = (torch.empty(pages, page, kv, dim, dtype=E4M3, device="cuda") for _ in range(2))
    x = torch.randn(2, 6, dim).to(BF16).cuda()
    slots = torch.tensor([pages * page - 1, 7]).cuda()
    torch.ops.b200q.qk_norm_rope_append(x[:, :2], x[:, 2:4], x[:, 4:], None, None, 1e-6, None, None, False, slots, kc, vc)
    for cache, src in ((kc, x[:, 2:4]), (vc, x[:, 4:])):
        want = src.float().to(E4M3).view(torch.uint8)
        assert torch.equal(cache[-1, -1].view(torch.uint8), want[0]) and torch.equal(cache[0, 7].view(torch.uint8), want[1])


def test_append_refusals():
    x = torch.randn(4, 6, 64).to(BF16).cuda()
    q, k, v = x[:, :2], x[:, 2:4], x[:, 4:]
    kc, vc = torch.zeros(2, 2, 16, 2, 64, dtype=BF16).cuda()
    slots, t, w = torch.arange(4).cuda(), _table(64).cuda(), torch.ones(64, dtype=BF16).cuda()
    ok = dict(q=q, k=k, v=v, q_weight=w, k_weight=w, eps=1e-6, cos_sin=t, positions=slots, interleaved=False, slot_map=slots, k_cache=kc, v_cache=vc)
    torch.ops.b200q.qk_norm_rope_append(**ok)
    odd = torch.zeros(2, 16, 2, 65, dtype=BF16).cuda()[..., 1:]
    for bad in (dict(q=q.half()), dict(k=k.float()), dict(k=k[:3]), dict(v=v[:, :1]), dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), dict(q_weight=w[:32]),
                dict(q_weight=w.float()), dict(k_weight=w.half()), dict(cos_sin=t.bfloat16()), dict(cos_sin=_table(12).cuda()), dict(cos_sin=_table(128).cuda()),
                dict(positions=None), dict(positions=slots.int()), dict(positions=slots[:2]), dict(slot_map=slots.int()), dict(slot_map=slots[:2]),
                dict(k_cache=kc.float(), v_cache=vc.float()), dict(k_cache=kc.to(E4M3)), dict(k_cache=kc[:, :, :1], v_cache=vc[:, :, :1]),
                dict(k_cache=odd, v_cache=odd), dict(k_cache=kc[:1].expand(2, 16, 2, 64)), dict(v_cache=vc[:, :, :1].expand(2, 16, 2, 64)), dict(k_cache=kc.transpose(2, 3), v_cache=vc.transpose(2, 3)), dict(k_scale=torch.ones(2).cuda()),
                dict(k_scale=torch.ones(1)), dict(q_dtype=F32), dict(slot_map=slots.cpu())):
        with pytest.raises(RuntimeError):
            torch.ops.b200q.qk_norm_rope_append(**{**ok, **bad})


# ----------------------------------------------------------------------------- attention
class _Paged:
    """A cache of shuffled pages; everything that no request may look at is NaN."""

    def __init__(self, lens, kv, dim, cache, page, seed=0, spare=2, hnd=False, scale=1.0, width=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in lens]
        self.width = max(need + [0]) + 1 if width is None else width
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        data = torch.full((2, total, page, kv, dim), math.nan).to(cache)
        at = 0
        for b, n in enumerate(lens):
            own = order[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = own
            rows = (torch.randn(2, need[b] * page, kv, dim, generator=g) * scale).to(cache)
            rows[:, n:] = torch.full((2, need[b] * page - n, kv, dim), math.nan).to(cache)
            data[:, own.long()] = rows.reshape(2, need[b], page, kv, dim)
        self.k, self.v = data[0], data[1]
        dev = data.transpose(2, 3).contiguous().cuda().transpose(2, 3) if hnd else data.cuda()
        self.kd, self.vd = dev[0], dev[1]
        self.lens, self.g = _i32(lens), g


def _attend_check(lens, heads, kv, dim, cache, page, window=0, out_dtype=BF16, seed=0, hnd=False, q_std=2.0, paged=None, q=None, **kw):
    p = paged or _Paged(lens, kv, dim, cache, page, seed, hnd=hnd, **kw)
    fp8 = cache != BF16
    ks, vs = (0.75, 1.5) if fp8 else (1.0, 1.0)
    scale = 1.0 / math.sqrt(dim)
    if q is None:
        q = (torch.randn(len(lens), heads, dim, generator=p.g) * q_std).to(BF16)
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, scale, ks, vs, window)
    out_scale = 20.0 if out_dtype == E4M3 else None
    inv = (_one(ks).cuda(), _one(vs).cuda()) if fp8 else (None, None)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.kd, p.vd, p.table.cuda(), p.lens.cuda(), scale, *inv, window,
                                                   None if out_scale is None else _one(out_scale).cuda(), out_dtype)
    assert got.dtype == out_dtype
    s = out_scale or 1.0
    want = (want * s).clamp(-LIMIT[out_dtype], LIMIT[out_dtype])
    _close(got.float(), want, HALF_STEP[out_dtype] * want.abs() + FLOOR[out_dtype] + (2.0 ** -11 + 2.0 ** -13) * s * size)
    _close(got_lse, lse, 2.0 ** -13 + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), 0.0))
    return got, got_lse


LENS = [0, 1, 15, 16, 17, 33, 100, 257]


@pytest.mark.parametrize("cache", [E4M3, BF16, E5M2])
@pytest.mark.parametrize("heads,kv,dim,page", [(8, 1, 128, 16), (1, 1, 64, 16), (12, 4, 128, 48), (9, 1, 64, 32), (16, 1, 256, 16), (20, 1, 128, 64), (4, 4, 256, 128),
                                               (34, 2, 64, 16), (6, 2, 80, 16), (3, 1, 8, 4), (5, 5, 200, 7), (4, 2, 128, 1), (8, 2, 128, 24)])
def test_attention(cache, heads, kv, dim, page):
    _attend_check(LENS, heads, kv, dim, cache, page, seed=heads + dim)


@pytest.mark.parametrize("cache,out_dtype", [(E4M3, F32), (E4M3, E4M3), (BF16, F32), (BF16, E4M3), (E5M2, E4M3)])
@pytest.mark.parametrize("dim,page", [(128, 16), (72, 16)])
def test_attention_output_types(cache, out_dtype, dim, page):
    _attend_check(LENS, 8, 2, dim, cache, page, out_dtype=out_dtype)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 100, 5000])
@pytest.mark.parametrize("cache,dim,page", [(E4M3, 128, 16), (BF16, 64, 32), (BF16, 48, 5)])
def test_attention_window(window, cache, dim, page):
    _attend_check(LENS + [1000], 4, 2, dim, cache, page, window=window)


@pytest.mark.parametrize("cache,dim", [(E4M3, 128), (BF16, 128), (BF16, 256), (E4M3, 64)])
@pytest.mark.parametrize("lens", [[1], [3000], [20000, 5], [1, 1, 1, 900, 0, 0, 4097, 2], [37] * 150, [16] * 400])
def test_attention_lengths(lens, cache, dim):
    _attend_check(lens, 8, 1, dim, cache, 16, seed=len(lens))


@pytest.mark.parametrize("heads,kv,dim,cache,window", [(8, 8, 128, E4M3, 0), (64, 8, 64, BF16, 0), (80, 4, 128, E4M3, 0), (4, 4, 256, E4M3, 0), (16, 16, 64, E5M2, 33),
                                                       (24, 8, 128, BF16, 20)])
def test_attention_heads_side_by_side(heads, kv, dim, cache, window):
    """Rows enough for all warps: neighbouring heads go side by side, and rows are cut between CTAs in all places."""
    lens = [0, 1, 200, 15, 16, 17] + [(37 * i) % 150 for i in range(90)] + [0, 0, 333]
    _attend_check(lens, heads, kv, dim, cache, 16, window=window, seed=dim)


@pytest.mark.parametrize("heads,kv,dim,cache,lens", [(8, 8, 64, E4M3, [23000, 9000]), (8, 4, 128, BF16, [1, 0, 70000]), (3, 1, 64, BF16, [300000])])
def test_attention_long_rows(heads, kv, dim, cache, lens):
    """Rows that every CTA has a part of, with a warp's share above and below what puts heads side by side."""
    _attend_check(lens, heads, kv, dim, cache, 64)


@pytest.mark.parametrize("requests", [4096, 4097, 8192])
def test_attention_many_requests(requests):
    """Up to 4096 requests' lengths are kept on chip; 8192 is the most."""
    _attend_check([(i * 7) % 19 for i in range(requests)], 1, 1, 64, BF16, 16)


def test_attention_too_many_requests():
    q, kc = torch.zeros(8193, 1, 64, dtype=BF16).cuda(), torch.zeros(1, 16, 1, 64, dtype=BF16).cuda()
    with pytest.raises(RuntimeError, match="maximum"):
        torch.ops.b200q.paged_attention(q, kc, kc, torch.zeros(8193, 1, dtype=torch.int32).cuda(), torch.zeros(8193, dtype=torch.int32).cuda(), 1.0)


def test_attention_repeats_its_bytes():
    p = _Paged([5000, 1, 777, 2048, 64, 3000], 4, 128, E4M3, 16)
    q = torch.randn(6, 16, 128, generator=p.g).to(BF16).cuda()
    args = (q, p.kd, p.vd, p.table.cuda(), p.lens.cuda(), 0.1)
    first, first_lse = torch.ops.b200q.paged_attention(*args)
    for _ in range(20):
        out, lse = torch.ops.b200q.paged_attention(*args)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


@pytest.mark.parametrize("heads,kv", [(64, 8), (32, 32), (128, 1), (7, 7), (14, 2)])
@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_attention_heads(heads, kv, cache):
    _attend_check([700, 3, 129], heads, kv, 128, cache, 32)


@pytest.mark.parametrize("cache,dim", [(E4M3, 128), (BF16, 64), (E4M3, 40)])
def test_attention_layouts(cache, dim):
    """Heads before slots in the cache, keys and values as halves of one tensor, a q that is a slice, table rows with a pitch."""
    p = _Paged([100, 260, 31], 4, dim, cache, 16, hnd=True)
    q = torch.randn(3, 8, dim).to(BF16)
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, 0.2)
    both = torch.stack([p.k, p.v], 1).cuda()
    wide = torch.zeros(3, 11, dim + 5, dtype=BF16).cuda()
    wide[:, 2:10, 3:dim + 3] = q.cuda()
    table = torch.zeros(3, p.width + 9, dtype=torch.int32).cuda()
    table[:, 4:4 + p.width] = p.table.cuda()
    for kc, vc in ((p.kd, p.vd), (both[:, 0], both[:, 1])):
        for qq in (q.cuda(), wide[:, 2:10, 3:dim + 3], q.transpose(0, 1).contiguous().cuda().transpose(0, 1)):
            got, got_lse = torch.ops.b200q.paged_attention(qq, kc, vc, table[:, 4:4 + p.width], p.lens.cuda(), 0.2)
            _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
            _close(got_lse, lse, 2.0 ** -13 + 2.0 ** -22 * lse.abs())


@pytest.mark.parametrize("cache,dim", [(E4M3, 128), (BF16, 128), (BF16, 24)])
def test_attention_pages_that_do_not_exist(cache, dim):
    """Entries outside the cache are keys that do not exist; lengths beyond the table end with it; negative lengths are empty."""
    p = _Paged([100, 64, 33, 200, 5], 2, dim, cache, 16)
    p.table[0, 2], p.table[1, :] = -1, 1 << 30
    p.table[2, 0], p.table[3, 12] = p.k.shape[0], -2147483648
    p.lens = _i32([100, 64, 33, 2147483647, -7])
    p.table = p.table[:, :13].clone()
    _attend_check([0] * 5, 4, 2, dim, cache, 16, paged=p)


@pytest.mark.parametrize("cache,dim", [(E4M3, 128), (BF16, 64), (E4M3, 72)])
def test_attention_is_not_finite_where_its_row_is_not(cache, dim):
    p = _Paged([50, 300, 20], 2, dim, cache, 16)
    spot = p.table[1, 17], 3
    for t, d in ((p.k, p.kd), (p.v, p.vd)):
        row = torch.full((dim,), math.nan).to(cache)
        t[spot[0], spot[1], 0] = row
        d[spot[0], spot[1], 0] = row.cuda()
    q = torch.randn(3, 4, dim).to(BF16)
    out, lse = torch.ops.b200q.paged_attention(q.cuda(), p.kd, p.vd, p.table.cuda(), p.lens.cuda(), 0.1)
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[1, :2] = True
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad) and torch.equal(lse.isnan().cpu(), bad)


@pytest.mark.parametrize("cache,dim", [(E4M3, 128), (BF16, 128)])
@pytest.mark.parametrize("q_std", [1e-30, 1e-3, 30.0, 1e4])
def test_attention_scores_of_all_sizes(cache, dim, q_std):
    """From flat rows to ones where a single key has everything; the scale keeps the scores in range."""
    p = _Paged([500, 40, 1], 2, dim, cache, 16, spare=3)
    q = (torch.randn(3, 4, dim, generator=p.g) * q_std).to(BF16)
    scale = 1.0 / math.sqrt(dim) / max(1.0, q_std / 4)
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, scale)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.kd, p.vd, p.table.cuda(), p.lens.cuda(), scale)
    _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
    _close(got_lse, lse, 2.0 ** -13 + 2.0 ** -22 * lse.abs())


@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_attention_rising_scores(cache):
    """Scores that rise along the cache: the running maximum moves at every step."""
    p = _Paged([1500], 1, 128, cache, 16)
    ramp = torch.linspace(-3, 3, 1500)
    pages = p.table[0, :-(-1500 // 16)].long()
    keys = torch.zeros(len(pages) * 16, 1, 128)
    keys[:1500, 0, 0] = ramp
    p.k[pages] = keys.to(cache).reshape(-1, 16, 1, 128)
    p.kd.copy_(p.k)
    q = torch.zeros(1, 8, 128)
    q[0, :, 0] = torch.linspace(-200, 200, 8)
    _attend_check([1500], 8, 1, 128, cache, 16, paged=p, q=q.to(BF16))


def test_attention_offsets_beyond_32_bits():
    pages, page, kv, dim = 1100000, 16, 2, 128
    kc, vc = (torch.empty(pages, page, kv, dim, dtype=E4M3, device="cuda") for _ in range(2))
    last = [pages - 1, pages - 2, 3]
    k, v = ((torch.randn(3, page, kv, dim)).to(E4M3) for _ in range(2))
    for i, pg in enumerate(last):
        kc[pg], vc[pg] = k[i].cuda(), v[i].cuda()
    q = torch.randn(1, 4, dim).to(BF16)
    want, lse, size = O.paged_attention(q, k, v, _i32([[0, 1, 2]]), _i32([40]), 0.1)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), kc, vc, _i32([last]).cuda(), _i32([40]).cuda(), 0.1)
    _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
    _close(got_lse, lse, 2.0 ** -13 + 2.0 ** -22 * lse.abs())


def test_attention_of_nothing():
    kc = torch.zeros(4, 16, 2, 128, dtype=BF16).cuda()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32).cuda()  # noqa: E731
    out, lse = torch.ops.b200q.paged_attention(torch.zeros(0, 4, 128, dtype=BF16).cuda(), kc, kc, i(0, 3), i(0), 1.0)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    q = torch.ones(3, 4, 128, dtype=BF16).cuda()
    for table, cache in ((i(3, 0), kc), (i(3, 5), kc[:0])):  # no table, no cache: nothing to see
        out, lse = torch.ops.b200q.paged_attention(q, cache, cache, table, i(3) + 9, 1.0)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_attention_kernels_agree():
    """The plain kernel through the C ABI and the one that the operator takes."""
    from b200_hpu_ops import abi
    p = _Paged([300, 0, 45, 1111], 2, 128, E4M3, 16)
    q = torch.randn(4, 8, 128).to(BF16).cuda()
    table, lens = p.table.cuda(), p.lens.cuda()
    got, got_lse = torch.ops.b200q.paged_attention(q, p.kd, p.vd, table, lens, 0.1, out_dtype=F32)
    out, lse = torch.empty_like(got), torch.empty_like(got_lse)
    a = abi.PagedAttentionArgs()
    a.q, a.q_token_stride, a.q_head_stride, a.requests, a.heads, a.kv_heads, a.dim = q.data_ptr(), 1024, 128, 4, 8, 2, 128
    a.k_cache, a.v_cache, a.cache_dtype, a.num_pages, a.page_size = p.kd.data_ptr(), p.vd.data_ptr(), abi.E4M3, p.kd.shape[0], 16
    a.k_page_stride, a.k_slot_stride, a.k_head_stride = a.v_page_stride, a.v_slot_stride, a.v_head_stride = p.kd.stride()[:3]
    a.block_table, a.table_width, a.table_stride, a.kv_lens = table.data_ptr(), p.width, p.width, lens.data_ptr()
    a.softmax_scale, a.out, a.out_dtype, a.lse, a.force_plain = 0.1, out.data_ptr(), abi.F32, lse.data_ptr(), 1
    a.stream = torch.cuda.current_stream().cuda_stream
    assert abi.lib.b200q_paged_attention(C.byref(a)) == 0
    assert torch.allclose(out, got, rtol=2e-3, atol=2e-3) and torch.allclose(lse, got_lse, rtol=1e-5)


def test_attention_refusals():
    q = torch.zeros(2, 4, 64, dtype=BF16).cuda()
    kc, vc = torch.zeros(2, 3, 16, 2, 64, dtype=BF16).cuda()
    table, lens = torch.zeros(2, 3, dtype=torch.int32).cuda(), torch.zeros(2, dtype=torch.int32).cuda()
    ok = dict(q=q, k_cache=kc, v_cache=vc, block_table=table, kv_lens=lens, softmax_scale=1.0)
    torch.ops.b200q.paged_attention(**ok)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(k_cache=kc.to(E4M3)), dict(k_cache=kc[:2]),
                dict(k_cache=kc.float(), v_cache=vc.float()), dict(k_cache=kc.transpose(2, 3), v_cache=vc.transpose(2, 3)), dict(block_table=table.long()),
                dict(block_table=table[:1]), dict(block_table=table.t().contiguous().t()), dict(kv_lens=lens.long()), dict(kv_lens=lens[:1]), dict(window=-1),
                dict(k_scale_inv=torch.ones(2).cuda()), dict(v_scale_inv=torch.ones(1)), dict(out_scale=torch.ones(1, dtype=BF16).cuda()), dict(out_dtype=E5M2),
                dict(kv_lens=lens.cpu())):
        with pytest.raises(RuntimeError):
            torch.ops.b200q.paged_attention(**{**ok, **bad})


# ----------------------------------------------------------------------------- together
class _Model:
    """One attention layer's decode path: plan, append, attend, with every length on the device."""

    def __init__(self, cache, requests=5, heads=8, kv=2, dim=128, page=16, pages=64, width=12):
        g = torch.Generator().manual_seed(3)
        self.heads, self.kv, self.dim, self.page, self.cache = heads, kv, dim, page, cache
        self.kc, self.vc = (torch.full((pages, page, kv, dim), math.nan).to(cache).cuda() for _ in range(2))
        self.free = torch.randperm(pages, generator=g).to(torch.int32).cuda()
        self.table = torch.full((requests, width), -1, dtype=torch.int32).cuda()
        self.lens, self.head = torch.zeros(requests, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
        self.qw, self.kw = (torch.randn(dim, generator=g).to(BF16).cuda() for _ in range(2))
        self.cos_sin = _table(dim).cuda()
        self.scale, self.inv = (None, None) if cache == BF16 else (_one(16.0).cuda(), _one(1 / 16.0).cuda())

    def append(self, qkv, new):
        h, g = self.heads, self.kv
        slots, pos, start, lens, head = torch.ops.b200q.paged_plan(self.lens, new, self.table, self.free, self.head, self.page, qkv.shape[0])
        q = torch.ops.b200q.qk_norm_rope_append(qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:], self.qw, self.kw, 1e-6, self.cos_sin, pos, False, slots, self.kc, self.vc,
                                                self.scale, self.scale)
        self.lens.copy_(lens)
        self.head.copy_(head)
        return q

    def attend(self, q):
        return torch.ops.b200q.paged_attention(q, self.kc, self.vc, self.table, self.lens, 1 / math.sqrt(self.dim), self.inv, self.inv)[0]


def _dense_check(m, seen, out):
    """seen: each request's projections so far; out: the answer to its last token."""
    h, g = m.heads, m.kv
    for b, rows in enumerate(seen):
        if not len(rows):
            assert bool((out[b] == 0).all())
            continue
        x, pos = torch.stack(rows), torch.arange(len(rows))
        q = O.norm_rope(x[-1:, :h], m.qw.cpu(), 1e-6, m.cos_sin.cpu(), pos[-1:], False).to(BF16)
        k = O.norm_rope(x[:, h:h + g], m.kw.cpu(), 1e-6, m.cos_sin.cpu(), pos, False)
        v = x[:, h + g:].double()
        if m.cache != BF16:
            k, v = ((t * 16).clamp(-448, 448).float().to(m.cache).double() / 16 for t in (k, v))
        else:
            k, v = k.to(BF16).double(), v
        s = torch.einsum("hd,nhd->hn", q[0].double(), k.repeat_interleave(h // g, 1)) / math.sqrt(m.dim)
        want = torch.einsum("hn,nhd->hd", s.softmax(-1), v.repeat_interleave(h // g, 1))
        # a q or k that rounds the other way than fp64's moves scores by up to a step of its type
        assert O.rel_frobenius(out[b].float(), want) < (2e-2 if m.cache == BF16 else 4e-2)


@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_prompt_then_decode_steps(cache):
    m = _Model(cache)
    gen = torch.Generator().manual_seed(9)
    prompts = _i32([37, 0, 16, 5, 64])
    rows = torch.randn(int(prompts.sum()) + 6, 12, 128, generator=gen).to(BF16)  # six padded rows
    m.append(rows.cuda(), prompts.cuda())
    at, seen = 0, []
    for n in prompts.tolist():
        seen.append(list(rows[at:at + n]))
        at += n
    for step in range(20):
        new = _i32([1, step % 3 == 0, 1, 1, 1])
        x = torch.randn(5, 12, 128, generator=gen).to(BF16)
        q = m.append(x[:int(new.sum())].cuda(), new.cuda())
        t, answers = 0, torch.zeros(5, 8, 128, dtype=BF16).cuda()
        for b, n in enumerate(new.tolist()):
            if n:
                seen[b].append(x[t])
                answers[b] = q[t]
                t += 1
        out = m.attend(answers).cpu()
        if step % 3 == 0:  # (a request without a new token has no query of its own)
            _dense_check(m, seen, out)
    assert m.lens.tolist() == [len(s) for s in seen]
    used = m.table[m.table >= 0]
    assert used.unique().numel() == used.numel() == int(m.head)  # no page twice, none left out


def test_decode_steps_in_graphs_and_on_other_streams():
    """Two captured steps of two caches, replayed on streams of their own at the same time, give what plain calls give."""
    def steps(m, x, run):
        return [run(m, x[i]).clone() for i in range(len(x))]

    ones = torch.ones(5, dtype=torch.int32).cuda()
    step = lambda m, x: m.attend(m.append(x, ones))  # noqa: E731
    x = torch.randn(2, 25, 5, 12, 128).to(BF16).cuda()
    plain = [steps(_Model(E4M3), x[i], step) for i in range(2)]
    models, graphs, outs, ins = [_Model(E4M3) for _ in range(2)], [], [], []
    step(_Model(E4M3), x[0, 0])
    torch.cuda.synchronize()
    for m in models:
        ins.append(torch.zeros_like(x[0, 0]))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(m, ins[-1]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for t in range(25):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ins[i].copy_(x[i, t])
                graphs[i].replay()
                got[i].append(outs[i].clone())
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(got[i], plain[i]):
            assert torch.equal(a, b)
    # and eagerly on another stream, behind work that is still running
    m, s = _Model(E4M3), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-2
        other = steps(m, x[0], step)
    s.synchronize()
    for a, b in zip(other, plain[0]):
        assert torch.equal(a, b)
