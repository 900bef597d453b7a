"""The paged key/value cache where it is easily wrong: precision of fp32 outputs, sizes near the ends of their types, tables and
caches of unusual form.  The oracle and the helpers are those of test_gpu_paged.py."""
import ctypes as C
import math

import pytest
import torch

from oracle import hpu_oracle as O
from test_gpu_paged import BF16, E4M3, E5M2, F32, _close, _dense_check, _i32, _Model, _one, _Paged, _status, _table  # noqa: F401 (_status: device status after each test)

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


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,cache", [(F32, E4M3), (BF16, E4M3), (F32, E5M2), (F32, BF16)])
def test_append_large_values_times_a_scale(interleaved, src, cache):
    """Values whose product with the scale passes the end of fp32: they turn first, and then saturate (or become infinite in bf16) with the sign
    that the turned value has."""
    g = torch.Generator().manual_seed(2)
    x = ((torch.rand(5, 4, 64, generator=g) + 0.1) * torch.where(torch.rand(5, 4, 64, generator=g) < 0.5, -1e37, 1e37)).to(src)
    kc, vc = (torch.zeros(1, 16, 1, 64).to(cache).cuda() for _ in range(2))
    at, table, scale = torch.arange(5), _table(64), _one(1000.0).cuda()
    q_dtype = E4M3 if cache == BF16 else cache
    q = torch.ops.b200q.qk_norm_rope_append(x[:, :2].cuda(), x[:, 2:3].cuda(), x[:, 3:].cuda(), None, None, 1e-6, table.cuda(), at.cuda(), interleaved, at.cuda(), kc, vc,
                                            scale, scale, scale, q_dtype)
    limit = {E4M3: 448.0, E5M2: 57344.0, BF16: math.inf}
    for got, dtype, rows in ((q, q_dtype, x[:, :2]), (kc[0, :5], cache, x[:, 2:3])):
        want = O.norm_rope(rows, None, 0.0, table, at, interleaved)
        far = want.abs() > 1e36  # (of the others a few may end below fp32's end)
        assert float(far.double().mean()) > 0.8
        assert torch.equal(got.float().cpu().double()[far], (want.sign() * limit[dtype])[far])
    assert torch.equal(vc[0, :5].float().cpu(), x[:, 3:].float().sign() * limit[cache])


@pytest.mark.parametrize("heads,kv", [(0, 2), (3, 0), (0, 0)])
def test_append_without_queries_or_without_keys(heads, kv):
    x = torch.randn(9, heads + 2 * kv, 64).to(BF16).cuda()
    kc, vc = (torch.zeros(2, 16, kv, 64, dtype=BF16).cuda() for _ in range(2))
    slots, pos = torch.randperm(32)[:9], torch.arange(9)
    q = torch.ops.b200q.qk_norm_rope_append(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], None, None, 1e-6, _table(64).cuda(), pos.cuda(), False, slots.cuda(),
                                            kc, vc)
    assert q.shape == (9, heads, 64)
    y = O.norm_rope(x.cpu(), None, 0.0, _table(64), pos, False)
    tol = 2.0 ** -8 * y.abs() + 2.0 ** -20 * y.abs().amax(-1, keepdim=True) if heads + kv else y
    _close(q.float(), y[:, :heads], tol[:, :heads])
    _close(kc.view(32, kv, 64)[slots.cuda()].float(), y[:, heads:heads + kv], tol[:, heads:heads + kv])
    assert torch.equal(vc.view(32, kv, 64)[slots.cuda()], x[:, heads + kv:])


def _append_to(kc, vc, tokens=7):
    kv, dim = kc.shape[2:]
    x = torch.randn(tokens, 3 * kv, dim).to(BF16).cuda()
    slots = torch.randperm(kc.shape[0] * kc.shape[1])[:tokens].cuda()
    torch.ops.b200q.qk_norm_rope_append(x[:, :kv], x[:, kv:2 * kv], x[:, 2 * kv:], None, None, 1e-6, None, None, False, slots, kc, vc)
    return x[:, kv:2 * kv], x[:, 2 * kv:], slots


def test_append_refuses_caches_that_overlap():
    """Strides too short for what lies inside them, one tensor as both caches, two that share part of an allocation."""
    flat = torch.zeros(1 << 14, dtype=BF16).cuda()
    view = lambda s, at=0, n=(4, 16, 2, 64): flat.as_strided(n, (*s, 1), at)  # noqa: E731
    good, far = view((2048, 128, 64)), torch.zeros(4, 16, 2, 64, dtype=BF16).cuda()
    _append_to(good, far)
    for bad in ((2048, 128, 4), (2048, 64, 64), (1024, 128, 64), (0, 128, 64), (2048, 0, 64), (2048, 128, 60)):
        for kc, vc in ((view(bad), far), (far, view(bad))):
            with pytest.raises(RuntimeError, match="must not overlap"):
                _append_to(kc, vc)
    for other in (good, view((2048, 128, 64), 64), view((2048, 128, 64), 6144), view((2048, 64, 1024), 2048)):
        with pytest.raises(RuntimeError, match="must not overlap"):
            _append_to(good, other)


@pytest.mark.parametrize("form", ["halves", "pages", "slots", "heads", "values", "orders"])
def test_append_to_caches_in_one_allocation(form):
    n, page, kv, dim = 5, 16, 3, 64
    if form == "orders":  # a page of keys slot by slot, then one of values head by head
        pool = torch.zeros(n, 2, page * kv * dim, dtype=BF16).cuda()
        kc, vc = pool[:, 0].view(n, page, kv, dim), pool[:, 1].view(n, kv, page, dim).transpose(1, 2)
    else:
        at = ("halves", "pages", "slots", "heads", "values").index(form)
        sizes = [n, page, kv]
        if form == "values":
            pool = torch.zeros(n, page, kv, 2 * dim, dtype=BF16).cuda()
            kc, vc = pool[..., :dim], pool[..., dim:]
        else:
            pool = torch.zeros(*sizes[:at], 2, *sizes[at:], dim, dtype=BF16).cuda()
            kc, vc = pool.select(at, 0), pool.select(at, 1)
    k, v, slots = _append_to(kc, vc)
    for cache, x in ((kc, k), (vc, v)):
        want = torch.zeros(n, page, kv, dim, dtype=BF16).cuda()
        want.view(-1, kv, dim)[slots] = x
        assert torch.equal(cache, want)


# ----------------------------------------------------------------------------- plan
def test_plan_of_almost_2_to_the_31_pages():
    """The largest table that is taken, all of it new: the pages are counted to within 2^14 of the type's end."""
    requests, width = 8192, 262143
    whole = torch.full((requests * width + 2048,), 7, dtype=torch.int32, device="cuda")
    table = whole[1024:-1024].view(requests, width)
    ctx, new = torch.zeros(requests, dtype=torch.int32).cuda(), torch.full((requests,), width, dtype=torch.int32).cuda()
    slots, pos, start, lens, head = torch.ops.b200q.paged_plan(ctx, new, table, _i32([5, 6]).cuda(), None, 1, 200000)
    assert head.tolist() == [requests * width] and lens.tolist() == [width] * requests
    assert table[0, :3].tolist() == [5, 6, -1] and int((table == -1).sum()) == requests * width - 2
    assert bool((whole[:1024] == 7).all()) and bool((whole[-1024:] == 7).all())
    assert slots[:3].tolist() == [5, 6, -1] and bool((slots[2:] == -1).all()) and torch.equal(pos.cpu(), torch.arange(200000))
    assert torch.equal(start.cpu(), (torch.arange(requests + 1) * width).int())


# ----------------------------------------------------------------------------- attention: sizes
def test_attention_empty_rows_of_very_many_heads():
    """2^31 values of four in one request's output, which are all to be cleared."""
    heads, dim = 1 << 25, 256
    dirty = torch.ones(1, heads, dim, dtype=BF16, device="cuda")
    del dirty  # (the output takes its place)
    q, kc = torch.ones(1, heads, 1, dtype=BF16, device="cuda").expand(1, heads, dim).contiguous(), torch.ones(1, 16, 1, dim, dtype=BF16).cuda()
    out, lse = torch.ops.b200q.paged_attention(q, kc, kc, _i32([[0]]).cuda(), _i32([0]).cuda(), 1.0)
    assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("cache,heads,kv,dim", [(E4M3, 8, 1, 128), (BF16, 4, 2, 64), (E5M2, 12, 1, 64), (BF16, 2, 1, 256), (E4M3, 2, 1, 72)])
@pytest.mark.parametrize("size", [-3e8, 1e9, -1e12, 3e20, -1e38, 2.2e38, -2.2e38, -2.35e38])
def test_attention_large_scores(cache, heads, kv, dim, size):
    """All keys of a row score the same, up to 3.39e38 away from 0 in powers of two, where neighbouring numbers are far apart, and a row
    of the lowest ones is not an empty one.  The roundings of
    a score (its factor's three, its own, two of the way back to powers of e) are 6 * 2^-24 of lse."""
    p = _Paged([0, 1, 5, 40, 300, 5000], kv, dim, cache, 16, seed=3)
    k = torch.where(p.k.float().isnan(), math.nan, 0.0)
    k[..., 0] += 1.0
    p.k = k.to(cache)
    q = torch.zeros(6, heads, dim)
    q[..., 0] = size
    q = q.to(BF16)
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, 1.0)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.k.cuda(), p.vd, p.table.cuda(), p.lens.cuda(), 1.0)
    _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
    _close(got_lse, lse, 2.0 ** -21 * torch.where(lse.isfinite(), lse.abs(), 0.0))


# ----------------------------------------------------------------------------- attention: a copy that does not arrive
@pytest.mark.parametrize("lens,kv,drops", [
    ([200], 1, [(0, 0, 0), (0, 3, 1), (0, 6, 0)]),                                       # one CTA, no joining kernel
    ([700, 40, 0, 1500, 16, 900], 8, [(0, 0, 0), (0, 7, 1), (1, 0, 0), (50, 3, 0), (99, 7, 0)]),  # rows cut between warps and CTAs; the last CTA has 15 steps
    ([3000 + 7 * i for i in range(16)], 8, [(0, 0, 0), (10, 3, 5), (73, 0, 15), (147, 7, 12)]),   # heads side by side
    ([131072], 8, [(0, 0, 0), (80, 4, 7)]),                                               # rows that every CTA has a part of
])
def test_attention_rows_whose_copies_do_not_arrive_are_nan(lens, kv, drops):
    """The wait runs out (no GPU fault), the status says so, the rows that missed their keys are NaN as a whole, all others have the bytes
    of an undisturbed call."""
    import b200_hpu_ops
    from b200_hpu_ops import abi
    heads, dim, page = 8 * kv, 128, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    need = [-(-n // page) for n in lens]
    kc, vc = (torch.randint(0, 256, (sum(need), page, kv, dim), generator=g, device="cuda", dtype=torch.uint8).bitwise_and(0xBF).view(E4M3) for _ in range(2))
    table, at = torch.full((len(lens), max(need)), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    table, kv_lens = table.cuda(), _i32(lens).cuda()
    q = torch.randn(len(lens), heads, dim, generator=g, device="cuda").to(BF16)
    run = lambda: torch.ops.b200q.paged_attention(q, kc, vc, table, kv_lens, 0.05)  # noqa: E731
    want, want_lse = run()
    assert bool(want.isfinite().all())
    for cta, warp, step in drops:
        out, lse = torch.zeros_like(want), torch.zeros_like(want_lse)
        space = torch.full((abi.lib.b200q_paged_attention_workspace_bytes(len(lens), heads, kv, dim, abi.E4M3),), 0x11, dtype=torch.uint8, device="cuda")
        a = abi.PagedAttentionArgs()
        a.q, a.q_token_stride, a.q_head_stride, a.requests, a.heads, a.kv_heads, a.dim = q.data_ptr(), heads * dim, dim, len(lens), heads, kv, dim
        a.k_cache, a.v_cache, a.cache_dtype, a.num_pages, a.page_size = kc.data_ptr(), vc.data_ptr(), abi.E4M3, kc.shape[0], page
        a.k_page_stride, a.k_slot_stride, a.k_head_stride = a.v_page_stride, a.v_slot_stride, a.v_head_stride = kc.stride()[:3]
        a.block_table, a.table_width, a.table_stride, a.kv_lens = table.data_ptr(), table.shape[1], table.shape[1], kv_lens.data_ptr()
        a.softmax_scale, a.out, a.out_dtype, a.lse = 0.05, out.data_ptr(), abi.BF16, lse.data_ptr()
        a.workspace, a.workspace_bytes, a.stream = space.data_ptr(), space.numel(), torch.cuda.current_stream().cuda_stream
        assert abi.lib.b200q_selftest_paged_wait_timeout(C.byref(a), cta, warp, step) == 0
        assert b200_hpu_ops.device_status() == 801
        lost = lse.isnan()
        assert torch.equal(out.isnan().all(-1), lost) and torch.equal(out.isnan().any(-1), lost)
        assert torch.equal(out[~lost], want[~lost]) and torch.equal(lse[~lost], want_lse[~lost])
        if (cta, warp, step) == (0, 0, 0):
            assert bool(lost[0, :8].all())  # (the first step of the list: request 0, key/value head 0)
        assert 8 <= int(lost.sum()) <= 128 and (len(lens) == 1 or not bool(lost.all()))  # (no CTA has a part of more than 16 rows of 8 heads)
        for x, y in zip(run(), (want, want_lse)):
            assert torch.equal(x, y)
    assert b200_hpu_ops.device_status() == 0


def test_attention_selftest_refusals():
    from b200_hpu_ops import abi
    test = abi.lib.b200q_selftest_paged_wait_timeout
    assert test(None, 0, 0, 0) == -1
    a = abi.PagedAttentionArgs()
    x = torch.zeros(1 << 16, dtype=torch.uint8).cuda()
    a.q = a.k_cache = a.v_cache = a.out = a.block_table = a.kv_lens = x.data_ptr()
    a.requests, a.heads, a.kv_heads, a.dim, a.num_pages, a.page_size, a.table_width, a.cache_dtype, a.out_dtype = 1, 8, 1, 128, 1, 16, 1, abi.E4M3, abi.BF16
    assert test(C.byref(a), -1, 0, 0) == -1 and test(C.byref(a), 0, 0, -1) == -1
    assert test(C.byref(a), 0, 0, 0) == -1  # no workspace
    for name, value in (("dim", 64), ("cache_dtype", abi.BF16), ("out_dtype", abi.F32), ("heads", 9)):
        old = getattr(a, name)
        setattr(a, name, value)
        assert test(C.byref(a), 0, 0, 0) == -2
        setattr(a, name, old)


# ----------------------------------------------------------------------------- attention: workspace
@pytest.mark.parametrize("cache,heads,kv,dim", [(E4M3, 8, 1, 64), (BF16, 16, 1, 64), (E4M3, 64, 8, 128), (E5M2, 20, 1, 128), (E4M3, 16, 1, 256), (BF16, 8, 4, 256)])
def test_attention_stays_within_its_workspace(cache, heads, kv, dim):
    """A workspace of just the size that is asked for, filled with NaN, between guards: rows cut between warps and between all CTAs, empty
    ones and whole ones.  A workspace that is smaller by one byte is refused."""
    from b200_hpu_ops import abi
    lens = [40000, 0, 17, 3000, 1]
    p = _Paged(lens, kv, dim, cache, 16, seed=4)
    q = torch.randn(5, heads, dim, generator=p.g).to(BF16).cuda()
    table, kv_lens = p.table.cuda(), p.lens.cuda()
    want, want_lse = torch.ops.b200q.paged_attention(q, p.kd, p.vd, table, kv_lens, 0.1)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    size = abi.lib.b200q_paged_attention_workspace_bytes(5, heads, kv, dim, abi.DTYPE[cache])
    space = torch.full((size + 2 * 65536,), 0xFF, dtype=torch.uint8, device="cuda")
    a = abi.PagedAttentionArgs()
    a.q, a.q_token_stride, a.q_head_stride, a.requests, a.heads, a.kv_heads, a.dim = q.data_ptr(), heads * dim, dim, 5, heads, kv, dim
    a.k_cache, a.v_cache, a.cache_dtype, a.num_pages, a.page_size = p.kd.data_ptr(), p.vd.data_ptr(), abi.DTYPE[cache], p.kd.shape[0], 16
    a.k_page_stride, a.k_slot_stride, a.k_head_stride = a.v_page_stride, a.v_slot_stride, a.v_head_stride = p.kd.stride()[:3]
    a.block_table, a.table_width, a.table_stride, a.kv_lens = table.data_ptr(), p.width, p.width, kv_lens.data_ptr()
    a.softmax_scale, a.out, a.out_dtype, a.lse = 0.1, out.data_ptr(), abi.BF16, lse.data_ptr()
    a.workspace, a.workspace_bytes, a.stream = space.data_ptr() + 65536, size, torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        assert abi.lib.b200q_paged_attention(C.byref(a)) == 0
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert bool((space[:65536] == 0xFF).all()) and bool((space[65536 + size:] == 0xFF).all())
    a.workspace_bytes = size - 1
    assert abi.lib.b200q_paged_attention(C.byref(a)) == -1


# ----------------------------------------------------------------------------- a server's steps
def _captured(m, tokens, requests):
    """A step of plan, append and the attention of each request's newest token, captured: (new lengths, projections, answers, replay)."""
    new, qkv = torch.zeros(requests, dtype=torch.int32).cuda(), torch.zeros(tokens, m.heads + 2 * m.kv, m.dim, dtype=BF16).cuda()

    def step():
        h, g = m.heads, m.kv
        slots, pos, start, lens, head = torch.ops.b200q.paged_plan(m.lens, new, m.table, m.free, m.head, m.page, tokens)
        q = torch.ops.b200q.qk_norm_rope_append(qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:], m.qw, m.kw, 1e-6, m.cos_sin, pos, False, slots, m.kc, m.vc, m.scale,
                                                m.scale)
        last = (start[1:] - 1).clamp(min=0)
        out = torch.ops.b200q.paged_attention(q.index_select(0, last), m.kc, m.vc, m.table, lens, 1 / math.sqrt(m.dim), m.inv, m.inv)[0]
        return slots, lens, head, out

    lens, head, table = m.lens.clone(), m.head.clone(), m.table.clone()
    step()  # (each operator runs once before the capture; with no new tokens nothing is written)
    torch.cuda.synchronize()
    assert torch.equal(m.table, table) and torch.equal(m.lens, lens) and torch.equal(m.head, head)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    return new, qkv, outs, graph


@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_captured_steps_with_idle_requests_and_prompts(cache):
    """From 0 to 9 new tokens for each request, other ones in every replay; a request's answer is that of its newest token."""
    m, gen = _Model(cache, requests=5), torch.Generator().manual_seed(11)
    new, qkv, (slots, lens, head, out), graph = _captured(m, 24, 5)
    seen = [[] for _ in range(5)]
    for step in range(24):
        counts = [[1, 1, 1, 1, 1], [1, 0, 1, 0, 1], [0, 0, 1, 1, 0], [9, 0, 1, 7, 1], [0, 0, 0, 0, 0], [0, 1, 0, 0, 5]][step % 6]
        x = torch.randn(24, 12, 128, generator=gen).to(BF16)
        new.copy_(_i32(counts))
        qkv.copy_(x)
        graph.replay()
        t = 0
        for b, n in enumerate(counts):
            seen[b] += list(x[t:t + n])
            t += n
        assert bool((slots[t:] == -1).all()) and lens.tolist() == [len(s) for s in seen]
        if step % 4 == 3 or step == 4:
            busy = [b for b, n in enumerate(counts) if n]
            answers = out.cpu()
            _dense_check(m, [seen[b] for b in busy], answers[busy])
        m.lens.copy_(lens)
        m.head.copy_(head)


@pytest.mark.parametrize("cache", [E4M3, BF16])
def test_captured_steps_while_requests_come_and_go(cache):
    """The pool is gone through several times.  Its list has one length and one address for the graph: a host that finds `free_head` above the
    number of free pages keeps the lengths and the head of before, puts what was not taken and what has come back to the front of
    the list with the head at 0, and runs the step again."""
    m, gen = _Model(cache, requests=4, pages=24, width=8), torch.Generator().manual_seed(12)
    new, qkv, (slots, lens, head, out), graph = _captured(m, 4, 4)
    seen, life = [[] for _ in range(4)], [40, 70, 55, 100]
    count, retired, short, taken = 24, [], 0, 0
    new.fill_(1)
    for step in range(400):
        x = torch.randn(4, 12, 128, generator=gen).to(BF16)
        qkv.copy_(x)
        graph.replay()
        if int(head) > count:
            short += 1
            begin = int(m.head)
            assert bool((slots < 0).any())  # a token without a page
            pool = m.free[begin:count].tolist() + retired
            taken, count, retired = taken + begin, len(pool), []
            m.free.copy_(_i32(pool + [-1] * (24 - count)))
            m.head.zero_()
            graph.replay()
            assert int(head) <= count
        assert bool((slots >= 0).all()) and slots.unique().numel() == 4
        for b in range(4):
            seen[b].append(x[b])
        if step % 40 == 39 or step in (0, 97, 98):
            _dense_check(m, seen, out.cpu())
        m.lens.copy_(lens)
        m.head.copy_(head)
        held = [m.table[b, :-(-len(seen[b]) // m.page)].tolist() for b in range(4)]
        left = m.free[int(m.head):count].tolist()
        assert sorted(sum(held, []) + left + retired) == list(range(24))  # every page once: held, free or retired
        for b in range(4):
            if len(seen[b]) == life[b]:  # its pages go back, and another request takes its row
                retired += held[b]
                seen[b] = []
                m.lens[b] = 0
    assert short >= 4 and taken > 48


def test_prompts_through_the_fp8_attention():
    """Prompts without a cached prefix: their keys and values gathered from the pages, one request at a time, for fp8_sdpa_recomp_fwd."""
    m, gen = _Model(E4M3, requests=4), torch.Generator().manual_seed(13)
    prompts, h, g, rep = [37, 0, 130, 5], m.heads, m.kv, m.heads // m.kv
    x = torch.randn(sum(prompts) + 4, h + 2 * g, 128, generator=gen).to(BF16)
    qkv, q_scale = x.cuda(), _one(32.0).cuda()
    slots, pos, start, lens, head = torch.ops.b200q.paged_plan(m.lens, _i32(prompts).cuda(), m.table, m.free, m.head, m.page, len(x))
    q = torch.ops.b200q.qk_norm_rope_append(qkv[:, :h], qkv[:, h:h + g], qkv[:, h + g:], m.qw, m.kw, 1e-6, m.cos_sin, pos, False, slots, m.kc, m.vc, m.scale,
                                            m.scale, q_scale, E4M3)
    at = 0
    for b, n in enumerate(prompts):
        if not n:
            continue
        pages = m.table[b, :-(-n // m.page)].long()
        k, v = (c.view(torch.uint8)[pages].view(E4M3).flatten(0, 1)[:n].transpose(0, 1).unsqueeze(1) for c in (m.kc, m.vc))  # [kv_heads, 1, n, dim]
        rows = q[at:at + n].view(n, g, rep, 128).permute(1, 2, 0, 3)                                                       # [kv_heads, heads of each, n, dim]
        got = torch.ops.hpu.fp8_sdpa_recomp_fwd(rows, k, v, None, 0.0, 128 ** -0.5, True, False, "None", 1 / q_scale, m.inv, m.inv, None, None, None,
                                                False, False, None, "None")[0]
        # keys and values as the oracle makes them from the projections; what is left is the output's rounding (2^-8 at most, of each value) and the
        # few e4m3 values that round the other way from fp32
        kk = (O.norm_rope(x[at:at + n, h:h + g], m.kw.cpu(), 1e-6, m.cos_sin.cpu(), torch.arange(n), False) * 16).clamp(-448, 448).float().to(E4M3)
        vv = (x[at:at + n, h + g:].float() * 16).clamp(-448, 448).to(E4M3)
        want = O.fp8_sdpa_recomp_fwd(rows.cpu(), kk.transpose(0, 1).unsqueeze(1), vv.transpose(0, 1).unsqueeze(1), None, 0.0, 128 ** -0.5, True,
                                     d_scale_q=_one(1 / 32.0), d_scale_k=_one(1 / 16.0), d_scale_v=_one(1 / 16.0))[0]
        assert O.rel_frobenius(got.float().cpu(), want.float()) < 2.0 ** -7
        at += n


@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (4, 2, 64), (2, 1, 256), (12, 1, 64), (2, 1, 72)])
@pytest.mark.parametrize("rising", [False, True])
def test_attention_large_values_of_a_bf16_cache(heads, kv, dim, rising):
    """Values of 3e36: an average of them is nowhere near the end of fp32, 2^7 times one of them is beyond it.  With scores that rise by 7
    from one step of 16 keys to the next the running maximum trails behind the scores as far as it may."""
    p = _Paged([0, 1, 5, 40, 300], kv, dim, BF16, 16, seed=6)
    p.v = (p.v.float() * 3e36).to(BF16)
    scale = 0.1
    if rising:
        k = torch.zeros(p.k.shape)
        for b, n in enumerate(p.lens.tolist()):
            for i in range(-(-n // 16)):
                k[int(p.table[b, i]), :, :, 0] = 7 * math.log(2) * i
        p.k = torch.where(p.k.float().isnan(), math.nan, k).to(BF16)
        scale = 1.0
    q = torch.randn(5, heads, dim, generator=p.g)
    if rising:
        q = torch.zeros(5, heads, dim)
        q[..., 0] = 1.0
    q = q.to(BF16)
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, scale)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.k.cuda(), p.v.cuda(), p.table.cuda(), p.lens.cuda(), scale)
    _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
    _close(got_lse, lse, 2.0 ** -13 + 2.0 ** -22 * torch.where(lse.isfinite(), lse.abs(), 0.0))


@pytest.mark.parametrize("cache", [E4M3, E5M2, BF16])
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 1), (128, 12), (256, 4)])
@pytest.mark.parametrize("base,rise", [(base * 2.0 ** i, rise) for base in (1.5, -1.5) for i, rise in ((24, 8), (25, 8), (26, 8), (27, 16), (28, 32))])
def test_attention_scores_that_rise_far_from_0(cache, dim, heads, base, rise):
    """Scores of 1.5 times 2^24 to 2^28 (in powers of two, exactly), where the neighbours of a number are 2 to 32 away, and a little more for
    every 16 keys: probabilities of up to 2^16 against the maximum so far, less the 7 that it is held below, which f16 does not hold.  (Not for the plain kernel, whose
    scores are in powers of e and not exact here: spacing 8 against a difference of 8 ln 2 and 16 ln 2.)"""
    p = _Paged([0, 16, 17, 40, 128, 128, 128], 1, dim, cache, 16, seed=8)
    k = torch.zeros(p.k.shape)
    k[..., 0] = 256.0
    for b, n in enumerate(p.lens.tolist()):
        for i in range(-(-n // 16)):
            k[int(p.table[b, i]), :, :, 1] = i
    p.k = torch.where(p.k.float().isnan(), math.nan, k).to(cache)
    q = torch.zeros(7, heads, dim)
    q[..., 0], q[..., 1] = base / 256, rise
    q, scale = q.to(BF16), float.fromhex("0x1.62e42fefa39efp-1")
    as_held = float(torch.tensor(scale, dtype=F32))
    assert float(torch.tensor(as_held, dtype=F32) * torch.tensor(1.44269504088896341, dtype=F32)) == 1.0
    want, lse, size = O.paged_attention(q, p.k, p.v, p.table, p.lens, scale)
    got, got_lse = torch.ops.b200q.paged_attention(q.cuda(), p.k.cuda(), p.vd, p.table.cuda(), p.lens.cuda(), scale)
    _close(got.float(), want, 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size)
    _close(got_lse, lse, 2.0 ** -21 * torch.where(lse.isfinite(), lse.abs(), 0.0))
