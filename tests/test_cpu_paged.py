"""The paged key/value cache without a GPU: what the C ABI refuses before any CUDA call, the schemas and Meta kernels, and the
oracle against dense definitions."""
import ctypes
import math

import pytest
import torch

from b200_hpu_ops import abi
from oracle import hpu_oracle as O

E4M3, E5M2, BF16, F32 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32
BAD, UNSUPPORTED, TOO_LARGE = -1, -2, -4
AT = 1 << 20  # an address that nothing reads


def test_layouts_of_the_argument_structs():
    assert abi.lib.b200q_sizeof_args(2) == ctypes.sizeof(abi.AppendArgs)
    assert abi.lib.b200q_sizeof_args(3) == ctypes.sizeof(abi.PagedAttentionArgs)


def _plan(**kw):
    a = dict(context=AT, new=AT, requests=4, table=AT, width=8, stride=8, free=AT, free_count=9, head=None, page=16, tokens=4, slots=AT, positions=AT,
             start=AT, lens=AT, next=AT, stream=None)
    a.update(kw)
    return abi.lib.b200q_paged_plan(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(requests=-1), BAD), (dict(width=-1), BAD), (dict(stride=7), BAD), (dict(page=0), BAD), (dict(tokens=-1), BAD), (dict(free_count=-1), BAD),
    (dict(requests=8193), TOO_LARGE), (dict(requests=8192, width=1 << 18, stride=1 << 18), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE), (dict(page=1 << 31), TOO_LARGE),
    (dict(context=None), BAD), (dict(new=None), BAD), (dict(table=None), BAD), (dict(free=None), BAD), (dict(slots=None), BAD), (dict(positions=None), BAD),
    (dict(start=None), BAD), (dict(lens=None), BAD), (dict(next=None), BAD),
])
def test_plan_refuses(kw, rc):
    assert _plan(**kw) == rc


def _append(**kw):
    a = abi.AppendArgs()
    for p in ("q", "k", "v", "slot_map", "k_cache", "v_cache", "q_out"):
        setattr(a, p, AT)
    a.src_dtype, a.cache_dtype, a.q_out_dtype, a.weight_dtype = abi.BF16, abi.E4M3, abi.BF16, abi.BF16
    a.tokens, a.heads, a.kv_heads, a.dim, a.num_pages, a.page_size = 3, 4, 2, 64, 8, 16
    a.q_token_stride, a.q_head_stride = 256, 64
    a.k_token_stride = a.v_token_stride = 128
    a.k_head_stride = a.v_head_stride = a.k_cache_head_stride = a.v_cache_head_stride = 64
    a.k_page_stride = a.v_page_stride = 2048
    a.k_slot_stride = a.v_slot_stride = 128
    for name, value in kw.items():
        setattr(a, name, value)
    return abi.lib.b200q_qk_norm_rope_append(ctypes.byref(a))


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=-1), BAD), (dict(heads=-1), BAD), (dict(kv_heads=-1), BAD), (dict(num_pages=-1), BAD), (dict(page_size=0), BAD),
    (dict(src_dtype=abi.E4M3), BAD), (dict(q_out_dtype=abi.F32), BAD), (dict(cache_dtype=abi.F32), BAD), (dict(cache_dtype=9), BAD),
    (dict(q_weight=AT, weight_dtype=abi.E4M3), BAD), (dict(cos_sin=AT, rotary_dim=64), BAD), (dict(slot_map=None), BAD), (dict(q=None), BAD),
    (dict(k=None), BAD), (dict(v=None), BAD), (dict(k_cache=None), BAD), (dict(v_cache=None), BAD), (dict(q_out=None), BAD),
    (dict(dim=0), UNSUPPORTED), (dict(dim=60), UNSUPPORTED), (dict(dim=264), UNSUPPORTED),
    (dict(cos_sin=AT, positions=AT, rotary_dim=0), UNSUPPORTED), (dict(cos_sin=AT, positions=AT, rotary_dim=12), UNSUPPORTED),
    (dict(cos_sin=AT, positions=AT, rotary_dim=72), UNSUPPORTED), (dict(cos_sin=AT + 8, positions=AT, rotary_dim=64), UNSUPPORTED),
    (dict(q=AT + 2), UNSUPPORTED), (dict(k_cache=AT + 1), UNSUPPORTED), (dict(q_weight=AT + 2), UNSUPPORTED), (dict(q_out=AT + 4), UNSUPPORTED),
    (dict(q_token_stride=254), UNSUPPORTED), (dict(v_slot_stride=66), UNSUPPORTED), (dict(k_page_stride=2), UNSUPPORTED),
    (dict(tokens=1 << 31), TOO_LARGE), (dict(num_pages=1 << 28), TOO_LARGE), (dict(heads=65535), TOO_LARGE),
])
def test_append_refuses(kw, rc):
    assert _append(**kw) == rc


def _attend(**kw):
    a = abi.PagedAttentionArgs()
    for p in ("q", "k_cache", "v_cache", "block_table", "kv_lens", "out"):
        setattr(a, p, AT)
    a.cache_dtype, a.out_dtype = abi.E4M3, abi.BF16
    a.requests, a.heads, a.kv_heads, a.dim, a.num_pages, a.page_size, a.table_width, a.table_stride = 3, 4, 2, 128, 8, 16, 4, 4
    for name, value in kw.items():
        setattr(a, name, value)
    return abi.lib.b200q_paged_attention(ctypes.byref(a))


@pytest.mark.parametrize("kw,rc", [
    (dict(requests=-1), BAD), (dict(heads=-4), BAD), (dict(kv_heads=0), BAD), (dict(heads=5), BAD), (dict(dim=0), BAD), (dict(num_pages=-1), BAD),
    (dict(page_size=0), BAD), (dict(table_width=-1), BAD), (dict(window=-1), BAD), (dict(cache_dtype=abi.F32), BAD), (dict(out_dtype=abi.E5M2), BAD),
    (dict(q=None), BAD), (dict(out=None), BAD), (dict(kv_lens=None), BAD), (dict(block_table=None), BAD), (dict(k_cache=None), BAD), (dict(v_cache=None), BAD),
    (dict(requests=8193), TOO_LARGE), (dict(requests=8192, table_width=1 << 18, page_size=16), TOO_LARGE), (dict(table_width=1 << 30, page_size=1 << 30), TOO_LARGE),
    (dict(kv_heads=128, heads=128 * 20, requests=1024, table_width=8192), TOO_LARGE), (dict(workspace=None), BAD), (dict(workspace=AT, workspace_bytes=1000), BAD),
    (dict(workspace=AT + 8, workspace_bytes=1 << 30), BAD),
    (dict(dim=257), UNSUPPORTED), (dict(num_pages=1 << 31), TOO_LARGE), (dict(page_size=1 << 31), TOO_LARGE), (dict(table_width=1 << 31), TOO_LARGE),
])
def test_attention_refuses(kw, rc):
    assert _attend(**kw) == rc


def test_nothing_to_do_is_no_error():
    assert _append(tokens=0) == 0 and _append(heads=0, kv_heads=0) == 0
    assert _attend(requests=0) == 0 and _attend(heads=0) == 0
    assert abi.lib.b200q_qk_norm_rope_append(None) == BAD and abi.lib.b200q_paged_attention(None) == BAD
    assert abi.lib.b200q_paged_attention_workspace_bytes(0, 8, 1, 128, abi.E4M3) == 0
    assert abi.lib.b200q_paged_attention_workspace_bytes(4, 8, 3, 128, abi.E4M3) == 0


def test_meta_kernels():
    m = lambda *s, dtype=BF16: torch.empty(*s, device="meta", dtype=dtype)  # noqa: E731
    i = lambda *s: m(*s, dtype=torch.int32)  # noqa: E731
    slots, positions, start, lens, head = torch.ops.b200q.paged_plan(i(5), i(5), i(5, 7), i(30), None, 16, 12)
    assert [(tuple(t.shape), t.dtype) for t in (slots, positions, start, lens, head)] == [
        ((12,), torch.int64), ((12,), torch.int64), ((6,), torch.int32), ((5,), torch.int32), ((1,), torch.int32)]
    kc, vc = m(30, 16, 2, 128, dtype=E4M3), m(30, 16, 2, 128, dtype=E4M3)
    q = torch.ops.b200q.qk_norm_rope_append(m(12, 8, 128), m(12, 2, 128), m(12, 2, 128), None, None, 1e-6, None, None, False, slots, kc, vc)
    assert q.shape == (12, 8, 128) and q.dtype == BF16
    q = torch.ops.b200q.qk_norm_rope_append(m(12, 8, 128), m(12, 2, 128), m(12, 2, 128), None, None, 1e-6, None, None, False, slots, kc, vc,
                                            q_dtype=E4M3)
    assert q.dtype == E4M3
    out, lse = torch.ops.b200q.paged_attention(m(5, 8, 128), kc, vc, i(5, 7), i(5), 0.1)
    assert out.shape == (5, 8, 128) and out.dtype == BF16 and lse.shape == (5, 8) and lse.dtype == F32
    assert torch.ops.b200q.paged_attention(m(5, 8, 128), kc, vc, i(5, 7), i(5), 0.1, out_dtype=F32)[0].dtype == F32


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        torch.ops.b200q.paged_plan(z, z, z.reshape(1, 1), z, None, 16, 1)


def test_oracle_plan_by_hand():
    ctx, new = torch.tensor([3, 0, 8], dtype=torch.int32), torch.tensor([3, 0, 1], dtype=torch.int32)
    table = torch.tensor([[7, -1, -1], [-1, -1, -1], [5, 6, -1]], dtype=torch.int32)
    slots, pos, start, lens, head, after = O.paged_plan(ctx, new, table, torch.tensor([9, 4, 1], dtype=torch.int32), None, 4, 6)
    assert slots.tolist() == [7 * 4 + 3, 9 * 4, 9 * 4 + 1, 4 * 4, -1, -1] and pos.tolist() == [3, 4, 5, 8, 0, 0]
    assert start.tolist() == [0, 3, 3, 4] and lens.tolist() == [6, 0, 9] and head.tolist() == [2]
    assert after.tolist() == [[7, 9, -1], [-1, -1, -1], [5, 6, 4]]


def test_oracle_rotation_is_a_rotation():
    x = torch.randn(5, 3, 16)
    a = torch.rand(32, 4, dtype=torch.float64) * 6
    table, pos = torch.cat([a.cos(), a.sin()], 1), torch.tensor([0, 3, 31, 7, 7])
    for inter in (False, True):
        y = O.norm_rope(x, None, 0.0, table, pos, inter)
        assert torch.equal(y[..., 8:], x[..., 8:].double())
        i, j = (2, 3) if inter else (1, 5)
        want = x[2, 1, i].double() * a[31, 1].cos() - x[2, 1, j].double() * a[31, 1].sin()
        assert abs(y[2, 1, i] - want) < 1e-14
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1))


def test_oracle_attention_against_dense():
    q, k, v = torch.randn(2, 4, 8), torch.randn(6, 4, 2, 8), torch.randn(6, 4, 2, 8)
    table, lens = torch.tensor([[3, 0, -1], [1, 5, 2]], dtype=torch.int32), torch.tensor([7, 12], dtype=torch.int32)
    out, lse, _ = O.paged_attention(q, k, v, table, lens, 0.3, 0.5, 2.0)
    for b, pages, n in ((0, [3, 0], 7), (1, [1, 5, 2], 12)):
        kk, vv = (t[pages].reshape(-1, 2, 8)[:n].double().repeat_interleave(2, 1) for t in (k, v))
        s = torch.einsum("hd,nhd->hn", q[b].double(), kk) * 0.15
        assert torch.allclose(lse[b], s.logsumexp(-1))
        assert torch.allclose(out[b], torch.einsum("hn,nhd->hd", s.softmax(-1), vv) * 2.0)
    assert math.isinf(O.paged_attention(q, k, v, table, torch.tensor([0, -3]), 0.3)[1].max())


def test_paged_attention_kernels_do_not_spill():
    """Nothing of the attention kernels lives in local memory (a step of theirs is some 200 instructions)."""
    import os
    import re
    from conftest import ROOT
    path = os.path.join(ROOT, "gaudi-pytorch-bridge_b200", "build", "paged_attention.ptxas")
    if not os.path.exists(path):
        pytest.skip("the kernels were not built in this tree")
    with open(path) as f:
        kernels = re.findall(r"Compiling entry function '(\S*paged\S*)'.*?\n.*?\n\s*(\d+) bytes stack frame, (\d+) bytes spill stores", f.read())
    assert len(kernels) > 15
    assert [k for k in kernels if k[1:] != ("0", "0")] == []
