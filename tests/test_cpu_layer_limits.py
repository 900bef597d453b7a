"""The norm, the adapters and the experts, without a GPU: what their self-tests, and they themselves, refuse before any CUDA call."""
import ctypes

import pytest
import torch

from b200_hpu_ops import abi
from test_cpu_layer import AT, BAD, UNSUPPORTED, _call, _lora, _norm

SOME = 1 << 40  # bytes of a workspace that nothing reads
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would reach the GPU")


def _moe_selftest(lost=0, **kw):
    a = abi.MoeArgs()
    a.x, a.router, a.gate_up, a.down, a.out, a.weights, a.ids, a.workspace = (AT,) * 8
    a.router_dtype, a.weight_dtype, a.out_dtype = abi.BF16, abi.E4M3, abi.BF16
    a.tokens, a.hidden, a.inner, a.experts, a.top_k, a.x_stride, a.workspace_bytes = 45, 64, 32, 8, 2, 64, SOME
    return _call(lambda p: abi.lib.b200q_selftest_moe_wait_timeout(p, lost), a, kw)


@pytest.mark.parametrize("kw,rc", [(dict(lost=-1), BAD), (dict(lost=4), BAD), (dict(workspace=None), BAD), (dict(workspace_bytes=100), BAD), (dict(tokens=-1), BAD), (dict(tokens=0), BAD),
                                   (dict(tokens=44), UNSUPPORTED), (dict(tokens=257), UNSUPPORTED), (dict(weight_dtype=abi.BF16), UNSUPPORTED), (dict(router_dtype=abi.F32), UNSUPPORTED),
                                   (dict(force_plain=1), UNSUPPORTED), (dict(hidden=40), UNSUPPORTED)])
def test_moe_selftest_refuses(kw, rc):
    assert _moe_selftest(**kw) == rc


def test_selftests_refuse_nothing():
    assert abi.lib.b200q_selftest_moe_wait_timeout(ctypes.POINTER(abi.MoeArgs)(), 0) == BAD


def _lora_selftest(lost=0, **kw):
    a = abi.LoraArgs()
    a.x, a.y, a.a, a.b, a.adapter, a.workspace = AT, AT << 4, AT << 5, AT << 6, AT, AT
    a.y_dtype = abi.BF16
    a.tokens, a.k, a.n, a.rank, a.adapters = 3, 64, 32, 16, 2
    a.x_stride, a.y_stride, a.a_stride, a.a_row_stride, a.b_stride, a.b_row_stride, a.workspace_bytes = 64, 32, 1024, 64, 512, 16, SOME
    return _call(lambda p: abi.lib.b200q_selftest_lora_wait_timeout(p, lost), a, kw)


@pytest.mark.parametrize("kw,rc", [(dict(lost=-1), BAD), (dict(lost=2), BAD), (dict(workspace=None), BAD), (dict(workspace_bytes=100), BAD), (dict(tokens=-1), BAD), (dict(tokens=0), BAD),
                                   (dict(rank=0), BAD), (dict(tokens=2048, rank=136, a_stride=136 * 64, b_row_stride=136, b_stride=136 * 32), UNSUPPORTED), (dict(tokens=8193), UNSUPPORTED), (dict(y_dtype=abi.F32), UNSUPPORTED),
                                   (dict(y=(AT << 4) + 2), UNSUPPORTED), (dict(force_plain=1), UNSUPPORTED), (dict(rank=12), UNSUPPORTED)])
def test_lora_selftest_refuses(kw, rc):
    assert _lora_selftest(**kw) == rc


def test_lora_selftest_refuses_nothing():
    assert abi.lib.b200q_selftest_lora_wait_timeout(ctypes.POINTER(abi.LoraArgs)(), 0) == BAD


def _norm_selftest(**kw):
    a = abi.NormArgs()
    a.x, a.weight, a.out = AT, AT, AT
    a.x_dtype, a.weight_dtype, a.out_dtype = abi.BF16, abi.BF16, abi.E4M3
    a.tokens, a.dim, a.x_stride, a.residual_stride = 149, 8192, 8192, 8192
    return _call(abi.lib.b200q_selftest_norm_wait_timeout, a, kw)


@pytest.mark.parametrize("kw,rc", [(dict(tokens=-1), BAD), (dict(tokens=0), BAD), (dict(dim=0), BAD), (dict(x=None), BAD), (dict(tokens=148), UNSUPPORTED), (dict(dim=4096), UNSUPPORTED),
                                   (dict(dim=8200, x_stride=8200), UNSUPPORTED), (dict(dim=8191, x_stride=8191), UNSUPPORTED), (dict(x_dtype=abi.F32), UNSUPPORTED), (dict(x=AT + 8), UNSUPPORTED)])
def test_norm_selftest_refuses(kw, rc):
    assert _norm_selftest(**kw) == rc


def test_norm_selftest_refuses_nothing():
    assert abi.lib.b200q_selftest_norm_wait_timeout(ctypes.POINTER(abi.NormArgs)()) == BAD


@pytest.mark.parametrize("kw", [dict(residual=AT + 64, weight=AT, x=AT << 6), dict(residual=(AT << 4), weight=(AT << 4) + 3 * 128 - 2), dict(residual=AT << 4, scale=(AT << 4) + 256, out_dtype=abi.BF16),
                                dict(residual=AT << 4, weight=(AT << 4) + 380, weight_dtype=abi.F32)])
def test_norm_refuses_to_write_its_inputs(kw):
    assert _norm(**kw) == BAD


@pytest.mark.parametrize("kw", [dict(x=(AT << 4) + 190), dict(a=(AT << 4) - 2 * 2 * 16 * 64 + 2), dict(b=(AT << 4) + 64), dict(adapter=(AT << 4) + 188), dict(scales=(AT << 4) + 100),
                                dict(y_stride=40, scales=(AT << 4) + 72), dict(x=(AT << 4) - 32 * 2, x_stride=0), dict(x=(AT << 4) + 64, x_stride=32)])
def test_lora_refuses_to_write_its_inputs(kw):
    assert _lora(workspace=AT, workspace_bytes=SOME, force_plain=1, **kw) == BAD
