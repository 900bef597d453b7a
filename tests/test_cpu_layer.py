"""The norm before, the adapters beside and the experts in place of the FP8 products, without a GPU: what the C ABI refuses before any CUDA call,
the schemas and Meta kernels, and the oracle against dense definitions."""
import ctypes

import pytest
import torch

from b200_hpu_ops import abi
from oracle import hpu_oracle as O

E4M3, E5M2, BF16, F32 = torch.float8_e4m3fn, torch.float8_e5m2, torch.bfloat16, torch.float32
BAD, UNSUPPORTED, TOO_LARGE = -1, -2, -4
AT = 1 << 20  # an address that nothing reads


def test_layouts_of_the_argument_structs():
    for i, args in enumerate((abi.NormArgs, abi.LoraArgs, abi.MoeArgs)):
        assert abi.lib.b200q_sizeof_args(4 + i) == ctypes.sizeof(args)


def _call(function, a, kw):
    for name, value in kw.items():
        setattr(a, name, value)
    return function(ctypes.byref(a))


def _norm(**kw):
    a = abi.NormArgs()
    a.x, a.weight, a.out = AT, AT, AT
    a.x_dtype, a.weight_dtype, a.out_dtype = abi.BF16, abi.BF16, abi.E4M3
    a.tokens, a.dim, a.x_stride, a.residual_stride = 3, 64, 64, 64
    return _call(abi.lib.b200q_add_rms_norm_cast, a, kw)


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=-1), BAD), (dict(dim=-1), BAD), (dict(x=None), BAD), (dict(out=None), BAD), (dict(x_dtype=abi.E4M3), BAD), (dict(out_dtype=abi.F32), BAD),
    (dict(weight_dtype=abi.E5M2), BAD), (dict(scale=AT, scale_inv=AT), BAD), (dict(scale_inv=AT, out_dtype=abi.BF16), BAD),
    (dict(residual=AT << 4, residual_stride=63), BAD), (dict(residual=AT), BAD), (dict(residual=AT + 128), BAD), (dict(residual=AT + 64, residual_stride=96, x_stride=96), BAD),
    (dict(tokens=1 << 31), TOO_LARGE), (dict(dim=1 << 31), TOO_LARGE),
    (dict(x=AT + 1), UNSUPPORTED), (dict(residual=(AT << 4) + 1), UNSUPPORTED), (dict(weight=AT + 1), UNSUPPORTED), (dict(kept=AT + 1), UNSUPPORTED),
    (dict(scale=AT + 2), UNSUPPORTED), (dict(scale_inv=AT + 2), UNSUPPORTED), (dict(out=AT + 1, out_dtype=abi.BF16), UNSUPPORTED),
    (dict(tokens=0), 0), (dict(dim=0), 0),
])
def test_norm_refuses(kw, rc):
    assert _norm(**kw) == rc


def _lora(**kw):
    a = abi.LoraArgs()
    a.x, a.y, a.a, a.b, a.adapter, a.workspace = AT, AT << 4, AT << 5, AT << 6, AT, AT
    a.y_dtype = abi.BF16
    a.tokens, a.k, a.n, a.rank, a.adapters = 3, 64, 32, 16, 2
    a.x_stride, a.y_stride, a.a_stride, a.a_row_stride, a.b_stride, a.b_row_stride = 64, 32, 1024, 64, 512, 16
    a.workspace_bytes = 0  # (what is not refused before stops here)
    return _call(abi.lib.b200q_lora_add, a, kw)


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=-1), BAD), (dict(k=-1), BAD), (dict(n=-1), BAD), (dict(rank=-1), BAD), (dict(adapters=-1), BAD), (dict(y_dtype=abi.E4M3), BAD), (dict(y_stride=31), BAD),
    (dict(x=None), BAD), (dict(y=None), BAD), (dict(a=None), BAD), (dict(b=None), BAD), (dict(adapter=None), BAD), (dict(), BAD), (dict(workspace=None), BAD),
    (dict(workspace=AT + 8, workspace_bytes=1 << 40), BAD),
    (dict(rank=257), TOO_LARGE), (dict(adapters=2049), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE), (dict(k=1 << 31), TOO_LARGE),
    (dict(n=1 << 31, y_stride=1 << 31), TOO_LARGE),
    (dict(x=AT + 1), UNSUPPORTED), (dict(a=AT + 1), UNSUPPORTED), (dict(b=AT + 1), UNSUPPORTED), (dict(y=AT + 1), UNSUPPORTED), (dict(y=AT + 2, y_dtype=abi.F32), UNSUPPORTED),
    (dict(adapter=AT + 2), UNSUPPORTED), (dict(scales=AT + 2), UNSUPPORTED),
    (dict(tokens=0), 0), (dict(k=0), 0), (dict(n=0), 0), (dict(rank=0), 0), (dict(adapters=0), 0),
])
def test_lora_refuses(kw, rc):
    assert _lora(**kw) == rc


def _moe(**kw):
    a = abi.MoeArgs()
    a.x, a.router, a.gate_up, a.down, a.out, a.weights, a.ids, a.workspace = (AT,) * 8
    a.router_dtype, a.weight_dtype, a.out_dtype = abi.BF16, abi.E4M3, abi.BF16
    a.tokens, a.hidden, a.inner, a.experts, a.top_k, a.x_stride = 3, 64, 32, 8, 2, 64
    a.workspace_bytes = 0
    return _call(abi.lib.b200q_moe_layer, a, kw)


@pytest.mark.parametrize("kw,rc", [
    (dict(tokens=-1), BAD), (dict(hidden=-1), BAD), (dict(inner=-1), BAD), (dict(experts=0), BAD), (dict(top_k=0), BAD), (dict(top_k=9), BAD),
    (dict(router_dtype=abi.E4M3), BAD), (dict(weight_dtype=abi.E5M2), BAD), (dict(weight_dtype=abi.F32), BAD), (dict(out_dtype=abi.E4M3), BAD),
    (dict(x=None), BAD), (dict(router=None), BAD), (dict(gate_up=None), BAD), (dict(down=None), BAD), (dict(out=None), BAD), (dict(weights=None), BAD), (dict(ids=None), BAD),
    (dict(), BAD), (dict(workspace=None), BAD), (dict(workspace=AT + 8, workspace_bytes=1 << 40), BAD),
    (dict(experts=513), TOO_LARGE), (dict(experts=32, top_k=17), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE), (dict(hidden=1 << 31), TOO_LARGE), (dict(inner=1 << 30), TOO_LARGE),
    (dict(x=AT + 1), UNSUPPORTED), (dict(router=AT + 1), UNSUPPORTED), (dict(router=AT + 2, router_dtype=abi.F32), UNSUPPORTED), (dict(gate_up=AT + 1, weight_dtype=abi.BF16), UNSUPPORTED),
    (dict(down=AT + 1, weight_dtype=abi.BF16), UNSUPPORTED), (dict(out=AT + 1), UNSUPPORTED), (dict(gate_up_scale=AT + 2), UNSUPPORTED), (dict(down_scale=AT + 2), UNSUPPORTED),
    (dict(num_tokens=AT + 2), UNSUPPORTED), (dict(weights=AT + 2), UNSUPPORTED), (dict(ids=AT + 2), UNSUPPORTED), (dict(tokens=0), 0),
])
def test_moe_refuses(kw, rc):
    assert _moe(**kw) == rc


def test_workspaces():
    assert abi.lib.b200q_lora_workspace_bytes(0, 64, 64, 16, 2) == 0 == abi.lib.b200q_lora_workspace_bytes(4, 64, 64, 257, 2)
    assert abi.lib.b200q_lora_workspace_bytes(4, 64, 64, 16, 2) >= 4 * 16 * 4
    assert abi.lib.b200q_moe_workspace_bytes(0, 64, 64, 16, 2) == 0 == abi.lib.b200q_moe_workspace_bytes(4, 64, 64, 513, 2)
    assert abi.lib.b200q_moe_workspace_bytes(4, 64, 32, 16, 2) >= 4 * 2 * (64 + 32) * 4


@pytest.mark.parametrize("adapters", [1, 40, 85, 300])
@pytest.mark.parametrize("last", [1, 100, 4000, 7936])
def test_lora_workspace_holds_the_last_tokens_of_a_long_call(adapters, last):
    bytes_of = abi.lib.b200q_lora_workspace_bytes
    for whole in (8192, 3 * 8192):
        assert bytes_of(whole + last, 4096, 64, 64, adapters) >= max(bytes_of(8192, 4096, 64, 64, adapters), bytes_of(last, 4096, 64, 64, adapters))


def test_schemas_and_meta():
    m = dict(device="meta")
    x = torch.empty(5, 64, dtype=BF16, **m)
    ops = torch.ops.b200q
    for dtype, scale, keep in ((E4M3, None, True), (E5M2, torch.empty((), **m), False), (BF16, None, False)):
        out, inv, kept = ops.add_rms_norm_cast(x, torch.empty_like(x), None, 1e-6, dtype, scale, keep)
        assert out.shape == x.shape and out.dtype == dtype
        assert inv.shape == ((5, 1) if dtype == E4M3 else (0,)) and inv.dtype == F32
        assert kept.shape == (x.shape if keep else (0,)) and kept.dtype == BF16
    y = torch.empty(5, 32, **m)
    assert ops.lora_add_(y, x, torch.empty(2, 8, 64, dtype=BF16, **m), torch.empty(2, 32, 8, dtype=BF16, **m), torch.empty(5, dtype=torch.int32, **m)) is y
    w = dict(dtype=E4M3, **m)
    for dtype in (None, F32):
        out, weights, ids = ops.moe_layer(x, torch.empty(4, 64, **m), torch.empty(4, 64, 64, **w), torch.empty(4, 64, 32, **w), None, None, 2, out_dtype=dtype)
        assert out.shape == x.shape and out.dtype == (dtype or BF16) and weights.shape == ids.shape == (5, 2) and (weights.dtype, ids.dtype) == (F32, torch.int32)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 16, dtype=BF16)
    with pytest.raises(NotImplementedError):
        torch.ops.b200q.add_rms_norm_cast(x, None, None, 1e-6, E4M3)
    with pytest.raises(NotImplementedError):
        torch.ops.b200q.lora_add_(x, x, x[None], x[None], torch.zeros(2, dtype=torch.int32))
    with pytest.raises(NotImplementedError):
        torch.ops.b200q.moe_layer(x, x, x[None], x[None], None, None, 1)


# ----------------------------------------------------------------------------- the oracle
def test_oracle_norm():
    g = torch.Generator().manual_seed(1)
    x, r, w = torch.randn(4, 33, generator=g), torch.randn(4, 33, generator=g), torch.randn(33, generator=g)
    z, y = O.add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(z, r + x)
    assert torch.allclose(y, torch.nn.functional.rms_norm(z.double(), (33,), w.double(), 1e-5), rtol=1e-12)
    assert torch.allclose(O.add_rms_norm(x, None, None, 0.0)[1].square().mean(-1), torch.ones(4, dtype=torch.float64))


def test_oracle_lora_is_a_merged_weight():
    g = torch.Generator().manual_seed(2)
    x, w, a, b = (torch.randn(*s, generator=g).double() for s in ((3, 10), (7, 10), (2, 4, 10), (2, 7, 4)))
    which, scales = torch.tensor([1, -1, 0]), torch.tensor([0.5, 2.0])
    got, size, live = O.lora_add(x @ w.T, x, a, b, which, scales)
    for t in range(3):
        merged = w if which[t] < 0 else w + float(scales[which[t]]) * b[which[t]] @ a[which[t]]
        assert torch.allclose(got[t], merged @ x[t], rtol=1e-12)
    assert live.tolist() == [True, False, True] and bool((size[1] == 0).all()) and bool((size[0] >= (got[0] - x[0] @ w.T).abs()).all())


def test_oracle_route():
    x = torch.eye(3)
    clean = torch.tensor([[0.0, 3.0, 3.0, 2.0], [1.0, 1.0, 1.0, 1.0], [-5.0, -6.0, -7.0, -4.0]])
    weights, ids = O.moe_route(x, clean.T.contiguous(), 2, True)
    assert ids.tolist() == [[1, 2], [0, 1], [3, 0]]
    assert torch.allclose(weights.sum(-1), torch.ones(3, dtype=torch.float64))
    weights, ids = O.moe_route(x, clean.T.contiguous(), 3, False, count=2)
    assert ids.tolist() == [[1, 2, 3], [0, 1, 2], [-1, -1, -1]] and bool((weights[2] == 0).all())
    assert torch.allclose(weights[1], torch.full((3,), 0.25, dtype=torch.float64))
    y = torch.tensor([[float("nan")], [1.0]])
    assert O.moe_route(y, torch.ones(3, 1), 2, True)[1].tolist() == [[0, 1], [0, 1]]


def test_oracle_experts_against_dense_sums():
    g = torch.Generator().manual_seed(3)
    e, h, f = 5, 12, 6
    x, router, gu, down = (torch.randn(*s, generator=g) for s in ((4, h), (e, h), (e, 2 * f, h), (e, h, f)))
    s1, s2 = torch.rand(e, 2 * f, generator=g), torch.rand(e, h, generator=g)
    weights, ids = O.moe_route(x, router, e, False)  # all experts: the dense mixture
    out, bound = O.moe_experts(x, weights, ids, gu, down, s1, s2)
    p = torch.softmax(x.double() @ router.double().T, -1)
    mid = torch.einsum("th,efh->tef", x.double(), gu.double()) * s1.double()
    hid = torch.nn.functional.silu(mid[..., :f]) * mid[..., f:]
    want = torch.einsum("te,tef,ehf,eh->th", p, hid, down.double(), s2.double())
    assert torch.allclose(out, want, rtol=1e-10) and bool((bound >= 0).all())
