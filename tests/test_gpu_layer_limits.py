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
