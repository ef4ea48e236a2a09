"""Four-bit weights beside another current device: refused before anything is launched (the addresses are none of that device's)."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_another_current_device_is_refused(monkeypatch):
    from flambeau_b200.engine.runtime import Runtime
    from flambeau_b200.kernels import ops
    from flambeau_b200.kernels.library import KernelError
    rt = Runtime("cuda:0", "bfloat16")
    ctx = SimpleNamespace(runtime=rt, ws=rt.ws)
    x = torch.randn(64, 96, device="cuda")
    codes, scales = ops.quantize_mxfp4(x)
    w, stack = ops.Mxfp4Weight(codes, scales, 96), ops.Mxfp4Weight(codes.view(2, 32, 48), scales.view(2, 32, 3), 96)
    a, out = torch.randn(16, 96, device="cuda").bfloat16(), torch.full((16, 64), 7.0, device="cuda")
    slabs = torch.empty(2, 16, 64, device="cuda")
    group = torch.zeros(1, dtype=torch.int32, device="cuda")
    index = torch.arange(16, dtype=torch.int32, device="cuda")
    calls = [lambda: ops.quantize_mxfp4(x), lambda: ops.dequantize_mxfp4(codes, scales, 96), lambda: ops.Mxfp4Weight(codes, scales, 96),
             lambda: ops.linear(a, w, out, ctx), lambda: ops.gated_linear(a, w, out[:, :32], "silu", ctx),
             lambda: ops.activated_linear(a, w, out, "gelu", ctx), lambda: ops.linear_slabs(a, w, slabs, ctx),
             lambda: ops.grouped_linear(a, index, stack, group, 16, out[:, :32], None, ctx),
             lambda: ops.grouped_gated_linear(a, None, stack, group, 16, out[:, :16], "silu", ctx)]
    top = rt.ws.top
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "current_device", lambda: 1)
        for i, call in enumerate(calls):
            with pytest.raises(KernelError, match="current device is cuda:1"):
                call()
                pytest.fail(f"call {i} was not refused")
    assert rt.ws.top == top and bool((out == 7.0).all())
    for call in calls:                           # each is in order on its own device
        call()
    # a step's scratch elsewhere (the check looks at its device alone)
    elsewhere = SimpleNamespace(runtime=rt, ws=SimpleNamespace(counters=torch.zeros(8, dtype=torch.int32)))
    for call in (lambda: ops.linear(a, w, out, elsewhere), lambda: ops.grouped_linear(a, index, stack, group, 16, out[:, :32], None, elsewhere)):
        with pytest.raises(KernelError, match="the step's scratch"):
            call()
    rt.check_status()
