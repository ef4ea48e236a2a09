"""A folder stored in float16: both modes of the engine hold the four-bit weights of the numbers that it stores."""
import pytest
import torch

import tiny
from test_mxfp4_models_gpu import engine_of, logits_of, worst
from test_mxfp4_weights import restored

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["A", "B"])
def test_float16_folders(name, tmp_path):
    from flambeau_b200.kernels import ops
    cfg = tiny.CONFIGS[name]
    folder = tiny.make_folder(tmp_path / "m", cfg, seed=31, dtype="float32", sharp=0.1)
    stored = restored(folder, lambda n, t: t.half())
    narrow, wide = engine_of(folder, "bfloat16"), engine_of(folder, "float32")
    for i, (a, b) in enumerate(zip(narrow.model.layers, wide.model.layers)):
        def of(*names):
            return [stored[f"model.layers.{i}.{n}.weight"].float().cuda() for n in names]
        q, k, v, o = of(*(f"self_attn.{m}_proj" for m in "qkvo"))
        gate, up, down = of(*(f"mlp.{m}_proj" for m in ("gate", "up", "down")))
        pairs = [(a.mixer.qkv, b.mixer.qkv, torch.cat([q, k, v])), (a.mixer.o, b.mixer.o, o), (a.feed_forward.down, b.feed_forward.down, down),
                 (a.feed_forward.gate_up, b.feed_forward.gate_up, torch.stack([gate, up], 1).flatten(0, 1))]
        for packed, held, w in pairs:
            assert torch.equal(packed.weight.tiles, ops.Mxfp4Weight.from_dense(w).tiles)
            assert torch.equal(held.weight, ops.dequantize_mxfp4(*ops.quantize_mxfp4(w), w.shape[1]))
    requests = tiny.random_requests(cfg, [60, 17], seed=2)
    assert worst(logits_of(narrow, requests, 6), logits_of(wide, requests, 6)) <= tiny.TOL["bfloat16"]
