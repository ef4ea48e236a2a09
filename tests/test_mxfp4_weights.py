"""What the loader hands to the maps that a runtime holds in four bits (CPU)."""
import warnings

import pytest
import torch

import tiny
from flambeau_b200.config.mistral import MistralConfig
from flambeau_b200.weights.loader import load_tensors
from flambeau_b200.weights.random_init import model_tensor_specs, write_random_model
from test_weights import FakeRuntime

MAPS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


class PackingRuntime(FakeRuntime):
    weight_format = "mxfp4"


def is_map(name):
    return any(m in name for m in MAPS)


def loaded(folder, specs, runtime):
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        got = load_tensors(folder, specs, runtime)
    return got, [str(w.message) for w in seen]


def test_the_large_maps_say_that_they_pack():
    specs = model_tensor_specs(MistralConfig.from_dict(tiny.CONFIGS["A"]))
    assert {n for n, s in specs.items() if s.packs} == {n for n in specs if is_map(n)} != set()


def test_maps_that_are_packed_are_not_warned_about(tmp_path):
    """A map stored in 32 bits does not stay so where it is packed: no product with it runs on the float32 FMA kernel."""
    cfg = MistralConfig.from_dict(tiny.CONFIGS["A"])
    write_random_model(tmp_path / "m", cfg, seed=1, dtype="bfloat16", float32_names=MAPS)
    specs = model_tensor_specs(cfg)
    assert loaded(tmp_path / "m", specs, PackingRuntime())[1] == []
    assert len(loaded(tmp_path / "m", specs, FakeRuntime())[1]) == 1
    write_random_model(tmp_path / "f32", cfg, seed=1, dtype="float32")
    said = loaded(tmp_path / "f32", specs, PackingRuntime())[1]
    assert len(said) == 1 and not is_map(said[0]) and "32-bit" in said[0]            # (the embedding or the head, which stay)


def restored(folder, change):
    """The folder's tensors through `change` (name, tensor) and back into it."""
    from flambeau_b200.weights.safetensors_io import SafetensorsFile, write_safetensors
    f = SafetensorsFile(folder / "model.safetensors")
    tensors = {n: change(n, f.tensor(n).clone()) for n in f.names()}
    f.close()
    write_safetensors(folder / "model.safetensors", tensors)
    return tensors


@pytest.mark.parametrize("full_precision", [False, True])
def test_maps_come_with_the_bits_that_they_are_stored_with(tmp_path, full_precision):
    """float16 has three bits more than bfloat16: a map is quantised from them in both modes, so that both have the same numbers."""
    cfg = MistralConfig.from_dict(tiny.CONFIGS["A"])
    write_random_model(tmp_path, cfg, seed=2, dtype="float32")
    stored = restored(tmp_path, lambda n, t: t.half())
    got, said = loaded(tmp_path, model_tensor_specs(cfg), PackingRuntime(full_precision))
    for n, t in stored.items():
        if is_map(n):
            assert got[n].dtype == torch.float32 and torch.equal(got[n], t.float())
        else:
            assert got[n].dtype == (torch.float32 if full_precision else torch.bfloat16)
    assert said == []


@pytest.mark.parametrize("kinds", [("half", "bfloat16"), ("bfloat16", "float"), ("bfloat16", "bfloat16")])
def test_maps_of_one_part_come_in_one_dtype(tmp_path, kinds):
    """What a part stacks may be stored in several types."""
    cfg = MistralConfig.from_dict(tiny.CONFIGS["A"])
    write_random_model(tmp_path, cfg, seed=3, dtype="float32")
    stored = restored(tmp_path, lambda n, t: getattr(t, kinds[0] if "q_proj" in n or "gate_proj" in n else kinds[1])())
    got, _ = loaded(tmp_path, model_tensor_specs(cfg), PackingRuntime())
    want = torch.bfloat16 if set(kinds) == {"bfloat16"} else torch.float32
    for n, t in stored.items():
        if is_map(n):
            assert got[n].dtype == want and torch.equal(got[n].float(), t.float())


def test_the_benchmark_takes_the_weight_format(capsys):
    from flambeau_b200.cli import main
    assert main(["bench", "--gpus", "4", "--weights", "mxfp4"]) == 2
    assert "one GPU" in capsys.readouterr().out
    with pytest.raises(SystemExit):
        main(["bench", "--weights", "int4"])
