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
