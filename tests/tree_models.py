"""Models for the tests of drafted trees and shortened caches whose layers differ in what a configuration file cannot say."""
import dataclasses
import importlib

import torch

from conftest import TINY_LLAMA


def two_value_sizes(cfg, sizes, *, dtype, device, ops, seed=7, std=0.15):
    """A model of ``cfg``'s design whose layer i has values of ``sizes[i]`` elements, and random weights."""
    model_of = importlib.import_module("daisi-llogos_b200.engine.model").DecoderModel
    loader = importlib.import_module("daisi-llogos_b200.weights.loader")
    spec = loader.build_model(cfg, dtype=dtype, device="cpu", ops=ops).spec
    layers = []
    for layer, size in zip(spec.layers, sizes):
        mixer = layer.parts["mixer"]
        parts = dict(layer.parts, mixer=dataclasses.replace(mixer, params=dict(mixer.params, value_dim=size)))
        layers.append(dataclasses.replace(layer, parts=parts))
    model = model_of(dataclasses.replace(spec, layers=tuple(layers)), dtype=dtype, device=torch.device(device), ops=ops)
    made = loader.random_tensors(model.tensor_decls(), seed, std=std, dtype=torch.bfloat16, device="cpu")
    model.bind({name: t.to(device=device, dtype=torch.float32 if dtype == torch.float32 else t.dtype) for name, t in made.items()})
    return model


CFG = dict(TINY_LLAMA, head_dim=64, hidden_size=256, num_attention_heads=4, num_key_value_heads=2)
