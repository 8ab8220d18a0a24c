"""Models for the tests of drafted trees and shortened caches whose layers differ in what a configuration file cannot say."""
import dataclasses
import importlib

import torch

from conftest import TINY_LLAMA


def two_value_sizes(cfg, sizes, **kw):
    """A model of ``cfg``'s design whose layer i has values of ``sizes[i]`` elements, and random weights."""
    return with_mixers(cfg, [dict(value_dim=size) for size in sizes], **kw)


def with_mixers(cfg, changes, *, dtype, device, ops, seed=7, std=0.15, cache_of=()):
    """A model of ``cfg``'s design with the parameters ``changes[i]`` for layer i's attention, and random weights.  ``cache_of``: (entry, the
    earlier one whose cache it reads)."""
    model_of = importlib.import_module("daisi-llogos_b200.engine.model").DecoderModel
    loader = importlib.import_module("daisi-llogos_b200.weights.loader")
    spec = loader.build_model(cfg, dtype=dtype, device="cpu", ops=ops).spec
    layers = []
    for layer, change in zip(spec.layers, changes):
        mixer = layer.parts["mixer"]
        parts = dict(layer.parts, mixer=dataclasses.replace(mixer, params=dict(mixer.params, **change)))
        layers.append(dataclasses.replace(layer, parts=parts))
    schedule = [dataclasses.replace(e, cache_of=dict(cache_of).get(i, e.cache_of)) for i, e in enumerate(spec.schedule)]
    model = model_of(dataclasses.replace(spec, layers=tuple(layers), schedule=tuple(schedule)), dtype=dtype, device=torch.device(device), ops=ops)
    made = loader.random_tensors(model.tensor_decls(), seed, std=std, dtype=torch.bfloat16, device="cpu")
    model.bind({name: t.to(device=device, dtype=torch.float32 if dtype == torch.float32 else t.dtype) for name, t in made.items()})
    return model


CFG = dict(TINY_LLAMA, head_dim=64, hidden_size=256, num_attention_heads=4, num_key_value_heads=2)
