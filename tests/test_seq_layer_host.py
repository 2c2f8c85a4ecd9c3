"""GatedDeltaMixer as a module, without a GPU."""
import copy

import torch

import tdc_sequence as S

SHAPE = dict(key_dim=64, value_dim=64, rotary_dim=32, max_positions=20)


def test_layer_made_on_the_meta_device():
    # to_empty leaves parameters to the state dict; the tables are not in it and are made again
    want = S.GatedDeltaMixer(64, 1, **SHAPE)
    m = S.GatedDeltaMixer(64, 1, device="meta", **SHAPE)
    assert m.cos.is_meta
    m = m.to(torch.float16)                                   # still without memory
    assert m.cos.is_meta and m.cos.dtype == torch.float32
    m = m.to_empty(device="cpu")
    m.load_state_dict(want.state_dict())
    assert torch.equal(m.cos, want.cos) and torch.equal(m.sin, want.sin)
    assert torch.equal(m.in_proj.weight.float(), want.in_proj.weight.half().float())


def test_tables_of_copies_and_moves():
    want = S.GatedDeltaMixer(64, 1, **SHAPE)
    for m in (copy.deepcopy(want), copy.deepcopy(want).half(), copy.deepcopy(want).to_empty(device="cpu")):
        assert torch.equal(m.cos, want.cos) and torch.equal(m.sin, want.sin)
