"""A replaced model whose Seer gates have no weights, or not all of them, says so."""
from __future__ import annotations

import os
import warnings

import pytest
import torch

pytest.importorskip("transformers")

from compactattention_amd.load_attention_replacement import load_llama_attention_replacement_model  # noqa: E402
from tests.test_replacement_cpu import _stock  # noqa: E402


def test_gates_without_weights_warn(tmp_path):
    with pytest.warns(UserWarning, match="without gate weights"):
        r = load_llama_attention_replacement_model(base_model=_stock(), variant="seer_compactattn")
    state = {k: torch.randn_like(v) for k, v in r.state_dict().items() if ".attn_gate." in k}
    assert len(state) == 2
    path = os.path.join(tmp_path, "attn_gate_weights.pth")
    torch.save({k: state[k] for k in list(state)[:1]}, path)
    with pytest.warns(UserWarning, match="lacks 1 gate weights"):
        load_llama_attention_replacement_model(base_model=_stock(), variant="seer_compactattn", model_id=str(tmp_path))
    torch.save(state, path)
    with warnings.catch_warnings():
        warnings.simplefilter("error", UserWarning)
        got = load_llama_attention_replacement_model(base_model=_stock(), variant="seer_compactattn", model_id=path).state_dict()
        load_llama_attention_replacement_model(base_model=_stock(), variant="flashprefill_compactattn")
    assert all(torch.equal(got[k], v) for k, v in state.items())
