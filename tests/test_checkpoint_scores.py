"""A checkpoint of a model with capped or biased scores is rebuilt with them: its state dict is the
plain model's, so only the stored configuration tells them apart."""

from __future__ import annotations

import dataclasses
import json

import pytest
import torch
from safetensors.torch import save_file

from local_ai_training.generate import generate, load_for_generation
from local_ai_training.model import ModelConfig, build_seeded_model

LETTERS = tuple(chr(48 + i) for i in range(40))


@pytest.mark.parametrize("kw", [{}, {"attention_softcap": 0.5}, {"distance_bias": True},
                                {"attention_softcap": 0.5, "distance_bias": True}])
@pytest.mark.parametrize("stored", ["all", "given"])
def test_the_loaded_model_computes_what_was_trained(tmp_path, kw, stored):
    shape = dict(block_size=32, n_layer=2, n_head=2, n_embd=32)
    config = ModelConfig(vocab_size=40, **shape, **kw)
    model = build_seeded_model(config, max_code=2, seed=4).eval()
    fields = dataclasses.asdict(config) if stored == "all" else {**shape, **kw}
    (tmp_path / "step.json").write_text(json.dumps({
        "max_code": 2, "vocabulary": LETTERS, "experiment_config": fields}))
    save_file({"model::" + name: t.contiguous() for name, t in model.state_dict().items()},
              tmp_path / "step.safetensors")
    loaded, letters = load_for_generation(tmp_path / "step")
    assert letters == LETTERS
    tokens = torch.randint(0, 40, (2, 24), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        assert torch.equal(loaded(tokens)[0], model(tokens)[0])
    texts = [generate(m, LETTERS, "0123", max_new_tokens=8, temperature=0.0)
             for m in (model, loaded)]
    assert texts[0] == texts[1]
