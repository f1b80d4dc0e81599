"""Room for the adapters that ``LLM`` is given, without a GPU."""

from __future__ import annotations

import json

import pytest
import torch

from miniserve_b200.engine import llm as llm_module


class Engine:
    def __init__(self, model, **kwargs):
        self.kwargs, self.loaded = kwargs, []

    def load_adapter(self, name, source):
        self.loaded.append(name)


def folder(path, **config):
    path.mkdir()
    (path / "adapter_config.json").write_text(json.dumps(config))
    return path


def made(monkeypatch, adapters, **kwargs):
    monkeypatch.setattr(llm_module, "Engine", Engine)
    return llm_module.LLM(random="tiny-b", dtype="float32", device="cpu", adapters=adapters, **kwargs).engine


def test_there_is_room_for_the_ranks_of_the_folders(tmp_path, monkeypatch):
    narrow, wide = folder(tmp_path / "narrow", r=4), folder(tmp_path / "wide", r=32)
    tensors = {"a.lora_A.weight": torch.zeros((24, 8)), "a.lora_B.weight": torch.zeros((99, 24))}
    room = lambda adapters, **kw: [made(monkeypatch, adapters, **kw).kwargs[k] for k in ("max_adapters", "max_adapter_rank")]  # noqa: E731
    assert room({"n": narrow}) == [1, 16] and room({"n": narrow, "w": str(wide)}) == [2, 32] and room({"t": tensors}) == [1, 24]
    assert room({"w": wide}, max_adapters=5, max_adapter_rank=64) == [5, 64] and room({"w": wide}, max_adapters=1, max_adapter_rank=16) == [1, 32]
    engine = made(monkeypatch, {"n": narrow, "w": wide})
    assert engine.loaded == ["n", "w"]
    assert "max_adapters" not in made(monkeypatch, None, max_running=4).kwargs


def test_a_folder_without_a_rank_is_refused_before_anything_is_built(tmp_path, monkeypatch):
    monkeypatch.setattr(llm_module, "random_model", lambda *a, **kw: pytest.fail("the model was built"))
    for config in (dict(), dict(r=None), dict(r="many")):
        path = tmp_path / f"bad{len(list(tmp_path.iterdir()))}"
        with pytest.raises(ValueError, match="no rank"):
            made(monkeypatch, {"bad": folder(path, **config)})
    with pytest.raises(FileNotFoundError, match="adapter_config"):
        made(monkeypatch, {"none": tmp_path / "nowhere"})
