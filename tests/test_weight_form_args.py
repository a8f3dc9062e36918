"""Arguments that would name a form of weights or rows and change nothing: refused, wherever they are given."""
import pytest
import torch

import tiny
from arle_amd import models  # noqa: F401
from arle_amd.config.registry import detect_architecture
from arle_amd.engine import Engine, EngineError
from arle_amd.engine import engine as engine_module
from arle_amd.engine.api import LLM
from arle_amd.parts.base import Runtime


def _spec():
    qwen3 = detect_architecture({"architectures": [tiny.ARCH]})
    return qwen3.recipe(qwen3.config_class.from_dict(tiny.TINY["A"][0]), ())


@pytest.mark.parametrize("args", [dict(row_form="mxfp4"), dict(row_form="mxfp16"), dict(weight_form="mxfp4", row_form="mxfp16"), dict(weight_form="mxfp8")])
def test_an_engine_refuses_forms_that_it_would_not_use(args, monkeypatch):
    monkeypatch.setattr(engine_module, "_device", lambda device: torch.device("cpu"))
    with pytest.raises(EngineError, match="row_form|weight_form"):
        Engine(_spec(), {}, **args)


def test_an_engine_that_is_built_keeps_its_forms():
    engine = object.__new__(Engine)
    for held in ((None, "mxfp8"), ("mxfp4", "mxfp8"), ("mxfp4", "mxfp4")):
        engine.rt = Runtime(device=torch.device("cpu"), act_dtype=torch.bfloat16, weight_form=held[0], row_form=held[1])
        for asked in (dict(weight_form="mxfp4"), dict(weight_form="mxfp4", row_form="mxfp4"), dict(row_form="mxfp4")):
            if held == (asked.get("weight_form"), asked.get("row_form", "mxfp8")):
                continue
            with pytest.raises(EngineError, match="was built with"):
                LLM(engine, **asked)
