"""bench.py --weight-form: heard by the default workload, refused where it would print figures of weights in bfloat16."""
import sys

import pytest

import bench


@pytest.mark.parametrize("mode", [["--sweep"], ["--generate"], ["--first-token"], ["--gaps"], ["--tune-products", "4b"], ["--ceilings"], ["--parts-only"],
                                  *(["--workload", w] for w in ("qwen3-8b-mixed", "qwen3-32b-decode", "gufasun", "sovutar", "tazitar", "retudra", "nafezen", "pozirax"))])
def test_modes_that_would_not_use_it_end_with_a_usage_error(mode, monkeypatch, capsys):
    for name in ("sweep", "generate_workload", "first_token", "step_gaps", "tune_products", "ceilings", "mixed_8b", "decode_32b", "gufasun_bench",
                 "sovutar_bench", "tazitar_bench", "retudra_bench", "nafezen_bench", "pozirax_bench"):
        monkeypatch.setattr(bench, name, lambda *args, name=name: pytest.fail(f"{name} ran"))
    monkeypatch.setattr(sys, "argv", ["bench.py", "--weight-form", "mxfp4", *mode])
    with pytest.raises(SystemExit) as end:
        bench.main()
    assert end.value.code == 2 and "--weight-form is for the default workload" in capsys.readouterr().err


def test_rows_go_with_weights(monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--row-form", "mxfp4"])
    with pytest.raises(SystemExit) as end:
        bench.main()
    assert end.value.code == 2 and "--row-form goes with --weight-form" in capsys.readouterr().err


@pytest.mark.parametrize("args", [[], ["--weight-form", "mxfp4"], ["--weight-form", "mxfp4", "--row-form", "mxfp4", "--prefill-only"]])
def test_the_default_workload_takes_them(args, monkeypatch, capsys):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--gpus", "2", *args])      # ends behind the arguments: no engine for two GPUs
    assert bench.main() == 2 and "one GPU" in capsys.readouterr().out
