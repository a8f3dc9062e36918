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


def test_a_step_reads_its_projections_in_the_form_that_they_are_held_in():
    c = bench.QWEN3_4B
    layers = c["num_hidden_layers"] * bench.layer_params(c)
    whole, held = bench.decode_bytes(c, 8, 2064.0), bench.decode_bytes(c, 8, 2064.0, 2, bench.MXFP4_BYTES)
    assert whole == bench.decode_bytes(c, 8, 2064.0, 2, 2) and whole - held == layers * (2 - 17 / 32)
    # 36 layers of q|k|v, o, gate|up and down: 4.25 bits a number, 1.9 GB of them; embedding and norms stay as they are
    assert layers * bench.MXFP4_BYTES == 36 * (6144 * 2560 + 2560 * 4096 + 3 * 2560 * 9728) * 17 / 32
