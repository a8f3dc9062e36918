"""The longest rows and the largest weights that the microscaled entry points take, and the engine's ways through them that other tests leave out."""
import pytest
import torch

import replay
import tiny
from arle_amd.engine import Engine, StepEntry
from arle_amd.engine.api import LLM
from arle_amd.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _signs(rows, width, seed, form):
    """Codes of -1, 0, 0 and 1, and those numbers in 32 bits: sums of up to 2^22 of them are exact."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    at = torch.randint(0, 4, (rows, width), generator=g, device=DEV, dtype=torch.uint8)
    one, minus = (0x38, 0xB8) if form == "mxfp8" else (2, 10)
    return torch.where(at == 0, minus, torch.where(at == 1, one, 0)).to(torch.uint8), (at == 1).float() - (at == 0).float()


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("M,variants", [(5, (0, 1)), (70, (2, 3, 7)), (300, (4, 5, 6, 8))])
def test_the_longest_rows(form, M, variants):
    K, N = mx.MAX_K, 72
    (xe, xv), (we, wv) = _signs(M, K, 1, form), _signs(N, K, 2, "mxfp4")
    ones = lambda n: torch.full((n, K // 32), 127, dtype=torch.uint8, device=DEV)
    x, w = mx.rows_from_codes(xe, ones(M), K, form), mx.lay_weight(mx.rows_from_codes(we, ones(N), K, "mxfp4"))
    # rows as far apart as they may be: the same elements in a wider buffer
    wide = torch.zeros(M, 2 * mx.MAX_K, dtype=torch.uint8, device=DEV)
    wide[:, :x.elements.shape[1]] = x.elements.view(torch.uint8)
    far = mx.MXRows(wide[:, :x.elements.shape[1]].view(x.elements.dtype), x.scales, K, form)
    assert torch.equal(mx.values(x), xv) and torch.equal(mx.values(far), xv)
    want = sum(xv[:, k:k + 2**18].double() @ wv[:, k:k + 2**18].double().T for k in range(0, K, 2**18)).float()
    for variant in variants:
        assert torch.equal(mx.gemm(x, w, torch.float32, variant=variant), want), variant
        assert torch.equal(mx.gemm(far, w, torch.float32, variant=variant), want), variant
    parts = mx.gemm(x, w, torch.float32, partials_ok=True, variant=variants[0], splits=8)
    assert torch.equal(parts.sum(0), want) and torch.equal(mx.gemm(x, w, torch.float32), want)
    assert torch.equal(mx.values(mx.quantize(xv[:5], form)), xv[:5])


@pytest.mark.parametrize("variant", [0, 1, 3, 6, 8])
def test_a_weight_past_2_to_the_31_numbers(variant):
    """Its tiles' places pass 32 bits, and so do a step's from the next one's."""
    N, K, M = 2**20 + 16, 2100, 16
    xe, xv = _signs(M, K, 1, "mxfp4")
    we, wv = _signs(N, K, 2, "mxfp4")
    x = mx.rows_from_codes(xe, torch.full((M, 66), 127, dtype=torch.uint8, device=DEV), K, "mxfp4")
    w = mx.lay_weight(mx.rows_from_codes(we, torch.full((N, 66), 127, dtype=torch.uint8, device=DEV), K, "mxfp4"))
    assert N * K > 2**31
    want = torch.cat([xv @ wv[n:n + 2**18].T for n in range(0, N, 2**18)], 1)
    assert torch.equal(mx.gemm(x, w, torch.float32, variant=variant), want)


@pytest.mark.parametrize("row_form", ["mxfp8", "mxfp4"])
def test_steps_from_graphs_that_were_captured_ahead(tmp_path, row_form):
    """Engine.warm_up and then decoding: every step replays, and gives the bits of an engine without graphs."""
    d = tiny.make_model_dir(tmp_path, "D")
    cfg, _ = tiny.read_folder(d)
    toks = {f"r{i}": tiny.random_tokens(n, cfg["vocab_size"], i) for i, n in enumerate([30, 19, 44])}
    steps = [s for rid, t in toks.items() for s in replay.prefill_then_decode(rid, t, 8)]
    make = lambda graphs: Engine.from_folder(d, page_size=32, max_tokens=1024, max_slots=4, cuda_graph=graphs, weight_form="mxfp4", row_form=row_form)
    warm, eager = make(True), make(False)
    assert warm.warm_up() > 0
    held = warm.graph_replays
    a, b = replay.run_steps(eager, steps), replay.run_steps(warm, steps)
    assert warm.graph_replays > held and a.keys() == b.keys() and all(torch.equal(a[k], b[k]) for k in a)


def test_tokens_with_a_warm_start_and_more_prompts_than_slots(tmp_path):
    d = tiny.make_model_dir(tmp_path, "B")
    prompts = [list(range(3 + i, 9 + 5 * i)) for i in range(7)]
    one = LLM(d, num_slots=2, kv_cache_tokens=256, max_seq_len=96, weight_form="mxfp4", warm_up=True).generate(prompts, max_tokens=10)
    two = LLM(d, num_slots=2, kv_cache_tokens=256, max_seq_len=96, weight_form="mxfp4", cuda_graph=False, async_overlap=False).generate(prompts, max_tokens=10)
    assert [o.response_token_ids for o in one] == [o.response_token_ids for o in two] and all(len(o.response_token_ids) == 10 for o in one)


def test_the_debug_dump_of_such_a_model(tmp_path, monkeypatch, capsys):
    monkeypatch.setenv("ARLE_AMD_DEBUG_DUMP", "1")
    d = tiny.make_model_dir(tmp_path, "A")
    engine = Engine.from_folder(d, max_tokens=64, page_size=4, weight_form="mxfp4")
    engine.add_request("x")
    assert torch.isfinite(engine.step([StepEntry("x", [1, 2, 3], [2])])).all()
    engine.step([StepEntry("x", [4], [0])])
    lines = [line for line in capsys.readouterr().err.splitlines() if line.startswith("[debug-dump]")]
    assert len(lines) == 2 * (1 + len(engine.model.schedule)) and all("nan=False inf=False" in line for line in lines)
