"""Microscaled rows and weights on the host: layouts of weights, and the calls that the entry points refuse before anything is launched."""
import copy

import pytest
import torch

import plain_mx as plain
from arle_amd.kernels import mx, ops


@pytest.fixture
def no_gpu(monkeypatch):
    """CPU tensors pass, and no kernel may be asked for."""
    monkeypatch.setattr(mx, "_here", lambda *t: 0)
    monkeypatch.setattr(mx, "_current", lambda: 0)
    monkeypatch.setattr(mx, "_DEVICES", {d: torch.device("cpu") for d in (-1, 0)})

    class Functions(dict):
        def get(self, name):
            raise AssertionError(f"{name} was launched")

    monkeypatch.setattr(mx, "_functions", Functions())


def _rows(T, width, form="mxfp8", seed=0):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(0, 16 if form == "mxfp4" else 120, (T, width), generator=g, dtype=torch.uint8)
    s = torch.randint(100, 140, (T, -(-width // 32)), generator=g, dtype=torch.uint8)
    return e, s, mx.rows_from_codes(e, s, width, form)


@pytest.mark.parametrize("form", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("T,width", [(0, 32), (1, 1), (3, 255), (5, 256), (2, 257), (4, 700)])
def test_rows_from_codes(no_gpu, form, T, width):
    e, s, rows = _rows(T, width, form)
    assert rows.rows == T and rows.padded % 512 == 0 and 0 <= rows.padded - width < 512
    got_e, got_s = plain.unpack(rows)
    assert torch.equal(got_e[:, :width], e) and not got_e[:, width:].any()
    blocks = s.shape[1]
    assert torch.equal(got_s[:, :blocks], s) and not got_s[:, blocks:].any()


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (40, 700), (33, 1100)])
def test_weight_tiles(no_gpu, n, k):
    """Lane 16 g + i of tile (t, s) holds row 16 t + i, k 128 s + 32 g ..; byte s % 4 of its scale word is that block's."""
    e, s, rows = _rows(n, k, "mxfp4")
    w = mx.lay_weight(rows)
    assert (w.n, w.k, w.gated) == (n, k, False)
    codes, scales = plain.unpack(rows)
    for t in range(w.tiles.shape[1]):
        for st in range(w.tiles.shape[0]):
            for lane in range(64):
                g, i = divmod(lane, 16)
                row = 16 * t + i
                piece = w.tiles[st, t, lane]
                got = torch.stack([piece & 15, piece >> 4], dim=-1).flatten()
                at = 128 * st + 32 * g
                want = codes[row, at:at + 32] if row < n else torch.zeros(32, dtype=torch.uint8)
                assert torch.equal(got, want)
                assert w.scales[st // 4, t, lane, st % 4] == (scales[row, at // 32] if row < n else 0)


@pytest.mark.parametrize("ff", [1, 16, 100, 256, 300])
def test_gated_weight_is_turns_of_sixteen(no_gpu, ff):
    e, s, rows = _rows(2 * ff, 64, "mxfp4")
    w = mx.lay_weight(rows, gated=True)
    padded = -(-ff // 512) * 512
    assert w.n == 2 * ff and w.tiles.shape[1] == 2 * padded // 16
    codes, _ = plain.unpack(rows)
    for c in range(0, padded, 7):
        for which in (0, 1):
            piece = w.tiles[0, 2 * (c // 16) + which, c % 16]
            got = torch.stack([piece & 15, piece >> 4], dim=-1).flatten()
            assert torch.equal(got, codes[which * ff + c, :32] if c < ff else torch.zeros(32, dtype=torch.uint8))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64)
    for call in (lambda: mx.quantize(x), lambda: mx.add_rmsnorm(x, None, torch.ones(64), 1e-6),
                 lambda: mx.rows_from_codes(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 64, "mxfp8")):
        with pytest.raises(ops.ShapeError, match="GPU only"):
            call()


def _e8(T, W):
    return torch.zeros(T, W, dtype=torch.uint8).view(torch.float8_e4m3fn)


def _s(T, B):
    return torch.zeros(T, B, dtype=torch.uint8).view(torch.float8_e8m0fnu)


def test_refused_rows(no_gpu):
    bad = [
        lambda: mx.quantize(torch.zeros(2, 64), "mxfp6"),
        lambda: mx.quantize(torch.zeros(2, 64, dtype=torch.float16)),
        lambda: mx.quantize(torch.zeros(64)),
        lambda: mx.quantize(torch.zeros(2, 0)),
        lambda: mx.quantize(torch.zeros(64, 4).T),                                      # columns apart
        lambda: mx.rows_from_codes(torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.uint8), 64, "mxfp8"),
        lambda: mx.rows_from_codes(torch.zeros(2, 63, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 64, "mxfp8"),
        lambda: mx.rows_from_codes(torch.full((2, 64), 16, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8), 64, "mxfp4"),
        lambda: mx.rows_from_codes(torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.uint8), 64, "mxfp8"),
        lambda: _rows(2, 64, "mxfp4")[2].elements_e4m3(),
        lambda: mx.values(torch.zeros(2, 64)),
        lambda: mx.values(_rows(2, 64)[2], torch.float16),
        lambda: mx.MXRows(_e8(2, 600)[:, 1:513], _s(2, 16), 512, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 513)[:, :512], _s(2, 16), 512, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(2, 20)[:, :16], 512, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(2, 16), 600, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(1, 16), 512, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(2, 16).view(torch.uint8), 512, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(2, 16), 0, "mxfp8"),
        lambda: mx.MXRows(_e8(2, 512), _s(2, 32), 1024, "mxfp4"),
        lambda: mx.MXRows(_e8(2, 2**23 + 16)[:, :512], _s(2, 16), 512, "mxfp8"),      # rows further apart than offsets of 32 bits reach over 256 of them
        lambda: mx.MXRows(_e8(2, 512), _s(2, 2**23 + 16)[:, :16], 512, "mxfp8"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ops.ShapeError):
            call()
            pytest.fail(f"call {i} passed")


@pytest.mark.parametrize("copied", [copy.copy, copy.deepcopy])
def test_rows_and_weights_can_be_copied(no_gpu, copied):
    rows, weight = _rows(3, 600)[2], mx.lay_weight(_rows(34, 600, "mxfp4")[2], gated=True)
    for a in (rows, weight):
        b = copied(a)
        assert type(b) is type(a) and all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(a[:2], b[:2])) and a[2:] == b[2:]


def test_refused_norms(no_gpu):
    res, w = torch.zeros(3, 64), torch.ones(64)
    bad = [
        lambda: mx.add_rmsnorm(res.bfloat16(), None, w, 1e-6),
        lambda: mx.add_rmsnorm(res[:, :32], None, w[:32], 1e-6),
        lambda: mx.add_rmsnorm(res, res[:2], w, 1e-6),
        lambda: mx.add_rmsnorm(res, torch.zeros(0, 3, 64), w, 1e-6),
        lambda: mx.add_rmsnorm(res, res.half(), w, 1e-6),
        lambda: mx.add_rmsnorm(res, torch.zeros(64), w, 1e-6),
        lambda: mx.add_rmsnorm(res, torch.zeros(1, 1, 3, 64), w, 1e-6),
        lambda: mx.add_rmsnorm(res, None, w[:63], 1e-6),
        lambda: mx.add_rmsnorm(res, None, w.half(), 1e-6),
        lambda: mx.add_rmsnorm(res, None, w, 1e-6, "fp8"),
        lambda: mx.add_rmsnorm(res, None, w, 1e-6, rows=torch.zeros(2, dtype=torch.int64)),
        lambda: mx.add_rmsnorm(torch.zeros(1, mx.MAX_WIDTH + 1), None, torch.ones(mx.MAX_WIDTH + 1), 1e-6),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ops.ShapeError):
            call()
            pytest.fail(f"call {i} passed")


def test_refused_products(no_gpu):
    x = _rows(3, 300)[2]
    w = mx.lay_weight(_rows(40, 300, "mxfp4")[2])
    wg = mx.lay_weight(_rows(40, 300, "mxfp4")[2], gated=True)
    bad = [
        lambda: mx.lay_weight(_rows(40, 300)[2]),                        # weights are held in 4 bits
        lambda: mx.lay_weight(_rows(0, 300, "mxfp4")[2]),
        lambda: mx.lay_weight(_rows(41, 300, "mxfp4")[2], gated=True),
        lambda: mx.gemm(torch.zeros(3, 300), w),
        lambda: mx.gemm(x, torch.zeros(40, 300)),
        lambda: mx.gemm(x, wg),
        lambda: mx.gate_up_act(x, w),
        lambda: mx.gate_up_act(x, wg, "fp4"),
        lambda: mx.gemm(_rows(3, 299)[2], w),
        lambda: mx.gemm(x, w, torch.float16),
        lambda: mx.gemm(x, mx.MXWeight(w.tiles[:, :1], w.scales, 40, 300)),
        lambda: mx.gemm(x, mx.MXWeight(w.tiles, w.scales, 60, 300)),
        lambda: mx.MXWeight(w.tiles[:, :2], w.scales[:, :2].contiguous()[:, :, :32], 32, 300),
        lambda: mx.MXWeight(w.tiles.transpose(2, 3).contiguous().transpose(2, 3), w.scales, 40, 300),
        lambda: w.first(24), lambda: w.first(48), lambda: w.first(0), lambda: wg.first(16),
        lambda: mx.gemm(_rows(17, 300)[2], w, variant=0),                # more rows than the kernel holds
        lambda: mx.gemm(x, w, variant=20),
        lambda: mx.gate_up_act(x, wg, variant=8),
        lambda: mx.gate_up_act(x, wg, variant=0),
        lambda: mx.gemm(x, w, variant=0, splits=5),                      # four steps of 128
        lambda: mx.gemm(_rows(3, 300, "mxfp4")[2], w, variant=3, splits=2),   # one round of 512
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ops.ShapeError):
            call()
            pytest.fail(f"call {i} passed")


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("bits", [4, 8])
def test_every_size_has_a_plan(bits, gated, whole):
    """A variant that takes the rows, and parts of K of which none is empty."""
    for M in (1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 129, 500, 1000, 2048, 5000, 70000):
        for n_tiles in (1, 3, 64, 96, 160, 384, 1216, 9496):
            for k_tiles in (4, 8, 20, 32, 76, 96, 1000):
                variant, splits, per_split = mx._plan(M, n_tiles, k_tiles, bits, gated, whole)
                few = variant in (*mx.ROW_VARIANTS, mx.GATED_ROWS)
                steps = k_tiles if few else k_tiles // 4
                assert splits >= 1 and (splits - 1) * per_split < steps <= splits * per_split
                assert M <= 16 if few else variant in mx._TILES
                assert (splits == 1 and variant in (3, 4, 5, 6, mx.GATED_ROWS)) if gated else variant != mx.GATED_ROWS


def test_no_rows_launch_nothing(no_gpu):
    w, wg = mx.lay_weight(_rows(40, 300, "mxfp4")[2]), mx.lay_weight(_rows(40, 300, "mxfp4")[2], gated=True)
    none = _rows(0, 300)[2]
    assert mx.gemm(none, w).shape == (0, 40) and mx.gate_up_act(none, wg).rows == 0
    assert mx.quantize(torch.zeros(0, 64)).rows == 0 and mx.values(none).shape == (0, 300)
    assert mx.add_rmsnorm(torch.zeros(0, 64), None, torch.ones(64), 1e-6).rows == 0


def test_designs_without_that_form_are_refused():
    from arle_amd import models  # noqa: F401
    from arle_amd.config.registry import detect_architecture
    from arle_amd.engine.engine import Engine, EngineError

    import tiny
    import tiny_gufasun

    qwen3 = detect_architecture({"architectures": [tiny.ARCH]})
    spec = qwen3.recipe(qwen3.config_class.from_dict(tiny.TINY["A"][0]), ())
    engine = object.__new__(Engine)
    engine.dtype = torch.bfloat16
    engine._check_weight_form(spec, "mxfp4", "mxfp8")
    for form, rows in (("int4", "mxfp8"), ("mxfp4", "bf16")):
        with pytest.raises(EngineError):
            engine._check_weight_form(spec, form, rows)
    engine.dtype = torch.float32
    with pytest.raises(EngineError, match="bfloat16"):
        engine._check_weight_form(spec, "mxfp4", "mxfp8")
    engine.dtype = torch.bfloat16
    raw = next(v for v in vars(tiny_gufasun).values() if isinstance(v, dict) and "layers" in v)
    other = detect_architecture(raw)
    with pytest.raises(EngineError, match="not built for"):
        engine._check_weight_form(other.recipe(other.config_class.from_dict(raw), ()), "mxfp4", "mxfp8")


def test_few_gated_rows_have_a_kernel_of_their_own(no_gpu):
    x, wg, w = _rows(3, 64)[2], mx.lay_weight(_rows(64, 64, "mxfp4")[2], gated=True), mx.lay_weight(_rows(64, 64, "mxfp4")[2])
    assert mx._plan(16, wg.n_tiles, wg.k_tiles, 8, True, True)[0] == mx.GATED_ROWS and mx._plan(17, wg.n_tiles, wg.k_tiles, 8, True, True)[0] in mx._TILES
    for call in (lambda: mx.gemm(x, w, variant=mx.GATED_ROWS), lambda: mx.gate_up_act(_rows(17, 64)[2], wg, variant=mx.GATED_ROWS)):
        with pytest.raises(ops.ShapeError):
            call()


def test_empty_rows(no_gpu):
    for form in ("mxfp8", "mxfp4"):
        rows = mx.empty_rows(5, 700, form)
        again = mx.MXRows(rows.elements, rows.scales, 700, form)      # as a user would make them, checked
        assert rows[2:] == again[2:] and rows.rows == 5 and rows.elements.is_contiguous()
    for args in ((5, 0, "mxfp8"), (-1, 32, "mxfp8"), (5, 32, "fp8"), (5, mx.MAX_K + 1, "mxfp4")):
        with pytest.raises(ops.ShapeError):
            mx.empty_rows(*args)


def test_blocks_that_attention_cannot_fill(no_gpu, monkeypatch):
    monkeypatch.setattr(ops, "_gpu", lambda *tensors: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    calls = []
    monkeypatch.setattr(ops.lib, "call", lambda name, *args: calls.append((name, args)))
    i32 = lambda values: torch.tensor(list(values), dtype=torch.int32)

    def run(blocks):
        out = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
        return ops.attn_decode_prep(torch.zeros(2, 3, 12 * 64), out, torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16),
                                    torch.zeros(6, 2, 64, 16, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), i32(range(4)), i32(range(3)),
                                    i32([20] * 3), max_kv_len=21, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16, scale=1.0, eps=1e-6,
                                    splits=1, blocks=blocks)

    rows = mx.empty_rows(3, 512, "mxfp8")._replace(device=-1)      # the device number of a tensor on the host
    assert run(rows) is rows and calls[-1][0] == "arle_attn_decode_prep_blocks" and calls[-1][1][-3:-1] == (8, 512)
    assert run(None).shape == (3, 512) and calls[-1][0] == "arle_attn_decode_prep"
    wide = mx.empty_rows(3, 1024, "mxfp8")
    apart = rows._replace(elements=wide.elements[:, :512])
    for bad in (rows._replace(rows=4), rows._replace(width=500), apart, rows._replace(device=0), rows.elements):
        with pytest.raises(ops.ShapeError):
            run(bad)


def test_views_without_the_padding(no_gpu):
    e, s, rows = _rows(9, 700)
    for part in (rows, rows.part(2, 7), rows.part(4, 4), mx.MXRows(rows.elements[1::3], rows.scales[1::3], 700, "mxfp8")):
        a, b = part.elements_e4m3(), part.scales_e8m0()
        assert torch.equal(a.view(torch.uint8), part.elements[:, :700].view(torch.uint8)) and a.data_ptr() == part.elements.data_ptr()
        assert torch.equal(b.view(torch.uint8), part.scales[:, :22].view(torch.uint8)) and b.shape == (part.rows, 22)
