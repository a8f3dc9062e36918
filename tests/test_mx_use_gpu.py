"""The microscaled kernels as programs use them: one behind the other, captured, on several streams and threads, with numbers that are none,
and at sizes past 32 bits."""
import threading

import pytest
import torch

import plain_mx as plain
import tiny
from arle_amd.engine import Engine, StepEntry
from arle_amd.kernels import mx

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMS = ["mxfp8", "mxfp4"]


def _g(seed):
    return torch.Generator().manual_seed(seed)


class _FeedForward:
    """Norm, gated first half, second half and the norm behind it, which adds the stack that a product may leave."""

    def __init__(self, H, ff, form, seed):
        n = lambda *shape: torch.randn(*shape, generator=_g(seed + len(shape) + shape[0]))
        self.form = form
        self.plain = [(1 + 0.1 * n(H)).double(), n(2 * ff, H).double() * H**-0.5, n(H, ff).double() * ff**-0.5]
        self.norm = self.plain[0].float().to(DEV)
        self.gate_up = mx.lay_weight(mx.quantize(self.plain[1].float().to(DEV), "mxfp4"), gated=True)
        self.down = mx.lay_weight(mx.quantize(self.plain[2].float().to(DEV), "mxfp4"))

    def __call__(self, residual, x):
        rows = mx.add_rmsnorm(residual, x, self.norm, 1e-6, self.form)
        stack = mx.gemm(mx.gate_up_act(rows, self.gate_up, self.form), self.down, partials_ok=True)
        return mx.values(mx.add_rmsnorm(residual, stack, self.norm, 1e-6, self.form))

    def in_64_bits(self, residual, x, rounded):
        norm, gate_up, down = self.plain
        held = lambda w: plain.round_rows(w, "mxfp4")
        rows = (lambda v: plain.round_rows(v, self.form)) if rounded else (lambda v: v)
        h, y = plain.norm(residual, x, norm, 1e-6)
        d = rows(plain.gated(rows(y), held(gate_up))) @ held(down).T
        h, y = plain.norm(h, d, norm, 1e-6)
        return h, rows(y)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("T,H,ff", [(1, 260, 700), (7, 1100, 300), (40, 512, 1530)])
def test_one_behind_the_other(form, T, H, ff):
    """Off from the same blocks in 64 bits by less than rounding every number to its element is off from not rounding: the two differ
    where 32 bits, or a product's bfloat16, put a number on the other side of a border between two elements."""
    part = _FeedForward(H, ff, form, 3)
    residual, x = torch.randn(T, H, generator=_g(1)), torch.randn(T, H, generator=_g(2)).bfloat16()
    h, y = part.in_64_bits(residual, x, True)
    h0, y0 = part.in_64_bits(residual, x, False)
    r = residual.to(DEV)
    got = part(r, x.to(DEV)).cpu().double()
    assert (r.cpu().double() - h).norm() <= (h - h0).norm() and (got - y).norm() <= (y - y0).norm()


def test_captured_at_the_first_call_and_replayed():
    """Two graphs of the same program, replayed several times in turn on two streams with new inputs, eager calls and synchronisations
    between; each keeps its own results."""
    parts = [_FeedForward(520, 300, form, 5) for form in FORMS]
    w = mx.lay_weight(mx.quantize(torch.randn(600, 520, generator=_g(7)).to(DEV), "mxfp4"))
    make = lambda: (torch.zeros(16, 520, device=DEV), torch.zeros(16, 520, dtype=torch.bfloat16, device=DEV))

    def program(residual, x):
        q = mx.quantize(x, "mxfp8")
        outs = [mx.gemm(q, w, torch.float32, variant=v) for v in range(9)] + [p(residual, x) for p in parts]
        return outs + [mx.values(q), mx.gemm(q, w, variant=2, splits=2)]

    torch.cuda.synchronize()
    held = []
    for _ in range(2):
        inputs = make()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = program(*inputs)
        held.append((inputs, graph, outs))
    streams = [torch.cuda.Stream() for _ in held]
    for turn in range(4):
        given = [(torch.randn(16, 520, generator=_g(10 * turn + i)), torch.randn(16, 520, generator=_g(10 * turn + i + 5)).bfloat16()) for i in range(2)]
        for (inputs, _, _), new in zip(held, given):
            for t, v in zip(inputs, new):
                t.copy_(v)
        torch.cuda.synchronize()
        for (_, graph, _), s in zip(held, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (inputs, _, outs), (residual, x) in zip(held, given):
            r = residual.to(DEV)
            want = program(r, x.to(DEV))
            assert torch.equal(inputs[0], r)
            for i, (a, b) in enumerate(zip(outs, want)):
                assert torch.equal(a, b), (turn, i)


def test_threads_with_streams_of_their_own():
    part = _FeedForward(300, 200, "mxfp8", 9)
    given = [(torch.randn(5 + i, 300, generator=_g(i)).to(DEV), torch.randn(5 + i, 300, generator=_g(i + 9)).to(DEV)) for i in range(4)]
    want = [part(r.clone(), x) for r, x in given]
    torch.cuda.synchronize()
    off, done = [], []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                if not torch.equal(part(given[i][0].clone(), given[i][1]), want[i]):
                    off.append(i)
            s.synchronize()
        done.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not off and len(done) == 4


@pytest.mark.parametrize("form", FORMS)
def test_numbers_that_are_none(form):
    """A block that is no number makes its row's results none, or its column's, and nobody else's; sums past the type are infinite."""
    M, N, K = 70, 150, 300
    x, w = torch.randn(M, K, generator=_g(1)), torch.randn(N, K, generator=_g(2))
    clean_x, clean_w = x.clone(), w.clone()
    x[3, 40], x[69, 299], w[10, 0], w[149, 64] = float("nan"), float("inf"), float("-inf"), float("nan")
    lay = lambda t, **kw: mx.lay_weight(mx.quantize(t.to(DEV), "mxfp4"), **kw)
    q, clean = mx.quantize(x.to(DEV), form), mx.quantize(clean_x.to(DEV), form)
    bad_rows, bad_columns = torch.zeros(M, dtype=torch.bool, device=DEV), torch.zeros(N, dtype=torch.bool, device=DEV)
    bad_rows[[3, 69]], bad_columns[[10, 149]] = True, True
    bad = bad_rows[:, None] | bad_columns[None]
    for variant in range(2, 9):
        want = mx.gemm(clean, lay(clean_w), torch.float32, variant=variant)
        got = mx.gemm(q, lay(w), torch.float32, variant=variant)
        assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], want[~bad]), variant
    rows = q.part(0, 9), clean.part(0, 9)
    for variant in (0, 1):
        got, want = mx.gemm(rows[0], lay(w), torch.float32, variant=variant), mx.gemm(rows[1], lay(clean_w), torch.float32, variant=variant)
        assert torch.equal(got.isnan(), bad[:9]) and torch.equal(got[~bad[:9]], want[~bad[:9]]), variant
    # gated: column 10 of the gate's half and 149 - 75 = 74 of the up's; each one's block of 32 is none
    blocks = torch.zeros(M, 3, dtype=torch.bool, device=DEV)
    blocks[:, [0, 2]] = True
    blocks[bad_rows] = True
    for variant in (3, 4, 5, 6):
        e, s = plain.unpack(mx.gate_up_act(q, lay(w, gated=True), form, variant=variant))
        ce, cs = plain.unpack(mx.gate_up_act(clean, lay(clean_w, gated=True), form, variant=variant))
        b = blocks.cpu()
        assert torch.equal(s[:, :3] == 255, b) and torch.equal(s[:, :3][~b], cs[:, :3][~b]), variant
        wide = b.repeat_interleave(32, 1)[:, :75]
        assert not e[:, :75][wide].any() and torch.equal(e[:, :75][~wide], ce[:, :75][~wide]), variant
    # 2^100 times 2^100; a column without weights stays zero
    huge = mx.quantize(torch.full((20, 64), 2.0**100, device=DEV), form)
    big = torch.full((40, 64), 2.0**100)
    big[1] = 0
    for variant in (2, 4, 8):
        got = mx.gemm(huge, lay(big), torch.float32, variant=variant)
        assert got[:, 1].eq(0).all() and got[:, [0, 2, 39]].isinf().all()


def test_results_past_32_bits_of_numbers():
    M, N = 70001, 32768
    e = torch.randint(0, 100, (M, 64), generator=_g(1), dtype=torch.uint8)
    s = torch.randint(120, 130, (M, 2), generator=_g(2), dtype=torch.uint8)
    x = mx.rows_from_codes(e.to(DEV), s.to(DEV), 64, "mxfp8")
    w = mx.lay_weight(mx.quantize(torch.randn(N, 64, generator=_g(3)).to(DEV), "mxfp4"))
    whole = mx.gemm(x, w)
    assert whole.numel() > 2**31
    for start in (0, 35000, M - 40):
        assert torch.equal(whole[start:start + 40], mx.gemm(x.part(start, start + 40), w))
    del whole
    wide = torch.randn(1, 8192, generator=_g(4)).to(DEV).bfloat16().expand(280000, 8192).contiguous()
    wide[-1] = wide[-1] * 3
    q = mx.quantize(wide)
    last = mx.quantize(wide[-3:])
    assert all(torch.equal(a, b) for a, b in zip(plain.unpack(q.part(279997, 280000)), plain.unpack(last)))
    assert torch.equal(mx.values(q, torch.bfloat16)[-3:], mx.values(last, torch.bfloat16))


def test_tuning_leaves_such_projections_alone(tmp_path):
    """The table of measured products is of products in bfloat16: the head's here."""
    d = tiny.make_model_dir(tmp_path, "A")
    engine = Engine.from_folder(d, max_tokens=64, weight_form="mxfp4")
    engine.tune_products(rows=[1, 8])
    engine.add_request("x")
    assert torch.isfinite(engine.step([StepEntry("x", [1, 2, 3], [2])])).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("K", [130, 1100, 1600])
def test_workgroups_with_several_tiles(form, K):
    """Products of more tiles than workgroups that run at once, whose last row and column blocks overlap the ones in front, with one, three and
    four rounds of K: exact, as numbers up to 3 and weights up to 6 with scales from 1/4 to 4 have sums under 2^20 of multiples of 1/32."""
    M, N = 4100, 4700
    few = torch.tensor([0, 2, 4, 5, 8, 10, 12, 13] if form == "mxfp4" else [0, 0x38, 0x40, 0x44, 0x80, 0xB8, 0xC0, 0xC4], dtype=torch.uint8)
    xe, we = few[torch.randint(0, 8, (M, K), generator=_g(1))], torch.randint(0, 16, (N, K), generator=_g(2), dtype=torch.uint8)
    xs, ws = (torch.randint(125, 130, (n, -(-K // 32)), generator=_g(n), dtype=torch.uint8) for n in (M, N))
    x, wide = mx.rows_from_codes(xe.to(DEV), xs.to(DEV), K, form), mx.rows_from_codes(we.to(DEV), ws.to(DEV), K, "mxfp4")
    w, gated = mx.lay_weight(wide), mx.lay_weight(wide, gated=True)
    want = (plain.dequantize(xe, xs, form).float().to(DEV).double() @ plain.dequantize(we, ws, "mxfp4").float().to(DEV).double().T)
    gate = plain.unpack(mx.gate_up_act(x, gated, form, variant=3))      # whose workgroups have one tile each
    for variant in sorted(mx._TILES):
        for dtype in (torch.float32, torch.bfloat16):
            assert torch.equal(mx.gemm(x, w, dtype, variant=variant), want.to(dtype)), (variant, dtype)
        if variant not in mx._PLAIN_TILES:
            assert all(torch.equal(p, q) for p, q in zip(gate, plain.unpack(mx.gate_up_act(x, gated, form, variant=variant)))), variant
    parts = mx.gemm(x, w, torch.float32, partials_ok=True, variant=5, splits=min(2, x.padded // 512))
    assert torch.equal(parts.double().sum(0) if parts.dim() == 3 else parts.double(), want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("out", FORMS)
@pytest.mark.parametrize("ff,K", [(1, 40), (32, 256), (100, 300), (700, 1100), (4000, 520)])
def test_gated_products_of_few_rows(form, out, ff, K):
    """The few rows' kernel against the tiles' one: whole numbers, whose sums are exact in any order, give the same blocks bit for bit; a block
    that is no number in a row, and one in a column of each half, give none where they enter."""
    few = torch.tensor([0, 2, 4, 5, 8, 10, 12, 13] if form == "mxfp4" else [0, 0x38, 0x40, 0x44, 0x80, 0xB8, 0xC0, 0xC4], dtype=torch.uint8)
    for M in (1, 7, 16):
        xe, we = few[torch.randint(0, 8, (M, K), generator=_g(M))], torch.randint(0, 16, (2 * ff, K), generator=_g(ff), dtype=torch.uint8)
        xs, ws = (torch.randint(122, 125, (n, -(-K // 32)), generator=_g(n + 1), dtype=torch.uint8) for n in (M, 2 * ff))
        for none in (False, True):
            if none:
                xs[M // 2, -1] = ws[ff // 2, 0] = ws[ff + ff // 3, -1] = 255
            x = mx.rows_from_codes(xe.to(DEV), xs.to(DEV), K, form)
            w = mx.lay_weight(mx.rows_from_codes(we.to(DEV), ws.to(DEV), K, "mxfp4"), gated=True)
            want, got = plain.unpack(mx.gate_up_act(x, w, out, variant=3)), plain.unpack(mx.gate_up_act(x, w, out, variant=mx.GATED_ROWS))
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (M, none)
            if not none:
                xv, wv = plain.dequantize(xe, xs, form), plain.dequantize(we, ws, "mxfp4")
                y, held = plain.gated(xv, wv), plain.dequantize(got[0][:, :ff], got[1][:, :-(-ff // 32)], out)
                half, least = {"mxfp8": (2.0**-4, 2.0**-10), "mxfp4": (2.0**-2, 2.0**-2)}[out]
                step = torch.maximum(half * y.abs(), least * plain.scale_values(got[1]).repeat_interleave(32, 1)[:, :ff])
                assert ((held - y).abs() <= step * (1 + 2.0**-10) + 2.0**-18 * y.abs() + 2.0**-100).all()
    assert all(torch.equal(a, b) for a, b in zip(plain.unpack(mx.gate_up_act(x, w, out)), plain.unpack(mx.gate_up_act(x, w, out, variant=mx.GATED_ROWS))))


def _at_the_end(t):
    """The same numbers in the last bytes of an allocation that ends with its mapping (of its own, a multiple of 2 MiB): a kernel that reads past
    what it was given, wherever that is the last of it, does not get away with it."""
    whole = torch.empty(32 * 2**20, dtype=torch.uint8, device=DEV)
    flat = t.contiguous().view(torch.uint8).flatten()
    whole[-flat.numel():] = flat
    return whole[-flat.numel():].view(t.dtype).view(t.shape)


@pytest.mark.parametrize("form", FORMS)
def test_operands_at_the_end_of_their_memory(form):
    """Every variant with rows and columns that fill its last tile, end inside it, or are fewer than it has."""
    torch.cuda.empty_cache()
    N, K = 600, 1100
    q = mx.quantize(torch.randn(520, K, generator=_g(1)).to(DEV), form)
    held = mx.quantize(torch.randn(N, K, generator=_g(2)).to(DEV), "mxfp4")
    w, wg = mx.lay_weight(held), mx.lay_weight(held, gated=True)
    ends = [mx.MXWeight(_at_the_end(v.tiles), _at_the_end(v.scales), v.n, v.k, v.gated) for v in (w, wg)]
    for M in (1, 16, 17, 32, 33, 64, 65, 100, 130, 256, 300, 520):
        rows = q.part(0, M)
        x = mx.MXRows(_at_the_end(rows.elements), _at_the_end(rows.scales), K, form)
        for variant in range(9):
            if variant > 1 or M <= 16:
                assert torch.equal(mx.gemm(x, ends[0], torch.float32, variant=variant), mx.gemm(rows, w, torch.float32, variant=variant)), (M, variant)
        for variant in (3, 4, 5, 6, mx.GATED_ROWS):
            if variant != mx.GATED_ROWS or M <= 16:
                got, want = mx.gate_up_act(x, ends[1], form, variant=variant), mx.gate_up_act(rows, wg, form, variant=variant)
                assert all(torch.equal(a, b) for a, b in zip(plain.unpack(got), plain.unpack(want))), (M, variant)
        assert torch.equal(mx.values(x), mx.values(rows))
    for n in (1, 16, 100):      # fewer columns than a tile has
        few = mx.lay_weight(mx.quantize(torch.randn(n, K, generator=_g(n)).to(DEV), "mxfp4"))
        end = mx.MXWeight(_at_the_end(few.tiles), _at_the_end(few.scales), n, K)
        for variant in range(2, 9):
            assert torch.equal(mx.gemm(x, end, torch.float32, variant=variant), mx.gemm(rows, few, torch.float32, variant=variant)), (n, variant)
    for T, W in ((1, 264), (5, 1530), (1100, 513)):
        numbers = torch.randn(T, W, generator=_g(T)).bfloat16().to(DEV)
        assert all(torch.equal(a, b) for a, b in zip(plain.unpack(mx.quantize(_at_the_end(numbers), form)), plain.unpack(mx.quantize(numbers, form))))
        residual, weight = torch.randn(T, W, generator=_g(3)).to(DEV), _at_the_end(torch.ones(W, device=DEV))
        a = mx.add_rmsnorm(_at_the_end(residual), _at_the_end(torch.stack([numbers, numbers])), weight, 1e-6, form)
        b = mx.add_rmsnorm(residual, torch.stack([numbers, numbers]), weight, 1e-6, form)
        assert all(torch.equal(p, q) for p, q in zip(plain.unpack(a), plain.unpack(b)))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("D,nq,nkv", [(128, 32, 8), (128, 6, 2), (64, 12, 4), (64, 32, 8)])
@pytest.mark.parametrize("contexts", [[0], [2047], [31, 32, 700, 0, 63], [900] * 9, [3000] + [40] * 40])
def test_attention_that_leaves_blocks(form, D, nq, nkv, contexts):
    """A step of decoded tokens whose results leave in blocks, bit for bit those that quantize makes of the same step's: splits that are merged
    by a kernel, or inside a workgroup, or one wave a request, and shared-out keys with some requests of one wave."""
    from arle_amd.kernels import lib, ops

    P, T = 16, len(contexts)
    pages = [(c + 1 + P - 1) // P for c in contexts]
    order = torch.randperm(sum(pages), generator=_g(1)).to(torch.int32)
    table = torch.zeros(T, max(pages), dtype=torch.int32)
    for i, part in enumerate(order.split(pages)):
        table[i, :len(part)] = part
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(sum(pages), nkv, *shape, generator=_g(2)).bfloat16().to(DEV) for shape in ((P, D), (D, P)))
    parts = torch.randn(2, T, (nq + 2 * nkv) * D, generator=_g(3)).to(DEV)

    def run(inwg=-1, **kw):
        out = torch.zeros(T, nq * D, dtype=torch.bfloat16, device=DEV)
        lib.function("arle_attn_decode_inwg")(inwg)
        try:
            return ops.attn_decode_prep(parts, out, k.clone(), v.clone(), table.to(DEV), i32(list(range(T + 1))), i32(list(range(T))), i32(contexts),
                                        max_kv_len=max(contexts) + 1, num_q_heads=nq, num_kv_heads=nkv, head_dim=D, page_size=P, scale=D**-0.5,
                                        eps=1e-6, **kw)
        finally:
            lib.function("arle_attn_decode_inwg")(-1)

    for kw in (dict(splits=1), dict(splits=5), dict(splits=2, inwg=1), dict(splits=2, inwg=0), dict(total_kv_len=sum(contexts) + T), dict()):
        want = mx.quantize(run(**kw), form)
        blocks = mx.empty_rows(T, nq * D, form)
        blocks.elements.view(torch.uint8).fill_(0x77)
        blocks.scales.view(torch.uint8).fill_(0x77)
        got = run(blocks=blocks, **kw)
        assert got is blocks and _same_rows(got, want), kw
    with pytest.raises(ops.ShapeError):
        run(blocks=mx.empty_rows(T, nq * D + 32, form))


def _same_rows(a, b):
    return a[2:5] == b[2:5] and all(torch.equal(p, q) for p, q in zip(plain.unpack(a), plain.unpack(b)))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("nq,nkv,window", [(32, 8, 0), (8, 2, 0), (4, 4, 40), (12, 4, 0)])
@pytest.mark.parametrize("portions", [[(0, 300)], [(0, 2048)], [(700, 64), (0, 33), (5, 500)], [(0, 20), (100, 1)]])
def test_portions_that_leave_blocks(form, nq, nkv, window, portions):
    """Prompt portions (position, tokens) whose results leave in blocks, bit for bit those that quantize makes of the same step's; where the step
    holds decoded tokens too, or rows have padding, the results come as they are."""
    from arle_amd.kernels import ops

    P, D, T = 16, 128, sum(n for _, n in portions)
    pages = [(at + n + P - 1) // P for at, n in portions]
    order = torch.randperm(sum(pages), generator=_g(1)).to(torch.int32)
    table = torch.zeros(len(portions), max(pages), dtype=torch.int32)
    for i, part in enumerate(order.split(pages)):
        table[i, :len(part)] = part
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(sum(pages), nkv, *shape, generator=_g(2)).bfloat16().to(DEV) for shape in ((P, D), (D, P)))
    q = torch.randn(T, nq * D, generator=_g(3)).bfloat16().to(DEV)
    row0 = [0]
    for _, n in portions:
        row0.append(row0[-1] + n)
    lengths = [n for _, n in portions]

    def run(**kw):
        out = torch.zeros(T, nq * D, dtype=torch.bfloat16, device=DEV)
        return ops.attn_paged_mfma(q, out, k, v, table.to(DEV), i32(row0), i32(list(range(len(portions)))), i32([at for at, _ in portions]),
                                   max_qlen=max(lengths), min_qlen=min(lengths), max_kv_len=max(at + n for at, n in portions), num_q_heads=nq,
                                   num_kv_heads=nkv, head_dim=D, page_size=P, scale=D**-0.5, window=window, **kw)

    for kw in (dict(portion_splits=1), dict(), dict(portion_splits=2)):
        want = mx.quantize(run(**kw), form)
        blocks = mx.empty_rows(T, nq * D, form)
        blocks.elements.view(torch.uint8).fill_(0x77)
        blocks.scales.view(torch.uint8).fill_(0x77)
        got = run(blocks=blocks, **kw)
        whole = kw == dict(portion_splits=1) and min(lengths) * nq // nkv > 16 and nq * D % 512 == 0
        assert (got is blocks) or not whole
        if got is not blocks:
            assert kw == dict(portion_splits=2) or kw == dict() or not whole
            got = mx.quantize(got, form)
        assert _same_rows(got, want), kw
    with pytest.raises(ops.ShapeError):
        run(blocks=mx.empty_rows(T + 1, nq * D, form))
