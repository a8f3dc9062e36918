"""Typed Python entry points of the microscaled kernels: rows and weights in blocks of 32 numbers that share a power of two.

Two forms of a row: "mxfp8" holds its numbers as e4m3 (8 bits, largest 448), "mxfp4" as e2m1 (4 bits, largest 6).  A block's scale
is 2^(code - 127), the smallest with which none of its numbers is past the largest; elements round to nearest, ties to even.  A
block with a NaN or an infinity has a NaN for its scale, and its numbers and every sum that they enter are NaN.  Weights are held
as "mxfp4", laid out once by `lay_weight`; the rows that meet them may be either form.

As everywhere in this package the host checks what a kernel assumes, the kernels run on torch's current stream, and there is no CPU
path.
"""
from __future__ import annotations

import dataclasses
import math

import torch

from . import lib, ops
from .ops import BF16, F32, ShapeError, _code, _i32, _need, _ptr, _rows, _stream

BLOCK = 32
PAD = 256                # a row's numbers are padded with zeros to a multiple of this, for products that walk whole steps
TILE = 128               # k of an operand tile
MAX_WIDTH = 16384        # of a norm's rows, which the kernel keeps in registers
BITS = {"mxfp8": 8, "mxfp4": 4}
_GRID_MAX = 2**31 - 1


def _here(*tensors) -> None:
    """All on one GPU, the current one: the stream that a kernel runs on is the current device's."""
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise ShapeError("arle_amd kernels run on the GPU only; got a CPU tensor")
        if t.device.index != torch.cuda.current_device():
            raise ShapeError(f"tensor on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


def _bits(form: str) -> int:
    _need(form in BITS, f"unknown form {form!r} (known: {', '.join(BITS)})")
    return BITS[form]


def padded_width(width: int) -> int:
    return -(-width // PAD) * PAD


@dataclasses.dataclass(frozen=True)
class MXRows:
    """Rows in blocks.  elements uint8: [T, padded] (mxfp8) or [T, padded / 2] (mxfp4, the number with the lower index in the lower
    half of a byte); scales uint8 [T, padded / 32]; zeros from `width` to `padded`, the next multiple of 256."""
    elements: torch.Tensor
    scales: torch.Tensor
    width: int
    form: str

    @property
    def rows(self) -> int:
        return self.elements.shape[0]

    @property
    def padded(self) -> int:
        return padded_width(self.width)

    def elements_e4m3(self) -> torch.Tensor:
        """The elements of "mxfp8" rows as torch's type, a view."""
        _need(self.form == "mxfp8", f"{self.form} elements are no e4m3")
        return self.elements[:, :self.width].view(torch.float8_e4m3fn)

    def scales_e8m0(self) -> torch.Tensor:
        """The scales as torch's type of bare exponents, a view [T, ceil(width / 32)]."""
        return self.scales[:, :-(-self.width // BLOCK)].view(torch.float8_e8m0fnu)

    def __getitem__(self, rows: slice) -> "MXRows":
        _need(isinstance(rows, slice), "MXRows take a slice of rows")
        return MXRows(self.elements[rows], self.scales[rows], self.width, self.form)


def _empty_rows(rows: int, width: int, form: str, device) -> MXRows:
    padded = padded_width(width)
    return MXRows(torch.empty((rows, padded * BITS[form] // 8), dtype=torch.uint8, device=device),
                  torch.empty((rows, padded // BLOCK), dtype=torch.uint8, device=device), width, form)


def _check_rows(x: MXRows, name: str = "x") -> None:
    """The kernels read 16 bytes of elements and words of scales at a time."""
    _need(type(x) is MXRows, f"{name} must be MXRows (see quantize), got {type(x).__name__}")
    bits = _bits(x.form)
    _here(x.elements, x.scales)
    e, s = x.elements, x.scales
    _need(x.width > 0, f"{name}: no columns")
    _need(e.dtype == torch.uint8 and e.dim() == 2 and e.shape[1] == x.padded * bits // 8 and s.dtype == torch.uint8
          and tuple(s.shape) == (e.shape[0], x.padded // BLOCK),
          f"{name}: {x.form} rows of {x.width} are uint8 [T, {x.padded * bits // 8}] and [T, {x.padded // BLOCK}]")
    _need(e.shape[0] <= 1 or (e.stride(0) % 16 == 0 and s.stride(0) % 4 == 0), f"{name}: rows must be 16 bytes apart, scales 4")
    _need(e.stride(1) == 1 and s.stride(1) == 1 and e.data_ptr() % 16 == 0 and s.data_ptr() % 4 == 0,
          f"{name}: elements must start at 16 bytes, scales at 4, both with contiguous rows")


def rows_from_codes(elements: torch.Tensor, scales: torch.Tensor, width: int, form: str) -> MXRows:
    """Rows from codes that exist already: elements uint8 [T, at least width], a code a byte in both forms; scales uint8 [T, ceil(width / 32)]."""
    bits = _bits(form)
    _here(elements, scales)
    _need(elements.dtype == torch.uint8 and elements.dim() == 2 and scales.dtype == torch.uint8 and scales.dim() == 2, "codes are uint8 [T, ...]")
    T = elements.shape[0]
    blocks = -(-width // BLOCK)
    _need(width > 0 and elements.shape[1] >= width and tuple(scales.shape) == (T, blocks), f"codes of rows of {width} are [T, {width}] and [T, {blocks}]")
    padded = padded_width(width)
    e = torch.nn.functional.pad(elements[:, :width], (0, padded - width))
    if bits == 4:
        _need(T == 0 or int(e.max()) < 16, "a code of 4 bits is under 16")
        e = e[:, 0::2] | (e[:, 1::2] << 4)
    return MXRows(e.contiguous(), torch.nn.functional.pad(scales, (0, padded // BLOCK - blocks)).contiguous(), width, form)


# ----------------------------------------------------------------------- rows


def quantize(x: torch.Tensor, form: str = "mxfp8") -> MXRows:
    """x [T, K] float32 or bfloat16 in blocks of 32 along K."""
    bits = _bits(form)
    _here(x)
    _rows(x, "x")
    T, K = x.shape
    _need(K > 0, "quantize: no columns")
    _need(T <= _GRID_MAX and padded_width(K) < 2**27, "quantize: too large for one launch")
    out = _empty_rows(T, K, form, x.device)
    if T == 0:
        return out
    size = x.element_size()
    aligned = K % 8 == 0 and x.data_ptr() % (4 * size) == 0 and x.stride(0) % 4 == 0
    lib.call("arle_mx_quantize", x.data_ptr(), _code(x), x.stride(0), out.elements.data_ptr(), out.scales.data_ptr(), bits, T, K, out.padded,
             int(aligned), _stream())
    return out


def values(x: MXRows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The numbers that the elements stand for, [T, width] in float32 (exact) or bfloat16 (exact but for numbers under its smallest normal one)."""
    _check_rows(x)
    _need(dtype in (torch.float32, torch.bfloat16), "values come in float32 or bfloat16")
    out = torch.empty((x.rows, x.width), dtype=dtype, device=x.elements.device)
    if x.rows:
        lib.call("arle_mx_values", x.elements.data_ptr(), x.elements.stride(0), x.scales.data_ptr(), x.scales.stride(0), BITS[x.form],
                 out.data_ptr(), _code(out), x.rows, x.width, _stream())
    return out


def add_rmsnorm(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, form: str = "mxfp8",
                rows: torch.Tensor | None = None) -> MXRows:
    """residual += delta (float32, in place unless `rows` is given); its root-mean-square norm in blocks, made from the 32-bit products.

    delta is None, [T, H], or a stack [S, T, H] of partial sums that are added in the order of the stack, as for ops.add_rmsnorm;
    rows (int32): the rows of the residual that are wanted, the last time it is read."""
    bits = _bits(form)
    _here(residual, delta, weight, rows)
    _need(residual.dtype == torch.float32 and residual.dim() == 2 and residual.is_contiguous(), "residual must be contiguous float32 [T, H]")
    T, width = residual.shape
    _need(0 < width <= MAX_WIDTH, f"a norm's rows have 1 to {MAX_WIDTH} columns, got {width}")
    n_delta, delta_code = 0, F32
    if delta is not None:
        _need(delta.dim() in (2, 3) and tuple(delta.shape[-2:]) == (T, width) and delta.is_contiguous() and delta.dtype in ops._CODES
              and (delta.dim() == 2 or delta.shape[0] >= 1), "delta must match the residual ([T, H] or a stack [S, T, H])")
        n_delta, delta_code = (delta.shape[0] if delta.dim() == 3 else 1), _code(delta)
    _need(weight.shape == (width,) and weight.is_contiguous(), "norm weight must be [width]")
    n_rows = T
    if rows is not None:
        _i32(rows, "rows")
        n_rows = rows.numel()
    out = _empty_rows(n_rows, width, form, residual.device)
    if n_rows == 0:
        return out
    ops_of = [t for t in (residual, delta, weight) if t is not None]
    aligned = width % 4 == 0 and all(t.data_ptr() % (4 * t.element_size()) == 0 for t in ops_of)
    lib.call("arle_mx_add_rmsnorm", residual.data_ptr(), _ptr(delta), n_delta, residual.numel(), delta_code, weight.data_ptr(), _code(weight),
             out.elements.data_ptr(), out.scales.data_ptr(), bits, _ptr(rows), n_rows, width, out.padded, int(aligned), float(eps), _stream())
    return out


# ------------------------------------------------------------------- products


@dataclasses.dataclass(frozen=True)
class MXWeight:
    """A weight [n, k] in 4 bits, laid out for the products.  tiles uint8 [tiles of 16 rows, tiles of 128 k, 64, 16], scales uint8
    [tiles of 16 rows, groups of 512 k, 64, 4].  gated: n = 2 * ff rows, the gate's and then the up's, held in turns of 16 with both
    halves padded with zeros to a multiple of 256."""
    tiles: torch.Tensor
    scales: torch.Tensor
    n: int
    k: int
    gated: bool = False

    @property
    def nbytes(self) -> int:
        return self.tiles.numel() + self.scales.numel()


def lay_weight(rows: MXRows, gated: bool = False) -> MXWeight:
    """The operand tiles of a weight given as "mxfp4" rows (quantize(w, "mxfp4")): a rearrangement at load time, the codes are untouched."""
    _check_rows(rows, "weight")
    _need(rows.form == "mxfp4", "weights are held in 4 bits (mxfp4)")
    n, padded = rows.rows, rows.padded
    _need(n > 0, "weight: no rows")
    e, s = rows.elements, rows.scales
    if gated:
        _need(n % 2 == 0, "a gated weight has as many gate rows as up rows")
        ff = n // 2
        more = padded_width(ff) - ff
        turns = lambda t: torch.nn.functional.pad(t.reshape(2, ff, -1), (0, 0, 0, more)).view(2, (ff + more) // 16, 16, -1).transpose(0, 1).flatten(0, 2)
        e, s = turns(e), turns(s)
    more = -e.shape[0] % 16
    e, s = torch.nn.functional.pad(e, (0, 0, 0, more)), torch.nn.functional.pad(s, (0, -s.shape[1] % 16, 0, more))
    tiles = e.reshape(-1, 16, padded // TILE, 4, 16).permute(0, 2, 3, 1, 4).reshape(-1, padded // TILE, 64, 16).contiguous()
    scales = s.reshape(s.shape[0] // 16, 16, -1, 4, 4).permute(0, 2, 4, 1, 3).reshape(s.shape[0] // 16, -1, 64, 4).contiguous()
    return MXWeight(tiles, scales, n, rows.width, gated)


def _check_weight(w: MXWeight, x: MXRows, gated: bool) -> None:
    _need(type(w) is MXWeight, f"the weight must be MXWeight (see lay_weight), got {type(w).__name__}")
    _here(w.tiles, w.scales)
    _need(w.gated == gated, "gate_up_act takes a weight laid out with gated=True, gemm one without")
    _need(w.k == x.width, f"inner sizes differ ({x.width} vs {w.k})")
    k_tiles = x.padded // TILE
    n_tiles = 2 * padded_width(w.n // 2) // 16 if gated else -(-w.n // 16)
    _need(w.tiles.dtype == torch.uint8 and tuple(w.tiles.shape) == (n_tiles, k_tiles, 64, 16) and w.tiles.is_contiguous()
          and w.tiles.data_ptr() % 16 == 0 and w.scales.dtype == torch.uint8 and w.scales.is_contiguous()
          and tuple(w.scales.shape) == (n_tiles, -(-k_tiles // 4), 64, 4) and w.scales.data_ptr() % 4 == 0,
          f"the tiles of a [{w.n}, {w.k}] weight are [{n_tiles}, {k_tiles}, 64, 16], their scales [{n_tiles}, {-(-k_tiles // 4)}, 64, 4]")


_EPI_F32, _EPI_BF16, _EPI_GATE = 0, 1, {"mxfp8": 2, "mxfp4": 3}
_ROW_TILES = {0: 1, 1: 2, 2: 4}                                             # variant -> tiles of 16 rows (mx_gemm_rows_kernel)
_TILE_SHAPES = {3: (64, 128), 4: (128, 128), 5: (128, 256), 6: (256, 256)}  # variant -> rows and columns (mx_gemm_tiles_kernel)


def _variant(M: int, n: int) -> int:
    if M <= 64:
        return 0 if M <= 16 else 1 if M <= 32 else 2
    for v in (6, 5, 4):
        rows, cols = _TILE_SHAPES[v]
        if -(-M // rows) * -(-n // cols) >= 256:
            return v
    return 3


def _launch(x: MXRows, w: MXWeight, epilogue: int, variant: int, splits: int, out, ldo: int, split_stride: int, out_scales, ldos: int, n: int,
            vec: bool) -> None:
    M = x.rows
    k_tiles, bits = w.tiles.shape[1], BITS[x.form]
    _need(variant not in _ROW_TILES or M <= 16 * _ROW_TILES[variant], f"variant {variant} takes {16 * _ROW_TILES.get(variant, 0)} rows")
    steps = k_tiles if variant in _ROW_TILES or bits == 8 else k_tiles // 2     # what the kernel walks K in
    per_split = -(-steps // splits)
    _need(splits >= 1 and (splits - 1) * per_split < steps, f"{splits} parts of {steps} steps: some would have none")
    lib.call("arle_mx_gemm", bits, epilogue, variant, x.elements.data_ptr(), x.elements.stride(0), x.scales.data_ptr(), x.scales.stride(0),
             w.tiles.data_ptr(), w.scales.data_ptr(), out.data_ptr(), ldo, split_stride, _ptr(out_scales), ldos, M, n, w.tiles.shape[0], k_tiles,
             splits, per_split, int(vec), _stream())


def gemm(x: MXRows, w: MXWeight, out_dtype: torch.dtype = torch.bfloat16, partials_ok: bool = False, *, variant: int | None = None,
         splits: int | None = None) -> torch.Tensor:
    """x [T, K] . w [N, K]^T with sums of 32 bits -> [T, N] in `out_dtype`; with `partials_ok` possibly a float32 stack [S, T, N] whose
    sum over S, in order, is the product (as Linear's)."""
    _check_rows(x)
    _check_weight(w, x, False)
    _need(out_dtype in (torch.float32, torch.bfloat16), "products come in float32 or bfloat16")
    M, N, device = x.rows, w.n, x.elements.device
    if M == 0:
        return torch.empty((0, N), dtype=out_dtype, device=device)
    if variant is None:
        variant = _variant(M, N)
    splits = splits or 1
    parts = splits > 1
    out = torch.empty((splits, M, N) if parts else (M, N), dtype=torch.float32 if parts else out_dtype, device=device)
    _launch(x, w, _EPI_F32 if out.dtype == torch.float32 else _EPI_BF16, variant, splits, out, N, M * N, None, 0, N, N % 8 == 0)
    if parts and not partials_ok:
        return ops.sum_partials(out, out_dtype)
    return out


def gate_up_act(x: MXRows, w: MXWeight, form: str = "mxfp8", *, variant: int | None = None) -> MXRows:
    """silu(x . gate^T) * (x . up^T) in blocks, [T, ff] from a weight laid out with gated=True: the rows of the second half's product,
    made from the 32-bit sums in one kernel."""
    _check_rows(x)
    _check_weight(w, x, True)
    _bits(form)
    out = _empty_rows(x.rows, w.n // 2, form, x.elements.device)
    if x.rows == 0:
        return out
    if variant is None:
        variant = _variant(x.rows, 16 * w.tiles.shape[0])
    _launch(x, w, _EPI_GATE[form], variant, 1, out.elements, out.elements.stride(0), 0, out.scales, out.scales.stride(0), 16 * w.tiles.shape[0], True)
    return out
