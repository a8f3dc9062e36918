"""Typed Python entry points of the microscaled kernels: rows and weights in blocks of 32 numbers that share a power of two.

Two forms of a row: "mxfp8" holds its numbers as e4m3 (8 bits, largest 448), "mxfp4" as e2m1 (4 bits, largest 6).  A block's scale
is 2^(code - 127), the smallest with which none of its numbers is past the largest; elements round to nearest, ties to even.  A
block with a NaN or an infinity has a NaN for its scale, and its numbers and every sum that they enter are NaN.  Weights are held
as "mxfp4", laid out once by `lay_weight`; the rows that meet them may be either form.

How wide a product's sums are depends on the form of its rows.  With "mxfp4" rows the instruction's products lose nothing, and they are added in 32 bits.
With "mxfp8" rows it aligns the products of eight neighbouring k (8 i to 8 i + 7) to the largest of them and drops of the others what is under 2^-13 of that one's
power of two: up to 7 * 2^-13 of an eight's largest product, where 32 bits would lose 2^-24 of it; the eights are added in 32 bits.  That is a 2^-9th of what rounding
to e4m3 has taken from numbers before, but a caller whose e4m3 numbers are exact gets 13 bits of an eight's sum, also as float32.

As everywhere in this package the host checks what a kernel assumes, the kernels run on torch's current stream, and there is no CPU
path.
"""
from __future__ import annotations

import collections
import functools

import torch

from . import lib, ops
from .ops import _CODES, F32, ShapeError, _ptr

BLOCK = 32
PAD = 512                # a row's numbers are padded with zeros to a multiple of this, for products that walk whole steps
TILE = 128               # k of an operand tile
MAX_K = 2**22            # numbers of a row: 256 rows of elements are within 32 bits of offsets
MAX_WEIGHT = 2**35       # numbers of a weight: its scales are
MAX_WIDTH = 16384        # of a norm's rows, which the kernel keeps in registers
BITS = {"mxfp8": 8, "mxfp4": 4}
_ELEMENTS = {"mxfp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}
_SCALES = torch.float8_e8m0fnu


# The checks below are plain `if`s whose message is made only where it is raised, and rows and weights are checked where they are
# made, not at every call: with eagerly made messages and checks at every use a product of a few rows cost the host 14 us, so 6.


_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _here(*tensors) -> int:
    """The current device, the one whose stream a kernel runs on and that all of the tensors have to be on."""
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ShapeError("arle_amd kernels run on the GPU only; got a CPU tensor")
    device = _current()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ShapeError(f"tensor on {t.device}, the current device is cuda:{device}")
    return device


def _same_device(held: int) -> int:
    """The current device, which has to be the one that rows and weights are held on."""
    device = _current()
    if held != device:
        raise ShapeError(f"rows or weights on cuda:{held}, the current device is cuda:{device}")
    return device


_functions: dict = {}


def _function(name: str):
    fn = _functions[name] = lib.function(name)
    return fn


def _failed(name: str, status: int) -> None:
    raise lib.KernelError(f"{name} failed with HIP error {status}")


_stream = ops._raw_stream or (lambda device: torch.cuda.current_stream(device).cuda_stream)      # handle of the current stream of a device


def _bits(form: str) -> int:
    bits = BITS.get(form)
    if bits is None:
        raise ShapeError(f"unknown form {form!r} (known: {', '.join(BITS)})")
    return bits


def padded_width(width: int) -> int:
    return -(-width // PAD) * PAD


_Rows = collections.namedtuple("_Rows", "elements scales width form rows padded bits device")


def _checked_fields(cls, fields: tuple, given: int, derived: tuple):
    if derived and derived != fields[given:]:
        raise ShapeError(f"{cls.__name__} of {fields[given:]} cannot be {derived}")
    return tuple.__new__(cls, fields)


class MXRows(_Rows):
    """Rows in blocks, MXRows(elements, scales, width, form).  elements: float8_e4m3fn [T, padded] (mxfp8) or uint8 [T, padded / 2] (mxfp4, the number
    with the lower index in the lower half of a byte); scales float8_e8m0fnu [T, padded / 32]; zeros (codes of 0) from `width` to `padded`, the next
    multiple of 512.  Views whose rows lie apart are fine where rows start at multiples of 16 bytes."""
    __slots__ = ()

    def __new__(cls, elements: torch.Tensor, scales: torch.Tensor, width: int, form: str, *derived):
        """derived: the other fields, if given (a tuple put together again from its fields): they have to be what the first four say."""
        bits = _bits(form)
        device = _here(elements, scales)
        if not 1 <= width <= MAX_K:
            raise ShapeError(f"rows have 1 to {MAX_K} columns, got {width}")
        padded = padded_width(width)
        e, s = elements, scales
        if not (e.dtype == _ELEMENTS[form] and e.dim() == 2 and e.shape[1] == padded * bits // 8 and s.dtype == _SCALES
                and tuple(s.shape) == (e.shape[0], padded // BLOCK)):
            raise ShapeError(f"{form} rows of {width} are {_ELEMENTS[form]} [T, {padded * bits // 8}] with scales {_SCALES} [T, {padded // BLOCK}], got "
                             f"{e.dtype} {tuple(e.shape)} with {s.dtype} {tuple(s.shape)}")
        if (e.stride(1) != 1 or s.stride(1) != 1 or e.data_ptr() % 16 or s.data_ptr() % 16
                or (e.shape[0] > 1 and (e.stride(0) % 16 or s.stride(0) % 16 or max(e.stride(0), s.stride(0)) > 2 * MAX_K))):
            raise ShapeError(f"rows of elements and scales must lie together and start at multiples of 16 bytes, up to {2 * MAX_K} apart")
        return _checked_fields(cls, (e, s, int(width), form, e.shape[0], padded, bits, device), 4, derived)

    def __getnewargs__(self):      # of a copy: what it is made from, which is checked again
        return self[:4]

    @classmethod
    def _make(cls, fields):
        """What `_replace` makes too: a plain tuple of the fields, which no kernel takes, as nothing has checked them."""
        return _Rows._make(fields)

    def part(self, start: int, stop: int) -> "MXRows":
        """Rows start .. stop - 1, a view."""
        return MXRows(self.elements[start:stop], self.scales[start:stop], self.width, self.form)

    def elements_e4m3(self) -> torch.Tensor:
        """The elements of "mxfp8" rows without the padding, a view [T, width]."""
        if self.bits != 8:
            raise ShapeError(f"{self.form} elements are no e4m3")
        return self.elements if self.width == self.padded else self.elements[:, :self.width]

    def scales_e8m0(self) -> torch.Tensor:
        """The scales without the padding, a view [T, ceil(width / 32)]."""
        return self.scales if self.width == self.padded else self.scales[:, :-(-self.width // BLOCK)]


_new = tuple.__new__
_empty = torch.empty


def _new_rows(rows: int, width: int, form: str, bits: int, device: int) -> MXRows:
    padded, on = -(-width // PAD) * PAD, _DEVICES.get(device) or _device(device)
    return _new(MXRows, (_empty(rows, padded * bits // 8, dtype=_ELEMENTS[form], device=on), _empty(rows, padded // BLOCK, dtype=_SCALES, device=on),
                         width, form, rows, padded, bits, device))


def empty_rows(rows: int, width: int, form: str) -> MXRows:
    """Rows that a kernel is to fill, on the current device."""
    bits = _bits(form)
    if rows < 0 or not 1 <= width <= MAX_K:
        raise ShapeError(f"rows have 1 to {MAX_K} columns, got [{rows}, {width}]")
    return _new_rows(rows, width, form, bits, _current())


_DEVICES: dict = {}


def _device(index: int) -> torch.device:
    return _DEVICES.setdefault(index, torch.device("cuda", index))


def rows_from_codes(elements: torch.Tensor, scales: torch.Tensor, width: int, form: str) -> MXRows:
    """Rows from codes that exist already: elements uint8 [T, at least width], a code a byte in both forms; scales uint8 [T, ceil(width / 32)]."""
    bits = _bits(form)
    _here(elements, scales)
    blocks = -(-width // BLOCK)
    if not (elements.dtype == torch.uint8 and elements.dim() == 2 and scales.dtype == torch.uint8 and width > 0 and elements.shape[1] >= width
            and tuple(scales.shape) == (elements.shape[0], blocks)):
        raise ShapeError(f"codes of rows of {width} are uint8 [T, {width}] and [T, {blocks}], got {elements.dtype} {tuple(elements.shape)} and "
                         f"{scales.dtype} {tuple(scales.shape)}")
    padded = padded_width(width)
    e = torch.nn.functional.pad(elements[:, :width], (0, padded - width))
    if bits == 4:
        if e.numel() and int(e.max()) > 15:
            raise ShapeError("a code of 4 bits is under 16")
        e = e[:, 0::2] | (e[:, 1::2] << 4)
    return MXRows(e.contiguous().view(_ELEMENTS[form]), torch.nn.functional.pad(scales, (0, padded // BLOCK - blocks)).contiguous().view(_SCALES), width, form)


# ----------------------------------------------------------------------- rows


def quantize(x: torch.Tensor, form: str = "mxfp8") -> MXRows:
    """x [T, K] float32 or bfloat16 in blocks of 32 along K."""
    bits = BITS.get(form) or _bits(form)
    device = x.get_device()
    if device < 0 or device != _current():
        _here(x)
    code = _CODES.get(x.dtype)
    if code is None or x.dim() != 2:
        raise ShapeError(f"quantize takes float32 or bfloat16 [T, K], got {x.dtype} {tuple(x.shape)}")
    T, K = x.shape
    stride, step = x.stride()
    if K < 1 or (step != 1 and K > 1) or K > MAX_K:
        raise ShapeError(f"quantize takes rows of 1 to {MAX_K} numbers that lie together, got {tuple(x.shape)} with strides {tuple(x.stride())}")
    out = _new_rows(T, K, form, bits, device)
    if T:
        at = x.data_ptr()
        aligned = K % 8 == 0 and stride % 4 == 0 and at % (16 if code == F32 else 8) == 0
        status = (_functions.get("arle_mx_quantize") or _function("arle_mx_quantize"))(
            at, code, stride, out[0].data_ptr(), out[1].data_ptr(), bits, T, K, out[5], aligned, _stream(device))
        if status:
            _failed("arle_mx_quantize", status)
    return out


def values(x: MXRows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The numbers that the elements stand for, [T, width] in float32 (exact) or bfloat16 (exact but for numbers under its smallest normal one)."""
    if type(x) is not MXRows:
        raise ShapeError(f"values takes MXRows (see quantize), got {type(x).__name__}")
    device = _same_device(x.device)
    if dtype not in _CODES:
        raise ShapeError("values come in float32 or bfloat16")
    out = torch.empty((x.rows, x.width), dtype=dtype, device=_device(device))
    if x.rows:
        status = (_functions.get("arle_mx_values") or _function("arle_mx_values"))(
            x.elements.data_ptr(), x.elements.stride(0), x.scales.data_ptr(), x.scales.stride(0), x.bits, out.data_ptr(),
            _CODES[dtype], x.rows, x.width, _stream(device))
        if status:
            _failed("arle_mx_values", status)
    return out


def add_rmsnorm(residual: torch.Tensor, delta: torch.Tensor | None, weight: torch.Tensor, eps: float, form: str = "mxfp8",
                rows: torch.Tensor | None = None) -> MXRows:
    """residual += delta (float32, in place unless `rows` is given); its root-mean-square norm in blocks, made from the 32-bit products.

    delta is None, [T, H], or a stack [S, T, H] of partial sums that are added in the order of the stack, as for ops.add_rmsnorm;
    rows (int32): the rows of the residual that are wanted, the last time it is read."""
    bits = BITS.get(form) or _bits(form)
    device = residual.get_device()
    if (device < 0 or device != _current() or weight.get_device() != device or (delta is not None and delta.get_device() != device)
            or (rows is not None and rows.get_device() != device)):
        _here(residual, delta, weight, rows)
    if residual.dtype is not torch.float32 or residual.dim() != 2 or not residual.is_contiguous():
        raise ShapeError("residual must be contiguous float32 [T, H]")
    T, width = residual.shape
    if not 0 < width <= MAX_WIDTH:
        raise ShapeError(f"a norm's rows have 1 to {MAX_WIDTH} columns, got {width}")
    at, w_at, w_code = residual.data_ptr(), weight.data_ptr(), _CODES.get(weight.dtype)
    if weight.dim() != 1 or weight.numel() != width or w_code is None or not weight.is_contiguous():
        raise ShapeError(f"norm weight must be float32 or bfloat16 [{width}]")
    aligned = width % 4 == 0 and at % 16 == 0 and w_at % (16 if w_code == F32 else 8) == 0
    n_delta = delta_at = delta_code = 0
    if delta is not None:
        n_delta, delta_code, dims = 1, _CODES.get(delta.dtype), delta.dim()
        if dims == 3:
            n_delta, rows_of, width_of = delta.shape
        elif dims == 2:
            rows_of, width_of = delta.shape
        else:
            rows_of = width_of = -1
        if rows_of != T or width_of != width or delta_code is None or n_delta < 1 or not delta.is_contiguous():
            raise ShapeError("delta must match the residual ([T, H] or a stack [S, T, H]) in float32 or bfloat16")
        delta_at = delta.data_ptr()
        aligned = aligned and delta_at % (16 if delta_code == F32 else 8) == 0
    n_rows = T
    if rows is not None:
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous():
            raise ShapeError("rows must be int32 1-D")
        n_rows = rows.numel()
    out = _new_rows(n_rows, width, form, bits, device)
    if n_rows:
        status = (_functions.get("arle_mx_add_rmsnorm") or _function("arle_mx_add_rmsnorm"))(
            at, delta_at, n_delta, T * width, delta_code, w_at, w_code, out[0].data_ptr(), out[1].data_ptr(), bits,
            _ptr(rows), n_rows, width, out[5], aligned, eps, _stream(device))
        if status:
            _failed("arle_mx_add_rmsnorm", status)
    return out


# ------------------------------------------------------------------- products


_Weight = collections.namedtuple("_Weight", "tiles scales n k gated n_tiles k_tiles device pitch")


class MXWeight(_Weight):
    """A weight [n, k] in 4 bits, laid out for the products (see lay_weight).  tiles uint8 [tiles of 128 k, tiles of 16 rows, 64, 16], scales uint8
    [groups of 512 k, tiles of 16 rows, 64, 4]; both may be the first rows' tiles of a larger weight.  gated: n = 2 * ff rows, the gate's and then
    the up's, held in turns of 16 with both halves padded with zeros to a multiple of 512."""
    __slots__ = ()

    def __new__(cls, tiles: torch.Tensor, scales: torch.Tensor, n: int, k: int, gated: bool = False, *derived):
        device = _here(tiles, scales)
        if n < 1 or k < 1 or (gated and n % 2):
            raise ShapeError(f"a weight of {n} rows of {k} ({'gated' if gated else 'plain'})")
        if k > MAX_K or n * k > MAX_WEIGHT:
            raise ShapeError(f"a weight has up to {MAX_K} columns and {MAX_WEIGHT} numbers, got [{n}, {k}]")
        k_tiles = padded_width(k) // TILE
        n_tiles = 2 * padded_width(n // 2) // 16 if gated else -(-n // 16)
        if not (tiles.dtype == torch.uint8 and tuple(tiles.shape) == (k_tiles, n_tiles, 64, 16) and scales.dtype == torch.uint8
                and tuple(scales.shape) == (k_tiles // 4, n_tiles, 64, 4)):
            raise ShapeError(f"the tiles of a [{n}, {k}] weight are uint8 [{k_tiles}, {n_tiles}, 64, 16], their scales [{k_tiles // 4}, {n_tiles}, 64, 4]")
        pitch = tiles.stride(0) // 1024
        if (tiles.stride() != (1024 * pitch, 1024, 16, 1) or scales.stride()[1:] != (256, 4, 1) or (k_tiles > 4 and scales.stride(0) != 256 * pitch)
                or pitch < n_tiles or pitch * k_tiles * 2048 > MAX_WEIGHT or tiles.data_ptr() % 16 or scales.data_ptr() % 16):
            raise ShapeError("a step's tiles and scales must lie together, start at multiples of 16 bytes and be equally many apart")
        return _checked_fields(cls, (tiles, scales, int(n), int(k), bool(gated), n_tiles, k_tiles, device, pitch), 5, derived)

    def __getnewargs__(self):
        return self[:5]

    @classmethod
    def _make(cls, fields):      # as for rows: nothing that a kernel takes
        return _Weight._make(fields)

    def first(self, rows: int) -> "MXWeight":
        """The weight's first `rows` rows, a multiple of 16: a view."""
        if self.gated or rows % 16 or not 0 < rows <= self.n:
            raise ShapeError(f"the first {rows} rows of a {'gated' if self.gated else 'plain'} weight of {self.n} are no whole tiles")
        return MXWeight(self.tiles[:, :rows // 16], self.scales[:, :rows // 16], rows, self.k)

    @property
    def nbytes(self) -> int:
        return self.tiles.numel() + self.scales.numel()


def lay_weight(rows: MXRows, gated: bool = False) -> MXWeight:
    """The operand tiles of a weight given as "mxfp4" rows (quantize(w, "mxfp4")): a rearrangement at load time, the codes are untouched."""
    if type(rows) is not MXRows or rows.bits != 4:
        raise ShapeError("weights are held in 4 bits: lay_weight takes mxfp4 rows")
    n, padded = rows.rows, rows.padded
    if n < 1 or (gated and n % 2):
        raise ShapeError("a gated weight has as many gate rows as up rows" if n else "a weight without rows")
    e, s = rows.elements, rows.scales.view(torch.uint8)
    if gated:
        ff = n // 2
        more = padded_width(ff) - ff
        turns = lambda t: torch.nn.functional.pad(t.reshape(2, ff, -1), (0, 0, 0, more)).view(2, (ff + more) // 16, 16, -1).transpose(0, 1).flatten(0, 2)
        e, s = turns(e), turns(s)
    more = -e.shape[0] % 16
    e, s = torch.nn.functional.pad(e, (0, 0, 0, more)), torch.nn.functional.pad(s, (0, -s.shape[1] % 16, 0, more))
    tiles = e.reshape(-1, 16, padded // TILE, 4, 16).permute(2, 0, 3, 1, 4).reshape(padded // TILE, -1, 64, 16).contiguous()
    scales = s.reshape(s.shape[0] // 16, 16, -1, 4, 4).permute(2, 0, 4, 1, 3).reshape(padded // 512, -1, 64, 4).contiguous()
    return MXWeight(tiles, scales, n, rows.width, gated)


_EPI_F32, _EPI_GATE = F32, {"mxfp8": 2, "mxfp4": 3}                         # (sums leave as the type whose code this is)
ROW_VARIANTS, GATED_ROWS = (0, 1), 9                                        # of up to 16 rows (mx_gemm_rows_kernel), sums or gated
# variant of mx_gemm_tiles_kernel -> rows, columns, workgroups a compute unit holds, us to start and end a launch, and us of 128 k for one workgroup
# alone and for a compute unit that is as full as all others, for rows of 8 bits and of 4.  What they were read from (MI355X, us in a captured graph,
# 2.4 of which are the launch; rows x N x K, 8 bits if not said):
#                                  32x64  64x128  128x128  128x256  256x256  128x192  256x192
#   64 x 2,560 x 9,728              16.3    26.4     36.1     41.5     75.5     35.5     58.8
#   128 x 6,144 x 2,560             10.2    10.4     14.3     17.6     24.8     17.2     20.8
#   512 x 2,560 x 9,728             36.8    25.3     39.0     48.3     80.8     43.3     67.4
#   2,048 x 2,560 x 9,728                   64.9     52.3     44.3     77.6     44.1     63.5
#   2,048 x 6,144 x 2,560                   34.8     28.1     31.0     30.4     30.5     27.1
#   4,096 x 6,144 x 4,096                            85.3     77.6     86.6     85.3     75.3
#   4,096 x 4,096 x 12,288                          158.8    143.6    134.0    164.4    181.7
#   8,192 x 6,144 x 2,560                           103.3     98.6     93.3    110.7     94.9
#   8,192 x 2,560 x 9,728                           156.6    154.1    180.0    171.7    152.2
#   2,048 x 2,560 x 9,728, 4 bits                    38.3     33.0     50.6     34.0     46.5
#   4,096 x 6,144 x 4,096, 4 bits                    67.1     59.2     60.2     69.6     55.2
#   gate|up, 64 x 9,728 x 2,560             12.3     14.1     16.4     26.6
#   gate|up, 2,048 x 9,728 x 2,560         143.0     81.4     78.9     85.3
#   gate|up, 4,096 x 12,288 x 4,096        546.3    325.0    298.1    276.2
#   the same, 4 bits                                279.4    241.4    197.2
# (gate|up before the activation's last bits, 1 to 3 % more since).  What the choice comes to, us, with add_rmsnorm behind it that reads the parts of K
# (variant, parts): chosen / best of all
#   32 x 4,096 x 12,288   (2, 4) 13.4 / -           64 x 2,560 x 9,728    (3, 7) 14.8 / (2, 4) 14.4     the same, 4 bits       (3, 7) 14.1 / (3, 4) 13.9
#   128 x 4,096 x 12,288  (3, 4) 18.1 / -           256 x 4,096 x 12,288  (3, 2) 23.8 / -               384 x 4,096 x 12,288   (4, 2) 33.0 / (5, 4) 32.6
#   512 x 2,560 x 9,728   (7, 4) 27.7 / (3, 1) 26.9 768 x 4,096 x 12,288  (4, 1) 54.5 / (5, 2) 47.7     1,024 x 4,096 x 12,288 (4, 1) 57.4 / 54.7 (itself again)
#   1,024 x 2,560 x 9,728 (7, 2) 39.2 / -           64 x 5,120 x 25,600   (3, 4) 29.0 / -               512 x 5,120 x 25,600   (7, 2) 75.2 / 72.8 (itself)
# and gate|up, ff x K of 25,600 x 5,120: 1 row (3) 31.7 / (9) 28.0, 16 rows of 4 bits (5) 35.6 / (9) 31.2, 64 rows (3) 38.3 / (5) 36.8, 512 rows (6) 112 / -.
_TILES = {2: (32, 64, 2, 1.5, 0.15, 0.36, 0.15, 0.36), 3: (64, 128, 1, 2.5, 0.28, 0.28, 0.25, 0.25), 4: (128, 128, 2, 2.5, 0.43, 0.78, 0.38, 0.68),
          5: (128, 256, 1, 3.0, 0.48, 0.715, 0.30, 0.55), 6: (256, 256, 1, 5.0, 0.95, 1.32, 0.55, 0.92), 7: (128, 192, 1, 3.0, 0.44, 0.59, 0.36, 0.47),
          8: (256, 192, 1, 4.0, 0.80, 1.05, 0.53, 0.73)}
_PLAIN_TILES = (2, 7, 8)  # whose waves own no whole blocks of 32 gated results
_UNITS = 256             # compute units
_SUM_US, _STACK_BYTES_A_US = 5.0, 5e6      # a launch more, which an eager caller pays the host for too; the stack written and read


def _tiles_us(variant: int, M: int, N: int, k_tiles: int, bits: int, splits: int) -> float:
    """What a product is expected to take, as far as variants and parts of K are compared by it."""
    rows, cols, held, start, *us = _TILES[variant]
    alone, full = us[:2] if bits == 8 else us[2:]
    turns, rest = divmod(-(-M // rows) * -(-N // cols) * splits, _UNITS * held)
    # the last turn has fewer workgroups; up to one a unit each of them has its unit to itself
    busy = 0.0 if held > 1 and rest <= _UNITS else rest / (_UNITS * held)
    steps = 4 * -(-k_tiles // (4 * splits))
    return start / 2 + turns * (steps * full + start / 2) + (steps * (alone + (full - alone) * busy) + start / 2 if rest else 0.0)


@functools.lru_cache(maxsize=4096)
def _plan(M: int, n_tiles: int, k_tiles: int, bits: int, gated: bool, whole: bool) -> tuple:
    """(variant, parts of K, steps a part) for sizes; whole: the sums have to come whole."""
    variant, splits = _choose(M, n_tiles, k_tiles, bits, gated, whole)
    return variant, splits, _per_split(M, k_tiles, bits, variant, splits)


def _choose(M: int, n_tiles: int, k_tiles: int, bits: int, gated: bool, whole: bool) -> tuple:
    N = 16 * n_tiles
    if M <= 16 and not gated:
        # us at 8 rows, pairs of columns tiles in 4 waves and K in as many parts as stand / the same whole / single tiles in 8 waves, whole:
        # 2,560 x 4,096  4.1 (8) / 5.7 / 5.0;  2,560 x 9,728  5.4 (8) / 9.6 / 7.7;  6,144 x 2,560  4.3 (4) / 4.7 / 5.4;
        # 10,240 x 5,120  8.6 (2) / 10.4 / 10.3.  Who reads the parts pays for each of them, so that with a norm behind it 1, 2, 4 and 8 parts take
        # 8.9, 8.1, 8.5 and 9.4 (2,560 x 4,096), 12.8, 10.3, 10.4 and 11.0 (2,560 x 9,728), and a decode step of 8 requests at the Qwen3-4B
        # widths 2.17, 2.12, 2.11, 2.07 and 2.08 ms with 640, 400, 320, 240 and 160 pairs and parts in all
        pairs = -(-n_tiles // 2)
        if whole:
            return (0 if pairs >= 192 else 1), 1
        return 0, _even(min(max(1, round(240 / pairs)), 8, max(1, k_tiles // 4)), k_tiles)
    if M <= 16 and n_tiles <= 1024:
        # us, the few rows' kernel / tiles of 64 x 128, of which there are too few to fill the chip then: 8 x 1,024 x 4,096 6.6 / 10.6, 8 x 3,200 x 1,024 3.7 /
        # 5.4, 16 x 6,144 x 2,048 6.1 / 8.0 (ff x K); 8 x 9,728 x 2,560 9.2 / 9.3, 16 rows 10.0 / 9.3, 8 x 12,288 x 4,096 13.5 / 12.7
        return GATED_ROWS, 1
    found = []
    for variant in _TILES:
        if gated and variant in _PLAIN_TILES:
            continue
        for splits in (1,) if gated else (1, 2, 4, 8):
            splits = _even(splits, k_tiles // 4)
            us = _tiles_us(variant, M, N, k_tiles, bits, splits)
            if splits > 1:
                us += 8 * splits * M * N / _STACK_BYTES_A_US + (_SUM_US if whole else 0)
            found.append((us, variant, splits))
    _, variant, splits = min(found)
    return variant, splits


def _even(splits: int, steps: int) -> int:
    """As many parts as `splits` parts of equal length make of `steps`, none of them empty."""
    return -(-steps // -(-steps // min(splits, steps)))


def _per_split(M: int, k_tiles: int, bits: int, variant: int, splits: int) -> int:
    """Steps of K that a part walks; refuses what the kernel was not written for."""
    few = variant in ROW_VARIANTS or variant == GATED_ROWS
    if not few and variant not in _TILES:
        raise ShapeError(f"no variant {variant}")
    if few and M > 16:
        raise ShapeError(f"variant {variant} takes 16 rows, got {M}")
    steps = k_tiles if few else k_tiles // 4
    if splits == 1:
        return steps
    per_split = -(-steps // splits) if splits > 0 else 0
    if splits < 1 or splits > 65535 or (splits - 1) * per_split >= steps:
        raise ShapeError(f"{splits} parts of {steps} steps: some would have none")
    return per_split


def _checked(x: MXRows, w: MXWeight, gated: bool) -> int:
    if type(x) is not MXRows or type(w) is not MXWeight:
        raise ShapeError(f"products take MXRows and an MXWeight (see quantize, lay_weight), got {type(x).__name__} and {type(w).__name__}")
    device = x[7]
    if x[2] != w[3] or w[4] is not gated or w[7] != device:
        if x.width != w.k:
            raise ShapeError(f"inner sizes differ ({x.width} vs {w.k})")
        if w.gated != gated:
            raise ShapeError("gate_up_act takes a weight laid out with gated=True, gemm one without")
        raise ShapeError(f"rows on cuda:{x.device}, the weight on cuda:{w.device}")
    if device != _current():
        _same_device(device)
    return device


def gemm(x: MXRows, w: MXWeight, out_dtype: torch.dtype = torch.bfloat16, partials_ok: bool = False, *, variant: int | None = None,
         splits: int | None = None) -> torch.Tensor:
    """x [T, K] . w [N, K]^T -> [T, N] in `out_dtype`, with sums of 32 bits behind what "mxfp8" rows lose inside every eight k (up to 7 * 2^-13 of its
    largest product: see the module); with `partials_ok` possibly a float32 stack [S, T, N] whose sum over S, in order, is the product (as Linear's).
    The sizes choose the kernel, or `variant` names it and `splits` its parts of K (default: 1)."""
    device = _checked(x, w, False)
    code = _CODES.get(out_dtype)
    if code is None:
        raise ShapeError("products come in float32 or bfloat16")
    elements, held, _, _, M, _, bits, _ = x
    tiles, tile_scales, N, _, _, n_tiles, k_tiles, _, pitch = w
    on = _DEVICES.get(device) or _device(device)
    if M == 0:
        return _empty(0, N, dtype=out_dtype, device=on)
    if variant is None:
        if splits is not None:
            raise ShapeError(f"{splits} parts of K without the variant that walks them: the sizes choose both, or the caller does")
        variant, splits, per_split = _plan(M, n_tiles, k_tiles, bits, False, not partials_ok)
    else:
        splits = 1 if splits is None else splits
        if variant == GATED_ROWS:
            raise ShapeError(f"variant {variant} makes blocks")
        per_split = _per_split(M, k_tiles, bits, variant, splits)
    parts = splits > 1
    out = _empty(splits, M, N, dtype=torch.float32, device=on) if parts else _empty(M, N, dtype=out_dtype, device=on)
    status = (_functions.get("arle_mx_gemm") or _function("arle_mx_gemm"))(
        bits, _EPI_F32 if parts else code, variant, elements.data_ptr(), elements.stride(0), held.data_ptr(), held.stride(0),
            tiles.data_ptr(), tile_scales.data_ptr(), out.data_ptr(), N, 0, 0, M, N, n_tiles, k_tiles, pitch, splits, per_split, _stream(device))
    if status:
        _failed("arle_mx_gemm", status)
    if parts and not partials_ok:
        return ops.sum_partials(out, out_dtype)
    return out


def gate_up_act(x: MXRows, w: MXWeight, form: str = "mxfp8", *, variant: int | None = None) -> MXRows:
    """silu(x . gate^T) * (x . up^T) in blocks, [T, ff] from a weight laid out with gated=True: the rows of the second half's product,
    made from the sums (as wide as gemm's: see the module) in one kernel.  (A row with a block that is no number is none throughout, its padding too.)"""
    device = _checked(x, w, True)
    out_bits = BITS.get(form) or _bits(form)
    elements, held, _, _, M, _, bits, _ = x
    tiles, tile_scales, n, _, _, n_tiles, k_tiles, _, pitch = w
    out = _new_rows(M, n // 2, form, out_bits, device)
    if M == 0:
        return out
    if variant is None:
        variant, _, per_split = _plan(M, n_tiles, k_tiles, bits, True, True)
    else:
        if variant in ROW_VARIANTS or variant in _PLAIN_TILES:
            raise ShapeError(f"variant {variant} makes no blocks")
        per_split = _per_split(M, k_tiles, bits, variant, 1)
    padded = out[5]
    status = (_functions.get("arle_mx_gemm") or _function("arle_mx_gemm"))(
        bits, _EPI_GATE[form], variant, elements.data_ptr(), elements.stride(0), held.data_ptr(), held.stride(0), tiles.data_ptr(),
            tile_scales.data_ptr(), out[0].data_ptr(), padded * out_bits // 8, out[1].data_ptr(), padded // BLOCK, M, 16 * n_tiles, n_tiles, k_tiles, pitch, 1,
            per_split, _stream(device))
    if status:
        _failed("arle_mx_gemm", status)
    return out
