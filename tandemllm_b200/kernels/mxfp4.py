"""Matrices in microscaled 4-bit numbers (MXFP4) and the bfloat16 products with them (`csrc/mxfp4*.cu`).

  quantize(w)     -> `Mxfp4Matrix`: blocks of 32 values of a row share a power of two, each value is one of 0 1/2 1 3/2 2 3 4 6 times it
                     with a sign (4.25 bits a value); `.values(dtype)` gives the values back
  linear(...)     x W^T (+ bias): what `parts.linear.linear` calls for such a matrix
  gated(...)      act(x G^T) * (x U^T), gate and up matrices side by side
  experts(...)    a layer of routed experts, from the rows' chosen experts and weights to their sum

Rows are bfloat16 and every sum is 32-bit: the weights are exact in bfloat16, so a product is what the bfloat16 path would give for the
rounded weights. The compute happens on the device of the rows, which has to be the current one, on its current stream; nothing is kept
between calls but what the caller passes in. There is no 32-bit product: a 32-bit runtime takes the values as a plain matrix. Products of
up to 8 rows take a row relative to its largest number: what is below 2^-31 of it loses bits, what is below 2^-39 counts as zero, and weights
beyond 2^95 can make their sums infinite.
"""

from __future__ import annotations

import ctypes
import functools
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from . import ops
from .build import Launchers, load

BLOCK = 32                      # values a scale
BYTES_A_VALUE = 17 / 32         # half a byte, and a scale's share
TILE_ROWS, TILE_K = 8, 128      # the layout's tiles
# Rows up to which a product goes to the register-only kernel. Its and the tensor cores' us at 8 rows: 12000 outputs of 4096 15.3 and 16.9, 7168 gated
# ones of 2048 9.9 and 14.2, 2048 of 2048 5.2 and 6.0, but 2048 of 7168 10.9 and 9.4. A form of it for 16 rows, which is gone, took at 12 rows 21.4
# (17.3), 14.4 (14.1), 7.6 (6.4) and 9.6 (9.7), and was ahead only where there is little to do (1000 of 600 5.2 and 5.8).
FEW_ROWS = 8
# Rows up to which, and experts a row with which, a layer of experts goes to the two-kernel form. Its us and the sorted form's at 8 rows: top-4 of 32
# experts of 1792 x 2048 46 and 65, top-6 of 64 of 768 x 2048 42 and 47, top-2 of 8 of 4096 x 2048 41 and 53; at one row 17 and 26.
EXPERT_ROWS, EXPERT_TOP = 8, 32
# Pairs an expert, on average, up to which the sorted form's tiles are of 64 rows, else of 160. Us of 64 and of 160 at 4, 16, 32 and 48 pairs: top-4 of 32
# experts of 1792 x 2048 84 and 87, 87 and 88, 94 and 92, 99 and 94; top-6 of 64 of 768 x 2048 76 and 79, 80 and 81, 86 and 85, 97 and 90. With half of
# the rows at one expert the same to 3 us (up to 24 pairs; at 64 116 and 100).
LOW_PAIRS = 20
TILE_CODES, TILE_BYTES = TILE_ROWS * TILE_K // 2, TILE_ROWS * TILE_K * 17 // 32

ACTIVATIONS = tuple(ops.ACTIVATIONS[a] for a in ("silu", "gelu", "relu2", "identity"))     # those a plain product may end with

_SIGNATURES = {
    "tl_mxfp4_quantize": [c_void_p, c_longlong, c_longlong, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p],
    "tl_mxfp4_values": [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p],
    "tl_mxfp4_few_fits": [c_int, c_int, c_int, c_int],
    "tl_mxfp4_few": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_float, c_float,
                     c_int, c_void_p, c_void_p],
    "tl_mxfp4_experts_fit": [c_int, c_int, c_int, c_int],
    "tl_mxfp4_experts_first": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int,
                               c_int, c_float, c_float, c_void_p, c_void_p],
    "tl_mxfp4_experts_second": [c_void_p, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_void_p, c_int, c_int, c_int, c_int,
                                c_void_p, c_void_p],
    "tl_mxfp4_tc": [c_void_p, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_float,
                    c_float, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p],
    "tl_mxfp4_plan": [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p],
    "tl_mxfp4_gather": [c_void_p, c_longlong, c_void_p, c_int, c_void_p, c_longlong, c_int, c_int, c_void_p],
    "tl_mxfp4_sum": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p],
}
_lib = None


def lib():
    global _lib
    if _lib is None:
        l = load("mxfp4")
        for name, args in _SIGNATURES.items():
            fn = getattr(l, name)
            fn.argtypes = args
            fn.restype = c_int
        l.tl_mx_last_error.restype = ctypes.c_char_p
        l.tl_mxfp4_experts_between.argtypes, l.tl_mxfp4_experts_between.restype = [c_int, c_int], c_longlong
        _lib = Launchers(l, _SIGNATURES)
    return _lib


def _check(code: int, what: str, kernels: int = 1) -> None:
    if code == 0:
        ops.launches += kernels
        return
    if code == ops.TL_BAD_ARGUMENT:
        raise ops.KernelError(lib().tl_mx_last_error().decode())
    raise ops.KernelError(f"{what}: CUDA error {code}: {ops.core().tl_cuda_error_string(code).decode()}")


def _here(t: torch.Tensor, what: str) -> int:
    """The number of the current device, which `t` has to be on."""
    index = t.get_device()
    if index < 0:
        raise ops.KernelError(f"{what} is on {t.device}; the kernels run on CUDA tensors only")
    if index != torch._C._cuda_getDevice():
        raise ops.KernelError(f"{what} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return index


def data_bytes(shape: tuple[int, ...]) -> int:
    """Bytes of the matrix or matrices of this shape."""
    return (1 if len(shape) == 2 else shape[0]) * -(-shape[-2] // TILE_ROWS) * -(-shape[-1] // TILE_K) * TILE_BYTES


class Mxfp4Matrix:
    """`groups` matrices [n, k] in 4-bit blocks, in the kernels' layout (csrc/mxfp4.cuh): `data` (uint8, contiguous) holds the codes of all tiles
    of 8 rows by 128 k, both sizes rounded up, and behind them their scales. `shape` is the shape of the tensor it was made of. A copy, also a
    pickled one, has the bytes of its own `data`."""

    def __init__(self, data: torch.Tensor, shape: tuple[int, ...]):
        shape = tuple(int(s) for s in shape)
        if len(shape) not in (2, 3) or min(shape) < 0:
            raise ops.KernelError(f"mxfp4: a matrix of shape {shape}; [n, k] or [groups, n, k] is wanted")
        self.groups, self.n, self.k = (1 if len(shape) == 2 else shape[0]), shape[-2], shape[-1]
        size = data_bytes(shape)
        if data.dtype is not torch.uint8 or data.numel() != size or not data.is_contiguous() or data.data_ptr() % 16:
            raise ops.KernelError(f"mxfp4: {data.dtype} data of {data.numel()} bytes for a matrix of shape {shape}; {size} contiguous bytes (uint8) "
                                  "from a multiple of 16 on are wanted")
        self._data, self.shape, self.device, self.index = data, shape, data.device, data.get_device()
        self._codes_bytes = size // TILE_BYTES * TILE_CODES

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @property
    def codes(self) -> int:
        """The address of the codes."""
        return self._data.data_ptr()

    @property
    def scales(self) -> int:
        """The address of the scales."""
        return self._data.data_ptr() + self._codes_bytes

    def __reduce__(self):
        return Mxfp4Matrix, (self._data, self.shape)

    @property
    def nbytes(self) -> int:
        return self._data.numel()

    def numel(self) -> int:
        return self.groups * self.n * self.k

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as a plain tensor of `shape`, exact in either dtype."""
        code = ops.dtype_code(dtype)
        _here(self._data, "the matrix")
        out = self._data.new_empty(self.shape, dtype=dtype)
        _check(lib().tl_mxfp4_values(self.codes, self.scales, out.data_ptr(), code, self.groups, self.n, self.k, ops.stream()), "mxfp4_values",
               kernels=int(out.numel() > 0))
        return out


def quantize(w: torch.Tensor) -> Mxfp4Matrix:
    """The matrix w [n, k], or the matrices [groups, n, k], 32-bit or bfloat16, rounded to MXFP4: a block of 32 values along k has the
    scale 2^s with s = floor(log2(largest)) - 2 (at least -127), each value becomes the nearest (ties to even) multiple it has a code for, and
    what lies beyond 6 * 2^s becomes that. A block with an infinity or a NaN is not a number as a whole."""
    if w.dim() not in (2, 3):
        raise ops.KernelError(f"mxfp4: a tensor of shape {tuple(w.shape)}; [n, k] or [groups, n, k] is wanted")
    code = ops.dtype_code(w.dtype)
    _here(w, "the matrix")
    shape, stride = w.shape, w.stride()
    if stride[-1] != 1 and shape[-1] > 1:
        w = w.contiguous()
        stride = w.stride()
    groups, n, k = (1, *shape) if len(shape) == 2 else shape
    data = w.new_empty(data_bytes(shape), dtype=torch.uint8)
    m = Mxfp4Matrix(data, shape)
    _check(lib().tl_mxfp4_quantize(w.data_ptr(), stride[-2], stride[0] if len(shape) == 3 else 0, code, m.codes, m.scales, groups, n, k,
                                   ops.stream()), "mxfp4_quantize", kernels=int(data.numel() > 0))
    return m


def _rows(runtime, x: torch.Tensor, w: Mxfp4Matrix) -> tuple[int, int]:
    """(rows, elements from one to the next) of x, which has to be what the products take; the runtime's status word is where x is."""
    if x.dim() != 2 or x.shape[1] != w.k:
        raise ops.KernelError(f"mxfp4 product: rows of shape {tuple(x.shape)} with a matrix of shape {w.shape}")
    if x.dtype is not torch.bfloat16:
        raise ops.KernelError(f"mxfp4 product: rows of {x.dtype}; bfloat16 is implemented")
    if _here(x, "x") != w.index:
        raise ops.KernelError(f"mxfp4 product: rows on {x.device}, the matrix on {w.device}")
    if runtime.status is None or runtime.status.get_device() != w.index:
        raise ops.KernelError(f"mxfp4 product: rows on {x.device}, the runtime on {runtime.device}")
    ld, inner = x.stride()
    if inner != 1 and w.k > 1:
        raise ops.KernelError(f"mxfp4 product: rows of {w.k} elements that lie {inner} apart; unit inner stride is implemented")
    return x.shape[0], ld


def _boxed(x: torch.Tensor, rows: int, k: int, ld: int, order: int | None = None, div: int = 1) -> tuple[torch.Tensor, int]:
    """(x, its row stride) for the tensor-core product: as it is where its rows lie behind one another from multiples of 16 bytes, else a copy
    that does. With
    `order` (`rows` row numbers on the device, to be divided by `div`) a copy of these rows."""
    if order is None and ld % 8 == 0 and ld >= k and x.data_ptr() % 16 == 0:
        return x, ld
    wide = -(-k // 8) * 8
    copy = x.new_empty(rows, wide)
    _check(lib().tl_mxfp4_gather(x.data_ptr(), ld, order, div, copy.data_ptr(), wide, rows, k, ops.stream()), "mxfp4_gather")
    return copy, wide


def _vector(v: torch.Tensor | None, size: int, name: str, index: int) -> int | None:
    if v is None:
        return None
    if v.dtype is not torch.float32 or v.numel() != size or v.get_device() != index or not v.is_contiguous():
        raise ops.KernelError(f"mxfp4 product: {name} is {v.dtype} {tuple(v.shape)} on {v.device}; {size} contiguous float32 numbers on "
                              f"cuda:{index} are wanted")
    return v.data_ptr()


def _output(out, rows: int, n: int, dtype: torch.dtype, x: torch.Tensor) -> torch.Tensor:
    if out is None:
        return x.new_empty(rows, n, dtype=dtype)
    if tuple(out.shape) != (rows, n) or out.dtype != dtype or out.device != x.device or (out.stride(1) != 1 and n > 1) or \
            (out.stride(0) < n and rows > 1):
        raise ops.KernelError(f"mxfp4 product: an output of {out.dtype} {tuple(out.shape)}, strides {out.stride()}, on {out.device}; {dtype} ({rows}, "
                              f"{n}) with unit inner stride, a row behind the other, on {x.device} is wanted")
    return out


@functools.lru_cache(maxsize=4096)
def shape_of(rows: int, row_tiles: int, k: int, sms: int, gated: bool) -> tuple[int, int]:
    """(token rows a tile, CTAs that share a tile's k, or 0 for the persistent form) of the tensor-core product of `rows` rows with
    `row_tiles` tiles of 128 weight rows.

    The form with the smallest estimated time, in us: `blocks` (of 128 k) one after the other in every round of CTAs, each as long as its
    weights take to convert or, persistent, as its tokens take to multiply; a round's start and end; and, where CTAs share a tile's k, adding
    their sums. The numbers are fitted to 2800 timings of 8 products with 17 to 4096 rows (9 to 16 take what they give); over these the
    choice is 1.1 % slower than the fastest form on average. What decides, at 7168 gated outputs of 2048: 100 rows 14 us in one persistent
    tile, 18 where two CTAs share its k; 2048 rows 92 in tiles of 160, 106 in tiles of 192. At 2048 outputs of 7168: 256 rows 17 with
    eight CTAs a tile, 29 without; 700 rows 30 without, 35 with two."""
    blocks = -(-k // TILE_K)
    best = None
    for h in range(64, min(256, max(64, -(-rows // 16) * 16)) + 1, 16):
        rounds = -(-row_tiles * -(-rows // h) // sms)
        alone = 0.024 * h if h > 160 else 0.0                           # (one accumulator: a tile is stored before the next is multiplied)
        cost = 4.2 + rounds * (blocks * max(0.45, 0.0021 * h) + 0.96 + alone) + 0.0045 * h
        if best is None or cost < best[0]:
            best = cost, h, 0
    for bn in (16, 32, 64, 128):
        if 4 * bn < min(rows, 128) or bn >= max(32, 2 * rows):
            continue
        for splits in (1, 2, 4, 8):
            ctas = row_tiles * -(-rows // bn) * splits
            if splits > 1 and (splits > blocks or 4 * ctas > 7 * sms):      # (clusters do not fill every SM twice: 288 CTAs take two rounds)
                break
            rounds, rest = divmod(ctas, 2 * sms)                        # two CTAs an SM; one alone is faster
            rounds += 0.0 if rest == 0 else 0.585 if rest <= sms else 1.0
            cost = 4.4 + rounds * (-(-blocks // splits) * (0.66 + 0.0014 * bn) * (1.18 if gated else 1.0) + 0.34 + 0.009 * bn) + 0.008 * bn
            cost += 1.0 + 0.0265 * bn if splits > 1 else 0.0
            if cost < best[0]:
                best = cost, bn, splits
    return best[1:]


def _product(runtime, x, rows: int, ld: int, w: Mxfp4Matrix, bias: int | None, out: torch.Tensor, act: int, constants) -> None:
    """out = the product of x's rows with w: act 0 plain, a gate's code gated, negated an activation on a plain product."""
    if rows == 0:
        return
    code = ops.dtype_code(out.dtype)
    if rows <= FEW_ROWS and lib().tl_mxfp4_few_fits(rows, w.n, w.k, act):
        _check(lib().tl_mxfp4_few(x.data_ptr(), ld, w.codes, w.scales, bias, out.data_ptr(), out.stride(0), rows, w.n, w.k, act, *constants, code,
                                  runtime.status.data_ptr(), ops.stream()), "mxfp4_few")
        return
    x, ld = _boxed(x, rows, w.k, ld)
    bn, splits = shape_of(rows, -(-w.n // (64 if act > 0 else 128)), w.k, ops.sm_count(), act > 0)
    _check(lib().tl_mxfp4_tc(x.data_ptr(), ld, rows, w.codes, w.scales, bias, out.data_ptr(), out.stride(0), rows, w.n, w.k, act, *constants, code,
                             bn, splits, None, None, None, None, 0, None, None, runtime.status.data_ptr(), ops.stream()), "mxfp4_tc")


def linear(runtime, x: torch.Tensor, w: Mxfp4Matrix, bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           out: torch.Tensor | None = None, act: str | int | None = None) -> torch.Tensor:
    """x [rows, k] times the one matrix w [n, k], plus `bias` (32-bit, [n]), through the activation `act` (silu, gelu, relu2 or identity, by
    name or code; None: as it is), in `out_dtype` (default: `out`'s, else x's). `out`, where it is given, shares no memory with the inputs."""
    if w.groups != 1:
        raise ops.KernelError(f"mxfp4 product: a stack of {w.groups} matrices where one is wanted")
    rows, ld = _rows(runtime, x, w)
    b = _vector(bias, w.n, "the bias", w.index)
    out = _output(out, rows, w.n, out_dtype or (out.dtype if out is not None else x.dtype), x)
    code = 0 if act is None else _gate(act)
    if code and code not in ACTIVATIONS:
        raise ops.KernelError(f"mxfp4 product: activation {act!r} behind a plain product; silu, gelu, relu2 and identity are implemented")
    _product(runtime, x, rows, ld, w, b, out, -code, (0.0, 0.0))
    return out


def _gate(act: str | int) -> int:
    code = ops.activation_code(act) if isinstance(act, str) else int(act)
    if code <= 0:
        raise ops.KernelError(f"mxfp4 product: activation {act!r} is none of {', '.join(ops.ACTIVATIONS)}")
    return code


def gated(runtime, x: torch.Tensor, w: Mxfp4Matrix, act: str | int = "silu", bias: torch.Tensor | None = None,
          constants: tuple[float, float] = (0.0, 0.0)) -> torch.Tensor:
    """act(x w[0]^T + b_gate) * (x w[1]^T + b_up) in bfloat16 for w of shape [2, n, k] (gate, up) and `bias` = [b_gate; b_up] (32-bit,
    [2 n]). `act`: a gate of `ops.ACTIVATIONS`, by name or code; `constants`: those of one that has some."""
    if w.groups != 2:
        raise ops.KernelError(f"mxfp4 gated product: {w.groups} matrices where a gate and an up matrix are wanted")
    rows, ld = _rows(runtime, x, w)
    b = _vector(bias, 2 * w.n, "the bias", w.index)
    out = x.new_empty(rows, w.n)
    _product(runtime, x, rows, ld, w, b, out, _gate(act), constants)
    return out


def experts(runtime, x: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor, w_first: Mxfp4Matrix, w_down: Mxfp4Matrix, act: str | int = "silu",
            weigh: str = "output", out_dtype: torch.dtype | None = None, constants: tuple[float, float] = (0.0, 0.0), defer: bool = False):
    """out[r] = sum over the experts e = ids[r, :] (int32) of wts[r, :] (32-bit) times expert e of x[r], in `out_dtype` (default: x's).

    `w_down` [E, hidden, inter]; `w_first` [2 E, inter, hidden], the gate and the up matrix of every expert in turn: an expert is
    down( act(gate x) * (up x) ); or [E, inter, hidden] without gates: down( act(up x) ). `weigh` "input": the weight multiplies what the
    first product makes of x, in front of the activation, and the experts' rows are added as they are. An id outside 0 .. E - 1 adds
    nothing and is recorded in the runtime's status word. With `defer` the result of many rows is an `ops.ExpertRows`, whose consumer
    weighs and adds the experts' rows itself; every id has to be an expert's then."""
    E = w_down.groups
    gates = w_first.groups // max(E, 1)
    if gates not in (1, 2) or w_first.groups != gates * E or w_first.n != w_down.k or w_first.k != w_down.n or w_first.index != w_down.index:
        raise ops.KernelError(f"mxfp4 experts: matrices of shapes {w_first.shape} on {w_first.device} and {w_down.shape} on {w_down.device}")
    if weigh not in ("input", "output"):
        raise ops.KernelError(f"experts weighed at their {weigh!r}: input or output")
    rows, ld = _rows(runtime, x, w_first)
    if ids.dtype is not torch.int32 or ids.dim() != 2 or ids.shape[0] != rows or ids.get_device() != w_down.index or not ids.is_contiguous():
        raise ops.KernelError(f"mxfp4 experts: ids {ids.dtype} {tuple(ids.shape)} on {ids.device}; contiguous int32 [{rows}, top] on {x.device} is "
                              "wanted")
    top = ids.shape[1]
    w = _vector(wts, rows * top, "the experts' weights", w_down.index)
    if not 1 <= top <= EXPERT_TOP or not 1 <= E <= 1024:
        raise ops.KernelError(f"mxfp4 experts: top-{top} of {E}; up to top-{EXPERT_TOP} of 1024 are implemented")
    code = _gate(act)
    if gates == 1 and code not in ACTIVATIONS:
        raise ops.KernelError(f"mxfp4 experts: activation {act!r} without a gate; silu, gelu, relu2 and identity are implemented")
    if rows == 0:
        return x.new_empty(0, w_down.n, dtype=out_dtype)
    form = _two_kernels if rows <= EXPERT_ROWS and lib().tl_mxfp4_experts_fit(rows, top, w_first.k, w_down.k) else _sorted
    return form(runtime, x, rows, ld, ids, top, w, wts, w_first, w_down, code if gates == 2 else -code, weigh == "input", constants,
                out_dtype or x.dtype, defer)


def _two_kernels(runtime, x, rows: int, ld: int, ids, top: int, w: int, wts, w_first, w_down, act: int, before: bool, constants, dtype, defer):
    out = x.new_empty(rows, w_down.n, dtype=dtype)
    E, inter, status, stream = w_down.groups, w_down.k, runtime.status.data_ptr(), ops.stream()
    between = x.new_empty(lib().tl_mxfp4_experts_between(rows * top, inter), dtype=torch.uint8)
    _check(lib().tl_mxfp4_experts_first(x.data_ptr(), ld, w_first.codes, w_first.scales, between.data_ptr(), rows, inter, w_first.k,
                                        ids.data_ptr(), w, int(before), top, E, act, *constants, status, stream), "mxfp4_experts_first")
    _check(lib().tl_mxfp4_experts_second(between.data_ptr(), w_down.codes, w_down.scales, out.data_ptr(), w_down.n, rows, w_down.n, inter,
                                         ids.data_ptr(), top, E, act, ops.dtype_code(dtype), status, stream), "mxfp4_experts_second")
    return out


def _sorted(runtime, x, rows: int, ld: int, ids, top: int, w: int, wts, w_first, w_down, act: int, before: bool, constants, dtype, defer):
    """The experts' token rows side by side, a tensor-core product over tiles of them for each half, and the rows' weighed sums. Between the halves
    a row is bfloat16, as the second product's rows have to be; what the second half makes is 32-bit until it is added."""
    E, inter, hidden, pairs, status, stream = w_down.groups, w_down.k, w_down.n, rows * top, runtime.status.data_ptr(), ops.stream()
    tile = 64 if pairs <= LOW_PAIRS * E else 160
    tiles = min(pairs // tile + E, pairs)
    ints = x.new_empty(2 * pairs + 3 * tiles + 1, dtype=torch.int32)
    order = ints.data_ptr()
    place = order + 4 * pairs
    group, row0, n_rows = (place + 4 * (pairs + i * tiles) for i in range(3))
    n_tiles = n_rows + 4 * tiles
    _check(lib().tl_mxfp4_plan(ids.data_ptr(), pairs, E, tile, order, place, group, row0, n_rows, n_tiles, status, stream), "mxfp4_plan")
    xs, ld = _boxed(x, pairs, w_first.k, ld, order, top)
    wide = -(-inter // 8) * 8
    a = x.new_empty(pairs, wide)
    y = x.new_empty(pairs, hidden, dtype=torch.float32)
    tail = (tile, 0, group, row0, n_rows, n_tiles, tiles)
    _check(lib().tl_mxfp4_tc(xs.data_ptr(), ld, pairs, w_first.codes, w_first.scales, None, a.data_ptr(), wide, pairs, inter, w_first.k, act,
                             *constants, ops.BF16, *tail, w if before else None, order if before else None, status, stream), "mxfp4_tc")
    _check(lib().tl_mxfp4_tc(a.data_ptr(), wide, pairs, w_down.codes, w_down.scales, None, y.data_ptr(), hidden, pairs, hidden, inter, 0, 0.0, 0.0,
                             ops.FP32, *tail, None, None, status, stream), "mxfp4_tc")
    if defer:
        return ops.ExpertRows(y, ints[pairs:2 * pairs], ids, None if before else wts)
    out = x.new_empty(rows, hidden, dtype=dtype)
    _check(lib().tl_mxfp4_sum(y.data_ptr(), place, ids.data_ptr(), None if before else w, out.data_ptr(), ops.dtype_code(dtype), rows, hidden, top,
                              E, stream), "mxfp4_sum")
    return out
