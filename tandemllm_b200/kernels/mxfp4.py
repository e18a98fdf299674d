"""Matrices in microscaled 4-bit numbers (MXFP4) and the bfloat16 products with them (`csrc/mxfp4*.cu`).

  quantize(w)     -> `Mxfp4Matrix`: blocks of 32 values of a row share a power of two, each value is one of 0 1/2 1 3/2 2 3 4 6 times it
                     with a sign (4.25 bits a value); `.values(dtype)` gives the values back
  linear(...)     x W^T (+ bias): what `parts.linear.linear` calls for such a matrix
  gated(...)      act(x G^T) * (x U^T), gate and up matrices side by side
  experts(...)    a layer of routed experts, from the rows' chosen experts and weights to their sum

Rows are bfloat16 and every sum is 32-bit: the weights are exact in bfloat16, so a product is what the bfloat16 path would give for the
rounded weights. The compute happens on the device of the rows, which has to be the current one, on its current stream; nothing is kept
between calls but what the caller passes in. There is no 32-bit product: a 32-bit runtime takes the values as a plain matrix.
"""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from . import ops
from .build import Launchers, load

BLOCK = 32                      # values a scale
TILE_ROWS, TILE_K = 8, 128      # the layout's tiles
FEW_ROWS = 32                   # rows up to which a product goes to the register-only kernel
EXPERT_ROWS, EXPERT_PAIRS, EXPERT_TOP = 8, 256, 32      # the experts' two-kernel form
BYTES_A_VALUE = 17 / 32

_SIGNATURES = {
    "tl_mxfp4_quantize": [c_void_p, c_longlong, c_longlong, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p],
    "tl_mxfp4_values": [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p],
    "tl_mxfp4_few": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_float, c_float,
                     c_int, c_void_p],
    "tl_mxfp4_experts_first": [c_void_p, c_longlong, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int,
                               c_int, c_int, c_int, c_float, c_float, c_void_p, c_void_p],
    "tl_mxfp4_experts_second": [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_void_p, c_int, c_int, c_int,
                                c_void_p, c_void_p],
    "tl_mxfp4_tc": [c_void_p, c_longlong, c_longlong, c_void_p, c_void_p, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_float,
                    c_float, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p],
    "tl_mxfp4_plan": [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p],
    "tl_mxfp4_gather": [c_void_p, c_longlong, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p],
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
        _lib = Launchers(l, _SIGNATURES)
    return _lib


def _check(code: int, what: str, kernels: int = 1) -> None:
    if code == 0:
        ops.launches += kernels
        return
    if code == ops.TL_BAD_ARGUMENT:
        raise ops.KernelError(lib().tl_mx_last_error().decode())
    raise ops.KernelError(f"{what}: CUDA error {code}: {ops.core().tl_cuda_error_string(code).decode()}")


def _here(device: torch.device, what: str) -> None:
    if device.type != "cuda":
        raise ops.KernelError(f"{what} is on {device}; the kernels run on CUDA tensors only")
    if device.index != torch.cuda.current_device():
        raise ops.KernelError(f"{what} is on {device}, the current device is cuda:{torch.cuda.current_device()}")


class Mxfp4Matrix:
    """`groups` matrices [n, k] in 4-bit blocks: codes uint8 [groups, n / 8, k / 128, 512] and scales uint8 [groups, n / 8, k / 128, 32]
    in the kernels' layout (csrc/mxfp4.cuh), both sizes rounded up. `shape` is the shape of the tensor it was made of."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape: tuple[int, ...]):
        self.codes, self.scales, self.shape = codes, scales, tuple(int(d) for d in shape)
        self.groups, self.n, self.k = (1 if len(shape) == 2 else self.shape[0]), self.shape[-2], self.shape[-1]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def numel(self) -> int:
        return self.groups * self.n * self.k

    def values(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as a plain tensor of `shape`, exact in either dtype."""
        _here(self.device, "the matrix")
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        _check(lib().tl_mxfp4_values(self.codes.data_ptr(), self.scales.data_ptr(), out.data_ptr(), ops.dtype_code(dtype), self.groups, self.n,
                                     self.k, ops.stream()), "mxfp4_values", kernels=int(out.numel() > 0))
        return out


def quantize(w: torch.Tensor) -> Mxfp4Matrix:
    """The matrix w [n, k], or the matrices [groups, n, k], 32-bit or bfloat16, rounded to MXFP4: a block of 32 values along k has the
    scale 2^s with s = floor(log2(largest)) - 2 (at least -127), each value becomes the nearest (ties to even) multiple it has a code for, and
    what lies beyond 6 * 2^s becomes that. A block with an infinity or a NaN is not a number as a whole."""
    if w.dim() not in (2, 3):
        raise ops.KernelError(f"mxfp4: a tensor of shape {tuple(w.shape)}; [n, k] or [groups, n, k] is wanted")
    code = ops.dtype_code(w.dtype)
    _here(w.device, "the matrix")
    if w.stride(-1) != 1 and w.shape[-1] > 1:
        w = w.contiguous()
    groups, (n, k) = (1 if w.dim() == 2 else w.shape[0]), w.shape[-2:]
    tiles = (groups, -(-n // TILE_ROWS), -(-k // TILE_K))
    codes = torch.empty(*tiles, TILE_ROWS * TILE_K // 2, dtype=torch.uint8, device=w.device)
    scales = torch.empty(*tiles, TILE_ROWS * TILE_K // BLOCK, dtype=torch.uint8, device=w.device)
    _check(lib().tl_mxfp4_quantize(w.data_ptr(), w.stride(-2), w.stride(0) if w.dim() == 3 else 0, code, codes.data_ptr(), scales.data_ptr(),
                                   groups, n, k, ops.stream()), "mxfp4_quantize", kernels=int(w.numel() > 0))
    return Mxfp4Matrix(codes, scales, tuple(w.shape))


def _rows(x: torch.Tensor, w: Mxfp4Matrix) -> torch.Tensor:
    """x as the kernels read it: rows of bfloat16 numbers that begin at multiples of 16 bytes, a multiple of 8 of them."""
    if x.dim() != 2 or x.shape[1] != w.k:
        raise ops.KernelError(f"mxfp4 product: rows of shape {tuple(x.shape)} with a matrix of shape {w.shape}")
    if x.dtype != torch.bfloat16:
        raise ops.KernelError(f"mxfp4 product: rows of {x.dtype}; bfloat16 is implemented")
    _here(x.device, "x")
    if w.device != x.device:
        raise ops.KernelError(f"mxfp4 product: rows on {x.device}, the matrix on {w.device}")
    if w.k % 8 or x.stride(-1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16:
        x = torch.nn.functional.pad(x, (0, -w.k % 8)).contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _vector(v: torch.Tensor | None, size: int, name: str, device) -> None:
    if v is None:
        return
    if v.dtype != torch.float32 or not v.is_contiguous() or v.numel() != size or v.device != device:
        raise ops.KernelError(f"mxfp4 product: {name} is {v.dtype} {tuple(v.shape)} on {v.device}; {size} contiguous float32 numbers on {device}")


def _output(out, rows: int, n: int, dtype: torch.dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(rows, n, dtype=dtype, device=device)
    if tuple(out.shape) != (rows, n) or out.dtype != dtype or out.device != device or out.stride(-1) != 1:
        raise ops.KernelError(f"mxfp4 product: an output of {out.dtype} {tuple(out.shape)} on {out.device}; {dtype} ({rows}, {n}) with unit inner "
                              f"stride on {device}")
    return out


def token_tile(rows: float) -> int:
    """Token rows of a tile of the tensor-core product for `rows` rows side by side."""
    return 16 if rows <= 16 else 32 if rows <= 32 else 64 if rows <= 64 else 128


def splits_of(ctas: int, k: int, sms: int) -> int:
    """CTAs that share a tile's k where `ctas` alone leave SMs idle (two CTAs an SM, each with at least two tiles of 128)."""
    return max(1, min(2 * sms // ctas, -(-k // TILE_K) // 2, 8))


def _product(runtime, x, w: Mxfp4Matrix, bias, out, act: int, constants) -> None:
    """out = the product of x's rows with w: act 0 plain, a gate's code gated, negated an activation on a plain product."""
    M = x.shape[0]
    if M == 0:
        return
    if M <= FEW_ROWS:
        _check(lib().tl_mxfp4_few(x.data_ptr(), x.stride(0), w.codes.data_ptr(), w.scales.data_ptr(), ops.ptr(bias), out.data_ptr(), out.stride(0),
                                  M, w.n, x.shape[1], act, *constants, ops.dtype_code(out.dtype), ops.stream()), "mxfp4_few")
        return
    bn = token_tile(M)
    ctas = -(-w.n // (64 if act > 0 else 128)) * -(-M // bn)
    _check(lib().tl_mxfp4_tc(x.data_ptr(), x.stride(0), M, w.codes.data_ptr(), w.scales.data_ptr(), ops.ptr(bias), out.data_ptr(), out.stride(0),
                             M, w.n, x.shape[1], act, *constants, ops.dtype_code(out.dtype), bn, splits_of(ctas, x.shape[1], ops.sm_count()),
                             None, None, None, None, 0, None, None, runtime.status.data_ptr(), ops.stream()), "mxfp4_tc")


def linear(runtime, x: torch.Tensor, w: Mxfp4Matrix, bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """x [rows, k] times the one matrix w [n, k], plus `bias` (32-bit, [n]), in `out_dtype` (default: x's)."""
    if w.groups != 1:
        raise ops.KernelError(f"mxfp4 product: a stack of {w.groups} matrices where one is wanted")
    x = _rows(x, w)
    _vector(bias, w.n, "the bias", x.device)
    out = _output(out, x.shape[0], w.n, out_dtype or (out.dtype if out is not None else x.dtype), x.device)
    _product(runtime, x, w, bias, out, 0, (0.0, 0.0))
    return out


def gated(runtime, x: torch.Tensor, w: Mxfp4Matrix, act: str | int = "silu", bias: torch.Tensor | None = None,
          constants: tuple[float, float] = (0.0, 0.0)) -> torch.Tensor:
    """act(x w[0]^T + b_gate) * (x w[1]^T + b_up) in bfloat16 for w of shape [2, n, k] (gate, up) and `bias` = [b_gate; b_up] (32-bit,
    [2 n]). `act`: a gate of `ops.ACTIVATIONS`, by name or code; `constants`: those of one that has some."""
    if w.groups != 2:
        raise ops.KernelError(f"mxfp4 gated product: {w.groups} matrices where a gate and an up matrix are wanted")
    x = _rows(x, w)
    _vector(bias, 2 * w.n, "the bias", x.device)
    code = ops.activation_code(act) if isinstance(act, str) else int(act)
    out = torch.empty(x.shape[0], w.n, dtype=torch.bfloat16, device=x.device)
    if code <= 0:
        raise ops.KernelError(f"mxfp4 gated product: activation {act!r} is no gate")
    _product(runtime, x, w, bias, out, code, constants)
    return out


def experts(runtime, x: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor, w_first: Mxfp4Matrix, w_down: Mxfp4Matrix, act: str | int = "silu",
            weigh: str = "output", out_dtype: torch.dtype | None = None, constants: tuple[float, float] = (0.0, 0.0)) -> torch.Tensor:
    """out[r] = sum over the experts e = ids[r, :] (int32) of wts[r, :] (32-bit) times expert e of x[r], in `out_dtype` (default: x's).

    `w_down` [E, hidden, inter]; `w_first` [2 E, inter, hidden], the gate and the up matrix of every expert in turn: an expert is
    down( act(gate x) * (up x) ); or [E, inter, hidden] without gates: down( act(up x) ). `weigh` "input": the weight multiplies what the
    first product makes of x, in front of the activation, and the experts' rows are added as they are. An id outside 0 .. E - 1 adds
    nothing and is recorded in the runtime's status word."""
    E, gates = w_down.groups, w_first.groups // max(w_down.groups, 1)
    if gates not in (1, 2) or w_first.groups != gates * E or (w_first.n, w_first.k) != (w_down.k, w_down.n):
        raise ops.KernelError(f"mxfp4 experts: matrices of shapes {w_first.shape} and {w_down.shape}")
    if weigh not in ("input", "output"):
        raise ops.KernelError(f"experts weighed at their {weigh!r}: input or output")
    code = ops.activation_code(act) if isinstance(act, str) else int(act)
    x = _rows(x, w_first)
    rows, top = ids.shape
    ops._need(ids, torch.int32, "expert ids"); ops._need(wts, torch.float32, "expert weights")
    if tuple(wts.shape) != (rows, top) or rows != x.shape[0] or ids.device != x.device or wts.device != x.device:
        raise ops.KernelError(f"mxfp4 experts: {tuple(x.shape)} rows with ids {tuple(ids.shape)} and weights {tuple(wts.shape)}")
    if not 1 <= top <= EXPERT_TOP or not 1 <= E <= 1024:
        raise ops.KernelError(f"mxfp4 experts: top-{top} of {E}; up to top-{EXPERT_TOP} of 1024 are implemented")
    out = torch.empty(rows, w_down.n, dtype=out_dtype or x.dtype, device=x.device)
    if rows == 0:
        return out
    form = _two_kernels if rows <= EXPERT_ROWS and rows * top <= EXPERT_PAIRS else _sorted
    form(runtime, x, ids, wts, w_first, w_down, code if gates == 2 else -code, weigh == "input", constants, out)
    return out


def _two_kernels(runtime, x, ids, wts, w_first, w_down, act: int, before: bool, constants, out) -> None:
    rows, top = ids.shape
    E, inter = w_down.groups, w_down.k
    ld = -(-inter // 8) * 8
    a = torch.empty(rows * top, ld, dtype=torch.bfloat16, device=x.device)
    _check(lib().tl_mxfp4_experts_first(x.data_ptr(), x.stride(0), w_first.codes.data_ptr(), w_first.scales.data_ptr(), a.data_ptr(), ld, rows,
                                        inter, x.shape[1], ids.data_ptr(), wts.data_ptr(), int(before), top, E, act, *constants,
                                        runtime.status.data_ptr(), ops.stream()), "mxfp4_experts_first")
    _check(lib().tl_mxfp4_experts_second(a.data_ptr(), ld, w_down.codes.data_ptr(), w_down.scales.data_ptr(), out.data_ptr(), out.stride(0), rows,
                                         w_down.n, inter, ids.data_ptr(), top, E, ops.dtype_code(out.dtype), runtime.status.data_ptr(),
                                         ops.stream()), "mxfp4_experts_second")


def _sorted(runtime, x, ids, wts, w_first, w_down, act: int, before: bool, constants, out) -> None:
    """The experts' token rows side by side, a tensor-core product over tiles of them for each half, and the rows' weighed sums."""
    rows, top = ids.shape
    E, inter, hidden, pairs, k = w_down.groups, w_down.k, w_down.n, rows * top, x.shape[1]
    tile = token_tile(1.4 * pairs / E)
    tiles = min(pairs // tile + E, pairs)
    ints = torch.empty(E + 2 * pairs + 3 * tiles + 1, dtype=torch.int32, device=x.device)
    counts = ints.data_ptr()
    order = counts + 4 * E
    place = order + 4 * pairs
    group, row0, n_rows = (place + 4 * (pairs + i * tiles) for i in range(3))
    n_tiles = n_rows + 4 * tiles
    _check(lib().tl_mxfp4_plan(ids.data_ptr(), pairs, E, tile, counts, order, place, group, row0, n_rows, n_tiles, runtime.status.data_ptr(),
                               ops.stream()), "mxfp4_plan")
    xs = torch.empty(pairs, k, dtype=torch.bfloat16, device=x.device)
    _check(lib().tl_mxfp4_gather(x.data_ptr(), x.stride(0), order, top, xs.data_ptr(), pairs, k, ops.stream()), "mxfp4_gather")
    ld = -(-inter // 8) * 8
    a = torch.empty(pairs, ld, dtype=torch.bfloat16, device=x.device)
    y = torch.empty(pairs, hidden, dtype=torch.float32, device=x.device)
    tail = (tile, 1, group, row0, n_rows, n_tiles, tiles)
    _check(lib().tl_mxfp4_tc(xs.data_ptr(), k, pairs, w_first.codes.data_ptr(), w_first.scales.data_ptr(), None, a.data_ptr(), ld, pairs, inter, k,
                             act, *constants, ops.BF16, *tail, wts.data_ptr() if before else None, order if before else None,
                             runtime.status.data_ptr(), ops.stream()), "mxfp4_tc")
    _check(lib().tl_mxfp4_tc(a.data_ptr(), ld, pairs, w_down.codes.data_ptr(), w_down.scales.data_ptr(), None, y.data_ptr(), hidden, pairs, hidden,
                             inter, 0, 0.0, 0.0, ops.FP32, *tail, None, None, runtime.status.data_ptr(), ops.stream()), "mxfp4_tc")
    _check(lib().tl_mxfp4_sum(y.data_ptr(), place, ids.data_ptr(), None if before else wts.data_ptr(), out.data_ptr(), ops.dtype_code(out.dtype),
                              rows, hidden, top, E, ops.stream()), "mxfp4_sum")
