"""Python face of the 8-bit linear layers' kernels (quantize_fp8.cu, gemm_fp8.cu): torch tensors in, launches on the current
stream of the tensors' device, which has to be the current one.

Values are held in ``torch.float8_e4m3fn`` with float32 scales: one for each 128 values of a row (the rows that go into a
product), or one for each block of 128 x 128 of a weight.  A value stands for ``q * scale``.  With amax the largest magnitude of
a block and a = max(amax, 448 * 2^-126), scale = a / 448 and q = round(x * (448 / a)), ties to even; a row's or a weight's last
blocks may be partial.  What is not a number makes its block's scale not a number, an infinite value makes it infinite.

Outputs are made when they are not given, in memory of the stream that the launch goes to, and returned; a call that gives none goes through one step of compiled code
(fp8_calls.cpp), any other through the checks here.  Given ones are contiguous, on the inputs' device, and overlap no input
(but ``add_rmsnorm`` adds into its residual where asked to).  The engine launches the same exported functions from its C++ parts.
"""
from __future__ import annotations

import ctypes
import functools
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional, Tuple

import torch

from . import ops
from .build import load_extension
from .ops import KernelError, call, register_signatures

register_signatures("fp8", {
    "ph_quantize_fp8": [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p],
    "ph_add_rmsnorm_fp8": [c_void_p, c_void_p, c_int, c_int, c_longlong, c_void_p, c_float, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p,
                           c_void_p, c_void_p],
    "ph_gated_fp8": [c_void_p, c_int, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p],
    "ph_fp8_take_error": [c_void_p],
    "ph_gemm_fp8": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_int, c_void_p,
                    c_void_p],
    "ph_gemm_fp8_gated": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p],
    "ph_gemm_fp8_plan": [c_int, c_int, c_int, c_int, c_void_p, c_void_p],
})

BLOCK = 128
E4M3, F32 = torch.float8_e4m3fn, torch.float32
MAX_NORM_WIDTH = 32768
_LIMIT = 2 ** 31 - 1                 # of every count: the launchers take 32-bit numbers, and ctypes cuts what is longer
ERRORS = {131: "the copies waited too long for a free stage", 132: "the products waited too long", 133: "the epilogue waited too long for an accumulator"}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


_raw_stream = torch._C._cuda_getCurrentRawStream       # a lookup of 0.1 us, where the stream as an object costs 3


def _stream(what: str, first: torch.Tensor, *others) -> int:
    """The current stream of the device that every tensor given is on, which has to be the current one."""
    if not first.is_cuda:
        raise KernelError(f"{what}: the tensors must be CUDA tensors; there is no host implementation")
    at = first.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise KernelError(f"{what}: the tensors are not all on one device")
    if at != torch.cuda.current_device():
        raise KernelError(f"{what}: the tensors are on device {at}, which is not the current one")
    scope = ops._scope.stream
    return scope if scope is not None else _raw_stream(at)


_calls = None


def _load_calls():
    """The extension that makes a plain call in one step (fp8_calls.cpp), with the launchers it needs.  Host tensors are refused by the
    faces' own checks, without compiling it."""
    global _calls
    calls = load_extension("fp8_calls")
    calls.set_launchers(*(ctypes.cast(ops._fn("fp8", f"ph_{n}")[0], c_void_p).value
                          for n in ("quantize_fp8", "add_rmsnorm_fp8", "gated_fp8", "gemm_fp8_plan", "gemm_fp8")))
    _calls = calls
    return calls


def _scope() -> int:
    scope = ops._scope.stream
    return -1 if scope is None else scope


def _made(got):
    """What a plain call gave: its outputs, or the status of a launcher that refused."""
    if got.__class__ is int:
        raise KernelError(ops._fn("fp8", "ph_quantize_fp8")[1]().decode("utf-8", "replace"))
    ops.launches += 1
    return got


def _check(what: str, name: str, t: torch.Tensor, shape: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
    """The output `name` that the caller has given."""
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise KernelError(f"{what}: {name} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t


def _empty(size, strides, dtype, device) -> torch.Tensor:
    """A new tensor of the stream that the launch goes to (empty_strided takes 1.5 us, new_empty 2.0 and empty 2.3)."""
    return ops.of_launch_stream(torch.empty_strided, size, strides, dtype=dtype, device=device)


def _matrix(what: str, name: str, t: torch.Tensor) -> Tuple[int, int]:
    shape = t.shape
    if len(shape) != 2 or not 0 < shape[1] <= _LIMIT or shape[0] > _LIMIT:
        raise KernelError(f"{what}: {name} must be a matrix with at least one column, got shape {tuple(shape)}")
    return shape


def quantize(x: torch.Tensor, out: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *,
             block_rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [T, K] (float32 or bfloat16, its rows ``x.stride(0)`` apart) in 8 bits: out [T, K] and scales [ceil(T / block_rows),
    ceil(K / 128)].  ``block_rows``: 1 for the rows of a product, 128 for a weight."""
    if out is None and scales is None:
        calls = _calls or (x.is_cuda and _load_calls())
        got = calls.quantize(x, block_rows, _scope()) if calls else None
        if got is not None:
            return _made(got)
    T, K = _matrix("quantize", "x", x)
    if block_rows not in (1, BLOCK):
        raise KernelError(f"quantize: block_rows is 1 or {BLOCK}, not {block_rows}")
    apart, step = x.stride()
    if (step != 1 and K > 1) or (T > 1 and apart < K):
        raise KernelError(f"quantize: the rows of x must be contiguous and apart, got strides {x.stride()}")
    code = ops._code(x.dtype)
    stream = _stream("quantize", x, out, scales)
    blocks = (T if block_rows == 1 else _blocks(T), _blocks(K))
    out = _empty((T, K), (K, 1), dtype=E4M3, device=x.device) if out is None else _check("quantize", "out", out, (T, K), E4M3)
    scales = _empty(blocks, (blocks[1], 1), dtype=F32, device=x.device) if scales is None else _check("quantize", "scales", scales, blocks, F32)
    call("fp8", "ph_quantize_fp8", x.data_ptr(), code, apart if T > 1 else K, out.data_ptr(), scales.data_ptr(), T, K, block_rows, stream)
    return out, scales


def add_rmsnorm(x: torch.Tensor, add: Optional[torch.Tensor], weight: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None,
                scales: Optional[torch.Tensor] = None, *, rows: Optional[torch.Tensor] = None, add_splits: int = 1, write_x: bool = True,
                x_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """v = x[t] + sum_s add[s][t]; out, scales = v * rsqrt(mean(v^2) + eps) * weight in 8 bits, out [T, E], scales [T, ceil(E / 128)].

    ``x`` [T, E] is the float32 residual, ``add`` [T, E] or, with ``add_splits`` > 1, [splits, T, E] (float32 or bfloat16, or
    None), ``weight`` float32 [E].  v is kept in ``x_out`` [T, E] where that is given, else in x itself (unless ``write_x`` is
    false or there is nothing to add).  ``rows`` (int32 [n]) picks the rows that are normed, in that order (out [n, E]); nothing is
    kept then, and a number outside 0 .. T - 1 leaves its row of out and scales as it was."""
    if out is None and scales is None and rows is None:
        calls = _calls or (x.is_cuda and _load_calls())
        got = calls.add_rmsnorm(x, add, weight, eps, add_splits, write_x, x_out, _scope()) if calls else None
        if got is not None:
            return _made(got)
    T, E = _matrix("add_rmsnorm", "x", x)
    if E > MAX_NORM_WIDTH:
        raise KernelError(f"add_rmsnorm: rows of at most {MAX_NORM_WIDTH} values, not {E}")
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise KernelError("add_rmsnorm: x must be contiguous float32")
    if weight.dtype != torch.float32 or weight.shape != (E,) or not weight.is_contiguous():
        raise KernelError(f"add_rmsnorm: weight must be contiguous float32 [{E}]")
    if add is not None and (not 1 <= add_splits <= _LIMIT or add.shape != ((T, E) if add_splits == 1 and add.dim() == 2 else (add_splits, T, E)) or not add.is_contiguous()):
        raise KernelError(f"add_rmsnorm: add must be contiguous {add_splits} x [{T}, {E}], got {tuple(add.shape)}")
    if not eps >= 0.0:
        raise KernelError(f"add_rmsnorm: eps must not be negative, got {eps}")
    n = T
    if rows is not None:
        if rows.dtype != torch.int32 or rows.dim() != 1 or rows.shape[0] > _LIMIT or not rows.is_contiguous() or x_out is not None:
            raise KernelError(f"add_rmsnorm: rows must be a contiguous int32 vector of at most {_LIMIT}, and x_out does not go with it")
        n = rows.shape[0]
    if n and not T:
        raise KernelError("add_rmsnorm: there are no rows to pick from")
    code = ops.F32 if add is None else ops._code(add.dtype)
    stream = _stream("add_rmsnorm", x, add, weight, out, scales, rows, x_out)
    blocks = (n, _blocks(E))
    out = _empty((n, E), (E, 1), dtype=E4M3, device=x.device) if out is None else _check("add_rmsnorm", "out", out, (n, E), E4M3)
    scales = _empty(blocks, (blocks[1], 1), dtype=F32, device=x.device) if scales is None else _check("add_rmsnorm", "scales", scales, blocks, F32)
    keep = None
    if x_out is not None:
        keep = _check("add_rmsnorm", "x_out", x_out, (T, E), F32).data_ptr()
    elif write_x and add is not None and rows is None:
        keep = x.data_ptr()
    call("fp8", "ph_add_rmsnorm_fp8", x.data_ptr(), None if add is None else add.data_ptr(), code, add_splits, T * E, weight.data_ptr(), eps,
         None if rows is None else rows.data_ptr(), n, T, E, keep, out.data_ptr(), scales.data_ptr(), stream)
    return out, scales


def _gate(gate):
    """The kernel's four floats on the host: alpha, limit, shift and the gate's kind."""
    if gate is None:
        return None
    if isinstance(gate, str) and gate != "gelu_tanh":
        raise KernelError(f"gated: gate {gate!r} is not known")
    if isinstance(gate, str):
        return (c_float * 4)(0, 0, 0, 2)
    if len(gate) != 3:
        raise KernelError(f"gated: the clamped swish has alpha, limit and shift, got {tuple(gate)}")
    return (c_float * 4)(*gate, 1)


def gated(gate_up: torch.Tensor, out: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *, splits: int = 1,
          gate=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """out, scales = silu(g) * u in 8 bits for rows [g0, u0, g1, u1, ...]: gate_up [T, 2 F], or [splits, T, 2 F] partial sums
    with ``splits`` > 1 (float32 or bfloat16), to out [T, F], scales [T, ceil(F / 128)].  ``gate``: None (silu), (alpha, limit,
    shift) of the clamped swish, or "gelu_tanh"."""
    if out is None and scales is None and gate is None:
        calls = _calls or (gate_up.is_cuda and _load_calls())
        got = calls.gated(gate_up, splits, _scope()) if calls else None
        if got is not None:
            return _made(got)
    shape = gate_up.shape
    if len(shape) != (2 if splits == 1 else 3) or shape[-1] % 2 or not 0 < shape[-1] <= _LIMIT or shape[-2] > _LIMIT or not 1 <= splits <= _LIMIT or \
            (splits > 1 and shape[0] != splits) or not gate_up.is_contiguous():
        raise KernelError(f"gated: gate_up must be contiguous (gate, up) pairs in {splits} parts, got {tuple(shape)}")
    T, F = shape[-2], shape[-1] // 2
    code = ops._code(gate_up.dtype)
    stream = _stream("gated", gate_up, out, scales)
    blocks = (T, _blocks(F))
    out = _empty((T, F), (F, 1), dtype=E4M3, device=gate_up.device) if out is None else _check("gated", "out", out, (T, F), E4M3)
    scales = _empty(blocks, (blocks[1], 1), dtype=F32, device=gate_up.device) if scales is None else _check("gated", "scales", scales, blocks, F32)
    call("fp8", "ph_gated_fp8", gate_up.data_ptr(), code, splits, T * 2 * F, out.data_ptr(), scales.data_ptr(), T, F, _gate(gate), stream)
    return out, scales


def check_errors() -> None:
    """Raise if a product on the current device gave up on a wait since the last check (waits for the device)."""
    code = c_int()
    call("fp8", "ph_fp8_take_error", ctypes.addressof(code))
    if code.value:
        raise KernelError(f"gemm_fp8: {ERRORS.get(code.value, 'error')} (status {code.value})")


@functools.lru_cache(maxsize=4096)
def plan(M: int, N: int, K: int, device: int = 0, tile: int = 0, splits: int = 0, whole: bool = True) -> Tuple[int, int]:
    """How a product is cut on the current device (number ``device``) where ``tile`` or ``splits`` is 0: tokens of a tile, parts of
    K.  ``whole``: the whole sum is wanted, not the parts."""
    t, s = c_int(tile), c_int(splits)
    call("fp8", "ph_gemm_fp8_plan", M, N, K, int(whole), ctypes.addressof(t), ctypes.addressof(s))
    return t.value, s.value


def gemm(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: Optional[torch.Tensor] = None, *,
         out_dtype: torch.dtype = torch.bfloat16, tile: int = 0, splits: int = 0, early_w: bool = False) -> torch.Tensor:
    """out [M, N] = (x * x_scales) @ (w * w_scales)^T: x [M, K] with x_scales [M, ceil(K / 128)], w [N, K] with w_scales
    [ceil(N / 128), ceil(K / 128)], K a multiple of 16, sums in float32, out float32 or bfloat16 (``out_dtype`` where out is not
    given).  ``splits`` > 1: K is cut into that many parts and out is [splits, M, N] float32, the sums of each, for a consumer that
    adds them up (``add_rmsnorm``, ``gated``); 0: cut as the kernel likes it, and out is the whole sum.  ``tile`` (0: the kernel's own
    choice): 16, 32, 64 or 96 tokens beside 128 features, or 256 x 256 on pairs of CTAs.  ``early_w``: w is not the result of a
    kernel that may still run when the product starts (a model's weight), so its first tiles may be read before the kernel in
    front has ended."""
    if out is None and not tile and not splits and (out_dtype is torch.bfloat16 or out_dtype is F32):
        calls = _calls or (x.is_cuda and _load_calls())
        got = calls.gemm(x, x_scales, w, w_scales, out_dtype is torch.bfloat16, early_w, _scope()) if calls else None
        if got is not None:
            return _made(got)
    M, K = _matrix("gemm_fp8", "x", x)
    N, K2 = _matrix("gemm_fp8", "w", w)
    if x.dtype is not E4M3 or w.dtype is not E4M3 or not x.is_contiguous() or not w.is_contiguous():
        raise KernelError("gemm_fp8: x and w must be contiguous float8_e4m3fn tensors")
    if K != K2 or N < 1:
        raise KernelError(f"gemm_fp8: x {tuple(x.shape)} and w {tuple(w.shape)} do not fit")
    kb = _blocks(K)
    if x_scales.dtype is not F32 or x_scales.shape != (M, kb) or not x_scales.is_contiguous():
        raise KernelError(f"gemm_fp8: x_scales must be contiguous float32 [{M}, {kb}]")
    if w_scales.dtype is not F32 or w_scales.shape != (_blocks(N), kb) or not w_scales.is_contiguous():
        raise KernelError(f"gemm_fp8: w_scales must be contiguous float32 [{_blocks(N)}, {kb}]")
    stream = _stream("gemm_fp8", x, x_scales, w, w_scales, out)
    if tile < 0 or splits < 0:
        raise KernelError(f"gemm_fp8: tile {tile} and splits {splits} must not be negative")
    device = x.device
    parted = splits > 1
    if not tile or not splits:
        if M:
            tile, splits = plan(M, N, K, device.index, tile, splits)
    if parted:
        out = _empty((splits, M, N), (M * N, N, 1), dtype=F32, device=device) if out is None else _check("gemm_fp8", "out", out, (splits, M, N), F32)
        code, whole, parts = ops.F32, None, out.data_ptr()
    else:
        out = _empty((M, N), (N, 1), dtype=out_dtype, device=device) if out is None else _check("gemm_fp8", "out", out, (M, N), out.dtype)
        code, whole, parts = ops._code(out.dtype), out.data_ptr(), None
        if splits > 1:
            held = _empty((splits, M, N), (M * N, N, 1), dtype=F32, device=device)
            parts = held.data_ptr()
    if not M:
        return out
    call("fp8", "ph_gemm_fp8", x.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), whole, code, M, N, K, tile, splits, parts,
         early_w, None, stream)
    return out


def gemm_gated(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: Optional[torch.Tensor] = None,
               scales: Optional[torch.Tensor] = None, *, gate=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """What ``gated`` makes of ``gemm``'s float32 product, without the product going to memory: w [N, K] holds the rows of gate and up in
    turn (N a multiple of 256, K of 16), out [M, N / 2], scales [M, N / 256]; ``gate`` as in ``gated``.  For many tokens: it runs on
    pairs of CTAs with K whole, whatever M is.  Where ``plan`` gives anything but (256, 1), ``gemm`` and ``gated`` can be faster."""
    M, K = _matrix("gemm_gated", "x", x)
    N, K2 = _matrix("gemm_gated", "w", w)
    if x.dtype is not E4M3 or w.dtype is not E4M3 or not x.is_contiguous() or not w.is_contiguous():
        raise KernelError("gemm_gated: x and w must be contiguous float8_e4m3fn tensors")
    kb = _blocks(K)
    if K != K2 or N < 1 or N % 256:
        raise KernelError(f"gemm_gated: x {tuple(x.shape)} and w {tuple(w.shape)} do not fit, or w's rows are no multiple of 256")
    for name, t, rows in (("x_scales", x_scales, M), ("w_scales", w_scales, N // BLOCK)):
        if t.dtype is not F32 or t.shape != (rows, kb) or not t.is_contiguous():
            raise KernelError(f"gemm_gated: {name} must be contiguous float32 [{rows}, {kb}]")
    stream = _stream("gemm_gated", x, x_scales, w, w_scales, out, scales)
    out = _empty((M, N // 2), (N // 2, 1), dtype=E4M3, device=x.device) if out is None else _check("gemm_gated", "out", out, (M, N // 2), E4M3)
    blocks = (M, N // 256)
    scales = _empty(blocks, (blocks[1], 1), dtype=F32, device=x.device) if scales is None else _check("gemm_gated", "scales", scales, blocks, F32)
    call("fp8", "ph_gemm_fp8_gated", x.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), out.data_ptr(), scales.data_ptr(), M, N, K,
         _gate(gate), None, stream)
    return out, scales
