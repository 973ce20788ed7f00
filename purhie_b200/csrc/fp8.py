"""Python face of the 8-bit linear layers' kernels (quantize_fp8.cu, gemm_fp8.cu): torch tensors in, launches on the current
stream of the tensors' device, which has to be the current one.

Values are held in ``torch.float8_e4m3fn`` with float32 scales: one for each 128 values of a row (the rows that go into a
product), or one for each block of 128 x 128 of a weight.  A value stands for ``q * scale``.  With amax the largest magnitude of
a block and a = max(amax, 448 * 2^-126), scale = a / 448 and q = round(x * (448 / a)), ties to even; a row's or a weight's last
blocks may be partial.  What is not a number makes its block's scale not a number, an infinite value makes it infinite.

Outputs are made when they are not given, and returned.  Given ones are contiguous, on the inputs' device, and overlap no input
(but ``add_rmsnorm`` adds into its residual where asked to).  The engine launches the same exported functions from its C++ parts.
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional, Tuple

import torch

from . import ops
from .gemm100 import _gate_pointer
from .ops import KernelError, call, register_signatures

register_signatures("fp8", {
    "ph_quantize_fp8": [c_void_p, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p],
    "ph_add_rmsnorm_fp8": [c_void_p, c_void_p, c_int, c_int, c_longlong, c_void_p, c_float, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p,
                           c_void_p, c_void_p],
    "ph_gated_fp8": [c_void_p, c_int, c_int, c_longlong, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p],
    "ph_gemm_fp8": [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p],
})

BLOCK = 128
E4M3 = torch.float8_e4m3fn
MAX_NORM_WIDTH = 32768
_LIMIT = 2 ** 31 - 1
_flags = {}
ERRORS = {131: "the copies waited too long for a free stage", 132: "the products waited too long", 133: "the epilogue waited too long for an accumulator"}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _on_device(what: str, first: torch.Tensor, **others) -> int:
    """The index of the device that every tensor given is on, which has to be the current one."""
    if not first.is_cuda:
        raise KernelError(f"{what}: the tensors must be CUDA tensors; there is no host implementation")
    at = first.get_device()
    for name, t in others.items():
        if t is not None and t.get_device() != at:
            raise KernelError(f"{what}: {name} is not on the device of the other tensors")
    if at != torch.cuda.current_device():
        raise KernelError(f"{what}: the tensors are on device {at}, which is not the current one")
    return at


def _given(what: str, name: str, t: Optional[torch.Tensor], shape: Tuple[int, ...], dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    """The output `name`: the tensor given, checked, or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=like.device)
    if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous():
        raise KernelError(f"{what}: {name} must be a contiguous {dtype} tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    return t


def _matrix(what: str, name: str, t: torch.Tensor) -> Tuple[int, int]:
    if t.dim() != 2 or t.shape[1] < 1 or t.shape[0] > _LIMIT or t.shape[1] > _LIMIT:
        raise KernelError(f"{what}: {name} must be a matrix with at least one column, got shape {tuple(t.shape)}")
    return t.shape[0], t.shape[1]


def quantize(x: torch.Tensor, out: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *,
             block_rows: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [T, K] (float32 or bfloat16, its rows ``x.stride(0)`` apart) in 8 bits: out [T, K] and scales [ceil(T / block_rows),
    ceil(K / 128)].  ``block_rows``: 1 for the rows of a product, 128 for a weight."""
    T, K = _matrix("quantize", "x", x)
    if block_rows not in (1, BLOCK):
        raise KernelError(f"quantize: block_rows is 1 or {BLOCK}, not {block_rows}")
    if (x.stride(1) != 1 and K > 1) or (T > 1 and x.stride(0) < K):
        raise KernelError(f"quantize: the rows of x must be contiguous and apart, got strides {x.stride()}")
    _on_device("quantize", x, out=out, scales=scales)
    out = _given("quantize", "out", out, (T, K), E4M3, x)
    scales = _given("quantize", "scales", scales, (T if block_rows == 1 else _blocks(T), _blocks(K)), torch.float32, x)
    call("fp8", "ph_quantize_fp8", x.data_ptr(), ops._code(x.dtype), x.stride(0) if T > 1 else K, out.data_ptr(), scales.data_ptr(), T, K,
         block_rows, ops._stream())
    return out, scales


def add_rmsnorm(x: torch.Tensor, add: Optional[torch.Tensor], weight: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None,
                scales: Optional[torch.Tensor] = None, *, rows: Optional[torch.Tensor] = None, add_splits: int = 1, write_x: bool = True,
                x_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """v = x[t] + sum_s add[s][t]; out, scales = v * rsqrt(mean(v^2) + eps) * weight in 8 bits, out [T, E], scales [T, ceil(E / 128)].

    ``x`` [T, E] is the float32 residual, ``add`` [T, E] or, with ``add_splits`` > 1, [splits, T, E] (float32 or bfloat16, or
    None), ``weight`` float32 [E].  v is kept in ``x_out`` [T, E] where that is given, else in x itself (unless ``write_x`` is
    false or there is nothing to add).  ``rows`` (int32 [n]) picks the rows that are normed, in that order (out [n, E]); nothing is
    kept then, and a number outside 0 .. T - 1 leaves its row of out and scales as it was."""
    T, E = _matrix("add_rmsnorm", "x", x)
    if E > MAX_NORM_WIDTH:
        raise KernelError(f"add_rmsnorm: rows of at most {MAX_NORM_WIDTH} values, not {E}")
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise KernelError("add_rmsnorm: x must be contiguous float32")
    if weight.dtype != torch.float32 or weight.shape != (E,) or not weight.is_contiguous():
        raise KernelError(f"add_rmsnorm: weight must be contiguous float32 [{E}]")
    if add is not None and (add_splits < 1 or add.shape != ((T, E) if add_splits == 1 and add.dim() == 2 else (add_splits, T, E)) or not add.is_contiguous()):
        raise KernelError(f"add_rmsnorm: add must be contiguous {add_splits} x [{T}, {E}], got {tuple(add.shape)}")
    if not eps >= 0.0:
        raise KernelError(f"add_rmsnorm: eps must not be negative, got {eps}")
    n = T
    if rows is not None:
        if rows.dtype != torch.int32 or rows.dim() != 1 or not rows.is_contiguous() or x_out is not None:
            raise KernelError("add_rmsnorm: rows must be a contiguous int32 vector, and x_out does not go with it")
        n = rows.shape[0]
    _on_device("add_rmsnorm", x, add=add, weight=weight, out=out, scales=scales, rows=rows, x_out=x_out)
    out = _given("add_rmsnorm", "out", out, (n, E), E4M3, x)
    scales = _given("add_rmsnorm", "scales", scales, (n, _blocks(E)), torch.float32, x)
    keep = None
    if x_out is not None:
        keep = _given("add_rmsnorm", "x_out", x_out, (T, E), torch.float32, x).data_ptr()
    elif write_x and add is not None and rows is None:
        keep = x.data_ptr()
    if n and not T:
        raise KernelError("add_rmsnorm: there are no rows to pick from")
    call("fp8", "ph_add_rmsnorm_fp8", x.data_ptr(), None if add is None else add.data_ptr(), ops.F32 if add is None else ops._code(add.dtype),
         add_splits, T * E, weight.data_ptr(), eps, None if rows is None else rows.data_ptr(), n, T, E, keep, out.data_ptr(),
         scales.data_ptr(), ops._stream())
    return out, scales


def gated(gate_up: torch.Tensor, out: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *, splits: int = 1,
          gate=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """out, scales = silu(g) * u in 8 bits for rows [g0, u0, g1, u1, ...]: gate_up [T, 2 F], or [splits, T, 2 F] partial sums
    with ``splits`` > 1 (float32 or bfloat16), to out [T, F], scales [T, ceil(F / 128)].  ``gate``: None (silu), (alpha, limit,
    shift) of the clamped swish, or "gelu_tanh"."""
    if gate_up.dim() != (2 if splits == 1 else 3) or gate_up.shape[-1] % 2 or not gate_up.shape[-1] or not gate_up.is_contiguous() or \
            (splits > 1 and gate_up.shape[0] != splits) or splits < 1 or gate_up.shape[-1] > _LIMIT:
        raise KernelError(f"gated: gate_up must be contiguous (gate, up) pairs in {splits} parts, got {tuple(gate_up.shape)}")
    T, F = gate_up.shape[-2], gate_up.shape[-1] // 2
    _on_device("gated", gate_up, out=out, scales=scales)
    out = _given("gated", "out", out, (T, F), E4M3, gate_up)
    scales = _given("gated", "scales", scales, (T, _blocks(F)), torch.float32, gate_up)
    call("fp8", "ph_gated_fp8", gate_up.data_ptr(), ops._code(gate_up.dtype), splits, T * 2 * F, out.data_ptr(), scales.data_ptr(), T, F,
         _gate_pointer(gate), ops._stream())
    return out, scales


def error_flag(device) -> torch.Tensor:
    flag = _flags.get(device)
    if flag is None:
        flag = _flags[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return flag


def check_errors(device) -> None:
    """Raise if a product gave up on a wait since the last check (synchronises the device)."""
    index = torch.device(device).index
    flag = _flags.get(torch.device("cuda", torch.cuda.current_device() if index is None else index))
    if flag is not None:
        code = int(flag.item())
        if code:
            flag.zero_()
            raise KernelError(f"gemm_fp8: {ERRORS.get(code, 'error')} (status {code})")


def gemm(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: Optional[torch.Tensor] = None, *,
         out_dtype: torch.dtype = torch.bfloat16, tile: int = 0, splits: int = 0, early_w: bool = False) -> torch.Tensor:
    """out [M, N] = (x * x_scales) @ (w * w_scales)^T: x [M, K] with x_scales [M, ceil(K / 128)], w [N, K] with w_scales
    [ceil(N / 128), ceil(K / 128)], K a multiple of 16, sums in float32, out float32 or bfloat16 (``out_dtype`` where out is not
    given).  ``tile`` and ``splits`` (0: the kernel's own choice): 16, 32 or 64 tokens beside 128 features, or 128 x 128; the CTAs that
    share a tile's K.  ``early_w``: w is not the result of a kernel that may still run when the product starts (a model's weight),
    so its first tiles may be read before the kernel in front has ended."""
    M, K = _matrix("gemm_fp8", "x", x)
    N, K2 = _matrix("gemm_fp8", "w", w)
    if x.dtype != E4M3 or w.dtype != E4M3 or not x.is_contiguous() or not w.is_contiguous():
        raise KernelError("gemm_fp8: x and w must be contiguous float8_e4m3fn tensors")
    if K != K2 or N < 1:
        raise KernelError(f"gemm_fp8: x {tuple(x.shape)} and w {tuple(w.shape)} do not fit")
    kb = _blocks(K)
    if x_scales.dtype != torch.float32 or x_scales.shape != (M, kb) or not x_scales.is_contiguous():
        raise KernelError(f"gemm_fp8: x_scales must be contiguous float32 [{M}, {kb}]")
    if w_scales.dtype != torch.float32 or w_scales.shape != (_blocks(N), kb) or not w_scales.is_contiguous():
        raise KernelError(f"gemm_fp8: w_scales must be contiguous float32 [{_blocks(N)}, {kb}]")
    _on_device("gemm_fp8", x, x_scales=x_scales, w=w, w_scales=w_scales, out=out)
    out = _given("gemm_fp8", "out", out, (M, N), out_dtype if out is None else out.dtype, x)
    call("fp8", "ph_gemm_fp8", x.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), out.data_ptr(), ops._code(out.dtype), M, N, K,
         tile, splits, 1 if early_w else 0, error_flag(x.device).data_ptr(), ops._stream())
    return out
