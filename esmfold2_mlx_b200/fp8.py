"""Linear layers with 8-bit operands and a scale for each block of 128 (K9).

The layers of the sequence dimension that are bound by their weights (the language model in front
of the trunk, whose weights the reference also holds in 8 bits, ``mlx_esmc.py:73,81``, in groups of 64
and as integers).  Here both operands are e4m3: the weight is laid out once with one fp32 scale a
128 x 128 block, and activations get one scale a row and 128 values at the call, so the tensor cores
run their 8-bit form and a block's largest value uses the whole range.

    w = fp8.quantize_weight(linear.weight)
    y = fp8.linear(x, w, bias=linear.bias)

Launches go on the current stream of the tensors' device; nothing synchronises.  Inference only: an
input that asks for gradients, or carries a tangent, is refused.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .attention import _heads_overlap, check_status_block, launch, pointer, refuse_grad, spans_overlap

BLOCK = 128
F8_MAX = 448.0          # the largest e4m3 value
SCALE_MIN = 2.0 ** -126  # the least scale: an all-zero block keeps a usable quotient
ROWS_MAX = 2 ** 30       # rows of x, and of a weight

_IN = {torch.float16: _lib.TMU_F16, torch.bfloat16: _lib.TMU_BF16, torch.float8_e4m3fn: _lib.TMU_E4M3}
_OUT = {torch.float16: _lib.TMU_F16, torch.bfloat16: _lib.TMU_BF16, torch.float32: _lib.TMU_F32}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


@dataclass
class BlockWeight:
    """An e4m3 weight [N, K] (``nn.Linear`` layout) with fp32 scales [ceil(N / 128), ceil(K / 128)]."""

    w8: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        w, s = self.w8, self.scales
        if w.dtype != torch.float8_e4m3fn or w.dim() != 2 or not w.is_contiguous():
            raise ValueError("w8 must be a contiguous float8_e4m3fn [N, K] tensor")
        if not 1 <= w.shape[0] <= ROWS_MAX or w.shape[1] < 1 or w.shape[1] % 16:
            raise ValueError(f"K must be a positive multiple of 16, N positive and at most {ROWS_MAX}")
        shape = (_blocks(w.shape[0]), _blocks(w.shape[1]))
        if s.dtype != torch.float32 or tuple(s.shape) != shape or not s.is_contiguous() or s.device != w.device:
            raise ValueError(f"scales must be a contiguous fp32 {list(shape)} tensor on w8's device")

    @property
    def shape(self) -> torch.Size:
        return self.w8.shape

    def dequantize(self) -> torch.Tensor:
        """The fp32 weight that the products see."""
        n, k = self.w8.shape
        s = self.scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        return self.w8.float() * s


def quantize_weight(weight: torch.Tensor, device="cuda") -> BlockWeight:
    """Lay out ``weight`` [N, K] once: scale = max(amax / 448, 2^-126) of each 128 x 128 block, values
    rounded to e4m3."""
    w = weight.detach().float().to(device)
    if w.dim() != 2:
        raise ValueError("weight must be [N, K]")
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    pad = torch.zeros(nb * BLOCK, kb * BLOCK, device=w.device)
    pad[:n, :k] = w
    blocks = pad.view(nb, BLOCK, kb, BLOCK)
    amax = blocks.abs().amax(dim=(1, 3))
    scales = torch.clamp(amax / torch.full_like(amax, F8_MAX), min=SCALE_MIN)
    q = (blocks / scales[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :k]
    return BlockWeight(q.to(torch.float8_e4m3fn).contiguous(), scales)


def _rows(name: str, x: torch.Tensor) -> torch.Tensor:
    """x as [M, K] rows of contiguous values, without a copy."""
    if x.dim() < 1 or (x.shape[-1] > 1 and x.stride(-1) != 1):
        raise ValueError(f"the last axis of {name} must be contiguous")
    if x.dim() == 2:
        return x
    try:
        return x.view(-1, x.shape[-1])
    except RuntimeError:
        raise ValueError(f"the leading axes of {name} must be one run of equally spaced rows") from None


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """K9's operands: fp16 or bf16 ``x`` [M, K] (K a multiple of 16) to ``(x8, scales)``, e4m3 [M, K] and
    fp32 [M, ceil(K / 128)], x ~ x8 * scale with scale = max(amax / 448, 2^-126) over 128 values of a row.
    A block that holds an infinity or a NaN becomes NaN."""
    if not x.is_cuda or x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError("x must be a CUDA fp16 or bf16 tensor")
    if x.dim() != 2:
        raise ValueError(f"x must be [M, K], got {tuple(x.shape)}")
    refuse_grad("quantize_rows", x)
    x = _rows("x", x)
    m, k = x.shape
    if m > ROWS_MAX:
        raise ValueError(f"x has {m} rows, more than {ROWS_MAX}")
    x8 = torch.empty(m, k, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(m, _blocks(k), dtype=torch.float32, device=x.device)
    launch(x.device, "tmu_quantize_rows", x.data_ptr(), _IN[x.dtype], _ld(x), m, k, x8.data_ptr(), scales.data_ptr())
    return x8, scales


def linear(x: torch.Tensor, weight: BlockWeight, bias: torch.Tensor | None = None, *,
           x_scales: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
           out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """K9: ``x @ weight^T + bias`` for fp16 or bf16 ``x`` [..., K], quantised at the call, or for e4m3 ``x``
    [..., K] with ``x_scales`` [..., ceil(K / 128)] from :func:`quantize_rows`; returns [..., N].

    ``bias`` is fp32 [N].  The output is ``out_dtype`` (fp16, bf16 or fp32; x's type by default, fp16 for
    e4m3 x) or ``out`` [..., N], which must not overlap an input.  Device errors go to ``status``, or to the
    record that ``ops.check_sequence_status`` reads."""
    code = _IN.get(x.dtype)
    if code is None or not x.is_cuda:
        raise TypeError("x must be a CUDA fp16, bf16 or float8_e4m3fn tensor")
    w8, scales, shape = weight.w8, weight.scales, x.shape
    n, k = w8.shape
    if len(shape) < 1 or shape[-1] != k:
        raise ValueError(f"x must be [..., {k}], got {tuple(shape)}")
    if w8.device != x.device:
        raise ValueError("the weight must be on x's device")
    refuse_grad("fp8.linear", x, bias, scales, x_scales, out)
    if status is not None:
        check_status_block(status, x.device)
    rows = _rows("x", x)
    m, ld = rows.shape[0], _ld(rows)
    if m > ROWS_MAX:
        raise ValueError(f"x has {m} rows, more than {ROWS_MAX}")
    xs = 0
    if code == _lib.TMU_E4M3:
        want = (*shape[:-1], _blocks(k))
        if (x_scales is None or x_scales.dtype is not torch.float32 or x_scales.shape != want
                or x_scales.device != x.device or not x_scales.is_contiguous()):
            raise ValueError(f"e4m3 x needs contiguous fp32 x_scales {list(want)} on its device")
        if not x.is_contiguous():
            raise ValueError("e4m3 x must be contiguous")
        xs = x_scales.data_ptr()
    elif x_scales is not None:
        raise ValueError("x_scales go with e4m3 x")
    if bias is not None and (bias.dtype is not torch.float32 or bias.dim() != 1 or bias.shape[0] != n
                             or bias.device != x.device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 [{n}] tensor on x's device")
    if out is None:
        dt = out_dtype or (torch.float16 if code == _lib.TMU_E4M3 else x.dtype)
        out_code = _OUT.get(dt)
        if out_code is None:
            raise TypeError("out_dtype must be fp16, bf16 or fp32")
        out = x.new_empty((*shape[:-1], n), dtype=dt)
        to, ldo = out.data_ptr(), n
    else:
        out_code = _OUT.get(out.dtype)
        if out_code is None or out.shape != (*shape[:-1], n) or out.device != x.device:
            raise ValueError(f"out must be an fp16, bf16 or fp32 {[*shape[:-1], n]} tensor on x's device")
        if out_dtype not in (None, out.dtype):
            raise ValueError("out_dtype differs from out's type")
        orow = _rows("out", out)
        # (out may be columns beside x's in one buffer)
        if (_heads_overlap(orow.unsqueeze(1), rows.unsqueeze(1))
                or any(t is not None and spans_overlap(out, t) for t in (w8, scales, bias, x_scales))):
            raise ValueError("out must not overlap an input")
        to, ldo = orow.data_ptr(), _ld(orow)
    lib = _lib._lib or _lib.load()
    need = (lib.tmu_linear_fp8_scaled_workspace_bytes if xs else lib.tmu_linear_fp8_workspace_bytes)(m, n, k)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None  # held until the launch is in the stream
    launch(x.device, "tmu_linear_fp8", rows.data_ptr(), code, ld, xs, w8.data_ptr(), scales.data_ptr(), pointer(bias), to,
           out_code, ldo, m, n, k, pointer(ws), need, pointer(status))
    return out
