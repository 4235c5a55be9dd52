"""Attention over packed sequences, and the norm and rotation of its queries and keys (K7, K8).

The sequence dimension's side of the model: the diffusion head's token transformer, whose additive
pair biases :func:`pair_cond.pair_biases` makes (``mlx_diffusion.py:259,369``), and the language
model in front of the trunk (``mlx_esmc.py``).  Tokens of all sequences lie behind one another,
``[T, heads, D]``, and ``cu_seqlens`` says where each sequence begins, so nothing is padded.

    q, k = qk_norm_rope(q, k, positions, rotary, norm="layer", q_weight=..., k_weight=...)
    o = attention(q, k, v, cu_seqlens)

``q``, ``k`` and ``v`` may be slices of one fused projection: the values of a head are contiguous and
the other strides are multiples of 8 elements.  Launches go on the current stream of the tensors'
device; nothing synchronises.  Inference only: an input that asks for gradients, or carries a tangent, is
refused.

A kernel's waits are bounded.  One that gives up leaves its output invalid and records it in the call's
``status`` block (``ops.new_status``, read by ``ops.check_status``), or without one in the device's own
record, which ``ops.check_sequence_status()`` reads where the program synchronises anyway.
"""

from __future__ import annotations

import math
from decimal import Context, Decimal, localcontext

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float16: _lib.TMU_F16, torch.bfloat16: _lib.TMU_BF16}
_PI = Decimal("3.141592653589793238462643383279502884197169399375105820974944592")
_NORMS = {None: _lib.TMU_NORM_NONE, "rms": _lib.TMU_NORM_RMS, "layer": _lib.TMU_NORM_LAYER}


# The current stream's handle by device index, without making a Stream object for it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def launch(device: torch.device, where: str, *args) -> None:
    """Call the C entry ``where`` with ``args`` and the current stream of ``device``, which is made the
    current device for the call if it is not."""
    fn = getattr(_lib._lib or _lib.load(), where)
    index = device.index
    if torch.cuda.current_device() == index:
        code = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            code = fn(*args, _raw_stream(index))
    if code:
        _lib.check(code, where)


def pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def refuse_grad(where: str, *tensors) -> None:
    """Raise if autograd would expect a gradient, or a tangent, from an operator that has none."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{where} has no backward pass: call it under torch.no_grad() or detach its inputs")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():  # inside forward_ad.dual_level()
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{where} has no forward derivative: unpack its inputs' primals")


def check_status_block(status: torch.Tensor | None, device: torch.device) -> None:
    """Raise unless ``status`` is None or a block as ``ops.new_status`` makes it."""
    if status is not None and (status.dtype is not torch.uint8 or status.numel() < _lib.TMU_STATUS_BYTES
                               or status.device != device or not status.is_contiguous() or status.data_ptr() % 16):
        raise ValueError("status must be ops.new_status of the tensors' device")


def spans_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges that two strided tensors reach over meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False

    def span(t):
        return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()

    return a.data_ptr() < b.data_ptr() + span(b) and b.data_ptr() < a.data_ptr() + span(a)


def _view(name: str, t: torch.Tensor, T: int, D: int, like: torch.Tensor) -> tuple[int, int, int, int]:
    """Address, token stride, head stride and heads of a [T, H, D] view of ``like``'s type and device."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[0] != T or shape[2] != D:
        raise ValueError(f"{name} must be [{T}, heads, {D}], got {tuple(shape)}")
    if t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} must have q's type and device")
    if stride[2] != 1 and D > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous")
    heads = shape[1]
    # an axis of length one is never stepped along: its stride is whatever the view happened to have
    return t.data_ptr(), stride[0] if T > 1 else 0, stride[1] if heads > 1 else 0, heads


def _check_first(name: str, q: torch.Tensor) -> int:
    code = _DTYPES.get(q.dtype)
    if code is None or not q.is_cuda:
        raise TypeError(f"{name} must be a CUDA fp16 or bf16 tensor")
    if q.dim() != 3:
        raise ValueError(f"{name} must be [T, heads, D], got {tuple(q.shape)}")
    return code


class Rotary:
    """Rotary position embedding of the first ``rot`` values of a head: pair i turns by
    ``position * base ** (-2 i / rot)`` radians.

    ``layout`` pairs (i, i + rot / 2) as ``"half"`` and (2 i, 2 i + 1) as ``"interleaved"``.
    ``scaling`` stretches it to contexts longer than the trained one:

    * ``{"type": "linear", "factor": s}``: every frequency divided by s.
    * ``{"type": "ntk", "factor": s}``: base times ``s ** (rot / (rot - 2))``, which leaves the fastest
      pair and divides the slowest by s.
    * ``{"type": "yarn", "factor": s, "original_length": n, "beta_fast": 32, "beta_slow": 1,
      "gain": 0.1 ln s + 1}``: pairs that turn more than ``beta_fast`` times over n positions stay, those
      below ``beta_slow`` are divided by s, with a linear ramp over the pair index between, and the
      rotated values are multiplied by ``gain``.

    Frequencies are kept as turns a position in 64-bit fixed point, each the nearest one, and multiplied
    by the 64-bit position in integers, negative ones too.  So the angle is off by at most
    ``abs(position) * 2**-65`` of a turn (2^-33 at 2^32 positions, 2^-26 at 2^39) and by its conversion to
    fp32, 2^-26 of a turn.  ``frequencies`` has them in radians a position, rounded to 64-bit floats."""

    def __init__(self, rot: int, base: float = 10000.0, layout: str = "half", scaling: dict | None = None,
                 device="cuda"):
        if rot < 16 or rot % 16:
            raise ValueError("rot must be a positive multiple of 16")
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be 'half' or 'interleaved'")
        self.rot, self.base, self.layout = int(rot), float(base), layout
        self.gain = 1.0
        with localcontext(Context(prec=60)):  # 64 bits of a turn need more digits than a float's 53
            exact = self._frequencies(scaling)
            fixed = [int((f / (2 * _PI) * 2**64).to_integral_value()) % 2**64 for f in exact]
        self.frequencies = [float(f) for f in exact]
        signed = [f - 2**64 if f >= 2**63 else f for f in fixed]
        self.turns = torch.tensor(signed, dtype=torch.int64).to(device)

    def _frequencies(self, scaling: dict | None) -> list[Decimal]:
        """Radians a position, to the digits of the current decimal context."""
        half, base = self.rot // 2, Decimal(self.base)
        kind = None if scaling is None else scaling.get("type")
        if kind not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"unknown scaling {kind!r}")
        s = 1.0 if kind is None else float(scaling["factor"])
        if not (0.0 < s < math.inf and 1.0 < self.base < math.inf):
            raise ValueError("the factor must be positive and the base above 1, both finite")
        factor = Decimal(s)
        if kind == "ntk":
            base *= factor ** (Decimal(self.rot) / (self.rot - 2))
        # one power and a product a pair: a power each took 1.7 ms for 32 pairs
        step, freq = base ** (Decimal(-1) / half), [Decimal(1)]
        while len(freq) < half:
            freq.append(freq[-1] * step)
        if kind == "linear":
            return [f / factor for f in freq]
        if kind == "yarn":
            n = float(scaling["original_length"])

            def pair_at(turns):  # the pair index that turns `turns` times over n positions
                return half * math.log(n / (turns * 2.0 * math.pi)) / math.log(self.base)

            lo = max(math.floor(pair_at(float(scaling.get("beta_fast", 32.0)))), 0)
            hi = min(math.ceil(pair_at(float(scaling.get("beta_slow", 1.0)))), self.rot - 1)
            self.gain = float(scaling.get("gain", 0.1 * math.log(s) + 1.0 if s > 1.0 else 1.0))
            width = Decimal(hi - lo) if hi > lo else Decimal("0.001")
            ramp = [min(Decimal(1), max(Decimal(0), (i - lo) / width)) for i in range(half)]
            return [f * (1 - r) + f / factor * r for f, r in zip(freq, ramp)]
        return freq


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor | None = None, rotary: Rotary | None = None,
                 *, norm: str | None = None, q_weight=None, k_weight=None, q_bias=None, k_bias=None,
                 eps: float = 1e-5, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """K8: the norm of every head of ``q`` [T, Hq, D] and ``k`` [T, Hkv, D] over its D values, then the
    rotation by ``positions`` [T] (int32 or int64), in one pass; returns ``(q_out, k_out)``.  (A norm over
    all heads of a token together, as some models have before they split the heads, is another one: apply
    it first and rotate with ``norm=None``.)

    ``norm`` is None, ``"rms"`` or ``"layer"``, with fp32 weights and biases [D] (None: 1 and 0), ``eps`` 0 or
    above (the mean square plus eps counts as 0 below 2^-126); without ``rotary`` only the norm is applied.  D is a multiple of 16, at most 256.  ``q_out`` may be ``q`` and
    ``k_out`` may be ``k``; other overlaps are refused."""
    dtype = _check_first("q", q)
    T, hq, D = q.shape
    qp, qt, qh, _ = _view("q", q, T, D, q)
    kp, kt, kh, hk = _view("k", k, T, D, q)
    kind = _NORMS.get(norm)
    if kind is None:
        raise ValueError("norm must be None, 'rms' or 'layer'")
    refuse_grad("qk_norm_rope", q, k, q_weight, k_weight, q_bias, k_bias, q_out, k_out)
    if norm is None:
        if not (q_weight is k_weight is q_bias is k_bias is None):
            raise ValueError("weights and biases need a norm")
    else:
        for p in (q_weight, k_weight, q_bias, k_bias):
            if p is not None and (p.dtype is not torch.float32 or p.dim() != 1 or p.shape[0] != D
                                  or p.device != q.device or not p.is_contiguous()):
                raise ValueError(f"weights and biases must be contiguous fp32 [{D}] tensors on q's device")
    rot = (0, 4, 0, 1.0, 0, 0)
    if rotary is not None:
        if rotary.rot > D:
            raise ValueError(f"the rotary's {rotary.rot} values exceed the head's {D}")
        if positions is None:
            raise ValueError("a rotary needs positions")
        if (positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or positions.shape[0] != T
                or positions.device != q.device or not positions.is_contiguous()):
            raise ValueError(f"positions must be a contiguous int32 or int64 [{T}] tensor on q's device")
        if rotary.turns.device != q.device:
            raise ValueError("the rotary must be on q's device")
        rot = (positions.data_ptr(), positions.element_size(), rotary.turns.data_ptr(), rotary.gain, rotary.rot,
               1 if rotary.layout == "interleaved" else 0)
    given = q_out is not None or k_out is not None
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        qo = (q_out.data_ptr(), hq * D, D, hq)
    else:
        qo = (qp, qt, qh, hq) if q_out is q else _view("q_out", q_out, T, D, q)
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        ko = (k_out.data_ptr(), hk * D, D, hk)
    else:
        ko = (kp, kt, kh, hk) if k_out is k else _view("k_out", k_out, T, D, q)
    if given:
        _check_rope_outputs((qp, qt, qh, hq), (kp, kt, kh, hk), qo, ko, T, D)
    args = _lib.QK_NORM_ROPE_ARGS.pack(qp, qt, qh, kp, kt, kh, *qo[:3], *ko[:3], kind, eps, pointer(q_weight),
                                       pointer(q_bias), pointer(k_weight), pointer(k_bias), *rot, T, hq, hk, D, dtype)
    launch(q.device, "tmu_qk_norm_rope", args)
    return q_out, k_out


def _check_rope_outputs(q, k, q_out, k_out, T: int, D: int) -> None:
    """The views (address, token stride, head stride, heads) of 16-bit tensors."""
    for name, src, dst, other in (("q_out", q, q_out, k), ("k_out", k, k_out, q)):
        if dst[3] != src[3]:
            raise ValueError(f"{name} must be shaped like its input")
        if _folded(dst, T, D):
            raise ValueError(f"{name} must not overlap itself")
        if _meet(dst, other, T, D, T, D) or (dst != src and _meet(dst, src, T, D, T, D)):
            raise ValueError(f"{name} may be its own input, and must not overlap one otherwise")
    if _meet(q_out, k_out, T, D, T, D):
        raise ValueError("q_out and k_out must not overlap")


def _folded(view, T: int, D: int) -> bool:
    """Whether two heads of a [T, H, D] view share memory (exact for non-negative strides)."""
    _, st, sh, H = view
    axes = [(s, n) for s, n in ((st, T), (sh, H)) if n > 1]
    span = D
    for s, n in sorted(axes):
        if s < span:
            return True
        span += s * (n - 1)
    return False


def _meet(a, b, Ta: int, Da: int, Tb: int, Db: int, size_a: int = 2, size_b: int = 2) -> bool:
    """Whether two [T, H, D] views of elements of the given sizes share memory.  Views of one
    projection interleave without sharing: with one token stride, their heads' ranges are compared
    within a token."""
    (pa, sta, sha, ha), (pb, stb, shb, hb) = a, b
    if Ta == 0 or Tb == 0 or ha == 0 or hb == 0:
        return False
    wa, wb = ((ha - 1) * sha + Da) * size_a, ((hb - 1) * shb + Db) * size_b  # bytes that a token's heads reach over
    if pa + (Ta - 1) * sta * size_a + wa <= pb or pb + (Tb - 1) * stb * size_b + wb <= pa:
        return False
    step = sta * size_a
    if Ta > 1 and step == stb * size_b and step >= wa and step >= wb:
        off = (pb - pa) % step  # b's heads begin `off` bytes behind a's in each period
        return off < wa or off + wb > step
    return True


def _ints(t: torch.Tensor) -> tuple[int, int, int, int]:
    return t.data_ptr(), t.stride(0), t.stride(1), t.shape[1]


def _self_overlap(t: torch.Tensor) -> bool:
    return _folded(_ints(t), t.shape[0], t.shape[2])


def _heads_overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    return _meet(_ints(a), _ints(b), a.shape[0], a.shape[2], b.shape[0], b.shape[2], a.element_size(), b.element_size())


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, *, causal: bool = False,
              scale: float | None = None, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """K7: softmax attention within each packed sequence: ``q`` [T, Hq, D], ``k`` and ``v`` [T, Hkv, D]
    (Hq a multiple of Hkv: query head h reads key head h // (Hq / Hkv)), ``cu_seqlens`` int32 [S + 1]
    on the device, ascending; returns ``out`` [T, Hq, D].

    ``scale`` defaults to 1 / sqrt(D).  ``bias`` [S or 1, Hq, n, n] of q's type is added to the scaled
    scores of each sequence's first n positions (``pair_cond.pair_biases(...)[block]`` with a sequence a
    fold, or with one fold's bias for all of its samples); -inf hides a key, and a row whose keys are
    all hidden comes out as 0.  D is a multiple of 8, at most 128.  Tokens past the last sequence are
    left as they were in ``out`` (unset in a new one).  What a row does not see, a key that its bias hides, a
    later one if ``causal``, another sequence, a token of no sequence, does not reach it, be it an infinity or
    a NaN.  Device errors go to ``status``, or to the record that ``ops.check_sequence_status`` reads."""
    dtype = _check_first("q", q)
    T, hq, D = q.shape
    qp, qt, qh, _ = _view("q", q, T, D, q)
    kp, kt, kh, hk = _view("k", k, T, D, q)
    vp, vt, vh, hv = _view("v", v, T, D, q)
    if hv != hk:
        raise ValueError("k and v must have the same heads")
    refuse_grad("attention", q, k, v, bias, out)
    if status is not None:
        check_status_block(status, q.device)
    if (cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.device != q.device
            or not cu_seqlens.is_contiguous() or cu_seqlens.shape[0] < 1):
        raise ValueError("cu_seqlens must be a contiguous int32 [S + 1] tensor on q's device")
    S = cu_seqlens.shape[0] - 1
    b = (0, 0, 0, 0, 0)
    if bias is not None:
        shape = bias.shape
        if (len(shape) != 4 or shape[0] not in (1, S) or shape[1] != hq or shape[2] != shape[3]
                or bias.dtype is not q.dtype or bias.device != q.device):
            raise ValueError(f"bias must be [1 or {S}, {hq}, n, n] of q's type on its device")
        n, stride = shape[2], bias.stride()
        if n > 1 and stride[3] != 1:
            raise ValueError("the last axis of bias must be contiguous")
        b = (bias.data_ptr(), stride[0] if shape[0] > 1 else 0, stride[1], stride[2], n)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op, ot, oh = out.data_ptr(), hq * D, D
    else:
        if out.shape != q.shape:
            raise ValueError("out must be shaped like q")
        o = op, ot, oh, _ = _view("out", out, T, D, q)
        if _folded(o, T, D) or any(_meet(o, t, T, D, T, D) for t in ((qp, qt, qh, hq), (kp, kt, kh, hk), (vp, vt, vh, hk))):
            raise ValueError("out must not overlap itself, q, k or v")
        if bias is not None and spans_overlap(out, bias):
            raise ValueError("out must not overlap bias")
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    args = _lib.ATTENTION_ARGS.pack(qp, qt, qh, kp, kt, kh, vp, vt, vh, op, ot, oh,
                                    cu_seqlens.data_ptr(), *b, S, T, hq, hk, D, dtype, 1 if causal else 0, scale,
                                    pointer(status))
    launch(q.device, "tmu_attention", args)
    return out
