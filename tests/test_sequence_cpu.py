"""CPU checks of the sequence operators: the argument checks of their C entries (nothing is launched),
the rotary's frequencies, the layout of 8-bit weights, and the refusals of the Python side."""

from __future__ import annotations

import ctypes
import math
import os
import re
from fractions import Fraction

import pytest
import torch
from torch.autograd import forward_ad

from esmfold2_mlx_b200 import _lib, attention as att, build, fp8

OK, INVALID, MISALIGNED, WORKSPACE, UNSUPPORTED = 0, 1, 2, 3, 4
P = 0x1000  # a pointer that no check follows


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def heads(data=P, st=64, sh=64):
    return _lib.TmuHeads(data, st, sh)


def attention(lib, q=None, k=None, v=None, o=None, cu=P, bias=None, S=1, T=4, hq=2, hkv=1, d=64, dtype=0, scale=0.125):
    h = heads()
    a = _lib.TmuAttentionArgs(q or h, k or h, v or h, o or h, cu, bias or _lib.TmuAttnBias(), S, T, hq, hkv, d, dtype, 0,
                              scale, None)
    return lib.tmu_attention(ctypes.byref(a), None)


def test_attention_refusals(lib):
    assert attention(lib, T=-1) == INVALID
    assert attention(lib, hq=0) == INVALID
    assert attention(lib, hq=3, hkv=2) == INVALID
    assert attention(lib, S=-1) == INVALID
    assert attention(lib, d=60) == UNSUPPORTED
    assert attention(lib, d=136) == UNSUPPORTED
    assert attention(lib, dtype=_lib.TMU_F32) == UNSUPPORTED
    assert attention(lib, cu=None) == INVALID
    assert attention(lib, scale=math.nan) == INVALID and attention(lib, scale=math.inf) == INVALID
    assert attention(lib, T=(1 << 30) + 1) == UNSUPPORTED
    assert attention(lib, q=heads(st=0)) == UNSUPPORTED and attention(lib, k=heads(st=0)) == UNSUPPORTED
    assert attention(lib, hq=4, hkv=2, v=heads(sh=0)) == UNSUPPORTED
    for name in "qkvo":
        assert attention(lib, **{name: heads(None)}) == INVALID
        assert attention(lib, **{name: heads(P + 2)}) == MISALIGNED
        assert attention(lib, **{name: heads(st=65)}) == MISALIGNED
        assert attention(lib, **{name: heads(sh=4)}) == MISALIGNED
        assert attention(lib, **{name: heads(st=-64)}) == INVALID
    assert attention(lib, bias=_lib.TmuAttnBias(None, 0, 0, 0, 5)) == INVALID
    assert attention(lib, bias=_lib.TmuAttnBias(P, 0, 0, 0, -1)) == INVALID
    assert lib.tmu_attention(None, None) == INVALID


def test_packed_arguments_have_the_structures_layout():
    """struct.pack's formats against the ctypes mirrors, field by field."""
    for fmt, cls in ((_lib.ATTENTION_ARGS, _lib.TmuAttentionArgs), (_lib.QK_NORM_ROPE_ARGS, _lib.TmuQkNormRopeArgs)):
        assert fmt.size == ctypes.sizeof(cls)
    a = _lib.TmuAttentionArgs.from_buffer_copy(_lib.ATTENTION_ARGS.pack(*range(1, 19), 19, 20, 21, 22, 23, 24, 25, 0.5, 26))
    assert (a.q.data, a.k.stride_head, a.out.stride_token, a.cu_seqlens, a.bias.data, a.bias.stride_row, a.bias.n, a.S) == (
        1, 6, 11, 13, 14, 17, 18, 19)
    assert (a.T, a.dtype, a.causal, a.scale, a.status) == (20, 24, 25, 0.5, 26)
    r = _lib.TmuQkNormRopeArgs.from_buffer_copy(
        _lib.QK_NORM_ROPE_ARGS.pack(*range(1, 13), 13, 0.5, 14, 15, 16, 17, 18, 8, 19, 2.0, 20, 1, 21, 22, 23, 24, 25))
    assert (r.k_out.stride_head, r.norm.kind, r.norm.eps, r.norm.k_bias, r.rotary.positions, r.rotary.position_bytes) == (
        12, 13, 0.5, 17, 18, 8)
    assert (r.rotary.turns, r.rotary.gain, r.rotary.rot, r.rotary.interleaved, r.T, r.Hq, r.Hkv, r.D, r.dtype) == (
        19, 2.0, 20, 1, 21, 22, 23, 24, 25)


def test_empty_calls_do_nothing(lib):
    none = heads(None)
    assert attention(lib, q=none, k=none, v=none, o=none, T=0) == OK
    assert attention(lib, S=0) == OK
    assert lib.tmu_quantize_rows(None, 0, 64, 0, 64, None, None, None) == OK
    assert lib.tmu_linear_fp8(None, 0, 64, None, None, None, None, None, 0, 8, 0, 8, 64, None, 0, None, None) == OK
    assert lib.tmu_linear_fp8_workspace_bytes(0, 8, 64) == 0


def rope(lib, d=64, T=4, dtype=0, kind=1, rot=64, pos=P, turns=P, nbytes=4, q=None, w=None, hq=2):
    h = heads()
    nrm = _lib.TmuQkNorm(kind, 1e-5, w, None, None, None)
    r = _lib.TmuRotary(pos, nbytes, turns, 1.0, rot, 0)
    return lib.tmu_qk_norm_rope(ctypes.byref(_lib.TmuQkNormRopeArgs(q or h, h, h, h, nrm, r, T, hq, 1, d, dtype)), None)


def test_qk_norm_rope_refusals(lib):
    assert rope(lib, d=40, rot=16) == UNSUPPORTED
    assert rope(lib, d=272) == UNSUPPORTED
    assert rope(lib, rot=80) == UNSUPPORTED
    assert rope(lib, rot=24) == UNSUPPORTED
    assert rope(lib, dtype=2) == UNSUPPORTED
    assert rope(lib, kind=3) == INVALID
    assert rope(lib, pos=None) == INVALID
    assert rope(lib, turns=None) == INVALID
    assert rope(lib, nbytes=2) == INVALID
    assert rope(lib, T=-1) == INVALID
    assert rope(lib, hq=0) == INVALID
    assert rope(lib, q=heads(P + 8)) == MISALIGNED
    assert rope(lib, w=P + 4) == MISALIGNED
    assert rope(lib, T=0) == OK


@pytest.mark.parametrize("eps", [-1e-5, math.nan, math.inf])
def test_norm_eps_refusals(lib, eps):
    h = heads()
    for kind, want in ((1, INVALID), (2, INVALID), (0, OK)):  # (T = 0: nothing is launched)
        args = _lib.TmuQkNormRopeArgs(h, h, h, h, _lib.TmuQkNorm(kind, eps, None, None, None, None),
                                      _lib.TmuRotary(None, 4, None, 1.0, 0, 0), 0, 1, 1, 64, 0)
        assert lib.tmu_qk_norm_rope(ctypes.byref(args), None) == want


def linear(lib, x=P, xd=0, ldx=64, xs=None, w=P, ws=P, out=P, od=0, ldo=8, M=40, N=8, K=64, work=P, nb=1 << 20):
    return lib.tmu_linear_fp8(x, xd, ldx, xs, w, ws, None, out, od, ldo, M, N, K, work, nb, None, None)


def test_linear_refusals(lib):
    assert linear(lib, K=24, ldx=24) == UNSUPPORTED
    assert linear(lib, xd=_lib.TMU_F32) == UNSUPPORTED
    assert linear(lib, od=_lib.TMU_E4M3) == UNSUPPORTED
    assert linear(lib, M=-1) == INVALID
    assert linear(lib, N=0) == INVALID
    assert linear(lib, x=None) == INVALID
    assert linear(lib, out=None) == INVALID
    assert linear(lib, xd=_lib.TMU_E4M3) == INVALID  # no scales
    assert linear(lib, xd=_lib.TMU_E4M3, xs=P, ldx=80) == UNSUPPORTED
    assert linear(lib, ldo=4) == INVALID
    assert linear(lib, ldx=32) == INVALID
    assert linear(lib, w=P + 8) == MISALIGNED
    assert linear(lib, nb=16) == WORKSPACE
    assert linear(lib, work=None) == WORKSPACE
    assert linear(lib, work=P + 8) == MISALIGNED
    assert lib.tmu_quantize_rows(P, 0, 60, 2, 48, P, P, None) == MISALIGNED
    assert lib.tmu_quantize_rows(P, 0, 32, 2, 48, P, P, None) == INVALID
    assert lib.tmu_quantize_rows(P, 2, 48, 2, 48, P, P, None) == UNSUPPORTED


def test_workspace_of_e4m3_rows(lib):
    """x that is e4m3 already needs room for its scales alone."""
    e4m3 = {"xd": _lib.TMU_E4M3, "xs": P, "K": 1360, "ldx": 1360, "M": 700}
    need = lib.tmu_linear_fp8_scaled_workspace_bytes(700, 8, 1360)
    assert need == 768 * 11 * 4 and lib.tmu_linear_fp8_workspace_bytes(700, 8, 1360) == need + 700 * 1360
    assert linear(lib, nb=need - 1, **e4m3) == WORKSPACE
    assert linear(lib, nb=need, work=P + 8, **e4m3) == MISALIGNED  # large enough
    assert linear(lib, nb=need, work=P + 8, K=1360, ldx=1360, M=700) == WORKSPACE
    assert lib.tmu_linear_fp8_scaled_workspace_bytes(16, 8, 64) == 0


def test_pointers_off_their_types_alignment(lib):
    """Every pointer that a kernel follows one value at a time, an odd number of bytes off."""
    assert attention(lib, cu=P + 2) == MISALIGNED
    assert attention(lib, bias=_lib.TmuAttnBias(P + 1, 0, 0, 8, 4)) == MISALIGNED
    assert rope(lib, pos=P + 2) == MISALIGNED and rope(lib, pos=P + 4, nbytes=8) == MISALIGNED
    assert rope(lib, turns=P + 4) == MISALIGNED
    for m in (1, 40):  # both kernels' ranges of rows
        assert linear(lib, M=m, out=P + 1) == MISALIGNED
        assert linear(lib, M=m, out=P + 2, od=_lib.TMU_F32) == MISALIGNED
        assert linear(lib, M=m, ws=P + 2) == MISALIGNED
        assert linear(lib, M=m, xd=_lib.TMU_E4M3, xs=P + 2) == MISALIGNED
        assert lib.tmu_linear_fp8(P, 0, 64, None, P, P, P + 2, P, 0, 8, m, 8, 64, P, 1 << 20, None, None) == MISALIGNED
    assert lib.tmu_quantize_rows(P, 0, 48, 2, 48, P, P + 2, None) == MISALIGNED


def test_sizes_past_the_index_range(lib):
    big = (1 << 30) + 1
    assert linear(lib, M=big) == UNSUPPORTED and linear(lib, N=big, ldo=1 << 31) == UNSUPPORTED
    assert linear(lib, K=(1 << 30) + 16, ldx=1 << 31) == UNSUPPORTED
    assert lib.tmu_quantize_rows(P, 0, 64, big, 64, P, P, None) == UNSUPPORTED
    assert lib.tmu_linear_fp8_workspace_bytes(big, 8, 64) == 0


def test_sequence_status_needs_an_address(lib):
    assert lib.tmu_sequence_status(None) == INVALID


def test_status_block(lib):
    assert lib.tmu_linear_fp8(P, 0, 64, None, P, P, None, P, 0, 8, 40, 8, 64, P, 1 << 20, P + 8, None) == MISALIGNED
    dev = torch.device("cpu")
    att.check_status_block(None, dev)
    att.check_status_block(torch.zeros(_lib.TMU_STATUS_BYTES, dtype=torch.uint8), dev)
    for bad in (torch.zeros(_lib.TMU_STATUS_BYTES - 1, dtype=torch.uint8), torch.zeros(_lib.TMU_STATUS_BYTES),
                torch.zeros(2 * _lib.TMU_STATUS_BYTES, dtype=torch.uint8)[::2],
                torch.zeros(2 * _lib.TMU_STATUS_BYTES, dtype=torch.uint8)[8:]):
        with pytest.raises(ValueError):
            att.check_status_block(bad, dev)


def test_rows_beside_one_another():
    """Columns of one buffer, of one type or two, do not overlap; rows that meet do."""
    buf = torch.zeros(10, 48, dtype=torch.float32)
    x, y = buf[:, :16].unsqueeze(1), buf[:, 16:].unsqueeze(1)
    assert not att._heads_overlap(y, x) and att._heads_overlap(buf[:, 15:].unsqueeze(1), x)
    half = buf.view(torch.float16)[:, :32].unsqueeze(1)
    assert not att._heads_overlap(y, half) and att._heads_overlap(x, half)
    assert att._heads_overlap(buf[:, :17].unsqueeze(1), y)


def test_python_refusals():
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        att.attention(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        att.qk_norm_rope(x, x)
    with pytest.raises(TypeError):
        fp8.quantize_rows(x[0])
    w = torch.zeros(4, 32, dtype=torch.float8_e4m3fn)
    with pytest.raises(TypeError):
        fp8.linear(x[0], fp8.BlockWeight(w, torch.ones(1, 1)))
    for bad in (lambda: fp8.BlockWeight(w, torch.ones(1, 2)), lambda: fp8.BlockWeight(w.half(), torch.ones(1, 1)),
                lambda: fp8.BlockWeight(w[:, :24], torch.ones(1, 1)), lambda: fp8.BlockWeight(w.t(), torch.ones(1, 1)),
                lambda: att.Rotary(24, device="cpu"), lambda: att.Rotary(32, layout="pairs", device="cpu"),
                lambda: att.Rotary(32, scaling={"type": "x"}, device="cpu"),
                lambda: att.Rotary(32, scaling={"type": "linear", "factor": 0.0}, device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_gradients_and_tangents_are_refused():
    x = torch.zeros(3)
    y = torch.zeros(3, requires_grad=True)
    att.refuse_grad("op", None, x)
    with pytest.raises(ValueError):
        att.refuse_grad("op", x, y)
    with torch.no_grad():
        att.refuse_grad("op", y)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        att.refuse_grad("op", x, forward_ad.unpack_dual(dual).primal)
        for t in (dual, dual[1:]):
            with pytest.raises(ValueError):
                att.refuse_grad("op", None, x, t)
            with torch.no_grad(), pytest.raises(ValueError):  # tangents are made under it too
                att.refuse_grad("op", t)
    with torch.no_grad():
        att.refuse_grad("op", x)


def test_heads_overlap():
    buf = torch.zeros(10, 6, 64)
    q, k, v = buf[:, :2], buf[:, 2:4], buf[:, 4:]
    assert not att._heads_overlap(q, k) and not att._heads_overlap(v, q)
    assert att._heads_overlap(buf[:, :3], k) and att._heads_overlap(buf, v) and att._heads_overlap(q, q)
    assert not att._heads_overlap(buf[:5], buf[5:])
    assert att._heads_overlap(buf[:6], buf[5:])
    assert att._heads_overlap(buf[..., :32], buf[..., 32:])  # interleaved within a token: refused as if shared
    assert att._self_overlap(torch.zeros(1, 2, 64).expand(5, 2, 64)) and not att._self_overlap(q)
    assert att._self_overlap(torch.as_strided(buf, (3, 2, 64), (64, 32, 1)))


def test_rotary_frequencies():
    r = att.Rotary(64, device="cpu")
    turns = [t % 2**64 for t in r.turns.tolist()]
    for i, t in enumerate(turns):
        f = 10000.0 ** (-2 * i / 64) / (2 * math.pi)
        assert abs(t / 2.0**64 - f) <= 2.0 ** -52
    assert r.gain == 1.0
    lin = att.Rotary(64, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert all(abs(a * 4 - b) < 1e-12 for a, b in zip(lin.frequencies, r.frequencies))
    ntk = att.Rotary(64, scaling={"type": "ntk", "factor": 4.0}, device="cpu")
    assert ntk.frequencies[0] == 1.0 and abs(ntk.frequencies[-1] * 4 / r.frequencies[-1] - 1) < 1e-12
    y = att.Rotary(64, scaling={"type": "yarn", "factor": 16.0, "original_length": 4096}, device="cpu")
    ratio = [a / b for a, b in zip(y.frequencies, r.frequencies)]
    assert ratio[0] == 1.0 and abs(ratio[-1] * 16 - 1) < 1e-12 and all(a >= b for a, b in zip(ratio, ratio[1:]))
    assert abs(y.gain - (0.1 * math.log(16) + 1)) < 1e-15
    turned = [f * 4096 / (2 * math.pi) for f in r.frequencies]
    assert all(q == 1.0 for q, t in zip(ratio, turned) if t > 50) and all(q < 0.07 for q, t in zip(ratio, turned) if t < 0.7)


def test_weight_layout():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(200, 272, generator=g)
    w[130:] *= 100
    q = fp8.quantize_weight(w, "cpu")
    assert q.scales.shape == (2, 3) and q.shape == (200, 272)
    d = q.dequantize()
    s = q.scales.repeat_interleave(128, 0)[:200].repeat_interleave(128, 1)[:, :272]
    # half a step of 3 mantissa bits, or of the least subnormal 2^-9
    assert ((d - w).abs() <= torch.maximum(w.abs() * 2.0**-4, s * 2.0**-10) * (1 + 1e-6)).all()
    z = fp8.quantize_weight(torch.zeros(8, 16), "cpu")
    assert (z.dequantize() == 0).all() and (z.scales == fp8.SCALE_MIN).all()


def kernels(text):
    """Name and body of every __global__ function in a source file."""
    for m in re.finditer(r"__global__[^;{]*?(\w+)\(const __grid_constant__[^)]*\)\s*\{", text):
        depth, end = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield m.group(1), text[m.end():end]


def test_kernels_read_nothing_before_their_dependency_wait():
    """Whatever a call is given, weights too, may be the output of the kernel in front of it: no load of the
    sequence kernels stands before griddepcontrol.wait.  (Bodies of lambdas are left out: they run where
    they are called.)"""
    found = set()
    for name in ("k7_attention.cuh", "k8_qk_rope.cuh", "k9_linear8.cuh"):
        with open(os.path.join(build.CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for kernel, body in kernels(text):
            found.add(kernel)
            head, wait, _ = body.partition("griddep_wait();")
            assert wait, kernel
            while True:
                m = re.search(r"auto \w+ = \[&\]\(.*?\)\s*\{", head)
                if m is None:
                    break
                depth, end = 1, m.end()
                while depth:
                    depth += {"{": 1, "}": -1}.get(head[end], 0)
                    end += 1
                head = head[:m.start()] + head[end:]
            assert not re.search(r"\b(load\w*|__ldg|tma_load\w*|run)\(|ld\.global|cp\.async", head), kernel
    assert found == {"attention_kernel", "qk_rope_kernel", "quantize_kernel", "transpose_scales_kernel",
                     "linear8_rows_kernel", "linear8_kernel", "linear8_pair_kernel"}


def pi_bounds():
    """pi from Machin's formula in integers, to 2^-240 either way."""
    one = 1 << 256

    def arctan_inverse(x):
        total, term, k = 0, one // x, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= x * x
            k += 2
        return total

    pi = 4 * (4 * arctan_inverse(5) - arctan_inverse(239))
    return Fraction(pi - (1 << 16), one), Fraction(pi + (1 << 16), one)


@pytest.mark.parametrize("rot,base", [(16, 10000.0), (64, 10000.0), (64, 500000.0), (128, 10000.5)])
@pytest.mark.parametrize("kind", [None, "linear", "ntk", "yarn"])
def test_rotary_turns_are_the_nearest(rot, base, kind):
    """Each 64-bit turn against its definition in rational numbers: with f = 2 pi turns / 2^64, and the
    factors that the scaling gives it taken off, f^(rot / 2) base^i = 1 lies between half a unit below and
    above (ntk: f^(h (h - 1)) base^(i (h - 1)) s^(i h) = 1 with h = rot / 2)."""
    s = Fraction(4) if kind != "yarn" else Fraction(16)
    scaling = {None: None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 4.0},
               "yarn": {"type": "yarn", "factor": 16.0, "original_length": 4096}}[kind]
    half, b = rot // 2, Fraction(base)
    lo = max(math.floor(half * math.log(4096 / (32 * 2 * math.pi)) / math.log(base)), 0)
    hi = min(math.ceil(half * math.log(4096 / (2 * math.pi)) / math.log(base)), rot - 1)
    pi_lo, pi_hi = pi_bounds()
    unit = Fraction(1, 1 << 64)
    near = Fraction(1, 2) + Fraction(1, 1 << 32)
    for i, t in enumerate(att.Rotary(rot, base, scaling=scaling, device="cpu").turns.tolist()):
        take = Fraction(1)
        if kind == "linear":
            take = s
        if kind == "yarn":
            r = min(max(Fraction(i - lo, hi - lo), Fraction(0)), Fraction(1))
            take = 1 / (1 - r + r / s)
        low, high = 2 * pi_lo * (t - near) * unit * take, 2 * pi_hi * (t + near) * unit * take
        if kind == "ntk":
            rest = b ** (i * (half - 1)) * s ** (i * half)
            assert low ** (half * (half - 1)) * rest < 1 < high ** (half * (half - 1)) * rest, i
        else:
            assert low ** half * b ** i < 1 < high ** half * b ** i, i
    for bad in ({"base": math.inf}, {"base": math.nan}, {"scaling": {"type": "linear", "factor": math.inf}},
                {"scaling": {"type": "ntk", "factor": math.nan}}):
        with pytest.raises(ValueError):
            att.Rotary(rot, device="cpu", **bad)


def test_arrives_on_the_other_cta_have_the_clusters_scope():
    """An arrive on another CTA's barrier names the cluster's scope (the default is the CTA's), and the pair
    kernel of the 8-bit product waits in it for every barrier that the pair shares."""
    for name in sorted(os.listdir(build.CSRC)):
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        for m in re.finditer(r"mbarrier\.arrive\.[\w.:]*shared::cluster", text):
            assert re.search(r"\.(release|relaxed)\.cluster\.", m.group(0)), (name, m.group(0))
        if name == "k9_linear8.cuh":
            body = dict(kernels(re.sub(r"//[^\n]*", "", text)))["linear8_pair_kernel"]
            assert body.count("warp_poll_pair(") == 4 and "warp_poll(" not in body
