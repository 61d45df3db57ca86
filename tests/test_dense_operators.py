"""RMS norm, 8-bit rows, projections and beam search on the CPU (the branch of the same entry points that CPU tensors take) and on the
device, against the definitions in 64 bits.

Tolerances are sums of roundings, element by element from the exact values: u = 2^-24 is float32's half step, half(t) that of a type
that a value is rounded to.  A sum in which a term goes through d additions is off by d u sum |a_i|; the matrix cores' additions do not round
to nearest, so theirs count twice.
"""
import math

import numpy as np
import pytest
import torch

from difflut_amd import ops
from difflut_amd.utils import GroupSum, Linear, RMSNorm, TokenEmbedding, beam_reorder, beam_step, cross_entropy

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CPU_AND_GPU = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
E4M3_HALF, E4M3_LEAST = 2.0 ** -4, 2.0 ** -10  # half steps: relative, and of the values below 2^-6


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, bound, dtype):
    """|got - want| within `bound` (of what was computed) and the rounding to `dtype` (of what came out)."""
    got, want, bound = got.detach().double(), want.detach().double().to(got.device), bound.double().to(got.device)
    limit = bound * (1 + half(dtype)) + half(dtype) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - want).abs()
    assert got.shape == want.shape
    assert bool((off <= limit).all()), f"off by {float((off - limit).max())} more than allowed, {int((~(off <= limit)).sum())} of {off.numel()}"


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ----------------------------------------------------------------------------- RMS norm
def norm_64(x, weight, eps, residual, gy, gh):
    """Values and bounds of (y, h, gx, gw)."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    wide, D = h.double(), x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.double().cpu()
    wide = wide.cpu()
    rstd = 1 / torch.sqrt(wide.square().mean(-1, keepdim=True) + eps)
    hat = wide * rstd
    depth = 54 + D / 1024  # additions of a square: a thread's, its team's
    rel = depth / 2 + 6
    y = hat * w
    g = gy.double().cpu() * w
    mean = (g * hat).mean(-1, keepdim=True)
    gx = rstd * (g - hat * mean)
    gx_bound = rstd * (g.abs() * (rel + 4) + hat.abs() * (g * hat).abs().mean(-1, keepdim=True) * (2 * depth + 3 * rel + 8)) * U
    if gh is not None:
        gx = gx + gh.double().cpu()
        gx_bound = gx_bound + gx.abs() * U
    terms = (gy.double().cpu() * hat).reshape(-1, D)
    return (y, y.abs() * rel * U), h, (gx, gx_bound), (terms.sum(0), terms.abs().sum(0) * (len(terms) + rel) * U)


# one value, odd widths, a vector, one below and above the teams' limits, several rows a team
NORM = [(1, 1), (3, 2), (5, 7), (2, 8), (33, 96), (9, 255), (7, 256), (4, 257), (70, 784), (3, 1024), (5, 1032), (2, 2051), (3, 4096), (2, 8200), (1, 33000), (300, 16)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("rows,D", NORM)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(device, rows, D, dtype, residual):
    g = gen(rows + D)
    x, gy, gh = (torch.randn(rows, D, generator=g).to(dtype) for _ in range(3))
    r = (2 * torch.randn(rows, D, generator=g)).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    (y, y_bound), h, (gx, gx_bound), (gw, gw_bound) = norm_64(x, w, 1e-6, r, gy, gh if residual else None)
    leaves = [t.to(device).requires_grad_() for t in (x, w, r) if t is not None]
    out = ops.rms_norm(leaves[0], leaves[1], residual=leaves[2] if residual else None)
    outs = list(out) if residual else [out]
    close(outs[0], y, y_bound, dtype)
    if residual:
        assert torch.equal(outs[1].cpu(), h)
    grads = torch.autograd.grad(outs, leaves, [gy.to(device), gh.to(device)][:len(outs)])
    close(grads[0], gx, gx_bound, dtype)
    close(grads[1], gw, gw_bound, dtype)
    if residual:
        assert torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_rms_norm_of_zeros_of_strangers_and_of_nothing(device):
    x = torch.zeros(4, 24)
    x[1, 5], x[2, 3] = math.inf, math.nan
    x[3] = 2.0
    y = ops.rms_norm(x.to(device), None, eps=1e-6).cpu()
    assert not y[0].any() and y[1, 5].isnan() and y[2].isnan().all()
    close(y[3], torch.full((24,), 1 / math.sqrt(1 + 1e-6 / 4)), torch.full((24,), 40 * U), torch.float32)
    assert ops.rms_norm(torch.zeros(2, 5, device=device), None, eps=0.0).isnan().all()  # zero over zero
    for shape in ((0, 24), (3, 0, 24)):
        leaf = torch.zeros(shape, device=device).requires_grad_()
        y, h = ops.rms_norm(leaf, None, residual=torch.zeros(shape, device=device))
        assert y.shape == h.shape == shape and torch.autograd.grad(y.sum(), leaf)[0].shape == shape
    codes, scale = ops.quantize_rows(torch.zeros(0, 24, device=device))
    assert codes.shape == (0, 24) and scale.shape == (0,)
    one = ops.rms_norm(torch.full((24,), 3.0, device=device))  # a row without a batch
    assert one.shape == (24,)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_rms_norm_gradients_of_some_inputs_and_results(device):
    """Only one of the results reaches the loss; only some inputs ask; the weight in another type; none."""
    g = gen(9)
    x, r, gy, gh = (torch.randn(2, 5, 40, generator=g).bfloat16() for _ in range(4))
    w = 1 + 0.2 * torch.randn(40, generator=g)
    for used in ("y", "h", "both"):
        a, b = x.to(device).requires_grad_(), r.to(device).requires_grad_()
        y, h = ops.rms_norm(a, w.to(device), residual=b)
        zero = torch.zeros_like(gy)
        _, _, (gx, bound), _ = norm_64(x, w, 1e-6, r, gy if used != "h" else zero, gh if used != "y" else zero)
        outs = {"y": [y], "h": [h], "both": [y, h]}[used]
        grads = torch.autograd.grad(outs, [a, b], {"y": [gy], "h": [gh], "both": [gy, gh]}[used] if device == "cpu" else
                                    [t.cuda() for t in {"y": [gy], "h": [gh], "both": [gy, gh]}[used]])
        for got in grads:
            close(got, gx, bound, torch.bfloat16)
    weight = w.to(device).requires_grad_()
    y = ops.rms_norm(x.to(device), weight)
    got, = torch.autograd.grad(y, weight, gy.to(device))
    _, _, _, (gw, bound) = norm_64(x, w, 1e-6, None, gy, None)
    close(got, gw, bound, torch.float32)
    b = r.to(device).requires_grad_()
    y, h = ops.rms_norm(x.to(device), None, residual=b)
    got, = torch.autograd.grad(y, b, gy.to(device))
    _, _, (gx, bound), _ = norm_64(x, None, 1e-6, r, gy, None)
    close(got, gx, bound, torch.bfloat16)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_rms_norm_strides(device):
    """Rows apart, a start off a vector's boundary, a transposed matrix, an expanded gradient."""
    g = gen(4)
    wide = torch.randn(20, 64, generator=g)
    for cut in (lambda t: t[:, 8:40], lambda t: t[:, 3:35], lambda t: t.t()[:32, :16], lambda t: t[::2, :32], lambda t: t[:1, 4:36], lambda t: t[:, None, ::2]):
        base = wide.clone().to(device).requires_grad_()
        x = cut(base)
        gy = torch.randn(x.shape[-1], generator=g)
        y, h = ops.rms_norm(x, None, residual=cut(wide.to(device) * 2))
        (want, bound), _, (gx, gx_bound), _ = norm_64(cut(wide), None, 1e-6, cut(wide * 2), gy.expand(x.shape), None)
        close(y, want, bound, torch.float32)
        grad, = torch.autograd.grad(y, base, gy.to(device).expand(x.shape))
        close(cut(grad), gx, gx_bound, torch.float32)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("rows,D", [(1, 1), (5, 7), (33, 96), (70, 784), (3, 2051), (2, 33000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_in_8_bits(device, rows, D, dtype):
    g = gen(rows * D)
    x, r, w = torch.randn(rows, D, generator=g).to(dtype), torch.randn(rows, D, generator=g).to(dtype), (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)
    x[0, 0] = 0.0
    (y, y_bound), h, _, _ = norm_64(x, w, 1e-6, r, x, None)
    for got, want, bound in ((ops.rms_norm_codes(x.to(device), w.to(device), residual=r.to(device)), y, y_bound),
                             (ops.quantize_rows(x.to(device)), x.double(), torch.zeros(rows, D))):
        codes, scale = got[0], got[1]
        assert codes.dtype is torch.float8_e4m3fn and codes.shape == (rows, D) and scale.dtype is torch.float32 and scale.shape == (rows,)
        most = want.abs().amax(1)
        close(scale, most / 448, bound.amax(1) / 448 + most / 448 * U, torch.float32)
        s = scale.cpu().double()[:, None]
        # off by the code's half step, and by the quotient's roundings
        step = torch.maximum(want.abs() * E4M3_HALF, s * E4M3_LEAST)
        assert bool(((codes.cpu().double() * s - want).abs() <= (step + bound) * (1 + 8 * U) + want.abs() * 4 * U).all())
        assert bool((codes.cpu().double().abs().amax(1) == 448).all() | (most == 0).any())
    assert torch.equal(ops.rms_norm_codes(x.to(device), w.to(device), residual=r.to(device))[2].cpu(), h)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_rows_in_8_bits_of_zeros_and_strangers(device):
    x = torch.zeros(4, 32)
    x[1, 3], x[2, 7], x[3, 0] = math.nan, math.inf, 1e-30
    x[2, 8] = 1.0
    codes, scale = ops.quantize_rows(x.to(device))
    codes, scale = codes.cpu().float(), scale.cpu()
    assert not codes[0].any() and scale[0] == 0
    assert scale[1].isnan() and codes[1].isnan().all()
    assert scale[2] == math.inf and codes[2, 7].isnan() and codes[2, 8] == 0
    assert codes[3, 0] == 448 and not codes[3, 1:].any()


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [3, 32, 785, 33000])
def test_rows_in_8_bits_of_very_small_values(device, dtype, D):
    """From rows whose scale has no reciprocal in float32 down to its smallest subnormal; zeros among them stay zeros, other rows as they are."""
    g = gen(D)
    most = torch.tensor([1.0, 1e-28, 1e-30, 5e-34, 2e-36, 1.3e-36, 1e-36, 1e-37, 2.0 ** -126, 1e-39, 2.0 ** -133, 700 * 2.0 ** -149, 2.0 ** -140, 2.0 ** -149, 0.0])
    shape = torch.rand(len(most), D, generator=g) * 2 - 1
    shape[:, 0], shape[:, 1:2], shape[:, 2] = 1.0, 0.0, -0.5
    x = (shape.double() * most[:, None].double()).to(dtype)
    weight = torch.tensor([1.0, 0.5] * D)[:D]
    w = (1e-37 * weight).to(dtype)  # the norm's: a weight that has decayed
    y = x[:1].double() / torch.sqrt(x[:1].double().square().mean() + 1e-6) * w.double()
    for got, want, rel in ((ops.quantize_rows(x.to(device)), x.double(), 0.0), (ops.rms_norm_codes(x[:1].to(device), w.to(device)), y, (54 + D / 1024) / 2 + 6)):
        codes, scale = got[0].cpu().double(), got[1].cpu().double()
        assert bool(codes.isfinite().all())
        top = want.abs().amax(1)
        # the scale is off by its rounding, of a subnormal 2^-150; (rel + 1) 2^-150: what came out as a subnormal itself
        least = (1 + (rel > 0)) * 2.0 ** -150
        assert bool(((scale - top / 448).abs() <= (rel + 1) * U * top / 448 + least).all())
        s = scale[:, None]
        # values beyond 448 of a scale that was rounded down are off by 448 times what that was
        step = torch.maximum(want.abs() * E4M3_HALF, s * E4M3_LEAST)
        limit = step * (1 + 8 * U) + want.abs() * (rel + 4) * U + (448 + 2) * least
        assert bool(((codes * s - want).abs() <= limit).all())
        assert not codes[want == 0].any()
        if dtype is torch.float32 and rel == 0.0:
            assert bool((codes.abs().amax(1) == 448)[top >= 1e-30].all())
    # a row of a weight that has decayed: its column is next to nothing, the others are as they were
    full = torch.randn(6, D, generator=g).to(dtype)
    gone = full.clone()
    gone[2] = x[7, :D]
    rows = torch.randn(5, D, generator=g).to(dtype).to(device)
    want, got = (ops.linear_codes(*ops.quantize_rows(rows), *ops.quantize_rows(t.to(device)), dtype=torch.float32) for t in (full, gone))
    assert bool(got[:, 2].isfinite().all()) and float(got[:, 2].abs().max()) < 1e-30
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(got[:, keep], want[:, keep])


# ----------------------------------------------------------------------------- projections
def act_64(z, act):
    """Value, slope, and a bound of the slope's slope"""
    s = torch.sigmoid(z)
    return {"none": lambda: (z, torch.ones_like(z), 0.0), "relu": lambda: (z.clamp(min=0), (z > 0).double(), 0.0),
            "sigmoid": lambda: (s, s * (1 - s), 0.1), "silu": lambda: (z * s, s * (1 + z * (1 - s)), 0.5)}[act]()


def linear_64(x, w, b, r, act, gated, gy):
    """[(value, bound)] of y, gx, gw, gb."""
    dtype = x.dtype
    h = half(dtype)
    x, w, gy = x.double(), w.double(), gy.double()
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    times = 6 if dtype is torch.float32 else 1  # products of planes, each a sum

    def product(a, at_a, c, at_c):  # a c with what a and c are off by
        return a @ c, at_a @ c.abs() + a.abs() @ at_c + (a.abs() @ c.abs()) * (2 * (times * a.shape[1] + 16) * U)

    z, z_off = product(x, torch.zeros_like(x), w.t(), torch.zeros_like(w.t()))
    if b is not None:
        z = z + b.double()
        z_off = z_off + z.abs() * U
    zk_off = z_off + z.abs() * (0.0 if dtype is torch.float32 else 2.0 ** -16)  # as it is kept: 24 bits of a float, 16 of them the value's

    def followed(t, off):
        value, slope, curve = act_64(t, act)
        jump = (t.abs() <= off + 2.0 ** -24) if act == "relu" else torch.zeros_like(t)  # (float16's smallest)
        v_off = (slope.abs() + curve * off) * off + value.abs() * (t.abs() * 2 + 8) * U
        s_off = curve * off + jump + (2 * t.abs() + 12) * (1 + t.abs()) * U * (act not in ("none", "relu"))
        return value, v_off, slope, s_off

    if gated:
        F = N // 2
        a, a_off, _, _ = followed(z[:, :F], z_off[:, :F])
        u, u_off = z[:, F:], z_off[:, F:]
        y, y_off = a * u, a_off * u.abs() + a.abs() * u_off + a_off * u_off + (a * u).abs() * U
        a, a_off, s, s_off = followed(z[:, :F], zk_off[:, :F])
        u_off = zk_off[:, F:]
        up = gy * a
        gate = gy * u * s
        gz = torch.cat([gate, up], 1)
        off = torch.cat([gy.abs() * (u.abs() * s_off + u_off * s.abs() + u_off * s_off), gy.abs() * a_off], 1)
    else:
        y, y_off, _, _ = followed(z, z_off)
        _, _, s, s_off = followed(z, zk_off)
        gz, off = gy * s, gy.abs() * s_off
    if r is not None:
        y = y + r.double()
        y_off = y_off + y.abs() * U
    off = off + gz.abs() * 3 * U
    gb = gz.sum(0), off.sum(0) + (gz.abs() + off).sum(0) * (M + 2) * U
    if gated or act != "none":
        off = off + (gz.abs() + off) * h
    off = off + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    gx = product(gz, off, w, torch.zeros_like(w))
    gw = product(gz.t(), off.t(), x, torch.zeros_like(x))
    return (y, y_off), gx, gw, gb


def check_linear(device, M, K, N, dtype, act, gated, bias, residual, grads=True):
    g = gen(M + K + N)
    x, w = torch.randn(M, K, generator=g).to(dtype), (torch.randn(N, K, generator=g) / math.sqrt(K)).to(dtype)
    b = (0.5 * torch.randn(N, generator=g)).to(dtype) if bias else None
    out = N // 2 if gated else N
    r = torch.randn(M, out, generator=g).to(dtype) if residual else None
    gy = torch.randn(M, out, generator=g).to(dtype)
    move = [None if t is None else t.to(device) for t in (x, w, b, r, gy)]
    (y, y_off), *wants = linear_64(*move[:4], act, gated, move[4])
    leaves = [None if t is None else t.requires_grad_() for t in move[:4]]
    got = (ops.gated_linear if gated else ops.linear)(*leaves[:3], activation=act, residual=leaves[3])
    assert got.dtype is dtype and got.shape == (M, out)
    close(got, y, y_off, dtype)
    if not grads:
        return
    asked = [t for t in leaves if t is not None]
    result = list(torch.autograd.grad(got, asked, move[4]))
    for (want, off), leaf in zip(wants, leaves[:3]):
        if leaf is not None:
            close(result.pop(0), want, off, dtype)
    if residual:
        assert torch.equal(result.pop(0), move[4])


# one value, less than a unit, units and half units, tiles and a little more, several stages, a long reduction, few rows
LINEAR = [(1, 1, 2), (1, 8, 8), (2, 16, 6), (3, 7, 10), (5, 64, 34), (17, 100, 40), (1, 512, 300), (9, 1000, 130), (33, 264, 514), (64, 128, 256),
          (130, 257, 130), (129, 72, 520), (300, 40, 16), (257, 520, 258), (16, 2048, 64), (700, 24, 24)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("M,K,N", LINEAR)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,bias,residual", [("none", False, False), ("sigmoid", True, True), ("relu", True, False), ("silu", False, True)])
def test_linear(device, M, K, N, dtype, act, bias, residual):
    check_linear(device, M, K, N, dtype, act, False, bias, residual)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("M,K,N", LINEAR)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,bias,residual", [("silu", False, False), ("sigmoid", True, True), ("none", True, False)])
def test_gated_linear(device, M, K, N, dtype, act, bias, residual):
    check_linear(device, M, K, N, dtype, act, True, bias, residual)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,dtype,gated", [
    (4100, 200, 4104, torch.bfloat16, False), (4100, 200, 4104, torch.bfloat16, True), (4101, 129, 4098, torch.float16, True),
    (5000, 72, 4000, torch.float32, False), (4111, 64, 5002, torch.float32, True), (30011, 320, 200, torch.bfloat16, False),
    (9001, 1024, 512, torch.float16, True), (20000, 48, 96, torch.float32, False), (513, 4096, 1030, torch.bfloat16, True), (70001, 16, 24, torch.bfloat16, False)])
def test_linear_of_many_tiles(M, K, N, dtype, gated):
    check_linear("cuda", M, K, N, dtype, "silu", gated, True, True)


# few rows, small tiles, a split reduction, gated tiles, large tiles
HUGE = [pytest.param("cpu", 3, 72, 40), pytest.param("cpu", 40, 72, 130)] + [
    pytest.param("cuda", *s, marks=pytest.mark.gpu) for s in ((3, 72, 40), (32, 640, 514), (100, 72, 300), (300, 2080, 514), (1100, 96, 2050), (4100, 72, 4104))]


@pytest.mark.parametrize("device,M,K,N", HUGE)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_of_the_lowest_value_times_nothing(device, M, K, N, gated):
    """A mask of the type's lowest (or largest) value in front of weights of zero adds nothing, whichever operand holds it."""
    g = gen(M + N)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) / math.sqrt(K)
    f = ops.gated_linear if gated else ops.linear
    for value in (torch.finfo(torch.float32).min, torch.finfo(torch.float32).max):
        for k in (0, 37, K - 1):
            xs, ws = x.clone(), w.clone()
            xs[:, k], ws[:, k] = 0.0, 0.0
            want = f(xs.to(device), ws.to(device), activation="silu")
            for masked, other in ((xs, ws), (ws, xs)):
                a = masked.clone()
                a[1::2, k] = value
                assert torch.equal(f(*(t.to(device) for t in ((a, other) if masked is xs else (other, a))), activation="silu"), want)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(32, 640, 514), (300, 72, 300), (300, 2080, 514), (4100, 72, 4104)])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_of_one_largest_value_wherever_it_stands(M, K, N, gated):
    """In any row of a tile of either operand: nothing but its product with zero comes of it."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x, w = torch.randn(M, K, device="cuda", generator=g), torch.randn(N, K, device="cuda", generator=g) / math.sqrt(K)
    f = ops.gated_linear if gated else ops.linear
    k = 41
    x[:, k], w[:, k] = 0.0, 0.0
    want = f(x, w)
    same = torch.ones((), dtype=torch.bool, device="cuda")
    for t in (x, w):
        for r in [*range(min(300, t.shape[0])), t.shape[0] - 1]:
            t[r, k] = torch.finfo(torch.float32).max
            same &= (f(x, w) == want).all()
            t[r, k] = 0.0
    assert bool(same)


@pytest.mark.parametrize("device,M,K,N", HUGE)
@pytest.mark.parametrize("where", ["x", "w", "gy"])
def test_linear_of_values_up_to_the_largest(device, M, K, N, where):
    """Float32 above the largest bfloat16 here and there, next to small ones: results and gradients within the bounds of any other value."""
    g = gen(M * 3 + N)
    most = torch.finfo(torch.float32).max
    values = torch.tensor([most, -most, 2.0 ** 128 - 2.0 ** 119, -(2.0 ** 128 - 2.0 ** 119), 2.0 ** 128 - 2.0 ** 119 - 2.0 ** 104, 2.0 ** 128 - 2.0 ** 120, 3e38, 1e38])
    t = {"x": torch.randn(M, K, generator=g), "w": torch.randn(N, K, generator=g), "gy": torch.randn(M, N, generator=g)}
    for name in t:
        t[name] *= 1e-4
    some = torch.rand(t[where].shape, generator=g) < 0.02
    some[1, 1] = True
    t[where] = torch.where(some, values[torch.randint(0, len(values), t[where].shape, generator=g)], t[where])
    x, w, gy = (v.to(device) for v in t.values())
    (y, y_off), gx, gw, _ = linear_64(x, w, None, None, "none", False, gy)
    x.requires_grad_(), w.requires_grad_()
    got = ops.linear(x, w)
    close(got, y, y_off, torch.float32)
    for grad, (want, off) in zip(torch.autograd.grad(got, (x, w), gy), (gx, gw)):
        assert float(want.abs().max()) < most
        close(grad, want, off, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,dtype,act", [(2, 1, 1 << 21, torch.float32, "none"), (3, 2, 1 << 22, torch.bfloat16, "silu"), ((1 << 22) + 5, 8, 8, torch.bfloat16, "silu"), ((1 << 22) + 5, 3, 2, torch.float32, "none")])
def test_linear_up_to_its_limits(M, K, N, dtype, act):
    """The longest rows that have a backward, and more rows than that."""
    check_linear("cuda", M, K, N, dtype, act, False, True, False)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(5, 40), (5, 8), (70, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("far", ["x", "w"])
def test_linear_of_rows_far_apart(M, N, dtype, far):
    """Some columns of a matrix with rows of more than 2^23 bytes: forward and backward, of few rows and by tiles."""
    g = gen(M + N)
    D, K = (1 << 23) // dtype.itemsize + 64, 64
    x, w, gy = torch.randn(M, K, generator=g).to(dtype).cuda(), (torch.randn(N, K, generator=g) / 8).to(dtype).cuda(), torch.randn(M, N, generator=g).to(dtype).cuda()
    wide = torch.empty(M if far == "x" else N, D, dtype=dtype, device="cuda")
    cut = wide[:, 128:128 + K]
    cut.copy_(x if far == "x" else w)
    (y, y_off), gx, gw, _ = linear_64(x, w, None, None, "none", False, gy)
    leaves = [t.requires_grad_() for t in ((cut.detach(), w) if far == "x" else (x, cut.detach()))]
    got = ops.linear(*leaves)
    close(got, y, y_off, dtype)
    for grad, (want, off) in zip(torch.autograd.grad(got, leaves, gy), (gx, gw)):
        close(grad, want, off, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,gated", [("none", False), ("silu", False), ("sigmoid", True)])
def test_linear_of_rows_without_a_backward(dtype, act, gated):
    """Refused by the call itself where gradients are asked for; without them, and of the residual's alone, it runs."""
    N = (1 << 23) // dtype.itemsize + 2
    g = gen(7)
    x, w = torch.randn(2, 3, generator=g).to(dtype).cuda(), torch.randn(N, 3, generator=g).to(dtype).cuda()
    f = ops.gated_linear if gated else ops.linear
    (y, y_off), *_ = linear_64(x, w, None, None, act, gated, torch.zeros(2, N // 2 if gated else N, device="cuda"))
    close(f(x, w, activation=act), y, y_off, dtype)
    b = torch.zeros(N, dtype=dtype, device="cuda")
    for leaves in ((x.clone().requires_grad_(), w, b), (x, w.clone().requires_grad_(), b), (x, w, b.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradients"):
            f(*leaves, activation=act)
        with torch.no_grad():
            close(f(*leaves, activation=act), y, y_off, dtype)
    r = torch.ones(2, N // 2 if gated else N, dtype=dtype, device="cuda").requires_grad_()
    out = f(x, w, activation=act, residual=r)
    assert torch.equal(torch.autograd.grad(out, r, torch.full_like(out, 2.0))[0], torch.full_like(out, 2.0))


# few rows: short and long reductions, rows of w shared by two wavefronts or eight, the last group inside a block, up to 16, 32 and 64 rows
@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,dtype,gated", [
    (1, 33, 70001, torch.bfloat16, False), (3, 100, 40000, torch.float16, False), (16, 96, 66000, torch.bfloat16, True), (5, 40, 33002, torch.float32, True),
    (20, 64, 70010, torch.float16, False), (32, 1000, 4098, torch.float32, False), (31, 77, 66002, torch.float32, False), (48, 300, 2050, torch.bfloat16, True),
    (64, 2047, 1030, torch.float16, True), (2, 4001, 17, torch.bfloat16, False), (16, 8200, 40, torch.float32, False), (1, 1, 50000, torch.float32, False)])
def test_linear_of_few_rows(M, K, N, dtype, gated):
    check_linear("cuda", M, K, N // 2 * 2 if gated else N, dtype, "sigmoid" if gated else "silu", gated, True, True)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(5, 64, 34), (40, 72, 514), (130, 257, 130), (300, 129, 2050), (4100, 200, 4104), (4101, 130, 4098), (9001, 64, 512)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "sigmoid"])
def test_linear_of_inference_is_that_of_training(M, K, N, dtype, gated, act):
    """Kernels that keep nothing for a backward give the same bits."""
    g = torch.Generator(device="cuda").manual_seed(M + K)
    x, w, b = (torch.randn(s, device="cuda", generator=g).to(dtype) for s in ((M, K), (N, K), (N,)))
    r = torch.randn(M, N // 2 if gated else N, device="cuda", generator=g).to(dtype)
    f = ops.gated_linear if gated else ops.linear
    for bias, residual in ((b, r), (None, None)):
        with torch.no_grad():
            want = f(x, w, bias, activation=act, residual=residual)
        assert torch.equal(f(x, w.detach().requires_grad_(), bias, activation=act, residual=residual), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_two_streams_at_once(dtype):
    """The same operators on other data on two streams, turn by turn without waiting, are those of one after the other."""
    p = block_parameters(dtype, "cuda")
    data = []
    for seed in (1, 2):
        g = gen(seed)
        data.append(([torch.randn(1500, 64, generator=g).to(dtype).cuda() for _ in range(3)], torch.randn(4, 6, 20001, generator=g).to(dtype).cuda()))

    def everything(d):
        (x, r, gy), logits = d
        y = block_step(p, x, r)
        grads = torch.autograd.grad(y, list(p.values()), gy)
        step = ops.beam_step(logits, torch.zeros(4, 6, device="cuda"))
        return [y, *grads, *step, *ops.beam_reorder([logits], step[1])]

    want = [everything(d) for d in data]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in data], [[], []]
    for _ in range(3):
        for k, (s, d) in enumerate(zip(streams, data)):
            with torch.cuda.stream(s):
                got[k].append(everything(d))
    torch.cuda.synchronize()
    for a, runs in zip(want, got):
        for b in runs:
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("M,K,N", [(40, 100, 60), (300, 129, 257), (3, 640, 1000), (1, 24, 7)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_of_whole_numbers_is_exact(device, M, K, N, dtype, gated):
    """Small whole numbers: products, sums and results are exact in every type, whatever the order."""
    g = gen(M * K)
    N = N // 2 * 2
    out = N // 2 if gated else N
    x, w = torch.randint(-1, 2, (M, K), generator=g), torch.randint(-1, 2, (N, K), generator=g) * (torch.rand(N, K, generator=g) < 8 / K)
    b, gy = torch.randint(-1, 2, (N,), generator=g), torch.randint(-1, 2, (M, out), generator=g) * (torch.rand(M, out, generator=g) < min(1, 8 / max(M, out)))
    leaves = [t.to(dtype).to(device).requires_grad_() for t in (x, w, b)]
    z = x @ w.t() + b
    y = (ops.gated_linear if gated else ops.linear)(*leaves, activation="none")
    want = z[:, :out] * z[:, out:] if gated else z
    fits = want.abs() <= 256
    assert torch.equal(y.cpu().double()[fits], want.double()[fits])
    gz = torch.cat([gy * z[:, out:], gy * z[:, :out]], 1) if gated else gy
    for got, want in zip(torch.autograd.grad(y, leaves, gy.to(dtype).to(device)), (gz @ w, gz.t() @ x, gz.sum(0))):
        fits = want.abs() <= 256
        assert torch.equal(got.cpu().double()[fits], want.double()[fits])


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_linear_float32_products_keep_24_bits(device):
    """One product per result: off by the roundings of six plane products' additions (two half steps each) and of the rest left out."""
    g = gen(12)
    n = 200
    d = torch.randn(n, generator=g) * torch.exp(4 * torch.randn(n, generator=g))
    w = torch.randn(150, n, generator=g) * torch.exp(4 * torch.randn(150, n, generator=g))
    got = ops.linear(torch.diag(d).to(device), w.to(device)).cpu().double()
    want = d.double()[:, None] * w.double().t()
    assert bool(((got - want).abs() <= 14 * U * want.abs()).all())


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("gated", [False, True])
def test_linear_strides(device, gated):
    """Leading dimensions, rows apart, starts off a unit's boundary, a transposed weight, an expanded gradient, a sliced residual."""
    g = gen(7)
    f = ops.gated_linear if gated else ops.linear
    for dtype in (torch.float32, torch.bfloat16):
        wide, wide_w = torch.randn(24, 80, generator=g).to(dtype), (torch.randn(60, 80, generator=g) / 8).to(dtype)
        for cx, cw in ((lambda t: t[:, 8:72], lambda t: t[:40, 16:80]), (lambda t: t[:, 3:67], lambda t: t[::2, 1:65][:20]), (lambda t: t[::2, :64], lambda t: t[:40, :64]),
                       (lambda t: t.t()[:64, :24], lambda t: t.t()[:40, :24]), (lambda t: t[:, None, :64], lambda t: t[:1, :64].expand(8, 64)), (lambda t: t[3, 5:69], lambda t: t[:8, 5:69])):
            bx, bw = wide.clone().to(device).requires_grad_(), wide_w.clone().to(device).requires_grad_()
            x, w = cx(bx), cw(bw)
            out = w.shape[0] // 2 if gated else w.shape[0]
            r = torch.randn(*x.shape[:-1], out + 3, generator=g).to(dtype)[..., 2:2 + out]
            gy = torch.randn(out, generator=g).to(dtype)
            y = f(x, w, residual=r.to(device), activation="silu")
            rows = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
            (want, off), (gx, gx_off), (gw, gw_off), _ = linear_64(rows(cx(wide)), cw(wide_w), None, rows(r), "silu", gated, gy.expand(rows(r).shape))
            assert y.shape == (*x.shape[:-1], out)
            close(rows(y), want, off, dtype)
            got_x, got_w = torch.autograd.grad(y, [x, w], gy.to(device).expand(y.shape))
            close(rows(got_x), gx, gx_off, dtype)
            close(got_w, gw, gw_off, dtype)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_linear_of_no_rows_and_gradients_of_some_inputs(device):
    x, w, b = torch.zeros(0, 16, device=device).requires_grad_(), torch.ones(6, 16, device=device).requires_grad_(), torch.ones(6, device=device).requires_grad_()
    y = ops.linear(x, w, b, activation="silu")
    grads = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == (0, 6) and grads[0].shape == (0, 16) and not grads[1].any() and not grads[2].any()
    assert ops.gated_linear(torch.zeros(2, 0, 16, device=device), w).shape == (2, 0, 3)
    g = gen(1)
    x, w, b, r, gy = (torch.randn(s, generator=g) for s in ((9, 16), (6, 16), (6,), (9, 6), (9, 6)))
    wants = linear_64(x, w, b, r, "sigmoid", False, gy)[1:]
    for k in range(3):
        leaves = [t.to(device) for t in (x, w, b, r)]
        leaves[k].requires_grad_()
        got, = torch.autograd.grad(ops.linear(*leaves[:3], activation="sigmoid", residual=leaves[3]), leaves[k], gy.to(device))
        close(got, *wants[k], torch.float32)
    r = r.to(device).requires_grad_()
    got, = torch.autograd.grad(ops.linear(x.to(device), w.to(device), residual=r), r, gy.to(device))
    assert torch.equal(got.cpu(), gy)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_leaves_other_rows_alone_where_one_is_not_finite(device, dtype):
    g = gen(2)
    x, w = torch.randn(150, 70, generator=g).to(dtype), torch.randn(36, 70, generator=g).to(dtype)
    y = ops.linear(x.to(device), w.to(device))
    x[3, 5], x[140, 69] = math.nan, math.inf
    z = ops.linear(x.to(device), w.to(device))
    others = [i for i in range(150) if i not in (3, 140)]
    assert torch.equal(y[others], z[others]) and z[3].isnan().all() and not z[140].isfinite().any()


def test_gradients_against_differences():
    g = gen(3)
    x, r, w, n = (torch.randn(s, dtype=torch.float64, generator=g).requires_grad_() for s in ((3, 6), (3, 4), (8, 6), (6,)))
    b = torch.randn(8, dtype=torch.float64, generator=g).requires_grad_()
    for act in ("silu", "sigmoid"):
        assert torch.autograd.gradcheck(lambda *t: ops.gated_linear(t[0], t[1], t[2], act, t[3]), (x, w, b, r))
        assert torch.autograd.gradcheck(lambda *t: ops.linear(t[0], t[1], t[2], act), (x, w, b))
    other = torch.randn(3, 6, dtype=torch.float64, generator=g).requires_grad_()
    assert torch.autograd.gradcheck(lambda *t: ops.rms_norm(t[0], t[1], 1e-3, t[2]), (x, n, other))


# ----------------------------------------------------------------------------- projections on 8-bit rows
def coded(shape, g, std=1.0):
    return ops.quantize_rows(std * torch.randn(shape, generator=g))


def cut_64(x, w):
    """What the 8-bit matrix cores' sums may leave out.  They add the products of a step of 64 to the place of the largest, with 13 bits behind
    its leading one: 2^16 + 2^3 is exact, of 2^16 + 2^2 the second is gone (and 2^16 + 2^-7 is exact again where the two are
    not in one sum).  So a product is off by less than 2^-13 of the step's largest, a step by less than 64 times that."""
    return sum(64 * 2.0 ** -13 * (x[:, None, k:k + 64] * w[None, :, k:k + 64]).abs().amax(2) for k in range(0, x.shape[1], 64))


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("M,K,N", [(1, 1, 2), (1, 16, 8), (3, 7, 10), (5, 128, 34), (17, 100, 40), (33, 1040, 514), (130, 257, 130), (1, 2048, 300), (300, 144, 24)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,gated,extras", [("none", False, False), ("silu", True, True), ("sigmoid", False, True)])
def test_linear_codes(device, M, K, N, dtype, act, gated, extras):
    g = gen(M + K + N)
    (x, sx), (w, sw) = coded((M, K), g), coded((N, K), g, 1 / math.sqrt(K))
    out = N // 2 if gated else N
    b, r = ((torch.randn(s, generator=g).to(dtype)) if extras else None for s in ((N,), (M, out)))
    move = [None if t is None else t.to(device) for t in (x, sx, w, sw, b, r)]
    y = ops.linear_codes(*move[:5], activation=act, residual=move[5], gated=gated, dtype=dtype)
    wide_x, wide_w = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
    (want, off), *_ = linear_64(wide_x, wide_w, b, r, act, gated, torch.zeros(M, out))
    size = wide_x.abs() @ wide_w.abs().t() * 4 * U + cut_64(wide_x, wide_w)  # the scales' roundings, and what the sums leave out
    size = size[:, :out] + size[:, out:] if gated else size
    other = 1.0 if not gated else 1 + (wide_x @ wide_w.t() + (0 if b is None else b.double())).abs().amax()
    close(y, want, off + size * other, dtype)
    z = ops.linear_codes(*move[:5], activation=act, residual=move[5], gated=gated, dtype=dtype)
    assert torch.equal(y, z)


@pytest.mark.gpu
def test_linear_codes_of_many_tiles_and_strides():
    g = gen(4)
    (x, sx), (w, sw) = (tuple(t.cuda() for t in coded(s, g)) for s in ((4200, 300), (4300, 300)))
    for k0, k1 in ((0, 272), (16, 288), (5, 300)):  # whole units, the same further on, neither
        a, c = x[:, k0:k1], w[:, k0:k1]
        y = ops.linear_codes(a, sx, c, sw, dtype=torch.float32)
        wide, wide_w = a.double() * sx.double()[:, None], c.double() * sw.double()[:, None]
        cut = torch.cat([cut_64(part, wide_w) for part in wide.split(64)])
        close(y, wide @ wide_w.t(), (wide.abs() @ wide_w.abs().t()) * (2 * (k1 - k0 + 16) + 4) * U + cut, torch.float32)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_linear_codes_of_strangers(device):
    """A row of zeros has scale 0, a row with a NaN stays one."""
    x = torch.ones(3, 32)
    x[0], x[1, 4] = 0.0, math.nan
    codes, scale = ops.quantize_rows(x.to(device))
    w, sw = ops.quantize_rows(torch.ones(8, 32, device=device))
    y = ops.linear_codes(codes, scale, w, sw, dtype=torch.float32).cpu()
    assert not y[0].any() and y[1].isnan().all()
    close(y[2], torch.full((8,), 32.0), torch.full((8,), 32 * 40 * U), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,dtype,gated", [(1, 5000, 40000, torch.bfloat16, False), (7, 100, 33000, torch.float32, True), (30, 260, 4100, torch.float16, False), (60, 512, 2052, torch.bfloat16, True),
                                               (4200, 144, 4230, torch.bfloat16, True), (4200, 128, 4224, torch.float16, False)])
def test_linear_codes_of_few_and_many_rows(M, K, N, dtype, gated):
    g = gen(M + N)
    (x, sx), (w, sw) = (tuple(t.cuda() for t in coded(s, g, d)) for s, d in (((M, K), 1.0), ((N, K), 1 / math.sqrt(K))))
    out = N // 2 if gated else N
    b, r = torch.randn(N, generator=g).to(dtype).cuda(), torch.randn(M, out, generator=g).to(dtype).cuda()
    y = ops.linear_codes(x, sx, w, sw, b, "silu", r, gated, dtype)
    wide, wide_w = x.double() * sx.double()[:, None], w.double() * sw.double()[:, None]
    for rows in range(0, M, 600):  # (in pieces: what the sums leave out is a number for every product of a step)
        part = slice(rows, min(M, rows + 600))
        (want, off), *_ = linear_64(wide[part], wide_w, b, r[part], "silu", gated, torch.zeros(part.stop - part.start, out, device="cuda"))
        size = wide[part].abs() @ wide_w.abs().t() * 4 * U + torch.cat([cut_64(q, wide_w) for q in wide[part].split(8)])
        size = size[:, :out] + size[:, out:] if gated else size
        other = 1.0 if not gated else 1 + (wide[part] @ wide_w.t() + b.double()).abs().amax()
        close(y[part], want, off + size * other, dtype)


# ----------------------------------------------------------------------------- beam search
def beam_64(logits, scores, beams, finished, end):
    """Every continuation, sorted: numpy, in doubles."""
    x, s = logits.double().cpu().numpy().copy(), scores.double().cpu().numpy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    B, K, V = x.shape
    out = []
    for b in range(B):
        found = []
        for k in range(K):
            if finished is not None and finished[b, k]:
                found.append((s[b, k], k, end))
                continue
            top = x[b, k].max()
            if top == -np.inf:
                continue
            norm = top + np.log(np.exp(x[b, k] - top).sum())
            best = np.argsort(-x[b, k], kind="stable")[:beams]
            found += [(s[b, k] + (x[b, k, v] - norm), k, v) for v in best]
        found = sorted((f for f in found if f[0] > -np.inf), key=lambda f: (-f[0], f[1], f[2]))[:beams]
        out.append(found + [(-np.inf, 0, -1)] * (beams - len(found)))
    return out


def check_beam(device, logits, scores, beams=None, finished=None, end=0):
    got = ops.beam_step(logits.to(device), scores.to(device), beams, None if finished is None else finished.to(device), end)
    count = logits.shape[1] if beams is None else beams
    want = beam_64(logits, scores, count, finished, end)
    B = logits.shape[0]
    assert all(t.shape == (B, count) for t in got) and got[0].dtype is torch.float32 and got[1].dtype is got[2].dtype is torch.int64
    value, parent, token = (torch.tensor([[f[i] for f in row] for row in want], dtype=torch.float64 if i == 0 else torch.int64).reshape(B, count) for i in range(3))
    assert torch.equal(got[1].cpu(), parent) and torch.equal(got[2].cpu(), token)
    live = value > -math.inf
    assert torch.equal(got[0].cpu() > -math.inf, live)
    # the log of a sum of exponentials, each off by its own ulps and by what its argument's rounding makes of it
    off = value.abs() * U + 40 * U
    assert bool(((got[0].cpu().double() - value).abs() <= off)[live].all())
    return got


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("B,K,V,beams", [(1, 1, 1, 1), (2, 3, 2, 8), (3, 4, 10, 4), (1, 64, 7, 64), (2, 5, 257, 5), (3, 8, 1000, 3), (1, 4, 4096, 4), (2, 4, 4097, 16), (1, 2, 30011, 64),
                                         (1, 16, 8200, 16), (40, 2, 520, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_beam_step(device, B, K, V, beams, dtype):
    g = gen(B * K + V)
    logits, scores = (3 * torch.randn(B, K, V, generator=g)).to(dtype), -5 * torch.rand(B, K, generator=g)
    check_beam(device, logits, scores, beams)
    ended = torch.rand(B, K, generator=g) < 0.4
    check_beam(device, logits, scores, beams, ended, end=V // 2)
    first = torch.full((B, K), -math.inf)
    first[:, 0] = 0.0
    check_beam(device, logits, first, beams)


@pytest.mark.gpu
@pytest.mark.parametrize("B,K,V,beams,dtype", [(2, 3, 131072, 8, torch.float32), (1, 16, 100003, 16, torch.bfloat16), (1, 1, 1 << 20, 64, torch.float16), (300, 4, 5000, 4, torch.float16)])
def test_beam_step_of_long_rows(B, K, V, beams, dtype):
    g = gen(V)
    logits, scores = (3 * torch.randn(B, K, V, generator=g)).to(dtype), -5 * torch.rand(B, K, generator=g)
    check_beam("cuda", logits, scores, beams)
    rising = torch.arange(V, dtype=torch.float32).expand(B, K, V) * (8.0 / V)  # every round passes the bound of the ones before
    check_beam("cuda", rising.to(dtype).contiguous(), scores, beams)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [5, 300, 5000, 20000])
def test_beam_step_equal_logits(device, V):
    """All equal, few distinct values, equal beams: by beam, then token."""
    g = gen(V)
    check_beam(device, torch.zeros(2, 3, V), torch.zeros(2, 3), 7)
    check_beam(device, torch.randint(0, 2, (2, 3, V), generator=g).float(), torch.zeros(2, 3), 16)
    same = torch.randint(0, 5, (1, 1, V), generator=g).half().expand(2, 4, V).contiguous()
    check_beam(device, same, torch.tensor([[0.0, 0.0, -1.0, 0.0], [-2.0, -2.0, -2.0, -2.0]]))
    check_beam(device, torch.tensor([0.0, -0.0]).repeat(V)[:V].expand(1, 2, V).contiguous(), torch.zeros(1, 2), 4)


# (beams in, vocabulary, answers): a piece of a row and several, few candidates and more than are ranked at once
@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("K,V,beams", [(4, 5, 16), (3, 700, 8), (2, 20001, 16), (4, 40000, 64), (64, 300, 64), (20, 9000, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_beam_step_scores_that_swallow_logits(device, K, V, beams, dtype):
    """Different logits, the same score as a double: by beam, then logit, then token."""
    g = gen(K + V)
    x = (3 * torch.randn(2, K, V, generator=g)).to(dtype)
    x[1, 0, V - 1] = x[1, 0].max()  # (twice: the lower token first)
    tiny = (torch.randn(2, K, V, generator=g) * 1e-20).to(dtype)  # all of one probability as a double
    mixed = torch.full((2, K), -1e30)
    mixed[:, 0], mixed[0, K - 1] = 0.0, -1e9
    ended = torch.zeros(2, K, dtype=torch.bool)
    ended[:, 1] = True
    for logits, scores, finished in [(x, torch.full((2, K), s), None) for s in (-1e30, -1e9, torch.finfo(torch.float32).min, math.inf)] + [
            (x, mixed, None), (x, mixed, ended), (tiny, torch.zeros(2, K), None), (tiny, torch.full((2, K), -1e30), ended)]:
        z, s = logits.double(), scores.double()
        c = s[:, :, None] + torch.log_softmax(z, 2)
        rank = torch.sort(z, dim=2, descending=True, stable=True).indices.argsort(2)  # of a beam's tokens
        if finished is not None:
            alone = torch.full_like(c, -math.inf)
            alone[:, :, 3] = s
            c = torch.where(finished[:, :, None], alone, c)
        place = rank + V * torch.arange(K)[None, :, None]
        got = ops.beam_step(logits.to(device), scores.to(device), beams, None if finished is None else finished.to(device), 3)
        for b in range(2):
            order = np.lexsort((place[b].flatten().numpy(), -c[b].flatten().numpy()))[:beams]
            assert got[1][b].tolist() == (order // V).tolist() and got[2][b].tolist() == (order % V).tolist()
            want = c[b].flatten()[order]
            assert bool(((got[0][b].cpu().double() - want).abs() <= want.abs() * U + 40 * U).logical_or(want == math.inf).all()) and torch.equal(got[0][b].cpu() == math.inf, want == math.inf)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [6, 700, 9001])
def test_beam_step_masked_rows(device, V):
    """Nothing left of a beam, of a sequence; one token left; infinities, NaN, the type's lowest value; scores that are no numbers."""
    g = gen(V + 1)
    x = torch.randn(5, 3, V, generator=g)
    x[0, 1] = -math.inf
    x[1] = -math.inf
    x[2, 0] = -math.inf
    x[2, 0, V - 1] = 0.5
    x[2, 1, ::2] = math.nan
    x[3, 0, 2], x[3, 1, 1], x[3, 1, 3] = math.inf, math.inf, math.inf
    x[4] = torch.finfo(torch.float32).min
    x[4, 1, 0] = -math.inf
    scores = -torch.rand(5, 3, generator=g)
    check_beam(device, x, scores, 3)
    check_beam(device, x, scores, 9)
    scores[0, 0], scores[2, 2] = -math.inf, math.nan
    got = ops.beam_step(x.to(device), scores.to(device))
    assert not (got[1][0] == 0).any() and not (got[1][2] == 2).any()
    got = ops.beam_step(x.to(device), torch.full((5, 3), -math.inf, device=device))
    assert bool((got[0] == -math.inf).all()) and bool((got[1] == 0).all()) and bool((got[2] == -1).all())
    x = torch.zeros(1, 2, V)
    x[0, :, 3:] = -1e4  # a mask of the exponential's nothing
    check_beam(device, x, torch.zeros(1, 2), 8 if V > 6 else 6)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_beam_step_strides_finished_and_empty(device):
    g = gen(6)
    wide, scores = torch.randn(4, 6, 90, generator=g), -torch.rand(4, 6, generator=g)
    for cut in (lambda t: t[:, :, 8:72], lambda t: t[:, :, 3:80], lambda t: t[:, ::2, :64], lambda t: t.transpose(0, 1)[:4, :4], lambda t: t[:1, 1:3]):
        x = cut(wide)
        s = scores[:x.shape[0], :x.shape[1]]
        got, want = ops.beam_step(cut(wide.to(device)), s.to(device)), beam_64(x, s, x.shape[1], None, 0)
        assert got[2].tolist() == [[int(f[2]) for f in row] for row in want]
    everything = torch.ones(4, 6, dtype=torch.bool)
    best, parents, tokens = ops.beam_step(torch.full((4, 6, 9), math.nan, device=device), scores.to(device), finished=everything.to(device), end=7)
    assert torch.equal(best.cpu(), scores.sort(dim=1, descending=True).values) and bool((tokens == 7).all())
    empty = ops.beam_step(torch.zeros(0, 3, 5, device=device), torch.zeros(0, 3, device=device))
    assert all(t.shape == (0, 3) for t in empty)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype", TYPES)
def test_beam_step_strides_of_one_beam(device, dtype):
    """One beam, one sequence, one class: the stride of a dimension of one entry says nothing about where rows lie."""
    g = gen(16)
    wide, line, scores = torch.randn(4, 6, 90, generator=g).to(dtype), torch.randn(1, 5, 70, generator=g).to(dtype), -torch.rand(5, 6, generator=g)
    cuts = [lambda t: t[:, -1:], lambda t: t[:, -1:, 3:80], lambda t: t[::2, 1:2], lambda t: t[:1, 2:3], lambda t: t[:, 0][:, None], lambda t: t[:1, :, 5:69],
            lambda t: t[:, :, :1], lambda t: t[:, 2:3, 4:5], lambda t: t[:1, 1:2].expand(3, 1, 90), lambda t: t[0].t()[:, None], lambda t: t[0].t()[:5, :, None], lambda t: t[:, ::3].transpose(0, 1)]
    for source, cut in [(wide, c) for c in cuts] + [(line, lambda t: t.transpose(0, 1)), (line, lambda t: t.transpose(0, 1)[1:, :, 2:]), (line[:, :, :1].contiguous(), lambda t: t.transpose(0, 1))]:
        x = cut(source)
        s = scores.repeat(18, 1)[:x.shape[0], :x.shape[1]]
        got = ops.beam_step(cut(source.to(device)), s.to(device), 4)
        want = beam_64(x, s, 4, None, 0)
        assert got[1].tolist() == [[f[1] for f in row] for row in want] and got[2].tolist() == [[int(f[2]) for f in row] for row in want]


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_beam_reorder(device):
    g = gen(8)
    parents = torch.tensor([[2, 2, 0, 1], [0, 1, 2, 0], [-1, 3, 1, 2 ** 40]])
    shapes = [((3, 3), torch.bool), ((3, 3, 5), torch.int64), ((3, 3, 7), torch.float16), ((3, 3, 3, 3), torch.uint8), ((3, 3, 4000, 3), torch.float32), ((3, 3, 0), torch.float32),
              ((3, 3, 33), torch.bfloat16), ((3, 3, 2), torch.float64), ((3, 3, 16), torch.int8), ((3, 3), torch.float32)]
    states = [(torch.rand(s, generator=g) * 100).to(t) for s, t in shapes]
    states.append(torch.rand(3, 6, 8, generator=g)[:, ::2])
    got = ops.beam_reorder([s.to(device) for s in states], parents.to(device))
    assert len(got) == len(states)
    for s, r in zip(states, got):
        assert r.shape == (3, 4, *s.shape[2:]) and r.dtype is s.dtype and r.is_contiguous()
        for b in range(3):
            for j, p in enumerate(parents[b].tolist()):
                assert torch.equal(r[b, j].cpu(), s[b, p] if 0 <= p < 3 else torch.zeros_like(s[b, 0]))
    assert ops.beam_reorder([], parents.to(device)) == []


# ----------------------------------------------------------------------------- modules
@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("bias", [False, True])
def test_linear8_through_changes_of_type_and_device(device, bias):
    """Codes and scales stay as they are; the bias and the result follow the module's type; a saved state is that of another module."""
    from difflut_amd.utils import Linear8

    torch.manual_seed(3)
    linear = Linear(40, 24, bias=bias, activation="silu", gated=True).to(device)
    x, r = torch.randn(5, 40, device=device), torch.randn(5, 24, device=device)
    first = linear.to_codes()
    want = first(x, residual=r)
    codes, scale = first.weight.float().clone(), first.weight_scale.clone()
    holds = lambda m: m.weight.dtype is torch.float8_e4m3fn and m.weight_scale.dtype is torch.float32 and torch.equal(m.weight.float(), codes) and torch.equal(m.weight_scale, scale)  # noqa: E731
    for change, dtype in ((lambda m: m.to(torch.bfloat16), torch.bfloat16), (lambda m: m.half(), torch.float16), (lambda m: m.bfloat16(), torch.bfloat16), (lambda m: m.to(device, torch.float16), torch.float16),
                          (lambda m: m.cpu().to(device), torch.float32), (lambda m: m.type(torch.float16), torch.float16), (lambda m: m.to(torch.float64).float(), torch.float32)):
        m = change(torch.nn.Sequential(linear.to_codes()))[0]
        assert m.dtype is dtype and (m.bias is None or m.bias.dtype is dtype) and holds(m)
        assert sorted(m.state_dict()) == sorted(["weight", "weight_scale"] + ["bias"] * bias)
        got = m(x, residual=r.to(dtype))
        b = linear.bias.detach().to(dtype) if bias else None
        assert got.dtype is dtype and torch.equal(got, ops.linear_codes(*ops.quantize_rows(x), first.weight, first.weight_scale, b, "silu", r.to(dtype), True, dtype))
    empty = linear.to_codes().to("meta").to_empty(device=device)
    empty.load_state_dict(first.state_dict())
    assert holds(empty) and torch.equal(empty(x, residual=r), want)
    import copy
    assert torch.equal(copy.deepcopy(first)(x, residual=r), want)


# ----------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_refusals(device):
    z = lambda *s, **k: torch.zeros(*s, device=device, **k)  # noqa: E731
    for call in (lambda: ops.rms_norm(z(3, 4), z(5)), lambda: ops.rms_norm(z(3, 4), residual=z(4)), lambda: ops.rms_norm(z(3, 0)), lambda: ops.rms_norm(z(3, 4), eps=-1.0),
                 lambda: ops.rms_norm(z(3, 4), eps=math.nan), lambda: ops.quantize_rows(z(3, 0)), lambda: ops.rms_norm_codes(z(3, 4), z(5)),
                 lambda: ops.linear(z(3, 4), z(5, 3)), lambda: ops.linear(z(3, 4), z(0, 4)), lambda: ops.linear(z(3, 4), z(5, 4), z(4)), lambda: ops.linear(z(3, 4), z(5, 4), activation="tanh"),
                 lambda: ops.linear(z(3, 4), z(5, 4), residual=z(5)), lambda: ops.linear(z(3, 4), z(4)), lambda: ops.gated_linear(z(3, 4), z(5, 4)), lambda: ops.gated_linear(z(3, 4), z(6, 4), residual=z(3, 6)),
                 lambda: ops.beam_step(z(3, 4), z(3)), lambda: ops.beam_step(z(3, 4, 5), z(3, 5)), lambda: ops.beam_step(z(3, 4, 5), z(3, 4, dtype=torch.float64)), lambda: ops.beam_step(z(3, 65, 5), z(3, 65)),
                 lambda: ops.beam_step(z(3, 4, 5), z(3, 4), beams=0), lambda: ops.beam_step(z(3, 4, 5), z(3, 4), beams=65), lambda: ops.beam_step(z(3, 4, 5), z(3, 4), beams=2.0),
                 lambda: ops.beam_step(z(3, 4, 5), z(3, 4), finished=z(3, 4)), lambda: ops.beam_step(z(3, 4, 0), z(3, 4)), lambda: ops.beam_reorder([z(3, 4)], z(3, 4)),
                 lambda: ops.beam_reorder([z(2, 4)], z(3, 4, dtype=torch.int64)), lambda: ops.beam_reorder([z(3)], z(3, 4, dtype=torch.int64)),
                 lambda: ops.beam_reorder([z(3, 4), z(3, 5)], z(3, 4, dtype=torch.int64))):
        with pytest.raises(ValueError):
            call()
    codes, scale = ops.quantize_rows(torch.ones(3, 4, device=device))
    for call in (lambda: ops.linear_codes(codes, scale[:2], codes, scale), lambda: ops.linear_codes(codes, scale, codes, scale.double()), lambda: ops.linear_codes(codes, scale, codes[:, :3], scale)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.rms_norm(z(3, 4, dtype=torch.int32)), lambda: ops.rms_norm(z(3, 4), residual=z(3, 4, dtype=torch.float16)), lambda: ops.linear(z(3, 4), z(5, 4, dtype=torch.bfloat16)),
                 lambda: ops.linear(z(3, 4), z(5, 4), z(5, dtype=torch.float16)), lambda: ops.linear_codes(z(3, 4), scale, codes, scale), lambda: ops.linear_codes(codes, scale, codes, scale, dtype=torch.float64),
                 lambda: ops.linear_codes(codes, scale, codes, scale, bias=z(3)), lambda: ops.quantize_rows(z(3, 4, dtype=torch.int64))):
        with pytest.raises(TypeError):
            call()


def test_module_refusals():
    for call in (lambda: RMSNorm(0), lambda: Linear(0, 3), lambda: Linear(3, 2.0), lambda: Linear(3, 2, activation="tanh"), lambda: RMSNorm(4)(torch.zeros(2, 5)), lambda: Linear(3, 2)(torch.zeros(2, 4))):
        with pytest.raises(ValueError):
            call()


def test_c_entry_points_refuse():
    """Before anything is launched: no device is needed, and none of the pointers is followed."""
    from difflut_amd import _native as nat

    lib, p = nat.lib(), 4096
    NULL, SHAPE, UNSUPPORTED, WORKSPACE = -1, -2, -3, -4
    norm = lambda x=p, ldx=8, r=0, ldr=0, w=0, h=0, y=p, t=0, pt=0, n=2, D=8, eps=0.0: lib.dl_rms_norm_fwd(x, ldx, r, ldr, w, h, y, None, None, t, pt, n, D, eps, None)  # noqa: E731
    assert [norm(x=0), norm(y=0), norm(r=p, ldr=8)] == [NULL] * 3
    assert [norm(n=0), norm(D=0), norm(ldx=7), norm(r=p, h=p, ldr=7), norm(eps=-1.0), norm(n=2 ** 31)] == [SHAPE] * 6
    assert [norm(t=3), norm(w=p, pt=7)] == [UNSUPPORTED] * 2
    assert lib.dl_quantize_rows(p, 8, 0, p, 0, 2, 8, None) == NULL and lib.dl_quantize_rows(p, 7, p, p, 0, 2, 8, None) == SHAPE
    back = lambda h=p, gy=p, gh=0, w=p, rstd=p, gx=p, gw=p, D=8, ws=p, size=1 << 20, ldh=8: lib.dl_rms_norm_bwd(h, ldh, w, rstd, gy, gh, gx, gw, 0, 0, 2, D, ws, size, None)  # noqa: E731
    assert [back(h=0), back(rstd=0), back(gy=0), back(w=0), back(ws=0)] == [NULL] * 5
    assert back(size=8) == WORKSPACE and back(ldh=7) == SHAPE and back(D=0) == SHAPE

    def linear(x=p, ldx=64, sx=0, w=p, ldw=64, sw=0, r=0, ldr=0, y=p, t=1, ot=1, M=4, N=8, K=64, act=0, gated=0, ws=p, size=1 << 30):
        return lib.dl_linear_fwd(x, ldx, sx, w, ldw, sw, None, r, ldr, y, None, t, ot, M, N, K, act, gated, ws, size, None)
    assert [linear(x=0), linear(w=0), linear(y=0), linear(sx=p), linear(t=3), linear(t=3, sx=p), linear(ldx=72, x=p + 2, ws=0, M=100)] == [NULL] * 7
    assert [linear(M=0), linear(N=0), linear(K=0), linear(ldx=63), linear(ldw=63), linear(gated=1, N=7), linear(r=p, ldr=7), linear(M=2 ** 31)] == [SHAPE] * 8
    assert [linear(t=5), linear(ot=0), linear(t=3, sx=p, sw=p, ot=3), linear(act=4), linear(K=2 ** 22 + 8, ldx=2 ** 23, ldw=2 ** 23)] == [UNSUPPORTED] * 5
    assert linear(x=p + 2, size=16, M=100) == WORKSPACE and linear(x=p + 2, ws=p + 4, M=100) == WORKSPACE

    def linear_back(x=p, ldx=64, w=p, ldw=64, z=p, gy=p, gx=p, gw=p, gb=p, t=1, M=4, N=8, K=64, act=2, gated=0, ws=p, size=1 << 30):
        return lib.dl_linear_bwd(x, ldx, w, ldw, z, gy, gx, gw, gb, t, M, N, K, act, gated, ws, size, None)
    assert [linear_back(x=0), linear_back(w=0), linear_back(z=0), linear_back(gy=0), linear_back(z=0, act=0, gated=1), linear_back(ws=0)] == [NULL] * 6
    assert [linear_back(M=0), linear_back(ldx=63), linear_back(ldw=63), linear_back(gated=1, N=7)] == [SHAPE] * 4
    assert [linear_back(t=3), linear_back(act=9), linear_back(N=2 ** 22 + 2)] == [UNSUPPORTED] * 3
    assert linear_back(size=64) == WORKSPACE
    step = lambda x=p, ld=10, t=0, s=p, o=p, ws=p, size=1 << 30, B=2, K=3, V=10, n=3: lib.dl_beam_step(x, ld, t, s, None, 0, o, p, p, ws, size, B, K, V, n, None)  # noqa: E731
    assert [step(x=0), step(s=0), step(o=0), step(ws=0)] == [NULL] * 4
    assert [step(B=0), step(K=0), step(V=0), step(n=0), step(ld=9)] == [SHAPE] * 5
    assert [step(t=3), step(K=65), step(n=65), step(V=2 ** 30 + 1, ld=2 ** 31), step(B=2 ** 20, K=64)] == [UNSUPPORTED] * 5
    assert step(size=8) == WORKSPACE and step(ws=p + 8) == WORKSPACE
    import ctypes
    one, zero = (ctypes.c_void_p * 1)(p), (ctypes.c_void_p * 1)(None)
    sizes = (ctypes.c_longlong * 1)(16)
    order = lambda src=one, dst=one, n=1, parents=p, B=2: lib.dl_beam_reorder(src, dst, sizes, n, parents, B, 3, 3, None)  # noqa: E731
    assert [order(parents=0), order(src=zero), order(dst=zero)] == [NULL] * 3
    assert [order(n=0), order(B=0)] == [SHAPE] * 2 and order(n=9) == UNSUPPORTED


def test_c_entry_point_refuses_to_keep_rows_without_a_backward():
    from difflut_amd import _native as nat

    p = 4096
    call = lambda kept, N, t=1: nat.lib().dl_linear_fwd(p, 64, 0, p, 64, 0, None, 0, 0, p, kept, t, t, 4, N, 64, 2, 0, None, 0, None)  # noqa: E731
    assert [call(p, 2 ** 22 + 1), call(p, 2 ** 21 + 1, 0), call(p, 2 ** 22 + 1, 2)] == [-3] * 3


@pytest.mark.gpu
def test_refusals_of_mixed_devices_float64_and_second_derivatives():
    x, w = torch.ones(4, 16, device="cuda"), torch.ones(8, 16, device="cuda")
    for call in (lambda: ops.rms_norm(x, torch.ones(16)), lambda: ops.rms_norm(x, residual=torch.ones(4, 16)), lambda: ops.linear(x, w.cpu()), lambda: ops.linear(x, w, torch.ones(8)),
                 lambda: ops.beam_step(torch.ones(2, 2, 9, device="cuda"), torch.ones(2, 2)), lambda: ops.beam_reorder([torch.ones(2, 2)], torch.zeros(2, 2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: ops.rms_norm(x.double()), lambda: ops.linear(x.double(), w.double()), lambda: ops.quantize_rows(x.double()), lambda: ops.beam_step(torch.ones(2, 2, 9, device="cuda").double(), torch.ones(2, 2, device="cuda"))):
        with pytest.raises(TypeError):
            call()
    x = x.requires_grad_()
    for y in (ops.rms_norm(x), ops.linear(x, w, activation="silu")):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


# ----------------------------------------------------------------------------- streams and graphs
def block_step(p, x, stream):
    """A block as it is trained: norm of the stream, gated projection, projection back into the stream."""
    y, h = ops.rms_norm(x, p["n"], residual=stream)
    y = ops.gated_linear(y, p["up"], activation="silu")
    return ops.linear(y, p["down"], p["b"], residual=h)


def block_parameters(dtype, device, D=64, F=96):
    g = gen(0)
    p = {"n": 1 + 0.1 * torch.randn(D, generator=g), "up": torch.randn(2 * F, D, generator=g) / 8, "down": torch.randn(D, F, generator=g) / 10, "b": torch.randn(D, generator=g)}
    return {k: v.to(dtype).to(device).requires_grad_() for k, v in p.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_on_another_stream(dtype):
    p = block_parameters(dtype, "cuda")
    g = gen(2)
    x, r, gy = (torch.randn(300, 64, generator=g).to(dtype).cuda() for _ in range(3))
    logits, scores = torch.randn(3, 4, 9000, generator=g).cuda(), torch.zeros(3, 4).cuda()

    def everything():
        y = block_step(p, x, r)
        grads = torch.autograd.grad(y, list(p.values()), gy)
        codes, scale, h = ops.rms_norm_codes(x, p["n"], residual=r)
        w, sw = ops.quantize_rows(p["up"])
        step = ops.beam_step(logits, scores)
        return [y, *grads, codes.float(), scale, h, ops.linear_codes(codes, scale, w, sw, gated=True, activation="silu", dtype=dtype), *step, *ops.beam_reorder([logits], step[1])]

    want = everything()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = everything()
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(dtype):
    """Forward and backward of a block and a search step in one graph, replayed on new inputs with eager work in between."""
    p = block_parameters(dtype, "cuda")
    g = gen(3)
    x, r, gy = (torch.randn(130, 64, generator=g).to(dtype).cuda() for _ in range(3))
    logits, scores = torch.randn(2, 3, 5001, generator=g).to(dtype).cuda(), torch.zeros(2, 3).cuda()

    def everything():
        y = block_step(p, x, r)
        grads = torch.autograd.grad(y, list(p.values()), gy)
        codes, scale, _ = ops.rms_norm_codes(x, p["n"], residual=r)
        w, sw = ops.quantize_rows(p["up"].detach())
        step = ops.beam_step(logits, scores)
        return [y, *grads, ops.linear_codes(codes, scale, w, sw, dtype=dtype), *step, *ops.beam_reorder([logits], step[1])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            everything()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    for turn in range(4):
        with torch.no_grad():
            for t in (x, r, gy, logits, scores, p["up"], p["n"]):
                t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in captured]
        want = everything()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), turn


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_model_of_blocks_trains_and_searches(device, dtype):
    """Tokens -> embedding -> two blocks on a residual stream -> a look-up-table layer on features in (0, 1) -> logits: gradients against the
    definitions; then beam search over three steps, and the same projection on 8-bit rows."""
    from difflut_amd import REGISTRY
    from difflut_amd.nodes import NodeConfig

    torch.manual_seed(5)
    V, D, F, B, T = 50, 32, 48, 4, 3
    embed = TokenEmbedding(V, D)
    norms, ups, downs = ([make() for _ in range(2)] for make in (lambda: RMSNorm(D), lambda: Linear(D, F, bias=False, activation="silu", gated=True), lambda: Linear(F, D)))
    last, head = RMSNorm(D), Linear(T * D, 64, activation="sigmoid")
    lut = REGISTRY.get_layer("random")(64, 2 * V, REGISTRY.get_node("dwn"), NodeConfig(input_dim=4, output_dim=1), seed=1)
    modules = torch.nn.ModuleList([embed, *norms, *ups, *downs, last, head]).to(device)
    modules = modules.to(dtype)
    lut = lut.to(device)

    def features(tokens, use=ops):
        stream, update = embed(tokens), None
        for norm, up, down in zip(norms, ups, downs):
            if update is None:
                y, h = use.rms_norm(stream, norm.weight), stream
            else:
                y, h = use.rms_norm(update, norm.weight, residual=stream)
            stream, update = h, use.linear(use.gated_linear(y, up.weight, None, "silu"), down.weight, down.bias)
        y, _ = use.rms_norm(update, last.weight, residual=stream)
        return use.linear(y.flatten(1), head.weight, head.bias, "sigmoid")

    class Plain:
        @staticmethod
        def rms_norm(x, w, residual=None):
            h = x if residual is None else x + residual
            y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w
            return y if residual is None else (y, h)

        @staticmethod
        def linear(x, w, b, act="none"):
            z = x @ w.t() + b
            return torch.sigmoid(z) if act == "sigmoid" else z

        @staticmethod
        def gated_linear(x, w, b, act):
            gate, up = (x @ w.t()).chunk(2, -1)
            return gate * torch.sigmoid(gate) * up

    tokens, target = torch.randint(0, V, (B, T), device=device), torch.randint(0, V, (B,), device=device)
    for _ in range(3):  # training runs
        modules.zero_grad()
        logits = GroupSum(V, tau=1.0)(lut(features(tokens).float()))
        cross_entropy(logits, target).backward()
        with torch.no_grad():
            for q in [*modules.parameters(), *lut.parameters()]:
                assert q.grad is None or bool(q.grad.isfinite().all())
                if q.grad is not None:
                    q -= 0.1 * q.grad
    # the features' gradients against the same model in doubles
    gy = torch.randn(B, 64, generator=gen(1)).to(dtype).to(device)
    y = features(tokens)
    params = list(modules.parameters())
    grads = torch.autograd.grad(y, params, gy)
    wide = [q.detach().double().cpu() for q in params]
    for q, v in zip(params, wide):
        q.data = v
    exact = features(tokens.cpu(), Plain)
    want = torch.autograd.grad(exact, params, gy.double().cpu())
    # nine products one behind the other, each a rounding or two of what it is made of, in sums of up to 96 terms of either sign
    for got, ref in zip([y, *grads], [exact, *want]):
        scale = ref.abs().max()
        assert float((got.detach().double().cpu() - ref.detach()).abs().max()) <= float(scale) * (64 * half(dtype) * 4)
    for q, v in zip(params, wide):
        q.data = v.to(dtype).to(device)
    # search: three beams, two steps of new tokens
    beams = 3
    with torch.no_grad():
        so_far = tokens[:, None].expand(B, beams, T).contiguous()
        scores = torch.full((B, beams), -math.inf, device=device)
        scores[:, 0] = 0.0
        ended = torch.zeros(B, beams, dtype=torch.bool, device=device)
        for _ in range(3):
            logits = GroupSum(V, tau=1.0)(lut(features(so_far.view(B * beams, T)).float())).view(B, beams, V)
            scores, parents, new = beam_step(logits, scores, finished=ended, end=0)
            so_far, ended = beam_reorder([so_far, ended], parents)
            so_far = torch.cat([so_far[:, :, 1:], new[:, :, None].clamp(min=0)], 2)
            ended = ended | (new == 0)
            assert bool((scores[:, :-1] >= scores[:, 1:]).all()) and bool((new >= 0).all())
        # 8-bit rows in the place of the last projection's
        y = torch.randn(B, T * D, generator=gen(2)).to(dtype).to(device)
        near, coarse = head(y), head.to_codes()(y)
        assert coarse.dtype is dtype and float((near.float() - coarse.float()).abs().max()) < 0.1
        coded_norm = RMSNorm(D, codes=True).to(device).to(dtype)
        codes, scale, h = coded_norm(y.view(B, T, D), residual=y.view(B, T, D))
        assert codes.shape == (B, T, D) and scale.shape == (B, T) and ups[0].to_codes()(codes, scale).shape == (B, T, F)
