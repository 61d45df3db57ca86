"""Embedding, group norm, dropout and sampling on the CPU (the branch of the same entry points that CPU tensors take) and on the
device, against the definitions in 64 bits.

Tolerances are sums of roundings.  u = 2^-24 is float32's half step; a value that is rounded to type t at the end is off by
half a step of it, eps(t) / 2 times its size.  A float32 sum of terms a_i in which no term goes through more than d additions is
off by d u sum |a_i|; the bounds below are taken element by element from the exact values.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from difflut_amd import ops

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CPU_AND_GPU = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, bound, dtype):
    """|got - want| within `bound` (of what was computed) and the rounding to `dtype` (of what came out)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu() if not torch.is_tensor(bound) else bound.double().cpu()
    limit = bound * (1 + half(dtype)) + half(dtype) * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got - want).abs()
    assert bool((off <= limit).all()), f"off by {float((off - limit).max())} more than {float(limit.max())}"


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ----------------------------------------------------------------------------- embedding
def embedding_64(tokens, weight, scale, gy, padding=None):
    V, D = weight.shape
    flat = tokens.reshape(-1).long()
    known = (flat >= 0) & (flat < V)
    y = torch.zeros(flat.numel(), D, dtype=torch.float64)
    y[known] = weight.double()[flat[known]] * scale
    gw, size, terms = (torch.zeros(V, n, dtype=torch.float64) for n in (D, D, 1))
    summed = known if padding is None else known & (flat != padding)
    g = gy.double().reshape(-1, D)[summed]
    gw.index_add_(0, flat[summed], g)
    size.index_add_(0, flat[summed], g.abs())
    terms.index_add_(0, flat[summed], torch.ones(len(g), 1, dtype=torch.float64))
    return y.view(*tokens.shape, D), gw * scale, size * abs(scale), terms


# a single token; rows shorter than a vector, odd, of a vector, of several teams; pieces that end inside a token's run
EMBED = [((512,), 3, 20), ((513,), 3, 20), ((510,), 9000, 8), ((1,), 1, 1), ((1,), 7, 5), ((3, 5), 9, 8), ((16,), 3, 64), ((17,), 1, 33), ((33, 2), 5, 257), ((300,), 1000, 16), ((0,), 6, 12),
         ((4, 129), 2, 1030), ((2049,), 700, 4)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("shape,V,D", EMBED)
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding(device, shape, V, D, dtype):
    g = gen(V + D)
    tokens = (torch.rand(shape, generator=g) ** 3 * V).long().clamp_(0, V - 1)
    weight, gy = torch.randn(V, D, generator=g).to(dtype), torch.randn(*shape, D, generator=g).to(dtype)
    scale = 1.75
    want, want_g, size, terms = embedding_64(tokens, weight, scale, gy)
    for ids in (tokens, tokens.int()):
        w = weight.to(device).requires_grad_()
        y = ops.embedding(ids.to(device), w, scale)
        assert y.shape == want.shape and y.dtype is dtype
        close(y, want, want.abs() * U, dtype)
        grad, = torch.autograd.grad(y, w, gy.to(device))
        assert grad.dtype is dtype
        close(grad, want_g, size * (terms + 1) * U, dtype)  # the terms' additions and the product with scale


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_embedding_of_tokens_outside_and_padding(device):
    V, D, g = 10, 12, gen(3)
    weight, gy = torch.randn(V, D, generator=g), torch.randn(9, D, generator=g)
    tokens = torch.tensor([-1, 3, 10, 3, 0, 9, 2 ** 40, 0, -2 ** 40])
    want, want_g, size, terms = embedding_64(tokens, weight, 1.0, gy, padding=0)
    w = weight.to(device).requires_grad_()
    y = ops.embedding(tokens.to(device), w, padding_idx=0)
    assert torch.equal(y.cpu().double(), want) and torch.equal(y[4].cpu(), weight[0])  # padding is looked up all the same
    grad, = torch.autograd.grad(y, w, gy.to(device))
    close(grad, want_g, size * terms * U, torch.float32)
    assert not grad[0].any() and not grad[1].any()
    # nothing but padding, nothing but strangers
    for ids in (torch.zeros(40, dtype=torch.long), torch.full((40,), -7)):
        y = ops.embedding(ids.to(device), w, padding_idx=0)
        grad, = torch.autograd.grad(y, w, torch.ones_like(y))
        assert not grad.any()


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_embedding_strides(device):
    """Rows apart, a transposed matrix, tokens and a gradient that are not contiguous, one that is expanded."""
    g = gen(5)
    wide, tokens = torch.randn(20, 40, generator=g), torch.randint(0, 20, (6, 8), generator=g)
    for cut in (lambda t: t[:, 4:20], lambda t: t[:, 3:20], lambda t: t.t()[:16], lambda t: t[::2]):
        base = wide.clone().to(device).requires_grad_()
        w = cut(base)
        ids = tokens.to(device).t() % w.shape[0]
        y = ops.embedding(ids, w, 2.0)
        close(y, 2.0 * cut(wide).double()[ids.cpu()], 0.0, torch.float32)
        gy = torch.randn(1, 1, w.shape[1], generator=g).to(device).expand(*ids.shape, -1)
        grad, = torch.autograd.grad(y, base, gy)
        _, want, size, terms = embedding_64(ids.cpu(), cut(wide), 2.0, gy.cpu())
        close(cut(grad), want, size * (terms + 1) * U, torch.float32)


def test_embedding_gradient_against_differences():
    w = torch.randn(5, 3, dtype=torch.float64, generator=gen(1)).requires_grad_()
    tokens = torch.tensor([0, 4, 4, 1, -1])
    assert torch.autograd.gradcheck(lambda t: ops.embedding(tokens, t, 0.7), (w,))


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D,dtype", [(20011, 3000, 68, torch.float32), (5000, 1, 24, torch.float32), (9000, 70001, 8, torch.bfloat16),
                                         (40000, 5, 129, torch.float16), (131072, 9000, 4, torch.float32), (300001, 100, 8, torch.float32),
                                         (200003, 300001, 8, torch.bfloat16), (170003, 600001, 4, torch.float32), (150000, 1, 4, torch.float32), (140000, 140001, 12, torch.float32)])
def test_embedding_gradient_of_many_tokens(n, V, D, dtype):
    """Uneven frequencies, all tokens equal, more tokens of the vocabulary than of the text: the formula, and the same bits twice."""
    g = gen(n)
    tokens = ((V + 1.0) ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp_(0, V - 1)
    tokens[::17] = -1  # (some of no token)
    gy = torch.randn(n, D, generator=g).to(dtype)
    w = torch.zeros(V, D, dtype=dtype, device="cuda").requires_grad_()
    y = ops.embedding(tokens.cuda(), w)
    grad, = torch.autograd.grad(y, w, gy.cuda(), retain_graph=True)
    again, = torch.autograd.grad(y, w, gy.cuda())
    _, want, size, terms = embedding_64(tokens, w.cpu(), 1.0, gy)
    close(grad, want, size * terms.clamp_max(2 * math.sqrt(n) + 64) * U, dtype)  # pieces first, then the pieces' sums
    assert torch.equal(grad, again)


# ----------------------------------------------------------------------------- group norm
def sigmoid(z):
    return 1 / (1 + torch.exp(-z))


def norm_64(x, G, weight, bias, eps, act, gy, depth):
    """The definition, its gradients, and bounds of what float32 makes of them (depth: additions a term of a group's sum goes through)."""
    B, C = x.shape[0], x.shape[-1]
    x, gy = x.double().reshape(B, -1, G, C // G), gy.double().reshape(B, -1, G, C // G)
    ga = torch.ones(G, C // G, dtype=torch.float64) if weight is None else weight.double().view(G, -1)
    be = torch.zeros(G, C // G, dtype=torch.float64) if bias is None else bias.double().view(G, -1)
    mean = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    m = mean(x)
    rstd = 1 / torch.sqrt(mean((x - m) ** 2) + eps)
    hat = (x - m) * rstd
    z = hat * ga + be
    s = sigmoid(z)
    y, slope = {"none": (z, torch.ones_like(z)), "relu": (z.clamp_min(0), (z > 0).double()), "silu": (z * s, s * (1 + z * (1 - s))),
                "sigmoid": (s, s * (1 - s))}[act]
    d = depth * U
    off_m = d * mean(x.abs()) + 2 * U * x.abs()              # the mean, the difference with it
    off_hat = off_m * rstd + hat.abs() * (2 * d + (d * mean(x.abs()) * rstd) ** 2 + 4 * U)  # ... and 1 / sqrt(var + eps)
    off_z = off_hat * ga.abs() + 3 * U * ((hat * ga).abs() + be.abs())
    off_y = 1.1 * off_z + 8 * U * (1 + z.abs()) * y.abs()    # |act'| <= 1.1; an exponential of z is off by (1 + |z|) u
    g = gy * slope
    off_g = gy.abs() * (0.5 * off_z + 16 * U * (1 + z.abs()) * (s if act != "none" else 0 * s))  # |act''| <= 1/2
    gb, gw = g.sum((0, 1)), (g * hat).sum((0, 1))
    many = (depth + 4 * B) * U
    off_b = off_g.sum((0, 1)) + many * g.abs().sum((0, 1))
    off_w = (off_g * hat.abs() + g.abs() * off_hat).sum((0, 1)) + many * (g * hat).abs().sum((0, 1))
    gh, off_h = g * ga, (off_g + 2 * U * g.abs()) * ga.abs()
    a, q = mean(gh), mean(gh * hat)
    off_a = mean(off_h) + d * mean(gh.abs())
    off_q = mean(off_h * hat.abs() + gh.abs() * off_hat) + d * mean((gh * hat).abs())
    gx = rstd * (gh - a - hat * q)
    size = gh.abs() + a.abs() + (hat * q).abs()
    rel = 2 * d + (d * mean(x.abs()) * rstd) ** 2 + 4 * U    # of rstd
    off_x = rstd * (off_h + off_a + hat.abs() * off_q + q.abs() * off_hat + size * (rel + 6 * U))
    flat = lambda t: t.reshape(B, -1, C)  # noqa: E731
    return [(flat(y), flat(off_y)), (flat(gx), flat(off_x)), (gw.reshape(-1), off_w.reshape(-1)), (gb.reshape(-1), off_b.reshape(-1))]


# positions x channels: one value, one position, channels fewer than a vector, groups of odd width, groups across vectors, one group
# wider than a block's tile, as many groups as channels, many positions, positions and channels that end inside a tile
NORM = [(1, (1,), 1, 1), (3, (), 24, 4), (2, (5,), 3, 3), (2, (7, 9), 20, 4), (1, (64,), 30, 3), (4, (11,), 8, 2), (2, (3, 5), 36, 12),
        (2, (2,), 2500, 1), (1, (3,), 5001, 3), (3, (13,), 64, 64), (2, (700,), 16, 2), (1, (50, 60), 40, 8), (5, (19,), 320, 32)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("B,space,C,G", NORM)
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm(device, B, space, C, G, dtype):
    g = gen(C + G)
    x, gy = ((torch.randn(B, *space, C, generator=g) * 0.4 + m).to(dtype) for m in (0.5, 0.0))
    weight, bias = ((torch.randn(C, generator=g) * 0.2 + m).to(dtype) for m in (1.0, 0.0))
    for act in ("none", "silu", "sigmoid"):
        want = norm_64(x, G, weight, bias, 1e-2, act, gy, depth=256)
        leaves = [t.to(device).requires_grad_() for t in (x, weight, bias)]
        y = ops.group_norm(leaves[0], G, *leaves[1:], eps=1e-2, activation=act)
        assert y.shape == x.shape and y.dtype is dtype
        got = [y, *torch.autograd.grad(y, leaves, gy.to(device))]
        for t, (exact, bound) in zip(got, want):
            assert t.dtype is dtype
            close(t.reshape(exact.shape), exact, bound, dtype)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_parameters_of_another_type_or_none(device):
    g = gen(7)
    x, gy = torch.randn(3, 10, 24, generator=g).bfloat16(), torch.randn(3, 10, 24, generator=g).bfloat16()
    weight, bias = torch.randn(24, generator=g), torch.randn(24, generator=g)
    for w, b in ((weight, bias), (weight, None), (None, bias), (None, None)):
        want = norm_64(x, 3, w, b, 1e-5, "sigmoid", gy, depth=256)
        leaves = [t.to(device).requires_grad_() for t in (x, w, b) if t is not None]
        it = iter(leaves[1:])
        y = ops.group_norm(leaves[0], 3, next(it) if w is not None else None, next(it) if b is not None else None, activation="sigmoid")
        close(y, *want[0], torch.bfloat16)
        got = torch.autograd.grad(y, leaves, gy.to(device))
        close(got[0], *want[1], torch.bfloat16)
        for t, pair in zip(got[1:], [want[2 + i] for i, p in enumerate((w, b)) if p is not None]):
            assert t.dtype is torch.float32
            close(t, *pair, torch.float32)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_relu_and_constant_groups(device):
    """A group of equal values has no variance: xhat is 0 and the output the bias; relu's gradient stops below 0."""
    x = torch.tensor([[[2.0, 2.0, 1.0, 3.0]], [[-5.0, -5.0, 4.0, 0.0]]])
    leaf = x.to(device).requires_grad_()
    bias = torch.tensor([0.5, -0.5, 0.0, 0.0], device=device)
    y = ops.group_norm(leaf, 2, None, bias, eps=1e-5, activation="relu")
    want = torch.tensor([[[0.5, 0.0, 0.0, 1.0]], [[0.5, 0.0, 1.0, 0.0]]])
    close(y, want, 1e-5, torch.float32)  # eps: 1 / sqrt(1 + 1e-5), 1 / sqrt(4 + 1e-5) of a difference of 2
    gx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    scale = 1 / math.sqrt(1e-5)
    close(gx[0, 0, :2], torch.tensor([0.5, -0.5]) * scale, scale * 8 * U, torch.float32)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_far_from_zero(device):
    """Values around 1000 with a spread of 1: E[x^2] - mean^2 would have lost the variance."""
    x = (torch.randn(2, 900, 8, generator=gen(9)) + 1000.0)
    y = ops.group_norm(x.to(device), 2)
    wide = x.double().view(2, -1, 2, 4)
    want = ((wide - wide.mean((1, 3), keepdim=True)) / torch.sqrt(wide.var((1, 3), unbiased=False, keepdim=True) + 1e-5)).view(x.shape)
    # the mean is a float32 near 1000: off by its own rounding and the sum's, (1 + depth) u 1000
    close(y, want, 1000 * 64 * U, torch.float32)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_leaves_other_samples_alone_when_one_is_not_finite(device):
    x = torch.randn(3, 6, 8, generator=gen(2))
    x[1, 2, 3] = float("nan")
    y = ops.group_norm(x.to(device), 2).cpu()
    assert y[1, :, :4].isnan().all() and not y[1, :, 4:].isnan().any() and not y[0].isnan().any() and not y[2].isnan().any()


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_module_on_images(device):
    from difflut_amd.utils import GroupNorm

    torch.manual_seed(0)
    x = torch.randn(2, 12, 5, 7)
    norm = GroupNorm(3, 12, activation="sigmoid").to(device)
    with torch.no_grad():
        norm.weight.normal_(), norm.bias.normal_()
    want = norm_64(x.movedim(1, -1), 3, norm.weight.cpu(), norm.bias.cpu(), 1e-5, "sigmoid", x.movedim(1, -1), depth=256)[0]
    for layout in (torch.contiguous_format, torch.channels_last):
        y = norm(x.to(device).contiguous(memory_format=layout))
        assert y.shape == x.shape and y.is_contiguous(memory_format=torch.channels_last)
        close(y.movedim(1, -1).reshape(2, -1, 12), *want, torch.float32)
    flat = norm(x[:, :, 0, 0].to(device))
    assert flat.shape == (2, 12)
    with pytest.raises(ValueError):
        norm(x[:, :5].to(device))


def test_group_norm_gradient_against_differences():
    g = gen(4)
    x, w, b = (torch.randn(s, dtype=torch.float64, generator=g).requires_grad_() for s in ((2, 5, 6), (6,), (6,)))
    for act in ("none", "silu", "sigmoid"):
        assert torch.autograd.gradcheck(lambda *t: ops.group_norm(t[0], 2, *t[1:], activation=act), (x, w, b))


@pytest.mark.gpu
@pytest.mark.parametrize("B,space,C,G", [(2, (130, 130), 40, 8), (1, (40000,), 6, 3), (3, (900,), 1100, 1), (1, (6001,), 2500, 1), (1, (70, 300), 64, 64),
                                         (300, (64,), 96, 4), (9, (130,), 250, 5), (5000, (), 64, 8), (3001, (3,), 24, 6), (2049, (), 7, 7), (1100, (2,), 36, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_of_larger_tensors(B, space, C, G, dtype):
    """Samples split over blocks, wide groups in slices, what still fits one block, small samples that share one; twice the same bits."""
    g = gen(C + G)
    x, gy = ((torch.randn(B, *space, C, generator=g) * 0.4 + m).to(dtype) for m in (0.5, 0.0))
    weight, bias = ((torch.randn(C, generator=g) * 0.2 + m).to(dtype) for m in (1.0, 0.0))
    want = norm_64(x, G, weight, bias, 1e-2, "silu", gy, depth=256)
    leaves = [t.cuda().requires_grad_() for t in (x, weight, bias)]
    runs = []
    for _ in range(2):
        y = ops.group_norm(leaves[0], G, *leaves[1:], eps=1e-2, activation="silu")
        runs.append([y, *torch.autograd.grad(y, leaves, gy.cuda())])
    for t, again, (exact, bound) in zip(*runs, want):
        close(t.reshape(exact.shape), exact, bound, dtype)
        assert torch.equal(t, again)


@pytest.mark.gpu
def test_group_norm_far_from_zero_in_pieces():
    """The variance of a sample that is split over blocks, around 1000, and with an outlier where the sums begin."""
    x = torch.randn(1, 60000, 8, generator=gen(9)) + 1000.0
    x[0, 0] = -5000.0
    y = ops.group_norm(x.cuda(), 2)
    wide = x.double().view(1, -1, 2, 4)
    want = ((wide - wide.mean((1, 3), keepdim=True)) / torch.sqrt(wide.var((1, 3), unbiased=False, keepdim=True) + 1e-5)).view(x.shape)
    rstd = 1 / math.sqrt(float(wide.var((1, 3), unbiased=False).min()))
    close(y, want, 1000 * rstd * 64 * U + want.abs() * 512 * U, torch.float32)  # the mean's rounding; a thread's rows in the variance


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_group_norm_gradients_of_some_inputs(device):
    g = gen(14)
    x, gy, weight, bias = (torch.randn(s, generator=g).to(device) for s in ((3, 40, 12), (3, 40, 12), (12,), (12,)))
    leaves = [t.clone().requires_grad_() for t in (x, weight, bias)]
    full = torch.autograd.grad(ops.group_norm(leaves[0], 3, *leaves[1:], activation="silu"), leaves, gy)
    for i in range(3):
        some = [t.clone().requires_grad_(n == i) for n, t in enumerate((x, weight, bias))]
        got, = torch.autograd.grad(ops.group_norm(some[0], 3, *some[1:], activation="silu"), some[i], gy)
        assert torch.equal(got, full[i])


# [B, P, C] in G groups and the type's number, by form: rounds of blocks over many samples, small samples that share blocks, one launch for few;
# a tile per block of 1024 threads; groups wider than a tile, of one position and of many
NORM_FORMS = [(1, 65536, 1, 2048, 8), (1, 8192, 1, 16000, 16), (0, 8192, 1, 16000, 16), (0, 65536, 1, 64, 8), (0, 4, 1, 64, 8), (0, 256, 576, 32, 8),
              (2, 600, 3, 1800, 1), (0, 1024, 1, 1500, 1), (1, 8192, 1, 16000, 1), (0, 700, 1, 4104, 2), (1, 16, 9215, 320, 32), (0, 2, 40000, 5000, 1)]


@pytest.mark.parametrize("type,B,P,C,G", NORM_FORMS)
def test_group_norm_workspaces_hold_what_is_kept(type, B, P, C, G):
    """What a direction keeps between its launches, and no more: a mean and a sum of squares per group of a piece; two
    sums per channel, of a sample or of a piece, their means per group, and up to 64 shares of many samples' sums."""
    from difflut_amd import _native as nat

    if not nat.is_built():
        pytest.skip("not built")
    x = B * P * C * (4 if type == 0 else 2)
    forward, backward = nat.lib().dl_group_norm_fwd_workspace_bytes(type, B, P, C, G), nat.lib().dl_group_norm_bwd_workspace_bytes(type, B, P, C, G)
    assert 0 < forward <= max(x // 16, 4096)
    assert 0 < backward <= 8 * B * C * (1 if P == 1 else 1 + P / 4) + 8 * B * G + 512 * C + 1024
    if C // G <= 1024 and P == 1:  # a tile in one block of 256 threads: 2048 blocks' sums at most, of 2048 channels
        assert forward <= 256 and backward <= 2 ** 25 + 512 * C + 1024


@pytest.mark.gpu
@pytest.mark.parametrize("type,B,P,C,G", [(1, 6000, 1, 2048, 8), (0, 5000, 1, 64, 8), (0, 4, 1, 64, 8), (0, 256, 60, 32, 8), (2, 600, 3, 1800, 1), (0, 1024, 1, 1500, 1),
                                          (0, 700, 1, 4104, 2), (1, 3, 1, 5001, 3), (1, 3, 3001, 320, 32), (0, 2, 700, 5000, 1), (2, 5, 3, 2, 1)])
def test_group_norm_stays_within_its_workspaces(type, B, P, C, G):
    """Workspaces of exactly the size asked for: right results, and nothing written behind them."""
    from difflut_amd import _native as nat

    lib, dtype, g = nat.lib(), TYPES[type], gen(B + C)
    x, gy = ((torch.randn(B, P, C, generator=g) * 0.4 + m).to(dtype) for m in (0.5, 0.0))
    weight, bias = ((torch.randn(C, generator=g) * 0.2 + m).to(dtype) for m in (1.0, 0.0))
    want = norm_64(x, G, weight, bias, 1e-2, "silu", gy, depth=256)
    x, gy, weight, bias = (t.cuda() for t in (x, gy, weight, bias))
    y, gx, gw, gb, stats = torch.empty_like(x), torch.empty_like(x), torch.empty_like(weight), torch.empty_like(bias), torch.empty(B, G, 2, device="cuda")
    sizes = [lib.dl_group_norm_fwd_workspace_bytes(type, B, P, C, G), lib.dl_group_norm_bwd_workspace_bytes(type, B, P, C, G)]
    spaces = [torch.full((n + 8192,), 90, dtype=torch.uint8, device="cuda") for n in sizes]
    at = lambda t: t.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.dl_group_norm_fwd(at(x), at(weight), at(bias), at(y), at(stats), type, type, B, P, C, G, 1e-2, 2, at(spaces[0]), sizes[0], stream) == 0
    assert lib.dl_group_norm_bwd(at(x), at(gy), at(weight), at(bias), at(stats), at(gx), at(gw), at(gb), type, type, B, P, C, G, 2, at(spaces[1]), sizes[1],
                                 stream) == 0
    for t, (exact, bound) in zip((y, gx, gw, gb), want):
        close(t.reshape(exact.shape), exact, bound, dtype)
    for n, space in zip(sizes, spaces):
        assert bool((space[n:] == 90).all())


@pytest.mark.gpu
def test_group_norm_gradients_of_more_channels_than_a_launch_takes():
    """2^29 channels and more: 32 to a block of 256 threads would be 2^32 work items.  x of 1 and -1 in turn under statistics of 0 and 1:
    the gradients are gy and gy x as they are (one sample, one position: nothing is added)."""
    from difflut_amd import _native as nat

    G, C = 64, 2 ** 29 + 64 * 6
    x, ones = torch.ones(C, dtype=torch.bfloat16, device="cuda"), torch.ones(C, dtype=torch.bfloat16, device="cuda")
    x[1::2] = -1
    gy = (torch.arange(C, dtype=torch.int32, device="cuda") % 257 - 128).to(torch.bfloat16)  # (whole numbers that bf16 holds)
    stats = torch.tensor([0.0, 1.0], device="cuda").repeat(G)
    gw, gb = (torch.full((C,), 500.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    need = nat.lib().dl_group_norm_bwd_workspace_bytes(1, 1, 1, C, G)
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    at = lambda t: t.data_ptr()  # noqa: E731
    assert nat.lib().dl_group_norm_bwd(at(x), at(gy), at(ones), None, at(stats), None, at(gw), at(gb), 1, 1, 1, 1, C, G, 0, at(space), need,
                                       torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(gb, gy) and torch.equal(gw, gy * x)


# ----------------------------------------------------------------------------- dropout
def philox(seed, offset, numel, start=0):
    """By numpy's 64-bit products, from the generator's definition; words start .. (a multiple of 4)."""
    counter = np.arange(start // 4, start // 4 - (-numel // 4), dtype=np.uint64)
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [counter & low, counter >> s32, np.full_like(counter, offset & 0xFFFFFFFF), np.full_like(counter, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(key[0]), b & low, (a >> s32) ^ c[3] ^ np.uint64(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, axis=1).reshape(-1)[:numel]


def test_philox_known_answers():
    """The generator's published test vectors (counter and key all zeros; all ones)."""
    from difflut_amd.cpu_ops import philox_words

    assert [f"{w:08x}" for w in philox(0, 0, 4)] == ["6627e8d5", "e169c58d", "bc57ac4c", "9b00dbd8"]
    for seed, offset in ((0, 0), (1, 2), (2 ** 64 - 1, 2 ** 64 - 1), (0x0123456789ABCDEF, 0xFEDCBA9876543210)):
        assert philox_words(ops._signed64(seed), ops._signed64(offset), 1001).tolist() == philox(seed, offset, 1001).tolist()


def philox_4x32(counter, key):
    """Ten rounds on four words under two, in Python's whole numbers."""
    (c0, c1, c2, c3), (k0, k1) = counter, key
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ k0, b % 2 ** 32, (a >> 32) ^ c3 ^ k1, a % 2 ** 32
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return [c0, c1, c2, c3]


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_philox_words_where_they_belong(device):
    """The three answers that are published with the generator (zeros, ones, digits of pi), then the order of the words: seed and offset have
    four different ones, and each decides the mask."""
    ones = 0xFFFFFFFF
    for counter, key, answer in (((0,) * 4, (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"), ((ones,) * 4, (ones, ones), "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                                 ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join(f"{w:08x}" for w in philox_4x32(counter, key)) == answer
    low, high, k0, k1 = 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0
    words = [w for i in range(250) for w in philox_4x32((i, 0, low, high), (k0, k1))]
    for p in (0.5, 0.1, 0.9):
        hit = torch.tensor([w < math.floor(p * 2.0 ** 32 + 0.5) for w in words])
        y = ops.dropout(torch.full((1000,), 0.25, device=device), p, (k1 << 32 | k0, high << 32 | low), mode="flip")
        assert torch.equal(y.cpu() == 0.75, hit)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("shape", [(1,), (3, 5), (64, 100), (7, 1025), (0, 4)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.25, 1 / 3, 0.999, 1.0])
def test_dropout(device, shape, dtype, p):
    seed, offset = 2 ** 63 + 12345, 2 ** 40 + 7
    g = gen(11)
    x, gy = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    hit = torch.from_numpy(philox(seed, offset, x.numel()) < math.floor(p * 2.0 ** 32 + 0.5)).view(shape)
    if p in (0.0, 1.0):
        assert hit.all() == (p == 1.0) or not hit.numel()
    factor = 0.0 if p == 1.0 else 1 / (1 - p)
    for state in ((seed, offset), torch.tensor([ops._signed64(seed), offset], device=device)):
        leaf = x.to(device).requires_grad_()
        y = ops.dropout(leaf, p, state)
        gx, = torch.autograd.grad(y, leaf, gy.to(device))
        for got, of in ((y, x), (gx, gy)):
            assert got.dtype is dtype
            want = torch.where(hit, 0.0, of.double() * factor)
            close(got, want, want.abs() * 2 * U, dtype)  # the factor and the product
            assert not got.detach().cpu()[hit].any()
        y = ops.dropout(leaf, p, state, mode="flip")
        gx, = torch.autograd.grad(y, leaf, gy.to(device))
        assert torch.equal(y.detach().cpu(), torch.where(hit, 1 - x.float(), x.float()).to(dtype)) and torch.equal(gx.cpu(), gy)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_dropout_of_views_and_values_that_are_not_finite(device):
    """The mask goes by the row-major order whatever the strides and the alignment; what is hit is gone whatever it was."""
    base = torch.randn(40, 30, generator=gen(3))
    for view in (lambda t: t.t(), lambda t: t[:, 3:], lambda t: t.reshape(-1)[1:], lambda t: t[::3, ::2]):
        x = view(base.to(device))
        hit = torch.from_numpy(philox(5, 6, x.numel()) < 2 ** 31).view(x.shape)
        assert torch.equal(ops.dropout(x, 0.5, (5, 6)).cpu(), torch.where(hit, 0.0, view(base) * 2))
    for bad in (math.inf, -math.inf, math.nan):
        y = ops.dropout(torch.full((64,), bad, device=device), 0.5, (1, 1)).cpu()
        hit = torch.from_numpy(philox(1, 1, 64) < 2 ** 31)
        assert not y[hit].any() and not y[~hit].isfinite().any()


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_dropout_module(device):
    from difflut_amd.utils import Dropout

    x = torch.ones(50, 40, device=device)
    drop = Dropout(0.25, seed=9).to(device)
    first, second = drop(x), drop(x)
    assert not torch.equal(first, second) and drop.state.tolist() == [9, 2]
    other = Dropout(0.25).to(device)
    other.load_state_dict({"state": torch.tensor([9, 1])})
    assert torch.equal(other(x), second)  # a resumed run goes on with the same masks
    # the backward draws the mask of its forward, also after further calls
    leaf = x.clone().requires_grad_()
    y = drop(leaf)
    drop(x)
    gx, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert torch.equal(gx, y.detach())
    assert drop.eval()(x) is x


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("mode", ["zero", "flip"])
def test_dropout_modules_have_noise_of_their_own(device, mode):
    """Modules built without a seed draw different masks, and the same ones again after torch.manual_seed; a seed given is kept."""
    from difflut_amd.utils import Dropout

    def build():
        torch.manual_seed(5)
        return [Dropout(0.5, mode).to(device) for _ in range(3)]

    x = torch.full((64, 64), 0.25, device=device)
    hits = [drop(x) != x * (1 if mode == "flip" else 2) for drop in build()]
    for i in range(3):
        for j in range(i):  # of 4096 independent pairs half are equal, within 6 standard deviations of 32
            assert abs(int((hits[i] == hits[j]).sum()) - 2048) <= 192
    assert all(torch.equal(drop(x) != x * (1 if mode == "flip" else 2), hit) for drop, hit in zip(build(), hits))
    assert torch.equal(Dropout(0.5, mode, seed=0).to(device)(x), ops.dropout(x, 0.5, (0, 0), mode))
    assert Dropout(0.5, seed=7).state.tolist() == [7, 0]


@pytest.mark.gpu
def test_more_than_two_to_the_31_elements():
    """Offsets past 32 bits: the last entries of a dropout, a lookup and a gradient."""
    n = 2 ** 31 + 40
    y = ops.dropout(torch.ones(n, dtype=torch.float16, device="cuda"), 0.5, (3, 4))
    for start in (0, 2 ** 31 - 64, 2 ** 31):
        hit = torch.from_numpy(philox(3, 4, min(128, n - start), start) < 2 ** 31)
        assert torch.equal(y[start:start + len(hit)].cpu() == 0, hit)
    del y
    V, D = 2 ** 21 + 3, 1032
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    w[-1], w[-2] = 1.0, 2.0
    tokens = torch.tensor([V - 1, V - 2, 0, V - 1], device="cuda")
    w.requires_grad_()
    y = ops.embedding(tokens, w)
    assert y[:, 0].tolist() == [1.0, 2.0, 0.0, 1.0] and y[:, -1].tolist() == [1.0, 2.0, 0.0, 1.0]
    grad, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert grad[[0, 1, V // 2, V - 3, V - 2, V - 1]].float().mean(1).tolist() == [1.0, 0.0, 0.0, 0.0, 1.0, 2.0]
    assert float(grad.sum(dtype=torch.float32)) == 4.0 * D


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes():
    """A launch takes less than 2^32 work items: lookups and samples of more rows are as right at the end as at the beginning."""
    n, D = 2 ** 26 + 1001, 129
    w = torch.arange(5 * D, device="cuda").view(5, D).remainder(251).to(torch.bfloat16)  # (whole numbers that bf16 holds)
    tokens = torch.arange(n, dtype=torch.int32, device="cuda") * 7 % 5
    y = ops.embedding(tokens, w)
    for start in range(0, n, 2 ** 22):
        assert torch.equal(y[start:start + 2 ** 22], w[tokens[start:start + 2 ** 22].long()]), start
    del y, tokens
    B, V = 2 ** 22 + 9, 1030
    best = torch.arange(B, device="cuda") * 13 % V
    logits = torch.zeros(B, V, dtype=torch.float16, device="cuda").scatter_(1, best[:, None], 1.0)
    temperature = torch.full((B,), 1e-3, device="cuda")  # (the others weigh exp(-1000))
    temperature[1::2] = 0.0
    assert torch.equal(ops.sample(logits, torch.full((B,), 0.5, device="cuda"), temperature=temperature), best)


def test_dropout_gradient_against_differences():
    x = torch.randn(4, 9, dtype=torch.float64, generator=gen(8)).requires_grad_()
    assert torch.autograd.gradcheck(lambda t: ops.dropout(t, 0.4, (3, 1)), (x,))


# ----------------------------------------------------------------------------- sampling
def sample_64(logits, uniform, T, k, p, m):
    """Row by row from the definition, in float64 (settings: float32 values, a list per row)."""
    out = []
    for row, u, t, kk, pp, mm in zip(logits.double().numpy(), uniform.double().numpy(), T, k, p, m):
        row = np.where(np.isnan(row), -np.inf, row)
        order = np.argsort(-row, kind="stable")
        order = order[row[order] > -np.inf]
        if not len(order):
            out.append(-1)
            continue
        top = row[order[0]]
        if not t > 0:
            out.append(int(order[0]))
            continue
        if 0 < kk < len(order):
            order = order[:kk]
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            w = np.where(row[order] == top, 1.0, np.exp((row[order] - top) / t) if top < np.inf else 0.0)
        before = np.concatenate([[0.0], np.cumsum(w)])  # one after the other
        keep = np.ones(len(order), bool) if pp >= 1 else before[:-1] < pp * before[-1]
        keep &= w >= mm
        keep[0] = True
        by_index = np.argsort(order[keep])
        kept, running = order[keep][by_index], np.cumsum(w[keep][by_index])
        past = np.nonzero(running > u * running[-1])[0]
        out.append(int(kept[past[0]] if len(past) else kept[-1]))
    return torch.tensor(out)


def f32(v):
    return float(np.float32(v))


def check_sample(device, logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    B = len(logits)
    rows = [v.float().tolist() if torch.is_tensor(v) else [f32(v)] * B for v in (temperature, top_k, top_p, min_p)]
    want = sample_64(logits, uniform, rows[0], [int(v) for v in rows[1]], *rows[2:])
    args = [v.to(device) if torch.is_tensor(v) else v for v in (temperature, top_k, top_p, min_p)]
    got = ops.sample(logits.to(device), uniform.to(device), *args)
    assert got.dtype is torch.int64 and got.cpu().tolist() == want.tolist()


# columns: one, a few lanes per row, a wavefront per row (powers of two, odd), a block per row
COLUMNS = [1, 2, 10, 33, 64, 65, 128, 129, 300, 1000, 1024, 1025, 4096, 4097, 9001]
FILTERS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.95, min_p=0.05),
           dict(temperature=0.7, top_k=50, top_p=0.9), dict(temperature=3.0, top_k=3000, top_p=0.999, min_p=0.001)]


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", COLUMNS)
@pytest.mark.parametrize("dtype", TYPES)
def test_sample(device, V, dtype):
    g = gen(V)
    B = 5 if V > 2000 else 13
    logits, uniform = (torch.randn(B, V, generator=g) * 3).to(dtype), torch.rand(B, generator=g)
    for settings in FILTERS:
        check_sample(device, logits, uniform, **settings)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [12, 700, 6000])
def test_sample_settings_per_row(device, V):
    g = gen(V + 1)
    B = 24
    r = torch.rand(4, B, generator=g)
    T, k, p, m = r[0] * 2, (r[1] * 2 * V).int(), 0.3 + r[2], r[3] * 0.2
    T[3], k[4], p[5], m[6] = 0.0, 1, 1.0, 0.0
    check_sample(device, torch.randn(B, V, generator=g) * 2, torch.rand(B, generator=g), T, k.long(), p, m)
    check_sample(device, torch.randn(B, V, generator=g) * 2, torch.rand(B, generator=g), T, 5, p, 0.01)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [10, 64, 300, 5000, 20000])
def test_sample_equal_logits(device, V):
    """Sums of bits, as GroupSum's are, have many equal values: the cuts fall among those, by index."""
    g = gen(V + 2)
    B = 6
    uniform = torch.rand(B, generator=g)
    for levels in (1, 2, 7):
        logits = torch.randint(0, levels, (B, V), generator=g).float()
        for settings in (dict(), dict(top_k=3), dict(top_k=max(1, V // 3)), dict(top_p=0.3), dict(top_k=max(1, V // 2), top_p=0.7),
                         dict(top_k=max(1, V - 1), top_p=0.9, temperature=0.25)):
            check_sample(device, logits, uniform, **settings)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [9, 200, 4500])
def test_sample_masked_rows(device, V):
    """Masks of -infinity and of the type's lowest value, rows with one or nothing left, NaN and +infinity."""
    g = gen(V + 3)
    logits = torch.randn(9, V, generator=g)
    logits[0] = -math.inf
    logits[1, 1:] = -math.inf
    logits[2, :-1] = torch.finfo(torch.float32).min
    logits[3, ::2] = -math.inf
    logits[4] = torch.finfo(torch.float32).min
    logits[5, 3] = math.nan
    logits[6] = math.nan
    logits[7, 2] = logits[7, 5] = math.inf
    logits[8, 0], logits[8, 1] = 0.0, -0.0
    for u in (0.0, 0.3, 0.999999):
        for settings in FILTERS:
            check_sample(device, logits, torch.full((9,), u), **settings)


@pytest.mark.gpu
@pytest.mark.parametrize("B,V", [(1, 65537), (3, 131071), (33, 70001), (1, 300001)])
def test_sample_long_rows(B, V):
    """Rows split over blocks, and more rows than are split: every kind of cut, equal logits, masks."""
    g = gen(V)
    normal, equal = torch.randn(3, V, generator=g) * 3, torch.randint(0, 9, (3, V), generator=g).float()
    masked = torch.where(torch.rand(3, V, generator=g) < 0.999, torch.full((3, V), -math.inf), normal)
    masked[0] = -math.inf
    masked[1, 5] = math.nan
    for logits in (normal, normal.bfloat16(), equal, masked):
        rows = torch.arange(B) % 3  # (the oracle's time goes by the row)
        uniform = torch.rand(3, generator=g)
        for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.01), (1.0, 0, 0.8, 0.0), (1.5, 3000, 0.99, 0.0), (1.0, 60000, 0.7, 1e-3)):
            want = sample_64(logits, uniform, [f32(T)] * 3, [k] * 3, [f32(p)] * 3, [f32(m)] * 3)[rows]
            got = ops.sample(logits.cuda()[rows.cuda()], uniform.cuda()[rows.cuda()], T, k, p, m)
            assert got.cpu().tolist() == want.tolist(), (T, k, p, m)


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [20, 500, 5000])
def test_sample_extreme_settings(device, V):
    """Temperatures near nothing and without end, settings that leave the first index, a top-k past any row."""
    g = gen(V + 4)
    logits = torch.randn(6, V, generator=g) * 4
    logits[1, 3] = math.inf
    logits[2, ::2] = logits[2].max()
    uniform = torch.tensor([0.0, 0.2, 0.5, 0.9, 1.0 - 2.0 ** -24, 0.7])
    for T in (1e-30, 1e-3, 1e30, 3e38):
        for k, p in ((0, 1.0), (5, 1.0), (0, 0.4), (V, 0.9)):
            check_sample(device, logits, uniform, T, k, p)
    first = logits.argmax(1).tolist()
    for name, v in (("temperature", -1.0), ("temperature", math.nan), ("top_p", 0.0), ("top_p", -3.0), ("top_p", math.nan), ("min_p", 1.5),
                    ("min_p", math.nan)):
        assert ops.sample(logits.to(device), uniform.to(device), **{name: torch.full((6,), v, device=device)}).tolist() == first
    for k in (2 ** 31 - 1, 2 ** 40, -5):
        top_k = torch.full((6,), k, dtype=torch.int64, device=device)
        assert ops.sample(logits.to(device), uniform.to(device), top_k=top_k).tolist() == ops.sample(logits.to(device), uniform.to(device)).tolist()


@pytest.mark.parametrize("device", CPU_AND_GPU)
@pytest.mark.parametrize("V", [5, 64, 65, 1000, 3000, 70001])
def test_sample_weights_of_nothing(device, V):
    """A number of 0 takes the first index that weighs anything: exp(-60) < 2^-86 does not, exp(-25) > 2^-37 does."""
    logits = torch.zeros(2, V)
    logits[:, V - 1] = 60.0
    logits[1, 1] = 35.0
    for settings in (dict(), dict(top_p=1 - 2.0 ** -24), dict(top_k=V)):
        assert ops.sample(logits.to(device), torch.zeros(2, device=device), **settings).tolist() == [V - 1, 1 if settings.get("top_p", 1) == 1 else V - 1]


# columns, their distance from the largest logit, top-p: what is kept ends 2 to 5 parts in 10^12 from a logit's border.  Rows with a list of what
# is open, rows that are searched, rows over blocks.
BORDERS = [(4001, 1 / 64, "0x1.5d5a720000000p-1"), (4006, 1 / 64, "0x1.8f47920000000p-3"), (4013, 3 / 64, "0x1.feda0c0000000p-1"),
           (4021, 3 / 64, "0x1.d30f020000000p-2"), (1831, 1 / 64, "0x1.7f17a20000000p-1"), (1830, 3 / 64, "0x1.0629680000000p-1"),
           (5005, 1 / 64, "0x1.365f9c0000000p-2"), (5006, 3 / 64, "0x1.3341f20000000p-3")]


@pytest.mark.parametrize("device,V,distance,p", [pytest.param(d, *case, marks=[pytest.mark.gpu] * (d == "cuda")) for d in ("cpu", "cuda") for case in BORDERS] + [
    pytest.param("cuda", *case, marks=pytest.mark.gpu) for case in ((70001, 1 / 64, "0x1.621fb00000000p-3"), (70002, 3 / 64, "0x1.de66740000000p-3"))])
def test_sample_nucleus_ends_where_the_weights_say(device, V, distance, p):
    """The largest logit first, the others equal.  Weights are whole numbers, so what top-p keeps is known exactly; the last of it is drawn.
    The limit's roundings: a weight's, at most 2^-46 of it at these sizes, a few of a double's, the 64-bit oracle's V 2^-53 on the CPU - in
    all less than 10^-12 of it, and the border is more than 2 10^-12 away."""
    shift = min(51, 62 - (V - 1).bit_length())
    first, each = 1 << shift, round(math.exp(-distance) * 2 ** shift)
    limit = Fraction(float.fromhex(p)) * (first + (V - 1) * each)
    kept = 1 + max(0, math.ceil((limit - first) / each))
    borders = [abs(1 - (first + n * each) / limit) for n in (kept - 2, kept - 1)]
    assert 2e-12 < min(borders) < 5e-12 and kept < V
    logits = torch.full((1, V), -distance)
    logits[0, 0] = 0.0
    uniform = torch.tensor([1 - 2.0 ** -24])  # (short of the whole by 2^-24 of it, less than the last weight)
    assert ops.sample(logits.to(device), uniform.to(device), top_p=float.fromhex(p)).item() == kept - 1


@pytest.mark.gpu
@pytest.mark.parametrize("B,V,top_p", [(1, 50000, 1.0), (3, 40000, 1.0), (20, 40000, 1.0), (1, 300000, 1.0), (1, 70000, 0.5), (2, 900, 0.5)])
def test_sample_negative_top_k_keeps_all(B, V, top_p):
    """The C entry point's top_k_all <= 0 keeps all, with the workspace that is asked for with the same number."""
    from difflut_amd import _native as nat

    lib, g = nat.lib(), gen(V)
    logits, uniform = torch.randn(B, V, generator=g).cuda(), torch.rand(B, generator=g).cuda()
    want = ops.sample(logits, uniform, top_p=top_p)
    for k in (-5, -1, 0, -2 ** 31):
        need = lib.dl_sample_workspace_bytes(B, V, k, top_p)
        space, out = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda"), torch.full((B,), -7, device="cuda")
        assert lib.dl_sample(logits.data_ptr(), V, 0, uniform.data_ptr(), None, None, None, None, 1.0, k, top_p, 0.0, out.data_ptr(),
                             space.data_ptr() if need else None, need, B, V, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, want), k


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_sample_strides_and_empty(device):
    g = gen(6)
    wide, uniform = torch.randn(8, 6000, generator=g), torch.rand(8, generator=g)
    for view in (lambda t: t[:, 1:50], lambda t: t[:, 3:], lambda t: t[:, ::2], lambda t: t.t()[:8, :8], lambda t: t[:1].expand(8, -1)):
        logits = view(wide.to(device))
        got = ops.sample(logits, uniform.to(device), top_k=20, top_p=0.8)
        assert got.cpu().tolist() == sample_64(view(wide), uniform, [1.0] * 8, [20] * 8, [f32(0.8)] * 8, [0.0] * 8).tolist()
    assert ops.sample(wide[:0].to(device), uniform[:0].to(device)).shape == (0,)


def test_sample_frequencies():
    """What is drawn for evenly spaced numbers has the softmax's frequencies to one part in their count."""
    logits = torch.tensor([0.0, 1.0, 2.0, -1.0])
    n = 4096
    tokens = ops.sample(logits.expand(n, -1), torch.arange(n) / n)
    assert (torch.bincount(tokens, minlength=4) / n - torch.softmax(logits, 0)).abs().max() <= 1 / n


# ----------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_refusals(device):
    w, t = torch.zeros(4, 3, device=device), torch.zeros(2, dtype=torch.long, device=device)
    x = torch.zeros(2, 5, 6, device=device)
    u = torch.zeros(2, device=device)
    logits = torch.zeros(2, 5, device=device)
    for error, call in [
            (ValueError, lambda: ops.embedding(t, w[0])), (ValueError, lambda: ops.embedding(t, w[:0])),
            (TypeError, lambda: ops.embedding(t.float(), w)), (TypeError, lambda: ops.embedding(t.short(), w)),
            (ValueError, lambda: ops.embedding(t, w, padding_idx=4)), (ValueError, lambda: ops.embedding(t, w, padding_idx=-1)),
            (TypeError, lambda: ops.embedding(t, w.int())), (TypeError, lambda: ops.embedding(t, w, scale=torch.ones(1, requires_grad=True))),
            (ValueError, lambda: ops.group_norm(x, 4)), (ValueError, lambda: ops.group_norm(x, 0)), (ValueError, lambda: ops.group_norm(x, 2.0)),
            (ValueError, lambda: ops.group_norm(x[:0], 2)), (ValueError, lambda: ops.group_norm(x[0, 0], 2)),
            (ValueError, lambda: ops.group_norm(x, 2, activation="tanh")), (ValueError, lambda: ops.group_norm(x, 2, eps=-1.0)),
            (ValueError, lambda: ops.group_norm(x, 2, w[0])), (ValueError, lambda: ops.group_norm(x, 2, None, w[0])),
            (TypeError, lambda: ops.group_norm(x.int(), 2)),
            (TypeError, lambda: ops.group_norm(x, 2, torch.ones(6, device=device), torch.ones(6, device=device).half())),
            (ValueError, lambda: ops.dropout(x, -0.1, (0, 0))), (ValueError, lambda: ops.dropout(x, 1.1, (0, 0))),
            (ValueError, lambda: ops.dropout(x, math.nan, (0, 0))), (ValueError, lambda: ops.dropout(x, 0.1, (0, 0), mode="noise")),
            (TypeError, lambda: ops.dropout(x, 0.1, t.int())), (TypeError, lambda: ops.dropout(x, 0.1, torch.zeros(3, dtype=torch.long, device=device))),
            (TypeError, lambda: ops.dropout(x.int(), 0.1, (0, 0))),
            (ValueError, lambda: ops.sample(logits[0], u)), (ValueError, lambda: ops.sample(logits[:, :0], u)),
            (ValueError, lambda: ops.sample(logits, u[:1])), (ValueError, lambda: ops.sample(logits, t)),
            (ValueError, lambda: ops.sample(logits, u, temperature=-1.0)), (ValueError, lambda: ops.sample(logits, u, temperature=math.nan)),
            (ValueError, lambda: ops.sample(logits, u, top_k=-1)), (ValueError, lambda: ops.sample(logits, u, top_k=1.5)),
            (ValueError, lambda: ops.sample(logits, u, top_p=0.0)), (ValueError, lambda: ops.sample(logits, u, top_p=1.5)),
            (ValueError, lambda: ops.sample(logits, u, min_p=1.5)), (TypeError, lambda: ops.sample(logits, u, top_k=u)), (ValueError, lambda: ops.sample(logits, u, top_p=u[:1]))]:
        with pytest.raises(error):
            call()


def test_c_entry_points_refuse():
    """Null pointers, unknown types and options, sizes that do not fit, short workspaces: an error before anything is launched."""
    from difflut_amd import _native as nat

    if not nat.is_built():
        pytest.skip("not built")
    lib = nat.lib()
    at, null, shape, unsupported, short = 4096, -1, -2, -3, -4  # (an address that is never followed)
    big = 1 << 40
    for want, call in [
            (unsupported, lambda: lib.dl_dropout(at, at, 7, 10, 0.5, 0, 0, 0, None, None, None)),
            (unsupported, lambda: lib.dl_dropout(at, at, 0, 10, 0.5, 2, 0, 0, None, None, None)),
            (shape, lambda: lib.dl_dropout(at, at, 0, -1, 0.5, 0, 0, 0, None, None, None)),
            (shape, lambda: lib.dl_dropout(at, at, 0, 10, 1.5, 0, 0, 0, None, None, None)),
            (shape, lambda: lib.dl_dropout(at, at, 0, 10, math.nan, 0, 0, 0, None, None, None)),
            (null, lambda: lib.dl_dropout(None, at, 0, 10, 0.5, 0, 0, 0, None, None, None)),
            (0, lambda: lib.dl_dropout(None, None, 0, 0, 0.5, 0, 0, 0, None, None, None)),
            (unsupported, lambda: lib.dl_embedding_fwd(at, 16, at, 8, at, 0, 4, 5, 8, 1.0, None)),
            (unsupported, lambda: lib.dl_embedding_fwd(at, 64, at, 8, at, 3, 4, 5, 8, 1.0, None)),
            (shape, lambda: lib.dl_embedding_fwd(at, 64, at, 7, at, 0, 4, 5, 8, 1.0, None)),
            (shape, lambda: lib.dl_embedding_fwd(at, 64, at, 8, at, 0, big, 5, 8, 1.0, None)),
            (shape, lambda: lib.dl_embedding_fwd(at, 64, at, 8, at, 0, 4, big, 8, 1.0, None)),
            (null, lambda: lib.dl_embedding_fwd(at, 64, None, 8, at, 0, 4, 5, 8, 1.0, None)),
            (null, lambda: lib.dl_embedding_bwd(at, 64, at, None, 0, 4, 5, 8, 1.0, -1, at, big, None)),
            (null, lambda: lib.dl_embedding_bwd(at, 64, None, at, 0, 4, 5, 8, 1.0, -1, at, big, None)),
            (null, lambda: lib.dl_embedding_bwd(at, 64, at, at, 0, 4000, 5, 8, 1.0, -1, None, big, None)),
            (short, lambda: lib.dl_embedding_bwd(at, 64, at, at, 0, 4000, 5, 8, 1.0, -1, at, lib.dl_embedding_bwd_workspace_bytes(4000, 5, 8) - 1, None)),
            (null, lambda: lib.dl_group_norm_fwd(at, at, at, at, None, 0, 0, 2, 3, 8, 2, 1e-5, 0, at, big, None)),
            (unsupported, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 9, 2, 3, 8, 2, 1e-5, 0, at, big, None)),
            (unsupported, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 0, 2, 3, 8, 2, 1e-5, 4, at, big, None)),
            (shape, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 0, 2, 3, 8, 3, 1e-5, 0, at, big, None)),
            (shape, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 0, 2, 3, 8, 2, -1.0, 0, at, big, None)),
            (shape, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 0, 2, big, 8, 2, 1e-5, 0, at, big, None)),
            (short, lambda: lib.dl_group_norm_fwd(at, at, at, at, at, 0, 0, 2, 3, 8, 2, 1e-5, 0, at, 8, None)),
            (null, lambda: lib.dl_group_norm_bwd(at, at, at, at, at, None, None, None, 0, 0, 2, 3, 8, 2, 0, at, big, None)),
            (short, lambda: lib.dl_group_norm_bwd(at, at, at, at, at, at, None, None, 0, 0, 2, 3, 8, 2, 0, at, 8, None)),
            (unsupported, lambda: lib.dl_sample(at, 8, 5, at, None, None, None, None, 1.0, 0, 1.0, 0.0, at, None, 0, 2, 8, None)),
            (shape, lambda: lib.dl_sample(at, 7, 0, at, None, None, None, None, 1.0, 0, 1.0, 0.0, at, None, 0, 2, 8, None)),
            (shape, lambda: lib.dl_sample(at, 8, 0, at, None, None, None, None, 1.0, 0, 1.0, 0.0, at, None, 0, 2, 0, None)),
            (null, lambda: lib.dl_sample(at, 8, 0, None, None, None, None, None, 1.0, 0, 1.0, 0.0, at, None, 0, 2, 8, None)),
            (null, lambda: lib.dl_sample(at, 1 << 20, 0, at, None, None, None, None, 1.0, 0, 0.5, 0.0, at, None, 0, 1, 1 << 20, None)),
            (short, lambda: lib.dl_sample(at, 1 << 20, 0, at, None, None, None, None, 1.0, 0, 0.5, 0.0, at, at, 8, 1, 1 << 20, None)),
            (0, lambda: lib.dl_sample(None, 8, 0, None, None, None, None, None, 1.0, 0, 1.0, 0.0, None, None, 0, 0, 8, None))]:
        assert call() == want
    assert lib.dl_group_norm_fwd_workspace_bytes(0, 2, 3, 8, 3) == 0 and lib.dl_embedding_bwd_workspace_bytes(-1, 5, 8) == 0


def test_embedding_gradient_refuses_vocabularies_that_the_sort_cannot_launch():
    """More than 2^30 rows would take 2^32 work items to sort for: refused before the first launch."""
    from difflut_amd import _native as nat

    if not nat.is_built():
        pytest.skip("not built")
    at, unsupported = 4096, -3  # (an address that is never followed)
    for V in (2 ** 30 + 1, 2 ** 31 - 1):
        for n in (513, 100000):
            for bits in (32, 64):
                assert nat.lib().dl_embedding_bwd(at, bits, at, at, 1, n, V, 16, 1.0, -1, at, 1 << 40, None) == unsupported


def test_rows_whose_last_columns_do_not_fit_32_bits_are_refused():
    """Features and channels near 2^31: a step past the last column would be a negative number."""
    from difflut_amd import _native as nat

    if not nat.is_built():
        pytest.skip("not built")
    lib, at, shape, big = nat.lib(), 4096, -2, 1 << 40  # (an address that is never followed)
    for D in (2 ** 31 - 1, 2 ** 31 - 1024, 2 ** 31 - 65536):
        assert lib.dl_embedding_fwd(at, 64, at, D, at, 1, 3, 1, D, 1.0, None) == shape
        for n in (3, 600):
            assert lib.dl_embedding_bwd(at, 64, at, at, 1, n, 1, D, 1.0, -1, at, big, None) == shape
        assert lib.dl_group_norm_fwd(at, at, at, at, at, 1, 1, 1, 1, D, 1, 1e-5, 0, at, big, None) == shape
        assert lib.dl_group_norm_bwd(at, at, at, at, at, at, None, None, 1, 1, 1, 1, D, 1, 0, at, big, None) == shape


def test_module_refusals():
    from difflut_amd.utils import Dropout, GroupNorm, TokenEmbedding

    for call in (lambda: TokenEmbedding(0, 4), lambda: TokenEmbedding(4, 0), lambda: TokenEmbedding(4, 4, padding_idx=4),
                 lambda: GroupNorm(3, 8), lambda: GroupNorm(0, 8), lambda: GroupNorm(2, 8, activation="gelu"),
                 lambda: Dropout(1.5), lambda: Dropout(0.5, mode="bits")):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_refusals_of_mixed_devices_float64_and_second_derivatives():
    w, t = torch.zeros(4, 3, device="cuda"), torch.zeros(2, dtype=torch.long)
    x = torch.randn(2, 5, 6, device="cuda")
    for call in (lambda: ops.embedding(t, w), lambda: ops.group_norm(x, 2, torch.ones(6)), lambda: ops.dropout(x, 0.5, t),
                 lambda: ops.sample(x[0], torch.zeros(5)), lambda: ops.sample(x[0], x[0, :, 0].abs(), top_p=torch.ones(5))):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: ops.embedding(t.cuda(), w.double()), lambda: ops.group_norm(x.double(), 2), lambda: ops.dropout(x.double(), 0.5, (0, 0)),
                 lambda: ops.sample(x[0].double(), x[0, :, 0].abs())):
        with pytest.raises(TypeError):
            call()
    for call, leaf in ((lambda v: ops.embedding(t.cuda(), v), w), (lambda v: ops.group_norm(v, 2), x)):
        leaf = leaf.clone().requires_grad_()
        y = call(leaf)
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)
    leaf = x.clone().requires_grad_()  # dropout is linear: its gradient has one of its own
    gy = torch.ones_like(x).requires_grad_()
    gx, = torch.autograd.grad(ops.dropout(leaf, 0.5, (1, 2)), leaf, gy, create_graph=True)
    gg, = torch.autograd.grad(gx, gy, torch.ones_like(gx))
    assert torch.equal(gg, gx.detach())


# ----------------------------------------------------------------------------- streams, graphs, a model
@pytest.mark.gpu
def test_on_another_stream():
    g = gen(12)
    w, t = torch.randn(50, 20, generator=g), torch.randint(0, 50, (300,), generator=g)
    x, logits, uniform = torch.randn(4, 200, 16, generator=g), torch.randn(3, 7000, generator=g), torch.rand(3, generator=g)

    def everything():
        leaf, xl = w.cuda().requires_grad_(), x.cuda().requires_grad_()
        y = ops.embedding(t.cuda(), leaf, 3.0)
        z = ops.dropout(ops.group_norm(xl, 4, activation="silu"), 0.2, (1, 2))
        return [y, *torch.autograd.grad(y, leaf, y.detach()), z, *torch.autograd.grad(z, xl, z.detach()),
                ops.sample(logits.cuda(), uniform.cuda(), 0.9, 100, 0.9)]

    want = everything()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = everything()
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_captured_and_replayed():
    """Every operator, forward and backward, in a graph: replays with new inputs against eager calls, eager work between them; the
    dropout module draws a new mask on every replay."""
    from difflut_amd.utils import Dropout

    g = gen(13)
    w, x = torch.randn(900, 64, generator=g).cuda().requires_grad_(), torch.randn(6, 300, 64, generator=g).cuda().requires_grad_()
    gamma, beta = torch.randn(64, generator=g).cuda().requires_grad_(), torch.randn(64, generator=g).cuda().requires_grad_()
    tokens, gy = torch.zeros(6, 300, dtype=torch.long, device="cuda"), torch.zeros(6, 300, 64, device="cuda")
    logits, uniform = torch.zeros(5, 9000, device="cuda"), torch.zeros(5, device="cuda")
    few = torch.zeros(5, 300, device="cuda")
    drop = Dropout(0.3, seed=4).cuda()

    def step():
        y = ops.embedding(tokens, w, 2.0)
        gw, = torch.autograd.grad(y, w, gy)
        z = ops.group_norm(x, 8, gamma, beta, activation="sigmoid")
        grads = torch.autograd.grad(z, [x, gamma, beta], gy)
        d = drop(x)
        gd, = torch.autograd.grad(d, x, gy)
        return [y, gw, z, *grads, d, gd, ops.sample(logits, uniform, 0.8, 300, 0.9, 0.001), ops.sample(few, uniform, 1.0, 0, 0.8)]

    def fill(seed):
        s = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            tokens.copy_((torch.rand(6, 300, generator=s, device="cuda") ** 4 * 900).long())
            gy.normal_(generator=s), logits.normal_(0, 2, generator=s), uniform.uniform_(generator=s), few.normal_(generator=s)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    masks = set()
    for replay in range(4):
        fill(replay)
        before = drop.state.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert drop.state.tolist() == [4, int(before[1]) + 1]
        drop.state.copy_(before)
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b), replay
        masks.add(int((got[6] == 0).long().mul(torch.arange(got[6].numel(), device="cuda").view(got[6].shape) % 997).sum()))
    assert len(masks) == 4


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_token_model_trains_and_answers(device):
    """Tokens -> embedding -> group norm with a sigmoid -> bit flips -> LUT layers -> GroupSum -> cross-entropy, every parameter's
    gradient; then one token at a time with sampling."""
    from difflut_amd.layers import RandomLayer
    from difflut_amd.nodes import NodeConfig, ProbabilisticNode
    from difflut_amd.nodes.utils import uniform_init
    from difflut_amd.utils import BankAdam, Dropout, GroupNorm, GroupSum, TokenEmbedding, cross_entropy, sample

    torch.manual_seed(5)
    V, D, T = 30, 24, 4
    node = NodeConfig(input_dim=4, output_dim=1, init_fn=uniform_init, init_kwargs={"a": -1.0, "b": 1.0})
    embed, norm = TokenEmbedding(V, D, scale=math.sqrt(D)).to(device), GroupNorm(4, D, activation="sigmoid").to(device)
    drop = Dropout(0.1, mode="flip", seed=1).to(device)
    layer = RandomLayer(T * D, 10 * V, ProbabilisticNode, node, seed=3).to(device)
    head = GroupSum(V, tau=2.0, use_randperm=False)
    parts = [embed, norm, drop, layer]

    def logits_of(tokens):
        h = norm(embed(tokens).movedim(-1, 1)).movedim(1, -1)
        assert h.shape == (*tokens.shape, D) and bool(((h > 0) & (h < 1)).all())
        return head(layer(drop(h.flatten(1))))

    tokens, targets = torch.randint(0, V, (16, T), device=device), torch.randint(0, V, (16,), device=device)
    leaves = [embed.weight, norm.weight, norm.bias, *layer.bank_parameters()]
    optimizer = BankAdam(leaves, lr=1e-2)
    for _ in range(2):
        loss = cross_entropy(logits_of(tokens), targets)
        optimizer.zero_grad()
        loss.backward()
        for p in leaves:
            assert p.grad is not None and p.grad.isfinite().all() and p.grad.any()
        optimizer.step()
    assert drop.state.tolist() == [1, 2]
    for m in parts:
        m.eval()
    g = gen(1)
    with torch.no_grad():
        for _ in range(5):
            nxt = sample(logits_of(tokens[:, -T:]), torch.rand(16, generator=g).to(device), temperature=0.8, top_k=10, top_p=0.9)
            assert nxt.shape == (16,) and bool(((nxt >= 0) & (nxt < V)).all())
            tokens = torch.cat([tokens, nxt.unsqueeze(1)], dim=1)


@pytest.mark.parametrize("device", CPU_AND_GPU)
def test_convolution_with_norm_and_flips(device):
    """ConvolutionalLayer -> GroupNorm with a sigmoid -> bit flips -> a second layer: the norm takes the layer's memory as it is."""
    from difflut_amd.layers import ConvolutionalLayer, ConvolutionConfig, RandomLayer
    from difflut_amd.nodes import DWNNode, NodeConfig
    from difflut_amd.nodes.utils import uniform_init
    from difflut_amd.utils import Dropout, GroupNorm

    torch.manual_seed(6)
    node = NodeConfig(input_dim=3, output_dim=1, init_fn=uniform_init, init_kwargs={"a": -1.0, "b": 1.0})
    conv = ConvolutionalLayer(ConvolutionConfig(tree_depth=1, in_channels=2, out_channels=8, receptive_field=3, seed=1), DWNNode, node,
                              RandomLayer, n_inputs_per_node=3).to(device)
    norm, drop = GroupNorm(2, 8, activation="sigmoid").to(device), Dropout(0.05, mode="flip").to(device)
    layer = RandomLayer(8 * 16, 20, DWNNode, node, seed=2).to(device)
    x = torch.rand(4, 2, 6, 6, device=device).requires_grad_()
    h = conv(x)
    assert h.movedim(1, -1).is_contiguous()
    y = layer(drop(norm(h)).flatten(1))
    y.sum().backward()
    assert x.grad.isfinite().all() and norm.weight.grad.any() and norm.bias.grad.any()
