"""Operators of the dense blocks between look-up-table layers in models over tokens, and of the search over their answers, as cases
that can be timed and compared.

A case is a dict of plain values; `kind` says which operator it is:

  norm     root-mean-square norm with the residual's addition in front of it; `train`: also the gradients of the two
           inputs and the weight; `codes`: the result in 8 bits (e4m3) with a scale per row
  linear   matrix product with bias, activation and residual; `train`: also the gradients of all of them; `codes`: both
           operands in 8 bits with a scale per row
  gated    activation of one projection times another one; `train` as above
  beam     a step of beam search: the best continuations over beams and vocabulary, and the states put in their order

`own` chooses between the plain form (elementary torch operations) and the framework's operators.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
CODES = torch.float8_e4m3fn
CODE_MAX = 448.0
EPS = 1e-6


def _norm(name, train, dtype, T, D, residual=True, codes=False):
    return {"name": name, "kind": "norm", "train": train, "dtype": dtype, "T": T, "D": D, "residual": residual, "codes": codes}


def _linear(name, train, dtype, M, K, N, act, bias=True, residual=False, codes=False):
    return {"name": name, "kind": "linear", "train": train, "dtype": dtype, "M": M, "K": K, "N": N, "act": act, "bias": bias,
            "residual": residual, "codes": codes}


def _gated(name, train, dtype, M, K, F, act="silu", bias=False):
    return {"name": name, "kind": "gated", "train": train, "dtype": dtype, "M": M, "K": K, "F": F, "act": act, "bias": bias}


def _beam(name, dtype, B, beams, V, D, spread=3.0, finished=0.0):
    return {"name": name, "kind": "beam", "dtype": dtype, "B": B, "beams": beams, "V": V, "D": D, "spread": spread, "finished": finished}


def listed():
    return [
        # one decoding step of 64 sequences, 784 features each; launch and host work only
        _norm("norm_step_t64", False, "fp32", 64, 784),
        # a long training batch in 16 bits
        _norm("norm_train_wide_bf16", True, "bf16", 65521, 1024),
        # the same batch in inference, handed on in 8 bits
        _norm("norm_codes_bf16", False, "bf16", 65521, 1024, codes=True),
        # logits of one sequence's next token over a large vocabulary
        _linear("linear_one_token", False, "bf16", 1, 1024, 131072, "none", bias=False),
        # the thermometer code's projection in front of a look-up-table layer: 784 features of 4 bits to 2000 values in (0, 1)
        _linear("linear_train_sigmoid", True, "fp32", 512, 3136, 2000, "sigmoid"),
        # the narrowing projection of a block back into its stream, in training
        _linear("linear_train_bf16", True, "bf16", 12544, 4096, 1024, "none", residual=True),
        # a wide layer's projection in inference on 8-bit operands
        _linear("linear_codes_wide", False, "bf16", 8192, 4096, 16384, "silu", codes=True),
        # one decoding step of 64 sequences through a gated projection
        _gated("gated_step_b64", False, "bf16", 64, 1024, 4096),
        # a training batch of 256 short sequences through the same projection
        _gated("gated_train_bf16", True, "bf16", 12544, 1024, 4096),
        # sizes of no particular alignment
        _gated("gated_train_ragged", True, "fp16", 2049, 1000, 2731, act="sigmoid", bias=True),
        # one request's search with four beams
        _beam("beam_one", "bf16", 1, 4, 49999, 1024),
        # many requests over a large vocabulary, some of their beams at an end already
        _beam("beam_wide_b64", "fp32", 64, 8, 131072, 4096, finished=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ragged(rng, n, step=16):
    """n as it is now and then, a multiple of `step` more often"""
    return n if rng.random() < 0.3 else max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["norm", "linear", "gated", "beam"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.6
    if kind == "norm":
        D = _ragged(rng, _log(rng, 16, 8192))
        T = max(1, min(_log(rng, 1, 65536), 60_000_000 // D))
        codes = not train and rng.random() < 0.5
        return _norm(None, train, dtype, T, D, rng.random() < 0.7, codes)
    if kind == "beam":
        beams, V = rng.randint(1, 16), _log(rng, 10, 131072)
        B = max(1, min(_log(rng, 1, 256), 60_000_000 // (beams * V)))
        return _beam(None, dtype, B, beams, V, _log(rng, 1, 4096), rng.choice([1.0, 3.0, 6.0]), rng.choice([0.0, 0.1, 0.5]))
    act = rng.choice(["none", "relu", "silu", "sigmoid"])
    M, K, N = _log(rng, 1, 16384), _ragged(rng, _log(rng, 16, 4096)), _ragged(rng, _log(rng, 10, 16384))
    while M * K * N > (100_000_000_000 if dtype != "fp32" else 20_000_000_000):
        M, N = max(1, M // 2), max(10, N - N // 4)
    if kind == "gated":
        return _gated(None, train, dtype, M, K, max(8, N // 2), act, rng.random() < 0.5)
    codes = not train and dtype != "fp32" and rng.random() < 0.4
    return _linear(None, train, dtype, M, _ragged(rng, K) if codes else K, N, act, rng.random() < 0.7, rng.random() < 0.4, codes)


# ----------------------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * std + mean).to(dtype)


def _coded(gen, rows, cols, std):
    """Rows of e4m3 values up to the type's largest, and the scales that make normally distributed rows of them"""
    x = torch.randn((rows, cols), generator=gen, device=DEVICE) * std
    scale = x.abs().amax(1) / CODE_MAX
    return (x / scale[:, None]).clamp_(-CODE_MAX, CODE_MAX).to(CODES), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, state, train = TYPES[case["dtype"]], dict(case), case.get("train", False)
    leaves = []

    def leaf(name, shape, std=1.0, mean=0.0):
        state[name] = _randn(gen, shape, dtype, std, mean).requires_grad_(train)
        leaves.append(name)

    if case["kind"] == "norm":
        leaf("x", (case["T"], case["D"]))
        if case["residual"]:
            leaf("res", (case["T"], case["D"]), 2.0)
        leaf("weight", (case["D"],), 0.2, 1.0)
        if train:
            state["gy"] = _randn(gen, (case["T"], case["D"]), dtype)
            if case["residual"]:
                state["gh"] = _randn(gen, (case["T"], case["D"]), dtype)
    elif case["kind"] == "beam":
        B, beams, V = case["B"], case["beams"], case["V"]
        state["logits"] = _randn(gen, (B, beams, V), dtype, case["spread"])
        state["scores"] = -5.0 * torch.rand((B, beams), generator=gen, device=DEVICE)
        state["ended"] = torch.rand((B, beams), generator=gen, device=DEVICE) < case["finished"]
        state["end"] = V // 2
        # what travels with a beam: its features, and the tokens so far
        state["states"] = [_randn(gen, (B, beams, case["D"]), dtype),
                           torch.randint(0, V, (B, beams, 64), generator=gen, device=DEVICE)]
    else:
        M, K = case["M"], case["K"]
        N = case["N"] if case["kind"] == "linear" else 2 * case["F"]
        out = (M, N) if case["kind"] == "linear" else (M, case["F"])
        if case.get("codes"):
            state["x"], state["x_scale"] = _coded(gen, M, K, 1.0)
            state["weight"], state["weight_scale"] = _coded(gen, N, K, 1.0 / math.sqrt(K))
        else:
            leaf("x", (M, K))
            leaf("weight", (N, K), 1.0 / math.sqrt(K))
        if case["bias"]:
            leaf("b", (N,), 0.5)
        if case.get("residual"):
            leaf("res", out)
        if train:
            state["gy"] = _randn(gen, out, dtype)
    state["leaves"] = leaves
    return state


# ----------------------------------------------------------------------------- one pass
def run(state):
    kind, train = state["kind"], state.get("train", False)
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "gated": _plain_gated, "beam": _plain_beam}[kind](state)
    from difflut_amd import ops

    if kind == "beam":
        scores, parents, tokens = ops.beam_step(state["logits"], state["scores"], finished=state["ended"], end=state["end"])
        return [scores, parents, tokens, *ops.beam_reorder(state["states"], parents)]
    if kind == "norm":
        if state["codes"]:
            return list(ops.rms_norm_codes(state["x"], state["weight"], eps=EPS, residual=state.get("res")))
        out = ops.rms_norm(state["x"], state["weight"], eps=EPS, residual=state.get("res"))
        outs, grads = (list(out), [state.get("gy"), state.get("gh")]) if state["residual"] else ([out], [state.get("gy")])
    else:
        if state.get("codes"):
            return [ops.linear_codes(state["x"], state["x_scale"], state["weight"], state["weight_scale"], state.get("b"),
                                     activation=state["act"], residual=state.get("res"), dtype=TYPES[state["dtype"]])]
        if kind == "linear":
            out = ops.linear(state["x"], state["weight"], state.get("b"), activation=state["act"], residual=state.get("res"))
        else:
            out = ops.gated_linear(state["x"], state["weight"], state.get("b"), activation=state["act"])
        outs, grads = [out], [state.get("gy")]
    if not train:
        return outs
    return [*outs, *torch.autograd.grad(outs, [state[n] for n in state["leaves"]], grads)]


@torch.no_grad()
def _plain_norm(s):
    x, weight = s["x"], s["weight"].float()
    dtype = x.dtype
    # the norm is that of the stream that is handed on: of the sum as its type holds it
    h = x if not s["residual"] else (x.float() + s["res"].float()).to(dtype)
    wide = h.float()
    rstd = (wide.square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = wide * rstd
    y = hat * weight
    if s["codes"]:
        scale = y.abs().amax(1) / CODE_MAX
        inverse = torch.where(scale > 0, 1 / scale, 0.0)
        outs = [(y * inverse[:, None]).clamp(-CODE_MAX, CODE_MAX).to(CODES), scale]
    else:
        outs = [y.to(dtype)]
    if s["residual"]:
        outs.append(h)
    if not s["train"]:
        return outs
    gy = s["gy"].float()
    g = gy * weight
    gx = rstd * (g - hat * (g * hat).mean(1, keepdim=True))
    if s["residual"]:
        gx = gx + s["gh"].float()
    gx, gw = gx.to(dtype), (gy * hat).sum(0).to(dtype)
    return [*outs, gx, gx, gw] if s["residual"] else [*outs, gx, gw]


def _act(z, act):
    """The activation's value and slope"""
    if act == "relu":
        return z.clamp(min=0), (z > 0).float()
    if act == "none":
        return z, torch.ones_like(z)
    sig = 1 / (1 + torch.exp(-z))
    return (sig, sig * (1 - sig)) if act == "sigmoid" else (z * sig, sig * (1 + z * (1 - sig)))


def _operands(s):
    x, w = s["x"].float(), s["weight"].float()
    return (x * s["x_scale"][:, None], w * s["weight_scale"][:, None]) if s.get("codes") else (x, w)


def _plain_grads(s, x, w, gz):
    """Gradients in the order of the leaves, from that of the product"""
    of = {"x": lambda: gz @ w, "weight": lambda: gz.t() @ x, "b": lambda: gz.sum(0), "res": lambda: s["gy"]}
    return [of[n]().to(s["gy"].dtype) for n in s["leaves"]]


@torch.no_grad()
def _plain_linear(s):
    x, w = _operands(s)
    z = x @ w.t()
    if s["bias"]:
        z = z + s["b"].float()
    y, slope = _act(z, s["act"])
    if s["residual"]:
        y = y + s["res"].float()
    y = y.to(TYPES[s["dtype"]])
    return [y, *_plain_grads(s, x, w, s["gy"].float() * slope)] if s["train"] else [y]


@torch.no_grad()
def _plain_gated(s):
    x, w = _operands(s)
    z = x @ w.t()
    if s["bias"]:
        z = z + s["b"].float()
    gate, up = z[:, :s["F"]], z[:, s["F"]:]
    a, slope = _act(gate, s["act"])
    y = (a * up).to(TYPES[s["dtype"]])
    if not s["train"]:
        return [y]
    gy = s["gy"].float()
    return [y, *_plain_grads(s, x, w, torch.cat([gy * up * slope, gy * a], 1))]


@torch.no_grad()
def _plain_beam(s):
    """In 64 bits: neighbouring candidates of different beams lie close together. The best of all are among the best of each beam."""
    x, before, ended, end = s["logits"].double(), s["scores"].double(), s["ended"], s["end"]
    B, beams, V = x.shape
    top = x.amax(2, keepdim=True)
    norm = top + torch.exp(x - top).sum(2, keepdim=True).log()
    most = min(beams, V)
    ordered, order = torch.sort(x, dim=2, descending=True, stable=True)
    value, token = before[:, :, None] + (ordered[:, :, :most] - norm), order[:, :, :most]
    # a beam that has ended goes on as it is, by one candidate
    rank = torch.arange(most, device=x.device)
    value = torch.where(ended[:, :, None], torch.where(rank == 0, before[:, :, None], -math.inf), value)
    token = torch.where(ended[:, :, None], end, token)
    # equal values in the order of beam and token: beams lie in order, and so do equal logits of one
    value, pick = torch.sort(value.view(B, -1), dim=1, descending=True, stable=True)
    value, pick = value[:, :beams], pick[:, :beams]
    parents, tokens = pick // most, token.reshape(B, -1).gather(1, pick)
    lost = value == -math.inf
    parents, tokens = torch.where(lost, 0, parents), torch.where(lost, -1, tokens)
    rows = torch.arange(B, device=x.device)[:, None]
    return [value.float(), parents, tokens, *(t[rows, parents] for t in s["states"])]


# ----------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_act(z, act):
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "sigmoid": lambda: torch.sigmoid(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "beam":
        total = torch.log_softmax(s["logits"].double(), 2) + s["scores"].double()[:, :, None]
        alone = torch.full_like(total, -math.inf)
        alone[:, :, s["end"]] = s["scores"].double()
        total = torch.where(s["ended"][:, :, None], alone, total).flatten(1)
        best = torch.topk(total, min(case["beams"], total.shape[1]), dim=1).values
        return [best, None, None, None, None]  # whole numbers, and inputs that only move
    train = case["train"]
    leaves = {n: s[n].detach().double().requires_grad_(train) for n in s["leaves"]}
    if case["kind"] == "norm":
        h = leaves["x"]
        if case["residual"]:
            h = h + leaves["res"]
            kept = h.detach().to(s["x"].dtype).double()  # what the stream holds, with the sum's gradient
            h = h + (kept - h.detach())
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["D"] + EPS) * leaves["weight"]
        if case["codes"]:
            scale = torch.linalg.vector_norm(y, math.inf, dim=1) / CODE_MAX
            # (codes are steps: what they stand for without the rounding is no value of theirs)
            outs, grads = [None, scale.detach()], []
        else:
            outs, grads = [y], [s.get("gy")]
        if case["residual"]:
            outs.append(h.detach() if case["codes"] else h)
            grads.append(s.get("gh"))
    else:
        if case.get("codes"):
            x, w = s["x"].double() * s["x_scale"].double()[:, None], s["weight"].double() * s["weight_scale"].double()[:, None]
        else:
            x, w = leaves["x"], leaves["weight"]
        if case["kind"] == "linear":
            z = torch.matmul(x, w.t()) if not case["bias"] else torch.addmm(leaves["b"], x, w.t())
            y = _exact_act(z, case["act"])
            y = y + leaves["res"] if case["residual"] else y
        else:
            halves = [torch.matmul(x, part.t()) for part in w.split(case["F"])]
            if case["bias"]:
                halves = [h + b for h, b in zip(halves, leaves["b"].split(case["F"]))]
            y = _exact_act(halves[0], case["act"]) * halves[1]
        outs, grads = [y], [s.get("gy")]
    if not train:
        return [o if o is None else o.detach() for o in outs]
    return [*(o.detach() for o in outs), *torch.autograd.grad(outs, list(leaves.values()), [g.double() for g in grads])]


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "norm":
        T, D, res = case["T"], case["D"], 1 if case["residual"] else 0
        n = T * D
        if case["codes"]:
            return {"bytes": size * (n * (1 + 2 * res) + D) + n + 4 * T, "flops": 10 * n}
        if not case["train"]:
            return {"bytes": size * (n * (2 + 2 * res) + D), "flops": 6 * n}
        # forward: x and the residual, y and their sum; backward: the sum, the gradients of both results, that of the inputs
        return {"bytes": size * (n * (5 + 3 * res) + 2 * D), "flops": 18 * n}
    if case["kind"] == "beam":
        B, beams, V = case["B"], case["beams"], case["V"]
        moved = 2 * B * beams * (size * case["D"] + 8 * 64)
        return {"bytes": size * B * beams * V + moved + 25 * B * beams, "flops": 8 * B * beams * V}
    M, K = case["M"], case["K"]
    N = case["N"] if case["kind"] == "linear" else 2 * case["F"]
    out = M * (N if case["kind"] == "linear" else case["F"])
    res = out if case.get("residual") else 0
    if case.get("codes"):
        return {"bytes": (M + N) * (K + 4) + size * (out + res + (N if case["bias"] else 0)), "flops": 2 * M * N * K}
    elements = M * K + N * K + out + res + (N if case["bias"] else 0)
    if not case["train"]:
        return {"bytes": size * elements, "flops": 2 * M * N * K}
    # the products' values of a curved activation are read again, the gradients written
    kept = 0 if case["kind"] == "linear" and case["act"] == "none" else M * N
    elements += 2 * kept + out + 2 * (M * K + N * K) + (N if case["bias"] else 0) + res
    return {"bytes": size * elements, "flops": 6 * M * N * K}
