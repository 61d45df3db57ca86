"""Operators of models over tokens and images of look-up-table layers, as cases that can be timed and compared.

A case is a dict of plain values; `kind` says which operator it is:

  embed    rows of a weight matrix by token, scaled; `train`: also the weight's gradient, summed token by token
  norm     group norm over channels-last activations with an activation behind it; `train`: also the gradients of the
           input, the weight and the bias
  drop     dropout from a counter-based generator: an entry becomes 0 (the others are scaled up), or, as the bit-flip
           augmentation of the LUT layers does, 1 - value, which the gradient ignores; `train`: also the input's gradient
  sample   one token per row of logits, with temperature, top-k, top-p and min-p, from given random numbers

`own` chooses between the plain form (elementary torch operations) and the framework's operators.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def _embed(name, train, dtype, T, V, D, tokens="zipf"):
    return {"name": name, "kind": "embed", "train": train, "dtype": dtype, "T": T, "V": V, "D": D, "tokens": tokens}


def _norm(name, train, dtype, B, H, W, C, G, act):
    return {"name": name, "kind": "norm", "train": train, "dtype": dtype, "B": B, "H": H, "W": W, "C": C, "G": G, "act": act}


def _drop(name, train, dtype, rows, cols, p, mode):
    return {"name": name, "kind": "drop", "train": train, "dtype": dtype, "rows": rows, "cols": cols, "p": p, "mode": mode}


def _sample(name, dtype, B, V, temperature, top_k, top_p, min_p, per_row=False, spread=3.0):
    return {"name": name, "kind": "sample", "dtype": dtype, "B": B, "V": V, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p, "per_row": per_row, "spread": spread}


def listed():
    return [
        # one decoding step of 64 sequences: their last tokens' rows, 784 features each; launch and host work only
        _embed("embed_step_t64", False, "fp32", 64, 32768, 784),
        # a training batch of 256 short sequences, token frequencies as text has them
        _embed("embed_train_t12544", True, "fp32", 12544, 16384, 784),
        # a long training batch over a large vocabulary, 16-bit weights, a ragged number of tokens
        _embed("embed_train_wide_bf16", True, "bf16", 65521, 131072, 1024),
        # one image's convolutional activations (32 channels of 24 x 24 positions) in an online request
        _norm("norm_one_image", False, "fp32", 1, 24, 24, 32, 8, "sigmoid"),
        # the convolutional layer's output in training: 256 images, 32 channels of 24 x 24 positions
        _norm("norm_conv_b256", True, "fp32", 256, 24, 24, 32, 8, "sigmoid"),
        # wide feature maps of odd size in 16 bits
        _norm("norm_wide_bf16", True, "bf16", 16, 95, 97, 320, 32, "silu"),
        # the thermometer code of the first training configuration (256 rows, 784 features of 4 bits), some bits flipped
        _drop("flip_code_b256", True, "fp32", 256, 3136, 0.1, "flip"),
        # a wide layer's activations in a large batch
        _drop("drop_b4096_bf16", True, "bf16", 4096, 16384, 0.2, "zero"),
        # one sequence's next token, every filter on
        _sample("sample_one_row", "bf16", 1, 49999, 0.8, 50, 0.95, 0.01),
        # labels drawn from a classifier's logits: a large batch of ten classes
        _sample("sample_classes_b8192", "fp32", 8192, 10, 1.0, 0, 0.9, 0.0, spread=1.0),
        # a batch of requests, each with settings of its own
        _sample("sample_requests_b64", "fp16", 64, 32768, 1.0, 40, 0.95, 0.02, per_row=True),
        # many sequences over a large vocabulary with the nucleus alone
        _sample("sample_wide_b256", "fp32", 256, 131072, 1.0, 0, 0.9, 0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "drop", "sample"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "embed":
        V, D = _log(rng, 100, 131072), _log(rng, 16, 1024)
        return _embed(None, rng.random() < 0.75, dtype, _log(rng, 1, 65536), V, D if rng.random() < 0.3 else max(16, D // 16 * 16),
                      rng.choice(["zipf", "zipf", "flat"]))
    if kind == "norm":
        G = rng.choice([1, 2, 4, 8, 16, 32])
        C = G * rng.randint(1, max(1, 512 // G))
        B, H, W = _log(rng, 1, 256), _log(rng, 1, 96), _log(rng, 1, 96)
        while H * W * (C // G) < 64:  # statistics of a handful of values are of no use to anybody
            H, W = 2 * H, W + 1
        while B * H * W * C > 30_000_000:
            B, H = max(1, B // 2), max(1, H - H // 3)
        return _norm(None, rng.random() < 0.75, dtype, B, H, W, C, G, rng.choice(["none", "silu", "sigmoid"]))
    if kind == "drop":
        rows, cols = _log(rng, 1, 4096), _log(rng, 10, 16384)
        return _drop(None, rng.random() < 0.75, dtype, rows, cols, round(rng.uniform(0.01, 0.9), 3), rng.choice(["zero", "zero", "flip"]))
    V = _log(rng, 2, 131072)
    B = max(1, min(_log(rng, 1, 8192), 30_000_000 // V))
    return _sample(None, dtype, B, V, round(rng.uniform(0.3, 1.5), 3), rng.choice([0, 0, 1, 5, 40, 200, 3000]),
                   rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), rng.choice([0.0, 0.0, 0.02, 0.1]), rng.random() < 0.3,
                   rng.choice([1.0, 3.0, 6.0]))


# ----------------------------------------------------------------------------- inputs
def _randn(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * std + mean).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    state = dict(case)
    if case["kind"] == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        u = torch.rand(T, generator=gen, device=DEVICE, dtype=torch.float64)
        # frequencies fall off as 1 / rank where tokens are those of text
        ids = (V + 1.0) ** u - 1.0 if case["tokens"] == "zipf" else u * V
        state["tokens"] = ids.long().clamp_(0, V - 1)
        state["weight"] = _randn(gen, (V, D), dtype, 1.0 / math.sqrt(D)).requires_grad_(case["train"])
        state["scale"] = math.sqrt(D)
        if case["train"]:
            state["gy"] = _randn(gen, (T, D), dtype, 1e-2)
    elif case["kind"] == "norm":
        C = case["C"]
        shape = (case["B"], case["H"], case["W"], C)
        state["x"] = _randn(gen, shape, dtype, 0.4, 0.5).requires_grad_(case["train"])
        state["weight"] = _randn(gen, (C,), dtype, 0.2, 1.0).requires_grad_(case["train"])
        state["bias"] = _randn(gen, (C,), dtype, 0.2).requires_grad_(case["train"])
        if case["train"]:
            state["gy"] = _randn(gen, shape, dtype)
    elif case["kind"] == "drop":
        shape = (case["rows"], case["cols"])
        if case["mode"] == "flip":  # a binary code
            state["x"] = (torch.rand(shape, generator=gen, device=DEVICE) < 0.5).to(dtype).requires_grad_(case["train"])
        else:
            state["x"] = _randn(gen, shape, dtype).requires_grad_(case["train"])
        state["seed"], state["offset"] = 0x5DEECE66D * (seed + 1) % (1 << 64), 1 + seed % 1000
        if case["train"]:
            state["gy"] = _randn(gen, shape, dtype)
    else:
        B = case["B"]
        state["logits"] = _randn(gen, (B, case["V"]), dtype, case["spread"])
        state["uniform"] = torch.rand(B, generator=gen, device=DEVICE)
        if case["per_row"]:  # every request's own settings, around the case's
            r = torch.rand((4, B), generator=gen, device=DEVICE)
            state["temperature"] = case["temperature"] * (0.5 + r[0])
            state["top_k"] = (case["top_k"] * 2 * r[1]).to(torch.int32)
            state["top_p"] = case["top_p"] + (1.0 - case["top_p"]) * (2 * r[2] - 1)
            state["min_p"] = case["min_p"] * 2 * r[3]
    return state


# ----------------------------------------------------------------------------- one pass
def run(state):
    kind, train = state["kind"], state.get("train", False)
    if not own:
        return {"embed": _plain_embed, "norm": _plain_norm, "drop": _plain_drop, "sample": _plain_sample}[kind](state)
    from difflut_amd import ops

    if kind == "embed":
        y = ops.embedding(state["tokens"], state["weight"], scale=state["scale"])
        return [y, *torch.autograd.grad(y, [state["weight"]], state["gy"])] if train else [y]
    if kind == "norm":
        leaves = [state["x"], state["weight"], state["bias"]]
        y = ops.group_norm(state["x"], state["G"], state["weight"], state["bias"], eps=1e-5, activation=state["act"])
        return [y, *torch.autograd.grad(y, leaves, state["gy"])] if train else [y]
    if kind == "drop":
        y = ops.dropout(state["x"], state["p"], (state["seed"], state["offset"]), mode=state["mode"])
        return [y, *torch.autograd.grad(y, [state["x"]], state["gy"])] if train else [y]
    return [ops.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"],
                       top_p=state["top_p"], min_p=state["min_p"])]


@torch.no_grad()
def _plain_embed(s):
    weight, tokens = s["weight"], s["tokens"]
    y = (weight[tokens].float() * s["scale"]).to(weight.dtype)
    if not s["train"]:
        return [y]
    gw = torch.zeros(weight.shape, device=weight.device).index_add_(0, tokens, s["gy"].float())
    return [y, (gw * s["scale"]).to(weight.dtype)]


@torch.no_grad()
def _plain_norm(s):
    x, B, C, G = s["x"], s["B"], s["C"], s["G"]
    xg = x.float().view(B, -1, G, C // G)
    mean = xg.mean((1, 3), keepdim=True)
    centred = xg - mean
    rstd = (centred.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    xhat = centred * rstd
    gamma, beta = s["weight"].float().view(G, C // G), s["bias"].float().view(G, C // G)
    z = xhat * gamma + beta
    if s["act"] == "sigmoid":
        y = 1 / (1 + torch.exp(-z))
        slope = y * (1 - y)
    elif s["act"] == "silu":
        sig = 1 / (1 + torch.exp(-z))
        y, slope = z * sig, sig * (1 + z * (1 - sig))
    else:
        y, slope = z, None
    y = y.view(x.shape).to(x.dtype)
    if not s["train"]:
        return [y]
    gz = s["gy"].float().view(xg.shape)
    gz = gz if slope is None else gz * slope
    gw, gb = (gz * xhat).sum((0, 1)).view(C), gz.sum((0, 1)).view(C)
    gh = gz * gamma
    gx = rstd * (gh - gh.mean((1, 3), keepdim=True) - xhat * (gh * xhat).mean((1, 3), keepdim=True))
    return [y, gx.view(x.shape).to(x.dtype), gw.to(x.dtype), gb.to(x.dtype)]


def _philox(seed, offset, numel, device):
    """[numel] words of the Philox 4x32 generator with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as
    easy as 1, 2, 3", 2011), word e % 4 of counter (e // 4, offset) under the key `seed`, as int64 values below 2^32."""
    low = 0xFFFFFFFF

    def product(a, m):  # high and low word of a 32 by 32 bit product, by halves: int64 has no room for all of it
        part = a * (m & 0xFFFF)
        upper = a * (m >> 16) + (part >> 16)
        return upper >> 16, ((upper & 0xFFFF) << 16) | (part & 0xFFFF)

    count = torch.arange(-(-numel // 4), dtype=torch.int64, device=device)
    c0, c1 = count & low, count >> 32
    c2, c3 = torch.full_like(count, offset & low), torch.full_like(count, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        high0, low0 = product(c0, 0xD2511F53)
        high1, low1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = high1 ^ c1 ^ k0, low1, high0 ^ c3 ^ k1, low0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], dim=1).view(-1)[:numel]


@torch.no_grad()
def _plain_drop(s):
    x, p = s["x"], s["p"]
    hit = (_philox(s["seed"], s["offset"], x.numel(), x.device) < int(math.floor(p * 2.0 ** 32 + 0.5))).view(x.shape)
    if s["mode"] == "flip":
        y = torch.where(hit, 1 - x.float(), x.float()).to(x.dtype)
        return [y, s["gy"]] if s["train"] else [y]
    scale = 1.0 / (1.0 - p)
    y = torch.where(hit, 0.0, x.float() * scale).to(x.dtype)
    return [y, torch.where(hit, 0.0, s["gy"].float() * scale).to(x.dtype)] if s["train"] else [y]


@torch.no_grad()
def _plain_sample(s):
    """In 64 bits: a token is drawn where a running sum passes a number, and neighbouring sums lie close together."""
    x = s["logits"].double()
    B, V = x.shape

    def setting(name):  # float32 values, like the random numbers
        v = s[name]
        return v.double().view(B, 1) if torch.is_tensor(v) else torch.full((B, 1), v, device=x.device).double()

    T, k, p, m = (setting(n) for n in ("temperature", "top_k", "top_p", "min_p"))
    x = torch.where(x.isnan(), -math.inf, x)
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = ordered[:, :1]
    w = torch.where(ordered == top, 1.0, torch.exp((ordered - top) / T))
    w = torch.where((ordered == top) | (T > 0), w, 0.0)
    rank = torch.arange(V, device=x.device)
    keep = (ordered > -math.inf) & ((rank < k) | (k <= 0))
    sums = torch.cumsum(w * keep, 1)
    before = torch.cat([torch.zeros_like(top), sums[:, :-1]], 1)
    keep &= (before < p * sums[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= (w >= m) | (rank == 0)
    kept = torch.zeros_like(x).scatter_(1, order, w * keep)
    running = torch.cumsum(kept, 1)
    total = running[:, -1:]
    u = torch.where(T > 0, s["uniform"].double().view(B, 1), 0.0)
    last = torch.where(kept > 0, rank, -1).amax(1)
    token = torch.minimum((running <= u * total).sum(1), last)
    return [torch.where(top.view(B) > -math.inf, token, -1)]


# ----------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_words(seed, offset, numel):
    """The generator's words by numpy's unsigned 64-bit products, a piece at a time."""
    out = np.empty(-(-numel // 4) * 4, dtype=np.uint32)
    words = out.reshape(-1, 4)
    m32, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    for start in range(0, len(words), 1 << 18):
        ctr = np.arange(start, min(start + (1 << 18), len(words)), dtype=np.uint64)
        c = [ctr & m32, ctr >> s32, np.full_like(ctr, offset & 0xFFFFFFFF), np.full_like(ctr, offset >> 32)]
        key = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> s32) ^ c[1] ^ np.uint64(key[0]), b & m32, (a >> s32) ^ c[3] ^ np.uint64(key[1]), a & m32]
            key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
        for j in range(4):
            words[start:start + len(ctr), j] = c[j]
    return out[:numel]


def exact(case, seed):
    if case["kind"] == "sample":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["kind"] == "embed":
        w, tokens = s["weight"].detach().double(), s["tokens"]
        y = w.index_select(0, tokens) * s["scale"]
        if not case["train"]:
            return [y]
        # a token's rows are neighbours once sorted: its sum is a difference of running sums, taken piece by piece
        order = torch.argsort(tokens, stable=True)
        gw = torch.zeros_like(w)
        for at in range(0, len(order), 4096):
            pos = order[at:at + 4096]
            ids, length = torch.unique_consecutive(tokens[pos], return_counts=True)
            run_ = torch.cumsum(s["gy"][pos].double(), 0)[torch.cumsum(length, 0) - 1]
            gw[ids] += torch.diff(run_, dim=0, prepend=torch.zeros_like(run_[:1]))
        return [y, gw * s["scale"]]
    if case["kind"] == "drop":
        if case["rows"] * case["cols"] > 70_000_000:
            return None
        words = _exact_words(s["seed"], s["offset"], case["rows"] * case["cols"])
        hit = torch.from_numpy(words < np.uint64(math.floor(case["p"] * 2.0 ** 32 + 0.5))).to(DEVICE).view(case["rows"], case["cols"])
        x = s["x"].detach().double()
        if case["mode"] == "flip":
            y = x + hit * (1 - 2 * x)
            return [y, s["gy"].double()] if case["train"] else [y]
        factor = (~hit).double() / (1.0 - case["p"])
        return [x * factor, s["gy"].double() * factor] if case["train"] else [x * factor]
    B, C, G = case["B"], case["C"], case["G"]
    leaves = [s[n].detach().double().requires_grad_(case["train"]) for n in ("x", "weight", "bias")]
    rows = leaves[0].reshape(B, -1, G, C // G).transpose(1, 2).reshape(B, G, -1)
    var, mean = torch.var_mean(rows, dim=2, unbiased=False, keepdim=True)
    hat = ((rows - mean) / torch.sqrt(var + 1e-5)).view(B, G, -1, C // G).transpose(1, 2).reshape(s["x"].shape)
    z = hat * leaves[1] + leaves[2]
    y = {"none": lambda: z, "sigmoid": lambda: torch.sigmoid(z), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
    if not case["train"]:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"].double())]


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = BYTES[case["dtype"]]
    if case["kind"] == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        moved = 8 * T + size * D * (min(T, V) + T)  # each row at most once, the outputs
        flops = T * D
        if case["train"]:
            moved, flops = moved + size * D * (T + V), flops + (T + V) * D
        return {"bytes": moved, "flops": flops}
    if case["kind"] == "norm":
        n = case["B"] * case["H"] * case["W"] * case["C"]
        if case["train"]:  # forward: x, y; backward: x, gy, gx
            return {"bytes": size * (5 * n + 6 * case["C"]), "flops": 35 * n}
        return {"bytes": size * (2 * n + 2 * case["C"]), "flops": 12 * n}
    if case["kind"] == "drop":
        n = case["rows"] * case["cols"]
        both = case["train"] and case["mode"] == "zero"  # a flip leaves the gradient as it is
        return {"bytes": size * n * (4 if both else 2), "flops": 30 * n * (2 if both else 1)}
    B, V = case["B"], case["V"]
    return {"bytes": size * B * V + (28 if case["per_row"] else 12) * B, "flops": 30 * B * V}
