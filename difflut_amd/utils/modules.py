"""GroupSum head (difflut/utils/modules.py:20-163): split the features into k contiguous groups
(zero-padded to a multiple of k), sum each group, divide by tau; its loss; and what stands around LUT layers in models over tokens and
in deep stacks (no counterpart in the reference): token embedding, group norm, counter-based dropout, sampling."""
import math
import warnings

import torch
import torch.nn as nn

from .. import ops
from .warnings import warn_default_value

DEFAULT_GROUPSUM_K = 1
DEFAULT_GROUPSUM_TAU = 1.0
DEFAULT_GROUPSUM_USE_RANDPERM = False


class GroupSum(nn.Module):
    def __init__(self, k=None, tau=None, use_randperm=None):
        super().__init__()
        if k is None:
            k = DEFAULT_GROUPSUM_K
            warn_default_value("k (GroupSum)", k, stacklevel=2)
        if tau is None:
            tau = DEFAULT_GROUPSUM_TAU
            warn_default_value("tau (GroupSum)", tau, stacklevel=2)
        if use_randperm is None:
            use_randperm = DEFAULT_GROUPSUM_USE_RANDPERM
            warn_default_value("use_randperm (GroupSum)", use_randperm, stacklevel=2)
        if not isinstance(k, int) or k <= 0:
            raise ValueError(f"k must be a positive integer, got {k}")
        if not isinstance(tau, (int, float)) or tau <= 0:
            raise ValueError(f"tau must be a positive number, got {tau}")
        self.k, self.tau, self.use_randperm = k, tau, use_randperm

    def forward(self, x):
        if x.dim() != 2:
            raise ValueError(f"GroupSum expects 2D input (batch_size, num_features), but got shape {x.shape} "
                             f"with {x.dim()} dimensions.")
        batch, features = x.shape
        if batch == 0:
            raise ValueError(f"GroupSum requires non-empty batch, got batch_size={batch}")
        if features == 0:
            raise ValueError(f"GroupSum requires non-zero features, got num_features={features}.")
        if features < self.k:
            warnings.warn(f"GroupSum input has fewer features ({features}) than output groups ({self.k}).",
                          UserWarning, stacklevel=2)
        if self.use_randperm:
            x = x[:, torch.randperm(features, device=x.device)]
        if features % self.k != 0:
            warnings.warn(f"GroupSum: Input has {features} features which is not divisible by k={self.k}. Adding "
                          f"{self.k - features % self.k} zero-padded features.", UserWarning, stacklevel=2)
        return ops.group_sum(x, self.k, self.tau)


def cross_entropy(logits, labels):
    """Mean cross-entropy of [batch, classes] logits (e.g. what GroupSum returns) against int64 class labels, loss and
    gradient from one pass on the device: a drop-in for `torch.nn.functional.cross_entropy(logits, labels)` with
    its default mean reduction (no class weights, no label smoothing, no ignore_index)."""
    return ops.cross_entropy(logits, labels)


class TokenEmbedding(nn.Module):
    """Rows of `weight` [num_tokens, features] by token, times `scale`: the first module of a model over tokens, in the place
    of an encoder.  The rows begin normally distributed with standard deviation 1 / sqrt(features).  Tokens outside [0, num_tokens)
    give zeros; `padding_idx` gets no gradient."""

    def __init__(self, num_tokens, features, scale=1.0, padding_idx=None):
        super().__init__()
        if not isinstance(num_tokens, int) or num_tokens <= 0 or not isinstance(features, int) or features <= 0:
            raise ValueError(f"num_tokens and features must be positive integers, got {num_tokens} and {features}")
        if padding_idx is not None and not 0 <= padding_idx < num_tokens:
            raise ValueError(f"padding_idx must be in [0, {num_tokens}), got {padding_idx}")
        self.num_tokens, self.features, self.scale, self.padding_idx = num_tokens, features, float(scale), padding_idx
        self.weight = nn.Parameter(torch.randn(num_tokens, features) / math.sqrt(features))

    def forward(self, tokens):
        return ops.embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return f"{self.num_tokens}, {self.features}, scale={self.scale}, padding_idx={self.padding_idx}"


class GroupNorm(nn.Module):
    """Group norm with an activation behind it ("none", "relu", "silu", "sigmoid") for [batch, channels] and
    [batch, channels, *positions] (the channel dimension second, as torch.nn.GroupNorm has it).  The work is done on channels-last
    memory, which is how ConvolutionalLayer leaves its output: such tensors are neither copied before nor after; others are
    copied once.  "sigmoid" brings activations to (0, 1) around the 1/2 that LUT nodes threshold at."""

    def __init__(self, groups, channels, eps=1e-5, affine=True, activation="none"):
        super().__init__()
        if not isinstance(groups, int) or not isinstance(channels, int) or groups <= 0 or channels <= 0 or channels % groups != 0:
            raise ValueError(f"groups must be a positive divisor of channels, got {groups} and {channels}")
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(ops.ACTIVATIONS)}, got {activation!r}")
        self.groups, self.channels, self.eps, self.activation = groups, channels, eps, activation
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(channels)) if affine else None

    def forward(self, x):
        if x.dim() < 2 or x.shape[1] != self.channels:
            raise ValueError(f"GroupNorm expects (batch, {self.channels}, ...), got {tuple(x.shape)}")
        y = ops.group_norm(x.movedim(1, -1), self.groups, self.weight, self.bias, self.eps, self.activation)
        return y.movedim(-1, 1)

    def extra_repr(self):
        return f"{self.groups}, {self.channels}, eps={self.eps}, affine={self.weight is not None}, activation={self.activation!r}"


class Dropout(nn.Module):
    """Dropout, or (mode "flip") bit flips in front of a layer, whose mask is drawn from (seed, number of the call) and never
    stored.  The pair is the int64 buffer `state`: it travels with the state dict, so a resumed run goes on with the same masks, and
    it is read and moved on by the device, so that every replay of a captured step draws a new mask.  In evaluation the
    input is returned as it is.  Without a `seed` one is drawn from torch's default generator, so that modules have noise of their own,
    and the same again after torch.manual_seed; where the state is the same (a seed given twice, a copied module, buffers broadcast from one
    data-parallel rank) the masks are.  A module is used on one stream at a time.
    Each forward moves the state on, also one that activation checkpointing runs again: `ops.dropout` with a pair of one's own
    is the call for that."""

    def __init__(self, p=0.5, mode="zero", seed=None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1], got {p}")
        if mode not in ops.DROP_MODES:
            raise ValueError(f"mode must be one of {list(ops.DROP_MODES)}, got {mode!r}")
        self.p, self.mode = p, mode
        if seed is None:
            seed = int(torch.randint(-(1 << 63), (1 << 63) - 1, (), dtype=torch.int64, device="cpu"))
        self.register_buffer("state", torch.tensor([ops._signed64(seed), 0], dtype=torch.int64))

    def forward(self, x):
        if not self.training:
            return x
        y = ops.dropout(x, self.p, self.state, self.mode)
        with torch.no_grad():
            self.state[1].add_(1)
        return y

    def extra_repr(self):
        return f"p={self.p}, mode={self.mode!r}"


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One class per row of logits [batch, classes] (e.g. what GroupSum returns), drawn with the random numbers `uniform` [batch]:
    see `ops.sample`."""
    return ops.sample(logits, uniform, temperature, top_k, top_p, min_p)
