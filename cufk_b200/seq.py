"""Operators of a model along chains: what reads tokens and speaks in torsions next to their reconstruction.

The reconstruction takes what a model says about a chain and returns its coordinates; these are the operators that such a
model is made of, over the same packed chains: a short causal convolution and a selective scan (an affine recurrence per
channel, as the reconstruction is one per chain), their single-token steps for chains that grow row by row, log
probabilities of the tokens (torsion bins, fragments) that it answers with, and gradient clipping by the global norm, which
the lever arm of a chain makes a necessity (a dihedral at its start moves every later atom).  The reference has none of
them.  Each is a hand-written sm_100a kernel behind the C ABI of ``include/cufkb_seq.h``.

Rows and chains.  Activations are ``(rows, width)`` with ``chain_points``, the ``(chains + 1,)`` int64 offsets of the
chains on the device (a chain may be empty; rows past the last offset are padding, whose results and gradients are zero);
``(chains, length, width)``; or ``(rows, width)`` for one chain.  Columns are contiguous, rows may have any stride (a slice
of a wider projection is read in place; rows of a scan that are more than 2^24 elements apart are copied first).  They are float32, float16 or bfloat16, computed in float32 and rounded once on
output; parameters, scan states and their gradients are float32.  ``chain_points`` stays on the device and is not
checked there beyond what keeps every access inside the arrays: it must start at 0 and not decrease.

Gradients are first derivatives: under ``create_graph`` they are the same, and differentiating them again is an error.

All calls run on the current stream and never synchronise with the host.  Sums over rows, channels and arrays are taken in an
order that depends on sizes and on the alignment of the arrays alone, so results of the same call repeat bit by bit.  Exponentials are the
hardware's, good to 2^-22; in chains of up to 16384 rows the last states and the gradient of A were off by less than 1e-6 of their norms.

These are plain functions of the extension, not ``torch.library`` operators like those of ``cufk_b200.ops``: ``torch.compile`` breaks its
graph at them.  CUDA graphs capture them.
"""

from __future__ import annotations

from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from ._native import _C

__all__ = [
    "TokenLogprobs",
    "clip_gradients",
    "selective_scan",
    "selective_scan_step",
    "short_conv",
    "short_conv_step",
    "token_logprobs",
]


def short_conv(
    x: Tensor,
    weight: Tensor,
    bias: Tensor | None = None,
    *,
    chain_points: Tensor | None = None,
    initial_state: Tensor | None = None,
    silu: bool = True,
    return_state: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    r"""Causal convolution of each channel with its own filter of 2 to 4 taps, along packed chains.

    ``pre[t] = bias + sum_k weight[:, k] x[t - taps + 1 + k]`` within a chain, and ``y = pre * sigmoid(pre)`` (``silu``) or ``pre``.

    Args:
        x: ``(rows, width)`` or ``(chains, length, width)``.
        weight: ``(width, taps)`` float32; the last tap meets the row itself.
        bias: ``(width,)`` float32.
        chain_points: offsets of packed chains (see the module's notes).
        initial_state: ``(chains, taps - 1, width)`` in the dtype of ``x``: the rows before each chain's first, oldest first;
            zero when omitted.
        return_state: also return the last ``taps - 1`` rows of each chain (of the initial state, where the chain is shorter),
            which ``short_conv_step`` continues from.

    Returns:
        ``y`` in the shape and dtype of ``x``, or ``(y, state)``.  Gradients flow to ``x``, ``weight``, ``bias`` and
        ``initial_state``, from both results.
    """
    out = _C.short_conv(x, weight, bias, chain_points, initial_state, silu, return_state)
    return (out[0], out[1]) if return_state else out[0]


def short_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Tensor | None = None, *, silu: bool = True) -> Tensor:
    r"""One more row of every chain: ``short_conv`` of ``x`` ``(chains, width)`` after the rows in ``state``.

    ``state``, ``(chains, taps - 1, width)`` contiguous in the dtype of ``x``, is updated in place: its oldest row leaves, ``x`` is
    its newest.  No gradients: with grad mode on, an argument that asks for one is refused.
    """
    return _C.short_conv_step(x, state, weight, bias, silu)


def selective_scan(
    x: Tensor,
    delta: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    delta_bias: Tensor | None = None,
    *,
    delta_softplus: bool = True,
    chain_points: Tensor | None = None,
    initial_state: Tensor | None = None,
    return_state: bool = False,
) -> Tensor | tuple[Tensor, Tensor]:
    r"""Selective scan along packed chains.

    Per channel d and state n, with ``dt = softplus(delta + delta_bias)`` (or ``delta + delta_bias``)::

        h_t = exp(dt_t A[d, n]) h_{t-1} + dt_t x_t B_t[n]
        y_t = (sum_n C_t[n] h_t[n] + D[d] x_t) * z_t sigmoid(z_t)

    Args:
        x, delta, z: ``(rows, width)`` or ``(chains, length, width)``; ``z`` (the gate) may be omitted.
        A: ``(width, states)`` float32, 1 to 64 states, negative for decay.
        B, C: ``(rows, states)``, or ``(rows, groups, states)`` where each group serves ``width / groups`` consecutive channels
            (``(chains, length, ...)`` with a three-dimensional ``x``), in the dtype of ``x``.
        D, delta_bias: ``(width,)`` float32.
        chain_points: offsets of packed chains (see the module's notes).
        initial_state: ``(chains, width, states)`` float32, the state before each chain's first row; zero when omitted.
        return_state: also return each chain's last state, which ``selective_scan_step`` continues from.

    Returns:
        ``y`` in the shape and dtype of ``x``, or ``(y, state)``.  Gradients flow to every floating argument, from both results.
        When one is asked for, the forward keeps the state every 8 rows (``width * states / 2`` bytes per row, states rounded up to 8, 16, 32 or 64), and
        the backward's workspace holds ``width * states**2 / 128`` more (partial sums for B and C).
    """
    out = _C.selective_scan(x, delta, A, B, C, D, z, delta_bias, chain_points, initial_state, delta_softplus, return_state)
    return (out[0], out[1]) if return_state else out[0]


def selective_scan_step(
    x: Tensor,
    delta: Tensor,
    A: Tensor,
    B: Tensor,
    C: Tensor,
    state: Tensor,
    D: Tensor | None = None,
    z: Tensor | None = None,
    delta_bias: Tensor | None = None,
    *,
    delta_softplus: bool = True,
) -> Tensor:
    r"""One more row of every chain: ``selective_scan`` of ``(chains, width)`` rows from ``state``.

    ``B`` and ``C`` are ``(chains, states)`` or ``(chains, groups, states)``.  ``state``, ``(chains, width, states)`` contiguous
    float32, is updated in place.  No gradients: with grad mode on, an argument that asks for one is refused.
    """
    return _C.selective_scan_step(x, delta, A, B, C, state, D, z, delta_bias, delta_softplus)


class TokenLogprobs(NamedTuple):
    logp: Tensor
    entropy: Tensor
    top_logp: Tensor
    top_tokens: Tensor


def token_logprobs(logits: Tensor, tokens: Tensor, *, top: int = 0) -> TokenLogprobs:
    r"""Log probabilities of given tokens under ``softmax(logits)``, each row's entropy, and its likeliest tokens.

    Args:
        logits: ``(..., tokens)`` float32, float16 or bfloat16; ``-inf`` rules a token out.
        tokens: ``(...)`` int64.  A negative token means "none here": its log probability is 0 and passes no gradient.  One
            past the last gives NaN.
        top: how many of the likeliest tokens to return, 0 to 32: largest logit first, equal ones by lower id (NaN counts as
            largest).

    Returns:
        ``(logp, entropy, top_logp, top_tokens)``: ``(...)`` and ``(..., top)``, float32 and int64.  ``logp`` and ``entropy``
        (natural logarithms) pass gradients to ``logits``; the alternatives do not.  A row that rules out every token has
        log probabilities ``-inf``, entropy 0 and no gradient.
    """
    return TokenLogprobs(*_C.token_logprobs(logits, tokens, top))


def clip_gradients(grads: Sequence[Tensor], max_norm: float, *, out: Sequence[Tensor] | None = None, eps: float = 1e-6) -> Tensor:
    r"""Scales gradients so that their global norm is at most ``max_norm``: ``g * min(1, max_norm / (norm + eps))``.

    Args:
        grads: CUDA tensors of any of the four dtypes, mixed at will, on one device.  Empty ones are allowed.
        max_norm: largest norm; ``inf`` only measures it and leaves the values as they are, whatever the norm.
        out: where the clipped gradients go, one tensor of equal shape and dtype per gradient; the gradients themselves
            when omitted (which are then not written at all where nothing needs clipping).
            A gradient that is listed twice (that of both terms of a sum, say) counts twice in the norm and is scaled once;
            apart from that, what is written for one may not be read or written for another.
            An expanded gradient (of a sum, say) needs an output of its own.

    Returns:
        The norm before clipping, a 0-d tensor on the device: float32, or float64 when some gradient is.  Squares are summed
        in float64.  With a finite ``max_norm`` a NaN norm makes every gradient NaN, and an infinite one makes the finite ones zero.
    """
    grads = list(grads)
    return _C.clip_gradients(grads, float(max_norm), float(eps), grads if out is None else list(out))
