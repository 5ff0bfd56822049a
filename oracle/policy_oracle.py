"""The policy operators in 64 bits on the CPU: the delta rule step by step, the gated feed-forward and the block norms,
with torch's derivatives of these definitions. Test infrastructure only."""
from __future__ import annotations

import math

import torch


def delta_rule(q, k, v, g, beta, state=None, reset=None, scale=None):
    """As isaac_net_amd.delta_rule, in float64, one step after the other; a memory that is emptied holds zeros."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    rep = H // Hk
    scale = K ** -0.5 if scale is None else scale
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if state is None else state.double()
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    q, k = q.repeat_interleave(rep, 2), k.repeat_interleave(rep, 2)
    out = []
    for t in range(T):
        empty = g[:, t] < -104.0
        if reset is not None:
            empty = empty | (reset[:, t] != 0)[:, None]
        d = torch.where(empty, torch.zeros_like(g[:, t]), torch.exp(torch.where(empty, torch.zeros_like(g[:, t]), g[:, t])))
        S = torch.where(empty[..., None, None], torch.zeros_like(S), d[..., None, None] * S)
        e = v[:, t] - (S * k[:, t, :, :, None]).sum(-2)
        S = S + (beta[:, t, :, None] * k[:, t])[..., None] * e[..., None, :]
        out.append(scale * (S * q[:, t, :, :, None]).sum(-2))
    return torch.stack(out, 1) if out else v.new_zeros(B, 0, H, V), S


def gated_ffn(x, w_gate, w_up, activation="silu"):
    x, w_gate, w_up = x.double(), w_gate.double(), w_up.double()
    a = x @ w_gate.T
    if activation == "silu":
        h = a * torch.sigmoid(a)
    elif activation == "gelu":
        h = 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)))
    else:
        h = torch.where(a <= 0, torch.zeros_like(a), a)          # (NaN stays)
    return h * (x @ w_up.T)


def block_norm(x, f=None, gate=None, scale=None, post_weight=None, pre_weight=None, eps=1e-6):
    norm = lambda z: z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)  # noqa: E731
    y = x.double()
    if f is not None:
        h = f.double()
        if post_weight is not None:
            h = norm(h) * post_weight.double()
        for m in (gate, scale):
            if m is not None:
                h = h * m.double()
        y = y + h
    return y, None if pre_weight is None else norm(y) * pre_weight.double()
