"""The measured operators of the learning loop: what a recurrent robot policy computes between two control steps.

The engines give a batch of robots their step outputs; the policy beside them turns those into the next messages and is
trained on windows of what it saw. A robot is one row of the batch (E envs x R robots), its memory one matrix a head.

  step    delta_rule_step: one control step of every robot's memory, the state updated in place (a rollout)
  window  delta_rule: a window of T control steps of every robot, from the state that its rollout held, with episode
          ends inside (training, or a forward pass alone)
  ffn     gated_ffn: both projections, the activation and the product
  norm    block_norm: the norm after a block, its gate and residual scale, and the norm before the next

`own` false: the operators in their plain form, elementary torch operations in 32 bits rounded once at the end, with
torch's own derivatives. `own` true: the package's operators.

Batches come from the framework's configurations: 64 x 8 (its debugging batch), 256 x 16, 1024 x 16, 4096 x 32 (its
headline workload); the window of 24 steps, head sizes and widths are generic.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def _package():
    """The package (its folder's name is no identifier), from the working folder."""
    if "isaac_net_amd" not in sys.modules:
        d = os.path.join(os.getcwd(), "isaac-net_amd")
        spec = importlib.util.spec_from_file_location("isaac_net_amd", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["isaac_net_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["isaac_net_amd"]


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a rollout of the debugging batch (64 envs x 8 robots): launches and latency only
        {"name": "step_512", "op": "step", "B": 512, "Hk": 2, "H": 2, "K": 32, "V": 32, "dtype": "f32", "end": 0.01},
        # a rollout of the headline workload (4096 envs x 32 robots), two heads of 64 x 64: the state is 4.3 GB
        {"name": "step_131072", "op": "step", "B": 131072, "Hk": 2, "H": 2, "K": 64, "V": 64, "dtype": "bf16",
         "end": 0.005},
        # a training batch: 1024 envs x 16 robots, windows of 24 steps, episode ends inside, the rollout's state given
        {"name": "window_16384x24", "op": "window", "B": 16384, "T": 24, "Hk": 2, "H": 2, "K": 64, "V": 64,
         "dtype": "bf16", "end": 0.02, "state": "given", "train": True},
        # truncated backpropagation carried over windows: a gradient into and out of the state, shared query and key
        # heads, sizes that fill no tile, 32-bit values
        {"name": "window_300x77_f32", "op": "window", "B": 300, "T": 77, "Hk": 2, "H": 6, "K": 40, "V": 56,
         "dtype": "f32", "end": 0.03, "state": "grad", "train": True},
        # whole episodes of a few robots: a long axis with few rows
        {"name": "window_2x4096", "op": "window", "B": 2, "T": 4096, "Hk": 8, "H": 8, "K": 64, "V": 64,
         "dtype": "bf16", "end": 0.0, "state": "none", "train": True},
        # large heads
        {"name": "window_4x2048_d128", "op": "window", "B": 4, "T": 2048, "Hk": 4, "H": 8, "K": 128, "V": 128,
         "dtype": "bf16", "end": 0.001, "state": "none", "train": True},
        # a small policy's rollout
        {"name": "ffn_512x128", "op": "ffn", "N": 512, "D": 128, "F": 344, "dtype": "bf16", "act": "silu",
         "train": False},
        # a training minibatch in float16, widths that fill no tile
        {"name": "ffn_16383x504", "op": "ffn", "N": 16383, "D": 504, "F": 1352, "dtype": "f16", "act": "gelu",
         "train": True},
        # a training step over every robot of the headline workload
        {"name": "ffn_131072x512", "op": "ffn", "N": 131072, "D": 512, "F": 2048, "dtype": "bf16", "act": "silu",
         "train": True},
        # a small policy's rollout
        {"name": "norm_512x128", "op": "norm", "N": 512, "D": 128, "dtype": "bf16", "gate": "full", "train": False},
        # 32-bit values, a gate for each robot, a width of no power of two
        {"name": "norm_5001x999_f32", "op": "norm", "N": 5001, "D": 999, "dtype": "f32", "gate": "row", "train": True},
        # a training step over every robot of the headline workload
        {"name": "norm_131072x512", "op": "norm", "N": 131072, "D": 512, "dtype": "bf16", "gate": "full",
         "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _head(rng):
    return rng.choice((16, 24, 32, 40, 48, 64, 64, 64, 96, 128))


def draw(rng):
    op = rng.choice(("step", "window", "window", "window", "ffn", "ffn", "norm"))
    if op == "step":
        Hk, K, V = rng.choice((1, 2, 2, 4)), _head(rng), _head(rng)
        H = Hk * rng.choice((1, 1, 2))
        return {"op": op, "B": min(_log(rng, 8, 131072), 131072 * 2 * 4096 // (H * K * V)), "Hk": Hk, "H": H, "K": K,
                "V": V, "dtype": rng.choice(("bf16", "bf16", "f32")), "end": rng.choice((0.0, 0.005))}
    if op == "window":
        Hk, K, V = rng.choice((1, 2, 4)), _head(rng), _head(rng)
        H, T = Hk * rng.choice((1, 1, 2, 3)), _log(rng, 2, 4096)
        most = 16384 * 24 * 2 * 4096 // (2 * T * H * K * V)
        return {"op": op, "B": max(1, min(_log(rng, 1, 16384), most)), "T": T, "Hk": Hk, "H": H, "K": K, "V": V,
                "dtype": rng.choice(("bf16", "bf16", "bf16", "f32")), "end": rng.choice((0.0, 0.002, 0.02)),
                "state": rng.choice(("given", "grad", "none")), "train": rng.random() < 0.7}
    if op == "ffn":
        D, F = 8 * _log(rng, 8, 128), 8 * _log(rng, 16, 320)
        N = max(1, min(_log(rng, 8, 131072), 131072 * 512 * 2048 // (D * F)))
        return {"op": op, "N": N, "D": D, "F": F, "dtype": rng.choice(("bf16", "bf16", "f16")),
                "act": rng.choice(("silu", "silu", "gelu", "relu")), "train": rng.random() < 0.6}
    D = _log(rng, 32, 2816)
    return {"op": op, "N": max(1, min(_log(rng, 8, 131072), 131072 * 512 // D)), "D": D,
            "dtype": rng.choice(("bf16", "bf16", "f16", "f32")), "gate": rng.choice(("full", "row", "none")),
            "train": rng.random() < 0.6}


# ------------------------------------------------------------------------------------------------ inputs
class _State:
    pass


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 29)
    n = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    u = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    dt = DTYPES[case["dtype"]]
    s = _State()
    s.case = case
    train = case.get("train", False)
    leaf = lambda x: x.requires_grad_(train)  # noqa: E731
    if case["op"] in ("step", "window"):
        B, Hk, H, K, V = (case[x] for x in ("B", "Hk", "H", "K", "V"))
        lead = (B,) if case["op"] == "step" else (B, case["T"])
        unit = lambda x: x / (x.norm(dim=-1, keepdim=True) + 1e-6)  # noqa: E731
        # queries and keys of unit length; a robot's observations change slowly, so its keys share a direction
        s.q = leaf(unit(n(*lead, Hk, K)).to(dt))
        s.k = leaf(unit(n(*lead, Hk, K) + 0.7 * n(B, *(1,) * (len(lead) - 1), Hk, K)).to(dt))
        s.v = leaf(n(*lead, H, V).to(dt))
        # decays from one step's half-life to thousands of steps, write strengths around one half
        s.g = leaf((-torch.exp(2.0 * n(*lead, H) - 3.5)).to(dt))
        s.beta = leaf(torch.sigmoid(n(*lead, H)).to(dt))
        s.reset = (u(*lead) < case["end"]) if case["end"] else None
        if case["op"] == "step" or case["state"] != "none":
            s.state = torch.empty(B, H, K, V, device=DEV).normal_(generator=g).mul_(0.3)
        else:
            s.state = None
        if case["op"] == "window" and train:
            s.d_o = n(*lead, H, V).to(dt)
            if case["state"] == "grad":
                s.state.requires_grad_(True)
                s.d_state = 0.3 * n(B, H, K, V)
    elif case["op"] == "ffn":
        N, D, F = case["N"], case["D"], case["F"]
        s.x = leaf(n(N, D).to(dt))
        s.w_gate = leaf((n(F, D) * (1.0 / math.sqrt(D))).to(dt))
        s.w_up = leaf((n(F, D) * (1.0 / math.sqrt(D))).to(dt))
        if train:
            s.d_y = n(N, F).to(dt)
    else:
        N, D = case["N"], case["D"]
        s.x = leaf((n(N, D) * 2.0).to(dt))
        s.f = leaf((n(N, D) * u(N, 1) * 3.0).to(dt))
        s.gate = {"full": lambda: leaf(torch.sigmoid(n(N, D)).to(dt)),
                  "row": lambda: leaf(torch.sigmoid(n(N, 1)).to(dt)), "none": lambda: None}[case["gate"]]()
        s.scale = leaf(0.1 + 0.02 * n(D))
        s.post_weight = leaf(1.0 + 0.1 * n(D))
        s.pre_weight = leaf(1.0 + 0.1 * n(D))
        if train:
            s.d_y, s.d_n = n(N, D).to(dt), n(N, D).to(dt)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_step(q, k, v, g, beta, state, reset):
    rep = v.shape[1] // q.shape[1]
    qf = q.float().repeat_interleave(rep, 1) * (q.shape[-1] ** -0.5)
    kf = k.float().repeat_interleave(rep, 1)
    keep = torch.exp(g.float())
    if reset is not None:
        keep = torch.where(reset[:, None], torch.zeros_like(keep), keep)
    state.mul_(keep[..., None, None])
    read = (state * kf[..., None]).sum(-2)
    write = beta.float()[..., None] * (v.float() - read)
    state.add_(kf[..., None] * write[..., None, :])
    return (state * qf[..., None]).sum(-2).to(v.dtype)


def _plain_window(q, k, v, g, beta, state, reset):
    """Chunks of up to 64 steps: products within a chunk, the state handed from chunk to chunk."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    C = min(64, 1 << (T - 1).bit_length())
    N = -(-T // C)

    def chunks(x, rep):
        x = x.float().repeat_interleave(rep, 2) if rep > 1 else x.float()
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, N * C - T))
        return x.transpose(1, 2).reshape(B, H, N, C, x.shape[-1])

    qc, kc, vc = chunks(q, H // Hk) * K ** -0.5, chunks(k, H // Hk), chunks(v, 1)
    bc = chunks(beta[..., None], 1)
    gc = chunks(g[..., None], 1)[..., 0]
    if reset is None:
        seg = torch.zeros(B, 1, N, C, dtype=torch.int32, device=q.device)
    else:
        rc = torch.nn.functional.pad(reset, (0, N * C - T)).reshape(B, 1, N, C)
        gc = torch.where(rc, torch.zeros_like(gc), gc)
        seg = rc.cumsum(-1)
    G = gc.cumsum(-1)
    zero = torch.zeros((), device=q.device)
    at = torch.arange(C, device=q.device)
    near = (seg[..., :, None] == seg[..., None, :]) & (at[:, None] >= at)
    dec = torch.where(near, torch.exp(torch.where(near, G[..., :, None] - G[..., None, :], zero)), zero)
    a = torch.where(seg == 0, torch.exp(G), zero)[..., None]                     # from the chunk's start
    c = torch.where(seg == seg[..., -1:], torch.exp(G[..., -1:] - G), zero)[..., None]   # to the chunk's end
    L = torch.where(at[:, None] > at, bc * (kc @ kc.transpose(-1, -2)) * dec, zero)
    inv = torch.eye(C, device=q.device).expand(B, H, N, C, C)
    s = 1
    while s < C:                              # (I + L)^-1: the inverses of blocks of s joined to blocks of 2 s
        cross = (at[:, None] // s % 2 == 1) & (at // s == at[:, None] // s - 1)
        inv = inv - inv @ torch.where(cross, L, zero) @ inv
        s *= 2
    P = (qc @ kc.transpose(-1, -2)) * dec
    S = torch.zeros(B, H, K, V, device=q.device) if state is None else state
    out = []
    for i in range(N):
        x = inv[:, :, i] @ (bc[:, :, i] * (vc[:, :, i] - a[:, :, i] * (kc[:, :, i] @ S)))
        out.append(a[:, :, i] * (qc[:, :, i] @ S) + P[:, :, i] @ x)
        S = a[:, :, i, -1:] * S + kc[:, :, i].transpose(-1, -2) @ (c[:, :, i] * x)
    o = torch.stack(out, 2).reshape(B, H, N * C, V)[:, :, :T]
    return o.transpose(1, 2).to(v.dtype), S


def _act(a, act):
    if act == "silu":
        return a / (1.0 + torch.exp(-a))
    if act == "gelu":
        return 0.5 * a * (1.0 + torch.tanh(0.7978845608028654 * (a + 0.044715 * a * a * a)))
    return torch.where(a > 0, a, torch.zeros_like(a))


def _plain_ffn(x, w_gate, w_up, act):
    xf = x.float()
    return (_act(xf @ w_gate.float().t(), act) * (xf @ w_up.float().t())).to(x.dtype)


def _plain_norm(x, f, gate, scale, post_weight, pre_weight):
    ff = f.float()
    h = ff * torch.rsqrt((ff * ff).mean(-1, keepdim=True) + EPS) * post_weight * scale
    y = x.float() + (h if gate is None else h * gate.float())
    return y.to(x.dtype), (y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * pre_weight).to(x.dtype)


# ------------------------------------------------------------------------------------------------ a pass
def run(s):
    case = s.case
    P = _package() if own else None
    if case["op"] == "step":
        o = P.delta_rule_step(s.q, s.k, s.v, s.g, s.beta, s.state, reset=s.reset) if own else \
            _plain_step(s.q, s.k, s.v, s.g, s.beta, s.state, s.reset)
        return o, s.state
    if case["op"] == "window":
        with torch.set_grad_enabled(case["train"]):
            o, S = P.delta_rule(s.q, s.k, s.v, s.g, s.beta, state=s.state, reset=s.reset) if own else \
                _plain_window(s.q, s.k, s.v, s.g, s.beta, s.state, s.reset)
        if not case["train"]:
            return o, S
        leaves, heads, grads = [s.q, s.k, s.v, s.g, s.beta], [o], [s.d_o]
        if case["state"] == "grad":
            leaves, heads, grads = leaves + [s.state], heads + [S], grads + [s.d_state]
        return o.detach(), S.detach(), torch.autograd.grad(heads, leaves, grads)
    if case["op"] == "ffn":
        with torch.set_grad_enabled(case["train"]):
            y = P.gated_ffn(s.x, s.w_gate, s.w_up, activation=case["act"]) if own else \
                _plain_ffn(s.x, s.w_gate, s.w_up, case["act"])
        if not case["train"]:
            return y
        return y.detach(), torch.autograd.grad([y], [s.x, s.w_gate, s.w_up], [s.d_y])
    with torch.set_grad_enabled(case["train"]):
        y, n = P.block_norm(s.x, s.f, gate=s.gate, scale=s.scale, post_weight=s.post_weight,
                            pre_weight=s.pre_weight, eps=EPS) if own else \
            _plain_norm(s.x, s.f, s.gate, s.scale, s.post_weight, s.pre_weight)
    if not case["train"]:
        return y, n
    leaves = [s.x, s.f] + ([s.gate] if s.gate is not None else []) + [s.scale, s.post_weight, s.pre_weight]
    return y.detach(), n.detach(), torch.autograd.grad([y, n], leaves, [s.d_y, s.d_n])


# ------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("step", "window"):
        B, Hk, H, K, V = (case[x] for x in ("B", "Hk", "H", "K", "V"))
        T = case.get("T", 1)
        train = case.get("train", False)
        io = B * T * (2 * Hk * K + H * V + 2 * H) * e           # q, k, v and the gates
        o = B * T * H * V * e
        st = B * H * K * V * 4
        states = {"step": 2, "window": {"none": 1, "given": 2, "grad": 2}[case.get("state", "given")]}[case["op"]]
        b = io + o + states * st + (B * T if case["end"] else 0)
        f = 6 * B * T * H * K * V                               # read, write and query the state
        if train:
            b += io + o + (2 * st if case["state"] == "grad" else 0)      # the gradients, and those of the outputs
            f += 14 * B * T * H * K * V
        return {"bytes": b, "flops": f}
    if case["op"] == "ffn":
        N, D, F = case["N"], case["D"], case["F"]
        b, f = (N * D + 2 * D * F + N * F) * e, 4 * N * D * F
        if case["train"]:
            b, f = b + (N * F + N * D + 2 * D * F) * e, 3 * f
        return {"bytes": b, "flops": f}
    N, D = case["N"], case["D"]
    gate = {"full": N * D, "row": N, "none": 0}[case["gate"]]
    b, f = (4 * N * D + gate) * e + 12 * D, 12 * N * D
    if case["train"]:
        b, f = b + (4 * N * D + gate) * e + 12 * D, f + 30 * N * D
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------------------------------------ 64 bits
def _steps64(q, k, v, g, beta, S, reset, scale):
    """The recurrence itself, step by step: [B, T, H, ...] with one query and key head a head."""
    outs = []
    for t in range(v.shape[1]):
        d = torch.exp(g[:, t])
        if reset is not None:
            d = d * (~reset[:, t])[:, None].double()
        S = d[..., None, None] * S
        e = v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t])
        S = S + torch.einsum("bhk,bhv->bhkv", k[:, t] * beta[:, t][..., None], e)
        outs.append(scale * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    return torch.stack(outs, 1), S


def _exact_delta(s, case):
    B, Hk, H, K, V = (case[x] for x in ("B", "Hk", "H", "K", "V"))
    step, train = case["op"] == "step", case.get("train", False)
    T = 1 if step else case["T"]
    rep = H // Hk
    rows = max(1, int((24 << 30) // (T * H * K * V * 8 * (5 if train else 1) + 4 * H * K * V * 8)))
    if -(-B // rows) * T * (60 if train else 20) * 1e-5 > 15 or T * H * K * V * 40 > 40 << 30:
        return None
    got = []
    for r in range(0, B, rows):
        cut = lambda x: x.detach()[r:r + rows].double()  # noqa: E731
        x = [cut(y) for y in (s.q, s.k, s.v, s.g, s.beta)]
        if step:
            x = [y[:, None] for y in x]
        S = cut(s.state) if s.state is not None else torch.zeros(x[0].shape[0], H, K, V, dtype=torch.float64,
                                                                 device=DEV)
        res = None if s.reset is None else s.reset[r:r + rows][:, None] if step else s.reset[r:r + rows]
        leaves = x + ([S] if case.get("state") == "grad" else [])
        for y in leaves:
            y.requires_grad_(train)
        # shared heads: head h reads query and key head h // rep
        sh = [x[i][:, :, :, None].expand(-1, -1, -1, rep, -1).reshape(x[i].shape[0], T, H, K) for i in (0, 1)]
        with torch.set_grad_enabled(train):
            o, S1 = _steps64(sh[0], sh[1], x[2], x[3], x[4], S, res, 1.0 / math.sqrt(K))
        if train:
            loss = (o * cut(s.d_o)).sum()
            if case["state"] == "grad":
                loss = loss + (S1 * cut(s.d_state)).sum()
            got.append([o.detach(), S1.detach()] + list(torch.autograd.grad(loss, leaves)))
            del loss
        else:
            got.append([o[:, 0] if step else o, S1])
        del o, S1, S, sh, leaves, x
    whole = [torch.cat(y) if len(y) > 1 else y[0] for y in zip(*got)]
    return (whole[0], whole[1], tuple(whole[2:])) if train else (whole[0], whole[1])


def _exact_ffn(s, case):
    x, wg, wu = (y.detach().double() for y in (s.x, s.w_gate, s.w_up))
    a, up = torch.matmul(x, wg.T), torch.matmul(x, wu.T)
    if case["act"] == "silu":
        sg = torch.sigmoid(a)
        h, dh = a * sg, sg * (1 + a * (1 - sg))
    elif case["act"] == "gelu":
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (a + 0.044715 * a ** 3))
        h = 0.5 * a * (1 + th)
        dh = 0.5 * (1 + th) + 0.5 * a * (1 - th ** 2) * c * (1 + 3 * 0.044715 * a ** 2)
    else:
        h, dh = a.clamp(min=0), (a > 0).double()
    y = h * up
    if not case["train"]:
        return y
    dy = s.d_y.double()
    da, du = dy * up * dh, dy * h
    del a, up, h, dh
    return y, (da @ wg + du @ wu, da.T @ x, du.T @ x)


def _exact_norm(s, case):
    x, f = s.x.detach().double(), s.f.detach().double()
    D = x.shape[1]
    sc, wp, wn = (y.detach().double() for y in (s.scale, s.post_weight, s.pre_weight))
    gate = torch.ones((), dtype=torch.float64, device=DEV) if s.gate is None else s.gate.detach().double()
    rf = 1.0 / torch.sqrt((f * f).sum(1, keepdim=True) / D + EPS)
    h = f * rf
    y = x + gate * sc * wp * h
    ry = 1.0 / torch.sqrt((y * y).sum(1, keepdim=True) / D + EPS)
    z = y * ry
    n = z * wn
    if not case["train"]:
        return y, n
    dy, dn = s.d_y.double(), s.d_n.double()
    dz = dn * wn
    dy = dy + ry * (dz - z * (dz * z).sum(1, keepdim=True) / D)
    dh = dy * gate * sc * wp
    df = rf * (dh - h * (dh * h).sum(1, keepdim=True) / D)
    grads = [dy, df]
    if s.gate is not None:
        dg = dy * sc * wp * h
        grads.append(dg if case["gate"] == "full" else dg.sum(1, keepdim=True))
    grads += [(dy * gate * wp * h).sum(0), (dy * gate * sc * h).sum(0), (dn * z).sum(0)]
    return y, n, tuple(grads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("step", "window"):
        return _exact_delta(s, case)
    return _exact_ffn(s, case) if case["op"] == "ffn" else _exact_norm(s, case)
