"""The policy operators' library and checks without a GPU: the exported symbols, the ctypes mirrors' layout, what the
Python entry points refuse and what the C entry points refuse before any launch."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

import isaac_net_amd as P
from conftest import ROOT
from isaac_net_amd import _lib, policy
from oracle import policy_oracle as O

HEADER = os.path.join(ROOT, "include", "inet_policy.h")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.POLICY_LIB_PATH):
        from isaac_net_amd import build
        build.build_policy()
    return _lib.load_policy()


def test_library_exports_every_declared_symbol(lib):
    names = re.findall(r"^\s*(?:int32_t|int64_t|const char \*)\s*(inet_policy_\w+)\s*\(", open(HEADER).read(), re.M)
    assert len(names) == 13
    for n in names:
        assert hasattr(lib, n), n
    assert lib.inet_policy_abi_version() == _lib.POLICY_ABI_VERSION
    assert b"gfx950" in lib.inet_policy_build_info()


def test_ctypes_layout_matches_header(tmp_path):
    structs = ("InetDelta", "InetDeltaGrad", "InetFfn", "InetFfnGrad", "InetNorm", "InetNormGrad")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for n in structs:
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for f in getattr(_lib, n)._fields_]
    c = tmp_path / "layout.c"
    c.write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(c)], check=True)
    out = dict(x.rsplit(" ", 1) for x in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True,
                                                        text=True).stdout.split("\n") if x)
    for n in structs:
        cls = getattr(_lib, n)
        assert int(out[n]) == ctypes.sizeof(cls), n
        for f in cls._fields_:
            assert int(out[f"{n}.{f[0]}"]) == getattr(cls, f[0]).offset, f"{n}.{f[0]}"


def test_loader_refuses(tmp_path):
    saved, _lib._POLICY_LIB = _lib._POLICY_LIB, None
    try:
        with pytest.raises(RuntimeError, match="missing"):
            _lib.load_policy(str(tmp_path / "nope.so"))
        (tmp_path / "old.c").write_text("int inet_policy_abi_version(void) { return 0; }\n"
                                        'const char *inet_policy_build_info(void) { return ""; }')
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(tmp_path / "old.so"), str(tmp_path / "old.c")], check=True)
        with pytest.raises(RuntimeError, match="ABI version"):
            _lib.load_policy(str(tmp_path / "old.so"))
    finally:
        _lib._POLICY_LIB = saved


def test_entry_points_need_the_gpu():
    x = torch.zeros(2, 4, 1, 8)
    g = torch.zeros(2, 4, 1)
    for call in (lambda: P.delta_rule(x, x, x, g, g), lambda: P.gated_ffn(torch.zeros(2, 8), x[0, 0], x[0, 0]),
                 lambda: P.block_norm(torch.zeros(2, 8), pre_weight=torch.ones(8)),
                 lambda: P.delta_rule_step(x[:, 0], x[:, 0], x[:, 0], g[:, 0], g[:, 0], torch.zeros(2, 1, 8, 8))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(ValueError, match="tensor"):
        P.delta_rule([1.0], x, x, g, g)


class _OnGpu:
    """Lets the shape and type checks run on CPU tensors."""
    def __enter__(self):
        self.saved, policy._on_gpu = policy._on_gpu, lambda **x: 0
        self.call, policy._call = policy._call, lambda *a: pytest.fail("a refused call reached the library")

    def __exit__(self, *a):
        policy._on_gpu, policy._call = self.saved, self.call


def test_delta_refusals():
    ok = dict(q=torch.zeros(2, 5, 1, 8), k=torch.zeros(2, 5, 1, 8), v=torch.zeros(2, 5, 2, 4), g=torch.zeros(2, 5, 2),
              beta=torch.zeros(2, 5, 2), state=torch.zeros(2, 2, 8, 4), reset=torch.zeros(2, 5, dtype=torch.bool))
    bad = [dict(q=torch.zeros(2, 5, 8)), dict(k=torch.zeros(2, 5, 1, 7)), dict(v=torch.zeros(2, 4, 2, 4)),
           dict(v=torch.zeros(2, 5, 0, 4)), dict(g=torch.zeros(2, 5, 1)), dict(beta=torch.zeros(2, 5)),
           dict(k=torch.zeros(2, 5, 1, 8).half()), dict(g=torch.zeros(2, 5, 2).half()),
           dict(state=torch.zeros(2, 2, 4, 8)), dict(state=torch.zeros(2, 2, 8, 4).half()),
           dict(reset=torch.zeros(2, 5)), dict(reset=torch.zeros(2, 4, dtype=torch.bool)),
           dict(q=torch.zeros(2, 5, 3, 8), k=torch.zeros(2, 5, 3, 8))]
    with _OnGpu():
        for b in bad:
            with pytest.raises(ValueError):
                P.delta_rule(**{**ok, **b})
        big = torch.zeros(2, 5, 1, 129)
        with pytest.raises(P.HipUnsupported, match="128"):
            P.delta_rule(**{**ok, "q": big, "k": big, "state": None})
        with pytest.raises(P.HipUnsupported, match="float64"):
            P.delta_rule(*(ok[n].double() for n in ("q", "k", "v", "g", "beta")))
        wide = torch.zeros(1, 1, 1, 8).expand(1 << 24, 1, 1, 8)
        with pytest.raises(P.HipUnsupported, match="fewer"):
            P.delta_rule(wide, wide, wide, wide[..., 0], wide[..., 0])
        one = {n: t[:, 0] for n, t in ok.items() if n != "state"}
        with pytest.raises(ValueError, match="contiguous"):
            P.delta_rule_step(**one, state=None)
        with pytest.raises(ValueError, match="contiguous"):
            P.delta_rule_step(**one, state=torch.zeros(2, 2, 4, 8).transpose(2, 3))
        with pytest.raises(ValueError, match="out"):
            P.delta_rule_step(**one, state=ok["state"], out=torch.zeros(2, 2, 5))


def test_ffn_and_norm_refusals():
    x, w = torch.zeros(3, 8).half(), torch.zeros(5, 8).half()
    with _OnGpu():
        for call in (lambda: P.gated_ffn(x, w, w[:4]), lambda: P.gated_ffn(x[:, :7], w, w),
                     lambda: P.gated_ffn(x, w, w.float()), lambda: P.gated_ffn(x, w, w, activation="tanh"),
                     lambda: P.gated_ffn(x, w[:0], w[:0])):
            with pytest.raises(ValueError):
                call()
        with pytest.raises(P.HipUnsupported, match="float32"):
            P.gated_ffn(x.float(), w.float(), w.float())
        y, one = torch.zeros(3, 8), torch.ones(8)
        for kw in (dict(f=torch.zeros(3, 7)), dict(f=y.half()), dict(f=y, gate=torch.zeros(3)),
                   dict(f=y, gate=torch.zeros(3, 2)), dict(f=y, scale=one[:7]), dict(f=y, post_weight=one.half()),
                   dict(pre_weight=torch.ones(1, 8)), dict(gate=y, pre_weight=one), dict(scale=one)):
            with pytest.raises(ValueError):
                P.block_norm(y, **kw)
        with pytest.raises(P.HipUnsupported, match="8192"):
            P.block_norm(torch.zeros(1, 8193), pre_weight=torch.ones(8193))
        assert P.block_norm(y) == (y, None)


def test_c_entry_points_refuse_before_any_launch(lib):
    B, none = ctypes.byref, None
    d, dg = _lib.InetDelta(), _lib.InetDeltaGrad()
    assert lib.inet_policy_delta_forward(none, none) == -1
    assert lib.inet_policy_delta_forward(B(d), none) == -1                          # no heads
    d.B, d.T, d.Hk, d.H, d.K, d.V = 2, 40, 1, 2, 16, 16
    assert lib.inet_policy_delta_forward(B(d), none) == -1                          # chunk not set
    for key, value, chunk in (("T", 4000, 32), ("dtype", 1, 64), ("B", 96, 32), ("K", 129, 0), ("dtype", 3, 0)):
        setattr(d, key, value)
        assert lib.inet_policy_delta_chunk(B(d)) == chunk, key
    d.B, d.T, d.K, d.dtype, d.chunk = 2, 40, 16, 0, 32
    assert lib.inet_policy_delta_forward(B(d), none) == -1                          # no tensors
    assert lib.inet_policy_delta_backward(B(d), B(dg), none) == -1
    assert lib.inet_policy_delta_step(B(d), none) == -1                             # T is not 1
    d.H = 3
    d.Hk = 2
    assert lib.inet_policy_delta_forward(B(d), none) == -1
    d.H, d.K = 2, 200
    assert lib.inet_policy_delta_forward(B(d), none) == -2
    d.K, d.B = 16, 0
    assert lib.inet_policy_delta_forward(B(d), none) == 0                           # nothing to do
    f, fg = _lib.InetFfn(), _lib.InetFfnGrad()
    assert lib.inet_policy_ffn_forward(none, none) == lib.inet_policy_ffn_forward(B(f), none) == -1
    f.N, f.D, f.F, f.dtype = 4, 8, 8, 0
    assert lib.inet_policy_ffn_forward(B(f), none) == -2                            # float32
    f.dtype = 1
    assert lib.inet_policy_ffn_forward(B(f), none) == lib.inet_policy_ffn_backward(B(f), B(fg), none) == -1
    f.x = f.w_gate = f.w_up = 8                                                     # rows off the 16-byte grid
    f.x_s = f.w_gate_s = f.w_up_s = 8
    f.y = 16
    assert lib.inet_policy_ffn_forward(B(f), none) == -1
    assert lib.inet_policy_ffn_work(-1, 8, 8, 0) == -1 and lib.inet_policy_ffn_work(4, 8, 8, 0) == 0
    n, ng = _lib.InetNorm(), _lib.InetNormGrad()
    assert lib.inet_policy_norm_forward(none, none) == lib.inet_policy_norm_forward(B(n), none) == -1
    n.N, n.D = 2, 9000
    assert lib.inet_policy_norm_forward(B(n), none) == -2
    n.D = 8
    assert lib.inet_policy_norm_forward(B(n), none) == lib.inet_policy_norm_backward(B(n), B(ng), none) == -1
    assert lib.inet_policy_norm_work(2, 9000) == -1


def test_oracle_known_answers():
    """One step by hand, and the memory read back: a unit key written in full is answered with its value."""
    k = torch.zeros(1, 2, 1, 4, dtype=torch.float64)
    k[0, 0, 0, 1] = k[0, 1, 0, 1] = 1.0
    v = torch.tensor([[[[2.0, -1.0]], [[5.0, 5.0]]]], dtype=torch.float64)
    one, zero = torch.ones(1, 2, 1, dtype=torch.float64), torch.zeros(1, 2, 1, dtype=torch.float64)
    o, s = O.delta_rule(k, k, v, zero, one, scale=1.0)
    assert torch.equal(o, v) and torch.equal(s[0, 0, 1], v[0, 1, 0])
    o, s = O.delta_rule(k, k, v, zero + math.log(0.5), one * 0.5, scale=1.0)
    assert torch.allclose(o[0, :, 0], torch.tensor([[1.0, -0.5], [2.75, 2.375]], dtype=torch.float64))
    o, s = O.delta_rule(k, k, v, zero, one * 0.5, reset=torch.tensor([[0, 1]]), scale=1.0)
    assert torch.equal(o[0, 1, 0], 0.5 * v[0, 1, 0])
