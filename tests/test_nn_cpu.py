"""Refusals of the layer entry points (amcuda.nn and its C ABI): bad types,
shapes, strides and sizes are errors before any device work."""
import ctypes as C
import math
import os
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from amcuda import _abi as A
from amcuda import nn

ROOT = Path(__file__).resolve().parents[1]


def test_rope_freqs_kinds():
    f, ms = nn.rope_freqs(8)
    assert ms == 1.0 and torch.allclose(f, 10000.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8), rtol=1e-14)
    g, ms = nn.rope_freqs(8, kind="linear", factor=4.0)
    assert ms == 1.0 and torch.allclose(g, f / 4, rtol=1e-14)
    g, ms = nn.rope_freqs(8, kind="base", factor=4.0)
    assert ms == 1.0 and math.isclose(g[0], f[0]) and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-12)
    g, ms = nn.rope_freqs(8, kind="parts", factor=4.0, original_len=4096)
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    assert torch.allclose(g, f * keep + f / 4 * (1 - keep), rtol=1e-14)
    assert math.isclose(ms, 0.1 * math.log(4.0) + 1, rel_tol=1e-6)


@pytest.mark.parametrize("bad", [dict(rot=0), dict(rot=3), dict(rot=8, base=0.0), dict(rot=8, factor=0.0),
                                 dict(rot=8, kind="parts", factor=2.0), dict(rot=2, kind="base", factor=2.0),
                                 dict(rot=8, kind="parts", original_len=10, slow=3.0, fast=2.0)])
def test_rope_freqs_refusals(bad):
    with pytest.raises(A.AmcError):
        nn.rope_freqs(**bad)


def test_rope_freqs_unknown_kind():
    with pytest.raises(ValueError):
        nn.rope_freqs(8, kind="other")


def rope_args(**change):
    a = dict(x=torch.zeros(2, 3, 5, 8), pos=torch.arange(5), freqs=torch.ones(4, dtype=torch.float64),
             out=torch.zeros(2, 3, 5, 8))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    {},                                                                     # not on a GPU
    {"x": torch.zeros(3, 5, 8)},
    {"x": torch.zeros(2, 3, 8, 5).transpose(2, 3)},
    {"out": torch.zeros(2, 3, 5, 6)},
    {"out": torch.zeros(2, 3, 5, 8, dtype=torch.bfloat16)},
    {"out": torch.zeros(2, 1, 5, 8).expand(2, 3, 5, 8)},
    {"pos": torch.arange(5, dtype=torch.int32)},
    {"pos": torch.arange(4)},
    {"freqs": torch.ones(4)},
    {"x2": torch.zeros(2, 1, 5, 8)},
    {"x2": torch.zeros(2, 1, 4, 8), "out2": torch.zeros(2, 1, 4, 8)},
])
def test_rope_refusals(change):
    with pytest.raises(ValueError):
        nn.rope(**rope_args(**change))


def c_rope(count=1, dtype=A.F32, batch=1, n=1, d=8, rot=8, pos=16, freqs=16, x=16, out=32, heads=1):
    t = (A.RopeTensor * 2)()
    for e in t:
        e.x, e.out, e.heads = x, out, heads
    return A.load().amc_rope(C.cast(t, C.c_void_p), count, dtype, batch, n, d, rot, pos, 0, freqs, 1.0, 0, 0, None)


@pytest.mark.parametrize("bad", [dict(count=0), dict(count=3), dict(dtype=A.F64), dict(d=0), dict(rot=10), dict(rot=3),
                                 dict(rot=0), dict(rot=1026, d=1100), dict(batch=-1), dict(n=-1), dict(pos=None), dict(freqs=None),
                                 dict(x=None), dict(heads=-1), dict(heads=40000), dict(batch=1 << 30, n=1 << 30)])
def test_c_rope_refusals(bad):
    assert c_rope(**bad) == 1


def test_c_rope_nothing_to_do():
    assert c_rope(n=0) == 0 and c_rope(batch=0) == 0 and c_rope(heads=0) == 0


def diff_args(**change):
    B, H, K, nq, nk, d = 2, 4, 2, 5, 7, 16
    a = dict(q=torch.zeros(B, 2 * H, nq, d), k=torch.zeros(B, 2 * K, nk, d), v=torch.zeros(B, K, nk, 2 * d),
             lam=torch.zeros(H, 4, d), o=torch.zeros(B, H, nq, 2 * d), lse=torch.zeros(B, 2 * H, nq), lam_init=0.8,
             scale=0.25)
    a.update(change)
    return a


@pytest.mark.parametrize("change", [
    {},                                                                     # not on a GPU
    {"q": torch.zeros(2, 7, 5, 16)},
    {"q": torch.zeros(2, 6, 5, 16)},
    {"q": torch.zeros(2, 8, 5, 16, dtype=torch.float64)},
    {"q": torch.zeros(2, 8, 16, 5).transpose(2, 3)},
    {"k": torch.zeros(2, 4, 7, 8)},
    {"k": torch.zeros(2, 4, 7, 16, dtype=torch.bfloat16)},
    {"v": torch.zeros(2, 2, 6, 32)},
    {"lam": torch.zeros(2, 4, 16)},
    {"lam": torch.zeros(4, 4, 8)},
    {"lam": torch.zeros(4, 4, 16, dtype=torch.bfloat16)},
    {"o": torch.zeros(2, 4, 5, 16)},
    {"o": torch.zeros(2, 1, 5, 32).expand(2, 4, 5, 32)},
    {"o2": torch.zeros(2, 4, 4, 32)},
    {"lse": torch.zeros(2, 4, 5)},
    {"lse": torch.zeros(2, 8, 5, dtype=torch.float64)},
    {"q_lens": torch.zeros(2, dtype=torch.int64)},
    {"kv_lens": torch.zeros(3, dtype=torch.int32)},
])
def test_diff_attention_refusals(change):
    with pytest.raises(ValueError):
        nn.diff_attention_fwd(**diff_args(**change))


@pytest.mark.parametrize("change", [{}, {"dq": torch.zeros(2, 8, 4, 16)}, {"dlam": torch.zeros(1, 4, 16)}, {"lse": None},
                                    {"do": torch.zeros(2, 4, 5, 16)},
                                    {"dk": torch.zeros(2, 1, 7, 16).expand(2, 4, 7, 16)}])
def test_diff_attention_bwd_refusals(change):
    a = diff_args()
    a.update(o2=torch.zeros(2, 4, 5, 32), do=torch.zeros(2, 4, 5, 32), dq=torch.zeros(2, 8, 5, 16),
             dk=torch.zeros(2, 4, 7, 16), dv=torch.zeros(2, 2, 7, 32), dlam=torch.zeros(4, 4, 16))
    a.update(change)
    with pytest.raises(ValueError):
        nn.diff_attention_bwd(**a)


def c_diff(entry="amc_diff_attention_fwd", **change):
    a = dict(dtype=A.BF16, batch=1, heads=2, kv_heads=1, nq=3, nk=4, d=64, dv=128, lam_rows=1, q=16, k=16, v=16, lam=16,
             o=16)
    a.update(change)
    p = A.DiffAttention(**a)
    return getattr(A.load(), entry)(C.byref(p), None)


@pytest.mark.parametrize("bad", [dict(dtype=A.F64), dict(dtype=A.E4M3), dict(heads=3, kv_heads=2), dict(heads=0),
                                 dict(kv_heads=0), dict(d=0), dict(d=129), dict(dv=257), dict(dv=0), dict(nq=-1),
                                 dict(nk=-1), dict(batch=-1), dict(batch=70000), dict(lam_rows=3), dict(q=None),
                                 dict(k=None), dict(v=None), dict(lam=None), dict(o=None)])
def test_c_diff_attention_refusals(bad):
    assert c_diff(**bad) == 1


def test_c_diff_attention_nothing_to_do():
    assert c_diff(batch=0) == 0 and c_diff(nq=0) == 0


def test_c_diff_attention_bwd_refusals():
    full = dict(o2=16, lse=16, d_o=16, dq=16, dk=16, dv_=16, dlam=16, workspace=16, workspace_bytes=1 << 30)
    for name in ("o2", "lse", "d_o", "dq", "dk", "dv_", "dlam"):
        assert c_diff("amc_diff_attention_bwd", **{**full, name: None}) == 1
    for bad in (dict(workspace=None), dict(workspace_bytes=8), dict(workspace=20)):
        assert c_diff("amc_diff_attention_bwd", **{**full, **bad}) == 1
        assert "workspace" in A.last_error()


def adamw_args(n=2, **change):
    def f(k=300, t=torch.float32):
        return [torch.zeros(k, dtype=t) for _ in range(n)]
    a = dict(params=f(), grads=f(), m=f(), v=f(), state=torch.zeros(2, dtype=torch.int64))
    a.update(change)
    return a


F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("change", [
    {"grads": [torch.zeros(300)]},
    {"m": [torch.zeros(300), torch.zeros(299)]},
    {"m": [torch.zeros(300, dtype=F8)] * 2, "v": [torch.zeros(300, dtype=F8)] * 2},
    {"m": [torch.zeros(300, dtype=F8)] * 2, "v": [torch.zeros(300)] * 2, "m_scales": [torch.zeros(2)] * 2,
     "v_scales": [torch.zeros(2)] * 2},
    {"m": [torch.zeros(300, dtype=F8)] * 2, "v": [torch.zeros(300, dtype=F8)] * 2, "m_scales": [torch.zeros(1)] * 2,
     "v_scales": [torch.zeros(2)] * 2},
    {"m_scales": [torch.zeros(2)] * 2, "v_scales": [torch.zeros(2)] * 2},
    {"params": [torch.zeros(300)] * 2},
    {"params": [torch.zeros(300), torch.zeros(300, dtype=torch.bfloat16)]},
    {"params": [torch.zeros(600)[::2], torch.zeros(300)]},
    {"params": [torch.zeros(300, dtype=torch.float64) for _ in range(2)]},
    {"masters": [torch.zeros(300)]},
    {"state": torch.zeros(1, dtype=torch.int64)},
    {"state": torch.zeros(2, dtype=torch.int32)},
    {"lr": torch.zeros(2)},
])
def test_adamw_refusals(change):
    with pytest.raises(ValueError):
        nn.AdamW(**adamw_args(**change))


def test_adamw_step_needs_a_gpu():
    with pytest.raises(ValueError):
        nn.AdamW(**adamw_args()).step()


def c_adamw(count=1, p=A.F32, g=A.F32, s=A.F32, state=16, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, **e):
    t = (A.AdamwTensor * 2)()
    for x in t:
        x.p = x.g = x.m = x.v = 16
        x.n = 4
    for k, v in e.items():
        setattr(t[count - 1], k, v)
    return A.load().amc_adamw(C.cast(t, C.c_void_p), count, p, g, s, state, None, lr, b1, b2, eps, wd, None)


@pytest.mark.parametrize("bad", [dict(state=None), dict(p=A.F64), dict(g=A.E4M3), dict(s=A.BF16), dict(s=A.E4M3),
                                 dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(lr=math.nan),
                                 dict(n=-1), dict(m=None), dict(count=2, master=16)])
def test_c_adamw_refusals(bad):
    assert c_adamw(**bad) == 1


def test_injected_launch_failures():
    code = r"""
import sys
sys.path[:0] = [%r, %r]
import test_nn_cpu as T
from amcuda import _abi as A
for f in (T.c_rope, T.c_diff, T.c_adamw):
    assert f() == 6, f
    assert "AMC_FAULT=launch" in A.last_error()
""" % (str(ROOT / "array-morphisms_b200"), str(ROOT / "tests"))
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, AMC_FAULT="launch"), capture_output=True,
                         text=True, timeout=120)
    assert out.returncode == 0, out.stderr


def test_c_rope_refuses_results_on_the_other_tensor():
    def call(x0, o0, x1, o1, heads1=1):
        t = (A.RopeTensor * 2)()
        (t[0].x, t[0].out, t[0].heads), (t[1].x, t[1].out, t[1].heads) = (x0, o0, 1), (x1, o1, heads1)
        return A.load().amc_rope(C.cast(t, C.c_void_p), 2, A.F32, 1, 1, 8, 8, None, 0, 16, 1.0, 0, 0, None)
    for bad in ((16, 32, 48, 32), (16, 48, 48, 64), (16, 32, 48, 16)):
        assert call(*bad) == 1 and "on one another" in A.last_error()
    # separate ones, two turns of one tensor, and an empty second pass this check and meet the next
    for fine in ((16, 16, 48, 48), (16, 32, 16, 48), (16, 32, 48, 32, 0)):
        assert call(*fine) == 1 and "null positions" in A.last_error()


def c_diff_apart(entry, **change):
    """A call with every tensor in a place of its own (addresses only) but for the changes; it never reaches a launch."""
    p = A.DiffAttention(dtype=A.F32, batch=1, heads=2, kv_heads=1, nq=3, nk=5, d=8, dv=8, lam_rows=1, scale=1.0)
    p.workspace, p.workspace_bytes = 4096 * 30, 1 << 30
    for i, name in enumerate(("q", "k", "v", "lam", "o", "o2", "d_o", "dq", "dk", "dv_", "dlam")):
        setattr(p, name, 4096 * (i + 1))
    p.lse = 4096 * 20
    for k, v in change.items():
        setattr(p, k, v)
    rc = getattr(A.load(), entry)(C.byref(p), None)
    return rc, A.last_error()


@pytest.mark.parametrize("entry,change", [
    ("amc_diff_attention_fwd", {"o": 4096}), ("amc_diff_attention_fwd", {"o2": 4096 * 5}),
    ("amc_diff_attention_fwd", {"o2": 4096 * 3}), ("amc_diff_attention_fwd", {"lse": 4096 * 5}),
    ("amc_diff_attention_bwd", {"dq": 4096}), ("amc_diff_attention_bwd", {"dk": 4096 * 8}),
    ("amc_diff_attention_bwd", {"dv_": 4096 * 7}), ("amc_diff_attention_bwd", {"dlam": 4096 * 4}),
    ("amc_diff_attention_bwd", {"dq": 4096 * 20}),
])
def test_c_diff_attention_refuses_results_on_other_tensors(entry, change):
    rc, text = c_diff_apart(entry, **change)
    assert rc == 1 and "lies on another tensor" in text


def test_adamw_refuses_a_tensor_in_two_places():
    z = torch.zeros(300)
    for change in ({"m": [z, torch.zeros(300)], "v": [z, torch.zeros(300)]}, {"v": [z, z]},
                   {"masters": [z, z]}, {"params": [z, torch.zeros(300)], "m": [torch.zeros(300), z]}):
        with pytest.raises(ValueError, match="as well"):
            nn.AdamW(**adamw_args(**change))
    p = [torch.zeros(300), torch.zeros(300)]
    nn.AdamW(**adamw_args(params=p, masters=p))
    nn.AdamW(**adamw_args(grads=[z, z]))
    e = torch.zeros(0)
    nn.AdamW(params=[e, e], grads=[e, e], m=[e, e], v=[e, e], state=torch.zeros(2, dtype=torch.int64))


def test_adamw_keeps_the_memory_it_was_made_with():
    a = adamw_args()
    opt = nn.AdamW(**a)
    at = a["params"][0].data_ptr()
    a["params"][0].data = torch.zeros(300)
    assert opt._table[0].p == at and any(s.data_ptr() == at for s in opt._keep)


def test_c_adamw_refuses_more_than_it_can_count():
    assert c_adamw(n=1 << 45) == 1
    assert "too many" in A.last_error()
    assert c_adamw(count=2, n=(1 << 42) - (1 << 12)) == 1
    assert "too many" in A.last_error()


def test_adamw_takes_an_assigned_rate(monkeypatch):
    """A rate assigned after the object was made is the next step's, whether it or the first was a tensor."""
    given = []
    monkeypatch.setattr(nn, "_run", lambda name, device, stream, *args: given.append(args[6:8]))
    rate = torch.tensor([0.25])
    opt = nn.AdamW(**adamw_args(lr=rate))
    opt.step()
    opt.lr = 0.5
    assert opt.lr == 0.5
    opt.step()
    opt.lr = rate
    assert opt.lr is rate
    opt.step()
    assert given == [(rate.data_ptr(), 0.0), (0, 0.5), (rate.data_ptr(), 0.0)]
    for bad in (torch.zeros(2), torch.zeros(1, dtype=torch.float64)):
        with pytest.raises(ValueError):
            opt.lr = bad
    assert opt.lr is rate


def test_adamw_refuses_tensors_that_share_some_memory():
    z = torch.zeros(600)
    nn.AdamW(**adamw_args(params=[z[:300], z[300:]]))
    for change in ({"params": [z[:300], z[299:599]]}, {"m": [z[1:301], torch.zeros(300)], "v": [z[:300], torch.zeros(300)]},
                   {"params": [torch.zeros(300), z[:300]], "masters": [z[200:500], torch.zeros(300)]}):
        with pytest.raises(ValueError, match="as well"):
            nn.AdamW(**adamw_args(**change))
