"""The differential-attention layer's operators (amcuda.nn) against plain
64-bit implementations on the device.

Tolerances count roundings.  u is the half step of the stored type (bf16 2^-8,
fp16 2^-11, fp32 2^-24 relative).  A 16-bit result carries its own rounding
(u of the value) and, in the tensor-core and split forms, the rounding of the
probabilities (and in the backward of dS) to 16 bits, u of each term: bounded
by u * sum |terms|, the same product with absolute values, so every comparison
is element by element against u * (|result| + 2 * absolute product) plus f32
accumulation, 2^-24 times the length of the sums, on the same absolute product.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    return torch.finfo(t).eps / 2


@pytest.fixture(scope="module")
def nn(amc):
    from amcuda import nn
    return nn


def randn(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


# ---------------------------------------------------------------------------- rope
def rope_ref(x, pos, freqs, mscale, interleaved, inverse):
    """The rotation in 64 bits, and sum |terms| of each element."""
    r = 2 * len(freqs)
    B, n = x.shape[0], x.shape[2]
    a = pos.expand(B, n).double()[:, None, :, None] * freqs
    c, s = a.cos() * mscale, a.sin() * (-mscale if inverse else mscale)
    xd = x.double()
    y, t = xd.clone(), xd.abs()
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    xa, xb = xd[..., ia], xd[..., ib]
    y[..., ia], y[..., ib] = xa * c - xb * s, xb * c + xa * s
    t[..., ia] = t[..., ib] = (xa.abs() + xb.abs()) * mscale
    return y, t


def rope_close(got, ref, terms, dtype):
    # f32: the reduced angle (half a turn) is rounded to 2^-25 turns and the
    # sine and cosine carry 2 ulp, so 2^-25 * 2 pi + 2 * 2^-23 < 2^-21 of the
    # terms, and the products and their sum 3 more half steps
    tol = half_step(dtype) * ref.abs() + (2.0 ** -21 + 3 * 2.0 ** -24) * terms + 1e-30
    if dtype is torch.float16:
        tol = tol + 2.0 ** -25          # half of fp16's subnormal step
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), ((got.double() - ref).abs() / tol).max().item()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,H,H2,n,d,rot", [(2, 3, 1, 17, 64, 64), (1, 1, 0, 1, 2, 2), (3, 2, 5, 1, 80, 48),
                                           (2, 4, 4, 130, 20, 6), (1, 16, 4, 33, 128, 128)])
def test_rope(nn, dtype, interleaved, B, H, H2, n, d, rot):
    t = TYPES[dtype]
    x, x2 = randn((B, n, H, d), 1, t).transpose(1, 2), randn((B, H2, n, d), 2, t) if H2 else None
    pos = torch.randint(0, 1 << 20, (B, n), device="cuda")
    freqs, ms = nn.rope_freqs(rot, kind="parts", factor=4.0, original_len=4096)
    freqs = freqs.cuda()
    for inverse in (False, True):
        out, out2 = torch.full_like(x, 7), torch.full_like(x2, 7) if H2 else None
        nn.rope(x, pos, freqs, out, x2, out2, mscale=ms, interleaved=interleaved, inverse=inverse)
        for a, o in ((x, out), (x2, out2)):
            if a is not None:
                rope_close(o, *rope_ref(a, pos, freqs, ms, interleaved, inverse), t)


def test_rope_in_place_strided_and_far(nn):
    """In place on a slice of a wider projection (rows not 16-byte aligned), at
    positions past 2^32, with one (n,) position vector."""
    for offset in (0, 3):
        wide = randn((2, 40, 3, 64 + 8), 3, torch.bfloat16)
        x = wide[..., offset:offset + 64].transpose(1, 2)
        keep = wide.clone()
        pos = (1 << 33) + torch.arange(40, device="cuda") * 12345677
        freqs, _ = nn.rope_freqs(64)
        freqs = freqs.cuda()
        ref, terms = rope_ref(x, pos, freqs, 1.0, False, False)
        nn.rope(x, pos, freqs, x)
        rope_close(x, ref, terms, torch.bfloat16)
        assert torch.equal(wide[..., :offset], keep[..., :offset])
        assert torch.equal(wide[..., offset + 64:], keep[..., offset + 64:])


def test_rope_gradient_by_differences(nn):
    """<w, R(x + h v) - R(x - h v)> / 2h = <R^T w, v>: R is linear."""
    x, v, w = (randn((1, 2, 9, 12), s, torch.float32) for s in (4, 5, 6))
    pos = torch.arange(9, device="cuda") * 37
    freqs, ms = nn.rope_freqs(8, kind="parts", factor=16.0, original_len=512)
    freqs = freqs.cuda()
    up, down, back = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    nn.rope(x + v, pos, freqs, up, mscale=ms, interleaved=True)
    nn.rope(x - v, pos, freqs, down, mscale=ms, interleaved=True)
    nn.rope(w, pos, freqs, back, mscale=ms, interleaved=True, inverse=True)
    lhs = ((up.double() - down.double()) * w).sum() / 2
    rhs = (back.double() * v).sum()
    # 216 products of values of a few units, each 2^-21 of its terms
    assert abs(lhs - rhs) < 216 * 64 * 2.0 ** -21


# ---------------------------------------------------------------------------- differential attention
LAM_INIT = 0.8


class Case:
    def __init__(self, B, H, K, nq, nk, d, dtype, causal=False, q_lens=None, kv_lens=None, dv=None, lam_rows=None,
                 seed=0, scale=None, heads_inner=True):
        t = TYPES[dtype]
        dv = 2 * d if dv is None else dv
        self.t, self.causal, self.scale = t, causal, scale or 1 / math.sqrt(d)

        def make(h, n, w, s):
            if heads_inner:
                return randn((B, n, h, w), seed + s, t).transpose(1, 2)
            return randn((B, h, n, w), seed + s, t)
        self.q, self.k, self.v, self.do = make(2 * H, nq, d, 1), make(2 * K, nk, d, 2), make(K, nk, dv, 3), make(H, nq, dv, 4)
        self.lam = randn((lam_rows or H, 4, d), seed + 5, t, 0.1)
        lens = [None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda") for x in (q_lens, kv_lens)]
        self.q_lens, self.kv_lens = lens
        self.H, self.K = H, K

    def fwd(self, nn, o2=True, **more):
        B, _, nq, _ = self.q.shape
        o = torch.full((B, self.H, nq, self.v.shape[3]), 7.0, dtype=self.t, device="cuda")
        lse = torch.full((B, 2 * self.H, nq), 7.0, device="cuda")
        second = torch.full_like(o, 7) if o2 else None
        ws = torch.empty(nn.diff_attention_workspace(self.q, self.k, self.v), dtype=torch.uint8, device="cuda")
        nn.diff_attention_fwd(self.q, self.k, self.v, self.lam, o, lse, LAM_INIT, self.scale, causal=self.causal,
                              q_lens=self.q_lens, kv_lens=self.kv_lens, o2=second, workspace=ws, **more)
        return o, lse, second

    def bwd(self, nn, o, lse, o2, **more):
        g = [torch.full_like(x, 7) for x in (self.q, self.k, self.v, self.lam)]
        n = nn.diff_attention_workspace(self.q, self.k, self.v, backward=True)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        nn.diff_attention_bwd(self.q, self.k, self.v, self.lam, o, o2, lse, self.do, *g, LAM_INIT, self.scale,
                              causal=self.causal, q_lens=self.q_lens, kv_lens=self.kv_lens, workspace=ws, **more)
        return dict(zip(("dq", "dk", "dv", "dlam"), g))

    def reference(self, backward=False):
        """name -> (value, sum |terms|) in 64 bits, from the formulas."""
        B, H2, nq, d = self.q.shape
        nk, dv, H, K = self.k.shape[2], self.v.shape[3], self.H, self.K
        G = H // K
        ql = self.q_lens.tolist() if self.q_lens is not None else [nq] * B
        kl = self.kv_lens.tolist() if self.kv_lens is not None else [nk] * B
        ok = torch.zeros(B, 1, 1, nq, nk, dtype=torch.bool, device="cuda")
        for b in range(B):
            i, j = torch.arange(ql[b], device="cuda")[:, None], torch.arange(kl[b], device="cuda")[None]
            ok[b, 0, 0, :ql[b], :kl[b]] = (j <= i + kl[b] - ql[b]) if self.causal else True

        def clean(x, lens):
            x = x.double().clone()
            for b in range(B):
                x[b, :, lens[b]:] = 0
            return x
        q = clean(self.q, ql).reshape(B, H, 2, nq, d)
        k = clean(self.k, kl).reshape(B, K, 2, nk, d).repeat_interleave(G, 1)
        v = clean(self.v, kl).reshape(B, K, 1, nk, dv).repeat_interleave(G, 1)
        x = (q @ k.transpose(-1, -2)) * self.scale
        x = x.masked_fill(~ok, -math.inf)
        lse = torch.logsumexp(x, -1)
        p = torch.exp(x - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
        lam4 = self.lam.double().expand(H, 4, d)
        e1, e2 = torch.exp((lam4[:, 0] * lam4[:, 1]).sum(-1)), torch.exp((lam4[:, 2] * lam4[:, 3]).sum(-1))
        lam = (e1 - e2 + LAM_INIT).reshape(1, H, 1, 1)
        om, oa = p @ v, p @ v.abs()
        r = {"o": (om[:, :, 0] - lam * om[:, :, 1], oa[:, :, 0] + lam.abs() * oa[:, :, 1]),
             "o2": (om[:, :, 1], oa[:, :, 1]), "lse": (lse.reshape(B, H2, nq), None)}
        if not backward:
            return r
        g = clean(self.do, ql)
        G1, Ga = (g @ v[:, :, 0].transpose(-1, -2))[:, :, None], (g.abs() @ v[:, :, 0].abs().transpose(-1, -2))[:, :, None]
        D, Da = (g[:, :, None] * om).sum(-1, keepdim=True), (g.abs()[:, :, None] * (oa + r["o"][1][:, :, None])).sum(-1, keepdim=True)
        sign = torch.stack([torch.ones_like(lam), -lam], 2)
        ds, dsa = p * (G1 - D) * sign * self.scale, p * (G1.abs() + D.abs()) * sign.abs() * self.scale
        # D is formed from outputs stored in 16 bits: a half step of each of its terms
        dd = p * Da * sign.abs() * self.scale

        def shared(t):
            return t.reshape(B, K, G, *t.shape[2:]).sum(2)
        r["dq"] = [(a @ b).reshape(B, H2, nq, d) for a, b in ((ds, k), (dsa + dd, k.abs()))]
        r["dk"] = [shared(a.transpose(-1, -2) @ b).reshape(B, 2 * K, nk, d) for a, b in ((ds, q), (dsa + dd, q.abs()))]
        r["dv"] = [shared(a.transpose(-1, -2) @ b) for a, b in ((p[:, :, 0] - lam * p[:, :, 1], g),
                                                               (p[:, :, 0] + lam.abs() * p[:, :, 1], g.abs()))]
        w = torch.stack([e1, -e2], 1)
        dl, dla = -D[:, :, 1].sum((0, 2, 3)), (p[:, :, 1] * Ga[:, :, 0]).sum((0, 2, 3))
        out = []
        for t, f in ((dl, 1.0), (dla, -1.0)):
            lam_t, w_t = (lam4, w) if f > 0 else (lam4.abs(), w.abs())
            rows = (t[:, None] * w_t).repeat_interleave(2, 1)[..., None] * lam_t[:, [1, 0, 3, 2]]
            out.append(rows if len(self.lam) == H else rows.sum(0, keepdim=True))
        r["dlam"] = out
        return r

    def check(self, got, ref, sums):
        """|got - ref| <= u |ref| + (2 u' + 2^-24 * sums) * sum |terms| with u
        the half step of the type; u' is u again where probabilities may be
        rounded to the type (16-bit types), 0 for f32 and dlam.  The scores
        themselves: an f32 dot of d terms, exponentiated, moves p by
        (d + 4) 2^-24 |score terms| <= 2^-16 here (|scores| < 40)."""
        u = half_step(self.t)
        for name, x in got.items():
            y, terms = ref[name]
            x = x.double()
            if name == "lse":
                fine = y > -math.inf
                assert torch.equal(x == -math.inf, ~fine)
                # f32 scores and sums: 40 * (d + 8) half steps at most
                assert ((x - y)[fine].abs() < 2.0 ** -24 * 40 * 72).all(), (x - y)[fine].abs().max()
                continue
            u2 = 0.0 if self.t is torch.float32 or name == "dlam" else 2 * u
            tol = u * y.abs() + (u2 + 2.0 ** -24 * sums + 2.0 ** -16) * terms + 1e-30
            if self.t is torch.float16:
                tol = tol + 2.0 ** -24
            worst = ((x - y).abs() / tol).max().item() if x.numel() else 0.0
            assert worst <= 1.0 and torch.isfinite(x).all(), (name, worst)


FWD = [
    dict(B=1, H=1, K=1, nq=1, nk=1, d=64),
    dict(B=2, H=2, K=1, nq=5, nk=7, d=64, causal=True),
    dict(B=1, H=2, K=2, nq=128, nk=128, d=64),
    dict(B=2, H=2, K=1, nq=129, nk=257, d=64, causal=True),
    dict(B=1, H=3, K=1, nq=300, nk=300, d=48, causal=True),
    dict(B=2, H=1, K=1, nq=200, nk=100, d=32, causal=True),           # rows that see no key
    dict(B=1, H=2, K=2, nq=64, nk=190, d=8, dv=24),
    dict(B=4, H=2, K=1, nq=150, nk=150, d=64, causal=True, q_lens=[150, 0, 1, 77], kv_lens=[150, 0, 1, 77]),
    dict(B=4, H=2, K=2, nq=130, nk=260, d=64, q_lens=[130, 20, 1, 128], kv_lens=[0, 260, 129, 128]),
    dict(B=3, H=2, K=1, nq=40, nk=300, d=64, causal=True, q_lens=[40, 3, 40], kv_lens=[300, 256, 20]),
    dict(B=3, H=4, K=1, nq=1, nk=1500, d=64, causal=True, q_lens=[1, 1, 0], kv_lens=[1500, 257, 9]),   # one token
    dict(B=2, H=4, K=2, nq=4, nk=1030, d=64, causal=True, kv_lens=[1029, 2]),    # a few; rows that see no key
    dict(B=1, H=16, K=1, nq=1, nk=700, d=32),
    dict(B=7, H=4, K=2, nq=1, nk=3001, d=64, causal=True, q_lens=[1, 1, 0, 1, 1, 1, 1],      # shared out unevenly
         kv_lens=[3001, 64, 500, 0, 65, 1, 2900]),
    dict(B=40, H=2, K=1, nq=3, nk=5000, d=16),                                               # shares of several units
    dict(B=300, H=2, K=2, nq=1, nk=300, d=32, causal=True, kv_lens=[(7 * i) % 301 for i in range(300)]),
    dict(B=3, H=2, K=1, nq=1, nk=700, d=64, q_lens=[0, 0, 0]),
    dict(B=1, H=2, K=2, nq=16, nk=530, d=40, dv=72),
    dict(B=2, H=3, K=3, nq=2, nk=137, d=64, heads_inner=False),
    # many tiles: pairs of CTAs, several tiles each
    dict(B=10, H=16, K=4, nq=130, nk=257, d=64, causal=True, q_lens=[130, 0, 1, 129, 128, 127, 77, 130, 130, 2],
         kv_lens=[257, 257, 0, 5, 256, 255, 129, 64, 65, 200]),
    dict(B=5, H=16, K=16, nq=300, nk=300, d=32, kv_lens=[300, 0, 299, 128, 1]),
    dict(B=3, H=25, K=5, nq=513, nk=700, d=48, causal=True),
    dict(B=1, H=2, K=1, nq=70, nk=70, d=100, dv=200, causal=True),    # wide head
    dict(B=1, H=1, K=1, nq=33, nk=65, d=13, dv=7),                    # odd dims
    dict(B=1, H=2, K=1, nq=33, nk=65, d=64, heads_inner=False, lam_rows=1),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(FWD)))
def test_diff_attention_forward(nn, dtype, case):
    c = Case(dtype=dtype, **FWD[case])
    o, lse, o2 = c.fwd(nn)
    c.check({"o": o, "lse": lse, "o2": o2}, c.reference(), c.k.shape[2])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(FWD)))
def test_diff_attention_gradients(nn, dtype, case):
    c = Case(dtype=dtype, **FWD[case])
    got = c.bwd(nn, *c.fwd(nn))
    c.check(got, c.reference(backward=True), max(c.k.shape[2], c.q.shape[2] * c.H // c.K))
    again = c.bwd(nn, *c.fwd(nn))
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_diff_attention_ignores_what_is_behind_the_lengths(nn, dtype):
    """NaN and infinities behind the lengths change nothing."""
    def make():
        return Case(B=3, H=2, K=1, nq=140, nk=140, d=64, dtype=dtype, causal=True, q_lens=[140, 65, 0],
                    kv_lens=[140, 65, 0])
    c, e = make(), make()
    for x in (e.q, e.k, e.v, e.do):
        x[1, :, 65:] = math.nan
        x[2] = math.inf
    a, b = c.fwd(nn), e.fwd(nn)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ga, gb = c.bwd(nn, *a), e.bwd(nn, *b)
    assert all(torch.equal(ga[n], gb[n]) for n in ga)
    assert ga["dk"][2].abs().max() == 0 and ga["dq"][1, :, 65:].abs().max() == 0


def test_diff_attention_gradients_by_differences(nn):
    """f32: (f(x + h v) - f(x - h v)) / 2h of f = <o, do> against <grad, v>, for each input."""
    c = Case(B=1, H=2, K=1, nq=12, nk=15, d=16, dtype="f32", causal=True, heads_inner=False)
    g = c.bwd(nn, *c.fwd(nn))
    h = 2.0 ** -7
    for name, x in (("dq", c.q), ("dk", c.k), ("dv", c.v), ("dlam", c.lam)):
        v = randn(x.shape, 99, torch.float32)
        v = v / v.norm()
        x0 = x.clone()
        f = []
        for s in (h, -h):
            x.copy_(x0 + s * v)
            f.append((c.fwd(nn)[0].double() * c.do).sum().item())
        x.copy_(x0)
        # third derivatives along a unit direction are below 60 here, so h^2/6 of them is below 1e-3;
        # f itself is a sum of 768 f32 values, 1e-5 over 2h
        assert abs((f[0] - f[1]) / (2 * h) - (g[name].double() * v).sum().item()) < 2e-3, name


# ---------------------------------------------------------------------------- AdamW
def adamw_ref(p, g, m, v, t, lr, b1, b2, eps, wd):
    """p, m, v after the step, and how far f32 may take p: every operation
    rounds once (a half step, 2^-24 of its result), and the errors are linear
    in the terms.  p keep: keep and the product, and the difference, 3 of |p|
    and 1 of the step (counted in the 4 and 16 below).  The step is
    rate * (m / (u / root + eps)): m has 3 of its terms b1 |m| and (1-b1) |g|
    (constant, product, sum); v has 4 of itself, so u = sqrt(v) 2 + 1; u / root
    2 more, + eps 1, the quotient 1, rate 1 and the product 1: 12 of the step
    formed with |terms| for m, which near cancellation in m exceeds the step
    itself."""
    terms = m.abs() * b1 + g.abs() * (1 - b1)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    f = lr / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + eps)
    q = p * (1 - lr * wd) - f * m
    return q, m, v, 2.0 ** -24 * (4 * (p.abs() + q.abs()) + 16 * f * terms)


SIZES = [1, 255, 256, 257, 4096, 4097, 0, 100003]
HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)


def make_tensors(sizes, dtype, seed, scale, shift=0):
    """Tensors of one flat buffer; `shift` elements off its alignment."""
    flat = randn((sum(sizes) + 4 * len(sizes) + shift,), seed, dtype, scale)
    out, at = [], shift
    for n in sizes:
        out.append(flat[at:at + n])
        at += n if shift else -(-n // 4) * 4
    return out


@pytest.mark.parametrize("p_type,g_type,masters", [("f32", "f32", False), ("bf16", "bf16", True), ("f16", "f32", True),
                                                   ("bf16", "bf16", False), ("f32", "f16", False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_32(nn, p_type, g_type, masters, shift):
    t = TYPES[p_type]
    p, g = make_tensors(SIZES, t, 1, 1.0, shift), make_tensors(SIZES, TYPES[g_type], 2, 1e-2, shift)
    w = [x.float() for x in p] if masters else None
    m = make_tensors(SIZES, torch.float32, 3, 1e-2, shift)
    v = [x.square_() for x in make_tensors(SIZES, torch.float32, 4, 1e-2, shift)]
    state = torch.tensor([6, 0], device="cuda")
    a = (0.9, 0.99, 1e-8, 0.1)
    ref = [adamw_ref((w or p)[i].double(), g[i].double(), m[i].double(), v[i].double(), 7, 3e-3, *a) for i in range(len(p))]
    nn.AdamW(p, g, m, v, state, masters=w, **HYPER).step()
    assert state.tolist() == [7, 0]
    for i in range(len(p)):
        pr, mr, vr, tol = ref[i]
        gd = g[i].double()
        # three roundings of each term of m, four of v
        assert ((m[i] - mr).abs() <= 3 * 2.0 ** -24 * (mr.abs() + 2 * gd.abs())).all()
        assert ((v[i] - vr).abs() <= 4 * 2.0 ** -24 * vr.abs() + 1e-37).all()
        if masters:
            assert ((w[i] - pr).abs() <= tol).all()
            assert torch.equal(p[i], w[i].to(t))
        else:
            assert ((p[i].double() - pr).abs() <= tol + half_step(t) * pr.abs() * (t is not torch.float32)).all()


def mix(n, tensor, t):
    low = 0xFFFFFFFF
    x = (torch.arange(n, device="cuda") * 0x9E3779B1 + t * 0x85EBCA77 + tensor * 0xC2B2AE3D) & low
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & low
    x = ((x ^ (x >> 15)) * 0x846CA68B) & low
    return x ^ (x >> 16)


E4M3 = sorted({(k / 512 if k < 8 else (8 + k % 8) / 8 * 2.0 ** (k // 8 - 7)) for k in range(127)})


@pytest.mark.parametrize("shift", [0, 1])
def test_adamw_8bit(nn, shift):
    """Each code is one of the two neighbours of the exact 64-bit value, the
    upper with the probability of the remainder by the same random bits; three
    steps, from zero states."""
    grid = torch.tensor(E4M3, dtype=torch.float64, device="cuda")
    p = make_tensors(SIZES, torch.float32, 1, 1.0, shift)
    m = [x.zero_() for x in make_tensors(SIZES, torch.float32, 3, 1.0, shift)]
    m = [torch.zeros(x.numel() + shift, dtype=torch.float8_e4m3fn, device="cuda")[shift:] for x in m]
    v = [torch.zeros_like(x) for x in m]
    ms, vs = ([torch.zeros(-(-n // 256), device="cuda") for n in SIZES] for _ in range(2))
    state = torch.tensor([0, 0], device="cuda")
    g = make_tensors(SIZES, torch.float32, 2, 1e-2, shift)
    opt = nn.AdamW(p, g, m, v, state, m_scales=ms, v_scales=vs, **HYPER)
    for t in (1, 2, 3):
        for i, x in enumerate(g):
            x.copy_(randn(x.shape, 10 * t + i, torch.float32, 1e-2))
        old = []
        for i, n in enumerate(SIZES):
            sm, sv = (s[i].double().repeat_interleave(256)[:n] for s in (ms, vs))
            old.append((p[i].double(), g[i].double(), m[i].double() * sm, (v[i].double() * sv) ** 2))
        opt.step()
        assert state.tolist() == [t, 0]
        for i, n in enumerate(SIZES):
            if not n:
                continue
            pr, mr, vr, tol = adamw_ref(*old[i], t, 3e-3, 0.9, 0.99, 1e-8, 0.1)
            assert ((p[i] - pr).abs() <= tol).all()
            r = mix(n, i, t)
            for code, scale, x, rnd, least in ((m[i], ms[i], mr, r & 0xFFFFF, False), (v[i], vs[i], vr.sqrt(), r >> 12, True)):
                pad = torch.cat([x.abs(), x.new_zeros(-n % 256)]).view(-1, 256).amax(1)
                assert ((scale.double() * 448 - pad).abs() <= 8 * 2.0 ** -24 * pad).all()
                a = x.abs() / (pad / 448).repeat_interleave(256)[:n]
                at = torch.searchsorted(grid, a.clamp(max=448.0), right=True) - 1
                lo, hi = grid[at], grid[(at + 1).clamp(max=126)]
                got = code.double().abs()
                # a is right to 16 half steps: a value that close to a code may fall to either side of it
                near = 16 * 2.0 ** -24 * a
                ok = ((got == lo) | (got == hi) | ((got - a).abs() <= near) |
                      ((got < lo) & (a - lo <= near)) | ((got > hi) & (hi - a <= near)))
                if least:
                    ok |= (got == 2.0 ** -9) & (a < 2.0 ** -9)
                assert ok.all()
                # the random bits decide: up where remainder + bits reach a whole step
                up = (a - lo) / (hi - lo).clamp(min=1e-30) + rnd.double() * 2.0 ** -20
                sure = ((up - 1).abs() > 2.0 ** -12) & (a < 448) & (a > 2.0 ** -9)
                assert torch.equal(got[sure], torch.where(up >= 1, hi, lo)[sure])
                assert ((code.double() < 0) <= (x < 0)).all()


def test_adamw_more_tensors_than_one_launch_holds(nn):
    sizes = [37 + i % 5 for i in range(600)]
    p = make_tensors(sizes, torch.float32, 1, 1.0)
    g, m, v = (make_tensors(sizes, torch.float32, s, 1e-2) for s in (2, 3, 4))
    v = [x.square_() for x in v]
    state = torch.tensor([0, 0], device="cuda")
    ref = [adamw_ref(p[i].double(), g[i].double(), m[i].double(), v[i].double(), 1, 3e-3, 0.9, 0.99, 1e-8, 0.1)
           for i in range(600)]
    nn.AdamW(p, g, m, v, state, **HYPER).step()
    assert state.tolist() == [1, 0]
    assert all(((p[i] - ref[i][0]).abs() <= ref[i][3]).all() for i in range(600))
    empty = torch.tensor([4, 0], device="cuda")
    nn.AdamW([], [], [], [], empty).step()
    assert empty.tolist() == [5, 0]


# ---------------------------------------------------------------------------- how calls are made
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,H,K,nq,nk", [(3, 4, 2, 1, 3000), (3, 12, 1, 1, 700), (300, 2, 2, 1, 300), (2, 2, 1, 7, 137),
                                         (10, 16, 4, 130, 257), (6, 4, 2, 300, 333)])
def test_diff_attention_over_caches_that_are_not_filled(nn, dtype, B, H, K, nq, nk):
    """Keys and rows behind the lengths hold NaN and infinities, in every form
    of the forward (the single-token one with 8 rows or fewer and with more, CTA
    pairs, single CTAs, f32): the result is that of zeros there."""
    kv = [nk - (37 * i + 16) % nk for i in range(B)]
    ql = [max(nq - 5 * i, 0) if nq > 1 else 1 for i in range(B)]
    make = lambda: Case(B=B, H=H, K=K, nq=nq, nk=nk, d=64, dtype=dtype, causal=True, q_lens=ql, kv_lens=kv)
    c, e = make(), make()
    for i in range(B):
        c.k[i, :, kv[i]:], c.v[i, :, kv[i]:], c.q[i, :, ql[i]:] = 0, 0, 0
        e.k[i, :, kv[i]:], e.v[i, :, kv[i]:], e.q[i, :, ql[i]:] = math.nan, math.inf if i % 2 else math.nan, math.nan
    assert all(torch.equal(x, y) for x, y in zip(c.fwd(nn), e.fwd(nn)))


def test_single_tokens_one_after_another_in_one_workspace(nn):
    """The joining kernel of a step, launched early, and the first kernel of the
    next share a workspace: each step's result is its own, also in a graph."""
    cases = [Case(B=8, H=16, K=4, nq=1, nk=9000, d=64, dtype="bf16", seed=10 * s, kv_lens=[9000 - 1000 * i for i in range(8)])
             for s in range(3)]
    want = [c.fwd(nn)[0] for c in cases]
    outs = [[torch.empty_like(want[0]) for _ in cases] for _ in range(20)]
    c = cases[0]
    ws = torch.empty(nn.diff_attention_workspace(c.q, c.k, c.v), dtype=torch.uint8, device="cuda")
    assert ws.numel()

    def steps(outs, stream=None):
        for row in outs:
            for c, o in zip(cases, row):
                nn.diff_attention_fwd(c.q, c.k, c.v, c.lam, o, None, LAM_INIT, c.scale, kv_lens=c.kv_lens, workspace=ws,
                                      stream=stream)
    steps(outs)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for row in outs for o, w in zip(row, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(outs)
    for row in outs:
        for o in row:
            o.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for row in outs for o, w in zip(row, want))


def test_diff_attention_alignments_and_strides_other_than_the_kernels_like(nn):
    """Rows off 16 bytes, keys broadcast over the batch, a negative scale."""
    c = Case(B=2, H=2, K=1, nq=70, nk=90, d=64, dtype="bf16", causal=True)
    wide = randn((2, 90, 2 * 64 + 3), 7, torch.bfloat16)
    c.k = wide[..., 3:].unflatten(-1, (2, 64)).transpose(1, 2)
    o, lse, o2 = c.fwd(nn)
    c.check({"o": o, "lse": lse, "o2": o2}, c.reference(), 90)
    c.k = randn((1, 2, 90, 64), 8, torch.bfloat16).expand(2, 2, 90, 64)
    got = c.fwd(nn)
    c.check(dict(zip(("o", "lse", "o2"), got)), c.reference(), 90)
    c.k = c.k.contiguous()
    c.scale = -0.125
    got = c.fwd(nn)
    c.check({**dict(zip(("o", "lse", "o2"), got)), **c.bwd(nn, *got)}, c.reference(backward=True), 140)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,nq,nk", [(2, 5, 0), (2, 0, 5), (0, 5, 5), (2, 1, 0)])
def test_diff_attention_of_nothing(nn, dtype, B, nq, nk):
    """No keys, no rows, no sequences: zeros where there is something to write."""
    c = Case(B=B, H=2, K=1, nq=nq, nk=nk, d=64, dtype=dtype, causal=True)
    o, lse, o2 = c.fwd(nn)
    g = c.bwd(nn, o, lse, o2)
    assert all((x == 0).all() for x in (o, o2, *g.values())) and (lse == -math.inf).all()
    empty = randn((2, 0, 5, 8), 1, TYPES[dtype])
    nn.rope(empty, torch.arange(5, device="cuda"), nn.rope_freqs(8)[0].cuda(), empty)


def test_diff_attention_offsets_past_32_bits(nn):
    """The last head of a cache whose rows stand 8192 elements apart, 2.4e9 elements in all."""
    n = 300_000
    cache = torch.zeros((1, n, 128, 64), dtype=torch.bfloat16, device="cuda")
    cache[:, :, -4:] = randn((1, n, 4, 64), 3, torch.bfloat16)
    c = Case(B=1, H=2, K=1, nq=1, nk=n, d=64, dtype="bf16", causal=True)
    c.k = cache[:, :, -4:-2].transpose(1, 2)
    c.v = cache[:, :, -2:].reshape(1, n, 1, 128).transpose(1, 2)
    assert c.k.stride(2) * n > 2 ** 31
    got = dict(zip(("o", "lse", "o2"), c.fwd(nn)))
    c.check(got, c.reference(), n)


def _everything(nn, dtype, nq, nk):
    """A layer's operators on fixed tensors: (call, its outputs)."""
    c = Case(B=3, H=4, K=2, nq=nq, nk=nk, d=64, dtype=dtype, causal=True)
    freqs = nn.rope_freqs(64)[0].cuda()
    pos = torch.arange(nq, device="cuda")
    q = torch.empty_like(c.q)
    o = torch.empty((3, 4, nq, 128), dtype=c.t, device="cuda")
    o2, lse = torch.empty_like(o), torch.empty((3, 8, nq), device="cuda")
    grads = [torch.empty_like(x) for x in (c.q, c.k, c.v, c.lam)]
    ws = torch.empty(nn.diff_attention_workspace(q, c.k, c.v, backward=True), dtype=torch.uint8, device="cuda")

    def call(stream=None):
        nn.rope(c.q, pos, freqs, q, stream=stream)
        nn.diff_attention_fwd(q, c.k, c.v, c.lam, o, lse, LAM_INIT, c.scale, causal=True, o2=o2, workspace=ws, stream=stream)
        nn.diff_attention_bwd(q, c.k, c.v, c.lam, o, o2, lse, c.do, *grads, LAM_INIT, c.scale, causal=True, workspace=ws,
                              stream=stream)
        nn.rope(grads[0], pos, freqs, grads[0], inverse=True, stream=stream)
    return call, [q, o, o2, lse, *grads]


# pairs of CTAs, single ones, the single-token form, f32
@pytest.mark.parametrize("dtype,nq,nk", [("bf16", 5000, 5000), ("f16", 300, 300), ("bf16", 1, 2000), ("f32", 70, 70)])
def test_captured_and_on_other_streams(nn, dtype, nq, nk):
    """An eager run, a captured one replayed twice over cleared outputs, and two
    runs at once on two streams give the same bits."""
    call, outs = _everything(nn, dtype, nq, nk)
    call()
    torch.cuda.synchronize()
    want = [x.clone() for x in outs]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call()
    for _ in range(2):
        for x in outs:
            x.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    other, outs2 = _everything(nn, dtype, nq, nk)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        call(s1)
        other(s2)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(outs, want, outs2))
    from amcuda import _abi
    _abi.call("amc_synchronize")      # no wait of the kernels gave up


def test_adamw_captured_with_a_rate_on_the_device(nn):
    """Each replay counts a step and reads the rate anew."""
    p, g = [randn((1000,), 1, torch.float32)], [randn((1000,), 2, torch.float32)]
    m, v = [torch.zeros(1000, device="cuda")], [torch.zeros(1000, device="cuda")]
    state, lr = torch.tensor([0, 0], device="cuda"), torch.tensor([0.5], device="cuda")
    opt = nn.AdamW(p, g, m, v, state, lr=lr, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)
    start = p[0].clone()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opt.step()
    assert state.tolist() == [0, 0] and torch.equal(p[0], start)
    x, mm, vv = start.double(), torch.zeros(1000, device="cuda").double(), torch.zeros(1000, device="cuda").double()
    for t, rate in ((1, 0.5), (2, 0.25), (3, 0.125)):
        lr.fill_(rate)
        graph.replay()
        torch.cuda.synchronize()
        x, mm, vv, tol = adamw_ref(x, g[0].double(), mm, vv, t, rate, 0.9, 0.99, 1e-8, 0.0)
        assert state.tolist() == [t, 0]
        assert ((p[0] - x).abs() <= t * tol).all()


def test_a_layer_trains(nn):
    """Projections, rotated queries and keys, differential attention and the
    optimizer as one training step: gradients of every parameter against
    autograd in 64 bits, then an AdamW step on them."""
    B, n, H, K, d, width = 2, 75, 4, 2, 16, 48
    t = torch.float32
    x, target = randn((B, n, width), 1, t), randn((B, n, H * 2 * d), 2, t)
    wq, wk, wv = (randn((width, k), 3 + i, t, 0.2) for i, k in enumerate((2 * H * d, 2 * K * d, 2 * K * d)))
    lam = randn((H, 4, d), 6, t, 0.2)
    params = [wq, wk, wv, lam]
    pos = torch.arange(n, device="cuda")
    freqs, _ = nn.rope_freqs(d)
    freqs, scale = freqs.cuda(), 1 / math.sqrt(d)

    def heads(y, h):
        return y.view(B, n, h, -1).transpose(1, 2)
    q, k, v = (x.view(B * n, width) @ w for w in params[:3])
    q, k, v = heads(q, 2 * H), heads(k, 2 * K), heads(v, K)
    nn.rope(q, pos, freqs, q, k, k)
    o = torch.empty((B, n, H, 2 * d), device="cuda").transpose(1, 2)
    o2, lse = torch.empty_like(o), torch.empty((B, 2 * H, n), device="cuda")
    nn.diff_attention_fwd(q, k, v, lam, o, lse, LAM_INIT, scale, causal=True, o2=o2)
    do = o - heads(target, H)
    dq, dk, dv, dlam = (torch.empty_like(y) for y in (q, k, v, lam))
    ws = torch.empty(nn.diff_attention_workspace(q, k, v, backward=True), dtype=torch.uint8, device="cuda")
    nn.diff_attention_bwd(q, k, v, lam, o, o2, lse, do, dq, dk, dv, dlam, LAM_INIT, scale, causal=True, workspace=ws)
    nn.rope(dq, pos, freqs, dq, dk, dk, inverse=True)
    flat = [y.transpose(1, 2).reshape(B * n, -1) for y in (dq, dk, dv)]
    grads = [x.view(B * n, width).t() @ y for y in flat] + [dlam]

    leaves = [y.double().requires_grad_() for y in params]
    q, k, v = (x.view(B * n, width).double() @ w for w in leaves[:3])
    q, k, v = heads(q, 2 * H), heads(k, 2 * K), heads(v, K)
    ang = pos.double()[:, None] * freqs
    co, si = ang.cos(), ang.sin()

    def turn(y):
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * co - b * si, b * co + a * si], -1)
    q, k = turn(q).unflatten(1, (H, 2)), turn(k).unflatten(1, (K, 2)).repeat_interleave(H // K, 1)
    s = (q @ k.transpose(-1, -2)) * scale
    p = torch.softmax(s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf), -1)
    l4 = leaves[3]
    lm = torch.exp((l4[:, 0] * l4[:, 1]).sum(-1)) - torch.exp((l4[:, 2] * l4[:, 3]).sum(-1)) + LAM_INIT
    out = (p[:, :, 0] - lm[:, None, None] * p[:, :, 1]) @ v.repeat_interleave(H // K, 1)
    loss = 0.5 * (out - heads(target, H)).square().sum()
    want = torch.autograd.grad(loss, leaves)
    for a, b in zip(grads, want):
        # f32 throughout: sums of at most 150 products of products, each a few
        # half steps off, and scores below 40 whose exponentials move 2^-16
        assert (a - b).abs().max() < 2.0 ** -13 * b.abs().max()
    m, v2 = [torch.zeros_like(y) for y in params], [torch.zeros_like(y) for y in params]
    state = torch.tensor([0, 0], device="cuda")
    before = [y.clone() for y in params]
    nn.AdamW(params, grads, m, v2, state, lr=1e-2, weight_decay=0.0).step()
    for y, z, g in zip(params, before, grads):
        # the first step is lr against the gradient's sign, but where |g| is near eps
        sure = g.abs() > 1e-4
        assert ((z - y - 1e-2 * g.sign()).abs()[sure] < 1e-5).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f16", 64), ("bf16", 32)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq", [300, 400])      # 400 without a mask: pairs of CTAs
def test_pairs_of_ctas_see_the_values_that_either_cleared(nn, dtype, d, causal, nq):
    """Both CTAs of a pair clear their columns of V behind the length, and one of
    them issues the products that read both: over lengths on every side of a
    step of 64 keys, and many launches, NaN there never reaches a result."""
    lens = [521, 520, 513, 512, 449, 447, 385, 383, 65, 1]
    make = lambda: Case(B=10, H=16, K=4, nq=nq, nk=521, d=d, dtype=dtype, causal=causal, kv_lens=lens)
    c, e = make(), make()
    for i, n in enumerate(lens):
        c.k[i, :, n:], c.v[i, :, n:] = 0, 0
        e.k[i, :, n:], e.v[i, :, n:] = math.nan, math.nan
    want = c.fwd(nn)
    for _ in range(30):
        assert all(torch.equal(x, y) for x, y in zip(want, e.fwd(nn)))


@pytest.mark.parametrize("b2", [0.0, 0.5])
def test_adamw_8bit_roots_are_rounded_to_nearest(nn, b2):
    """One element a block: its scale is sqrt(v) / 448, the root and the product
    each rounded to nearest.  From zero states v = (1 - b2) g^2, at b2 = 0 and 1/2
    one rounding of g^2 and both parities of its exponent; over the range of f32
    with its edges, in which the smallest root, 2^-74.5, is above the least scale."""
    n = 1 << 15
    g1 = torch.rand(n, generator=torch.Generator().manual_seed(3)) + 1
    g1 = g1 * 2.0 ** torch.randint(-72, 62, (n,), generator=torch.Generator().manual_seed(4)).float()
    g1[:6] = torch.tensor([2.0 ** -74, 2.0 ** -63, 1.5 * 2.0 ** -50, 2.0 ** -50 * (1 - 2.0 ** -24), 1.8e19, 1.0])
    g = torch.zeros(n, 256)
    g[:, 0] = g1
    g = g.view(-1).cuda()
    p, m, v = torch.zeros_like(g), *(torch.zeros(g.shape, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ms, vs = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    state = torch.tensor([0, 0], device="cuda")
    nn.AdamW([p], [g], [m], [v], state, beta2=b2, m_scales=[ms], v_scales=[vs]).step()
    x = (g1 * g1) * (1 - b2)                         # f32, IEEE on the host
    root = x.double().sqrt().float()                 # 53 bits, then 24: no double rounding for a root of 24 bits
    assert torch.equal(vs.cpu(), root * torch.tensor(1 / 448, dtype=torch.float32))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,H,K,nq,nk,d", [(2, 2, 1, 5, 40, 64),       # single tokens, 16 rows a key head
                                           (1, 2, 2, 1, 2000, 64),     # their parts joined
                                           (2, 4, 1, 1, 2000, 32),
                                           (1, 2, 1, 130, 140, 64),    # single CTAs
                                           (6, 16, 8, 260, 270, 64),   # pairs of CTAs
                                           (1, 1, 1, 20, 40, 100)])    # wide heads
def test_diff_attention_rows_that_hold_nan(nn, dtype, B, H, K, nq, nk, d):
    """A row of Q that holds NaN has NaN for its log-sum-exp, not the -inf of a row
    that sees no key, and NaN for its outputs and gradients; the other rows'
    results are those of a call without it."""
    make = lambda: Case(B=B, H=H, K=K, nq=nq, nk=nk, d=d, dtype=dtype)
    c, e = make(), make()
    at = nq // 2
    e.q[0, 1, at, 3] = math.nan               # map 2 of head 0
    (o, lse, o2), (on, lsen, o2n) = c.fwd(nn), e.fwd(nn)
    assert lsen[0, 1, at].isnan() and on[0, 0, at].isnan().all() and o2n[0, 0, at].isnan().all()
    assert lsen.isnan().sum() == 1 and on.isnan().sum() == o2n.isnan().sum() == on.shape[3]
    for x, y in ((o, on), (o2, o2n), (lse, lsen)):
        fine = ~y.isnan()
        assert torch.equal(x[fine], y[fine])
    g = e.bwd(nn, on, lsen, o2n)
    assert g["dq"][0, :2, at].isnan().all() and g["dv"][0, 0].isnan().all() and g["dlam"][0].isnan().all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nk,d", [(1, 700, 64), (140, 150, 64), (20, 30, 100)])
def test_diff_attention_rows_whose_scores_are_all_minus_infinity(nn, dtype, nq, nk, d):
    """Finite queries and keys whose products pass the range of f32: such a row
    weighs no key, so its results and its gradients are 0, like those of a row
    that sees none, and the other rows' are finite."""
    c = Case(B=1, H=1, K=1, nq=nq, nk=nk, d=d, dtype=dtype, heads_inner=False)
    c.q[..., 0], c.k[..., 0] = 0, -1e20
    at = nq // 2
    c.q[0, :, at, 0] = 1e25
    o, lse, o2 = c.fwd(nn)
    assert (lse[0, :, at] == -math.inf).all() and (o[0, 0, at] == 0).all() and (o2[0, 0, at] == 0).all()
    g = c.bwd(nn, o, lse, o2)
    assert (g["dq"][0, :, at] == 0).all()
    assert all(torch.isfinite(x).all() for x in g.values())


def test_adamw_8bit_keeps_a_nan(nn):
    """A gradient's NaN stays in its element's parameter and states, as in 32-bit
    states, and its block's other elements are as without it; an infinity makes
    its block's scales infinite, and the block NaN at the next step."""
    n = 1024

    def run(bad):
        p = randn((n,), 1, torch.float32)
        m, v = (torch.zeros(n, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
        ms, vs = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
        g = randn((n,), 2, torch.float32)
        g[5], g[256:512] = 0.0, 0.0
        for i, x in bad.items():
            g[i] = x
        opt = nn.AdamW([p], [g], [m], [v], torch.tensor([0, 0], device="cuda"), m_scales=[ms], v_scales=[vs], **HYPER)
        opt.step()
        first = [p.clone(), m.float(), v.float(), ms.clone(), vs.clone()]
        g.copy_(randn((n,), 3, torch.float32))
        opt.step()
        return first, [p.clone(), m.float(), v.float(), ms, vs]
    nan = {5: math.nan, **{i: math.nan for i in range(256, 512)}}
    where = torch.zeros(n, dtype=torch.bool, device="cuda")
    where[list(nan)] = True
    for a, b in zip(run({}), run(nan)):
        for x, y in zip(a[:3], b[:3]):
            assert torch.equal(y.isnan(), where) and torch.equal(x[~where], y[~where])
        keep = [0, 2, 3]
        assert torch.equal(a[3][keep], b[3][keep]) and torch.equal(a[4][keep], b[4][keep])
    first, second = run({600: math.inf})
    block = torch.arange(n, device="cuda") // 256 == 2
    assert first[3].isinf().tolist() == first[4].isinf().tolist() == [False, False, True, False]
    assert first[1][600].isnan() and first[2][600].isnan() and first[1].isnan().sum() == 1
    assert second[0].isnan()[block].all() and not second[0].isnan()[~block].any()


def turns_exactly(pos, freq):
    """pos * freq / 2 pi less whole turns, in rationals (freq is a double, 1 / 2 pi to 60 digits)."""
    from fractions import Fraction
    tau = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)
    t = pos * Fraction(freq) / tau
    return float(t - round(t))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_far_positions_in_32_bits(nn, interleaved):
    """Positions up to 2^53 keep the angle of position times frequency, against an
    exact reduction on the host: the allowance is that of near positions."""
    d = 64
    at = [0, 1, 4097, (1 << 20) + 7, (1 << 30) + 12345, (1 << 33) + 987654321, (1 << 40) + 1234567, (1 << 47) - 1,
          (1 << 53) - 1, -((1 << 40) + 77)]
    freqs, _ = nn.rope_freqs(d)
    turns = torch.tensor([[turns_exactly(p, f) for f in freqs.tolist()] for p in at], dtype=torch.float64, device="cuda")
    c, s = (2 * math.pi * turns).cos(), (2 * math.pi * turns).sin()
    x = randn((1, 2, len(at), d), 7, torch.float32)
    out = torch.empty_like(x)
    nn.rope(x, torch.tensor(at, device="cuda"), freqs.cuda(), out, interleaved=interleaved)
    ia, ib = (slice(0, d, 2), slice(1, d, 2)) if interleaved else (slice(0, d // 2), slice(d // 2, d))
    xd = x.double()
    y, terms = torch.empty_like(xd), torch.empty_like(xd)
    y[..., ia], y[..., ib] = xd[..., ia] * c - xd[..., ib] * s, xd[..., ib] * c + xd[..., ia] * s
    terms[..., ia] = terms[..., ib] = xd[..., ia].abs() + xd[..., ib].abs()
    rope_close(out, y, terms, torch.float32)


SMALL_AND_LARGE = [
    # upstream gradients far below 1, as before a loss is scaled up: dS is below fp16's least number, its sums are not
    dict(B=2, H=2, K=2, nq=300, nk=2000, d=64, up=2.0 ** -17, shift=4.0),
    dict(B=2, H=4, K=1, nq=1000, nk=1000, d=64, up=2.0 ** -19, shift=4.0, causal=True, q_lens=[1000, 700], kv_lens=[1000, 900]),
    dict(B=1, H=2, K=1, nq=1500, nk=1500, d=32, up=2.0 ** -19, shift=4.0),
    # and far above it: dS passes 65504, and the products with a small scale do not
    dict(B=1, H=2, K=1, nq=40, nk=4, d=64, up=2.0 ** 13, gain=8.0, scale=1 / 64),
    dict(B=2, H=4, K=2, nq=40, nk=3, d=32, up=2.0 ** 13, gain=8.0, scale=1 / 64, causal=True),
    # keys whose weight is below fp16's least in every row: dV is a sum of many
    dict(B=1, H=2, K=2, nq=2000, nk=64, d=64, up=8.0, far=17.0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(SMALL_AND_LARGE)))
def test_diff_attention_gradients_of_any_size(nn, dtype, case):
    """Where the operands of the gradients' products would leave the range of
    fp16, the gradients are still as near as `check` has them."""
    a = dict(SMALL_AND_LARGE[case])
    up, shift, gain, far = (a.pop(n, 0.0) for n in ("up", "shift", "gain", "far"))
    c = Case(dtype=dtype, **a)
    c.do *= up
    c.q[..., 0] += shift
    c.lam *= 0.25
    if gain:
        c.q *= gain
    if far:
        # half of the keys lie 17 nats behind the others: weights of about 2^-30
        c.q[..., 1], c.k[..., 1] = 4.0, 0.0
        c.k[:, :, ::2, 1] = -far / 4 / c.scale
    got, ref = c.bwd(nn, *c.fwd(nn)), c.reference(backward=True)
    for name, x in got.items():
        # a result within its rounding, u and twice u of its terms, of the type's
        # largest number may be infinite; there are few of them
        y, terms = ref[name]
        over = y.abs() + 4 * half_step(c.t) * terms > torch.finfo(c.t).max
        assert over.sum() < 0.1 * over.numel() and ((x[over].double() - y[over]).abs() < 2 * terms[over]).logical_or(x[over] == y[over].sign() * math.inf).all()
        x[over] = y[over] = 0
    c.check(got, ref, max(c.k.shape[2], c.q.shape[2] * c.H // c.K))


SINGLE_TOKENS = [dict(B=40, H=2, K=1, nq=3, nk=5000, d=16), dict(B=3, H=4, K=1, nq=1, nk=1500, d=64, causal=True),
                 dict(B=7, H=4, K=2, nq=1, nk=3001, d=64, causal=True, kv_lens=[3001, 64, 500, 0, 65, 1, 2900]),
                 dict(B=1, H=16, K=1, nq=1, nk=20000, d=64), dict(B=2, H=12, K=1, nq=1, nk=4099, d=32, dv=128),
                 dict(B=300, H=2, K=2, nq=1, nk=900, d=64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(SINGLE_TOKENS)))
def test_single_tokens_round_no_weight(nn, dtype, case):
    """The single-token form carries a weight as two 16-bit values: what is left
    out is u^2 of it, not u, so a box of 16 keys that went missing would show.
    Beside it the scores' 2^-16 (as in `check`), and f32 sums: a warp's chain of
    nk / 64 products at most, 16 terms in each, and one of all CTAs' parts."""
    c = Case(dtype=dtype, **SINGLE_TOKENS[case])
    assert c.H // c.K * c.q.shape[2] <= 16
    u, nk = half_step(c.t), c.k.shape[2]
    o, _, o2 = c.fwd(nn)
    ref = c.reference()
    for x, (y, terms) in ((o, ref["o"]), (o2, ref["o2"])):
        tol = u * y.abs() + (2.0 ** -16 + u * u + 2.0 ** -23 * (nk / 64 + 16 + 296)) * terms + 1e-30
        if dtype == "f16":
            tol = tol + 2.0 ** -24
        assert ((x.double() - y).abs() <= tol).all(), ((x.double() - y).abs() / tol).max()


EVERY_KEY = [dict(B=2, H=4, K=1, nq=1, nk=3001, d=64, kv_lens=[3001, 2900]), dict(B=1, H=16, K=1, nq=1, nk=9000, d=64),
             dict(B=300, H=2, K=2, nq=1, nk=300, d=64), dict(B=1, H=2, K=1, nq=140, nk=700, d=64, kv_lens=[641]),
             dict(B=20, H=8, K=2, nq=200, nk=521, d=64, kv_lens=[521 - 7 * i for i in range(20)]),
             dict(B=1, H=2, K=1, nq=40, nk=300, d=100, dv=128)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", range(len(EVERY_KEY)))
def test_every_key_counts(nn, dtype, case):
    """Each column of V is 1 at one key and 0 elsewhere, keys at the edges of boxes,
    steps and tiles among them: a result is that key's weight alone, to the
    rounding of that weight."""
    c = Case(dtype=dtype, **EVERY_KEY[case])
    nk, dv = c.k.shape[2], c.v.shape[3]
    keys = sorted({k for e in (0, 16, 32, 48, 64, 128, 256, 512, 1024, nk) for k in (e - 1, e, e + 1) if 0 <= k < nk})
    rest = torch.randperm(nk, generator=torch.Generator().manual_seed(1)).tolist()
    keys += [k for k in rest if k not in keys][:dv - len(keys)]
    c.v.zero_()
    c.v[:, :, keys, list(range(dv))] = 1
    o, lse, o2 = c.fwd(nn)
    c.check({"o": o, "lse": lse, "o2": o2}, c.reference(), 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("d,dv", [(128, 256), (128, 8), (72, 136), (96, 192), (64, 256), (65, 129), (1, 1), (8, 8)])
@pytest.mark.parametrize("nq", [1, 70])
def test_head_dims_up_to_their_limits(nn, dtype, d, dv, nq):
    c = Case(B=2, H=4, K=2, nq=nq, nk=100, d=d, dv=dv, dtype=dtype, causal=True, q_lens=[nq, min(nq, 40)], kv_lens=[100, 61])
    o, lse, o2 = c.fwd(nn)
    got = {"o": o, "lse": lse, "o2": o2, **c.bwd(nn, o, lse, o2)}
    c.check(got, c.reference(backward=True), 140)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("a", [dict(B=4, H=6, K=2, nq=333, nk=333, d=48, causal=True),      # heads of a key head shared by a cluster
                               dict(B=4, H=2, K=2, nq=150, nk=290, d=32),
                               dict(B=10, H=16, K=4, nq=150, nk=290, d=64, causal=True),
                               dict(B=4, H=4, K=1, nq=1, nk=300, d=64, causal=True),
                               dict(B=4, H=2, K=1, nq=45, nk=70, d=100, causal=True)])
def test_gradients_of_batches_that_are_not_filled(nn, dtype, a):
    """NaN and infinities behind the lengths change no gradient, in every form of the backward."""
    B, nq, nk = a["B"], a["nq"], a["nk"]
    kv = [nk - (37 * i + 1) % nk for i in range(B)]
    ql = kv if nq == nk else [max(nq - 5 * i, 0) if nq > 1 else 1 for i in range(B)]
    make = lambda: Case(dtype=dtype, q_lens=ql, kv_lens=kv, **a)
    c, e = make(), make()
    for i in range(B):
        for x, n in ((c.q, ql), (c.do, ql), (c.k, kv), (c.v, kv)):
            x[i, :, n[i]:] = 0
        for x, n in ((e.q, ql), (e.do, ql), (e.k, kv), (e.v, kv)):
            x[i, :, n[i]:] = math.inf if i % 2 else math.nan
    ga, gb = c.bwd(nn, *c.fwd(nn)), e.bwd(nn, *e.fwd(nn))
    assert all(torch.equal(ga[n], gb[n]) for n in ga) and all(torch.isfinite(x).all() for x in ga.values())


PAIRS = [dict(B=10, H=16, K=4, nq=400, nk=257, d=64, q_lens=[400, 0, 1, 129, 128, 127, 257, 400, 256, 2],
              kv_lens=[257, 257, 0, 5, 256, 255, 129, 64, 65, 200]),
         dict(B=5, H=16, K=16, nq=512, nk=300, d=32, kv_lens=[300, 0, 299, 128, 1]),
         dict(B=3, H=25, K=5, nq=390, nk=700, d=48),
         dict(B=19, H=8, K=8, nq=256, nk=1, d=64),
         dict(B=2, H=40, K=8, nq=1024, nk=2048, d=64, q_lens=[1024, 900], kv_lens=[2048, 1985])]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(PAIRS)))
def test_many_rows_over_few_keys(nn, dtype, case):
    """The form of the forward on pairs of CTAs, several tiles a pair: its results,
    their repetition, in a graph too, and rows that hold NaN."""
    c = Case(dtype=dtype, **PAIRS[case])
    got = c.fwd(nn)
    c.check(dict(zip(("o", "lse", "o2"), got)), c.reference(), c.k.shape[2])
    again = [torch.empty_like(x) for x in got]
    ws = torch.empty(nn.diff_attention_workspace(c.q, c.k, c.v), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nn.diff_attention_fwd(c.q, c.k, c.v, c.lam, again[0], again[1], LAM_INIT, c.scale, q_lens=c.q_lens,
                              kv_lens=c.kv_lens, o2=again[2], workspace=ws)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    c.q[0, 3, 140, 5] = math.nan
    o, lse, o2 = c.fwd(nn)
    assert lse[0, 3, 140].isnan() and lse.isnan().sum() == 1 and o[0, 1, 140].isnan().all()
    assert all(torch.equal(x[~y.isnan()], y[~y.isnan()]) for x, y in zip(got, (o, lse, o2)))
    from amcuda import _abi
    _abi.call("amc_synchronize")      # no wait of the kernels gave up
