"""The operators of a differential-attention layer and of its training step,
as measured cases: rotary positions, differential attention (forward,
training step, single-token decode) and the AdamW step over many tensors.

`run` computes a case in its plain form (elementary torch operations in 32
bits, 64 where 32 lose what matters) or, with `own` set, by the calls a user
makes of `amcuda.nn`.  `exact` gives the same outputs in 64 bits.
"""
import itertools
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path("array-morphisms_b200").resolve()))

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LAM_INIT = 0.8
QBLOCK = 256            # elements that share one scale of an 8-bit state
QMAX = 448.0            # the largest e4m3 value


def listed():
    return [
        # one decode step's rotation: 16 sequences, each at its own far position
        {"name": "rope_token", "op": "rope", "dtype": "bf16", "batch": 16, "heads": 16, "heads2": 4, "n": 1, "d": 64,
         "rot": 64, "interleaved": False, "inverse": False, "far": 200000, "factor": 16.0},
        # a training batch's query and key maps (16 x 2048 tokens, head dim 64)
        {"name": "rope_train", "op": "rope", "dtype": "bf16", "batch": 16, "heads": 16, "heads2": 16, "n": 2048, "d": 64,
         "rot": 64, "interleaved": False, "inverse": False, "far": 0, "factor": 1.0},
        # the gradient of an interleaved rotation of part of the head, odd length
        {"name": "rope_grad_partial", "op": "rope", "dtype": "f32", "batch": 3, "heads": 12, "heads2": 4, "n": 1037,
         "d": 80, "rot": 48, "interleaved": True, "inverse": True, "far": 30000, "factor": 8.0},
        # a long prompt: causal, four query heads to a key head
        {"name": "diff_prompt", "op": "diff_fwd", "dtype": "bf16", "batch": 4, "heads": 16, "kv_heads": 4, "nq": 4096,
         "nk": 4096, "d": 64, "causal": True, "ragged": False},
        # a padded batch of prompts that continue a cached prefix
        {"name": "diff_padded", "op": "diff_fwd", "dtype": "f16", "batch": 6, "heads": 8, "kv_heads": 2, "nq": 333,
         "nk": 777, "d": 64, "causal": True, "ragged": True},
        # 32-bit inference on short sequences
        {"name": "diff_f32", "op": "diff_fwd", "dtype": "f32", "batch": 4, "heads": 8, "kv_heads": 8, "nq": 512,
         "nk": 512, "d": 64, "causal": False, "ragged": False},
        # the training step at the attention workload's size: 16 x 16 maps x 2048 x 64
        {"name": "diff_train", "op": "diff_train", "dtype": "bf16", "batch": 16, "heads": 8, "kv_heads": 8, "nq": 2048,
         "nk": 2048, "d": 64, "causal": False, "ragged": False},
        # the training step of a padded causal batch with shared key heads and a narrow head
        {"name": "diff_train_padded", "op": "diff_train", "dtype": "bf16", "batch": 5, "heads": 6, "kv_heads": 2,
         "nq": 1000, "nk": 1000, "d": 48, "causal": True, "ragged": True},
        # one new token for each of 8 sequences over long caches
        {"name": "diff_token_long", "op": "diff_fwd", "dtype": "bf16", "batch": 8, "heads": 16, "kv_heads": 4, "nq": 1,
         "nk": 32768, "d": 64, "causal": True, "ragged": True},
        # one new token over a short cache: latency
        {"name": "diff_token_short", "op": "diff_fwd", "dtype": "bf16", "batch": 1, "heads": 8, "kv_heads": 8, "nq": 1,
         "nk": 137, "d": 64, "causal": True, "ragged": False},
        # the optimizer step of a mixed-precision model: 16-bit parameters, 32-bit masters and states
        {"name": "adamw_masters", "op": "adamw", "dtype": "bf16", "masters": True, "bits": 32, "layers": 24, "width": 1024,
         "step": 1000},
        # the same step with the states in 8 bits and 32-bit parameters
        {"name": "adamw_8bit", "op": "adamw", "dtype": "f32", "masters": False, "bits": 8, "layers": 12, "width": 1024,
         "step": 100},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "diff_fwd", "diff_fwd", "diff_train", "diff_token", "adamw"])
    if op == "rope":
        d = rng.choice([32, 48, 64, 80, 128])
        rot = rng.choice([d, d, d // 2 // 2 * 2])
        n = _log(rng, 1, 4096)
        batch = rng.randint(1, max(1, min(16, 32768 // n)))
        return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "batch": batch, "heads": rng.randint(1, 16),
                "heads2": rng.choice([0, 1, 4, 8]), "n": n, "d": d, "rot": rot, "interleaved": rng.random() < 0.5,
                "inverse": rng.random() < 0.5, "far": rng.choice([0, 100000]), "factor": rng.choice([1.0, 4.0, 32.0])}
    if op == "adamw":
        bits = rng.choice([8, 32])
        dtype = rng.choice(["f32", "bf16", "f16"])
        return {"op": op, "dtype": dtype, "masters": dtype != "f32" and rng.random() < 0.7, "bits": bits,
                "layers": rng.randint(1, 12), "width": _log(rng, 31, 1024), "step": _log(rng, 1, 100000)}
    kv = rng.choice([1, 2, 4])
    heads = kv * rng.choice([1, 2, 4])
    d = rng.choice([32, 48, 64, 64, 64])
    ragged = rng.random() < 0.5
    if op == "diff_token":
        nk = _log(rng, 64, 32768)
        batch = rng.randint(1, 8)
        return {"op": "diff_fwd", "dtype": rng.choice(["bf16", "f16"]), "batch": batch, "heads": heads, "kv_heads": kv,
                "nq": rng.choice([1, 1, 2, 4]), "nk": nk, "d": d, "causal": True, "ragged": ragged}
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    n = _log(rng, 32, 512 if dtype == "f32" else 2048)
    batch = rng.randint(1, max(1, min(8, 8192 // n)))
    if op == "diff_train":
        return {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv, "nq": n, "nk": n, "d": d,
                "causal": rng.random() < 0.6, "ragged": ragged}
    return {"op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv, "nq": n,
            "nk": n + (rng.randint(0, 500) if rng.random() < 0.5 else 0), "d": d, "causal": rng.random() < 0.6,
            "ragged": ragged}


# ------------------------------------------------------------------ inputs
def _randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _heads_first(batch, n, heads, d, g, dtype):
    """A projection's output (batch, n, heads, d), seen heads first."""
    return _randn((batch, n, heads, d), g, dtype).transpose(1, 2)


def _freqs(c):
    """Radians per position of each rotated pair; positions interpolated by `factor` where a pair turns less than
    once in the original 4096 positions, kept where it turns more than 32 times, and a ramp between."""
    i = torch.arange(0, c["rot"], 2, dtype=torch.float64)
    f = 10000.0 ** (-i / c["rot"])
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return f * keep + f / c["factor"] * (1 - keep)


def _mscale(c):
    return 1.0 if c["factor"] <= 1 else 0.1 * math.log(c["factor"]) + 1.0


def _adamw_sizes(c):
    """The tensors of `layers` blocks of a model of this width: four square and two wide matrices, a vector of odd
    length; matrices are counted by their elements."""
    w = c["width"]
    return [w * w, w * w, w * w, w * w, 4 * w * w, 4 * w * w, 2 * w + 1] * c["layers"]


def _pieces(sizes, dtype, block=1):
    """One flat buffer and a view of it for each tensor, each on a boundary of 64 elements."""
    n = [-(-s // block) for s in sizes]
    starts = list(itertools.accumulate(((k + 63) // 64 * 64 for k in n), initial=0))
    flat = torch.zeros(starts[-1], dtype=dtype, device="cuda")
    return flat, [flat[s:s + k] for s, k in zip(starts, n)]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "rope":
        t = DTYPES[c["dtype"]]
        s["x"] = _heads_first(c["batch"], c["n"], c["heads"], c["d"], g, t)
        s["x2"] = _heads_first(c["batch"], c["n"], c["heads2"], c["d"], g, t) if c["heads2"] else None
        at = torch.randint(0, c["far"] + 1, (c["batch"], 1), generator=g, device="cuda")
        s["pos"] = at + torch.arange(c["n"], device="cuda")
        s["freqs"], s["mscale"] = _freqs(c).cuda(), _mscale(c)
    elif c["op"] == "adamw":
        t, sizes = DTYPES[c["dtype"]], _adamw_sizes(c)
        s["p_flat"], s["p"] = _pieces(sizes, t)
        s["g_flat"], s["g"] = _pieces(sizes, t)
        p = torch.randn(s["p_flat"].shape, generator=g, device="cuda") * 0.02
        s["p_flat"].copy_(p)
        s["g_flat"].copy_(torch.randn(p.shape, generator=g, device="cuda") * 1e-3)
        s["w_flat"], s["w"] = _pieces(sizes, torch.float32) if c["masters"] else (None, None)
        if c["masters"]:
            s["w_flat"].copy_(p)
        m = torch.randn(p.shape, generator=g, device="cuda") * 3e-4
        v = (torch.randn(p.shape, generator=g, device="cuda") * 1e-3).square() + 1e-8
        kind = torch.float32 if c["bits"] == 32 else torch.float8_e4m3fn
        s["m_flat"], s["m"] = _pieces(sizes, kind)
        s["v_flat"], s["v"] = _pieces(sizes, kind)
        if c["bits"] == 32:
            s["m_flat"].copy_(m)
            s["v_flat"].copy_(v)
        else:
            # codes and scales as a running optimizer holds them
            s["m_flat"].copy_((m * (QMAX / 2e-3)).clamp(-QMAX, QMAX))
            s["v_flat"].copy_((v.sqrt() * (QMAX / 5e-3)).clamp(2.0 ** -9, QMAX))
            s["ms_flat"], s["ms"] = _pieces(sizes, torch.float32, QBLOCK)
            s["vs_flat"], s["vs"] = _pieces(sizes, torch.float32, QBLOCK)
            s["ms_flat"].fill_(2e-3 / QMAX)
            s["vs_flat"].fill_(5e-3 / QMAX)
        s["t"] = torch.tensor([c["step"], 0], dtype=torch.int64, device="cuda")
    else:
        t = DTYPES[c["dtype"]]
        B, H, K, d = c["batch"], c["heads"], c["kv_heads"], c["d"]
        s["q"] = _heads_first(B, c["nq"], 2 * H, d, g, t)
        s["k"] = _heads_first(B, c["nk"], 2 * K, d, g, t)
        s["v"] = _heads_first(B, c["nk"], K, 2 * d, g, t)
        s["lam"] = _randn((H, 4, d), g, t, 0.1)
        s["q_lens"] = s["kv_lens"] = None
        if c["ragged"]:
            # lengths of a padded batch; one sequence at full length, later ones down to nothing
            u = torch.rand(B, generator=g, device="cuda")
            u[0] = 1.0
            s["kv_lens"] = (u * c["nk"]).round().to(torch.int32)
            full = c["nq"] == c["nk"]
            s["q_lens"] = s["kv_lens"].clone() if full else (u * c["nq"]).ceil().to(torch.int32)
        if c["op"] == "diff_train":
            s["do"] = _heads_first(B, c["nq"], H, 2 * d, g, t)
        s["scale"] = 1.0 / math.sqrt(d)
    return s


# ------------------------------------------------------------------ plain forms
def _rope_plain(x, pos, freqs, mscale, rot, interleaved, inverse):
    ang = pos[:, None, :, None].double() * freqs
    co, si = (ang.cos() * mscale).float(), (ang.sin() * (-mscale if inverse else mscale)).float()
    y = x.float().clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a], y[..., b] = xa * co - xb * si, xb * co + xa * si
    return y.to(x.dtype)


def _visible(s, c):
    """(B, 1, 1, 1, nq, nk): the keys that a row attends to."""
    i = torch.arange(c["nq"], device="cuda")[:, None]
    j = torch.arange(c["nk"], device="cuda")[None, :]
    nq = s["q_lens"][:, None, None] if s["q_lens"] is not None else c["nq"]
    nk = s["kv_lens"][:, None, None] if s["kv_lens"] is not None else c["nk"]
    ok = (i < nq) & (j < nk)
    if c["causal"]:
        ok = ok & (j <= i + nk - nq)
    return ok.reshape(-1, 1, 1, 1, c["nq"], c["nk"])


def _diff_plain(s, c):
    B, H, K, d = c["batch"], c["heads"], c["kv_heads"], c["d"]
    G = H // K
    q = s["q"].float().reshape(B, K, G, 2, c["nq"], d)
    k = s["k"].float().reshape(B, K, 1, 2, c["nk"], d)
    v = s["v"].float().reshape(B, K, 1, 1, c["nk"], 2 * d)
    ok = _visible(s, c)
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    x = torch.where(ok, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = p / torch.where(total == 0, 1.0, total)
    om = p @ v
    e = torch.exp((s["lam"][:, 0::2].float() * s["lam"][:, 1::2].float()).sum(-1))
    lam = (e[:, 0] - e[:, 1] + LAM_INIT).reshape(1, K, G, 1, 1)
    o = om[:, :, :, 0] - lam * om[:, :, :, 1]
    out = {"o": o.reshape(B, H, c["nq"], 2 * d).to(s["q"].dtype), "lse": lse.reshape(B, 2 * H, c["nq"])}
    if c["op"] != "diff_train":
        return out
    t = s["q"].dtype
    do = s["do"].float().reshape(B, K, G, c["nq"], 2 * d)
    dp = do @ v[:, :, 0].transpose(-1, -2)
    row = (do.unsqueeze(3) * om).sum(-1, keepdim=True)
    sign = torch.cat([torch.ones_like(lam), -lam], 3).unsqueeze(-1)
    ds = p * (dp.unsqueeze(3) - row) * sign * s["scale"]
    dlam = -row[:, :, :, 1].double().sum((0, 3, 4)).reshape(H, 1).float()
    w = dlam * e * torch.tensor([1.0, -1.0], device="cuda")
    w = w.repeat_interleave(2, 1).unsqueeze(-1)
    out["dq"] = (ds @ k).reshape(B, 2 * H, c["nq"], d).to(t)
    out["dk"] = (ds.transpose(-1, -2) @ q).sum(2).reshape(B, 2 * K, c["nk"], d).to(t)
    both = p[:, :, :, 0] - lam * p[:, :, :, 1]
    out["dv"] = (both.transpose(-1, -2) @ do).sum(2).to(t)
    out["dlam"] = (w * s["lam"].float()[:, [1, 0, 3, 2]]).to(t)
    return out


def _hash(n, tensor, t):
    """32 mixed bits for each element of a tensor, from its place, its tensor and the step (the lowbias32 mixer)."""
    low = 0xFFFFFFFF
    x = (torch.arange(n, device="cuda") * 0x9E3779B1 + t * 0x85EBCA77 + tensor * 0xC2B2AE3D) & low
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & low
    x = ((x ^ (x >> 15)) * 0x846CA68B) & low
    return x ^ (x >> 16)


def _blocks(x):
    n = x.numel()
    return torch.cat([x, x.new_zeros(-n % QBLOCK)]).view(-1, QBLOCK)


def _spread(scale, n):
    return scale.repeat_interleave(QBLOCK)[:n]


def _to_8bit(x, rnd, least):
    """x >= 0 over its block's largest value as e4m3, rounded up or down at random (20 random bits), and the scales."""
    top = _blocks(x).amax(1)
    some = top >= 2.0 ** -100
    scale = torch.where(some, top * (1 / QMAX), 0.0)
    a = x * _spread(torch.where(some, QMAX / torch.where(some, top, 1.0), 0.0), x.numel())
    coarse = ((a.view(torch.int32) + rnd.to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    fine = torch.floor(a * 512.0 + rnd.float() * 2.0 ** -20) * (1 / 512.0)
    code = torch.where(a < 2.0 ** -6, fine, coarse).clamp(max=QMAX)
    if least:
        code = torch.where((a > 0) & (code == 0), 2.0 ** -9, code)
    return code, scale


LR, B1, B2, EPS, DECAY = 1e-3, 0.9, 0.95, 1e-8, 0.1


def _adamw_one(s, c, i, t, rate, root):
    n = s["p"][i].numel()
    p = (s["w"] or s["p"])[i].float()
    g = s["g"][i].float()
    m, v = s["m"][i].float(), s["v"][i].float()
    if c["bits"] == 8:
        m = m * _spread(s["ms"][i], n)
        v = (v * _spread(s["vs"][i], n)).square()
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    p = p * (1 - LR * DECAY) - rate * (m / (v.sqrt() / root + EPS))
    if c["masters"]:
        s["w"][i].copy_(p)
    s["p"][i].copy_(p)
    if c["bits"] == 32:
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
        return
    x = _hash(n, i, t)
    code, scale = _to_8bit(m.abs(), x & 0xFFFFF, False)
    s["m"][i].copy_(torch.copysign(code, m))
    s["ms"][i].copy_(scale)
    code, scale = _to_8bit(v.sqrt(), x >> 12, True)
    s["v"][i].copy_(code)
    s["vs"][i].copy_(scale)


def _adamw_plain(s, c):
    s["t"][0] += 1
    t = s["t"][0]
    rate = (LR / (1 - B1 ** t.double())).float()
    root = (1 - B2 ** t.double()).sqrt().float()
    [_adamw_one(s, c, i, t, rate, root) for i in range(len(s["p"]))]


def _adamw_outputs(s):
    return {k: s[k] for k in ("p_flat", "w_flat", "m_flat", "v_flat", "ms_flat", "vs_flat", "t") if s.get(k) is not None}


# ------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"] == "rope":
        more = (s["mscale"], c["rot"], c["interleaved"], c["inverse"])
        return [_rope_plain(x, s["pos"], s["freqs"], *more) for x in (s["x"], s["x2"]) if x is not None]
    if c["op"] == "adamw":
        _adamw_plain(s, c)
        return _adamw_outputs(s)
    return _diff_plain(s, c)


def _own(s, c):
    from amcuda import nn
    if c["op"] == "rope":
        out, out2 = torch.empty_like(s["x"]), torch.empty_like(s["x2"]) if s["x2"] is not None else None
        nn.rope(s["x"], s["pos"], s["freqs"], out, s["x2"], out2, mscale=s["mscale"], interleaved=c["interleaved"],
                inverse=c["inverse"])
        return [out] if out2 is None else [out, out2]
    if c["op"] == "adamw":
        if "opt" not in s:
            s["opt"] = nn.AdamW(s["p"], s["g"], s["m"], s["v"], s["t"], LR, B1, B2, EPS, DECAY, masters=s["w"],
                                m_scales=s.get("ms"), v_scales=s.get("vs"))
        s["opt"].step()
        return _adamw_outputs(s)
    q, k, v, train = s["q"], s["k"], s["v"], c["op"] == "diff_train"
    if "ws" not in s:
        n = nn.diff_attention_workspace(q, k, v, backward=train)
        s["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    o = torch.empty((c["batch"], c["heads"], c["nq"], 2 * c["d"]), dtype=q.dtype, device="cuda")
    lse = torch.empty((c["batch"], 2 * c["heads"], c["nq"]), dtype=torch.float32, device="cuda")
    o2 = torch.empty_like(o) if train else None
    more = {"causal": c["causal"], "q_lens": s["q_lens"], "kv_lens": s["kv_lens"], "workspace": s["ws"]}
    nn.diff_attention_fwd(q, k, v, s["lam"], o, lse, LAM_INIT, s["scale"], o2=o2, **more)
    if not train:
        return {"o": o, "lse": lse}
    dq, dk, dv, dlam = (torch.empty_like(x) for x in (q, k, v, s["lam"]))
    nn.diff_attention_bwd(q, k, v, s["lam"], o, o2, lse, s["do"], dq, dk, dv, dlam, LAM_INIT, s["scale"], **more)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


# ------------------------------------------------------------------ work
def _pairs(c):
    """(row, key) pairs of one map of the whole batch at full lengths, and the keys that any row sees."""
    nq, nk = c["nq"], c["nk"]
    if not c["causal"]:
        return c["batch"] * nq * nk
    first = nk - nq
    return c["batch"] * sum(min(nk, max(0, first + i + 1)) for i in (0, nq - 1)) * nq // 2


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["batch"] * c["n"] * (c["heads"] + c["heads2"])
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": 2 * n * c["d"] * size + 8 * c["batch"] * c["n"] + 4 * c["rot"], "flops": 3 * n * c["rot"]}
    if c["op"] == "adamw":
        n = sum(_adamw_sizes(c))
        size = 4 if c["dtype"] == "f32" else 2
        states = 16 if c["bits"] == 32 else 4 + 16 / QBLOCK
        params = size + 8 if c["masters"] else 2 * size
        return {"bytes": n * (size + params + states), "flops": 14 * n}
    size = 4 if c["dtype"] == "f32" else 2
    q = c["batch"] * c["nq"] * 2 * c["heads"] * c["d"] * size
    kv = c["batch"] * c["nk"] * 4 * c["kv_heads"] * c["d"] * size
    lse = c["batch"] * c["nq"] * 2 * c["heads"] * 4
    # a map's scores cost d products a pair and its values 2d; ragged lengths are uniform over the range
    part = 1.0
    if c["ragged"]:
        part = (1 + (c["batch"] - 1) * (1 / 3 if c["nq"] > 4 else 1 / 2)) / c["batch"]
    fwd = 2 * 6 * c["d"] * c["heads"] * _pairs(c) * part
    if c["op"] == "diff_fwd":
        return {"bytes": 2 * q + kv * (part if c["nq"] <= 4 else 1) + lse, "flops": fwd}
    # forward, then scores again (2d), dP (2d), dV (2d), dK (2d) and dQ (2d)
    return {"bytes": 4 * q + 2 * kv + lse, "flops": fwd + 2 * 10 * c["d"] * c["heads"] * _pairs(c) * part}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        turn = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda"),
                           s["pos"][:, None, :, None].double() * s["freqs"])
        turn = turn.conj() if c["inverse"] else turn
        res = []
        for x in (s["x"], s["x2"]):
            if x is None:
                continue
            r = x[..., :c["rot"]].double()
            pair = r.unflatten(-1, (-1, 2)) if c["interleaved"] else r.unflatten(-1, (2, -1)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            y = y.flatten(-2) if c["interleaved"] else y.transpose(-1, -2).flatten(-2)
            res.append(torch.cat([y, x[..., c["rot"]:].double()], -1))
        return res
    if c["op"] == "adamw":
        return _adamw_exact(s, c)
    return _diff_exact(s, c)


def _adamw_exact(s, c):
    """One step in 64 bits.  The 8-bit codes depend on the last bit of what is rounded and are left to the plain form."""
    t = c["step"] + 1
    out = {k: s[k].double() for k in ("p_flat", "m_flat", "v_flat")}
    if c["masters"]:
        out["w_flat"] = s["w_flat"].double()
    for i in range(len(s["p"])):
        at, n = s["p"][i].storage_offset(), s["p"][i].numel()
        m, v, g = s["m"][i].double(), s["v"][i].double(), s["g"][i].double()
        if c["bits"] == 8:
            m, v = m * _spread(s["ms"][i].double(), n), (v * _spread(s["vs"][i].double(), n)) ** 2
        m.lerp_(g, 1 - B1)
        v.lerp_(g ** 2, 1 - B2)
        step = (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
        p = (s["w"] or s["p"])[i].double()
        for name, x in (("p_flat", p - LR * (DECAY * p + step)), ("m_flat", m), ("v_flat", v)):
            out[name][at:at + n] = x
        if c["masters"]:
            out["w_flat"][at:at + n] = out["p_flat"][at:at + n]
    if c["bits"] == 8:
        out["m_flat"] = out["v_flat"] = out["ms_flat"] = out["vs_flat"] = None
    out["t"] = None
    return out


def _diff_exact(s, c):
    train = c["op"] == "diff_train"
    H, K = c["heads"], c["kv_heads"]
    lam = s["lam"].double().requires_grad_(train)
    acc, dlam = {}, 0
    with torch.enable_grad() if train else torch.no_grad():
        for b in range(c["batch"]):
            q, k, v = (s[x][b].double().requires_grad_(train) for x in ("q", "k", "v"))
            nq = int(s["q_lens"][b]) if s["q_lens"] is not None else c["nq"]
            nk = int(s["kv_lens"][b]) if s["kv_lens"] is not None else c["nk"]
            kk = k.unflatten(0, (K, 2)).repeat_interleave(H // K, 0)
            logits = torch.einsum("hmid,hmjd->hmij", q.unflatten(0, (H, 2)), kk) * s["scale"]
            hide = torch.ones(c["nq"], c["nk"], dtype=torch.bool, device="cuda")
            hide[:nq, :nk] = False
            if c["causal"]:
                hide |= torch.ones_like(hide).triu(1 + nk - nq)
            empty = hide.all(1)
            logits = logits.masked_fill(hide & ~empty[:, None], -math.inf)
            p = torch.softmax(logits, -1).masked_fill(empty[:, None], 0.0)
            maps = torch.einsum("hmij,hjd->mhid", p, v.repeat_interleave(H // K, 0))
            e = torch.exp((lam[:, 0::2] * lam[:, 1::2]).sum(-1))
            o = maps[0] - (e[:, 0] - e[:, 1] + LAM_INIT)[:, None, None] * maps[1]
            lse = torch.logsumexp(logits, -1).masked_fill(empty, -math.inf).flatten(0, 1)
            got = {"o": o.detach(), "lse": lse.detach()}
            if train:
                dq, dk, dv, dl = torch.autograd.grad(o, (q, k, v, lam), s["do"][b].double())
                got |= {"dq": dq, "dk": dk, "dv": dv}
                dlam = dlam + dl
            for name, x in got.items():
                acc.setdefault(name, []).append(x)
            del logits, p, maps, o, lse
    out = {name: torch.stack(x) for name, x in acc.items()}
    if train:
        out["dlam"] = dlam
    return out
