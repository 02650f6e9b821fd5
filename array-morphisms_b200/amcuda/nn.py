"""The operators of a differential-attention layer and of its training step,
on torch CUDA tensors: rotary positions, differential attention (forward,
gradient, and the single-token form) and the AdamW step.

Tensors are (batch, heads, rows, dim) with unit stride along dim and any
strides over the other axes, so a projection's (batch, rows, heads, dim)
output is passed as its transpose(1, 2).  Types are float32, bfloat16 and
float16; arithmetic is f32 or wider, but for the weights (and the gradients'
operands made of them) that the attention of 16-bit tensors with d up to 64 and
dv up to 128 rounds once to their type for the tensor cores; its single-token
form rounds none.  Results go into tensors the caller gives; nothing is
allocated, and torch's autograd does not see the calls.  Calls run on `stream` (the current stream of the
tensors' device when None) and may be captured into CUDA graphs.

    freqs, mscale = rope_freqs(64, factor=8.0, kind="parts", original_len=4096)
    rope(q, pos, freqs.cuda(), q_rot, k, k_rot, mscale=mscale)
    diff_attention_fwd(q_rot, k_rot, v, lam, o, lse, lam_init, scale, causal=True, o2=o2)
    diff_attention_bwd(q_rot, k_rot, v, lam, o, o2, lse, do, dq, dk, dv, dlam, lam_init, scale, causal=True,
                       workspace=ws)
    rope(dq, pos, freqs, dq, dk, dk, mscale=mscale, inverse=True)
    opt.step()                       # opt = AdamW(params, grads, m, v, state, lr=1e-3)
"""
from __future__ import annotations

import ctypes as C
import struct

from . import _abi as A

ROPE_KINDS = {"plain": 0, "linear": 1, "base": 2, "parts": 3}


def _dtypes():
    import torch
    return {torch.float32: A.F32, torch.bfloat16: A.BF16, torch.float16: A.F16}


_DTYPES = None


def _dtype(t, who: str) -> int:
    global _DTYPES
    if _DTYPES is None:
        _DTYPES = _dtypes()
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{who}: float32, bfloat16 or float16 expected, not {t.dtype}")
    return code


def _run(name: str, device, stream, *args) -> None:
    """The entry point on `stream` (the device's current one when None), with
    the tensors' device current for the call."""
    import torch
    if device.type != "cuda":
        raise ValueError("expected CUDA tensors")
    # the handle alone: making torch's stream object costs 2 us of a call's 10
    handle = torch._C._cuda_getCurrentRawStream(device.index) if stream is None else stream.cuda_stream
    # handle 0, torch's default stream, is the legacy stream (1 in the C ABI's
    # terms: NULL would mean the library's own stream)
    if device.index == torch.cuda.current_device():
        A.call(name, *args, handle or 1)
    else:
        with torch.cuda.device(device):
            A.call(name, *args, handle or 1)


# What a call checks depends on its tensors' layouts alone, so a layout that
# passed is remembered with what was derived from it; addresses and contents
# are read at every call.
_LAYOUTS: dict = {}


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _remember(key, value):
    if len(_LAYOUTS) >= 4096:
        _LAYOUTS.clear()
    _LAYOUTS[key] = value
    return value


def _same(who: str, first, *tensors) -> None:
    for t in tensors:
        if t is not None and (t.device != first.device or t.dtype != first.dtype):
            raise ValueError(f"{who}: tensors differ in device or type")


def _rows(t, who: str, shape=None):
    """Checks a (batch, heads, rows, dim) tensor; its strides over the first three axes."""
    if t.dim() != 4 or (t.stride(3) != 1 and t.shape[3] > 1):
        raise ValueError(f"{who}: expected (batch, heads, rows, dim) with unit stride along dim")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{who}: expected shape {tuple(shape)}, not {tuple(t.shape)}")
    return t.stride()[:3]


def _written(t, strides, who: str) -> None:
    """An output must not map two elements to one place."""
    for n, s in zip(t.shape, strides):
        if n > 1 and s == 0 and t.numel():
            raise ValueError(f"{who}: an output cannot be broadcast (stride 0)")


# ---------------------------------------------------------------------------- rotary positions
def rope_freqs(rot: int, base: float = 10000.0, kind: str = "plain", factor: float = 1.0, original_len: int = 0,
               slow: float = 1.0, fast: float = 32.0):
    """(freqs, mscale) of rope for rotated dim `rot`: radians per position of
    each of the rot/2 pairs (a float64 CPU tensor) and the factor on the
    rotated values.  `kind` stretches them to contexts `factor` times the
    original: "linear" (positions divided by factor), "base" (the base
    raised), "parts" (pairs that turn often over original_len kept, slow ones
    divided, a ramp between)."""
    import torch
    if kind not in ROPE_KINDS:
        raise ValueError(f"rope_freqs: kind is one of {sorted(ROPE_KINDS)}")
    out = torch.empty(max(rot // 2, 0), dtype=torch.float64)
    ms = C.c_float()
    A.call("amc_rope_freqs", C.cast(C.c_void_p(out.data_ptr()), C.POINTER(C.c_double)), rot, base, ROPE_KINDS[kind],
           factor, original_len, slow, fast, C.byref(ms))
    return out, ms.value


def rope(x, pos, freqs, out, x2=None, out2=None, mscale: float = 1.0, interleaved: bool = False,
         inverse: bool = False, stream=None) -> None:
    """out = x (batch, heads, n, d) with its first 2 * len(freqs) dims turned
    by the rows' positions, the rest copied; a second tensor (the keys) of the
    same batch, n and d goes along in the same launch.  `pos` is int64 (n,) or
    (batch, n).  Pairs are the halves of the rotated dims, or neighbours when
    `interleaved`.  `inverse` turns back: the gradient.  out may be x."""
    key = ("rope", _layout(x), _layout(out), _layout(x2), _layout(out2), _layout(pos), _layout(freqs))
    known = _LAYOUTS.get(key)
    if known is None:
        known = _remember(key, _rope_layout(x, pos, freqs, out, x2, out2))
    first, second, sizes, pos_stride = known
    tensors = _ROPE.pack(x.data_ptr(), out.data_ptr(), *first)
    if second is not None:
        tensors += _ROPE.pack(x2.data_ptr(), out2.data_ptr(), *second)
    _run("amc_rope", x.device, stream, tensors, *sizes, pos.data_ptr(), pos_stride, freqs.data_ptr(), mscale,
         int(interleaved), int(inverse))


_ROPE = struct.Struct("=2Q7q")
assert _ROPE.size == C.sizeof(A.RopeTensor)


def _rope_layout(x, pos, freqs, out, x2, out2):
    """Checks rope's tensors; (heads and strides of each tensor, the entry point's sizes, the stride of pos)."""
    import torch
    B, _, n, d = x.shape if x.dim() == 4 else (0, 0, 0, 0)
    pairs = [(x, out)] if x2 is None else [(x, out), (x2, out2)]
    if x2 is not None and out2 is None:
        raise ValueError("rope: x2 needs out2")
    rows = []
    for a, o in pairs:
        xs, os = _rows(a, "rope", (B, a.shape[1], n, d) if a.dim() == 4 else None), _rows(o, "rope", a.shape)
        _same("rope", x, a, o)
        _written(o, os, "rope")
        rows.append((a.shape[1], *xs, *os))
    if pos.dtype != torch.int64 or tuple(pos.shape) not in ((n,), (B, n)) or (n > 1 and pos.stride(-1) != 1):
        raise ValueError("rope: positions are int64 (n,) or (batch, n) with unit stride along n")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise ValueError("rope: freqs is a contiguous float64 vector")
    if pos.device != x.device or freqs.device != x.device:
        raise ValueError("rope: positions and freqs live on the tensors' device")
    return (rows[0], rows[1] if x2 is not None else None,
            (len(pairs), _dtype(x, "rope"), B, n, d, 2 * freqs.shape[0]), pos.stride(0) if pos.dim() == 2 else 0)


# ---------------------------------------------------------------------------- differential attention
_DIFF = struct.Struct("=10i2f15Qq27q")
assert _DIFF.size == C.sizeof(A.DiffAttention)
_NONE3 = (0, 0, 0)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _diff_sizes(q, k, v, who: str):
    qs, ks, vs = _rows(q, who), _rows(k, who), _rows(v, who)
    B, H2, nq, d = q.shape
    K2, nk = k.shape[1], k.shape[2]
    dv = v.shape[3]
    if H2 % 2 or K2 % 2 or not K2 or not H2 or H2 % K2:
        raise ValueError(f"{who}: q and k hold two maps a head; query heads are a multiple of key heads")
    if tuple(k.shape) != (B, K2, nk, d) or tuple(v.shape) != (B, K2 // 2, nk, dv):
        raise ValueError(f"{who}: q (B, 2H, nq, d), k (B, 2K, nk, d) and v (B, K, nk, dv) expected")
    _same(who, q, k, v)
    return (B, H2 // 2, K2 // 2, nq, nk, d, dv), qs, ks, vs


def _check_lens(t, B: int, device, who: str) -> None:
    import torch
    if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,) or t.device != device or
                          (B > 1 and t.stride(0) != 1)):
        raise ValueError(f"{who}: lengths are int32 (batch,) on the tensors' device")


def _diff_layout(q, k, v, lam, o, lse, o2, q_lens, kv_lens, workspace, grads, who: str):
    """Checks the tensors of a call; (sizes, strides, workspace bytes) as the C
    struct holds them.  grads: None, or (do, dq, dk, dv, dlam)."""
    import torch
    (B, H, K, nq, nk, d, dv), qs, ks, vs = _diff_sizes(q, k, v, who)
    _same(who, q, lam)
    if lam.dim() != 3 or lam.shape[0] not in (1, H) or tuple(lam.shape[1:]) != (4, d) or not lam.is_contiguous():
        raise ValueError(f"{who}: lam is a contiguous (1 or H, 4, d) tensor")
    _check_lens(q_lens, B, q.device, who)
    _check_lens(kv_lens, B, q.device, who)
    shape = (B, H, nq, dv)
    os = _rows(o, who, shape)
    o2s = _NONE3 if o2 is None else _rows(o2, who, shape)
    _same(who, q, o, o2)
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (B, 2 * H, nq) or
                            not lse.is_contiguous() or lse.device != q.device):
        raise ValueError(f"{who}: lse is a contiguous float32 (B, 2H, nq) tensor")
    if workspace is not None and (workspace.device != q.device or not workspace.is_contiguous()):
        raise ValueError(f"{who}: the workspace is contiguous, on the tensors' device")
    if grads is None:
        written, more = ((o, os), (o2, o2s)), _NONE3 * 4
    else:
        do, dq, dk, dv_, dlam = grads
        if lse is None or o2 is None:
            raise ValueError(f"{who}: lse and o2 of the forward are needed")
        dos = _rows(do, who, shape)
        dqs, dks, dvs = _rows(dq, who, q.shape), _rows(dk, who, k.shape), _rows(dv_, who, v.shape)
        _same(who, q, do, dq, dk, dv_, dlam)
        if tuple(dlam.shape) != tuple(lam.shape) or not dlam.is_contiguous():
            raise ValueError(f"{who}: dlam is contiguous and shaped like lam")
        written, more = ((dq, dqs), (dk, dks), (dv_, dvs)), (*dos, *dqs, *dks, *dvs)
    for t, s in written:
        if t is not None:
            _written(t, s, who)
    return ((B, H, K, nq, nk, d, dv, lam.shape[0]), (*qs, *ks, *vs, *os, *o2s, *more),
            0 if workspace is None else workspace.numel() * workspace.element_size(), _dtype(q, who))


def _diff_call(who: str, q, k, v, lam, o, lse, o2, q_lens, kv_lens, workspace, grads, causal, scale, lam_init, stream):
    key = (who, _layout(q), _layout(k), _layout(v), _layout(lam), _layout(o), _layout(lse), _layout(o2),
           _layout(q_lens), _layout(kv_lens), _layout(workspace), None if grads is None else tuple(map(_layout, grads)))
    known = _LAYOUTS.get(key)
    if known is None:
        known = _remember(key, _diff_layout(q, k, v, lam, o, lse, o2, q_lens, kv_lens, workspace, grads, who))
    sizes, strides, ws_bytes, dtype = known
    args = _DIFF.pack(dtype, int(bool(causal)), *sizes, scale, lam_init, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                      lam.data_ptr(), _ptr(q_lens), _ptr(kv_lens), o.data_ptr(), _ptr(o2), _ptr(lse),
                      *((0, 0, 0, 0, 0) if grads is None else [t.data_ptr() for t in grads]), _ptr(workspace), ws_bytes,
                      *strides)
    _run("amc_" + who, q.device, stream, args)


def diff_attention_workspace(q, k, v, backward: bool = False) -> int:
    """Bytes of workspace that diff_attention_fwd (and, with `backward`,
    diff_attention_bwd) needs for tensors like these; it may be 0."""
    who = "diff_attention_workspace"
    (B, H, K, nq, nk, d, dv), *_ = _diff_sizes(q, k, v, who)
    p = A.DiffAttention(dtype=_dtype(q, who), batch=B, heads=H, kv_heads=K, nq=nq, nk=nk, d=d, dv=dv, lam_rows=1)
    n = C.c_int64()
    A.call("amc_diff_attention_workspace", C.byref(p), int(backward), C.byref(n))
    return n.value


def diff_attention_fwd(q, k, v, lam, o, lse, lam_init: float, scale: float, causal: bool = False, q_lens=None,
                       kv_lens=None, o2=None, workspace=None, stream=None) -> None:
    """o (B, H, nq, dv) = (softmax(scale Q1 K1^T) - lam softmax(scale Q2 K2^T)) V.

    q (B, 2H, nq, d): heads 2h and 2h + 1 are the two maps of head h; k
    (B, 2K, nk, d) likewise; v (B, K, nk, dv); H a multiple of K.  lam
    (1 or H, 4, d) holds the learned rows, lam = exp(l0 . l1) - exp(l2 . l3) +
    lam_init.  Row i of sequence b sees the keys below kv_lens[b], and with
    `causal` those up to i + kv_lens[b] - q_lens[b]; without lengths, nk and
    nq stand for them.  Rows behind q_lens and rows that see no key give 0.
    What the tensors hold behind the lengths is not used.  lse (B, 2H, nq)
    float32 (or None) receives the row log-sum-exps; o2 (like o) the second
    map's part, which the backward needs.  One query row (or few) a head runs
    the single-token form, split over the keys.  A cache that fills up is best
    given whole with its kv_lens: each new shape of a slice of it is checked anew
    on the host, which costs more than a short call's kernel."""
    _diff_call("diff_attention_fwd", q, k, v, lam, o, lse, o2, q_lens, kv_lens, workspace, None, causal, scale,
               lam_init, stream)


def diff_attention_bwd(q, k, v, lam, o, o2, lse, do, dq, dk, dv, dlam, lam_init: float, scale: float,
                       causal: bool = False, q_lens=None, kv_lens=None, workspace=None, stream=None) -> None:
    """Gradients of diff_attention_fwd for upstream `do` (like o), from its o,
    o2 and lse: dq, dk, dv and dlam, shaped like their tensors, gradients of
    shared heads summed, zero behind the lengths.  No sums by atomics: repeated calls
    give identical bits."""
    _diff_call("diff_attention_bwd", q, k, v, lam, o, lse, o2, q_lens, kv_lens, workspace, (do, dq, dk, dv, dlam),
               causal, scale, lam_init, stream)


# ---------------------------------------------------------------------------- AdamW
STATE_BLOCK = 256     # elements that share one scale of an 8-bit state


class AdamW:
    """The AdamW step over a list of tensors, in one launch for every 256:
        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    The tensors are the caller's, contiguous, on one device, and are updated
    in place by every step(); gradients are read from the given buffers.
    params and grads are float32, bfloat16 or float16.  With `masters`
    (float32) the update is made on those and params receive them rounded.  m
    and v are float32, or torch.float8_e4m3fn codes of m and sqrt(v) with a
    float32 scale for every STATE_BLOCK elements in m_scales and v_scales
    (zeros are a fresh state).  A NaN gradient makes its own element's
    parameter and states NaN; an infinite one, with 8-bit states, its whole
    block's at the next step.  `state` is an int64 pair on the device, (steps
    done, 0); each step counts it, so a step captured into a CUDA graph goes
    on counting at its replays.  lr is a number, or a float32 tensor of one
    element on the device that is read at every step.  Two steps of the same
    tensors must not overlap.  Tensors that are given other memory later
    (`p.data = ...`) need an AdamW of their own: this one keeps the memory it
    was made with."""

    def __init__(self, params, grads, m, v, state, lr=1e-3, beta1: float = 0.9, beta2: float = 0.999,
                 eps: float = 1e-8, weight_decay: float = 0.01, masters=None, m_scales=None, v_scales=None):
        import torch
        params, grads, m, v = list(params), list(grads), list(m), list(v)
        n = len(params)
        lists = {"grads": grads, "m": m, "v": v}
        for name, x in (("masters", masters), ("m_scales", m_scales), ("v_scales", v_scales)):
            if x is not None:
                lists[name] = list(x)
        if any(len(x) != n for x in lists.values()):
            raise ValueError("AdamW: one tensor of each kind for every parameter")
        self.device = state.device
        if state.dtype != torch.int64 or tuple(state.shape) != (2,) or not state.is_contiguous():
            raise ValueError("AdamW: state is an int64 pair, (steps done, 0)")
        bits8 = bool(m) and m[0].dtype == torch.float8_e4m3fn
        state_type = torch.float8_e4m3fn if bits8 else torch.float32
        if bits8 and ("m_scales" not in lists or "v_scales" not in lists):
            raise ValueError("AdamW: 8-bit states need m_scales and v_scales")
        if not bits8 and (m_scales is not None or v_scales is not None):
            raise ValueError("AdamW: scales belong to 8-bit states")
        kinds = {"m": state_type, "v": state_type, "masters": torch.float32, "m_scales": torch.float32,
                 "v_scales": torch.float32, "grads": grads[0].dtype if n else None}
        table = (A.AdamwTensor * max(n, 1))()
        written = []
        for i, p in enumerate(params):
            if p.dtype != params[0].dtype or p.device != self.device or not p.is_contiguous():
                raise ValueError("AdamW: parameters share a type and device and are contiguous")
            for name, x in lists.items():
                t = x[i]
                blocks = name.endswith("_scales")
                want = -(-p.numel() // STATE_BLOCK) if blocks else p.numel()
                if t.dtype != kinds[name] or t.device != self.device or not t.is_contiguous() or t.numel() != want:
                    raise ValueError(f"AdamW: {name}[{i}] does not match its parameter in type, device, layout or size")
            e = table[i]
            e.p, e.n, e.g, e.m, e.v = p.data_ptr(), p.numel(), grads[i].data_ptr(), m[i].data_ptr(), v[i].data_ptr()
            for name, x in (("params", params), *lists.items()):
                # a master may be its parameter (both f32); nothing else is written twice
                at = x[i].data_ptr()
                if name == "grads" or not x[i].numel() or (name == "masters" and at == p.data_ptr()):
                    continue
                written.append((at, at + x[i].numel() * x[i].element_size(), name, i))
            if masters is not None:
                e.master = lists["masters"][i].data_ptr()
            if bits8:
                e.m_scale, e.v_scale = lists["m_scales"][i].data_ptr(), lists["v_scales"][i].data_ptr()
        written.sort()
        for (_, end, *_), (at, _, name, i) in zip(written, written[1:]):
            if at < end:
                raise ValueError(f"AdamW: memory of {name}[{i}] is another tensor of the step as well")
        self.lr, self.betas, self.eps, self.weight_decay = lr, (beta1, beta2), eps, weight_decay
        self.state, self._table, self._n = state, table, n
        self._kinds = (_dtype(params[0], "AdamW"), _dtype(grads[0], "AdamW")) if n else (A.F32, A.F32)
        self._kinds += (A.E4M3 if bits8 else A.F32,)
        # the table's addresses stay valid, even if a tensor is given other memory
        self._keep = [t.untyped_storage() for x in (params, *lists.values()) for t in x]

    @property
    def lr(self):
        """The rate of the next step, as it was given: a number or a tensor on the device."""
        return self._lr if self._lr_dev is None else self._lr_dev

    @lr.setter
    def lr(self, lr) -> None:
        import torch
        if not isinstance(lr, torch.Tensor):
            self._lr, self._lr_dev = float(lr), None
        elif lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != self.device:
            raise ValueError("AdamW: lr is a number or a float32 tensor of one element on the device")
        else:
            self._lr, self._lr_dev = 0.0, lr

    def step(self, stream=None) -> None:
        """One update of every tensor; `lr`, a number or a tensor, may be assigned
        between steps (a captured step keeps the one it was captured with)."""
        _run("amc_adamw", self.device, stream, self._table, self._n, *self._kinds, self.state.data_ptr(),
             _ptr(self._lr_dev), self._lr, *self.betas, self.eps, self.weight_decay)
