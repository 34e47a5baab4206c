"""Attention operators with relative positions on the HIP engine (include/fact_hip.h FactAttention, FactQkNorm).

    qk_norm_rope / qk_norm_rope_backward   RMS norm of each query and key head with a learned gain, then rotation by position
    attention / attention_backward         sliding window, sinks, learned relative position bias by buckets
    relative_buckets                       the logarithmic bucket map of the clipped distances

Tensors are [batch, token, head, dh] CUDA tensors of any strides whose last dimension is contiguous (views of one packed
projection are read in place; what the kernels cannot address is copied first).  Calls run on the current stream of the
tensors' device, never synchronise, and take their scratch memory from torch's allocator per call, so they can be captured into
graphs and run on several streams at once.  There is no autograd: as in the engine, the backward is a call of its own, and a
tensor that requires grad is refused while grad mode is on (its gradient would be lost without a word): detach it, or call under
torch.no_grad().
Models use the same kernels through the transformer options of their config (mint_amd/protos.py).
"""
import collections
import ctypes as C

import torch

from mint_amd import _lib as L

AttentionSaved = collections.namedtuple("AttentionSaved", ["lse", "out_lo"])
AttentionSaved.__doc__ = """What attention(training=True) leaves for the backward: the base-2 log-sum-exp of every row, fp32
[batch, heads, queries], and - with a relative bias, up to EXACT_KEYS keys, or where a window and its sinks leave up to EXACT_WINDOW
to a row - the fp32 rounding residual of the output, [batch, queries, heads, dh]: the backward's row sums dO . O need it where they
are added up (the fp32 gradient of the table) or rows average the rounding of few probabilities."""

# The residual is worth its price where rows average the rounding of few probabilities: without it dq and dk of 2 keys a row are
# 3.8e-3 off (norm), of 9 keys 2.65e-3, of 57 causal ones 2.7e-3, of 65 2.5e-3; with it all are 2.35e-3, what the rounding of dS and of
# the result costs.  At 512 keys nothing is left of the gain (2.38e-3 and 2.36e-3).  It costs two products more in the forward: B 16,
# H 10, dh 80, 512 keys 42 instead of 27 us, n 1440, H 12, dh 128, window +-8 27 + 60 us instead of 20 + 56.
EXACT_KEYS = 512   # short sequences
EXACT_WINDOW = 64  # and rows that see this many keys of a long one

DTYPES = {torch.bfloat16: 0, torch.float32: 1}


def _need(cond, msg, *args):
    if not cond:
        raise ValueError(msg % args)


def _int32(x, name):
    """ctypes would drop the upper bits."""
    x = int(x)
    _need(-1 << 31 <= x < 1 << 31, "%s must fit 32 bits, not %d", name, x)
    return x


def _detached(t, name):
    _need(not (t.requires_grad and torch.is_grad_enabled()),
          "%s requires grad, and these calls record no graph: detach it or call under torch.no_grad(), and take the gradients from "
          "the backward call", name)


def relative_buckets(num_buckets, max_distance, bidirectional=True, device=None):
    """int32 [2 * max_distance + 1]: bucket of each distance key - query clipped to +-max_distance.  Half of a side's buckets
    hold one distance each, the rest grow by equal ratios up to max_distance; with `bidirectional` keys after the query have the
    upper half of the buckets, without it they share bucket 0."""
    num_buckets, max_distance = _int32(num_buckets, "num_buckets"), _int32(max_distance, "max_distance")
    got = (C.c_int32 * (2 * min(max(0, max_distance), 1024) + 1))()  # (a wider map is refused)
    L.check(L.lib().fact_relative_buckets(num_buckets, max_distance, 1 if bidirectional else 0, got))
    return torch.tensor(list(got), dtype=torch.int32, device=device)


def _heads(t, name, dtype, device=None):
    """A [batch, token, head, dh] tensor that the kernels can read in place, or a contiguous copy of it."""
    _need(torch.is_tensor(t) and t.dim() == 4, "%s must be a [batch, token, head, dh] tensor", name)
    _detached(t, name)
    _need(t.is_cuda, "%s must be a CUDA tensor: there is no CPU path", name)
    _need(device is None or t.device == device, "%s is on %s, expected %s", name, t.device, device)
    if dtype is not None:
        _need(t.dtype == dtype, "%s must be %s, not %s", name, dtype, t.dtype)
    return t if _addressable(t) else t.clone(memory_format=torch.contiguous_format)


def _addressable(t):
    s = t.stride()
    return s[3] == 1 and not (s[0] | s[1] | s[2]) & 7 and s[1] <= 1 << 25 and not t.data_ptr() & 15


def _dest(t, name, shape, dtype, device):
    """A caller's output tensor (written in place: it has to be addressable), or a new one."""
    if t is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _need(torch.is_tensor(t) and t.shape == torch.Size(shape) and t.dtype == dtype and t.device == device,
          "%s must be a %s tensor of shape %s on %s", name, dtype, tuple(shape), device)
    _detached(t, name)
    _need(_addressable(t), "%s must have a contiguous last dimension, 16-byte alignment and strides that are multiples of 8", name)
    _need(all(t.stride(i) for i in range(3) if t.shape[i] > 1), "%s must not be a broadcast tensor", name)
    return t


def _vector(t, name, shape, dtype, device):
    if t is None:
        return None
    _need(torch.is_tensor(t) and t.dtype == dtype and t.device == device and t.shape == torch.Size(shape),
          "%s must be a %s tensor of shape %s on %s", name, dtype, tuple(shape), device)
    _detached(t, name)
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)


def _p(t):
    return None if t is None else t.data_ptr()


def _set(a, name, t):
    setattr(a, name, t.data_ptr())
    getattr(a, name + "_stride")[:] = t.stride()[:3]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(fn, a, ws_bytes, device):
    """fn(args, workspace, bytes, stream) on the device's current stream, with scratch memory of this call's own."""
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    index, before = device.index, torch.cuda.current_device()
    if before != index:
        torch.cuda.set_device(index)
    try:
        rc = fn(C.byref(a), ws.data_ptr() if ws_bytes else None, ws_bytes, _raw_stream(index))
    finally:
        if before != index:
            torch.cuda.set_device(before)
    if rc:
        L.check(rc)


def _ws_bytes(name, a, backward):
    n = C.c_size_t(0)
    L.check(getattr(L.lib(), name)(C.byref(a), backward, C.byref(n)))
    return n.value


# Calls of one geometry (shapes, strides, types, devices, options) share their checks: the first one leaves its filled-in argument
# struct and workspace size, the next ones copy it and set the pointers.  Nothing of the tensors themselves is kept.  (A call
# costs the host 9-11 instead of 18 us; one new token of 32 sequences takes the GPU 4.)
_PLANS = {}
_MOST_PLANS = 512
_Plan = collections.namedtuple("_Plan", ["args", "fn", "ws", "extra"])


def _keep(key, args, fn, ws, extra=None):
    if key is not None:
        if len(_PLANS) >= _MOST_PLANS:
            _PLANS.clear()
        _PLANS[key] = _Plan(bytes(args), fn, ws, extra)


def _key(op, tensors, options):
    """None where an argument is no tensor or has to be refused: the checks say so."""
    try:
        if torch.is_grad_enabled():
            for t in tensors:
                if t is not None and t.requires_grad:
                    return None
        return (op,) + tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors]) + options
    except AttributeError:
        return None


# ---- attention ------------------------------------------------------------------------------------------------------
def _attention_args(q, k, v, scale, window, sinks, rel_table, rel_map, kv_len, q_start):
    q = _heads(q, "q", torch.bfloat16)
    dev = q.device
    k, v = _heads(k, "k", torch.bfloat16, dev), _heads(v, "v", torch.bfloat16, dev)
    B, nq, H, dh = q.shape
    _need(k.shape == v.shape and k.shape[0] == B and k.shape[3] == dh, "k and v must be [%d, tokens, heads, %d], got %s and %s",
          B, dh, tuple(k.shape), tuple(v.shape))
    nk, Hkv = k.shape[1], k.shape[2]
    _need(Hkv > 0 and H % Hkv == 0, "the %d query heads must be a multiple of the %d key heads", H, Hkv)
    _need(len(window) == 2, "window must be (left, right)")
    a = L.FactAttention(B=B, H=H, Hkv=Hkv, nq=nq, nk=nk, dh=dh, window_left=_int32(window[0], "window"),
                        window_right=_int32(window[1], "window"), sinks=_int32(sinks, "sinks"),
                        scale=float(dh ** -0.5 if scale is None else scale))
    _need((rel_table is None) == (rel_map is None), "rel_table and rel_map belong together")
    if rel_table is not None:
        _need(torch.is_tensor(rel_table) and rel_table.dim() == 2 and rel_table.shape[1] == H,
              "rel_table must be [buckets, %d]", H)
        _need(torch.is_tensor(rel_map) and rel_map.dim() == 1 and rel_map.numel() >= 3 and rel_map.numel() % 2 == 1,
              "rel_map must hold the bucket of 2 * max_distance + 1 distances")
        rel_table = _vector(rel_table, "rel_table", rel_table.shape, torch.float32, dev)
        rel_map = _vector(rel_map, "rel_map", rel_map.shape, torch.int32, dev)
        a.rel_buckets, a.rel_max_distance = rel_table.shape[0], rel_map.numel() // 2
    kv_len = _vector(kv_len, "kv_len", (B,), torch.int32, dev)
    q_start = _vector(q_start, "q_start", (B,), torch.int32, dev)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _set(a, name, t)
    held = (q, k, v, rel_table, rel_map, kv_len, q_start)
    _inputs(a, held)
    return a, held  # (the copies live until the launch is enqueued)


def _inputs(a, held):
    """Pointers of the forward's inputs; their alignment bits."""
    q, k, v, rel_table, rel_map, kv_len, q_start = held
    a.q, a.k, a.v = x, y, z = q.data_ptr(), k.data_ptr(), v.data_ptr()
    bits = x | y | z
    if rel_table is not None:
        a.rel_table, a.rel_map = x, y = rel_table.data_ptr(), rel_map.data_ptr()
        bits |= x | y
    if kv_len is not None:
        a.kv_len = x = kv_len.data_ptr()
        bits |= x
    if q_start is not None:
        a.q_start = x = q_start.data_ptr()
        bits |= x
    return bits


def _options(scale, window, sinks):
    return (None if scale is None else float(scale), (-1, -1) if window is None else tuple([int(w) for w in window]), int(sinks))


def attention(q, k, v, scale=None, window=None, sinks=0, rel_table=None, rel_map=None, kv_len=None, q_start=None,
              training=False, out=None):
    """Attention of q [B, nq, H, dh] over k, v [B, nk, Hkv, dh], bf16; head h reads key head h // (H // Hkv).

    Query row i of sequence b stands at position q_start[b] + i (0 + i without q_start) and sees the keys j with j < kv_len[b],
    j <= position + window[1] and (j >= position - window[0] or j < sinks); a negative window side is open.  rel_table
    [buckets, H] fp32 adds rel_table[rel_map[clip(j - position)]][h] to scale * q . k; -inf hides a key, finite values count up to
    +-2^14.  A row that sees no key gives zeros.
    What stands at keys and values that no row of their sequence sees (from kv_len on, behind the window, in a cache's free places)
    reaches no result.  `out` may be q, and must not overlap k or v.  Returns out [B, nq, H, dh], with `training`
    (out, AttentionSaved)."""
    options = _options(scale, window, sinks)
    held = (q, k, v, rel_table, rel_map, kv_len, q_start)
    key = _key("attention", held + (out,), options + (bool(training),))
    plan = _PLANS.get(key)
    if plan is not None:
        a = L.FactAttention.from_buffer_copy(plan.args)
        if out is None:
            out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
        a.out = x = out.data_ptr()
        if not (_inputs(a, held) | x) & 15:
            dev, saved = q.device, None
            if training:
                lse = torch.empty(plan.extra[0], dtype=torch.float32, device=dev)
                lo = torch.empty(q.shape, dtype=torch.float32, device=dev) if plan.extra[1] else None
                a.lse, a.out_lo, saved = lse.data_ptr(), _p(lo), AttentionSaved(lse, lo)
            _launch(plan.fn, a, plan.ws, dev)
            return (out, saved) if training else out
    a, given = _attention_args(*held[:3], *options, *held[3:])
    dev = given[0].device
    shape = (a.B, a.nq, a.H, a.dh)
    out = _dest(out, "out", shape, torch.bfloat16, dev)
    if 0 in shape:
        return (out, AttentionSaved(out.new_empty((a.B, a.H, a.nq), dtype=torch.float32), None)) if training else out
    if a.nk == 0:
        out.zero_()
        lse = torch.full((a.B, a.H, a.nq), float("inf"), device=dev) if training else None
        return (out, AttentionSaved(lse, None)) if training else out
    _set(a, "out", out)
    saved = None
    if training:
        lse = torch.empty((a.B, a.H, a.nq), dtype=torch.float32, device=dev)
        narrow = min(a.window_left, a.window_right) >= 0 and a.window_left + 1 + a.window_right + a.sinks <= EXACT_WINDOW
        exact = rel_table is not None or a.nk <= EXACT_KEYS or narrow
        lo = torch.empty(shape, dtype=torch.float32, device=dev) if exact else None
        saved = AttentionSaved(lse, lo)
        a.lse, a.out_lo = lse.data_ptr(), _p(lo)
    ws, fn = _ws_bytes("fact_attention_workspace", a, 0), L.lib().fact_attention
    _launch(fn, a, ws, dev)
    if all(x is y for x, y in zip(held, given)):
        _keep(key, a, fn, ws, (saved.lse.shape, saved.out_lo is not None) if training else None)
    return (out, saved) if training else out


def attention_backward(dout, q, k, v, out, saved, scale=None, window=None, sinks=0, rel_table=None, rel_map=None, kv_len=None,
                       q_start=None, dq=None, dk=None, dv=None):
    """Gradients of attention(..., training=True) for dout [B, nq, H, dh]: (dq, dk, dv), with a relative bias also the fp32
    gradient of rel_table.  `out` and `saved` are what the forward returned; dq, dk, dv may be given (views of one packed
    gradient, for instance; they must not overlap the inputs)."""
    _need(isinstance(saved, AttentionSaved), "saved must be what attention(training=True) returned")
    options = _options(scale, window, sinks)
    held = (q, k, v, rel_table, rel_map, kv_len, q_start)
    lse, lo = saved
    key = _key("backward", held + (dout, out, lse, lo, dq, dk, dv), options)
    plan = _PLANS.get(key)
    if plan is not None:
        dev = q.device
        a = L.FactAttention.from_buffer_copy(plan.args)
        dq = torch.empty(q.shape, dtype=torch.bfloat16, device=dev) if dq is None else dq
        dk = torch.empty(k.shape, dtype=torch.bfloat16, device=dev) if dk is None else dk
        dv = torch.empty(k.shape, dtype=torch.bfloat16, device=dev) if dv is None else dv
        bits = _inputs(a, held)
        for name, t in (("dout", dout), ("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
            x = t.data_ptr()
            setattr(a, name, x)
            bits |= x
        if lo is not None:
            a.out_lo = x = lo.data_ptr()
            bits |= x
        if not bits & 15:
            if rel_table is None:
                _launch(plan.fn, a, plan.ws, dev)
                return dq, dk, dv
            drel = torch.empty(rel_table.shape, dtype=torch.float32, device=dev)
            a.drel = drel.data_ptr()
            _launch(plan.fn, a, plan.ws, dev)
            return dq, dk, dv, drel
    a, given = _attention_args(*held[:3], *options, *held[3:])
    dev = given[0].device
    shape = torch.Size((a.B, a.nq, a.H, a.dh))
    more = (dout, out, lse, lo)
    dout, out = _heads(dout, "dout", torch.bfloat16, dev), _heads(out, "out", torch.bfloat16, dev)
    _need(dout.shape == shape and out.shape == shape, "dout and out must be %s", tuple(shape))
    dq = _dest(dq, "dq", q.shape, torch.bfloat16, dev)
    dk = _dest(dk, "dk", k.shape, torch.bfloat16, dev)
    dv = _dest(dv, "dv", v.shape, torch.bfloat16, dev)
    drel = None
    if rel_table is not None:
        drel = torch.empty((a.rel_buckets, a.H), dtype=torch.float32, device=dev)
    if 0 in shape or a.nk == 0:
        for t in (dq, dk, dv, drel):
            if t is not None:
                t.zero_()
        return (dq, dk, dv) if drel is None else (dq, dk, dv, drel)
    lse = _vector(lse, "saved.lse", (a.B, a.H, a.nq), torch.float32, dev)
    lo = _vector(lo, "saved.out_lo", shape, torch.float32, dev)
    for name, t in (("out", out), ("dout", dout), ("dq", dq), ("dk", dk), ("dv", dv)):
        _set(a, name, t)
    a.lse, a.out_lo, a.drel = lse.data_ptr(), _p(lo), _p(drel)
    ws, fn = _ws_bytes("fact_attention_workspace", a, 1), L.lib().fact_attention_backward
    _launch(fn, a, ws, dev)
    if all(x is y for x, y in zip(held + more, given + (dout, out, lse, lo))):
        _keep(key, a, fn, ws)
    return (dq, dk, dv) if drel is None else (dq, dk, dv, drel)


# ---- norm of queries and keys with rotation ---------------------------------------------------------------------------
def _norm_args(q, k, q_gamma, k_gamma, positions, eps, rotary_dim, base, interleaved, position0):
    q = _heads(q, "q", None)
    _need(q.dtype in DTYPES, "q must be bfloat16 or float32, not %s", q.dtype)
    dev = q.device
    k = _heads(k, "k", q.dtype, dev)
    B, n, H, dh = q.shape
    _need(k.shape[0] == B and k.shape[1] == n and k.shape[3] == dh, "k must be [%d, %d, heads, %d], got %s", B, n, dh,
          tuple(k.shape))
    q_gamma = _vector(q_gamma, "q_gamma", (dh,), torch.float32, dev)
    k_gamma = _vector(k_gamma, "k_gamma", (dh,), torch.float32, dev)
    a = L.FactQkNorm(B=B, n=n, H=H, Hkv=k.shape[2], dh=dh, interleaved=1 if interleaved else 0, dtype=DTYPES[q.dtype],
                     rotary_dim=dh if rotary_dim is None else _int32(rotary_dim, "rotary_dim"),
                     position0=_int32(position0, "position0"), eps=eps, base=base)
    if positions is not None:
        _need(torch.is_tensor(positions) and positions.dtype == torch.int32 and positions.device == dev
              and tuple(positions.shape) in ((B, n), (n,)), "positions must be an int32 tensor of shape %s or %s on %s",
              (B, n), (n,), dev)
        a.position_stride[:] = positions.expand(B, n).stride()
    for name, t in (("q", q), ("k", k)):
        _set(a, name, t)
    held = (q, k, q_gamma, k_gamma, positions)
    _norm_inputs(a, held)
    return a, held


def _norm_inputs(a, held):
    q, k, q_gamma, k_gamma, positions = held
    a.q, a.k = x, y = q.data_ptr(), k.data_ptr()
    bits = x | y
    if q_gamma is not None:
        a.q_gamma = x = q_gamma.data_ptr()
        bits |= x
    if k_gamma is not None:
        a.k_gamma = x = k_gamma.data_ptr()
        bits |= x
    if positions is not None:
        a.positions = positions.data_ptr()
    return bits


def _norm_options(eps, rotary_dim, base, interleaved, position0):
    return float(eps), None if rotary_dim is None else int(rotary_dim), float(base), bool(interleaved), int(position0)


def qk_norm_rope(q, k, q_gamma=None, k_gamma=None, eps=1e-6, rotary_dim=None, base=10000.0, interleaved=False, positions=None,
                 position0=0, q_out=None, k_out=None):
    """x * rsqrt(mean(x^2) + eps) * gamma of every head of q [B, n, H, dh] and k [B, n, Hkv, dh] (bf16 or fp32; gains fp32 [dh],
    None: 1), then the first rotary_dim values (None: all, 0: none) of each head turned in pairs by
    position * base^(-2 i / rotary_dim).  Pair i is (i, i + rotary_dim / 2), `interleaved` (2 i, 2 i + 1).  positions: int32
    [B, n] or [n]; without it position0 + token.  Returns (q, k); q_out / k_out may be q / k themselves."""
    options = _norm_options(eps, rotary_dim, base, interleaved, position0)
    held = (q, k, q_gamma, k_gamma, positions)
    key = _key("norm", held + (q_out, k_out), options)
    plan = _PLANS.get(key)
    if plan is not None:
        dev = q.device
        a = L.FactQkNorm.from_buffer_copy(plan.args)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=dev) if q_out is None else q_out
        k_out = torch.empty(k.shape, dtype=q.dtype, device=dev) if k_out is None else k_out
        a.q_out, a.k_out = x, y = q_out.data_ptr(), k_out.data_ptr()
        if not (_norm_inputs(a, held) | x | y) & 15:
            _launch(plan.fn, a, 0, dev)
            return q_out, k_out
    a, given = _norm_args(*held, *options)
    dev = given[0].device
    q_out = _dest(q_out, "q_out", q.shape, q.dtype, dev)
    k_out = _dest(k_out, "k_out", k.shape, q.dtype, dev)
    if a.B == 0 or a.n == 0:
        return q_out, k_out
    _set(a, "q_out", q_out)
    _set(a, "k_out", k_out)
    fn = L.lib().fact_qk_norm
    _launch(fn, a, 0, dev)
    if all(x is y for x, y in zip(held, given)):
        _keep(key, a, fn, 0)
    return q_out, k_out


def qk_norm_rope_backward(dq_out, dk_out, q, k, q_gamma=None, k_gamma=None, eps=1e-6, rotary_dim=None, base=10000.0,
                          interleaved=False, positions=None, position0=0, dq=None, dk=None):
    """Gradients of qk_norm_rope for (dq_out, dk_out), from the forward's INPUTS q, k: (dq, dk, dq_gamma, dk_gamma), the last two
    fp32 [dh].  dq / dk may be dq_out / dk_out themselves."""
    options = _norm_options(eps, rotary_dim, base, interleaved, position0)
    held = (q, k, q_gamma, k_gamma, positions)
    key = _key("norm backward", held + (dq_out, dk_out, dq, dk), options)
    plan = _PLANS.get(key)
    if plan is not None:
        dev = q.device
        a = L.FactQkNorm.from_buffer_copy(plan.args)
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev) if dq is None else dq
        dk = torch.empty(k.shape, dtype=q.dtype, device=dev) if dk is None else dk
        bits = _norm_inputs(a, held)
        for name, t in (("dq_out", dq_out), ("dk_out", dk_out), ("dq", dq), ("dk", dk)):
            x = t.data_ptr()
            setattr(a, name, x)
            bits |= x
        if not bits & 15:
            gains = torch.empty((2, a.dh), dtype=torch.float32, device=dev)
            x = gains.data_ptr()
            a.dq_gamma, a.dk_gamma = x, x + 4 * a.dh
            _launch(plan.fn, a, plan.ws, dev)
            return dq, dk, gains[0], gains[1]
    a, given = _norm_args(*held, *options)
    dev = given[0].device
    more = (dq_out, dk_out)
    dq_out, dk_out = _heads(dq_out, "dq_out", q.dtype, dev), _heads(dk_out, "dk_out", q.dtype, dev)
    _need(dq_out.shape == q.shape and dk_out.shape == k.shape, "dq_out and dk_out must have the shapes of q and k")
    dq, dk = _dest(dq, "dq", q.shape, q.dtype, dev), _dest(dk, "dk", k.shape, q.dtype, dev)
    gains = torch.empty((2, a.dh), dtype=torch.float32, device=dev)
    if a.B == 0 or a.n == 0:
        gains.zero_()
        return dq, dk, gains[0], gains[1]
    for name, t in (("dq_out", dq_out), ("dk_out", dk_out), ("dq", dq), ("dk", dk)):
        _set(a, name, t)
    a.dq_gamma, a.dk_gamma = gains.data_ptr(), gains.data_ptr() + 4 * a.dh
    ws, fn = _ws_bytes("fact_qk_norm_workspace", a, 1), L.lib().fact_qk_norm_backward
    _launch(fn, a, ws, dev)
    if all(x is y for x, y in zip(held + more, given + (dq_out, dk_out))):
        _keep(key, a, fn, ws)
    return dq, dk, gains[0], gains[1]
