"""Cases for timing the attention operators: the per-head norm of queries and keys with rotation, and attention with a
sliding window, sinks and a learned relative position bias by buckets (forward, backward and the few-row form).

`own = False` computes them from elementary torch operations in 32 bits, `own = True` calls mint_amd.attention.
"""
import math

import torch

own = False

EPS = 1e-6
BASE = 10000.0


# ---- cases ----------------------------------------------------------------------------------------------------------
def _norm(name, B, n, H, Hkv, dh, dtype="bf16", train=False, rot=None, interleaved=False, start=0):
    """start: position of the first token of each sequence (a far one for a long track's continuation)."""
    return {"name": name, "op": "norm", "B": B, "n": n, "H": H, "Hkv": Hkv, "dh": dh, "dtype": dtype, "train": train,
            "rot": dh if rot is None else rot, "interleaved": interleaved, "start": start}


def _attn(name, B, nq, nk, H, Hkv, dh, left=-1, right=-1, sinks=0, buckets=0, dist=0, both=True, ragged=False,
          train=False, step=False, wide_scale=False):
    """step: the queries are the last `nq` tokens of each sequence; ragged: sequences of different lengths in one batch;
    wide_scale: softmax scale (H * dh)^-0.5, the model's, instead of dh^-0.5."""
    return {"name": name, "op": "attn", "B": B, "nq": nq, "nk": nk, "H": H, "Hkv": Hkv, "dh": dh, "left": left,
            "right": right, "sinks": sinks, "buckets": buckets, "dist": dist, "both": both, "ragged": ragged,
            "train": train, "step": step, "wide_scale": wide_scale}


def listed():
    return [
        # one new frame of 32 sequences that are being generated: nothing but latency
        _norm("norm_step", 32, 1, 10, 10, 80, start=4096),
        # the cross-modal stack of the default model, one training step's worth of q and k
        _norm("norm_train", 16, 360, 10, 10, 80, train=True),
        # the scaled model kept in fp32, half of each head rotated, pairs side by side
        _norm("norm_train_fp32", 8, 1440, 12, 12, 128, dtype="fp32", train=True, rot=64, interleaved=True),
        # the cross-modal stack of the default model with a relative bias, trained
        _attn("bias_train", 16, 360, 360, 10, 10, 80, buckets=32, dist=128, train=True, wide_scale=True),
        # evaluation on tracks of different lengths padded to one odd length
        _attn("bias_padded", 32, 237, 237, 10, 10, 80, buckets=32, dist=128, ragged=True, wide_scale=True),
        # the sampler's last layer: only one row of each sequence's output is kept
        _attn("bias_one_row", 32, 1, 360, 10, 10, 80, buckets=32, dist=128, wide_scale=True),
        # the scaled model with local attention to both sides, trained
        _attn("window_train", 4, 1440, 1440, 12, 12, 128, left=128, right=128, sinks=4, train=True),
        # causal, heads that share keys, an odd length, bias and window together, trained
        _attn("window_bias_train_gqa", 2, 2047, 2047, 12, 4, 64, left=255, right=0, sinks=4, buckets=32, dist=128, both=False,
              train=True),
        # one long track (136 s of frames), forward only
        _attn("window_long", 1, 8192, 8192, 10, 10, 80, left=1023, right=0, sinks=16),
        # one new token of 32 sequences against a long cache through the window
        _attn("window_step", 32, 1, 16384, 12, 4, 128, left=1023, right=0, sinks=4, ragged=True, step=True),
        # one new token of few sequences against the whole of a long cache
        _attn("bias_step_long", 4, 1, 32767, 10, 10, 80, right=0, buckets=32, dist=128, both=False, ragged=True, step=True),
        # the scaled model's cross-modal stack, full attention with a relative bias, trained: the largest
        _attn("bias_train_scaled", 8, 1440, 1440, 12, 12, 128, buckets=64, dist=512, train=True, wide_scale=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = 3.5e11  # operations of a drawn attention case at the most: the largest listed one has more
    dh = rng.choice([32, 64, 80, 96, 128])
    if rng.random() < 0.3:
        while True:
            B, n, H, group = _log_int(rng, 1, 32), _log_int(rng, 1, 2048), rng.randint(1, 16), rng.choice([1, 1, 2, 4])
            if B * n * H * (1 + group) * dh <= 3.5e7:  # values of q and k: the largest listed case has more
                break
        c = _norm("", B, n, H * group, H, dh, dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.6,
                  rot=rng.choice([0, dh // 2, dh, dh]), interleaved=rng.random() < 0.3, start=rng.choice([0, 0, rng.randint(0, 100000)]))
    else:
        kind = rng.choice(["train", "train", "forward", "step"])
        while True:
            B, Hkv, group = _log_int(rng, 1, 32), rng.randint(1, 12), rng.choice([1, 1, 2, 4])
            H = Hkv * group
            nk = _log_int(rng, 1, 2048) if kind != "step" else _log_int(rng, 16, 16384)
            nq = nk if kind != "step" else min(nk, rng.choice([1, 1, 1, 2, 3]))
            if 14 * B * H * nq * nk * dh <= most and B * H * nq * nk <= 1 << 28 and B * nk * H * dh <= 1 << 27:
                break
        causal = rng.random() < 0.5
        windowed = rng.random() < 0.6
        left = _log_int(rng, 1, 1024) if windowed else -1
        right = 0 if causal or kind == "step" else (left if windowed else -1)
        bias = rng.random() < 0.6
        c = _attn("", B, nq, nk, H, Hkv, dh, left=left, right=right, sinks=rng.choice([0, 1, 4, 17]) if windowed else 0,
                  buckets=rng.choice([8, 32, 64]) if bias else 0, dist=rng.choice([20, 128, 512]) if bias else 0,
                  both=right != 0, ragged=rng.random() < 0.5, train=kind == "train", step=kind == "step",
                  wide_scale=rng.random() < 0.3)
    del c["name"]
    return c


# ---- what the two forms share: the data ----------------------------------------------------------------------------
def _lengths(case):
    """Lengths of the sequences of a ragged batch: from the whole length down, one odd step each."""
    B, n = case["B"], case["nk"]
    low = max(1, n // 2) if case["step"] else 1
    low = max(low, case["nq"]) if case["step"] else low
    return [n - ((n - low) * b) // max(1, B - 1) for b in range(B)]


def _bucket_map(buckets, dist, both):
    """Bucket of every clipped distance key - query in -dist .. dist: half of a side's buckets one distance each, the rest
    in steps of equal ratio up to `dist`; with `both`, keys after the query have the upper half of the buckets."""
    per = buckets // 2 if both else buckets
    near = per // 2
    got = []
    for d in range(-dist, dist + 1):
        far, base = (abs(d), per if d > 0 else 0) if both else (max(-d, 0), 0)
        if far < near:
            b = far
        else:
            b = near + int(math.log(far / near) / math.log(dist / near) * (per - near) + 1e-9)
            b = min(b, per - 1)
        got.append(base + b)
    return got


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(1000003 * seed + 17)

    def normal(*shape, dtype=torch.bfloat16, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * std).to(dtype)

    B, H, Hkv, dh = case["B"], case["H"], case["Hkv"], case["dh"]
    st = {"case": case}
    if case["op"] == "norm":
        n, dt = case["n"], torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        # q, k and v of a token lie side by side, as one projection leaves them
        packed = normal(B, n, H + 2 * Hkv, dh, dtype=dt, std=1.5)
        st["q"], st["k"] = packed[:, :, :H], packed[:, :, H:H + Hkv]
        st["q_gamma"] = 1.0 + normal(dh, dtype=torch.float32, std=0.1)
        st["k_gamma"] = 1.0 + normal(dh, dtype=torch.float32, std=0.1)
        st["positions"] = (case["start"] + torch.arange(n, device=dev, dtype=torch.int32)).expand(B, n).contiguous()
        if case["train"]:
            st["dq"], st["dk"] = normal(B, n, H, dh, dtype=dt), normal(B, n, Hkv, dh, dtype=dt)
        return st
    nq, nk = case["nq"], case["nk"]
    if case["step"] or nq != nk:  # the queries are new, keys and values lie in a cache
        st["q"], st["k"], st["v"] = normal(B, nq, H, dh), normal(B, nk, Hkv, dh), normal(B, nk, Hkv, dh)
    else:
        packed = normal(B, nk, H + 2 * Hkv, dh)
        st["q"], st["k"], st["v"] = packed[:, :, :H], packed[:, :, H:H + Hkv], packed[:, :, H + Hkv:]
    st["scale"] = (H * dh if case["wide_scale"] else dh) ** -0.5
    st["kv_len"] = st["q_start"] = None
    if case["ragged"]:
        st["kv_len"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    if case["step"]:
        last = st["kv_len"] if case["ragged"] else torch.full((B,), nk, dtype=torch.int32, device=dev)
        st["q_start"] = last - nq
    st["table"] = st["map"] = None
    if case["buckets"]:
        st["table"] = normal(case["buckets"], H, dtype=torch.float32)
        st["map"] = torch.tensor(_bucket_map(case["buckets"], case["dist"], case["both"]), dtype=torch.int32, device=dev)
    if case["train"]:
        st["dout"] = normal(B, nq, H, dh)
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, rot, interleaved):
    """Rotate the pairs of the first `rot` dims of [B, n, heads, dh]; cos, sin are [B, n, 1, rot / 2]."""
    if not rot:
        return x
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    u, w = a * cos - b * sin, b * cos + a * sin
    r = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((r, rest), -1)


def _plain_norm(st):
    c = st["case"]
    rot, inter = c["rot"], c["interleaved"]
    cos = sin = None
    if rot:
        freq = BASE ** (-torch.arange(0, rot, 2, device=st["q"].device, dtype=torch.float64) / rot)
        ang = st["positions"].double()[:, :, None, None] * freq
        cos, sin = ang.cos().float(), ang.sin().float()

    def forward(x, gamma):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        return _turn(x * r * gamma, cos, sin, rot, inter)

    def backward(dz, x, gamma):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        dy = _turn(dz.float(), cos, None if sin is None else -sin, rot, inter)
        xn = x * r
        dgamma = (dy * xn).double().sum((0, 1, 2)).float()
        gd = gamma * dy
        return r * (gd - xn * (gd * xn).mean(-1, keepdim=True)), dgamma

    dt = st["q"].dtype
    out = {"q": forward(st["q"], st["q_gamma"]).to(dt), "k": forward(st["k"], st["k_gamma"]).to(dt)}
    if c["train"]:
        dq, out["dq_gamma"] = backward(st["dq"], st["q"], st["q_gamma"])
        dk, out["dk_gamma"] = backward(st["dk"], st["k"], st["k_gamma"])
        out["dq"], out["dk"] = dq.to(dt), dk.to(dt)
    return out


def _plain_attn(st):
    c = st["case"]
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    B, nq, H, dh = q.shape
    nk, Hkv = k.shape[1], k.shape[2]
    rows = H // Hkv * nq  # the query rows that share a key head
    dev = q.device
    j = torch.arange(nk, device=dev)
    p = torch.arange(nq, device=dev)[None]
    if st["q_start"] is not None:
        p = p + st["q_start"][:, None]
    d = j[None, None] - p[:, :, None]  # [B or 1, nq, nk]
    seen = torch.ones_like(d, dtype=torch.bool)
    if c["right"] >= 0:
        seen = seen & (d <= c["right"])
    if c["left"] >= 0:
        seen = seen & ((d >= -c["left"]) | (j < c["sinks"]))
    if st["kv_len"] is not None:
        seen = seen & (j[None, None] < st["kv_len"][:, None, None])
    qg = q.permute(0, 2, 1, 3).reshape(B, Hkv, rows, dh)
    kg, vg = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    s = (qg @ kg.transpose(-1, -2)).view(B, H, nq, nk) * st["scale"]
    bucket = None
    if st["table"] is not None:
        bucket = st["map"].long()[d.clamp(-c["dist"], c["dist"]) + c["dist"]]
        s = s + st["table"][bucket].permute(0, 3, 1, 2)
    s = s.masked_fill(~seen[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    w = (s - torch.where(m == -math.inf, torch.zeros_like(m), m)).exp()
    del s
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    wg = w.view(B, Hkv, rows, nk)
    o = (wg @ vg).view(B, H, nq, dh).permute(0, 2, 1, 3)
    out = {"out": o.to(torch.bfloat16)}
    if c["train"]:
        dog = st["dout"].float().permute(0, 2, 1, 3).reshape(B, Hkv, rows, dh)
        dv = wg.transpose(-1, -2) @ dog
        dw = dog @ vg.transpose(-1, -2)
        ds = wg * (dw - (wg * dw).sum(-1, keepdim=True))
        del dw
        dq = (ds @ kg) * st["scale"]
        dk = (ds.transpose(-1, -2) @ qg) * st["scale"]
        out["dq"] = dq.view(B, H, nq, dh).permute(0, 2, 1, 3).to(torch.bfloat16)
        out["dk"] = dk.permute(0, 2, 1, 3).to(torch.bfloat16)
        out["dv"] = dv.permute(0, 2, 1, 3).to(torch.bfloat16)
        if st["table"] is not None:
            # sum over the batch, then along the diagonals: with the rows turned over, laid side by side and cut one value
            # shorter each, the values of one distance lie in one column
            ds = ds.view(B, H, nq, nk).sum(0, dtype=torch.float64).flip(1)
            ds = torch.nn.functional.pad(ds, (0, nq)).view(H, -1)[:, :nq * (nk + nq - 1)].view(H, nq, nk + nq - 1).sum(1)
            d = torch.arange(1 - nq, nk, device=dev).clamp(-c["dist"], c["dist"]) + c["dist"]
            got = torch.zeros(H, c["buckets"], dtype=torch.float64, device=dev)
            out["dtable"] = got.index_add_(1, st["map"].long()[d], ds).t().contiguous().float()
    return out


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _own_norm(st):
    from mint_amd import attention as A
    c = st["case"]
    kw = dict(eps=EPS, rotary_dim=c["rot"], base=BASE, interleaved=c["interleaved"], positions=st["positions"])
    q, k = A.qk_norm_rope(st["q"], st["k"], st["q_gamma"], st["k_gamma"], **kw)
    out = {"q": q, "k": k}
    if c["train"]:
        out["dq"], out["dk"], out["dq_gamma"], out["dk_gamma"] = A.qk_norm_rope_backward(
            st["dq"], st["dk"], st["q"], st["k"], st["q_gamma"], st["k_gamma"], **kw)
    return out


def _own_attn(st):
    from mint_amd import attention as A
    c = st["case"]
    kw = dict(scale=st["scale"], window=(c["left"], c["right"]), sinks=c["sinks"], rel_table=st["table"], rel_map=st["map"],
              kv_len=st["kv_len"], q_start=st["q_start"])
    if not c["train"]:
        return {"out": A.attention(st["q"], st["k"], st["v"], **kw)}
    o, saved = A.attention(st["q"], st["k"], st["v"], training=True, **kw)
    g = A.attention_backward(st["dout"], st["q"], st["k"], st["v"], o, saved, **kw)
    out = {"out": o, "dq": g[0], "dk": g[1], "dv": g[2]}
    if st["table"] is not None:
        out["dtable"] = g[3]
    return out


def run(state):
    if state["case"]["op"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_attn(state) if own else _plain_attn(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def _seen_pairs(case):
    """(visible query-key pairs of one head over the batch, keys that any query sees over the batch)."""
    lens = _lengths(case) if case["ragged"] else [case["nk"]] * case["B"]
    pairs = keys = 0
    for n in lens:
        first = n - case["nq"] if case["step"] else 0
        p = torch.arange(first, first + case["nq"], dtype=torch.int64)
        hi = torch.clamp(p + case["right"] + 1, max=n) if case["right"] >= 0 else torch.full_like(p, n)
        lo = torch.clamp(p - case["left"], min=0) if case["left"] >= 0 else torch.zeros_like(p)
        sink = torch.clamp(torch.minimum(torch.full_like(p, min(case["sinks"], n)), hi), min=0)
        pairs += int((torch.clamp(hi - torch.maximum(lo, sink), min=0) + sink).sum())
        low, top, s = int(lo.min()), int(hi.max()), int(sink.max())
        keys += max(0, top - max(low, s)) + s
    return pairs, keys


def work(case):
    B, H, Hkv, dh = case["B"], case["H"], case["Hkv"], case["dh"]
    if case["op"] == "norm":
        values = B * case["n"] * (H + Hkv) * dh
        size = 2 if case["dtype"] == "bf16" else 4
        if case["train"]:  # reads x and dz, writes z and dx
            return {"bytes": 4 * size * values + 16 * dh, "flops": 22 * values}
        return {"bytes": 2 * size * values + 8 * dh, "flops": 8 * values}
    pairs, keys = _seen_pairs(case)
    rows = B * case["nq"] * H * dh
    moved = 2 * (2 * rows + 2 * keys * Hkv * dh)
    if case["train"]:  # dout in, dq, dk and dv out
        moved += 2 * (2 * rows + 2 * B * case["nk"] * Hkv * dh)
    return {"bytes": moved + 8 * case["buckets"] * H, "flops": (14 if case["train"] else 4) * pairs * H * dh}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _exact_norm(st):
    c = st["case"]
    rot = c["rot"]
    q, k, gq, gk = (t.double().detach().requires_grad_(True) for t in (st["q"], st["k"], st["q_gamma"], st["k_gamma"]))

    def one(x, g):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * g
        if not rot:
            return y
        i = torch.arange(rot // 2, device=x.device)
        first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + rot // 2)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                           st["positions"].double()[..., None] * torch.exp(-math.log(BASE) * 2.0 * i.double() / rot))
        z = torch.complex(y[..., first], y[..., second]) * turn[:, :, None]
        whole = torch.cat((z.real, z.imag, y[..., rot:]), -1)
        place = torch.cat((first, second, torch.arange(rot, c["dh"], device=x.device)))
        return whole[..., torch.argsort(place)]

    zq, zk = one(q, gq), one(k, gk)
    out = {"q": zq.detach(), "k": zk.detach()}
    if c["train"]:
        g = torch.autograd.grad((zq, zk), (q, k, gq, gk), (st["dq"].double(), st["dk"].double()))
        out["dq"], out["dk"], out["dq_gamma"], out["dk_gamma"] = g
    return out


def _exact_attn(st):
    c = st["case"]
    B, nq, H, dh = st["q"].shape
    group = H // c["Hkv"]
    train = c["train"]
    dev = st["q"].device
    grads = {n: torch.zeros(st[n[1:]].shape, dtype=torch.float64, device=dev) for n in ("dq", "dk", "dv")} if train else {}
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=dev)
    dtable = torch.zeros(c["buckets"], H, dtype=torch.float64, device=dev)
    for b in range(B):
        n = c["nk"] if st["kv_len"] is None else int(st["kv_len"][b])
        first = 0 if st["q_start"] is None else int(st["q_start"][b])
        at = torch.arange(first, first + nq, device=dev).unsqueeze(1)
        key = torch.arange(n, device=dev).unsqueeze(0)
        ok = torch.ones(nq, n, dtype=torch.bool, device=dev)
        if c["right"] >= 0:
            ok &= key <= at + c["right"]
        if c["left"] >= 0:
            ok &= (key + c["left"] >= at) | (key < c["sinks"])
        if st["map"] is not None:
            index = st["map"][(key - at).clamp(min=-c["dist"], max=c["dist"]) + c["dist"]].long()
        live = ok.any(1, keepdim=True)
        shut = torch.zeros(nq, n, dtype=torch.float64, device=dev).masked_fill(live & ~ok, -math.inf)
        for h in range(H):
            q = st["q"][b, :, h].double().requires_grad_(train)
            k = st["k"][b, :n, h // group].double().requires_grad_(train)
            v = st["v"][b, :n, h // group].double().requires_grad_(train)
            leaves = [q, k, v]
            with torch.set_grad_enabled(train):
                x = st["scale"] * q.matmul(k.t()) + shut
                if st["map"] is not None:
                    t = st["table"][:, h].double().requires_grad_(train)
                    leaves.append(t)
                    x = x + t.gather(0, index.reshape(-1)).view(nq, n)
                o = torch.softmax(x, 1).matmul(v) * live
            out[b, :, h] = o.detach()
            if train:
                g = torch.autograd.grad(o, leaves, st["dout"][b, :, h].double())
                grads["dq"][b, :, h] += g[0]
                grads["dk"][b, :n, h // group] += g[1]
                grads["dv"][b, :n, h // group] += g[2]
                if st["map"] is not None:
                    dtable[:, h] += g[3]
    got = {"out": out, **grads}
    if train and st["table"] is not None:
        got["dtable"] = dtable
    return got


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_norm(st) if case["op"] == "norm" else _exact_attn(st)
