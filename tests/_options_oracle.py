"""The oracle's FACT model with the attention options of the transformer config: RMS norm of queries and keys with rotation,
symmetric window with sinks, relative position bias by buckets (float64, autograd)."""
import math

import torch

from oracle import fact_oracle as O


def bucket_map(buckets, dist):
    """Both directions: half of a side's buckets one distance each, then equal ratios up to dist (tests of the map itself use
    exact arithmetic: tests/test_attention_args.py)."""
    n = buckets // 2
    e = n // 2
    got = []
    for d in range(-dist, dist + 1):
        far = abs(d)
        b = far if far < e else min(n - 1, e + int(math.log(far / e) / math.log(dist / e) * (n - e) + 1e-9))
        got.append(b + (n if d > 0 else 0))
    return torch.tensor(got)


def attention(x, params, base, heads, opt, eps=1e-5):
    b, n, dim = x.shape
    dh = dim // heads
    qkv = (x @ params[base + "/attn/to_qkv/kernel"]).view(b, n, 3, heads, dh).permute(2, 0, 3, 1, 4)
    q, k, v = qkv[0], qkv[1], qkv[2]
    if opt.get("qk_norm"):
        def norm(t, g):
            t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * params[base + "/attn/%s_norm/gamma" % g]
            rd = opt.get("rotary_dim", 0)
            if rd:
                i = torch.arange(rd // 2, dtype=t.dtype)
                ang = torch.arange(n, dtype=t.dtype)[:, None] * opt.get("rotary_base", 10000.0) ** (-2 * i / rd)
                c, s = ang.cos(), ang.sin()
                a, w = t[..., :rd // 2], t[..., rd // 2:rd]
                t = torch.cat((a * c - w * s, w * c + a * s, t[..., rd:]), -1)
            return t
        q, k = norm(q, "q"), norm(k, "k")
    dots = q @ k.transpose(-1, -2) * dim ** -0.5
    d = torch.arange(n)[None] - torch.arange(n)[:, None]
    if opt.get("rel_buckets"):
        D = opt["rel_max_distance"]
        table = params[base + "/attn/relative_bias/table"]
        dots = dots + table[bucket_map(opt["rel_buckets"], D)[d.clamp(-D, D) + D]].permute(2, 0, 1)
    if opt.get("window"):
        seen = (d.abs() <= opt["window"]) | ((torch.arange(n)[None] < opt.get("sinks", 0)) & (d <= opt["window"]))
        dots = dots.masked_fill(~seen, -math.inf)
    out = (torch.softmax(dots, -1) @ v).permute(0, 2, 1, 3).reshape(b, n, dim)
    return out @ params[base + "/attn/to_out/kernel"] + params[base + "/attn/to_out/bias"]


def transformer(x, params, prefix, c, opt):
    for l in range(c["layers"]):
        base = "%s/layer_%d" % (prefix, l)
        p = {k: params[v] for k, v in O.layer_names(prefix, l).items()}
        x = attention(O.layer_norm(x, p["ln1_g"], p["ln1_b"]), params, base, c["heads"], opt) + x
        x = O.mlp(O.layer_norm(x, p["ln2_g"], p["ln2_b"]), p["w1"], p["b1"], p["w2"], p["b2"]) + x
    return x


def forward(params, cfg, opts, motion, audio):
    feats = []
    for name, inp in (("motion", motion), ("audio", audio)):
        f = inp @ params[name + "_linear_embedding/kernel"] + params[name + "_linear_embedding/bias"]
        f = f + params[name + "_pos_embedding/position_embedding"]
        feats.append(transformer(f, params, name + "_transformer", cfg[name], opts.get(name, {})))
    x = transformer(torch.cat(feats, 1), params, "cross_modal_layer/transformer", cfg["cross"], opts.get("cross", {}))
    return x @ params["cross_modal_layer/output/kernel"] + params["cross_modal_layer/output/bias"]


def loss_and_grads(params, cfg, opts, batch):
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in params.items()}
    pred = forward(leaves, cfg, opts, batch["motion_input"], batch["audio_input"])
    loss = O.motion_loss(batch["target"], pred)
    loss.backward()
    return loss.detach(), {k: v.grad if v.grad is not None else torch.zeros_like(v) for k, v in leaves.items()}, pred.detach()


def set_options(config, opts):
    """Write {stack: options} into a MultiModalModel config."""
    fm = config.fact_model
    targets = {m.feature_name: m.model[0].transformer for m in fm.modality}
    targets["cross"] = fm.cross_modal_model.transformer
    for name, o in opts.items():
        t = targets[name]
        t.qk_norm = bool(o.get("qk_norm", 0))
        t.rotary_dim = o.get("rotary_dim", 0)
        t.rotary_base = o.get("rotary_base", 10000.0)
        t.attention_window = o.get("window", 0)
        t.attention_sinks = o.get("sinks", 0)
        t.relative_attention_num_buckets = o.get("rel_buckets", 0)
        t.relative_attention_max_distance = o.get("rel_max_distance", 128)
    return config
