"""FACTModel with the attention options of the transformer config (q / k norm with rotation, window with sinks, relative
position bias) against the float64 oracle with the same options: forward, every gradient, the sampler, optimizer steps,
checkpoints.  Tolerances are those of the model tests without options (bf16 operands): forward 2e-2, loss 1e-2, per-tensor
gradient cosine 0.99 and relative error 8e-2."""
import ctypes

import pytest
import torch

from mint_amd import _lib as L
from mint_amd import checkpoint, model_builder
from mint_amd.trainer import Adam, SingleTaskTrainer
from oracle import fact_oracle as O
from tests import _options_oracle as P
from tests.test_gpu_model import cos, gpu_batch, make_config, oracle_params, rel

pytestmark = pytest.mark.gpu

ALL = dict(qk_norm=1, rotary_dim=32, window=20, sinks=4, rel_buckets=16, rel_max_distance=40)
SETS = {
    "all": {"motion": ALL, "audio": dict(ALL, window=12, rotary_dim=16), "cross": dict(ALL, window=30, sinks=33)},
    "norm": {"motion": dict(qk_norm=1), "cross": dict(qk_norm=1, rotary_dim=32, rotary_base=500.0)},
    "bias": {"cross": dict(rel_buckets=32, rel_max_distance=128)},
    "window": {"audio": dict(window=9), "cross": dict(window=25, sinks=1)},
}


def _model(cfg, opts, B, training=True, seed=1):
    model = model_builder.build(P.set_options(make_config(cfg), opts), training)
    model.build(B, 225, 35)
    g = torch.Generator().manual_seed(seed)
    for name, v in zip(model.variable_names, model.trainable_variables):
        if name.endswith("/bias") or name.endswith("/beta"):
            v.copy_(torch.randn(v.shape, generator=g) * 0.05)
        elif name.endswith("/gamma"):
            v.copy_(1.0 + torch.randn(v.shape, generator=g) * 0.1)
        elif name.endswith("/table"):
            v.copy_(torch.randn(v.shape, generator=g))
        if "_norm/gamma" in name and "/attn/" in name:  # logits large enough for the options to matter at scale dim^-0.5
            v.mul_(2.0)
    model.sync_weights()
    return model


@pytest.mark.parametrize("name", sorted(SETS))
@pytest.mark.parametrize("sr", [0, 1])
def test_tiny_forward_and_every_gradient(name, sr):
    cfg, opts, B, T = O.TINY_CFG, SETS[name], 4, 8
    model = _model(cfg, opts, B)
    model.set_option("sr_rows", sr)
    batch = O.synthetic_batch(cfg, B, T, seed=2)
    gb = gpu_batch(batch)
    params = oracle_params(model)
    inputs = {k: gb[k] for k in ("motion_input", "audio_input")}
    out = model(inputs)
    loss, grads, pred = P.loss_and_grads(params, cfg, opts, batch)
    assert rel(out, pred) < 2e-2
    plain = O.fact_forward(params, cfg, batch["motion_input"], batch["audio_input"])
    assert rel(pred, plain) > 3e-2  # the options matter here
    for _ in range(2):  # gradients accumulate into the arena, the second call doubles them
        got = model.forward_backward(inputs, gb["target"])
    assert abs(float(got) - float(loss)) / float(loss) < 1e-2
    for n, g in zip(model.variable_names, model.gradients):
        ref = 2 * grads[n]
        if float(ref.norm()) < 1e-9:
            assert float(g.norm()) < 1e-6, n
            continue
        assert cos(g, ref) > 0.99 and rel(g, ref) < 8e-2, (n, cos(g, ref), rel(g, ref))


def test_fact_v5_dims_forward_and_gradients():
    cfg = {k: (dict(v, layers=1) if isinstance(v, dict) else v) for k, v in O.FACT_V5_CFG.items()}
    opts = {"motion": dict(rel_buckets=32, rel_max_distance=64), "audio": dict(window=64, sinks=4),
            "cross": dict(qk_norm=1, rotary_dim=80, window=100, sinks=8, rel_buckets=32, rel_max_distance=128)}
    B, T = 2, 20
    model = _model(cfg, opts, B)
    batch = O.synthetic_batch(cfg, B, T, seed=3)
    gb = gpu_batch(batch)
    loss, grads, pred = P.loss_and_grads(oracle_params(model), cfg, opts, batch)
    inputs = {k: gb[k] for k in ("motion_input", "audio_input")}
    assert rel(model(inputs), pred) < 2e-2
    got = model.forward_backward(inputs, gb["target"])
    assert abs(float(got) - float(loss)) / float(loss) < 1e-2
    for n, g in zip(model.variable_names, model.gradients):
        if float(grads[n].norm()) < 1e-9:
            continue
        assert cos(g, grads[n]) > 0.99 and rel(g, grads[n]) < 8e-2, (n, cos(g, grads[n]), rel(g, grads[n]))


def test_sampler_matches_oracle_and_the_full_rows():
    """The sampler keeps one row of the last layer: the single-row kernel against the whole, and both against the oracle."""
    cfg, opts, B = O.TINY_CFG, SETS["all"], 3
    got = {}
    for sr in (1, 0):
        model = _model(cfg, opts, B, training=False)
        model.set_option("sr_rows", sr)
        batch = O.synthetic_batch(cfg, B, 8, seed=4)
        g = torch.Generator().manual_seed(9)
        audio = torch.randn(B, 64 + 5, 35, generator=g, dtype=torch.float64)
        got[sr] = model.infer_auto_regressive({"motion_input": batch["motion_input"].float().cuda(),
                                               "audio_input": audio.float().cuda()}, steps=20)
    params = oracle_params(model)
    motion, outs = batch["motion_input"], []
    for i in range(6):
        out = P.forward(params, cfg, opts, motion, audio[:, i:i + 64])[:, :1]
        outs.append(out)
        motion = torch.cat([motion[:, 1:], out], 1)
    ref = torch.cat(outs, 1)
    for sr in (0, 1):
        assert got[sr].shape == ref.shape and rel(got[sr], ref) < 3e-2, (sr, rel(got[sr], ref))


@pytest.mark.parametrize("fused", [False, True])
def test_trainer_steps_update_the_new_variables(fused):
    cfg, opts = O.TINY_CFG, SETS["all"]
    model = _model(cfg, opts, 4)
    gb = gpu_batch(O.synthetic_batch(cfg, 4, 8, seed=5))
    before = {n: v.clone() for n, v in zip(model.variable_names, model.trainable_variables)}
    trainer = SingleTaskTrainer([gb], "target", model, optimizer=Adam(1e-3), grad_clip_norm=0.0 if fused else 1.0)
    losses = [float(trainer.train_step(iter([gb]))) for _ in range(6)]
    assert all(x == x for x in losses)
    for n, v in zip(model.variable_names, model.trainable_variables):
        if "/attn/q_norm" in n or "/attn/k_norm" in n or "/relative_bias/" in n:
            moved = (v - before[n]).abs()
            assert float(moved.max()) > 1e-4 and torch.isfinite(v).all(), n
    used = [n for n in model.variable_names if "/relative_bias/" in n]
    assert len(used) == 6  # one table a layer


def test_two_streams_of_encoders_and_repeat():
    """Motion and audio stacks run beside each other with their own workspaces: the same step twice gives the same gradients."""
    cfg, opts = O.TINY_CFG, SETS["all"]
    model = _model(cfg, opts, 4)
    gb = gpu_batch(O.synthetic_batch(cfg, 4, 8, seed=6))
    inputs = {k: gb[k] for k in ("motion_input", "audio_input")}
    seen = []
    for _ in range(3):
        model.grad_arena.zero_()
        model.forward_backward(inputs, gb["target"])
        seen.append({n: g.clone() for n, g in zip(model.variable_names, model.gradients)})
    for n in seen[0]:  # (bias and split-K sums of the engine use fp32 atomics: equal up to their order)
        assert rel(seen[1][n], seen[0][n]) < 1e-3 and rel(seen[2][n], seen[0][n]) < 1e-3, n


@pytest.mark.parametrize("name", ["all", "window", "bias"])
def test_batches_smaller_than_the_handle(name):
    """Fewer sequences are cut into more pieces: a handle for 24 has the workspace of every smaller batch, too."""
    cfg, opts = {k: (dict(v, layers=1) if isinstance(v, dict) else v) for k, v in O.TINY_CFG.items()}, SETS[name]
    cfg["motion"]["seq_len"], cfg["audio"]["seq_len"] = 256, 512
    ask = L.FactAttention(H=4, Hkv=4, nq=768, nk=768, dh=32, window_left=-1, window_right=-1, scale=1.0)
    for i, t in enumerate(("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv")):
        setattr(ask, t, 4096 * (i + 1))
        if t != "lse":
            getattr(ask, t + "_stride")[:] = (1 << 20, 128, 32)
    need, bytes_ = {}, ctypes.c_size_t(0)
    for ask.B in (1, 24):
        L.check(L.lib().fact_attention_workspace(ctypes.byref(ask), 1, ctypes.byref(bytes_)))
        need[ask.B] = bytes_.value
    assert need[1] > need[24]  # (what makes this more than a repetition)
    big = _model(cfg, opts, 24)
    for B in (1, 2, 5, 11, 24):
        one = _model(cfg, opts, B)
        gb = gpu_batch(O.synthetic_batch(cfg, B, 8, seed=B))
        inputs = {k: gb[k] for k in ("motion_input", "audio_input")}
        seen = []
        for model in (big, one):
            model.grad_arena.zero_()
            loss = float(model.forward_backward(inputs, gb["target"]))
            seen.append((loss, {n: g.clone() for n, g in zip(model.variable_names, model.gradients)}, model(inputs).clone()))
        assert seen[0][0] == pytest.approx(seen[1][0], rel=1e-5) and rel(seen[0][2], seen[1][2]) < 1e-5
        # The engine's fp32 atomics (bias and split-K sums) add in any order, also between two runs of one handle; a sum that lies
        # at a border of bf16 rounds to either neighbour, one step of 2^-7 apart, so no value downstream is off by more than that
        # share of what it sums.  Pieces written over each other would be off by whole terms.
        for n in seen[0][1]:
            assert rel(seen[0][1][n], seen[1][1][n]) < 2.0 ** -7, (B, n)


def test_checkpoint_round_trip_with_options(tmp_path):
    cfg, opts = O.TINY_CFG, SETS["all"]
    a = _model(cfg, opts, 2)
    prefix = str(tmp_path / "ckpt-1")
    checkpoint.export_tf_checkpoint(a, prefix)
    b = _model(cfg, opts, 2, seed=8)
    checkpoint.import_tf_checkpoint(b, prefix)
    for n, x, y in zip(a.variable_names, a.trainable_variables, b.trainable_variables):
        assert torch.equal(x, y), n
    batch = O.synthetic_batch(cfg, 2, 8, seed=7)
    inputs = {k: batch[k].float().cuda() for k in ("motion_input", "audio_input")}
    assert torch.equal(a(inputs), b(inputs))


def test_defaults_leave_the_model_as_it_was():
    cfg = O.TINY_CFG
    model = model_builder.build(make_config(cfg), True)
    model.build(2, 225, 35)
    assert model.variable_names == [n for n, _ in O.param_shapes(cfg)]
