"""The training step with gated MLPs, rotary positions and a largest norm of the gradients: the operators of test_gated_linear.py,
test_rotary.py and test_grad_norm.py run together, as TinyTransformer runs them.

Tolerances are those of tests/test_tiny_transformer.py and tests/test_residual_transformer.py for the same reasons.
"""
import numpy as np
import pytest

from helpers import integers
from oracle import oracle_np as O
from test_residual_transformer import _flat, _kept, _params, _rounded

from mograd_amd import BF16, F16, F32, I64, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype
from mograd_amd.tiny_transformer import TinyTransformer, init_params


def _gated_params(seed, V, d, ff, L, post_norm=False):
    """As _params, with both projections of a gated MLP."""
    params = _params(seed, V, d, ff, L, post_norm)
    wide = init_params(np.random.Generator(np.random.PCG64(seed + 1)), V, d, ff, L, gated_ff=True)
    for b, w in zip(params["blocks"], wide["blocks"]):
        b["w1"], b["b1"] = w["w1"], w["b1"]
    return params


def _turns(model, positions, B, T):
    """The oracle's argument for a model's rotary positions."""
    if not model.rotary_base:
        return None
    pairs = model.dh // 2
    freq = (model.rotary_base ** (-np.arange(pairs) / pairs)).astype(np.float32)
    at = np.broadcast_to(np.arange(T), (1, B, T)) if positions is None else positions
    return at, freq, [i * model.rotary_axes // pairs for i in range(pairs)]


def test_oracle_against_autograd():
    import torch

    F = torch.nn.functional
    V, d, ff, L, H, B, T = 11, 16, 20, 2, 2, 3, 9
    params = _gated_params(3, V, d, ff, L)
    rng = np.random.default_rng(4)
    ids, labels = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T))
    positions, freq, axis = rng.integers(0, 50, (2, B, T)), rng.random(4), [0, 0, 1, 1]
    loss, grads = O.residual_transformer_step(params, ids, labels, H, gated="silu", turns=(positions, freq, axis))
    leaf = lambda a: torch.tensor(np.asarray(a, np.float64), requires_grad=True)
    p = {k: leaf(v) if k != "blocks" else [{n: leaf(a) for n, a in b.items()} for b in v] for k, v in params.items()}
    angle = torch.tensor(np.moveaxis(positions[axis], 0, -1) * freq)[:, :, None, :]

    def turn(x):
        a, b = x[..., :4], x[..., 4:]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], dim=-1)

    h = F.embedding(torch.from_numpy(ids), p["embed"])
    for b in p["blocks"]:
        x = F.layer_norm(h, (d,), b["ln1_g"], b["ln1_b"], 1e-5)
        q, k, v = (F.linear(x, b[w]).reshape(B, T, H, d // H) for w in ("wq", "wk", "wv"))
        o = F.scaled_dot_product_attention(turn(q).transpose(1, 2), turn(k).transpose(1, 2), v.transpose(1, 2), is_causal=True)
        h = h + F.linear(o.transpose(1, 2).reshape(B, T, d), b["wo"])
        gu = F.linear(F.layer_norm(h, (d,), b["ln2_g"], b["ln2_b"], 1e-5), b["w1"], b["b1"])
        h = h + F.linear(F.silu(gu[..., :ff]) * gu[..., ff:], b["w2"])
    want = F.cross_entropy(F.linear(h, p["lm_head"]).reshape(B * T, -1), torch.from_numpy(labels).reshape(-1))
    want.backward()
    assert abs(loss - want.item()) < 1e-12
    got = _flat(grads)
    for name, t in _flat(p).items():
        np.testing.assert_allclose(got[name], t.grad.numpy(), atol=1e-11, err_msg=name)


def test_refusals():
    class Nothing:
        device = lib = stream = None

    for bad in (dict(gated_ff=5), dict(gated_ff=-1), dict(rotary_base=-1.0), dict(rotary_base=10.0, rotary_axes=0), dict(rotary_base=10.0, rotary_axes=9)):
        with pytest.raises(MogradError):
            TinyTransformer(Nothing(), 5, 32, 64, 1, 2, **bad)
    with pytest.raises(MogradError):
        TinyTransformer(Nothing(), 5, 30, 64, 1, 2, rotary_base=10.0)


# ---- on the GPU ----------------------------------------------------------------------------

OPTIONS = [dict(gated_ff=0), dict(rotary_base=100.0), dict(gated_ff=2, rotary_base=100.0, rotary_axes=3), dict(gated_ff=1, post_norm=True, rotary_base=50.0),
           dict(gated_ff=0, act8=True, rotary_base=50.0), dict(gated_ff=4, post_norm=True, act8=True, residual_scale=1.25), dict(gated_ff=3, deferred=False)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(F32, 2e-4), (BF16, 8e-2)])
@pytest.mark.parametrize("V,d,ff,L,H,B,T", [(17, 64, 128, 2, 2, 2, 24), (29, 72, 100, 3, 2, 3, 41)])
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: ",".join(f"{k}={v}" for k, v in o.items()))
def test_step_matches_oracle(device, dtype, tol, V, d, ff, L, H, B, T, options):
    gated = options.get("gated_ff")
    make = _params if gated is None else _gated_params
    params = make(80 + V, V, d, ff, L, options.get("post_norm", False))
    ids, labels = integers(81, 1, (B, T), 0, V, np.int32), integers(81, 2, (B, T), 0, V, np.int32)
    model = TinyTransformer(device, V, d, ff, L, H, compute_dtype=dtype, **options)
    model.load_params(params)
    at = integers(81, 3, (model.rotary_axes, B, T), 0, 60, np.int64) if model.rotary_axes > 1 else None
    positions = None if at is None else AnyBuffer.from_numpy(device, at)
    got_loss = model.step(AnyBuffer.from_numpy(device, ids), AnyBuffer.from_numpy(device, labels), B, T, positions=positions).item()
    got = _flat(model.gradients())
    want_loss, want = O.residual_transformer_step(_rounded(params, dtype), ids, labels, H, options.get("residual_scale", 1.0),
                                                  store=lambda a: round_to_dtype(a, dtype), kept=_kept(model, B * T),
                                                  gated=None if gated is None else O.GATES[gated], turns=_turns(model, at, B, T))
    want = _flat(want)
    assert abs(got_loss - want_loss) <= (2e-4 if dtype == F32 else 2.0 ** -8) * abs(want_loss), (got_loss, want_loss)
    assert set(got) == set(want)
    for name in want:
        assert np.isfinite(got[name]).all(), name
        if dtype == F32:
            err, scale = np.abs(got[name] - want[name]).max(), np.abs(want[name]).max()
            assert err <= tol * scale, f"{name}: max err {err:.3g} vs max |grad| {scale:.3g}"
        else:
            rel = np.linalg.norm(got[name] - want[name]) / np.linalg.norm(want[name])
            assert rel <= tol, f"{name}: relative L2 error {rel:.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("post_norm", [False, True])
def test_deferred_sums_and_immediate_ones(device, post_norm):
    V, d, ff, L, H, B, T = 21, 64, 256, 2, 2, 3, 50
    params = _gated_params(95, V, d, ff, L, post_norm)
    ids, labels = (AnyBuffer.from_numpy(device, integers(96, i, (B, T), 0, V, np.int32)) for i in (1, 2))
    grads = []
    for deferred in (True, False):
        model = TinyTransformer(device, V, d, ff, L, H, compute_dtype=F16, deferred=deferred, gated_ff=0, rotary_base=1e4, post_norm=post_norm)
        model.load_params(params)
        model.step(ids, labels, B, T)
        grads.append(model.grads.to_numpy())
        model.step(ids, labels, B, T)
        assert np.array_equal(model.grads.to_numpy(), grads[-1])  # no atomics anywhere: the second step is the first one
    # the same fp32 sums, rounded to fp16 (half a step, at least 2^-25) before they are cast in the second
    assert (np.abs(grads[0] - grads[1]) <= np.maximum(2.0 ** -11 * np.abs(grads[0]), 2.0 ** -25)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_training_steps_with_a_largest_norm(device, share):
    """Three steps: the norm is that of all gradients, and each update bit for bit Adam's from gradients scaled by max_norm / norm."""
    V, d, ff, L, H, B, T = 13, 32, 48, 2, 2, 3, 20
    model, plain = (TinyTransformer(device, V, d, ff, L, H, gated_ff=0, rotary_base=1e4) for _ in range(2))
    for m in (model, plain):
        m.load_params(_gated_params(97, V, d, ff, L))
    ids, labels = (AnyBuffer.from_numpy(device, integers(98, i, (B, T), 0, V, np.int32)) for i in (1, 2))
    for step in range(3):
        for m in (model, plain):
            m.step(ids, labels, B, T)
        g = model.grads.to_numpy()
        assert np.array_equal(plain.grads.to_numpy(), g)
        norm = O.grad_norm(list(_flat(model.gradients()).values()))
        most = float(np.float32(share * norm))
        model.adam_step(lr=1e-2, weight_decay=0.01, decoupled=True, max_norm=most)
        got = model.grad_norm.to_numpy()[0]
        assert abs(got - norm) <= 2.0 ** -23 * norm
        assert np.array_equal(model.grads.to_numpy(), g)
        scale = np.float32(most) / got if got > np.float32(most) else np.float32(1)
        scaled = (g * scale).astype(np.float32)
        device.lib.mg_copy_to_device(plain.grads.data_ptr(), scaled.ctypes.data, scaled.nbytes, device.stream)
        plain.adam_step(lr=1e-2, weight_decay=0.01, decoupled=True)
        assert np.array_equal(model.master.to_numpy(), plain.master.to_numpy()), step


@pytest.mark.gpu
def test_positions_and_rule_tables(device):
    model = TinyTransformer(device, 13, 32, 64, 1, 2, compute_dtype=F32, gated_ff=0, rotary_base=1e4, rotary_axes=2)
    model.load_params(_gated_params(97, 13, 32, 64, 1))
    ids = AnyBuffer.from_numpy(device, integers(98, 1, (2, 8), 0, 13, np.int32))
    good = AnyBuffer.from_numpy(device, np.zeros((2, 2, 8), np.int64))
    assert good.dtype == I64
    model.step(ids, ids, 2, 8, positions=good)
    for bad in (None, AnyBuffer.from_numpy(device, np.zeros((2, 8), np.int64)), AnyBuffer.from_numpy(device, np.zeros((2, 2, 8), np.float32), F32)):
        with pytest.raises(MogradError):
            model.step(ids, ids, 2, 8, positions=bad)
    with pytest.raises(MogradError):
        model.step_via_rules(ids, ids, 2, 8)
    with pytest.raises(MogradError):
        TinyTransformer(device, 13, 32, 64, 1, 2).step(ids, ids, 2, 8, positions=good)
