"""The training step with norms and gates after the blocks, a scaled stream and activations kept in 8 bits: the operators of
tests/test_residual_norm.py and tests/test_act8.py run together, as TinyTransformer runs them.

The oracle of the step sees, for the backward, the activations that the GPU kept: the bytes are downloaded and restored, so that
a value on the border between two steps, which another rounding in the forward puts on the other side, is not counted as an
error of the backward.  Tolerances are those of tests/test_tiny_transformer.py for the same reasons.
"""
import numpy as np
import pytest

from helpers import integers
from oracle import oracle_np as O

from mograd_amd import BF16, F16, F32, AnyBuffer, MogradError
from mograd_amd.runtime import round_to_dtype
from mograd_amd.tiny_transformer import POST_NORM_PARAMS, TinyTransformer, init_params


def _params(seed, V, d, ff, L, post_norm):
    rng = np.random.Generator(np.random.PCG64(seed))
    params = init_params(rng, V, d, ff, L, post_norm)
    for b in params["blocks"]:  # off the defaults, which would hide a swapped or dropped one
        for name in b:
            if name.endswith("_g") or name.startswith("gate"):
                b[name] = rng.uniform(0.5, 1.5, b[name].shape).astype(np.float32)
            elif name.endswith("_b"):
                b[name] = rng.normal(0, 0.1, b[name].shape).astype(np.float32)
    return params


def _flat(tree):
    out = {k: v for k, v in tree.items() if k != "blocks"}
    for i, b in enumerate(tree["blocks"]):
        out.update({f"blocks.{i}.{k}": v for k, v in b.items()})
    return out


def _rounded(params, dtype):
    r = lambda a: round_to_dtype(a, dtype).astype(np.float64)
    return {k: r(v) if k != "blocks" else [{n: r(a) for n, a in b.items()} for b in v] for k, v in params.items()}


# ---- the oracle, no GPU --------------------------------------------------------------------


def test_oracle_without_options_is_the_plain_step():
    params = _params(1, 11, 16, 40, 2, False)
    rng = np.random.default_rng(2)
    ids, labels = rng.integers(0, 11, (3, 9)), rng.integers(0, 11, (3, 9))
    loss, grads = O.residual_transformer_step(params, ids, labels, 2)
    want_loss, want = O.tiny_transformer_step(params, ids, labels, 2)
    assert abs(loss - want_loss) < 1e-12
    got, want = _flat(grads), _flat(want)
    assert set(got) == set(want)
    for name in want:
        np.testing.assert_allclose(got[name], want[name], atol=1e-11, err_msg=name)


def test_oracle_against_autograd():
    import torch

    F = torch.nn.functional
    V, d, ff, L, H, B, T, scale = 11, 16, 40, 2, 2, 3, 9, 0.8
    params = _params(3, V, d, ff, L, True)
    rng = np.random.default_rng(4)
    ids, labels = rng.integers(0, V, (B, T)), rng.integers(0, V, (B, T))
    loss, grads = O.residual_transformer_step(params, ids, labels, H, scale)
    leaf = lambda a: torch.tensor(np.asarray(a, np.float64), requires_grad=True)
    p = {k: leaf(v) if k != "blocks" else [{n: leaf(a) for n, a in b.items()} for b in v] for k, v in params.items()}
    norm = lambda x, b, name: F.layer_norm(x, (d,), b[name + "_g"], b[name + "_b"], 1e-5)
    h = F.embedding(torch.from_numpy(ids), p["embed"])
    for b in p["blocks"]:
        x = norm(h, b, "ln1")
        q, k, v = (F.linear(x, b[w]).reshape(B, T, H, d // H).transpose(1, 2) for w in ("wq", "wk", "wv"))
        f = F.linear(F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(B, T, d), b["wo"])
        h = scale * h + b["gate1"] * norm(f, b, "post1")
        f = F.linear(F.relu(F.linear(norm(h, b, "ln2"), b["w1"], b["b1"])), b["w2"])
        h = scale * h + b["gate2"] * norm(f, b, "post2")
    want = F.cross_entropy(F.linear(h, p["lm_head"]).reshape(B * T, -1), torch.from_numpy(labels).reshape(-1))
    want.backward()
    assert abs(loss - want.item()) < 1e-12
    got = _flat(grads)
    for name, t in _flat(p).items():
        np.testing.assert_allclose(got[name], t.grad.numpy(), atol=1e-11, err_msg=name)


def test_init_params_of_the_post_norms():
    b = init_params(np.random.default_rng(0), 5, 8, 16, 1, post_norm=True)["blocks"][0]
    assert set(POST_NORM_PARAMS) <= set(b)
    assert (b["gate1"] == 1).all() and (b["post2_g"] == 1).all() and (b["post1_b"] == 0).all()


# ---- on the GPU ----------------------------------------------------------------------------


def _kept(model, n):
    """What the backward saw: the restored bytes where an activation is kept in 8 bits."""
    def of(layer, name, value):
        buf = model.saved[layer].get(name + "_8")
        if buf is None:
            return value
        cols = value.shape[1]
        return O.act8_load(buf.to_numpy().view(np.uint8)[:model.lib.mg_act8_bytes(n, cols)], n, cols)
    return of


OPTIONS = [dict(post_norm=True), dict(post_norm=True, act8=True), dict(act8=True), dict(residual_scale=0.75),
           dict(post_norm=True, act8=True, residual_scale=1.25)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(F32, 2e-4), (BF16, 8e-2)])
@pytest.mark.parametrize("V,d,ff,L,H,B,T", [(17, 64, 128, 2, 2, 2, 24), (29, 72, 100, 3, 2, 3, 41)])
@pytest.mark.parametrize("options", OPTIONS)
def test_step_matches_oracle(device, dtype, tol, V, d, ff, L, H, B, T, options):
    params = _params(80 + V, V, d, ff, L, options.get("post_norm", False))
    ids, labels = integers(81, 1, (B, T), 0, V, np.int32), integers(81, 2, (B, T), 0, V, np.int32)
    model = TinyTransformer(device, V, d, ff, L, H, compute_dtype=dtype, **options)
    model.load_params(params)
    got_loss = model.step(AnyBuffer.from_numpy(device, ids), AnyBuffer.from_numpy(device, labels), B, T).item()
    got = _flat(model.gradients())
    want_loss, want = O.residual_transformer_step(_rounded(params, dtype), ids, labels, H, options.get("residual_scale", 1.0),
                                                  store=lambda a: round_to_dtype(a, dtype), kept=_kept(model, B * T))
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
def test_forward_is_the_same_with_activations_in_8_bits(device, post_norm):
    """Only the backward reads them: the same loss, bit for bit; gradients off by the steps of 8 bits; fewer bytes kept."""
    V, d, ff, L, H, B, T = 33, 128, 512, 2, 4, 4, 64
    params = _params(90, V, d, ff, L, post_norm)
    ids, labels = (AnyBuffer.from_numpy(device, integers(91, i, (B, T), 0, V, np.int32)) for i in (1, 2))
    runs = []
    for act8 in (False, True):
        model = TinyTransformer(device, V, d, ff, L, H, post_norm=post_norm, act8=act8, residual_scale=0.9)
        model.load_params(params)
        loss = model.step(ids, labels, B, T).item()
        first = model.grads.to_numpy()
        assert model.step(ids, labels, B, T).item() == loss
        assert np.array_equal(model.grads.to_numpy(), first)  # no atomics anywhere: the second step is the first one
        runs.append((loss, first, model.kept_bytes()))
    (loss, grads, plain), (loss8, grads8, less) = runs
    assert loss == loss8
    rel = np.linalg.norm(grads8 - grads) / np.linalg.norm(grads)
    # a value is off by at most half a step, 2^-7 of its block's largest: its share of a gradient by no more on average
    assert 0 < rel <= 2.0 ** -7
    assert less <= 0.8 * plain


@pytest.mark.gpu
def test_deferred_sums_and_immediate_ones(device):
    V, d, ff, L, H, B, T = 21, 64, 256, 2, 2, 3, 50
    params = _params(95, V, d, ff, L, True)
    ids, labels = (AnyBuffer.from_numpy(device, integers(96, i, (B, T), 0, V, np.int32)) for i in (1, 2))
    grads = []
    for deferred in (True, False):
        model = TinyTransformer(device, V, d, ff, L, H, compute_dtype=F16, deferred=deferred, post_norm=True, act8=True)
        model.load_params(params)
        model.step(ids, labels, B, T)
        grads.append(model.grads.to_numpy())
    # the same fp32 sums, rounded to fp16 (half a step, at least 2^-25) before they are cast in the second
    assert (np.abs(grads[0] - grads[1]) <= np.maximum(2.0 ** -11 * np.abs(grads[0]), 2.0 ** -25)).all()


@pytest.mark.gpu
def test_optimizer_and_rule_tables(device):
    model = TinyTransformer(device, 13, 32, 64, 1, 2, compute_dtype=F32, post_norm=True, act8=True)
    model.load_params(_params(97, 13, 32, 64, 1, True))
    ids = AnyBuffer.from_numpy(device, integers(98, 1, (2, 8), 0, 13, np.int32))
    before = _flat(model.parameters())
    model.step(ids, ids, 2, 8)
    model.adam_step()
    after = _flat(model.parameters())
    assert all((before[n] != after[n]).any() for n in before)
    with pytest.raises(MogradError):
        model.step_via_rules(ids, ids, 2, 8)
