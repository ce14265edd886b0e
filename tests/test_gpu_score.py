"""Model.score (nk_model_score) on the GPU, and the operators at the model's end
run together as a distillation step: a teacher's scores, the student's loss and
gradient, back through the logits product and the final norm, and an update."""

import numpy as np
import pytest

from conftest import c1_cfg, same_model, tiny_cfg

pytestmark = pytest.mark.gpu


def _seq(orc, n, vocab, seed):
    r = orc.Rng(seed)
    return np.array([r.below(vocab) for _ in range(n)], dtype=np.uint32)


def _softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


@pytest.mark.parametrize("batch,t,top", [(1, 1, 0), (1, 9, 1), (3, 17, 20), (5, 40, 128)])
def test_score_matches_the_loss_call_and_the_definition(gpu, orc, batch, t, top):
    kw = c1_cfg(dict)
    om, gm = same_model(orc, gpu, kw, seed=0)
    ids = _seq(orc, batch * t, kw["vocab"], 100 + t)
    tg = np.roll(ids, -1)
    tg[::7] = 0xFFFFFFFF
    loss, lg = gm.loss(ids, tg, batch, t, want_logits=True)
    out = gm.score(ids, tg, batch, t, top)
    live = tg != 0xFFFFFFFF
    z = lg.astype(np.float64)
    logp = z - np.log(np.exp(z - z.max(-1, keepdims=True)).sum(-1, keepdims=True)) - z.max(-1, keepdims=True)
    lp, ent = out["logprob"].reshape(-1), out["entropy"].reshape(-1)
    rows = np.arange(batch * t)
    assert (lp[~live] == 0).all() and (ent[~live] == 0).all()
    # f32 sums of 1024 terms: below 2e-5 by (4 * 24 + 52) roundings of 2^-24 of the sum, log V times that for H.
    assert np.abs(lp - logp[rows, np.where(live, tg, 0)])[live].max(initial=0) <= 2e-5
    assert np.abs(ent + (np.exp(logp) * logp).sum(-1))[live].max(initial=0) <= 2e-4
    if live.any():
        assert abs(-lp[live].mean() - loss) <= 1e-4 * max(1.0, abs(loss))
    if top:
        want = np.argsort(-lg, axis=-1, kind="stable")[:, :top].astype(np.uint32)
        got = out["top_ids"].reshape(batch * t, top)
        assert np.array_equal(got[live], want[live]) and (got[~live] == 0xFFFFFFFF).all()
        tl = out["top_logprobs"].reshape(batch * t, top)
        assert np.abs(tl - np.take_along_axis(logp, want.astype(np.int64), -1))[live].max(initial=0) <= 2e-5
        assert np.isneginf(tl[~live]).all()
    # The oracle's own logits, at its tolerance.
    _, ref = om.loss(ids, tg, batch, t, want_logits=True)
    r = ref.astype(np.float64)
    rl = r - r.max(-1, keepdims=True) - np.log(np.exp(r - r.max(-1, keepdims=True)).sum(-1, keepdims=True))
    assert np.abs(lp - rl[rows, np.where(live, tg, 0)])[live].max(initial=0) <= 2e-3


def test_score_refusals_and_other_decoders(gpu, orc):
    kw = tiny_cfg(dict, 19)
    _, gm = same_model(orc, gpu, kw, seed=2)
    ids = _seq(orc, 12, 19, 3)
    for bad in (dict(ids=np.full(12, 19, np.uint32)), dict(targets=np.full(12, 19, np.uint32)), dict(top=129)):
        a = {"ids": ids, "targets": ids, "top": 4, **bad}
        with pytest.raises(gpu.NoeticError) as e:
            gm.score(a["ids"], a["targets"], 2, 6, a["top"])
        assert e.value.status == gpu.NK_ERR_INVALID
    with pytest.raises(ValueError):
        gm.score(ids, ids, 3, 6)
    dec = gpu.Decoder(gm, 2)
    dec.step([1, 2])
    before = dec.get_state()
    # More alternatives than the vocabulary has.
    out = gm.score(ids, ids, 2, 6, 40)
    assert (out["top_ids"][..., 19:] == 0xFFFFFFFF).all() and (np.sort(out["top_ids"][..., :19], -1) == np.arange(19)).all()
    assert np.array_equal(dec.get_state()[0], before[0])


def test_a_distillation_step_of_the_final_norm_and_the_embedding(gpu, orc):
    # The student's final RMSNorm and tied embedding, trained on the teacher's
    # top 16 for one step, against the same step in 64 bits.
    V, d, batch, t, K, eps = 256, 64, 2, 33, 16, 1e-5
    kw = dict(vocab=V, d_model=d, n_layer=2, expand=1, conv_k=4, mlp_mult=2, eps=eps, tau_max=64.0)
    _, teacher = same_model(orc, gpu, kw, seed=5)
    ids = _seq(orc, batch * t, V, 9)
    tg = np.roll(ids, -1)
    tg[t - 1::t] = 0xFFFFFFFF  # nothing follows a sequence's last token
    sc = teacher.score(ids, tg, batch, t, K)
    rng = np.random.default_rng(1)
    n = batch * t
    x = rng.standard_normal((n, d)).astype(np.float32)
    gain = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)
    emb = (0.3 * rng.standard_normal((V, d))).astype(np.float32)
    T, live = 2.0, tg != 0xFFFFFFFF
    scale = 1.0 / live.sum()

    fw = gpu.layer_norm(x, gain, eps=eps, rms=True)
    logits = gpu.gemm_tn(np.ascontiguousarray(fw["y"].T), np.ascontiguousarray(emb.T), d, n, V)
    tids, tlp = sc["top_ids"].reshape(n, K), sc["top_logprobs"].reshape(n, K)
    loss, dz = gpu.distill(logits, tids, tlp, temperature=T, grad_scale=scale)
    dy = gpu.gemm_tn(np.ascontiguousarray(dz.T), emb, V, n, d)
    demb = gpu.gemm_tn(dz, fw["y"], n, V, d)
    dx, dgain, _ = gpu.layer_norm_backward(x, dy, gain, None, fw["rstd"])
    new, _, _ = gpu.adamw_step(gain, dgain, np.zeros(d), np.zeros(d), lr=1e-2, t=1, decay=False)

    x6, g6, e6 = x.astype(np.float64), gain.astype(np.float64), emb.astype(np.float64)
    r = 1 / np.sqrt((x6 * x6).mean(-1, keepdims=True) + eps)
    h = x6 * r
    z = (h * g6) @ e6.T
    q = np.zeros((n, V))
    qk = np.where(live[:, None], _softmax(np.where(live[:, None], tlp.astype(np.float64), 0) / T), 0)
    np.put_along_axis(q, np.where(live[:, None], tids, 0).astype(np.int64), qk, -1)
    q[~live] = 0
    p = _softmax(z / T)
    with np.errstate(divide="ignore", invalid="ignore"):
        kl = T * T * np.where(q > 0, q * (np.log(q) - np.log(p)), 0).sum(-1)
    dz6 = scale * T * np.where(live[:, None], p - q, 0)
    dy6 = dz6 @ e6
    c = dy6 * g6
    dx6 = r * (c - h * (c * h).mean(-1, keepdims=True))
    near = lambda a, b: np.abs(a - b).max() <= 2e-5 * np.abs(b).max()  # noqa: E731  (f32 products of up to 256 terms)
    assert near(loss, kl) and near(dz, dz6) and near(dy, dy6) and near(demb, dz6.T @ (h * g6))
    assert near(dx, dx6) and near(dgain, (dy6 * h).sum(0))
    assert (loss[~live] == 0).all() and (dz[~live] == 0).all() and (dx[~live] == 0).all()
    # AdamW's first step moves every value by lr against its gradient's sign.
    assert np.abs((gain - new) - 1e-2 * np.sign(dgain)).max() < 1e-4
    # A loss that falls along the gradient at the rate it says: first-order change for a small step.
    step = 1e-3 / np.abs(dz6).max()
    z2 = z - step * dz6
    with np.errstate(divide="ignore", invalid="ignore"):
        kl2 = T * T * np.where(q > 0, q * (np.log(q) - np.log(_softmax(z2 / T))), 0).sum(-1)
    assert abs(scale * (kl.sum() - kl2.sum()) / step / (dz6 * dz6).sum() - 1) < 1e-2
