"""A semantic feature field end to end: render, decode, distil from the teacher
cache, gradients into the per-Gaussian features and the decoder."""

import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from feature_helpers import distill64
from helpers import random_scene
from mlx3d_b200 import splatting as gs
from mlx3d_b200.losses import distill_loss, distill_loss_and_grad
from mlx3d_b200.splatting import FeatureDecoder, GaussianModel, GaussianTrainer, decode_features
from mlx3d_b200.staging import TeacherCache

pytestmark = pytest.mark.gpu


def _scene(channels):
    cam, means, quats, scales, opac, colors = random_scene(3)
    t = lambda a: torch.tensor(a, device="cuda")  # noqa: E731
    n = means.shape[0]
    params = {"means": t(means), "quats": t(quats), "scales": torch.log(t(scales)), "opacities": torch.logit(t(opac)),
              "sh_dc": t(colors).reshape(n, 1, 3).clone(), "sh_rest": torch.zeros((n, 0, 3), device="cuda")}
    g = torch.Generator(device="cuda").manual_seed(4)
    feats = torch.randn((n, channels), device="cuda", generator=g).requires_grad_(True)
    return cam, GaussianModel(params, sh_degree=0), feats, g


@pytest.mark.parametrize("channels,hidden,classes,decoded", [(16, 40, 7, True), (12, 0, 12, False)])
def test_distill_view_against_the_plain_pipeline(channels, hidden, classes, decoded):
    cam, model, feats, g = _scene(channels)
    pixels = cam.width * cam.height
    teacher = torch.randn((2, cam.height, cam.width, classes), device="cuda", generator=g) * 3
    cache = TeacherCache(2 * pixels, 4, classes)
    for view in range(2):
        cache.write(view * pixels, teacher[view])
    dec = FeatureDecoder.create(channels, hidden, classes, generator=g) if decoded else None
    trainer = GaussianTrainer(model)
    rows = cache.at(slice(pixels, 2 * pixels))
    out = trainer.distill_view(cam, feats, rows, dec, temperature=2.0)
    assert all(p.grad is None for p in model.params.values())  # the geometry is left alone
    got = [feats.grad] + ([dec.params[k].grad for k in ("w_gate", "w_up", "w_down")] if decoded else [])

    # the same from the rendered channels on, in 64 bits
    leaf = feats.detach().clone().requires_grad_(True)
    r = model.render_features(cam, leaf, normalize=True)
    x = r["features"].detach().double().requires_grad_(True)
    ws = [dec.params[k].detach().double().requires_grad_(True) for k in ("w_gate", "w_up", "w_down")] if decoded else []
    logits = x
    if decoded:
        gate = x @ ws[0].T
        logits = (gate * torch.sigmoid(gate) * (x @ ws[1].T)) @ ws[2].T
    values, index = cache.read(slice(pixels, 2 * pixels))
    shape = (cam.height, cam.width, 4)
    loss, dl = distill64(logits.detach(), values.reshape(shape), index.reshape(shape), 2.0, r["alpha"].detach())
    grads = torch.autograd.grad(logits, [x, *ws], dl / pixels)
    r["features"].backward(grads[0].float())
    want = [leaf.grad, *grads[1:]]
    # Roundings to 16 bits (half a step e = 2^-9): weights, features, h, logits, dlogits, dg or du, and the result: 8 in a
    # row at most.  A logit's rounding changes the softmax by 2 |s| e / T.  dlogits = q - p cancels: relative to what is
    # left, the errors of q and p grow by kappa.
    kappa = float((dl.abs() + 2 * torch.softmax(logits.detach() / 2, -1) * r["alpha"].detach()[..., None] * 2).norm()
                  / dl.norm())
    tol = 2.0 ** -9 * (8 + kappa * float(logits.detach().abs().max())) if decoded else 1e-4
    assert abs(float(out["loss"]) - float(loss.mean())) <= tol * float(loss.mean())
    for a, b in zip(got, want):
        assert a.shape == b.shape
        assert float((a.double() - b.double()).norm()) <= tol * float(b.double().norm())


def test_distill_view_accumulates_and_takes_arrays():
    cam, model, feats, g = _scene(5)
    trainer = GaussianTrainer(model)
    values = torch.randn((cam.width * cam.height, 3), device="cuda", generator=g)
    index = torch.randint(0, 5, (cam.width * cam.height, 3), device="cuda", generator=g)
    first = trainer.distill_view(cam, feats, (values, index))
    once = feats.grad.clone()
    trainer.distill_view(cam, feats, (values, index))
    assert torch.allclose(feats.grad, 2 * once, rtol=1e-4, atol=1e-9)  # (the compositor's atomics change the order)
    shape = (cam.height, cam.width, 3)
    again = distill_loss(first["logits"], (values.reshape(shape), index.reshape(shape)), weight=first["alpha"])
    assert torch.equal(again, first["loss"])


def test_render_features_decodes():
    cam, model, feats, g = _scene(8)
    dec = FeatureDecoder.create(8, 16, 3, activation="gelu", generator=g)
    out = model.render_features(cam, feats, decoder=dec)
    assert out["logits"].shape == (cam.height, cam.width, 3) and out["logits"].dtype == torch.bfloat16
    assert torch.equal(out["logits"], dec(out["features"]))
    plain = gs.render_gaussian_features(cam, model.params["means"], model.params["quats"], model.scales_act,
                                        model.opacities_act, feats)
    assert "logits" not in plain and torch.equal(plain["features"], out["features"])


def test_distill_view_refuses_float16_decoders():
    cam, model, feats, g = _scene(8)
    dec = FeatureDecoder.create(8, 16, 3, dtype=torch.float16, generator=g)
    with pytest.raises(ValueError, match="bfloat16"):
        GaussianTrainer(model).distill_view(cam, feats, (torch.zeros(1, 1), torch.zeros(1, 1).int()), dec)


def test_calls_of_several_threads_at_once():
    """Different sizes of every operator from threads with streams of their own, again and again."""
    def work(seed, n, d, f, c, k):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
        leaves = [t.requires_grad_(True) for t in (rnd(n, d), rnd(f, d), rnd(f, d), rnd(c, f))]
        cache = TeacherCache(n, k, c)
        cache.write(0, rnd(n, c))

        def once():
            y = decode_features(*leaves)
            loss, grad = distill_loss_and_grad(y.detach(), cache.at(slice(0, n)))
            return [loss, *torch.autograd.grad(y, leaves, grad)]
        return once

    jobs = [work(1, 3000, 64, 256, 150, 8), work(2, 700, 16, 64, 20, 5), work(3, 5000, 128, 128, 250, 32),
            work(4, 40, 9, 30, 201, 3)]
    wants = [job() for job in jobs]
    torch.cuda.synchronize()
    failed = []

    def run(job, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = job()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    failed.append("different results")
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    threads = [threading.Thread(target=run, args=a) for a in zip(jobs, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_forward_mode_is_refused():
    """There are no forward-mode derivatives: a tangent must not get lost on the way."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    for n in (5, 300):  # both ways of decoding
        args = [rnd(n, 8).bfloat16(), rnd(16, 8).bfloat16(), rnd(16, 8).bfloat16(), rnd(4, 16).bfloat16()]
        logits, teacher = rnd(n, 4), (rnd(n, 2), torch.zeros((n, 2), device="cuda", dtype=torch.int32))
        want = decode_features(*args), distill_loss(logits, teacher)
        with fwAD.dual_level():
            assert torch.equal(decode_features(*args), want[0])  # no tangents: as ever
            assert torch.equal(distill_loss(logits, teacher), want[1])
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    for at in range(4):
                        dual = [fwAD.make_dual(t, torch.ones_like(t)) if i == at else t for i, t in enumerate(args)]
                        with pytest.raises(NotImplementedError, match="forward mode"):
                            decode_features(*dual)
                    with pytest.raises(NotImplementedError, match="forward mode"):
                        distill_loss(fwAD.make_dual(logits, torch.ones_like(logits)), teacher)


def test_calls_without_gradients_bypass_autograd():
    x, w = torch.zeros((3, 8), device="cuda").bfloat16(), torch.zeros((16, 8), device="cuda").bfloat16()
    down = torch.zeros((4, 16), device="cuda").bfloat16()
    assert not decode_features(x, w, w, down).requires_grad
    assert decode_features(x, w.clone().requires_grad_(True), w, down).requires_grad
    with torch.no_grad():
        assert not decode_features(x, w.clone().requires_grad_(True), w, down).requires_grad
