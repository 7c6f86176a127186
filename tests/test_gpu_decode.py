"""Gated feature decoder on the GPU against the plain 64-bit form."""

import ctypes
import math
import threading

import pytest
import torch

from feature_helpers import DTYPES, decode64, decode_norm_bound, decode_tolerances, norm_off
from mlx3d_b200 import _native as nat
from mlx3d_b200.splatting import FeatureDecoder, decode_features

pytestmark = pytest.mark.gpu


def _inputs(n, d, f, c, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    ty = DTYPES[dtype]
    x = rnd(n, d)
    x[: n // 10] = 0.0  # uncovered pixels
    return (x.to(ty), (rnd(f, d) / math.sqrt(d)).to(ty), (rnd(f, d) / math.sqrt(d)).to(ty),
            (rnd(c, f) * 2 / math.sqrt(f)).to(ty), (rnd(n, c) * 0.1).to(ty))


def _wait_failures():
    cnt = ctypes.c_uint64(0)
    nat.call("gs_wait_failures", ctypes.byref(cnt), 0)
    return cnt.value


def _within(got, want, tol):
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() / tol.clamp(min=1e-30)).max()
    assert float(worst) <= 1.0, float(worst)


SIZES = [
    (1, 1, 1, 1), (1, 32, 64, 20), (2, 3, 5, 7), (127, 16, 64, 16), (128, 64, 64, 64), (129, 17, 65, 33),
    (300, 47, 171, 133), (1000, 128, 256, 256), (513, 64, 200, 150), (260, 65, 40, 129), (130, 8, 600, 250),
    (77, 120, 128, 2), (40000, 64, 128, 150), (20001, 33, 70, 31),
]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,c", SIZES)
def test_forward_matches_the_definition(n, d, f, c, dtype, act):
    x, wg, wu, wd, _ = _inputs(n, d, f, c, dtype, seed=n + d)
    y = decode_features(x, wg, wu, wd, act)
    assert y.shape == (n, c) and y.dtype == x.dtype
    _within(y, decode64(x, wg, wu, wd, act), decode_tolerances(x, wg, wu, wd, act))
    assert _wait_failures() == 0


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,c", SIZES)
def test_gradients_match_the_definition(n, d, f, c, dtype, act):
    x, wg, wu, wd, dy = _inputs(n, d, f, c, dtype, seed=n + c)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = decode_features(*leaves, act)
    grads = torch.autograd.grad(y, leaves, dy)
    plain = [t.detach() for t in leaves]
    want = decode64(*plain, act, dy)
    tol = decode_tolerances(*plain, act, dy)
    for got, w, t, leaf in zip((y.detach(), *grads), want, tol, (y, *leaves)):
        assert got.shape == leaf.shape and got.dtype == leaf.dtype
        _within(got, w, t)
    assert _wait_failures() == 0


def test_gradients_on_demand_are_the_same_numbers():
    x, wg, wu, wd, dy = _inputs(700, 40, 100, 30, "bf16")
    full = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    want = torch.autograd.grad(decode_features(*full), full, dy)
    for need in ((True, False, False, False), (False, True, False, False), (False, False, False, True)):
        leaves = [t.clone().requires_grad_(r) for t, r in zip((x, wg, wu, wd), need)]
        decode_features(*leaves).backward(dy)
        for leaf, w, r in zip(leaves, want, need):
            assert (leaf.grad is None) if not r else torch.equal(leaf.grad, w)


def test_repeated_calls_are_bitwise_equal():
    x, wg, wu, wd, dy = _inputs(30000, 64, 256, 150, "bf16")
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    runs = []
    for _ in range(3):
        y = decode_features(*leaves)
        runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_images_strides_types_and_unaligned_rows():
    x, wg, wu, wd, _ = _inputs(20 * 30, 24, 50, 11, "fp16")
    want = decode_features(x, wg, wu, wd)
    assert torch.equal(decode_features(x.reshape(20, 30, 24), wg, wu, wd), want.reshape(20, 30, 11))
    wide = torch.zeros((600, 40), device="cuda", dtype=x.dtype)
    wide[:, 5:29] = x
    assert torch.equal(decode_features(wide[:, 5:29], wg, wu, wd), want)
    flat = torch.zeros((600 * 24 + 1,), device="cuda", dtype=x.dtype)
    flat[1:] = x.reshape(-1)
    assert torch.equal(decode_features(flat[1:].reshape(600, 24), wg, wu, wd), want)
    assert torch.equal(decode_features(x.float(), wg, wu, wd), want)  # rounded to the weights' type
    assert torch.equal(decode_features(x, wg.T.contiguous().T, wu, wd), want)
    assert torch.equal(decode_features(x[0], wg, wu, wd), want[0])


def test_gradient_through_float32_features():
    x, wg, wu, wd, dy = _inputs(50, 8, 16, 5, "bf16")
    a = x.float().requires_grad_(True)
    b = x.clone().requires_grad_(True)
    decode_features(a, wg, wu, wd).backward(dy)
    decode_features(b, wg, wu, wd).backward(dy)
    assert a.grad.dtype == torch.float32 and torch.equal(a.grad, b.grad.float())


def test_no_rows():
    x, wg, wu, wd, dy = _inputs(0, 8, 16, 5, "bf16")
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = decode_features(*leaves)
    assert y.shape == (0, 5)
    grads = torch.autograd.grad(y, leaves, dy)
    assert grads[0].shape == (0, 8) and all((g == 0).all() for g in grads[1:])


def test_one_bad_pixel_stays_alone():
    x, wg, wu, wd, _ = _inputs(300, 16, 32, 9, "bf16")
    want = decode_features(x, wg, wu, wd)
    x[200] = math.nan
    x[201, 0] = math.inf
    got = decode_features(x, wg, wu, wd)
    keep = [i for i in range(300) if i not in (200, 201)]
    assert torch.equal(got[keep], want[keep]) and got[200].isnan().all()


def test_large_gates_do_not_overflow():
    x = torch.tensor([[300.0], [-300.0], [0.0]], device="cuda", dtype=torch.bfloat16)
    one = torch.ones((1, 1), device="cuda", dtype=torch.bfloat16)
    for act in ("silu", "gelu"):
        a = x.clone().requires_grad_(True)
        y = decode_features(a, one, one, one, act)
        assert y[:, 0].tolist() == [90112.0, 0.0, 0.0]  # 300^2 rounded to bf16
        y.sum().backward()
        assert torch.isfinite(a.grad).all() and a.grad[1] == 0


def test_weights_changed_before_the_backward_are_refused():
    x, wg, wu, wd, dy = _inputs(10, 8, 16, 5, "bf16")
    wg.requires_grad_(True)
    y = decode_features(x, wg, wu, wd)
    with torch.no_grad():
        wg.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_captured_and_on_another_stream():
    x, wg, wu, wd, dy = _inputs(3000, 32, 96, 40, "bf16")
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]

    def work():
        y = decode_features(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(work())
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        x.copy_(_inputs(3000, 32, 96, 40, "bf16", seed=8)[0])
    want = work()
    for _ in range(2):
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_decoder_object_trains_float32_leaves():
    dec = FeatureDecoder.create(16, 32, 7, generator=torch.Generator(device="cuda").manual_seed(1))
    x = torch.randn((64, 16), device="cuda")
    y = dec(x)
    assert y.dtype == torch.bfloat16
    y.float().square().sum().backward()
    for p in dec.params.values():
        assert p.grad is not None and p.grad.dtype == torch.float32 and torch.isfinite(p.grad).all()


def test_first_call_of_a_thread():
    x, wg, wu, wd, dy = _inputs(300, 64, 64, 64, "bf16")
    size = nat.load().gs_decode_image_bytes(64, 64, 64)
    image = torch.empty((size,), device="cuda", dtype=torch.uint8)
    nat.call("gs_decode_prepare", wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 2, 64, 64, 64, image.data_ptr(), size,
             nat.stream())
    leaf = x.clone().requires_grad_(True)
    want = torch.autograd.grad(decode_features(leaf, wg, wu, wd), leaf, dy)[0]
    dx = torch.zeros_like(x)
    torch.cuda.synchronize()
    args = (x.data_ptr(), dy.data_ptr(), 2, 300, 64, 64, 64, 0, image.data_ptr(), size, dx.data_ptr(), None, None, None,
            None, 0, None)
    status = []
    t = threading.Thread(target=lambda: status.append(nat.load().gs_decode_backward(*args)))  # no CUDA call before it
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert status == [nat.GS_OK] and torch.equal(dx, want)


@pytest.mark.parametrize("f,d,c", [(256, 64, 152), (256, 64, 128), (256, 128, 256), (1100, 40, 24), (64, 128, 200)])
def test_many_tiles_of_every_plan(f, d, c):
    """Several tiles per SM, with weights resident beside one or more input stages, or streamed through three or two."""
    x, wg, wu, wd, dy = _inputs(60001, d, f, c, "bf16", seed=f + c)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = decode_features(*leaves)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    with torch.no_grad():
        want, tol = decode64(x, wg, wu, wd, "silu", dy), decode_tolerances(x, wg, wu, wd, "silu", dy)
        for g, w, t in zip(got, want, tol):
            _within(g, w, t)
    assert _wait_failures() == 0


@pytest.mark.parametrize("c", [1, 2, 7, 33, 64, 150, 161, 163, 192, 225, 255])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_outputs_at_any_element_leave_their_surroundings(c, offset):
    n, d, f = 1301, 24, 96
    x, wg, wu, wd, _ = _inputs(n, d, f, c, "bf16")
    want = decode_features(x, wg, wu, wd)
    lib = nat.load()
    size = lib.gs_decode_image_bytes(d, f, c)
    image = torch.empty((size,), device="cuda", dtype=torch.uint8)
    nat.call("gs_decode_prepare", wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 2, d, f, c, image.data_ptr(), size,
             nat.stream())
    flat = torch.full((n * c + 64,), 5.0, device="cuda", dtype=torch.bfloat16)
    nat.call("gs_decode_forward", x.data_ptr(), 2, n, d, f, c, 0, image.data_ptr(), size,
             flat.data_ptr() + 2 * offset, None, 0, nat.stream())
    assert torch.equal(flat[offset:offset + n * c].reshape(n, c), want)
    assert (flat[:offset] == 5.0).all() and (flat[offset + n * c:] == 5.0).all()


def test_offsets_beyond_32_bits():
    """More than 2^31 outputs, and gradients of them through padded rows: the last rows are those of a call of their own."""
    n, d, f, c = 14_400_003, 15, 64, 150
    _, wg, wu, wd, _ = _inputs(1, d, f, c, "bf16")
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty((n, d), device="cuda", dtype=torch.bfloat16).normal_(generator=g).requires_grad_(True)
    y = decode_features(x, wg, wu, wd)
    dy = y.detach() * 0.5
    dx, = torch.autograd.grad(y, x, dy)
    tail = x.detach()[-999:].clone().requires_grad_(True)
    own = decode_features(tail, wg, wu, wd)
    assert torch.equal(y.detach()[-999:], own.detach())
    assert torch.equal(dx[-999:], torch.autograd.grad(own, tail, dy[-999:])[0])


def test_weight_gradients_of_like_signed_sums():
    """One CTA sums 16384 equal tiles of positive terms: the sums must not drift away from 16384 times one tile's.

    A matrix instruction takes 2^-22.2 of a float32 accumulator away, 8 instructions a tile, sums of at most 256 tiles
    in a row: 256 * 8 / 2 * 2^-22.2 = 2.1e-4 < 2^-12, always in one direction.  Rounding the results to float16
    averages out over thousands of elements; a single one is off by half a step (2^-11) on either side besides."""
    d, f, c, times = 8, 4800, 8, 16384
    g = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda lo, hi, *s: (torch.rand(s, device="cuda", generator=g) * (hi - lo) + lo).half()  # noqa: E731
    x = rnd(0.5, 1.0, 128, d)
    leaves = [w.requires_grad_(True) for w in (rnd(0.1, 0.2, f, d), rnd(0.1, 0.2, f, d), rnd(0.1, 0.2, c, f))]
    dy = rnd(0.5, 1.5, 128, c) * 2.0 ** -10
    one = torch.autograd.grad(decode_features(x, *leaves), leaves, dy)
    all_ = torch.autograd.grad(decode_features(x.repeat(times, 1), *leaves), leaves, dy.repeat(times, 1))
    for a, b in zip(all_, one):
        off = a.double() / (times * b.double()) - 1.0
        assert abs(float(off.mean())) <= 2.0 ** -12 + 2.0 ** -16
        assert float(off.abs().max()) <= 2.0 ** -12 + 2 * 2.0 ** -11 + 2.0 ** -16
    assert _wait_failures() == 0


def test_weight_gradients_of_long_walks():
    """Every tile of a walk of more than 256 counts once: first, around the places where sums leave TMEM, last."""
    n, d, f, c = 128 * 1600 + 77, 40, 4800, 24
    x, wg, wu, wd, dy = _inputs(n, d, f, c, "bf16", seed=3)
    leaves = [w.requires_grad_(True) for w in (wg, wu, wd)]
    for tile in (0, 255, 256, 257, 511, 512, 1023, 1024, 1300, 1599, 1600):
        rows = slice(128 * tile, min(n, 128 * (tile + 1)))
        only = torch.zeros_like(dy)
        only[rows] = dy[rows]
        got = torch.autograd.grad(decode_features(x, *leaves), leaves, only)
        want = torch.autograd.grad(decode_features(x[rows], *leaves), leaves, dy[rows])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), tile
    assert _wait_failures() == 0


LONG = [(20001, 33, 70, 31), (40000, 64, 128, 150), (60001, 64, 256, 152), (60001, 64, 256, 128), (60001, 128, 256, 256),
        (60001, 40, 1100, 24), (60001, 128, 64, 200)]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,c", LONG)
def test_gradients_of_many_tiles_by_norm(n, d, f, c, dtype, act):
    """Bounds element by element grow with n, the gradients with its root: by norm, one lost tile shows."""
    x, wg, wu, wd, dy = _inputs(n, d, f, c, dtype, seed=n + f)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = decode_features(*leaves, act)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = decode64(*(t.detach() for t in leaves), act, dy)
    for a, b in zip(got, want):
        assert norm_off(a, b) <= decode_norm_bound(a.dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,c", LONG)
def test_every_tile_of_a_walk_counts_once(n, d, f, c, dtype):
    """All of dy but one tile is zero: the weights' gradients are those of a call on that tile alone (the other tiles
    add exact zeros), wherever it lies in its CTA's walk."""
    x, wg, wu, wd, dy = _inputs(n, d, f, c, dtype, seed=n + c)
    x = torch.randn((n, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)).to(x.dtype)
    leaves = [w.requires_grad_(True) for w in (wg, wu, wd)]
    y = decode_features(x, *leaves)
    chunks, tiles = (f + 63) // 64, (n + 127) // 128
    splits = 148 // chunks
    for tile in {0, 1, splits - 1, splits, 2 * splits + 1, tiles // 2, tiles - splits, tiles - 2, tiles - 1}:
        if not 0 <= tile < tiles:
            continue
        rows = slice(128 * tile, min(n, 128 * (tile + 1)))
        only = torch.zeros_like(dy)
        only[rows] = dy[rows]
        got = torch.autograd.grad(y, leaves, only, retain_graph=True)
        want = torch.autograd.grad(decode_features(x[rows], *leaves), leaves, dy[rows])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), tile
        assert all((w != 0).any() for w in want)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_one_feature_vector(dtype, act):
    x, wg, wu, wd, _ = _inputs(600, 24, 50, 11, dtype, seed=4)
    for row in (77, 599):  # covered pixels
        one = x[row]
        assert (one != 0).all()
        y = decode_features(one, wg, wu, wd, act)
        assert y.shape == (11,) and (y != 0).any()
        _within(y, decode64(one[None], wg, wu, wd, act)[0], decode_tolerances(one[None], wg, wu, wd, act)[0])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_large_gates_in_many_rows(act):
    """As many rows as the matrix kernels take: gates of 300 and -300, bf16, every output and gradient."""
    n = 300
    sign = torch.ones((n, 1), device="cuda", dtype=torch.bfloat16)
    sign[1::3], sign[2::3] = -1.0, 0.0
    x = (300.0 * sign).requires_grad_(True)
    one = lambda: torch.ones((1, 1), device="cuda", dtype=torch.bfloat16).requires_grad_(True)  # noqa: E731
    wg, wu, wd = one(), one(), one()
    y = decode_features(x, wg, wu, wd, act)
    grads = torch.autograd.grad(y, (x, wg, wu, wd), torch.ones_like(y))
    up = sign[:, 0] > 0
    assert (y[up, 0] == 90112.0).all() and (y[~up] == 0).all()  # 300^2 rounded to bf16
    # up: h = 90000 (bf16 90112), dg = u = 300, du = 300; below and at zero nothing is left
    assert (grads[0][up] == 600.0).all() and (grads[0][~up] == 0).all()
    # Sums of 100 rows are whole numbers below 2^24, exact in 32 bits, and rounded once: 9000000 lies between 137 and
    # 138 steps of 2^16 (bf16 has 8 bits), nearer the first, 8978432, off by 2.4e-3 <= 2^-8.
    rows = int(up.sum())
    want = [300.0 * 300.0 * rows, 300.0 * 300.0 * rows, 90112.0 * rows]
    for g, w in zip(grads[1:], want):
        assert float(g.detach()) == float(torch.tensor(w).bfloat16())
