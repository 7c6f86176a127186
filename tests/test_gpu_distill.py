"""Distillation loss and teacher cache on the GPU against plain 64-bit forms."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch

from feature_helpers import DTYPES, distill64, distill_tolerance, half_step, read64, write64
from mlx3d_b200 import _native as nat
from mlx3d_b200.losses import distill_loss, distill_loss_and_grad
from mlx3d_b200.staging import TeacherCache

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(n, c, k, dtype, vdtype="fp16", seed=0):
    g = _gen(seed)
    s = (torch.randn((n, c), device="cuda", generator=g) * 2).to(DTYPES[dtype])
    v = (torch.randn((n, k), device="cuda", generator=g) * 2 + 3).to(DTYPES[vdtype])
    i = torch.randint(-1, c + 1, (n, k), device="cuda", generator=g, dtype=torch.int32)  # absent and repeated ones
    w = torch.rand((n,), device="cuda", generator=g)
    return s, v, i, w


def _check(s, v, i, w, t, loss, grad, g_row=1.0):
    want_l, want_g = distill64(s, v, i, t, w)
    tol_l, rel = distill_tolerance(s, v, t, v.shape[-1])
    ww = torch.ones(s.shape[:-1], device="cuda", dtype=torch.float64) if w is None else w.double()
    tol = ww * t * t * tol_l + 2.0 ** -22 * want_l.abs()
    assert ((loss.double() - want_l).abs() <= tol).all()
    if grad is not None:
        # q and p are at most 1 and each off by rel: 2 rel (w T); factors and the final rounding
        want_g = want_g * g_row
        size = (ww * t * g_row if not isinstance(g_row, float) else ww * t * abs(g_row))[..., None]
        tiny = 2.0 ** -25 if s.dtype == torch.float16 else 0.0  # half a subnormal step
        tol = size * 2 * rel[..., None] + want_g.abs() * (half_step(s.dtype) + 2.0 ** -21) + tiny
        assert ((grad.double() - want_g).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,c,k,t", [
    (1, 1, 1, 1.0), (1, 2, 3, 1.0), (3, 7, 1, 2.0), (257, 20, 5, 1.0), (64, 32, 32, 0.5), (1000, 133, 8, 2.0),
    (515, 150, 8, 4.0), (130, 151, 33, 1.0), (33, 1024, 64, 1.0), (17, 1201, 256, 1.0), (9, 4099, 16, 2.0),
    (5, 32001, 32, 1.0), (2, 70001, 7, 1.0), (4097, 16, 4, 1.0), (2049, 8, 8, 1.0),
])
def test_distill_matches_the_definition(n, c, k, t, dtype):
    vdtype = {"fp32": "fp32", "fp16": "fp16", "bf16": "bf16"}[dtype]
    s, v, i, w = _inputs(n, c, k, dtype, vdtype, seed=n + c)
    loss, grad = distill_loss_and_grad(s, (v, i), temperature=t, weight=w, reduction="none")
    assert loss.dtype == torch.float32 and grad.dtype == s.dtype and grad.shape == s.shape
    _check(s, v, i, w, t, loss, grad)
    # the loss alone, and autograd's gradient, are the same numbers
    leaf = s.clone().requires_grad_(True)
    alone = distill_loss(leaf, (v, i), temperature=t, weight=w, reduction="none")
    assert torch.equal(alone, loss)
    alone.backward(torch.ones_like(alone))
    assert torch.equal(leaf.grad, grad)


@pytest.mark.parametrize("k", [1, 3, 8, 9, 40])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_every_split_of_a_row(dtype, k):
    """Class counts on both sides of every split; odd ones start every second row inside a pair of classes."""
    for c in (1, 2, 3, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 97, 127, 128, 129, 159, 160, 161, 255, 257, 509, 510, 513,
              1017, 1018, 1021, 1022, 1025, 1533, 1534, 1537, 2041, 2043):
        s, v, i, w = _inputs(75, c, k, dtype, dtype, seed=c)
        loss, grad = distill_loss_and_grad(s, (v, i), temperature=1.0, weight=w, reduction="none")
        _check(s, v, i, w, 1.0, loss, grad)


@pytest.mark.parametrize("c", [3, 31, 133, 301, 1201])
def test_odd_rows_do_not_see_their_neighbours(c):
    for dtype in ("fp32", "bf16"):
        s, v, i, w = _inputs(41, c, 5, dtype, dtype)
        want_l, want_g = distill_loss_and_grad(s, (v, i), weight=w, reduction="none")
        s[1::2] = math.nan
        loss, grad = distill_loss_and_grad(s, (v, i), weight=w, reduction="none")
        assert torch.equal(loss[::2], want_l[::2]) and torch.equal(grad[::2], want_g[::2])
        here = ((i >= 0) & (i < c)).any(1)[1::2]
        assert loss[1::2][here].isnan().all() and (loss[1::2][~here] == 0).all()


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reductions_and_cotangents(reduction):
    n, c, k = 1031, 77, 6
    s, v, i, w = _inputs(n, c, k, "fp32")
    rows, _ = distill64(s, v, i, 2.0, w)
    div = n if reduction == "mean" else 1
    leaf = s.clone().requires_grad_(True)
    loss = distill_loss(leaf, (v, i), 2.0, w, reduction)
    tol_l, _ = distill_tolerance(s, v, 2.0, k)
    got = float(loss.detach())
    assert abs(got - float(rows.sum() / div)) <= float((w * 4.0 * tol_l).sum() / div) + 1e-6 * got
    (loss * -3.0).backward()
    _check(s, v, i, w, 2.0, distill_loss(s, (v, i), 2.0, w, "none"), leaf.grad, g_row=-3.0 / div)
    l2, g2 = distill_loss_and_grad(s, (v, i), 2.0, w, reduction)
    assert torch.equal(l2, loss.detach())
    _check(s, v, i, w, 2.0, distill_loss(s, (v, i), 2.0, w, "none"), g2, g_row=1.0 / div)


def test_per_row_cotangents_and_no_weight():
    s, v, i, _ = _inputs(300, 41, 5, "bf16", "bf16")
    leaf = s.clone().requires_grad_(True)
    loss = distill_loss(leaf, (v, i), reduction="none")
    g = torch.linspace(0.0, 2.0, 300, device="cuda")
    loss.backward(g)
    _check(s, v, i, None, 1.0, loss.detach(), leaf.grad, g_row=g.double()[:, None])


def test_images_strides_and_unaligned_bases():
    s, v, i, w = _inputs(24 * 20, 30, 4, "fp32")
    want = distill_loss(s, (v, i), weight=w, reduction="none")
    img = s.reshape(24, 20, 30)
    got = distill_loss(img, (v.reshape(24, 20, 4), i.reshape(24, 20, 4)), weight=w.reshape(24, 20), reduction="none")
    assert got.shape == (24, 20) and torch.equal(got.reshape(-1), want)
    wide = torch.zeros((480, 37), device="cuda")
    wide[:, 3:33] = s
    assert torch.equal(distill_loss(wide[:, 3:33], (v, i), weight=w, reduction="none"), want)
    for dtype in ("fp32", "fp16", "bf16"):  # contiguous, but off every vector boundary
        x = s.to(DTYPES[dtype])
        flat = torch.zeros((480 * 30 + 1,), device="cuda", dtype=x.dtype)
        flat[1:] = x.reshape(-1)
        off = flat[1:].reshape(480, 30)
        a = distill_loss_and_grad(x, (v, i), weight=w)
        b = distill_loss_and_grad(off, (v, i), weight=w)
        tol = 2.0 ** -20 * float(a[0].abs()) if dtype == "fp32" else 2.0 ** -18 * float(a[0].abs())
        assert abs(float(a[0]) - float(b[0])) <= tol
        assert torch.allclose(a[1].float(), b[1].float(), rtol=2 * half_step(x.dtype) + 2.0 ** -18, atol=1e-9)


def test_masked_values():
    inf, low = math.inf, torch.finfo(torch.float32).min
    s = torch.tensor([[0.0, 1.0, 2.0, -1.0]] * 8, device="cuda")
    s[3, 1] = -inf  # a student class masked out, not among the teacher's
    s[4, 0] = -inf  # ... among the teacher's: infinite loss, finite gradient
    s[5, 1] = low
    v = torch.tensor([[1.0, 0.0]] * 8, device="cuda")
    i = torch.tensor([[0, 2]] * 8, device="cuda", dtype=torch.int32)
    i[0] = -1  # nothing left
    v[1] = -inf  # nothing left
    v[2, 1] = -inf  # one entry left
    v[6] = low  # two equal entries
    v[7, 1] = low  # an entry with probability 0
    i[7, 1] = 3
    s[7, 3] = -inf  # ... on a masked class: contributes nothing
    loss, grad = distill_loss_and_grad(s, (v, i), reduction="none")
    want_l, want_g = distill64(s, v, i)
    assert loss[4] == inf
    keep = [0, 1, 2, 3, 5, 6, 7]
    assert torch.allclose(loss[keep].double(), want_l[keep], rtol=1e-6, atol=1e-6)
    assert torch.allclose(grad.double(), want_g, rtol=1e-6, atol=1e-6)
    assert (loss[:2] == 0).all() and (grad[:2] == 0).all()
    # NaN stays NaN in its row only
    s[3, 0] = math.nan
    v[2, 0] = math.nan
    loss, grad = distill_loss_and_grad(s, (v, i), reduction="none")
    assert loss[[2, 3]].isnan().all() and not loss[[0, 1, 5, 6, 7]].isnan().any()
    assert not grad[[0, 1, 5, 6, 7]].isnan().any()


def test_no_rows():
    s = torch.zeros((0, 5), device="cuda", requires_grad=True)
    v, i = torch.zeros((0, 2), device="cuda"), torch.zeros((0, 2), device="cuda", dtype=torch.int32)
    loss = distill_loss(s, (v, i), reduction="sum")
    assert float(loss) == 0.0
    loss.backward()
    assert s.grad.shape == (0, 5)
    assert distill_loss(s, (v, i), reduction="none").shape == (0,)


def test_wide_index_types():
    s, v, i, _ = _inputs(50, 11, 3, "fp32")
    want = distill_loss(s, (v, i))
    assert torch.equal(distill_loss(s, (v, i.short())), want)
    far = i.long()
    far[i < 0] = (1 << 33) + 2  # 2 if cut to 32 bits
    far[i >= 11] = -(1 << 40)
    assert torch.equal(distill_loss(s, (v, far)), want)


# ---------------------------------------------------------------- the cache
def _cache_logits(n, c, dtype, seed):
    g = _gen(seed)
    z = (torch.randn((n, c), device="cuda", generator=g) * 3).to(DTYPES[dtype])
    return z


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,c,k", [
    (1, 1, 1), (1, 5, 8), (3, 2, 2), (100, 20, 5), (257, 32, 32), (300, 33, 31), (1000, 150, 8), (515, 133, 7),
    (64, 1201, 32), (31, 4096, 16), (9, 32767, 32), (4100, 64, 3), (70, 257, 1),
    # one thread per row: many rows
    (4736, 1, 1), (5003, 150, 8), (4801, 133, 5), (4999, 128, 16), (4750, 7, 16), (4736, 300, 12), (5000, 64, 2),
    (4737, 384, 9), (4900, 20, 20),
])
def test_write_and_read_match_the_definition(n, c, k, dtype, bits):
    z = _cache_logits(n, c, dtype, n * 7 + c)
    if c > 4:
        z[:, 1] = -math.inf
        z[:, 3] = torch.finfo(z.dtype).min
        z[n // 2] = -math.inf  # a row with nothing
        z[n // 3, 2:] = math.nan  # a row with one usable class
        z[0, 2] = math.inf
    cache = TeacherCache(n + 5, k, c, bits=bits)
    before = cache.records.clone()
    cache.write(3, z)
    values, index = cache.read(slice(3, 3 + n))
    first, scale, want_i, code = write64(z, k, bits)
    assert torch.equal(index.cpu(), want_i)
    assert torch.equal(values.cpu(), read64(first, scale, want_i, code))  # the codes exactly
    assert torch.equal(cache.records[:3], before[:3]) and torch.equal(cache.records[3 + n:], before[3 + n:])


def test_write_equal_logits_take_the_lowest_indices():
    z = torch.zeros((4, 100), device="cuda")
    z[1] = -0.0
    z[2, ::3] = -0.0
    z[3, 50:] = 1.0
    cache = TeacherCache(4, 6, 100)
    cache.write(0, z)
    values, index = cache.read(slice(None))
    assert index[:3].tolist() == [[0, 1, 2, 3, 4, 5]] * 3
    assert index[3].tolist() == [50, 51, 52, 53, 54, 55]
    assert (values[:3] == 0).all() and (values[3] == 1).all()


def test_write_extreme_ranges():
    big = torch.finfo(torch.float32).max
    z = torch.tensor([[big, -1e38, 0.0, 5.0], [1e-44, 0.0, -1e-44, -3e-44], [big, big, big, big],
                      [3.0, 3.0, 3.0, 2.0]], device="cuda")
    for bits in (8, 4):
        cache = TeacherCache(4, 4, 4, bits=bits)
        cache.write(0, z)
        values, index = cache.read(slice(None))
        first, scale, want_i, code = write64(z, 4, bits)
        assert torch.equal(index.cpu(), want_i)
        assert torch.equal(values.cpu(), read64(first, scale, want_i, code))


def test_write_a_span_beyond_float32():
    # last - first overflows; the second entry lies 0.9 of a step below the first
    z = torch.tensor([[3.3e38, 3.3e38 - 0.9 * 6.6e38 / 255, 1e38, -3.3e38]], device="cuda")
    for rows in (1, 5000):  # both ways of writing
        cache = TeacherCache(rows, 4, 4)
        cache.write(0, z.repeat(rows, 1))
        values, index = cache.read(slice(rows - 1, rows))
        first, scale, want_i, code = write64(z, 4, 8)
        assert code[0, 1] == 1 and torch.equal(index.cpu(), want_i)
        assert torch.equal(values.cpu(), read64(first, scale, want_i, code))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_write_subnormals_and_signed_zeros_in_order(dtype):
    """Even rows of 16-bit logits in their many: the quick path has to order what rounds and flushes easily."""
    t = torch.finfo(DTYPES[dtype])
    tiny = t.smallest_normal * t.eps
    line = torch.tensor([-0.0, 0.0, tiny, -tiny, 2 * tiny, t.min, t.max, -t.smallest_normal, t.smallest_normal, -1.0],
                        device="cuda", dtype=DTYPES[dtype])
    assert (line[2] > 0) and (line[4] > line[2])
    z = line.repeat(5000, 1)
    cache = TeacherCache(5000, 9, 10)
    cache.write(0, z)
    _, index = cache.read(slice(None))
    assert (index == torch.tensor([6, 8, 4, 2, 0, 1, 3, 7, 9], device="cuda")).all()


@pytest.mark.parametrize("k,bits", [(7, 8), (8, 8), (8, 4), (16, 8), (16, 4), (32, 8), (32, 4), (3, 4), (1, 8), (20, 4)])
def test_read_rows_in_any_order(k, bits):
    z = _cache_logits(500, 40, "fp32", 1)
    z[:100, 5:] = -math.inf  # rows with absent entries
    cache = TeacherCache(500, k, 40, bits=bits)
    cache.write(0, z)
    all_v, all_i = cache.read(slice(None))
    rows = torch.tensor([[3, 499, 3], [0, -1, 500], [250, 1 << 40, -(1 << 50)]], device="cuda")
    v, i = cache.read(rows)
    assert v.shape == (3, 3, k)
    assert torch.equal(all_v.cpu(), read64(*write64(z, k, bits)))
    inside = (rows >= 0) & (rows < 500)
    assert torch.equal(v[inside], all_v[rows[inside]]) and torch.equal(i[inside], all_i[rows[inside]])
    assert (v[~inside] == -math.inf).all() and (i[~inside] == -1).all()
    v32, i32 = cache.read(rows[:2].int())
    assert torch.equal(v32, v[:2]) and torch.equal(i32, i[:2])
    assert cache.read(slice(7, 7))[0].shape == (0, k)
    assert cache.read(rows[:0])[0].shape == (0, 3, k)


def test_cache_starts_empty_and_saves():
    cache = TeacherCache(10, 3, 9, bits=4)
    v, i = cache.read(slice(None))
    assert (v == -math.inf).all() and (i == -1).all()
    cache.write(2, _cache_logits(4, 9, "bf16", 2).reshape(2, 2, 9))
    other = TeacherCache(10, 3, 9, bits=4)
    other.load_state_dict(cache.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(cache.read(slice(None)), other.read(slice(None))))
    with pytest.raises(ValueError, match="bits"):
        TeacherCache(10, 3, 9, bits=8).load_state_dict(cache.state_dict())
    with pytest.raises(ValueError, match="shape"):
        TeacherCache(11, 3, 9, bits=4).load_state_dict(cache.state_dict())


def test_cache_argument_checks():
    cache = TeacherCache(10, 3, 9)
    z = torch.zeros((4, 9), device="cuda")
    with pytest.raises(ValueError, match="outside"):
        cache.write(7, z)
    with pytest.raises(ValueError, match="outside"):
        cache.write(-1, z)
    with pytest.raises(ValueError, match="shape"):
        cache.write(0, z[:, :8])
    with pytest.raises(ValueError, match="CUDA"):
        cache.write(0, z.cpu())
    for bad in (slice(0, 11), slice(-2, 3), slice(5, 2)):
        with pytest.raises(ValueError, match="outside"):
            cache.read(bad)
    with pytest.raises(ValueError, match="step"):
        cache.read(slice(0, 4, 2))
    with pytest.raises(TypeError):
        cache.read([1, 2])
    with pytest.raises(TypeError):
        cache.read(torch.ones(3, device="cuda"))
    with pytest.raises(ValueError, match="rows"):
        distill_loss(z, cache.at(slice(0, 3)))
    with pytest.raises(ValueError, match="classes"):
        distill_loss(torch.zeros((3, 8), device="cuda"), cache.at(slice(0, 3)))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,c,k,dtype", [(1, 5, 2, "fp32"), (300, 20, 5, "fp32"), (999, 133, 8, "fp16"),
                                         (65, 1201, 32, "bf16"), (3, 20011, 17, "fp32")])
def test_loss_from_the_cache_is_the_loss_of_what_it_reads(n, c, k, dtype, bits):
    cache = TeacherCache(n + 40, k, c, bits=bits)
    cache.write(40, _cache_logits(n, c, "fp32", 9))  # the first 40 rows stay empty
    rows = torch.randint(-2, n + 43, (n,), device="cuda", generator=_gen(4))
    s = _cache_logits(n, c, dtype, 11)
    for at in (rows, slice(40, 40 + n)):
        v, i = cache.read(at)
        want = distill_loss_and_grad(s, (v, i), 2.0, reduction="none")
        got = distill_loss_and_grad(s, cache.at(at), 2.0, reduction="none")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        _check(s, v, i, None, 2.0, *got)


def test_backward_refuses_rows_written_since_the_loss():
    cache = TeacherCache(8, 2, 5)
    cache.write(0, torch.randn((8, 5), device="cuda"))
    s = torch.randn((8, 5), device="cuda", requires_grad=True)
    loss = distill_loss(s, cache.at(slice(0, 8)))
    cache.write(0, torch.randn((8, 5), device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_captured_and_on_another_stream():
    z, s = _cache_logits(2000, 60, "fp32", 5), _cache_logits(2000, 60, "fp32", 6)
    cache = TeacherCache(2000, 8, 60)

    def work():
        cache.write(0, z)
        return distill_loss_and_grad(s, cache.at(slice(None)), 2.0)

    want = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
        graphs, outs = [], []
        for _ in range(2):  # two graphs, replayed in turn
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(work())
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    z.copy_(_cache_logits(2000, 60, "fp32", 7))
    want = work()
    for _ in range(2):
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_kernels_are_counted():
    lib = nat.load()
    before = lib.gs_kernel_launch_count()
    cache = TeacherCache(4, 2, 5)
    cache.write(0, torch.zeros((4, 5), device="cuda"))
    assert lib.gs_kernel_launch_count() > before


def test_offsets_beyond_32_bits():
    """More than 2^31 logits: the last rows are those of a call of their own."""
    n, c, k = 14_400_003, 150, 8
    s = torch.empty((n, c), device="cuda", dtype=torch.bfloat16).normal_(generator=_gen(1))
    cache = TeacherCache(n, k, c)
    cache.write(0, s)
    v, i = cache.read(slice(n - 999, n))
    own = TeacherCache(999, k, c)
    own.write(0, s[-999:])
    want_v, want_i = own.read(slice(None))
    assert torch.equal(v, want_v) and torch.equal(i, want_i)
    picked = torch.arange(n - 999, n, device="cuda")
    assert torch.equal(cache.read(picked)[1], want_i)
    s.mul_(-0.5)  # not the teacher's own logits
    loss, grad = distill_loss_and_grad(s, cache.at(slice(0, n)), 2.0, reduction="none")
    want_l, want_g = distill_loss_and_grad(s[-999:], own.at(slice(0, 999)), 2.0, reduction="none")
    assert torch.equal(loss[-999:], want_l) and torch.equal(grad[-999:], want_g)


@pytest.mark.parametrize("c", [300, 700, 1201, 2041, 5001])
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_long_rows_off_their_vectors(dtype, c):
    """Logits one element off a 16-byte boundary, the gradient on one."""
    n, k = 37, 9
    s, v, i, w = _inputs(n, c, k, dtype, dtype, seed=c)
    flat = torch.zeros((n * c + 1,), device="cuda", dtype=s.dtype)
    flat[1:] = s.reshape(-1)
    off = flat[1:].reshape(n, c)
    loss, grad = distill_loss_and_grad(off, (v, i), weight=w, reduction="none")
    assert off.data_ptr() % 16 and grad.data_ptr() % 16 == 0
    _check(s, v, i, w, 1.0, loss, grad)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,c", [(1_000_003, 20), (300_001, 133), (300_001, 150), (150_001, 300)])
def test_gradients_off_their_vectors(n, c, dtype):
    """Logits on a 16-byte boundary, the gradient one element off one, several tiles a warp: what is written over a
    tile must not meet the copy that fills its buffer next."""
    k = 4
    s, v, i, w = _inputs(n, c, k, dtype, dtype, seed=c)
    want_l, want_g = distill_loss_and_grad(s, (v, i), weight=w, reduction="none")
    flat = torch.full((n * c + 64,), 5.0, device="cuda", dtype=s.dtype)
    out = flat[1:1 + n * c].view(n, c)
    loss = torch.empty((n,), device="cuda")
    teacher = nat.GsTeacher(v.data_ptr(), i.data_ptr(), None, None, 0, 0, nat.DTYPES[v.dtype], k, 0)
    for _ in range(3):
        out.zero_()
        assert s.data_ptr() % 16 == 0 and out.data_ptr() % 16 == s.element_size()
        nat.call("gs_distill", s.data_ptr(), nat.DTYPES[s.dtype], n, c, ctypes.byref(teacher), 1.0, w.data_ptr(), 1.0,
                 None, 1, loss.data_ptr(), None, out.data_ptr(), None, 0, nat.stream())
        assert torch.equal(loss, want_l) and torch.equal(out, want_g)
    assert flat[0] == 5.0 and (flat[1 + n * c:] == 5.0).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows", [3, 5001])  # both ways of writing
def test_codes_next_to_a_border_by_far_less_than_64_bits_hold(rows, dtype, bits):
    """The quotients of the exact differences decide: halves go to the even code, less than a half does not."""
    tiny = {"fp32": 2.0 ** -149, "bf16": 2.0 ** -133}[dtype]
    line = []
    for big in (1.0, 2.0 ** 127, 2.0 ** -60):
        for mid in (0.0, tiny, -tiny, 2.0 ** -100, -(2.0 ** -100)):
            line.append([big, mid, -big])
            line.append([big, mid + big / 2, -big])  # (on the code's own value: far from a border)
    z = torch.tensor(line, device="cuda", dtype=torch.float64).to(DTYPES[dtype])
    z = z.repeat((rows + len(line) - 1) // len(line), 1)[:rows] if rows > 3 else z
    cache = TeacherCache(z.shape[0], 3, 3, bits=bits)
    cache.write(0, z)
    levels = 2 ** bits - 1
    at = 8 + 2 * 3
    codes = cache.records[:, at:at + (3 * bits + 7) // 8].cpu()
    for r in range(min(z.shape[0], len(line))):
        first, mid, last = (Fraction(float(v)) for v in z[r].cpu())
        want = round((first - mid) * levels / (first - last))  # (halves to even)
        got = int(codes[r, 1]) if bits == 8 else int(codes[r, 0]) >> 4
        assert got == want, (r, z[r].tolist())


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows", [2000, 5000])  # both ways of writing
def test_write_the_whole_range_of_float32(rows, bits):
    """From next to the largest float32 to next to the lowest: nothing that is kept reads as absent."""
    big = torch.finfo(torch.float32).max
    z = torch.zeros((rows, 3), device="cuda")
    z[:, 0] = (big - torch.arange(rows, device="cuda", dtype=torch.float64) * 2.0 ** 105).float()
    z[:, 2] = -(big - 2.0 ** 104)  # the lowest value that is kept
    cache = TeacherCache(rows, 3, 3, bits=bits)
    cache.write(0, z)
    values, index = cache.read(slice(None))
    assert (index == torch.arange(3, device="cuda")).all()
    assert torch.equal(values[:, 0], z[:, 0])
    # the step's half a rounding (or one, where it was taken down), 2^bits - 1 times; the value's own half
    tol = z[:, 0].double() * 2 * (2.0 ** -23 + 2.0 ** -24)
    assert ((values[:, 2].double() - z[:, 2].double()).abs() <= tol).all()
    assert torch.isfinite(values).all()


@pytest.mark.parametrize("t", [1e-18, 1e-9, 1e9, 1e18])
@pytest.mark.parametrize("c,k", [(20, 5), (401, 9), (5001, 40)])
def test_temperatures_far_from_one(c, k, t):
    s, v, i, w = _inputs(70, c, k, "fp32", "fp32", seed=c)
    t = float(torch.tensor(t))  # as the kernels have it
    loss, grad = distill_loss_and_grad(s * t, (v * t, i), temperature=t, weight=w, reduction="none")
    _check(s * t, v * t, i, w, t, loss, grad)


def test_cache_made_in_inference_mode():
    """The teacher runs in inference mode, the student trains: the cache serves both."""
    s = torch.randn((6, 9), device="cuda", requires_grad=True)
    with torch.inference_mode():
        cache = TeacherCache(6, 3, 9)
        cache.write(0, torch.randn((6, 9), device="cuda", generator=_gen(1)))
        saved = cache.state_dict()
    want, want_g = distill_loss_and_grad(s.detach(), cache.read(slice(None)))
    loss = distill_loss(s, cache.at(slice(0, 6)))
    loss.backward()
    assert torch.equal(loss.detach(), want) and torch.equal(s.grad, want_g)
    loss = distill_loss(s, cache.at(slice(0, 6)))
    with torch.inference_mode():
        cache.load_state_dict(saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dtype,sizes", [
    ("fp32", (319, 320, 321, 508, 509, 510, 511, 512, 1020, 1021, 1022, 1532, 1533, 1534)),
    ("fp16", (511, 512, 513, 639, 640, 641, 1016, 1017, 1018, 2040, 2041, 2042, 3063, 3064, 3065, 3066, 3067)),
    ("bf16", (511, 512, 513, 640, 641, 1017, 1018, 2041, 2042, 3064, 3065, 3066)),
])
def test_both_sides_of_every_limit_of_long_rows(dtype, sizes, off):
    """The last and first row lengths of the tiles, of 4, 8 and 12 units a lane, of a block a row; logits on a 16-byte
    boundary and one element off it."""
    for c in sizes:
        n, k = 70, 9
        s, v, i, w = _inputs(n, c, k, dtype, dtype, seed=c)
        if off:
            flat = torch.zeros((n * c + 1,), device="cuda", dtype=s.dtype)
            flat[1:] = s.reshape(-1)
            s = flat[1:].view(n, c)
        loss, grad = distill_loss_and_grad(s, (v, i), weight=w, reduction="none")
        _check(s, v, i, w, 1.0, loss, grad)
        alone = distill_loss(s, (v, i), weight=w, reduction="none")
        assert torch.equal(alone, loss)


@pytest.mark.parametrize("k", [128, 255, 256])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_more_teacher_entries_than_classes(dtype, k):
    """As many entries as there may be, most classes several times: the largest tiles, one warp a block."""
    for c in (1, 5, 16, 17, 32, 33, 64, 96, 150, 256, 300, 700, 4001):
        n = 100
        s, v, i, w = _inputs(n, c, k, dtype, dtype, seed=c + k)
        loss, grad = distill_loss_and_grad(s, (v, i), weight=w, reduction="none")
        want_l, want_g = distill64(s, v, i, 1.0, w)
        tol_l, rel = distill_tolerance(s, v, 1.0, k)
        # the entries of one class are added one by one, and the row's on as few as one lane: k roundings more
        tol_l, rel = tol_l + 2.0 ** -24 * k * (1 + tol_l / rel), rel + 2.0 ** -24 * k
        assert ((loss.double() - want_l).abs() <= w * tol_l + 2.0 ** -22 * want_l.abs()).all()
        tol = (w * 2 * rel)[:, None] + want_g.abs() * (half_step(s.dtype) + 2.0 ** -21)
        assert ((grad.double() - want_g).abs() <= tol).all()
