"""Feature-field operators without a GPU: refusals of the Python entry points
and of the C ABI, and the plain forms the GPU tests compare against."""

import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from feature_helpers import DTYPES, decode64, decode_norm_bound, distill64, norm_off
from mlx3d_b200 import _native as nat
from mlx3d_b200.losses import distill_loss, distill_loss_and_grad
from mlx3d_b200.splatting import FeatureDecoder, decode_features
from mlx3d_b200.staging import TeacherCache


def _teacher(n=3, k=2):
    return torch.zeros(n, k), torch.zeros(n, k, dtype=torch.int32)


@pytest.mark.parametrize("fn", [distill_loss, distill_loss_and_grad])
def test_distill_refusals(fn):
    s = torch.zeros(3, 5)
    v, i = _teacher()
    with pytest.raises(ValueError, match="CUDA"):
        fn(s, (v, i))
    with pytest.raises(ValueError, match="reduction"):
        fn(s, (v, i), reduction="batchmean")
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            fn(s, (v, i), temperature=t)
    with pytest.raises(ValueError, match="shape"):
        fn(torch.zeros(3, 0), (v, i))
    with pytest.raises(ValueError, match="shape"):
        fn(s, (v[:2], i[:2]))
    with pytest.raises(ValueError, match="shape"):
        fn(s, (v, i[:, :1]))
    with pytest.raises(ValueError, match="entries"):
        fn(s, (v[:, :0], i[:, :0]))
    with pytest.raises(ValueError, match="entries"):
        fn(s, _teacher(3, nat.GS_TEACHER_MAX_K + 1))
    with pytest.raises(TypeError, match="index"):
        fn(s, (v, i.float()))
    with pytest.raises(TypeError, match="teacher"):
        fn(s, v)
    with pytest.raises(ValueError, match="weight"):
        fn(s, (v, i), weight=torch.ones(2))
    with pytest.raises(ValueError, match="at least one row"):
        fn(s[:0], (v[:0], i[:0]))
    with pytest.raises(TypeError, match="floating"):
        fn(s.int(), (v, i))


def test_teacher_cache_refusals():
    for bad in (dict(k=0), dict(k=33), dict(num_classes=0), dict(num_classes=32768), dict(bits=2), dict(rows=-1)):
        with pytest.raises(ValueError):
            TeacherCache(**{**dict(rows=4, k=8, num_classes=20), **bad})
    with pytest.raises(ValueError, match="CUDA"):
        TeacherCache(4, 8, 20, device="cpu")


def _native_teacher(**kw):
    t = nat.GsTeacher(None, None, None, None, 0, 0, 0, 4, 8)
    for name, v in kw.items():
        setattr(t, name, v)
    return t


def test_native_distill_rejects_bad_arguments_before_the_device():
    lib = nat.load()

    def call(dtype=0, n=2, classes=5, t=None, temp=1.0, loss=None, ws=0):
        t = _native_teacher() if t is None else t
        return lib.gs_distill(None, dtype, n, classes, ctypes.byref(t), temp, None, 1.0, None, 0, None, loss, None,
                              None, ws, None)

    assert call(dtype=3) == nat.GS_ERR_INVALID_ARG
    assert call(n=-1) == nat.GS_ERR_INVALID_ARG
    assert call(classes=0) == nat.GS_ERR_INVALID_ARG
    assert call(classes=1 << 31) == nat.GS_ERR_INVALID_ARG
    assert call(classes=nat.GS_DISTILL_MAX_CLASSES + 1) == nat.GS_ERR_INVALID_ARG  # 16 bytes of a row stay countable
    assert b"classes" in lib.gs_last_error()
    assert call(t=_native_teacher(k=0)) == nat.GS_ERR_INVALID_ARG
    assert call(t=_native_teacher(k=33)) == nat.GS_ERR_INVALID_ARG  # a cache's limit
    assert call(t=_native_teacher(bits=0, k=257)) == nat.GS_ERR_INVALID_ARG
    assert call(t=_native_teacher(bits=5)) == nat.GS_ERR_INVALID_ARG
    assert call(t=_native_teacher(records=8, n_records=4)) == nat.GS_ERR_INVALID_ARG
    assert b"aligned" in lib.gs_last_error()
    for temp in (0.0, -2.0, math.nan, math.inf, 1e-39):
        assert call(temp=temp) == nat.GS_ERR_INVALID_ARG
        assert b"temperature" in lib.gs_last_error()
    assert call() == nat.GS_ERR_INVALID_ARG  # NULL logits
    assert call(t=_native_teacher(bits=0)) == nat.GS_ERR_INVALID_ARG
    assert b"NULL" in lib.gs_last_error()
    assert call(n=0, loss=16, ws=8) == nat.GS_ERR_CAPACITY
    assert lib.gs_distill(None, 0, 2, 5, None, 1.0, None, 1.0, None, 0, None, None, None, None, 0,
                          None) == nat.GS_ERR_INVALID_ARG


def test_native_cache_rejects_bad_arguments_before_the_device():
    lib = nat.load()
    assert lib.gs_teacher_record_bytes(8, 8) == 32
    assert lib.gs_teacher_record_bytes(32, 4) == 96
    assert [lib.gs_teacher_record_bytes(k, b) for k, b in ((0, 8), (33, 8), (8, 3))] == [0, 0, 0]

    def write(dtype=0, n=2, classes=5, records=16, held=4, first=0, k=4, bits=8):
        return lib.gs_teacher_write(None, dtype, n, classes, records, held, first, k, bits, None)

    for bad in (dict(dtype=9), dict(n=-1), dict(classes=0), dict(classes=32768), dict(records=8), dict(k=0),
                dict(k=33), dict(bits=16), dict(first=-1), dict(first=3), dict(first=5, n=0), dict(records=None),
                dict(n=1 << 62, held=4)):
        assert write(**bad) == nat.GS_ERR_INVALID_ARG, bad
    assert write() == nat.GS_ERR_INVALID_ARG  # NULL logits
    assert write(n=0) == nat.GS_OK

    def read(n=2, records=16, held=4, k=4, bits=8):
        return lib.gs_teacher_read(records, held, None, 0, n, k, bits, None, None, None)

    for bad in (dict(n=-1), dict(records=24), dict(k=0), dict(k=40), dict(bits=0), dict(held=-2), {}):
        assert read(**bad) == nat.GS_ERR_INVALID_ARG, bad
    assert read(n=0) == nat.GS_OK


def test_plain_distillation_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    s = torch.randn(6, 9, generator=g, dtype=torch.float64)
    v = torch.randn(6, 4, generator=g, dtype=torch.float64)
    i = torch.randint(-1, 10, (6, 4), generator=g)  # absent ones, one past the end, repeats
    i[2] = -1
    loss, grad = distill64(s, v, i, t=1.7)
    assert loss[2] == 0 and (grad[2] == 0).all()
    h = 1e-6
    for c in range(9):
        d = torch.zeros_like(s)
        d[:, c] = h
        diff = (distill64(s + d, v, i, t=1.7)[0] - distill64(s - d, v, i, t=1.7)[0]) / (2 * h)
        # third-order remainder h^2 / 6 * |L'''| <= 1e-11, cancellation 2^-52 * |L| / h <= 1e-8
        assert torch.allclose(diff, grad[:, c], rtol=0, atol=1e-8)


def _weights(d=4, f=8, c=3, dtype=torch.bfloat16):
    return torch.zeros(f, d, dtype=dtype), torch.zeros(f, d, dtype=dtype), torch.zeros(c, f, dtype=dtype)


def test_decode_refusals():
    x = torch.zeros(5, 4, dtype=torch.bfloat16)
    wg, wu, wd = _weights()
    with pytest.raises(ValueError, match="CUDA"):
        decode_features(x, wg, wu, wd)
    with pytest.raises(ValueError, match="activation"):
        decode_features(x, wg, wu, wd, activation="relu")
    for bad in ((x[:, :3], wg, wu, wd), (x, wg[:7], wu, wd), (x, wg, wu, wd[:, :7]), (x, wg[0], wu, wd),
                (x[0, 0], wg, wu, wd)):
        with pytest.raises(ValueError):
            decode_features(*bad)
    with pytest.raises(ValueError, match="channels"):
        decode_features(torch.zeros(5, 129), *_weights(129))
    with pytest.raises(ValueError, match="channels"):
        decode_features(torch.zeros(5, 0), *_weights(0))
    with pytest.raises(ValueError, match="outputs"):
        decode_features(x, *_weights(c=257))
    with pytest.raises(ValueError, match="hidden"):
        decode_features(x, *_weights(f=0))
    with pytest.raises(TypeError, match="float16"):
        decode_features(x, *_weights(dtype=torch.float32))
    with pytest.raises(TypeError, match="float16"):
        decode_features(x, wg, wu.half(), wd)
    with pytest.raises(TypeError, match="floating"):
        decode_features(x.int(), wg, wu, wd)
    with pytest.raises(ValueError, match="params"):
        FeatureDecoder({"w_gate": wg})
    with pytest.raises(TypeError, match="dtype"):
        FeatureDecoder(dict(w_gate=wg, w_up=wu, w_down=wd), dtype=torch.float32)


def test_native_decode_rejects_bad_arguments_before_the_device():
    lib = nat.load()
    size = lib.gs_decode_image_bytes(32, 100, 20)
    assert size == 2 * (16384 + 32 * 128)
    for d, f, c in ((0, 8, 8), (129, 8, 8), (8, 0, 8), (8, 65537, 8), (8, 8, 0), (8, 8, 257)):
        assert lib.gs_decode_image_bytes(d, f, c) == 0
        assert lib.gs_decode_workspace_bytes(16, 16, 10, d, f, c, 1) == 0
        assert lib.gs_decode_prepare(16, 16, 16, 1, d, f, c, 16, 1 << 30, None) == nat.GS_ERR_INVALID_ARG
        assert lib.gs_decode_forward(16, 1, 4, d, f, c, 0, 16, 1 << 30, 16, None, 0, None) == nat.GS_ERR_INVALID_ARG
        assert lib.gs_decode_backward(16, 16, 1, 4, d, f, c, 0, 16, 1 << 30, 16, None, None, None, None, 0,
                                      None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_prepare(16, 16, 16, 0, 32, 100, 20, 16, size, None) == nat.GS_ERR_INVALID_ARG  # float32
    assert lib.gs_decode_prepare(16, 16, 16, 1, 32, 100, 20, 16, size - 1, None) == nat.GS_ERR_CAPACITY
    assert lib.gs_decode_prepare(16, 16, 16, 1, 32, 100, 20, 8, size, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_prepare(None, 16, 16, 1, 32, 100, 20, 16, size, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_forward(16, 1, -1, 32, 100, 20, 0, 16, size, 16, None, 0, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_forward(16, 1, 4, 32, 100, 20, 2, 16, size, 16, None, 0, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_forward(None, 1, 4, 32, 100, 20, 0, 16, size, 16, None, 0, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_forward(16, 1, 4, 32, 100, 20, 0, 16, size - 16, 16, None, 0, None) == nat.GS_ERR_CAPACITY
    assert lib.gs_decode_forward(None, 1, 0, 32, 100, 20, 0, None, 0, None, None, 0, None) == nat.GS_OK
    assert lib.gs_decode_forward(16, 1, nat.GS_DECODE_MAX_N + 1, 32, 100, 20, 0, 16, size, 16, None, 0,
                                 None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_is_few(64, 32, 256, 100) == 1 and lib.gs_decode_is_few(65, 32, 256, 100) == 0
    assert lib.gs_decode_is_few(1, 128, 256, 250) == 0 and lib.gs_decode_is_few(-1, 8, 8, 8) == 0
    few = (16, 16, 16, 16, 1, 1, 32, 64, 20, 0, 16, None)
    for at, bad in ((0, None), (3, None), (10, None), (4, 0), (5, 65), (5, -1), (6, 129), (7, 1 << 16), (9, 2)):
        assert lib.gs_decode_forward_few(*few[:at], bad, *few[at + 1:]) == nat.GS_ERR_INVALID_ARG, at
    assert lib.gs_decode_forward_few(None, None, None, None, 1, 0, 32, 64, 20, 0, None, None) == nat.GS_OK
    # aligned rows need no copy; 20 classes (40 bytes a row) and unaligned addresses do
    assert lib.gs_decode_workspace_bytes(16, None, 1000, 32, 100, 20, 0) == 0
    assert lib.gs_decode_workspace_bytes(18, None, 1000, 32, 100, 20, 0) >= 1000 * 64
    assert lib.gs_decode_workspace_bytes(16, 16, 1000, 32, 100, 20, 0) >= 1000 * 48
    assert lib.gs_decode_forward(18, 1, 1000, 32, 100, 20, 0, 16, size, 16, None, 0, None) == nat.GS_ERR_CAPACITY
    need = lib.gs_decode_workspace_bytes(16, 16, 1000, 32, 100, 20, 1)
    assert need >= 4 * (2 * 32 * 100 + 20 * 100) + 1000 * 48
    args = (16, 16, 1, 1000, 32, 100, 20, 0, 16, size, None, 16, 16)
    assert lib.gs_decode_backward(*args, None, 16, need, None) == nat.GS_ERR_INVALID_ARG
    assert lib.gs_decode_backward(*args, 16, 16, need - 1, None) == nat.GS_ERR_CAPACITY


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_plain_decoder_gradients_against_differences(act):
    g = torch.Generator().manual_seed(5)
    leaves = [torch.randn(*s, generator=g, dtype=torch.float64) for s in ((4, 3), (5, 3), (5, 3), (2, 5))]
    dy = torch.randn(4, 2, generator=g, dtype=torch.float64)
    grads = decode64(*leaves, act, dy)[1:]
    h = 1e-6
    for t, grad in zip(leaves, grads):
        for i in range(t.numel()):
            keep = float(t.view(-1)[i])
            t.view(-1)[i] = keep + h
            up = (decode64(*leaves, act) * dy).sum()
            t.view(-1)[i] = keep - h
            down = (decode64(*leaves, act) * dy).sum()
            t.view(-1)[i] = keep
            # third derivatives are below 1e3 here: remainder 2e-10; cancellation 2^-52 * 100 / h = 2e-8
            assert abs(float((up - down) / (2 * h) - grad.view(-1)[i])) < 1e-7


def test_differentiated_sees_leaves_and_tangents():
    a, leaf = torch.zeros(3), torch.zeros(3, requires_grad=True)
    assert not nat.differentiated(a) and nat.differentiated(a, leaf)
    with torch.no_grad():
        assert not nat.differentiated(leaf)
        with fwAD.dual_level():
            assert nat.differentiated(fwAD.make_dual(a, torch.ones(3)))
    assert not nat.differentiated(a)


def test_temperatures_whose_square_is_no_normal_number_are_refused():
    """T^2 would be 0 or infinite in 32 bits and the loss 0 or NaN instead of its value."""
    lib, (v, i) = nat.load(), _teacher()
    for t in (1e-39, 3e-39, 1e-30, 1e-23, 9e-19, 1.1e18, 2e19, 1e30, 3e38):
        for fn in (distill_loss, distill_loss_and_grad):
            with pytest.raises(ValueError, match="temperature"):
                fn(torch.zeros(3, 5), (v, i), temperature=t)
        status = lib.gs_distill(None, 0, 2, 5, ctypes.byref(_native_teacher()), t, None, 1.0, None, 0, None, None, None,
                                None, 0, None)
        assert status == nat.GS_ERR_INVALID_ARG and b"temperature" in lib.gs_last_error()
    for t in (1e-18, 1e18):  # the limits are allowed (and refused for the CPU tensor)
        with pytest.raises(ValueError, match="CUDA"):
            distill_loss(torch.zeros(3, 5), (v, i), temperature=t)
        lib.gs_distill(None, 0, 2, 5, ctypes.byref(_native_teacher()), t, None, 1.0, None, 0, None, None, None, None, 0,
                       None)
        assert b"NULL" in lib.gs_last_error()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,d,f,c", [(20001, 33, 70, 31), (60001, 16, 24, 9)])
def test_norm_bound_tells_a_lost_tile(n, d, f, c, dtype):
    """Planted in the plain form: gradients without one tile, the first, a middle or the ragged last one, or with a
    tile counted twice, are out of the bound the GPU tests use; gradients rounded as the kernels round are within."""
    g = torch.Generator().manual_seed(7)
    ty = DTYPES[dtype]
    r = lambda *s: torch.randn(*s, generator=g).to(ty)  # noqa: E731
    x, wg, wu, wd, dy = r(n, d), r(f, d) / d ** 0.5, r(f, d) / d ** 0.5, r(c, f) / f ** 0.5, r(n, c)
    full = decode64(x, wg, wu, wd, "silu", dy)[2:]
    bound = decode_norm_bound(ty)
    for w in full:
        assert norm_off(w.to(ty), w) <= bound / 2
    for tile in (0, n // 256, n // 128):
        rows = slice(128 * tile, min(n, 128 * tile + 128))
        part = decode64(x[rows], wg, wu, wd, "silu", dy[rows])[2:]
        for w, p in zip(full, part):
            assert norm_off(w - p, w) > 2 * bound and norm_off(w + p, w) > 2 * bound
