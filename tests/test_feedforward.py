"""The gated feed-forward block's operators (gated projections, counter-based dropout, root-mean-square norm) against a plain
implementation in 64 bits.

Bounds.  u = 2^-11 (fp16) or 2^-24 (fp32) is half a step of the stored type, relative to the value; below the normal range fp16 steps
are 2^-24, so half of one, 2^-25, is added.  An fp32 sum of n terms is off by at most n * 2^-23 of the sum of the terms' magnitudes
(2^-23, not 2^-24: the tensor core drops what does not fit).  fp16 products are exact in fp32; an fp32 product in three tf32 parts is
off by at most 2^-19 of its magnitude (each operand is hi + lo with |lo| <= 2^-10 |hi|, lo kept to 2^-21 of the operand; lo * lo <= 2^-20 is
dropped).  The activations are good to 2^-18 of (1 + |a|) times their size: the fast exponential is off by (2 + 1.2 |a|) * 2^-23, erfc's
rounded argument z by 2 z^2 * 2^-24 < 2^-18 for |z| < 5.
"""
import copy
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import cases
from deep8_b200 import _lib, ops

DEV = "cuda:0"
ACTS = sorted(ops.ACTIVATIONS)
TYPES = [torch.float16, torch.float32]
U = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126}
PRODUCT = {torch.float16: 0.0, torch.float32: 2.0 ** -19}
ACT_ERR = 2.0 ** -18


# ------------------------------------------------------------------------------------------------ plain implementations
def philox_words(seed, offset, first, count):
    """Words [first, first + count) of the stream, numpy, 64-bit integers."""
    m = np.uint64(0xFFFFFFFF)
    g0 = first // 4
    g = np.arange(g0, (first + count + 3) // 4, dtype=np.uint64)
    c = [g & m, g >> np.uint64(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[first - 4 * g0:first - 4 * g0 + count]


def keep_mask(drop, shape, first=0):
    n = int(np.prod(shape))
    return torch.from_numpy(philox_words(drop.seed, drop.offset, first, n) >= np.uint64(round(drop.p * 2 ** 32))).reshape(shape)


def dropped(drop, t):
    if drop is None:
        return t
    if drop.p == 1.0:
        return torch.zeros_like(t)
    return torch.where(keep_mask(drop, t.shape).to(t.device), t / (1.0 - drop.p), torch.zeros_like(t))


def act64(name, a):
    """act(a), act'(a) in 64 bits."""
    if name == "relu":
        return a.clamp(min=0), (a > 0).double()
    if name == "sigmoid":
        return torch.sigmoid(a), torch.sigmoid(a) * torch.sigmoid(-a)
    if name == "silu":
        s = torch.sigmoid(a)
        return a * s, s + a * s * torch.sigmoid(-a)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
    k = math.sqrt(2.0 / math.pi)
    z = 2 * k * (a + 0.044715 * a ** 3)
    s = torch.sigmoid(z)  # (1 + tanh(z / 2)) / 2, which for a < -5 would cancel to 0 even in 64 bits (1 - |tanh| < 2^-53)
    return a * s, s + a * s * torch.sigmoid(-z) * 2 * k * (1 + 3 * 0.044715 * a * a)


def gated64(x, w, name, drop=None):
    """h, pre for x [rows, xc], w [2, xc, yc] in 64 bits."""
    pre = torch.matmul(x, w)
    return dropped(drop, act64(name, pre[0])[0] * pre[1]), pre


def gated_back64(x, w, pre, dz, name, drop=None):
    value, slope = act64(name, pre[0])
    d = dropped(drop, dz)
    dpre = torch.stack((d * pre[1] * slope, d * value))
    return dpre, torch.matmul(dpre, w.transpose(1, 2)).sum(0), torch.matmul(x.t(), dpre)


def norm64(x, weight, eps):
    rstd = 1.0 / torch.sqrt((x * x).mean(-1) + eps)
    return x * rstd.unsqueeze(-1) * weight, rstd


def norm_back64(x, weight, rstd, dy):
    n = x * rstd.unsqueeze(-1)
    u = dy * weight
    return rstd.unsqueeze(-1) * (u - n * (u * n).mean(-1, keepdim=True)), (dy * n).reshape(-1, x.shape[-1]).sum(0)


def within(got, want, bound, what=""):
    got = got.double().cpu()
    want, bound = want.cpu(), bound.cpu()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), "%s: %d of %d elements out of bounds, the worst %.3g of its bound" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() / bound.clamp(min=1e-300)).max()))


def stored(want, err, dtype):
    """Bound of a value known to `err` once it is stored in dtype."""
    return err + (want.abs() + err) * U[dtype] + TINY[dtype]


def tensor(seed, shape, dtype, std=1.0):
    return torch.from_numpy(cases.normal(seed, shape, std)).to(DEV).to(dtype)


def product_err(a, b, dtype, n):
    """Bound of an fp32 product a b with n terms per sum."""
    return torch.matmul(a.abs(), b.abs()) * (PRODUCT[dtype] + n * 2.0 ** -23)


def check_gated(x, w, name, h, pre, drop=None):
    dtype = x.dtype
    x64, w64 = x.double().reshape(-1, x.shape[-1]), w.double()
    h64, pre64 = gated64(x64, w64, name, drop)
    e = product_err(x64, w64, dtype, x64.shape[1])
    if pre is not None:
        within(pre, pre64, stored(pre64, e, dtype), "pre")
    value, _ = act64(name, pre64[0])
    scale = 1.0 if drop is None or drop.p == 1.0 else 1.0 / (1.0 - drop.p)
    # |act'| <= 1.13 for all of them; relu's kink adds nothing beyond that
    e_value = 1.13 * e[0] + ACT_ERR * (1.0 + pre64[0].abs()) * value.abs()
    err = (e_value * pre64[1].abs() + value.abs() * e[1] + e_value * e[1]) * scale + h64.abs() * 2.0 ** -21
    if drop is not None:
        assert torch.equal(h.reshape(h64.shape) != 0, (h64 != 0) & (h.reshape(h64.shape) != 0))  # dropped elements are exactly 0
    within(h.reshape(h64.shape), h64, stored(h64, err, dtype), "h")


# rows, cols, width: single elements, one token, ragged sizes, one past the tile edges, sizes whose rows start on 16-byte
# boundaries, enough tiles for every tile shape of the fp16 kernels, contractions that are split
GATED = [((1, 1, 1), 1), ((1, 1, 64), 64), ((1, 3, 17), 9), ((2, 65, 40), 72), ((1, 129, 128), 192), ((1, 257, 130), 250), ((3, 100, 64), 1000),
         ((1, 1, 4096), 512), ((1, 7, 2048), 1032), ((1, 48, 1600), 264), ((1, 127, 1000), 504), ((1, 300, 512), 520)]
GATED_LARGE = [((1, 1500, 512), 2496), ((2, 1024, 320), 4992), ((1, 2047, 128), 2504), ((1, 1300, 72), 2002), ((1, 1999, 333), 2503)]


# ------------------------------------------------------------------------------------------------ on the CPU
def test_generator_known_answers():
    """The published vectors of Philox4x32-10 at the all-zero and all-one counter and key."""
    assert [int(v) for v in philox_words(0, 0, 0, 4)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = (1 << 64) - 1
    with np.errstate(over="ignore"):
        g = philox_words(ones, ones, 4 * ((1 << 61) - 1), 4)  # any counter: the four words of one group belong together
    assert len(set(int(v) for v in g)) == 4


@pytest.mark.parametrize("name", ACTS)
def test_plain_gradients_against_differences(name):
    """The formulas the kernels are held to are the derivatives of the forward formulas (central differences in 64 bits)."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(5, 7, generator=g, dtype=torch.float64), torch.randn(2, 7, 6, generator=g, dtype=torch.float64)
    dz = torch.randn(5, 6, generator=g, dtype=torch.float64)
    drop = ops.Dropout(0.3, 11, 4)
    h, pre = gated64(x, w, name, drop)
    _, dx, dw = gated_back64(x, w, pre, dz, name, drop)
    for t, grad, f in ((x, dx, lambda v: gated64(v, w, name, drop)[0]), (w, dw, lambda v: gated64(x, v, name, drop)[0])):
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        step = 1e-6
        diff = ((f(t + step * v) - f(t - step * v)) * dz).sum() / (2 * step)
        assert abs(float(diff - (grad * v).sum())) < 1e-7 * (1 + abs(float(diff)))  # step^2 and 2^-53 / step


def test_plain_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(6)
    x, weight = torch.randn(4, 9, generator=g, dtype=torch.float64), torch.randn(9, generator=g, dtype=torch.float64)
    dy = torch.randn(4, 9, generator=g, dtype=torch.float64)
    _, rstd = norm64(x, weight, 1e-3)
    dx, dweight = norm_back64(x, weight, rstd, dy)
    for t, grad, f in ((x, dx, lambda v: norm64(v, weight, 1e-3)[0]), (weight, dweight, lambda v: norm64(x, v, 1e-3)[0])):
        v = torch.randn(t.shape, generator=g, dtype=torch.float64)
        step = 1e-6
        diff = ((f(t + step * v) - f(t - step * v)) * dy).sum() / (2 * step)
        assert abs(float(diff - (grad * v).sum())) < 1e-7 * (1 + abs(float(diff)))


def test_dropout_arguments_are_checked():
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            ops.Dropout(p, 1)
    for seed, offset in ((-1, 0), (1 << 64, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError):
            ops.Dropout(0.1, seed, offset)
    with pytest.raises(ValueError):
        ops.Dropout(0.1, 1, counter=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.Dropout(0.1, 1, counter=torch.zeros(2, dtype=torch.int64))


class _NoLaunchLib:
    def __getattr__(self, name):
        def refuse(*a, **k):
            raise AssertionError("%s was reached: the argument check did not fire" % name)
        return refuse


class _AnyDevice(ops.Context):
    """A context without a GPU behind it whose device check is the type and layout check alone."""

    def _on_device(self, *ts):
        return ops._same(*ts)


@pytest.fixture
def bare():
    c = _AnyDevice.__new__(_AnyDevice)
    c.lib, c.h, c.device, c._device, c.stream = _NoLaunchLib(), None, 0, torch.device("cuda", 0), None
    return c


def test_front_end_checks(bare):
    x, w = torch.zeros(1, 4, 8), torch.zeros(2, 8, 6)
    pre, dz, rows = torch.zeros(2, 4, 6), torch.zeros(1, 4, 6), torch.zeros(4)
    bad = [
        lambda: bare.gated_forward(x[0], w),                                        # three dimensions
        lambda: bare.gated_forward(x, torch.zeros(1, 8, 6)),                        # two projections
        lambda: bare.gated_forward(x, torch.zeros(2, 7, 6)),
        lambda: bare.gated_forward(x, w, "swish"),
        lambda: bare.gated_forward(x, w, out=torch.zeros(1, 4, 7)),
        lambda: bare.gated_forward(x, w.half()),
        lambda: bare.gated_forward(x.transpose(1, 2), torch.zeros(2, 4, 6)),        # not contiguous
        lambda: bare.gated_forward(x, w, pre=torch.zeros(2, 5, 6)),
        lambda: bare.gated_grad_pre(pre, torch.zeros(1, 4, 5)),
        lambda: bare.gated_grad_pre(pre, dz, dpre=torch.zeros(2, 4, 5)),
        lambda: bare.gated_backward(x, w, pre, torch.zeros(1, 5, 6), None, None),
        lambda: bare.gated_backward(x, w, pre, dz, torch.zeros(1, 4, 7), None),
        lambda: bare.gated_backward(x, w, pre, dz, None, torch.zeros(2, 8, 5)),
        lambda: bare.gated_backward(x, w, pre, dz, x.clone().half(), None),
        lambda: bare.dropout_forward(x, ops.Dropout(0.1, 1), residual=torch.zeros(1, 4, 7)),
        lambda: bare.dropout_forward(x, ops.Dropout(0.1, 1), out=torch.zeros(4, 8)),
        lambda: bare.dropout_forward(x, ops.Dropout(0.1, 1, counter=torch.zeros(1, dtype=torch.int64))),  # a counter on the host
        lambda: bare.dropout_backward(x, torch.zeros(1, 4, 7), ops.Dropout(0.1, 1)),
        lambda: bare.rms_norm_forward(x, torch.zeros(7)),
        lambda: bare.rms_norm_forward(x, torch.zeros(8), rstd=torch.zeros(5)),
        lambda: bare.rms_norm_forward(x, torch.zeros(8), rstd=rows.double()),
        lambda: bare.rms_norm_backward(x, torch.zeros(8), rows, x.clone(), torch.zeros(7), x.clone()),
        lambda: bare.rms_norm_backward(x, torch.zeros(8), rows, torch.zeros(1, 4, 7), None, x.clone()),
        lambda: bare.rms_norm_backward(x, torch.zeros(8), rows, None, None, torch.zeros(1, 5, 8)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was not refused" % k)
    with pytest.raises(TypeError):
        bare.gated_forward(x.double(), w.double())


def test_tensors_of_the_host_are_refused():
    c = ops.Context.__new__(ops.Context)
    c.lib, c.h, c.device, c._device, c.stream = _NoLaunchLib(), None, 0, torch.device("cuda", 0), None
    with pytest.raises(ValueError):
        c.gated_forward(torch.zeros(1, 4, 8), torch.zeros(2, 8, 6))
    with pytest.raises(ValueError):
        c.dropout_forward(torch.zeros(4), ops.Dropout(0.1, 1))
    with pytest.raises(ValueError):
        c.rms_norm_forward(torch.zeros(4, 8), torch.zeros(8))


class _RecordingLib:
    """Stands in for the library: keeps what the dropout argument of a call points at."""

    def d8k_dropout_forward(self, h, dtype, x, residual, y, n, drop):
        spec = drop._obj
        self.got = (spec.p, spec.seed, spec.offset, spec.device_offset)
        return 0


def test_dropout_fields_set_after_construction_reach_the_library(bare):
    """A training loop that advances the offset (or exchanges the counter) gets another mask; what a constructor refuses a setter does, too."""
    bare.lib = _RecordingLib()
    x, top = torch.zeros(4), (1 << 64) - 1
    first, second = torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64)
    drop = ops.Dropout(0.1, 5)

    def handed():
        bare.dropout_forward(x, drop)
        assert (drop.p, drop.seed, drop.offset) == bare.lib.got[:3]
        return bare.lib.got

    bare._device = torch.device("cpu")  # where this test's counters are
    assert handed() == (0.1, 5, 0, None)
    drop.offset += 1
    drop.seed = top
    drop.p = 0.5
    assert handed() == (0.5, top, 1, None)
    for counter in (first, second):
        drop.counter = counter
        assert drop.counter is counter and handed() == (0.5, top, 1, counter.data_ptr())
    second.set_(torch.zeros(1, dtype=torch.int64))  # the same tensor over other memory
    assert handed()[3] == second.data_ptr()
    drop.counter = None
    assert handed() == (0.5, top, 1, None)
    for field, value in (("p", 1.5), ("p", -0.1), ("p", float("nan")), ("seed", -1), ("seed", 1 << 64), ("offset", 1 << 64),
                         ("counter", torch.zeros(1)), ("counter", torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(ValueError):
            setattr(drop, field, value)
    assert handed() == (0.5, top, 1, None)
    drop.counter = first
    bare._device = torch.device("cuda", 0)
    with pytest.raises(ValueError):
        bare.dropout_forward(x, drop)  # the counter that is set now is checked, not the constructor's
    twin = copy.copy(drop)
    twin.offset, twin.counter = 7, None
    assert (drop.offset, drop.counter) == (1, first) and (twin.p, twin.seed, twin.offset, twin.counter) == (0.5, top, 7, None)


def test_library_refuses_a_null_context():
    lib = _lib.load()
    assert lib.d8k_gated_forward(None, 0, 0, None, 1, 1, 1, None, 1, None, None, None) == 1
    assert lib.d8k_dropout_forward(None, 0, None, None, None, 1, None) == 1
    assert lib.d8k_rms_norm_forward(None, 0, None, None, 1e-6, None, None, 1, 1) == 1
    assert b"context" in lib.d8k_last_error()


def test_cpp_gradient_checks():
    """What the C++ gradients refuse before they touch a device (tests/cpp/test_feedforward_checks.cu)."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "test_feedforward_checks")
    assert os.path.exists(exe), "tests/cpp/bin/test_feedforward_checks is missing: run __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


def _philox_raw(counter, key):
    """Philox4x32-10 of one 128-bit counter under a 64-bit key, lists of 32-bit words, lowest first, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


# counter, key, words: the generator's published answers (the authors' Random123 distribution, its known-answer list for philox4x32 10)
PHILOX_ANSWERS = [([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
                  ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
                  ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])]


def test_generator_published_answers():
    """All three published vectors, and the plain generator of this file against them where its element index can reach the counter: the words
    of seed and offset have a place of their own each."""
    for counter, key, words in PHILOX_ANSWERS:
        assert _philox_raw(counter, key) == words
    seed, offset, group = 0x299f31d0a4093822, 0x0370734413198a2e, 0x05a308d3243f6a88
    want = _philox_raw([group & 0xFFFFFFFF, group >> 32, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])
    assert [int(v) for v in philox_words(seed, offset, 4 * group, 4)] == want
    counter, key, words = PHILOX_ANSWERS[2]
    assert [int(v) for v in philox_words(key[0] | key[1] << 32, counter[2] | counter[3] << 32, 8, 1)] == _philox_raw([2, 0] + counter[2:], key)[:1]


# ------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GATED, ids=str)
def test_gated_forward(ctx, shape, dtype):
    (xb, xr, xc), yc = shape
    x, w = tensor(1, (xb, xr, xc), dtype), tensor(2, (2, xc, yc), dtype, 1.0 / math.sqrt(xc))
    for k, name in enumerate(ACTS if xb * xr * xc * yc < 1 << 22 else ["silu"]):
        drop = ops.Dropout(0.2, 77, k) if k % 2 else None
        pre = torch.full((2, xb * xr, yc), float("nan"), dtype=dtype, device=DEV)
        h = ctx.gated_forward(x, w, name, pre=pre, dropout=drop)
        check_gated(x, w, name, h, pre, drop)
        assert torch.equal(ctx.gated_forward(x, w, name, dropout=drop), h)  # h does not depend on pre being kept, nor on the run
    assert ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GATED_LARGE, ids=str)
def test_gated_forward_many_tiles(ctx, shape, dtype):
    (xb, xr, xc), yc = shape
    x, w = tensor(3, (xb, xr, xc), dtype), tensor(4, (2, xc, yc), dtype, 1.0 / math.sqrt(xc))
    drop = ops.Dropout(0.1, 5, 1 << 40)
    pre = torch.full((2, xb * xr, yc), float("nan"), dtype=dtype, device=DEV)
    h = ctx.gated_forward(x, w, "gelu_tanh", pre=pre, dropout=drop)
    check_gated(x, w, "gelu_tanh", h, pre, drop)
    assert torch.equal(ctx.gated_forward(x, w, "gelu_tanh", dropout=drop), h)
    assert ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_forward_on_views_off_the_16_byte_boundary(ctx, dtype):
    for shift_x, shift_w, shift_h in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (3, 2, 1)):
        x = torch.empty(64 * 64 + 8, dtype=dtype, device=DEV)[shift_x:shift_x + 64 * 64].view(1, 64, 64)
        w = torch.empty(2 * 64 * 128 + 8, dtype=dtype, device=DEV)[shift_w:shift_w + 2 * 64 * 128].view(2, 64, 128)
        x.copy_(tensor(5, (1, 64, 64), dtype))
        w.copy_(tensor(6, (2, 64, 128), dtype, 0.125))
        h_all = torch.full((64 * 128 + 8,), 7.0, dtype=dtype, device=DEV)
        pre_all = torch.full((2 * 64 * 128 + 8,), 7.0, dtype=dtype, device=DEV)
        h, pre = h_all[shift_h:shift_h + 64 * 128].view(1, 64, 128), pre_all[shift_h:shift_h + 2 * 64 * 128].view(2, 64, 128)
        ctx.gated_forward(x, w, "silu", out=h, pre=pre)
        check_gated(x, w, "silu", h, pre)
        for whole, n in ((h_all, 64 * 128), (pre_all, 2 * 64 * 128)):  # nothing beside the outputs is written
            assert (whole[:shift_h] == 7).all() and (whole[shift_h + n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_forward_leaves_what_follows_alone(ctx, dtype):
    """Rows behind the last one and columns behind the last one, at sizes that do not fill a tile."""
    for rows, cols, width in ((5, 64, 72), (130, 96, 200), (257, 64, 256)):
        x, w = tensor(7, (1, rows, cols), dtype), tensor(8, (2, cols, width), dtype, 0.1)
        h_all = torch.full((rows * width + 4096,), 7.0, dtype=dtype, device=DEV)
        pre_all = torch.full((2 * rows * width + 4096,), 7.0, dtype=dtype, device=DEV)
        h, pre = h_all[:rows * width].view(1, rows, width), pre_all[:2 * rows * width].view(2, rows, width)
        ctx.gated_forward(x, w, "gelu", out=h, pre=pre)
        check_gated(x, w, "gelu", h, pre)
        assert (h_all[rows * width:] == 7).all() and (pre_all[2 * rows * width:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_forward_infinities_and_nan(ctx, dtype):
    """A NaN in a row of x reaches that row alone; overflowing projections give infinities, not NaN."""
    x, w = tensor(9, (1, 40, 64), dtype), tensor(10, (2, 64, 64), dtype, 0.1)
    clean = ctx.gated_forward(x, w, "silu")
    x[0, 7, 3] = float("nan")
    h = ctx.gated_forward(x, w, "silu")
    assert torch.isnan(h[0, 7]).all()
    rest = [r for r in range(40) if r != 7]
    assert torch.equal(h[0, rest], clean[0, rest])
    big = 60000.0 if dtype == torch.float16 else 1e30
    x = torch.full((1, 2, 64), big, dtype=dtype, device=DEV)
    w = torch.full((2, 64, 64), 1.0, dtype=dtype, device=DEV)
    w[0, :, 1] = -1.0  # act(-large) vanishes for silu, gelu, relu
    for name in ("silu", "gelu", "gelu_tanh", "relu"):
        h = ctx.gated_forward(x, w, name)
        assert (h[0, :, 0] == float("inf")).all() and (h[0, :, 1] == 0).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_gated_grad_pre(ctx, name, dtype):
    for rows, width, p in ((1, 1, 0.0), (3, 5, 0.5), (64, 256, 0.1), (33, 1001, 0.0), (257, 520, 0.3), (2, 8, 1.0)):
        pre, dz = tensor(11, (2, rows, width), dtype, 2.0), tensor(12, (1, rows, width), dtype)
        drop = ops.Dropout(p, 3, 9) if p else None
        n = torch.zeros(1, dtype=torch.float64)
        dpre64, _, _ = gated_back64(torch.zeros(rows, 1, dtype=torch.float64, device=DEV), torch.zeros(2, 1, width, dtype=torch.float64, device=DEV),
                                    pre.double(), dz[0].double(), name, drop)
        got = ctx.gated_grad_pre(pre, dz, name, dropout=drop)
        scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
        a = pre[0].double().abs()
        # the slope's error in absolute terms: its parts are at most 1 + |a|
        err = torch.stack((dz[0].double().abs() * scale * pre[1].double().abs() * ACT_ERR * (1 + a) ** 2, dpre64[1].abs() * ACT_ERR * (1 + a))) \
            + dpre64.abs() * 2.0 ** -21
        within(got, dpre64, stored(dpre64, err, dtype), "dpre")
        inplace = pre.clone()
        assert ctx.gated_grad_pre(inplace, dz, name, dpre=inplace, dropout=drop) is inplace and torch.equal(inplace, got)


@pytest.mark.gpu
def test_gated_grad_pre_drops_whatever_is_there(ctx):
    """Positions the mask drops have zero gradients even where the projections hold infinities or NaN."""
    drop = ops.Dropout(0.5, 21, 2)
    pre = torch.full((2, 4, 64), float("inf"), dtype=torch.float16, device=DEV)
    pre[0, 1] = float("nan")
    got = ctx.gated_grad_pre(pre, torch.ones(1, 4, 64, dtype=torch.float16, device=DEV), "silu", dropout=drop)
    off = ~keep_mask(drop, (4, 64)).to(DEV)
    assert (got[:, off] == 0).all() and off.any()


def check_backward(x, w, pre, dz, dx, dw, name, drop, dx0=None, dw0=None):
    dtype = x.dtype
    x64, w64 = x.double().reshape(-1, x.shape[-1]), w.double()
    pre64, dz64 = pre.double(), dz.double().reshape(-1, dz.shape[-1])
    dpre, dx64, dw64 = gated_back64(x64, w64, pre64, dz64, name, drop)
    a = pre64[0].abs()
    scale = 1.0 / (1.0 - drop.p) if drop is not None else 1.0
    e = torch.stack((dz64.abs() * scale * pre64[1].abs() * ACT_ERR * (1 + a) ** 2, dpre[1].abs() * ACT_ERR * (1 + a))) + dpre.abs() * 2.0 ** -21
    e = stored(dpre, e, dtype)  # dpre is stored in dtype between the kernels
    size = dpre.abs() + e
    if dx is not None:
        n = 2 * w.shape[2]
        err = torch.matmul(e, w64.abs().transpose(1, 2)).sum(0) + torch.matmul(size, w64.abs().transpose(1, 2)).sum(0) * (PRODUCT[dtype] + n * 2.0 ** -23)
        if dx0 is not None:
            dx64 = dx64 + dx0.double().reshape(dx64.shape)
            err = err + dx64.abs() * 2.0 ** -23
        within(dx.reshape(dx64.shape), dx64, stored(dx64, err, dtype), "dx")
    if dw is not None:
        n = x64.shape[0]
        err = torch.matmul(x64.abs().t(), e) + torch.matmul(x64.abs().t(), size) * (PRODUCT[dtype] + n * 2.0 ** -23)
        if dw0 is not None:
            dw64 = dw64 + dw0.double()
            err = err + dw64.abs() * 2.0 ** -23
        within(dw, dw64, stored(dw64, err, dtype), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", GATED + GATED_LARGE, ids=str)
def test_gated_backward(ctx, shape, dtype):
    (xb, xr, xc), yc = shape
    x, w = tensor(13, (xb, xr, xc), dtype), tensor(14, (2, xc, yc), dtype, 1.0 / math.sqrt(xc))
    pre, dz = tensor(15, (2, xb * xr, yc), dtype), tensor(16, (xb, xr, yc), dtype, 0.1)
    for name, drop in (("silu", None), ("gelu_tanh", ops.Dropout(0.25, 1, 2))):
        dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
        assert ctx.gated_backward(x, w, pre, dz, dx, dw, name, accumulate=False, dropout=drop) == (dx, dw)
        check_backward(x, w, pre, dz, dx, dw, name, drop)
        again_x, again_w = torch.empty_like(x), torch.empty_like(w)
        ctx.gated_backward(x, w, pre, dz, again_x, None, name, accumulate=False, dropout=drop)
        ctx.gated_backward(x, w, pre, dz, None, again_w, name, accumulate=False, dropout=drop)
        assert torch.equal(again_x, dx) and torch.equal(again_w, dw)  # same bits, one gradient at a time
    dx0, dw0 = tensor(17, (xb, xr, xc), dtype), tensor(18, (2, xc, yc), dtype)
    dx, dw, kept = dx0.clone(), dw0.clone(), pre.clone()
    ctx.gated_backward(x, w, kept, dz, dx, dw, "gelu", dpre=kept)  # accumulates; the workspace over pre
    check_backward(x, w, pre, dz, dx, dw, "gelu", None, dx0, dw0)
    assert ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_without_rows(ctx, dtype):
    x, w = torch.empty(1, 0, 8, dtype=dtype, device=DEV), tensor(1, (2, 8, 6), dtype)
    pre = torch.empty(2, 0, 6, dtype=dtype, device=DEV)
    assert ctx.gated_forward(x, w, pre=pre).shape == (1, 0, 6)
    dw = torch.ones_like(w)
    ctx.gated_backward(x, w, pre, torch.empty(1, 0, 6, dtype=dtype, device=DEV), torch.empty_like(x), dw)
    assert (dw == 1).all()
    ctx.gated_backward(x, w, pre, torch.empty(1, 0, 6, dtype=dtype, device=DEV), torch.empty_like(x), dw, accumulate=False)
    assert (dw == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 1000, 4099, 1 << 20])
def test_dropout(ctx, n, dtype):
    x, r = tensor(19, (n,), dtype), tensor(20, (n,), dtype)
    for p in (0.0, 0.1, 0.5, 0.999, 1.0):
        drop = ops.Dropout(p, 0xFEDCBA9876543210, (1 << 63) + n)
        want = dropped(drop, x.double())
        got = ctx.dropout_forward(x, drop)
        within(got, want, stored(want, want.abs() * 2.0 ** -22, dtype), "y")
        assert torch.equal(got == 0, (want == 0) | (got == 0))
        got_r = ctx.dropout_forward(x, drop, residual=r)
        sum64 = want + r.double()
        within(got_r, sum64, stored(sum64, (want.abs() + r.double().abs()) * 2.0 ** -22, dtype), "residual + y")
        dx = torch.full_like(x, float("nan"))
        assert torch.equal(ctx.dropout_backward(dx, x, drop, accumulate=False), got)  # the same mask
        assert torch.equal(ctx.dropout_backward(r.clone(), x, drop), got_r)           # accumulated
        for inplace in (x.clone(), r.clone()):  # over x, over the residual
            out = ctx.dropout_forward(inplace if torch.equal(inplace, x) else x, drop, residual=r if torch.equal(inplace, x) else inplace, out=inplace)
            assert out is inplace and torch.equal(out, got_r)
        dy = x.clone()
        assert torch.equal(ctx.dropout_backward(dy, dy, drop, accumulate=False), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_off_the_16_byte_boundary(ctx, dtype):
    drop = ops.Dropout(0.3, 4, 4)
    x, r = tensor(21, (5000,), dtype), tensor(22, (5000,), dtype)
    want = ctx.dropout_forward(x, drop, residual=r)
    for sx, sr, sy in ((1, 0, 0), (0, 1, 0), (0, 0, 3)):
        parts = []
        for t, s in ((x, sx), (r, sr), (torch.zeros_like(x), sy)):
            whole = torch.full((5016,), 7.0, dtype=dtype, device=DEV)
            whole[s:s + 5000].copy_(t)
            parts.append(whole)
        y = parts[2][sy:sy + 5000]
        ctx.dropout_forward(parts[0][sx:sx + 5000], drop, residual=parts[1][sr:sr + 5000], out=y)
        assert torch.equal(y, want)
        assert (parts[2][:sy] == 7).all() and (parts[2][sy + 5000:] == 7).all()


@pytest.mark.gpu
def test_dropout_drops_infinities_and_nan(ctx):
    drop = ops.Dropout(0.5, 8, 1)
    x = torch.full((4096,), float("nan"), dtype=torch.float32, device=DEV)
    x[::2] = float("inf")
    y = ctx.dropout_forward(x, drop)
    keep = keep_mask(drop, (4096,)).to(DEV)
    assert (y[~keep] == 0).all() and torch.isnan(y[keep & torch.isnan(x)]).all() and (y[keep & torch.isinf(x)] == float("inf")).all()
    assert (ctx.dropout_forward(x, ops.Dropout(1.0, 8, 1)) == 0).all()


@pytest.mark.gpu
def test_dropout_beyond_32_bit_offsets(ctx):
    n = (1 << 32) + 4099
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    drop = ops.Dropout(0.5, 17, 3)
    y = ctx.dropout_forward(x, drop)
    for first in (0, (1 << 31) - 100, (1 << 32) - 100, n - 4099):
        count = min(4000, n - first)
        want = keep_mask(drop, (count,), first).to(DEV).half() * 2
        assert torch.equal(y[first:first + count], want)
    assert torch.equal(y[-3:], keep_mask(drop, (3,), n - 3).to(DEV).half() * 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 5), (7, 64), (33, 257), (65, 1000), (300, 1024), (5, 8200), (40, 12288), (3, 40000), (2, 70001),
                                   (2000, 96)], ids=str)
def test_rms_norm(ctx, shape, dtype):
    rows, cols = shape
    x, weight, dy = tensor(23, shape, dtype, 3.0), tensor(24, (cols,), dtype), tensor(25, shape, dtype, 0.1)
    eps = 1e-5
    y64, rstd64 = norm64(x.double(), weight.double(), eps)
    rstd = torch.full((rows,), float("nan"), device=DEV)
    y = ctx.rms_norm_forward(x, weight, eps, rstd=rstd)
    # a sum of n squares, at most n / 32 of them in a row and a tree above: far less than n steps; its root halves the error
    e = (cols * 2.0 ** -24 + 4 * 2.0 ** -23)
    within(rstd, rstd64, rstd64 * e + 1e-30, "rstd")
    within(y, y64, stored(y64, y64.abs() * (e + 2.0 ** -22), dtype), "y")
    assert torch.equal(ctx.rms_norm_forward(x, weight, eps), y)
    inplace = x.clone()
    assert torch.equal(ctx.rms_norm_forward(inplace, weight, eps, out=inplace), y)

    dx64, dweight64 = norm_back64(x.double(), weight.double(), rstd.double(), dy.double())
    n = (x.double() * rstd.double()[:, None]).abs()
    u = (dy.double() * weight.double()).abs()
    e_dx = rstd.double()[:, None] * (u * 2.0 ** -21 + n * (u * n).mean(1, keepdim=True) * (cols * 2.0 ** -23 + 2.0 ** -20))
    e_dw = (dy.double().abs() * n).sum(0) * (rows * 2.0 ** -23 + 2.0 ** -20)
    dx, dweight = torch.full_like(x, float("nan")), torch.full_like(weight, float("nan"))
    assert ctx.rms_norm_backward(x, weight, rstd, dx, dweight, dy, accumulate=False) == (dx, dweight)
    within(dx, dx64, stored(dx64, e_dx, dtype), "dx")
    within(dweight, dweight64, stored(dweight64, e_dw, dtype), "dweight")
    once_x, once_w = torch.empty_like(x), torch.empty_like(weight)
    ctx.rms_norm_backward(x, weight, rstd, once_x, None, dy, accumulate=False)
    ctx.rms_norm_backward(x, weight, rstd, None, once_w, dy, accumulate=False)
    assert torch.equal(once_x, dx)
    within(once_w, dweight64, stored(dweight64, e_dw, dtype), "dweight alone")
    acc_x, acc_w = x.clone(), weight.clone()
    ctx.rms_norm_backward(x, weight, rstd, acc_x, acc_w, dy)
    within(acc_x, dx64 + x.double(), stored(dx64 + x.double(), e_dx + (dx64 + x.double()).abs() * 2.0 ** -22, dtype), "dx accumulated")
    within(acc_w, dweight64 + weight.double(), stored(dweight64 + weight.double(), e_dw + (dweight64 + weight.double()).abs() * 2.0 ** -22, dtype),
           "dweight accumulated")
    for _ in range(2):  # same bits every run
        ctx.rms_norm_backward(x, weight, rstd, once_x, once_w, dy, accumulate=False)
        assert torch.equal(once_x, dx) and torch.equal(once_w, dweight)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm_off_the_16_byte_boundary(ctx, dtype):
    rows, cols = 33, 512
    x, weight, dy = tensor(26, (rows, cols), dtype), tensor(27, (cols,), dtype), tensor(28, (rows, cols), dtype)
    rstd = torch.empty(rows, device=DEV)
    y = ctx.rms_norm_forward(x, weight, rstd=rstd)
    dx, dweight = torch.empty_like(x), torch.empty_like(weight)
    ctx.rms_norm_backward(x, weight, rstd, dx, dweight, dy, accumulate=False)

    def shifted(t, s):
        whole = torch.full((t.numel() + 16,), 7.0, dtype=t.dtype, device=DEV)
        whole[s:s + t.numel()].copy_(t.reshape(-1))
        return whole, whole[s:s + t.numel()].view(t.shape)

    for k in range(5):
        s = [1 if i == k else 0 for i in range(5)]
        (_, xs), (_, ws), (ya, ys), (_, gs), (da, ds) = shifted(x, s[0]), shifted(weight, s[1]), shifted(y * 0, s[2]), shifted(dy, s[3]), shifted(dx * 0, s[4])
        r2, dw2 = torch.empty_like(rstd), torch.empty_like(dweight)
        ctx.rms_norm_forward(xs, ws, out=ys, rstd=r2)
        ctx.rms_norm_backward(xs, ws, rstd, ds, dw2, gs, accumulate=False)
        # another order of the sums: a few steps of fp32, at most one of the stored type
        for got, want in ((r2, rstd), (ys, y), (ds, dx), (dw2, dweight)):
            close = (got.double() - want.double()).abs() <= want.double().abs() * (2 * U[got.dtype] + 2.0 ** -19) + want.double().abs().max() * 2.0 ** -18
            assert close.all()
        assert (ya[:s[2]] == 7).all() and (ya[s[2] + y.numel():] == 7).all() and (da[:s[4]] == 7).all() and (da[s[4] + dx.numel():] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rms_norm_zero_rows_and_zero_values(ctx, dtype):
    weight = tensor(29, (64,), dtype)
    empty = torch.empty(0, 64, dtype=dtype, device=DEV)
    none = torch.empty(0, device=DEV)
    assert ctx.rms_norm_forward(empty, weight, rstd=none).shape == (0, 64)
    dweight = torch.ones_like(weight)
    ctx.rms_norm_backward(empty, weight, none, empty.clone(), dweight, empty.clone())
    assert (dweight == 1).all()
    ctx.rms_norm_backward(empty, weight, none, empty.clone(), dweight, empty.clone(), accumulate=False)
    assert (dweight == 0).all()
    rstd = torch.empty(3, device=DEV)
    y = ctx.rms_norm_forward(torch.zeros(3, 64, dtype=dtype, device=DEV), weight, 1e-6, rstd=rstd)  # an all-zero row: eps alone
    assert (y == 0).all() and ((rstd - 1000.0).abs() < 1e-3).all()


@pytest.mark.gpu
def test_library_refusals(ctx):
    """Calls that the Python front-end cannot make, at the C interface."""
    lib = _lib.load()
    x, w = tensor(1, (1, 4, 8), torch.float32), tensor(2, (2, 8, 8), torch.float32)
    h, p = torch.empty(1, 4, 8, device=DEV), ops._p
    ok = dict(ctx=ctx.h, dtype=1, act=0, x=p(x), xb=1, xr=4, xc=8, w=p(w), yc=8, pre=None, h=p(h), drop=None)

    def call(**change):
        a = dict(ok, **change)
        return lib.d8k_gated_forward(a["ctx"], a["dtype"], a["act"], a["x"], a["xb"], a["xr"], a["xc"], a["w"], a["yc"], a["pre"], a["h"], a["drop"])

    assert call() == 0
    import ctypes
    bad_p = ctypes.byref(_lib.DropoutSpec(1.5, 1, 1, None))
    odd = ctypes.byref(_lib.DropoutSpec(0.5, 1, 1, x.data_ptr() + 4))
    for change in (dict(dtype=7), dict(act=-1), dict(act=5), dict(x=None), dict(w=None), dict(h=None), dict(xc=0), dict(yc=0), dict(xr=-1),
                   dict(xb=1 << 16, xr=1 << 16), dict(h=p(x)), dict(pre=p(w)), dict(h=p(w)), dict(pre=p(h)), dict(drop=bad_p), dict(drop=odd)):
        assert call(**change) == 1, change
    n = x.numel()
    d = ops.Dropout(0.5, 1).arg
    assert lib.d8k_dropout_forward(ctx.h, 1, p(x), None, p(h), n, None) == 1
    assert lib.d8k_dropout_forward(ctx.h, 1, None, None, p(h), n, d) == 1
    assert lib.d8k_dropout_forward(ctx.h, 1, p(x), None, ctypes.c_void_p(x.data_ptr() + 4), n - 1, d) == 1  # overlaps, shifted
    assert lib.d8k_dropout_backward(ctx.h, 1, p(x), p(x), n, 1, d) == 1                                    # accumulates over dy
    rstd = torch.empty(4, device=DEV)
    weight = torch.ones(8, device=DEV)
    for eps in (-1.0, float("nan"), float("inf")):
        assert lib.d8k_rms_norm_forward(ctx.h, 1, p(x), p(weight), eps, p(h), None, 4, 8) == 1
    assert lib.d8k_rms_norm_forward(ctx.h, 1, p(x), p(weight), 1e-6, p(h), None, 4, 0) == 1
    assert lib.d8k_rms_norm_forward(ctx.h, 1, p(x), p(weight), 1e-6, ctypes.c_void_p(x.data_ptr() + 16), None, 4, 8) == 1
    assert lib.d8k_rms_norm_backward(ctx.h, 1, p(x), p(weight), p(rstd), p(x), None, p(h), 4, 8, 0) == 1
    assert lib.d8k_rms_norm_backward(ctx.h, 1, p(x), p(weight), None, p(h), None, p(x), 4, 8, 0) == 1
    pre = torch.empty(2, 4, 8, device=DEV)
    assert lib.d8k_gated_backward(ctx.h, 1, 0, p(x), 1, 4, 8, p(w), 8, p(pre), p(h), p(pre), p(x), None, 0, None) == 1   # dx over x
    assert lib.d8k_gated_backward(ctx.h, 1, 0, p(x), 1, 4, 8, p(w), 8, p(pre), p(h), None, None, None, 0, None) == 1     # no workspace
    assert lib.d8k_gated_backward(ctx.h, 1, 9, p(x), 1, 4, 8, p(w), 8, p(pre), p(h), p(pre), None, None, 0, None) == 1
    torch.cuda.synchronize()
    assert ctx.status() == 0


def _block_step(c, dtype, t, drop_in, drop_out, out):
    """One training step of y = r + dropout((act(n w0) (n w1)) w2), n = rms_norm(r): forward, then all gradients."""
    r, gain, w, w2, dy = t["r"], t["gain"], t["w"], t["w2"], t["dy"]
    rows, cols, width = r.shape[1], r.shape[2], w.shape[2]
    rstd, pre, dpre = out["rstd"], out["pre"], out["dpre"]
    n = c.rms_norm_forward(r, gain, out=out["n"], rstd=rstd)
    h = c.gated_forward(n, w, "silu", out=out["h"], pre=pre, dropout=drop_in)
    z = c.matmul_forward(h, w2, out=out["z"])
    c.dropout_forward(z, drop_out, residual=r, out=out["y"])
    c.dropout_backward(out["dz"], dy, drop_out, accumulate=False)
    c.matmul_grad_x(h, out["dh"], w2, out["dz"], accumulate=False)
    c.matmul_grad_y(h, w2, out["dw2"], out["dz"], accumulate=False)
    c.gated_backward(n, w, pre, out["dh"], out["dn"], out["dw"], "silu", dpre=dpre, accumulate=False, dropout=drop_in)
    out["dr"].copy_(dy)  # the residual path
    c.rms_norm_backward(r, gain, rstd, out["dr"], None, out["dn"])
    c.rms_norm_backward(r, gain, rstd, None, out["dgain"], out["dn"], accumulate=False)


def _block(dtype, rows, cols, width):
    t = {"r": tensor(31, (1, rows, cols), dtype, 2.0), "gain": 1 + tensor(32, (cols,), dtype, 0.1), "w": tensor(33, (2, cols, width), dtype, cols ** -0.5),
         "w2": tensor(34, (1, width, cols), dtype, width ** -0.5), "dy": tensor(35, (1, rows, cols), dtype, 0.1)}
    new = lambda *shape, d=dtype: torch.full(shape, float("nan"), dtype=d, device=DEV)
    out = {"rstd": new(rows, d=torch.float32), "n": new(1, rows, cols), "pre": new(2, rows, width), "dpre": new(2, rows, width), "h": new(1, rows, width),
           "z": new(1, rows, cols), "y": new(1, rows, cols), "dz": new(1, rows, cols), "dh": new(1, rows, width), "dw2": new(1, width, cols),
           "dn": new(1, rows, cols), "dw": new(2, cols, width), "dr": new(1, rows, cols), "dgain": new(cols)}
    return t, out


def _block64(t, drop_in, drop_out, eps=1e-6):
    v = {k: a.double() for k, a in t.items()}
    n, rstd = norm64(v["r"][0], v["gain"], eps)
    h, pre = gated64(n, v["w"], "silu", drop_in)
    y = v["r"][0] + dropped(drop_out, h @ v["w2"][0])
    dz = dropped(drop_out, v["dy"][0])
    dh, dw2 = dz @ v["w2"][0].t(), h.t() @ dz
    _, dn, dw = gated_back64(n, v["w"], pre, dh, "silu", drop_in)
    dr, dgain = norm_back64(v["r"][0], v["gain"], rstd, dn)
    return {"y": y, "dw2": dw2, "dw": dw, "dr": dr + v["dy"][0], "dgain": dgain}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 64, 128), (37, 96, 200), (300, 256, 520)], ids=str)
def test_block(ctx, sizes, dtype):
    """The operators together, as a training step calls them, against the whole block in 64 bits."""
    t, out = _block(dtype, *sizes)
    drop_in, drop_out = ops.Dropout(0.1, 91, 0), ops.Dropout(0.1, 91, 1)
    _block_step(ctx, dtype, t, drop_in, drop_out, out)
    # a chain of at most eight stored tensors, each off by u of its size, and sums whose errors average: eight half steps of the result's size
    tol = 8 * U[dtype] + 8 * PRODUCT[dtype]
    for k, want in _block64(t, drop_in, drop_out).items():
        got = out[k].double().reshape(want.shape)
        err = float((got - want).norm() / want.norm())
        assert err <= tol, "%s: %.3g > %.3g" % (k, err, tol)
    assert ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_block_captured_and_replayed(dtype):
    """The same step captured once on a stream of its own and replayed: same bits as the eager step; with a counter in device
    memory every replay draws its own masks; two graphs of one context replay one after the other; an eager step in between."""
    import deep8_b200
    c = deep8_b200.Context(0)
    side = torch.cuda.Stream()
    t, out = _block(dtype, 130, 1600, 264)  # split contractions among the gradients
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)
    d_in, d_out = ops.Dropout(0.2, 7, 0, counter), ops.Dropout(0.2, 7, 1 << 32, counter)
    c.use_stream(side)
    wanted = []
    with torch.cuda.stream(side):
        for step in range(3):
            counter.fill_(step)
            _block_step(c, dtype, t, ops.Dropout(0.2, 7, step), ops.Dropout(0.2, 7, (1 << 32) + step), out)  # eager, the offset given
            wanted.append({k: v.clone() for k, v in out.items()})
        side.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                _block_step(c, dtype, t, d_in, d_out, out)
                counter.add_(1)
            graphs.append(g)
        counter.zero_()
        for step in range(3):
            for v in out.values():
                v.fill_(float("nan"))
            graphs[step % 2].replay()
            side.synchronize()
            for k, v in out.items():
                assert k == "dpre" or torch.equal(v, wanted[step][k]), (step, k)  # dpre is workspace
            x = tensor(step, (1, 50, 1600), dtype)
            c.gated_forward(x, t["w"])  # eager use of the same context between replays
        assert int(counter) == 3
    assert c.status() == 0
    del graphs
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_odd_rows_captured(dtype):
    """Sizes whose rows are copied with padding: captured in a context that has no memory for the copies yet (kernels without copies run),
    then eagerly (the memory comes), then captured again, then a larger size while the older graph, which reads the older memory,
    is still replayed."""
    import deep8_b200
    c = deep8_b200.Context(0)
    side = torch.cuda.Stream()
    c.use_stream(side)
    sizes = [(70, 51, 133), (300, 1001, 2003)]
    with torch.cuda.stream(side):
        held = []
        for rows, cols, width in sizes:
            x, w = tensor(1, (1, rows, cols), dtype), tensor(2, (2, cols, width), dtype, cols ** -0.5)
            pre, dz = tensor(3, (2, rows, width), dtype), tensor(4, (1, rows, width), dtype, 0.1)
            for eager_first in (False, True):
                h, kept, dx, dw, dpre = (torch.empty_like(t) for t in (dz, pre, x, w, pre))

                def step():
                    c.gated_forward(x, w, "silu", out=h, pre=kept)
                    c.gated_backward(x, w, pre, dz, dx, dw, "silu", dpre=dpre, accumulate=False)

                if eager_first:
                    step()
                side.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side):
                    step()
                held.append((g, x, w, pre, dz, h, kept, dx, dw))
            for g, x, w, pre, dz, h, kept, dx, dw in held:
                for t in (h, kept, dx, dw):
                    t.fill_(float("nan"))
                g.replay()
                side.synchronize()
                check_gated(x, w, "silu", h, kept)
                check_backward(x, w, pre, dz, dx, dw, "silu", None)
    assert c.status() == 0
    del held, g
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 2048, 200), (5, 1024, 2048), (48, 1600, 264), (256, 4096, 512), (1000, 192, 320), (300, 1001, 2003)], ids=str)
def test_accumulating_calls_captured(sizes, dtype):
    """Kernels that join partial sums (in a cluster, by a last arrival, by tickets, by a second launch), captured and replayed with new inputs in
    the same memory and gradients that grow: the bits of the eager calls."""
    import deep8_b200
    rows, cols, width = sizes
    c = deep8_b200.Context(0)
    side = torch.cuda.Stream()
    c.use_stream(side)
    with torch.cuda.stream(side):
        x, w, dz = torch.empty(1, rows, cols, dtype=dtype, device=DEV), torch.empty(2, cols, width, dtype=dtype, device=DEV), tensor(3, (1, rows, width), dtype, 0.1)
        h, pre, dpre = torch.empty_like(dz), torch.empty(2, rows, width, dtype=dtype, device=DEV), torch.empty(2, rows, width, dtype=dtype, device=DEV)
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)

        def step():
            c.gated_forward(x, w, "gelu", out=h, pre=pre)
            c.gated_backward(x, w, pre, dz, dx, dw, "gelu", dpre=dpre)

        def fill(k):
            x.copy_(tensor(50 + k, x.shape, dtype))
            w.copy_(tensor(60 + k, w.shape, dtype, cols ** -0.5))

        wanted = []
        for k in range(3):
            fill(k)
            step()
            wanted.append([t.clone() for t in (h, pre, dx, dw)])
        side.synchronize()
        check_gated(x, w, "gelu", h, pre)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step()
        dx.zero_()
        dw.zero_()
        for k in range(3):
            fill(k)
            h.fill_(float("nan"))
            g.replay()
            side.synchronize()
            for got, want in zip((h, pre, dx, dw), wanted[k]):
                assert torch.equal(got, want), k
    assert c.status() == 0
    del g
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_backward_on_views_off_the_16_byte_boundary(ctx, dtype):
    rows, cols, width = 300, 256, 520

    def view(t, shift):
        whole = torch.full((t.numel() + 8,), 7.0, dtype=dtype, device=DEV)
        part = whole[shift:shift + t.numel()].view(t.shape)
        return whole, part.copy_(t)

    x, w = tensor(13, (1, rows, cols), dtype), tensor(14, (2, cols, width), dtype, 1.0 / 16)
    pre, dz = tensor(15, (2, rows, width), dtype), tensor(16, (1, rows, width), dtype, 0.1)
    zx, zw = torch.zeros_like(x), torch.zeros_like(w)
    for place in range(8):
        shifts = [(1 + k % 3) * (place in (k, 7)) for k in range(7)]
        parts = [view(t, s) for t, s in zip((x, w, pre, dz, zx, zw, pre), shifts)]
        (_, x1), (_, w1), (_, pre1), (_, dz1), (dx_all, dx), (dw_all, dw), (dpre_all, dpre) = parts
        ctx.gated_backward(x1, w1, pre1, dz1, dx, dw, "silu", dpre=dpre, accumulate=place % 2 == 0)
        check_backward(x, w, pre, dz, dx, dw, "silu", None)
        for whole, part, shift in ((dx_all, dx, shifts[4]), (dw_all, dw, shifts[5]), (dpre_all, dpre, shifts[6])):
            assert (whole[:shift] == 7).all() and (whole[shift + part.numel():] == 7).all()
    assert ctx.status() == 0


@pytest.mark.gpu
def test_padding_memory_grows_while_another_stream_is_captured():
    """Two contexts: one's call is captured while the other, on its own stream, needs more memory for its padded copies."""
    import deep8_b200
    a, b = deep8_b200.Context(0), deep8_b200.Context(0)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    a.use_stream(sa)
    b.use_stream(sb)
    x, w = tensor(1, (1, 48, 256), torch.float16), tensor(2, (2, 256, 512), torch.float16, 1.0 / 16)
    h = a.gated_forward(x, w)
    x1, w1 = tensor(3, (1, 40, 255), torch.float16), tensor(4, (2, 255, 511), torch.float16, 1.0 / 16)
    small = b.gated_forward(x1, w1)
    x2, w2 = tensor(5, (1, 40, 4095), torch.float16), tensor(6, (2, 4095, 2003), torch.float16, 1.0 / 64)  # 33 MB of copies
    large, out = torch.empty(1, 40, 2003, dtype=torch.float16, device=DEV), torch.empty_like(h)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=sa):
        a.gated_forward(x, w, out=out)
        b.gated_forward(x2, w2, out=large)
        a.dropout_forward(out, ops.Dropout(0.5, 1), out=out)
    torch.cuda.synchronize()
    check_gated(x1, w1, "silu", small, None)
    check_gated(x2, w2, "silu", large, None)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, a.dropout_forward(h, ops.Dropout(0.5, 1)))
    assert a.status() == 0 and b.status() == 0
    del g
    a.close()
    b.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_two_contexts_on_two_streams(dtype):
    """Each context owns its scratch memory, arrival words, tickets and padding memory: calls of two on two streams do not meet."""
    import deep8_b200
    held = [(deep8_b200.Context(0), torch.cuda.Stream()) for _ in range(2)]
    for sizes in ((1, 2048, 200), (5, 1024, 2048), (48, 1600, 264), (256, 1024, 512), (100, 1001, 203)):
        rows, cols, width = sizes
        calls = []
        for k, (c, stream) in enumerate(held):
            x, w = tensor(70 + k, (1, rows, cols), dtype), tensor(80 + k, (2, cols, width), dtype, cols ** -0.5)
            pre, dz, gain = tensor(90 + k, (2, rows, width), dtype), tensor(100 + k, (1, rows, width), dtype, 0.1), tensor(110 + k, (cols,), dtype)
            c.use_stream(stream)

            def call(c=c, x=x, w=w, pre=pre, dz=dz, gain=gain):
                dx, dw, dgain, rstd = torch.empty_like(x), torch.empty_like(w), torch.empty_like(gain), torch.empty(x.shape[1], device=DEV)
                n = c.rms_norm_forward(x, gain, rstd=rstd)
                h = c.gated_forward(n, w)
                c.gated_backward(n, w, pre, dz, dx, dw, accumulate=False)
                dn = torch.empty_like(x)
                c.rms_norm_backward(x, gain, rstd, dn, dgain, dx, accumulate=False)
                return h, dx, dw, dn, dgain

            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                alone = call()
            torch.cuda.synchronize()
            calls.append((call, stream, alone))
        together = []
        for _ in range(4):
            for call, stream, alone in calls:
                with torch.cuda.stream(stream):
                    together.append((call(), alone))
        torch.cuda.synchronize()
        for got, want in together:
            assert all(torch.equal(g, w) for g, w in zip(got, want)), sizes
    for c, _ in held:
        assert c.status() == 0
        c.close()


@pytest.mark.gpu
def test_gated_beyond_32_bit_offsets(ctx):
    """More than 2^32 elements of h: the last rows, with dropout, against the plain form."""
    rows, cols, width = 66000, 64, 66048
    x = torch.randn(1, rows, cols, device=DEV, dtype=torch.float32, generator=torch.Generator(DEV).manual_seed(1)).half()
    w = tensor(41, (2, cols, width), torch.float16, 0.125)
    drop = ops.Dropout(0.1, 3, 5)
    h = ctx.gated_forward(x, w, "silu", dropout=drop)
    for first in (0, 65020, rows - 3):  # the rows around element 2^32 and the last ones
        part = ctx.gated_forward(x[:, first:first + 3].contiguous(), w, "silu")[0].double()
        keep = keep_mask(drop, (3, width), first * width).to(DEV)
        got = h[0, first:first + 3].double()
        assert (got[~keep] == 0).all()
        want = part[keep] / 0.9
        # both sides are rounded to fp16 once (2 u) and may add their 64 products in different orders: |x w| <= 5.5 * 0.7 in each, so the
        # sums differ by 2 * 64 * 2^-23 * 64 * 3.9 < 2^-8.0 at the very most, times the other factor (below 16)
        assert ((got[keep] - want).abs() <= want.abs() * 2.0 ** -9.9 + 2.0 ** -8 * 16).all()
    assert ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["sigmoid", "silu"])
def test_gates_far_below_zero(ctx, name):
    """fp32 gates between -87 and -64, whose sigmoids are small but normal numbers, times an up projection of 2^100.  Gates of ten bits: their
    products with 1 and 2^100 are exact.  The exponential is off by 2^-22, at most four operations and four more of the product by 2^-24."""
    a = torch.arange(-87.0, -64.0, 0.125, dtype=torch.float64)
    w = torch.tensor([1.0, 2.0 ** 100], device=DEV).view(2, 1, 1).repeat(1, 1, 4)
    for rows in (a.numel(), 5):  # the tensor cores, the streaming kernel
        x = a[:rows].float().to(DEV).view(1, rows, 1)
        h64 = gated64(x[0].double(), w.double(), name)[0]
        within(ctx.gated_forward(x, w, name)[0], h64, stored(h64, h64.abs() * 2.0 ** -21, torch.float32), "h")
    gate = x.new_tensor(a.tolist()).view(1, 1, -1)
    pre, dz = torch.cat((gate, torch.full_like(gate, 2.0 ** 100))), torch.ones_like(gate)
    value, slope = act64(name, gate[0].double())
    want = torch.stack((slope * 2.0 ** 100, value))
    within(ctx.gated_grad_pre(pre, dz, name), want, stored(want, want.abs() * 2.0 ** -20, torch.float32), "dpre")


def _slopes64(name, dtype, limit):
    """Gates on both sides from 3 to `limit`, the plain form's slopes, and how far a slope may be off, relative to it.  One exponential e is off
    by 2^-22 (fp32) or (2 + 1.2 |z|) 2^-23 (the fast one of fp16), enters s (1 - s) = e / (1 + e)^2 at most twice, beside at most four
    divisions and products of 2^-22 (fast) each.  silu and gelu_tanh: z is the gate or gelu_tanh's polynomial in it, whose own
    rounding moves the exponential by |z| 2^-22; outside +-3 their two terms cancel to no less than a third of their sizes."""
    a = torch.linspace(3.0, limit, 4001, dtype=torch.float64).to(dtype)
    a = torch.cat((a, -a)).to(DEV)
    a64 = a.double()
    slope = act64(name, a64)[1]
    z = a64.abs() if name != "gelu_tanh" else 2 * math.sqrt(2 / math.pi) * (a64.abs() + 0.044715 * a64.abs() ** 3)
    e = 2 * (2.0 ** -22 if dtype == torch.float32 else (2 + 1.2 * z) * 2.0 ** -23) + 4 * 2.0 ** -22
    if name != "sigmoid":
        e = 3 * (e + (2 * z * 2.0 ** -22 if name == "gelu_tanh" else 0.0))
    return a, slope, e


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["sigmoid", "silu", "gelu_tanh"])
def test_gradients_of_saturated_gates(ctx, name, dtype):
    """act' relative to itself where 1 - sigmoid(a) is far below the spacing of floats around 1."""
    a, slope, e = _slopes64(name, dtype, 30.0 if dtype == torch.float32 else 16.0)
    factor = 512.0 if name == "sigmoid" else 1.0  # keeps fp16's dpre normal
    pre = torch.stack((a, torch.full_like(a, factor))).view(2, 1, -1)
    got = ctx.gated_grad_pre(pre, torch.full_like(pre[:1], factor), name)
    want = slope * factor * factor
    within(got[0, 0], want, stored(want, want.abs() * (e + 2.0 ** -23), dtype), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
def test_a_nan_gate_stays_visible(ctx, name, dtype):
    """A NaN among the gate's weights makes that column of h NaN whatever the activation, and its gradients of the up projection."""
    for rows in (1, 6, 40, 300):
        x, w = tensor(51, (1, rows, 64), dtype), tensor(52, (2, 64, 72), dtype, 0.1)
        w[0, 5, 3] = float("nan")
        pre = torch.empty(2, rows, 72, dtype=dtype, device=DEV)
        h = ctx.gated_forward(x, w, name, pre=pre)
        column = torch.arange(72, device=DEV) == 3
        assert torch.equal(torch.isnan(h[0]), column.expand(rows, 72)) and not torch.isnan(pre[1]).any()
        dpre = ctx.gated_grad_pre(pre, torch.ones_like(h), name)
        assert torch.equal(torch.isnan(dpre[1]), column.expand(rows, 72))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("accumulate", [0, 1])
@pytest.mark.parametrize("sizes", [(700, 512, 520), (2000, 1024, 1000), (333, 250, 1001), (300, 256, 512), (64, 72, 4104), (1500, 250, 2056),
                                   (4096, 1024, 1000)], ids=str)
def test_gradient_products_by_themselves(ctx, sizes, accumulate, dtype):
    """d8k_gated_grad_x_into and d8k_gated_grad_w_into, which take dpre as it lies in the caller's memory."""
    lib, p = _lib.load(), ops._p
    rows, xc, yc = sizes
    x, w, dpre = tensor(61, (1, rows, xc), dtype), tensor(62, (2, xc, yc), dtype, yc ** -0.5), tensor(63, (2, rows, yc), dtype)
    dx0, dw0 = tensor(64, (1, rows, xc), dtype), tensor(65, (2, xc, yc), dtype)
    dx, dw, kept = dx0.clone(), dw0.clone(), dpre.clone()
    code = 0 if dtype == torch.float16 else 1
    before = ctx.launch_count()
    assert lib.d8k_gated_grad_x_into(ctx.h, code, p(dx), 1, rows, xc, p(w), yc, p(dpre), accumulate) == 0
    # yc: rows that TMA reads as they are, but no whole 128-byte pieces.  Without a padded dpre the paired kernel, for which w or x would be copied
    # with padding, cannot run.
    copies_in_vain = dtype == torch.float16 and yc % 8 == 0 and yc % 64 != 0
    if copies_in_vain:
        assert ctx.launch_count() - before == 1
    before = ctx.launch_count()
    assert lib.d8k_gated_grad_w_into(ctx.h, code, p(x), 1, rows, xc, p(dw), yc, p(dpre), accumulate) == 0
    if copies_in_vain and xc % 8 == 0:
        assert ctx.launch_count() - before == 1
    x64, w64, d64 = x[0].double(), w.double(), dpre.double()
    for got, want, size, n, old in ((dx[0], torch.matmul(d64, w64.transpose(1, 2)).sum(0), torch.matmul(d64.abs(), w64.abs().transpose(1, 2)).sum(0), 2 * yc, dx0[0]),
                                    (dw, torch.matmul(x64.t(), d64), torch.matmul(x64.abs().t(), d64.abs()), rows, dw0)):
        err = size * (PRODUCT[dtype] + n * 2.0 ** -23)
        if accumulate:
            want = want + old.double()
            err = err + want.abs() * 2.0 ** -23
        within(got, want, stored(want, err, dtype))
    assert torch.equal(dpre, kept) and ctx.status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_backward_with_shifted_workspace_of_whole_pieces(dtype):
    """A workspace off the 16-byte boundary whose rows are whole 128-byte pieces: the copy's rows have nothing behind them to clear.  Eagerly and
    captured."""
    import deep8_b200
    c, side = deep8_b200.Context(0), torch.cuda.Stream()
    c.use_stream(side)
    rows, cols, width = 40, 96, 192
    with torch.cuda.stream(side):
        x, w = tensor(1, (1, rows, cols), dtype), tensor(2, (2, cols, width), dtype, 0.1)
        pre, dz = tensor(3, (2, rows, width), dtype), tensor(4, (1, rows, width), dtype, 0.1)
        whole = torch.full((pre.numel() + 8,), 7.0, dtype=dtype, device=DEV)
        dpre, dx, dw = whole[1:1 + pre.numel()].view(pre.shape), torch.empty_like(x), torch.empty_like(w)
        step = lambda: c.gated_backward(x, w, pre, dz, dx, dw, "silu", dpre=dpre, accumulate=False)
        step()
        check_backward(x, w, pre, dz, dx, dw, "silu", None)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step()
        dx.fill_(float("nan"))
        dw.fill_(float("nan"))
        g.replay()
        check_backward(x, w, pre, dz, dx, dw, "silu", None)
        assert whole[0] == 7 and (whole[1 + pre.numel():] == 7).all()
    assert c.status() == 0
    del g
    c.close()


@pytest.mark.gpu
def test_device_generator_against_raw_counters(ctx):
    """The device's decisions for the first groups, bit by bit: with p = 1/2 an element stays when its word's top bit is set; p = 2^-k masks the
    bits further down."""
    seed, offset = 0x299f31d0a4093822, 0x0370734413198a2e
    words = [w for group in range(64) for w in _philox_raw([group, 0, offset & 0xFFFFFFFF, offset >> 32], [seed & 0xFFFFFFFF, seed >> 32])]
    for p in (0.5, 0.25, 1.0 / 3, 0.9, 2.0 ** -32, 1.0 - 2.0 ** -32):
        y = ctx.dropout_forward(torch.ones(256, device=DEV), ops.Dropout(p, seed, offset))
        assert [bool(v) for v in (y != 0).tolist()] == [w >= round(p * 2 ** 32) for w in words], p


@pytest.mark.gpu
def test_dropout_beyond_the_counters_low_word():
    """2^34 elements and more: their groups no longer fit the counter's first word, and a second launch takes them.  In place, 34 GB."""
    import deep8_b200
    n = (1 << 34) + 4099
    if torch.cuda.mem_get_info()[0] < 2 * n + (2 << 30):
        pytest.skip("needs 36 GB of device memory")
    c = deep8_b200.Context(0)
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    drop = ops.Dropout(0.5, 17, 3)
    c.dropout_forward(x, drop, out=x)
    for first, count in ((0, 4000), ((1 << 34) - 100, 4099), (n - 3, 3)):
        assert torch.equal(x[first:first + count], keep_mask(drop, (count,), first).to(DEV).half() * 2), first
    c.close()
    del x
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scratch", [4096, 1 << 20])
def test_contexts_with_little_scratch_memory(scratch, dtype):
    """Plans that would split a contraction have to do with what the context was given."""
    import deep8_b200
    c = deep8_b200.Context(0, scratch)
    for rows, xc, yc in ((1, 4096, 512), (7, 2048, 1032), (48, 1600, 264), (127, 1000, 504), (300, 512, 520), (256, 4096, 128), (700, 512, 2048)):
        x, w = tensor(1, (1, rows, xc), dtype), tensor(2, (2, xc, yc), dtype, xc ** -0.5)
        pre = torch.empty(2, rows, yc, dtype=dtype, device=DEV)
        h = c.gated_forward(x, w, "silu", pre=pre)
        check_gated(x, w, "silu", h, pre)
        pre, dz = tensor(3, (2, rows, yc), dtype), tensor(4, (1, rows, yc), dtype, 0.1)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        c.gated_backward(x, w, pre, dz, dx, dw, "silu", accumulate=False)
        check_backward(x, w, pre, dz, dx, dw, "silu", None)
    rows, cols = 600, 1000
    x, weight, dy, rstd = tensor(5, (rows, cols), dtype), tensor(6, (cols,), dtype), tensor(7, (rows, cols), dtype), torch.empty(rows, device=DEV)
    c.rms_norm_forward(x, weight, rstd=rstd)
    dx, dweight = torch.empty_like(x), torch.empty_like(weight)
    c.rms_norm_backward(x, weight, rstd, dx, dweight, dy, accumulate=False)
    want_x, want_w = norm_back64(x.double(), weight.double(), rstd.double(), dy.double())
    n = (x.double() * rstd.double()[:, None]).abs()
    u = (dy.double() * weight.double()).abs()
    within(dx, want_x, stored(want_x, rstd.double()[:, None] * (u * 2.0 ** -21 + n * (u * n).mean(1, keepdim=True) * (cols * 2.0 ** -23 + 2.0 ** -20)), dtype), "dx")
    within(dweight, want_w, stored(want_w, (dy.double().abs() * n).sum(0) * (rows * 2.0 ** -23 + 2.0 ** -20), dtype), "dweight")
    assert c.status() == 0
    c.close()


@pytest.mark.gpu
def test_cpp_nodes():
    """The C++ nodes (tests/cpp/test_feedforward_host.cu): the block as a graph, forward and backward walk."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "test_feedforward_host")
    assert os.path.exists(exe), "tests/cpp/bin/test_feedforward_host is missing: run __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.gpu
def test_cpp_node_graphs():
    """Graphs of several blocks and shared variables, both types, every activation (tests/cpp/test_feedforward_nodes.cu)."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "test_feedforward_nodes")
    assert os.path.exists(exe), "tests/cpp/bin/test_feedforward_nodes is missing: run __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
