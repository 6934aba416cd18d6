"""4-bit projections, rotary positions and shared-prefix attention on the GPU,
against plain forms in float64.

Tolerances.  A rounding to bf16 is off by at most U = 2^-8 of the value, to fp16
2^-11, to fp32 2^-24.

* linear_w4: products of exact operands summed in fp32.  An element's terms are
  (16 + c) x and (16 + z) x, at most 31 |x| each, scaled by s; it passes at most
  32 sums in an MFMA, 4 in a group, 2 in the correction, K / G over the groups
  and 8 over the waves: (48 + K / G) 2^-24 62 sum |x| s, then U |y|.  Where the
  zeros' part is a product of its own, the K / G sums over the groups come twice
  but hold one of the two terms more than the other for at most four groups: what
  they round is at most 31 |x| s in all, and the bound is the same.
* rotary: sine and cosine are off by at most 2^-22 (truncation 3e-8 and a few
  roundings below one), the products and sums by three roundings:
  2^-21 factor (|x| + |y|), then the type's own rounding.
* attention: a probability is rounded to bf16 (U each), its fp32 score and
  exponential are off by less than 2e-4 of it (128 products of operands of
  about one, exp2 to a few ulps): (U + 2e-4) sum p |v| / l, then U |o|.
"""
import ctypes
import math
import random

import pytest
import torch

from nanovllm_amd import kernels as K
from nanovllm_amd.layers import rope_frequencies

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -8
D = 128


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    over = (got - want).abs() - tol.double().cpu()
    assert torch.isfinite(got).all()
    assert over.max() <= 0, f"off by {float(over.max()):.3g} more than allowed"


# ---------------------------------------------------------------- linear_w4

def w4_case(rows, n, k, group, zeros, bias, seed=0):
    g = gen(seed)
    x = torch.randn(rows, k, generator=g, device="cuda").to(BF16)
    qw = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.randn(k // group, n, generator=g, device="cuda") * 0.02).to(BF16)
    z = torch.randint(0, 16, (k // group, n), generator=g, device="cuda",
                      dtype=torch.uint8) if zeros else None
    b = torch.randn(n, generator=g, device="cuda").to(BF16) if bias else None
    return x, qw, s, z, b


def w4_reference(x, qw, s, z, b):
    n, k = qw.shape[0], 2 * qw.shape[1]
    group = k // s.shape[0]
    c = torch.empty(n, k, dtype=torch.float64, device=qw.device)
    c[:, 0::2], c[:, 1::2] = (qw & 15).double(), (qw >> 4).double()
    zz = torch.full_like(s, 8.0).double() if z is None else z.double()
    step = s.double().t().repeat_interleave(group, 1)
    w = (c - zz.t().repeat_interleave(group, 1)) * step
    y = x.double() @ w.t()
    if b is not None:
        y = y + b.double()
    terms = x.double().abs() @ step.abs().t()
    return y, U * y.abs() + (48 + k // group) * 2.0 ** -24 * 62 * terms


@pytest.mark.parametrize("rows,n,k,group", [
    (1, 16, 32, 32), (1, 1, 64, 64), (2, 7, 96, 32), (3, 33, 128, 128), (4, 100, 160, 32),
    (5, 18, 192, 64), (8, 130, 256, 128), (15, 64, 1024, 128), (16, 255, 544, 32),
    (17, 48, 384, 64), (31, 20, 1152, 128), (32, 512, 2048, 256), (33, 96, 640, 32),
    (61, 77, 1280, 64), (64, 260, 4096, 128), (65, 34, 320, 32), (130, 50, 768, 384),
    (1, 4096, 4096, 128), (6, 1030, 4160, 64), (16, 2048, 2560, 32), (1, 40, 96, 96),
    (17, 5000, 544, 32), (20, 9000, 288, 96), (24, 2500, 1088, 64), (40, 1100, 6400, 256),
    (48, 16400, 512, 128), (64, 8200, 1056, 32), (64, 600, 9728, 128), (81, 4000, 2080, 32),
    (130, 700, 4416, 64), (257, 130, 2048, 128)])
@pytest.mark.parametrize("zeros,bias", [(False, False), (True, True)])
def test_linear_w4(cuda, rows, n, k, group, zeros, bias):
    case = w4_case(rows, n, k, group, zeros, bias, seed=rows + n)
    want, tol = w4_reference(*case)
    close(K.linear_w4(*case), want, tol)


def test_linear_w4_strides_out_and_alignment(cuda):
    x, qw, s, z, b = w4_case(9, 36, 256, 64, True, True)
    want, tol = w4_reference(x, qw, s, z, b)
    wide = torch.zeros(9, 300, dtype=BF16, device="cuda")
    for at in (0, 3, 8):            # rows on odd strides and addresses are taken too
        view = wide[:, at:at + 256]
        view.copy_(x)
        close(K.linear_w4(view, qw, s, z, b), want, tol)
    columns = x.t().contiguous().t()
    close(K.linear_w4(columns, qw, s, z, b), want, tol)
    out = torch.full((9, 41), 7.0, dtype=BF16, device="cuda")
    got = K.linear_w4(x, qw, s, z, b, out=out[:, 2:38])
    assert got.data_ptr() == out[:, 2:].data_ptr()
    close(out[:, 2:38], want, tol)
    assert (out[:, :2] == 7).all() and (out[:, 38:] == 7).all()


def test_linear_w4_codes_past_two_to_the_31_bytes(cuda):
    n, k, group = 215000, 20480, 128
    qw = torch.randint(0, 256, (n, k // 2), generator=gen(11), device="cuda", dtype=torch.uint8)
    assert qw.numel() > 2 ** 31
    s = (torch.randn(k // group, n, generator=gen(12), device="cuda") * 0.02).to(BF16)
    for rows in (3, 20):
        x = torch.randn(rows, k, generator=gen(rows), device="cuda").to(BF16)
        got = K.linear_w4(x, qw, s)
        for at in (0, 104800, n - 48):
            part = slice(at, at + 48)
            want, tol = w4_reference(x, qw[part], s[:, part], None, None)
            close(got[:, part], want, tol)


@pytest.mark.parametrize("rows,k", [(33, 288), (64, 256), (17, 5440)])
def test_linear_w4_rows_far_apart(cuda, rows, k):
    """Columns of a wide tensor up to the largest stride that the kernel takes
    and past it, NaN around them: nothing beside a row comes into its sum."""
    x, qw, s, z, b = w4_case(rows, 36, k, 32, True, True)
    want, tol = w4_reference(x, qw, s, z, b)
    for stride in ((1 << 24) - 8, 1 << 24):
        flat = torch.full((rows * stride,), float("nan"), dtype=BF16, device="cuda")
        far = flat.view(rows, stride)[:, 128:128 + k]
        far.copy_(x)
        close(K.linear_w4(far, qw, s, z, b), want, tol)
        del flat, far


def test_linear_w4_a_bad_row_stays_alone_in_a_slab(cuda):
    for rows, n in ((29, 4100), (70, 70)):
        x, qw, s, z, b = w4_case(rows, n, 512, 64, True, False)
        want, tol = w4_reference(x, qw, s, z, b)
        bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
        bad[::9] = True
        x[::9, 7::100], x[::18, 300] = float("inf"), float("nan")
        got = K.linear_w4(x, qw, s, z, b)
        assert got[bad].isnan().all()
        close(got[~bad], want[~bad], tol[~bad])


def test_linear_w4_a_bad_row_stays_alone(cuda):
    x, qw, s, z, b = w4_case(5, 40, 256, 128, True, False)
    want, tol = w4_reference(x, qw, s, z, b)
    x[1, 7], x[3, 200] = float("inf"), float("nan")
    got = K.linear_w4(x, qw, s, z, b)
    assert got[1].isnan().all() and got[3].isnan().all()
    keep = torch.tensor([0, 2, 4], device="cuda")
    close(got[keep], want[keep], tol[keep])


@pytest.mark.parametrize("rows,n,k,group", [
    (1, 40, 256, 128), (4, 130, 1024, 32), (9, 64, 4096, 64), (16, 70, 8192, 128), (17, 100, 1024, 128),
    (33, 72, 2048, 32), (64, 130, 4096, 64), (70, 40, 672, 96)])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_w4_large_finite_x(cuda, rows, n, k, group, zeros):
    """x up to bf16's largest value: outputs are finite where their definition is."""
    x, qw, s, z, b = w4_case(rows, n, k, group, zeros, True)
    s = (s * 0.01).clamp(-6e-4, 6e-4)
    top = torch.finfo(BF16).max
    x[0, :group] = top                          # a whole group of one sign
    x[rows // 2, 7], x[rows - 1, k - 1] = 1e37, -top
    want, tol = w4_reference(x, qw, s, z, b)
    assert (want.abs() < top).all()
    close(K.linear_w4(x, qw, s, z, b), want, tol)


def test_linear_w4_out_over_an_input_is_refused(cuda):
    x, qw, s, z, b = w4_case(6, 128, 128, 64, True, True)
    want = K.linear_w4(x, qw, s, z, b)
    flat = torch.zeros(6 * 128 + 64, dtype=BF16, device="cuda")
    moved = flat[:6 * 128].view(6, 128)
    moved.copy_(x)
    scales = torch.zeros(2 * 128 + 8, dtype=BF16, device="cuda")
    scales[:2 * 128] = s.flatten()
    held = scales[:2 * 128].view(2, 128)
    codes = qw.clone()
    for args, out in [((moved, qw, s, z, b), moved), ((moved, qw, s, z, b), flat[64:].view(6, 128)),
                      ((x[:1], qw, held, z, b), scales[8:136].view(1, 128)),
                      ((x, codes, s, z, b), codes.view(-1).view(BF16)[:6 * 128].view(6, 128)),
                      ((x[:1], qw, s, z, held[0]), held[:1])]:
        with pytest.raises(ValueError, match="overlap"):
            K.linear_w4(*args, out=out)
    assert torch.equal(moved, x)
    # x and out as different columns of the same rows do not
    both = torch.zeros(6, 272, dtype=BF16, device="cuda")
    both[:, :128] = x
    assert torch.equal(K.linear_w4(both[:, :128], qw, s, z, b, out=both[:, 136:264]), want)
    assert torch.equal(both[:, :128], x) and (both[:, 128:136] == 0).all()


def test_linear_w4_empty(cuda):
    x, qw, s, z, b = w4_case(3, 8, 64, 32, False, False)
    assert K.linear_w4(x[:0], qw, s).shape == (0, 8)
    assert K.linear_w4(x, qw[:0], s[:, :0].contiguous()).shape == (3, 0)


@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (256, True)])
def test_quantized_weights(cuda, group, zeros):
    w = torch.randn(72, 768, generator=gen(1), device="cuda").to(BF16) * 0.05
    w[3] = 0                        # a group of zeros has scale zero
    qw, s, z = K.quantize_w4(w, group, zeros)
    x = torch.randn(4, 768, generator=gen(2), device="cuda").to(BF16)
    want, tol = w4_reference(x, qw, s, z, None)
    close(K.linear_w4(x, qw, s, z), want, tol)
    assert (K.linear_w4(x, qw, s, z)[:, 3] == 0).all()


def test_linear_w4_refusals(cuda):
    x, qw, s, z, b = w4_case(3, 8, 128, 64, True, True)
    bad = [(x.float(), qw, s, z, b), (x[0], qw, s, z, b), (x[:, :96].contiguous(), qw, s, z, b),
           (x, qw.to(torch.int8), s, z, b), (x, qw[:, :32], s, z, b), (x, qw, s.float(), z, b),
           (x, qw, s[:, :4], z, b), (x, qw, s.t().contiguous().t(), z, b),
           (x, qw, s, z.int(), b), (x, qw, s, z[:1], b), (x, qw, s, z, b.float()),
           (x, qw, s, z, b[:4]), (x.cpu(), qw, s, z, b), (x, qw, s.cpu(), z, b),
           (x, qw, torch.ones(8, 8, dtype=BF16, device="cuda"), None, b)]   # groups of 16
    for args in bad:
        with pytest.raises((ValueError, TypeError)):
            K.linear_w4(*args)
    for out in (torch.empty(3, 9, dtype=BF16, device="cuda"), torch.empty(3, 8, device="cuda"),
                torch.empty(8, 3, dtype=BF16, device="cuda").t(),
                torch.empty(1, 8, dtype=BF16, device="cuda").expand(3, 8)):
        with pytest.raises(ValueError):
            K.linear_w4(x, qw, s, z, b, out=out)
    with pytest.raises(ValueError, match="gradients"):
        K.linear_w4(x.clone().requires_grad_(), qw, s, z, b)


# ---------------------------------------------------------------- rotary positions

HALF_STEP = {BF16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotary_reference(x, positions, freq, interleaved, factor):
    """(rotated heads, tolerance) in float64."""
    rot = 2 * freq.numel()
    a = positions.double()[:, None, None] * freq.double()
    y = x.double().clone()
    p = y[..., :rot]
    u, v = (p[..., 0::2], p[..., 1::2]) if interleaved else (p[..., :rot // 2], p[..., rot // 2:])
    ru, rv = factor * (u * a.cos() - v * a.sin()), factor * (v * a.cos() + u * a.sin())
    size = (u.abs() + v.abs()) * abs(factor)
    tol = torch.zeros_like(y)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ru.clone(), rv.clone()
        tol[..., 0:rot:2] = tol[..., 1:rot:2] = size
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = ru.clone(), rv.clone()
        tol[..., :rot // 2] = tol[..., rot // 2:rot] = size
    rounding = torch.where(tol > 0, HALF_STEP[x.dtype] * y.abs(), 0.0)
    if x.dtype == torch.float16:
        # below its least normal value 2^-14 fp16 keeps steps of 2^-24: a
        # rounding there is off by up to 2^-25 whatever the value
        rounding = torch.where(tol > 0, rounding.clamp(min=2.0 ** -25), 0.0)
    return y, 2.0 ** -21 * tol + rounding


def test_rotary_in_place_turns_once_where_an_earlier_error_is_reported(cuda):
    """An error that another call has left (here a device number that does not
    exist) is reported by the launch that follows it; q and k are rotated all the
    same, and only once."""
    hip = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    hip = ctypes.CDLL(hip)
    q = torch.randn(3, 4, 64, generator=gen(5), device="cuda")
    k = torch.randn(3, 2, 64, generator=gen(6), device="cuda")
    pos = torch.tensor([1, 5, 9], device="cuda")
    freq = torch.rand(32, generator=gen(7), device="cuda", dtype=torch.float64)
    want = K.rotary_embedding(pos, q, k, freq)
    rows = torch.cat([q, k], 1)
    qi, ki = rows[:, :4], rows[:, 4:]
    torch.cuda.synchronize()
    assert hip.hipSetDevice(1 << 20) != 0
    with pytest.raises(RuntimeError):
        K.rotary_embedding(pos, qi, ki, freq, q_out=qi, k_out=ki)
    assert torch.equal(qi, want[0]) and torch.equal(ki, want[1])
    K.rotary_embedding(pos, q, k, freq)      # nothing stays behind


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,hq,hk,d,rot", [
    (1, 16, 8, 128, 128), (1, 1, 1, 2, 2), (3, 5, 1, 64, 32), (7, 24, 4, 128, 64),
    (129, 32, 8, 128, 128), (33, 6, 2, 80, 20), (17, 3, 3, 96, 24), (5, 7, 2, 192, 96),
    (4, 2, 1, 256, 256), (2, 3, 1, 512, 512), (2, 1, 1, 1024, 10), (6, 2, 0, 20, 14)])
def test_rotary(cuda, interleaved, dtype, t, hq, hk, d, rot):
    g = gen(t + d)
    q = torch.randn(t, hq, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(t, hk, d, generator=g, device="cuda").to(dtype) if hk else None
    pos = torch.randint(0, 131072, (t,), generator=g, device="cuda")
    pos[0] = 0 if t > 1 else 131071
    freq = rope_frequencies(rot, 10000.0)[0].cuda()
    qo, ko = K.rotary_embedding(pos, q, k, freq, interleaved=interleaved, factor=1.25)
    close(qo, *rotary_reference(q, pos, freq, interleaved, 1.25))
    assert (ko is None) == (k is None)
    if k is not None:
        close(ko, *rotary_reference(k, pos, freq, interleaved, 1.25))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_far_positions_and_quadrants(cuda, interleaved):
    # all four quadrants, their borders, negative and far positions, in float32
    pos = torch.tensor([0, 1, 2, 3, 4, 5, 6, -1, -7, 11, 999983, 2 ** 24 + 1, 2 ** 31 + 5],
                       device="cuda")
    x = torch.randn(13, 2, 64, generator=gen(5), device="cuda")
    freq = torch.cat([torch.tensor([math.pi / 2, math.pi / 4, math.pi, 1.0], dtype=torch.float64),
                      rope_frequencies(56, 1e6)[0]]).cuda()
    got, _ = K.rotary_embedding(pos, x, None, freq, interleaved=interleaved)
    want, tol = rotary_reference(x, pos, freq, interleaved, 1.0)
    # an angle p f is one rounding of float64 off: 2^-53 of it
    angle = pos.double().abs().max() * freq.max() * 2.0 ** -53
    close(got, want, tol + 2 * angle * x.abs().max().double())


@pytest.mark.parametrize("dtype,interleaved", [(BF16, False), (BF16, True), (torch.float32, False)])
@pytest.mark.parametrize("rot", [128, 64, 12])
def test_rotary_views_and_in_place(cuda, dtype, interleaved, rot):
    t, hq, hk, d = 19, 8, 2, 128
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=gen(3), device="cuda").to(dtype)
    before = qkv.clone()
    q, k = qkv[:, :hq * d].view(t, hq, d), qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
    pos = torch.randint(0, 40960, (t,), generator=gen(4), device="cuda")
    freq = rope_frequencies(rot, 1e6)[0].cuda()
    wq = rotary_reference(q, pos, freq, interleaved, 1.0)
    wk = rotary_reference(k, pos, freq, interleaved, 1.0)
    qo, ko = K.rotary_embedding(pos, q, k, freq, interleaved)
    assert qo.is_contiguous() and ko.is_contiguous() and torch.equal(qkv, before)
    close(qo, *wq)
    close(ko, *wk)
    # head-major outputs, and one head apart from the next by an odd number
    q2 = torch.zeros(hq, t, d, dtype=dtype, device="cuda").transpose(0, 1)
    k2 = torch.zeros(t, hk, d + 3, dtype=dtype, device="cuda")[:, :, 1:d + 1]
    K.rotary_embedding(pos, q, k, freq, interleaved, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    # in place
    q3, k3 = K.rotary_embedding(pos, q, k, freq, interleaved, 1.0, q, k)
    assert q3.data_ptr() == q.data_ptr() and torch.equal(q3, qo) and torch.equal(k3, ko)
    assert torch.equal(qkv[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
@pytest.mark.parametrize("t,hq,hk,d,rot", [
    (3, 2, 1, 65, 64), (1, 1, 1, 3, 2), (5, 4, 2, 33, 32), (4, 3, 1, 129, 64), (2, 2, 2, 1023, 512),
    (7, 5, 1, 67, 6), (260, 8, 1, 65, 62)])
def test_rotary_odd_heads_are_whole(cuda, interleaved, dtype, t, hq, hk, d, rot):
    g = gen(d + rot)
    q = torch.randn(t, hq, d, generator=g, device="cuda").to(dtype)
    k = torch.randn(t, hk, d, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 40960, (t,), generator=g, device="cuda")
    freq = rope_frequencies(rot, 10000.0)[0].cuda()
    # one element more behind each head, which stays
    qo, ko = (torch.full((t, h, d + 1), float("nan"), dtype=dtype, device="cuda") for h in (hq, hk))
    K.rotary_embedding(pos, q, k, freq, interleaved, q_out=qo[..., :d], k_out=ko[..., :d])
    for x, out in ((q, qo), (k, ko)):
        close(out[..., :d], *rotary_reference(x, pos, freq, interleaved, 1.0))
        assert torch.equal(out[..., rot:d], x[..., rot:]) and out[..., d].isnan().all()
    # in place, whole heads side by side
    both = torch.cat([q, k], 1)
    K.rotary_embedding(pos, both[:, :hq], both[:, hq:], freq, interleaved, q_out=both[:, :hq],
                       k_out=both[:, hq:])
    assert torch.equal(both, torch.cat([qo[..., :d], ko[..., :d]], 1))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, torch.float16, torch.float32])
def test_rotary_heads_at_every_alignment(cuda, interleaved, dtype):
    """Heads that begin 1 to 16 elements behind a 16-byte border, with and without
    elements behind the rotated ones."""
    t, h = 5, 3
    for d, rot in ((64, 32), (64, 64), (40, 16), (24, 8)):
        pos = torch.randint(0, 40960, (t,), generator=gen(d), device="cuda")
        freq = rope_frequencies(rot, 10000.0)[0].cuda()
        for at in (1, 2, 4, 8, 16):
            for gap in (0, 1, 2, 4, 8):
                row = torch.randn(t, h, d + gap, generator=gen(at), device="cuda").to(dtype)
                store = torch.zeros(row.numel() + at, dtype=dtype, device="cuda")
                x = store[at:].view(t, h, d + gap)
                x.copy_(row)
                out = torch.full_like(store, float("nan"))[at:].view(t, h, d + gap)
                K.rotary_embedding(pos, x[..., :d], None, freq, interleaved, q_out=out[..., :d])
                close(out[..., :d], *rotary_reference(x[..., :d], pos, freq, interleaved, 1.0))
                assert out[..., d:].isnan().all()


def test_rotary_nothing_to_do(cuda):
    freq = rope_frequencies(64, 1e4)[0].cuda()
    x = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
    qo, ko = K.rotary_embedding(torch.empty(0, dtype=torch.int64, device="cuda"), x, x, freq)
    assert qo.shape == ko.shape == (0, 4, 64)


def test_rotary_refusals(cuda):
    x = torch.randn(4, 2, 64, device="cuda").to(BF16)
    pos = torch.arange(4, device="cuda")
    freq = rope_frequencies(64, 1e4)[0].cuda()
    for args in [(pos.int(), x, x, freq), (pos[:3], x, x, freq), (pos, x, x, freq.float()),
                 (pos, x, x[:, :, :32], freq), (pos, x, x.float(), freq), (pos, x, x[:3], freq),
                 (pos, x[:, 0], None, freq), (pos, x.double(), None, freq),
                 (pos, x, x, rope_frequencies(66, 1e4)[0].cuda()), (pos, x, x, freq[:0]),
                 (pos.cpu(), x, x, freq), (pos, x, x, freq.cpu()),
                 (pos, x.transpose(1, 2), None, freq[:1])]:
        with pytest.raises((ValueError, TypeError)):
            K.rotary_embedding(*args)
    big = torch.zeros(5, 2, 64, dtype=BF16, device="cuda")
    for q_out, k_out in [(big[1:], big[:4]), (x[:, :, :32], None), (x.float(), None),
                         (big[:1].expand(4, 2, 64), None), (x, x)]:
        with pytest.raises(ValueError):
            K.rotary_embedding(pos, big[:4], x, freq, q_out=q_out, k_out=k_out)
    with pytest.raises(ValueError, match="k_out"):
        K.rotary_embedding(pos, x, None, freq, k_out=big[:4])
    with pytest.raises(ValueError, match="gradients"):
        K.rotary_embedding(pos, x.float().requires_grad_(), None, freq)


# ---------------------------------------------------------------- shared prefix

def pages_case(rows, keys, prefix, hq, hkv, block=256, fp8=False, seed=0, token_major=False,
               spare=3):
    """A cache whose sequences list the same pages for the prefix's whole pages
    and copies of the page it ends in; keys may be fewer than the prefix."""
    g = gen(seed)
    shared, rest = divmod(prefix, block)
    blocks = [max(-(-n // block), 1) for n in keys]
    cols = max(max(blocks), -(-prefix // block), 1)
    table, at = [], shared
    for i in range(len(keys)):
        row = list(range(shared)) + list(range(at, at + cols - shared))
        at += cols - shared
        table.append(row)
    order = list(range(at + spare))
    random.Random(seed).shuffle(order)
    table = torch.tensor([[order[b] for b in r] for r in table], dtype=torch.int32, device="cuda")
    shape = (at + spare, block, hkv, 2, D) if token_major else (at + spare, hkv, 2, block, D)
    pages = torch.randn(shape, generator=g, device="cuda").to(BF16)
    perm = (3, 0, 1, 2, 4) if token_major else (2, 0, 3, 1, 4)
    if rest:
        own = table[:, shared].long()
        view = pages.permute(*perm)
        view[:, own, :rest] = view[:, own[0], :rest][:, None].clone()
    if fp8:
        pages = pages.to(FP8)
    view = pages.permute(*perm)
    q = torch.randn(sum(rows), hq, D, generator=g, device="cuda").to(BF16)
    cu = [torch.tensor([0] + list(torch.tensor(v).cumsum(0)), dtype=torch.int32, device="cuda")
          for v in (rows, keys)]
    return q, view[0], view[1], cu[0], cu[1], table


def prefix_reference(q, kc, vc, rows, keys, table, scale, ks=1.0, vs=1.0):
    """(output, tolerance) in float64 on the CPU; blocks outside the cache hold
    no keys."""
    block, hkv = kc.shape[1], kc.shape[2]
    group = q.shape[1] // hkv
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    start = 0
    for i, (r, n) in enumerate(zip(rows, keys)):
        if r and n > 0:
            ids = table[i, :-(-n // block)].long()
            ok = ((ids >= 0) & (ids < kc.shape[0])).repeat_interleave(block)[:n]
            ids = ids.clamp(0, kc.shape[0] - 1)
            k = kc[ids].double().flatten(0, 1)[:n] * ks
            v = vc[ids].double().flatten(0, 1)[:n] * vs
            s = torch.einsum("rhgd,nhd->hgrn", q[start:start + r].double().unflatten(1, (hkv, group)),
                             k) * scale
            last = torch.arange(n - r, n, device="cuda")
            seen = (torch.arange(n, device="cuda")[None] <= last[:, None]) & ok
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            p = torch.where(seen.any(-1)[:, None], p, 0.0)
            out[start:start + r] = torch.einsum("hgrn,nhd->rhgd", p, v).flatten(1, 2).cpu()
            tol[start:start + r] = torch.einsum("hgrn,nhd->rhgd", p, v.abs()).flatten(1, 2).cpu()
        start += r
    return out, (U + 2e-4) * tol + U * out.abs()


SCALE = D ** -0.5

PREFIX_CASES = {
    # one row each, whole pages, pages the prefix ends in, short of one chunk
    "decode": dict(rows=[1] * 9, keys=[600, 513, 700, 512 + 256, 530, 1000, 514, 600, 2000],
                   prefix=512, hq=16, hkv=8),
    "inside_a_page": dict(rows=[1] * 5, keys=[612, 613, 900, 700, 611], prefix=611, hq=8, hkv=2),
    "under_a_chunk": dict(rows=[1, 1, 1], keys=[40, 90, 31], prefix=31, hq=4, hkv=4),
    "no_prefix": dict(rows=[1, 1], keys=[300, 5], prefix=0, hq=8, hkv=8),
    "one_sequence": dict(rows=[1], keys=[3000], prefix=2816, hq=16, hkv=8),
    # rows of several, ragged, a sequence without rows, more than a tile's
    "verify": dict(rows=[6] * 7, keys=[1030, 1500, 1031, 1100, 1026, 1290, 1024 + 6], prefix=1024,
                   hq=32, hkv=8),
    "ragged": dict(rows=[3, 0, 1, 9, 5, 2], keys=[300, 700, 257, 1000, 400, 258], prefix=256, hq=12,
                   hkv=2),
    "tile_64": dict(rows=[8] * 5, keys=[520, 2000, 530, 777, 1300], prefix=512, hq=64, hkv=8),
    "prompts": dict(rows=[70, 200, 33], keys=[400, 900, 320], prefix=256, hq=16, hkv=4),
    "group_5": dict(rows=[4, 30, 7], keys=[300, 500, 280], prefix=224, hq=10, hkv=2),
    "group_64": dict(rows=[2, 3], keys=[300, 500], prefix=256, hq=64, hkv=1),
    "group_33": dict(rows=[1, 5], keys=[300, 500], prefix=256, hq=33, hkv=1),
    # sequences that end within the prefix, see nothing, or have no key
    "shorter": dict(rows=[1, 1, 1, 1, 1, 1], keys=[700, 100, 0, 1, 32, 512], prefix=512, hq=8,
                    hkv=4),
    "rows_before_keys": dict(rows=[5, 9, 3, 4], keys=[300, 4, 3, 0], prefix=256, hq=8, hkv=4),
    "rows_into_prefix": dict(rows=[40, 2, 60], keys=[520, 513, 530], prefix=512, hq=8, hkv=2),
    # small pages: more than a wave's lanes of them in one part
    "block_32": dict(rows=[1] * 4, keys=[4200, 4100, 6500, 4099], prefix=4096, hq=8, hkv=8, block=32),
    "block_96": dict(rows=[2] * 3, keys=[1000, 1200, 990], prefix=960 + 17, hq=8, hkv=8, block=96),
    "many": dict(rows=[1] * 300, keys=[300 + i for i in range(300)], prefix=256, hq=8, hkv=2),
}


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("name", sorted(PREFIX_CASES))
def test_shared_prefix(cuda, name, fp8):
    c = dict(PREFIX_CASES[name])
    rows, keys, prefix = c.pop("rows"), c.pop("keys"), c.pop("prefix")
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, fp8=fp8, seed=len(name), **c)
    ks, vs = torch.tensor([0.5], device="cuda"), torch.tensor([1.5], device="cuda")
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE, *((0.5, 1.5) if fp8 else ()))
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, max(rows), max(max(keys), prefix),
                                           prefix, SCALE, table, k_scale=ks, v_scale=vs)
    close(got, want, tol)
    # bounds that are far above the lengths change the split alone
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, max(rows) + 3, 4 * max(keys) + 999,
                                           prefix, SCALE, table, k_scale=ks, v_scale=vs)
    close(got, want, tol)
    if all(r == 1 for r in rows):
        lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
        for bound in (None, max(max(keys), prefix)):
            got = K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, SCALE,
                                                   max_seqlen_k=bound, k_scale=ks, v_scale=vs)
            close(got, want, tol)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("block", [32, 256])
def test_shared_prefix_prompts_whose_keys_stay_in_one_part(cuda, block, fp8):
    # more keys a part than a wave's lanes hold small pages
    rows, keys, prefix = [1500, 548, 3], [3300, 2900, 2600], 224
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 64, 8, block=block, fp8=fp8)
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    one = torch.ones(1, device="cuda")
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 1500, 3300, prefix, SCALE, table,
                                           k_scale=one, v_scale=one)
    close(got, want, tol)


@pytest.mark.parametrize("fp8", [False, True])
def test_shared_prefix_layouts(cuda, fp8):
    rows, keys, prefix = [2, 5, 1], [900, 600, 512], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 16, 4, fp8=fp8, token_major=True)
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    wide = torch.randn(8, 16 * D + 64, device="cuda").to(BF16)
    view = wide[:, 64:].view(8, 16, D)
    view.copy_(q)
    out = torch.full((8, 17, D), 5.0, dtype=BF16, device="cuda")
    long_table = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
    long_table[:3, :table.shape[1]] = table
    got = K.shared_prefix_attention_varlen(view, kc, vc, cu_q, cu_k, 5, 900, prefix, SCALE,
                                           long_table, out=out[:, 1:])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    close(out[:, 1:], want, tol)
    assert (out[:, 0] == 5).all()


def test_shared_prefix_padded_batch_leaves_rows(cuda):
    rows, keys, prefix = [3, 1, 4], [700, 513, 600], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 2)
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    for before, behind in ((0, 5), (2, 3)):
        t = before + 8 + behind
        qq = torch.randn(t, 8, D, device="cuda").to(BF16)
        qq[before:before + 8] = q
        out = torch.full((t, 8, D), 9.0, dtype=BF16, device="cuda")
        K.shared_prefix_attention_varlen(qq, kc, vc, cu_q + before, cu_k, 4, 700, prefix, SCALE,
                                         table, out=out)
        close(out[before:before + 8], want, tol)
        assert (out[:before] == 9).all() and (out[before + 8:] == 9).all()
    # padding sequences of no rows and no keys behind the real ones
    pad = lambda cu: torch.cat([cu, cu[-1:].repeat(2)])  # noqa: E731
    padded = torch.cat([table, torch.full_like(table[:2], -1)])
    got = K.shared_prefix_attention_varlen(q, kc, vc, pad(cu_q), pad(cu_k), 4, 700, prefix, SCALE,
                                           padded)
    close(got, want, tol)


def test_shared_prefix_blocks_outside_the_cache_hold_no_keys(cuda):
    rows, keys, prefix = [2, 1, 3], [1100, 900, 1025], 768
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    table[:, 1] = kc.shape[0]           # a prefix page
    table[0, 3], table[1, 3] = -1, 1 << 30
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 3, 1100, prefix, SCALE, table)
    close(got, want, tol)
    table[:] = -1
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 3, 1100, prefix, SCALE, table)
    assert (got == 0).all()


def put(pages, at, value):
    """pages[at] = value, FP8 pages too (which hold no infinity: NaN)."""
    if pages.dtype == FP8:
        pages.view(torch.uint8)[at] = 0x7F
    else:
        pages[at] = value


NAN_CASES = [   # the last keys' units on 16, 32, 64 and 128 rows; one part, some, more than a join's batch
    ([1] * 4, [70, 100, 90, 300], 64, 8, 4), ([1] * 3, [8000, 9000, 8200], 7936, 4, 1),
    ([4, 2, 3], [900, 540, 2700], 512, 8, 1), ([8, 8], [600, 2000], 512, 64, 8),
    ([40, 3], [600, 3000], 512, 16, 4), ([1] * 70, [530 + i for i in range(70)], 512, 8, 2)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,keys,prefix,hq,hkv", NAN_CASES)
@pytest.mark.parametrize("shared", [True, False])
def test_attention_nan_reaches_the_rows_that_see_it(cuda, shared, rows, keys, prefix, hq, hkv, fp8):
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, hq, hkv, fp8=fp8, seed=prefix)
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    group, t = hq // hkv, sum(rows)
    one = torch.ones(1, device="cuda")

    def check(q, kc, vc, bad):
        if shared:
            got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, max(rows), max(keys), prefix,
                                                   SCALE, table, k_scale=one, v_scale=one)
        else:
            got = K.paged_attention_varlen(q, kc, vc, cu_q, cu_k, max(rows), max(keys), SCALE, table,
                                           k_scale=one, v_scale=one)
        got = got.cpu()
        assert got[bad].isnan().all()
        if not bad.all():
            close(got[~bad], want[~bad], tol[~bad])

    bad = torch.zeros(t, hq, dtype=torch.bool)
    bad[::3, 1] = True
    broken = q.clone()
    broken[::3, 1, 5] = float("nan")
    check(broken, kc, vc, bad)
    # a key that all see, one of the prefix's last, and one of the last sequence's own
    for seq, key in ((0, 3), (0, prefix - 1), (len(keys) - 1, keys[-1] - rows[-1])):
        broken, values = kc.clone(), vc.clone()      # of the same strides
        block = (table[seq:seq + 1] if seq else table)[:, key // 256].long()
        put(broken, (block, key % 256, 0, 9), float("nan"))
        bad = torch.zeros(t, hq, dtype=torch.bool)
        start = 0
        for i, (r, n) in enumerate(zip(rows, keys)):
            if i == seq or seq == 0:
                bad[start + max(0, key - (n - r)):start + r, :group] = True
            start += r
        check(q, broken, values, bad)


def test_shared_prefix_clips_like_paged_attention(cuda):
    # longer than the bounds on the device: rows past max_seqlen_q are zeros,
    # keys past max_seqlen_k unseen
    rows, keys, prefix = [6, 2, 4], [900, 700, 560], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    for mq, mk in ((4, 900), (6, 640), (3, 512), (2, 100)):
        want = K.paged_attention_varlen(q, kc, vc, cu_q, cu_k, mq, mk, SCALE, table)
        got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, mq, mk, prefix, SCALE, table)
        # both are within the bound of the header from the same values
        tol = 2 * ((U + 2e-4) * 4.0 + U * want.double().abs())
        close(got, want, tol)
        assert torch.equal((got == 0).all(-1), (want == 0).all(-1))


HIDDEN_CASES = [
    ([1] * 6, [700, 100, 6, 1, 32, 512], 512, 8, 4), ([5, 9, 3, 4], [300, 4, 3, 0], 256, 8, 4),
    ([40, 2, 60], [520, 513, 530], 512, 8, 2), ([1] * 3, [5000, 1500, 4097], 4096, 4, 1),
    ([1] * 90, [520 + 7 * i if i % 3 else 8 * i + 1 for i in range(90)], 512, 8, 2),
    ([130, 3], [400, 90], 256, 16, 4)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,keys,prefix,hq,hkv", HIDDEN_CASES)
def test_shared_prefix_values_that_are_not_finite_stay_with_the_rows_that_see_them(
        cuda, rows, keys, prefix, hq, hkv, fp8):
    """An infinity or NaN in V of a shared key: rows that end before it are as if it
    were not there, the others are not finite in that element."""
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, hq, hkv, fp8=fp8, seed=prefix + 1)
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    one, group = torch.ones(1, device="cuda"), hq // hkv
    last = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, keys)])
    bad = torch.zeros(want.shape, dtype=torch.bool)
    for i, value in enumerate((float("nan"), float("inf"), float("-inf"))):
        for j, key in enumerate((5, 40, prefix // 2 + 3, prefix - 1)):
            d, head = 37 * i + 11 * j, (i + j) % hkv
            put(vc, (table[:, key // 256].long(), key % 256, head, d), value)
            bad[last >= key, head * group:(head + 1) * group, d] = True
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, max(rows), max(max(keys), prefix),
                                           prefix, SCALE, table, k_scale=one, v_scale=one).cpu()
    assert not got[bad].isfinite().any()
    close(got[~bad], want[~bad], tol[~bad])


def test_shared_prefix_no_query_rows_within_the_bound(cuda):
    """max_seqlen_q of 0 leaves every row of the batch past it: zeros, and rows of no
    sequence as they were."""
    rows, keys, prefix = [2, 1], [600, 540], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    q = torch.cat([q, q[:2]])
    out = torch.full((5, 8, D), 3.0, dtype=BF16, device="cuda")
    K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 0, 600, prefix, SCALE, table, out=out)
    assert (out[:3] == 0).all() and (out[3:] == 3).all()


def clipped_lengths(rows, keys, max_q, max_k):
    """What a call with these bounds computes: (rows, keys) of every sequence."""
    kept = [min(r, max_q) for r in rows]
    return kept, [min(n - (r - a), max_k) for r, a, n in zip(rows, kept, keys)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("mq,mk", [(4, 900), (6, 899), (6, 700), (6, 699), (6, 559), (3, 512), (5, 511),
                                   (2, 100), (1, 33), (6, 1)])
def test_shared_prefix_clips_to_the_bounds(cuda, mq, mk, fp8):
    """Against the definition on the clipped lengths, where the first key that a
    bound cuts off would take all the weight."""
    rows, keys, prefix = [6, 2, 4], [900, 700, 560], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4, fp8=fp8)
    kept, seen = clipped_lengths(rows, keys, mq, mk)
    starts = [0, 6, 8]
    planted = [i for i, n in enumerate(seen) if n < keys[i] and (n >= prefix or (n == max(seen) and i == 0))]
    for i in planted:       # the key behind the last one that the sequence sees
        page, at = int(table[i, seen[i] // 256]), seen[i] % 256
        row = q[starts[i] + kept[i] - 1].view(4, 2, D)[:, 0].float() * 4
        kc[page, at], vc[page, at] = row.to(kc.dtype), torch.full_like(row, 400.0).to(vc.dtype)
    assert planted
    first = torch.cat([torch.arange(s, s + r) for s, r in zip(starts, kept)])
    want, tol = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    want[first], tol[first] = prefix_reference(q[first.cuda()], kc, vc, kept, seen, table, SCALE)
    over, _ = prefix_reference(q[first.cuda()], kc, vc, kept,
                               [n + (i in planted) for i, n in enumerate(seen)], table, SCALE)
    ends = torch.tensor(kept).cumsum(0) - 1
    for i in planted:       # seen all the same, it would show
        assert ((over - want[first]).abs() > 100 * tol[first])[ends[i]].any()
    one = torch.ones(1, device="cuda")
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, mq, mk, prefix, SCALE, table,
                                           k_scale=one, v_scale=one)
    close(got, want, tol)


def test_shared_prefix_large_scores_and_stale_slots(cuda):
    # rows whose parts differ by hundreds in the exponent, infinities and NaN in
    # slots that no row sees
    rows, keys, prefix = [1] * 4, [700, 530, 520, 1300], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    q[0] *= 60
    kc[table[0, 2].long(), :100] *= 20
    want, tol = prefix_reference(q, kc, vc, rows, keys, table, SCALE)
    for i, n in enumerate(keys):
        page = table[i, n // 256].long()
        kc[page, n % 256:] = float("nan")
        vc[page, n % 256:] = float("inf")
    got = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 1, 1300, prefix, SCALE, table)
    # scores of up to some thousand: 2^-24 of them in the exponent besides
    close(got, want, tol + 4e-3 * want.abs() + 4e-3)


def test_shared_prefix_offsets_past_32_bits(cuda):
    # a cache of more than 2^31 elements whose pages lie at its end
    block, hkv = 256, 8
    nb = (1 << 31) // (2 * block * hkv * D) + 40
    pages = torch.zeros(nb, hkv, 2, block, D, dtype=BF16, device="cuda")
    small = pages_case([1, 3, 2], [1100, 900, 801], 768, 16, hkv)
    q, kc, vc, cu_q, cu_k, table = small
    used = table.unique().long()
    view = pages.permute(2, 0, 3, 1, 4)
    moved = table + (nb - kc.shape[0])
    view[0][used + (nb - kc.shape[0])] = kc[used]
    view[1][used + (nb - kc.shape[0])] = vc[used]
    want, tol = prefix_reference(q, kc, vc, [1, 3, 2], [1100, 900, 801], table, SCALE)
    got = K.shared_prefix_attention_varlen(q, view[0], view[1], cu_q, cu_k, 3, 1100, 768, SCALE, moved)
    close(got, want, tol)


def test_shared_prefix_lengths_on_the_host(cuda):
    rows, keys, prefix = [2, 1], [600, 540], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    want = K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 2, 600, prefix, SCALE, table)
    got = K.shared_prefix_attention_varlen(q, kc, vc, [0, 2, 3], [0, 600, 1140], 2, 600, prefix, SCALE,
                                           table)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="max_seqlen_k"):
        K.shared_prefix_attention_varlen(q, kc, vc, [0, 2, 3], [0, 600, 1140], 2, 599, prefix, SCALE,
                                         table)


def test_shared_prefix_refusals(cuda):
    rows, keys, prefix = [1, 1], [600, 540], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    lens = torch.tensor(keys, dtype=torch.int32, device="cuda")

    def call(q=q, kc=kc, vc=vc, lens=lens, table=table, prefix=prefix, scale=SCALE, **kw):
        return K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, scale, **kw)

    call()
    for kw in (dict(prefix=-1), dict(prefix=257 * table.shape[1]), dict(scale=0.0), dict(scale=-1.0),
               dict(scale=float("nan")), dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[:, :, :64]),
               dict(kc=kc[..., :64], vc=vc[..., :64], q=q[..., :64].contiguous()),
               dict(kc=kc.float(), vc=vc.float()), dict(vc=vc[:2]), dict(lens=lens.long()),
               dict(lens=lens[:1]), dict(table=table.long()), dict(table=table[:1]),
               dict(table=table[0]), dict(out=torch.empty(2, 8, D, device="cuda")),
               dict(out=torch.empty(2, 9, D, dtype=BF16, device="cuda")), dict(max_seqlen_k=-1),
               dict(k_scale=torch.ones(2, device="cuda")), dict(q=q.cpu()),
               dict(q=torch.cat([q, q], -1)[..., 4:4 + D])):
        with pytest.raises((ValueError, TypeError)):
            call(**kw)


def test_shared_prefix_refuses_gradients(cuda):
    rows, keys, prefix = [1, 1], [600, 540], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
    one = torch.ones(1, device="cuda")
    want = K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, SCALE)
    wants = lambda t: t.detach().requires_grad_()  # noqa: E731
    for a, kw in (((wants(q), kc, vc), {}), ((q, wants(kc), vc), {}), ((q, kc, wants(vc)), {}),
                  ((q, kc, vc), dict(k_scale=wants(one), v_scale=one)),
                  ((q, kc, vc), dict(k_scale=one, v_scale=wants(one)))):
        with pytest.raises(ValueError, match="gradients"):
            K.shared_prefix_attention_decode(*a, lens, table, prefix, SCALE, **kw)
        with pytest.raises(ValueError, match="gradients"):
            K.shared_prefix_attention_varlen(*a, cu_q, cu_k, 1, 600, prefix, SCALE, table, **kw)
        with torch.no_grad():
            assert torch.equal(K.shared_prefix_attention_decode(*a, lens, table, prefix, SCALE, **kw),
                               want)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_shared_prefix_scales_on_another_device_are_refused(cuda):
    q, kc, vc, _, _, table = pages_case([1, 1], [600, 540], 512, 8, 4, fp8=True)
    lens = torch.tensor([600, 540], dtype=torch.int32, device="cuda")
    one, far = torch.ones(1, device="cuda"), torch.ones(1, device="cuda:1")
    for kw in (dict(k_scale=far, v_scale=one), dict(k_scale=one, v_scale=far)):
        with pytest.raises(ValueError, match="same device"):
            K.shared_prefix_attention_decode(q, kc, vc, lens, table, 512, SCALE, **kw)


def test_shared_prefix_out_that_overlaps_itself_is_refused(cuda):
    rows, keys, prefix = [1, 1, 1], [600, 540, 513], 512
    q, kc, vc, cu_q, cu_k, table = pages_case(rows, keys, prefix, 8, 4)
    lens = torch.tensor(keys, dtype=torch.int32, device="cuda")
    want = K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, SCALE)
    flat = torch.zeros(3 * 8 * D, dtype=BF16, device="cuda")
    for strides in ((0, D, 1), (8 * D, 0, 1), (D, D, 1), (4 * D, D, 1), (8 * D, 64, 1)):
        out = flat.as_strided((3, 8, D), strides)
        with pytest.raises(ValueError, match="overlap"):
            K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, SCALE, out=out)
        with pytest.raises(ValueError, match="overlap"):
            K.shared_prefix_attention_varlen(q, kc, vc, cu_q, cu_k, 1, 600, prefix, SCALE, table, out=out)
    assert (flat == 0).all()
    for out in (torch.zeros(8, 3, D, dtype=BF16, device="cuda").transpose(0, 1),
                torch.zeros(3, 8, 2 * D, dtype=BF16, device="cuda")[..., D:]):
        K.shared_prefix_attention_decode(q, kc, vc, lens, table, prefix, SCALE, out=out)
        assert torch.equal(out, want)


# ---------------------------------------------------------------- streams, graphs, a step

def step_state(seed=0, batch=6, hidden=512, hq=8, hkv=2, prefix=512):
    """A decoding step's attention block: 4-bit q/k/v and output projections,
    scaled rotary positions, a cache over a shared prefix."""
    g = gen(seed)
    keys = [prefix + 1 + 37 * i for i in range(batch)]
    _, kc, vc, _, _, table = pages_case([1] * batch, keys, prefix, hq, hkv, seed=seed)
    scaling = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=40960)
    freq, factor = rope_frequencies(D, 1e6, scaling)
    w = [torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
         for n, k in (((hq + 2 * hkv) * D, hidden), (hidden, hq * D))]
    pos = torch.tensor([n - 1 for n in keys], device="cuda")
    block = kc.shape[1]
    slots = torch.gather(table, 1, (pos // block)[:, None])[:, 0] * block + pos % block
    return dict(x=torch.randn(batch, hidden, generator=g, device="cuda").to(BF16), kc=kc, vc=vc,
                table=table, keys=keys, pos=pos, slots=slots.int(), freq=freq.cuda(), factor=factor,
                qkv=K.quantize_w4(w[0], 128), o=K.quantize_w4(w[1], 64, zeros=True), hq=hq, hkv=hkv,
                prefix=prefix, lens=torch.tensor(keys, dtype=torch.int32, device="cuda"))


def step(s):
    hq, hkv, b = s["hq"], s["hkv"], s["x"].shape[0]
    qkv = K.linear_w4(s["x"], *s["qkv"])
    q, k, v = (p.view(b, -1, D) for p in qkv.split([hq * D, hkv * D, hkv * D], 1))
    K.rotary_embedding(s["pos"], q, k, s["freq"], factor=s["factor"], q_out=q, k_out=k)
    K.store_kvcache(k, v, s["kc"], s["vc"], s["slots"])
    o = K.shared_prefix_attention_decode(q, s["kc"], s["vc"], s["lens"], s["table"], s["prefix"],
                                         SCALE, max_seqlen_k=max(s["keys"]))
    return K.linear_w4(o.flatten(1), *s["o"])


def test_a_decoding_step(cuda):
    s = step_state()
    hq, hkv, b = s["hq"], s["hkv"], s["x"].shape[0]
    got = step(s)
    # each part against its plain form on the rounded outputs of the one before
    want, tol = w4_reference(s["x"], *s["qkv"], None)
    qkv = K.linear_w4(s["x"], *s["qkv"])
    close(qkv, want, tol)
    q, k, v = (p.view(b, -1, D) for p in qkv.split([hq * D, hkv * D, hkv * D], 1))
    qr, kr = K.rotary_embedding(s["pos"], q, k, s["freq"], factor=s["factor"])
    close(qr, *rotary_reference(q, s["pos"], s["freq"], False, s["factor"]))
    close(kr, *rotary_reference(k, s["pos"], s["freq"], False, s["factor"]))
    rows = s["slots"].long()
    assert torch.equal(s["kc"][rows // 256, rows % 256], kr)
    assert torch.equal(s["vc"][rows // 256, rows % 256], v)
    o = K.shared_prefix_attention_decode(qr, s["kc"], s["vc"], s["lens"], s["table"], s["prefix"],
                                         SCALE, max_seqlen_k=max(s["keys"]))
    close(o, *prefix_reference(qr, s["kc"], s["vc"], [1] * b, s["keys"], s["table"], SCALE))
    want, tol = w4_reference(o.flatten(1), *s["o"], None)
    close(got, want, tol)


def test_steps_captured_and_on_two_streams(cuda):
    states = [step_state(seed) for seed in (1, 2)]
    want = [step(s) for s in states]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    for turn in range(3):
        for graph, out, w in zip(graphs, outs, want):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w), f"replay {turn}"
            step(states[1 - turn % 2])          # eager work of its own between the replays
    # two streams at once: no scratch memory is shared
    streams = [torch.cuda.Stream() for _ in states]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i, s in enumerate(states):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(s))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for g in got[i]:
            assert torch.equal(g, w)


def test_repeated_calls_give_the_same_bits(cuda):
    s = step_state(3)
    first = step(s)
    for _ in range(5):
        assert torch.equal(step(s), first)
