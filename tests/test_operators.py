"""Host side of the 4-bit projections, rotary positions and shared-prefix
attention: quantizer, frequencies, plans and refusals (no GPU)."""
import math

import pytest
import torch

from nanovllm_amd import _native
from nanovllm_amd import kernels as K
from nanovllm_amd.layers import rope_frequencies

BF16 = torch.bfloat16
P = 4096                # a pointer that no refused call reads


# ---------------------------------------------------------------- quantizer

def dequantized(qw, s, z):
    n, k = qw.shape[0], 2 * qw.shape[1]
    c = torch.stack((qw & 15, qw >> 4), -1).view(n, k).double()
    step = s.double().t().repeat_interleave(k // s.shape[0], 1)
    zero = 8.0 if z is None else z.double().t().repeat_interleave(k // s.shape[0], 1)
    return (c - zero) * step, step


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 256])
def test_quantize_w4_rounds_to_the_nearest_level(group, zeros):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(24, 512, generator=g) * torch.rand(24, 1, generator=g)
    w[5] = w[5].abs() + 1.0             # a row of one sign
    w[6] = -w[6].abs()
    w[7, :group] = 0.0
    qw, s, z = K.quantize_w4(w, group, zeros)
    assert qw.shape == (24, 256) and qw.dtype == torch.uint8
    assert s.shape == (512 // group, 24) and s.dtype == BF16 and s.is_contiguous()
    assert (z is None) == (not zeros)
    back, step = dequantized(qw, s, z)
    # half a step, and at the ends of the range what the scale's rounding to
    # bf16 (2^-8 of at most 15 steps) and the rounded zero (half a step) cut off
    slack = 0.5 + 15 * 2.0 ** -8 + (0.5 if zeros else 0.0)
    assert ((back - w.double()).abs() <= slack * step + 1e-12).all()
    assert (back[7, :group] == 0).all()
    inside = (back - w.double()).abs() <= 0.5 * step * (1 + 1e-6)
    assert inside.double().mean() > 0.95


def test_quantize_w4_keeps_what_four_bits_hold():
    codes = torch.randint(-8, 8, (16, 128), generator=torch.Generator().manual_seed(0))
    codes[:, 0], codes[:, 64] = -8, -8
    w = codes.double() * 0.125
    qw, s, z = K.quantize_w4(w.float(), 64)
    assert z is None and torch.equal(dequantized(qw, s, z)[0], w)


@pytest.mark.parametrize("lo,hi,scale", [(-8.0, 8.0, 8 / 7), (-8.0, 3.0, 1.0), (-3.0, 7.0, 1.0),
                                         (1.0, 14.0, 2.0), (-16.0, -1.0, 2.0)])
def test_quantize_w4_takes_the_least_scale_that_holds_both_ends(lo, hi, scale):
    w = torch.linspace(lo, hi, 64)[None]
    qw, s, _ = K.quantize_w4(w, 64)
    assert float(s) == float(torch.tensor(scale).to(BF16))
    back, step = dequantized(qw, s, None)
    assert ((back - w.double()).abs() <= (0.5 + 8 * 2.0 ** -8) * step).all()   # 8 steps of the scale's rounding


def test_quantize_w4_refusals():
    w = torch.zeros(4, 128)
    for args in [(w, 16), (w, 96), (w, 0), (w, -32), (w[0], 32), (w.int(), 32), (w[:, :0], 32)]:
        with pytest.raises(ValueError):
            K.quantize_w4(*args)


# ---------------------------------------------------------------- frequencies

def test_frequencies_default_and_linear():
    freq, factor = rope_frequencies(128, 1e6)
    assert factor == 1.0 and freq.dtype == torch.float64 and freq.shape == (64,)
    assert freq[0] == 1.0 and math.isclose(freq[32], 1e-3, rel_tol=1e-12)
    slow, factor = rope_frequencies(128, 1e6, dict(rope_type="linear", factor=4.0))
    assert factor == 1.0 and torch.equal(slow, freq / 4)


def test_frequencies_yarn():
    o, s, base = 32768, 4.0, 1e6
    freq, _ = rope_frequencies(128, base)
    got, factor = rope_frequencies(128, base, dict(rope_type="yarn", factor=s,
                                                   original_max_position_embeddings=o))
    assert math.isclose(factor, 0.1 * math.log(4) + 1)
    turns = o * freq / (2 * math.pi)
    ratio = got / freq
    # the ramp's ends are whole pairs: one pair beyond each is past them
    step = base ** (2 / 128)
    assert torch.allclose(ratio[turns > 32 * step], torch.ones(1, dtype=torch.float64))
    assert torch.allclose(ratio[turns < 1 / step], torch.full((1,), 1 / s, dtype=torch.float64))
    assert (ratio.diff() <= 1e-12).all() and ratio.min() >= 1 / s - 1e-12
    given, factor = rope_frequencies(128, base, dict(type="yarn", factor=s, attention_factor=1.5,
                                                     original_max_position_embeddings=o))
    assert factor == 1.5 and torch.equal(given, got)


def test_frequencies_yarn_amplitude():
    def factor(s=40.0, **kw):
        return rope_frequencies(64, 1e4, dict(type="yarn", factor=s, original_max_position_embeddings=4096,
                                              **kw))[1]

    m = 0.1 * math.log(40)
    assert math.isclose(factor(), m + 1)
    assert factor(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert math.isclose(factor(mscale=0.707, mscale_all_dim=1.0), (0.707 * m + 1) / (m + 1))
    assert math.isclose(factor(mscale=1.0, mscale_all_dim=0.0), m + 1)
    assert factor(mscale=2.0, mscale_all_dim=0.5, attention_factor=1.25) == 1.25
    assert factor(s=1.0, mscale=2.0, mscale_all_dim=0.5) == 1.0
    for kw in (dict(mscale=0.707), dict(mscale_all_dim=1.0)):
        with pytest.raises(ValueError, match="mscale"):
            factor(**kw)


def test_frequencies_yarn_ends_of_the_ramp():
    """factor 8, 4096 positions, base 1e4, 64 elements: the pair that turns 32 times is
    64 ln(4096 / (64 pi)) / (2 ln 1e4) = 10.47, the one that turns once 22.51."""
    scaling = dict(type="yarn", factor=8.0, original_max_position_embeddings=4096)
    freq, _ = rope_frequencies(64, 1e4)
    low, high = (64 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(1e4)) for t in (32, 1))
    assert 10.4 < low < 10.5 and 22.5 < high < 22.6
    for truncate, a, b in ((None, 10, 23), (True, 10, 23), (False, low, high)):
        got, factor = rope_frequencies(64, 1e4, dict(scaling, truncate=truncate))
        assert math.isclose(factor, 0.1 * math.log(8) + 1)
        for i in range(32):
            ramp = min(max((i - a) / (b - a), 0.0), 1.0)
            want = float(freq[i]) * ((1 - ramp) + ramp / 8)
            assert math.isclose(float(got[i]), want, rel_tol=1e-12), (truncate, i)


def test_frequencies_refuse_keys_they_do_not_read():
    base = {"default": {}, "linear": dict(factor=2.0), "dynamic": dict(factor=2.0),
            "yarn": dict(factor=2.0), "llama3": dict(factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0),
            "longrope": dict(short_factor=[1.0] * 32, long_factor=[2.0] * 32)}
    for kind, keys in base.items():
        scaling = dict(rope_type=kind, original_max_position_embeddings=4096, **keys)
        want = rope_frequencies(64, 1e4, scaling, seq_len=8192)
        kept = dict(scaling, rope_theta=1e4, partial_rotary_factor=0.5, finetuned=True, attn_factor=None)
        got = rope_frequencies(64, 1e4, kept, seq_len=8192)
        assert torch.equal(got[0], want[0]) and got[1] == want[1]
        for extra in (dict(attn_factor=2.0), dict(short_mscale=1.2), dict(mrope_section=[8, 12, 12]),
                      dict(extrapolation_factor=1.0), dict(alpha=2.0)):
            with pytest.raises(ValueError, match="not read"):
                rope_frequencies(64, 1e4, dict(scaling, **extra), seq_len=8192)
        if kind != "yarn":
            with pytest.raises(ValueError, match="not read"):
                rope_frequencies(64, 1e4, dict(scaling, truncate=False), seq_len=8192)
        with pytest.raises(ValueError, match="rope_theta"):
            rope_frequencies(64, 1e4, dict(scaling, rope_theta=5e5), seq_len=8192)


def test_frequencies_llama3():
    scaling = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192)
    freq, _ = rope_frequencies(128, 5e5)
    got, factor = rope_frequencies(128, 5e5, scaling)
    wave = 2 * math.pi / freq
    assert factor == 1.0
    assert torch.allclose(got[wave < 2048], freq[wave < 2048])
    assert torch.allclose(got[wave > 8192], freq[wave > 8192] / 8)
    mid = (wave > 2048) & (wave < 8192)
    smooth = (8192 / wave[mid] - 1) / 3
    assert mid.any() and torch.allclose(got[mid], (1 - smooth) * freq[mid] / 8 + smooth * freq[mid])


def test_frequencies_dynamic_and_longrope():
    freq, _ = rope_frequencies(64, 1e4)
    scaling = dict(rope_type="dynamic", factor=2.0)
    short, _ = rope_frequencies(64, 1e4, scaling, max_position=4096, seq_len=4096)
    assert torch.equal(short, freq)
    grown, _ = rope_frequencies(64, 1e4, scaling, max_position=4096, seq_len=8192)
    # the last pair turns (2 * 8192 / 4096 - 1) times slower
    assert grown[0] == 1.0 and math.isclose(freq[-1] / grown[-1], 3.0, rel_tol=1e-9)
    scaling = dict(rope_type="longrope", short_factor=[1.0] * 32, long_factor=[2.0] * 32,
                   original_max_position_embeddings=4096)
    a, fa = rope_frequencies(64, 1e4, scaling, max_position=131072, seq_len=4096)
    b, fb = rope_frequencies(64, 1e4, scaling, max_position=131072, seq_len=4097)
    assert torch.equal(a, freq) and torch.equal(b, freq / 2)
    assert fa == fb and math.isclose(fa, math.sqrt(1 + math.log(32) / math.log(4096)))


def test_frequencies_refusals():
    for args, kw in [((127, 1e4), {}), ((0, 1e4), {}), ((64, 1e4, dict(type="linear")), {}),
                     ((64, 1e4, dict(type="odd", factor=2.0)), dict(max_position=64)),
                     ((64, 1e4, dict(type="yarn", factor=2.0)), {}),
                     ((64, 1e4, dict(type="llama3", factor=2.0)), dict(max_position=64)),
                     ((64, 1e4, dict(type="longrope", short_factor=[1.0], long_factor=[1.0])),
                      dict(max_position=64))]:
        with pytest.raises(ValueError):
            rope_frequencies(*args, **kw)


# ---------------------------------------------------------------- refusals

def test_the_library_refuses_bad_products_on_the_host():
    lib = _native.load()

    def call(x=P, stride=128, w=P, s=P, z=None, b=None, out=P, out_stride=8, rows=2, n=8, k=128,
             group=32):
        return lib.nva_linear_w4(x, stride, w, s, z, b, out, out_stride, rows, n, k, group, None, 0,
                                 None)

    assert call(rows=0) == _native.NVA_OK
    for kw in (dict(rows=-1), dict(n=0), dict(k=0), dict(group=0), dict(group=48), dict(x=None),
               dict(w=None), dict(s=None), dict(out=None), dict(stride=120), dict(out_stride=7)):
        assert call(**kw) == _native.NVA_ERR_ARG, kw
    for kw in (dict(group=16), dict(stride=132), dict(x=P + 8), dict(w=P + 4),
               dict(rows=64, stride=1 << 24), dict(rows=17, stride=1 << 26),
               dict(rows=64 * 65535 + 1), dict(k=(1 << 20) + 32, stride=1 << 21),
               dict(n=1 << 27, out_stride=1 << 27)):
        assert call(**kw) == _native.NVA_ERR_UNSUPPORTED, kw


def test_the_library_refuses_bad_rotations_on_the_host():
    lib = _native.load()

    def call(pos=P, freq=P, dtype=0, q=P, hq=2, k=P, hk=1, t=4, d=64, rot=64, qo=P, ko=P):
        return lib.nva_rotary_embedding(pos, freq, 1.0, 0, dtype, q, 128, 64, hq, k, 64, 64, hk, t, d,
                                        rot, qo, 128, 64, ko, 64, 64, None)

    assert call(t=0) == _native.NVA_OK
    for kw in (dict(t=-1), dict(hq=-1), dict(hk=-1), dict(d=0), dict(rot=0), dict(rot=33),
               dict(rot=66), dict(dtype=3), dict(pos=None), dict(freq=None), dict(q=None),
               dict(k=None), dict(qo=None), dict(ko=None)):
        assert call(**kw) == _native.NVA_ERR_ARG, kw
    for kw in (dict(d=1026), dict(d=1024, rot=514)):
        assert call(**kw) == _native.NVA_ERR_UNSUPPORTED, kw


def test_the_library_refuses_bad_prefix_attention_on_the_host():
    lib = _native.load()

    def call(q=P, kc=P, kv=0, blocks=8, bs=256, cu=P, table=P, cols=4, seqs=2, t=2, mq=1, mk=1024,
             prefix=512, hq=8, hkv=2, d=128, scale=0.1, out=P, ws=P, nbytes=1 << 30, tok=128,
             stride=4):
        return lib.nva_shared_prefix_attention_varlen(
            q, hq * 128, 128, kc, kc, kv, 256 * 2 * 128, tok, 256 * 128, blocks, bs, cu, cu, table,
            stride, cols, seqs, t, mq, mk, prefix, hq, hkv, d, scale, None, None, out, hq * 128, 128,
            ws, nbytes, None)

    assert call(seqs=0) == _native.NVA_OK and call(t=0) == _native.NVA_OK
    for kw in (dict(q=None), dict(kc=None), dict(cu=None), dict(table=None), dict(out=None),
               dict(kv=2), dict(seqs=-1), dict(t=-1), dict(mq=-1), dict(mk=-1), dict(prefix=-1),
               dict(hq=0), dict(hkv=0), dict(hq=7), dict(scale=0.0), dict(scale=float("nan")),
               dict(cols=-1), dict(stride=3)):
        assert call(**kw) == _native.NVA_ERR_ARG, kw
    for kw in (dict(d=64), dict(bs=48), dict(bs=0), dict(blocks=0), dict(hq=130, hkv=2),
               dict(q=P + 8), dict(out=P + 2), dict(tok=132),
               dict(seqs=1 << 20, t=1 << 20, mq=1 << 20)):
        assert call(**kw) == _native.NVA_ERR_UNSUPPORTED, kw
    for kw in (dict(ws=None), dict(nbytes=64), dict(ws=P + 8)):
        assert call(**kw) == _native.NVA_ERR_WORKSPACE, kw


def test_prefix_workspace_holds_every_part():
    size = _native.load().nva_shared_prefix_workspace_size
    for seqs, t, hq, hkv, mq, mk, prefix in [(1, 1, 8, 8, 1, 100, 0), (8, 8, 16, 8, 1, 968, 768),
                                             (64, 384, 32, 8, 6, 9000, 8192),
                                             (128, 1024, 64, 8, 8, 5611, 4111)]:
        # at least one part of each row's prefix (if there is one) and own keys
        parts = (1 if min(prefix, mk) >= 32 else 0) + 1
        assert size(seqs, t, hq, hkv, 128, mq, mk, prefix) >= t * hq * parts * 129 * 4
    for bad in [(0, 1, 8, 8, 128, 1, 8, 0), (1, 0, 8, 8, 128, 1, 8, 0), (1, 1, 8, 8, 64, 1, 8, 0),
                (1, 1, 8, 3, 128, 1, 8, 0), (1, 1, 8, 8, 128, 1, 8, -1), (1, 1, 130, 2, 128, 1, 8, 0)]:
        assert size(*bad) == 0


@pytest.mark.parametrize("seqs,t,hq,hkv,mq,mk,prefix,parts", [
    (8, 16384, 64, 8, 2048, 8192, 4096, 2), (1, 4096, 64, 8, 4096, 40960, 4096, 2),
    (1, 4096, 64, 8, 4096, 40960, 36864, 3), (2, 2000, 16, 2, 1000, 31024, 1024, 10),
    (4, 8192, 32, 8, 2048, 2048, 0, 1)])
def test_prefix_workspace_of_prompts_stays_with_few_parts(seqs, t, hq, hkv, mq, mk, prefix, parts):
    """A part costs 516 bytes a row and head: rows that fill the device by themselves
    are not split as far as a decode batch's."""
    size = _native.load().nva_shared_prefix_workspace_size(seqs, t, hq, hkv, 128, mq, mk, prefix)
    assert size <= t * (hq * parts * 129 * 4 + 4)


def test_prefix_attention_bounds_past_2_to_the_30_keys_are_refused():
    lib = _native.load()
    size = lib.nva_shared_prefix_workspace_size
    for max_k in ((1 << 30) + 1, 2 ** 31 - 64, 2 ** 31 - 1):
        assert size(8, 16384, 64, 8, 128, 2048, max_k, 4096) == 0
        assert lib.nva_shared_prefix_attention_varlen(
            P, 64 * 128, 128, P, P, 0, 256 * 128, 128, 256 * 128, 8, 256, P, P, P, 4, 4, 8, 16384,
            2048, max_k, 512, 64, 8, 128, 0.1, None, None, P, 64 * 128, 128, P, 1 << 40,
            None) == _native.NVA_ERR_UNSUPPORTED
    # the largest bound is planned without coming round: a slot for every row and head
    assert 16384 * 64 * 516 <= size(8, 16384, 64, 8, 128, 2048, 1 << 30, 4096) < 1 << 40


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="device"):
        K.linear_w4(x, torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(2, 8, dtype=BF16))
    with pytest.raises(ValueError, match="device"):
        K.rotary_embedding(torch.arange(2), x.view(2, 1, 64), None, torch.ones(32, dtype=torch.float64))
    cache = torch.zeros(2, 256, 1, 128, dtype=BF16)
    with pytest.raises(ValueError, match="device"):
        K.shared_prefix_attention_decode(torch.zeros(2, 1, 128, dtype=BF16), cache, cache,
                                         torch.ones(2, dtype=torch.int32),
                                         torch.zeros(2, 1, dtype=torch.int32), 0, 1.0)
