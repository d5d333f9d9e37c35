"""Angle tables of RotaryEmbedding's forms against the formulas in 64 bits, and the constructor's refusals (CPU)."""
import math

import pytest
import torch

from diffulex_amd import _lib
from diffulex_amd.rotary_embedding import RotaryEmbedding, get_rope
from oracle import rotary as orot


def _check(rope, angle, gain=1.0):
    """angle(position, pair) in 64 bits; cosines and sines rounded once: within half a step of fp32 (2^-24), and the 64-bit
    angle itself is off by at most a few steps of 64 bits of positions below 2^18."""
    table = rope.cos_sin_cache.double()
    n, rot = table.shape
    g = torch.Generator().manual_seed(0)
    for p in [0, 1, n - 1] + torch.randint(0, n, (40,), generator=g).tolist():
        for i in range(rot // 2):
            a = angle(p, i)
            assert abs(table[p, i] - gain * math.cos(a)) <= gain * 2.0 ** -24 + 1e-9
            assert abs(table[p, rot // 2 + i] - gain * math.sin(a)) <= gain * 2.0 ** -24 + 1e-9


def test_plain_form_keeps_the_reference_bits():
    assert torch.equal(RotaryEmbedding(128, 128, 500, 1e6).cos_sin_cache, orot.cos_sin_cache(128, 500, 1e6))
    assert torch.equal(RotaryEmbedding(128, 128, 500, 1e6, rope_scaling=dict(rope_type="default")).cos_sin_cache,
                       orot.cos_sin_cache(128, 500, 1e6))


@pytest.mark.parametrize("hd,rot,neox", [(128, 64, True), (128, 128, False), (64, 16, False)])
def test_unscaled(hd, rot, neox):
    rope = RotaryEmbedding(hd, rot, 100000, 1e4, is_neox_style=neox)
    assert rope.cos_sin_cache.shape == (100000, rot)
    _check(rope, lambda p, i: p * 1e4 ** (-2 * i / rot))


def test_linear_and_dynamic():
    _check(RotaryEmbedding(64, 64, 9000, 1e6, rope_scaling=dict(type="linear", factor=4)), lambda p, i: p / 4 * 1e6 ** (-2 * i / 64))
    s = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=2048)
    base = 1e4 * (2.0 * 8192 / 2048 - 1) ** (64 / 62)
    _check(RotaryEmbedding(64, 64, 8192, 1e4, rope_scaling=s), lambda p, i: p * base ** (-2 * i / 64))


@pytest.mark.parametrize("factor,extra,gain", [(8.0, {}, 0.1 * math.log(8) + 1), (1.0, {}, 1.0),
                                               (4.0, dict(attention_factor=1.5, beta_fast=16, beta_slow=2), 1.5)])
def test_yarn(factor, extra, gain):
    dim, base, orig = 64, 1e4, 2048
    rope = RotaryEmbedding(128, dim, int(orig * factor), base, rope_scaling=dict(
        rope_type="yarn", factor=factor, original_max_position_embeddings=orig, **extra))
    fast, slow = extra.get("beta_fast", 32), extra.get("beta_slow", 1)
    # pair i turns orig * base^(-2i/dim) / 2 pi times over the original length
    low = max(math.floor(dim / 2 * math.log(orig / (2 * math.pi * fast), base)), 0)
    high = min(math.ceil(dim / 2 * math.log(orig / (2 * math.pi * slow), base)), dim - 1)

    def angle(p, i):
        r = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        f = base ** (-2 * i / dim)
        return p * (f * (1 - r) + f / factor * r)
    _check(rope, angle, gain)


def test_get_rope_keeps_one_module():
    s = dict(rope_type="linear", factor=2.0)
    a = get_rope(64, 32, 128, 1e4, s, False)
    assert get_rope(64, 32, 128, 1e4, dict(s), is_neox_style=False) is a
    assert get_rope(64, 32, 128, 1e4) is not a


def test_refusals():
    for bad in (dict(rope_type="other", factor=2.0), dict(factor=2.0), dict(rope_type="linear", factor=0.5), dict(type="yarn", factor=float("inf")),
                dict(type="dynamic", factor=2.0, original_max_position_embeddings=-4)):
        with pytest.raises(ValueError):
            RotaryEmbedding(64, 64, 128, 1e4, rope_scaling=bad)
    for rot in (0, 65, 66, 7):
        with pytest.raises(AssertionError):
            RotaryEmbedding(64, rot, 128, 1e4)
    lib = _lib.load()
    import ctypes as C
    p = _lib.RopeParams()
    p.n_tokens, p.num_q_heads, p.num_kv_heads, p.head_dim, p.max_position = 4, 1, 1, 64, 16
    for field, value, status in (("rotary_dim", -16, -1), ("rotary_dim", 80, -1), ("rotary_dim", 24, -2), ("interleaved", 2, -1), ("kv_dtype", 4, -1)):
        p.rotary_dim, p.interleaved, p.kv_dtype = 0, 0, 0
        p.q = p.k = p.q_out = p.k_out = p.positions = p.cos_sin_cache = 4096
        p.q_stride_token = p.k_stride_token = p.q_out_stride_token = p.k_out_stride_token = 64
        setattr(p, field, value)
        assert lib.dfx_rope_kv_store(C.byref(p), None) == status, field
    # microscaled stores: blocks that straddle the halves, missing scales
    p.kv_dtype, p.rotary_dim, p.interleaved = 2, 32, 0
    p.v = p.k_cache = p.v_cache = p.slot_mapping = 4096
    p.v_stride_token, p.n_slots = 64, 16
    assert lib.dfx_rope_kv_store(C.byref(p), None) == -1
    p.k_block_scales = p.v_block_scales = 4096
    assert lib.dfx_rope_kv_store(C.byref(p), None) == -2


def test_mx_entry_points_refuse_without_launching():
    lib = _lib.load()
    ok = [4096, 4096, 128, 128, 4096, 4096, 4096, 4096, 4096, 0, 8, 64, 2, 64, 2, None]

    def store(**kw):
        names = ["key", "value", "ks", "vs", "kc", "vc", "ksc", "vsc", "slots", "type", "n", "slots_n", "heads", "hd", "fmt", "stream"]
        a = dict(zip(names, ok))
        a.update(kw)
        return lib.dfx_kv_store_mx(*[a[n] for n in names])
    assert store(n=0) == 0
    for bad, status in ((dict(fmt=1), -1), (dict(hd=48), -2), (dict(ks=120), -1), (dict(ks=132), -1), (dict(key=4098), -1), (dict(type=2), -1),
                        (dict(vsc=None), -1), (dict(n=-1), -1), (dict(heads=0), -1), (dict(n=1 << 40), -2)):
        assert store(**bad) == status, bad


@pytest.mark.parametrize("extra", [dict(mscale=0.7), dict(truncate=False), dict(low_freq_factor=1.0)])
@pytest.mark.parametrize("kind", ["linear", "dynamic", "yarn"])
def test_settings_that_are_not_understood_are_refused(kind, extra):
    with pytest.raises(ValueError, match=next(iter(extra))):
        RotaryEmbedding(64, 64, 32, 1e4, rope_scaling=dict(rope_type=kind, factor=2.0, **extra))
    if kind != "yarn":
        with pytest.raises(ValueError, match="beta_fast"):
            RotaryEmbedding(64, 64, 32, 1e4, rope_scaling=dict(rope_type=kind, factor=2.0, beta_fast=16))


def test_get_rope_is_still_a_cache():
    a = get_rope(64, 64, 16, 1e4)
    assert get_rope.cache_info().currsize == 1
    get_rope.cache_clear()
    assert get_rope.cache_info().currsize == 0 and get_rope(64, 64, 16, 1e4) is not a


def test_settings_with_lists_reach_the_constructor():
    with pytest.raises(ValueError, match="unknown rope_scaling"):
        get_rope(64, 64, 16, 1e4, dict(rope_type="other", short_factor=[1.0, 2.0], nested=dict(a=[1])))
    with pytest.raises(ValueError, match="short_factor"):
        get_rope(64, 64, 16, 1e4, dict(rope_type="yarn", factor=2.0, short_factor=[1.0, 2.0]))
