"""GPU parity of the rotary embedding's other forms: interleaved pairs, part of the head, scaled frequencies, and their stores.

Rotated values: the kernel's fp32 arithmetic (two rounded products, one rounded sum) is restated on the CPU from the module's
table and compared bit for bit; the table itself is compared with the formulas in 64 bits (tests/test_rotary_tables.py)."""
import pytest
import torch

from diffulex_amd import _lib
from diffulex_amd.rotary_embedding import RotaryEmbedding
from oracle import fp8_e4m3, mx

pytestmark = pytest.mark.gpu
MAXPOS, BASE = 4096, 1.0e6
YARN = dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=1024)


def _want(x, pos, table, hd, rot, neox):
    """fp32, each product and sum rounded on its own, then bf16 (CPU tensors; x: [T, H * hd])."""
    T = x.shape[0]
    f = x.float().reshape(T, -1, hd)
    cs = table[pos.long().clamp(0, table.shape[0] - 1)]
    c, s = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    a, b = (f[..., :rot // 2], f[..., rot // 2:rot]) if neox else (f[..., 0:rot:2], f[..., 1:rot:2])
    y1, y2 = a * c - b * s, b * c + a * s
    y = torch.cat((y1, y2), -1) if neox else torch.stack((y1, y2), -1).flatten(-2)
    return torch.cat((y, f[..., rot:]), -1).to(torch.bfloat16).reshape(x.shape)


def _inputs(T, hq, hkv, hd, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, (hq + 2 * hkv) * hd, generator=g).to(torch.bfloat16), torch.randint(0, MAXPOS, (T,), generator=g).to(dtype))


def _bits(t):
    t = t.cpu().contiguous()
    return t.view({1: torch.uint8, 2: torch.int16}[t.element_size()])


FORMS = [(128, 128, False, None), (128, 64, True, None), (128, 64, False, YARN), (128, 32, True, dict(type="linear", factor=2.5)),
         (64, 16, False, None), (64, 32, True, YARN), (96, 48, True, None), (80, 80, False, None), (16, 16, False, None),
         (128, 128, True, YARN)]


@pytest.mark.parametrize("hd,rot,neox,scaling", FORMS)
@pytest.mark.parametrize("T,hq,hkv,dtype", [(1, 1, 1, torch.int64), (77, 6, 2, torch.int32), (1500, 28, 4, torch.int64)])
def test_forward_bit_exact(dev, hd, rot, neox, scaling, T, hq, hkv, dtype):
    qkv, pos = _inputs(T, hq, hkv, hd, seed=T + hd + rot, dtype=dtype)
    rope = RotaryEmbedding(hd, rot, MAXPOS, BASE, is_neox_style=neox, rope_scaling=scaling).to(dev)
    table = rope.cos_sin_cache.cpu()
    q, k = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd]
    g = qkv.to(dev)
    got_q, got_k = rope(pos.to(dev), g[:, :hq * hd], g[:, hq * hd:(hq + hkv) * hd])
    torch.cuda.synchronize()
    assert torch.equal(_bits(got_q), _bits(_want(q, pos, table, hd, rot, neox)))
    assert torch.equal(_bits(got_k), _bits(_want(k, pos, table, hd, rot, neox)))
    assert torch.equal(_bits(g), _bits(qkv))


def test_positions_outside_the_table_read_nothing_outside(dev):
    rope = RotaryEmbedding(64, 32, 16, BASE, is_neox_style=False).to(dev)
    x, _ = _inputs(4, 1, 1, 64, seed=1)
    pos = torch.tensor([-5, 15, 16, 1 << 40])
    got, _ = rope(pos.to(dev), x[:, :64].to(dev), x[:, 64:128].to(dev))
    assert torch.equal(_bits(got), _bits(_want(x[:, :64], pos, rope.cos_sin_cache.cpu(), 64, 32, False)))


@pytest.mark.parametrize("hd,rot,neox", [(128, 128, True), (128, 64, True), (128, 32, False), (64, 64, False), (128, 32, True), (96, 32, True)])
@pytest.mark.parametrize("cache", ["bf16", "fp8", "e4m3", "e2m1"])
@pytest.mark.parametrize("slot_dtype", [torch.int32, torch.int64])
def test_store_of_rotated_rows(dev, hd, rot, neox, cache, slot_dtype):
    """(128, 32, True) and (96, 32, True) with microscaled caches: blocks straddle the rotated halves, two launches."""
    T, hq, hkv, page, pages = 333, 5, 2, 16, 24
    qkv, pos = _inputs(T, hq, hkv, hd, seed=11)
    q, k, v = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd], qkv[:, (hq + hkv) * hd:]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(12))[:T].to(slot_dtype)
    slots[::6] = -1
    slots[5] = pages * page + 3
    keep = (slots >= 0) & (slots < pages * page)
    rope = RotaryEmbedding(hd, rot, MAXPOS, BASE, is_neox_style=neox, rope_scaling=YARN).to(dev)
    table = rope.cos_sin_cache.cpu()
    width = {"bf16": hd, "fp8": hd, "e4m3": hd, "e2m1": hd // 2}[cache]
    kc = [torch.full((pages, page, hkv, width), 7, dtype=torch.uint8, device=dev) for _ in range(2)]
    if cache == "bf16":
        kc = [c.bfloat16() for c in kc]
    if cache == "fp8":
        sc = [torch.tensor([0.01, 0.02], device=dev), torch.tensor([0.015, 0.03], device=dev)]
        kc = [c.view(torch.float8_e4m3fn) for c in kc]
    elif cache == "bf16":
        sc = [None, None]
    else:
        sc = [torch.full((pages, page, hkv, hd // 32), 7, dtype=torch.uint8, device=dev) for _ in range(2)]
    g = qkv.to(dev)
    got_q, got_k = rope.forward_and_store(pos.to(dev), g[:, :hq * hd], g[:, hq * hd:(hq + hkv) * hd], g[:, (hq + hkv) * hd:], kc[0],
                                          kc[1], slots.to(dev), k_scale=sc[0], v_scale=sc[1])
    torch.cuda.synchronize()
    want_k = _want(k, pos, table, hd, rot, neox)
    assert torch.equal(_bits(got_q), _bits(_want(q, pos, table, hd, rot, neox))) and torch.equal(_bits(got_k), _bits(want_k))
    for rows, got, s in ((want_k, kc[0], sc[0]), (v, kc[1], sc[1])):
        rows = rows.reshape(T, hkv, hd)
        want = torch.full((pages * page, hkv, width), 7, dtype=torch.uint8)
        if cache == "bf16":
            want = want.bfloat16()
            want[slots[keep].long()] = rows[keep]
        elif cache == "fp8":
            want[slots[keep].long()] = torch.from_numpy(fp8_e4m3.quantize_per_head(rows.float().numpy(), s.cpu().numpy()))[keep]
        else:
            codes, b = mx.quantise(rows, cache)
            want[slots[keep].long()] = mx.pack(codes, cache)[keep]
            want_s = torch.full((pages * page, hkv, hd // 32), 7, dtype=torch.uint8)
            want_s[slots[keep].long()] = b[keep]
            assert torch.equal(s.cpu().flatten(0, 1), want_s)
        assert torch.equal(_bits(got).flatten(0, 1), _bits(want))


def test_distinct_layout_takes_two_launches(dev):
    T, hkv, hd, page, pages = 70, 2, 64, 16, 8
    qkv, pos = _inputs(T, hkv, hkv, hd, seed=3)
    rope = RotaryEmbedding(hd, 32, MAXPOS, BASE, is_neox_style=False).to(dev)
    g = qkv.to(dev)
    q, k, v = g[:, :hkv * hd], g[:, hkv * hd:2 * hkv * hd], g[:, 2 * hkv * hd:]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(4))[:T].to(torch.int32)
    kc = torch.zeros(pages, hkv, hd // 8, page, 8, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros(pages, hkv, hd, page, dtype=torch.bfloat16, device=dev)
    _, got_k = rope.forward_and_store(pos.to(dev), q, k, v, kc, vc, slots.to(dev))
    torch.cuda.synchronize()
    want = _want(qkv[:, hkv * hd:2 * hkv * hd], pos, rope.cos_sin_cache.cpu(), hd, 32, False)
    assert torch.equal(_bits(got_k), _bits(want))
    for t in range(0, T, 13):
        p, o = int(slots[t]) // page, int(slots[t]) % page
        assert torch.equal(kc[p, :, :, o].reshape(hkv, hd).cpu(), want[t].view(hkv, hd))
        assert torch.equal(vc[p, :, :, o].cpu(), qkv[t, 2 * hkv * hd:].view(hkv, hd))


def test_in_place_through_the_c_abi(dev):
    import ctypes as C
    T, hq, hkv, hd, rot = 200, 8, 2, 128, 64
    for inter in (0, 1):
        qkv, pos = _inputs(T, hq, hkv, hd, seed=4)
        rope = RotaryEmbedding(hd, rot, MAXPOS, BASE, is_neox_style=not inter).to(dev)
        tab = rope.cos_sin_cache.cpu()
        want = qkv.clone()
        want[:, :(hq + hkv) * hd] = _want(qkv[:, :(hq + hkv) * hd], pos, tab, hd, rot, not inter)
        g, gp = qkv.to(dev), pos.to(dev)
        p = _lib.RopeParams()
        p.q = p.q_out = g.data_ptr()
        p.k = p.k_out = g.data_ptr() + hq * hd * 2
        p.q_stride_token = p.k_stride_token = p.q_out_stride_token = p.k_out_stride_token = g.stride(0)
        p.positions, p.position_index_type = gp.data_ptr(), _lib.DFX_INDEX_I64
        p.cos_sin_cache, p.max_position = rope.cos_sin_cache.data_ptr(), MAXPOS
        p.n_tokens, p.num_q_heads, p.num_kv_heads, p.head_dim, p.rotary_dim, p.interleaved = T, hq, hkv, hd, rot, inter
        assert _lib.load().dfx_rope_kv_store(C.byref(p), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(_bits(g), _bits(want))


def test_refusals(dev):
    x = torch.zeros(4, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(_lib.DfxError, match="unsupported"):
        RotaryEmbedding(128, 24, 64, BASE).to(dev)(pos, x, x)          # not a multiple of 16
    rope = RotaryEmbedding(128, 64, 64, BASE).to(dev)
    with pytest.raises(RuntimeError):
        rope(pos[:3], x, x)
    with pytest.raises(RuntimeError):
        rope(pos, x.half(), x)


@pytest.mark.parametrize("interleaved", [False, True])
def test_tensors_the_kernel_cannot_reach_are_refused(dev, interleaved):
    """Positions, slots, caches or scales in host memory, outputs of other shapes: an error before anything is launched."""
    op = _lib.ops().rope_kv_store
    t, hq, hk, hd = 4, 4, 2, 64
    bf = dict(dtype=torch.bfloat16, device=dev)
    q, k, v = torch.zeros(t, hq * hd, **bf), torch.zeros(t, hk * hd, **bf), torch.zeros(t, hk * hd, **bf)
    good = dict(positions=torch.arange(t, device=dev), query=q, key=k, q_out=torch.empty_like(q), k_out=torch.empty_like(k),
                cos_sin_cache=torch.zeros(8, hd, device=dev), head_size=hd, value=v,
                k_cache=torch.zeros(2, 16, hk, hd, dtype=torch.uint8, device=dev), v_cache=torch.zeros(2, 16, hk, hd, dtype=torch.uint8, device=dev),
                slot_mapping=torch.arange(t, device=dev), k_scale=torch.zeros(2, 16, hk, hd // 32, dtype=torch.uint8, device=dev),
                v_scale=torch.zeros(2, 16, hk, hd // 32, dtype=torch.uint8, device=dev), rotary_dim=0, interleaved=interleaved)
    fp8 = dict(good, k_scale=torch.ones(hk, device=dev), v_scale=torch.ones(hk, device=dev))
    for args in (good, fp8):
        op(**args)
        for name in ("positions", "cos_sin_cache", "value", "k_cache", "v_cache", "slot_mapping", "k_scale", "v_scale", "q_out", "k_out"):
            with pytest.raises(RuntimeError):
                op(**dict(args, **{name: args[name].cpu()}))
        for bad in (dict(q_out=torch.empty(t - 1, hq * hd, **bf)), dict(k_out=torch.empty(t, hd, **bf)), dict(q_out=torch.empty(t, hq * hd, device=dev)),
                    dict(k_out=torch.empty(t, 2 * hk * hd, **bf)[:, ::2])):
            with pytest.raises(RuntimeError):
                op(**dict(args, **bad))
    torch.cuda.synchronize()
