"""GPU parity of the microscaled KV cache's store and load against the 64-bit oracle: equal bits (powers of two as scales make
every code and every widened value exact)."""
import pytest
import torch

import diffulex_amd as dfx
from diffulex_amd import _lib
from oracle import mx

pytestmark = pytest.mark.gpu
FMTS = ["e4m3", "e2m1"]


def _empty(fmt, pages, page, heads, hd, dev, fill=7):
    """(k_cache, v_cache, k_scale, v_scale) filled with a byte that a store has to leave where it writes nothing."""
    width = hd if fmt == "e4m3" else hd // 2
    c = [torch.full((pages, page, heads, width), fill, dtype=torch.uint8, device=dev) for _ in range(2)]
    s = [torch.full((pages, page, heads, hd // 32), fill, dtype=torch.uint8, device=dev) for _ in range(2)]
    return (*c, *s)


def _rows(n, heads, hd, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, hd, generator=g) * torch.exp2(torch.randint(-9, 10, (n, heads, hd), generator=g).float())
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n,heads,hd,slot_dtype", [(1, 1, 32, torch.int32), (77, 4, 128, torch.int64), (300, 3, 96, torch.int32),
                                                   (2049, 2, 64, torch.int32)])
def test_store_bit_exact(dev, fmt, n, heads, hd, slot_dtype):
    page = 16
    pages = n // page + 9
    k, v = _rows(n, heads, hd, 1), _rows(n, heads, hd, 2)
    g = torch.Generator().manual_seed(3)
    slots = torch.randperm(pages * page, generator=g)[:n].to(slot_dtype)
    slots[::5] = -1
    if n > 8:
        slots[1], slots[7] = pages * page, pages * page + 12345   # behind the cache: skipped
    kc, vc, ks, vs = _empty(fmt, pages, page, heads, hd, dev)
    qkv = torch.cat([k.flatten(1), torch.zeros(n, 8, dtype=torch.bfloat16), v.flatten(1)], 1).to(dev)   # rows with a longer stride
    gk, gv = qkv[:, :heads * hd].unflatten(1, (heads, hd)), qkv[:, heads * hd + 8:].unflatten(1, (heads, hd))
    dfx.store_kvcache_unified_layout(gk, gv, kc, vc, slots.to(dev), None, k_scale=ks, v_scale=vs.view(torch.float8_e8m0fnu))
    torch.cuda.synchronize()
    keep = (slots >= 0) & (slots < pages * page)
    for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
        codes, b = mx.quantise(x, fmt)
        want, want_s = (t.cpu().clone().flatten(0, 1).fill_(7) for t in (cache, scale))
        want[slots[keep].long()], want_s[slots[keep].long()] = mx.pack(codes, fmt)[keep], b[keep]
        assert torch.equal(cache.cpu().flatten(0, 1), want)
        assert torch.equal(scale.cpu().flatten(0, 1), want_s)


@pytest.mark.parametrize("fmt", FMTS)
def test_store_every_bf16(dev, fmt):
    """Every bf16 pattern, alone in its block and beside a larger neighbour: zeros of both signs, subnormals, ties, the largest
    values, infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536, 2, 32, dtype=torch.bfloat16)
    x[:, 0, 3] = bits
    x[:, 1, 11], x[:, 1, 30] = bits, 1.75
    kc, vc, ks, vs = _empty(fmt, 4096, 16, 2, 32, dev)
    slots = torch.arange(65536, dtype=torch.int32, device=dev)
    g = x.to(dev)
    dfx.store_kvcache_unified_layout(g, g, kc, vc, slots, None, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    codes, b = mx.quantise(x, fmt)
    assert torch.equal(ks.cpu().flatten(0, 1), b) and torch.equal(vs, ks)
    assert torch.equal(kc.cpu().flatten(0, 1), mx.pack(codes, fmt)) and torch.equal(vc, kc)


class _MD:
    pass


def _contexts(lens, new, page, seed, skip=None):
    """Metadata of a read: pages dealt at random, one spare column of -1."""
    g = torch.Generator().manual_seed(seed)
    b = len(lens)
    need = [-(-c // page) for c in lens]
    perm = torch.randperm(sum(need) + 2, generator=g).to(torch.int32)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    if skip is not None:
        table[skip] = -1
    m = _MD()
    m.block_tables, m.context_lens = table, torch.tensor(lens, dtype=torch.int32)
    m.seq_lens_ts, m.seq_lens = torch.tensor(new, dtype=torch.int32), None
    m.cu_seqlens_q = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    m.cu_seqlens_k = torch.tensor([0] + [c + n for c, n in zip(lens, new)]).cumsum(0).to(torch.int32)
    m.max_seqlen_k = max(c + n for c, n in zip(lens, new))
    return m, sum(need) + 2


def _to(m, dev):
    for k, v in vars(m).items():
        if isinstance(v, torch.Tensor):
            setattr(m, k, v.to(dev))
    return m


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,new,page,heads,hd", [([1], [0], 16, 1, 32), ([0, 65, 64, 7], [3, 1, 0, 32], 16, 2, 64),
                                                    ([1000, 333], [5, 6], 256, 4, 128), ([50, 20], [1, 1], 7, 3, 96)])
def test_load_bit_exact(dev, fmt, lens, new, page, heads, hd):
    m, pages = _contexts(lens, new, page, 5)
    g = torch.Generator().manual_seed(6)
    kc, vc, ks, vs = _empty(fmt, pages, page, heads, hd, "cpu")
    top = 254                                             # (all codes but E4M3's NaN; scales of every size, one NaN block)
    for c in (kc, vc):
        c.copy_(torch.randint(0, 127, c.shape, generator=g) + 128 * torch.randint(0, 2, c.shape, generator=g))
    for s in (ks, vs):
        s.copy_(torch.randint(90, 150, s.shape, generator=g))
    ks[0, 0, 0, 0], vs[0, 0, 0, 0], ks[-1, 0, 0, 0], vs[-1, 0, 0, 0] = 255, 0, top - 8, 255
    t = sum(new)
    kn, vn = _rows(t, heads, hd, 7), _rows(t, heads, hd, 8)
    want = []
    for c, s, fresh in ((kc, ks, kn), (vc, vs, vn)):
        val = mx.values(c, s, fmt).flatten(0, 1)
        rows = []
        for i, (n, q) in enumerate(zip(lens, new)):
            pos = torch.arange(n)
            rows.append(val[m.block_tables[i][pos // page].long() * page + pos % page])
            a = int(m.cu_seqlens_q[i])
            rows.append(fresh[a:a + q].double())
        want.append(torch.cat(rows).to(torch.bfloat16))
    dm = _to(m, dev)
    got = dfx.load_kvcache(kc.to(dev), vc.to(dev), dm, kn.to(dev), vn.to(dev), k_scale=ks.to(dev), v_scale=vs.to(dev))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert a.dtype == torch.bfloat16
        a = a.cpu()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(a.view(torch.int16)[~torch.isnan(b)], b.view(torch.int16)[~torch.isnan(b)])


@pytest.mark.parametrize("fmt", FMTS)
def test_store_then_load_in_place_out_and_skipped_page(dev, fmt):
    page, heads, hd, lens = 16, 2, 128, [40, 33]
    m, pages = _contexts(lens, [0, 0], page, 9)
    rows = _rows(sum(lens), heads, hd, 10)
    slots = torch.cat([m.block_tables[i][torch.arange(n) // page] * page + torch.arange(n) % page for i, n in enumerate(lens)])
    kc, vc, ks, vs = _empty(fmt, pages, page, heads, hd, dev)
    dfx.store_kvcache_unified_layout(rows.to(dev), (-rows).to(dev), kc, vc, slots.to(dev), None, k_scale=ks, v_scale=vs)
    m.block_tables[0, 1] = -1                              # rows 16..31 of the first sequence: left as they were
    out = tuple(torch.full((sum(lens), heads, hd), 3.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    empty = torch.empty(0, heads, hd, dtype=torch.bfloat16, device=dev)
    got = dfx.load_kvcache(kc, vc, _to(m, dev), empty, empty, k_scale=ks, v_scale=vs, out=out)
    torch.cuda.synchronize()
    assert got[0] is out[0] and got[1] is out[1]
    codes, b = mx.quantise(rows, fmt)
    want = mx.values(mx.pack(codes, fmt), b, fmt)
    want[16:32] = 3.0
    assert torch.equal(out[0].cpu().double(), want)
    want[:16], want[32:] = -want[:16], -want[32:]
    assert torch.equal(out[1].cpu().double(), want)


def test_refusals(dev):
    kc, vc, ks, vs = _empty("e4m3", 4, 16, 2, 64, dev)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(3, dtype=torch.int32, device=dev)
    store = dfx.store_kvcache_unified_layout
    for bad in (dict(key=x.half()), dict(key=x[:2]), dict(slot_mapping=slots[:2]), dict(slot_mapping=slots.float()),
                dict(k_cache=kc.bfloat16()), dict(k_cache=kc[..., :32]), dict(k_scale=ks[..., :1]), dict(v_scale=vs[:2]),
                dict(key=x[..., :32], value=x[..., :32]), dict(k_cache=kc[:, :, :1], v_cache=vc[:, :, :1])):
        a = dict(key=x, value=x, k_cache=kc, v_cache=vc, slot_mapping=slots, attn_metadata=None, k_scale=ks, v_scale=vs)
        a.update(bad)
        with pytest.raises((RuntimeError, AssertionError)):
            store(**a)
    # head_dim 48 is no number of blocks, a key row off 16 bytes cannot be moved in chunks
    flat = torch.zeros(3 * 2 * 64 + 8, dtype=torch.bfloat16, device=dev)
    off = flat[1:1 + 3 * 128].view(3, 2, 64)
    with pytest.raises(_lib.DfxError, match="invalid argument"):
        store(off, x, kc, vc, slots, None, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert (kc == 7).all() and (vc == 7).all() and (ks == 7).all() and (vs == 7).all()
    with pytest.raises(AssertionError):
        dfx.load_kvcache(x.view(1, 3, 2, 64), x.view(1, 3, 2, 64), _MD(), x, x, out=(x, x))


def test_store_recorded_into_a_graph_and_on_another_stream(dev):
    page, heads, hd, n = 16, 2, 128, 40
    rows = [_rows(n, heads, hd, s).to(dev) for s in (20, 21, 22)]
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:n].to(torch.int32).to(dev)
    x = rows[0].clone()
    kc, vc, ks, vs = _empty("e4m3", 4, page, heads, hd, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dfx.store_kvcache_unified_layout(x, x, kc, vc, slots, None, k_scale=ks, v_scale=vs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dfx.store_kvcache_unified_layout(x, x, kc, vc, slots, None, k_scale=ks, v_scale=vs)
    for r in rows:
        x.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        codes, b = mx.quantise(r.cpu(), "e4m3")
        assert torch.equal(kc.cpu().flatten(0, 1)[slots.cpu().long()], codes) and torch.equal(ks.cpu().flatten(0, 1)[slots.cpu().long()], b)


def _load_all(kc, vc, ks, vs, dev):
    """Every row of a cache, loaded as one context."""
    m = _MD()
    n = kc.shape[0] * kc.shape[1]
    i32 = dict(dtype=torch.int32, device=dev)
    m.block_tables, m.context_lens = torch.arange(kc.shape[0], **i32)[None], torch.tensor([n], **i32)
    m.seq_lens_ts, m.seq_lens, m.max_seqlen_k = torch.zeros(1, **i32), None, n
    m.cu_seqlens_q, m.cu_seqlens_k = torch.zeros(2, **i32), torch.tensor([0, n], **i32)
    none = torch.empty(0, kc.shape[2], ks.shape[3] * 32, dtype=torch.bfloat16, device=dev)
    out = dfx.load_kvcache(kc.to(dev), vc.to(dev), m, none, none, k_scale=ks.to(dev), v_scale=vs.to(dev))
    torch.cuda.synchronize()
    return tuple(x.cpu() for x in out)


@pytest.mark.parametrize("fmt", FMTS)
def test_load_every_scale_and_code(dev, fmt):
    """All 256 scale bytes with all codes: code * 2^(b - 127) rounded to bf16 (which it is already, but for products below bf16's smallest
    subnormal), 2^128 and more an infinity."""
    codes = 256 if fmt == "e4m3" else 16
    rows = max(codes // 32, 1)
    c = torch.arange(codes).repeat(32 // min(codes, 32)).view(rows, 32).to(torch.uint8).repeat(256, 1)
    kc = mx.pack(c, fmt).reshape(-1, 8, 1, 32 if fmt == "e4m3" else 16)
    ks = torch.arange(256, dtype=torch.uint8).repeat_interleave(rows).view(-1, 8, 1, 1)
    want = mx.values(kc, ks, fmt).flatten(0, 1).to(torch.bfloat16)
    for got in _load_all(kc, kc.clone(), ks, ks.clone(), dev):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got.view(torch.int16)[ok], want.view(torch.int16)[ok])


@pytest.mark.parametrize("fmt", FMTS)
def test_every_finite_bf16_stored_and_loaded_is_finite(dev, fmt):
    """What a store writes is a bf16 for every finite row: the load widens it exactly.  Up to half a step of the code's grid from the row, or one step in
    the last binade, where the nearest code would stand for 2^128."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    bits = bits[torch.isfinite(bits)]
    n = bits.numel()                                       # 65280 = 4080 pages of 16
    x = torch.zeros(n, 2, 32, dtype=torch.bfloat16)
    x[:, 0, 3] = bits
    x[:, 1, 11], x[:, 1, 30] = bits, 1.75
    kc, vc, ks, vs = _empty(fmt, n // 16, 16, 2, 32, dev)
    g = x.to(dev)
    dfx.store_kvcache_unified_layout(g, -g, kc, vc, torch.arange(n, dtype=torch.int32, device=dev), None, k_scale=ks, v_scale=vs)
    got, negated = _load_all(kc, vc, ks, vs, dev)
    assert torch.isfinite(got).all() and torch.equal(negated.double(), -got.double())
    codes, b = mx.quantise(x, fmt)
    assert torch.equal(got.double(), mx.values(mx.pack(codes, fmt), b, fmt))
