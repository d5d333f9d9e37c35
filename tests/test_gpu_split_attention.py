"""GPU parity of dfx_split_attn (microscaled caches, shared prefixes) against 64-bit attention.

Tolerance.  The kernel's scores are fp32 sums of exact products, its weights 2^x in fp32 rounded to bf16 for the second product, its
sums fp32, its output rounded to bf16.  With w_j the true weights and d the largest relative error of a rounded weight against its
unrounded share of l, |o' - o| <= d * sum_j w_j |v_j| + half a step of the output.  d: half a step of bf16, 2^-8, plus
the scores' and the exponential's fp32 error: scores here are below 2^6 in units of log2 with 128 products each, at most
128 * 2^-24 * 2^6 < 2^-10.9 in the exponent in the worst case and 2^-14 in any real one.  A margin of 1 / 16 of 2^-8 covers
it and the fp32 sums: |o' - o| <= 2^-8 (1 + 1/16) (spread + |o|) + 1e-7, element by element."""
import types

import pytest
import torch

import diffulex_amd as dfx
from diffulex_amd import _lib
from oracle import mx, split

pytestmark = pytest.mark.gpu
FMTS = ["bf16", "e4m3", "e2m1"]


class Problem:
    """A batch: lengths, pages dealt at random, caches whose every byte behind the contexts is NaN."""

    def __init__(self, fmt, ctx, new, hq, hkv, hd, page, seed=0, groups=(), block_causal=False, dbs=4, spare_columns=1):
        """groups: (first sequence, one behind the last, prefix length); their sequences share whole pages of the prefix, and
        hold copies of the page in which it ends."""
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.ctx, self.new, self.hq, self.hkv, self.hd, self.page = fmt, ctx, new, hq, hkv, hd, page
        self.groups, self.block_causal, self.dbs = list(groups), block_causal, dbs
        b, t = len(ctx), sum(new)
        need = [-(-c // page) for c in ctx]
        shared = {s: (a, p) for a, e, p in groups for s in range(a, e)}
        self.table = torch.full((b, max(need + [1]) + spare_columns), -1, dtype=torch.int32)
        ids = torch.randperm(sum(need) + 3, generator=g).tolist()
        rows = lambda *shape: (torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-1, 2, (shape[-1],), generator=g).float())).to(torch.bfloat16)  # noqa: E731
        pages = len(ids)
        k, v = (torch.full((pages, page, hkv, hd), float("nan"), dtype=torch.bfloat16) for _ in range(2))
        for s in range(b):
            first, prefix = shared.get(s, (s, 0))
            for p in range(need[s]):
                n = min(page, ctx[s] - p * page)
                if first != s and (p + 1) * page <= min(prefix, ctx[first]):
                    self.table[s, p] = self.table[first, p]
                    continue
                i = ids.pop()
                self.table[s, p] = i
                k[i, :n], v[i, :n] = rows(n, hkv, hd), rows(n, hkv, hd)
                copy = min(prefix, ctx[first]) - p * page
                if first != s and copy > 0:
                    f = int(self.table[first, p])
                    m = min(copy, n)
                    k[i, :m], v[i, :m] = k[f, :m], v[f, :m]
        self.q, self.k, self.v = rows(t, hq, hd), rows(t, hkv, hd), rows(t, hkv, hd)
        self.scale = hd ** -0.5
        self.ks = self.vs = None
        if fmt == "bf16":
            self.kc, self.vc = k, v
            self.kv, self.vv = k.double(), v.double()
        else:
            (kc, self.ks), (vc, self.vs) = mx.quantise(k, fmt), mx.quantise(v, fmt)
            self.kc, self.vc = mx.pack(kc, fmt), mx.pack(vc, fmt)
            self.kv, self.vv = mx.values(self.kc, self.ks, fmt), mx.values(self.vc, self.vs, fmt)
        self.context_lens = torch.tensor(ctx, dtype=torch.int32)
        self.cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)

    def metadata(self, dev):
        m = types.SimpleNamespace(
            is_prefill=False, cu_seqlens_q=self.cu.to(dev), cu_seqlens_k=self.cu.to(dev), max_seqlen_q=max(self.new + [1]), max_seqlen_k=0,
            slot_mapping=None, context_lens=self.context_lens.to(dev), block_tables=self.table.to(dev), attn_type="block_attention",
            diffusion_block_size=self.dbs, decode_mode="static", kv_cache_layout="unified", need_kv_cache_store=False, seq_lens=None,
            seq_lens_ts=None, decode_mask="block_causal" if self.block_causal else "full")
        if self.groups:
            # (neighbouring groups; sequences between them are groups of their own with no prefix)
            cu, lens, at = [self.groups[0][0]], [], self.groups[0][0]
            for a, e, p in self.groups:
                if a > at:
                    lens.append(0)
                    cu.append(a)
                lens.append(p)
                cu.append(e)
                at = e
            m.prefix_cu_seqs, m.prefix_lens = torch.tensor(cu, dtype=torch.int32).to(dev), torch.tensor(lens, dtype=torch.int32).to(dev)
        return m

    def scales(self, dev):
        return dict(k_scale=None, v_scale=None) if self.ks is None else dict(k_scale=self.ks.to(dev), v_scale=self.vs.to(dev))

    def run(self, dev, **kw):
        m = self.metadata(dev)
        out = torch.full(self.q.shape, 77.0, dtype=torch.bfloat16, device=dev)
        args = dict(block_tables=m.block_tables, context_lens=m.context_lens, cu_seqlens_q=m.cu_seqlens_q, cu_seqlens_new=m.cu_seqlens_k,
                    max_seqlen_q=m.max_seqlen_q, mask_mode=int(self.block_causal), diffusion_block_size=self.dbs, out=out,
                    # (a bf16 cache without groups: one of no sequences, which routes the call here)
                    prefix_cu_seqs=getattr(m, "prefix_cu_seqs", torch.zeros(1, dtype=torch.int32, device=dev)),
                    prefix_lens=getattr(m, "prefix_lens", torch.zeros(0, dtype=torch.int32, device=dev)), **self.scales(dev))
        args.update(kw)
        dfx.paged_attention(self.q.to(dev), self.k.to(dev), self.v.to(dev), self.kc.to(dev), self.vc.to(dev), self.scale, **args)
        torch.cuda.synchronize()
        return out.cpu()

    def want(self):
        return split.attention(self.q, self.k, self.v, self.kv, self.vv, self.table, self.context_lens, self.cu, self.cu, self.scale,
                               self.block_causal, self.dbs)

    def check(self, got, want=None):
        o, spread, written = want if want is not None else self.want()
        assert (got[~written] == 77.0).all(), "a row without a key was written"
        got = got.double()
        tol = 2.0 ** -8 * (1 + 1 / 16) * (spread + o.abs()) + 1e-7
        bad = ~((got - o).abs() <= tol) & written[:, None, None]
        assert not bad.any(), f"{int(bad.sum())} elements off, worst {float(((got - o).abs() / tol)[written].max())} of the tolerance"


SHAPES = [  # hq, hkv, hd, page
    (1, 1, 128, 16), (28, 4, 128, 32), (4, 2, 64, 7), (16, 1, 64, 256), (32, 32, 128, 64), (6, 3, 128, 1)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
def test_single_tokens(dev, fmt, hq, hkv, hd, page):
    p = Problem(fmt, [0, 1, 31, 32, 33, 64, 65, 127, 128, 129, 700, 0], [1] * 11 + [0], hq, hkv, hd, page, seed=1)
    p.check(p.run(dev))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
@pytest.mark.parametrize("block_causal", [False, True])
def test_ragged_blocks(dev, fmt, hq, hkv, hd, page, block_causal):
    p = Problem(fmt, [5, 0, 300, 64, 63, 1, 0, 130], [7, 33, 32, 1, 65, 0, 3, 12], hq, hkv, hd, page, seed=2, block_causal=block_causal)
    p.check(p.run(dev))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("prefix", [32, 100, 256])
@pytest.mark.parametrize("hq,hkv,hd,page", SHAPES)
def test_shared_prefix(dev, fmt, prefix, hq, hkv, hd, page):
    ctx = [prefix + x for x in (0, 1, 40, 17, 70, 5)]
    p = Problem(fmt, ctx, [1, 3, 1, 4, 2, 0], hq, hkv, hd, page, seed=3, groups=[(0, 6, prefix)], block_causal=True, dbs=2)
    p.check(p.run(dev))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new", [[1] * 14, [32] * 14, [1, 9, 0, 33, 2, 1, 70, 4, 1, 1, 5, 6, 7, 8]])
def test_several_groups_and_sequences_outside_them(dev, fmt, new):
    """Groups of 5, 1 and 4 sequences, prefixes that end inside a page and a tile, one of nothing; sequences before, between and
    behind them; contexts that end inside their group's prefix, one of them empty."""
    ctx = [40, 200, 230, 150, 0, 201, 33, 97, 300, 90, 91, 45, 90, 10]
    p = Problem(fmt, ctx, new, 14, 2, 128, 16, seed=4, groups=[(1, 6, 200), (7, 8, 70), (8, 12, 90)], block_causal=True, dbs=4)
    p.check(p.run(dev))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("n_wg", [1, 2, 5, 64, 513])
def test_any_number_of_workgroups(dev, fmt, n_wg):
    """Every way of cutting the work: whole items, pieces of several, pieces of one key tile."""
    p = Problem(fmt, [700, 650, 1, 900], [1, 20, 3, 1], 28, 4, 128, 32, seed=5, groups=[(0, 2, 600)])
    want = p.want()
    got = p.run(dev, max_workgroups=n_wg)
    p.check(got, want)
    assert torch.equal(got, p.run(dev, max_workgroups=n_wg)), "two calls differ"


@pytest.mark.parametrize("fmt", FMTS)
def test_long_context_one_sequence(dev, fmt):
    p = Problem(fmt, [30011], [1], 8, 2, 128, 64, seed=6)
    p.check(p.run(dev))


@pytest.mark.parametrize("fmt", FMTS)
def test_skipped_pages_and_ids_outside_the_cache(dev, fmt):
    p = Problem(fmt, [200, 64, 32, 100], [1, 2, 0, 40], 8, 2, 128, 16, seed=7)
    p.table[0, 3], p.table[0, 5], p.table[3, 0] = -1, p.kc.shape[0], 1 << 30
    p.table[1, :4] = -7                                    # nothing but the fresh rows
    p.check(p.run(dev))
    q = Problem(fmt, [64, 40], [2, 1], 8, 2, 128, 16, seed=8)
    q.table[0] = -1
    cu_new = torch.tensor([0, 0, 0], dtype=torch.int32, device=dev)   # no fresh rows either: zeros, the reference divides 0 by 0
    got = q.run(dev, cu_seqlens_new=cu_new)
    assert (got[:2] == 0).all()
    o, spread, written = split.attention(q.q, q.k, q.v, q.kv, q.vv, q.table, q.context_lens, q.cu, cu_new.cpu(), q.scale)
    q.check(got, (o, spread, written))


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_non_finite_blocks_reach_their_own_sequence_only(dev, fmt):
    p = Problem(fmt, [50, 50], [1, 1], 2, 1, 64, 16, seed=9)
    p.vs[int(p.table[0, 0]), 3, 0, 1] = 255
    got = p.run(dev)
    assert torch.isnan(got[0, :, 32:]).all() and not torch.isnan(got[0, :, :32]).any() and not torch.isnan(got[1]).any()
    p.vv = mx.values(p.vc, p.vs, fmt)
    p.vv[int(p.table[0, 0])] = 0.0
    want = p.want()
    p.check(torch.cat([torch.full_like(got[:1], 77.0), got[1:]]), (want[0], want[1], torch.tensor([False, True])))


def test_large_scores_and_infinities(dev):
    """Scores thousands apart (the running maximum moves often, first weights vanish), one key that is infinite."""
    p = Problem("bf16", [300], [4], 4, 1, 128, 16, seed=10)
    p.kc = p.kc * torch.linspace(0.1, 60, p.kc.shape[0]).view(-1, 1, 1, 1).to(torch.bfloat16)
    p.kv = p.kc.double()
    got = p.run(dev)
    o, spread, written = p.want()
    # scores up to 2^12: 128 products' sums are off by at most 128 * 2^-24 * 2^12 = 2^-5 in the exponent
    assert ((got.double() - o).abs() <= (2.0 ** -8 + 2.0 ** -5) * (spread + o.abs()) + 1e-7).all()


def test_operand_strides_and_a_layer_view_of_the_cache(dev):
    """q, k, v as column slices of one projection, out as a slice, the cache a view whose pages are not neighbours."""
    p = Problem("bf16", [100, 40, 260], [5, 1, 33], 6, 2, 128, 16, seed=11, groups=[(0, 2, 32)])
    t = p.q.shape[0]
    proj = torch.cat([p.q.flatten(1), p.k.flatten(1), p.v.flatten(1), torch.zeros(t, 16, dtype=torch.bfloat16)], 1).to(dev)
    q, k, v = (proj[:, a * 128:(a + n) * 128].unflatten(1, (n, 128)) for a, n in ((0, 6), (6, 2), (8, 2)))
    pages = torch.full((p.kc.shape[0], 3, 16, 2, 128), float("nan"), dtype=torch.bfloat16, device=dev)
    pages[:, 0], pages[:, 2] = p.kc.to(dev), p.vc.to(dev)
    out = torch.full((t, 8, 128), 77.0, dtype=torch.bfloat16, device=dev)
    m = p.metadata(dev)
    dfx.paged_attention(q, k, v, pages[:, 0], pages[:, 2], p.scale, block_tables=m.block_tables, context_lens=m.context_lens,
                        cu_seqlens_q=m.cu_seqlens_q, cu_seqlens_new=m.cu_seqlens_k, max_seqlen_q=0, out=out[:, 1:7],
                        prefix_cu_seqs=m.prefix_cu_seqs, prefix_lens=m.prefix_lens)
    torch.cuda.synchronize()
    p.check(out[:, 1:7].cpu())
    assert (out[:, 0] == 77.0).all() and (out[:, 7] == 77.0).all()


def test_rows_behind_the_last_sequence_and_offsets_beyond_the_operands(dev):
    p = Problem("e4m3", [50, 60, 0, 0], [2, 3, 0, 0], 4, 2, 64, 16, seed=12)
    p.q = torch.cat([p.q, torch.full((6, 4, 64), float("nan"), dtype=torch.bfloat16)])   # a padded batch
    m = p.metadata(dev)
    got = p.run(dev)
    assert (got[5:] == 77.0).all()
    want = p.want()
    p.check(got, want)
    # offsets that promise more rows than there are
    cu_new = torch.tensor([0, 2, 900, 900, 900], dtype=torch.int32, device=dev)
    cu_q = torch.tensor([0, 2, 5, 1 << 20, 1 << 20], dtype=torch.int32, device=dev)
    got = p.run(dev, cu_seqlens_new=cu_new, cu_seqlens_q=cu_q)
    p.check(got[:5], tuple(x[:5] for x in want))
    del m


def test_offsets_beyond_32_bits(dev):
    """Pages at the end of caches of more than 2^32 bytes (bf16: more than 2^32 elements)."""
    for fmt, page, hkv, hd in (("bf16", 256, 8, 128), ("e4m3", 256, 8, 128), ("e2m1", 256, 8, 128)):
        p = Problem(fmt, [600, 520], [1, 3], 16, hkv, hd, page, seed=13)
        width = p.kc.shape[-1] * p.kc.element_size()
        pages = (1 << 32) * p.kc.element_size() // (page * hkv * width) + p.kc.shape[0]
        shift = pages - p.kc.shape[0]
        big = [torch.empty((pages,) + tuple(p.kc.shape[1:]), dtype=p.kc.dtype, device=dev) for _ in range(2)]
        sc = dict(k_scale=None, v_scale=None)
        for b, c in zip(big, (p.kc, p.vc)):
            b[:256].zero_()
            b[shift:] = c.to(dev)
        if fmt != "bf16":
            sc = {n: torch.empty((pages,) + tuple(s.shape[1:]), dtype=torch.uint8, device=dev) for n, s in (("k_scale", p.ks), ("v_scale", p.vs))}
            sc["k_scale"][shift:], sc["v_scale"][shift:] = p.ks.to(dev), p.vs.to(dev)
        m = p.metadata(dev)
        m.block_tables = torch.where(m.block_tables >= 0, m.block_tables + shift, m.block_tables)
        out = dfx.paged_attention(p.q.to(dev), p.k.to(dev), p.v.to(dev), *big, p.scale, block_tables=m.block_tables,
                                  context_lens=m.context_lens, cu_seqlens_q=m.cu_seqlens_q, cu_seqlens_new=m.cu_seqlens_k, max_seqlen_q=0,
                                  prefix_lens=torch.zeros(0, dtype=torch.int32, device=dev),
                                  prefix_cu_seqs=torch.zeros(1, dtype=torch.int32, device=dev), **sc)
        torch.cuda.synchronize()
        p.check(out.cpu())
        if fmt != "bf16":
            slots = (m.block_tables[0, :1].long() * page + torch.arange(4, device=dev)).to(torch.int64)
            rows = torch.randn(4, hkv, hd, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
            dfx.store_kvcache_unified_layout(rows.to(dev), rows.to(dev), *big, slots, None, **sc)
            codes, b = mx.quantise(rows, fmt)
            at = int(m.block_tables[0, 0])
            assert torch.equal(big[0][at, :4].cpu(), mx.pack(codes, fmt)) and torch.equal(sc["v_scale"][at, :4].cpu(), b)
            md = types.SimpleNamespace(block_tables=m.block_tables[:1], context_lens=torch.tensor([4], dtype=torch.int32, device=dev),
                                       seq_lens_ts=torch.zeros(1, dtype=torch.int32, device=dev), max_seqlen_k=4,
                                       cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=dev),
                                       cu_seqlens_k=torch.tensor([0, 4], dtype=torch.int32, device=dev))
            none = torch.empty(0, hkv, hd, dtype=torch.bfloat16, device=dev)
            kk, _ = dfx.load_kvcache(*big, md, none, none, **sc)
            assert torch.equal(kk.cpu().double(), mx.values(mx.pack(codes, fmt), b, fmt))
        del big, sc
        torch.cuda.empty_cache()


def test_two_graphs_replayed_with_other_lengths(dev):
    """Captured once at full lengths, replayed with the lengths and tables of other steps, in turn with another graph and eager
    calls on another stream."""
    ps = [Problem("e4m3", c, [2, 1, 4, 1], 8, 2, 128, 16, seed=20 + i, groups=[(0, 3, 48)]) for i, c in
          enumerate(([400, 300, 90, 33], [48, 49, 50, 0], [64, 399, 200, 70]))]
    pages = max(p.kc.shape[0] for p in ps)
    width = max(p.table.shape[1] for p in ps)
    kc, vc = (torch.zeros((pages,) + tuple(ps[0].kc.shape[1:]), dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((pages,) + tuple(ps[0].ks.shape[1:]), dtype=torch.uint8, device=dev) for _ in range(2))
    m = ps[0].metadata(dev)
    m.block_tables = torch.full((4, width), -1, dtype=torch.int32, device=dev)
    q, k, v = (x.to(dev) for x in (ps[0].q, ps[0].k, ps[0].v))

    def load(p):
        for dst, src in ((kc, p.kc), (vc, p.vc), (ks, p.ks), (vs, p.vs)):
            dst[:src.shape[0]] = src.to(dev)
        m.block_tables.fill_(-1)
        m.block_tables[:, :p.table.shape[1]] = p.table.to(dev)
        m.context_lens.copy_(p.context_lens)
        for dst, src in ((q, p.q), (k, p.k), (v, p.v)):
            dst.copy_(src)

    def call():
        return dfx.dllm_flash_attn_decode(q, k, v, kc, vc, ps[0].scale, m, k_scale=ks, v_scale=vs)

    load(ps[0])
    call()
    graphs, outs = [], []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    side = torch.cuda.Stream()
    for p in (*ps, ps[1], ps[0]):
        load(p)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = call()
        for g, o in zip(graphs, outs):
            o.fill_(77.0)
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], eager)
        p.check(outs[0].cpu())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_store_travels_with_the_call(dev, fmt):
    p = Problem(fmt, [40, 20], [3, 2], 4, 2, 64, 16, seed=30)
    m = p.metadata(dev)
    kc, vc, ks, vs = (x.to(dev) for x in (p.kc, p.vc, p.ks, p.vs))
    slots = torch.tensor([40, 41, 42, 20, 21])
    rows = [0, 0, 0, 1, 1]
    slots = torch.stack([p.table[r, int(x) // 16] * 16 + int(x) % 16 for r, x in zip(rows, slots)]).to(torch.int32)
    out = dfx.dllm_flash_attn_decode(p.q.to(dev), p.k.to(dev), p.v.to(dev), kc, vc, p.scale, m, k_scale=ks, v_scale=vs,
                                     store_slot_mapping=slots.to(dev))
    torch.cuda.synchronize()
    p.check(out.cpu())
    codes, b = mx.quantise(p.k, fmt)
    assert torch.equal(kc.cpu().flatten(0, 1)[slots.long()], mx.pack(codes, fmt)) and torch.equal(ks.cpu().flatten(0, 1)[slots.long()], b)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1", "bf16"])
def test_decoding_steps_through_the_attention_module(dev, fmt):
    """A run as a model makes it: two steps of a batch that shares a prompt, scaled and partly rotated positions, each step rotated,
    stored and attended through Attention.forward, the second reading what the first wrote."""
    hq, hkv, hd, page, prefix, n = 8, 2, 128, 16, 96, 4
    g = torch.Generator().manual_seed(40)
    rope = dfx.get_rope(hd, 64, 512, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=128), False).to(dev)
    att = dfx.Attention(hq, hd, hd ** -0.5, hkv)
    p = Problem(fmt, [prefix + 3, prefix + 20, prefix], [n, n, n], hq, hkv, hd, page, seed=41, groups=[(0, 3, prefix)], spare_columns=2)
    # pages for the steps' rows
    pages = p.kc.shape[0]
    extra = torch.arange(pages, pages + 6, dtype=torch.int32).view(3, 2)
    for s in range(3):
        have = -(-p.ctx[s] // page)
        p.table[s, have:have + 2] = extra[s]
    grow = lambda x: torch.cat([x, torch.zeros((6,) + tuple(x.shape[1:]), dtype=x.dtype)])  # noqa: E731
    att.k_cache, att.v_cache = grow(p.kc).to(dev), grow(p.vc).to(dev)
    if fmt != "bf16":
        att.k_scale, att.v_scale = grow(p.ks).to(dev), grow(p.vs).to(dev)
    p.kv, p.vv = grow(p.kv), grow(p.vv)
    m = p.metadata(dev)
    m.need_kv_cache_store = True
    dfx.set_fetch_fn_for_attn_metadata(lambda: m)
    for step in range(2):
        x = torch.randn(3 * n, (hq + 2 * hkv) * hd, generator=g).to(torch.bfloat16)
        pos = torch.cat([c + torch.arange(n) for c in p.ctx])
        row = torch.arange(3).repeat_interleave(n)
        slots = p.table[row, pos // page] * page + pos % page
        m.slot_mapping = slots.to(torch.int32).to(dev)
        m.context_lens = torch.tensor(p.ctx, dtype=torch.int32, device=dev)
        d = x.to(dev)
        q, k, v = d[:, :hq * hd], d[:, hq * hd:(hq + hkv) * hd], d[:, (hq + hkv) * hd:]
        out = att(q, k, v, rope=(rope, pos.to(dev)))
        torch.cuda.synchronize()
        # what the module should have computed, from the oracle of each part
        f = x[:, :(hq + hkv) * hd].float().view(3 * n, -1, hd)
        cs = rope.cos_sin_cache.cpu()[pos]
        c, s = cs[:, None, :32], cs[:, None, 32:]
        a, b = f[..., 0:64:2], f[..., 1:64:2]
        f = torch.cat([torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2), f[..., 64:]], -1).to(torch.bfloat16)
        p.q, p.k, p.v = f[:, :hq], f[:, hq:], x[:, (hq + hkv) * hd:].view(3 * n, hkv, hd)
        p.context_lens = torch.tensor(p.ctx, dtype=torch.int32)
        p.check(out.view(3 * n, hq, hd).cpu())
        for rows, values, cache, scale in ((p.k, p.kv, att.k_cache, att.k_scale), (p.v, p.vv, att.v_cache, att.v_scale)):
            if fmt == "bf16":
                values.flatten(0, 1)[slots.long()] = rows.double()
                assert torch.equal(cache.cpu().flatten(0, 1)[slots.long()], rows)
            else:
                codes, sb = mx.quantise(rows, fmt)
                values.flatten(0, 1)[slots.long()] = mx.values(mx.pack(codes, fmt), sb, fmt)
                assert torch.equal(cache.cpu().flatten(0, 1)[slots.long()], mx.pack(codes, fmt))
                assert torch.equal(scale.cpu().flatten(0, 1)[slots.long()], sb)
        p.ctx = [c + n for c in p.ctx]


def test_agrees_with_the_unshared_kernel(dev):
    """The same batch with and without the promise of a shared prefix: two kernels, each within the tolerance of the truth."""
    p = Problem("bf16", [300, 280, 301], [4, 4, 4], 28, 4, 128, 32, seed=50, groups=[(0, 3, 256)])
    m = p.metadata(dev)
    got = dfx.dllm_flash_attn_decode(p.q.to(dev), p.k.to(dev), p.v.to(dev), p.kc.to(dev), p.vc.to(dev), p.scale, m)
    del m.prefix_lens, m.prefix_cu_seqs
    plain = dfx.dllm_flash_attn_decode(p.q.to(dev), p.k.to(dev), p.v.to(dev), p.kc.to(dev), p.vc.to(dev), p.scale, m)
    torch.cuda.synchronize()
    want = p.want()
    p.check(got.cpu(), want)
    p.check(plain.cpu(), want)


def test_refusals(dev):
    p = Problem("e4m3", [40, 20], [3, 2], 4, 2, 64, 16, seed=60, groups=[(0, 2, 16)])
    i32 = dict(dtype=torch.int32, device=dev)
    m = p.metadata(dev)
    for kw in (dict(prefix_cu_seqs=None), dict(prefix_cu_seqs=torch.zeros(3, **i32)), dict(prefix_lens=m.prefix_lens.long()),
               dict(prefix_lens=torch.zeros(9, **i32), prefix_cu_seqs=torch.zeros(10, **i32)),   # more groups than sequences
               dict(static_scratch=True), dict(cache_layout="distinct"), dict(rope=(torch.zeros(8, 64, device=dev), torch.zeros(5, **i32))),
               dict(mask_mode=2), dict(mask_mode=1, diffusion_block_size=0), dict(max_workgroups=-1), dict(max_workgroups=1 << 20),
               dict(context_lens=m.context_lens[:1]), dict(block_tables=m.block_tables.long()), dict(k_scale=p.ks[..., :1].to(dev))):
        with pytest.raises((RuntimeError, AssertionError)):
            p.run(dev, **kw)
    kc = p.kc.to(dev)
    with pytest.raises(RuntimeError, match="shared prefixes"):   # FP8 codes with one scale per head
        dfx.paged_attention(p.q.to(dev), p.k.to(dev), p.v.to(dev), kc.view(torch.float8_e4m3fn), kc.view(torch.float8_e4m3fn), p.scale,
                            block_tables=m.block_tables, context_lens=m.context_lens, cu_seqlens_q=m.cu_seqlens_q,
                            cu_seqlens_new=m.cu_seqlens_k, max_seqlen_q=0, prefix_cu_seqs=m.prefix_cu_seqs, prefix_lens=m.prefix_lens,
                            k_scale=torch.ones(2, device=dev), v_scale=torch.ones(2, device=dev))
    for bad_scale in (0.0, -1.0, float("nan"), float("inf")):
        p.scale = bad_scale
        with pytest.raises(_lib.DfxError):
            p.run(dev)


def test_nothing_to_do(dev):
    p = Problem("e4m3", [40, 20], [0, 0], 4, 2, 64, 16, seed=61)
    assert p.run(dev).shape == (0, 4, 64)
    no_cache = Problem("bf16", [0, 0], [5, 2], 4, 2, 64, 16, seed=62)
    out = torch.full(no_cache.q.shape, 77.0, dtype=torch.bfloat16, device=dev)
    m = no_cache.metadata(dev)
    dfx.paged_attention(no_cache.q.to(dev), no_cache.k.to(dev), no_cache.v.to(dev), None, None, no_cache.scale, block_tables=None,
                        context_lens=None, cu_seqlens_q=m.cu_seqlens_q, cu_seqlens_new=m.cu_seqlens_k, max_seqlen_q=5, out=out,
                        prefix_cu_seqs=torch.zeros(1, dtype=torch.int32, device=dev), prefix_lens=torch.zeros(0, dtype=torch.int32, device=dev))
    torch.cuda.synchronize()
    no_cache.check(out.cpu())


@pytest.mark.parametrize("n_wg", [7, 9, 10, 13, 15, 37, 100])
def test_numbers_of_workgroups_that_the_dies_do_not_share_evenly(dev, n_wg):
    """No range of the work may be left without a workgroup."""
    p = Problem("e2m1", [900, 650, 40, 1200], [1, 20, 3, 1], 28, 4, 128, 32, seed=6, groups=[(0, 2, 600)])
    p.check(p.run(dev, max_workgroups=n_wg))


@pytest.mark.parametrize("batch,groups", [(300, 0), (700, 0), (640, 600), (1100, 3)])
def test_more_virtual_sequences_than_threads(dev, batch, groups):
    """A thread then lists several of them, and the merge looks a row block's up among several per thread (from 1025 blocks on with four waves)."""
    ctx = [(s * 37) % 61 + (8 if groups else 0) for s in range(batch)]
    new = [(s * 7) % 4 for s in range(batch)]
    each = max(batch // groups, 1) if groups else 0
    p = Problem("e4m3", ctx, new, 4, 2, 64, 8, seed=7, groups=[(g * each, (g + 1) * each, 8) for g in range(groups)])
    p.check(p.run(dev))


def test_narrow_and_wide_items_side_by_side(dev):
    p = Problem("bf16", [50, 10, 900] * 20, [1, 3, 20] * 20, 28, 4, 128, 32, seed=8, groups=[(0, 20, 7)])
    want = p.want()
    for n_wg in (0, 2, 12):
        p.check(p.run(dev, max_workgroups=n_wg), want)


def test_two_calls_at_once_on_two_streams(dev):
    """Each call has a workspace of its own."""
    a = Problem("e4m3", [400, 900, 33], [5, 1, 2], 28, 4, 128, 32, seed=9)
    b = Problem("e2m1", [1300, 64], [40, 7], 8, 2, 64, 16, seed=10)
    wa, wb = a.want(), b.want()
    ma, mb = a.metadata(dev), b.metadata(dev)
    on = lambda p: [x.to(dev) for x in (p.q, p.k, p.v, p.kc, p.vc)]  # noqa: E731
    ta, tb, sa, sb = on(a), on(b), a.scales(dev), b.scales(dev)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(one):
            ga = dfx.dllm_flash_attn_decode(*ta, a.scale, ma, **sa)
        with torch.cuda.stream(two):
            gb = dfx.dllm_flash_attn_decode(*tb, b.scale, mb, **sb)
        got.append((ga, gb))
    torch.cuda.synchronize()
    for ga, gb in got:
        a.check(ga.cpu(), wa)
        b.check(gb.cpu(), wb)


def _check_with_non_finite(p, got, want):
    """NaN and infinities where the oracle has them, its values within the tolerance elsewhere."""
    o, spread, written = want
    assert (got[~written] == 77.0).all()
    got = got.double()
    assert torch.equal(torch.isnan(got)[written], torch.isnan(o)[written])
    inf = torch.isinf(o) & written[:, None, None]
    assert (got[inf] == o[inf]).all()
    ok = torch.isfinite(o) & written[:, None, None]
    tol = 2.0 ** -8 * (1 + 1 / 16) * (spread + o.abs()) + 1e-7
    assert ((got - o).abs() <= tol)[ok].all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("hq,hkv,hd", [(28, 4, 128), (4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("n_wg", [0, 3, 40])
def test_non_finite_values_of_a_prefix_reach_the_rows_that_see_them_only(dev, fmt, new, hq, hkv, hd, n_wg):
    """Values of two keys of a shared prefix are infinite or NaN; some sequences of the group end before the second, or before
    both, one has no context at all: for them these keys do not exist, whatever shares their tiles."""
    p = Problem(fmt, [200, 40, 230, 0, 130, 200, 90], [new] * 7, hq, hkv, hd, 16, seed=70, groups=[(0, 7, 200)])
    for pos in (70, 150):
        at, off = int(p.table[0, pos // 16]), pos % 16
        if fmt == "bf16":
            p.vc[at, off, 0, 3], p.vc[at, off, -1, 40], p.vc[at, off, -1, 41] = float("nan"), float("inf"), float("-inf")
        else:
            p.vs[at, off, 0, 0] = p.vs[at, off, -1, 1] = 255
    p.vv = p.vc.double() if fmt == "bf16" else mx.values(p.vc, p.vs, fmt)
    want = p.want()
    rows = torch.arange(7).repeat_interleave(new)
    clean = (rows == 1) | (rows == 3)
    assert torch.isfinite(want[0][clean]).all() and not torch.isfinite(want[0][~clean]).flatten(1).all(-1).any()
    _check_with_non_finite(p, p.run(dev, max_workgroups=n_wg), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("hq,hkv,hd", [(28, 4, 128), (4, 2, 64), (1, 1, 128)])
@pytest.mark.parametrize("n_wg", [0, 5])
def test_non_finite_values_of_fresh_rows_reach_the_blocks_that_see_them_only(dev, fmt, hq, hkv, hd, n_wg):
    p = Problem(fmt, [50, 0, 300], [12, 9, 40], hq, hkv, hd, 16, seed=71, block_causal=True, dbs=4)
    bad = {0: 6, 1: 8, 2: 37}                              # sequence: fresh row, in its blocks 1, 2 and 9
    clean = Problem(fmt, [50, 0, 300], [12, 9, 40], hq, hkv, hd, 16, seed=71, block_causal=True, dbs=4)
    sees = torch.zeros(p.q.shape[0], dtype=torch.bool)
    for s, j in bad.items():
        a = int(p.cu[s])
        p.v[a + j, :, 5], p.v[a + j, :, 33] = float("nan"), float("inf")
        sees[a + j // 4 * 4:int(p.cu[s + 1])] = True
    got = p.run(dev, max_workgroups=n_wg)
    assert torch.isnan(got[sees][..., 5]).all() and (got[sees][..., 33] == float("inf")).all()
    want = clean.want()
    keep = ~sees[:, None, None].expand_as(got) | (torch.arange(hd) != 5) & (torch.arange(hd) != 33)
    clean.check(torch.where(keep, got.double(), want[0]), want)


@pytest.mark.parametrize("n_wg", [0, 1, 30])
@pytest.mark.parametrize("new", [1, 40])
def test_an_infinite_key(dev, new, n_wg):
    """An element of one cached key is infinite: its score is +inf for the rows whose element there is positive -- they have no softmax, NaN --
    and -inf for the others, which go on as if the key were not there."""
    p = Problem("bf16", [300, 64], [new, new], 8, 2, 128, 16, seed=72)
    p.q[:, :, 9] = torch.where(p.q[:, :, 9] == 0, torch.ones_like(p.q[:, :, 9]), p.q[:, :, 9])
    p.kc[int(p.table[0, 7]), 3, :, 9] = float("inf")
    p.kv = p.kc.double()
    nan = (p.q[:, :, 9] > 0) & (torch.arange(2 * new) < new)[:, None]
    assert nan.any() and not nan[:new].all()
    got = p.run(dev, max_workgroups=n_wg)
    assert torch.isnan(got[nan]).all() and not torch.isnan(got[~nan]).any()
    p.kv[int(p.table[0, 7]), 3, :, 9] = 1e9                # for the oracle: weight exp(-1e9 |q|) = 0 in 64 bits where the element is negative
    o, spread, written = p.want()
    p.check(torch.where(nan[..., None], o, got.double()), (o, spread, written))
