"""Cases that measure the rotary embedding's forms, the microscaled KV cache and the attention that reads it.

An operator is named by a case's "op":

* ``rope``: rotary embedding of q and k (half or interleaved pairs, part of the head, scaled frequencies);
* ``rope_write``: the same with the store of k and v into a microscaled cache in the same call;
* ``write``: store of fresh k and v rows into an MXFP8 cache (E4M3 codes, one power-of-two scale per 32 elements);
* ``read``: gather of every sequence's context through its block table, widened to bf16, fresh rows appended;
* ``write_read``: the store of the step's rows followed by the read of the whole contexts;
* ``attn``: decode attention over a microscaled cache (``mx8``: E4M3, ``mx4``: E2M1) and the fresh rows;
* ``prefix``: decode attention of groups of sequences that share a prefix (bf16 or microscaled cache).
"""
import math
import random

import torch

own = False

BLOCK = 32                                                   # elements per scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)              # magnitudes of the 4-bit codes 0..7


def listed():
    return [
        # one token of each of 64 sequences, pairs interleaved over half of each head
        dict(name="rope_step_interleaved", op="rope", tokens=64, hq=32, hkv=32, hd=128, rot=64, neox=False, scaling="none", maxpos=8192),
        # one decoding step of 64 blocks of 32 tokens, frequencies scaled for a long context, k and v into the cache
        dict(name="rope_write_step", op="rope_write", tokens=2048, hq=28, hkv=4, hd=128, rot=128, neox=True, scaling="yarn",
             maxpos=131072, page=256, slots=32768),
        # prompts of 65 thousand tokens in all, position interpolation
        dict(name="rope_prompt", op="rope", tokens=65521, hq=28, hkv=4, hd=128, rot=64, neox=True, scaling="linear", maxpos=65536),
        # one block of 32 tokens of each of 8 sequences
        dict(name="write_step", op="write", tokens=256, hkv=4, hd=128, page=32, slots=16384),
        # a packed prompt batch of odd length, 32 KV heads
        dict(name="write_prompt", op="write", tokens=16385, hkv=32, hd=128, page=256, slots=32768),
        # contexts of a batch of 64 read back
        dict(name="read_batch", op="read", fmt="mx8", seqs=64, hkv=4, hd=128, page=256, lo=256, hi=2048, new=32),
        # a few long contexts in 4 bits: the step's rows written, then everything read back
        dict(name="write_read_long", op="write_read", fmt="mx4", seqs=3, hkv=4, hd=128, page=32, lo=9000, hi=33000, new=5),
        # single tokens of a small batch: latency
        dict(name="attn_token", op="attn", fmt="mx8", seqs=8, hq=28, hkv=4, hd=128, page=32, lo=100, hi=1000, new=1, mask="full", dbs=32),
        # single tokens over long contexts in 4 bits
        dict(name="attn_token_long", op="attn", fmt="mx4", seqs=5, hq=32, hkv=32, hd=128, page=64, lo=20000, hi=60000, new=1, mask="full", dbs=32),
        # blocks of 32 tokens, 28 / 4 heads, a batch of 128 at prefixes of 2048 to 8192
        dict(name="attn_block_batch", op="attn", fmt="mx8", seqs=128, hq=28, hkv=4, hd=128, page=256, lo=2048, hi=8192, new=32, mask="full", dbs=32),
        # 64 samples of one prompt, one token each
        dict(name="prefix_token", op="prefix", fmt="bf16", seqs=64, groups=1, prefix=4096, hq=28, hkv=4, hd=128, page=256, lo=1, hi=512, new=1,
             mask="full", dbs=32),
        # four prompts with 64 samples each, blocks of 4 tokens, of which up to 12 are in flight
        dict(name="prefix_groups", op="prefix", fmt="mx8", seqs=256, groups=4, prefix=8192, hq=28, hkv=4, hd=128, page=32, lo=16, hi=700, new=12,
             mask="block_causal", dbs=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "rope_write", "write", "read", "write_read", "attn", "attn", "prefix", "prefix"))
    hd = rng.choice((64, 128, 128))
    hq, hkv = rng.choice(((28, 4), (32, 32), (4, 2), (32, 8), (16, 1)))
    page = rng.choice((16, 32, 64, 256))
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 40000), hq=hq, hkv=hkv, hd=hd, rot=rng.choice((hd // 4, hd // 2, hd)), neox=rng.random() < 0.5,
                    scaling=rng.choice(("none", "linear", "dynamic", "yarn")), maxpos=rng.choice((8192, 65536, 131072)))
    if op == "rope_write":
        tokens = _log(rng, 1, 8000)
        return dict(op=op, tokens=tokens, hq=hq, hkv=hkv, hd=hd, rot=rng.choice((hd // 2, hd)), neox=rng.random() < 0.5,
                    scaling=rng.choice(("none", "dynamic", "yarn")), maxpos=32768, page=page, slots=256 * (-(-tokens // 256) + 8))
    if op == "write":
        tokens = _log(rng, 1, 16000)
        return dict(op=op, tokens=tokens, hkv=hkv, hd=hd, page=page, slots=256 * (-(-tokens // 256) + 8))
    if op in ("read", "write_read"):
        hi = _log(rng, 40, 30000)
        return dict(op=op, fmt=rng.choice(("mx8", "mx4")), seqs=_log(rng, 1, max(2, 2_000_000 // (hi * hkv))), hkv=hkv, hd=hd, page=page,
                    lo=max(1, hi // 4), hi=hi, new=rng.choice((1, 3, 32)))
    new = rng.choice((1, 1, 4, 7, 32))
    mask = rng.choice(("full", "block_causal"))
    dbs = rng.choice((1, 4, 32))
    if op == "attn":
        hi = _log(rng, 60, 60000)
        return dict(op=op, fmt=rng.choice(("mx8", "mx4")), seqs=_log(rng, 1, max(2, 1_200_000 // (hi * hkv))), hq=hq, hkv=hkv, hd=hd, page=page,
                    lo=max(0, hi // 5), hi=hi, new=new, mask=mask, dbs=dbs)
    prefix = page * max(1, _log(rng, 128, 12000) // page)
    groups = rng.choice((1, 1, 2, 5))
    return dict(op=op, fmt=rng.choice(("bf16", "mx8", "mx4")), seqs=groups * rng.randint(1, max(2, min(60, 8_000_000 // (prefix * groups * hkv)))),
                groups=groups, prefix=prefix, hq=hq, hkv=hkv, hd=hd, page=page, lo=0, hi=_log(rng, 8, 600), new=new, mask=mask, dbs=dbs)


# ---- what a case's sizes are -------------------------------------------------------------------
def _lengths(case):
    """(context lengths, fresh rows) of the case's sequences: of the case alone, so that work() knows them."""
    rng = random.Random("%d %d %d %d" % (case["seqs"], case["lo"], case["hi"], case["new"]))
    ctx = [case.get("prefix", 0) + rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    # (one row, three rows or a whole block per sequence; more than one block where several are in flight)
    new = [case["new"] if case["new"] in (1, 32) else rng.randint(1, case["new"]) for _ in range(case["seqs"])]
    return ctx, new


def _row_bytes(fmt, hd):
    return {"bf16": 2 * hd, "mx8": hd + hd // BLOCK, "mx4": hd // 2 + hd // BLOCK}[fmt]


def work(case):
    hd, hkv = case["hd"], case["hkv"]
    if case["op"] in ("rope", "rope_write"):
        t, rows = case["tokens"], case["hq"] + hkv
        size = t * rows * hd * 4 + t * (4 * case["rot"] + 8)
        if case["op"] == "rope_write":
            size += t * hkv * (hd * 2 + 2 * _row_bytes("mx8", hd)) + 8 * t
        return {"bytes": size, "flops": 3 * t * rows * case["rot"]}
    if case["op"] == "write":
        return {"bytes": case["tokens"] * (hkv * (4 * hd + 2 * _row_bytes("mx8", hd)) + 4), "flops": 4 * case["tokens"] * hkv * hd}
    ctx, new = _lengths(case)
    row = hkv * _row_bytes(case["fmt"], hd)
    if case["op"] in ("read", "write_read"):
        size = 2 * sum(ctx) * (row + 2 * hkv * hd) + 2 * sum(new) * hkv * hd * 4
        if case["op"] == "write_read":
            size += 2 * sum(new) * (row + hkv * hd * 2)
        return {"bytes": size, "flops": 2 * sum(ctx) * hkv * hd}
    shared = case.get("prefix", 0)
    keys = sum(c - shared for c in ctx) + case.get("groups", 0) * shared
    size = 2 * keys * row + sum(new) * (case["hq"] * hd * 4 + hkv * hd * 4)
    return {"bytes": size, "flops": 4 * hd * case["hq"] * sum(n * (c + n) for c, n in zip(ctx, new))}


# ---- inputs -----------------------------------------------------------------------------------
def _scaling(case):
    return {"none": None, "linear": dict(rope_type="linear", factor=4.0), "dynamic": dict(rope_type="dynamic", factor=2.0,
            original_max_position_embeddings=4096),
            "yarn": dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=16384)}[case["scaling"]]


def _angles(case, positions):
    """cos and sin in 64 bits of the given positions for every rotated pair, scaled as the case says (without its repository's code)."""
    dim, base, maxpos = case["rot"], 1.0e6, case["maxpos"]
    i = torch.arange(0, dim, 2, dtype=torch.float64, device=positions.device)
    gain = 1.0
    if case["scaling"] == "dynamic":     # the base grows so that the table's last position keeps the original's resolution
        base = base * (2.0 * maxpos / 4096 - 1.0) ** (dim / (dim - 2))
    freq = base ** (-i / dim)
    if case["scaling"] == "linear":
        freq = freq / 4.0
    if case["scaling"] == "yarn":        # slow pairs are interpolated, fast ones kept, a ramp between
        turn = [dim * math.log(16384 / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32, 1)]
        low, high = max(math.floor(turn[0]), 0), min(math.ceil(turn[1]), dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / 8.0 * ramp + freq * (1 - ramp)
        gain = 0.1 * math.log(8.0) + 1.0
    a = positions.double()[:, None] * freq[None, :]
    return a.cos() * gain, a.sin() * gain


def _quantise(x, fmt):
    """bf16 rows [.., hd] -> (codes, scale bytes): per 32 elements the smallest power of two that brings them into the codes' range."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(amax)
    e = (p - 9 + (m > 0.875).int() if fmt == "mx8" else p - 3 + (m > 0.75).int()).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    bad = ~torch.isfinite(amax)
    y = torch.where(bad, torch.zeros_like(b), torch.ldexp(b, -e))
    scales = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8).squeeze(-1)
    if fmt == "mx8":
        return y.flatten(-2).to(torch.float8_e4m3fn), scales
    a = y.abs()
    # ties go to the even code
    code = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int()
    code = (code + 8 * torch.signbit(y).int()).flatten(-2).unflatten(-1, (-1, 2))
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scales


def _values(codes, scales, fmt):
    """What the codes stand for, in 32 bits."""
    if fmt == "bf16":
        return codes.float()
    if fmt == "mx8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
        c = codes.view(torch.uint8).int()
        v = table[torch.stack((c & 15, c >> 4), -1).flatten(-2)]
    e = scales.view(torch.uint8).int() - 127
    s = torch.where(e == 128, torch.full(e.shape, float("nan"), device=e.device), torch.ldexp(torch.ones(e.shape, device=e.device), e))
    return (v.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _bf16(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _cache(g, fmt, pages, page, hkv, hd):
    """K or V rows of a cache: channels of unequal size, as keys have them."""
    x = _bf16(g, pages, page, hkv, hd) * torch.exp2(torch.randint(-1, 2, (hkv, hd), generator=g, device="cuda").float()).to(torch.bfloat16)
    if fmt == "bf16":
        return x, None
    done = [_quantise(p, fmt) for p in x.split(max(1, (1 << 25) // (page * hkv * hd)))]
    return torch.cat([d[0].view(torch.uint8) for d in done]).view(done[0][0].dtype), torch.cat([d[1] for d in done])


class _Metadata:
    """The attributes of a decoding step's metadata object that the operators read."""

    is_prefill, kv_cache_layout, need_kv_cache_store, decode_mode, attn_type = False, "unified", True, "static", "block_attention"


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    op, hd, hkv = case["op"], case["hd"], case["hkv"]
    s = {"case": case}
    if op in ("rope", "rope_write"):
        t, hq = case["tokens"], case["hq"]
        qkv = _bf16(g, t, (hq + 2 * hkv) * hd)           # column slices of one projection
        s["q"], s["k"], s["v"] = qkv[:, :hq * hd], qkv[:, hq * hd:(hq + hkv) * hd], qkv[:, (hq + hkv) * hd:]
        s["positions"] = torch.randint(0, case["maxpos"], (t,), generator=g, device="cuda")
        if own:
            from diffulex_amd import RotaryEmbedding
            s["rope"] = RotaryEmbedding(hd, case["rot"], case["maxpos"], 1.0e6, is_neox_style=case["neox"], rope_scaling=_scaling(case)).to("cuda")
        else:
            cos, sin = _angles(case, torch.arange(case["maxpos"], device="cuda"))
            s["table"] = torch.cat((cos, sin), -1).float()
    if op in ("rope_write", "write"):
        t = case["tokens"]
        if op == "write":
            kv = _bf16(g, t, 2, hkv, hd)
            s["k"], s["v"] = kv[:, 0], kv[:, 1]
        s["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:t].to(torch.int32)
        for n in "kv":
            s[n + "_cache"] = torch.zeros(case["slots"] // case["page"], case["page"], hkv, hd, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
            s[n + "_scale"] = torch.zeros(case["slots"] // case["page"], case["page"], hkv, hd // BLOCK, dtype=torch.uint8, device="cuda")
        return s
    if op == "rope":
        return s
    ctx, new = _lengths(case)
    page, shared = case["page"], case.get("prefix", 0)
    b, per = case["seqs"], case["seqs"] // max(1, case.get("groups", 0))
    first = shared // page                               # pages that a group's sequences have in common
    n_pages = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    pages = case.get("groups", 0) * first + sum(n - first for n in n_pages)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((b, max(n_pages) + 1), -1, dtype=torch.int32)
    at = case.get("groups", 0) * first
    for i, n in enumerate(n_pages):
        if first:
            table[i, :first] = perm[(i // per) * first:(i // per + 1) * first]
        table[i, first:n] = perm[at:at + n - first]
        at += n - first
    m = _Metadata()
    m.block_tables = table.cuda()
    m.context_lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    m.seq_lens_ts = torch.tensor(new, dtype=torch.int32).cuda()
    m.seq_lens = None
    m.cu_seqlens_q = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    m.max_seqlen_q = max(new)
    m.cu_seqlens_k = m.cu_seqlens_q
    m.diffusion_block_size = case.get("dbs", 32)
    m.decode_mask = case.get("mask", "full")
    s["k_cache"], s["k_scale"] = _cache(g, case["fmt"], pages, page, hkv, hd)
    s["v_cache"], s["v_scale"] = _cache(g, case["fmt"], pages, page, hkv, hd)
    t = sum(new)
    s["k"], s["v"] = _bf16(g, t, hkv, hd), _bf16(g, t, hkv, hd)
    if op in ("read", "write_read"):
        m.cu_seqlens_k = torch.tensor([0] + [c + n for c, n in zip(ctx, new)]).cumsum(0).to(torch.int32).cuda()
        m.max_seqlen_k = max(c + n for c, n in zip(ctx, new))
        total = sum(ctx) + t
        # where the step's rows go: behind the contexts, in the sequences' own pages
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, new)])
        row = torch.repeat_interleave(torch.arange(b), torch.tensor(new))
        s["slots"] = (table[row, pos // page] * page + pos % page).to(torch.int32).cuda()
        s["out"] = tuple(torch.empty(total, hkv, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    else:
        s["q"] = _bf16(g, t, case["hq"], hd)
        if op == "prefix":
            m.prefix_cu_seqs = torch.arange(0, b + 1, per, dtype=torch.int32).cuda()
            m.prefix_lens = torch.full((case["groups"],), shared, dtype=torch.int32).cuda()
    # index arrays of the plain form, which knows the lengths as a host program does
    s["rows"] = torch.repeat_interleave(torch.arange(b), torch.tensor(new)).cuda()
    s["place"] = torch.cat([torch.arange(n) for n in new]).cuda()
    s["ctx_rows"] = torch.repeat_interleave(torch.arange(b), torch.tensor(ctx)).cuda()
    s["ctx_place"] = torch.cat([torch.arange(c) for c in ctx]).cuda()
    s["metadata"], s["longest"], s["most"] = m, max(ctx), max(new)
    return s


# ---- plain forms -------------------------------------------------------------------------------
def _rotate(x, cos, sin, case):
    """x: [T, H * hd]; cos, sin: [T, rot / 2]."""
    hd, rot = case["hd"], case["rot"]
    x = x.float().unflatten(-1, (-1, hd))
    r, rest = x[..., :rot], x[..., rot:]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if case["neox"] else (r[..., 0::2], r[..., 1::2])
    cos, sin = cos[:, None, :], sin[:, None, :]
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.cat((a, b), -1) if case["neox"] else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((y, rest), -1).flatten(-2).to(torch.bfloat16)


def _plain_write(s, k, v, fmt):
    slots = s["slots"].long()
    for n, x in (("k", k), ("v", v)):
        codes, scales = _quantise(x, fmt)
        s[n + "_cache"].view(torch.uint8).flatten(0, 1)[slots] = codes.view(torch.uint8)
        s[n + "_scale"].flatten(0, 1)[slots] = scales


def _plain_read(s):
    case, m = s["case"], s["metadata"]
    page, start = case["page"], m.cu_seqlens_k.long()
    slot = m.block_tables[s["ctx_rows"], s["ctx_place"] // page].long() * page + s["ctx_place"] % page
    for n, out in zip("kv", s["out"]):
        cached = s[n + "_cache"].view(torch.uint8).flatten(0, 1)[slot]
        out[start[s["ctx_rows"]] + s["ctx_place"]] = _values(cached, s[n + "_scale"].flatten(0, 1)[slot], case["fmt"]).to(torch.bfloat16)
        out[start[s["rows"]] + m.context_lens.long()[s["rows"]] + s["place"]] = s[n]
    return s["out"]


def _plain_attention(s):
    case, m = s["case"], s["metadata"]
    hq, hkv, hd, page, longest, most = case["hq"], case["hkv"], case["hd"], case["page"], s["longest"], s["most"]
    b, g = m.context_lens.numel(), hq // hkv
    pos = torch.arange(longest, device="cuda")
    slot = (m.block_tables[:, pos // page].long() * page + pos % page).clamp(min=0)
    seen = pos[None, :] < m.context_lens[:, None]                                       # [B, L]
    padded = [torch.zeros(b, most, h, hd, device="cuda") for h in (hq, hkv, hkv)]
    for p, n in zip(padded, "qkv"):
        p[s["rows"], s["place"]] = s[n].float()
    keys = [torch.cat((torch.where(seen[:, :, None, None], _values(
        s[n + "_cache"].flatten(0, 1)[slot] if case["fmt"] == "bf16" else s[n + "_cache"].view(torch.uint8).flatten(0, 1)[slot],
        None if case["fmt"] == "bf16" else s[n + "_scale"].flatten(0, 1)[slot], case["fmt"]), 0.0), p), 1).transpose(1, 2)
        for n, p in (("k", padded[1]), ("v", padded[2]))]                               # [B, Hkv, L + most, hd]
    q = padded[0].unflatten(2, (hkv, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)           # [B, Hkv, most * G, hd]
    scores = q @ keys[0].transpose(2, 3) * hd ** -0.5
    i = torch.arange(most, device="cuda")
    last = (i // case["dbs"] + 1) * case["dbs"] if case["mask"] == "block_causal" else torch.full_like(i, most)
    fresh = (i[None, :] < last[:, None])[None] & (i[None, None, :] < m.seq_lens_ts[:, None, None])   # [B, row, key]
    mask = torch.cat((seen[:, None, :].expand(b, most, longest), fresh), 2).repeat_interleave(g, 1)[:, None]
    scores = torch.where(mask, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    o = (p @ keys[1]) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (most, g)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return o[s["rows"], s["place"]].to(torch.bfloat16)


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from diffulex_amd import dllm_flash_attn_decode, load_kvcache, store_kvcache_unified_layout
    if op in ("rope", "rope_write"):
        if own:
            if op == "rope":
                return s["rope"](s["positions"], s["q"], s["k"])
            q, k = s["rope"].forward_and_store(s["positions"], s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"],
                                               k_scale=s["k_scale"], v_scale=s["v_scale"])
        else:
            cs = s["table"][s["positions"]]
            cos, sin = cs[:, :case["rot"] // 2], cs[:, case["rot"] // 2:]
            q, k = _rotate(s["q"], cos, sin, case), _rotate(s["k"], cos, sin, case)
            if op == "rope":
                return q, k
            _plain_write(s, k.unflatten(-1, (-1, case["hd"])), s["v"].unflatten(-1, (-1, case["hd"])), "mx8")
        return q, k, s["k_cache"], s["v_cache"], s["k_scale"].view(torch.float8_e8m0fnu), s["v_scale"].view(torch.float8_e8m0fnu)
    if op in ("write", "write_read"):
        if own:
            store_kvcache_unified_layout(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], None, k_scale=s["k_scale"], v_scale=s["v_scale"])
        else:
            _plain_write(s, s["k"], s["v"], case.get("fmt", "mx8"))
        if op == "write":
            return s["k_cache"], s["v_cache"], s["k_scale"].view(torch.float8_e8m0fnu), s["v_scale"].view(torch.float8_e8m0fnu)
    if op in ("read", "write_read"):
        if own:
            return load_kvcache(s["k_cache"], s["v_cache"], s["metadata"], s["k"], s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], out=s["out"])
        return _plain_read(s)
    if own:
        return dllm_flash_attn_decode(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], case["hd"] ** -0.5, s["metadata"],
                                      k_scale=s["k_scale"], v_scale=s["v_scale"])
    return _plain_attention(s)


# ---- the definitions, in 64 bits ---------------------------------------------------------------
def _grid_round(y, fmt):
    """y (64 bits) to the nearest value of the code's grid, ties to even: steps of 2^(exponent - mantissa bits), down to the subnormals'."""
    bits, low = (3, -6) if fmt == "mx8" else (1, 0)
    ex = torch.floor(torch.log2(y.abs().clamp(min=1e-300))).clamp(min=low)
    ex = torch.where(torch.exp2(ex) > y.abs().clamp(min=2.0 ** low), ex - 1, ex)
    step = torch.exp2(ex - bits)
    return torch.round(y / step) * step


def _exact_codes(x, fmt):
    """(code values, scale values) in 64 bits of rows x."""
    b = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    big = 448.0 if fmt == "mx8" else 6.0
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / big))
    e = torch.where(top > big * torch.exp2(e), e + 1, torch.where(top <= big * torch.exp2(e - 1), e - 1, e)).clamp(min=-127)
    return _grid_round(b / torch.exp2(e), fmt).reshape(x.shape), torch.exp2(e)[..., 0]


def _exact_values(codes, scales, fmt):
    if fmt == "bf16":
        return codes.double()
    c = codes.view(torch.uint8).long()
    if fmt == "mx4":
        c = torch.stack((c % 16, c // 16), -1).reshape(*c.shape[:-1], -1)
    m, low = (3, 7) if fmt == "mx8" else (1, 1)
    sign, c = 1.0 - 2.0 * (c >> (4 + m if fmt == "mx8" else 3)).double(), c & (127 if fmt == "mx8" else 7)
    ex, frac = c >> m, (c & ((1 << m) - 1)).double() / (1 << m)
    v = sign * torch.where(ex == 0, frac * 2.0 ** (1 - low), (1 + frac) * torch.exp2((ex - low).double()))
    return (v.reshape(*v.shape[:-1], -1, BLOCK) * torch.exp2(scales.long().double() - 127)[..., None]).reshape(v.shape)


def _exact_rope(s, case):
    cos, sin = _angles(case, s["positions"])
    z = torch.complex(cos, sin)[:, None, :]
    done = []
    for n in "qk":
        x = s[n].double().reshape(case["tokens"], -1, case["hd"])
        half = case["rot"] // 2
        pair = torch.arange(half, device="cuda")
        at = (pair, pair + half) if case["neox"] else (2 * pair, 2 * pair + 1)
        y = torch.complex(x[..., at[0]], x[..., at[1]]) * z
        x = x.clone()
        x[..., at[0]], x[..., at[1]] = y.real, y.imag
        done.append(x)
    return done


def exact(case, seed):
    s = prepare(case, seed)
    op, hd = case["op"], case["hd"]
    if op == "rope":
        return tuple(x.reshape(case["tokens"], -1) for x in _exact_rope(s, case))
    if op in ("rope_write", "write"):
        if op == "rope_write":
            q, k = _exact_rope(s, case)
            # what is written is the rotated key as it is returned, rounded to its type: from 64 bits it may round the other
            # way, so the cache's keys have no value here, and its values do
            v = s["v"].reshape(case["tokens"], -1, hd)
        else:
            k, v = s["k"], s["v"]
        got = []
        for x in (k, v):
            codes, scales = _exact_codes(x, "mx8")
            c = torch.zeros(case["slots"], case["hkv"], hd, dtype=torch.float64, device="cuda")
            e = torch.full((case["slots"], case["hkv"], hd // BLOCK), 2.0 ** -127, dtype=torch.float64, device="cuda")
            c[s["slots"].long()], e[s["slots"].long()] = codes, scales
            got.append((c.reshape(s["k_cache"].shape), e.reshape(s["k_scale"].shape)))
        if op == "write":
            return got[0][0], got[1][0], got[0][1], got[1][1]
        return q.reshape(case["tokens"], -1), k.reshape(case["tokens"], -1), None, got[1][0], None, got[1][1]
    ctx, new = _lengths(case)
    m, page = s["metadata"], case["page"]
    out, at = [[], []], 0                # (the rows that write_read writes lie behind the contexts that it reads)
    for i, (c, n) in enumerate(zip(ctx, new)):
        table = m.block_tables[i, :-(-c // page)].long()
        rows = []
        for name in "kv":
            codes = s[name + "_cache"].view(torch.uint8)[table] if case["fmt"] != "bf16" else s[name + "_cache"][table]
            x = _exact_values(codes, None if case["fmt"] == "bf16" else s[name + "_scale"][table], case["fmt"]).flatten(0, 1)[:c]
            rows.append(torch.cat((x, s[name][at:at + n].double())))
        if op in ("read", "write_read"):
            out[0].append(rows[0])
            out[1].append(rows[1])
        else:
            g = case["hq"] // case["hkv"]
            q = s["q"][at:at + n].double().reshape(n, case["hkv"], g, hd)
            dots = torch.einsum("nhgd,khd->hngk", q, rows[0]) / math.sqrt(hd)
            if case["mask"] == "block_causal":
                r = torch.arange(n, device="cuda")
                hidden = r[None, :] // case["dbs"] > r[:, None] // case["dbs"]
                dots[..., c:] = dots[..., c:].masked_fill(hidden[None, :, None, :], -math.inf)
            out[0].append(torch.einsum("hngk,khd->nhgd", torch.softmax(dots, -1), rows[1]).reshape(n, case["hq"], hd))
        at += n
    if op in ("read", "write_read"):
        return tuple(torch.cat(x) for x in out)
    return torch.cat(out[0])
