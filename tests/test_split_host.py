"""CPU tests of dfx_split_attn's host side: struct mirror, refusals, workspace; the 64-bit oracle against the fp32 one."""
import ctypes as C
import os
import subprocess
import types

import pytest
import torch

import diffulex_amd as dfx
from diffulex_amd import _lib
from oracle import attention as oat
from oracle import split

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layout_matches_header(tmp_path):
    names = [f[0] for f in _lib.SplitAttnParams._fields_]
    prints = "".join(f'printf("%zu\\n", offsetof(dfx_split_attn_params, {n}));' for n in names)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "diffulex_amd.h"\n'
                   'int main(void){printf("%zu\\n", sizeof(dfx_split_attn_params));' + prints + 'return 0;}\n')
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert got[0] == C.sizeof(_lib.SplitAttnParams) and got[1:] == [getattr(_lib.SplitAttnParams, n).offset for n in names]


def _params(**kw):
    p = _lib.SplitAttnParams()
    p.q = p.k_new = p.v_new = p.out = p.k_cache = p.v_cache = p.k_scales = p.v_scales = 4096
    p.block_tables = p.context_lens = p.cu_seqlens_q = p.cu_seqlens_new = 4096
    p.num_seqs, p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size, p.max_pages_per_seq, p.n_pages = 3, 8, 2, 128, 16, 4, 12
    p.num_q_tokens = p.num_new_tokens = 5
    for n in ("q_stride_token", "o_stride_token", "kn_stride_token", "vn_stride_token"):
        setattr(p, n, 1024)
    for n in ("q_stride_head", "o_stride_head", "kn_stride_head", "vn_stride_head"):
        setattr(p, n, 128)
    p.block_table_stride, p.kv_dtype, p.scale, p.diffusion_block_size, p.max_workgroups = 4, 2, 0.1, 32, 8
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_refuses_without_launching():
    lib = _lib.load()
    call = lambda **kw: lib.dfx_split_attn(C.byref(_params(**kw)), None)  # noqa: E731
    assert lib.dfx_split_attn(None, None) == -1
    assert call(num_seqs=0) == 0 and call(num_q_tokens=0) == 0
    assert call() == _lib.load().dfx_split_attn(C.byref(_params()), None) == -3                     # no workspace
    assert call(workspace=4096, workspace_bytes=1000) == -3
    for bad in (dict(head_dim=96), dict(num_seqs=70000), dict(num_q_tokens=1 << 31), dict(max_workgroups=1 << 17), dict(num_groups=9)):
        assert call(**bad) == -2, bad
    for bad in (dict(kv_dtype=1), dict(kv_dtype=4), dict(mask_mode=3), dict(mask_mode=1, diffusion_block_size=0), dict(scale=0.0), dict(num_q_heads=7),
                dict(q=4098), dict(k_cache=4100), dict(kn_stride_token=1020), dict(k_scales=None), dict(kv_dtype=0), dict(v_cache=None),
                dict(page_size=0), dict(num_groups=1), dict(max_workgroups=-1), dict(cu_seqlens_new=None), dict(k_new=None), dict(num_seqs=-1)):
        assert call(**bad) == -1, bad
    need = lib.dfx_split_attn_workspace_bytes(C.byref(_params()))
    assert need > 0 and lib.dfx_split_attn_workspace_bytes(C.byref(_params(head_dim=80))) == -2
    assert lib.dfx_split_attn_workspace_bytes(C.byref(_params(num_groups=2))) > need
    assert call(workspace=4096 + 16, workspace_bytes=need) == -1                                     # misaligned


@pytest.mark.parametrize("block_causal", [False, True])
def test_oracle_agrees_with_the_fp32_oracle(block_causal):
    g = torch.Generator().manual_seed(0)
    ctx, new, page, hq, hkv, hd = [20, 0, 33], [3, 5, 9], 8, 4, 2, 64
    table = torch.arange(15, dtype=torch.int32).view(3, 5)
    kc, vc = (torch.randn(15, page, hkv, hd, generator=g).to(torch.bfloat16) for _ in range(2))
    q, k, v = (torch.randn(17, h, hd, generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
    cu = torch.tensor([0, 3, 8, 17], dtype=torch.int32)
    table[2, 1] = -1
    got, spread, written = split.attention(q, k, v, kc.double(), vc.double(), table, torch.tensor(ctx), cu, cu, 0.125, block_causal, 4)
    want = oat.paged_attention_fp32(q, k, v, kc, vc, table, torch.tensor(ctx, dtype=torch.int32), cu, cu, 0.125,
                                    mask_mode=int(block_causal), dbs=4)
    # fp32 sums of 64 products and of at most 42 weights: a few thousand steps of 2^-24 at most
    assert (got - want.double()).abs().max() < 1e-4 and written.all() and (spread >= got.abs() - 1e-12).all()


def test_half_a_pair_of_prefix_tensors_is_refused():
    x, one = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for kw in (dict(prefix_cu_seqs=one), dict(prefix_lens=one[:1])):
        with pytest.raises(_lib.DfxError, match="go together"):
            dfx.paged_attention(x, x, x, None, None, 1.0, block_tables=None, context_lens=None, cu_seqlens_q=one, cu_seqlens_new=one,
                                max_seqlen_q=1, **kw)


def test_microscaled_caches_in_the_distinct_layout_are_refused():
    md = types.SimpleNamespace(is_prefill=False, kv_cache_layout="distinct")
    layer = dfx.Attention(1, 64, 1.0, 1)
    layer.k_scale = layer.v_scale = torch.zeros(2, 8, 1, 2, dtype=torch.uint8)
    layer.fetch_attn_metadata = lambda: md
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="unified"):
        layer(x, x, x)
