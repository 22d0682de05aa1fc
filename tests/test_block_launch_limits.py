"""Calls of more threads than one launch holds (2^32) are refused before anything runs, as what they are.  No GPU is needed, and none reached."""
import ctypes

import pytest

from torch_dist_ext_amd import _capi
from test_block_abi_host import attention, batch, head_rows, product


@pytest.mark.parametrize("kw", [
    dict(tokens=1, n=1 << 28, k=1), dict(tokens=2, n=(1 << 31) - 1, k=1), dict(tokens=4, n=1 << 30, k=131071),       # 16 channels a workgroup of 256 threads
    dict(tokens=5, n=1 << 30, k=4), dict(tokens=40, n=1 << 29, k=4), dict(tokens=9, n=(1 << 31) - 1, k=3),            # 32 channels and 256 or 512 threads; rows that begin anywhere 16 and 512
    dict(tokens=1 << 25, n=1 << 20, k=128), dict(tokens=1 << 25, n=1 << 20, k=127),                                   # tiles
])
def test_int8_linear(kw):
    assert _capi.load().tde_int8_linear(ctypes.byref(product(**kw)), None) == _capi.ETOOBIG


@pytest.mark.parametrize("kw", [
    dict(tokens=1 << 26, q_heads=1, kv_heads=0, dim=7, rot_dim=0), dict(tokens=1 << 26, q_heads=1, kv_heads=0, dim=8, rot_dim=8),
    dict(tokens=(1 << 26) - 3, q_heads=1, kv_heads=0, dim=7, rot_dim=0), dict(tokens=1 << 23, q_heads=64, kv_heads=8, dim=1024, rot_dim=0),
])
def test_head_rows(kw):
    lib = _capi.load()
    assert lib.tde_qk_norm_rope(ctypes.byref(head_rows(**kw)), None) == _capi.ETOOBIG
    assert lib.tde_append_kv(ctypes.byref(head_rows(**kw)), None) == _capi.ETOOBIG


@pytest.mark.parametrize("kw", [
    dict(tokens=1 << 24, batch=batch(seqs=1 << 24)),                                              # a decode step of as many sequences
    dict(tokens=1, q_heads=64, kv_heads=64, batch=batch(seqs=1 << 20, table_pages=4096)),         # mostly empty: the second launch is the larger one
    dict(tokens=1 << 30, q_heads=1, kv_heads=1, dim=256, batch=batch(seqs=1 << 24)),
])
def test_attention(kw):
    lib, n = _capi.load(), ctypes.c_int64()
    assert lib.tde_paged_attention_workspace(ctypes.byref(attention(**kw)), ctypes.byref(n)) == _capi.ETOOBIG
    assert lib.tde_paged_attention(ctypes.byref(attention(**kw)), None) == _capi.ETOOBIG


def test_largest_plans_are_still_made():
    """Sizes just inside: the workspace entry, which launches nothing, takes them."""
    lib, n = _capi.load(), ctypes.c_int64()
    for kw in (dict(tokens=(1 << 23) - 600, batch=batch(seqs=(1 << 23) - 600), kv_heads=1, q_heads=8), dict(tokens=1, q_heads=64, kv_heads=64, batch=batch(seqs=1 << 15, table_pages=4096)),
               dict(tokens=1 << 23, q_heads=64, kv_heads=8, batch=batch(seqs=1))):
        assert lib.tde_paged_attention_workspace(ctypes.byref(attention(**kw)), ctypes.byref(n)) == _capi.OK, kw
