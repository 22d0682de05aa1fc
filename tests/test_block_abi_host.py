"""The attention block's C entry points without a GPU: what they refuse, what they plan, and the arithmetic of paged addresses."""
import ctypes
import os
import subprocess

import pytest
import torch

import torch_dist_ext_amd as tde
from torch_dist_ext_amd import _capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
SOMEWHERE = 1 << 20   # an address that no refused call may touch


def test_quotients_and_page_numbers(tmp_path):
    program = str(tmp_path / "unit_test_pages")
    build = [HIPCC, "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "include"),
             "-I", os.path.join(ROOT, "torch_dist_ext_amd", "csrc"), os.path.join(ROOT, "tests", "native", "unit_test_pages.cpp"), "-o", program]
    built = subprocess.run(build, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert built.returncode == 0, built.stdout
    ran = subprocess.run([program], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout


def test_structures_have_the_headers_sizes(tmp_path):
    names = {"tde_int8_product": _capi.Int8Product, "tde_heads": _capi.Heads, "tde_cache": _capi.Cache, "tde_paged_batch": _capi.PagedBatch,
             "tde_head_rows": _capi.HeadRows, "tde_attention": _capi.Attention}
    source = tmp_path / "sizes.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tde_abi.h"', "int main(void) {"]
    for name, struct in names.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (name, name))
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (name, field) for field, _ in struct._fields_]
        lines.append('printf("\\n");')
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], stdout=subprocess.PIPE, text=True, check=True).stdout
    for line in out.splitlines():
        name, size, *offsets = line.split()
        struct = names[name]
        assert ctypes.sizeof(struct) == int(size), name
        assert [getattr(struct, f).offset for f, _ in struct._fields_] == [int(x) for x in offsets], name


def product(**kw):
    base = dict(tokens=4, k=64, n=8, out_dtype=_capi.BF16, codes=SOMEWHERE, weight=SOMEWHERE, scales=SOMEWHERE, weight_scales=SOMEWHERE, out=SOMEWHERE)
    base.update(kw)
    return _capi.Int8Product(**base)


@pytest.mark.parametrize("kw,status", [
    (dict(out_dtype=_capi.F64), _capi.EDTYPE), (dict(out_dtype=9), _capi.EDTYPE), (dict(reserved=1), _capi.EINVAL),
    (dict(tokens=-1), _capi.ESHAPE), (dict(n=-1), _capi.ESHAPE), (dict(k=0), _capi.ESHAPE), (dict(tokens=1 << 31), _capi.ESHAPE),
    (dict(k=131072), _capi.EHIDDEN), (dict(codes=None), _capi.EINVAL), (dict(weight=None), _capi.EINVAL), (dict(scales=None), _capi.EINVAL),
    (dict(weight_scales=None), _capi.EINVAL), (dict(out=None), _capi.EINVAL), (dict(tokens=(1 << 31) - 1, n=(1 << 31) - 1), _capi.ETOOBIG),
    (dict(tokens=0, codes=None, out=None), _capi.OK), (dict(n=0, weight=None), _capi.OK),
])
def test_int8_linear_refuses(kw, status):
    assert _capi.load().tde_int8_linear(ctypes.byref(product(**kw)), None) == status
    assert _capi.load().tde_int8_linear(None, None) == _capi.EINVAL


def batch(**kw):
    base = dict(page_table=SOMEWHERE, q_starts=SOMEWHERE, kv_lens=SOMEWHERE, table_stride=8, seqs=2, table_pages=8, cache_pages=16, page_size=16)
    base.update(kw)
    return _capi.PagedBatch(**base)


HEADS, CACHE = _capi.Heads(SOMEWHERE, 512, 128), _capi.Cache(SOMEWHERE, 4096, 256, 128)


def head_rows(**kw):
    base = dict(dtype=_capi.BF16, dim=128, rot_dim=128, q_heads=4, kv_heads=2, tokens=4, eps=1e-6, positions_bytes=8, positions=SOMEWHERE,
                cos_sin=SOMEWHERE, cos_sin_rows=64, cos_sin_stride=128, q_gamma=SOMEWHERE, k_gamma=SOMEWHERE, q=HEADS, k=HEADS, v=HEADS, q_out=HEADS,
                k_out=HEADS, k_cache=CACHE, v_cache=CACHE, batch=batch())
    base.update(kw)
    return _capi.HeadRows(**base)


NOTHING = _capi.Heads(None, 512, 128)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=_capi.F64), _capi.EDTYPE), (dict(dim=0), _capi.ESHAPE), (dict(dim=1025, rot_dim=0), _capi.EHIDDEN), (dict(rot_dim=130), _capi.ESHAPE),
    (dict(rot_dim=63), _capi.ESHAPE), (dict(rot_dim=-2), _capi.ESHAPE), (dict(tokens=-1), _capi.ESHAPE), (dict(tokens=1 << 31), _capi.ESHAPE),
    (dict(q_heads=-1), _capi.ESHAPE), (dict(kv_heads=-1), _capi.ESHAPE), (dict(q_heads=70000), _capi.ESHAPE), (dict(interleaved=2), _capi.EINVAL),
    (dict(positions_bytes=2), _capi.EINVAL), (dict(eps=-1.0), _capi.EINVAL), (dict(eps=float("nan")), _capi.EINVAL), (dict(eps=float("inf")), _capi.EINVAL),
    (dict(cos_sin=None), _capi.EINVAL), (dict(q=NOTHING), _capi.EINVAL), (dict(k=NOTHING), _capi.EINVAL), (dict(q_out=NOTHING), _capi.EINVAL),
    (dict(q=_capi.Heads(SOMEWHERE, -1, 1)), _capi.ESHAPE), (dict(reserved=1), _capi.EINVAL), (dict(cos_sin_rows=-1), _capi.ESHAPE),
    (dict(tokens=0, q=NOTHING, k=NOTHING), _capi.OK), (dict(q_heads=0, kv_heads=0, k=NOTHING), _capi.OK),
    (dict(tokens=(1 << 31) - 1, q_heads=64), _capi.ETOOBIG),
])
def test_head_rows_refuse(kw, status):
    lib = _capi.load()
    assert lib.tde_qk_norm_rope(ctypes.byref(head_rows(**kw)), None) == status
    assert lib.tde_append_kv(ctypes.byref(head_rows(**kw)), None) == status
    assert lib.tde_qk_norm_rope(None, None) == lib.tde_append_kv(None, None) == _capi.EINVAL


BAD_BATCHES = [
    (dict(seqs=-1), _capi.ESHAPE), (dict(table_pages=-1), _capi.ESHAPE), (dict(cache_pages=-1), _capi.ESHAPE), (dict(page_size=0), _capi.ESHAPE),
    (dict(table_stride=-1), _capi.ESHAPE), (dict(q_starts=None), _capi.EINVAL), (dict(kv_lens=None), _capi.EINVAL), (dict(page_table=None), _capi.EINVAL),
    (dict(seqs=(1 << 24) + 1), _capi.ESHAPE),
]


def test_append_refuses_its_own():
    lib = _capi.load()
    assert lib.tde_qk_norm_rope(ctypes.byref(head_rows(positions=None)), None) == _capi.EINVAL
    assert lib.tde_qk_norm_rope(ctypes.byref(head_rows(k_out=NOTHING)), None) == _capi.EINVAL
    no_cache, backwards = _capi.Cache(None, 4096, 256, 128), _capi.Cache(SOMEWHERE, 4096, -256, 128)
    for kw, status in ((dict(v=NOTHING), _capi.EINVAL), (dict(k_cache=no_cache), _capi.EINVAL), (dict(v_cache=no_cache), _capi.EINVAL),
                       (dict(v_cache=backwards), _capi.ESHAPE)):
        assert lib.tde_append_kv(ctypes.byref(head_rows(**kw)), None) == status, kw
    for kw, status in BAD_BATCHES:
        assert lib.tde_append_kv(ctypes.byref(head_rows(batch=batch(**kw))), None) == status, kw


def attention(**kw):
    base = dict(dtype=_capi.BF16, dim=128, q_heads=8, kv_heads=2, tokens=4, scale=0.1, q=HEADS, out=HEADS, k_cache=CACHE, v_cache=CACHE, batch=batch(),
                workspace=SOMEWHERE, workspace_bytes=1 << 40)
    base.update(kw)
    return _capi.Attention(**base)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=_capi.F32), _capi.EDTYPE), (dict(dim=12), _capi.ESHAPE), (dict(dim=0), _capi.ESHAPE), (dict(dim=264), _capi.EHIDDEN),
    (dict(q_heads=7), _capi.ESHAPE), (dict(q_heads=0), _capi.ESHAPE), (dict(kv_heads=0), _capi.ESHAPE), (dict(tokens=-1), _capi.ESHAPE),
    (dict(tokens=1 << 31), _capi.ESHAPE), (dict(tokens=(1 << 31) - 1), _capi.ETOOBIG), (dict(scale=0.0), _capi.EINVAL), (dict(scale=-1.0), _capi.EINVAL),
    (dict(scale=float("nan")), _capi.EINVAL), (dict(scale=float("inf")), _capi.EINVAL), (dict(zero_tail=2), _capi.EINVAL), (dict(reserved=5), _capi.EINVAL),
    (dict(k_cache=_capi.Cache(SOMEWHERE, 1 << 31, 256, 128)), _capi.ESHAPE), (dict(v_cache=_capi.Cache(SOMEWHERE, 4096, 1 << 31, 128)), _capi.ESHAPE),
] + [(dict(batch=batch(**kw)), status) for kw, status in BAD_BATCHES])
def test_attention_refuses(kw, status):
    lib, n = _capi.load(), ctypes.c_int64()
    t = attention(**kw)
    assert lib.tde_paged_attention_workspace(ctypes.byref(t), ctypes.byref(n)) == status
    assert lib.tde_paged_attention(ctypes.byref(t), None) == status


def test_attention_refuses_buffers():
    lib, n = _capi.load(), ctypes.c_int64()
    for kw, status in ((dict(q=NOTHING), _capi.EINVAL), (dict(out=NOTHING), _capi.EINVAL), (dict(k_cache=_capi.Cache(None, 4096, 256, 128)), _capi.EINVAL),
                       (dict(v_cache=_capi.Cache(SOMEWHERE + 8, 4096, 256, 128)), _capi.EALIGN), (dict(k_cache=_capi.Cache(SOMEWHERE, 4096, 252, 128)), _capi.EALIGN),
                       (dict(k_cache=_capi.Cache(SOMEWHERE, 4100, 256, 128)), _capi.EALIGN), (dict(v_cache=_capi.Cache(SOMEWHERE, 4096, 256, 100)), _capi.EALIGN)):
        assert lib.tde_paged_attention(ctypes.byref(attention(**kw)), None) == status, kw
    # a call whose keys are split needs its workspace
    split = dict(tokens=1, batch=batch(seqs=1, table_pages=4096))
    assert lib.tde_paged_attention_workspace(ctypes.byref(attention(**split)), ctypes.byref(n)) == _capi.OK
    assert n.value > 0
    for kw, status in ((dict(workspace=None), _capi.EINVAL), (dict(workspace_bytes=n.value - 1), _capi.EINVAL), (dict(workspace=SOMEWHERE + 4), _capi.EALIGN)):
        assert lib.tde_paged_attention(ctypes.byref(attention(**split, **kw)), None) == status, kw
    assert lib.tde_paged_attention_workspace(ctypes.byref(attention(tokens=0)), ctypes.byref(n)) == _capi.OK and n.value == 0
    assert lib.tde_paged_attention(ctypes.byref(attention(tokens=0, q=NOTHING)), None) == _capi.OK
    assert lib.tde_paged_attention_workspace(ctypes.byref(attention()), None) == _capi.EINVAL
    assert lib.tde_paged_attention(None, None) == _capi.EINVAL


def test_tracing_sees_shapes_and_types():
    meta = torch.device("meta")
    codes, weight = torch.empty((2, 3, 64), dtype=torch.int8, device=meta), torch.empty((40, 64), dtype=torch.int8, device=meta)
    s = torch.empty(6, device=meta)
    y = tde.int8_linear(codes, s, weight, torch.empty(40, device=meta), None, torch.float16)
    assert y.shape == (2, 3, 40) and y.dtype == torch.float16 and tde.int8_linear(codes, s, weight, s).dtype == torch.bfloat16
    qkv = torch.empty((5, 8, 32), dtype=torch.bfloat16, device=meta)
    q, k = tde.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], s, s, 1e-6, s, s)
    assert q.shape == (5, 4, 32) and k.shape == (5, 2, 32) and q.is_contiguous()
    cache = torch.empty((4, 16, 2, 32), dtype=torch.bfloat16, device=meta)
    assert tde.append_kv(k, k, cache, cache, s, s, s) is None
    assert tde.append_kv(k, k, cache, cache, s, s, s, q=q).shape == q.shape
    assert tde.paged_attention(q, cache, cache, s, s, s).shape == q.shape
    assert tde.paged_attention_out(q, cache, cache, s, s, s, q) is None


def test_there_is_no_cpu_path():
    with pytest.raises(NotImplementedError):
        tde.int8_linear(torch.zeros((1, 8), dtype=torch.int8), torch.ones(1), torch.zeros((1, 8), dtype=torch.int8), torch.ones(1))
