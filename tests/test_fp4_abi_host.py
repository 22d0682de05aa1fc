"""The C entry points over a cache in 4 bits and of page updates without a GPU: what they refuse, and their structures."""
import ctypes
import subprocess

import pytest
import torch

import torch_dist_ext_amd as tde
from torch_dist_ext_amd import _capi
from test_block_abi_host import BAD_BATCHES, NOTHING, ROOT, SOMEWHERE, attention, batch, head_rows

CODES, SCALES = _capi.Cache(SOMEWHERE, 4096, 64, 1024), _capi.Cache(SOMEWHERE, 256, 4, 64)
NO_CACHE = _capi.Cache(None, 4096, 64, 1024)


def test_structures_have_the_headers_sizes(tmp_path):
    names = {"tde_append_fp4": _capi.AppendFp4, "tde_attention_fp4": _capi.AttentionFp4, "tde_unpack_fp4_rows": _capi.UnpackFp4Rows, "tde_page_update": _capi.PageUpdate}
    source = tmp_path / "sizes.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tde_abi.h"', "int main(void) {"]
    for name, struct in names.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (name, name))
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (name, field) for field, _ in struct._fields_]
        lines.append('printf("\\n");')
    lines.append('printf("%d %d\\n", TDE_FP4_BLOCK, TDE_FP4_MAX_DIM);')
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", ROOT + "/include", str(source), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], stdout=subprocess.PIPE, text=True, check=True).stdout.splitlines()
    for line in out[:-1]:
        name, size, *offsets = line.split()
        assert ctypes.sizeof(names[name]) == int(size), name
        assert [getattr(names[name], f).offset for f, _ in names[name]._fields_] == [int(x) for x in offsets], name
    assert out[-1].split() == [str(_capi.FP4_BLOCK), str(_capi.FP4_MAX_DIM)]


def append(k_scales=SCALES, v_scales=SCALES, reserved=0, **kw):
    kw = dict(dict(k_cache=CODES, v_cache=CODES), **kw)
    return _capi.AppendFp4(rows=head_rows(**kw), k_scales=k_scales, v_scales=v_scales, reserved=reserved)


def test_append_refuses():
    lib = _capi.load()
    assert lib.tde_append_kv_fp4(None, None) == _capi.EINVAL
    for kw, status in ((dict(reserved=1), _capi.EINVAL), (dict(dtype=_capi.F64), _capi.EDTYPE), (dict(dim=16, rot_dim=16), _capi.ESHAPE), (dict(dim=80, rot_dim=0), _capi.ESHAPE),
                       (dict(dim=288, rot_dim=0), _capi.EHIDDEN), (dict(k=NOTHING), _capi.EINVAL), (dict(q=NOTHING), _capi.EINVAL), (dict(k_cache=NO_CACHE), _capi.EINVAL),
                       (dict(k_scales=NO_CACHE), _capi.EINVAL), (dict(v_scales=NO_CACHE), _capi.EINVAL), (dict(v_scales=_capi.Cache(SOMEWHERE, -1, 4, 64)), _capi.ESHAPE),
                       (dict(rot_dim=130), _capi.ESHAPE), (dict(eps=float("nan")), _capi.EINVAL), (dict(tokens=(1 << 31) - 1, q_heads=64), _capi.ETOOBIG),
                       (dict(tokens=0, k=NOTHING), _capi.OK), (dict(q_heads=0, kv_heads=0), _capi.OK)):
        assert lib.tde_append_kv_fp4(ctypes.byref(append(**kw)), None) == status, kw
    for kw, status in BAD_BATCHES:
        assert lib.tde_append_kv_fp4(ctypes.byref(append(batch=batch(**kw))), None) == status, kw


def attention_fp4(k_scales=SCALES, v_scales=SCALES, reserved=0, **kw):
    kw = dict(dict(k_cache=CODES, v_cache=CODES), **kw)
    return _capi.AttentionFp4(attention=attention(**kw), k_scales=k_scales, v_scales=v_scales, reserved=reserved)


def test_attention_refuses():
    lib, n = _capi.load(), ctypes.c_int64()
    assert lib.tde_paged_attention_fp4(None, None) == lib.tde_paged_attention_fp4_workspace(None, ctypes.byref(n)) == _capi.EINVAL
    assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(attention_fp4()), None) == _capi.EINVAL
    far = _capi.Cache(SOMEWHERE, 1 << 31, 4, 64)
    for kw, status in ((dict(reserved=1), _capi.EINVAL), (dict(dtype=_capi.F32), _capi.EDTYPE), (dict(dim=16), _capi.ESHAPE), (dict(dim=72), _capi.ESHAPE),
                       (dict(dim=288), _capi.EHIDDEN), (dict(q_heads=3, kv_heads=2), _capi.ESHAPE), (dict(scale=0.0), _capi.EINVAL),
                       (dict(k_scales=_capi.Cache(SOMEWHERE, -256, 4, 64)), _capi.ESHAPE), (dict(v_scales=far), _capi.ESHAPE), (dict(k_cache=far), _capi.ESHAPE)):
        for call in (lambda t: lib.tde_paged_attention_fp4(t, None), lambda t: lib.tde_paged_attention_fp4_workspace(t, ctypes.byref(n))):
            assert call(ctypes.byref(attention_fp4(**kw))) == status, kw
    off = _capi.Cache(SOMEWHERE + 8, 4096, 64, 1024)
    for kw, status in ((dict(q=NOTHING), _capi.EINVAL), (dict(k_cache=NO_CACHE), _capi.EINVAL), (dict(v_scales=NO_CACHE), _capi.EINVAL), (dict(k_cache=off), _capi.EALIGN),
                       (dict(v_cache=_capi.Cache(SOMEWHERE, 4096, 72, 1024)), _capi.EALIGN), (dict(tokens=0, q=NOTHING), _capi.OK)):
        kw = dict(kw, workspace=SOMEWHERE, workspace_bytes=1 << 40)
        assert lib.tde_paged_attention_fp4(ctypes.byref(attention_fp4(**kw)), None) == status, kw
    # a call with few rows over a long table splits its keys and needs a workspace
    split = dict(tokens=1, batch=batch(seqs=1, table_pages=4096))
    assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(attention_fp4(**split)), ctypes.byref(n)) == _capi.OK and n.value > 0
    for kw, status in ((dict(workspace=None, workspace_bytes=1 << 40), _capi.EINVAL), (dict(workspace=SOMEWHERE, workspace_bytes=n.value - 1), _capi.EINVAL),
                       (dict(workspace=SOMEWHERE + 4, workspace_bytes=1 << 40), _capi.EALIGN)):
        assert lib.tde_paged_attention_fp4(ctypes.byref(attention_fp4(**split, **kw)), None) == status, kw


def test_launches_that_do_not_fit():
    """Calls of more threads than one launch holds (2^32), or of more tiles than are counted, are refused before anything runs, or planned another way."""
    lib, n = _capi.load(), ctypes.c_int64()
    for kw in (dict(tokens=1 << 26, q_heads=1, kv_heads=0, dim=32, rot_dim=0), dict(tokens=1 << 23, q_heads=64, kv_heads=8, dim=256, rot_dim=0, dtype=_capi.F32),
               dict(tokens=1 << 30, q_heads=8, kv_heads=8, dim=256, rot_dim=0)):
        assert lib.tde_append_kv_fp4(ctypes.byref(append(**kw)), None) == _capi.ETOOBIG, kw
    for kw in (dict(tokens=1 << 24, batch=batch(seqs=1 << 24)), dict(tokens=1 << 30, q_heads=1, kv_heads=1, dim=256, batch=batch(seqs=1 << 24)),
               dict(tokens=1 << 24, q_heads=1, kv_heads=1, batch=batch(seqs=1 << 24))):
        kw = dict(kw, workspace=SOMEWHERE, workspace_bytes=1 << 62)
        assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(attention_fp4(**kw)), ctypes.byref(n)) == _capi.ETOOBIG, kw
        assert lib.tde_paged_attention_fp4(ctypes.byref(attention_fp4(**kw)), None) == _capi.ETOOBIG, kw
    for kw in (dict(tokens=1 << 20, batch=batch(seqs=1 << 20)), dict(tokens=1, q_heads=64, kv_heads=64, batch=batch(seqs=1 << 15, table_pages=4096)),
               dict(tokens=1, q_heads=1, kv_heads=1, batch=batch(seqs=1, table_pages=(1 << 31) // 128)), dict(tokens=1 << 23, q_heads=64, kv_heads=8, batch=batch(seqs=1))):
        assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(attention_fp4(**kw)), ctypes.byref(n)) == _capi.OK, kw


def test_slots_far_apart_are_planned_another_way():
    """Decode rows whose keys' offsets do not hold 32 bits take the tiles of 64 rows, as those over pages that 8 does not divide."""
    lib, n = _capi.load(), ctypes.c_int64()

    def workspace(page_size=16, **kw):
        t = attention_fp4(tokens=1, batch=batch(seqs=1, page_size=page_size, table_pages=4096), **kw)
        assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(t), ctypes.byref(n)) == _capi.OK
        return n.value

    near, other = workspace(), workspace(page_size=17)
    assert near != other
    for name, base in (("k_cache", 64), ("v_cache", 64), ("k_scales", 4), ("v_scales", 4)):
        assert workspace(**{name: _capi.Cache(SOMEWHERE, 4096, (1 << 27) - 64, base)}) == near
        assert workspace(**{name: _capi.Cache(SOMEWHERE, 4096, 1 << 27, base)}) == workspace(page_size=12, **{name: _capi.Cache(SOMEWHERE, 4096, 64, base)}), name


def test_scales_of_scores():
    """A scale whose product with log2(e) is no fp32 number would make every weight NaN."""
    lib, n = _capi.load(), ctypes.c_int64()
    for scale, status in ((2e38, _capi.OK), (2.4e38, _capi.EINVAL), (float("inf"), _capi.EINVAL), (1e-45, _capi.OK), (1e-46, _capi.EINVAL), (float("nan"), _capi.EINVAL)):
        assert lib.tde_paged_attention_fp4_workspace(ctypes.byref(attention_fp4(scale=scale)), ctypes.byref(n)) == status, scale


def unpack(sizes=(2, 3, 4), code_strides=(768, 256, 64), scale_strides=(48, 16, 4), **kw):
    base = dict(dim=128, out_dtype=_capi.BF16, codes=SOMEWHERE, scales=SOMEWHERE, out=SOMEWHERE)
    base.update(kw)
    three = ctypes.c_int64 * 3
    return _capi.UnpackFp4Rows(sizes=three(*sizes), code_strides=three(*code_strides), scale_strides=three(*scale_strides), **base)


@pytest.mark.parametrize("kw,status", [
    (dict(reserved=1), _capi.EINVAL), (dict(out_dtype=_capi.F64), _capi.EDTYPE), (dict(dim=48), _capi.ESHAPE), (dict(dim=0), _capi.ESHAPE), (dict(dim=288), _capi.EHIDDEN),
    (dict(sizes=(-1, 3, 4)), _capi.ESHAPE), (dict(code_strides=(1, -1, 1)), _capi.ESHAPE), (dict(scale_strides=(1, 1, 1 << 41)), _capi.ESHAPE),
    (dict(sizes=(1 << 20, 1 << 20, 1)), _capi.ETOOBIG), (dict(sizes=(1 << 28, 1, 1)), _capi.ETOOBIG), (dict(sizes=(1 << 31, 1, 1)), _capi.ETOOBIG), (dict(codes=None), _capi.EINVAL),
    (dict(scales=None), _capi.EINVAL), (dict(out=None), _capi.EINVAL), (dict(sizes=(0, 1 << 40, 1 << 40), codes=None, out=None), _capi.OK),
])
def test_unpack_refuses(kw, status):
    assert _capi.load().tde_unpack_fp4(ctypes.byref(unpack(**kw)), None) == status
    assert _capi.load().tde_unpack_fp4(None, None) == _capi.EINVAL


def update(**kw):
    base = dict(page_table=SOMEWHERE, kv_lens=SOMEWHERE, new_tokens=SOMEWHERE, keep_lens=SOMEWHERE, free_pages=SOMEWHERE, free_count=SOMEWHERE, q_starts=SOMEWHERE,
                positions=SOMEWHERE, slots=SOMEWHERE, table_stride=8, tokens=4, seqs=2, table_pages=8, free_capacity=16, page_size=16)
    base.update(kw)
    return _capi.PageUpdate(**base)


@pytest.mark.parametrize("kw,status", [
    (dict(reserved=1), _capi.EINVAL), (dict(seqs=-1), _capi.ESHAPE), (dict(seqs=(1 << 24) + 1), _capi.ESHAPE), (dict(table_pages=-1), _capi.ESHAPE), (dict(page_size=0), _capi.ESHAPE),
    (dict(free_capacity=-1), _capi.ESHAPE), (dict(tokens=-1), _capi.ESHAPE), (dict(tokens=1 << 31), _capi.ESHAPE), (dict(table_stride=-1), _capi.ESHAPE),
    (dict(seqs=1 << 20, table_pages=1 << 11), _capi.ETOOBIG), (dict(page_table=None), _capi.EINVAL), (dict(kv_lens=None), _capi.EINVAL), (dict(new_tokens=None), _capi.EINVAL),
    (dict(free_pages=None), _capi.EINVAL), (dict(free_count=None), _capi.EINVAL), (dict(q_starts=None), _capi.EINVAL), (dict(positions=None), _capi.EINVAL),
    (dict(slots=None), _capi.EINVAL),
])
def test_update_refuses(kw, status):
    assert _capi.load().tde_update_pages(ctypes.byref(update(**kw)), None) == status
    assert _capi.load().tde_update_pages(None, None) == _capi.EINVAL


def test_shapes_without_data():
    """What compiled graphs see."""
    meta = dict(device="meta")
    codes, scales = torch.empty((3, 16, 2, 32), dtype=torch.uint8, **meta), torch.empty((3, 16, 2, 2), dtype=torch.uint8, **meta)
    table, starts, lens = (torch.empty(s, dtype=torch.int32, **meta) for s in ((4, 5), (5,), (4,)))
    q, k = (torch.empty((7, n, 64), dtype=torch.bfloat16, **meta) for n in (4, 2))
    assert tde.unpack_fp4(codes, scales, torch.float16).shape == (3, 16, 2, 64) and tde.unpack_fp4(codes, scales).dtype == torch.bfloat16
    assert tde.append_kv_fp4(k, k, codes, scales, codes, scales, table, starts, lens, q=q).shape == q.shape
    assert tde.append_kv_fp4(k, k, codes, scales, codes, scales, table, starts, lens) is None
    assert tde.paged_attention_fp4(q, codes, scales, codes, scales, table, starts, lens).shape == q.shape
    assert tde.paged_attention_fp4_out(q, codes, scales, codes, scales, table, starts, lens, q) is None
    got = tde.update_pages(table, lens, lens, starts, starts[:1], 16, 9, keep_lens=lens)
    assert [(t.shape[0], t.dtype) for t in got] == [(5, torch.int32), (9, torch.int32), (9, torch.int64)]


def test_tensors_have_to_be_on_a_gpu():
    codes, scales = torch.zeros((3, 16, 2, 32), dtype=torch.uint8), torch.zeros((3, 16, 2, 2), dtype=torch.uint8)
    with pytest.raises((RuntimeError, NotImplementedError)):
        tde.unpack_fp4(codes, scales)
    with pytest.raises(RuntimeError, match="q_gamma without q"):
        tde.append_kv_fp4(None, None, codes, scales, codes, scales, None, None, None, q_gamma=codes)
