"""Refusals of the operators over 8-bit pages, before anything is launched (all on the CPU)."""
import ctypes
import itertools
import os
import subprocess
import sys

import pytest
import torch

from deserve_amd import _lib
from deserve_amd.quant_ops import BatchQuantizedWithPagedKVCacheWrapper, PageRecord, move_accepted_quantized_rows, rope_append_quantized

bf16 = torch.bfloat16


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_records():
    r = PageRecord(16, 8, 128)
    assert r.page_bytes == 32896 == _lib.lib().dskv_quant_page_bytes(16, 8, 128)
    for page, hkv, dim in ((1, 1, 8), (12, 5, 80), (8, 8, 128), (64, 1, 256), (3, 17, 64)):
        r = PageRecord(page, hkv, dim)
        assert r.page_bytes == _lib.lib().dskv_quant_page_bytes(page, hkv, dim) and r.page_bytes % 128 == 0
        pages = torch.zeros((5, r.page_bytes), dtype=torch.uint8)
        assert r.codes(pages).shape == (5, 2, hkv, page, dim) and r.scales(pages).shape == (5, 2, hkv)
        r.scales(pages)[3, 1, hkv - 1] = 2.0
        r.codes(pages)[3, 1, hkv - 1, page - 1, dim - 1] = 1.5
        values = r.values(pages, bf16)
        assert values.shape == (5, 2, page, hkv, dim) and values[3, 1, page - 1, hkv - 1, dim - 1] == 3 and values.abs().sum() == 3
    for bad in ((0, 8, 128), (16, 0, 128), (16, 8, 12), (16, 8, 264)):
        refused("pages of", PageRecord, *bad)


def test_append():
    r = PageRecord(16, 8, 64)
    pages = torch.zeros((4, r.page_bytes), dtype=torch.uint8)
    q, k, table = torch.zeros((3, 32, 64), dtype=bf16), torch.zeros((3, 8, 64), dtype=bf16), torch.zeros((3, 64))
    csr = (i32(0, 3), i32(0), i32(0, 1), i32(3))

    def call(q=q, k=k, v=k, pages=pages, csr=csr, page=16, table=table, **kw):
        return rope_append_quantized(q, k, v, csr[0], pages, csr[1], csr[2], csr[3], page, table, **kw)
    refused("on the GPU", call)
    refused("pages must be", call, pages=pages[:, :-1])
    refused("pages must be", call, pages=pages.view(torch.float8_e4m3fn))
    refused("pages must be", call, pages=pages[::2])
    refused("pages must be", call, page=8)
    refused("pages of 0", call, page=0)
    refused("k must be", call, k=k[0])
    refused("v must be", call, v=k[:, :4])
    refused("v must be", call, v=k.half())
    refused("q must be", call, q=q[:2])
    refused("q is missing", call, q=None)
    refused("unsupported", call, q=q.double(), k=k.double(), v=k.double())
    refused("rope_table", call, table=table[:2])
    refused("rope_table", call, table=table.double())
    refused("out must be", call, out=q[:2])
    refused("out is for", call, table=None, out=q)
    refused("qo_indptr", call, csr=(csr[0].long(), *csr[1:]))
    refused("kv_indptr holds 1", call, csr=(csr[0], csr[1], i32(0), csr[3]))
    refused("disagree", call, csr=(csr[0], csr[1], i32(0, 1, 2), csr[3]))
    refused("kv_last_page_len holds 0", call, csr=(*csr[:3], i32()))


def test_attention():
    refused("HND", BatchQuantizedWithPagedKVCacheWrapper, torch.empty(1), "NHD")
    w = BatchQuantizedWithPagedKVCacheWrapper(torch.empty(16, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="before begin_forward"):
        w.forward(torch.zeros(1), torch.zeros(1))
    csr = (i32(0, 2), i32(0, 1), i32(0), i32(5))
    begin = lambda csr=csr, hq=32, hkv=8, dim=128, page=16, **kw: w.begin_forward(*csr, hq, hkv, dim, page, **{"max_qo_len": 2, **kw})
    refused("on the GPU", begin)
    refused("qo_indptr", begin, (torch.zeros(2), *csr[1:]))
    refused("disagree", begin, (csr[0], i32(0, 1, 2), *csr[2:]))
    refused("multiple of num_kv_heads", begin, hq=30)
    refused("pages of", begin, dim=100)
    refused("pages of", begin, page=0)
    refused("not be negative", begin, max_qo_len=-1)
    refused("not be negative", begin, min_qo_len=-1)
    refused("masks hold 64", begin, max_qo_len=65, masks=torch.zeros(2).long())
    refused("masks", begin, masks=torch.zeros(2))


def test_move():
    r = PageRecord(16, 8, 64)
    pages = torch.zeros((2, 4, r.page_bytes), dtype=torch.uint8)
    csr, path, counts = (i32(0, 3), i32(0), i32(0, 1), i32(3)), i32(0, 2, -1), i32(2)
    call = lambda pages=pages, csr=csr, path=path, counts=counts, sizes=(16, 8, 64): move_accepted_quantized_rows(pages, *csr, path, counts, *sizes)
    refused("on the GPU", call)
    refused("pages must be", call, pages[0])
    refused("pages must be", call, pages[:, ::2])
    refused("pages must be", call, sizes=(16, 4, 64))
    refused("path", call, path=path.long())
    refused("counts holds 0", call, counts=i32())


def test_c_entries():
    lib = _lib.lib()
    rows = lambda **kw: ctypes.byref(_lib.QuantRows(**{**dict(qo_indptr=16, kv_page_indices=16, kv_page_indptr=16, kv_last_page_lens=16,
                                                              n_page_indices=4, batch=1, nnz=2, num_pages=4, page_size=16, n_kv_heads=8,
                                                              head_dim=128), **kw}))

    def append(r, q_out=16, pages=16, q=16, k=16, v=16, qs=4096, ks=1024, vs=1024, table=16, hq=32, dtype=_lib.BF16):
        return lib.dskv_rope_append_quant(r, q_out, pages, q, k, v, qs, ks, vs, table, hq, dtype, None), _lib.last_error()
    for want, args in (("batch", (rows(batch=-1),)), ("page shape", (rows(num_pages=0),)), ("head_dim", (rows(head_dim=12),)),
                       ("head_dim", (rows(head_dim=264),)), ("null", (rows(qo_indptr=None),)), ("too large", (rows(page_size=1 << 30),))):
        rc, said = append(*args)
        assert rc == _lib.E_INVAL and want in said, (want, said)
    for want, kw in (("null", dict(k=None)), ("null", dict(q_out=None)), ("dtype", dict(dtype=7)), ("overlap", dict(ks=1000)),
                     ("overlap", dict(qs=4095)), ("aligned", dict(v=24)), ("aligned", dict(vs=1028)), ("n_qo_heads", dict(hq=0))):
        rc, said = append(rows(), **kw)
        assert rc == _lib.E_INVAL and want in said, (want, said)
    assert lib.dskv_rope_append_quant(None, *[16] * 5, 1, 1, 1, 16, 1, 2, None) == _lib.E_INVAL
    assert append(rows(batch=0))[0] == 0 and append(rows(nnz=0))[0] == 0
    move = lambda r, pages=16, stride=1 << 20, layers=2, path=16, counts=16: (
        lib.dskv_move_quant_rows(r, pages, stride, layers, path, counts, None), _lib.last_error())
    for want, kw in (("null", dict(pages=None)), ("null", dict(path=None)), ("aligned", dict(pages=8)), ("overlap", dict(stride=1024)),
                     ("layers", dict(layers=-1)), ("layers", dict(layers=1 << 20))):
        rc, said = move(rows(), **kw)
        assert rc == _lib.E_INVAL and want in said, (want, said)
    assert move(rows(batch=0))[0] == 0 and move(rows(), layers=0)[0] == 0
    base = dict(qo_indptr=16, kv_page_indptr=16, kv_page_indices=16, kv_last_page_lens=16, masks=None, workspace=None, workspace_bytes=0,
                n_page_indices=4, batch=1, nnz=2, max_qo_len=2, n_qo_heads=32, n_kv_heads=8, head_dim=128, page_size=16, num_pages=4,
                dtype=_lib.BF16, sm_scale=0.1)

    def attend(out=16, q=16, stride=4096, pages=16, min_qo_len=0, **kw):
        step = _lib.QuantStep(_lib.TreeStep(**{**base, **kw}), None, 0, min_qo_len)
        return lib.dskv_quant_attn(ctypes.byref(step), out, q, stride, pages, None), _lib.last_error()
    for want, kw in (("negative", dict(batch=-1)), ("negative", dict(min_qo_len=-1)), ("dtype", dict(dtype=5)), ("multiple", dict(n_qo_heads=30)),
                     ("head_dim", dict(head_dim=100)), ("page shape", dict(num_pages=0)), ("sm_scale", dict(sm_scale=0.0)),
                     ("sm_scale", dict(sm_scale=float("nan"))), ("masks hold", dict(masks=16, max_qo_len=65)), ("null", dict(out=None)),
                     ("null", dict(qo_indptr=None)), ("overlap", dict(stride=4000)), ("aligned", dict(q=8)), ("aligned", dict(stride=4100))):
        rc, said = attend(**kw)
        assert rc == _lib.E_INVAL and want in said, (want, rc, said)
    for kw in (dict(batch=0), dict(nnz=0), dict(max_qo_len=0)):
        assert attend(**kw)[0] == 0
    rc, said = attend()
    assert rc == _lib.E_NOMEM and "workspace of 0" in said
    need = lib.dskv_quant_attn_workspace(1, 2, 2, 32, 8, 128, _lib.BF16)
    rc, said = attend(workspace=16, workspace_bytes=need)
    assert rc == _lib.E_NOMEM and "0 counters" in said
    rc, said = attend(workspace=24, workspace_bytes=need)
    assert rc == _lib.E_INVAL and "workspace must be 16-byte aligned" in said
    assert lib.dskv_quant_attn_workspace(0, 2, 2, 32, 8, 128, 2) == 0 == lib.dskv_quant_attn_workspace(1, 2, 2, 32, 8, 80, 2)
    assert lib.dskv_quant_attn_counters(8) == 1024 and lib.dskv_quant_attn_counters(1000) == 2000 and lib.dskv_quant_attn_counters(0) == 0
    assert lib.dskv_quant_attn(None, 16, 16, 4096, 16, None) == _lib.E_INVAL


def test_workspaces_of_all_forms():
    """Every pair of heads, rows and type has a form and asks for a workspace; head dims without a matrix form ask for none."""
    lib = _lib.lib()
    for dtype in (_lib.F32, _lib.F16, _lib.BF16):
        for hkv, group in itertools.product((1, 2, 8, 600), (1, 2, 4, 7, 16, 17, 31, 32, 33, 48, 64, 65, 71, 128, 130)):
            for rows in (1, 2, 5, 8, 9, 16, 17, 64, 128, 2000):
                for dim in (64, 128):
                    assert lib.dskv_quant_attn_workspace(8, 8 * rows, rows, hkv * group, hkv, dim, dtype) > 0
                assert lib.dskv_quant_attn_workspace(8, 8 * rows, rows, hkv * group, hkv, 80, dtype) == 0


def test_workspaces_for_any_number_of_rows():
    """max_qo_len as large as its type goes, with every group: an answer, and not the end of the process."""
    code = ("from deserve_amd import _lib\n"
            "for rows in (1 << 24, 1 << 28, 1 << 29, 1 << 30, (1 << 31) - 1):\n"
            "    for group in (1, 4, 16, 32, 64, 128, 256, 512, 1024, 1 << 16):\n"
            "        for dtype in (_lib.F32, _lib.F16, _lib.BF16):\n"
            "            for dim in (64, 128):\n"
            "                assert _lib.lib().dskv_quant_attn_workspace(3, 9, rows, group, 1, dim, dtype) > 0, (rows, group, dtype, dim)\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
