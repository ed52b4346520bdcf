"""What the paged-cache and cross-attention entry points refuse, before any
device is touched: the torch wrappers by shape, type and layout, the C ABI by
null pointers, alignment, strides and sizes."""

import ctypes as C

import pytest
import torch

from waveforcing_b200 import _lib as L
from waveforcing_b200 import kernels as K

bf, i32 = torch.bfloat16, torch.int32


def _passes(fn, *a, **kw):
    with pytest.raises(RuntimeError, match="CUDA"):
        fn(*a, **kw)


def _rejects(fn, *a, **kw):
    with pytest.raises(ValueError):
        fn(*a, **kw)


def pages(dtype=torch.uint8, n=3, heads=2, ps=16):
    return K.KVPages.empty(n, heads, ps, dtype, "cpu")


def plan(B=2, width=2):
    return torch.zeros(B, width, dtype=i32), torch.zeros(B + 1, dtype=i32), torch.zeros(B, dtype=i32)


def test_pages():
    k = torch.zeros(3, 2, 16, 128, dtype=torch.uint8)
    s = torch.zeros(3, 2, 16)
    K.KVPages(k, k, s, s)
    for bad in [(k, k), (k, k, s, None), (k, k, s.double(), s), (k, k, s, s[:2]), (k, k.to(torch.int8), s, s),
                (k[..., :64].float(), k, s, s), (k.to(bf), k.to(bf), s, s), (k, k[:2], s, s),
                (k.transpose(2, 3), k.transpose(2, 3), s, s), (k.half(), k.half())]:
        _rejects(K.KVPages, *bad)


def test_write():
    p, (table, cu, lens) = pages(), plan()
    x = torch.zeros(5, 2, 128, dtype=bf)
    _passes(K.paged_kv_write, p, x, x, table, cu, lens)
    _rejects(K.paged_kv_write, p, x, x[:4], table, cu, lens)
    _rejects(K.paged_kv_write, p, x.float(), x.float(), table, cu, lens)
    _rejects(K.paged_kv_write, p, torch.zeros(5, 3, 128, dtype=bf), torch.zeros(5, 3, 128, dtype=bf), table, cu, lens)
    _rejects(K.paged_kv_write, p, torch.zeros(5, 2, 64, dtype=bf), torch.zeros(5, 2, 64, dtype=bf), table, cu, lens)
    _rejects(K.paged_kv_write, p, x, x, table.long(), cu, lens)
    _rejects(K.paged_kv_write, p, x, x, table, cu[:-1], lens)
    _rejects(K.paged_kv_write, p, x, x, table[:1], cu, lens)
    _rejects(K.paged_kv_write, p, x, x, table.t().contiguous().t(), cu, lens)
    _rejects(K.paged_kv_write, p, x, x, table, torch.zeros(6, dtype=i32)[::2], lens)
    _rejects(K.paged_kv_write, p, x.clone().requires_grad_(), x, table, cu, lens)


def test_read():
    p, (table, cu, lens) = pages(), plan()
    out = torch.zeros(5, 2, 128, dtype=bf)
    _passes(K.paged_kv_read, p, table, cu, lens, rows=5)
    _passes(K.paged_kv_read, p, table, cu, lens, out_k=out, out_v=out.clone())
    _rejects(K.paged_kv_read, p, table, cu, lens)
    _rejects(K.paged_kv_read, p, table, cu, lens, out_k=out)
    _rejects(K.paged_kv_read, p, table, cu, lens, rows=4, out_k=out, out_v=out)
    _rejects(K.paged_kv_read, p, table, cu, lens, out_k=out.float(), out_v=out.float())


def test_attention():
    p, (table, cu, lens) = pages(), plan()
    q = torch.zeros(5, 4, 128, dtype=bf)
    _passes(K.paged_attention, q, p, table, cu, lens)
    _passes(K.paged_attention, q, p, table, cu, lens, block=1, window=3, sink=1, out=torch.empty_like(q))
    _rejects(K.paged_attention, torch.zeros(5, 3, 128, dtype=bf), p, table, cu, lens)  # 3 heads over 2
    _rejects(K.paged_attention, q.half(), p, table, cu, lens)
    _rejects(K.paged_attention, q[None], p, table, cu, lens)
    _rejects(K.paged_attention, q, p, table, cu, lens, out=torch.empty(4, 4, 128, dtype=bf))
    _rejects(K.paged_attention, q, p, table, cu, lens.float())
    _rejects(K.paged_attention, q.clone().requires_grad_(), p, table, cu, lens)
    with torch.no_grad():
        _passes(K.paged_attention, q.clone().requires_grad_(), p, table, cu, lens)


def test_attention_ranges():
    """Beyond 32 bits ctypes would pass on what is left of a number."""
    p, (table, cu, lens) = pages(), plan()
    q = torch.zeros(5, 4, 128, dtype=bf)
    _passes(K.paged_attention, q, p, table, cu, lens, block=2**31 - 1, window=2**31 - 1, sink=2**31 - 1)
    for bad in [dict(block=2**32 + 1), dict(window=2**32 + 5), dict(window=3, sink=2**32), dict(block=-1), dict(window=-(2**32) + 1)]:
        _rejects(K.paged_attention, q, p, table, cu, lens, **bad)


def test_cross_attention():
    q, k = torch.zeros(2, 5, 4, 128, dtype=bf), torch.zeros(2, 7, 2, 128, dtype=bf)
    idx = torch.zeros(2, dtype=i32)
    mask = torch.ones(2, 7, dtype=torch.bool)
    _passes(K.cross_attention, q, k, k)
    _passes(K.cross_attention, q, k[:1], k[:1])
    _passes(K.cross_attention, q, k, k, kv_lens=idx, key_mask=mask, kv_index=idx)
    three = torch.zeros(3, 7, 2, 128, dtype=bf)
    _passes(K.cross_attention, q, three, three, kv_index=idx)
    _rejects(K.cross_attention, q, three, three)
    _rejects(K.cross_attention, q, k, k[:, :6])
    _rejects(K.cross_attention, q, torch.zeros(2, 7, 3, 128, dtype=bf), torch.zeros(2, 7, 3, 128, dtype=bf))
    _rejects(K.cross_attention, q, torch.zeros(2, 0, 2, 128, dtype=bf), torch.zeros(2, 0, 2, 128, dtype=bf))
    _rejects(K.cross_attention, q, k, k, kv_lens=idx.long())
    _rejects(K.cross_attention, q, k, k, kv_index=idx[:1])
    _rejects(K.cross_attention, q, k, k, key_mask=mask[:, :6])
    _rejects(K.cross_attention, q, k, k, key_mask=mask.to(torch.uint8))
    _rejects(K.cross_attention, q.float(), k, k)
    _rejects(K.cross_attention, q, k, k, out=torch.empty(2, 5, 4, 128))
    _rejects(K.cross_attention, q, k.clone().requires_grad_(), k)


def desc(**kw):
    d = dict(k=256, v=256, k_scale=256, v_scale=256, n_pages=4, page_size=16, heads=2, head_dim=128,
             dtype=L.WF_DTYPE_E4M3, k_stride=(4096, 2048, 128), v_stride=(4096, 2048, 128), k_scale_stride=(32, 16),
             v_scale_stride=(32, 16))
    d.update(kw)
    return C.byref(L.KvPagesDesc(**d))


def batch(**kw):
    d = dict(table=256, table_stride=4, cu=256, lens=256, seqs=2, max_pages=4, rows=8)
    d.update(kw)
    return C.byref(L.KvBatchDesc(**d))


BAD_PAGES = [(dict(k=None), 1), (dict(v=264), 1), (dict(head_dim=64), 2), (dict(dtype=9), 2), (dict(n_pages=0), 1),
             (dict(page_size=0), 1), (dict(heads=0), 1), (dict(k_stride=(4096, 2048, 120)), 1),
             (dict(v_stride=(4096, 0, 128)), 1), (dict(k_scale=None), 1), (dict(dtype=L.WF_DTYPE_BF16), 1),
             (dict(v_scale_stride=(32, -1)), 1), (dict(n_pages=1 << 40), 1)]
BAD_BATCH = [(dict(seqs=-1), 1), (dict(seqs=1 << 30), 1), (dict(max_pages=0), 1), (dict(rows=-1), 1),
             (dict(rows=1 << 40), 1), (dict(max_pages=1 << 30), 1), (dict(table=None), 1), (dict(cu=None), 1),
             (dict(lens=None), 1), (dict(table_stride=-1), 1)]


def calls(p, b):
    lib = L.lib()
    s = L.i64_array((256, 128))
    return [lambda: lib.wf_paged_kv_write(p, b, 256, 256, s, s, None),
            lambda: lib.wf_paged_kv_read(p, b, 256, 256, s, s, None),
            lambda: lib.wf_paged_attn(p, b, 256, s, 256, s, None, 4, 0, 0, 0, 8, 64, 0.1, None, 0, None)]


@pytest.mark.parametrize("change,code", BAD_PAGES, ids=str)
def test_abi_refuses_bad_pages(change, code):
    for call in calls(desc(**change), batch()):
        assert call() == code and L.last_error()
    assert L.lib().wf_paged_attn_workspace(desc(**change), batch(), 4, 0, 0, 8, 64) == -1


@pytest.mark.parametrize("change,code", BAD_BATCH, ids=str)
def test_abi_refuses_bad_batches(change, code):
    for call in calls(desc(), batch(**change)):
        assert call() == code and L.last_error()


def test_abi_empty_calls_launch_nothing():
    for change in (dict(rows=0), dict(seqs=0)):
        for call in calls(desc(), batch(**change)):
            assert call() == L.WF_OK


@pytest.mark.parametrize("args", [
    dict(q=None), dict(o=264), dict(H=3), dict(H=0), dict(H=2 * 129), dict(block=-1), dict(window=-1), dict(sink=-2),
    dict(sink=4), dict(max_new=-1), dict(max_len=-1), dict(scale=0.0), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(qs=(100, 128)), dict(os=(0, 128)),
], ids=str)
def test_abi_attention_refusals(args):
    a = dict(q=256, o=256, H=4, block=0, window=0, sink=0, max_new=8, max_len=64, scale=0.1, qs=(512, 128),
             os=(512, 128))
    a.update(args)
    rc = L.lib().wf_paged_attn(desc(), batch(), a["q"], L.i64_array(a["qs"]), a["o"], L.i64_array(a["os"]), None, a["H"],
                               a["block"], a["window"], a["sink"], a["max_new"], a["max_len"], a["scale"], None, 0, None)
    assert rc == L.WF_ERR_INVALID_ARG and L.last_error()


@pytest.mark.parametrize("at,short", [(None, 0), (264, 0), (256, 1)], ids=["none", "not aligned", "too small"])
def test_abi_attention_workspace(at, short):
    """A call whose keys are split needs the workspace that it asked for."""
    b = batch(seqs=1, rows=1, max_pages=4096)
    need = L.lib().wf_paged_attn_workspace(desc(), b, 4, 0, 0, 1, 60000)
    assert need > 0
    rc = L.lib().wf_paged_attn(desc(), b, 256, L.i64_array((512, 128)), 256, L.i64_array((512, 128)), None, 4, 0, 0, 0, 1,
                               60000, 0.1, at, need - short, None)
    assert rc == L.WF_ERR_INVALID_ARG and "workspace" in L.last_error()


@pytest.mark.parametrize("args,code", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=264), 1), (dict(o=None), 1), (dict(D=64), 2), (dict(H=5), 1),
    (dict(kv=0), 1), (dict(states=3), 1), (dict(states=0), 1), (dict(Lk=0), 1), (dict(batch=-1), 1),
    (dict(batch=70000), 1), (dict(batch=60000, Lq=60000, states=60000), 1), (dict(qs=(4, 512, 128)), 1),
    (dict(ks=(0, 256, 128)), 1), (dict(mask=256, ms=-1), 1), (dict(scale=-1.0), 1),
], ids=str)
def test_abi_cross_attention_refusals(args, code):
    a = dict(q=256, k=256, v=256, o=256, batch=2, Lq=3, states=2, Lk=7, H=4, kv=2, D=128, qs=(1536, 512, 128),
             ks=(1792, 256, 128), mask=None, ms=7, scale=0.1)
    a.update(args)
    i3 = L.i64_array
    rc = L.lib().wf_cross_attn(a["q"], a["k"], a["v"], a["o"], None, a["batch"], a["Lq"], a["states"], a["Lk"], a["H"],
                               a["kv"], a["D"], i3(a["qs"]), i3(a["ks"]), i3(a["ks"]), i3(a["qs"]), None, None,
                               a["mask"], a["ms"], a["scale"], None, 0, None)
    assert rc == code and L.last_error()


def test_descriptors_match_the_header():
    """The packed bytes and the ctypes structures have the layout a C compiler gives the header's."""
    import os
    import subprocess
    import tempfile

    src = '#include "wfk.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(){printf("%zu %zu %zu %zu",' \
          'sizeof(wf_kv_pages),sizeof(wf_kv_batch),offsetof(wf_kv_pages,k_stride),offsetof(wf_kv_batch,rows));}'
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "a.c"), "w").write(src)
        subprocess.run(["gcc", "-I" + os.path.dirname(L.HEADER_PATH), os.path.join(d, "a.c"), "-o",
                        os.path.join(d, "a")], check=True)
        got = subprocess.run([os.path.join(d, "a")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got[:2]] == [len(K._PACK_PAGES(*range(19))), len(K._PACK_BATCH(*range(7)))]
    for pack, desc, n in ((K._PACK_PAGES, L.KvPagesDesc, 19), (K._PACK_BATCH, L.KvBatchDesc, 7)):
        d = desc.from_buffer_copy(pack(*range(1, n + 1)))
        flat = []
        for name, _ in desc._fields_:
            x = getattr(d, name)
            flat += list(x) if hasattr(x, "__len__") else [x]
        assert flat == list(range(1, n + 1))
    assert [int(x) for x in got] == [C.sizeof(L.KvPagesDesc), C.sizeof(L.KvBatchDesc), L.KvPagesDesc.k_stride.offset,
                                     L.KvBatchDesc.rows.offset]
